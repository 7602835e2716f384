// A few tokens times NVFP4 weights on the tensor cores, sm_100a:
// y = x . Wᵀ, the SiLU-gated pair silu(x . W1ᵀ) * (x . W2ᵀ), and both with the
// weights of each token's chosen experts.  x is fp16, bf16 or fp32 and loses
// nothing that an fp32 sum keeps; sums are fp32.
//
// Mathematics.  The block-scaled MMA (tcgen05.mma kind::mxf4nvf4) multiplies
// e2m1 by e2m1, so x is written as a sum of kGemvTerms = 8 e2m1 digits in base 8.  For
// 16 consecutive elements with largest magnitude a, let s be the smallest
// power of two with a <= 4.5 s.  Then
//   t_1 = x / s,   q_j = e2m1(t_j) (nearest),   t_(j+1) = 8 (t_j - q_j),
//   x = s (q_1 + q_2 / 8 + ... + q_8 / 8^7) + error,   |error| <= s / 2 / 8^7 < 2^-23 a.
// It converges because below 5 the e2m1 values are at most 1 apart: |t_j| <= 4.5
// gives |t_j - q_j| <= 1/2 and |t_(j+1)| <= 4.  Every step is exact in fp32, s
// is an e4m3 scale (of all eight digits, 2^-6 <= s <= 2^8 after x is multiplied by a power
// of two 2^e chosen for the token and K range), and the MMA's products are exact.  The digits
// are eight rows of the MMA's B operand, the weights are its A operand (128
// rows), read by the tensor core as they are stored:
//   D[row][8 token + j] = sum over k of W[row][k] s q_(j+1),
//   y[token][row] = 2^-e (D_0 + (D_1 + (D_2 + ...) / 8) / 8).
// Nothing touches the weights between HBM and the tensor core, so a token
// costs no instructions per weight, and 16 tokens (N = 128) stay within the
// time that the weights take to arrive.  (The same products with mma.m16n8k16 and
// the weights converted to fp16 in registers, 560 instructions for each 8192 weights, were bound
// by instruction issue: 18.2 us for one token of 16384 x 7168, 59 us for 16 of 7168 x 16384.)
//
// An infinite or NaN element makes its 16 elements' scale NaN, and with it
// every output of that token.
//
// Two kernels.  gemv_expand_kernel writes the digits and scales as images of the
// shared memory that the MMAs read.  gemv_kernel streams the weights.  It may
// start loading them before the expansion is done: the expansion lets
// it start only after its own wait for all earlier work in the stream.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cstdint>
#include "kernel_common.cuh"
#include "ptx.cuh"
#include "quantize.cuh"

namespace nvfp4 {

constexpr int kDtF32 = 0, kDtF16 = 1, kDtBF16 = 2;

constexpr int kGemvTerms = 8;            // e2m1 digits of an element
constexpr int kGemvTokens = 16;          // tokens of a group: 128 columns of the MMA
constexpr int kGemvTokenBytes = kGemvTerms * kBK / 2;   // digits of one token, one 256-deep K block
constexpr int kGemvXSfBytes = kSfStageBytes;             // and the scale atoms of a group's K block
constexpr int kGemvMaxPairs = 256;       // rows of an expert call
constexpr int kGemvMaxExperts = 1024;
constexpr int kGemvMaxSplits = 8;

// One expert's weights as the kernel finds them in device memory.
struct alignas(64) GemvExpert {
  CUtensorMap map;                       // as GemvParams::map1
  const uint8_t* sf;
};

// Groups of an expert call, written by the expansion: an expert and up to 16 of its rows.
struct GemvGroups {
  int count;
  int expert[kGemvMaxPairs];
  int rows[kGemvMaxPairs];
  int before[kGemvMaxPairs];             // rows in the groups before
  int pair[kGemvMaxPairs];               // [before + i]: row of x's pairs
};

struct GemvParams {
  CUtensorMap map1, map2;                // weights [l][n][k/2] bytes, box {128 B, 128 rows, 1}
  const uint8_t *sf1, *sf2;              // scale atoms; map2 / sf2: gated only
  const void* x;                         // [l][m][k], rows ldx elements apart
  int64_t ldx, x_batch;
  void* out;                             // [l][m][n], rows ldo elements apart
  int64_t ldo, out_batch;
  int m, n, k, l;
  int x_dtype, out_dtype;
  int x_vec;                             // every 8 elements of x are 16-byte aligned
  int k_blocks, row_blocks;              // 256-deep K blocks, 128-row blocks
  int passes;                            // groups of 16 tokens of a batch entry
  int splits;                            // CTAs of a cluster, each with a part of K
  int group_rows;                        // tokens of the largest group
  int w_slots, x_slots;                  // shared-memory ring slots
  // expansion
  float* back;                           // [group][16][splits]: 2^-e
  uint8_t* image;                        // [k_block][group]: digits, scale atoms
  // experts
  const int* ids;                        // [pairs]
  int pairs, topk, experts;
  int x_per_pair;                        // x has a row for each pair, not for each token
  const GemvExpert *table1, *table2;
  GemvGroups* groups;
  unsigned* status;
  long long wait_limit;
};

// 2^e as fp32, -126 <= e <= 127.
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
  if (dtype == kDtF32) static_cast<float*>(out)[i] = v;
  else if (dtype == kDtF16) static_cast<__half*>(out)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// silu(g) * u = g / (1 + e^-g) * u in fp32 with the library's expf and an IEEE
// division: the output may be fp32 here, and there are few values.
__device__ __forceinline__ float silu_gate_f32(float g, float u) { return __fdiv_rn(g, 1.f + expf(-g)) * u; }

// Byte offset of (K block, group) in the images: the groups of a K block lie
// one behind the other, each with its rows' digits and its scale atoms.
__device__ __forceinline__ size_t gemv_image_at(int kb, int rows_all, int groups_all, int before, int group) {
  return (size_t)kb * ((size_t)rows_all * kGemvTokenBytes + (size_t)groups_all * kGemvXSfBytes) +
         (size_t)before * kGemvTokenBytes + (size_t)group * kGemvXSfBytes;
}

// ---------------------------------------------------------------------------
// Expansion
// ---------------------------------------------------------------------------
constexpr int kExpandThreads = 128;                       // a thread has 16 elements
constexpr int kExpandBlocks = kExpandThreads / 16;        // K blocks of a CTA

// Eight consecutive elements as fp32.
__device__ __forceinline__ void gemv_load8(const GemvParams& p, int64_t at, float (&f)[8]) {
  uint32_t v[8];
  if (p.x_dtype == kDtF32) {
    const uint32_t* q = static_cast<const uint32_t*>(p.x) + at;
    if (p.x_vec) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(q)), b = __ldg(reinterpret_cast<const uint4*>(q) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      #pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __ldg(q + i);
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i]);
    return;
  }
  const uint16_t* q = static_cast<const uint16_t*>(p.x) + at;
  if (p.x_vec) {
    const uint4 a = __ldg(reinterpret_cast<const uint4*>(q));
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (uint32_t)__ldg(q + 2 * i) | (uint32_t)__ldg(q + 2 * i + 1) << 16;
  }
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (p.x_dtype == kDtBF16) {
      f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
}

__device__ __forceinline__ void take_largest(uint32_t& top, float f) {   // of the finite magnitudes, as bits
  const uint32_t bits = __float_as_uint(f) & 0x7fffffffu;
  if (bits < 0x7f800000u && bits > top) top = bits;
}

// Pairs of one expert in ascending order, 16 at a time; one warp, the result in shared memory.
__device__ __forceinline__ void gemv_group_pairs(const GemvParams& p, GemvGroups& out, int* seen, int* open,
                                                 int* group_of, int* place_of) {
  const int lane = (int)(threadIdx.x & 31u);
  const uint32_t lt = (1u << lane) - 1u;
  for (int i = lane; i < p.experts; i += 32) seen[i] = 0;
  __syncwarp();
  int groups = 0;
  for (int i0 = 0; i0 < p.pairs; i0 += 32) {
    const int i = i0 + lane;
    const int id = i < p.pairs ? __ldg(p.ids + i) : -1;
    const bool valid = (unsigned)id < (unsigned)p.experts;
    const uint32_t same = __match_any_sync(0xffffffffu, valid ? id : -1);
    const int before = valid ? seen[id] : 0, at = before + __popc(same & lt);
    const int old = valid && before > 0 ? open[id] : 0;
    const bool first = valid && at % kGemvTokens == 0;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    int grp = groups + __popc(firsts & lt);
    const uint32_t mine = firsts & same & (lt | (1u << lane));   // the group's first row, if it is among these 32
    const int theirs = __shfl_sync(0xffffffffu, grp, mine ? 31 - __clz(mine) : lane);
    grp = mine ? theirs : old;
    if (first) out.expert[grp] = id, out.rows[grp] = 0;
    __syncwarp();
    if (valid) atomicAdd(&out.rows[grp], 1);
    if (valid && (same >> lane) == 1u) seen[id] = at + 1, open[id] = grp;   // the expert's last row among these
    if (i < p.pairs) group_of[i] = valid ? grp : -1, place_of[i] = at % kGemvTokens;
    groups += __popc(firsts);
    __syncwarp();
  }
  int sum = 0;                                            // exclusive sums of the groups' rows
  for (int g0 = 0; g0 < groups; g0 += 32) {
    const int rows = g0 + lane < groups ? out.rows[g0 + lane] : 0;
    int x = rows;
    #pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (g0 + lane < groups) out.before[g0 + lane] = sum + x - rows;
    sum += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) out.count = groups;
  __syncwarp();
  for (int i = lane; i < p.pairs; i += 32)
    if (group_of[i] >= 0) out.pair[out.before[group_of[i]] + place_of[i]] = i;
}

// grid: (row of x, chunk of 8 K blocks of a split).  A CTA takes the largest magnitude
// of its row in the whole split (every CTA of the split reads it: a few KB from L2),
// then each thread expands 16 elements.
template <bool kMoe>
__global__ void __launch_bounds__(kExpandThreads) gemv_expand_kernel(const __grid_constant__ GemvParams p) {
  __shared__ uint32_t s_top[kExpandThreads / 32];
  __shared__ GemvGroups s_groups;
  __shared__ int s_seen[kMoe ? kGemvMaxExperts : 1], s_open[kMoe ? kGemvMaxExperts : 1];
  __shared__ int s_group_of[kMoe ? kGemvMaxPairs : 1], s_place_of[kMoe ? kGemvMaxPairs : 1];
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();                            // after the wait: see the head of this file
  const int r = (int)blockIdx.x;
  int group, place, rows, before, rows_all, groups_all;
  int64_t src;
  if constexpr (kMoe) {
    if (warp == 0) gemv_group_pairs(p, s_groups, s_seen, s_open, s_group_of, s_place_of);
    __syncthreads();
    if (r == 0 && blockIdx.y == 0) {
      if (tid == 0) p.groups->count = s_groups.count;
      for (int i = tid; i < p.pairs; i += kExpandThreads) {
        p.groups->expert[i] = s_groups.expert[i], p.groups->rows[i] = s_groups.rows[i];
        p.groups->before[i] = s_groups.before[i], p.groups->pair[i] = s_groups.pair[i];
      }
    }
    group = s_group_of[r], place = s_place_of[r];
    if (group < 0) {                                      // not an expert: a row of zeros
      for (int c = (int)blockIdx.y * kExpandThreads + tid; c < p.n; c += (int)gridDim.y * kExpandThreads)
        store_out(p.out, p.out_dtype, (int64_t)r * p.ldo + c, 0.f);
      return;
    }
    rows = s_groups.rows[group], before = s_groups.before[group];
    rows_all = groups_all = p.pairs;
    src = (int64_t)(p.x_per_pair ? r : r / p.topk) * p.ldx;
  } else {
    const int batch = r / p.m, row = r % p.m, pass = row / kGemvTokens;
    place = row % kGemvTokens;
    group = batch * p.passes + pass;
    rows = min(kGemvTokens, p.m - pass * kGemvTokens);
    before = batch * p.m + pass * kGemvTokens;
    rows_all = p.l * p.m, groups_all = p.l * p.passes;
    src = (int64_t)batch * p.x_batch + (int64_t)row * p.ldx;
  }
  const int chunks = (int)gridDim.y / p.splits;
  const int split = (int)blockIdx.y / chunks, chunk = (int)blockIdx.y % chunks;
  const int kb0 = p.k_blocks * split / p.splits, kb1 = p.k_blocks * (split + 1) / p.splits;
  if (kb0 + chunk * kExpandBlocks >= kb1) return;

  // this thread's 16 elements, and the largest of the split
  const int kb = kb0 + chunk * kExpandBlocks + tid / 16, b = tid % 16;
  const int k0 = kb * kBK + b * 16;
  const bool mine = kb < kb1 && k0 < p.k;
  float v[16];
  uint32_t top = 0;
  {
    float lo[8], hi[8];
    #pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = hi[i] = 0.f;
    if (mine) gemv_load8(p, src + k0, lo), gemv_load8(p, src + k0 + 8, hi);
    #pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = lo[i], v[8 + i] = hi[i];
  }
  for (int c = kb0 * (kBK / 8) + tid; c < min(kb1 * kBK, p.k) / 8; c += kExpandThreads) {
    float f[8];
    gemv_load8(p, src + (int64_t)c * 8, f);
    #pragma unroll
    for (int i = 0; i < 8; ++i) take_largest(top, f[i]);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  #pragma unroll
  for (int i = 0; i < kExpandThreads / 32; ++i) top = max(top, s_top[i]);
  // the largest magnitude goes into [2^9, 2^10): scales reach 2^8 at most
  const int e = min(9 - ((int)(top >> 23) - 127), 126);
  if (chunk == 0 && tid == 0) p.back[((int64_t)group * kGemvTokens + place) * p.splits + split] = exp2_int(-e);

  const float up = exp2_int(e);
  uint32_t amax = 0;
  bool finite = true;
  #pragma unroll
  for (int i = 0; i < 16; ++i) {
    finite = finite && (__float_as_uint(v[i]) & 0x7fffffffu) < 0x7f800000u;
    v[i] *= up;
    take_largest(amax, v[i]);
  }
  // s = 2^q: the smallest with amax <= 4.5 s (1.125 * 2^(q + 2)), in [2^-6, 2^8]
  int q = (int)(amax >> 23) - 127 - ((amax & 0x7fffffu) <= 0x100000u ? 2 : 1);
  q = max(q, -6);
  const float down = exp2_int(-q);
  #pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = finite ? v[i] * down : 0.f;
  uint8_t* const image = p.image + gemv_image_at(kb, rows_all, groups_all, before, group);
  uint8_t* const digits = image + place * kGemvTokenBytes + (b & 1) * 8;
  #pragma unroll
  for (int j = 0; j < kGemvTerms; ++j) {
    uint32_t word[2] = {0u, 0u};
    #pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t two = e2m1x2(v[2 * i], v[2 * i + 1]);
      word[i / 4] |= two << (8 * (i % 4));
      uint32_t h;
      asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(two));
      const float2 d = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = (v[2 * i] - d.x) * 8.f;
      v[2 * i + 1] = (v[2 * i + 1] - d.y) * 8.f;
    }
    // row j of the token's 8 x 128 bytes, 16-byte pieces exchanged as the 128-byte swizzle has them
    if (mine) *reinterpret_cast<uint2*>(digits + j * 128 + (((b >> 1) ^ j) << 4)) = make_uint2(word[0], word[1]);
  }
  const uint32_t s8 = finite ? (uint32_t)(q + 7) << 3 : 0x7fu;   // e4m3 of 2^q, or NaN
  const uint32_t pair = s8 | (__shfl_down_sync(0xffffffffu, s8, 1) << 8);
  const uint32_t four = pair | (__shfl_down_sync(0xffffffffu, pair, 2) << 16);
  if (mine && b % 4 == 0) {
    uint8_t* const atom = image + rows * kGemvTokenBytes + (b / 4) * kSfAtom;
    #pragma unroll
    for (int j = 0; j < kGemvTerms; ++j) {
      const int row = place * kGemvTerms + j;
      *reinterpret_cast<uint32_t*>(atom + (row % 32) * 16 + (row / 32) * 4) = four;
    }
  }
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------
constexpr int kGemvWBytes = kBM * kBK / 2 + kSfStageBytes;   // a weight slot: 128 rows x 256, scale atoms
constexpr int kGemvMaxWSlots = 8, kGemvMaxXSlots = 4;
constexpr int kGemvThreads = 7 * 32;     // epilogue warps 0-3, weights 4, x 5, MMA and TMEM 6

// Copy one scale atom into TMEM: row i to lane i of each lane quadrant, 4 columns.
__device__ __forceinline__ void tc_cp_32x128b_x4(uint32_t taddr, uint64_t s_desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(s_desc) : "memory");
}

// What a cluster works on: tile t of the call.
struct GemvTile { int group, row_block, batch, rows, before, expert; };

template <bool kMoe>
__device__ __forceinline__ GemvTile gemv_tile(const GemvParams& p, int t) {
  GemvTile r;
  if constexpr (kMoe) {
    r.group = t / p.row_blocks, r.row_block = t % p.row_blocks, r.batch = 0;
    r.expert = __ldcg(&p.groups->expert[r.group]);
    r.rows = __ldcg(&p.groups->rows[r.group]), r.before = __ldcg(&p.groups->before[r.group]);
  } else {
    // groups of the same weights next to one another: they share them in L2
    const int pass = t % p.passes, rest = t / p.passes;
    r.row_block = rest % p.row_blocks, r.batch = rest / p.row_blocks;
    r.group = r.batch * p.passes + pass;
    r.rows = min(kGemvTokens, p.m - pass * kGemvTokens), r.before = r.batch * p.m + pass * kGemvTokens;
    r.expert = 0;
  }
  return r;
}

// A cluster of `splits` CTAs owns a 128-row block and a group; each CTA has a
// part of K.  Shared memory holds a ring of weight slots (one matrix' K block,
// 18 KB) and a ring of x slots; it is kept to half of the SM's, so that the next
// kernel's CTAs can be resident and start their loads while this one ends.  The sums of
// the CTAs of a cluster meet in distributed shared memory: each CTA owns 128 / splits rows,
// gets the others' sums for them and adds them in the order of the CTAs.
template <bool kDual, bool kMoe, int kTmemCols>
__global__ void __launch_bounds__(kGemvThreads) gemv_kernel(const __grid_constant__ GemvParams p) {
  constexpr int kMats = kDual ? 2 : 1;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_w_full[kGemvMaxWSlots], bar_w_free[kGemvMaxWSlots];
  __shared__ uint64_t bar_x_full[kGemvMaxXSlots], bar_x_free[kGemvMaxXSlots];
  __shared__ uint64_t bar_acc_full, bar_acc_free, bar_drain;
  __shared__ uint64_t bar_sums, bar_sums_free;            // this CTA's rows: all sums there; its sums taken everywhere
  __shared__ uint32_t s_tmem_base;
  __shared__ volatile int s_abort;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = (int)threadIdx.x >> 5;
  const int splits = p.splits;
  const int rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int cluster = (int)blockIdx.x / splits, clusters = (int)gridDim.x / splits;
  const int kb0 = p.k_blocks * rank / splits, kb1 = p.k_blocks * (rank + 1) / splits;
  // shared memory: weight slots, x slots, the cluster's sums
  const int x_bytes = p.group_rows * kGemvTokenBytes + kGemvXSfBytes;   // a multiple of 1024
  // odd numbers of tokens: 8 columns more, whose digits are whatever lies behind; they are not used
  const int n_pad = (p.group_rows * kGemvTerms + 15) / 16 * 16;
  const uint32_t w_base = smem_base, x_base = smem_base + p.w_slots * kGemvWBytes;
  const uint32_t sums_base = x_base + p.x_slots * x_bytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.w_slots; ++i) mbar_init(smem_u32(&bar_w_full[i]), 1), mbar_init(smem_u32(&bar_w_free[i]), 1);
    for (int i = 0; i < p.x_slots; ++i) mbar_init(smem_u32(&bar_x_full[i]), 1), mbar_init(smem_u32(&bar_x_free[i]), 1);
    mbar_init(smem_u32(&bar_acc_full), 1);
    mbar_init(smem_u32(&bar_acc_free), 4);
    mbar_init(smem_u32(&bar_drain), 1);
    mbar_init(smem_u32(&bar_sums), splits);
    mbar_init(smem_u32(&bar_sums_free), splits);
    s_abort = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 6) tmem_alloc<kTmemCols>(smem_u32(&s_tmem_base));
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync();                         // the others' barriers exist
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  const AbortCtl ctl{&s_abort, p.status, p.wait_limit};
  // experts: the groups come from the expansion
  if (kMoe) griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int tiles = kMoe ? __ldcg(&p.groups->count) * p.row_blocks : p.l * p.passes * p.row_blocks;
  const int atoms_all = p.k / kKStep;                     // 64-deep atoms of a 128-row block

  if (warp == 4) {
    // ------------------------------------------------------------ weights
    if (elect_one()) {
      const uint64_t pol = policy_evict_normal();
      int slot = 0;
      uint32_t phase = 0, issued = 0, last_phase = 0;
      bool ok = true;
      for (int t = cluster; t < tiles && ok; t += clusters) {
        const GemvTile tc = gemv_tile<kMoe>(p, t);
        const void *map[2] = {&p.map1, &p.map2};
        const uint8_t* sf[2] = {p.sf1, p.sf2};
        if constexpr (kMoe) {
          map[0] = &p.table1[tc.expert].map, sf[0] = p.table1[tc.expert].sf;
          if constexpr (kDual) map[1] = &p.table2[tc.expert].map, sf[1] = p.table2[tc.expert].sf;
        }
        const size_t atom0 = ((size_t)tc.batch * p.row_blocks + tc.row_block) * (size_t)atoms_all;
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          const int atoms = min(kBK / kKStep, atoms_all - kb * (kBK / kKStep));
          #pragma unroll
          for (int mat = 0; mat < kMats; ++mat) {
            if (!ctl.wait(smem_u32(&bar_w_free[slot]), phase ^ 1u, kDevTimeoutStageFree)) {
              ok = false;
              break;
            }
            const uint32_t dst = w_base + slot * kGemvWBytes, bar = smem_u32(&bar_w_full[slot]);
            mbar_arrive_expect_tx(bar, kBM * kBK / 2 + atoms * kSfAtom);
            tma_load_3d(dst, map[mat], bar, kb * (kBK / 2), tc.row_block * kBM, tc.batch, pol);
            bulk_load(dst + kBM * kBK / 2, sf[mat] + (atom0 + (size_t)kb * (kBK / kKStep)) * kSfAtom, atoms * kSfAtom,
                      bar, pol);
            issued |= 1u << slot;
            last_phase = (last_phase & ~(1u << slot)) | (phase << slot);
            if (++slot == p.w_slots) slot = 0, phase ^= 1u;
          }
        }
      }
      if (!ok)                                            // copies in flight land before the CTA winds down
        for (int s = 0; s < p.w_slots; ++s)
          if ((issued >> s) & 1u) ctl.drain_copies(smem_u32(&bar_w_full[s]), (last_phase >> s) & 1u);
    }
  } else if (warp == 5) {
    // ------------------------------------------------------------ x
    if (elect_one()) {
      griddep_wait();                                     // the expansion is done
      const uint64_t pol = policy_evict_normal();
      const int rows_all = kMoe ? p.pairs : p.l * p.m, groups_all = kMoe ? p.pairs : p.l * p.passes;
      int slot = 0;
      uint32_t phase = 0, issued = 0, last_phase = 0;
      bool ok = true;
      for (int t = cluster; t < tiles && ok; t += clusters) {
        const GemvTile tc = gemv_tile<kMoe>(p, t);
        const uint32_t bytes = tc.rows * kGemvTokenBytes + kGemvXSfBytes;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!ctl.wait(smem_u32(&bar_x_free[slot]), phase ^ 1u, kDevTimeoutStageFree)) {
            ok = false;
            break;
          }
          const uint32_t bar = smem_u32(&bar_x_full[slot]);
          mbar_arrive_expect_tx(bar, bytes);
          bulk_load(x_base + slot * x_bytes, p.image + gemv_image_at(kb, rows_all, groups_all, tc.before, tc.group),
                    bytes, bar, pol);
          issued |= 1u << slot;
          last_phase = (last_phase & ~(1u << slot)) | (phase << slot);
          if (++slot == p.x_slots) slot = 0, phase ^= 1u;
        }
      }
      if (!ok)
        for (int s = 0; s < p.x_slots; ++s)
          if ((issued >> s) & 1u) ctl.drain_copies(smem_u32(&bar_x_full[s]), (last_phase >> s) & 1u);
    }
  } else if (warp == 6) {
    // ------------------------------------------------------------ MMA
    if (elect_one()) {
      const uint64_t w_desc0 = kmajor_sw128_desc(w_base), x_desc0 = kmajor_sw128_desc(x_base);
      const uint64_t sf_desc0 = sf_atom_desc(w_base + kBM * kBK / 2), xsf_desc0 = sf_atom_desc(x_base);
      // accumulators, then each slot's scales: 16 columns for a weight slot, 16 for an x slot
      const uint32_t sf_col = tmem + kMats * n_pad, xsf_col = sf_col + 16 * p.w_slots;
      int ws = 0, xs = 0;
      uint32_t w_phase = 0, x_phase = 0, acc_phase = 0;
      bool ok = true, any = false;
      for (int t = cluster; t < tiles && ok; t += clusters) {
        const GemvTile tc = gemv_tile<kMoe>(p, t);
        const int n_cols = (tc.rows * kGemvTerms + 15) / 16 * 16;
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(n_cols >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
        if (!ctl.wait(smem_u32(&bar_acc_free), acc_phase ^ 1u, kDevTimeoutAccFree)) break;
        tc_fence_after();
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          const int atoms = min(kBK / kKStep, atoms_all - kb * (kBK / kKStep));
          if (!ctl.wait(smem_u32(&bar_x_full[xs]), x_phase, kDevTimeoutTmaFull)) {
            ok = false;
            break;
          }
          const uint64_t dx = desc_advance(x_desc0, xs * x_bytes);
          const uint64_t dxs = desc_advance(xsf_desc0, xs * x_bytes + tc.rows * kGemvTokenBytes);
          const uint32_t xsf = xsf_col + 16 * xs;
          #pragma unroll
          for (int mat = 0; mat < kMats; ++mat) {
            if (!ctl.wait(smem_u32(&bar_w_full[ws]), w_phase, kDevTimeoutTmaFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint64_t dw = desc_advance(w_desc0, ws * kGemvWBytes), dws = desc_advance(sf_desc0, ws * kGemvWBytes);
            const uint32_t sf = sf_col + 16 * ws;
            for (int j = 0; j < atoms; ++j) {
              if (mat == 0) tc_cp_32x128b_x4(xsf + 4 * j, desc_advance(dxs, j * kSfAtom));
              tc_cp_32x128b_x4(sf + 4 * j, desc_advance(dws, j * kSfAtom));
              tc_mma_nvf4(tmem + mat * n_pad, desc_advance(dw, 32 * j), desc_advance(dx, 32 * j), idesc, sf + 4 * j,
                          xsf + 4 * j, kb != kb0 || j != 0);
            }
            tc_commit(smem_u32(&bar_w_free[ws]));
            any = true;
            if (++ws == p.w_slots) ws = 0, w_phase ^= 1u;
          }
          if (!ok) break;
          tc_commit(smem_u32(&bar_x_free[xs]));
          if (++xs == p.x_slots) xs = 0, x_phase ^= 1u;
        }
        if (!ok) break;
        tc_commit(smem_u32(&bar_acc_full));
        acc_phase ^= 1u;
      }
      if (s_abort && any) {
        tc_commit(smem_u32(&bar_drain));
        ctl.drain(smem_u32(&bar_drain), 0);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    griddep_wait();                                       // the expansion's factors; and nothing is written before
    const int lane = (int)(threadIdx.x & 31u), row = warp * 32 + lane;
    const int own_rows = kBM / splits, owner = row / own_rows;   // the CTA that finishes this thread's row
    uint32_t phase = 0;
    for (int t = cluster; t < tiles; t += clusters) {
      const GemvTile tc = gemv_tile<kMoe>(p, t);
      if (!ctl.wait(smem_u32(&bar_acc_full), phase, kDevTimeoutAccFull)) break;
      tc_fence_after();
      if (splits > 1 && t != cluster &&
          !ctl.wait_cluster(smem_u32(&bar_sums_free), phase ^ 1u, kDevTimeoutAccFree)) break;
      const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16);
      // sums of a sender in an owner's shared memory: [sender][matrix][token][row of the owner]
      const uint32_t slice = sums_base + (uint32_t)((rank * kMats * tc.rows) * own_rows + row % own_rows) * 4u;
      const uint32_t remote = splits > 1 ? mapa_shared(slice, (uint32_t)owner) : 0u;
      auto out_at = [&](int tok) -> int64_t {              // where the token's row of this tile starts
        const int64_t at = kMoe ? (int64_t)__ldcg(&p.groups->pair[tc.before + tok]) * p.ldo
                                : (int64_t)tc.batch * p.out_batch + (int64_t)(tc.before - tc.batch * p.m + tok) * p.ldo;
        return at + (int64_t)tc.row_block * kBM;
      };
      for (int t0 = 0; t0 < tc.rows; t0 += 2) {
        uint32_t d[kMats][16];
        #pragma unroll
        for (int mat = 0; mat < kMats; ++mat) tmem_ld_32x32b_x16(acc + mat * n_pad + t0 * kGemvTerms, d[mat]);
        tmem_ld_wait();
        #pragma unroll
        for (int mat = 0; mat < kMats; ++mat) tmem_regs_ready16(d[mat]);
        #pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int tok = t0 + i;
          if (tok >= tc.rows) break;
          const float back = __ldcg(p.back + ((int64_t)tc.group * kGemvTokens + tok) * splits + rank);
          float v[kMats];
          #pragma unroll
          for (int mat = 0; mat < kMats; ++mat) {
            v[mat] = __uint_as_float(d[mat][8 * i + 7]);
            #pragma unroll
            for (int j = 6; j >= 0; --j) v[mat] = fmaf(v[mat], 0.125f, __uint_as_float(d[mat][8 * i + j]));
            v[mat] *= back;
          }
          if (splits > 1) {
            #pragma unroll
            for (int mat = 0; mat < kMats; ++mat)
              st_shared_cluster_f32(remote + (uint32_t)((mat * tc.rows + tok) * own_rows) * 4u, v[mat]);
          } else if (tc.row_block * kBM + row < p.n) {
            store_out(p.out, p.out_dtype, out_at(tok) + row, kDual ? silu_gate_f32(v[0], v[kMats - 1]) : v[0]);
          }
        }
      }
      // the accumulators may be overwritten
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_acc_free));
      if (splits > 1) {
        named_bar_sync(1, 128);
        if ((int)threadIdx.x < splits) mbar_arrive_cluster(mapa_shared(smem_u32(&bar_sums), threadIdx.x));
        if (!ctl.wait_cluster(smem_u32(&bar_sums), phase, kDevTimeoutAccFull)) break;
        for (int i = (int)threadIdx.x; i < own_rows * tc.rows; i += 128) {
          const int r = i % own_rows, tok = i / own_rows;
          float v[kMats];
          #pragma unroll
          for (int mat = 0; mat < kMats; ++mat) {
            v[mat] = 0.f;
            for (int s = 0; s < splits; ++s)
              v[mat] += __uint_as_float(lds_u32(sums_base + (uint32_t)(((s * kMats + mat) * tc.rows + tok) * own_rows + r) * 4u));
          }
          const int at = rank * own_rows + r;
          if (tc.row_block * kBM + at < p.n)
            store_out(p.out, p.out_dtype, out_at(tok) + at, kDual ? silu_gate_f32(v[0], v[kMats - 1]) : v[0]);
        }
        named_bar_sync(1, 128);                           // all of this CTA's rows are read
        if ((int)threadIdx.x < splits) mbar_arrive_cluster(mapa_shared(smem_u32(&bar_sums_free), threadIdx.x));
      }
      phase ^= 1u;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync();                         // nobody writes to a CTA that is gone
  tc_fence_after();
  if (warp == 6) tmem_dealloc<kTmemCols>(tmem);
}

}  // namespace nvfp4
