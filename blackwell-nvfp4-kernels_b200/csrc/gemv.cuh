// A few tokens times NVFP4 weights on the tensor cores, sm_100a:
// y = x . Wᵀ, the SiLU-gated pair silu(x . W1ᵀ) * (x . W2ᵀ), and both with the
// weights of each token's chosen experts.  x is fp16, bf16 or fp32, held to 24 bits under the
// largest of 16 neighbours; sums are fp32.
//
// Mathematics.  The block-scaled MMA (tcgen05.mma kind::mxf4nvf4) multiplies
// e2m1 by e2m1, so x is written as eight balanced base-8 digits.  For 16
// consecutive elements with largest magnitude a, let s be the smallest power of two
// with a <= 1.5 s.  Then
//   x = s (q_1 + q_2 / 8 + ... + q_8 / 8^7) + error,   q_j in {-2, -1.5, ..., 1.5},
// where the q_j are the digits (in halves) of the integer nearest to 2 * 8^7 x / s:
// they are e2m1 values, and |error| <= s / 4 / 8^7 = 2^-23 s < 2^-22 a.  s is an
// e4m3 scale (of all eight digits; 2^-6 <= s <= 2^8 after x is multiplied by a
// power of two 2^e chosen for the token and K range), and the MMA's products are exact.
// So x is a fixed-point number under its block's largest, and under 2^-14 of the K range's largest: the error
// is below 2^-22 of the one or 2^-36 of the other.  Against 64 bits a result with weights everywhere is off by
// as much as an fp32 sum or less.  But where a block's largest element meets a zero code, what its neighbours lose to it
// is not hidden by its product: one element of 1e4 among 7168 normal ones makes the rows whose weight there is
// zero off by 1.3e-5 (bf16) to 2.6e-5 (fp32) relative, an fp32 sum's by about 1e-6 or less.  (Eight digits are all that N = 128 columns have room for
// with 16 tokens.)
// The digits are eight rows of the MMA's B operand, the weights are its A
// operand (128 rows), read by the tensor core as they are stored:
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
// With few tokens gemv_kernel expands x itself, eight warps of each CTA for its
// part of K, while the first weights are on their way.  With more that would
// be the slowest part (about 300 warp instructions for a token's 256
// elements), and gemv_expand_kernel does it once, as images of the shared memory that the MMAs
// read; gemv_kernel may then load weights before the expansion is done, because the expansion lets
// it start only after its own wait for all earlier work in the stream.
#pragma once
#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_bf16.h>
#include <cstdint>
#include <type_traits>
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

// Groups of an expert call: an expert and up to 16 of its rows.  Both kernels make
// them for themselves from the ids.
struct GemvGroups {
  int count;
  int rows[kGemvMaxPairs];
  uint16_t expert[kGemvMaxPairs];
  uint16_t before[kGemvMaxPairs];        // rows in the groups before
  uint16_t pair[kGemvMaxPairs];          // [before + i]: row of x's pairs
};
struct GemvGroupScratch {
  uint16_t seen[kGemvMaxExperts], open[kGemvMaxExperts];        // an expert's rows so far, its last group
  int16_t group_of[kGemvMaxPairs], place_of[kGemvMaxPairs];
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
  int splits, split_bits;                // CTAs of a cluster, each with a part of K; splits = 1 << split_bits
  int room, group_rows;                  // tokens that a group can have, and the largest has
  int w_slots, x_slots, acc_bufs;        // shared-memory ring slots, accumulators
  // expansion
  float* back;                           // [group][16][splits]: 2^-e
  uint8_t* image;                        // [k_block][group]: digits, scale atoms
  // experts
  const int* ids;                        // [pairs]
  int pairs, topk, experts;
  int x_per_pair;                        // x has a row for each pair, not for each token
  const GemvExpert *table1, *table2;
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
constexpr int kExpandThreads = 256;                       // a warp has a K block, a thread 8 elements
constexpr int kExpandBlocks = kExpandThreads / 32;        // K blocks of a CTA

// Eight consecutive elements as they lie in memory (b: fp32 only).  kVec: 16-byte aligned.
struct Raw8 { uint4 a, b; };
// From L2, and not by the path of read-only data (ld.global.nc): a kernel of this file starts while the one before
// it may still write x and the ids.  Volatile: the load stays in front of a signal that follows it.
__device__ __forceinline__ uint4 ldcg_v4(const void* q) {
  uint4 v;
  asm volatile("ld.global.cg.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(q));
  return v;
}
template <bool kWide, bool kVec>
__device__ __forceinline__ Raw8 gemv_raw8(const void* x, int64_t at) {
  Raw8 r;
  r.b = make_uint4(0, 0, 0, 0);
  if constexpr (kWide) {
    const uint32_t* q = static_cast<const uint32_t*>(x) + at;
    if constexpr (kVec) {
      r.a = ldcg_v4(q), r.b = ldcg_v4(q + 4);
    } else {
      r.a = make_uint4(__ldcg(q), __ldcg(q + 1), __ldcg(q + 2), __ldcg(q + 3));
      r.b = make_uint4(__ldcg(q + 4), __ldcg(q + 5), __ldcg(q + 6), __ldcg(q + 7));
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(x) + at;
    if constexpr (kVec) {
      r.a = ldcg_v4(q);
    } else {
      uint32_t v[4];
      #pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (uint32_t)__ldcg(q + 2 * i) | (uint32_t)__ldcg(q + 2 * i + 1) << 16;
      r.a = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
  return r;
}

// As fp32.
__device__ __forceinline__ void widen8(const Raw8& r, int dtype, float (&f)[8]) {
  const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
  if (dtype == kDtF32) {
    #pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
  } else if (dtype == kDtBF16) {
    #pragma unroll
    for (int i = 0; i < 4; ++i)
      f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  } else {
    #pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x, f[2 * i + 1] = t.y;
    }
  }
}

// Calls f with the loader of x's type and alignment: the choice is made once, outside
// of the loops, so that their loads can be in flight together.
template <class F>
__device__ __forceinline__ void gemv_with_loader(const GemvParams& p, F f) {
  const void* x = p.x;
  if (p.x_dtype == kDtF32) {
    if (p.x_vec) f([x](int64_t at) { return gemv_raw8<true, true>(x, at); });
    else f([x](int64_t at) { return gemv_raw8<true, false>(x, at); });
  } else {
    if (p.x_vec) f([x](int64_t at) { return gemv_raw8<false, true>(x, at); });
    else f([x](int64_t at) { return gemv_raw8<false, false>(x, at); });
  }
}

// Largest finite magnitude (bits) of eight elements.
__device__ __forceinline__ uint32_t largest8(const Raw8& r, int dtype) {
  float f[8];
  widen8(r, dtype, f);
  uint32_t top = 0;
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = __float_as_uint(f[i]) & 0x7fffffffu;
    top = max(top, bits < 0x7f800000u ? bits : 0u);
  }
  return top;
}

// The exponent that takes a largest magnitude (bits) into [2^7, 2^8): scales
// reach 2^8 at most; as far as it and its inverse are normal numbers.
__device__ __forceinline__ int gemv_exponent(uint32_t top) { return min(7 - ((int)(top >> 23) - 127), 126); }

// Transposes 8 words of 8 nibbles: word c's nibble r becomes word r's nibble c.
__device__ __forceinline__ void transpose_nibbles(uint32_t* w) {
  #pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint32_t a = w[r], b = w[r + 4];
    w[r] = __byte_perm(a, b, 0x5410), w[r + 4] = __byte_perm(a, b, 0x7632);
  }
  #pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i < 2 ? i : i + 2;
    const uint32_t a = w[r], b = w[r + 2];
    w[r] = __byte_perm(a, b, 0x6240), w[r + 2] = __byte_perm(a, b, 0x7351);
  }
  #pragma unroll
  for (int r = 0; r < 8; r += 2) {
    const uint32_t a = w[r], b = w[r + 1];
    w[r] = (a & 0x0f0f0f0fu) | ((b & 0x0f0f0f0fu) << 4);
    w[r + 1] = ((a >> 4) & 0x0f0f0f0fu) | (b & 0xf0f0f0f0u);
  }
}

// Digits of a warp's 256 elements, eight in each lane (two lanes a block of
// 16): store(j, eight codes) for j = 0..7; returns the four scale bytes of 64 elements,
// valid in lanes 0, 8, 16 and 24.  `up`: 2^e.
template <class Store>
__device__ __forceinline__ uint32_t gemv_digits(float (&v)[8], float up, Store store) {
  uint32_t amax = 0;
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] *= up;
    amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
  }
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const bool finite = amax < 0x7f800000u;
  // s = 2^q: the smallest with amax <= 1.5 s, in [2^-6, 2^8]
  const int q = max((int)(amax >> 23) - 127 + ((amax & 0x7fffffu) > 0x400000u ? 1 : 0), -6);
  const float units = finite ? exp2_int(22 - q) : 0.f;    // of s / 2 / 8^7
  uint32_t w[8];
  #pragma unroll
  for (int i = 0; i < 8; ++i) {
    // balanced base-8 digits: 4 added to each makes them the 3-bit fields of one number
    const uint32_t y = (uint32_t)(__float2int_rn(finite ? v[i] * units : 0.f) + 0x924924);
    uint32_t x = (y & 0xfffu) | ((y & 0xfff000u) << 4);
    x = (x & 0x003f003fu) | ((x & 0x0fc00fc0u) << 2);
    x = (x & 0x07070707u) | ((x & 0x38383838u) << 1);     // fields f in nibbles
    // code of (f - 4) / 2: f - 4 for f >= 4, else sign and 4 - f
    const uint32_t neg = (~x >> 2) & 0x11111111u;
    w[i] = (((x & 0x33333333u) ^ (neg * 3u)) + neg) | (neg << 3);
  }
  transpose_nibbles(w);
  #pragma unroll
  for (int j = 0; j < kGemvTerms; ++j) store(j, w[7 - j]);
  const uint32_t s8 = finite ? (uint32_t)(q + 7) << 3 : 0x7fu;   // e4m3 of 2^q, or NaN
  const uint32_t pair = s8 | (__shfl_down_sync(0xffffffffu, s8, 2) << 8);
  return pair | (__shfl_down_sync(0xffffffffu, pair, 4) << 16);
}

// Offset of lane's four bytes of digit j among a token's 8 x 128 bytes: 16-byte
// pieces exchanged as the 128-byte swizzle has them.
__device__ __forceinline__ int gemv_digit_at(int lane, int j) { return j * 128 + (((lane >> 2) ^ j) << 4) + (lane & 3) * 4; }

// Where digit row `row` of a group has its scale word in an atom.
__device__ __forceinline__ int gemv_scale_at(int row) { return (row % 32) * 16 + (row / 32) * 4; }

// Digits and scales of one token's 256 elements (a warp's) to an image: `token`
// its digits, `atoms` the group's scale atoms.  Lane 8a + j writes digit j's scales of atom a.
__device__ __forceinline__ void gemv_put(float (&v)[8], float up, uint8_t* token, uint8_t* atoms, int place) {
  const int lane = (int)(threadIdx.x & 31u);
  const uint32_t four = gemv_digits(v, up, [&](int j, uint32_t w) {
    *reinterpret_cast<uint32_t*>(token + gemv_digit_at(lane, j)) = w;
  });
  const uint32_t mine = __shfl_sync(0xffffffffu, four, lane & 24);
  *reinterpret_cast<uint32_t*>(atoms + (lane >> 3) * kSfAtom + gemv_scale_at(place * kGemvTerms + (lane & 7))) = mine;
}

// Pairs of one expert in ascending order, p.room at a time; one warp, the result in shared memory.
__device__ __forceinline__ void gemv_group_pairs(const GemvParams& p, GemvGroups& out, GemvGroupScratch& tmp) {
  const int lane = (int)(threadIdx.x & 31u);
  const uint32_t lt = (1u << lane) - 1u;
  for (int i = lane; i < p.experts; i += 32) tmp.seen[i] = 0;
  __syncwarp();
  int groups = 0;
  for (int i0 = 0; i0 < p.pairs; i0 += 32) {
    const int i = i0 + lane;
    const int id = i < p.pairs ? __ldcg(p.ids + i) : -1;
    const bool valid = (unsigned)id < (unsigned)p.experts;
    const uint32_t same = __match_any_sync(0xffffffffu, valid ? id : -1);
    const int before = valid ? tmp.seen[id] : 0, at = before + __popc(same & lt);
    const int old = valid && before > 0 ? tmp.open[id] : 0;
    const bool first = valid && at % p.room == 0;
    const uint32_t firsts = __ballot_sync(0xffffffffu, first);
    int grp = groups + __popc(firsts & lt);
    const uint32_t mine = firsts & same & (lt | (1u << lane));   // the group's first row, if it is among these 32
    const int theirs = __shfl_sync(0xffffffffu, grp, mine ? 31 - __clz(mine) : lane);
    grp = mine ? theirs : old;
    if (first) out.expert[grp] = (uint16_t)id, out.rows[grp] = 0;
    __syncwarp();
    if (valid) atomicAdd(&out.rows[grp], 1);
    if (valid && (same >> lane) == 1u) tmp.seen[id] = (uint16_t)(at + 1), tmp.open[id] = (uint16_t)grp;   // the expert's last row among these
    if (i < p.pairs) tmp.group_of[i] = (int16_t)(valid ? grp : -1), tmp.place_of[i] = (int16_t)(at % p.room);
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
    if (g0 + lane < groups) out.before[g0 + lane] = (uint16_t)(sum + x - rows);
    sum += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) out.count = groups;
  __syncwarp();
  for (int i = lane; i < p.pairs; i += 32)
    if (tmp.group_of[i] >= 0) out.pair[out.before[tmp.group_of[i]] + tmp.place_of[i]] = (uint16_t)i;
}

// grid: (row of x, chunk of 8 K blocks, split).  A CTA takes the largest magnitude
// of its row in the whole split (every CTA of the split reads it: a few KB from L2),
// then each warp expands one K block.
template <bool kMoe>
__global__ void __launch_bounds__(kExpandThreads) gemv_expand_kernel(const __grid_constant__ GemvParams p) {
  __shared__ uint32_t s_top[kExpandThreads / 32];
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  griddep_wait();
  griddep_launch_dependents();                            // after the wait: see the head of this file
  const int r = (int)blockIdx.x;
  int group, place, rows, before, rows_all, groups_all;
  int64_t src;
  if constexpr (kMoe) {
    __shared__ GemvGroups s_groups;
    __shared__ GemvGroupScratch s_tmp;
    if (warp == 0) gemv_group_pairs(p, s_groups, s_tmp);
    __syncthreads();
    group = s_tmp.group_of[r], place = s_tmp.place_of[r];
    if (group < 0) {                                      // not an expert: a row of zeros
      for (int c = (int)(blockIdx.z * gridDim.y + blockIdx.y) * kExpandThreads + tid; c < p.n; c += (int)(gridDim.y * gridDim.z) * kExpandThreads)
        store_out(p.out, p.out_dtype, (int64_t)r * p.ldo + c, 0.f);
      return;
    }
    rows = s_groups.rows[group], before = s_groups.before[group];
    rows_all = groups_all = p.pairs;
    src = (int64_t)(p.x_per_pair ? r : r / p.topk) * p.ldx;
  } else {
    const int batch = p.l == 1 ? 0 : r / p.m, row = r - batch * p.m, pass = row / kGemvTokens;
    place = row % kGemvTokens;
    group = batch * p.passes + pass;
    rows = min(kGemvTokens, p.m - pass * kGemvTokens);
    before = batch * p.m + pass * kGemvTokens;
    rows_all = p.l * p.m, groups_all = p.l * p.passes;
    src = (int64_t)batch * p.x_batch + (int64_t)row * p.ldx;
  }
  const int split = (int)blockIdx.z, chunk = (int)blockIdx.y;
  const int kb0 = (p.k_blocks * split) >> p.split_bits, kb1 = (p.k_blocks * (split + 1)) >> p.split_bits;
  if (kb0 + chunk * kExpandBlocks >= kb1) return;

  // this thread's elements, and the largest of the split
  const int kb = kb0 + chunk * kExpandBlocks + warp, k0 = kb * kBK + lane * 8;
  Raw8 raw;
  raw.a = raw.b = make_uint4(0, 0, 0, 0);
  uint32_t top = 0;
  gemv_with_loader(p, [&](auto load) {
    if (kb < kb1 && k0 < p.k) raw = load(src + k0);
    const int c1 = min(kb1 * kBK, p.k) / 8;
    for (int c = kb0 * (kBK / 8) + tid; c < c1; c += 4 * kExpandThreads) {
      Raw8 r[4];
      #pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = load(src + (int64_t)(c + u * kExpandThreads < c1 ? c + u * kExpandThreads : c) * 8);
      #pragma unroll
      for (int u = 0; u < 4; ++u) top = max(top, largest8(r[u], p.x_dtype));
    }
  });
  float v[8];
  widen8(raw, p.x_dtype, v);
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_top[warp] = top;
  __syncthreads();
  #pragma unroll
  for (int i = 0; i < kExpandThreads / 32; ++i) top = max(top, s_top[i]);
  const int e = gemv_exponent(top);
  if (chunk == 0 && tid == 0) p.back[((int64_t)group * kGemvTokens + place) * p.splits + split] = exp2_int(-e);
  if (kb >= kb1) return;
  uint8_t* const image = p.image + gemv_image_at(kb, rows_all, groups_all, before, group);
  gemv_put(v, exp2_int(e), image + place * kGemvTokenBytes, image + rows * kGemvTokenBytes, place);
}

// ---------------------------------------------------------------------------
// Products
// ---------------------------------------------------------------------------
constexpr int kGemvWBytes = kBM * kBK / 2 + kSfStageBytes;   // a weight slot: 128 rows x 256, scale atoms
constexpr int kBMBits = 7;
static_assert(1 << kBMBits == kBM, "rows of a block");
constexpr int kGemvSfCols = 32;          // TMEM columns of a weight slot: its scales and x's
constexpr int kGemvMaxWSlots = 12, kGemvMaxXSlots = 8;        // even; 8 x slots where the kernel expands x
constexpr int kGemvSelfTokens = 2;       // largest group that gemv_kernel expands itself
constexpr int kGemvSelfPairs = 32;       // and the most rows of an expert call
// warps: epilogue 0-3, expansion 0-7 (without it x copies: 4), then weights, two for the MMAs
constexpr int gemv_threads(bool self) { return 32 * (self ? 11 : 8); }

// Copy one scale atom into TMEM: row i to lane i of each lane quadrant, 4 columns.
__device__ __forceinline__ void tc_cp_32x128b_x4(uint32_t taddr, uint64_t s_desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(s_desc) : "memory");
}

// Store to shared memory of any CTA of the cluster, its bytes counted on an
// mbarrier there: the data and the signal in one, no fence.
__device__ __forceinline__ void st_async(uint32_t cluster_addr, const float (&v)[1], uint32_t cluster_bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.f32 [%0], %1, [%2];" ::"r"(cluster_addr),
               "f"(v[0]), "r"(cluster_bar)
               : "memory");
}
__device__ __forceinline__ void st_async(uint32_t cluster_addr, const float (&v)[4], uint32_t cluster_bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                   cluster_addr),
               "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "r"(cluster_bar)
               : "memory");
}
__device__ __forceinline__ void lds_vec(uint32_t addr, float (&v)[1]) {
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[0]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void lds_vec(uint32_t addr, float (&v)[4]) {
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Tokens of an epilogue step, which waits once for its loads; the columns behind
// the last token's are other accumulators or scales, and not used.  And tokens of one
// store between the CTAs of a cluster (16 tokens 7168 x 16384 19.2 us, 20.0 with stores of one
// token; two tokens at once cost the self-expanding form 0.2 us).
template <bool kSelf> constexpr int kGemvStep = kSelf ? 2 : 4;
template <bool kSelf> constexpr int kGemvSend = kSelf ? 1 : 4;
// Accumulator columns of a step.
__device__ __forceinline__ void tmem_ld_terms(uint32_t taddr, uint32_t (&d)[16]) { tmem_ld_32x32b_x16(taddr, d); }
__device__ __forceinline__ void tmem_ld_terms(uint32_t taddr, uint32_t (&d)[32]) { tmem_ld_32x32b_x32(taddr, d); }
template <int N>
__device__ __forceinline__ void tmem_terms_ready(uint32_t (&d)[N]) {
  #pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(d[i]));
}

// What a cluster works on: tile t of the call.
struct GemvTile { int group, row_block, batch, rows, before, expert; };

// Groups of a small expert call, made by each CTA for itself.
struct GemvSmallGroups {
  int count;
  int expert[kGemvSelfPairs], rows[kGemvSelfPairs];
  int pair[kGemvSelfPairs][kGemvSelfTokens], x_row[kGemvSelfPairs][kGemvSelfTokens];
};

__device__ __forceinline__ int gemv_pair(const GemvSmallGroups& g, const GemvTile& t, int row) { return g.pair[t.group][row]; }
__device__ __forceinline__ int gemv_pair(const GemvGroups& g, const GemvTile& t, int row) { return g.pair[t.before + row]; }

template <bool kMoe, bool kSelf, class Groups>
__device__ __forceinline__ GemvTile gemv_tile(const GemvParams& p, const Groups& groups, int t) {
  GemvTile r;
  if constexpr (kMoe) {
    r.group = t / p.row_blocks, r.row_block = t - r.group * p.row_blocks, r.batch = 0;
    r.expert = groups.expert[r.group], r.rows = groups.rows[r.group];
    if constexpr (kSelf) r.before = 0;
    else r.before = groups.before[r.group];
  } else {
    // groups of the same weights next to one another: they share them in L2 (the branches spare
    // two divisions, about 0.1 us, where they are not needed)
    const int rest = p.passes == 1 ? t : t / p.passes, pass = t - rest * p.passes;
    r.batch = p.l == 1 ? 0 : rest / p.row_blocks, r.row_block = rest - r.batch * p.row_blocks;
    r.group = r.batch * p.passes + pass;
    r.rows = min(kGemvTokens, p.m - pass * kGemvTokens), r.before = r.batch * p.m + pass * kGemvTokens;
    r.expert = 0;
  }
  return r;
}

// A cluster of `splits` CTAs owns a 128-row block and a group; each CTA has a
// part of K.  Shared memory holds a ring of weight slots (one matrix' K block,
// 18 KB) and a ring of x slots.  The sums of the CTAs of a cluster meet in distributed
// shared memory: each CTA owns 128 / splits rows, gets the others' sums for them and
// adds them in the order of the CTAs.
//
// Bound: the weights' way from HBM.  One token 16384 x 7168 (66 MB) takes 13.4 us (4.9
// TB/s); a ring of eight such slots alone, one CTA on each SM copying 66 MB and computing nothing, takes 13.2, plain
// 32-byte loads 12.3 (10.1 us at the rate of a long copy: what is short here is the time).  The
// gated pair 14336 x 4096 (66 MB) 13.9 us, 8 experts of a token, gated, 2048 x 7168 (132 MB) 24.0 (the
// ring 22.7), 64 rows of experts 7168 x 2048 (348 MB) 55 us (the ring 53.5), one token 128256 x 4096 (296 MB) 45.8 us,
// 6.5 TB/s.  Smaller calls are bound by the
// chain from the end of the work before to the first product and from the last to the output, about
// 4 us: 4.4 us for 1001 x 1536 (0.9 MB).  More tokens cost the expansion, 0.1 us of epilogue each
// and room for fewer weights on their way: 7168 x 16384 14.3 us for one, 18.8 for 16.
template <bool kDual, bool kMoe, bool kSelf, int kTmemCols>
__global__ void __launch_bounds__(gemv_threads(kSelf), 2) gemv_kernel(const __grid_constant__ GemvParams p) {
  constexpr int kMats = kDual ? 2 : 1;
  constexpr int kWWarp = kSelf ? 8 : 5, kMmaWarp = kWWarp + 1;   // and kMmaWarp + 1
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t bar_w_full[kGemvMaxWSlots], bar_w_free[kGemvMaxWSlots];
  __shared__ uint64_t bar_x_full[kGemvMaxXSlots], bar_x_free[kGemvMaxXSlots];
  __shared__ uint64_t bar_acc_full[2], bar_acc_free[2], bar_drain[2], bar_go;
  __shared__ uint64_t bar_sums, bar_sums_free;            // this CTA's rows: all sums there; its sums taken everywhere
  __shared__ uint32_t s_tmem_base;
  __shared__ volatile int s_abort;
  __shared__ uint32_t s_top[kGemvSelfTokens];             // expansion: largest magnitudes
  // Of the tokens of a tile: 2^-e (tile index % kBackSlots), and the row of out (index % 2, experts).  finish(i) reads
  // both, and its first barrier lies behind all that finish(i - 1) reads: written inside finish(i), two slots do.
  // expand(i) writes 2^-e before finish(i - 1), when a warp may still be in finish(i - 2) (no barrier of the whole CTA
  // comes between them where the group stays the same and nothing is exchanged): slots i, i - 1 and i - 2 differ.
  constexpr int kBackSlots = kSelf ? 4 : 2;
  __shared__ float s_back[kBackSlots][kSelf ? kGemvSelfTokens : kGemvTokens];
  __shared__ int s_row[2][kGemvTokens];
  __shared__ std::conditional_t<!kMoe, char, std::conditional_t<kSelf, GemvSmallGroups, GemvGroups>> s_groups;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const int warp = (int)threadIdx.x >> 5, lane = (int)(threadIdx.x & 31u);
  const int splits = p.splits;
  const int rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int cluster = (int)blockIdx.x >> p.split_bits, clusters = (int)gridDim.x >> p.split_bits;
  const int kb0 = (p.k_blocks * rank) >> p.split_bits, kb1 = (p.k_blocks * (rank + 1)) >> p.split_bits;
  // shared memory: weight slots, x slots, the cluster's sums
  const int x_bytes = p.group_rows * kGemvTokenBytes + kGemvXSfBytes;   // a multiple of 1024
  // odd numbers of tokens: 8 columns more, whose digits are whatever lies behind; they are not used
  const int n_pad = (p.group_rows * kGemvTerms + 15) / 16 * 16;
  const uint32_t w_base = smem_base, x_base = smem_base + p.w_slots * kGemvWBytes;
  const uint32_t sums_base = x_base + p.x_slots * x_bytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.w_slots; ++i) mbar_init(smem_u32(&bar_w_full[i]), 1), mbar_init(smem_u32(&bar_w_free[i]), 1);
    for (int i = 0; i < p.x_slots; ++i) {
      mbar_init(smem_u32(&bar_x_full[i]), kSelf ? p.group_rows : 1);
      mbar_init(smem_u32(&bar_x_free[i]), kMats);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 2);
      mbar_init(smem_u32(&bar_acc_free[i]), 4);
      mbar_init(smem_u32(&bar_drain[i]), 1);
    }
    mbar_init(smem_u32(&bar_sums), 1);
    mbar_init(smem_u32(&bar_go), 8);
    mbar_init(smem_u32(&bar_sums_free), splits);
    s_abort = 0;
    for (int i = 0; i < kGemvSelfTokens; ++i) s_top[i] = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == kMmaWarp) tmem_alloc<kTmemCols>(smem_u32(&s_tmem_base));
  if constexpr (kMoe && !kSelf) {
    // like the weights the ids are there when the expansion lets this kernel start (64 rows of experts
    // 7168 x 2048 55.0 us, 57.3 with the expansion's groups); the ring is scratch until its first load
    if (warp == 0) {
      gemv_group_pairs(p, s_groups, *reinterpret_cast<GemvGroupScratch*>(smem_raw));
      fence_proxy_async_smem();
    }
  }
  if constexpr (kMoe && kSelf) griddep_wait();            // the experts' ids
  if constexpr (kMoe && kSelf) {
    // rows of one expert in ascending order, kGemvSelfTokens at a time
    if (warp == 0) {
      const uint32_t lt = (1u << lane) - 1u;
      const int id = lane < p.pairs ? __ldcg(p.ids + lane) : -1;
      const bool valid = (unsigned)id < (unsigned)p.experts;
      const uint32_t same = __match_any_sync(0xffffffffu, valid ? id : -1);
      const int at = __popc(same & lt);
      const bool first = valid && at % kGemvSelfTokens == 0;
      const uint32_t firsts = __ballot_sync(0xffffffffu, first);
      const uint32_t mine = firsts & same & (lt | (1u << lane));
      const int from = valid ? 31 - __clz(mine) : lane;
      const int grp = __shfl_sync(0xffffffffu, __popc(firsts & lt), from);
      if (valid) {
        s_groups.pair[grp][at % kGemvSelfTokens] = lane;
        s_groups.x_row[grp][at % kGemvSelfTokens] = p.x_per_pair ? lane : lane / p.topk;
      }
      if (first) s_groups.expert[grp] = id, s_groups.rows[grp] = min(kGemvSelfTokens, __popc(same) - at);
      if (lane == 0) s_groups.count = __popc(firsts);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (splits > 1) cluster_sync();                         // the others' barriers exist
  tc_fence_after();
  const uint32_t tmem = s_tmem_base;
  const AbortCtl ctl{&s_abort, p.status, p.wait_limit};
  if (threadIdx.x == 0) griddep_launch_dependents();
  int tiles;
  if constexpr (kMoe) tiles = s_groups.count * p.row_blocks;
  else tiles = p.l * p.passes * p.row_blocks;
  const int atoms_all = p.k / kKStep;                     // 64-deep atoms of a 128-row block

  if (warp == kWWarp) {
    // ------------------------------------------------------------ weights
    if (elect_one()) {
      // Weights that are read once leave L2 to what is read again (x's images, the next kernel's input): 3 tokens 14336 x
      // 4096 10.3 us, 11.2 with the normal policy.  More groups of one matrix find it in L2.  An expert's groups
      // are too far apart for that: evict-first is better for any number of tokens, the normal policy hardly ever (64 rows of
      // experts 7168 x 2048 60.6 and 63.2; 256 rows of 64 experts 2048 x 4096 63.0 and 68.9, all of 8 experts 37.0 and 38.3;
      // 32 of 8 experts 4096 x 14336 102.7 and 107.5; 256 of 8 experts 7168 x 2048 49.0 and 48.8).
      const uint64_t pol = kMoe || p.passes == 1 ? policy_evict_first() : policy_evict_normal();
      int slot = 0;
      uint32_t phase = 0, issued = 0, last_phase = 0;
      // The tables are in global memory, where the caller may have written others since the last call.  A tile's maps are
      // acquired ahead, behind the loads of the first K block of the tile before (64 rows of experts 7168 x 2048 55.3 us;
      // 56.8 where each tile starts with it).
      [[maybe_unused]] int acquired = -1;
      [[maybe_unused]] auto acquire = [&](int expert) {
        if (expert == acquired) return;
        tensor_map_acquire(&p.table1[expert].map);
        if constexpr (kDual) tensor_map_acquire(&p.table2[expert].map);
        acquired = expert;
      };
      bool ok = true;
      if constexpr (kSelf) {
        // x's loads first: behind the weights' first slots they would take twice as long
        griddep_wait();
        if (cluster < tiles) {
          if constexpr (kMoe) acquire(gemv_tile<kMoe, kSelf>(p, s_groups, cluster).expert);
          ctl.wait(smem_u32(&bar_go), 0, kDevTimeoutStageFree);
        }
      }
      for (int t = cluster; t < tiles && ok; t += clusters) {
        const GemvTile tc = gemv_tile<kMoe, kSelf>(p, s_groups, t);
        const void *map[2] = {&p.map1, &p.map2};
        const uint8_t* sf[2] = {p.sf1, p.sf2};
        if constexpr (kMoe) {
          map[0] = &p.table1[tc.expert].map, sf[0] = p.table1[tc.expert].sf;
          if constexpr (kDual) map[1] = &p.table2[tc.expert].map, sf[1] = p.table2[tc.expert].sf;
          acquire(tc.expert);                             // the first tile's; the others' have been
        }
        const size_t atom0 = ((size_t)tc.batch * p.row_blocks + tc.row_block) * (size_t)atoms_all;
        for (int kb = kb0; kb < kb1 && ok; ++kb) {
          const int atoms = min(kBK / kKStep, atoms_all - kb * (kBK / kKStep));
          #pragma unroll
          for (int mat = 0; mat < kMats; ++mat) {
            if (!kSelf && slot == 0 && phase == 1u) griddep_wait();   // the ring is full: again, no polling
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
          if constexpr (kMoe)
            if (kb == kb0 && t + clusters < tiles) acquire(gemv_tile<kMoe, kSelf>(p, s_groups, t + clusters).expert);
        }
      }
      if (!ok)                                            // copies in flight land before the CTA winds down
        for (int s = 0; s < p.w_slots; ++s)
          if ((issued >> s) & 1u) ctl.drain_copies(smem_u32(&bar_w_full[s]), (last_phase >> s) & 1u);
    }
  } else if (!kSelf && warp == 4) {
    // ------------------------------------------------------------ x: copied
    griddep_wait();                                       // the expansion is done
    if (elect_one()) {
      const uint64_t pol = policy_evict_normal();
      const int rows_all = kMoe ? p.pairs : p.l * p.m, groups_all = kMoe ? p.pairs : p.l * p.passes;
      int slot = 0;
      uint32_t phase = 0, issued = 0, last_phase = 0;
      bool ok = true;
      for (int t = cluster; t < tiles && ok; t += clusters) {
        const GemvTile tc = gemv_tile<kMoe, kSelf>(p, s_groups, t);
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
  } else if (warp >= kMmaWarp) {
    // ------------------------------------------------------------ MMA
    // Two issuing threads, each with its own accumulator: an instruction or a
    // barrier check costs its thread 30 to 100 cycles, and one thread's 770 cycles for a
    // K block (two waits, eight copies, four MMAs, two commits; measured) were as long as
    // the block takes to arrive.  They take the weight slots in turn: gate and up, or even and
    // odd K blocks, whose sums the epilogue adds.  (The numbers of slots, x's too, are even, so that
    // a slot is always the same thread's and its phases are waited for one after the other: a thread that
    // tested a phase the other had not waited for could take the one before for it.)
    griddep_wait();                                       // nothing to do before; and no polling beside a kernel at work
    if (elect_one()) {
      const int me = warp - kMmaWarp;
      const uint64_t w_desc0 = kmajor_sw128_desc(w_base), x_desc0 = kmajor_sw128_desc(x_base);
      const uint64_t sf_desc0 = sf_atom_desc(w_base + kBM * kBK / 2), xsf_desc0 = sf_atom_desc(x_base);
      // accumulators, then for each weight slot 16 columns of its scales and 16 of x's with them (free
      // when the slot is: the MMAs that read them are done)
      const uint32_t sf_col = tmem + p.acc_bufs * 2 * n_pad;
      const int span = kb1 - kb0;
      int ws = me, xs = kDual ? 0 : me, acc = 0, done = 0;   // done: K blocks before this tile
      uint32_t w_phase = 0, x_phase = 0, acc_phase = 0;
      bool ok = true, any = false;
      for (int t = cluster; t < tiles && ok; t += clusters, done += span) {
        const GemvTile tc = gemv_tile<kMoe, kSelf>(p, s_groups, t);
        const int n_cols = (tc.rows * kGemvTerms + 15) / 16 * 16;
        const int xsf_at = (kSelf ? p.group_rows : tc.rows) * kGemvTokenBytes;
        const uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(n_cols >> 3) << 17) | ((uint32_t)(kBM >> 4) << 24);
        const uint32_t d_acc = tmem + (acc * 2 + me) * n_pad;
        if (!ctl.wait(smem_u32(&bar_acc_free[acc]), acc_phase ^ 1u, kDevTimeoutAccFree)) break;
        tc_fence_after();
        uint32_t more = 0;
        for (int kb = kb0 + (kDual ? 0 : (done ^ me) & 1); kb < kb1; kb += kDual ? 1 : 2) {
          if (!ctl.wait(smem_u32(&bar_x_full[xs]), x_phase, kDevTimeoutTmaFull) ||
              !ctl.wait(smem_u32(&bar_w_full[ws]), w_phase, kDevTimeoutTmaFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t dx = desc_advance(x_desc0, xs * x_bytes), dw = desc_advance(w_desc0, ws * kGemvWBytes);
          const uint64_t dxs = desc_advance(xsf_desc0, xs * x_bytes + xsf_at);
          const uint64_t dws = desc_advance(sf_desc0, ws * kGemvWBytes);
          const uint32_t sf = sf_col + kGemvSfCols * ws, xsf = sf + kGemvSfCols / 2;
          const int atoms = atoms_all - kb * (kBK / kKStep);
          #pragma unroll
          for (int j = 0; j < kBK / kKStep; ++j) {
            if (j < atoms) {
              tc_cp_32x128b_x4(xsf + 4 * j, desc_advance(dxs, j * kSfAtom));
              tc_cp_32x128b_x4(sf + 4 * j, desc_advance(dws, j * kSfAtom));
              tc_mma_nvf4(d_acc, desc_advance(dw, 32 * j), desc_advance(dx, 32 * j), idesc, sf + 4 * j, xsf + 4 * j, more);
              more = 1;
            }
          }
          tc_commit(smem_u32(&bar_w_free[ws]));
          tc_commit(smem_u32(&bar_x_free[xs]));
          any = true;
          if ((ws += 2) >= p.w_slots) ws -= p.w_slots, w_phase ^= 1u;
          if ((xs += kDual ? 1 : 2) >= p.x_slots) xs -= p.x_slots, x_phase ^= 1u;
        }
        if (!ok) break;
        tc_commit(smem_u32(&bar_acc_full[acc]));
        if (++acc == p.acc_bufs) acc = 0, acc_phase ^= 1u;
      }
      if (s_abort && any) {
        tc_commit(smem_u32(&bar_drain[me]));
        ctl.drain(smem_u32(&bar_drain[me]), 0);
      }
    }
  } else {
    // ------------------------------------------------------------ workers: expansion, epilogue
    griddep_wait();                                       // x or its expansion; and nothing is written before
    const int row = warp * 32 + lane;
    const int own_bits = kBMBits - p.split_bits, own_rows = 1 << own_bits, owner = row >> own_bits;   // the CTA that finishes this thread's row
    if constexpr (kMoe && kSelf) {                        // rows without an expert are zero
      for (int i = (int)blockIdx.x; i < p.pairs; i += (int)gridDim.x)
        if ((unsigned)__ldcg(p.ids + i) >= (unsigned)p.experts)
          for (int c = row; c < p.n; c += 256) store_out(p.out, p.out_dtype, (int64_t)i * p.ldo + c, 0.f);
    }
    // Expansion of a tile's x.  A warp takes one token's K block at a time, a lane
    // 8 elements; 8 of them a round.  The warps end each round together: a slot's next
    // user then cannot wait for its barrier before this round's user has (the parity of a
    // phase says nothing about the phase two before), and all give up if one has to.
    const int me = warp, tid = (int)threadIdx.x, span = kb1 - kb0;
    const int slot_mask = p.x_slots - 1, slot_bits = __popc(slot_mask);
    int seen = -1;                                        // the group whose s_top is there
    auto expand = [&](int t, int index) -> bool {
      bool ok = true;
      if constexpr (kSelf) {                              // x in 16 bits, 16-byte aligned
        const GemvTile tc = gemv_tile<kMoe, kSelf>(p, s_groups, t);
        auto x_at = [&](int tok) -> int64_t {
          if constexpr (kMoe) return (int64_t)s_groups.x_row[tc.group][tok] * p.ldx;
          return (int64_t)tc.batch * p.x_batch + (int64_t)(tc.before - tc.batch * p.m + tok) * p.ldx;
        };
        static_assert(kGemvSelfTokens == 2, "token of an item: its last bit");
        const int two = tc.rows - 1;                        // tokens of the group: 1 or 2
        const int items = span << two, done = index * span;
        // the elements of four rounds' items at a time
        auto load_batch = [&](uint4 (&r)[4], int i0) {
          #pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = i0 + 8 * u + me, k0 = (kb0 + (i >> two)) * kBK + lane * 8;
            r[u] = make_uint4(0, 0, 0, 0);
            if (i < items && k0 < p.k) r[u] = ldcg_v4(static_cast<const uint16_t*>(p.x) + x_at(i & two) + k0);
          }
        };
        uint4 raw[4];
        load_batch(raw, 0);
        if (index == 0 && lane == 0) mbar_arrive(smem_u32(&bar_go));
        if (tc.group != seen) {
          if (seen >= 0) {
            named_bar_sync(2, 256);                       // everybody has read the last group's
            if (tid < kGemvSelfTokens) s_top[tid] = 0;
            named_bar_sync(2, 256);
          }
          auto take = [&](const uint4 (&r)[4], int i0) {
            #pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int i = i0 + 8 * u + me;
              if (i >= items) break;
              const uint32_t top = __reduce_max_sync(0xffffffffu, largest8(Raw8{r[u], {}}, p.x_dtype));
              if (lane == 0) atomicMax(&s_top[i & two], top);
            }
          };
          take(raw, 0);
          for (int i0 = 32; i0 < items; i0 += 32) {
            uint4 r[4];
            load_batch(r, i0);
            take(r, i0);
          }
          named_bar_sync(2, 256);
          seen = tc.group;
        }
        if (tid < tc.rows) s_back[index % kBackSlots][tid] = exp2_int(-gemv_exponent(s_top[tid]));
        __syncwarp();
        for (int i0 = 0; i0 < items && ok; i0 += 32) {
          if (i0 > 0) load_batch(raw, i0);
          #pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (i0 + 8 * u >= items || !ok) break;
            const int i = i0 + 8 * u + me, tok = i & two;
            const int c = done + (i >> two), slot = c & slot_mask;
            bool free = true;
            if (i < items) {                              // the same for the whole warp
              free = ctl.wait(smem_u32(&bar_x_free[slot]), (uint32_t)((c >> slot_bits) & 1) ^ 1u, kDevTimeoutStageFree);
              free = __all_sync(0xffffffffu, free);
              if (free) {
                uint8_t* const image = smem_raw + (x_base - smem_u32(smem_raw)) + slot * x_bytes;
                float v[8];
                widen8(Raw8{raw[u], {}}, p.x_dtype, v);
                gemv_put(v, exp2_int(gemv_exponent(s_top[tok])), image + tok * kGemvTokenBytes,
                         image + p.group_rows * kGemvTokenBytes, tok);
                fence_proxy_async_smem();
                __syncwarp();
                // the barrier counts group_rows arrivals: the last row makes up for those that the group lacks
                if (lane == 0)
                  mbar_arrive_n(smem_u32(&bar_x_full[slot]), tok == tc.rows - 1 ? p.group_rows - tc.rows + 1 : 1);
              }
            }
            ok = !named_bar_any(2, 256, !free);
          }
        }
      }
      return ok;
    };
    // A tile's sums: from TMEM, over the cluster, to the output.
    uint32_t phase = 0, acc_phase = 0;
    int acc_buf = 0;
    auto finish = [&](int t, int index) -> bool {
        constexpr int kStep = kGemvStep<kSelf>, kSend = kGemvSend<kSelf>;
        const GemvTile tc = gemv_tile<kMoe, kSelf>(p, s_groups, t);
        // before the wait: a load for each token in the loops below is 0.3 us a token
        if (row < tc.rows) {
          if constexpr (!kSelf) s_back[index % kBackSlots][row] = __ldcg(p.back + ((int64_t)tc.group * kGemvTokens + row) * splits + rank);
          if constexpr (kMoe) s_row[index % 2][row] = gemv_pair(s_groups, tc, row);
        }
        bool ok = ctl.wait(smem_u32(&bar_acc_full[acc_buf]), acc_phase, kDevTimeoutAccFull);
        if (splits > 1 && t != cluster)
          ok = ok && ctl.wait_cluster(smem_u32(&bar_sums_free), phase ^ 1u, kDevTimeoutPeers);
        if (named_bar_any(1, 128, !ok)) return false;       // all of the epilogue's warps or none
        tc_fence_after();
        const uint32_t acc = tmem + ((uint32_t)(warp * 32) << 16) + acc_buf * 2 * n_pad;
        // one K block: only the thread whose turn it was has written its accumulator
        const bool both = kDual || kb1 - kb0 > 1;
        const int only = index * (kb1 - kb0) & 1;
        // sums of a sender in an owner's shared memory: [sender][matrix][token / kSend][row of the owner][token % kSend]
        constexpr uint32_t kVec = 4u * kSend;
        const int sends = (tc.rows + kSend - 1) / kSend;
        const uint32_t slice = sums_base + (uint32_t)((rank * kMats * sends) * own_rows + (row & (own_rows - 1))) * kVec;
        const uint32_t remote = splits > 1 ? mapa_shared(slice, (uint32_t)owner) : 0u;
        const uint32_t remote_bar = splits > 1 ? mapa_shared(smem_u32(&bar_sums), (uint32_t)owner) : 0u;
        if (splits > 1 && threadIdx.x == 0)                 // every CTA's sums of this CTA's rows
          mbar_arrive_expect_tx(smem_u32(&bar_sums), (uint32_t)(kMats * sends * kBM) * kVec);
        auto out_at = [&](int tok) -> int64_t {              // where the token's row of this tile starts
          int64_t at;
          if constexpr (kMoe) at = (int64_t)s_row[index % 2][tok] * p.ldo;
          else at = (int64_t)tc.batch * p.out_batch + (int64_t)(tc.before - tc.batch * p.m + tok) * p.ldo;
          return at + (int64_t)tc.row_block * kBM;
        };
        for (int t0 = 0; t0 < tc.rows; t0 += kStep) {
          uint32_t d[2][kStep * kGemvTerms];
          tmem_ld_terms(acc + (both ? 0 : only * n_pad) + t0 * kGemvTerms, d[0]);
          if (both) tmem_ld_terms(acc + n_pad + t0 * kGemvTerms, d[1]);
          tmem_ld_wait();
          tmem_terms_ready(d[0]), tmem_terms_ready(d[1]);
          float v[2][kStep];
          #pragma unroll
          for (int i = 0; i < kStep; ++i) {
            // without a branch for each token their chains of sums overlap (16 tokens 7168 x 16384 19.2 us, with
            // it 20.0); sums behind the last token's are not stored
            v[0][i] = v[1][i] = 0.f;
            if (!kSelf || t0 + i < tc.rows) {
              const float back = s_back[index % kBackSlots][t0 + i];
              #pragma unroll
              for (int a = 0; a < 2; ++a)
                if (a == 0 || both) {
                  v[a][i] = __uint_as_float(d[a][8 * i + 7]);
                  #pragma unroll
                  for (int j = 6; j >= 0; --j) v[a][i] = fmaf(v[a][i], 0.125f, __uint_as_float(d[a][8 * i + j]));
                  v[a][i] *= back;
                }
            }
            if constexpr (!kDual) v[0][i] += v[1][i];
          }
          if (splits > 1) {
            #pragma unroll
            for (int mat = 0; mat < kMats; ++mat)
              #pragma unroll
              for (int i = 0; i < kStep; i += kSend)
                if (t0 + i < tc.rows) {
                  float some[kSend];
                  #pragma unroll
                  for (int j = 0; j < kSend; ++j) some[j] = v[mat][i + j];
                  st_async(remote + (uint32_t)((mat * sends + (t0 + i) / kSend) * own_rows) * kVec, some, remote_bar);
                }
          } else if (tc.row_block * kBM + row < p.n) {
            #pragma unroll
            for (int i = 0; i < kStep; ++i)
              if (t0 + i < tc.rows)
                store_out(p.out, p.out_dtype, out_at(t0 + i) + row, kDual ? silu_gate_f32(v[0][i], v[1][i]) : v[0][i]);
          }
        }
        // the accumulators may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar_acc_free[acc_buf]));
        if (++acc_buf == p.acc_bufs) acc_buf = 0, acc_phase ^= 1u;
        if (splits > 1) {
          ok = ctl.wait_cluster(smem_u32(&bar_sums), phase, kDevTimeoutPeers);
          if (named_bar_any(1, 128, !ok)) return false;
          for (int i = (int)threadIdx.x; i < own_rows * sends; i += 128) {
            const int r = i & (own_rows - 1), send = i >> own_bits;
            float v[kMats][kSend];
            #pragma unroll
            for (int mat = 0; mat < kMats; ++mat) {
              float part[kGemvMaxSplits][kSend];           // all loads before the first sum
              #pragma unroll
              for (int s = 0; s < kGemvMaxSplits; ++s)
                if (s < splits) lds_vec(sums_base + (uint32_t)(((s * kMats + mat) * sends + send) * own_rows + r) * kVec, part[s]);
              #pragma unroll
              for (int j = 0; j < kSend; ++j) {
                v[mat][j] = part[0][j];
                #pragma unroll
                for (int s = 1; s < kGemvMaxSplits; ++s)
                  if (s < splits) v[mat][j] += part[s][j];
              }
            }
            const int at = rank * own_rows + r;
            if (tc.row_block * kBM + at < p.n) {
              #pragma unroll
              for (int j = 0; j < kSend; ++j) {
                const int tok = send * kSend + j;
                if (tok < tc.rows)
                  store_out(p.out, p.out_dtype, out_at(tok) + at, kDual ? silu_gate_f32(v[0][j], v[kMats - 1][j]) : v[0][j]);
              }
            }
          }
          if (t + clusters < tiles) {
            named_bar_sync(1, 128);                         // all of this CTA's rows are read: the next may come
            if ((int)threadIdx.x < splits) mbar_arrive_cluster(mapa_shared(smem_u32(&bar_sums_free), threadIdx.x));
          }
          phase ^= 1u;
        }
      return true;
    };
    // the next tile's x before a tile's end: that has a second accumulator to wait in
    bool finishing = warp < 4;
    const int count = cluster < tiles ? (tiles - 1 - cluster) / clusters + 1 : 0;
    #pragma unroll 1
    for (int i = 0; i < count + (kSelf ? 1 : 0); ++i) {
      if (kSelf && i < count && !expand(cluster + i * clusters, i)) break;
      const int f = kSelf ? i - 1 : i;
      if (f >= 0 && finishing) finishing = finish(cluster + f * clusters, f);
    }
  }
  tc_fence_before();
  __syncthreads();
  // Nobody writes to a CTA that is gone: each has waited for all that the others
  // send it, unless it gave up a wait.
  if (splits > 1) {
    cluster_arrive();
    if (s_abort) cluster_wait();
  }
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc<kTmemCols>(tmem);
}

}  // namespace nvfp4
