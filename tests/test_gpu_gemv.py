"""GPU: a few tokens times NVFP4 weights (gemv, dual_gemv, moe.gemv,
moe.dual_gemv) against the products in 64 bits.

Tolerance, for y = sum_k w_k x_k with A = sum_k |w_k| a_k, a_k the largest |x| of
the 16 elements around k (and never below 2^-14 of the token's largest, where the digits'
scale stops):
  the digits of x are off by less than 2^-22 a_k: 2^-22 A;
  the first digit's sum has terms of magnitude <= 2 |w_k| a_k, the others' together a
  seventh of that; K/64 MMAs add in fp32, and 16 more roundings follow (eight digits, two
  accumulators, splits), each off by at most 2^-23 of what it adds: (K/64 + 16) 2^-23 * 16/7 A;
  the output is rounded once: eps/2 |y|, or half its smallest step.
"""
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib
from nvfp4_b200 import build as B
from nvfp4_b200 import gemv as V
from nvfp4_b200 import moe
from nvfp4_b200.formats import quantize_nvfp4, swizzle_sf
from oracle import nvfp4_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _ready(cuda_device):
    B.build()
    _lib.load()


def make_weights(n, k, seed, l=1, scale=0.05):
    """(Weights, dense fp64 [l, n, k]) with scales over most of e4m3's range."""
    g = torch.Generator().manual_seed(seed)
    packed, sf, dense = [], [], []
    for _ in range(l):
        w = torch.randn(n, k, generator=g) * scale * torch.exp2(torch.randint(-3, 4, (n, k // 16, 1), generator=g).float()).expand(
            n, k // 16, 16).reshape(n, k)
        p, s = quantize_nvfp4(w)
        packed.append(p)
        sf.append(s)
        dense.append(O.dequantize(p.numpy(), s.numpy()).astype(np.float64))
    b = torch.stack(packed).cuda().permute(1, 2, 0).view(torch.float4_e2m1fn_x2)
    return V.Weights(b, swizzle_sf(torch.stack(sf, -1)).cuda()), np.stack(dense)


def products(x, w):
    """(y, error bound without the output's rounding) in 64 bits: x [m, k], w [n, k]."""
    x = x.double().cpu().numpy()
    m, k = x.shape
    a = np.abs(x).reshape(m, k // 16, 16).max(2, keepdims=True)
    a = np.maximum(a, 2.0 ** -14 * np.abs(x).max(1)[:, None, None] if m else a)
    a = np.broadcast_to(a, (m, k // 16, 16)).reshape(m, k)
    with np.errstate(invalid="ignore"):
        y = x @ w.T
        bound = (a @ np.abs(w).T) * (2.0 ** -22 + (k / 64 + 16) * 2.0 ** -23 * 16 / 7)
    return y, bound


def check(got, y, bound, rounding=1):
    t = torch.finfo(got.dtype)
    got = got.double().cpu().numpy()
    tol = bound + rounding * (t.eps / 2) * (np.abs(y) + bound) + t.smallest_normal * t.eps / 2
    bad = ~(np.abs(got - y) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.nanmax(np.abs(got - y) / tol)))


def gate(g, eg, u, eu):
    """silu(g) u and its bound: |silu'| <= 1.1; exp, the sum, the quotient and the product
    are together off by less than 8 * 2^-24 and the exponential's argument by eg."""
    s = g / (1 + np.exp(-g))
    y = s * u
    return y, 1.1 * eg * (np.abs(u) + eu) + np.abs(s) * eu + 8 * 2.0 ** -24 * np.abs(y)


SIZES = [(1, 1, 64), (1, 128, 256), (2, 129, 320), (1, 300, 1024), (3, 127, 192), (5, 4099, 448), (8, 33, 2048),
         (16, 257, 960), (1, 2048, 7168), (1, 1000, 9216), (4, 512, 2304), (15, 200, 4096)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gemv(m, n, k, dtype):
    w, dense = make_weights(n, k, seed=m * n + k)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k), dtype=torch.float32).to(TYPES[dtype])
    y, bound = products(x, dense[0])
    for out in (None, torch.float32, torch.float16):
        got = V.gemv(x.cuda(), w, out_dtype=out)
        assert got.dtype == (out or x.dtype) and got.shape == (m, n)
        check(got, y, bound)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("m,n,k", SIZES)
def test_dual_gemv(m, n, k, dtype):
    w1, d1 = make_weights(n, k, seed=m * n + k)
    w2, d2 = make_weights(n, k, seed=m * n + k + 1)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(k + 1)).to(TYPES[dtype])
    y, bound = gate(*products(x, d1[0]), *products(x, d2[0]))
    for out in (None, torch.float32):
        check(V.dual_gemv(x.cuda(), w1, w2, out_dtype=out), y, bound)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("m,l", [(1, 3), (2, 2), (17, 1), (40, 2), (100, 1)])
def test_gemv_batches_and_more_rows_than_a_group(m, l):
    n, k = 200, 640
    w, dense = make_weights(n, k, seed=m, l=l)
    x = torch.randn(l, m, k, generator=torch.Generator().manual_seed(m)).bfloat16()
    got = V.gemv(x.cuda(), w, out_dtype=torch.float32)
    assert got.shape == (l, m, n)
    for b in range(l):
        check(got[b], *products(x[b], dense[b]))
    if l == 1:
        assert torch.equal(V.gemv(x[0].cuda(), w, out_dtype=torch.float32), got[0])


def test_gemv_without_rows():
    w, _ = make_weights(40, 128, seed=0)
    assert V.gemv(torch.empty(0, 128, dtype=torch.float16, device="cuda"), w).shape == (0, 40)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_gemv_strided_and_unaligned(dtype):
    n, k, m = 150, 512, 3
    w, dense = make_weights(n, k, seed=7)
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(m, k + 24, generator=g).to(TYPES[dtype])
    for x in (wide[:, 8:8 + k], wide[:, 1:1 + k], wide[:, :k].T.contiguous().T, wide[:1, 3:3 + k].expand(m, k)):
        dev = wide.cuda()
        xd = torch.as_strided(dev, x.shape, x.stride(), x.storage_offset()) if x.data_ptr() >= wide.data_ptr() and \
            x.untyped_storage().data_ptr() == wide.untyped_storage().data_ptr() else x.cuda().T.contiguous().T
        y, bound = products(x, dense[0])
        check(V.gemv(xd, w), y, bound)
        big = torch.full((m, n + 9), float("nan"), dtype=TYPES[dtype], device="cuda")
        out = big[:, 4:4 + n]
        assert V.gemv(xd, w, out=out) is out
        check(out, y, bound)
        assert bool(torch.isnan(big[:, :4]).all()) and bool(torch.isnan(big[:, 4 + n:]).all())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("power", [-140, -126, -100, 0, 60, 100])
def test_gemv_over_the_types_range(dtype, power):
    """Magnitudes far outside fp16's and e4m3's range, tokens of very different ones side by side."""
    n, k = 130, 768
    w, dense = make_weights(n, k, seed=5)
    x = torch.randn(2, k, generator=torch.Generator().manual_seed(9), dtype=torch.float64)
    x = torch.stack((x[0] * 2.0 ** power, x[1])).to(TYPES[dtype])
    y, bound = products(x, dense[0])
    check(V.gemv(x.cuda(), w, out_dtype=torch.float32), y, bound)


def test_gemv_wide_range_within_a_token():
    n, k = 140, 4096
    w, dense = make_weights(n, k, seed=6)
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(1, k, generator=g) * torch.exp2(torch.randint(-30, 8, (1, k // 16, 1), generator=g).float()).expand(
        1, k // 16, 16).reshape(1, k)).bfloat16()
    x[0, 100] = 3000.0
    check(V.gemv(x.cuda(), w, out_dtype=torch.float32), *products(x, dense[0]))
    check(V.gemv(torch.zeros_like(x).cuda(), w, out_dtype=torch.float32), np.zeros((1, n)), np.zeros((1, n)))


@pytest.mark.parametrize("m", [2, 6])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_gemv_non_finite_tokens_are_nan_and_leave_the_others(m, value):
    n, k = 260, 1024
    w, dense = make_weights(n, k, seed=8)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).half()
    y, bound = products(x, dense[0])
    x[1, 700] = value
    got = V.gemv(x.cuda(), w)
    assert bool(torch.isnan(got[1]).all())
    keep = [i for i in range(m) if i != 1]
    check(got[keep], y[keep], bound[keep])


def test_gemv_weights_written_just_before():
    """Each call sees the weights that the stream wrote before it, also by its very last kernel."""
    n, k = 2048, 4096
    w, _ = make_weights(n, k, seed=1)
    sets = [make_weights(n, k, seed=s)[0] for s in (2, 3)]
    for m in (1, 6):
        x = torch.randn(m, k, device="cuda").bfloat16()
        want = [V.gemv(x, s) for s in sets]
        torch.cuda.synchronize()
        for i in range(30):
            w.b.view(torch.uint8).copy_(sets[i % 2].b.view(torch.uint8))
            w.sfb_perm.view(torch.uint8).copy_(sets[i % 2].sfb_perm.view(torch.uint8))
            assert torch.equal(V.gemv(x, w), want[i % 2]), (m, i)


def test_gemv_repeats_bit_for_bit_and_without_dependent_launch():
    w1, _ = make_weights(1500, 3584, seed=1)
    w2, _ = make_weights(1500, 3584, seed=2)
    for m in (1, 2, 7, 16):
        x = torch.randn(m, 3584, device="cuda").half()
        a = V.dual_gemv(x, w1, w2)
        for _ in range(5):
            assert torch.equal(V.dual_gemv(x, w1, w2), a)
        os.environ["NVFP4_PDL"] = "0"
        try:
            assert torch.equal(V.dual_gemv(x, w1, w2), a)
        finally:
            del os.environ["NVFP4_PDL"]


def test_gemv_on_two_streams_at_once():
    w1, _ = make_weights(2048, 7168, seed=1)
    w2, _ = make_weights(4096, 2048, seed=2)
    cases = [(torch.randn(m, w.k, device="cuda").bfloat16(), w) for m in (1, 4, 16) for w in (w1, w2)]
    want = [V.gemv(x, w) for x, w in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        got = []
        for i, (x, w) in enumerate(cases * 3):
            with torch.cuda.stream(streams[i % 3]):
                got.append(V.gemv(x, w))
        torch.cuda.synchronize()
        for i, y in enumerate(got):
            assert torch.equal(y, want[i % len(cases)])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("m,n", [(1, 2048), (2, 2048), (5, 2048), (1, 192)])
def test_gemv_to_and_fro_between_two_buffers(m, n):
    """A chain of calls that each overwrite what the call before read, and that may start before it ends: as with
    a pause after each."""
    g = torch.Generator("cuda").manual_seed(n)
    b = torch.randint(0, 256, (n, n // 2), generator=g, dtype=torch.uint8, device="cuda")
    # codes of mean square 8.6 at scale 2^-7 (2^-5 for 192): a step's growth is about 1
    sf = torch.full((-(-n // 128), n // 64, 32, 4, 4), 0x04 if n == 2048 else 0x10, dtype=torch.uint8, device="cuda")
    w = V.Weights(b, sf)
    start = torch.randn(m, n, generator=g, device="cuda").bfloat16()

    def chain(pause):
        bufs = [start.clone(), torch.empty_like(start)]
        torch.cuda.synchronize()
        seen = []
        for i in range(40):
            V.gemv(bufs[i % 2], w, out=bufs[1 - i % 2])
            if pause:
                torch.cuda.synchronize()
            if i % 10 == 9:
                seen.append(bufs[1 - i % 2].clone())
        return seen

    want = chain(True)
    assert all(bool(torch.isfinite(t).all()) and bool(t.any()) for t in want)
    for _ in range(10):
        for a, c in zip(chain(False), want):
            assert torch.equal(a, c)
    graph, out = _capture(lambda: chain_captured(w, start))
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[-1])
    del graph


def chain_captured(w, start):
    bufs = [start.clone(), torch.empty_like(start)]
    for i in range(40):
        V.gemv(bufs[i % 2], w, out=bufs[1 - i % 2])
    return bufs[0]


def test_gemv_of_32_matrices_of_four_row_blocks():
    """Their scales' memory has the permuted view's first two extents."""
    packed, atoms, dense = raw_weights(500, 128, seed=3, l=32)
    x = torch.randn(32, 1, 128, generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    y = V.gemv(x, V.Weights(packed.permute(1, 2, 0), atoms))
    assert torch.equal(y, V.gemv(x, V.Weights(packed.permute(1, 2, 0), atoms.permute(3, 4, 1, 5, 2, 0))))
    for b in range(32):
        check(y[b], *products_there(x[b], dense[b]))


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_gemv_on_another_device():
    w, dense = make_weights(200, 512, seed=4)
    other = V.Weights(w.b.to("cuda:1"), w.sfb_perm.contiguous().to("cuda:1"))
    x = torch.randn(3, 512).bfloat16()
    check(V.gemv(x.to("cuda:1"), other), *products(x, dense[0]))


def test_gemv_broadcast_batches_and_out_batches_apart():
    l, m, n, k = 3, 4, 140, 384
    w, dense = make_weights(n, k, seed=12, l=l)
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(1)).half().cuda()
    big = torch.full((l, m + 2, n + 3), float("nan"), dtype=torch.float32, device="cuda")
    got = V.gemv(x[None].expand(l, m, k), w, out=big[:, 1:1 + m, :n])
    for b in range(l):
        check(got[b], *products(x, dense[b]))
    assert int(torch.isnan(big).sum()) == big.numel() - l * m * n


def test_gemv_weights_past_32_bit_offsets():
    """More than 2^31 bytes of weights: the last row blocks against their own products."""
    n, k, m = 70016, 65536, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    b = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    sf = torch.randint(0x20, 0x40, (n // 128, k // 64, 32, 4, 4), generator=g, dtype=torch.uint8, device="cuda")
    x = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    got = {rows: V.gemv(x[:rows], V.Weights(b, sf), out_dtype=torch.float32) for rows in (1, m)}
    for blk in (0, n // 128 - 1):
        rows = slice(128 * blk, 128 * blk + 128)
        plain = sf[blk].permute(2, 1, 0, 3).reshape(128, k // 16).cpu().numpy()
        dense = O.dequantize(b[rows].cpu().numpy(), plain).astype(np.float64)
        y, bound = products(x, dense)
        for r, out in got.items():
            check(out[:, rows], y[:r], bound[:r])
    assert _lib.device_status() == 0


def test_gemv_two_captured_graphs_at_once():
    """Each graph's workspace is its own: replays of both on two streams give what the calls give."""
    w, _ = make_weights(1300, 2560, seed=2)
    xs = [torch.randn(m, 2560, device="cuda").bfloat16() for m in (5, 11)]
    graphs = [_capture(lambda x=x: V.gemv(V.gemv(x, w)[:, :64].repeat(1, 40), w)) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    for seed in range(4):
        for x in xs:
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(seed)).bfloat16())
        torch.cuda.synchronize()
        for _ in range(3):
            for s, (graph, _) in zip(streams, graphs):
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for x, (_, out) in zip(xs, graphs):
            assert torch.equal(out, V.gemv(V.gemv(x, w)[:, :64].repeat(1, 40), w))


# ---------------------------------------------------------------------------
# experts
# ---------------------------------------------------------------------------
def make_experts(e, n, k, seed):
    ws = [make_weights(n, k, seed=seed + i) for i in range(e)]
    return moe.ExpertWeights([(w.b, w.sfb_perm) for w, _ in ws]), np.stack([d[0] for _, d in ws])


MOE_SIZES = [(1, 1, 1, 64, 128), (1, 8, 16, 200, 640), (4, 8, 12, 129, 1024), (5, 3, 7, 130, 320), (16, 2, 64, 60, 256),
             (33, 1, 3, 100, 512), (32, 8, 9, 257, 192), (2, 4, 4, 1500, 2304)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("t,topk,e,n,k", MOE_SIZES)
def test_moe_gemv(t, topk, e, n, k, dtype):
    """Choices drawn with repetitions, some outside the experts; a row for each token and for each choice."""
    w1, d1 = make_experts(e, n, k, seed=100 * t)
    w2, d2 = make_experts(e, n, k, seed=100 * t + 50)
    g = torch.Generator().manual_seed(t + k)
    ids = torch.randint(-1, e + 1, (t, topk), generator=g, dtype=torch.int32)
    flat = ids.reshape(-1).tolist()
    for rows in {t, t * topk}:
        x = torch.randn(rows, k, generator=g).to(TYPES[dtype])
        one = moe.gemv(x.cuda(), ids.cuda(), w1, out_dtype=torch.float32)
        two = moe.dual_gemv(x.cuda(), ids.cuda(), w1, w2)
        assert one.shape == two.shape == (t * topk, n) and two.dtype == x.dtype
        for p, ex in enumerate(flat):
            if not 0 <= ex < e:
                assert not bool(one[p].any()) and not bool(two[p].any())
                continue
            xr = x[p if rows == t * topk else p // topk][None]
            y1, b1 = products(xr, d1[ex])
            check(one[p:p + 1], y1, b1)
            check(two[p:p + 1], *gate(y1, b1, *products(xr, d2[ex])))
    assert _lib.device_status() == 0


@pytest.mark.parametrize("ids", [[[-1, 9], [100, -5]], [[2, 2], [2, 2]], [[0, 1], [1, 0]]])
def test_moe_gemv_no_expert_one_expert_and_swapped(ids):
    w, d = make_experts(4, 150, 256, seed=3)
    ids = torch.tensor(ids, dtype=torch.int32)
    for scale in (1, 20):                                  # few rows, and more than one CTA groups by itself
        x = torch.randn(2 * scale, 256).half()
        big = ids.repeat(scale, 1)
        got = moe.gemv(x.cuda(), big.cuda(), w)
        for p, ex in enumerate(big.reshape(-1).tolist()):
            if 0 <= ex < 4:
                check(got[p:p + 1], *products(x[p // 2][None], d[ex]))
            else:
                assert not bool(got[p].any())


def test_moe_gemv_out_rows_apart_and_one_choice_vector():
    w, d = make_experts(5, 96, 192, seed=9)
    x = torch.randn(6, 192).bfloat16()
    ids = torch.tensor([0, 4, 2, 2, 1, 3], dtype=torch.int32)
    big = torch.full((6, 128), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = moe.gemv(x.cuda(), ids.cuda(), w, out=big[:, 16:112])
    for p in range(6):
        check(got[p:p + 1], *products(x[p][None], d[int(ids[p])]))
    assert bool(torch.isnan(big[:, :16]).all()) and bool(torch.isnan(big[:, 112:]).all())


@pytest.mark.parametrize("tokens", [3, 12, 50])
def test_moe_gemv_ids_weights_and_x_written_just_before(tokens):
    """What the stream's last kernels wrote, the ids and weights too, which the call reads first."""
    w, _ = make_experts(8, 1024, 2048, seed=1)
    other, _ = make_experts(8, 1024, 2048, seed=60)
    g = torch.Generator().manual_seed(tokens)
    sets = [(torch.randint(-1, 8, (tokens, 4), generator=g, dtype=torch.int32).cuda(),
             torch.randn(tokens, 2048, generator=g).bfloat16().cuda(), e) for e in (w, other, w)]
    want = [moe.gemv(x, ids, e) for ids, x, e in sets]
    live, _ = make_experts(8, 1024, 2048, seed=1)
    ids, x = sets[0][0].clone(), sets[0][1].clone()
    torch.cuda.synchronize()
    for i in range(30):
        now_ids, now_x, now_w = sets[i % 3]
        for (b, sf), (nb, ns) in zip(live.w, now_w.w):
            b.view(torch.uint8).copy_(nb.view(torch.uint8))
            sf.view(torch.uint8).copy_(ns.view(torch.uint8))
        x.copy_(now_x)
        ids.copy_(now_ids)
        assert torch.equal(moe.gemv(x, ids, live), want[i % 3]), i
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", list(TYPES))
def test_moe_gemv_unaligned_x_and_strided_choices(dtype):
    w, d = make_experts(6, 160, 448, seed=20)
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(5, 470, generator=g).to(TYPES[dtype]).cuda()
    ids = torch.randint(0, 6, (3, 5), generator=g, dtype=torch.int32).cuda().T
    for off in (0, 8, 3):
        x = wide[:, off:off + 448]
        got = moe.gemv(x, ids, w, out_dtype=torch.float32)
        for p, ex in enumerate(ids.reshape(-1).tolist()):
            check(got[p:p + 1], *products(x[p // 3][None], d[ex]))


def test_moe_gemv_non_finite_tokens_are_nan_and_leave_the_others():
    w, d = make_experts(3, 140, 512, seed=30)
    for tokens in (3, 30):
        x = torch.randn(tokens, 512, generator=torch.Generator().manual_seed(1)).half()
        ids = torch.zeros(tokens, 2, dtype=torch.int32)        # all of them in the groups of one expert
        ids[:, 1] = 2
        y = [products(x, d[0]), products(x, d[2])]
        x[1, 300] = float("inf")
        got = moe.gemv(x.cuda(), ids.cuda(), w)
        for t in range(tokens):
            for j in range(2):
                row = got[2 * t + j][None]
                if t == 1:
                    assert bool(torch.isnan(row).all())
                else:
                    check(row, y[j][0][t:t + 1], y[j][1][t:t + 1])


# ---------------------------------------------------------------------------
# many tiles for each CTA
# ---------------------------------------------------------------------------
def raw_weights(n, k, seed, l=1):
    """(packed [l, n, k/2], atoms [l, rows/128, k/64, 32, 4, 4], dense fp64 [l, n, k]) on the GPU, of random
    codes and scales: large ones quickly."""
    g = torch.Generator("cuda").manual_seed(seed)
    rb = -(-n // 128)
    packed = torch.randint(0, 256, (l, n, k // 2), generator=g, dtype=torch.uint8, device="cuda")
    atoms = torch.randint(0x20, 0x40, (l, rb, k // 64, 32, 4, 4), generator=g, dtype=torch.uint8, device="cuda")
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device="cuda")
    codes = torch.stack((packed & 15, packed >> 4), -1).reshape(l, n, k // 16, 16)
    # [l, row block, quarter, row of 32, atom, block of 16]
    scales = atoms.view(torch.float8_e4m3fn).double().permute(0, 1, 4, 3, 2, 5).reshape(l, rb * 128, k // 16)[:, :n]
    return packed, atoms, (table[codes.int()] * scales.unsqueeze(-1)).reshape(l, n, k)


def products_there(x, w):
    """:func:`products` on the GPU, for large weights."""
    x = x.double()
    m, k = x.shape
    a = torch.maximum(x.abs().reshape(m, k // 16, 16).amax(2), 2.0 ** -14 * x.abs().amax(1, keepdim=True))
    bound = a.repeat_interleave(16, 1) @ w.abs().T * (2.0 ** -22 + (k / 64 + 16) * 2.0 ** -23 * 16 / 7)
    return (x @ w.T).cpu().numpy(), bound.cpu().numpy()


def scaled_rows(rows, k, seed, dtype=torch.bfloat16):
    """Rows whose magnitudes differ by powers of two: a sum taken back with another row's factor shows."""
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn(rows, k, generator=g, device="cuda")
    return (x * torch.exp2(((torch.arange(rows, device="cuda") * 5) % 7 - 3).float())[:, None]).to(dtype)


@pytest.mark.parametrize("l,m,n,k", [(2, 1, 20480, 2048), (2, 2, 20480, 512), (3, 1, 20000, 320), (7, 2, 3000, 512)])
def test_gemv_batch_entries_that_share_a_ctas_tiles(l, m, n, k):
    """A CTA's tiles go over from one batch entry to the next: each row gets its own factor."""
    packed, atoms, dense = raw_weights(n, k, seed=n + l, l=l)
    w = V.Weights(packed.permute(1, 2, 0), atoms)
    x = scaled_rows(l * m, k, seed=k).view(l, m, k)
    first = V.gemv(x, w, out_dtype=torch.float32)
    for b in range(l):
        check(first[b], *products_there(x[b], dense[b]))
        gated = V.dual_gemv(x, w, w, out_dtype=torch.float32)
        y, e = products_there(x[b], dense[b])
        with np.errstate(over="ignore"):
            check(gated[b], *gate(y, e, y, e))
    for _ in range(20):
        assert torch.equal(V.gemv(x, w, out_dtype=torch.float32), first)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("rows", [3, 16])
def test_moe_gemv_choices_that_share_a_ctas_tiles(rows):
    """The same with one expert's tiles after another's."""
    e, n, k = 3, 19200, 256
    packed, atoms, dense = raw_weights(n, k, seed=rows, l=e)
    w = moe.ExpertWeights(list(zip(packed, atoms)))
    x = scaled_rows(rows, k, seed=rows, dtype=torch.float16)
    ids = (torch.arange(rows, dtype=torch.int32, device="cuda") * 2) % e
    first = moe.gemv(x, ids, w, out_dtype=torch.float32)
    for p, ex in enumerate(ids.tolist()):
        check(first[p:p + 1], *products_there(x[p:p + 1], dense[ex]))
    for _ in range(20):
        assert torch.equal(moe.gemv(x, ids, w, out_dtype=torch.float32), first)
    assert _lib.device_status() == 0


# (batch entries, rows, N, K): more row blocks than a GPU has SMs, so that a CTA takes several tiles; the last two with the K
# of a tile shared between CTAs
WIDE = [(1, 1, 20000, 1024), (1, 2, 20000, 2048), (1, 1, 128256, 1024), (1, 2, 128256, 512), (3, 1, 20000, 704),
        (20, 2, 2300, 2304), (1, 5, 20000, 512), (1, 1, 25600, 8192), (2, 1, 12800, 8192)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("l,m,n,k", WIDE)
def test_gemv_several_tiles_a_cta(l, m, n, k, dtype):
    packed, atoms, dense = raw_weights(n, k, seed=n + k, l=l)
    w = V.Weights(packed.permute(1, 2, 0), atoms)
    x = scaled_rows(l * m, k, seed=m, dtype=TYPES[dtype]).view(l, m, k)
    one, two = V.gemv(x, w, out_dtype=torch.float32), V.dual_gemv(x, w, w, out_dtype=torch.float32)
    for b in range(l):
        y, e = products_there(x[b], dense[b])
        check(one[b], y, e)
        with np.errstate(over="ignore"):
            check(two[b], *gate(y, e, y, e))
    del dense
    torch.cuda.empty_cache()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("tokens,topk,e,n,k", [(1, 8, 8, 7168, 2048), (4, 8, 10, 7168, 2048), (16, 2, 8, 7168, 512), (32, 1, 1, 2048, 1024),
                                               (1, 8, 8, 3200, 8192), (5, 8, 8, 7168, 512)])
def test_moe_gemv_several_tiles_a_cta(tokens, topk, e, n, k):
    """One token's experts, and choices that repeat an expert up to 32 times."""
    packed, atoms, dense = raw_weights(n, k, seed=tokens + n, l=e)
    w = moe.ExpertWeights(list(zip(packed, atoms)))
    g = torch.Generator().manual_seed(tokens)
    ids = torch.randint(0, e, (tokens, topk), generator=g, dtype=torch.int32) if tokens > 1 else torch.randperm(e, generator=g)[None, :topk].int()
    for rows in {tokens, tokens * topk}:
        x = scaled_rows(rows, k, seed=rows)
        one = moe.gemv(x, ids.cuda(), w, out_dtype=torch.float32)
        two = moe.dual_gemv(x, ids.cuda(), w, w, out_dtype=torch.float32)
        per = x if rows == tokens * topk else x.repeat_interleave(topk, 0)
        for ex in set(ids.reshape(-1).tolist()):
            at = (ids.reshape(-1) == ex).nonzero()[:, 0].cuda()
            y, err = products_there(per[at], dense[ex])
            check(one[at], y, err)
            with np.errstate(over="ignore"):
                check(two[at], *gate(y, err, y, err))
    del dense
    torch.cuda.empty_cache()
    assert _lib.device_status() == 0


@pytest.mark.parametrize("tokens,topk,e,n,k,before", [(16, 2, 8, 4096, 1024, True), (4, 8, 16, 4096, 768, True), (16, 2, 8, 512, 1024, False),
                                                       (2, 8, 4, 14336, 1024, False), (8, 1, 8, 14336, 1024, False)])
def test_moe_gemv_repeated_experts_with_and_without_space(tokens, topk, e, n, k, before):
    """A call whose choices repeat the experts expands x before the product, where it has the space for that; either
    way the products are right."""
    packed, atoms, dense = raw_weights(n, k, seed=n, l=e)
    w = moe.ExpertWeights(list(zip(packed, atoms)))
    ids = torch.randint(0, e, (tokens, topk), generator=torch.Generator().manual_seed(n), dtype=torch.int32).cuda()
    x = scaled_rows(tokens, k, seed=tokens)
    lib, rows = _lib.load(), tokens * topk
    results = []
    for space in (None, lib.nvfp4_moe_gemv_workspace_bytes(_lib.NVFP4_BF16, 0, tokens, topk, k), "python"):
        out = torch.full((rows, n), float("nan"), device="cuda")
        count = lib.nvfp4_launch_count()
        if space == "python":
            moe.gemv(x, ids, w, out=out)
        else:
            ws = torch.empty(space, dtype=torch.uint8, device="cuda") if space else None
            _lib.check(lib.nvfp4_moe_gemv(x.data_ptr(), _lib.NVFP4_BF16, k, 0, ids.data_ptr(), tokens, topk, w.table().data_ptr(), None, e,
                                          out.data_ptr(), _lib.NVFP4_F32, n, n, k, ws.data_ptr() if space else None, space or 0,
                                          torch.cuda.current_stream().cuda_stream))
        assert lib.nvfp4_launch_count() - count == (2 if before and space else 1)
        results.append(out)
        torch.cuda.synchronize()
    each = x.double().repeat_interleave(topk, 0)
    for ex in set(ids.reshape(-1).tolist()):
        at = ids.reshape(-1) == ex
        for out in results:
            check(out[at], *products_there(each[at], dense[ex]))
    assert _lib.device_status() == 0


def test_expert_table_is_kept_for_calls_on_other_streams():
    """Dropped while a call on another stream is still to read it, the table's memory is not handed out again."""
    packed, atoms, dense = raw_weights(256, 128, seed=1, l=2)
    pairs = list(zip(packed, atoms))
    x, ids = torch.randn(2, 128, device="cuda").half(), torch.tensor([[0], [1]], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    for form in (moe.gemv, lambda x, ids, w: moe.dual_gemv(x, ids, w, w)):
        w = moe.ExpertWeights(pairs)
        at, size = w.table().data_ptr(), w.table().numel()
        want = form(x, ids, w)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(200_000_000)                # about 0.1 s
            got = form(x, ids, w)
        del w
        fresh = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(64)]     # never written
        busy = not side.query()
        assert busy and at not in {t.data_ptr() for t in fresh}
        side.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("tokens", [2, 12])
def test_moe_gemv_table_rewritten_in_place(tokens):
    """Another table at the same address: its descriptors count, not the ones that a call before has read.
    All weights stay alive."""
    sets = [make_experts(6, 640, 1024, seed=s)[0] for s in (1, 30, 60)]
    x = torch.randn(tokens, 1024, generator=torch.Generator().manual_seed(tokens)).bfloat16().cuda()
    ids = (torch.arange(tokens * 4, dtype=torch.int32, device="cuda") % 6).view(tokens, 4)
    want = [(moe.gemv(x, ids, w), moe.dual_gemv(x, ids, w, w)) for w in sets]
    live = make_experts(6, 640, 1024, seed=1)[0]
    for i in range(60):
        live.table().copy_(sets[i % 3].table())
        assert torch.equal(moe.gemv(x, ids, live), want[i % 3][0]), i
        assert torch.equal(moe.dual_gemv(x, ids, live, live), want[i % 3][1]), i
    at = set()
    for i in range(6):                                     # and a new object's table where a dropped one's was
        fresh = moe.ExpertWeights(sets[i % 3].w)
        at.add(fresh.table().data_ptr())
        assert torch.equal(moe.gemv(x, ids, fresh), want[i % 3][0]), i
        del fresh
    assert len(at) < 6 and _lib.device_status() == 0


# ---------------------------------------------------------------------------
# a run of the operators together, captured and replayed
# ---------------------------------------------------------------------------
def _capture(fn):
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        fn()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = fn()
    return graph, out


@pytest.mark.parametrize("m", [1, 3, 12])
def test_dense_block_together_and_captured(m):
    """norm -> gated products -> down product -> norm, as one decoding step runs a block."""
    from nvfp4_b200 import norm
    hidden, inner = 768, 1152
    w1, d1 = make_weights(inner, hidden, seed=1)
    w2, d2 = make_weights(inner, hidden, seed=2)
    w3, d3 = make_weights(hidden, inner, seed=3)
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, hidden, generator=g).bfloat16().cuda()
    residual = torch.randn(m, hidden, generator=g).bfloat16().cuda()
    gain = (1 + 0.1 * torch.randn(hidden, generator=g)).bfloat16().cuda()

    def block():
        y, h = norm.rms_norm(x, gain, residual)
        mid = V.dual_gemv(y, w1, w2)
        down = V.gemv(mid, w3)
        return (y, h, mid, down) + norm.rms_norm(down, gain, h)

    graph, out = _capture(block)
    for seed in (5, 6):
        gg = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(m, hidden, generator=gg).bfloat16())
        residual.copy_(torch.randn(m, hidden, generator=gg).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, block()):
            assert torch.equal(a, b)
        y, h, mid, down, last, h2 = out
        check(mid, *gate(*products(y, d1[0]), *products(y, d2[0])))
        check(down, *products(mid, d3[0]))
        assert torch.equal(h2, (down.float() + h.float()).bfloat16())
    del graph


@pytest.mark.parametrize("t,topk", [(1, 4), (9, 6)])
def test_expert_block_together_and_captured(t, topk):
    """norm -> experts' gated products -> experts' down products -> weighted sum."""
    from nvfp4_b200 import norm
    hidden, inner, e = 512, 640, 16
    w1, _ = make_experts(e, inner, hidden, seed=10)
    w2, _ = make_experts(e, inner, hidden, seed=40)
    w3, d3 = make_experts(e, hidden, inner, seed=70)
    g = torch.Generator().manual_seed(t)
    x = torch.randn(t, hidden, generator=g).bfloat16().cuda()
    gain = torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    ids = torch.randint(0, e, (t, topk), generator=g, dtype=torch.int32).cuda()
    share = torch.rand(t, topk, generator=g).cuda()
    order = moe.pair_order(t, topk, "cuda")

    def block():
        y, _ = norm.rms_norm(x, gain)
        mid = moe.dual_gemv(y, ids, w1, w2)
        down = moe.gemv(mid, ids, w3, out_dtype=torch.float16)
        return mid, down, moe.combine(down, order, share)

    graph, out = _capture(block)
    for seed in (5, 6):
        gg = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(t, hidden, generator=gg).bfloat16())
        ids.copy_(torch.randint(0, e, (t, topk), generator=gg, dtype=torch.int32))
        share.copy_(torch.rand(t, topk, generator=gg))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, block()):
            assert torch.equal(a, b)
        mid, down, total = out
        flat = ids.reshape(-1).tolist()
        for p, ex in enumerate(flat):
            check(down[p:p + 1], *products(mid[p:p + 1], d3[ex]))
        want = O.moe_combine(down.cpu().numpy(), np.arange(t * topk, dtype=np.int32), share.cpu().numpy(), t, topk)
        assert np.array_equal(total.cpu().numpy(), want)
    del graph


FIRST_CALLS = """
import sys
import torch
from nvfp4_b200 import _lib, gemv, norm
g = torch.Generator().manual_seed(0)
b = torch.randint(0, 256, (300, 320), generator=g, dtype=torch.uint8).cuda()
sf = torch.randint(0x20, 0x40, (3, 10, 32, 4, 4), generator=g, dtype=torch.uint8).cuda()
w = gemv.Weights(b, sf)
gain = torch.ones(640, dtype=torch.bfloat16, device="cuda")
xs = [torch.randn(m, 640, generator=g).bfloat16().cuda() for m in (1, 9)]
torch.cuda.synchronize()
s = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.cuda.stream(s):
    with torch.cuda.graph(graph, stream=s):
        out = [gemv.dual_gemv(norm.rms_norm(x, gain)[0], w, w) for x in xs]
    graph.replay()
torch.cuda.synchronize()
for x, y in zip(xs, out):
    assert torch.equal(y, gemv.dual_gemv(norm.rms_norm(x, gain)[0], w, w)) and bool(y.any())
assert _lib.device_status() == 0
"""


def test_first_calls_of_a_process_inside_a_capture():
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": str(Path(V.__file__).resolve().parents[1])})
    assert r.returncode == 0, r.stderr[-2000:]


def test_expert_table_is_not_made_inside_a_capture():
    w, _ = make_experts(2, 64, 128, seed=1)
    x = torch.randn(1, 128, device="cuda").half()
    ids = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=s):
                moe.gemv(x, ids, w)
    torch.cuda.synchronize()
    assert moe.gemv(x, ids, w).shape == (1, 64)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_gemv_refuses():
    w, _ = make_weights(64, 128, seed=1)
    w2, _ = make_weights(72, 128, seed=1)
    x = torch.randn(2, 128, device="cuda").half()
    for bad in (x.double(), x[:, :64], x.cpu(), x[0], x[None].expand(2, 2, 128)):
        with pytest.raises(ValueError):
            V.gemv(bad, w)
    for out in (torch.empty(2, 63, device="cuda").half(), torch.empty(2, 64), torch.empty(64, 2, device="cuda").half().T,
                torch.empty(2, 64, device="cuda", dtype=torch.int32), torch.empty(1, 64, device="cuda").half().expand(2, 64)):
        with pytest.raises(ValueError):
            V.gemv(x, w, out=out)
    with pytest.raises(ValueError):
        V.gemv(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        V.dual_gemv(x, w, w2)
    with pytest.raises(_lib.Nvfp4Error):
        V.gemv(torch.zeros(4097, 128, device="cuda").half(), w)
    for b, sf in ((w.b.cpu(), w.sfb_perm), (w.b[:, :31], w.sfb_perm), (w.b, w.sfb_perm.view(torch.uint8)[..., :1, :]),
                  (w.b.view(torch.uint8).float(), w.sfb_perm)):
        with pytest.raises(ValueError):
            V.Weights(b, sf)


def test_moe_gemv_refuses():
    w, _ = make_experts(3, 64, 128, seed=1)
    other, _ = make_experts(2, 64, 128, seed=1)
    x = torch.randn(4, 128, device="cuda").half()
    ids = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    for bx, bi in ((x.double(), ids), (x, ids.long()), (x[:3], ids), (x, ids.cpu()), (x[:, :64], ids)):
        with pytest.raises(ValueError):
            moe.gemv(bx, bi, w)
    with pytest.raises(ValueError):
        moe.dual_gemv(x, ids, w, other)
    with pytest.raises(_lib.Nvfp4Error, match="at most 256"):
        moe.gemv(torch.zeros(129, 128, device="cuda").half(), torch.zeros(129, 2, dtype=torch.int32, device="cuda"), w)


def test_expert_weights_refuse_other_types_and_plain_scales():
    packed, atoms, _ = raw_weights(128, 128, seed=1)
    b, sf = packed[0], atoms[0]
    moe.ExpertWeights([(b, sf), (b.view(torch.float4_e2m1fn_x2).unsqueeze(-1), sf.view(-1))])
    for bad in ((b.half(), sf), (b, sf.float()), (b, sf.reshape(128, 8)), (b, sf.reshape(128, 8, 1))):
        with pytest.raises(ValueError):
            moe.ExpertWeights([(b, sf), bad])


def test_rows_past_32_bits_are_refused():
    """Counts of rows that a C int would cut off."""
    from nvfp4_b200 import norm
    packed, atoms, _ = raw_weights(1, 64, seed=1)
    many = torch.zeros(1, 64, device="cuda").half().expand(2 ** 32 + 1, 64)
    with pytest.raises(ValueError, match="rows"):
        V.gemv(many, V.Weights(packed[0], atoms[0]))
    ids = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(2 ** 32 + 1, 1)
    with pytest.raises(ValueError, match="rows"):
        moe.gemv(many, ids, moe.ExpertWeights([(packed[0], atoms[0])]))
    gain = torch.ones(64, device="cuda")
    for f in (norm.rms_norm, norm.rms_norm_fp8, norm.rms_norm_nvfp4):
        with pytest.raises(ValueError, match="rows"):
            f(many, gain, **({"group": None} if f is norm.rms_norm_fp8 else {}))
