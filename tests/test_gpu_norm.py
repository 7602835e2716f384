"""GPU: residual addition, RMS norm and quantised output.

h is the fp32 sum rounded once, compared bit for bit.  y in 64 bits from h; the
kernel rounds r, h * r and the product with the weight to fp32 (3 * 2^-24 |y|, and the root's own
2^-53), then to the output.  fp8: the scale is amax/448, one more rounding of an amax
that is off by 3 * 2^-24; the codes are the nearest ones (see there).  NVFP4: bit for bit what the quantiser makes of the same fp32 y."""
import numpy as np
import pytest
import torch

from nvfp4_b200 import _lib
from nvfp4_b200 import build as B
from nvfp4_b200 import norm
from nvfp4_b200.formats import quantize_nvfp4, swizzle_sf
from nvfp4_b200.quantize import quantize

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _ready(cuda_device):
    B.build()
    _lib.load()


def make(rows, k, x, r, w, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed + rows + k)
    return ((torch.randn(rows, k, generator=g) * scale).to(TYPES[x]),
            None if r is None else (3 * torch.randn(rows, k, generator=g)).to(TYPES[r]),
            (1 + 0.3 * torch.randn(k, generator=g)).to(TYPES[w]))


def stream(x, residual):
    return x if residual is None else (x.float() + residual.float()).to(residual.dtype)


def y64(h, w, eps):
    h = h.double()
    return h * (h.square().mean(1, keepdim=True) + eps).rsqrt() * w.double()


def y32(h, w, eps):
    """The kernel's fp32 y: the root in 64 bits, then one rounding after another."""
    r = (h.double().square().mean(1, keepdim=True) + eps).rsqrt().float()
    return h.float() * r * w.float()


MIXES = [("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp16"), ("fp32", "fp32", "fp32"), ("fp32", "bf16", "bf16"),
         ("bf16", None, "fp32"), ("fp16", "fp32", "bf16"), ("bf16", "fp16", "fp16")]
SHAPES = [(1, 7168), (1, 1), (3, 7), (5, 64), (2, 1001), (130, 256), (7, 16384), (2, 20000), (1, 32768), (700, 4096),
          (301, 5000)]


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_rms_norm(rows, k, mix):
    x, residual, w = make(rows, k, *mix)
    args = (x.cuda(), w.cuda(), None if residual is None else residual.cuda())
    h = stream(x, residual)
    want = y64(h, w, 1e-5)
    for out in (None, torch.float32):
        y, hg = norm.rms_norm(*args, eps=1e-5, out_dtype=out)
        assert y.dtype == (out or x.dtype)
        assert torch.equal(hg.cpu(), h)
        t = torch.finfo(y.dtype)
        tol = want.abs() * (3 * 2.0 ** -24 * 1.001 + t.eps / 2 * 1.001) + t.smallest_normal * t.eps / 2
        assert bool(((y.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("rows,k,group", [(1, 7168, 128), (1, 1001, None), (33, 256, 32), (5, 4096, 64), (3, 20480, None),
                                          (600, 4096, 128), (2, 128, 128), (4, 2, None)])
def test_rms_norm_fp8(rows, k, group, mix):
    x, residual, w = make(rows, k, *mix, seed=1)
    h = stream(x, residual)
    (q, scales), hg = norm.rms_norm_fp8(x.cuda(), w.cuda(), None if residual is None else residual.cuda(), group=group)
    assert torch.equal(hg.cpu(), h)
    want = y64(h, w, 1e-6).view(rows, -1, group or k)
    s64 = want.abs().amax(2) / 448
    s = scales.cpu().double()
    assert bool(((s - s64).abs() <= 5 * 2.0 ** -24 * s64).all())
    code = q.cpu().float().double().view(rows, -1, group or k)
    assert bool((code.abs().amax(2) == 448).all())           # the group's largest is the largest code
    t = want / s64.unsqueeze(2)
    # Every code is the nearest one to the 64-bit quotient but where that lies within fp32's roundings
    # of a border: h * weight and its largest (for fp32 inputs), 448 / largest and the product round once
    # each, 4 * 2^-24 |t| together; this test's own fp32 t rounds once more.  The codes of both ends then
    # enclose the kernel's.
    ends = [(t * (1 + d * 5.1 * 2.0 ** -24)).float().to(torch.float8_e4m3fn).double() for d in (-1, 1)]
    assert bool(((torch.minimum(*ends) <= code) & (code <= torch.maximum(*ends))).all())


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("rows,k", [(1, 7168), (1, 64), (127, 128), (128, 320), (129, 4096), (300, 1024), (385, 2048), (2, 16448)])
def test_rms_norm_nvfp4_is_the_quantiser_of_the_normed_values(rows, k, mix):
    x, residual, w = make(rows, k, *mix, seed=2)
    h = stream(x, residual)
    (packed, sf, sf_perm), hg = norm.rms_norm_nvfp4(x.cuda(), w.cuda(), None if residual is None else residual.cuda())
    assert torch.equal(hg.cpu(), h)
    y = y32(h, w, 1e-6)
    p, s = quantize_nvfp4(y)
    assert torch.equal(packed.view(torch.uint8)[:, :, 0].cpu(), p)
    assert torch.equal(sf.view(torch.uint8)[:, :, 0].cpu(), s)
    mem = lambda t: t.view(torch.uint8).permute(5, 2, 4, 0, 1, 3).contiguous().cpu()   # noqa: E731
    assert torch.equal(mem(sf_perm), mem(swizzle_sf(s.unsqueeze(-1))))
    # the same tensors as the quantiser's, shapes and strides too
    for a, b in zip((packed, sf, sf_perm), quantize(y.cuda())):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        assert all(p == q for p, q, n in zip(a.stride(), b.stride(), a.shape) if n > 1)


def test_rms_norm_in_place_strided_and_unaligned():
    rows, k = 40, 1024
    g = torch.Generator().manual_seed(1)
    big = torch.randn(rows, k + 40, generator=g).bfloat16().cuda()
    w = torch.rand(k + 3, generator=g).bfloat16().cuda()
    for off in (0, 8, 3):
        x, residual = big[:, off:off + k], big[:, 16 + off:16 + off + k].clone()
        gain = w[:k] if off != 3 else w[3:]
        want_h = (x.float() + residual.float()).bfloat16()
        ref, _ = norm.rms_norm(x.contiguous(), gain.clone(), residual)
        buf = torch.zeros(rows, k + 8, dtype=torch.bfloat16, device="cuda")
        out = buf[:, off % 8:off % 8 + k]
        y, h = norm.rms_norm(x, gain, residual, out=out, residual_out=residual)
        assert y is out and h is residual
        assert torch.equal(h, want_h) and torch.equal(y, ref)
        assert not bool(buf[:, k + off % 8:].any())
    y, _ = norm.rms_norm(big[:, :k].T.contiguous().T, w[:k])
    assert torch.equal(y, norm.rms_norm(big[:, :k].contiguous(), w[:k])[0])
    x = torch.randn(rows, k, generator=g).half().cuda()
    for f in (norm.rms_norm_fp8, norm.rms_norm_nvfp4):
        first, _ = f(x, w[:k])
        again, _ = f(x, w[:k], out=first)
        assert all(a.data_ptr() == b.data_ptr() for a, b in zip(first, again))


def test_rms_norm_onto_its_input():
    x = torch.randn(20, 3000, generator=torch.Generator().manual_seed(3)).half().cuda()
    w = torch.rand(3000, generator=torch.Generator().manual_seed(4)).half().cuda()
    want, _ = norm.rms_norm(x, w)
    y, h = norm.rms_norm(x, w, out=x)
    assert y is x and h is x and torch.equal(x, want)


def test_rms_norm_past_32_bit_offsets():
    rows, k = 66000, 32768
    x = torch.empty(rows, k, dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1))
    w = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    (q, s), _ = norm.rms_norm_fp8(x, w)
    (packed, sf, _), _ = norm.rms_norm_nvfp4(x, w)
    for part in (slice(0, 2), slice(rows - 2, rows)):
        (q2, s2), _ = norm.rms_norm_fp8(x[part].clone(), w)
        (packed2, sf2, _), _ = norm.rms_norm_nvfp4(x[part].clone(), w)
        for a, b in ((q[part], q2), (s[part], s2), (packed[part], packed2), (sf[part], sf2)):
            assert torch.equal(a.view(torch.uint8).cpu(), b.view(torch.uint8).cpu())


def test_rms_norm_special_rows():
    """Zero rows, tiny and huge ones, infinities and NaN, and a gain that is not finite."""
    k = 256
    x = torch.randn(9, k, generator=torch.Generator().manual_seed(4))
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e30
    x[3, 5] = float("inf")
    x[4, 6] = float("nan")
    x[5, 16:32] = 0
    x[6] = torch.finfo(torch.float32).max
    x[7] = 0
    x[7, 200] = 1e-38
    w = torch.ones(k)
    want = y64(x, w, 1e-6)
    y, _ = norm.rms_norm(x.cuda(), w.cuda())
    y = y.cpu().double()
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    fin = ~torch.isnan(want)
    assert bool(((y[fin] - want[fin]).abs() <= 4 * 2.0 ** -24 * want[fin].abs() + 2.0 ** -149).all())
    (q, s), _ = norm.rms_norm_fp8(x.cuda(), w.cuda(), group=32)
    assert not bool(s[0].any()) and not bool(q.float()[0].any())
    assert bool(torch.isnan(s[4]).all()) and bool(torch.isnan(q.float()[4]).all())
    assert bool(torch.isnan(s[3, 0])) and not bool(torch.isnan(s[3, 1:]).any())
    (packed, sf, _), _ = norm.rms_norm_nvfp4(x.cuda(), w.cuda())
    sf = sf.float()[:, :, 0]
    packed = packed.view(torch.uint8)[:, :, 0]
    assert not bool(sf[0].any()) and not bool(packed[0].any())
    assert bool(torch.isnan(sf[4]).all()) and bool(torch.isnan(sf[3, 0])) and not bool(torch.isnan(sf[3, 1:]).any())
    assert not bool(sf[5, 1]) and not bool(packed[5, 8:16].any())
    w[40] = float("nan")
    w[80] = float("inf")
    (_, sf, _), _ = norm.rms_norm_nvfp4(x[8:].cuda(), w.cuda())
    nan = torch.isnan(sf.float()[0, :, 0])
    assert bool(nan[2]) and int(nan.sum()) == 1              # the infinite gain saturates its scale
    assert _lib.device_status() == 0


def test_rms_norm_nvfp4_feeds_the_dual_gemm():
    """The prompt's side: normed and quantised in one pass, then the GEMM, as from the quantiser."""
    from nvfp4_b200 import dual_gemm
    m, n, k = 200, 256, 512
    g = torch.Generator().manual_seed(8)
    x, w = torch.randn(m, k, generator=g).bfloat16(), (1 + 0.1 * torch.randn(k, generator=g)).bfloat16()
    b1, _, s1 = quantize(torch.randn(n, k, generator=g).cuda())
    b2, _, s2 = quantize(torch.randn(n, k, generator=g).cuda())
    (packed, _, sf_perm), _ = norm.rms_norm_nvfp4(x.cuda(), w.cuda())
    c = torch.empty(1, m, n, dtype=torch.float16, device="cuda").permute(1, 2, 0)
    got = dual_gemm.dual_gemm(packed, b1, b2, sf_perm, s1, s2, c).clone()
    a, _, sa = quantize(y32(x, w, 1e-6).cuda())
    assert torch.equal(got, dual_gemm.dual_gemm(a, b1, b2, sa, s1, s2, c))
    assert _lib.device_status() == 0


def test_rms_norm_captured():
    x = torch.randn(5, 2048, device="cuda").bfloat16()
    residual = torch.randn(5, 2048, device="cuda").bfloat16()
    w = torch.rand(2048, device="cuda").bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm.rms_norm_fp8(x, w, residual)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = norm.rms_norm_fp8(x, w, residual), norm.rms_norm_nvfp4(x, w, residual), norm.rms_norm(x, w, residual)
    x.copy_(torch.randn(5, 2048).bfloat16())
    graph.replay()
    torch.cuda.synchronize()
    again = norm.rms_norm_fp8(x, w, residual), norm.rms_norm_nvfp4(x, w, residual), norm.rms_norm(x, w, residual)
    flat = lambda v: [t.view(torch.uint8) for p in v for q in (p if isinstance(p, tuple) else (p,))   # noqa: E731
                      for t in (q if isinstance(q, tuple) else (q,))]
    for a, b in zip(flat(out), flat(again)):
        assert torch.equal(a, b)
    del graph


def test_rms_norm_no_rows_and_refusals():
    w = torch.ones(128, device="cuda")
    x = torch.randn(2, 128, device="cuda")
    y, _ = norm.rms_norm(x[:0], w)
    assert y.shape == (0, 128)
    (q, s), _ = norm.rms_norm_fp8(x[:0], w)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    for args in ((x.double(), w), (x[0], w), (x, w[:64]), (x, w, x[:1]), (x, w, x.long()), (x, w.cpu())):
        with pytest.raises(ValueError):
            norm.rms_norm(*args)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, residual_out=x)
    with pytest.raises(ValueError):
        norm.rms_norm(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        norm.rms_norm_fp8(x, w, group=48)
    with pytest.raises(ValueError):
        norm.rms_norm_fp8(x[:, :96], w[:96], group=64)
    with pytest.raises(ValueError):
        norm.rms_norm_nvfp4(x[:, :100], w[:100])
    with pytest.raises(ValueError):
        norm.rms_norm_fp8(x, w, out=(torch.empty(2, 128, device="cuda"), torch.empty(2, 1, device="cuda")))
    with pytest.raises(_lib.Nvfp4Error, match="negative"):
        norm.rms_norm(x, w, eps=-1.0)
    with pytest.raises(_lib.Nvfp4Error, match="32768"):
        norm.rms_norm(torch.zeros(1, 32776, device="cuda"), torch.zeros(32776, device="cuda"))


def test_rms_norm_without_a_residual_returns_x_itself():
    """Also where the kernel reads a copy of it: what is returned is the stream that the next block adds to."""
    w = torch.ones(96, device="cuda")
    for x in (torch.randn(5, 96, device="cuda"), torch.randn(96, 5, device="cuda").T, torch.randn(5, 192, device="cuda")[:, ::2]):
        want = norm.rms_norm(x.contiguous(), w)[0]
        y, h = norm.rms_norm(x, w)
        assert h is x and torch.equal(y, want)
        assert norm.rms_norm_fp8(x, w, group=32)[1] is x
    x = torch.randn(64, 5, device="cuda").T
    assert norm.rms_norm_nvfp4(x, w[:64])[1] is x
