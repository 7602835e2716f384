"""CPU: the norm's and the products' entry points reject bad arguments before
touching a GPU, and their Python sides bad tensors."""
import ctypes

import pytest
import torch

from nvfp4_b200 import _lib
from nvfp4_b200 import build as B
from nvfp4_b200 import gemv, moe, norm

P, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4096 + 8)   # never dereferenced
F32, F16, BF16 = _lib.NVFP4_F32, _lib.NVFP4_F16, _lib.NVFP4_BF16
INVALID, SHAPE, ALIGNMENT = _lib.NVFP4_ERR_INVALID_ARG, _lib.NVFP4_ERR_SHAPE, _lib.NVFP4_ERR_ALIGNMENT


@pytest.fixture(scope="module")
def lib():
    B.build()
    return _lib.load()


def _gemv(lib, **k):
    a = dict(x=P, xt=F16, ldx=256, xb=0, b1=P, s1=P, b2=None, s2=None, out=P, ot=F16, ldo=128, ob=0, m=1, n=128, k=256,
             l=1, ws=P, size=1 << 30)
    a.update(k)
    return lib.nvfp4_gemv(a["x"], a["xt"], a["ldx"], a["xb"], a["b1"], a["s1"], a["b2"], a["s2"], a["out"], a["ot"],
                          a["ldo"], a["ob"], a["m"], a["n"], a["k"], a["l"], a["ws"], a["size"], None)


@pytest.mark.parametrize("change,status", [
    (dict(x=None), INVALID), (dict(b1=None), INVALID), (dict(s1=None), INVALID), (dict(out=None), INVALID),
    (dict(b2=P), INVALID), (dict(s2=P), INVALID), (dict(m=-1), INVALID), (dict(n=0), INVALID), (dict(k=0), INVALID),
    (dict(l=0), INVALID), (dict(xt=7), INVALID), (dict(ot=-1), INVALID), (dict(ldo=100), INVALID), (dict(ldx=-1), INVALID),
    (dict(k=96, ldx=96), SHAPE), (dict(m=5000), SHAPE), (dict(l=5000), SHAPE), (dict(k=1 << 21, ldx=1 << 21), SHAPE),
    (dict(m=4096, n=1 << 29, ldo=1 << 29), SHAPE), (dict(m=4096, l=4096, k=1 << 20), SHAPE),
    (dict(b1=ODD), ALIGNMENT), (dict(s1=ODD), ALIGNMENT), (dict(b2=ODD, s2=P), ALIGNMENT),
    (dict(x=ctypes.c_void_p(4097)), ALIGNMENT), (dict(out=ctypes.c_void_p(4098), ot=F32), ALIGNMENT)])
def test_gemv_rejects_without_gpu(lib, change, status):
    assert _gemv(lib, **change) == status
    assert lib.nvfp4_last_error()


def test_gemv_no_rows_and_workspace_sizes(lib):
    assert _gemv(lib, m=0, x=None) == _lib.NVFP4_OK
    small, large = (lib.nvfp4_gemv_workspace_bytes(F32, 0, m, 128, 4096, 1) for m in (16, 64))
    assert 0 < small < large
    assert lib.nvfp4_gemv_workspace_bytes(F16, 1, 0, 128, 256, 1) == 0
    assert lib.nvfp4_moe_gemv_workspace_bytes(F16, 1, 4, 8, 1024) == 0          # expanded by the kernel itself
    assert lib.nvfp4_moe_gemv_workspace_bytes(F16, 0, 4, 8, 1024) > 0
    assert lib.nvfp4_moe_gemv_workspace_bytes(F16, 1, 5, 8, 1024) > 0
    assert lib.nvfp4_moe_gemv_workspace_bytes(F16, 1, 1000, 8, 1024) == 0       # refused by the call


@pytest.mark.parametrize("change,status", [
    (dict(x=None), INVALID), (dict(ids=None), INVALID), (dict(t1=None), INVALID), (dict(out=None), INVALID),
    (dict(tokens=-1), INVALID), (dict(topk=0), INVALID), (dict(e=0), INVALID), (dict(n=0), INVALID),
    (dict(tokens=65, topk=4), SHAPE), (dict(e=1025), SHAPE), (dict(k=100), SHAPE), (dict(xt=3), INVALID),
    (dict(t1=ctypes.c_void_p(4096 + 16)), ALIGNMENT), (dict(tokens=9, ws=None, size=0), INVALID),
    (dict(tokens=9, size=64), INVALID), (dict(tokens=9, ws=ODD), ALIGNMENT)])
def test_moe_gemv_rejects_without_gpu(lib, change, status):
    a = dict(x=P, xt=F16, ldx=256, per=0, ids=P, tokens=1, topk=4, t1=P, t2=None, e=8, out=P, ot=F16, ldo=128, n=128, k=256,
             ws=P, size=1 << 30)
    a.update(change)
    assert lib.nvfp4_moe_gemv(a["x"], a["xt"], a["ldx"], a["per"], a["ids"], a["tokens"], a["topk"], a["t1"], a["t2"], a["e"],
                              a["out"], a["ot"], a["ldo"], a["n"], a["k"], a["ws"], a["size"], None) == status


def test_moe_table_rejects_without_gpu(lib):
    one = (ctypes.c_void_p * 1)(4096)
    odd = (ctypes.c_void_p * 1)(4100)
    none = (ctypes.c_void_p * 1)(None)
    buf = (ctypes.c_char * int(lib.nvfp4_moe_table_bytes(1)))()
    assert lib.nvfp4_moe_table_bytes(0) == 0 and lib.nvfp4_moe_table_bytes(3) == 3 * len(buf)
    assert lib.nvfp4_moe_table(one, one, 0, 128, 256, buf) == INVALID
    assert lib.nvfp4_moe_table(one, one, 1, 128, 256, None) == INVALID
    assert lib.nvfp4_moe_table(none, one, 1, 128, 256, buf) == INVALID
    assert lib.nvfp4_moe_table(one, odd, 1, 128, 256, buf) == ALIGNMENT
    assert lib.nvfp4_moe_table(one, one, 1, 128, 100, buf) == SHAPE


@pytest.mark.parametrize("change,status", [
    (dict(x=None), INVALID), (dict(w=None), INVALID), (dict(y=None), INVALID), (dict(h=None), INVALID),
    (dict(rows=-1), INVALID), (dict(k=0), INVALID), (dict(fmt=5), INVALID), (dict(xt=9), INVALID), (dict(eps=-1.0), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(k=40000, ldh=40000), SHAPE), (dict(fmt=1, scales=None), INVALID),
    (dict(fmt=1, group=48), SHAPE), (dict(fmt=1, group=128, k=192), SHAPE), (dict(fmt=2, k=100), SHAPE),
    (dict(fmt=2, sf=None), INVALID), (dict(fmt=2, y=ODD), ALIGNMENT), (dict(ldh=10), INVALID), (dict(fmt=0, ldy=10), INVALID),
    (dict(x=ctypes.c_void_p(4097)), ALIGNMENT), (dict(fmt=1, scales=ctypes.c_void_p(4098)), ALIGNMENT)])
def test_rms_norm_rejects_without_gpu(lib, change, status):
    a = dict(x=P, xt=BF16, ldx=256, r=P, rt=BF16, ldr=256, h=P, ldh=256, w=P, wt=BF16, eps=1e-6, rows=4, k=256, fmt=0, y=P,
             yt=BF16, ldy=256, scales=P, group=128, sf=P, sfp=None)
    a.update(change)
    assert lib.nvfp4_rms_norm(a["x"], a["xt"], a["ldx"], a["r"], a["rt"], a["ldr"], a["h"], a["ldh"], a["w"], a["wt"], a["eps"],
                              a["rows"], a["k"], a["fmt"], a["y"], a["yt"], a["ldy"], a["scales"], a["group"], a["sf"],
                              a["sfp"], None) == status
    assert a["rows"] == 0 or lib.nvfp4_last_error()


def test_python_sides_refuse_host_tensors():
    b, sf = torch.zeros(128, 128, dtype=torch.uint8), torch.zeros(1, 4, 32, 4, 4, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        gemv.Weights(b, sf)
    with pytest.raises(ValueError, match="CUDA"):
        norm.rms_norm(torch.zeros(2, 64), torch.zeros(64))
    with pytest.raises(ValueError):
        moe.ExpertWeights([(b, sf)])
    order = moe.pair_order(3, 2, "cpu")
    assert order.dst.tolist() == list(range(6)) and (order.tokens, order.topk) == (3, 2)


def test_digits_of_x_stay_within_their_bound():
    """The arithmetic of the products' digits on the host: eight balanced base-8 digits in
    halves are e2m1 values of at most 2 in magnitude and give back x to 2^-23 of the scale."""
    import numpy as np
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-1.5, 1.5, 100000), [1.5, -1.5, 0.0, 2.0 ** -24, -(2.0 ** -23)]])   # in units of s
    units = np.rint(x * 2.0 ** 22).astype(np.int64)
    fields = units + 0x924924
    assert (fields >= 0).all() and (fields < 1 << 24).all()
    digits = np.stack([((fields >> (3 * (7 - j))) & 7) - 4 for j in range(8)])
    assert digits.min() >= -4 and digits.max() <= 3
    back = sum(d / 2 * 8.0 ** -j for j, d in enumerate(digits))
    assert np.abs(back - x).max() <= 2.0 ** -23


def test_combine_refuses_an_order_out_or_rows_on_the_host():
    """Addresses of host memory never reach a kernel."""
    rows = torch.zeros(6, 64, dtype=torch.float16, device="meta")     # stands for another device
    with pytest.raises(ValueError, match="CUDA"):
        moe.combine(torch.zeros(6, 64, dtype=torch.float16), moe.pair_order(3, 2, "cpu"))
    with pytest.raises(ValueError, match="order"):
        moe.combine(rows, moe.pair_order(3, 2, "cpu"))
    for dst in (torch.zeros(6, dtype=torch.int64, device="meta"), torch.zeros(5, dtype=torch.int32, device="meta"),
                torch.zeros(12, dtype=torch.int32, device="meta")[::2]):
        with pytest.raises(ValueError, match="order"):
            moe.combine(rows, moe.PairOrder(dst, 3, 2))
    with pytest.raises(ValueError, match="out"):
        moe.combine(rows, moe.pair_order(3, 2, "meta"), out=torch.zeros(3, 64))


def test_scales_of_32_matrices_of_four_row_blocks_are_their_memory():
    """[32, 4, K/64, 32, 4, 4], contiguous, is the memory of 32 matrices and not the permuted view of one."""
    t = torch.zeros(32, 4, 2, 32, 4, 4, dtype=torch.uint8)
    gemv.check_scales("sf", t, 512, 128, 32, t.device)
    gemv.check_scales("sf", t.view(torch.float8_e4m3fn), 400, 128, 32, t.device)
    view = t.permute(3, 4, 1, 5, 2, 0)                       # the permuted view of the same
    gemv.check_scales("sf", view, 512, 128, 32, t.device)
    one = torch.zeros(4, 2, 32, 4, 4, dtype=torch.uint8)
    gemv.check_scales("sf", one, 512, 128, 1, t.device)
    for bad, n, k, l in ((t, 512, 128, 31), (t, 640, 128, 32), (t, 512, 192, 32), (view.contiguous(), 512, 128, 32),
                         (t.float(), 512, 128, 32), (one, 512, 128, 2), (one.transpose(0, 1), 256, 256, 1),
                         (t.to("meta"), 512, 128, 32)):
        with pytest.raises(ValueError):
            gemv.check_scales("sf", bad, n, k, l, t.device)


def test_experts_scales_are_checked_for_type_and_layout():
    n, k = 256, 128
    memory = torch.zeros(2, 2, 32, 4, 4, dtype=torch.uint8)
    view = memory.view(1, 2, 2, 32, 4, 4).permute(3, 4, 1, 5, 2, 0)
    dev = memory.device
    for good in (memory, memory.view(-1), memory.view(1, 2, 2, 32, 4, 4), memory.view(torch.float8_e4m3fn), view, view[..., 0],
                 memory.view(4, 512), memory.view(torch.int8)):
        moe._check_expert_scales("sf", good, n, k, dev)
    plain = torch.zeros(n, k // 16, dtype=torch.uint8)       # as many bytes, in another order
    for bad in (plain, plain.unsqueeze(-1), plain.view(torch.float8_e4m3fn), plain[None], view.contiguous(), memory.float(),
                memory.half(), memory.transpose(0, 1), memory[:1], memory.to("meta")):
        with pytest.raises(ValueError):
            moe._check_expert_scales("sf", bad, n, k, dev)


def test_grouped_gemm_refuses_weights_on_another_device():
    class Elsewhere:
        n, k, device = 128, 64, torch.device("cpu")

        def __len__(self):
            return 2

    i32 = torch.zeros(3, dtype=torch.int32, device="meta")
    d = moe.Dispatch(torch.zeros(4, 32, dtype=torch.uint8, device="meta"), i32, i32, i32, i32, i32, i32, i32, 4, 1, 64, 2)
    with pytest.raises(ValueError, match="weights are on"):
        moe.grouped_gemm(d, Elsewhere(), torch.zeros(4, 128, dtype=torch.float16, device="meta"))


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 128, 2 ** 31 - 2 ** 20])
def test_widths_next_to_32_bits_are_refused(lib, n):
    """The kernels count columns in 32 bits, in steps of up to 2^20."""
    assert _gemv(lib, n=n, ldo=n, k=64, ldx=64) == SHAPE
    one = ctypes.c_void_p(4096)
    assert lib.nvfp4_moe_gemv(one, F16, 64, 0, one, 1, 1, one, None, 8, one, F16, n, n, 64, one, 1 << 30, None) == SHAPE


def test_bound_of_one_elements_digits_tells_seven_digits_from_eight():
    """The bound that the GPU test of single elements uses, on the host: kept by eight digits, broken without the last."""
    import numpy as np
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(4000) * 2.0 ** rng.integers(-12, 12, 4000)).astype(np.float32).astype(np.float64)
    s = 2.0 ** np.ceil(np.log2(np.abs(x) / 1.5))
    fields = np.rint(x / s * 2.0 ** 22).astype(np.int64) + 0x924924
    digits = [(((fields >> (3 * (7 - j))) & 7) - 4) / 2 for j in range(8)]
    bound = np.abs(x) * (8 / 3 + 3.5) * 2.0 ** -24

    def joined(n):
        v = np.zeros(len(x), np.float32)
        for d in reversed(digits[:n]):
            v = (v.astype(np.float64) / 8 + d).astype(np.float32)     # one rounding, as fmaf
        return v * s
    assert (np.abs(joined(8) - x) <= bound).all()
    assert (np.abs(joined(7) - x) > bound).mean() > 0.2
