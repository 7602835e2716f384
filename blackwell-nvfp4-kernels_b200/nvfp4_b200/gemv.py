"""A few tokens times NVFP4 weights (``nvfp4_gemv`` in libnvfp4_b200.so).

The GEMMs of this package quantise the activations and work on 128-row tiles.
For the one to sixteen tokens of a decoding step these products read the same
weights in the same layout (``quantize.quantize``, ``formats``) once, and take the
activations as they are, fp16, bf16 or fp32, with fp32 sums (each element to 2^-22 of
the largest of its 16 neighbours, see :func:`gemv`):

    w1, w2 = gemv.Weights(b1, sfb1_perm), gemv.Weights(b2, sfb2_perm)
    h = gemv.dual_gemv(x, w1, w2)        # silu(x . W1ᵀ) * (x . W2ᵀ)
    y = gemv.gemv(h, w3)                 # h . W3ᵀ

The per-expert forms are ``moe.gemv`` and ``moe.dual_gemv``.  Counterparts in the
reference: the dual and the grouped GEMM (nvfp4_dual_gemm/reference.py:27-77,
nvfp4_group_gemm/reference.py:39-74), which take quantised activations.
"""
from __future__ import annotations

import torch

from . import _lib
from .dual_gemm import check_sf_perm, current_stream_on, on_device
from .formats import ceil_div

DTYPES = {torch.float32: _lib.NVFP4_F32, torch.float16: _lib.NVFP4_F16,
          torch.bfloat16: _lib.NVFP4_BF16}


def check_scales(name: str, t: torch.Tensor, n: int, k: int, l: int, device) -> None:
    """``t`` must be the permuted scales of L matrices [N, K] or their memory (see :class:`Weights`)."""
    atoms = (ceil_div(n, 128), k // 64, 32, 4, 4)
    shape = tuple(t.shape)
    if shape == (l,) + atoms or (l == 1 and shape == atoms):
        if t.dtype not in (torch.float8_e4m3fn, torch.uint8, torch.int8):
            raise ValueError(f"{name}: expected float8_e4m3fn, got {t.dtype}")
        if not t.is_contiguous() or t.device != device:
            raise ValueError(f"{name} must be contiguous on {device}")
    elif t.dim() == 6 and shape[:2] == (32, 4):
        check_sf_perm(name, t, n, k, l, device)
    else:
        raise ValueError(f"{name}: shape {shape} holds no scales of [{n}, {k}, {l}]")


class Weights:
    """One NVFP4 weight matrix (or L of them), checked once.

    ``b``: float4_e2m1fn_x2 (or uint8) [N, K/2] or [N, K/2, L], K-major, batch
    outermost; ``sfb_perm``: its permuted scales, float8_e4m3fn (or uint8)
    [32, 4, ceil(N/128), 4, K/64, L], or that tensor's memory, contiguous
    [(L,) ceil(N/128), K/64, 32, 4, 4].  K % 64 == 0.  The tensors are kept."""

    def __init__(self, b: torch.Tensor, sfb_perm: torch.Tensor):
        if not b.is_cuda or b.dim() not in (2, 3):
            raise ValueError("b must be a CUDA tensor [N, K/2] or [N, K/2, L]")
        if b.dtype not in (torch.float4_e2m1fn_x2, torch.uint8, torch.int8):
            raise ValueError(f"b: expected float4_e2m1fn_x2, got {b.dtype}")
        n, kh = int(b.shape[0]), int(b.shape[1])
        l = int(b.shape[2]) if b.dim() == 3 else 1
        k = 2 * kh
        if n < 1 or l < 1 or k < 64 or k % 64:
            raise ValueError(f"b: N={n}, L={l} must be positive and K={k} a positive multiple of 64")
        if b.stride(1) != 1 or (n > 1 and b.stride(0) != kh) or (l > 1 and b.stride(2) != n * kh):
            raise ValueError(f"b: strides {b.stride()} are not the K-major [L][{n}][{kh}] layout")
        check_scales("sfb_perm", sfb_perm, n, k, l, b.device)
        self.b, self.sfb_perm = b, sfb_perm
        self.n, self.k, self.l, self.device = n, k, l, b.device
        self.ptrs = (b.data_ptr(), sfb_perm.data_ptr())
        self.space: dict = {}       # workspace bytes by (rows, type and alignment of x)


def _rows_last(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


# the cheapest of torch's allocating calls with a shape of its own
_empty = torch.empty_strided


def _launch(fn, device, args) -> None:
    """fn(*args, stream) on the device's current stream, with the device current."""
    st = current_stream_on(device.index)
    status = fn(*args, st) if st is not None else on_device(device, lambda s: fn(*args, s))
    if status:
        _lib.check(status)


def _run(x, w, w2, out, out_dtype):
    code, dims = DTYPES.get(x.dtype), x.dim()
    if code is None or dims not in (2, 3):
        raise ValueError("x must be float16, bfloat16 or float32 [M, K] or [L, M, K]")
    if x.device != w.device:
        raise ValueError(f"x is on {x.device}, the weights on {w.device}")
    n, k, l, shape = w.n, w.k, w.l, x.shape
    if shape[-1] != k or (shape[0] if dims == 3 else 1) != l:
        raise ValueError(f"x {tuple(shape)} does not match weights of K={k}, L={l}")
    m = shape[-2]
    if m >> 31:
        raise ValueError(f"{m} rows: at most 4096 of a matrix")
    x = _rows_last(x)
    want = (l, m, n) if dims == 3 else (m, n)
    if out is None:
        out = _empty(want, (n, 1) if dims == 2 else (m * n, n, 1), dtype=out_dtype or x.dtype, device=x.device)
        if out.dtype not in DTYPES:
            raise ValueError(f"out_dtype {out_dtype} is none of float16, bfloat16 and float32")
    elif (tuple(out.shape) != want or out.dtype not in DTYPES or out.device != x.device
          or out.dtype != (out_dtype or out.dtype) or (out.stride(-1) != 1 and n > 1)
          or (m > 1 and out.stride(-2) < n)
          or (dims == 3 and l > 1 and out.stride(0) < (m - 1) * out.stride(1) + n)):
        raise ValueError(f"out must be {want}, float16, bfloat16 or float32, rows apart, on {x.device}")
    if m == 0:
        return out
    xs, os_, px, es = x.stride(), out.stride(), x.data_ptr(), x.element_size()
    xb, ob = (xs[0], os_[0]) if dims == 3 else (0, 0)
    lib = _lib.load()
    aligned = not (px | xs[-2] * es | xb * es) & 15
    size = w.space.get((m, code, aligned))
    if size is None:
        with torch.cuda.device(w.device):
            size = lib.nvfp4_gemv_workspace_bytes(code, aligned, m, n, k, l)
        w.space[(m, code, aligned)] = size
    space = _empty((size,), (1,), dtype=torch.uint8, device=x.device) if size else None
    _launch(lib.nvfp4_gemv, x.device, (
        px, code, xs[-2], xb, *w.ptrs, *(w2.ptrs if w2 is not None else (None, None)), out.data_ptr(),
        DTYPES[out.dtype], os_[-2] if os_[-2] > n else n, ob, m, n, k, l,
        space.data_ptr() if size else None, size))
    return out


def gemv(x: torch.Tensor, w: Weights, out: torch.Tensor | None = None,
         out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x . Wᵀ for x [M, K] (or [L, M, K], L matrices): [M, N] (or [L, M, N]) in
    ``out_dtype`` (x's type by default; fp16, bf16 or fp32), one rounding of an
    fp32 sum.  x enters the sums with an error below 2^-22 of the largest of its 16
    consecutive elements (or of 2^-14 of its row's largest, if that is more): no more than
    fp32 sums lose, but for outputs whose weights are zero where x is largest.
    ``out``: written and returned instead of a new tensor; its rows may
    be strided; it must not overlap x or the weights.  Meant for M <= 16; every 16
    further tokens read the weights again (M <= 4096, and L * M * K < 2^31)."""
    return _run(x, w, None, out, out_dtype)


def dual_gemv(x: torch.Tensor, w1: Weights, w2: Weights, out: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """silu(x . W1ᵀ) * (x . W2ᵀ), the gate in fp32; otherwise as :func:`gemv`."""
    if (w1.n, w1.k, w1.l, w1.device) != (w2.n, w2.k, w2.l, w2.device):
        raise ValueError("w1 and w2 must have the same N, K, L and device")
    return _run(x, w1, w2, out, out_dtype)
