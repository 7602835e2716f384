"""Residual addition, root-mean-square norm and quantised output in one pass
(``nvfp4_rms_norm`` in libnvfp4_b200.so): what stands before the projections of a block.

    h = x + residual                     (rounded to the residual's type)
    y = h / sqrt(mean(h^2) + eps) * weight

:func:`rms_norm` returns y in 16 or 32 bits (the input of ``gemv``),
:func:`rms_norm_fp8` in e4m3 with fp32 scales, :func:`rms_norm_nvfp4` in the
layouts of ``quantize.quantize`` (the A operand of the GEMMs).  Each returns
``(y, h)``; h is the residual of the next block, x itself where no residual is given.
The reference takes its operands quantised (nvfp4_dual_gemm/reference.py:113-187)
and has no counterpart.
"""
from __future__ import annotations

import torch

from . import _lib
from .gemv import DTYPES, _launch, _rows_last

_empty, _empty_like = torch.empty_strided, torch.empty_like


def _like(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor of x's shape (empty_like is the cheapest call, for contiguous x)."""
    return _empty_like(x, dtype=dtype) if x.is_contiguous() else _empty(x.shape, (x.shape[1], 1), dtype=dtype, device=x.device)


def _check(x, weight, residual, residual_out):
    """(x, weight, residual, h): checked, rows with unit stride."""
    if x.dim() != 2 or x.dtype not in DTYPES or not x.is_cuda:
        raise ValueError("x must be a CUDA float16, bfloat16 or float32 tensor [rows, K]")
    shape, device = x.shape, x.device
    rows, k = shape
    if weight.shape != (k,) or weight.dtype not in DTYPES or weight.device != device:
        raise ValueError(f"weight must be float16, bfloat16 or float32 [{k}] on {device}")
    if k < 1:
        raise ValueError("K must be positive")
    if rows >> 31:
        raise ValueError(f"{rows} rows: at most 2^31 - 1")
    x = _rows_last(x)
    if weight.stride(0) != 1:
        weight = weight.contiguous()
    if residual is None:
        if residual_out is not None:
            raise ValueError("residual_out without a residual")
        return x, weight, None, None
    if residual.shape != shape or residual.dtype not in DTYPES or residual.device != device:
        raise ValueError(f"residual must be float16, bfloat16 or float32 [{rows}, {k}] on {device}")
    h = residual_out
    if h is None:
        h = _like(residual, residual.dtype)
    elif (h.shape != shape or h.dtype != residual.dtype or h.device != device
          or (h.stride(1) != 1 and k > 1) or (rows > 1 and h.stride(0) < k)):
        raise ValueError(f"residual_out must be {residual.dtype} [{rows}, {k}], rows apart, on {device}")
    return x, weight, _rows_last(residual), h


def _run(x, weight, residual, h, eps, fmt, y, y_dtype=0, ldy=0, scales=None, group=0, sf_perm=None, sf=None):
    rows, k = x.shape
    if residual is None:
        res = (None, 0, 0, None, 0)
    else:
        ldh = h.stride(0)
        res = (residual.data_ptr(), DTYPES[residual.dtype], residual.stride(0), h.data_ptr(),
               ldh if ldh > k else k)
    _launch(_lib.load().nvfp4_rms_norm, x.device, (
        x.data_ptr(), DTYPES[x.dtype], x.stride(0), *res, weight.data_ptr(), DTYPES[weight.dtype], eps, rows, k,
        fmt, y, y_dtype, ldy, scales, group, sf_perm, sf))


def rms_norm(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
             eps: float = 1e-6, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
             residual_out: torch.Tensor | None = None):
    """(y, h) for x [rows, K], K <= 32768; y [rows, K] in ``out_dtype`` (x's type by
    default).  x, weight, residual and y may each be float16, bfloat16 or float32;
    ``residual_out`` may be ``residual`` itself and ``out`` may be ``x`` (then updated
    in place); nothing else may overlap."""
    given = x
    x, weight, residual, h = _check(x, weight, residual, residual_out)
    rows, k = x.shape
    if out is None:
        out = _like(x, out_dtype or x.dtype)
        if out.dtype not in DTYPES:
            raise ValueError(f"out_dtype {out_dtype} is none of float16, bfloat16 and float32")
    elif (tuple(out.shape) != (rows, k) or out.dtype not in DTYPES or out.device != x.device
          or out.dtype != (out_dtype or out.dtype) or (out.stride(1) != 1 and k > 1)
          or (rows > 1 and out.stride(0) < k)):
        raise ValueError(f"out must be [{rows}, {k}], float16, bfloat16 or float32, rows apart, on {x.device}")
    _run(x, weight, residual, h, eps, _lib.NVFP4_NORM_PLAIN, out.data_ptr(), DTYPES[out.dtype],
         max(out.stride(0), k))
    return out, given if h is None else h


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                 eps: float = 1e-6, group: int | None = 128, out=None,
                 residual_out: torch.Tensor | None = None):
    """((q, scales), h): q float8_e4m3fn [rows, K] and scales float32 [rows, K/group]
    with y = q * scale; scale = amax/448 over ``group`` columns (32, 64 or 128,
    dividing K; None: the row), q = e4m3(y / scale) to nearest even, zeros under a
    zero scale; a NaN gives its group a NaN scale.  The quotient is formed from
    h * weight, without the rounding of the root, in two roundings: a code on a border may
    differ from the one that the rounded y and scale give.  ``out``: the (q, scales) of an
    earlier call of the same sizes, reused."""
    given = x
    x, weight, residual, h = _check(x, weight, residual, residual_out)
    rows, k = x.shape
    if group not in (None, 32, 64, 128):
        raise ValueError(f"group {group} is none of 32, 64, 128 or None (the row)")
    if group is not None and k % group:
        raise ValueError(f"K={k} must be a multiple of the group ({group})")
    groups = 1 if group is None else k // group
    if out is None:
        q = _like(x, torch.float8_e4m3fn)
        scales = _empty((rows, groups), (groups, 1), dtype=torch.float32, device=x.device)
    else:
        q, scales = out
        if (tuple(q.shape) != (rows, k) or tuple(scales.shape) != (rows, groups)
                or q.dtype != torch.float8_e4m3fn or scales.dtype != torch.float32
                or any(t.device != x.device or not t.is_contiguous() for t in out)):
            raise ValueError("out does not match: pass the (q, scales) an earlier call returned")
    _run(x, weight, residual, h, eps, _lib.NVFP4_NORM_FP8, q.data_ptr(), scales=scales.data_ptr(),
         group=group or 0)
    return (q, scales), given if h is None else h


def rms_norm_nvfp4(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, *,
                   eps: float = 1e-6, out=None, residual_out: torch.Tensor | None = None):
    """((packed, sf, sf_perm), h): y quantised as ``quantize.quantize`` would
    quantise it, bit for bit, and in the same three tensors (K % 64 == 0);
    a NaN gives its 16 columns a NaN scale.  ``out``: the three tensors of an earlier
    call of the same sizes, reused."""
    given = x
    x, weight, residual, h = _check(x, weight, residual, residual_out)
    rows, k = x.shape
    if k % 64:
        raise ValueError(f"K={k} must be a multiple of 64")
    rb, ka = -(-rows // 128), k // 64
    # shapes and strides of quantize.quantize's tensors: views of [1][rows][K/2], [1][rows][K/16] and
    # [1][rb][ka][32][4][4] bytes
    views = (((rows, k // 2, 1), (k // 2, 1, rows * (k // 2))), ((rows, k // 16, 1), (k // 16, 1, rows * (k // 16))),
             ((32, 4, rb, 4, ka, 1), (16, 4, ka * 512, 1, 512, rb * ka * 512)))
    if out is not None:
        packed, sf, sf_perm = out
        for t, (shape, strides), kind in zip(out, views, (torch.float4_e2m1fn_x2,) + (torch.float8_e4m3fn,) * 2):
            if (tuple(t.shape) != shape or t.dtype != kind or t.device != x.device
                    or any(a != b for a, b, n in zip(t.stride(), strides, shape) if n > 1)):
                raise ValueError("out does not match: pass the three tensors an earlier call returned")
    else:
        packed = _empty(*views[0], dtype=torch.float4_e2m1fn_x2, device=x.device)
        sf = _empty(*views[1], dtype=torch.float8_e4m3fn, device=x.device)
        sf_perm = _empty(*views[2], dtype=torch.float8_e4m3fn, device=x.device)
    _run(x, weight, residual, h, eps, _lib.NVFP4_NORM_NVFP4, packed.data_ptr(), sf_perm=sf_perm.data_ptr(),
         sf=sf.data_ptr())
    return (packed, sf, sf_perm), given if h is None else h
