"""MoE dispatch and combine around the grouped GEMM (``nvfp4_moe_dispatch`` /
``nvfp4_moe_combine`` in libnvfp4_b200.so).

The reference's grouped GEMM takes each expert's A_g, its permuted scales and
M_g as given (nvfp4_group_gemm/reference.py:39-74, the task tuple of
reference.py:196).  ``dispatch`` produces them from routed tokens on the
device: fp32 activations ``x [T, K]`` and expert choices ``ids [T, topk]``
become one packed NVFP4 buffer whose rows are grouped by expert (stable in
token order), the per-expert scale atoms, and the row / block offsets.
``grouped_inputs`` turns a dispatch plus per-expert weights into the
``(abc, sfasfb, sfasfb_reordered, problem_sizes)`` tuple that
``group_gemm.custom_kernel`` takes, and ``combine`` maps the grouped output
rows back to tokens (weighted sum over each token's choices).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from .dual_gemm import _current_stream_handle, check_sf_perm, on_device
from .gemv import DTYPES, _empty, _launch, _rows_last


@dataclass
class Dispatch:
    """Device tensors of one dispatch (int32 index arrays, uint8 byte arrays)."""
    packed: torch.Tensor        # [T*topk, K/2]; rows >= row_offsets[E] unused
    sf: torch.Tensor            # flat scale atoms, nvfp4_moe_sf_bytes() bytes
    counts: torch.Tensor        # [E]
    row_offsets: torch.Tensor   # [E+1]
    atom_offsets: torch.Tensor  # [E+1]
    src: torch.Tensor           # [T*topk]: pair index t*topk + j of each permuted row
    dst: torch.Tensor           # [T*topk]: permuted row of each pair, -1 if dropped
    workspace: torch.Tensor
    tokens: int
    topk: int
    k: int
    experts: int


def _alloc(tokens, topk, k, experts, device) -> Dispatch:
    lib = _lib.load()
    pairs = tokens * topk
    i32 = dict(dtype=torch.int32, device=device)
    return Dispatch(
        packed=torch.empty((pairs, k // 2), dtype=torch.uint8, device=device),
        sf=torch.empty(int(lib.nvfp4_moe_sf_bytes(tokens, topk, k, experts)), dtype=torch.uint8,
                       device=device),
        counts=torch.empty(experts, **i32), row_offsets=torch.empty(experts + 1, **i32),
        atom_offsets=torch.empty(experts + 1, **i32), src=torch.empty(pairs, **i32),
        dst=torch.empty(pairs, **i32),
        workspace=torch.empty(int(lib.nvfp4_moe_workspace_bytes(tokens, topk, experts)) // 4,
                              **i32),
        tokens=tokens, topk=topk, k=k, experts=experts)


def dispatch(x: torch.Tensor, expert_ids: torch.Tensor, num_experts: int,
             out: Dispatch | None = None) -> Dispatch:
    """Route ``x`` (CUDA fp32 [T, K], K % 64 == 0) by ``expert_ids`` (int32
    [T] or [T, topk]; ids outside [0, num_experts) are dropped).  ``out``: a
    Dispatch of an earlier call with the same sizes, whose buffers are reused."""
    if x.dim() != 2 or x.dtype != torch.float32 or not x.is_cuda:
        raise ValueError("x must be a CUDA float32 tensor [tokens, K]")
    ids = expert_ids if expert_ids.dim() == 2 else expert_ids.unsqueeze(1)
    if ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.dtype != torch.int32:
        raise ValueError("expert_ids must be int32 [tokens] or [tokens, topk]")
    if ids.device != x.device:
        raise ValueError("x and expert_ids must be on the same device")
    tokens, k = x.shape
    topk = ids.shape[1]
    if k % 64:
        raise ValueError(f"K={k} must be a multiple of 64")
    x, ids = x.contiguous(), ids.contiguous()
    if out is None:
        out = _alloc(tokens, topk, k, num_experts, x.device)
    elif (out.tokens, out.topk, out.k, out.experts) != (tokens, topk, k, num_experts) or \
            out.packed.device != x.device:
        raise ValueError("out does not match: pass a Dispatch made for the same sizes")
    d = out
    lib = _lib.load()
    _lib.check(on_device(x.device, lambda st: lib.nvfp4_moe_dispatch(
        x.data_ptr(), ids.data_ptr(), tokens, topk, k, num_experts, d.packed.data_ptr(),
        d.sf.data_ptr(), d.counts.data_ptr(), d.row_offsets.data_ptr(),
        d.atom_offsets.data_ptr(), d.src.data_ptr(), d.dst.data_ptr(), d.workspace.data_ptr(),
        d.workspace.numel() * 4, st)))
    return d


def expert_operands(d: Dispatch, counts=None):
    """Per expert: (a [M, K/2, 1] float4_e2m1fn_x2, sfa_perm [32, 4, ceil(M/128),
    4, K/64, 1] float8_e4m3fn, M) as views into the dispatch buffers.  Reads
    the counts back to the host (a synchronisation) unless ``counts`` (a list
    of ints) is given."""
    counts = [int(v) for v in (d.counts.tolist() if counts is None else counts)]
    ka = d.k // 64
    ops, row, blk = [], 0, 0
    for m in counts:
        rb = -(-m // 128)
        a = d.packed[row:row + m].view(torch.float4_e2m1fn_x2).unsqueeze(-1)
        atoms = d.sf[blk * ka * 512:(blk + rb) * ka * 512].view(1, rb, ka, 32, 4, 4)
        sfa = atoms.permute(3, 4, 1, 5, 2, 0).view(torch.float8_e4m3fn)
        ops.append((a, sfa, m))
        row += m
        blk += rb
    return ops


def grouped_inputs(d: Dispatch, weights, c_all: torch.Tensor, counts=None):
    """The grouped-GEMM task tuple for C_e = A_e . W_eᵀ over the experts with
    tokens.  ``weights``: per expert (w [N, K/2, 1] float4_e2m1fn_x2, sfw_perm
    [32, 4, ceil(N/128), 4, K/64, 1]); ``c_all``: fp16 [T*topk, N], expert e's
    output lands in rows [row_offsets[e], +M_e).  Returns (data, experts) with
    ``experts`` the expert index of each group in ``data``."""
    ops = expert_operands(d, counts)
    n = c_all.shape[1]
    abc, sfab, sfab_perm, sizes, which = [], [], [], [], []
    row = 0
    for e, ((a, sfa, m), (w, sfw)) in enumerate(zip(ops, weights)):
        if m > 0:
            abc.append((a, w, c_all[row:row + m].unsqueeze(-1)))
            sfab.append((None, None))          # plain scales: unused by the kernels
            sfab_perm.append((sfa, sfw))
            sizes.append((m, n, d.k, 1))
            which.append(e)
        row += m
    return (abc, sfab, sfab_perm, sizes), which


BYTES = (torch.uint8, torch.int8)


def _check_expert_scales(name, t, n, k, device):
    """One expert's permuted scales or their memory in any contiguous shape, but not plain [N, K/16] ones, which
    hold as many bytes where N is a multiple of 128."""
    rn, rk = -(-n // 128), k // 64
    if t.numel() != rn * rk * 512 or t.device != device:
        raise ValueError(f"{name} must hold {rn * rk * 512} bytes on {device}")
    if t.dtype not in BYTES + (torch.float8_e4m3fn,):
        raise ValueError(f"{name}: expected float8_e4m3fn, got {t.dtype}")
    view = t.unsqueeze(-1) if t.dim() == 5 else t
    if tuple(view.shape) == (32, 4, rn, 4, rk, 1):
        check_sf_perm(name, view, n, k, 1, device)
    elif not t.is_contiguous() or tuple(t.shape) in ((n, k // 16), (n, k // 16, 1), (1, n, k // 16)):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, strides {t.stride()} are not the permuted layout of [{n}, {k}]")


class ExpertWeights:
    """Per-expert NVFP4 weights for :func:`grouped_gemm`: ``w[e]`` = (b [N, K/2, 1]
    float4_e2m1fn_x2 (or uint8 [N, K/2]), sfb_perm [32, 4, ceil(N/128), 4, K/64, 1] or its
    memory), all on one device.  The pointer arrays for the C call are built once."""

    def __init__(self, w):
        self.w = list(w)
        if not self.w:
            raise ValueError("no experts")
        b0 = self.w[0][0]
        self.n, self.k = int(b0.shape[0]), int(b0.shape[1]) * 2
        arr = ctypes.c_void_p * len(self.w)
        for i, (b, sfb) in enumerate(self.w):
            if tuple(b.shape[:2]) != (self.n, self.k // 2) or not b.is_cuda:
                raise ValueError(f"expert {i}: weights must be CUDA [{self.n}, {self.k // 2}(, 1)]")
            if b.stride(0) != self.k // 2 or b.stride(1) != 1 or b.device != b0.device:
                raise ValueError(f"expert {i}: weights must be row-major [N][K/2] on {b0.device}")
            if b.dtype not in BYTES + (torch.float4_e2m1fn_x2,):
                raise ValueError(f"expert {i}: expected float4_e2m1fn_x2 weights, got {b.dtype}")
            _check_expert_scales(f"expert {i}: scales", sfb, self.n, self.k, b0.device)
        self.b_ptrs = arr(*[b.data_ptr() for b, _ in self.w])
        self.sfb_ptrs = arr(*[s.data_ptr() for _, s in self.w])
        self.device = b0.device
        self._table = None
        self._streams: set = set()  # whose calls the allocator knows to read the table
        self.space: dict = {}       # workspace bytes by (tokens, topk, type and alignment of x)

    def table(self) -> torch.Tensor:
        """The experts' weights as :func:`gemv` finds them in device memory (made by
        the first call that needs it)."""
        if self._table is None:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("call ExpertWeights.table() (or one product) before capturing a CUDA graph")
            lib = _lib.load()
            host = (ctypes.c_char * int(lib.nvfp4_moe_table_bytes(len(self.w))))()
            with torch.cuda.device(self.device):
                _lib.check(lib.nvfp4_moe_table(self.b_ptrs, self.sfb_ptrs, len(self.w), self.n, self.k, host))
                self._table = torch.frombuffer(host, dtype=torch.uint8).to(self.device)
                self._streams.add(_current_stream_handle(self.device.index))
        return self._table

    def _address(self, stream: int) -> int:
        """The table's address for a call on the current stream (its handle).  The allocator is told of each stream but
        the one that made the table, so that a table dropped before such a call has run stays until it has."""
        table = self.table()
        if stream not in self._streams:
            table.record_stream(torch.cuda.current_stream(self.device))
            self._streams.add(stream)
        return table.data_ptr()

    def __len__(self):
        return len(self.w)


def grouped_gemm(d: Dispatch, weights: ExpertWeights, c_all: torch.Tensor) -> torch.Tensor:
    """C_e = A_e . W_eᵀ for every expert straight from the dispatch's device
    sizes (no host synchronisation): expert e's output lands in rows
    [row_offsets[e], +counts[e]) of ``c_all`` (fp16 [T*topk, N])."""
    if len(weights) != d.experts or weights.k != d.k:
        raise ValueError(f"weights are for {len(weights)} experts x K={weights.k}, "
                         f"dispatch has {d.experts} x K={d.k}")
    if weights.device != d.packed.device:
        raise ValueError(f"weights are on {weights.device}, the dispatch on {d.packed.device}")
    rows = d.tokens * d.topk
    if (c_all.dtype != torch.float16 or tuple(c_all.shape) != (rows, weights.n)
            or not c_all.is_contiguous() or c_all.device != d.packed.device):
        raise ValueError(f"c_all must be a contiguous float16 [{rows}, {weights.n}] tensor "
                         f"on {d.packed.device}")
    lib = _lib.load()
    _lib.check(on_device(c_all.device, lambda st: lib.nvfp4_moe_grouped_gemm(
        d.packed.data_ptr(), rows, d.sf.data_ptr(), d.counts.data_ptr(), d.row_offsets.data_ptr(),
        d.atom_offsets.data_ptr(), weights.b_ptrs, weights.sfb_ptrs, d.experts, weights.n, d.k,
        c_all.data_ptr(), st)))
    return c_all


def combine(c_all: torch.Tensor, d: Dispatch, weights: torch.Tensor | None = None,
            out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * c_all[dst[t*topk + j]] (fp32 [T, N]);
    ``weights`` fp32 [T] or [T, topk], None for all ones."""
    if c_all.dim() != 2 or c_all.dtype != torch.float16 or not c_all.is_contiguous():
        raise ValueError("c_all must be a contiguous float16 tensor [rows, N]")
    n, dst = c_all.shape[1], d.dst
    if (dst.device != c_all.device or dst.dtype != torch.int32 or dst.numel() != d.tokens * d.topk
            or not dst.is_contiguous()):
        raise ValueError(f"the order of {d.tokens} x {d.topk} rows must be contiguous int32 on c_all's device")
    if weights is not None:
        weights = weights.reshape(d.tokens, d.topk)
        if weights.dtype != torch.float32 or weights.device != c_all.device:
            raise ValueError("weights must be float32 on c_all's device")
        weights = weights.contiguous()
    if out is None:
        out = torch.empty((d.tokens, n), dtype=torch.float32, device=c_all.device)
    elif (tuple(out.shape) != (d.tokens, n) or out.dtype != torch.float32 or not out.is_contiguous()
          or out.device != c_all.device):
        raise ValueError("out must be a contiguous float32 tensor [tokens, N] on c_all's device")
    if not c_all.is_cuda:
        raise ValueError("c_all must be a CUDA tensor")
    lib = _lib.load()
    _lib.check(on_device(c_all.device, lambda st: lib.nvfp4_moe_combine(
        c_all.data_ptr(), c_all.shape[0], dst.data_ptr(),
        weights.data_ptr() if weights is not None else None,
        d.tokens, d.topk, n, out.data_ptr(), st)))
    return out


def _products(x, expert_ids, w, w2, out, out_dtype):
    ids = expert_ids if expert_ids.dim() == 2 else expert_ids.unsqueeze(1)
    if ids.dim() != 2 or ids.dtype != torch.int32:
        raise ValueError("expert_ids must be int32 [tokens] or [tokens, topk]")
    code = DTYPES.get(x.dtype)
    if x.dim() != 2 or code is None:
        raise ValueError("x must be float16, bfloat16 or float32 [tokens or tokens*topk, K]")
    if not (x.device == ids.device == w.device):
        raise ValueError(f"x, expert_ids and the weights must be on one device ({w.device})")
    tokens, topk = ids.shape
    rows, n, k = tokens * topk, w.n, w.k
    if x.shape[1] != k or x.shape[0] not in (tokens, rows):
        raise ValueError(f"x {tuple(x.shape)} is neither [{tokens}, {k}] nor [{rows}, {k}]")
    if rows >> 31:
        raise ValueError(f"{rows} rows: at most 256")
    x, ids = _rows_last(x), ids.contiguous()
    if out is None:
        out = _empty((rows, n), (n, 1), dtype=out_dtype or x.dtype, device=x.device)
        if out.dtype not in DTYPES:
            raise ValueError(f"out_dtype {out_dtype} is none of float16, bfloat16 and float32")
    elif (tuple(out.shape) != (rows, n) or out.dtype not in DTYPES or out.device != x.device
          or out.dtype != (out_dtype or out.dtype) or (out.stride(1) != 1 and n > 1)
          or (rows > 1 and out.stride(0) < n)):
        raise ValueError(f"out must be [{rows}, {n}], float16, bfloat16 or float32, rows apart, on {x.device}")
    if rows == 0:
        return out
    ldx, ldo, px = x.stride(0), out.stride(0), x.data_ptr()
    lib = _lib.load()
    aligned = not (px | ldx * x.element_size()) & 15
    size = w.space.get((tokens, topk, code, aligned))
    if size is None:
        # three and more tokens that choose more often than there are experts: with the space that an x without alignment
        # needs, the library takes the form that reads an expert less often where that is faster
        size = w.space[(tokens, topk, code, aligned)] = lib.nvfp4_moe_gemv_workspace_bytes(
            code, aligned and (tokens <= 2 or rows <= len(w)), tokens, topk, k)
    space = _empty((size,), (1,), dtype=torch.uint8, device=x.device) if size else None
    stream = _current_stream_handle(x.device.index)
    _launch(lib.nvfp4_moe_gemv, x.device, (
        px, code, ldx, x.shape[0] == rows and topk > 1, ids.data_ptr(), tokens, topk, w._address(stream),
        w2._address(stream) if w2 is not None else None, len(w), out.data_ptr(), DTYPES[out.dtype],
        ldo if ldo > n else n, n, k, space.data_ptr() if size else None, size))
    return out


def gemv(x: torch.Tensor, expert_ids: torch.Tensor, weights: ExpertWeights,
         out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Row t*topk + j of the result is x_row . W_eᵀ with e = expert_ids[t, j] (int32
    [T] or [T, topk]): a decoding step's experts without a dispatch, activations not
    quantised, each chosen expert's weights read once for every group of its rows (two rows
    up to 32 in all, unless three and more tokens choose more often than there are experts; else
    4 to 16 rows, about twice an expert's average).
    ``x``: float16, bfloat16 or float32, [T, K] (token t's row for all its choices)
    or [T*topk, K] (a row for each choice).  A row whose id is outside
    [0, experts) is zero.  Result [T*topk, N] in ``out_dtype`` (x's type by
    default); float16 goes into :func:`combine` with :func:`pair_order`.  At most
    256 rows: ``dispatch`` and ``grouped_gemm`` are for more."""
    return _products(x, expert_ids, weights, None, out, out_dtype)


def dual_gemv(x: torch.Tensor, expert_ids: torch.Tensor, w1: ExpertWeights, w2: ExpertWeights,
              out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """silu(x_row . W1_eᵀ) * (x_row . W2_eᵀ) for each choice; otherwise as :func:`gemv`."""
    if (len(w1), w1.n, w1.k, w1.device) != (len(w2), w2.n, w2.k, w2.device):
        raise ValueError("w1 and w2 must have the same number of experts, N, K and device")
    return _products(x, expert_ids, w1, w2, out, out_dtype)


@dataclass
class PairOrder:
    """Rows in the order of the choices (row t*topk + j), as :func:`gemv` leaves
    them: stands in for a Dispatch in :func:`combine`."""
    dst: torch.Tensor
    tokens: int
    topk: int


def pair_order(tokens: int, topk: int, device) -> PairOrder:
    """Made once for each (tokens, topk)."""
    return PairOrder(torch.arange(tokens * topk, dtype=torch.int32, device=device), tokens, topk)
