"""Attention inside the structures of a packed batch, differentiable: the operators of a readout on per-atom features.

The network's own attention stops at its 4.5 A cutoff.  These act on rows packed structure by structure, as `System(graph_start=...)` and
`So3lr(batch_segments=...)` pack atoms (or frame by frame, for the trajectories of a batch):

    packed = PackedStructures(graph_start)                        # the layout, once per batch
    q, k = norm_rotate(q, k, positions, frequencies, q_weight=wq, k_weight=wk)
    out = structure_attention(q, k, v, packed)                    # every row attends to the rows of its structure

Both run on the current stream of their inputs' device, support autograd once (not twice), and give the same bits every time.  No counterpart in
the reference.  Memory comes from torch's allocator, so a call can be captured into a CUDA graph (capture the backward pass with leaves
that no live eager graph holds: torch's own accumulation nodes remember the stream that they were made on).
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch
from torch.autograd.function import once_differentiable

from ._lib import AttentionShape, NormRotateArgs, Rows, check, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _stream(t):
    return C.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _head_rows(name, t, dtype, device, d=None):
    """`t` (rows, heads, d) in a form that the kernels read: as it is where its last axis is contiguous, 16-byte pieces are aligned and no axis
    is broadcast, else a contiguous copy."""
    if t.ndim != 3 or t.dtype != dtype or t.device != device or (d is not None and t.shape[2] != d):
        raise ValueError(f"{name} must be (rows, heads, {'d' if d is None else d}) {dtype} on {device}, not {tuple(t.shape)} {t.dtype} on {t.device}")
    unit = 16 // t.element_size()
    if t.stride(2) != 1 or t.stride(0) % unit or t.stride(1) % unit or t.data_ptr() % 16 or 0 in t.stride():
        t = t.contiguous()
        if t.data_ptr() % 16 or t.stride(2) != 1:
            t = t.clone(memory_format=torch.contiguous_format)
    return t


def _rows(t):
    return Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _first(q):
    if not isinstance(q, torch.Tensor) or q.device.type != "cuda" or q.dtype not in _TYPES or q.ndim != 3:
        got = f"{tuple(q.shape)} {q.dtype} on {q.device}" if isinstance(q, torch.Tensor) else type(q).__name__
        raise ValueError(f"rows must be (n, heads, d) float32, bfloat16 or float16 on a GPU, not {got}")


# ------------------------------------------------------------------------------------------------------------
# layout
# ------------------------------------------------------------------------------------------------------------
class PackedStructures:
    """The layout of a batch.  `graph_start` (n_structures + 1 ascending integers from 0) gives the first row of every structure and the number
    of rows; `graph_start_kv` the same for the keys where they are other rows than the queries (one query per structure, new frames
    of trajectories).  causal: query i of lq sees key j of lk where j <= i + lk - lq, so the last query sees all keys.  Structures
    may be empty on either side; a query that sees no key gives zero.  Make it outside of a graph capture: it copies its tables to the device
    and waits for that."""

    def __init__(self, graph_start, graph_start_kv=None, causal=False, device=0):
        q = self._starts("graph_start", graph_start)
        k = q if graph_start_kv is None else self._starts("graph_start_kv", graph_start_kv)
        if len(q) != len(k):
            raise ValueError(f"graph_start describes {len(q) - 1} structures, graph_start_kv {len(k) - 1}")
        self.device = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        if self.device.type != "cuda":
            raise ValueError(f"a layout lives on a GPU, not on {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.n_structures, self.rows_q, self.rows_kv, self.causal = len(q) - 1, int(q[-1]), int(k[-1]), bool(causal)
        qp, kp = q.ctypes.data_as(C.c_void_p), k.ctypes.data_as(C.c_void_p)
        size = lib.so3lr_b200_packing_size(self.n_structures, qp, kp)
        if size < 0:
            raise ValueError("graph_start must ascend from 0")
        self._image = np.empty(size, np.int32)
        self._host = self._image.ctypes.data_as(C.c_void_p)
        check(lib.so3lr_b200_packing_build(self.n_structures, qp, kp, int(self.causal), self._host, size), "packing_build")
        if not torch.cuda.is_available():
            raise RuntimeError("so3lr_b200 needs a CUDA device (sm_100a); there is no CPU path")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a PackedStructures layout cannot be made while a graph is captured")
        self._made_on = torch.cuda.current_stream(self.device)
        self._dev = torch.from_numpy(self._image).to(self.device)

    @staticmethod
    def _starts(name, x):
        x = x.detach().cpu().numpy() if isinstance(x, torch.Tensor) else np.asarray(x)
        if x.ndim != 1 or x.size < 1 or not np.issubdtype(x.dtype, np.integer):
            raise ValueError(f"{name} must be a list of n_structures + 1 integers, not {x.dtype} {x.shape}")
        x = x.astype(np.int64)
        if x[0] != 0 or np.any(np.diff(x) < 0) or x[-1] >= 2**31 - 1:
            raise ValueError(f"{name} must ascend from 0 and stay below 2**31")
        return np.ascontiguousarray(x, dtype=np.int32)

    def _table(self, t):
        """The device copy, kept alive for the stream that is about to read it."""
        s = torch.cuda.current_stream(t.device)
        if s != self._made_on:
            self._dev.record_stream(s)
        return C.c_void_p(self._dev.data_ptr())


# ------------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------------
def _workspace(packed, shape, vjp, device):
    size = lib.so3lr_b200_structure_attention_workspace(packed._host, C.byref(shape), vjp)
    return (torch.empty(size, dtype=torch.uint8, device=device), size) if size > 0 else (None, 0)


def _attention_forward(q, k, v, packed, shape, train):
    """(out, what rounding it left or None, lse or None)"""
    with torch.cuda.device(q.device):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        rest = torch.empty_like(out) if train and q.dtype != torch.float32 else None
        lse = torch.empty(q.shape[1], q.shape[0], dtype=torch.float32, device=q.device) if train else None
        if q.shape[0] > packed.rows_q:      # rows behind the last structure belong to none
            out[packed.rows_q:].zero_()
        if packed.rows_q:
            work, size = _workspace(packed, shape, 0, q.device)
            check(lib.so3lr_b200_structure_attention(packed._host, packed._table(q), _stream(q), C.byref(shape), C.byref(_rows(q)),
                                                     C.byref(_rows(k)), C.byref(_rows(v)), _p(out), _p(rest), _p(lse), _p(work), size),
                  "structure_attention")
    return out, rest, lse


class _StructureAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packed, shape):
        out, rest, lse = _attention_forward(q, k, v, packed, shape, True)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.packed, ctx.shape = packed, shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        q, k, v, out, rest, lse = ctx.saved_tensors
        packed = ctx.packed
        with torch.cuda.device(q.device):
            g = _head_rows("the cotangent", g, q.dtype, q.device)
            dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
            for t, n in ((dq, packed.rows_q), (dk, packed.rows_kv), (dv, packed.rows_kv)):
                if t.shape[0] > n:
                    t[n:].zero_()
            if packed.rows_q or packed.rows_kv:
                delta = torch.empty_like(lse)
                work, size = _workspace(packed, ctx.shape, 1, q.device)
                check(lib.so3lr_b200_structure_attention_vjp(packed._host, packed._table(q), _stream(q), C.byref(ctx.shape), C.byref(_rows(q)),
                                                             C.byref(_rows(k)), C.byref(_rows(v)), _p(out), _p(rest), _p(lse), C.byref(_rows(g)),
                                                             _p(delta), _p(dq), _p(dk), _p(dv), _p(work), size), "structure_attention_vjp")
        return dq, dk, dv, None, None


def structure_attention(q, k, v, packed, scale=None):
    """softmax(scale q k^T) v inside every structure of `packed`.

    q (n, heads, d); k, v (n_kv, heads_kv, d) with heads a multiple of heads_kv (query head h reads key head h // (heads // heads_kv));
    float32, bfloat16 or float16 on one GPU, d a multiple of 16 up to 128, any strides.  scale: 1 / sqrt(d) unless given, positive.  Returns
    (n, heads, d); rows behind the layout's last structure are zero.  Values that are not finite spoil the rows of their own structure
    only.  Sums and the softmax run in float32; 16-bit probabilities are rounded once to the inputs' type ahead of the product with v."""
    _first(q)
    if not isinstance(packed, PackedStructures):
        raise ValueError(f"packed must be a PackedStructures layout, not {type(packed).__name__}")
    d = q.shape[2]
    q = _head_rows("q", q, q.dtype, q.device)
    k, v = (_head_rows(name, t, q.dtype, q.device, d) for name, t in (("k", k), ("v", v)))
    if packed.device != q.device:
        raise ValueError(f"the layout is on {packed.device}, the rows on {q.device}")
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    if d % 16 or not 16 <= d <= 128:
        raise ValueError(f"d must be a multiple of 16 up to 128, not {d}")
    if not q.shape[1] or not k.shape[1] or q.shape[1] % k.shape[1] or q.shape[1] > 65535:
        raise ValueError(f"{q.shape[1]} query heads cannot share {k.shape[1]} key heads")
    if q.shape[0] < packed.rows_q or k.shape[0] < packed.rows_kv:
        raise ValueError(f"the layout has {packed.rows_q} and {packed.rows_kv} rows, q {q.shape[0]} and k {k.shape[0]}")
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, not {scale}")
    shape = AttentionShape(_TYPES[q.dtype], q.shape[1], k.shape[1], d, q.shape[0], k.shape[0], scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _StructureAttention.apply(q, k, v, packed, shape)
    return _attention_forward(q, k, v, packed, shape, False)[0]


# ------------------------------------------------------------------------------------------------------------
# norm and rotation
# ------------------------------------------------------------------------------------------------------------
def _rotate_args(q, k, positions, frequencies, wq, wk, eps, neighbors):
    w = wq if wq is not None else wk
    return NormRotateArgs(q.shape[0], q.shape[2], q.shape[1], 0 if k is None else k.shape[1], _TYPES[q.dtype],
                          0 if positions is None else positions.shape[1], int(neighbors), int(w is not None),
                          int(w is not None and w.dtype == torch.float32), int(positions is not None and positions.dtype == torch.float64), eps,
                          _p(positions), _p(frequencies), _p(wq), _p(wk))


def _norm_rotate_forward(q, k, positions, frequencies, wq, wk, eps, neighbors):
    with torch.cuda.device(q.device):
        oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ok = None if k is None else torch.empty(k.shape, dtype=q.dtype, device=q.device)
        a = _rotate_args(q, k, positions, frequencies, wq, wk, eps, neighbors)
        check(lib.so3lr_b200_norm_rotate(_stream(q), C.byref(a), C.byref(_rows(q)), None if k is None else C.byref(_rows(k)), _p(oq), _p(ok)),
              "norm_rotate")
    return oq, ok


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, wq, wk, eps, neighbors):
        ctx.save_for_backward(q, k, positions, frequencies, wq, wk)
        ctx.rest = eps, neighbors
        ctx.set_materialize_grads(False)
        return _norm_rotate_forward(q, k, positions, frequencies, wq, wk, eps, neighbors)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, positions, frequencies, wq, wk = ctx.saved_tensors
        if gq is None and gk is None:
            return (None,) * 8
        with torch.cuda.device(q.device):
            gq = torch.zeros_like(q) if gq is None else gq
            gq = _head_rows("the cotangent", gq, q.dtype, q.device)
            if k is not None:
                gk = _head_rows("the cotangent", torch.zeros_like(k) if gk is None else gk, q.dtype, q.device)
            dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            dk = None if k is None else torch.empty(k.shape, dtype=q.dtype, device=q.device)
            dpos = torch.empty_like(positions) if positions is not None and ctx.needs_input_grad[2] else None
            dwq, dwk = (torch.empty_like(w) if w is not None and n else None for w, n in ((wq, ctx.needs_input_grad[4]), (wk, ctx.needs_input_grad[5])))
            size = lib.so3lr_b200_norm_rotate_workspace(q.shape[2]) if dwq is not None or dwk is not None else 0
            work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
            a = _rotate_args(q, k, positions, frequencies, wq, wk, *ctx.rest)
            check(lib.so3lr_b200_norm_rotate_vjp(_stream(q), C.byref(a), C.byref(_rows(q)), None if k is None else C.byref(_rows(k)),
                                                 C.byref(_rows(gq)), None if k is None else C.byref(_rows(gk)), _p(dq), _p(dk), _p(dpos), _p(dwq),
                                                 _p(dwk), _p(work), size), "norm_rotate_vjp")
        return dq, dk, dpos, None, dwq, dwk, None, None


def norm_rotate(q, k=None, positions=None, frequencies=None, *, q_weight=None, k_weight=None, eps=1e-6, pairing="halves"):
    """(q, k) normalised per head and rotated by the rows' positions, in one pass.

    Norm, where weights (d) are given (both sides or neither; float32 or the rows' type): weight * x / sqrt(mean(x^2) + eps).
    Rotation, where positions (n, axes) float32 or float64 and frequencies (axes, d / 2) float32 are given: pair p of a head turns by
    theta_p = sum_a positions[:, a] frequencies[a, p], formed in float64; pairs are (p, p + d / 2) ("halves") or (2p, 2p + 1)
    ("neighbors").  The product of two rotated rows then depends on the difference of their positions only.  q (n, heads, d) and
    k (n, heads_k, d), or None, float32, bfloat16 or float16 on one GPU, d a multiple of 16 up to 256, any strides.  Gradients: q, k, positions and the
    weights (frequencies are constants).  Returns new (q, k), contiguous."""
    _first(q)
    d = q.shape[2]
    q = _head_rows("q", q, q.dtype, q.device)
    if k is not None:
        k = _head_rows("k", k, q.dtype, q.device, d)
        if k.shape[0] != q.shape[0]:
            raise ValueError(f"q has {q.shape[0]} rows, k {k.shape[0]}")
    if d % 16 or not 16 <= d <= 256:
        raise ValueError(f"d must be a multiple of 16 up to 256, not {d}")
    if pairing not in ("halves", "neighbors"):
        raise ValueError(f"pairing must be 'halves' or 'neighbors', not {pairing!r}")
    if (positions is None) != (frequencies is None):
        raise ValueError("positions and frequencies come together")
    norm = q_weight is not None or k_weight is not None
    if not norm and positions is None:
        raise ValueError("neither weights nor positions: nothing to do")
    if norm and (q_weight is None or (k_weight is None) != (k is None)):
        raise ValueError("weights come for both sides or for neither")
    if positions is not None:
        if positions.ndim != 2 or positions.shape[0] != q.shape[0] or not 1 <= positions.shape[1] <= 16 or positions.device != q.device or \
                positions.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"positions must be ({q.shape[0]}, axes) float32 or float64 on {q.device}, not {tuple(positions.shape)} {positions.dtype} "
                             f"on {positions.device}")
        if tuple(frequencies.shape) != (positions.shape[1], d // 2) or frequencies.dtype != torch.float32 or frequencies.device != q.device:
            raise ValueError(f"frequencies must be ({positions.shape[1]}, {d // 2}) float32 on {q.device}, not {tuple(frequencies.shape)} "
                             f"{frequencies.dtype} on {frequencies.device}")
        if frequencies.requires_grad and torch.is_grad_enabled():
            raise ValueError("frequencies are constants: no gradient is formed for them")
        positions, frequencies = positions.contiguous(), frequencies.contiguous()
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (d,) or w.device != q.device or w.dtype not in (torch.float32, q.dtype) or w.dtype != q_weight.dtype):
            raise ValueError(f"{name} must be ({d},) float32 or {q.dtype} on {q.device}, both sides alike, not {tuple(w.shape)} {w.dtype} on {w.device}")
    q_weight, k_weight = (None if w is None else w.contiguous() for w in (q_weight, k_weight))
    eps = float(eps)
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"eps must not be negative, not {eps}")
    args = (q, k, positions, frequencies, q_weight, k_weight, eps, pairing == "neighbors")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:6]):
        return _NormRotate.apply(*args)
    return _norm_rotate_forward(*args)
