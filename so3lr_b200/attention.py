"""Attention inside the structures of a packed batch, differentiable: the operators of a readout on per-atom features.

The network's own attention stops at its 4.5 A cutoff.  These act on rows packed structure by structure, as `System(graph_start=...)` and
`So3lr(batch_segments=...)` pack atoms (or frame by frame, for the trajectories of a batch):

    packed = PackedStructures(graph_start)                        # the layout, once per batch
    q, k = norm_rotate(q, k, positions, frequencies, q_weight=wq, k_weight=wk)
    out = structure_attention(q, k, v, packed)                    # every row attends to the rows of its structure

Both run on the current stream of their inputs' device, support autograd once (not twice, and not in forward mode), and give the same bits every time.
No counterpart in the reference.  Memory comes from torch's allocator, so a call can be captured into a CUDA graph (capture the backward pass with leaves
that no live eager graph holds: torch's own accumulation nodes remember the stream that they were made on).  Every wait inside the kernels is bounded;
should one run out, rows of that call are NaN and the next structure_attention on the device, forward or backward, raises So3lrB200Error, once.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch
import torch.autograd.forward_ad as _forward_ad
from torch.autograd.function import once_differentiable

from ._lib import AttentionShape, NormRotateArgs, Rows, check, lib

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_UNIT = {torch.float32: 4, torch.bfloat16: 8, torch.float16: 8}      # values of 16 bytes
_CONTIGUOUS = torch.contiguous_format
_raw_stream = torch._C._cuda_getCurrentRawStream                     # of a device ordinal: torch.cuda.current_stream(..).cuda_stream without its object


def _p(t):
    return 0 if t is None else t.data_ptr()


def _aligned(t, unit):
    """`t` (rows, heads, d) in a form that the kernels read: as it is where its last axis is contiguous, 16-byte pieces are aligned and no axis
    is broadcast, else a contiguous copy."""
    a, b, c = t.stride()
    if c != 1 or not a or not b or (a | b) % unit or t.data_ptr() % 16:
        t = t.contiguous()
        a, b, _ = t.stride()
        if not a or not b or (a | b) % unit or t.data_ptr() % 16:      # as it was: the stride of an axis of one is free
            t = t.clone(memory_format=torch.contiguous_format)
    return t


def _head_rows(name, t, dtype, device, d=None):
    if t.ndim != 3 or t.dtype != dtype or t.device != device or (d is not None and t.shape[2] != d):
        raise ValueError(f"{name} must be (rows, heads, {'d' if d is None else d}) {dtype} on {device}, not {tuple(t.shape)} {t.dtype} on {t.device}")


def _cotangent(g, like):
    """`g` as the kernels read it (autograd hands over what has the output's shape, type and device)."""
    return _aligned(g, _UNIT[like.dtype])


def _rows(t):
    return Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _first(q):
    if not isinstance(q, torch.Tensor) or q.device.type != "cuda" or q.dtype not in _TYPES or q.ndim != 3:
        got = f"{tuple(q.shape)} {q.dtype} on {q.device}" if isinstance(q, torch.Tensor) else type(q).__name__
        raise ValueError(f"rows must be (n, heads, d) float32, bfloat16 or float16 on a GPU, not {got}")


def _no_tangents(name, *tensors):
    """The kernels read a dual tensor's value through its pointer: its tangent would be dropped, which counts as zero."""
    if _forward_ad._current_level >= 0:
        for t in tensors:
            if isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} is not differentiable in forward mode")


def _constant(name, x):
    """The number x; raises where a gradient is asked of it."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} is a constant: no gradient is formed for it")
    return float(x)


class _On:
    """Makes a tensor's device the current one where it is not (a context object per call costs more than the launch of a kernel)."""
    __slots__ = ("index", "back")

    def __init__(self, index):
        self.index = index

    def __enter__(self):
        self.back = torch._C._cuda_getDevice()
        if self.back != self.index:
            torch._C._cuda_setDevice(self.index)

    def __exit__(self, *_):
        if self.back != self.index:
            torch._C._cuda_setDevice(self.back)


# ------------------------------------------------------------------------------------------------------------
# layout
# ------------------------------------------------------------------------------------------------------------
class PackedStructures:
    """The layout of a batch.  `graph_start` (n_structures + 1 ascending integers from 0) gives the first row of every structure and the number
    of rows; `graph_start_kv` the same for the keys where they are other rows than the queries (one query per structure, new frames
    of trajectories).  causal: query i of lq sees key j of lk where j <= i + lk - lq, so the last query sees all keys.  Structures
    may be empty on either side; a query that sees no key gives zero.  Make it outside of a graph capture: it copies its tables to the device
    and waits for that.  A captured graph reads these tables: the layout has to live as long as the graph is replayed."""

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
        self._index = self.device.index
        self._made_on = _raw_stream(self._index)
        self._dev = torch.from_numpy(self._image).to(self.device)
        self._dev_ptr = self._dev.data_ptr()
        self._calls = {}

    @staticmethod
    def _starts(name, x):
        x = x.detach().cpu().numpy() if isinstance(x, torch.Tensor) else np.asarray(x)
        if x.ndim != 1 or x.size < 1 or not np.issubdtype(x.dtype, np.integer):
            raise ValueError(f"{name} must be a list of n_structures + 1 integers, not {x.dtype} {x.shape}")
        x = x.astype(np.int64)
        if x[0] != 0 or np.any(np.diff(x) < 0) or x[-1] >= 2**31 - 1:
            raise ValueError(f"{name} must ascend from 0 and stay below 2**31")
        return np.ascontiguousarray(x, dtype=np.int32)

    def _stream(self):
        """The current stream, on which the layout's tables stay alive."""
        s = _raw_stream(self._index)
        if s != self._made_on:
            self._dev.record_stream(torch.cuda.current_stream(self.device))
        return s

    def _call(self, q, k, scale):
        """What calls with rows of these shapes have in common: (shape, workspace of the forward call, of its transpose); raises where the
        shapes do not fit."""
        scale = None if scale is None else _constant("scale", scale)
        key = (q.dtype, q.shape, k.shape, scale)
        call = self._calls.get(key)
        if call is None:
            (n, heads, d), (n_kv, heads_kv, _) = q.shape, k.shape
            if d % 16 or not 16 <= d <= 128:
                raise ValueError(f"d must be a multiple of 16 up to 128, not {d}")
            if not heads or not heads_kv or heads % heads_kv or heads > 65535:
                raise ValueError(f"{heads} query heads cannot share {heads_kv} key heads")
            if n < self.rows_q or n_kv < self.rows_kv:
                raise ValueError(f"the layout has {self.rows_q} and {self.rows_kv} rows, q {n} and k {n_kv}")
            if max(n, n_kv) >= 2**31 - 1:
                raise ValueError(f"q has {n} and k {n_kv} rows; at most 2**31 - 2 are supported")
            x = 1.0 / math.sqrt(d) if scale is None else scale
            if not (x > 0 and math.isfinite(x)):
                raise ValueError(f"scale must be positive and finite, not {scale}")
            shape = AttentionShape(_TYPES[q.dtype], heads, heads_kv, d, n, n_kv, x)
            call = C.byref(shape), *(lib.so3lr_b200_structure_attention_workspace(self._host, C.byref(shape), vjp) for vjp in (0, 1))
            if len(self._calls) >= 64:
                self._calls.clear()
            self._calls[key] = call
        return call


# ------------------------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------------------------
def _attention_forward(q, k, v, packed, call, train):
    """(out, what rounding it left or None, lse or None)"""
    shape, size, _ = call
    with _On(packed._index):
        out = torch.empty_like(q, memory_format=_CONTIGUOUS)
        rest = torch.empty_like(q, memory_format=_CONTIGUOUS) if train and q.dtype != torch.float32 else None
        lse = q.new_empty((q.shape[1], q.shape[0]), dtype=torch.float32) if train else None
        if q.shape[0] > packed.rows_q:      # rows behind the last structure belong to none
            out[packed.rows_q:].zero_()
        if packed.rows_q:
            work = q.new_empty(size, dtype=torch.uint8) if size > 0 else None
            check(lib.so3lr_b200_structure_attention(packed._host, packed._dev_ptr, packed._stream(), shape, C.byref(_rows(q)), C.byref(_rows(k)),
                                                     C.byref(_rows(v)), out.data_ptr(), _p(rest), _p(lse), _p(work), size), "structure_attention")
    return out, rest, lse


def _attention_backward(ctx, g):
    q, k, v, out, rest, lse = ctx.saved_tensors
    packed, (shape, _, size) = ctx.packed, ctx.call
    _no_tangents("structure_attention", g)
    with _On(packed._index):
        g = _cotangent(g, q)
        dq, dk, dv = torch.empty_like(q, memory_format=_CONTIGUOUS), torch.empty_like(k, memory_format=_CONTIGUOUS), torch.empty_like(k, memory_format=_CONTIGUOUS)
        if q.shape[0] > packed.rows_q:
            dq[packed.rows_q:].zero_()
        if k.shape[0] > packed.rows_kv:
            dk[packed.rows_kv:].zero_()
            dv[packed.rows_kv:].zero_()
        if packed.rows_q or packed.rows_kv:
            delta = torch.empty_like(lse)
            work = q.new_empty(size, dtype=torch.uint8) if size > 0 else None
            check(lib.so3lr_b200_structure_attention_vjp(packed._host, packed._dev_ptr, packed._stream(), shape, C.byref(_rows(q)), C.byref(_rows(k)),
                                                         C.byref(_rows(v)), out.data_ptr(), _p(rest), lse.data_ptr(), C.byref(_rows(g)),
                                                         delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _p(work), size),
                  "structure_attention_vjp")
    return dq, dk, dv, None, None


_attention_backward_once = once_differentiable(_attention_backward)


class _StructureAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, packed, call):
        out, rest, lse = _attention_forward(q, k, v, packed, call, True)
        ctx.save_for_backward(q, k, v, out, rest, lse)
        ctx.packed, ctx.call = packed, call
        return out

    @staticmethod
    def backward(ctx, g):      # differentiable once: the guard against a second time is only needed where a graph is recorded
        return _attention_backward_once(ctx, g) if torch.is_grad_enabled() else _attention_backward(ctx, g)


def structure_attention(q, k, v, packed, scale=None):
    """softmax(scale q k^T) v inside every structure of `packed`.

    q (n, heads, d); k, v (n_kv, heads_kv, d) with heads a multiple of heads_kv (query head h reads key head h // (heads // heads_kv));
    float32, bfloat16 or float16 on one GPU, d a multiple of 16 up to 128, any strides.  scale: 1 / sqrt(d) unless given, positive, a constant.  Returns
    (n, heads, d); rows behind the layout's last structure are zero.  Values that are not finite spoil the rows of their own structure
    only.  Sums and the softmax run in float32.  With 16-bit rows the probabilities, and in the backward pass their gradients dS = P (dP - delta),
    are rounded to the inputs' type on the way into a second product.  float16 takes powers of two out of both first: neither the tails of
    a softmax nor cotangents of any size are lost in its last steps."""
    _first(q)
    if not isinstance(packed, PackedStructures):
        raise ValueError(f"packed must be a PackedStructures layout, not {type(packed).__name__}")
    dtype, device = q.dtype, q.device
    if packed.device != device:
        raise ValueError(f"the layout is on {packed.device}, the rows on {device}")
    _head_rows("k", k, dtype, device, q.shape[2])
    _head_rows("v", v, dtype, device)
    if k.shape != v.shape:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    _no_tangents("structure_attention", q, k, v, scale)
    call = packed._call(q, k, scale)
    unit = _UNIT[dtype]
    q, k, v = _aligned(q, unit), _aligned(k, unit), _aligned(v, unit)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _StructureAttention.apply(q, k, v, packed, call)
    return _attention_forward(q, k, v, packed, call, False)[0]


# ------------------------------------------------------------------------------------------------------------
# norm and rotation
# ------------------------------------------------------------------------------------------------------------
def _rotate_args(q, k, positions, frequencies, wq, wk, eps, neighbors):
    n, heads, d = q.shape
    w = wq if wq is not None else wk
    return NormRotateArgs(n, d, heads, 0 if k is None else k.shape[1], _TYPES[q.dtype], 0 if positions is None else positions.shape[1], neighbors,
                          w is not None, w is not None and w.dtype == torch.float32, positions is not None and positions.dtype == torch.float64, eps,
                          _p(positions), _p(frequencies), _p(wq), _p(wk))


def _norm_rotate_forward(q, k, positions, frequencies, wq, wk, eps, neighbors):
    index = q.device.index
    with _On(index):
        oq = torch.empty_like(q, memory_format=_CONTIGUOUS)
        ok = None if k is None else torch.empty_like(k, memory_format=_CONTIGUOUS)
        a = _rotate_args(q, k, positions, frequencies, wq, wk, eps, neighbors)
        check(lib.so3lr_b200_norm_rotate(_raw_stream(index), C.byref(a), C.byref(_rows(q)), None if k is None else C.byref(_rows(k)), oq.data_ptr(),
                                         _p(ok)), "norm_rotate")
    return oq, ok


def _norm_rotate_backward(ctx, gq, gk):
    q, k, positions, frequencies, wq, wk = ctx.saved_tensors
    if gq is None and gk is None:
        return (None,) * 8
    _no_tangents("norm_rotate", gq, gk)
    index, need = q.device.index, ctx.needs_input_grad
    with _On(index):
        gq = _cotangent(torch.zeros_like(q) if gq is None else gq, q)
        dq, dk, gk_rows = torch.empty_like(q, memory_format=_CONTIGUOUS), None, None
        if k is not None:
            gk = _cotangent(torch.zeros_like(k) if gk is None else gk, k)
            dk, gk_rows = torch.empty_like(k, memory_format=_CONTIGUOUS), C.byref(_rows(gk))
        dpos = torch.empty_like(positions) if positions is not None and need[2] else None
        dwq = torch.empty_like(wq) if wq is not None and need[4] else None
        dwk = torch.empty_like(wk) if wk is not None and need[5] else None
        size = lib.so3lr_b200_norm_rotate_workspace(q.shape[2]) if dwq is not None or dwk is not None else 0
        work = q.new_empty(size, dtype=torch.uint8) if size else None
        a = _rotate_args(q, k, positions, frequencies, wq, wk, *ctx.rest)
        check(lib.so3lr_b200_norm_rotate_vjp(_raw_stream(index), C.byref(a), C.byref(_rows(q)), None if k is None else C.byref(_rows(k)),
                                             C.byref(_rows(gq)), gk_rows, dq.data_ptr(), _p(dk), _p(dpos), _p(dwq), _p(dwk), _p(work), size),
              "norm_rotate_vjp")
    return dq, dk, dpos, None, dwq, dwk, None, None


_norm_rotate_backward_once = once_differentiable(_norm_rotate_backward)


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, wq, wk, eps, neighbors):
        ctx.save_for_backward(q, k, positions, frequencies, wq, wk)
        ctx.rest = eps, neighbors
        ctx.set_materialize_grads(False)
        return _norm_rotate_forward(q, k, positions, frequencies, wq, wk, eps, neighbors)

    @staticmethod
    def backward(ctx, gq, gk):
        return _norm_rotate_backward_once(ctx, gq, gk) if torch.is_grad_enabled() else _norm_rotate_backward(ctx, gq, gk)


def norm_rotate(q, k=None, positions=None, frequencies=None, *, q_weight=None, k_weight=None, eps=1e-6, pairing="halves"):
    """(q, k) normalised per head and rotated by the rows' positions, in one pass.

    Norm, where weights (d) are given (both sides or neither; float32 or the rows' type): weight * x / sqrt(mean(x^2) + eps).
    Rotation, where positions (n, axes) float32 or float64 and frequencies (axes, d / 2) float32 are given: pair p of a head turns by
    theta_p = sum_a positions[:, a] frequencies[a, p], formed in float64; pairs are (p, p + d / 2) ("halves") or (2p, 2p + 1)
    ("neighbors").  The product of two rotated rows then depends on the difference of their positions only.  q (n, heads, d) and
    k (n, heads_k, d), or None, float32, bfloat16 or float16 on one GPU, d a multiple of 16 up to 256, any strides.  Gradients: q, k, positions and the
    weights (frequencies and eps are constants).  Returns new (q, k), contiguous."""
    _first(q)
    n, _, d = q.shape
    dtype, device = q.dtype, q.device
    if k is not None:
        _head_rows("k", k, dtype, device, d)
        if k.shape[0] != n:
            raise ValueError(f"q has {n} rows, k {k.shape[0]}")
    if d % 16 or not 16 <= d <= 256:
        raise ValueError(f"d must be a multiple of 16 up to 256, not {d}")
    if n > 2**31 - 2**20:
        raise ValueError(f"q has {n} rows; at most 2**31 - 2**20 are supported")
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
        if positions.ndim != 2 or positions.shape[0] != n or not 1 <= positions.shape[1] <= 16 or positions.device != device or \
                positions.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"positions must be ({n}, axes) float32 or float64 on {device}, not {tuple(positions.shape)} {positions.dtype} "
                             f"on {positions.device}")
        if frequencies.shape != (positions.shape[1], d // 2) or frequencies.dtype != torch.float32 or frequencies.device != device:
            raise ValueError(f"frequencies must be ({positions.shape[1]}, {d // 2}) float32 on {device}, not {tuple(frequencies.shape)} "
                             f"{frequencies.dtype} on {frequencies.device}")
        if frequencies.requires_grad and torch.is_grad_enabled():
            raise ValueError("frequencies are constants: no gradient is formed for them")
        positions, frequencies = positions.contiguous(), frequencies.contiguous()
    if norm:
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None and (w.shape != (d,) or w.device != device or w.dtype not in (torch.float32, dtype) or w.dtype != q_weight.dtype):
                raise ValueError(f"{name} must be ({d},) float32 or {dtype} on {device}, both sides alike, not {tuple(w.shape)} {w.dtype} on {w.device}")
        q_weight, k_weight = q_weight.contiguous(), None if k_weight is None else k_weight.contiguous()
    _no_tangents("norm_rotate", q, k, positions, frequencies, q_weight, k_weight, eps)
    eps = _constant("eps", eps)
    if not 0 <= eps < math.inf:
        raise ValueError(f"eps must not be negative, not {eps}")
    unit = _UNIT[dtype]
    q, k = _aligned(q, unit), None if k is None else _aligned(k, unit)
    args = (q, k, positions, frequencies, q_weight, k_weight, eps, pairing == "neighbors")
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad) or (positions is not None and positions.requires_grad) or
                                    (norm and (q_weight.requires_grad or (k_weight is not None and k_weight.requires_grad)))):
        return _NormRotate.apply(*args)
    return _norm_rotate_forward(*args)
