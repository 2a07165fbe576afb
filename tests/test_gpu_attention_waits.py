"""What a call of structure_attention leaves and tells when a bounded wait of its tensor-core kernels runs out.

With a negative count of tries the loading warps give up where a barrier is not over at once.  Every row then is NaN or right, none is left as it was,
and the next call on the device says so, once."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200 import PackedStructures, structure_attention  # noqa: E402
from so3lr_b200._lib import Rows, So3lrB200Error, lib  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BEFORE = 777.0


class _Tries:
    def __init__(self, tries):
        self.tries = tries

    def __enter__(self):
        self.before = lib.so3lr_b200_host_wait_tries(self.tries)

    def __exit__(self, *_):
        torch.cuda.synchronize()
        lib.so3lr_b200_host_wait_tries(self.before)


def _rows(t):
    return C.byref(Rows(t.data_ptr(), t.stride(0), t.stride(1)))


def _error():
    word = C.c_int(-1)
    assert lib.so3lr_b200_structure_attention_error(C.byref(word)) == 0
    return word.value


def _inputs(lengths, hq, hk, d, dtype, seed=0):
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = int(starts[-1])
    return starts, [torch.randn(n, h, d, generator=gen, device="cuda").to(TYPES[dtype]) for h in (hq, hk, hk, hq)]


def _forward(packed, shape, size, q, k, v, out, rest, lse):
    work = torch.full((max(size, 1),), 0x55, dtype=torch.uint8, device="cuda")
    return lib.so3lr_b200_structure_attention(packed._host, packed._dev_ptr, packed._stream(), shape, _rows(q), _rows(k), _rows(v), out.data_ptr(),
                                              0 if rest is None else rest.data_ptr(), lse.data_ptr(), work.data_ptr(), size)


def _backward(packed, shape, size, q, k, v, out, rest, lse, g, dq, dk, dv):
    work, delta = torch.full((max(size, 1),), 0x55, dtype=torch.uint8, device="cuda"), torch.empty_like(lse)
    return lib.so3lr_b200_structure_attention_vjp(packed._host, packed._dev_ptr, packed._stream(), shape, _rows(q), _rows(k), _rows(v), out.data_ptr(),
                                                  0 if rest is None else rest.data_ptr(), lse.data_ptr(), _rows(g), delta.data_ptr(), dq.data_ptr(),
                                                  dk.data_ptr(), dv.data_ptr(), work.data_ptr(), size)


def _right_or_nan(got, want):
    """Returns how many values are NaN."""
    nan = torch.isnan(got)
    assert torch.equal(got[~nan], want[~nan])
    return int(nan.sum())


CASES = [
    # one tile a CTA from a queue, two tiles from a queue, float32 (one and two tiles), walks in pieces, structures without keys among many
    ("bf16", [300, 257, 640, 5, 0, 400] * 12, 8, 4, 64, False), ("f16", [300, 257, 640, 5, 0, 400] * 12, 8, 4, 32, True),
    ("bf16", [900, 1300, 257, 0, 1], 16, 8, 128, True), ("f16", [1025], 1, 1, 112, False), ("f32", [300, 500, 20] * 8, 4, 4, 32, False),
    ("f32", [2100, 300], 4, 2, 32, True), ("f32", [300, 500, 20], 4, 2, 64, True),
]


@pytest.mark.parametrize("dtype,lengths,hq,hk,d,causal", CASES)
def test_waits_that_run_out(dtype, lengths, hq, hk, d, causal):
    starts, (q, k, v, g) = _inputs(lengths, hq, hk, d, dtype)
    packed = PackedStructures(starts, causal=causal)
    leaf = [x.clone().requires_grad_() for x in (q, k, v)]
    want = structure_attention(*leaf, packed)
    grads = torch.autograd.grad(want, leaf, g)
    want = want.detach()
    shape, size, size_vjp = packed._call(q, k, None)
    rest = None if dtype == "f32" else torch.empty_like(q)
    lse = torch.full((hq, len(q)), BEFORE, device="cuda")
    out = torch.full_like(q, BEFORE)
    good = out.clone(), None if rest is None else rest.clone(), lse.clone()
    assert _forward(packed, shape, size, q, k, v, *good) == 0 and torch.equal(good[0], want) and _error() == 0

    with _Tries(-1):
        assert _forward(packed, shape, size, q, k, v, out, rest, lse) == 0          # nothing is known of it yet
        torch.cuda.synchronize()
        held = out.clone()
        assert _forward(packed, shape, size, q, k, v, out, rest, lse) == 6          # told, and not run
        torch.cuda.synchronize()
        assert torch.equal(torch.nan_to_num(out), torch.nan_to_num(held)) and not (out == BEFORE).any() and not (lse == BEFORE).any()
        assert _right_or_nan(out, want) > 0 and _error() == 0                       # told once
        d_ = [torch.full_like(x, BEFORE) for x in (q, k, v)]
        assert _backward(packed, shape, size_vjp, q, k, v, *good, g, *d_) == 0
        torch.cuda.synchronize()
        assert _error() == 1 and _error() == 0
    for x, y in zip(d_, grads):
        assert not (x == BEFORE).any() and _right_or_nan(x, y) > 0

    # as it was before
    again = structure_attention(*leaf, packed)
    assert torch.equal(again, want) and all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(again, leaf, g), grads))
    assert _error() == 0


def test_the_next_call_raises():
    starts, (q, k, v, g) = _inputs([300, 400], 4, 2, 64, "bf16")
    packed = PackedStructures(starts)
    want = structure_attention(q, k, v, packed)
    with _Tries(-1):
        out = structure_attention(q, k, v, packed)
    assert torch.isnan(out).any()
    short = PackedStructures([0, 20])
    with pytest.raises(So3lrB200Error, match="wait"):            # whatever the next call is
        structure_attention(q[:20], k[:20], v[:20], short)
    assert torch.isfinite(structure_attention(q[:20], k[:20], v[:20], short)).all() and torch.equal(structure_attention(q, k, v, packed), want)
    # in a backward pass as well
    leaf = q.clone().requires_grad_()
    out = structure_attention(leaf, k, v, packed)
    with _Tries(-1):
        (dq,) = torch.autograd.grad(out, leaf, g, retain_graph=True)
    assert torch.isnan(dq).any()
    with pytest.raises(So3lrB200Error, match="wait"):
        torch.autograd.grad(out, leaf, g, retain_graph=True)
    (dq,) = torch.autograd.grad(out, leaf, g)
    assert torch.isfinite(dq).all()


def test_a_captured_call():
    """A graph whose kernels gave up tells the next plain call, and its other replays are right."""
    starts, (q, k, v, _) = _inputs([300, 400], 4, 2, 64, "bf16")
    packed = PackedStructures(starts)
    want = structure_attention(q, k, v, packed)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with _Tries(-1):
        with torch.cuda.graph(graph):
            out = structure_attention(q, k, v, packed)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.isnan(out).any() and _error() == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = structure_attention(q, k, v, packed)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and _error() == 0
