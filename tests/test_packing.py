"""Layouts of packed structures (host side of so3lr_b200.attention): work items cover every row once, what is refused. No GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from so3lr_b200 import attention as A
from so3lr_b200._lib import AttentionShape, NormRotateArgs, Rows, lib



def image(lq, lk, causal):
    sq, sk = (np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (lq, lk))
    p = [x.ctypes.data_as(C.c_void_p) for x in (sq, sk)]
    size = lib.so3lr_b200_packing_size(len(lq), *p)
    assert size > 0
    im = np.full(size + 8, -7, np.int32)
    assert lib.so3lr_b200_packing_build(len(lq), *p, int(causal), im.ctypes.data_as(C.c_void_p), size) == 0
    assert np.all(im[size:] == -7)
    return im[:size]


def items(im, at, n):
    return im[im[at]:im[at] + 4 * im[n]].reshape(-1, 4)


LAYOUTS = [([0], [0]), ([1], [1]), ([64], [64]), ([65, 0, 63], [65, 0, 63]), ([3, 70, 129], [200, 0, 65]), ([1] * 5, [17, 0, 513, 1024, 4000]),
           ([130, 5], [3, 1]), ([32, 0, 17, 5], [16, 3, 32, 1])]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", LAYOUTS)
def test_items_cover_what_is_allowed(lq, lk, causal):
    im = image(lq, lk, causal)
    allowed = [np.arange(b)[None, :] <= np.arange(a)[:, None] + (b - a) if causal else np.ones((a, b), bool) for a, b in zip(lq, lk)]
    # query tiles: once each, and the keys of a tile reach as far as any of its rows sees, no further
    short = max(lq + lk) <= 48          # tables of 16 rows only where all structures are short
    for at, n, tile in ((8, 9, 64), (17, 18, 128), (19, 20, 256)) + (((29, 30, 16),) if short else ()):
        seen = set()
        rows = items(im, at, n)
        assert np.all(np.diff(rows[:, 3] - rows[:, 2]) <= 0)          # the longest first
        for s, t, first, last in rows:
            assert (s, t) not in seen and first == 0
            seen.add((s, t))
            cols = allowed[s][t * tile:(t + 1) * tile].any(0)
            assert last == (cols.nonzero()[0].max() + 1 if cols.any() else 0)
        assert len(seen) == sum(-(-a // tile) for a in lq)
    # key tiles
    assert short or im[30] == im[32] == 0
    for at, n, tile in ((10, 11, 64), (21, 22, 128)) + (((31, 32, 16),) if short else ()):
        seen = set()
        for s, t, first, last in items(im, at, n):
            assert (s, t) not in seen and last == lq[s]
            seen.add((s, t))
            r = allowed[s][:, t * tile:(t + 1) * tile].any(1)
            assert first == (r.nonzero()[0].min() if r.any() else lq[s])
        assert len(seen) == sum(-(-b // tile) for b in lk)
    # stretches of the keys: disjoint, in order, all keys, and at least one item per structure with queries
    first_of = im[im[14]:im[14] + len(lq) + 1]
    split = items(im, 12, 13)
    for s, (a, b) in enumerate(zip(lq, lk)):
        mine = split[first_of[s]:first_of[s + 1]]
        assert len(mine) == 0 if a == 0 else np.all(mine[:, 0] == s) and np.all(mine[:, 1] == len(mine)) and mine[0, 2] == 0 and mine[-1, 3] == b
        assert np.all(mine[1:, 2] == mine[:-1, 3])
    assert im[13] == first_of[-1] and im[15] == int(len(split) > sum(a > 0 for a in lq)) and im[5] == max(lq) and im[23] == max(lk)


def test_refused_layouts():
    for sq, sk in (([1, 2], [0, 2]), ([0, 2], [1, 2]), ([0, 3, 2], [0, 1, 2]), ([0, 1, 2], [0, 2, 1])):
        sq, sk = np.asarray(sq, np.int32), np.asarray(sk, np.int32)
        assert lib.so3lr_b200_packing_size(len(sq) - 1, sq.ctypes.data_as(C.c_void_p), sk.ctypes.data_as(C.c_void_p)) == -1
    z = np.zeros(1, np.int32).ctypes.data_as(C.c_void_p)
    assert lib.so3lr_b200_packing_size(0, z, None) == -1 and lib.so3lr_b200_packing_size(-1, z, z) == -1
    buf = np.zeros(4, np.int32)
    assert lib.so3lr_b200_packing_build(0, z, z, 0, buf.ctypes.data_as(C.c_void_p), 4) == 1          # too small an image
    for bad in ([1, 2], [0, 3, 2], [[0, 1]], [0.0, 1.0], [], [0, 2**31]):
        with pytest.raises(ValueError):
            A.PackedStructures(bad)
    with pytest.raises(ValueError):
        A.PackedStructures([0, 2], [0, 1, 2])
    with pytest.raises(ValueError):
        A.PackedStructures([0, 2], device="cpu")


def test_refused_calls_at_the_c_entry():
    """Arguments that are checked ahead of any launch: status 1, nothing runs (the pointers are never followed)."""
    im = image([5], [5], False)
    h = im.ctypes.data_as(C.c_void_p)
    fake = 1 << 20
    good = dict(type=0, heads_q=4, heads_kv=2, d=32, rows_q=5, rows_kv=5, scale=1.0)
    r = Rows(fake, 128, 32)

    def call(shape=None, q=r, image=h, dev=fake, out=fake):
        s = AttentionShape(**{**good, **(shape or {})})
        a = (image, dev, None, C.byref(s), C.byref(q) if q else None, C.byref(r), C.byref(r))
        return {lib.so3lr_b200_structure_attention(*a, out, None, None, None, 0),
                lib.so3lr_b200_structure_attention_vjp(*a, out, None, fake, C.byref(q) if q else None, fake, out, fake, fake, None, 0)}

    for bad in (dict(type=3), dict(type=-1), dict(heads_q=3), dict(heads_kv=0), dict(heads_q=0), dict(d=24), dict(d=8), dict(d=144), dict(rows_q=4),
                dict(rows_kv=4), dict(rows_q=2**31), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        assert call(bad) == {1}, bad
    assert call(q=None) == {1} and call(q=Rows(fake + 4, 128, 32)) == {1} and call(q=Rows(fake, 126, 32)) == {1} and call(q=Rows(fake, 128, 2)) == {1}
    assert call(q=Rows(None, 128, 32)) == {1} and call(image=None) == {1} and call(dev=None) == {1} and call(out=None) == {1}
    other = im.copy()
    other[0] += 1
    assert call(image=other.ctypes.data_as(C.c_void_p)) == {1}

    good_r = dict(n=5, d=32, heads_q=4, heads_k=2, type=0, axes=1, neighbors=0, norm=1, weights_f32=1, positions_f64=0, eps=1e-6, positions=fake,
                  frequencies=fake, weight_q=fake, weight_k=fake)
    for bad in (dict(n=-1), dict(d=24), dict(d=8), dict(d=272), dict(type=3), dict(axes=17), dict(axes=-1), dict(positions=None), dict(frequencies=None),
                dict(heads_q=-1), dict(weight_q=None), dict(weight_k=None)):
        a = NormRotateArgs(**{**good_r, **bad})
        assert lib.so3lr_b200_norm_rotate(None, C.byref(a), C.byref(r), C.byref(r), fake, fake) == 1, bad
        assert lib.so3lr_b200_norm_rotate_vjp(None, C.byref(a), C.byref(r), C.byref(r), C.byref(r), C.byref(r), fake, fake, fake, fake, fake, fake, 1 << 30) == 1
    a = NormRotateArgs(**good_r)
    assert lib.so3lr_b200_norm_rotate(None, C.byref(a), None, C.byref(r), fake, fake) == 1
    assert lib.so3lr_b200_norm_rotate(None, C.byref(a), C.byref(r), C.byref(r), None, fake) == 1
    assert lib.so3lr_b200_norm_rotate_vjp(None, C.byref(a), C.byref(r), C.byref(r), C.byref(r), C.byref(r), fake, fake, fake, fake, fake, None, 0) == 1


def test_rows_must_be_on_a_gpu():
    q = torch.zeros(3, 2, 32)
    for bad in (q, q.double(), q[0], None, [1.0]):
        with pytest.raises(ValueError):
            A.structure_attention(bad, q, q, None)
        with pytest.raises(ValueError):
            A.norm_rotate(bad, q, q_weight=torch.ones(32), k_weight=torch.ones(32))
