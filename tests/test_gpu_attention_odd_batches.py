"""Batches that mix what the kernels are chosen by: many short structures beside a long one, many heads, sides without rows."""
import ctypes as C

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200 import PackedStructures, structure_attention  # noqa: E402
from so3lr_b200._lib import Rows, lib  # noqa: E402
from test_gpu_attention_cotangents import check  # noqa: E402
from test_gpu_structure_attention import TYPES, inputs, reference, starts, train, within  # noqa: E402


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("longest", [49, 230, 610])
def test_many_short_structures_beside_a_long_one(longest, dtype):
    rng = np.random.default_rng(longest)
    lengths = rng.integers(10, 41, 120).tolist()
    lengths.insert(70, longest)
    q, k, v, g = inputs(lengths, lengths, 4, 4, 32, TYPES[dtype], seed=longest)
    packed = PackedStructures(starts(lengths))
    val, err = reference(q, k, v, g, lengths, lengths, False, 32 ** -0.5, q.dtype)
    got = train(q, k, v, g, packed)
    within(got, val, err)
    for x, y in zip(got, train(q, k, v, g, packed)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("lengths,hq,hk", [([40, 21], 130, 65), ([150, 33], 130, 65), ([30, 140], 96, 3), ([17, 90], 1, 1)])
def test_many_heads_in_float16(lengths, hq, hk):
    n = sum(lengths)
    sizes = 10.0 ** (-4 * torch.rand(1, hk, 1, generator=torch.Generator().manual_seed(hk))).repeat_interleave(hq // hk, 1).expand(n, hq, 1)
    check(lengths, hq, hk, 64, False, sizes.cuda())


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lq,lk", [([0, 0, 0], [4, 0, 300]), ([4, 0, 300], [0, 0, 0]), ([0, 5, 200], [200, 0, 0])])
def test_a_side_without_rows_whatever_memory_holds(lq, lk, dtype):
    """Gradients of rows that meet nothing are zero; the workspace starts as anything."""
    hq, hk, d = 4, 2, 64
    q, k, v, g = inputs(lq, lk, hq, hk, d, TYPES[dtype], seed=1)
    packed = PackedStructures(starts(lq), starts(lk))
    shape, _, size = packed._call(q, k, None)
    rows = lambda t: C.byref(Rows(t.data_ptr(), t.stride(0), t.stride(1)))
    for word in (0, -1, 0x7F7F7F7F, 0x22D00000, 0x55555555):      # 0x22D00000: 2^-57.3, twice whose square is 2^-113.6
        work = torch.full((max(size, 4) // 4 + 1,), word, dtype=torch.int32, device="cuda")
        out, rest, lse = torch.zeros_like(q), None if dtype == "f32" else torch.zeros_like(q), torch.full((hq, len(q)), -float("inf"), device="cuda")
        d_ = [torch.full_like(x, 777.0) for x in (q, k, v)]
        assert lib.so3lr_b200_structure_attention_vjp(packed._host, packed._dev_ptr, packed._stream(), shape, rows(q), rows(k), rows(v), out.data_ptr(),
                                                      0 if rest is None else rest.data_ptr(), lse.data_ptr(), rows(g), torch.empty_like(lse).data_ptr(),
                                                      *(x.data_ptr() for x in d_), work.data_ptr(), size) == 0
        assert all((x == 0).all() for x in d_), hex(word)
    assert all((x == 0).all() for x in train(q, k, v, g, packed))
    assert (structure_attention(q, k, v, packed) == 0).all()


@pytest.mark.parametrize("d,lengths", [(64, [85, 40]), (32, [300]), (128, [60, 71]), (64, [150]), (128, [400])])
@pytest.mark.parametrize("rising", [True, False])
def test_gradients_that_grow_along_the_walk(d, lengths, rising):
    """float16: cotangents and values over five powers of ten from the first row to the last, or the other way; some rows without any."""
    n = sum(lengths)
    t = torch.linspace(0, 1, n, device="cuda") if rising else torch.linspace(1, 0, n, device="cuda")
    sizes = (10.0 ** (5 * t - 3))[:, None, None].clone()
    sizes[:7] = 0.0
    check(lengths, 2, 1, d, False, sizes, v_size=(10.0 ** (3 * t - 2))[:, None, None], qk_size=0.3)
    check(lengths, 2, 2, d, True, sizes, v_size=(10.0 ** (3 * t - 2))[:, None, None], qk_size=0.3)
