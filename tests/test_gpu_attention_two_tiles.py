"""The forward kernels whose CTAs work on two tiles of 128 queries (16-bit rows of more than 64 values from 800 keys on, float32 rows of up to 32 from
2,048 on) against the formula, with the bounds of test_gpu_structure_attention."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200.attention import PackedStructures, structure_attention  # noqa: E402
from test_gpu_structure_attention import TYPES, inputs, no_wait_ran_out, reference, starts, train, within  # noqa: E402

CASES = [
    # 16 bits: more jobs than SMs, with tiles of both kinds of count (an odd number of tiles, keys that only the second tile sees)
    ("bf16", [900, 1300, 257, 0, 1, 815, 130], None, 32, 8, 128, True), ("f16", [900, 1300, 257, 0, 1, 815, 130], None, 32, 8, 128, True),
    ("bf16", [900, 1300, 257, 0, 1], None, 24, 24, 112, False), ("f16", [1024, 385, 2], None, 40, 8, 80, True),
    # few jobs: walks cut into pieces
    ("bf16", [1300], None, 1, 1, 128, True), ("f16", [2100, 900], None, 2, 1, 112, False), ("bf16", [3000], None, 1, 1, 96, False),
    # other keys than queries: rows without keys, tiles of rows without keys, more keys than rows
    ("bf16", [900, 100, 300, 0, 128], [200, 1500, 300, 70, 0], 8, 2, 128, True), ("f16", [1000, 257], [100, 2000], 8, 4, 128, True),
    ("bf16", [129, 256], [900, 1111], 4, 4, 128, False),
    # float32
    ("f32", [2100, 300], None, 4, 2, 32, True), ("f32", [2100, 300, 0, 1], None, 2, 2, 32, False), ("f32", [2561], None, 12, 4, 16, True),
    ("f32", [600, 257], [2300, 40], 4, 1, 32, True), ("f32", [2049, 500], [300, 2048], 2, 2, 32, True),
]


@pytest.mark.parametrize("dtype,lq,lk,hq,hk,d,causal", CASES)
def test_two_tiles_against_the_formula(dtype, lq, lk, hq, hk, d, causal):
    lk = lq if lk is None else lk
    q, k, v, g = inputs(lq, lk, hq, hk, d, TYPES[dtype], seed=len(lq) + d, extra=2)
    packed = PackedStructures(starts(lq), starts(lk), causal=causal)
    n, m = sum(lq), sum(lk)
    got = train(q, k, v, g, packed)
    val, err = reference(q, k, v, g, lq, lk, causal, d ** -0.5, q.dtype)
    within(got, val, err)
    assert all((x[rows:] == 0).all() for x, rows in zip(got, (n, n, m, m)))
    assert torch.equal(structure_attention(q, k, v, packed), got[0])
    for x, y in zip(got, train(q, k, v, g, packed)):
        assert torch.equal(x, y)
    no_wait_ran_out()
