"""float16 attention where one key takes nearly all of a row's probability and has little to say: the output is the sum of what is left.

The probabilities are formed relative to a reference near the row's largest logit, times a power of two that keeps the largest below 2^16: off by
2^-11 of themselves, and by half of float16's smallest step, which is 2^-36 of the row's largest where the reference may lag four powers of two
behind (tensor cores), and 2^-40 else: 2^-36 below.  Other terms as in test_gpu_structure_attention."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200 import PackedStructures, structure_attention  # noqa: E402

U, F32 = 2.0 ** -11, 2.0 ** -24
CASES = [
    # lq, lk (None: the same), heads, key heads, d, causal: tensor cores (one tile, two, in pieces), warp-level, single queries (narrow, wide, one stretch)
    ([700, 300], None, 4, 2, 64, False), ([900, 1300], None, 16, 8, 128, True), ([2100], None, 1, 1, 112, False), ([4096], None, 2, 1, 32, True),
    ([100, 60], None, 4, 2, 64, False), ([40, 17], None, 4, 4, 32, False), ([150], None, 1, 1, 16, True), ([1] * 3, [5000, 700, 40], 8, 2, 128, True),
    ([3, 16], [4097, 900], 8, 2, 64, False), ([8], [60], 8, 1, 96, False),
]


@pytest.mark.parametrize("gap", [14.5, 19.5, 23.5, 24.5])
@pytest.mark.parametrize("lq,lk,hq,hk,d,causal", CASES)
def test_one_key_takes_it_all(lq, lk, hq, hk, d, causal, gap):
    """gap: of the first key's logit over the others', as a power of two of the probability."""
    lk = lq if lk is None else lk
    starts = [np.concatenate([[0], np.cumsum(x)]).astype(np.int32) for x in (lq, lk)]
    gen = torch.Generator(device="cuda").manual_seed(int(gap) + d)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v = normal(sum(lq), hq, d) * 0.05, normal(sum(lk), hk, d) * 0.05, 100 + 10 * normal(sum(lk), hk, d)
    q[..., 0], k[..., 0] = 4.0, 0.0
    first = torch.as_tensor(starts[1][:-1].astype(np.int64))
    k[first, :, 0], v[first] = gap / 1.4426950408889634 * d ** 0.5 / 4.0, 0.0
    q, k, v = q.half(), k.half(), v.half()
    out = structure_attention(q, k, v, PackedStructures(*starts, causal=causal))
    for a, b, c, e in zip(starts[0][:-1], starts[0][1:], starts[1][:-1], starts[1][1:]):
        n, m = int(b - a), int(e - c)
        ok = torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n) if causal else torch.ones(n, m, dtype=torch.bool, device="cuda")
        for h in range(hq):
            Q, K, V = q[a:b, h].double(), k[c:e, h // (hq // hk)].double(), v[c:e, h // (hq // hk)].double()
            P = torch.softmax((d ** -0.5 * Q @ K.T).masked_fill(~ok, -float("inf")), -1)
            O = P @ V
            logit = d ** -0.5 * (Q.abs() @ K.abs().T) * (d + 4) * F32
            rel = 3 * torch.where(ok, logit, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 + m * F32
            # the logits refer to a number of their size: its rounding, and that of a product with log2(e)
            rel = rel + 2 * gap * F32
            bound = (((rel + U + m * F32) * P + 2.0 ** -36 * ok) @ V.abs()) * 1.01 + U * O.abs() * 1.01 + 2.0 ** -25
            off = (out[a:b, h].double() - O).abs()
            assert (off <= bound).all(), f"{float((off / bound).max()):.3g} times the bound, {float((off / O.clamp(min=1e-9)).max()):.3g} of the value"


def test_their_gradients():
    """dv holds 2^15 P, and dS its own power of two: nothing of the rows' tails is lost there."""
    n, d = 600, 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v, g = normal(n, 1, d) * 0.05, normal(n, 1, d) * 0.05, 10 * normal(n, 1, d), 100 * normal(n, 1, d)
    q[..., 0], k[..., 0] = 4.0, 0.0
    k[0, :, 0], v[0] = 20 / 1.4426950408889634 * d ** 0.5 / 4.0, 0.0
    leaf = [x.half().requires_grad_() for x in (q, k, v)]
    out = structure_attention(*leaf, PackedStructures([0, n]))
    dq, dk, dv = torch.autograd.grad(out, leaf, g.half())
    Q, K, V = (x.detach()[:, 0].double().requires_grad_() for x in leaf)
    O = torch.softmax(d ** -0.5 * Q @ K.T, -1) @ V
    want = torch.autograd.grad(O, (Q, K, V), g.half()[:, 0].double())
    # keys other than the first: dv = 2^-20 of 600 cotangents of 100, in steps of 2^-24 where it is small
    off = (dv[1:, 0].double() - want[2][1:]).abs()
    assert (off <= 4 * U * want[2][1:].abs().amax() + 2.0 ** -25).all()
    assert ((dq[:, 0].double() - want[0]).abs() <= 8 * U * want[0].abs().amax() + 2.0 ** -25).all()
