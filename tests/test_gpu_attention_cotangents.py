"""Gradients of structure_attention in float16 for cotangents of any size, against the formula in 64 bits.

float16 has 11 bits down to 2^-14 and steps of 2^-24 below; a mean loss has cotangents of 1e-3 and less, a scaled one of 1e3 and more.  The kernels
form dS times a power of two (on the tensor cores a query row's own ahead of dS k, one of a structure and key head ahead of dS^T q) that brings
2 |g| sqrt(d) max |v_jc|, which no |dS| passes, between 2^14 and 2^15 (the warp-level ones: the largest |dS| so far).  So dS is off by 2^-11 of itself and by 2^-25 of that scale: 2^-38 of
|g| sqrt(d) max |v_jc|.
Bounds otherwise, with u = 2^-11: logits are off by (d + 4) 2^-24 of sum |q||k| (times scale: e), probabilities by 3 max e + 2^-20 + L 2^-24, o by a
rounding of P (u, and 2^-25 of the row's largest one) and of the result with its rest (2^-22 |o|, or half a step of 2^-24), delta by that times
|g|, dP by (d + 4) 2^-24 of sum |g||v|; a result is rounded once, to 2^-11 of itself or half a step.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200.attention import PackedStructures, structure_attention  # noqa: E402

U, F32 = 2.0 ** -11, 2.0 ** -24


def reference(q, k, v, g, starts, causal):
    """(values, bounds) of dq, dk, dv in float64."""
    q, k, v, g = (x.double() for x in (q, k, v, g))
    hq, hk, d = q.shape[1], k.shape[1], q.shape[2]
    scale, group = d ** -0.5, hq // hk
    val, err = [torch.zeros_like(x) for x in (q, k, v)], [torch.zeros_like(x) for x in (q, k, v)]
    for a, b in zip(starts[:-1], starts[1:]):
        n = int(b - a)
        for h in range(hq if n else 0):
            j = h // group
            Q, K, V, G = q[a:b, h], k[a:b, j], v[a:b, j], g[a:b, h]
            ok = torch.ones(n, n, dtype=torch.bool, device=q.device)
            if causal:
                ok = ok.tril()
            P = torch.softmax((scale * Q @ K.T).masked_fill(~ok, -float("inf")), -1)
            O, dP = P @ V, G @ V.T
            dS = P * (dP - (G * O).sum(-1, keepdim=True))
            e = scale * (Q.abs() @ K.abs().T) * (d + 4) * F32
            rel = 3 * torch.where(ok, e, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 + n * F32
            eO = ((rel + U + n * F32) * P + 2.0 ** -25 * ok) @ V.abs() + 2.0 ** -22 * O.abs() + 2.0 ** -25
            edelta = (G.abs() * (eO + O.abs() * (d + 4) * F32)).sum(-1, keepdim=True)
            edP = (G.abs() @ V.abs().T) * (d + 4) * F32
            eS = P * (edP + edelta) * (1 + rel) + rel * dS.abs() * 1.01 + (U + n * F32) * dS.abs()
            size = 2.0 ** -38 * d ** 0.5 * V.abs().amax()
            top = g[a:b, j * group:(j + 1) * group].norm(dim=-1).amax()
            val[0][a:b, h] += scale * dS @ K
            err[0][a:b, h] += scale * (eS * (1 + U) + size * G.norm(dim=-1, keepdim=True) * ok) @ K.abs()
            val[1][a:b, j] += scale * dS.T @ Q
            err[1][a:b, j] += scale * (eS * (1 + U) + size * top * ok).T @ Q.abs()
            val[2][a:b, j] += P.T @ G
            err[2][a:b, j] += ((rel + U + n * hq * F32) * P).T @ G.abs()
    return val, [x * 1.01 + U * (y.abs() + x) + 2.0 ** -25 for x, y in zip(err, val)]


def check(lengths, hq, hk, d, causal, sizes, v_size=1.0, qk_size=1.0, seed=0):
    """sizes: number or tensor that broadcasts against the cotangent."""
    starts = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    n = int(starts[-1])
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v = (normal(n, hq, d) * qk_size).half(), (normal(n, hk, d) * qk_size).half(), (normal(n, hk, d) * v_size).half()
    g = (normal(n, hq, d) * sizes).half()
    assert torch.isfinite(g).all()
    val, err = reference(q, k, v, g, starts, causal)
    leaf = [x.detach().requires_grad_() for x in (q, k, v)]
    packed = PackedStructures(starts, causal=causal)
    got = torch.autograd.grad(structure_attention(*leaf, packed), leaf, g)
    again = torch.autograd.grad(structure_attention(*leaf, packed), leaf, g)
    for name, x, y, z, e in zip(("dq", "dk", "dv"), got, again, val, err):
        assert torch.equal(x, y), name
        assert (z.abs() <= 6e4).all(), "the result has to fit float16"
        off = (x.double() - z).abs()
        assert (off <= e).all(), f"{name}: {float((off / e).max()):.3g} times the bound"
        # altogether: where the result holds its digits, well inside of what the roundings of dS and of the result add up to
        big = z.abs() >= 2.0 ** -14
        if big.any():
            assert (off[big].norm() <= 2 * U * z[big].norm()).all(), f"{name}: {float(off[big].norm() / z[big].norm()):.3g}"
    return got


LONG = ([2048], 2, 1, 64, False), ([700, 0, 301, 1], 2, 2, 128, True), ([400, 90], 4, 2, 32, False)      # tensor cores
SHORT = ([40, 7, 0, 21], 4, 2, 64, False), ([60, 65, 1], 2, 1, 112, True), ([12, 3], 2, 2, 16, False), ([300], 2, 2, 32, True)      # warp-level


@pytest.mark.parametrize("size", [1e-5, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize("lengths,hq,hk,d,causal", LONG + SHORT)
def test_cotangents_of_any_size(lengths, hq, hk, d, causal, size):
    check(lengths, hq, hk, d, causal, size, seed=d)


@pytest.mark.parametrize("lengths,d", [([30, 5, 2], 128), ([500], 128), ([20], 64), ([300], 64)])
def test_logits_gradients_beyond_the_type(lengths, d):
    # dS passes float16's 65504, the gradients do not
    check(lengths, 2, 1, d, True, 300.0, v_size=100.0, qk_size=0.2)


@pytest.mark.parametrize("lengths,d", [([130, 200, 90], 64), ([20, 33, 9], 64), ([150, 100], 128)])
def test_cotangents_of_different_sizes_side_by_side(lengths, d):
    gen = torch.Generator().manual_seed(3)
    n, hq, hk = sum(lengths), 4, 2
    # from structure to structure, and key head to key head
    sizes = torch.cat([torch.full((m, 1, 1), 10.0 ** (2 - 3 * i)) for i, m in enumerate(lengths)]) * torch.tensor([1.0, 1.0, 1e-2, 1e-2])[None, :, None]
    check(lengths, hq, hk, d, False, sizes.cuda())
    # from row to row
    sizes = 10.0 ** (-4 * torch.rand(n, hq, 1, generator=gen))
    check(lengths, hq, hk, d, True, sizes.cuda())


@pytest.mark.parametrize("lengths", [[200, 130], [30, 20]])
def test_no_cotangent_and_values_that_are_not_finite(lengths):
    hq, hk, d, n = 2, 1, 64, sum(lengths)
    check(lengths, hq, hk, d, False, torch.zeros(n, 1, 1, device="cuda"))
    got = check(lengths, hq, hk, d, False, torch.full((n, 1, 1), 1e-3, device="cuda"))
    # one in the first structure: the second one's gradients keep their bits
    gen = torch.Generator(device="cuda").manual_seed(0)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    q, k, v, g = normal(n, hq, d).half(), normal(n, hk, d).half(), normal(n, hk, d).half(), (normal(n, hq, d) * 1e-3).half()
    packed = PackedStructures([0, lengths[0], n])
    for spoiled in ("v", "g"):
        for bad in (float("inf"), float("nan")):
            x = {"v": v.clone(), "g": g.clone()}
            x[spoiled][3, 0, 5] = bad
            leaf = [t.detach().requires_grad_() for t in (q, k, x["v"])]
            new = torch.autograd.grad(structure_attention(*leaf, packed), leaf, x["g"])
            for a, b in zip(new, got):
                assert torch.equal(a[lengths[0]:], b[lengths[0]:])
