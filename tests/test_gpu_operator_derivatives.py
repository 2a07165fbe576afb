"""Derivatives that the operators on packed structures do not form are refused, none is dropped without a word."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu

from so3lr_b200 import PackedStructures, norm_rotate, structure_attention  # noqa: E402


def _rows(n=12, h=2, d=32):
    gen = torch.Generator(device="cuda").manual_seed(1)
    normal = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    return normal(n, h, d), normal(n, h, d), normal(n, h, d), normal(n, 3), normal(3, d // 2), normal(d)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(3))
def test_forward_mode_of_attention(which, grad):
    q, k, v, *_ = _rows()
    packed = PackedStructures([0, 5, 12])
    with fwAD.dual_level():
        x = [t.clone().requires_grad_(grad) for t in (q, k, v)]
        x[which] = fwAD.make_dual(x[which], torch.ones_like(q))
        with pytest.raises(RuntimeError):
            structure_attention(*x, packed)
        with torch.no_grad(), pytest.raises(RuntimeError):
            structure_attention(*x, packed)
        # a tangent elsewhere is none of its business
        assert torch.equal(structure_attention(q, k, v, packed), structure_attention(q, k, v, packed))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: structure_attention(*[t if i == which else y for i, y in enumerate((q, k, v))], packed), (q,), (q,))


@pytest.mark.parametrize("which", range(6))
def test_forward_mode_of_norm_and_rotation(which):
    q, k, _, pos, f, w = _rows()
    with fwAD.dual_level():
        x = [q, k, pos, f, w, w.clone()]
        x[which] = fwAD.make_dual(x[which], torch.ones_like(x[which]))
        with pytest.raises(RuntimeError):
            norm_rotate(*x[:4], q_weight=x[4], k_weight=x[5])
        with torch.no_grad(), pytest.raises(RuntimeError):
            norm_rotate(*x[:4], q_weight=x[4], k_weight=x[5])
        a, b = norm_rotate(q, k, pos, f, q_weight=w, k_weight=w)
        assert fwAD.unpack_dual(a).tangent is None and fwAD.unpack_dual(b).tangent is None
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: norm_rotate(t, None, pos, f)[0], (q,), (q,))


def test_scale_and_eps_that_would_learn():
    q, k, v, pos, f, w = _rows()
    packed = PackedStructures([0, 5, 12])
    scale = torch.tensor(0.3, requires_grad=True)
    for s in (scale, scale.cuda(), scale * 2):
        with pytest.raises(ValueError, match="scale"):
            structure_attention(q, k, v, packed, scale=s)
    eps = torch.tensor(1e-5, requires_grad=True)
    with pytest.raises(ValueError, match="eps"):
        norm_rotate(q, k, q_weight=w, k_weight=w, eps=eps)
    with torch.no_grad():
        assert torch.equal(structure_attention(q, k, v, packed, scale=scale), structure_attention(q, k, v, packed, scale=float(scale)))
        a, b = norm_rotate(q, k, q_weight=w, k_weight=w, eps=eps), norm_rotate(q, k, q_weight=w, k_weight=w, eps=float(eps))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    with fwAD.dual_level():
        dual = fwAD.make_dual(torch.tensor(0.3), torch.tensor(1.0))
        with pytest.raises(RuntimeError):
            structure_attention(q, k, v, packed, scale=dual)
        with pytest.raises(RuntimeError):
            norm_rotate(q, k, q_weight=w, k_weight=w, eps=dual)


def test_cotangents_with_tangents():
    q, k, v, pos, f, _ = _rows()
    packed = PackedStructures([0, 5, 12])
    x = q.clone().requires_grad_()
    for out in (structure_attention(x, k, v, packed), norm_rotate(x, k, pos, f)[0]):
        with fwAD.dual_level(), pytest.raises(RuntimeError):
            torch.autograd.grad(out, x, fwAD.make_dual(torch.ones_like(q), torch.ones_like(q)))
