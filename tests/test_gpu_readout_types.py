"""StructureReadout with 16-bit parameters and under autocast: the same operators on the same roundings, called by hand."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from so3lr_b200 import PackedStructures, StructureReadout, norm_rotate, structure_attention  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _setup(seed=4):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = StructureReadout(n_out=3, heads=4, d=32, seed=seed)
    with torch.no_grad():
        r.last.normal_(generator=gen)
        r.norm_q.add_(0.1 * torch.randn(32, generator=gen, device="cuda"))
    return r, torch.randn(301, 128, generator=gen, device="cuda"), torch.rand(301, 3, generator=gen, device="cuda") * 12, np.array([0, 7, 8, 60, 260, 301])


def _by_hand(r, x, pos, gs, dt, wide):
    """Products in `dt`; the sum of features and attention in float32 where `wide`."""
    p = {n: t.to(dt) for n, t in r.named_parameters()}
    norm = (r.norm_q, r.norm_k)
    atoms, pool = PackedStructures(gs), PackedStructures(np.arange(len(gs)), gs)
    q, k, v = (x.to(dt) @ p["qkv"]).unflatten(1, (3, r.heads, r.d)).unbind(1)
    q, k = norm_rotate(q, k, pos, r.frequencies, q_weight=norm[0], k_weight=norm[1])
    o = structure_attention(q, k, v, atoms).flatten(1) @ p["out"]
    y = (x if wide else x.to(dt)) + o
    k, v = (y.to(dt) @ p["pool_kv"]).unflatten(1, (2, r.heads, r.d)).unbind(1)
    o = structure_attention(p["pool_query"].expand(len(gs) - 1, r.heads, r.d), k, v, pool)
    return o.flatten(1) @ p["last"]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_16_bit_parameters(dtype):
    dt = TYPES[dtype]
    r, x, pos, gs = _setup()
    f = r.frequencies.clone()
    full = r(x, pos, gs)
    r = r.to(dt)
    assert all(p.dtype == dt for p in r.parameters())
    # the frequencies turn positions of tens of Angstrom, whose angles want more than 8 or 11 bits
    assert r.frequencies.dtype == torch.float32 and torch.equal(r.frequencies, f)
    for features in (x, x.to(dt)):
        got = r(features, pos, gs)
        assert got.dtype == dt and torch.equal(got, _by_hand(r, features, pos, gs, dt, False))
    # some ten roundings of the type one behind the other, through two softmaxes of logits of size one
    assert (got.float() - full).abs().max() <= 50 * torch.finfo(dt).eps * full.abs().max()
    got.float().square().sum().backward()
    assert all(torch.isfinite(p.grad).all() and (p.grad != 0).any() for p in r.parameters())
    # back, and elsewhere: the buffer follows the device only
    assert r.float().frequencies.dtype == torch.float32 and r.to("cpu").frequencies.device.type == "cpu"
    assert torch.equal(r.to("cuda").frequencies, f) and torch.equal(r.state_dict()["frequencies"], f)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_under_autocast(dtype):
    dt = TYPES[dtype]
    r, x, pos, gs = _setup()
    with torch.autocast("cuda", dtype=dt):
        got = r(x, pos, gs)
    want = _by_hand(r, x, pos, gs, dt, True)
    assert got.dtype == dt and torch.equal(got, want)
    g = torch.randn(got.shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(dt)
    grads = [torch.autograd.grad(y, list(r.parameters()), g) for y in (got, want)]
    for a, b in zip(*grads):
        assert a.dtype == torch.float32 and torch.isfinite(a).all()
        assert (a - b).abs().max() <= 2 * torch.finfo(dt).eps * b.abs().max()      # copies of a rounded parameter may meet in another order
