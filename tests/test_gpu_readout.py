"""Atom features and the attention readout on top of them, alone and through the batched calculator, against torch in 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import so3lr_oracle as O
from so3lr_b200 import workloads as W

pytestmark = pytest.mark.gpu


def _batch(n=5, seed=3):
    rng = np.random.default_rng(seed)
    mols = [W.molecule(rng, int(k)) for k in rng.integers(10, 41, n)]
    Z = np.concatenate([z for z, _ in mols]).astype(np.int32)
    R = np.concatenate([r for _, r in mols]).astype(np.float32)
    gs = np.concatenate([[0], np.cumsum([len(z) for z, _ in mols])]).astype(np.int32)
    return Z, R, gs


def _inputs(Z, R, gs, pad=0):
    """Inputs of the batched calculator; `pad` atoms behind the last structure form a masked graph."""
    n, g = len(Z), len(gs) - 1
    seg = np.repeat(np.arange(g), np.diff(gs))
    i, j, il, jl = [], [], [], []
    for a, b in zip(gs[:-1], gs[1:]):
        x, y = O.neighbor_list(R[a:b].astype(np.float64), None, 4.5)
        i.append(x + a), j.append(y + a)
        x, y = np.nonzero(~np.eye(b - a, dtype=bool))
        il.append(x + a), jl.append(y + a)
    i, j, il, jl = (np.concatenate(v).astype(np.int32) for v in (i, j, il, jl))
    if pad:
        Z, R = np.concatenate([Z, np.ones(pad, np.int32)]), np.concatenate([R, np.full((pad, 3), 50.0, np.float32) + 9 * np.arange(pad)[:, None].astype(np.float32)])
        seg = np.concatenate([seg, np.full(pad, g)])
    return dict(positions=R, atomic_numbers=Z, idx_i=i, idx_j=j, idx_i_lr=il, idx_j_lr=jl, cell=None, total_charge=None, num_unpaired_electrons=None,
                batch_segments=seg, node_mask=np.arange(n + pad) < n, graph_mask=np.arange(g + bool(pad)) < g)


def test_features_against_the_oracle_and_in_both_orders():
    from so3lr_b200 import System
    P = O.load_params()
    Z, R, _ = _batch(1)
    s = System(Z, None, cutoff_lr=12.0)
    with pytest.raises(RuntimeError):
        s.features()                      # nothing evaluated yet
    s.compute(torch.tensor(R, device="cuda"))
    seg = torch.as_tensor(R.astype(np.float64))
    i, j = O.neighbor_list(R.astype(np.float64), None, 4.5)
    il, jl = O.neighbor_list(R.astype(np.float64), None, 12.0, ordered=True)
    _, aux = O.energy_from_graph(P, Z, seg[j.astype(np.int64)] - seg[i.astype(np.int64)], i, j, seg[jl.astype(np.int64)] - seg[il.astype(np.int64)], il, jl)
    want = aux["x_final"].detach()
    got = s.features().cpu().double()
    # the features feed the charges and ratios, which agree to 1e-5 of order one
    assert got.shape == (len(Z), 128) and (got - want).abs().max() <= 2e-5 * want.abs().max()
    # a periodic box keeps its rows in another order inside: the rows follow their atoms
    Zb, Rb, cell = W.water_box(216, 18.64, 5)
    Rb = np.asarray(Rb, np.float32)
    perm = np.random.default_rng(0).permutation(len(Zb))
    f = []
    for p in (np.arange(len(Zb)), perm):
        b = System(np.asarray(Zb)[p], cell, cutoff_lr=9.0, skin=0.0)
        b.compute(torch.tensor(Rb[p], device="cuda"))
        f.append(b.features())
    assert (f[0][torch.as_tensor(perm, device="cuda")] - f[1]).abs().max() <= 2e-5 * f[0].abs().max()


def _plain(r, x, pos, gs):
    """The readout in float64 from its definition."""
    p = {n: t.detach().double().requires_grad_() for n, t in r.named_parameters()}
    x, theta = x.double(), pos.double() @ r.frequencies.double()
    c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]

    def rotate(y, w):
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w
        a, b = y.chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c], -1)

    def attend(q, k, v):
        a = torch.softmax(torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(r.d), -1)
        return torch.einsum("hij,jhd->ihd", a, v)

    q, k, v = (x @ p["qkv"]).unflatten(1, (3, r.heads, r.d)).unbind(1)
    q, k = rotate(q, p["norm_q"]), rotate(k, p["norm_k"])
    o = torch.cat([attend(q[a:b], k[a:b], v[a:b]) for a, b in zip(gs[:-1], gs[1:])])
    y = x + o.flatten(1) @ p["out"]
    k, v = (y @ p["pool_kv"]).unflatten(1, (2, r.heads, r.d)).unbind(1)
    o = torch.cat([attend(p["pool_query"][None], k[a:b], v[a:b]) for a, b in zip(gs[:-1], gs[1:])])
    return o.flatten(1) @ p["last"], p


@pytest.mark.parametrize("heads,d", [(4, 32), (3, 48)])
def test_readout_and_its_gradients(heads, d):
    from so3lr_b200 import StructureReadout
    gen = torch.Generator(device="cuda").manual_seed(1)
    gs = np.array([0, 7, 8, 60, 260, 301])
    x = torch.randn(301, 128, generator=gen, device="cuda")
    pos = torch.rand(301, 3, generator=gen, device="cuda") * 12
    r = StructureReadout(n_out=3, heads=heads, d=d, seed=4)
    assert (r(x, pos, gs) == 0).all()                     # as it starts
    with torch.no_grad():
        r.last.normal_(generator=gen)
    leaf = pos.clone().requires_grad_()
    got = r(x, leaf, gs)
    want, p = _plain(r, x, pos, gs)
    # float32 through two products of 128 and 4 x 32 terms, a softmax and one of 128 more: 1e-6 of the size of the result each
    assert got.shape == (5, 3) and (got.double() - want).abs().max() <= 1e-5 * want.abs().max()
    g = torch.randn(5, 3, generator=gen, device="cuda")
    (got * g).sum().backward()
    (want * g.double()).sum().backward()
    for n, t in r.named_parameters():
        assert (t.grad.double() - p[n].grad).abs().max() <= 2e-5 * p[n].grad.abs().max(), n
    # a shift of the structures changes nothing: the positions' gradient sums to zero in every structure
    for a, b in zip(gs[:-1], gs[1:]):
        assert leaf.grad[a:b].sum(0).abs().max() <= 1e-4 * max(float(leaf.grad[a:b].abs().sum()), 1e-6)
    with pytest.raises(ValueError):
        r(x[:, :64], pos, gs)
    with pytest.raises(ValueError):
        r(x, pos[:300], gs)
    with pytest.raises(ValueError):
        StructureReadout(d=20)


@pytest.mark.parametrize("pad", [0, 6])
def test_batched_calculator_with_a_readout(pad):
    from so3lr_b200 import So3lr, StructureReadout
    Z, R, gs = _batch(6)
    r = StructureReadout(n_out=2, seed=2)
    with torch.no_grad():
        r.last.normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    inputs = _inputs(Z, R, gs, pad)
    plain = So3lr(lr_cutoff=1000.0)(inputs)
    out = So3lr(lr_cutoff=1000.0, readout=r)(inputs)
    for k in plain:                                       # the rest of the outputs stays what it is
        assert torch.allclose(plain[k], out[k], rtol=1e-5, atol=1e-5), k
    assert out["features"].shape == (len(Z) + pad, 128) and out["readout"].shape == (len(gs) - 1 + bool(pad), 2)
    want, _ = _plain(r, out["features"][:len(Z)], torch.tensor(R, device="cuda"), gs)
    n = len(gs) - 1
    assert (out["readout"][:n].double() - want).abs().max() <= 1e-5 * want.abs().max()
    assert (out["readout"][n:] == 0).all() and (out["features"][len(Z):] == 0).all()
    # trained on the frozen features: every parameter gets a gradient, and a step along it changes the result
    (out["readout"] ** 2).sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() and (p.grad != 0).any() for p in r.parameters())


def test_copies_and_captured_readouts():
    import copy

    from so3lr_b200 import StructureReadout
    gen = torch.Generator(device="cuda").manual_seed(9)
    r = StructureReadout(n_out=2, seed=1)
    with torch.no_grad():
        r.last.normal_(generator=gen)
    x, pos, gs = torch.randn(50, 128, generator=gen, device="cuda"), torch.rand(50, 3, generator=gen, device="cuda") * 9, np.array([0, 30, 50])
    with torch.no_grad():
        want = r(x, pos, gs)
        assert torch.equal(copy.deepcopy(r)(x, pos, gs), want)      # its layouts stay with the original
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            r(x, pos, gs)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            got = r(x, pos, gs)
        for i in range(1, r.MAX_CACHED_LAYOUTS + 4):                # the graph's layout is not among those that make room
            r(x, pos, np.array([0, i, 50]))
        assert any(k[0] == np.asarray(gs, np.int32).tobytes() for k in r._captured)
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
