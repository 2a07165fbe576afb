"""A readout over a padded batch: masked atoms take no part in it, wherever they stand."""
import numpy as np
import pytest
import torch

from so3lr_b200 import workloads as W

pytestmark = pytest.mark.gpu


def _readout(seed=2, n_out=2):
    from so3lr_b200 import StructureReadout
    r = StructureReadout(n_out=n_out, seed=seed)
    with torch.no_grad():
        r.last.normal_(generator=torch.Generator(device="cuda").manual_seed(seed))
    return r


def _pairs(R, start, keep):
    i, j = np.nonzero(~np.eye(len(R), dtype=bool))
    near = np.linalg.norm(R[j] - R[i], axis=1) < 4.5
    there = keep[i] & keep[j]
    return [x + start for x in (i[near & there], j[near & there], i[there], j[there])]


def _inputs(mols, masked, one_graph=False):
    """mols: (Z, R) of every structure; masked: of every structure a mask of atoms that only fill it up."""
    Z, R = (np.concatenate([m[k] for m in mols]) for k in (0, 1))
    start = np.concatenate([[0], np.cumsum([len(z) for z, _ in mols])])
    keep = ~np.concatenate(masked)
    lists = [_pairs(r, a, ~m) for (_, r), a, m in zip(mols, start, masked)]
    i, j, il, jl = (np.concatenate(x).astype(np.int32) for x in zip(*lists))
    graphs = dict(batch_segments=None, graph_mask=None) if one_graph else dict(batch_segments=np.repeat(np.arange(len(mols)), np.diff(start)),
                                                                              graph_mask=np.ones(len(mols), bool))
    return dict(positions=R.astype(np.float32), atomic_numbers=Z.astype(np.int32), idx_i=i, idx_j=j, idx_i_lr=il, idx_j_lr=jl, cell=None, total_charge=None,
                num_unpaired_electrons=None, node_mask=keep, **graphs)


def _filled(rng, mol, many, where):
    """`many` atoms that are masked among or behind those of a structure."""
    z, r = mol
    at = np.full(many, len(z)) if where == "behind" else np.sort(rng.integers(0, len(z) + 1, many))
    mask = np.insert(np.zeros(len(z), bool), at, True)
    return (np.insert(z, at, 1), np.insert(r, at, rng.normal(size=(many, 3)) * 3 + 40, axis=0)), mask


@pytest.mark.parametrize("where", ["behind", "among"])
@pytest.mark.parametrize("one_graph", [True, False])
def test_masked_atoms_of_a_structure(one_graph, where):
    from so3lr_b200 import So3lr
    rng = np.random.default_rng(5)
    mols = [W.molecule(rng, n) for n in ((20,) if one_graph else (20, 13, 31))]
    r = _readout()
    fn = So3lr(lr_cutoff=1000.0, readout=r)
    want = fn(_inputs(mols, [np.zeros(len(z), bool) for z, _ in mols], one_graph))
    filled, masked = zip(*[_filled(rng, m, many, where) for m, many in zip(mols, (12, 0, 40))])
    got = fn(_inputs(filled, masked, one_graph))
    keep = torch.tensor(~np.concatenate(masked), device="cuda")
    assert got["features"].shape == (len(keep), 128) and (got["features"][~keep] == 0).all()
    # the network's own sums may be formed in another order where rows stand elsewhere: a few roundings of float32 through its layers.  (The
    # charges do differ: a structure's total is shared out among all atoms of its segment, as the reference does it.)
    assert (got["features"][keep] - want["features"]).abs().max() <= 2e-5 * want["features"].abs().max()
    assert (got["readout"] - want["readout"]).abs().max() <= 1e-4 * want["readout"].abs().max()
    for out in (want, got):
        r.zero_grad()
        (out["readout"] ** 2).sum().backward()
        out["grads"] = [p.grad.clone() for p in r.parameters()]
    for x, y in zip(got["grads"], want["grads"]):
        assert (x - y).abs().max() <= 2e-4 * y.abs().max()


def test_all_atoms_of_a_structure_masked_and_a_readout_of_ones_own():
    """A structure without atoms pools nothing; whatever a readout makes of that, masked graphs give zero."""
    from so3lr_b200 import So3lr
    rng = np.random.default_rng(6)
    mols = [W.molecule(rng, 12), W.molecule(rng, 9)]
    masked = [np.zeros(12, bool), np.ones(9, bool)]
    inputs = _inputs(mols, masked)
    inputs["graph_mask"] = np.array([True, False])
    seen = {}

    def mean(features, positions, graph_start):
        seen.update(features=features, positions=positions, graph_start=np.asarray(graph_start))
        return torch.stack([features[a:b].mean(0) for a, b in zip(graph_start[:-1], graph_start[1:])])

    out = So3lr(lr_cutoff=1000.0, readout=mean)(inputs)
    assert seen["features"].shape == (12, 128) and seen["graph_start"].tolist() == [0, 12, 12]
    assert torch.equal(seen["positions"].cpu(), torch.tensor(mols[0][1].astype(np.float32)))
    assert torch.equal(out["readout"][0], out["features"][:12].mean(0)) and (out["readout"][1] == 0).all()
    out = So3lr(lr_cutoff=1000.0, readout=_readout())(inputs)
    assert torch.isfinite(out["readout"]).all() and (out["readout"][0] != 0).any() and (out["readout"][1] == 0).all()
