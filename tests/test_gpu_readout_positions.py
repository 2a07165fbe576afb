"""What the batched calculator does with positions that ask for a derivative when there is a readout."""
import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as fwAD

pytestmark = pytest.mark.gpu


def test_positions_of_the_batched_calculator():
    """A readout's gradient in the positions would lack the part through the features, which carry no graph."""
    from so3lr_b200 import So3lr, StructureReadout
    from so3lr_b200 import workloads as W
    Z, R = W.molecule(np.random.default_rng(3), 15)
    i, j = np.nonzero(~np.eye(15, dtype=bool))
    near = np.linalg.norm(R[j] - R[i], axis=1) < 4.5
    inputs = dict(atomic_numbers=Z, idx_i=i[near], idx_j=j[near], idx_i_lr=i, idx_j_lr=j, cell=None)
    fn = So3lr(lr_cutoff=1000.0, readout=StructureReadout(seed=1))
    pos = torch.tensor(np.asarray(R, np.float32), device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="positions"):
        fn(dict(inputs, positions=pos))
    with torch.no_grad():
        want = fn(dict(inputs, positions=pos))
    # the network adds its neighbours' terms in any order: some 15 roundings of 2^-24 in each of three layers, and what these make of them
    assert (fn(dict(inputs, positions=pos.detach()))["features"] - want["features"]).abs().max() <= 2e-5 * want["features"].abs().max()
    # without a readout, positions are taken as they are
    assert "energy" in So3lr(lr_cutoff=1000.0)(dict(inputs, positions=pos))
    with fwAD.dual_level(), pytest.raises((ValueError, RuntimeError)):
        fn(dict(inputs, positions=fwAD.make_dual(pos.detach(), torch.ones_like(pos))))
