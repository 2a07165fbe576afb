"""System.features after an evaluation that failed on its way: the latest finished one's rows in the caller's order, or an error."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_rebuild_that_finds_no_memory():
    from so3lr_b200 import workloads as W
    from so3lr_b200._lib import lib
    from so3lr_b200.engine import System
    Z, R, _ = W.water_box(216, 18.7, 5)
    dense = torch.tensor(R, dtype=torch.float32, device="cuda")
    mol = torch.arange(len(Z), device="cuda") // 3
    centre = dense[::3][mol]
    thin = centre * 4.0 + (dense - centre)
    # the atoms in another order, so that the two structures are sorted differently
    thin = thin.flip(1)
    failed = 0
    for nth in range(1, 12):
        s = System(Z, np.eye(3) * 18.7 * 4.0, cutoff_lr=9.0, damping=2.0, skin=0.0)
        s.compute(thin)
        want = s.features()
        lib.so3lr_b200_host_fail_allocation(nth, 1)
        try:
            s.compute(dense)
            ok = True
        except RuntimeError:
            ok = False
        finally:
            lib.so3lr_b200_host_fail_allocation(0, 0)
        if ok:
            break
        failed += 1
        try:
            got = s.features()
        except RuntimeError:
            got = want
        assert torch.equal(got, want), nth
        s.compute(thin)
        assert (s.features() - want).abs().max() <= 2e-5 * want.abs().max()
    assert failed >= 1
