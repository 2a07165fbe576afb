"""Segments of the batched calculator that name no graph are refused ahead of any index on the device."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("segments", [[0] * 9 + [2] * 3, [0] * 9 + [7] * 3, [-1] * 9 + [0] * 3, [0] * 11, [0] * 13])
@pytest.mark.parametrize("with_readout", [False, True])
def test_segments_out_of_range(segments, with_readout):
    from so3lr_b200 import So3lr, StructureReadout
    from so3lr_b200 import workloads as W
    Z, R = W.molecule(np.random.default_rng(3), 12)
    i, j = (x.astype(np.int32) for x in np.nonzero(~np.eye(12, dtype=bool)))
    inputs = dict(positions=np.asarray(R, np.float32), atomic_numbers=Z, idx_i=i, idx_j=j, idx_i_lr=i, idx_j_lr=j, cell=None, node_mask=np.ones(12, bool))
    fn = So3lr(lr_cutoff=1000.0, readout=StructureReadout() if with_readout else None)
    with pytest.raises(ValueError, match="batch_segments"):
        fn(dict(inputs, batch_segments=np.array(segments), graph_mask=np.ones(2, bool)))
    out = fn(dict(inputs, batch_segments=np.zeros(12, np.int64), graph_mask=np.array([True, False])))
    assert torch.isfinite(out["energy"]).all() and out["energy"].shape == (2,)
