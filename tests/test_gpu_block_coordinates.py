"""The blocks on voxel features leave a tensor of raw voxels as wide as it was: ordered behind them, it
has the keys that it has ordered before them."""
import pytest
import torch

from spira_amd import SparseTensor
from spira_amd import nn as spnn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("double", [False, True])
@pytest.mark.parametrize("block", [lambda: spnn.AttentionBlock(32, 2, window=64), lambda: spnn.ExpertBlock(32, 64, 4, 1)])
def test_order_behind_a_block(dev, block, double):
    g = torch.Generator().manual_seed(1)
    far = 20000 if double else 200  # (more than 32 bits hold of the three)
    coords = torch.randint(0, far, (300, 3), generator=g, dtype=torch.int32).to(dev)
    x = SparseTensor(coords, torch.randn(300, 32, generator=g).to(dev), double=double)
    with torch.no_grad():
        y = block().to(dev).eval()(x).order()
    ref = SparseTensor(coords, x.features, double=double).order()
    assert y.coordinates.dtype == ref.coordinates.dtype and torch.equal(y.coordinates, ref.coordinates)
