"""Outputs of the feed-forward operators that share memory with inputs, and where the served block rounds."""
import pytest
import torch

from graphsage_amd import ops
from graphsage_amd.layers import GatedFeedForward

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(1, 7), (5, 64), (3, 2047), (2100, 600), (2, 40001)])
def test_norm_in_place_of_its_rows(dev, dtype, rows, dim):
    """Without a residual the sum is x: written over by y there is none to return, and so none to differentiate from."""
    torch.manual_seed(dim)
    x, w = torch.randn(rows, dim, device=dev).to(dtype), torch.randn(dim, device=dev)
    want, s = ops.rms_norm_fwd(x, w)
    assert s is x
    y, s = ops.rms_norm_fwd(x, w, out=x)
    assert y is x and s is None and torch.equal(y, want)
    x = torch.randn(rows, dim, device=dev).to(dtype)
    other = torch.empty_like(x)
    y, s = ops.rms_norm_fwd(x, w, out=other)
    assert y is other and s is x
    with pytest.raises(RuntimeError):
        ops.rms_norm_bwd(x, None, w)
