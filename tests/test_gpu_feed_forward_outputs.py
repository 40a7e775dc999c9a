"""Outputs of the feed-forward operators that share memory with inputs, and rows of any strides through the served block."""
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


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantised_rows_apart_from_their_inputs(dev, dtype):
    q, scale = ops.quantize_rows(torch.randn(6, 64, device=dev))
    size = torch.empty((), dtype=dtype).element_size()
    hold = torch.zeros(6 * 64 * (size + 1) + 64, dtype=torch.int8, device=dev)
    rows = hold[:6 * 64].view(6, 64)
    rows.copy_(q)
    for start in (0, 64, 5 * 64):
        out = hold[start:start + 6 * 64 * size].view(dtype).view(6, 64)
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.dequantize_rows(rows, scale, dtype, out=out)
    if dtype == torch.float32:
        both = torch.zeros(6 * 64, device=dev)
        both[:6] = scale
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.dequantize_rows(q, both[:6], dtype, out=both.view(6, 64))
    out = hold[6 * 64:6 * 64 * (size + 1)].view(dtype).view(6, 64)       # behind the last row
    assert torch.equal(ops.dequantize_rows(rows, scale, dtype, out=out), ops.dequantize_rows(q, scale, dtype))
    assert torch.equal(rows, q)


@pytest.mark.parametrize("rows", [3, 70])
def test_served_block_takes_rows_of_any_strides(dev, rows):
    """As the block does with its fp32 weights: transposed, every other column, one row repeated."""
    torch.manual_seed(rows)
    block = GatedFeedForward(96, 130).to(dev).eval()
    wide, row = torch.randn(192, rows, device=dev), torch.randn(1, 96, device=dev)
    for x, r in ((wide[:96].t(), wide[96:].t()), (wide[::2].t(), None), (wide[:96].t(), row.expand(rows, 96))):
        full = x.contiguous(), None if r is None else r.contiguous()
        for layout in (block.dequantize_, block.quantize_):
            layout()
            with torch.no_grad():
                assert torch.equal(block(x, r), block(*full))
    with torch.no_grad(), pytest.raises(RuntimeError, match="2-D"):
        block(torch.randn(2, 3, 96, device=dev))
