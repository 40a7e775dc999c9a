"""The gate's activations far from zero, where a sum of near-opposite terms would leave nothing of their value."""
import math

import pytest
import torch

from graphsage_amd import ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half a subnormal step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gate_values(dtype, dev):
    """-12 to 12 in the rows' type: gate products and their values are exact, one of the two weights' columns each."""
    g = torch.linspace(-12, 12, 1201, device=dev).to(dtype)
    x = torch.stack((g, torch.ones_like(g)), 1).contiguous()
    w_gate, w_up = (torch.tensor([[a, b]], dtype=dtype, device=dev) for a, b in ((1, 0), (0, 1)))
    return g.double(), x, w_gate, w_up


def within(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert float(over.max()) <= 0, f"{int((over > 0).sum())} beyond their bound"


def tail(g):
    """Phi(g) = erfc(-g / sqrt 2) / 2 and the density, in 64 bits and to the last digit for every g."""
    return 0.5 * torch.erfc(-g / math.sqrt(2)), torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)


# gelu(g) = g Phi(g).  An argument of the tail that is off by 2 E (g / sqrt 2, or the exponent g^2 / 2 and its change of
# base) changes Phi(-|g|) by at most 2 (g^2 + 1) E; the function itself is off by at most 16 E, the products by 2 E: relative
# errors all of them.
def value_bound(g, v):
    return v.abs() * (18 + 2 * (g * g + 1)) * E


# slope = Phi(g) + g density(g): Phi as above; of the density, -g^2 / 2 and its change of base are off by 2 E at most each,
# so the exponential by 2 g^2 E, and by 16 E of its own and of the products.
def slope_bound(g):
    phi, density = tail(g)
    return (phi * (18 + 2 * (g * g + 1)) + g.abs() * density * (16 + 2 * g * g)) * E


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 1201])
def test_gelu_keeps_its_relative_accuracy(dev, dtype, rows):
    g, x, w_gate, w_up = gate_values(dtype, dev)
    at = torch.linspace(0, 1200, rows, device=dev).long()
    g, x = g[at], x[at].contiguous()
    out, saved = ops.gated_linear_fwd(x, w_gate, w_up, "gelu", save=True)
    assert torch.equal(saved[0, :, 0].double(), g) and bool((saved[1] == 1).all())
    phi, density = tail(g)
    want = g * phi
    within(out[:, 0], want, value_bound(g, want) * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype])
    dx, dwg, dwu = ops.gated_linear_bwd(torch.ones_like(out), x, w_gate, w_up, saved, "gelu")
    slope = phi + g * density
    within(dx[:, 0], slope, slope_bound(g) * (1 + 2 ** -7) + slope.abs() * (U[dtype] + E) + TINY[dtype])
    within(dx[:, 1], want, value_bound(g, want) * (1 + 2 ** -7) + want.abs() * (U[dtype] + E) + TINY[dtype])


@pytest.mark.parametrize("rows", [5, 600])
def test_8_bit_gelu_keeps_its_relative_accuracy(dev, rows):
    """x rows of whole numbers with a scale of 1 / 8; their gate products are exact."""
    q = torch.linspace(-96, 96, rows, device=dev).round()
    x = torch.stack((q, torch.full_like(q, 8.0)), 1).to(torch.int8)
    scale, one = torch.full((rows,), 0.125, device=dev), torch.ones(1, device=dev)
    w_gate, w_up = (torch.tensor([[a, b]], dtype=torch.int8, device=dev) for a, b in ((1, 0), (0, 1)))
    g = q.double() / 8
    want = g * tail(g)[0]
    for dtype in DTYPES:
        out = ops.int8_gated_linear(x, scale, w_gate, one, w_up, one, "gelu", dtype)[:, 0]
        within(out, want, value_bound(g, want) * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype])


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_activations_behind_their_tails(dev, act):
    """Values that no type holds are zero, large ones are themselves, infinities and NaN stay what the formula gives."""
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([-3e38, -200.0, -100.0, 100.0, 3e38, inf, nan], device=dev)
    x = torch.stack((g, torch.ones_like(g)), 1).contiguous()
    w_gate, w_up = torch.tensor([[1.0, 0.0]], device=dev), torch.tensor([[0.0, 1.0]], device=dev)
    out = ops.gated_linear_fwd(x[:5].contiguous(), w_gate, w_up, act)[0][:, 0]
    assert bool((out[:3].abs() <= 1e-36).all()) and torch.equal(out[3:5], g[3:5])
    assert bool(torch.isnan(ops.gated_linear_fwd(x[6:].contiguous(), w_gate, w_up, act)[0]).all())
