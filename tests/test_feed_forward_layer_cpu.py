"""GatedFeedForward's and the autograd forms' choices, with recorders in place of the kernels: which form a call takes,
and which weights it serves."""
import copy
import io
import itertools

import pytest
import torch

from graphsage_amd import functional as SF
from graphsage_amd import _lib, ops
from graphsage_amd.layers import GatedFeedForward
from graphsage_amd.models import GraphSAGE


@pytest.fixture
def served(monkeypatch):
    """An 8-bit layout that is a copy of its weight, and a block that says which weights a call was served from."""
    monkeypatch.setattr(ops, "quantize_rows", lambda w, padded=False: (w.detach().clone(), torch.ones(w.size(0))))
    monkeypatch.setattr(SF, "rms_norm", lambda *a, **k: a[0])
    monkeypatch.setattr(SF, "gated_linear", lambda x, *a: x)
    monkeypatch.setattr(SF, "linear_concat", lambda h, w: "fp32")
    monkeypatch.setattr(GatedFeedForward, "_serve", lambda self, x, r: self._eight)
    monkeypatch.setattr(torch.Tensor, "__add__", lambda a, b: b)

    def call(block):
        with torch.no_grad():
            return block(torch.zeros(1, 8))
    return call


CHANGES = {
    "copy_": lambda b: b.up.weight.detach().copy_(torch.zeros(12, 8)),
    "in place": lambda b: b.gate.weight.detach().mul_(0.5),
    "another parameter": lambda b: setattr(b.down, "weight", torch.nn.Parameter(torch.zeros(8, 12))),
    "other data": lambda b: setattr(b.gate.weight, "data", torch.zeros(12, 8)),
    "a layer's load_state_dict": lambda b: b.up.load_state_dict({"weight": torch.zeros(12, 8)}),
    "a layer's reset": lambda b: b.up.reset_parameters(),
    "a step": lambda b: torch.optim.SGD(b.parameters(), lr=0.1).step(),
}


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("training", [False, True])
def test_changed_weights_are_not_served_from_old_8_bits(served, change, training):
    """In eval mode, and where the 8 bits were laid out in training mode."""
    block = GatedFeedForward(8, 12).train(training)
    block.quantize_()
    block.eval()
    assert served(block) is block._eight and block.quantized
    for p in block.parameters():
        p.grad = torch.ones_like(p)
    CHANGES[change](block)
    assert served(block) == "fp32" and not block.quantized
    block.quantize_()
    eight = served(block)
    for (q, _), layer in zip(eight, (block.gate, block.up, block.down)):
        assert torch.equal(q, layer.weight)


def test_the_norms_weight_is_not_quantised(served):
    block = GatedFeedForward(8, 12).eval().quantize_()
    with torch.no_grad():
        block.norm_weight.mul_(2)
    assert served(block) is block._eight


def test_parametrized_weights_are_served_until_they_change(served):
    block = GatedFeedForward(8, 12).eval()
    torch.nn.utils.parametrizations.weight_norm(block.up)
    block.quantize_()
    assert served(block) is block._eight and served(block) is block._eight
    with torch.no_grad():
        block.up.parametrizations.weight.original0.mul_(2)
    assert served(block) == "fp32"


def test_copies_keep_current_8_bits_and_no_others(served):
    block = GatedFeedForward(8, 12).eval().quantize_()
    stored = io.BytesIO()
    torch.save(block, stored)
    stored.seek(0)
    for other in (copy.deepcopy(block), torch.load(stored, weights_only=False)):
        assert other.quantized and served(other) is other._eight
        with torch.no_grad():
            other.gate.weight.zero_()
        assert not other.quantized and block.quantized
    with torch.no_grad():
        block.gate.weight.zero_()
    assert not copy.deepcopy(block).quantized


def test_inference_tensors_as_weights(served):
    """Weights made under inference_mode have no count of their changes; they are served."""
    with torch.inference_mode():
        block = GatedFeedForward(8, 12).eval().quantize_()
        assert served(block) is block._eight


# ------------------------------------------------------------------------------- what the backward pass keeps
@pytest.fixture
def kept(monkeypatch):
    """ops.gated_linear_fwd on the CPU; the list of what `save` was at each call."""
    calls = []

    def forward(x, w_gate, w_up, activation="silu", save=False, out=None):
        calls.append(save)
        g, u = x @ w_gate.t(), x @ w_up.t()
        return g.sigmoid() * g * u, (torch.stack((g, u)) if save else None)
    monkeypatch.setattr(ops, "gated_linear_fwd", forward)
    return calls


def test_products_are_kept_for_a_gradient_only(kept):
    plain, leaf = torch.randn(3, 8), torch.nn.Parameter(torch.randn(5, 8))
    w = torch.randn(5, 8)
    for args in ((plain, leaf, w), (plain, w, leaf), (plain.clone().requires_grad_(), w, w), (plain, leaf, leaf)):
        for mode in (torch.no_grad, torch.inference_mode):
            with mode():
                want = SF.gated_linear(*args)
            assert kept.pop() is False and not want.requires_grad
        got = SF.gated_linear(*args)
        assert kept.pop() is True and got.requires_grad and torch.equal(got, want)
        with torch.no_grad(), torch.enable_grad():
            SF.gated_linear(*args)
        assert kept.pop() is True
    SF.gated_linear(plain, w, w)
    assert kept == [False]


def test_blocks_evaluation_keeps_no_products(kept, monkeypatch):
    monkeypatch.setattr(ops, "rms_norm_fwd", lambda x, w, residual=None, eps=1e-6: (x * w, x if residual is None else x + residual))
    monkeypatch.setattr(ops, "linear_concat_fwd", lambda a1, w1, *a, **k: a1 @ w1.t())
    monkeypatch.setattr(ops, "aligned_rows", lambda t: t)
    block = GatedFeedForward(8, 12)
    for mode in (block.train, block.eval):
        mode()
        with torch.no_grad():
            block(torch.randn(2, 8), torch.randn(2, 8))
        assert kept.pop() is False
        block(torch.randn(2, 8))
        assert kept.pop() is True


# ------------------------------------------------------------------------------- shapes
@pytest.mark.parametrize("shape", [(3, 2, 8), (6, 8), (1, 6, 8), (2, 3, 1, 8), (8,), (2, 3, 4)])
def test_a_residual_of_another_shape_is_refused(monkeypatch, shape):
    """Also where it has as many rows: they would be other rows."""
    monkeypatch.setattr(ops, "rms_norm_fwd", lambda x, w, residual=None, eps=1e-6: (x * w, x + residual))
    with pytest.raises(RuntimeError, match="residual: expected shape"):
        SF.rms_norm(torch.zeros(2, 3, 8), torch.ones(8), torch.zeros(shape))


# ------------------------------------------------------------------------------- outputs
@pytest.mark.parametrize("shape", [(4, 8), (2, 3, 8), (8,)])
def test_outputs_may_be_changed_in_place(kept, monkeypatch, shape):
    """y and the gated product are not kept for the backward pass; s is, and torch says so."""
    monkeypatch.setattr(ops, "rms_norm_fwd", lambda x, w, residual=None, eps=1e-6: (x * w, x if residual is None else x + residual))
    monkeypatch.setattr(ops, "rms_norm_bwd", lambda dy, s, w, eps, ds, need_dx, need_dw: (dy * w, (dy * s).sum(0)))
    monkeypatch.setattr(ops, "gated_linear_bwd", lambda d, x, g, u, saved, act, need_dx, need_dw: (d @ u, d.t() @ x, d.t() @ x))
    x, r, w = torch.randn(shape, requires_grad=True), torch.randn(shape), torch.ones(8, requires_grad=True)
    wg, wu = torch.randn(5, 8, requires_grad=True), torch.randn(5, 8)
    for y in (SF.rms_norm(x, w), SF.rms_norm(x, w, r)[0]):
        assert y.shape == x.shape
        y.mul_(3.0).sum().backward()
        assert bool((x.grad == 3).all())
        x.grad = None
    h = SF.gated_linear(x, wg, wu)
    assert h.shape == (*shape[:-1], 5)
    h.mul_(2.0).sum().backward()
    assert x.grad.shape == x.shape and wg.grad.shape == wg.shape
    y, s = SF.rms_norm(x, w, r)
    s.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_16_bit_blocks_are_refused_before_any_work(monkeypatch):
    """The down projection is an fp32 product."""
    monkeypatch.setattr(SF, "rms_norm", lambda *a, **k: pytest.fail("launched"))
    block = GatedFeedForward(8, 12)
    with pytest.raises(RuntimeError, match="expected fp32 rows"):
        block(torch.zeros(2, 8, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="expected fp32 rows"):
        block.half()(torch.zeros(2, 8, dtype=torch.float16))
    with pytest.raises(RuntimeError, match="expected fp32 rows"):
        block.eval()(torch.zeros(2, 8))


# ------------------------------------------------------------------------------- the products' cuts
def test_product_cut_agrees_with_what_the_products_ask_for():
    """Its slices with the workspace (a tile's sums in 32 bits for each), its 0 with the sizes that take any rows."""
    lib = _lib.load()
    seen = set()
    for m, n, k, gated, fp32 in itertools.product((1, 16, 17, 300, 512, 513, 2049, 8192), (1, 64, 700, 4099, 8192), (16, 64, 1040, 4112, 40000),
                                                  (False, True), (False, True)):
        tile, slices = ops.product_cut(m, n, k, gated, fp32)
        seen.add((tile, slices > 1))
        assert lib.sage_product_any_rows(m, n, k, gated, fp32) == (tile == 0)
        across = tile // 2 if gated else tile
        want = 0 if slices == 1 else -(-m // tile) * -(-n // across) * tile * tile * 4 * slices
        assert lib.sage_product_workspace_bytes(m, n, k, gated, fp32) == want
        assert ops.product_cut(m, n, k, gated, fp32, few_rows=False)[0] in (128, 256)
    assert seen == {(0, False), (128, False), (128, True), (256, False), (256, True)}


def test_product_cut_refusals():
    for bad in ((0, 8, 64), (8, 0, 64), (8, 8, 0), (-1, 8, 64)):
        with pytest.raises(RuntimeError, match="sage_product_cut"):
            ops.product_cut(*bad)
    assert _lib.load().sage_product_cut(8, 8, 64, 0, 0, 1, None, None) == -1


# ------------------------------------------------------------------------------- stored models
def test_models_stored_before_there_were_blocks(served):
    """A whole model without the attribute loads as one without blocks; one with blocks keeps them."""
    old = GraphSAGE(8, 8)
    del old.blocks
    for model, count in ((old, None), (GraphSAGE(8, 8, num_layers=3, ffn_channels=12), 2)):
        stored = io.BytesIO()
        torch.save(model, stored)
        stored.seek(0)
        back = torch.load(stored, weights_only=False)
        assert (back.blocks if count is None else len(back.blocks)) == count
        x = torch.zeros(2, 8)
        assert back._feed_forward(0, x, x) is x if count is None else len(list(back.blocks.parameters())) == 8
