"""The feed-forward block as it is used: its operators one after the other, autograd, streams and graphs,
the layer, the model and the trainer, in fp32 and served in 8 bits."""
import copy
import math

import pytest
import torch
import torch.nn.functional as F

from graphsage_amd import functional as SF
from graphsage_amd import ops
from graphsage_amd.layers import GatedFeedForward
from graphsage_amd.models import GraphSAGE
from tests.helpers import random_graph

pytestmark = pytest.mark.gpu
E = 2.0 ** -24


def reference(block, x, residual=None):
    """The block in 64 bits on the CPU, from its parameters (leaves of their own, returned)."""
    p = {n: v.detach().cpu().double().requires_grad_() for n, v in block.named_parameters()}
    x = x.detach().cpu().double().requires_grad_()
    r = None if residual is None else residual.detach().cpu().double().requires_grad_()
    s = x if r is None else x + r
    y = s * (s.square().mean(-1, keepdim=True) + block.eps).rsqrt() * p["norm_weight"]
    g, u = y @ p["gate.weight"].t(), y @ p["up.weight"].t()
    a = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu}[block.activation](g)
    return s + (a * u) @ p["down.weight"].t(), p, x, r


# The chain in fp32: every stage's relative error is a few E times the sums' lengths (tests of the operators), and
# sums of n terms of random sign lose sqrt(n) of their magnitudes, so outputs and gradients that are of order one
# agree to some 1e-5; 2e-4 of the largest value leaves room for the few that cancel.
def near(got, want, what, tol=2e-4):
    got, want = got.detach().cpu().double(), want.detach()
    scale = float(want.abs().max())
    assert float((got - want).abs().max()) <= tol * scale, (what, float((got - want).abs().max()), scale)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,channels,hidden", [(1, 8, 12), (7, 33, 50), (200, 96, 257), (1000, 256, 512)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_block_forward_and_gradients(dev, act, rows, channels, hidden, with_residual):
    torch.manual_seed(rows + channels)
    block = GatedFeedForward(channels, hidden, act).to(dev)
    with torch.no_grad():
        block.norm_weight.add_(0.3 * torch.randn(channels, device=dev))
    x = torch.randn(rows, channels, device=dev, requires_grad=True)
    r = torch.randn(rows, channels, device=dev, requires_grad=True) if with_residual else None
    out = block(x, r)
    want, p, x64, r64 = reference(block, x, r)
    near(out, want, "out")
    dout = torch.randn(rows, channels, device=dev)
    out.backward(dout)
    want.backward(dout.cpu().double())
    near(x.grad, x64.grad, "dx")
    if with_residual:
        near(r.grad, r64.grad, "dr")
        assert torch.equal(r.grad, x.grad)
    for name, v in block.named_parameters():
        near(v.grad, p[name].grad, name)


def test_leading_dimensions_and_partial_gradients(dev):
    """[..., n] inputs; only some of the inputs ask for a gradient; an output that nothing uses; a
    gradient that is one value repeated (sum) or arrives transposed."""
    torch.manual_seed(3)
    x, r = torch.randn(2, 3, 5, 24, device=dev), torch.randn(2, 3, 5, 24, device=dev)
    w = torch.randn(24, device=dev, requires_grad=True)
    y, s = SF.rms_norm(x, w, r)
    assert y.shape == s.shape == x.shape
    y.sum().backward()
    s64 = x.double() + r.double()
    xh = s64 * (s64.square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    near(w.grad, xh.sum((0, 1, 2)).cpu(), "dw")
    r2 = r.clone().requires_grad_()
    y, s = SF.rms_norm(x, w.detach(), r2)
    (2 * s).sum().backward()                        # y unused: the sum's gradient passes through
    assert bool((r2.grad == 2).all())
    wg, wu = torch.randn(40, 24, device=dev), torch.randn(40, 24, device=dev, requires_grad=True)
    out = SF.gated_linear(x, wg, wu, "gelu")
    assert out.shape == (2, 3, 5, 40)
    flat = SF.gated_linear(x.reshape(-1, 24), wg, wu, "gelu")
    assert torch.equal(flat.view_as(out), out)
    flat.t().contiguous().t().mul(1.0).t().sum().backward()
    g = F.gelu(x.reshape(-1, 24).double() @ wg.double().t())
    near(wu.grad, (g.t() @ x.reshape(-1, 24).double()).cpu(), "dw_up")
    with torch.no_grad():
        assert torch.equal(SF.gated_linear(x, wg, wu, "gelu"), out)
    with pytest.raises(RuntimeError):
        z = x.clone().requires_grad_()
        (dz,) = torch.autograd.grad(SF.rms_norm(z, w).square().sum(), z, create_graph=True)
        dz.sum().backward()


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gradients_against_differences(dev, act):
    """Directional derivatives of the definition in 64 bits (central differences: their error is some 1e-9) against
    the kernels' gradients, whose error is below 64 E of the magnitudes that they add up at these sizes."""
    g = torch.Generator().manual_seed(5)
    m, k, h = 6, 9, 11
    v = {n: torch.randn(*s, generator=g) for n, s in (("x", (m, k)), ("r", (m, k)), ("w", (k,)), ("wg", (h, k)), ("wu", (h, k)), ("dh", (m, h)), ("ds", (m, k)))}

    def value(t):
        s = t["x"] + t["r"]
        y = s * (s.square().mean(1, keepdim=True) + 1e-6).rsqrt() * t["w"]
        a = {"silu": F.silu, "gelu": F.gelu}[act](y @ t["wg"].t())
        return (v["dh"].double() * a * (y @ t["wu"].t())).sum() + (v["ds"].double() * s).sum()

    d = {n: t.to(dev).requires_grad_() for n, t in v.items()}
    y, s = SF.rms_norm(d["x"], d["w"], d["r"])
    ((SF.gated_linear(y, d["wg"], d["wu"], act) * d["dh"]).sum() + (s * d["ds"]).sum()).backward()
    for name in ("x", "r", "w", "wg", "wu"):
        for seed in range(3):
            along = torch.randn(v[name].shape, generator=g).double()
            t = {n: u.double() for n, u in v.items()}
            step = 1e-5
            up, down = dict(t), dict(t)
            up[name], down[name] = t[name] + step * along, t[name] - step * along
            want = float((value(up) - value(down)) / (2 * step))
            got = float((d[name].grad.cpu().double() * along).sum())
            size = float((d[name].grad.cpu().double().abs() * along.abs()).sum()) + float(v["dh"].abs().sum())
            assert abs(got - want) <= 1e-7 + 64 * E * 10 * size, (name, got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 5, 70, 300])
def test_operators_one_after_the_other(dev, dtype, rows):
    """A row's stage outputs do not depend on the rows beside it, in one call or many, captured in a graph or not,
    on another stream than the default one."""
    torch.manual_seed(rows)
    k, h = 208, 130
    x, r = torch.randn(rows, k, device=dev).to(dtype), torch.randn(rows, k, device=dev).to(dtype)
    w = (1 + 0.2 * torch.randn(k, device=dev)).to(dtype)
    wg, wu, wd = (torch.randn(*s, device=dev) * s[1] ** -0.5 for s in ((h, k), (h, k), (k, h)))
    (gq, gs), (uq, us), (dq, ds) = (ops.quantize_rows(t, padded=True) for t in (wg, wu, wd))
    lg, lu = wg.to(dtype), wu.to(dtype)

    def chain(x, r):
        y, s = ops.rms_norm_fwd(x, w, residual=r)
        out, saved = ops.gated_linear_fwd(y, lg, lu, save=True)
        dx, dwg, dwu = ops.gated_linear_bwd(out, y, lg, lu, saved)
        dn, dw = ops.rms_norm_bwd(dx, s, w, dsum=s)
        q, qs, s2 = ops.rms_norm_int8(x, w, residual=r, padded=True)
        hq, hs = ops.quantize_rows(ops.int8_gated_linear(q, qs, gq, gs, uq, us, out_dtype=torch.bfloat16), padded=True)
        z = ops.int8_linear(hq, hs, dq, ds, out_dtype=dtype)
        return [y, s, out, dx, dwg, dwu, dn, dw, q, qs, s2, hq, hs, z]

    want = chain(x, r)
    for name, got in zip(range(14), chain(x, r)):
        assert torch.equal(got, want[name]), name
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = chain(x, r)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want))
    # two graphs over the same inputs, replayed in turn and together with eager calls
    x1, r1 = x.clone(), r.clone()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = chain(x1, r1)
        graphs.append((graph, outs))
    for turn in range(3):
        x1.copy_(torch.roll(x, turn, 0))
        r1.copy_(torch.roll(r, turn, 0))
        eager = chain(x1, r1)
        for graph, outs in graphs:
            for o in outs:
                o.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for graph, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


def test_backward_in_a_graph_beside_eager_training(dev):
    """forward and backward of the block captured in a graph, replayed between eager steps of a block of its own."""
    torch.manual_seed(0)
    block, other = GatedFeedForward(64, 96).to(dev), GatedFeedForward(64, 96).to(dev)
    x, dout = torch.randn(130, 64, device=dev), torch.randn(130, 64, device=dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            grads = torch.autograd.grad(block(x), list(block.parameters()), dout)
    torch.cuda.current_stream().wait_stream(side)
    want = [g.clone() for g in grads]
    with torch.no_grad():
        h = SF.gated_linear(SF.rms_norm(x, block.norm_weight), block.gate.weight, block.up.weight)
        most = 2 * 132 * E * (dout.abs().t() @ h.abs())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x)
        grads = torch.autograd.grad(out, list(block.parameters()), dout)
    for _ in range(3):
        for g in grads:
            g.zero_()
        other(x).sum().backward()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads[:3], want[:3]))
        # the down projection's gradient is linear_dweight's, whose slices meet by fp32 atomics in any order (two eager
        # calls differ as well): each of two sums of 130 terms is off by at most 132 E of the magnitudes
        assert bool(((grads[3] - want[3]).abs() <= most).all())


def served_bound(block, x, r):
    """|served - exact| element by element: half a step of each quantisation, carried through the block."""
    p = {n: v.detach().double() for n, v in block.named_parameters()}
    s = x.double() if r is None else x.double() + r.double()
    y = s * (s.square().mean(-1, keepdim=True) + block.eps).rsqrt() * p["norm_weight"]
    half = lambda t: 0.5001 * t.abs().amax(-1, keepdim=True) / 127          # noqa: E731
    g, u = y @ p["gate.weight"].t(), y @ p["up.weight"].t()

    def off(a, b, da, db):         # of a @ b^T
        return (a.abs() + da) @ db.t() + da @ b.abs().t()
    dy = half(y).expand_as(y)
    dg = off(y, p["gate.weight"], dy, half(p["gate.weight"]).expand_as(p["gate.weight"]))
    du = off(y, p["up.weight"], dy, half(p["up.weight"]).expand_as(p["up.weight"]))
    a = F.silu(g)
    h = a * u
    dh = 1.2 * dg * (u.abs() + du) + a.abs() * du
    dh = dh + (h.abs() + dh) * 2.0 ** -8
    dh = dh + 0.5001 * (h.abs() + dh).amax(-1, keepdim=True) / 127
    want = s + h @ p["down.weight"].t()
    return want, off(h, p["down.weight"], dh, half(p["down.weight"]).expand_as(p["down.weight"])) + 1e-4 * want.abs() + 1e-5


@pytest.mark.parametrize("rows,channels,hidden", [(1, 16, 32), (5, 50, 37), (300, 128, 200)])
def test_block_served_in_8_bits(dev, rows, channels, hidden):
    torch.manual_seed(rows)
    block = GatedFeedForward(channels, hidden).to(dev).eval()
    x, r = torch.randn(rows, channels, device=dev), torch.randn(rows, channels, device=dev)
    assert not block.quantized
    block.quantize_()
    for residual in (None, r):
        with torch.no_grad():
            got = block(x, residual)
        want, bound = served_bound(block, x, residual)
        assert bool(((got.double() - want).abs() <= bound).all())
        # far nearer than the bound, which adds up worst cases, and not the fp32 path
        err = (got.double() - want).norm() / (want - (x if residual is None else x + residual).double()).norm()
        exact = block(x, residual)                # gradients enabled: fp32 weights
        assert 1e-4 < float(err) < 0.1 and not torch.equal(exact.detach(), got)
        near(exact, reference(block, x, residual)[0], "fp32")
    assert block.quantized
    block.train()
    assert not block.quantized
    block.eval().quantize_().load_state_dict(copy.deepcopy(block.state_dict()))
    assert not block.quantized


@pytest.mark.parametrize("aggregator", ["mean", "max", "gcn", "max_pool"])
def test_model_with_blocks(dev, aggregator):
    """Pruned, unpruned and table-gather forms agree; the gradients reach every parameter; a model without blocks has
    the parameters it always had; 8-bit inference stays near."""
    from graphsage_amd.datasets import planted_partition
    from graphsage_amd.samplers import UniformLoader
    torch.manual_seed(1)
    data = planted_partition(500, 6000, 48, 4, seed=0)
    loader = UniformLoader(data, num_neighbors=[5, 4, 3], input_nodes=torch.arange(60), batch_size=60, seed=3)
    model = GraphSAGE(48, 32, aggregator, 3, 4, ffn_channels=80).to(dev)
    plain = GraphSAGE(48, 32, aggregator, 3, 4)
    assert len(model.blocks) == 2 and plain.blocks is None
    assert not any(n.startswith("blocks") for n in plain.state_dict())
    batch = next(iter(loader))
    x, y = batch.x.to(dev), batch.y[:60].to(dev)
    edge_index = batch.edge_index
    pruned = model(x, edge_index)
    assert pruned.shape == (60, 4)
    table = model.forward_batch(batch)
    torch.testing.assert_close(pruned, table, rtol=1e-4, atol=2e-5)
    model.prune_to_seeds = False
    whole = model(x, edge_index)
    torch.testing.assert_close(whole[:60], pruned, rtol=1e-4, atol=2e-5)
    model.prune_to_seeds = True
    F.cross_entropy(pruned, y).backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) and float(p.grad.abs().sum()) > 0
               for p in model.parameters())
    with pytest.raises(RuntimeError, match="eval"):
        model.quantize_()
    model.eval()
    with torch.no_grad():                          # one sampled batch: inference(loader) samples anew each time
        exact = model(x, edge_index)
        served = model.quantize_()(x, edge_index)
    assert not torch.equal(served, exact) and float((served - exact).norm() / exact.norm()) < 0.1
    assert model.inference(loader).shape == (60, 4)
    with pytest.raises(RuntimeError, match="no feed-forward"):
        plain.quantize_()


def test_block_inside_the_model_against_the_reference(dev):
    """Layer outputs fed to a block in 64 bits by hand: which rows are the residual, and from which layer on."""
    torch.manual_seed(2)
    n = 200
    ei = torch.from_numpy(random_graph(n, 3000, seed=4, isolated=3)).to(dev)
    x = torch.randn(n, 24, device=dev)
    model = GraphSAGE(24, 24, "mean", 3, 5, ffn_channels=40).to(dev)
    with torch.no_grad():
        out = model(x, ei)
        h0 = model.layers[0](x, ei).relu()
        b0 = reference(model.blocks[0], h0)[0].float().to(dev)
        h1 = model.layers[1](b0, ei).relu()
        b1 = reference(model.blocks[1], h1, b0)[0].float().to(dev)
        torch.testing.assert_close(out, model.layers[2](b1, ei), rtol=1e-4, atol=2e-5)


def test_trainer_runs_blocks_on_the_module_path(dev):
    from graphsage_amd.datasets import planted_partition
    from graphsage_amd.datasets.synthetic import _masks
    from graphsage_amd.engine import SageTrainEngine
    from graphsage_amd.samplers import NeighborSampler, UniformLoader
    from graphsage_amd.samplers.uniform_loader import device_graph
    from graphsage_amd.trainers import SupervisedGraphSageTrainerForNodeLevelTask
    torch.manual_seed(0)
    data = planted_partition(600, 6000, 24, 3, seed=1)
    _masks(data, 200, 100, 100, 0)
    model = GraphSAGE(24, 16, "mean", 2, 3, ffn_channels=32).to(dev)

    def trainer(**kw):
        return SupervisedGraphSageTrainerForNodeLevelTask(
            data, UniformLoader, 5, 5, loss_fn=F.cross_entropy, model=model, optimizer=torch.optim.Adam(model.parameters(), lr=1e-2),
            num_epochs=1, device=dev, supervised_only=True, **kw)
    before = [p.detach().clone() for p in model.parameters()]
    t = trainer()
    assert t.engine is None
    loss = t.train(1)
    assert math.isfinite(float(loss))
    assert all(not torch.equal(a, b) for a, b in zip(before, model.parameters()))
    assert 0 <= t.test()["test_acc"] <= 1
    with pytest.raises(RuntimeError, match="feed-forward"):
        trainer(use_engine=True)
    graph = device_graph(data)
    with pytest.raises(NotImplementedError, match="feed-forward"):
        SageTrainEngine(model, NeighborSampler(data, [5, 5], seed=0), graph.features(data), graph.labels(data), 64)
