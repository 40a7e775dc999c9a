"""Cases of the residual feed-forward block's operators (graphsage_amd/ops.py): the root-mean-square
norm with the residual's addition (own type, 8 bits with row scales, forward + backward), the 8-bit
product with token and channel scales, and the gated projections with their backward pass.

`own` chooses between the plain form (elementary torch operations in 32 bits) and the framework's
kernels; both take what `prepare` makes.
"""
import math

import torch

own = False

EPS = 1e-6
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # ---- norm: rows x dim
        # one decoding step of eight sequences: latency
        dict(name="norm_rows8", op="norm", rows=8, dim=4096, dtype="bf16", residual=True, mode="fwd"),
        # the norm in front of an 8-bit product, a prompt's worth of rows
        dict(name="norm_int8_prompt", op="norm", rows=8192, dim=5120, dtype="bf16", residual=True, mode="int8"),
        # hidden rows of the 25/10 fan-out with 512 seeds, width 256: one training step's norm
        dict(name="norm_train_sage", op="norm", rows=13312, dim=256, dtype="f32", residual=True, mode="train"),
        # a training batch, ragged row count, odd width
        dict(name="norm_train_ragged", op="norm", rows=16381, dim=2047, dtype="bf16", residual=True, mode="train"),
        # ---- 8-bit product: m x n over k
        # single token against a square layer: the weights' bytes are the floor
        dict(name="int8_token", op="int8", m=1, n=4096, k=4096, out="bf16", bias=False, gated=False),
        # a small decoding batch through the gated pair of an 8-bit block
        dict(name="int8_gated_batch", op="int8", m=24, n=8192, k=2048, out="bf16", bias=False, gated=True),
        # ragged: class count of a hidden layer, odd rows, sampled batch
        dict(name="int8_ragged", op="int8", m=1409, n=1031, k=608, out="f32", bias=True, gated=False),
        # whole-graph inference / a long prompt: compute bound
        dict(name="int8_large", op="int8", m=8192, n=8192, k=8192, out="bf16", bias=True, gated=False),
        # ---- gated projections: m x h over k
        # single tokens of a few sequences
        dict(name="gated_rows4", op="gated", m=4, h=5632, k=2048, dtype="bf16", act="silu", train=False),
        # one training step behind a 256-wide aggregation, the framework's own type
        dict(name="gated_train_sage", op="gated", m=13312, h=1024, k=256, dtype="f32", act="silu", train=True),
        # ragged rows and widths, half precision
        dict(name="gated_train_ragged", op="gated", m=1999, h=2730, k=1000, dtype="f16", act="gelu", train=True),
        # a training batch: compute bound
        dict(name="gated_train_large", op="gated", m=8192, h=8192, k=2048, dtype="bf16", act="silu", train=True),
    ]


def _spread(rng, low, high, step=1):
    """A whole number of [low, high], spread over the logarithm; rounded to `step` where it is not 1."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(step, min(high, (v + step - 1) // step * step))


def draw(rng):
    op = rng.choice(["norm", "int8", "gated"])
    step = rng.choice([1, 8, 64])          # odd widths, widths of whole vectors, widths of whole tiles
    if op == "norm":
        dim = _spread(rng, 64, 8192, step)
        rows = min(_spread(rng, 1, 32768), (1 << 26) // dim)
        return dict(op=op, rows=rows, dim=dim, dtype=rng.choice(["bf16", "f16", "f32"]),
                    residual=rng.random() < 0.75, mode=rng.choice(["fwd", "int8", "train"]))
    if op == "int8":
        gated = rng.random() < 0.3
        return dict(op=op, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 8192, step),
                    k=_spread(rng, 64, 4096 if gated else 8192, step),
                    out=rng.choice(["bf16", "f16", "f32"]), bias=not gated and rng.random() < 0.5, gated=gated)
    train = rng.random() < 0.5
    return dict(op=op, m=_spread(rng, 1, 8192), h=_spread(rng, 32, 8192, step), k=_spread(rng, 32, 2048, step),
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), act=rng.choice(["silu", "gelu", "relu"]), train=train)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device=dev) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "norm":
        rows, dim, dt = case["rows"], case["dim"], DTYPE[case["dtype"]]
        # a residual stream: rows of different loudness, a few channels far louder than the rest
        loud = torch.exp(0.5 * normal(rows, 1))
        channel = torch.where(torch.rand(dim, generator=gen, device=dev) < 0.01, 8.0, 1.0)
        s["x"] = (normal(rows, dim) * loud * channel).to(dt)
        s["r"] = normal(rows, dim, dtype=dt) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * normal(dim)).to(dt)
        if case["mode"] == "train":
            s["dy"] = normal(rows, dim, dtype=dt)
            s["ds"] = normal(rows, dim, dtype=dt) if case["residual"] else None
    elif case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]

        def eight(rows):
            q = torch.round(normal(rows, k, scale=36.0)).clamp_(-127, 127).to(torch.int8)
            return q, 0.005 * (0.5 + torch.rand(rows, generator=gen, device=dev))

        s["xq"], s["xs"] = eight(m)
        s["wq"], s["ws"] = eight(n)
        if case["gated"]:
            s["uq"], s["us"] = eight(n)
        s["bias"] = normal(n) if case["bias"] and not case["gated"] else None
    else:
        m, h, k, dt = case["m"], case["h"], case["k"], DTYPE[case["dtype"]]
        s["x"] = normal(m, k, dtype=dt)
        s["wg"] = normal(h, k, scale=k ** -0.5, dtype=dt)
        s["wu"] = normal(h, k, scale=k ** -0.5, dtype=dt)
        if case["train"]:
            s["dh"] = normal(m, h, dtype=dt)
    return s


# ------------------------------------------------------------------------------- plain forms
def _act(g, name):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "gelu":
        return 0.5 * g * (1.0 + torch.erf(g * 0.5 ** 0.5))
    return torch.clamp(g, min=0.0)


def _act_slope(g, name):
    if name == "silu":
        p = torch.sigmoid(g)
        return p * (1.0 + g * (1.0 - p))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5)) + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5
    return (g > 0).to(g.dtype)


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    w = s["w"].float()
    t = s["x"].float() if s["r"] is None else s["x"].float() + s["r"].float()
    rstd = torch.rsqrt(t.square().mean(dim=-1, keepdim=True) + EPS)
    out = {} if s["r"] is None else {"sum": t.to(dt)}
    if c["mode"] == "int8":
        # in 64 bits: a value next to the middle of two steps has to fall on its own side
        v = s["x"].double() if s["r"] is None else s["x"].double() + s["r"].double()
        v = v * s["w"].double()
        top = v.abs().amax(dim=-1, keepdim=True)
        q = torch.round(v * torch.where(top > 0, 127.0 / top, 0.0))
        scale = (top.float() * rstd / 127.0)
        out["y"] = (q.float() * scale).to(torch.bfloat16)     # the values that the 8 bits stand for
        out["scale"] = scale[:, 0]
        return out
    out["y"] = (t * rstd * w).to(dt)
    if c["mode"] == "train":
        dy = s["dy"].float()
        xh, dyw = t.to(dt).float() * rstd, dy * w             # the backward pass starts from the sum as it is stored
        dx = rstd * (dyw - xh * (dyw * xh).mean(dim=-1, keepdim=True))
        out["dx"] = (dx if s["ds"] is None else dx + s["ds"].float()).to(dt)
        out["dw"] = (dy * xh).sum(dim=0).to(s["w"].dtype)
    return out


def _plain_int8(s):
    c = s["case"]
    x = s["xq"].float()
    g = (x @ s["wq"].float().t()) * s["xs"][:, None] * s["ws"][None, :]
    if c["gated"]:
        g = _act(g, "silu") * ((x @ s["uq"].float().t()) * s["xs"][:, None] * s["us"][None, :])
    elif s["bias"] is not None:
        g = g + s["bias"]
    return g.to(DTYPE[c["out"]])


def _plain_gated(s):
    c, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["wg"].float(), s["wu"].float()
    g, u = x @ wg.t(), x @ wu.t()
    a = _act(g, c["act"])
    out = {"h": (a * u).to(dt)}
    if c["train"]:
        dh = s["dh"].float()
        dg, du = dh * u * _act_slope(g, c["act"]), dh * a
        out["dx"] = (dg @ wg + du @ wu).to(dt)
        out["dwg"] = (dg.t() @ x).to(dt)
        out["dwu"] = (du.t() @ x).to(dt)
    return out


# ------------------------------------------------------------------------------- the framework's calls
def _own_norm(s):
    from graphsage_amd import ops
    c = s["case"]
    if c["mode"] == "int8":
        q, scale, total = ops.rms_norm_int8(s["x"], s["w"], residual=s["r"], eps=EPS)
        out = {"y": ops.dequantize_rows(q, scale, torch.bfloat16), "scale": scale}
    else:
        y, total = ops.rms_norm_fwd(s["x"], s["w"], residual=s["r"], eps=EPS)
        out = {"y": y}
    if s["r"] is not None:
        out["sum"] = total
    if c["mode"] == "train":
        out["dx"], out["dw"] = ops.rms_norm_bwd(s["dy"], total, s["w"], eps=EPS, dsum=s["ds"])
    return out


def _own_int8(s):
    from graphsage_amd import ops
    c = s["case"]
    if c["gated"]:
        return ops.int8_gated_linear(s["xq"], s["xs"], s["wq"], s["ws"], s["uq"], s["us"], activation="silu",
                                     out_dtype=DTYPE[c["out"]])
    return ops.int8_linear(s["xq"], s["xs"], s["wq"], s["ws"], bias=s["bias"], out_dtype=DTYPE[c["out"]])


def _own_gated(s):
    from graphsage_amd import ops
    c = s["case"]
    if not c["train"]:
        return {"h": ops.gated_linear_fwd(s["x"], s["wg"], s["wu"], activation=c["act"])[0]}
    h, saved = ops.gated_linear_fwd(s["x"], s["wg"], s["wu"], activation=c["act"], save=True)
    dx, dwg, dwu = ops.gated_linear_bwd(s["dh"], s["x"], s["wg"], s["wu"], saved, activation=c["act"])
    return {"h": h, "dx": dx, "dwg": dwg, "dwu": dwu}


def run(state):
    op = state["case"]["op"]
    if op == "norm":
        return _own_norm(state) if own else _plain_norm(state)
    if op == "int8":
        return _own_int8(state) if own else _plain_int8(state)
    return _own_gated(state) if own else _plain_gated(state)


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "norm":
        rows, dim, size = case["rows"], case["dim"], SIZE[case["dtype"]]
        n, wide = rows * dim, 2 if case["residual"] else 1
        if case["mode"] == "int8":
            # x, r read; the sum, the 8 bits and the scales written; the 8 bits read back into 16
            return {"bytes": n * (size * (2 * wide - 1) + 1 + 1 + 2) + 8 * rows + dim * size, "flops": 9 * n}
        if case["mode"] == "fwd":
            return {"bytes": n * size * 2 * wide + dim * size, "flops": 5 * n}
        # x, dy read and y, dx written; with a residual r, ds read and the sum written too
        return {"bytes": n * size * (7 if case["residual"] else 4) + 2 * dim * size, "flops": 15 * n}
    if case["op"] == "int8":
        m, n, k, pair = case["m"], case["n"], case["k"], 2 if case["gated"] else 1
        return {"bytes": m * k + pair * n * k + m * n * SIZE[case["out"]] + 4 * (m + pair * n), "flops": 2 * pair * m * n * k}
    m, h, k, size = case["m"], case["h"], case["k"], SIZE[case["dtype"]]
    if not case["train"]:
        return {"bytes": size * (m * k + 2 * h * k + m * h), "flops": 4 * m * h * k}
    return {"bytes": size * (2 * m * k + 4 * h * k + 2 * m * h), "flops": 12 * m * h * k}


# ------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """From the definitions, apart from the forms above: derivatives by torch's differentiation where there are any."""
    s = prepare(case, seed)
    d = {name: v.double() for name, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "norm":
        total = d["x"] + d["r"] if case["residual"] else d["x"]
        size = torch.linalg.vector_norm(total, dim=1, keepdim=True) / math.sqrt(case["dim"])
        unit = total / torch.sqrt(size ** 2 + EPS)
        out = {"sum": total} if case["residual"] else {}
        if case["mode"] == "int8":
            v = unit * d["w"]
            scale = v.abs().max(dim=1).values / 127
            out["y"] = torch.round(v / scale[:, None]) * scale[:, None]
            out["scale"] = scale
            return out
        out["y"] = unit * d["w"]
        if case["mode"] == "train":
            with torch.enable_grad():
                leaf, w = total.to(s["x"].dtype).double().requires_grad_(), d["w"].clone().requires_grad_()
                y = leaf * (leaf.pow(2).sum(dim=1, keepdim=True) / case["dim"] + EPS).pow(-0.5)
                out["dx"], out["dw"] = torch.autograd.grad(y * w, (leaf, w), d["dy"])
            if case["residual"]:
                out["dx"] = out["dx"] + d["ds"]
        return out
    if case["op"] == "int8":
        g = torch.mm(d["xq"] * d["xs"][:, None], (d["wq"] * d["ws"][:, None]).t())
        if case["gated"]:
            return g / (1 + torch.exp(-g)) * torch.mm(d["xq"] * d["xs"][:, None], (d["uq"] * d["us"][:, None]).t())
        return g + d["bias"] if case["bias"] else g
    with torch.enable_grad():
        leaves = [d[name].requires_grad_(case["train"]) for name in ("x", "wg", "wu")]
        g = torch.mm(leaves[0], leaves[1].t())
        a = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.nn.functional.relu}[case["act"]](g)
        h = a * torch.mm(leaves[0], leaves[2].t())
        out = {"h": h.detach()}
        if case["train"]:
            out["dx"], out["dwg"], out["dwu"] = torch.autograd.grad(h, leaves, d["dh"])
    return out
