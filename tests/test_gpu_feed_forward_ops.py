"""Operators of the feed-forward block (norm with the residual's addition, 8-bit output, 8-bit
products, gated projections) against their definitions in 64 bits.

Tolerances are bounds by arithmetic, element by element, from the 64-bit values: u is half a step of
the output's type (relative to the value), E = 2^-24 that of an fp32 operation, and a sum of n terms
in fp32, in any order, is off by at most n E times the sum of the magnitudes.
"""
import math

import pytest
import torch

from graphsage_amd import _lib, ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}   # half a subnormal step
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    over = (got - want).abs() - bound
    assert bool((over <= 0).all()), f"{what}: {int((over > 0).sum())} beyond their bound, worst by {float(over.max()):.3g}"


def norm_ref(x, w, r, eps):
    s = x.double() + (0 if r is None else r.double())
    rstd = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    return s, rstd, s * rstd * w.double()


# a row's fp32 statistics: a term's path through the tree is at most 64 additions (vectors of a thread, lanes, waves),
# so the mean is off by 66 E and its root by half of that; x + r, the two products and the root add a few E
STAT = 40 * E

ROWS = [(1, 1), (1, 7), (3, 64), (5, 255), (2, 256), (130, 602), (9, 1023), (4, 2047), (3, 4104), (2, 8192), (2, 16390), (1, 40001)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", ROWS)
def test_rms_norm_forward(dev, dtype, rows, dim):
    g = gen(dev, rows * 7919 + dim)
    x, r = normal(g, rows, dim, dtype=dtype, scale=3.0), normal(g, rows, dim, dtype=dtype)
    for w in (normal(g, dim, dtype=dtype), normal(g, dim)):
        for res in (None, r):
            y, total = ops.rms_norm_fwd(x, w, residual=res, eps=1e-6)
            s, rstd, want = norm_ref(x, w, res, 1e-6)
            if res is None:
                assert total is x
            else:
                within(total, s, s.abs() * (U[dtype] + E) + TINY[dtype], "sum")
            within(y, want, want.abs() * (U[dtype] + STAT) * (1 + 2 ** -7) + TINY[dtype], "y")


@pytest.mark.parametrize("dtype", DTYPES)
def test_rms_norm_strides_and_outputs(dev, dtype):
    """Rows that start anywhere, one row repeated (stride 0), outputs inside larger buffers, the
    residual stream updated in place; what lies around the outputs stays as it was."""
    g = gen(dev, 5)
    rows, dim = 37, 203
    big = normal(g, rows, 3 * dim + 5, dtype=dtype)
    x, r = big[:, 1:1 + dim], normal(g, 1, dim, dtype=dtype).expand(rows, dim)
    w = normal(g, dim, dtype=dtype)
    hold = torch.full((rows + 2, dim + 9), 7.0, dtype=dtype, device=dev)
    y, total = ops.rms_norm_fwd(x, w, residual=r, out=hold[1:-1, 3:3 + dim])
    want_y, want_s = ops.rms_norm_fwd(x.contiguous(), w, residual=r.contiguous())
    assert torch.equal(y, want_y) and torch.equal(total, want_s)
    hold[1:-1, 3:3 + dim] = 7.0
    assert bool((hold == 7.0).all())
    stream = r.contiguous()
    y2, s2 = ops.rms_norm_fwd(x, w, residual=stream, sum_out=stream)
    assert s2 is stream and torch.equal(stream, want_s) and torch.equal(y2, want_y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", ROWS)
def test_rms_norm_int8(dev, dtype, rows, dim):
    g = gen(dev, rows * 31 + dim)
    x, r, w = normal(g, rows, dim, dtype=dtype, scale=2.0), normal(g, rows, dim, dtype=dtype), normal(g, dim, dtype=dtype)
    q, scale, total = ops.rms_norm_int8(x, w, residual=r)
    s, rstd, y = norm_ref(x, w, r, 1e-6)
    within(total, s, s.abs() * (U[dtype] + E) + TINY[dtype], "sum")
    want = y.abs().amax(1) / 127
    within(scale, want, want * (STAT + 4 * E), "scale")
    # q is 127 t / max|t| with t off by 2 E and the quotient by 3 E: rounding adds half a step
    v = (s * w.double()) / (s * w.double()).abs().amax(1, keepdim=True) * 127
    within(q, v, 0.5 + 127 * 8 * E, "q")
    assert int(q.abs().max()) == 127
    wide, scale2, _ = ops.rms_norm_int8(x, w, residual=r, padded=True)
    assert wide.size(1) == (dim + 15) // 16 * 16 and torch.equal(wide[:, :dim], q) and torch.equal(scale, scale2)
    assert not wide[:, dim:].any()
    q3, scale3 = ops.quantize_rows(x)
    top = x.double().abs().amax(1)
    within(scale3, top / 127, top / 127 * 2 * E, "quantize_rows scale")
    within(q3, x.double() / top[:, None] * 127, 0.5 + 127 * 8 * E, "quantize_rows q")
    for out in DTYPES:
        back = ops.dequantize_rows(q, scale, out)
        want = q.double() * scale.double()[:, None]
        within(back, want, want.abs() * (U[out] + 2 * E) + TINY[out], "dequantize_rows")


def test_quantised_rows_of_special_values(dev):
    """Zeros, subnormals, the type's largest values, infinities and NaN in a row; its neighbours are
    not touched by them."""
    x = torch.ones(9, 130, device=dev)
    x[1] = 0.0
    x[2] = 0.0
    x[2, 77] = 2.0 ** -149
    x[3] *= 1e-38
    x[4, 3] = 3.4e38
    x[5, 129] = float("inf")
    x[6, 64] = float("nan")
    x[7, 0] = -float("inf")
    q, scale = ops.quantize_rows(x)
    for row in (5, 6, 7):
        assert math.isnan(float(scale[row])) and not q[row].any()
        assert bool(torch.isnan(ops.dequantize_rows(q, scale)[row]).all())
    assert float(scale[1]) == 0 and not q[1].any()
    assert int(q[2, 77]) == 127 and int(q[2].abs().sum()) == 127
    assert bool((q[3] == 127).all()) and int(q[4, 3]) == 127 and int(q[4].abs().sum()) == 127
    for row in (0, 8):
        assert bool((q[row] == 127).all()) and abs(float(scale[row]) * 127 - 1) <= 4 * E
    y, _ = ops.rms_norm_fwd(x, torch.ones(130, device=dev))
    assert bool(torch.isnan(y[6]).all()) and float(y[5, 0]) == 0 and math.isnan(float(y[5, 129]))
    assert not y[1].any() and bool(torch.isfinite(y[[0, 1, 2, 3, 8]]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", ROWS + [(4999, 96), (3000, 1200), (1500, 4100)])
def test_rms_norm_backward(dev, dtype, rows, dim):
    g = gen(dev, rows * 17 + dim)
    s, dy, ds = (normal(g, rows, dim, dtype=dtype) for _ in range(3))
    for w in (1 + normal(g, dim, dtype=dtype), 1 + normal(g, dim)):
        for dsum in (None, ds):
            dx, dw = ops.rms_norm_bwd(dy, s, w, dsum=dsum)
            s64, rstd, _ = norm_ref(s, w, None, 1e-6)
            xh, gw = s64 * rstd, dy.double() * w.double()
            c, c_mag = (gw * xh).mean(1, keepdim=True), (gw * xh).abs().mean(1, keepdim=True)
            want = rstd * (gw - xh * c) + (0 if dsum is None else ds.double())
            # c: 66 terms' additions on the magnitudes and the statistics; the rest a few operations each
            mag = rstd * (gw.abs() + xh.abs() * c_mag) + (0 if dsum is None else ds.double().abs())
            within(dx, want, mag * (72 * E + 2 * STAT) + want.abs() * U[dtype] * (1 + 2 ** -7) + TINY[dtype], "dx")
            want_w, mag_w = (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0)
            # a column's sum: at most rows / groups terms in a thread, then the groups; no more than rows + 16 in all
            within(dw, want_w, mag_w * ((min(rows, rows / 1024 + 1100) + 16) * E + STAT) + want_w.abs() * U[w.dtype] * (1 + 2 ** -7)
                   + TINY[w.dtype], "dw")
            again = ops.rms_norm_bwd(dy, s, w, dsum=dsum)
            assert torch.equal(again[0], dx) and torch.equal(again[1], dw)
            only = ops.rms_norm_bwd(dy, s, w, dsum=dsum, need_dw=False)
            assert only[1] is None and torch.equal(only[0], dx)
            only = ops.rms_norm_bwd(dy, s, w, dsum=dsum, need_dx=False)
            assert only[0] is None and torch.equal(only[1], dw)


# ------------------------------------------------------------------------------- 8-bit product
def eight(g, rows, k):
    q = torch.randint(-128, 128, (rows, k), generator=g, device=g.device, dtype=torch.int32).to(torch.int8)
    return q, 0.01 * (0.5 + torch.rand(rows, generator=g, device=g.device))


PRODUCTS = [(1, 1, 1), (1, 48, 16), (3, 17, 250), (16, 33, 64), (17, 130, 4096), (31, 64, 1008), (33, 257, 129), (64, 100, 528),
            (65, 16, 48), (65, 300, 16), (129, 127, 272), (200, 515, 602), (513, 258, 128), (1000, 2100, 144), (4099, 5003, 80)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_int8_linear(dev, m, n, k):
    g = gen(dev, m + n + k)
    (x, xs), (w, ws), bias = eight(g, m, k), eight(g, n, k), normal(g, n)
    acc = torch.mm(x.double(), w.double().t())            # whole numbers below 2^53: exact
    for out_dtype in DTYPES:
        for b in (None, bias):
            got = ops.int8_linear(x, xs, w, ws, bias=b, out_dtype=out_dtype)
            prod = acc * xs.double()[:, None] * ws.double()
            want = prod + (0 if b is None else b.double())
            within(got, want, prod.abs() * 4 * E + want.abs() * (U[out_dtype] + 2 * E) + TINY[out_dtype], f"{out_dtype} {b is None}")


def test_int8_linear_largest_sums(dev):
    """The widest row whose sum cannot leave 32 bits, all products at their largest; one more is refused."""
    k = 131056
    x = torch.full((2, k), -128, dtype=torch.int8, device=dev)
    one = torch.ones(2, device=dev)
    assert ops.int8_linear(x, one, x, one).tolist() == [[float(k * 16384)] * 2] * 2      # 17 bits times 2^14: exact in fp32
    with pytest.raises(RuntimeError, match="32 bits"):
        y = torch.zeros((2, k + 1), dtype=torch.int8, device=dev)
        ops.int8_linear(y, one, y, one)


def act64(v, name):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v / math.sqrt(2)))
    return v.clamp_min(0)


def slope64(v, name):
    if name == "silu":
        p = torch.sigmoid(v)
        return p * (1 + v * (1 - p))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v / math.sqrt(2))) + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    return (v > 0).double()


# fp32 evaluation of an activation or its slope: the exponential's argument rounds by E |g| (times log2 e), its
# value by 2 E more; division, erf and products add a few E.  |value| <= |g| + 0.2, |slope| <= 1.2.
def act_error(g, name):
    return (12 * E + 4 * E * g.abs()) * (g.abs() + 0.2)


def slope_error(g, name):
    return (16 * E + 6 * E * g.abs() * (1 + g.abs())) * 1.2


def gated_bound(g, u, dg, du, name):
    """Bound of |act(g) u| when g, u are off by dg, du (slopes of the activations stay below 1.2)."""
    a = act64(g, name)
    return (1.2 * dg + act_error(g, name)) * (u.abs() + du) + a.abs() * du + (a * u).abs() * 2 * E


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 40, 64), (5, 17, 250), (24, 130, 2048), (64, 48, 112), (65, 65, 96), (300, 515, 602), (1000, 4200, 144)])
def test_int8_gated_linear(dev, act, m, n, k):
    g = gen(dev, m * 3 + n + k)
    (x, xs), (w, ws), (v, vs) = eight(g, m, k), eight(g, n, k), eight(g, n, k)
    xs = xs * 0.02
    gate = torch.mm(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()
    up = torch.mm(x.double(), v.double().t()) * xs.double()[:, None] * vs.double()
    want = act64(gate, act) * up
    bound = gated_bound(gate, up, gate.abs() * 4 * E, up.abs() * 4 * E, act)
    for out_dtype in DTYPES:
        got = ops.int8_gated_linear(x, xs, w, ws, v, vs, activation=act, out_dtype=out_dtype)
        within(got, want, bound * (1 + 2 ** -7) + want.abs() * U[out_dtype] + TINY[out_dtype], f"{out_dtype}")


# ------------------------------------------------------------------------------- gated projections
GATED = [(1, 1, 1), (1, 40, 64), (4, 130, 600), (17, 33, 8), (64, 70, 1000), (65, 16, 24), (66, 65, 33), (130, 257, 128), (700, 530, 602), (2050, 2100, 72)]


def gated_ref(x, wg, wu, act):
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    # k products (exact or E each) and their sum in fp32
    k = x.size(1) + 2
    return g, u, x.abs() @ wg.abs().t() * k * E, x.abs() @ wu.abs().t() * k * E


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h,k", GATED)
def test_gated_linear_forward(dev, dtype, act, m, h, k):
    rng = gen(dev, m + h * 3 + k)
    x, wg, wu = normal(rng, m, k, dtype=dtype, scale=2.0), normal(rng, h, k, dtype=dtype, scale=k ** -0.5), normal(rng, h, k, dtype=dtype, scale=k ** -0.5)
    out, saved = ops.gated_linear_fwd(x, wg, wu, activation=act, save=True)
    g, u, dg, du = gated_ref(x, wg, wu, act)
    within(saved[0], g, dg + g.abs() * E, "gate")
    within(saved[1], u, du + u.abs() * E, "up")
    want = act64(g, act) * u
    within(out, want, gated_bound(g, u, dg, du, act) * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype], "out")
    plain, none = ops.gated_linear_fwd(x, wg, wu, activation=act)
    assert none is None and torch.equal(plain, out)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h,k", GATED)
def test_gated_linear_backward(dev, dtype, act, m, h, k):
    rng = gen(dev, m + h * 5 + k)
    x, wg, wu = normal(rng, m, k, dtype=dtype), normal(rng, h, k, dtype=dtype, scale=k ** -0.5), normal(rng, h, k, dtype=dtype, scale=k ** -0.5)
    dh = normal(rng, m, h, dtype=dtype)
    _, saved = ops.gated_linear_fwd(x, wg, wu, activation=act, save=True)
    dx, dwg, dwu = ops.gated_linear_bwd(dh, x, wg, wu, saved, activation=act)
    # from the saved products, which the forward test bounds: what is left is the operands' rounding
    g, u, d = saved[0].double(), saved[1].double(), dh.double()
    slope, a = slope64(g, act), act64(g, act)
    dg, du = d * u * slope, d * a
    dg_off = (d * u).abs() * slope_error(g, act) + dg.abs() * (U[dtype] + 3 * E) * (1 + 2 ** -7) + TINY[dtype]
    du_off = d.abs() * act_error(g, act) + du.abs() * (U[dtype] + 3 * E) * (1 + 2 ** -7) + TINY[dtype]
    x64, g64, u64 = x.double(), wg.double(), wu.double()

    def check(got, want, mag, off, terms, what):
        within(got, want, off + (mag + off) * (terms + 2) * E + want.abs() * U[dtype] * (1 + 2 ** -7) + TINY[dtype], what)

    check(dx, dg @ g64 + du @ u64, dg.abs() @ g64.abs() + du.abs() @ u64.abs(), dg_off @ g64.abs() + du_off @ u64.abs(), 2 * h, "dx")
    check(dwg, dg.t() @ x64, dg.abs().t() @ x64.abs(), dg_off.t() @ x64.abs(), m, "dw_gate")
    check(dwu, du.t() @ x64, du.abs().t() @ x64.abs(), du_off.t() @ x64.abs(), m, "dw_up")
    one = ops.gated_linear_bwd(dh, x, wg, wu, saved, activation=act, need_dw=False)
    assert one[1] is None and one[2] is None and torch.equal(one[0], dx)
    one = ops.gated_linear_bwd(dh, x, wg, wu, saved, activation=act, need_dx=False)
    assert one[0] is None and torch.equal(one[1], dwg) and torch.equal(one[2], dwu)


@pytest.mark.parametrize("dtype", DTYPES + [torch.int8])
def test_products_take_any_rows(dev, dtype):
    """Views whose rows start anywhere or repeat, and an output inside a larger buffer."""
    rng = gen(dev, 11)
    for m in (9, 140):
        big = normal(rng, m, 400, scale=30.0).to(dtype)
        w = normal(rng, 77, 400, scale=30.0).to(dtype)
        x, wg, wu = big[:, 3:3 + 96], w[:, 16:112], w[:, 201:297]
        row = x[:1].expand(m, 96)
        hold = torch.full((m + 1, 90), 5.0, dtype=torch.float32 if dtype == torch.int8 else dtype, device=dev)
        for a in (x, row):
            if dtype == torch.int8:
                s, t = torch.ones(m, device=dev) * 1e-3, torch.ones(77, device=dev) * 1e-3
                got = ops.int8_gated_linear(a, s, wg, t, wu, t, out=hold[:m, 5:82])
                want = ops.int8_gated_linear(a.contiguous(), s, wg.contiguous(), t, wu.contiguous(), t)
                plain = ops.int8_linear(a, s, wg, t, out_dtype=torch.float32)
                assert torch.equal(plain, ops.int8_linear(a.contiguous(), s, wg.contiguous(), t))
            else:
                got = ops.gated_linear_fwd(a, wg, wu, out=hold[:m, 5:82])[0]
                want = ops.gated_linear_fwd(a.contiguous(), wg.contiguous(), wu.contiguous())[0]
            assert torch.equal(got, want)
            hold[:m, 5:82] = 5.0
            assert bool((hold == 5.0).all())


@pytest.mark.parametrize("dtype", DTYPES + [torch.int8])
@pytest.mark.parametrize("m,n,k", [(1, 9, 17), (4, 4100, 37), (16, 700, 1999), (20, 4099, 1023), (24, 50, 4111), (40, 33, 517), (200, 300, 65)])
def test_few_rows_of_odd_lengths(dev, dtype, m, n, k):
    """Rows of any length and start, with NaN (8 bits: 127) around them, give what whole pieces give."""
    rng = gen(dev, m + n + k)
    one = 127 if dtype == torch.int8 else float("nan")

    def inside(rows):
        hold = torch.full((rows + 2, k + 6), one, dtype=dtype, device=dev)
        hold[1:-1, 3:-3] = normal(rng, rows, k, scale=40.0 if dtype == torch.int8 else 1.0).clamp(-127, 127).to(dtype)
        view = hold[1:-1, 3:-3]
        return view, torch.nn.functional.pad(view, (0, 16 - k % 16))

    (x, x16), (wg, wg16), (wu, wu16) = inside(m), inside(n), inside(n)
    if dtype == torch.int8:
        s, t = torch.rand(m, generator=rng, device=dev) * 1e-2, torch.rand(n, generator=rng, device=dev) * 1e-2
        assert torch.equal(ops.int8_linear(x, s, wg, t), ops.int8_linear(x16, s, wg16, t))
        assert torch.equal(ops.int8_gated_linear(x, s, wg, t, wu, t), ops.int8_gated_linear(x16, s, wg16, t, wu16, t))
        return
    got, saved = ops.gated_linear_fwd(x, wg, wu, save=True)
    g, u, dg, du = gated_ref(x, wg, wu, "silu")
    within(saved[0], g, dg + g.abs() * E, "gate")
    within(saved[1], u, du + u.abs() * E, "up")
    want = act64(g, "silu") * u
    within(got, want, gated_bound(g, u, dg, du, "silu") * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype], "out")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gated_backward_takes_repeated_rows(dev, dtype):
    """x and both weights as one row repeated (stride 0), and weights that are every other row of a buffer."""
    rng = gen(dev, 5)
    x, w = normal(rng, 1, 64, dtype=dtype).expand(40, 64), normal(rng, 1, 64, dtype=dtype).expand(24, 64)
    v = normal(rng, 48, 64, dtype=dtype)[::2]
    for args in ((x, w, w), (x, v, w), (x.contiguous(), v, v)):
        dh = normal(rng, 40, 24, dtype=dtype)
        full = [t.contiguous() for t in args]
        saved = ops.gated_linear_fwd(*args, save=True)[1]
        assert torch.equal(saved, ops.gated_linear_fwd(*full, save=True)[1])
        for got, want in zip(ops.gated_linear_bwd(dh, *args, saved), ops.gated_linear_bwd(dh, *full, saved)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("rows,dim,dtype", [(2 ** 26 + 5, 8, torch.bfloat16), (2 ** 22 + 3, 2056, torch.bfloat16), (2 ** 22 + 3, 1032, torch.float32)])
def test_rms_norm_of_very_many_rows(dev, rows, dim, dtype):
    """More rows than one dimension of a grid takes threads for, as one row repeated and its last rows others."""
    rng = gen(dev, dim)
    row, w = normal(rng, 1, dim, dtype=dtype), normal(rng, dim, dtype=dtype)
    y, _ = ops.rms_norm_fwd(row.expand(rows, dim), w)
    want = ops.rms_norm_fwd(row.expand(2048, dim), w)[0][:1]
    for at in (0, 2 ** 20 - 1, 2 ** 20, 2 ** 22, rows - 1):
        assert torch.equal(y[at:at + 1], want), at
    q, scale = ops.quantize_rows(row.expand(rows, dim))
    want, one = ops.quantize_rows(row.expand(2048, dim))
    for at in (0, 2 ** 20, 2 ** 22, rows - 1):
        assert torch.equal(q[at], want[0]) and torch.equal(scale[at], one[0]), at


def test_products_behind_32_bit_offsets(dev):
    """More than 2^31 outputs, saved sums and weight bytes: the last rows against calls of their own.  Small whole
    numbers, so that every sum is exact and the order of its terms is free."""
    rng = gen(dev, 31)
    m, h, k, last = 66000, 33000, 32, 5

    def whole(rows, cols, dtype):
        return torch.randint(-1, 2, (rows, cols), generator=rng, device=dev, dtype=torch.int8).to(dtype)

    x, w, v = (whole(n, k, torch.int8) for n in (m, h, h))
    sx, sw = torch.rand(m, generator=rng, device=dev), torch.rand(h, generator=rng, device=dev)
    out = ops.int8_linear(x, sx, w, sw, out_dtype=torch.bfloat16)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-last:], ops.int8_linear(x[-last:], sx[-last:], w, sw, out_dtype=torch.bfloat16))
    del out
    x, w, v = x.bfloat16(), w.bfloat16(), v.bfloat16()
    out, saved = ops.gated_linear_fwd(x, w, v, "relu", save=True)
    end, end_saved = ops.gated_linear_fwd(x[-last:], w, v, "relu", save=True)
    assert torch.equal(out[-last:], end) and torch.equal(saved[:, -last:], end_saved)
    dh = out.zero_()
    dh[-last:] = whole(last, h, torch.bfloat16)
    got = ops.gated_linear_bwd(dh, x, w, v, saved, "relu")
    want = ops.gated_linear_bwd(dh[-last:], x[-last:], w, v, end_saved, "relu")
    assert torch.equal(got[0][-last:], want[0]) and not got[0][:-last].any()
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])
    del out, saved, dh
    n, k = 2 ** 24 + 21, 130           # weights of more than 2^31 bytes, few rows
    w = torch.randint(-2, 3, (n, k), generator=rng, device=dev, dtype=torch.int8)
    x, sx, sw = whole(3, k, torch.int8), torch.ones(3, device=dev), torch.ones(n, device=dev)
    out = ops.int8_linear(x, sx, w, sw)
    for at in (0, 2 ** 24 - 1, n - 40):
        assert torch.equal(out[:, at:at + 40].double(), x.double() @ w[at:at + 40].double().t()), at


def test_norm_outputs_that_share_memory(dev):
    """An output may be an input, row for row; shifted against one, or both outputs in one buffer, is refused."""
    rng = gen(dev, 3)
    hold, w = normal(rng, 41, 96), normal(rng, 96)
    x, r = hold[:20], hold[20:40]
    y, s = ops.rms_norm_fwd(x, w, r)
    for kw in (dict(out=hold[1:21]), dict(sum_out=hold[21:41]), dict(out=r, sum_out=r), dict(sum_out=hold.view(-1)[8:8 + 1920].view(20, 96))):
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.rms_norm_fwd(x, w, r, **kw)
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.rms_norm_int8(x, w, r, sum_out=hold[21:41])
    y2, s2 = ops.rms_norm_fwd(x, w, r, out=x, sum_out=r)
    assert torch.equal(y, y2) and torch.equal(s, s2)


def test_not_a_number_stays_in_its_row(dev):
    """A NaN in a row of x reaches that row's outputs and no others, also through rows that fill a tile."""
    for m in (3, 70, 300):
        for dtype in DTYPES:
            x, w = torch.ones(m, 72, dtype=dtype, device=dev), torch.ones(33, 72, dtype=dtype, device=dev)
            x[m - 1, 71] = float("nan")
            out, _ = ops.gated_linear_fwd(x, w, w)
            assert bool(torch.isnan(out[m - 1]).all()) and bool(torch.isfinite(out[:m - 1]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h,k", [(1, 1, 8), (1, 130, 208), (3, 17, 40), (40, 33, 24), (70, 130, 136), (300, 515, 200), (129, 257, 264)])
def test_backward_writes_its_outputs_only(dev, dtype, m, h, k):
    """dx and dw in the middle of buffers whose other elements stay as they were (widths that are no whole
    runs, rows that fill no tile), and the workspace's next bytes too."""
    rng = gen(dev, m + h + k)
    x, wg, wu, dh = normal(rng, m, k, dtype=dtype), normal(rng, h, k, dtype=dtype), normal(rng, h, k, dtype=dtype), normal(rng, m, h, dtype=dtype)
    _, saved = ops.gated_linear_fwd(x, wg, wu, save=True)
    want = ops.gated_linear_bwd(dh, x, wg, wu, saved)
    room = 256 * max(k, 64)
    dx = torch.full((m * k + 2 * room,), 3.0, dtype=dtype, device=dev)
    dw = torch.full((2 * h * k + 2 * room,), 3.0, dtype=dtype, device=dev)
    kind = ops.ROW_DTYPES[dtype]
    size = _lib.load().sage_gated_linear_bwd_workspace_bytes(m, h, k, kind)
    ws = torch.full((size + (1 << 20),), 77, dtype=torch.uint8, device=dev)
    one = x.element_size()
    ops._call("sage_gated_linear_bwd", dev, dh.data_ptr(), h, x.data_ptr(), k, wg.data_ptr(), k, wu.data_ptr(), k, saved.data_ptr(), 0,
              m, h, k, kind, dx.data_ptr() + room * one, k, dw.data_ptr() + room * one, ws.data_ptr(), size)
    assert torch.equal(dx[room:-room].view(m, k), want[0])
    assert torch.equal(dw[room:-room].view(2 * h, k), torch.cat(want[1:]))
    assert bool((dx[:room] == 3).all()) and bool((dx[-room:] == 3).all())
    assert bool((dw[:room] == 3).all()) and bool((dw[-room:] == 3).all())
    assert bool((ws[size:] == 77).all())


def test_refusals(dev):
    """Wrong types, shapes, strides and outputs, before anything is launched."""
    x, w = torch.zeros(4, 32, device=dev), torch.ones(32, device=dev)
    q, s = torch.zeros(4, 32, dtype=torch.int8, device=dev), torch.ones(4, device=dev)
    wide = torch.zeros(4, 64, device=dev)
    half, saved = x.bfloat16(), torch.zeros(2, 4, 4, device=dev)
    for call in (lambda: ops.rms_norm_fwd(x.double(), w), lambda: ops.rms_norm_fwd(x, w[:-1]), lambda: ops.rms_norm_fwd(x, w.bfloat16()),
                 lambda: ops.rms_norm_fwd(x, None), lambda: ops.rms_norm_fwd(x.t(), w[:4]), lambda: ops.rms_norm_fwd(x, w, residual=half),
                 lambda: ops.rms_norm_fwd(x, w, residual=wide), lambda: ops.rms_norm_fwd(x, w, sum_out=wide[:, :32]),
                 lambda: ops.rms_norm_fwd(x, w, out=x[:1].expand(4, 32)), lambda: ops.rms_norm_fwd(x, w, out=half),
                 lambda: ops.rms_norm_fwd(x[:, :0], w[:0]), lambda: ops.rms_norm_fwd(x[0], w), lambda: ops.rms_norm_fwd(x, w.cpu()),
                 lambda: ops.rms_norm_bwd(half, x, w), lambda: ops.rms_norm_bwd(x, x, w, dsum=wide), lambda: ops.rms_norm_bwd(x, x, w, need_dx=False, need_dw=False),
                 lambda: ops.rms_norm_int8(x, None), lambda: ops.quantize_rows(q), lambda: ops.dequantize_rows(q, s[:3]), lambda: ops.dequantize_rows(q, s, torch.float64),
                 lambda: ops.int8_linear(x, s, q, s), lambda: ops.int8_linear(q, s[:2], q, s), lambda: ops.int8_linear(q, s, q[:, :16], s),
                 lambda: ops.int8_linear(q, s, q, s, bias=w), lambda: ops.int8_linear(q, s, q, s, out_dtype=torch.int8),
                 lambda: ops.int8_linear(q, s, q, s.half()), lambda: ops.int8_linear(q, s, q, s, out=wide), lambda: ops.int8_linear(q, s, q[:0], s[:0]),
                 lambda: ops.int8_gated_linear(q, s, q, s, q[:2], s[:2]), lambda: ops.int8_gated_linear(q, s, q, s, q, s, activation="tanh"),
                 lambda: ops.gated_linear_fwd(x, half, x), lambda: ops.gated_linear_fwd(x, x, x[:2]), lambda: ops.gated_linear_fwd(x, wide, wide),
                 lambda: ops.gated_linear_fwd(x, x, x, activation="none"), lambda: ops.gated_linear_fwd(x, x, x, out=x[:, :4]),
                 lambda: ops.gated_linear_fwd(wide[:, 32:], x, x, out=wide[:, 30:34]),
                 lambda: ops.gated_linear_bwd(x, x, x, x, saved), lambda: ops.gated_linear_bwd(wide[:, :4], x, x, x, saved[:, :, :3]),
                 lambda: ops.gated_linear_bwd(wide[:, :4], x, x, x, None), lambda: ops.gated_linear_bwd(wide[:, :4], x, x, x, saved, need_dx=False, need_dw=False)):
        with pytest.raises(RuntimeError):
            call()
    ops.gated_linear_fwd(wide[:, 32:], x, x, out=wide[:, 28:32])       # columns of one buffer that lie apart


def test_empty_inputs(dev):
    for dtype in DTYPES:
        x, w = torch.zeros(0, 24, dtype=dtype, device=dev), torch.ones(24, dtype=dtype, device=dev)
        wg = torch.ones(5, 24, dtype=dtype, device=dev)
        y, s = ops.rms_norm_fwd(x, w, residual=x)
        assert y.shape == s.shape == (0, 24)
        dx, dw = ops.rms_norm_bwd(y, s, w)
        assert dx.shape == (0, 24) and not dw.any()
        q, scale, _ = ops.rms_norm_int8(x, w)
        assert q.shape == (0, 24) and scale.shape == (0,) and ops.dequantize_rows(q, scale).shape == (0, 24)
        h, saved = ops.gated_linear_fwd(x, wg, wg, save=True)
        assert h.shape == (0, 5)
        dx, dwg, dwu = ops.gated_linear_bwd(h, x, wg, wg, saved)
        assert dx.shape == (0, 24) and not dwg.any() and not dwu.any()
        wq, ws = ops.quantize_rows(wg)
        assert ops.int8_linear(q, scale, wq, ws).shape == (0, 5) and ops.int8_gated_linear(q, scale, wq, ws, wq, ws).shape == (0, 5)
