"""Every cut that the feed-forward block's products take: both tiles in each type and direction, k whole and in
slices, with few and many runs of 64 bytes a block and runs that k does not fill, rows and columns that fill no tile; the
few-rows kernels that aligned rows take; and the norm's kernels for many rows of two to four vectors a thread.  Each
case first asks the library whether these sizes still take the cut that they are here for.

Bounds as in the operators' tests: from the 64-bit values, by arithmetic.
"""
import pytest
import torch

from graphsage_amd import ops
from tests.test_gpu_feed_forward_ops import (DTYPES, E, STAT, TINY, U, act64, act_error, eight, gated_bound, gated_ref, gen, norm_ref,
                                             normal, slope64, slope_error, within)

pytestmark = pytest.mark.gpu
SIZE = {torch.float32: 4, torch.bfloat16: 2, torch.float16: 2, torch.int8: 1}


def row_bytes(k, size):
    """Of rows in whole pieces of 16 bytes, as the tile kernels take them."""
    return (k * size + 15) // 16 * 16


def in_a_last_slice(k_bytes, slices):
    """Runs of 64 bytes that the last slice of k has."""
    runs, steps = -(-k_bytes // 64), -(-k_bytes // 128)
    return runs - (slices - 1) * 2 * -(-steps // slices)


# ------------------------------------------------------------------------------- 8 bits
# (tile, slices): m, n, k.  The unsplit 256 tile with 5 to 12 and 29 runs, whole and not; last slices of 1 to 7 runs
EIGHT = [((256, 1), 3255, 3727, 282), ((256, 1), 3001, 4097, 384), ((256, 1), 3255, 3727, 447), ((256, 1), 3255, 3727, 512),
         ((256, 1), 3001, 4097, 560), ((256, 1), 3255, 3727, 767), ((256, 1), 3001, 4097, 1856),
         ((256, 2), 518, 7505, 6254), ((256, 3), 1153, 3324, 4139), ((256, 3), 1000, 4099, 4100), ((256, 4), 530, 4440, 15809),
         ((256, 6), 4171, 388, 9765), ((256, 10), 2748, 391, 17687), ((256, 16), 3325, 169, 39451),
         ((256, 24), 2138, 157, 64810), ((256, 32), 144, 1648, 87378), ((256, 24), 154, 2060, 64918), ((256, 24), 133, 2390, 70888),
         ((256, 32), 1665, 134, 83586), ((256, 24), 2099, 137, 68153),
         ((128, 1), 547, 1033, 600), ((128, 2), 514, 2220, 3484), ((128, 3), 4155, 38, 2182), ((128, 4), 1043, 137, 1947),
         ((128, 5), 543, 34, 1589), ((128, 6), 36, 45, 5361), ((128, 8), 525, 36, 1899), ((128, 12), 513, 43, 2856),
         ((128, 24), 517, 44, 8906), ((128, 32), 18, 33, 8100), ((128, 48), 520, 51, 30341), ((128, 64), 24, 35, 16322)]


@pytest.mark.parametrize("cut,m,n,k", EIGHT)
def test_int8_linear_cuts(dev, cut, m, n, k):
    assert ops.product_cut(m, n, row_bytes(k, 1)) == cut
    g = gen(dev, m + n + k)
    (x, xs), (w, ws), bias = eight(g, m, k), eight(g, n, k), normal(g, n)
    prod = torch.mm(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()       # whole numbers below 2^53: exact
    for out_dtype, b in ((torch.float32, None), (torch.bfloat16, bias), (torch.float16, bias)):
        got = ops.int8_linear(x, xs, w, ws, bias=b, out_dtype=out_dtype)
        want = prod if b is None else prod + b.double()
        bound = prod.abs() * 4 * E + want.abs() * (U[out_dtype] + 2 * E) + TINY[out_dtype]
        if out_dtype == torch.float16:               # sums of long rows leave the type
            inside = want.abs() < 65000
            got, want, bound = got[inside], want[inside], bound[inside]
        within(got, want, bound, f"{out_dtype}")


EIGHT_PAIR = [((256, 1), 904, 6299, 265), ((256, 1), 3001, 2049, 448), ((256, 1), 904, 6299, 513), ((256, 1), 3001, 2049, 1111),
              ((256, 2), 568, 3658, 5883), ((256, 3), 898, 2145, 4137), ((256, 6), 650, 1380, 10451), ((256, 12), 654, 726, 30571),
              ((256, 32), 1559, 77, 87320), ((256, 32), 1618, 66, 87368), ((256, 24), 137, 1091, 70828),
              ((128, 1), 547, 533, 1027), ((128, 2), 930, 663, 3481), ((128, 3), 2114, 67, 2049), ((128, 5), 543, 34, 1589),
              ((128, 16), 534, 40, 3859), ((128, 48), 520, 51, 30341)]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("cut,m,n,k", EIGHT_PAIR)
def test_int8_gated_linear_cuts(dev, act, cut, m, n, k):
    assert ops.product_cut(m, n, row_bytes(k, 1), gated=True) == cut
    g = gen(dev, m * 3 + n + k)
    (x, xs), (w, ws), (v, vs) = eight(g, m, k), eight(g, n, k), eight(g, n, k)
    xs = xs * 5 * k ** -0.5
    gate = torch.mm(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()
    up = torch.mm(x.double(), v.double().t()) * xs.double()[:, None] * vs.double()
    want = act64(gate, act) * up
    bound = gated_bound(gate, up, gate.abs() * 4 * E, up.abs() * 4 * E, act)
    for out_dtype in DTYPES:
        got = ops.int8_gated_linear(x, xs, w, ws, v, vs, activation=act, out_dtype=out_dtype)
        within(got, want, bound * (1 + 2 ** -7) + want.abs() * U[out_dtype] + TINY[out_dtype], f"{out_dtype}")


# ------------------------------------------------------------------------------- gated projections, forward
PAIR_16 = [((256, 1), 904, 6299, 132), ((256, 1), 3001, 2049, 192), ((256, 1), 904, 6299, 223), ((256, 1), 3001, 2049, 256), ((256, 1), 3001, 2049, 300),
           ((256, 2), 568, 3658, 2941), ((256, 3), 898, 2145, 2068), ((256, 5), 641, 1812, 5990), ((256, 8), 902, 779, 10600), ((256, 32), 1559, 77, 43660),
           ((128, 1), 547, 533, 400), ((128, 2), 930, 663, 1740), ((128, 3), 2114, 67, 1030), ((128, 4), 702, 131, 970), ((128, 6), 517, 36, 659),
           ((128, 32), 529, 34, 7962)]
PAIR_32 = [((256, 1), 904, 6299, 66), ((256, 1), 3001, 2049, 96), ((256, 1), 904, 6299, 111), ((256, 1), 3001, 2049, 128), ((256, 1), 3001, 2049, 150),
           ((256, 3), 682, 2794, 457), ((256, 5), 641, 1863, 1410), ((256, 10), 927, 657, 5397),
           ((128, 1), 547, 533, 60), ((128, 2), 3644, 140, 228), ((128, 3), 580, 33, 132), ((128, 8), 525, 36, 474), ((128, 48), 572, 36, 3068)]
PAIRS = [(dtype, *case) for dtype, cases in ((torch.bfloat16, PAIR_16), (torch.float16, PAIR_16), (torch.float32, PAIR_32)) for case in cases]


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype,cut,m,h,k", PAIRS)
def test_gated_linear_forward_cuts(dev, act, dtype, cut, m, h, k):
    assert ops.product_cut(m, h, row_bytes(k, SIZE[dtype]), gated=True, fp32=dtype == torch.float32) == cut
    rng = gen(dev, m + h * 3 + k)
    x, wg, wu = normal(rng, m, k, dtype=dtype, scale=2.0), normal(rng, h, k, dtype=dtype, scale=k ** -0.5), normal(rng, h, k, dtype=dtype, scale=k ** -0.5)
    out, saved = ops.gated_linear_fwd(x, wg, wu, activation=act, save=True)
    g, u, dg, du = gated_ref(x, wg, wu, act)
    within(saved[0], g, dg + g.abs() * E, "gate")
    within(saved[1], u, du + u.abs() * E, "up")
    want = act64(g, act) * u
    within(out, want, gated_bound(g, u, dg, du, act) * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype], "out")
    assert torch.equal(ops.gated_linear_fwd(x, wg, wu, activation=act)[0], out)


@pytest.mark.parametrize("dtype,cut,m,h,k", PAIRS)
def test_gated_linear_forward_cuts_in_whole_numbers(dev, dtype, cut, m, h, k):
    """Sums of whole numbers are exact in any order: the products have to be equal."""
    rng = gen(dev, m + h + k)
    x, wg, wu = (torch.randint(-2, 3, (n, k), generator=rng, device=dev).to(dtype) for n in (m, h, h))
    out, saved = ops.gated_linear_fwd(x, wg, wu, "relu", save=True)
    g, u = x.double() @ wg.double().t(), x.double() @ wu.double().t()
    assert torch.equal(saved[0].double(), g) and torch.equal(saved[1].double(), u)
    assert torch.equal(out, (g.clamp_min(0) * u).float().to(dtype))


# ------------------------------------------------------------------------------- gated projections, backward
# (dx's cut, dw's cut): m, h, k
BACK_16 = [((256, 1), (128, 6), 4704, 68, 2578), ((256, 1), (128, 3), 4704, 193, 2578), ((128, 4), (256, 1), 139, 1586, 4016),
           ((128, 4), (256, 1), 225, 1586, 4016), ((256, 2), (128, 2), 7178, 1441, 538), ((256, 3), (256, 1), 2049, 2049, 2050),
           ((256, 6), (128, 1), 1573, 2640, 1190), ((256, 12), (128, 1), 167, 8084, 4117), ((128, 1), (256, 6), 5424, 205, 4123)]
BACK_32 = [((256, 1), (128, 12), 4704, 33, 2578), ((256, 1), (128, 6), 4704, 97, 2578), ((128, 8), (256, 1), 65, 1586, 4016),
           ((128, 4), (256, 1), 129, 1586, 4016), ((256, 3), (128, 4), 2351, 232, 1691), ((256, 6), (128, 1), 1181, 1615, 2021),
           ((128, 3), (256, 3), 458, 783, 2469), ((128, 1), (256, 8), 6893, 197, 3354), ((256, 16), (128, 1), 192, 8094, 3501)]
BACKS = [(dtype, *case) for dtype, cases in ((torch.bfloat16, BACK_16), (torch.float16, BACK_16), (torch.float32, BACK_32)) for case in cases]


def backward_cuts(m, h, k, size):
    wide = -(-h // (64 // size)) * (64 // size)
    return tuple(ops.product_cut(*sizes, fp32=size == 4, few_rows=False) for sizes in ((m, k, 2 * wide * size), (wide + h, k, m * size)))


@pytest.mark.parametrize("dtype,dx_cut,dw_cut,m,h,k", BACKS)
def test_gated_linear_backward_cuts(dev, dtype, dx_cut, dw_cut, m, h, k):
    assert backward_cuts(m, h, k, SIZE[dtype]) == (dx_cut, dw_cut)
    rng, act = gen(dev, m + h * 5 + k), "silu"
    x, wg, wu = normal(rng, m, k, dtype=dtype), normal(rng, h, k, dtype=dtype, scale=k ** -0.5), normal(rng, h, k, dtype=dtype, scale=k ** -0.5)
    dh = normal(rng, m, h, dtype=dtype)
    _, saved = ops.gated_linear_fwd(x, wg, wu, activation=act, save=True)
    dx, dwg, dwu = ops.gated_linear_bwd(dh, x, wg, wu, saved, activation=act)
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


@pytest.mark.parametrize("dtype,dx_cut,dw_cut,m,h,k", BACKS)
def test_gated_linear_backward_cuts_in_whole_numbers(dev, dtype, dx_cut, dw_cut, m, h, k):
    """ReLU, whole saved products and gradients of -1, 0, 1: dg and du are exact in every type, and so are the sums."""
    rng = gen(dev, m + h + k)

    def whole(*shape, most=1):
        return torch.randint(-most, most + 1, shape, generator=rng, device=dev)
    x, wg, wu, dh = (whole(*s).to(dtype) for s in ((m, k), (h, k), (h, k), (m, h)))
    saved = whole(2, m, h, most=7).float()
    dx, dwg, dwu = ops.gated_linear_bwd(dh, x, wg, wu, saved, "relu")
    g, u, d = saved[0].double(), saved[1].double(), dh.double()
    dg, du = d * u * (g > 0), d * g.clamp_min(0)
    for got, want in ((dx, dg @ wg.double() + du @ wu.double()), (dwg, dg.t() @ x.double()), (dwu, du.t() @ x.double())):
        assert float(want.abs().max()) < 2 ** 24 and torch.equal(got, want.float().to(dtype))


def test_the_cases_reach_what_they_are_for():
    """Slices in every number up to 64, last slices of one run to more than four, each form with both tiles."""
    slices = {cut for cut, *_ in EIGHT}
    assert {s for t, s in slices if t == 128} >= {1, 2, 3, 4, 5, 6, 8, 12, 24, 32, 48, 64}
    assert {s for t, s in slices if t == 256} >= {1, 2, 3, 4, 6, 10, 16, 24, 32}
    for tile in (128, 256):
        assert {in_a_last_slice(row_bytes(k, 1), cut[1]) for cut, m, n, k in EIGHT if cut[0] == tile and cut[1] > 1} >= {1, 2, 3, 4, 5, 7}
    assert {-(-k // 64) for cut, m, n, k in EIGHT if cut == (256, 1)} >= {5, 6, 7, 8, 9, 12, 29}
    for cases in (EIGHT, EIGHT_PAIR, PAIR_16, PAIR_32):
        assert {(c[0][0], c[0][1] > 1) for c in cases} == {(256, False), (256, True), (128, False), (128, True)}
    for cases in (BACK_16, BACK_32):
        for i in (0, 1):
            assert {(c[i][0], c[i][1] > 1) for c in cases} >= {(256, False), (256, True), (128, False)}


# ------------------------------------------------------------------------------- few rows
# pairs: 8 columns a block (short rows and rows of 4 KB), 16 columns; up to 32 rows in blocks of 16 and of 32 columns; 64 rows a block
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h,kb", [(1, 1003, 1040), (4, 1003, 4112), (16, 1003, 8192), (16, 4090, 4128), (9, 4090, 512), (17, 515, 4096),
                                    (32, 4099, 2064), (25, 4099, 3104), (40, 333, 1040), (130, 77, 528)])
def test_few_aligned_rows(dev, dtype, m, h, kb):
    k, fp32 = kb // SIZE[dtype], dtype == torch.float32
    assert ops.product_cut(m, h, kb, gated=True, fp32=fp32)[0] == 0 and kb % 16 == 0
    rng = gen(dev, m + h + kb)
    x, wg, wu = normal(rng, m, k, dtype=dtype, scale=2.0), normal(rng, h, k, dtype=dtype, scale=k ** -0.5), normal(rng, h, k, dtype=dtype, scale=k ** -0.5)
    out, saved = ops.gated_linear_fwd(x, wg, wu, save=True)
    g, u, dg, du = gated_ref(x, wg, wu, "silu")
    within(saved[0], g, dg + g.abs() * E, "gate")
    within(saved[1], u, du + u.abs() * E, "up")
    want = act64(g, "silu") * u
    within(out, want, gated_bound(g, u, dg, du, "silu") * (1 + 2 ** -7) + want.abs() * U[dtype] + TINY[dtype], "out")


@pytest.mark.parametrize("m,n,k", [(1, 1003, 1040), (8, 1003, 8208), (8, 4090, 4096), (9, 1003, 4112), (16, 4090, 528), (17, 515, 4096), (32, 4099, 2064),
                                   (25, 4099, 3104), (40, 333, 1040), (130, 77, 528)])
def test_few_aligned_8_bit_rows(dev, m, n, k):
    assert ops.product_cut(m, n, k)[0] == ops.product_cut(m, n, k, gated=True)[0] == 0 and k % 16 == 0
    g = gen(dev, m + n + k)
    (x, xs), (w, ws), (v, vs), bias = eight(g, m, k), eight(g, n, k), eight(g, n, k), normal(g, n)
    prod = torch.mm(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()
    want = prod + bias.double()
    within(ops.int8_linear(x, xs, w, ws, bias=bias), want, prod.abs() * 4 * E + want.abs() * 3 * E, "product")
    xs = xs * 5 * k ** -0.5
    gate = torch.mm(x.double(), w.double().t()) * xs.double()[:, None] * ws.double()
    up = torch.mm(x.double(), v.double().t()) * xs.double()[:, None] * vs.double()
    want = act64(gate, "silu") * up
    within(ops.int8_gated_linear(x, xs, w, ws, v, vs), want, gated_bound(gate, up, gate.abs() * 4 * E, up.abs() * 4 * E, "silu") + want.abs() * E, "pair")


# ------------------------------------------------------------------------------- norm of many rows
# from 2048 rows on a wave takes a row of up to 256 vectors of 16 bytes, 1 to 4 a lane; longer ones a block, 2 or 4 a thread
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vectors", [(2048, 63.3), (2049, 65), (2050, 127.9), (2051, 130.2), (2100, 191), (2053, 193.1), (2051, 255.9), (2049, 257.2),
                                          (2048, 1500.4), (2050, 2049.3), (2048, 4095.9)])
def test_rms_norm_of_many_rows(dev, dtype, rows, vectors):
    dim = round(vectors * (16 // SIZE[dtype]))
    g = gen(dev, rows + dim)
    x, r, w = normal(g, rows, dim, dtype=dtype, scale=3.0), normal(g, rows, dim, dtype=dtype), normal(g, dim, dtype=dtype)
    for res in (None, r):
        y, total = ops.rms_norm_fwd(x, w, residual=res)
        s, rstd, want = norm_ref(x, w, res, 1e-6)
        if res is not None:
            within(total, s, s.abs() * (U[dtype] + E) + TINY[dtype], "sum")
        within(y, want, want.abs() * (U[dtype] + STAT) * (1 + 2 ** -7) + TINY[dtype], "y")
        q, scale, total8 = ops.rms_norm_int8(x, w, residual=res)
        assert torch.equal(total8, total)
        want = want.abs().amax(1) / 127
        within(scale, want, want * (STAT + 4 * E), "scale")
        v = s * w.double()
        v = v / v.abs().amax(1, keepdim=True) * 127
        within(q, v, 0.5 + 127 * 8 * E, "q")
        assert bool((q.abs().amax(1) == 127).all())
        del s, rstd, want, v
    q, scale = ops.quantize_rows(x)
    top = x.double().abs().amax(1)
    within(scale, top / 127, top / 127 * 2 * E, "quantize_rows scale")
    within(q, x.double() / top[:, None] * 127, 0.5 + 127 * 8 * E, "quantize_rows q")
