"""The row operators' sums on data whose sums are exact, so that a value lost, taken
twice or put into another row shows at any number of rows, and on random f32 data
within bounds that follow from the additions.

Exact data: values of 1 and 2, weights of 1/2, 1 and 2, mean 0 and rstd 1.  Every
product and every sum below 2^24 is then exact in f32 in whatever order it is
taken.  The two row means are correctly rounded quotients, so dx = g - m1 - h m2
is off by the roundings of m1, m2, the difference, the product's fma and a factor
rstd: 2^-24 of each, and 2^-24 of the result once more for dz or the scale."""
import pytest
import torch

from tests.test_gpu_rows import DTYPES, EPS, F16, F32, LARGE, UNIT, WIDTHS, rows_of, weights_of
from vauss_b200 import ops

pytestmark = pytest.mark.gpu

E = 2.0**-24
# small calls on the direct kernels, large ones on the streaming ones, rows that no kernel holds
SMALL = [(1, 1), (1, 5003), (37, 3), (300, 59), (500, 64), (2_000, 96), (20_000, 64), (40_001, 12), (19, 520), (7, 1030),
         (150, 4096), (1_000, 1031)]
LONG = [(67, 16_001), (70, 20_000), (43, 33_333), (2, 140_003)]
SHAPES = SMALL + LARGE + [(3_000_001 // c, c) for c in WIDTHS + [1, 900, 924, 956]] + LONG


def small_integers(cuda, rows, cols, dtype, seed, layout="plain"):
    gen = torch.Generator(device=cuda).manual_seed(seed)
    v = torch.randint(1, 3, (rows, cols), device=cuda, generator=gen)
    if layout == "strided":
        t = torch.full((rows, cols + 5), float("nan"), dtype=dtype, device=cuda)[:, 3:3 + cols]
    else:
        t = torch.empty(rows, cols, dtype=dtype, device=cuda)
    return t.copy_(v)


def within(got, want, bound, what):
    """got within `bound` and half a unit of its type of want (f64, all on the device)."""
    half = 0.5 * UNIT[got.dtype] * want.abs() if got.dtype != F32 else 0.0
    err = (got.double() - want).abs()
    assert bool((err <= bound + half + (2.0**-25 if got.dtype == F16 else 0.0)).all()), \
        f"{what}: off by {float((err - bound - half).max()):.3g} over its bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_backward_of_exact_sums(cuda, dtype, rows, cols):
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    w = torch.exp2(torch.randint(-1, 2, (cols,), device=cuda, generator=gen).float())
    mean, rstd = torch.zeros(rows, device=cuda), torch.ones(rows, device=cuda)
    for layout in ("plain", "strided"):
        z = small_integers(cuda, rows, cols, dtype, 1, layout)
        dy = small_integers(cuda, rows, cols, dtype, 2, layout)
        dz = small_integers(cuda, rows, cols, dtype, 3, layout)
        h, d = z.double(), dy.double()
        dw, db = (d * h).sum(0), d.sum(0)
        assert float(dw.max()) < 2**24
        g = d * w.double()
        m1, m2 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
        t = g - m1 - h * m2
        bound = E * (m1 + h * m2 + (g - m1).abs() + 2 * t.abs())
        o = ops.layer_norm_bwd(dy, z, w, mean, rstd)
        assert torch.equal(o.dweight.double(), dw) and torch.equal(o.dbias.double(), db), layout
        within(o.dx, t, bound, f"dx {layout}")
        for with_dz in (True, False):
            j = ops.dropout_add_norm_bwd(dy, dz if with_dz else None, z, w, mean, rstd, 0.25, 3, 5)
            assert torch.equal(j.dweight.double(), dw) and torch.equal(j.dbias.double(), db), f"joined {layout}"
            r = t + dz.double() if with_dz else t
            wide = bound + E * r.abs()
            within(j.dresidual, r, wide, f"dresidual {layout}")
            factor = ops.dropout(torch.ones(rows, cols, device=cuda), 0.25, 3, 5).double()
            # the factor's own rounding (4/3 is not f32's) and the product's
            within(j.dx, r * factor, (wide + 2 * E * r.abs()) * 4 / 3, f"joined dx {layout}")


@pytest.mark.parametrize("rows,cols", [(r, c) for r, c in SHAPES if c <= 4096 and r <= 70_000])
def test_f32_rounding(cuda, rows, cols):
    """f32 results within what their additions cost.  A row's sum of at most 4096 columns is at most 40 additions deep
    (32 values of a thread as 16 pairs, a warp's 5, its CTA's at most 8 + 2, and the ends), so it is off by at most
    40 E of the sum of magnitudes; a product or a difference by E of itself; rsqrt by 4 E.  dweight adds chains of at
    most 1024 rows: with partial sums of random sign the error is about E sqrt(L / 6) of the root of the sum of
    squares (L the chain), of which six are allowed, and 2 E for each term."""
    x, _ = rows_of(cuda, rows, cols, F32, rows + cols)
    w, b, _, _ = weights_of(cuda, cols, F32, cols)
    x64, w64, b64 = x.double(), w.double(), b.double()
    m64 = x64.mean(1, keepdim=True)
    c64 = x64 - m64
    v64 = (c64 * c64).mean(1, keepdim=True) + EPS
    q64 = v64.rsqrt()
    o = ops.layer_norm(x, w, b, EPS)
    dm = 41 * E * x64.abs().mean(1, keepdim=True)  # of the mean
    within(o.mean, m64[:, 0], dm[:, 0], "mean")
    # variance: the squares of x - m (each off by E, the mean's error adds its square and cancels in the sum to first
    # order), their sum, the quotient and eps; rstd half of that
    dq = (0.5 * (44 * E + dm * dm / v64) + 4 * E) * q64
    within(o.rstd, q64[:, 0], dq[:, 0], "rstd")
    y64 = c64 * q64 * w64 + b64
    within(o.y, y64, (w64 * q64).abs() * (dm + E * c64.abs()) + (c64 * w64).abs() * (dq + E * q64) + E * y64.abs(), "y")
    dy, _ = rows_of(cuda, rows, cols, F32, rows + cols + 1)
    g = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd)
    d64, m, q = dy.double(), o.mean.double()[:, None], o.rstd.double()[:, None]
    h = (x64 - m) * q
    e = d64 * w64
    m1, m2 = e.mean(1, keepdim=True), (e * h).mean(1, keepdim=True)
    t = q * (e - m1 - h * m2)
    d1, d2 = 42 * E * e.abs().mean(1, keepdim=True), 45 * E * (e * h).abs().mean(1, keepdim=True)
    within(g.dx, t, q * (d1 + h.abs() * d2 + E * (2 * e.abs() + m1.abs() + 4 * (h * m2).abs())) + 2 * E * t.abs(), "dx")
    share = E * (2 + 6 * (min(rows, 1024) / 6) ** 0.5)
    within(g.dweight, (d64 * h).sum(0), share * (d64 * h).square().sum(0).sqrt() + 40 * E * (d64 * h).sum(0).abs() +
           2 * E * (d64 * h).abs().max(), "dweight")


# 16-bit rows that a warp holds with 22 to 30 values a lane where there are many of them
MANY = [(14_300, c) for c in (487, 601, 703, 644, 700, 892, 706, 750, 822, 902, 958)] + \
    [(28_500, c) for c in (900, 924, 956)]
# rows on a CTA with 16 and 32 values a thread, whole vectors and ragged
ON_A_CTA = [(700, c) for c in (1536, 1538, 1543, 1544, 1601, 2040, 2047, 2048, 3500, 6001, 8192, 11_501, 12_288, 16_000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES + MANY + ON_A_CTA)
def test_forward_of_exact_sums(cuda, dtype, rows, cols):
    """The mean is the correctly rounded quotient of an exact sum, z of values without a mask exact.  For y and rstd:
    the squares' sum of like signs is at most 100 additions deep (a thread's share of 140003 columns and the CTA's),
    rsqrt is within 4 E, and y takes the mean's rounding, a difference, two products and a sum."""
    gen = torch.Generator(device=cuda).manual_seed(rows + cols)
    w = torch.exp2(torch.randint(-1, 2, (cols,), device=cuda, generator=gen).float())
    b = torch.randint(-1, 2, (cols,), device=cuda, generator=gen).float()
    for layout in ("plain", "strided"):
        x = small_integers(cuda, rows, cols, dtype, 1, layout)
        r = small_integers(cuda, rows, cols, dtype, 2, layout)
        for joined in (False, True):
            if joined:
                o = ops.dropout_add_norm(x, r, w, b, 0.0, 1, 2)
                assert torch.equal(o.z, x + r), layout
                z = x.double() + r.double()
            else:
                o, z = ops.layer_norm(x, w, b), x.double()
            mean = (z.sum(1) / cols).float()  # in f64: torch divides by a number as a product with its inverse
            assert torch.equal(o.mean, mean), f"mean {layout}"
            d = z - mean.double()[:, None]
            v = (d * d).mean(1, keepdim=True) + EPS
            q = v.rsqrt()
            dq = (0.5 * 104 * E + 4 * E) * q
            within(o.rstd, q[:, 0], dq[:, 0], f"rstd {layout}")
            y = d * q * w.double() + b.double()
            within(o.y, y, d.abs() * w.double() * (dq + 3 * E * q) + E * y.abs(), f"y {layout}")
        o = ops.dropout_add_norm(x, r, w, b, 0.25, 1, 2)
        factor = ops.dropout(torch.ones(rows, cols, device=cuda), 0.25, 1, 2).double()
        z = r.double() + x.double() * factor
        within(o.z, z, 3 * E * z.abs(), f"masked z {layout}")
        z = o.z.double()
        mean = z.mean(1, keepdim=True)
        q = ((z - mean).square().mean(1, keepdim=True) + EPS).rsqrt()
        dm, dq = 101 * E * mean, (0.5 * 104 * E + 4 * E) * q + 0.5 * q**3 * (101 * E * mean)**2
        within(o.mean, mean[:, 0], dm[:, 0], f"masked mean {layout}")
        y = (z - mean) * q * w.double() + b.double()
        within(o.y, y, w.double() * (q * dm + (z - mean).abs() * (dq + 3 * E * q)) + E * y.abs(), f"masked y {layout}")


@pytest.mark.parametrize("rows,cols,layout", [(100_000_000, 1, "plain"), (60_000_000, 2, "plain"), (100_000_000, 1, "strided"),
                                              (200_000, 1030, "plain"), (30_000, 12_300, "plain")])
def test_sums_of_many_alike_rows(cuda, rows, cols, layout):
    """The gradient of a mean: every term of dbias and dweight is the same, so that the roundings of a chain of sums all
    go one way.  No chain is longer than 256 terms: of a tile's sums (48 terms each) or of rows, then the lanes' (32),
    the warps' (16) and a share of the CTAs' (100 here); a chain of n alike terms is off by at most (n + 1) / 2 roundings
    of E: 230 E in all."""
    dy = torch.full((rows, cols), 0.7123, device=cuda)
    if layout == "strided":
        dy = torch.full((rows, cols + 1), 0.7123, device=cuda)[:, 1:]
    z = torch.ones(rows, cols, device=cuda)
    mean, rstd = torch.zeros(rows, device=cuda), torch.ones(rows, device=cuda)
    want = float(dy[0, 0].double()) * rows
    g = ops.layer_norm_bwd(dy, z, torch.ones(cols, device=cuda), mean, rstd)
    for got in (g.dweight, g.dbias):
        assert float((got.double() / want - 1).abs().max()) <= 230 * E
