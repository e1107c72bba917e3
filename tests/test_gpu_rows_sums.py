"""The row operators' sums on data whose sums are exact, so that a value lost, taken
twice or put into another row shows at any number of rows.

Exact data: values of 1 and 2, weights of 1/2, 1 and 2, mean 0 and rstd 1.  Every
product and every sum below 2^24 is then exact in f32 in whatever order it is
taken.  The two row means are correctly rounded quotients, so dx = g - m1 - h m2
is off by the roundings of m1, m2, the difference, the product's fma and a factor
rstd: 2^-24 of each, and 2^-24 of the result once more for dz or the scale."""
import pytest
import torch

from tests.test_gpu_rows import DTYPES, F16, F32, LARGE, UNIT, WIDTHS
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
