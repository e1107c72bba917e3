"""The row operators (dropout, layer norm and the two joined) against their
formulas in 64 bits, at the sizes, strides and masks where they can go wrong.

Tolerances, for inputs of order one.  Every kernel computes in f32 and rounds
each output once, so an output of type T is within half a unit of T's last
place (u/2, u = 2^-10 for f16, 2^-7 for bf16: the spacing relative to the
value) plus the f32 error.  A sum of n terms taken in order is off by at most
n 2^-24 of the sum of magnitudes; the kernels' sums are trees or strips whose
depth is far below 256, so 256 * 2^-24 = 1.6e-5 of the tensor's largest
magnitude bounds every f32 error here, doubled for the products around it."""
import ctypes

import numpy as np
import pytest
import torch

from vauss_b200 import _native, ops

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNIT = {F32: 2.0**-23, F16: 2.0**-10, BF16: 2.0**-7}
F32_ERR = 2 * 256 * 2.0**-24
EPS = 1e-5


def keep_mask(n, p, seed, offset):
    return keep_mask_at(0, n, p, seed, offset)


def keep_mask_at(first, n, p, seed, offset):
    """The definition in the header for indices [first, first + n), first a multiple of 8, in numpy's uint64."""
    t = 65536 if p == 1 else min(65535, int(p * 65536 + 0.5))
    g = np.arange(first // 8, first // 8 + (n + 7) // 8, dtype=np.uint64)
    m32 = np.uint64(0xFFFFFFFF)
    s32 = np.uint64(32)
    c = [g & m32, g >> s32, np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k[0]), b & m32, (a >> s32) ^ c[3] ^ np.uint64(k[1]), a & m32]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    lanes = np.stack([(w >> np.uint64(h)) & np.uint64(0xFFFF) for w in c for h in (0, 16)], 1).reshape(-1)[:n]
    return torch.from_numpy((lanes >= t).astype(np.bool_)), 65536.0 / (65536 - t) if t < 65536 else 0.0


def dropout_ref(x, p, seed, offset):
    keep, scale = keep_mask(x.numel(), p, seed, offset)
    return torch.where(keep.view(x.shape), x * scale, torch.zeros((), dtype=x.dtype))


def norm_ref(z, w, b, eps=EPS):
    mean = z.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((z - mean) ** 2).mean(-1, keepdim=True) + eps)
    return (z - mean) * rstd * w + b, mean, rstd


def norm_bwd_ref(dy, z, w, mean, rstd):
    h = (z - mean) * rstd
    g = dy * w
    t = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return t, (dy * h).sum(0), dy.sum(0)


def close(got, want, what, terms=1.0):
    """got within half a unit of its type and the f32 error (`terms` times the tensor's scale) of want (f64)."""
    assert got.shape == want.shape, f"{what}: {got.shape} {want.shape}"
    if got.numel() == 0:
        return
    g = got.detach().cpu().double()
    bound = 0.5 * UNIT[got.dtype] * want.abs() + F32_ERR * terms * max(float(want.abs().max()), 1e-30)
    if got.dtype == F16:
        bound = bound + 2.0**-25  # half the subnormal spacing
    err = (g - want).abs()
    assert bool(torch.isfinite(g).all()), f"{what}: not finite"
    assert bool((err <= bound).all()), f"{what}: off by {float((err - bound).max()):.3g} over its bound"


def rows_of(cuda, rows, cols, dtype, seed, layout="plain"):
    """A matrix on the device and its values in f64.  "strided": columns of a wider buffer; "shifted": contiguous,
    one element past an aligned base."""
    gen = torch.Generator().manual_seed(seed)
    v = torch.randn(rows, cols, generator=gen) * 0.8 + 0.3
    if layout == "strided":
        wide = torch.full((rows, cols + 5), float("nan"), dtype=dtype, device=cuda)
        t = wide[:, 3:3 + cols]
    elif layout == "shifted":
        t = torch.full((rows * cols + 1,), float("nan"), dtype=dtype, device=cuda)[1:].view(rows, cols)
    else:
        t = torch.empty(rows, cols, dtype=dtype, device=cuda)
    t.copy_(v)
    return t, t.cpu().double()


def weights_of(cuda, cols, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    w = (torch.randn(cols, generator=gen) * 0.2 + 1).to(cuda, dtype)
    b = (torch.randn(cols, generator=gen) * 0.2).to(cuda, dtype)
    return w, b, w.cpu().double(), b.cpu().double()


SHAPES = [(1, 1), (5, 1), (1, 8), (3, 7), (300, 2), (257, 16), (1000, 48), (513, 59), (64, 64), (37, 100), (129, 128),
          (33, 255), (19, 520), (7, 1030), (41, 1024), (5, 2049), (150, 4096), (1, 4096), (3, 5003), (2, 16384),
          (2, 16385), (1, 40001), (2100, 24), (40_001, 12)]
DTYPES = [F32, F16, BF16]


def test_generator_known_answers():
    """The published test vector of Philox 4x32-10 (counter and key all zeros) pins this file's reference."""
    words = (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)
    for t in range(0, 65536, 1024):
        got, _ = keep_mask(8, t / 65536, 0, 0)
        assert got.tolist() == [((w >> h) & 0xFFFF) >= t for w in words for h in (0, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count", [0, 1, 7, 8, 9, 255, 4096, 100_003])
def test_dropout(cuda, dtype, count):
    x, x64 = rows_of(cuda, 1, count, dtype, count + 1)
    x, x64 = x.view(-1), x64.view(-1)
    for p, seed, offset in ((0.0, 1, 0), (0.1, 12345678901234567, 3), (0.5, 2**64 - 1, 2**64 - 1), (0.9, 0, 2**40), (1.0, 5, 5)):
        want = dropout_ref(x64, p, seed, offset)
        close(ops.dropout(x, p, seed, offset), want, f"p {p}")
        close(ops.dropout_bwd(x, p, seed, offset), want, f"gradient, p {p}")
    y = x.clone()
    assert ops.dropout(y, 0.3, 9, 9, out=y) is y  # in place
    close(y, dropout_ref(x64, 0.3, 9, 9), "in place")


def test_dropout_is_a_mask_of_the_index(cuda):
    """The mask does not depend on the type, the alignment or the values, and differs by seed and offset."""
    n = 50_001
    masks = []
    for dtype in DTYPES:
        for shift in (0, 1, 3):
            base = torch.ones(n + shift, dtype=dtype, device=cuda)
            masks.append((ops.dropout(base[shift:], 0.4, 77, 8) != 0).cpu())
    assert all(torch.equal(masks[0], m) for m in masks[1:])
    kept = float(masks[0].double().mean())
    assert abs(kept - 0.6) < 5 * (0.24 / n) ** 0.5
    other = [(ops.dropout(torch.ones(n, device=cuda), 0.4, s, o) != 0).cpu() for s, o in ((78, 8), (77, 9))]
    for m in other:  # independent masks agree in 0.6^2 + 0.4^2 of the places
        assert abs(float((m == masks[0]).double().mean()) - 0.52) < 5 * (0.25 / n) ** 0.5


def test_dropout_drops_nan_and_infinities(cuda):
    n = 4096
    keep, _ = keep_mask(n, 0.5, 3, 4)
    for dtype in DTYPES:
        x = torch.ones(n, dtype=dtype, device=cuda)
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")]).repeat(n // 3 + 1)[:n]
        x[~keep.to(cuda)] = bad.to(cuda, dtype)[~keep.to(cuda)]
        y = ops.dropout(x, 0.5, 3, 4)
        assert torch.equal(y.cpu().double(), torch.where(keep, 2.0, 0.0).double())
        r = torch.zeros(8, n // 8, dtype=dtype, device=cuda)
        out = ops.dropout_add_norm(x.view(8, -1), r, None, None, 0.5, 3, 4)
        assert torch.equal(out.z.view(-1), y) and bool(torch.isfinite(out.y).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(cuda, dtype, rows, cols):
    for layout, wdtype in (("plain", F32), ("plain", dtype), ("strided", F32), ("shifted", F32)):
        x, x64 = rows_of(cuda, rows, cols, dtype, rows + cols, layout)
        w, b, w64, b64 = weights_of(cuda, cols, wdtype, cols)
        y64, m64, q64 = norm_ref(x64, w64, b64)
        o = ops.layer_norm(x, w, b, EPS)
        # rstd of a two-value row magnifies the mean's rounding by its own size
        close(o.y, y64, f"y {layout}", terms=max(1.0, float(q64.max())))
        close(o.mean, m64[:, 0], f"mean {layout}")
        close(o.rstd, q64[:, 0], f"rstd {layout}", terms=max(1.0, float(q64.max())))
    o2 = ops.layer_norm(x, w, b, EPS)
    assert torch.equal(o.y, o2.y) and torch.equal(o.mean, o2.mean)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm_bwd(cuda, dtype, rows, cols):
    for layout, wdtype in (("plain", F32), ("plain", dtype), ("strided", F32), ("shifted", F32)):
        x, x64 = rows_of(cuda, rows, cols, dtype, rows + cols, layout)
        dy, dy64 = rows_of(cuda, rows, cols, dtype, rows + cols + 1, layout)
        w, _, w64, _ = weights_of(cuda, cols, wdtype, cols)
        o = ops.layer_norm(x, w, None, EPS)
        m, q = o.mean.cpu().double()[:, None], o.rstd.cpu().double()[:, None]
        dx64, dw64, db64 = norm_bwd_ref(dy64, x64, w64, m, q)
        g = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd)
        # dx of a nearly constant row is a difference of terms of size rstd
        scale = float(q.max() * dy64.abs().max() * w64.abs().max()) / max(float(dx64.abs().max()), 1e-30)
        close(g.dx, dx64, f"dx {layout}", terms=max(1.0, scale))
        h = ((x64 - m) * q).abs()
        close(g.dweight, dw64, f"dweight {layout}",
              terms=max(1.0, float((dy64.abs() * h).sum(0).max()) / max(float(dw64.abs().max()), 1e-30)))
        close(g.dbias, db64, f"dbias {layout}",
              terms=max(1.0, float(dy64.abs().sum(0).max()) / max(float(db64.abs().max()), 1e-30)))
        assert g.dweight.dtype == wdtype
        again = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd)
        assert all(torch.equal(u, v) for u, v in ((g.dx, again.dx), (g.dweight, again.dweight), (g.dbias, again.dbias)))
        if layout == "plain":  # in place
            want = g.dx.clone()
            h = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd, out=ops.LayerNormGrads(dy, g.dweight, g.dbias))
            assert torch.equal(h.dx, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_dropout_add_norm(cuda, dtype, rows, cols):
    for layout, p in (("plain", 0.25), ("plain", 0.0), ("plain", 1.0), ("strided", 0.25), ("shifted", 0.25)):
        x, x64 = rows_of(cuda, rows, cols, dtype, rows + cols, layout)
        r, r64 = rows_of(cuda, rows, cols, dtype, rows + cols + 1, layout)
        w, b, w64, b64 = weights_of(cuda, cols, F32, cols)
        o = ops.dropout_add_norm(x, r, w, b, p, 99, 7, EPS)
        z64 = r64 + dropout_ref(x64, p, 99, 7)
        close(o.z, z64, f"z {layout}")
        y64, m64, q64 = norm_ref(o.z.cpu().double(), w64, b64)
        close(o.y, y64, f"y {layout}", terms=max(1.0, float(q64.max())))
        close(o.mean, m64[:, 0], f"mean {layout}")
        close(o.rstd, q64[:, 0], f"rstd {layout}", terms=max(1.0, float(q64.max())))
        if layout == "plain":  # in place
            want = [t.clone() for t in (o.y, o.z, o.mean, o.rstd)]
            v = ops.dropout_add_norm(x, r, w, b, p, 99, 7, EPS, out=ops.DropoutAddNormOutput(x, r, o.mean, o.rstd))
            assert all(torch.equal(a, c) for a, c in zip(want, (v.y, v.z, v.mean, v.rstd)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_dropout_add_norm_bwd(cuda, dtype, rows, cols):
    for layout, p, with_dz in (("plain", 0.25, True), ("plain", 0.0, True), ("plain", 0.25, False), ("plain", 1.0, True),
                               ("strided", 0.25, True), ("shifted", 0.25, True)):
        z, z64 = rows_of(cuda, rows, cols, dtype, rows + cols, layout)
        dy, dy64 = rows_of(cuda, rows, cols, dtype, rows + cols + 1, layout)
        dz, dz64 = rows_of(cuda, rows, cols, dtype, rows + cols + 2, layout)
        w, _, w64, _ = weights_of(cuda, cols, F32, cols)
        o = ops.layer_norm(z, w, None, EPS)
        m, q = o.mean.cpu().double()[:, None], o.rstd.cpu().double()[:, None]
        t64, dw64, db64 = norm_bwd_ref(dy64, z64, w64, m, q)
        scale = float(q.max() * dy64.abs().max() * w64.abs().max())
        t64 = t64 + (dz64 if with_dz else 0)
        g = ops.dropout_add_norm_bwd(dy, dz if with_dz else None, z, w, o.mean, o.rstd, p, 11, 2**33 + 5)
        terms = max(1.0, scale / max(float(t64.abs().max()), 1e-30))
        close(g.dresidual, t64, f"dresidual {layout}", terms=terms)
        dx64 = dropout_ref(t64, p, 11, 2**33 + 5)
        close(g.dx, dx64, f"dx {layout}",
              terms=max(1.0, 2 * scale / max(float(dx64.abs().max()), 1e-30)))
        ln = ops.layer_norm_bwd(dy, z, w, o.mean, o.rstd)
        assert torch.equal(ln.dweight, g.dweight) and torch.equal(ln.dbias, g.dbias)
        if layout == "plain" and with_dz:  # in place
            want = (g.dx.clone(), g.dresidual.clone())
            v = ops.dropout_add_norm_bwd(dy, dz, z, w, o.mean, o.rstd, p, 11, 2**33 + 5,
                                         out=ops.DropoutAddNormGrads(dy, dz, g.dweight, g.dbias))
            assert torch.equal(v.dx, want[0]) and torch.equal(v.dresidual, want[1])


# Calls large enough for the streaming backward kernels (over 16 MB of traffic) in every type, with tiles and rows
# that end inside 16-byte pieces.  The sums over the rows are strips of at most a few hundred rows each.
LARGE = [(250_001, 12), (900_000, 5), (60_001, 59), (50_003, 64), (30_001, 100), (10_001, 384), (7_001, 520),
         (3_701, 1030), (1_901, 2049), (1_001, 4096), (801, 5003), (331, 12_000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", LARGE)
def test_large_backward(cuda, dtype, rows, cols):
    z, z64 = rows_of(cuda, rows, cols, dtype, rows + cols)
    dy, dy64 = rows_of(cuda, rows, cols, dtype, rows + cols + 1)
    dz, dz64 = rows_of(cuda, rows, cols, dtype, rows + cols + 2)
    w, _, w64, _ = weights_of(cuda, cols, F32, cols)
    o = ops.layer_norm(z, w, None, EPS)
    y64, m64, q64 = norm_ref(z64, w64, 0.0)
    close(o.y, y64, "y", terms=max(1.0, float(q64.max())))
    m, q = o.mean.cpu().double()[:, None], o.rstd.cpu().double()[:, None]
    t64, dw64, db64 = norm_bwd_ref(dy64, z64, w64, m, q)
    scale = float(q.max() * dy64.abs().max() * w64.abs().max())
    g = ops.layer_norm_bwd(dy, z, w, o.mean, o.rstd)
    close(g.dx, t64, "dx", terms=max(1.0, scale / float(t64.abs().max())))
    h = ((z64 - m) * q).abs()
    close(g.dweight, dw64, "dweight", terms=max(1.0, float((dy64.abs() * h).sum(0).max()) / float(dw64.abs().max())))
    close(g.dbias, db64, "dbias", terms=max(1.0, float(dy64.abs().sum(0).max()) / float(db64.abs().max())))
    for d, d64 in ((dz, dz64), (None, 0.0)):
        j = ops.dropout_add_norm_bwd(dy, d, z, w, o.mean, o.rstd, 0.25, 11, 2**33 + 5)
        want = t64 + d64
        close(j.dresidual, want, "dresidual", terms=max(1.0, scale / float(want.abs().max())))
        dx64 = dropout_ref(want, 0.25, 11, 2**33 + 5)
        close(j.dx, dx64, "joined dx", terms=max(1.0, 2 * scale / float(dx64.abs().max())))
        assert torch.equal(j.dweight, g.dweight) and torch.equal(j.dbias, g.dbias)


# A width for each number of values that a lane holds, in runs of four, two and one.
WIDTHS = [2, 3, 6, 10, 17, 18, 20, 23, 28, 33, 36, 60, 76, 130, 170, 201, 250, 300, 401, 420, 602, 700, 703, 750, 822, 902]


@pytest.mark.parametrize("cols", WIDTHS)
def test_large_widths(cuda, cols):
    rows = 3_000_001 // cols
    test_large_backward(cuda, BF16, rows, cols)
    x, x64 = rows_of(cuda, rows, cols, BF16, cols + 3)
    r, r64 = rows_of(cuda, rows, cols, BF16, cols + 4)
    w, b, w64, b64 = weights_of(cuda, cols, F32, cols + 5)
    o = ops.dropout_add_norm(x, r, w, b, 0.25, 7, 9, EPS)
    z64 = r64 + dropout_ref(x64, 0.25, 7, 9)
    close(o.z, z64, "z")
    y64, _, q64 = norm_ref(o.z.cpu().double(), w64, b64)
    close(o.y, y64, "y", terms=max(1.0, float(q64.max())))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(67, 16_001), (70, 20_000), (43, 33_333), (2, 140_003)])
def test_longest_rows(cuda, dtype, rows, cols):
    """Rows that no kernel holds whole, from contiguous buffers and from columns of a wider one."""
    test_large_backward(cuda, dtype, rows, cols)
    x, x64 = rows_of(cuda, rows, cols, dtype, cols + 3)
    r, r64 = rows_of(cuda, rows, cols, dtype, cols + 4)
    w, b, w64, b64 = weights_of(cuda, cols, F32, cols + 5)
    o = ops.dropout_add_norm(x, r, w, b, 0.25, 7, 9, EPS)
    z64 = r64 + dropout_ref(x64, 0.25, 7, 9)
    close(o.z, z64, "z")
    y64, _, q64 = norm_ref(o.z.cpu().double(), w64, b64)
    close(o.y, y64, "y", terms=max(1.0, float(q64.max())))
    wide = torch.zeros(rows, cols + 3, dtype=dtype, device=cuda)
    wide[:, 1:1 + cols] = x
    v = ops.dropout_add_norm(wide[:, 1:1 + cols], r, w, b, 0.25, 7, 9, EPS)
    assert torch.equal(v.z, o.z)
    close(v.y, y64, "y of strided rows", terms=max(1.0, float(q64.max())))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(60_001, 59), (3_701, 1030), (1_001, 4096)])
def test_large_in_place_and_strided(cuda, dtype, rows, cols):
    """In place, and from columns of a wider buffer, the same bits as out of place from contiguous rows (the column
    sums of strided rows are taken by another kernel and only agree within rounding)."""
    z, _ = rows_of(cuda, rows, cols, dtype, 1)
    dy, _ = rows_of(cuda, rows, cols, dtype, 2)
    dz, _ = rows_of(cuda, rows, cols, dtype, 3)
    w, b, _, _ = weights_of(cuda, cols, F32, 4)
    o = ops.dropout_add_norm(dy, z, w, b, 0.25, 1, 2)
    g = ops.dropout_add_norm_bwd(dy, dz, z, w, o.mean, o.rstd, 0.25, 1, 2)
    wide = [torch.zeros(rows, cols + 3, dtype=dtype, device=cuda) for _ in range(3)]
    for k, t in zip(wide, (dy, dz, z)):
        k[:, 1:1 + cols] = t
    sdy, sdz, sz = (k[:, 1:1 + cols] for k in wide)
    s = ops.dropout_add_norm_bwd(sdy, sdz, sz, w, o.mean, o.rstd, 0.25, 1, 2)
    tol = 4 * UNIT[dtype] * float(g.dx.float().abs().max())
    assert float((s.dx.float() - g.dx.float()).abs().max()) <= tol
    assert float((s.dweight - g.dweight).abs().max()) <= F32_ERR * rows
    f = ops.dropout_add_norm(sdy, sz, w, b, 0.25, 1, 2)
    assert float((f.y.float() - o.y.float()).abs().max()) <= 4 * UNIT[dtype] * float(o.y.float().abs().max())
    assert torch.equal(f.z, o.z)
    v = ops.dropout_add_norm_bwd(dy, dz, z, w, o.mean, o.rstd, 0.25, 1, 2,
                                 out=ops.DropoutAddNormGrads(dy, dz, torch.empty_like(w), torch.empty_like(w)))
    assert torch.equal(v.dx, g.dx) and torch.equal(v.dresidual, g.dresidual) and torch.equal(v.dweight, g.dweight)


def test_no_weights_and_single_gradients(cuda):
    x, x64 = rows_of(cuda, 50, 72, F32, 1)
    dy, dy64 = rows_of(cuda, 50, 72, F32, 2)
    one = torch.ones(72, dtype=torch.float64)
    o = ops.layer_norm(x)
    y64, m64, q64 = norm_ref(x64, one, 0 * one)
    close(o.y, y64, "y")
    b = torch.full((72,), 0.5, device=cuda)
    close(ops.layer_norm(x, None, b).y, y64 + 0.5, "y with a bias alone")
    g = ops.layer_norm_bwd(dy, x, None, o.mean, o.rstd)
    dx64, _, db64 = norm_bwd_ref(dy64, x64, one, m64, q64)
    close(g.dx, dx64, "dx", terms=4.0)
    assert g.dweight is None and g.dbias is None
    g = ops.layer_norm_bwd(dy, x, None, o.mean, o.rstd, with_bias=True)
    assert g.dweight is None
    close(g.dbias, db64, "dbias", terms=8.0)
    w = torch.ones(72, device=cuda)
    assert ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd, with_bias=False).dbias is None


def test_gradients_against_differences(cuda):
    """The f32 gradients against central differences of a scalar sum of the outputs, formed in f64 from f32 calls.
    With a step of 2^-6 on values of order one the truncation error is of order step^2 = 2.4e-4 of the third
    derivative and the outputs' rounding gives 2 * 2^-24 * sqrt(values) / (2 * 2^-6) = 1e-4: 5e-3 covers both."""
    rows, cols, p, h = 6, 40, 0.3, 2.0**-6
    x, _ = rows_of(cuda, rows, cols, F32, 1)
    r, _ = rows_of(cuda, rows, cols, F32, 2)
    cy, _ = rows_of(cuda, rows, cols, F32, 3)
    cz, _ = rows_of(cuda, rows, cols, F32, 4)
    w, b, _, _ = weights_of(cuda, cols, F32, 5)

    def value(x, r, w, b):
        o = ops.dropout_add_norm(x, r, w, b, p, 21, 22, EPS)
        return float((o.y.double() * cy.double()).sum() + (o.z.double() * cz.double()).sum())

    o = ops.dropout_add_norm(x, r, w, b, p, 21, 22, EPS)
    g = ops.dropout_add_norm_bwd(cy, cz, o.z, w, o.mean, o.rstd, p, 21, 22)
    gen = torch.Generator().manual_seed(6)
    for name, grad, at in (("x", g.dx, 0), ("residual", g.dresidual, 1), ("weight", g.dweight, 2), ("bias", g.dbias, 3)):
        args = [x, r, w, b]
        dirn = torch.randn(args[at].shape, generator=gen).to(cuda)
        dirn /= dirn.norm()
        plus, minus = list(args), list(args)
        plus[at], minus[at] = args[at] + h * dirn, args[at] - h * dirn
        diff = (value(*plus) - value(*minus)) / (2 * h)
        want = float((grad.double() * dirn.double()).sum())
        assert abs(diff - want) <= 5e-3 * max(1.0, float(grad.norm())), f"{name}: {diff} {want}"


def test_constant_rows(cuda):
    """A row without variance gives its bias and gradients of size 1 / sqrt(eps), nothing infinite."""
    for dtype in DTYPES:
        for cols in (1, 8, 59, 1024):
            x = torch.full((3, cols), 5.0, dtype=dtype, device=cuda)
            b = torch.full((cols,), 0.25, device=cuda)
            o = ops.layer_norm(x, None, b, EPS)
            assert torch.equal(o.y.float().cpu(), torch.full((3, cols), 0.25))
            assert torch.allclose(o.rstd.cpu(), torch.full((3,), EPS**-0.5), rtol=1e-6)
            g = ops.layer_norm_bwd(torch.ones_like(x), x, None, o.mean, o.rstd)
            assert torch.equal(g.dx.float().cpu(), torch.zeros(3, cols))


def test_large_offset_rows(cuda):
    """Two passes over the row: a level of 1000 times the spread costs no more than the rounding of its sum, at most
    32 additions deep (a variance from the mean of squares would be off by 6 %)."""
    x = (torch.randn(64, 768, generator=torch.Generator().manual_seed(1)) + 1000).to(cuda)
    x64 = x.cpu().double()
    y64, m64, q64 = norm_ref(x64, 1.0, 0.0)
    o = ops.layer_norm(x, eps=EPS)
    assert float((o.y.cpu().double() - y64).abs().max()) <= 32 * 1000 * 2.0**-24 * float(q64.max()) + 1e-5


def test_indices_past_32_bits(cuda):
    """The last values of buffers of over 2^32 values: the mask's index and the rows' addresses are 64-bit."""
    rows, cols = (1 << 21) + 5, 2048
    n = rows * cols
    x = torch.ones(rows, cols, dtype=F16, device=cuda)
    x[-3:] = torch.linspace(-1, 1, 3 * cols, device=cuda, dtype=F16).view(3, cols)
    first = n - 3 * cols
    # the words of the groups that hold the last three rows, from counters over 2^29
    keep, scale = keep_mask_at(first, 3 * cols, 0.5, 7, 9)
    want = torch.where(keep.view(3, cols), x[-3:].cpu().double() * scale, 0.0)
    y = ops.dropout(x, 0.5, 7, 9)
    close(y[-3:], want, "dropout")
    del y
    o = ops.dropout_add_norm(x, x, None, None, 0.5, 7, 9)
    close(o.z[-3:], want + x[-3:].cpu().double(), "z")
    y64, m64, q64 = norm_ref(o.z[-3:].cpu().double(), 1.0, 0.0)
    close(o.y[-3:], y64, "y")
    close(o.mean[-3:], m64[:, 0], "mean", terms=64.0)
    g = ops.layer_norm_bwd(o.y, o.z, None, o.mean, o.rstd)
    assert bool(torch.isfinite(g.dx[-3:]).all())
    t64, _, _ = norm_bwd_ref(o.y[-3:].cpu().double(), o.z[-3:].cpu().double(), 1.0, o.mean[-3:].cpu().double()[:, None],
                             o.rstd[-3:].cpu().double()[:, None])
    close(g.dx[-3:], t64, "dx", terms=max(1.0, float(q64.max() * y64.abs().max()) / float(t64.abs().max())))


def test_no_rows(cuda):
    x = torch.empty(0, 16, device=cuda)
    w = torch.ones(16, device=cuda)
    o = ops.layer_norm(x, w, w)
    assert o.y.shape == (0, 16) and o.mean.shape == (0,)
    g = ops.layer_norm_bwd(x, x, w, o.mean, o.rstd, out=ops.LayerNormGrads(x.clone(), w.clone(), w.clone()))
    assert torch.equal(g.dweight, torch.zeros_like(w)) and torch.equal(g.dbias, torch.zeros_like(w))
    j = ops.dropout_add_norm(x, x, w, w, 0.5, 1)
    assert ops.dropout_add_norm_bwd(x, x, j.z, w, j.mean, j.rstd, 0.5, 1).dx.shape == (0, 16)


def test_leading_dimensions(cuda):
    x, _ = rows_of(cuda, 24, 36, BF16, 1)
    w, b, _, _ = weights_of(cuda, 36, F32, 2)
    flat, deep = ops.layer_norm(x, w, b), ops.layer_norm(x.view(2, 3, 4, 36), w, b)
    assert deep.y.shape == (2, 3, 4, 36) and torch.equal(deep.y.view(24, 36), flat.y)


def test_on_another_stream(cuda):
    """Calls follow torch's current stream, and calls of two streams do not share a workspace."""
    x, _ = rows_of(cuda, 20_000, 96, F32, 1)
    dy, _ = rows_of(cuda, 20_000, 96, F32, 2)
    w, b, _, _ = weights_of(cuda, 96, F32, 3)
    o = ops.layer_norm(x, w, b)
    want = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd)
    want2 = ops.layer_norm_bwd(x, x, w, o.mean, o.rstd)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for k in range(8):
        with torch.cuda.stream(streams[k % 2]):
            got.append(ops.layer_norm_bwd(dy if k % 2 == 0 else x, x, w, o.mean, o.rstd))
    torch.cuda.synchronize()
    for k, g in enumerate(got):
        ref = want if k % 2 == 0 else want2
        assert torch.equal(g.dx, ref.dx) and torch.equal(g.dweight, ref.dweight) and torch.equal(g.dbias, ref.dbias)


def test_many_streams(cuda):
    """More streams than the ctx keeps buffers for, each with calls of growing size, all in flight at once."""
    dy, _ = rows_of(cuda, 3000, 40, BF16, 1)
    x, _ = rows_of(cuda, 3000, 40, BF16, 2)
    w, _, _, _ = weights_of(cuda, 40, F32, 3)
    o = ops.layer_norm(x, w)
    sizes = (5, 200, 1000, 3000)
    want = [ops.layer_norm_bwd(dy[:n], x[:n], w, o.mean[:n], o.rstd[:n]) for n in sizes]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(20)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append([ops.layer_norm_bwd(dy[:n], x[:n], w, o.mean[:n], o.rstd[:n]) for n in sizes])
    torch.cuda.synchronize()
    for per_stream in got:
        for g, ref in zip(per_stream, want):
            assert torch.equal(g.dweight, ref.dweight) and torch.equal(g.dbias, ref.dbias) and torch.equal(g.dx, ref.dx)


def test_statistics_at_any_address(cuda):
    """mean and rstd one element past a 16-byte boundary: another kernel, the same values within rounding."""
    rows, cols = 60_000, 64
    dy, _ = rows_of(cuda, rows, cols, F32, 1)
    x, _ = rows_of(cuda, rows, cols, F32, 2)
    w, _, _, _ = weights_of(cuda, cols, F32, 3)
    o = ops.layer_norm(x, w)
    want = ops.layer_norm_bwd(dy, x, w, o.mean, o.rstd)
    off = torch.empty(2, rows + 1, device=cuda)
    off[0, 1:], off[1, 1:] = o.mean, o.rstd
    got = ops.layer_norm_bwd(dy, x, w, off[0, 1:], off[1, 1:])
    # the row sums are taken in another order: 2 * 64 * 2^-24 of values of order one, times rstd
    tol = 2 * 64 * 2.0**-24 * float(o.rstd.max()) * 8
    assert float((got.dx - want.dx).abs().max()) <= tol
    assert float((got.dweight - want.dweight).abs().max()) <= F32_ERR * float((dy.abs() * 4).sum(0).max())


def test_in_a_graph(cuda):
    x, _ = rows_of(cuda, 512, 80, BF16, 1)
    r, _ = rows_of(cuda, 512, 80, BF16, 2)
    w, b, _, _ = weights_of(cuda, 80, F32, 3)

    def step(fwd=None, bwd=None):
        o = ops.dropout_add_norm(x, r, w, b, 0.2, 5, 6, out=fwd)
        return o, ops.dropout_add_norm_bwd(x, r, o.z, w, o.mean, o.rstd, 0.2, 5, 6, out=bwd)

    o, g = step()
    want = [t.clone() for t in (o.y, g.dx, g.dresidual, g.dweight, g.dbias)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(o, g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step(o, g)
    for t in (o.y, g.dx, g.dresidual, g.dweight, g.dbias):
        t.zero_()
    torch.cuda.synchronize()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, (o.y, g.dx, g.dresidual, g.dweight, g.dbias)))


def test_refusals(cuda):
    ctx = ops.context(cuda)
    x = torch.zeros(4, 8, device=cuda)
    w = torch.ones(8, device=cuda)
    st = torch.zeros(4, device=cuda)
    for bad in (-0.1, 1.5, float("nan")):
        with pytest.raises(_native.VsError, match="not in"):
            ops.dropout(x, bad, 1)
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(_native.VsError, match="eps"):
            ops.layer_norm(x, w, w, eps)
    for call in (lambda: ops.dropout(x.cpu(), 0.1, 1), lambda: ops.dropout(x.t(), 0.1, 1),
                 lambda: ops.dropout(x.int(), 0.1, 1), lambda: ops.layer_norm(x.double()),
                 lambda: ops.layer_norm(x.t()), lambda: ops.layer_norm(x, w[:7]),
                 lambda: ops.layer_norm(x, w.half()), lambda: ops.layer_norm(x[:, :0]),
                 lambda: ops.layer_norm(x, w, w.half()),
                 lambda: ops.layer_norm(x[:1].expand(4, 8)),
                 lambda: ops.layer_norm(x, out=ops.LayerNormOutput(x.half(), st, st)),
                 lambda: ops.layer_norm_bwd(x.half(), x, w, st, st), lambda: ops.layer_norm_bwd(x, x, w, st[:3], st),
                 lambda: ops.dropout_add_norm(x, x[:2], w, w, 0.1, 1)):
        with pytest.raises(AssertionError):
            call()
    # through the C entry points: null buffers, unknown types, bad strides, misaligned buffers
    p, lib, z64 = x.data_ptr(), ctx.lib, ctypes.c_uint64(0)
    assert lib.vs_dropout(ctx.h, 8, 0, None, 0.1, 1, 1, p) == 1
    assert lib.vs_dropout(ctx.h, 8, 7, p, 0.1, 1, 1, p) == 5
    assert lib.vs_dropout(ctx.h, 4, 0, p + 2, 0.1, 1, 1, p) == 1
    assert lib.vs_layer_norm(ctx.h, 4, 0, 0, 0, p, 0, None, None, 1e-5, p, None, None) == 1
    assert lib.vs_layer_norm(ctx.h, 4, 8, 0, 1, p, 0, None, None, 1e-5, p, None, None) == 5
    assert lib.vs_layer_norm(ctx.h, 4, 8, 0, 0, p, 7, None, None, 1e-5, p, None, None) == 1
    assert lib.vs_layer_norm(ctx.h, 1 << 59, 8, 0, 0, p, 0, None, None, 1e-5, p, None, None) == 2
    assert lib.vs_layer_norm_backward(ctx.h, 4, 8, 0, 0, p, 0, p, 0, None, None, p, p, None, None) == 1
    assert lib.vs_dropout_add_norm(ctx.h, 4, 8, 0, 0, p, 0, None, 0, None, None, 0.1, 1, 1, 1e-5, p, p, None, None) == 1
    assert lib.vs_dropout_add_norm_backward(ctx.h, 4, 8, 0, 0, p, 0, None, 0, p, 0, None, p, p, 2.0, 1, 1, p, p, None,
                                            None) == 1
    assert b"p = 2" in lib.vs_ctx_last_error(ctx.h)
    assert lib.vs_layer_norm(None, 4, 8, 0, 0, p, 0, None, None, 1e-5, p, None, None) == 1
    # statistics are optional in the C entry point
    y = torch.empty_like(x)
    assert lib.vs_layer_norm(ctx.h, 4, 8, 0, 0, p, 0, None, None, 1e-5, y.data_ptr(), None, None) == 0
