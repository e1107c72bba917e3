"""The row operators where calls reach the edges of what the header allows:
buffers that serve as input and output, sums over very many rows, captured
graphs, streams and threads.

Helpers and the tolerances of `close` are those of test_gpu_rows.py."""
import ctypes
import threading

import pytest
import torch

from tests.test_gpu_rows import DTYPES, F32, rows_of, weights_of
from vauss_b200 import _native, ops

pytestmark = pytest.mark.gpu

# One shape for each backward kernel: rows on warps and on a CTA, direct and streaming, and rows that no kernel holds.
BACKWARD = [(1, 64), (40, 100), (3, 4096), (900, 64), (50_003, 64), (60_001, 59), (801, 5003), (70, 20_000), (5, 33_333)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", BACKWARD)
@pytest.mark.parametrize("over", ["dweight", "dbias"])
def test_weight_gradients_over_the_weight(cuda, dtype, rows, cols, over):
    """dweight or dbias in the weight's own buffer: the bits of a call with buffers of their own."""
    z, _ = rows_of(cuda, rows, cols, dtype, 1)
    dy, _ = rows_of(cuda, rows, cols, dtype, 2)
    dz, _ = rows_of(cuda, rows, cols, dtype, 3)
    w, _, _, _ = weights_of(cuda, cols, F32, 4)
    o = ops.layer_norm(z, w)
    wide = torch.zeros(rows, cols + 3, dtype=dtype, device=cuda)
    wide[:, 1:1 + cols] = dy
    for g in (dy, wide[:, 1:1 + cols]):
        want = ops.layer_norm_bwd(g, z, w, o.mean, o.rstd)
        own = w.clone()
        out = ops.LayerNormGrads(torch.empty_like(z), torch.empty_like(w), torch.empty_like(w))
        setattr(out, over, own)
        got = ops.layer_norm_bwd(g, z, own, o.mean, o.rstd, out=out)
        assert all(torch.equal(getattr(got, k), getattr(want, k)) for k in ("dx", "dweight", "dbias"))
        want = ops.dropout_add_norm_bwd(g, dz, z, w, o.mean, o.rstd, 0.25, 1, 2)
        own = w.clone()
        out = ops.DropoutAddNormGrads(torch.empty_like(z), torch.empty_like(z), torch.empty_like(w), torch.empty_like(w))
        setattr(out, over, own)
        got = ops.dropout_add_norm_bwd(g, dz, z, own, o.mean, o.rstd, 0.25, 1, 2, out=out)
        assert all(torch.equal(getattr(got, k), getattr(want, k)) for k in ("dx", "dresidual", "dweight", "dbias"))


def test_statistics_do_not_share_the_weights(cuda):
    """mean or rstd in the weight's or the bias's buffer (64 rows of 64): rows would read what others wrote."""
    x, _ = rows_of(cuda, 64, 64, F32, 1)
    w, b, _, _ = weights_of(cuda, 64, F32, 2)
    y, s = torch.empty_like(x), torch.empty(64, device=cuda)
    for mean, rstd in ((w, s), (b, s), (s, w), (s, b)):
        with pytest.raises(_native.VsError, match="mean and rstd"):
            ops.layer_norm(x, w, b, out=ops.LayerNormOutput(y, mean, rstd))
        with pytest.raises(_native.VsError, match="mean and rstd"):
            ops.dropout_add_norm(x, x, w, b, 0.1, 1, out=ops.DropoutAddNormOutput(y, torch.empty_like(x), mean, rstd))


def test_destroying_a_context_waits_for_every_stream(cuda):
    """A ctx whose calls went to one stream and that ends on another: its buffers are freed only after the first
    stream's work (held back by a long kernel before the calls) has ended."""
    z, _ = rows_of(cuda, 20_000, 96, F32, 1)
    dy, _ = rows_of(cuda, 20_000, 96, F32, 2)
    w, _, _, _ = weights_of(cuda, 96, F32, 3)
    o = ops.layer_norm(z, w)
    want = ops.layer_norm_bwd(dy, z, w, o.mean, o.rstd)
    got = [torch.empty_like(t) for t in (want.dx, want.dweight, want.dbias)]
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    ctx = ops.Context(cuda.index or 0)
    lib = ctx.lib
    assert lib.vs_ctx_set_stream(ctx.h, a.cuda_stream) == 0
    with torch.cuda.stream(a):
        torch.cuda._sleep(400_000_000)  # about 0.2 s
    assert lib.vs_layer_norm_backward(ctx.h, 20_000, 96, 0, 0, dy.data_ptr(), 0, z.data_ptr(), 0, w.data_ptr(),
                                      o.mean.data_ptr(), o.rstd.data_ptr(), *(t.data_ptr() for t in got)) == 0
    assert not a.query()
    assert lib.vs_ctx_set_stream(ctx.h, b.cuda_stream) == 0
    h, ctx.h = ctx.h, None
    lib.vs_ctx_destroy(h)
    assert a.query()
    assert all(torch.equal(t, u) for t, u in zip(got, (want.dx, want.dweight, want.dbias)))


def test_threads_on_streams_of_their_own(cuda):
    """Calls of several threads at once, each on its stream: the bits of calls one after another."""
    w, _, _, _ = weights_of(cuda, 96, F32, 1)
    data = [(rows_of(cuda, 20_000, 96, F32, 10 + k)[0], rows_of(cuda, 20_000, 96, F32, 20 + k)[0]) for k in range(3)]
    stats = [ops.layer_norm(z, w) for _, z in data]
    want = [ops.layer_norm_bwd(dy, z, w, o.mean, o.rstd) for (dy, z), o in zip(data, stats)]
    torch.cuda.synchronize()
    got, gate = [[] for _ in data], threading.Barrier(len(data))

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            gate.wait(30)
            for _ in range(50):
                got[k].append(ops.layer_norm_bwd(*data[k], w, stats[k].mean, stats[k].rstd))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for per_thread, ref in zip(got, want):
        assert len(per_thread) == 50
        for g in per_thread:
            assert all(torch.equal(getattr(g, k), getattr(ref, k)) for k in ("dx", "dweight", "dbias"))


def test_the_error_word_is_read(cuda):
    """A wait that runs out on the context of the row operators (a peer barrier that nobody else signals) raises from
    check_device, once; without one it returns."""
    ops.layer_norm(torch.ones(4, 8, device=cuda))
    ops.check_device(cuda)
    ctx = ops._row_context(cuda.index or 0)
    mine, other = (torch.zeros(2, dtype=torch.int32, device=cuda) for _ in range(2))
    ptrs = (ctypes.c_void_p * _native.PEER_MAX)(mine.data_ptr(), other.data_ptr())
    assert ctx.lib.vs_peer_barrier(ctx.h, ptrs, 2, 0, 1) == 0
    with pytest.raises(_native.VsError, match="TIMEOUT"):
        ops.check_device()
    ops.check_device(0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", BACKWARD + [(1_000, 64), (40_001, 12), (20_000, 64), (1_001, 4096)])
def test_every_kernel_in_a_graph(cuda, dtype, rows, cols):
    """Forward and backward of both norms and of dropout captured and replayed twice, the column sums by one CTA, by the
    last one and by the joining kernel: the bits of direct calls."""
    x, _ = rows_of(cuda, rows, cols, dtype, 1)
    r, _ = rows_of(cuda, rows, cols, dtype, 2)
    w, b, _, _ = weights_of(cuda, cols, F32, 3)

    def step(o=None, g=None, n=None, gn=None, d=None):
        o = ops.dropout_add_norm(x, r, w, b, 0.2, 5, 6, out=o)
        g = ops.dropout_add_norm_bwd(x, r, o.z, w, o.mean, o.rstd, 0.2, 5, 6, out=g)
        n = ops.layer_norm(x, w, b, out=n)
        gn = ops.layer_norm_bwd(r, x, w, n.mean, n.rstd, out=gn)
        return o, g, n, gn, ops.dropout(x, 0.2, 5, 7, out=d)

    outs = step()
    flat = [t for part in outs[:4] for t in vars(part).values()] + [outs[4]]
    want = [t.clone() for t in flat]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(*outs)
    for t in flat:
        t.zero_()
    torch.cuda.synchronize()
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, flat))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", BACKWARD + [(1_000, 3), (15_000, 750), (300, 703), (9, 1), (1_000, 1030)])
def test_nan_and_infinity_stay_in_their_rows(cuda, dtype, rows, cols):
    """Rows that hold a NaN or an infinity leave the other rows' results as they are, bit for bit, wherever the kernels
    keep rows side by side; their own are NaN (of one column: NaN too, from inf - inf)."""
    clean = [rows_of(cuda, rows, cols, dtype, k)[0] for k in range(3)]
    w, b, _, _ = weights_of(cuda, cols, F32, 4)
    bad = torch.arange(rows, device=cuda) % 7 == 3
    bad[0] = bad[-1] = True
    if rows == 1:
        bad[:] = True
    value = torch.where(torch.arange(rows, device=cuda) % 2 == 0, float("nan"), float("inf")).to(dtype)
    at = torch.arange(rows, device=cuda) % cols
    x = clean[0].clone()
    x[bad, at[bad]] = value[bad]
    for strided in (False, True):
        def lay(t):
            if not strided:
                return t
            wide = torch.full((rows, cols + 3), float("nan"), dtype=dtype, device=cuda)
            wide[:, 1:1 + cols] = t
            return wide[:, 1:1 + cols]
        want, got = ops.layer_norm(lay(clean[0]), w, b), ops.layer_norm(lay(x), w, b)
        for k in ("y", "mean", "rstd"):
            assert torch.equal(getattr(got, k)[~bad], getattr(want, k)[~bad]), f"{k} strided {strided}"
        assert bool(got.y[bad].isnan().all())
        want = ops.dropout_add_norm(lay(clean[1]), lay(clean[0]), w, b, 0.25, 1, 2)
        got = ops.dropout_add_norm(lay(clean[1]), lay(x), w, b, 0.25, 1, 2)
        for k in ("y", "z", "mean", "rstd"):
            assert torch.equal(getattr(got, k)[~bad], getattr(want, k)[~bad]), f"joined {k} strided {strided}"
        o = ops.layer_norm(clean[0], w, b)
        for args, ref in (((clean[1], x), (clean[1], clean[0])), ((x, clean[1]), (clean[0], clean[1]))):  # in z, in dy
            args, ref = [lay(t) for t in args], [lay(t) for t in ref]
            g, r = ops.layer_norm_bwd(*args, w, o.mean, o.rstd), ops.layer_norm_bwd(*ref, w, o.mean, o.rstd)
            assert torch.equal(g.dx[~bad], r.dx[~bad]), f"dx strided {strided}"
            j = ops.dropout_add_norm_bwd(args[0], lay(clean[2]), args[1], w, o.mean, o.rstd, 0.25, 1, 2)
            q = ops.dropout_add_norm_bwd(ref[0], lay(clean[2]), ref[1], w, o.mean, o.rstd, 0.25, 1, 2)
            assert torch.equal(j.dx[~bad], q.dx[~bad]) and torch.equal(j.dresidual[~bad], q.dresidual[~bad])
