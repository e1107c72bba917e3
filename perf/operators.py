"""Measured cases of the row operators: dropout from a counter-based generator,
layer norm, and the two joined over a residual stream, forward and backward.

Each case is one call on ``rows x cols`` values.  ``run`` computes it in
elementary torch operations in 32 bits, or, where ``own`` is set, through
``vauss_b200.ops``; ``exact`` computes it from the definition in 64 bits.

Definitions (i = row * cols + col, the value's index):
  dropout     t = round(65536 p); the value is kept when its 16-bit number is
              at least t, and then multiplied by 65536 / (65536 - t); the number
              is half-word i % 8 of the four words that Philox 4x32 with ten
              rounds gives for the counter (i / 8, offset) and the key seed
  layer norm  y = (x - mean) rstd weight + bias, rstd = 1 / sqrt(var + eps)
  joined      z = residual + dropout(x); y = layer norm of z
"""
import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
OPS = ("dropout", "dropout_bwd", "layer_norm", "layer_norm_bwd", "dropout_add_norm", "dropout_add_norm_bwd")
EPS = 1e-5

# Full-width values read and written per element of the matrix
STREAMS = {"dropout": 2, "dropout_bwd": 2, "layer_norm": 2, "layer_norm_bwd": 3, "dropout_add_norm": 4,
           "dropout_add_norm_bwd": 5}
# Operations per element: products, sums and comparisons of the formulas, and
# the generator's ten rounds of two products and four exclusive ors per eight elements
FLOPS = {"dropout": 10, "dropout_bwd": 10, "layer_norm": 8, "layer_norm_bwd": 15, "dropout_add_norm": 19,
         "dropout_add_norm_bwd": 26}
MOST = 3_000_000 * 64  # elements of the largest listed case
MOST_STREAMED = MOST * 3 * 2  # and the bytes that it moves


def _case(name, op, rows, cols, dtype, p=0.1):
    return {"name": name, "op": op, "rows": rows, "cols": cols, "dtype": dtype, "p": p}


def listed():
    return [
        # the opacities of the 20k-splat scene: a call that is all latency
        _case("dropout_20k_f32", "dropout", 20_000, 1, "f32"),
        # the half-precision degree-3 colour rows of the 3M-splat scene, gradient
        _case("dropout_bwd_3m_48_f16", "dropout_bwd", 3_000_000, 48, "f16", 0.25),
        # one row of a wide head: the smallest normalisation
        _case("norm_1_4096_bf16", "layer_norm", 1, 4096, "bf16"),
        # the 59 trained values of each of 1M splats, whitened: an odd width
        _case("norm_1m_59_f32", "layer_norm", 1_000_000, 59, "f32"),
        # a wide head over a batch of rows
        _case("norm_16k_4096_bf16", "layer_norm", 16_384, 4096, "bf16"),
        # the 20k-splat scene's features, gradient
        _case("norm_bwd_20k_64_f16", "layer_norm_bwd", 20_000, 64, "f16"),
        # 3M splats with 64 features: very many short rows into one weight gradient
        _case("norm_bwd_3m_64_bf16", "layer_norm_bwd", 3_000_000, 64, "bf16"),
        # a ragged matrix, odd in both directions
        _case("norm_bwd_1021_5003_f32", "layer_norm_bwd", 1021, 5003, "f32"),
        # between two blocks of a head over the 20k-splat scene
        _case("join_20k_64_bf16", "dropout_add_norm", 20_000, 64, "bf16"),
        # the same over 1M splats, with wider features
        _case("join_1m_128_bf16", "dropout_add_norm", 1_000_000, 128, "bf16"),
        # its gradient over a ragged matrix whose rows are not whole vectors
        _case("join_bwd_4099_1030_f16", "dropout_add_norm_bwd", 4099, 1030, "f16", 0.2),
        # its gradient over a batch of wide rows
        _case("join_bwd_8k_4096_bf16", "dropout_add_norm_bwd", 8192, 4096, "bf16"),
    ]


def draw(rng):
    """Any operator and type; widths from 1 to 16384 (every third one a multiple of 8) and any number of rows that
    the largest listed case's traffic allows, both spread over their logarithm; a listed case's size is not drawn."""
    op, dtype = rng.choice(OPS), rng.choice(sorted(DTYPES))
    cols = int(2 ** rng.uniform(0, 14))
    if rng.randrange(3) == 0:
        cols = max(8, cols // 8 * 8)
    most = min(MOST, MOST_STREAMED // (STREAMS[op] * SIZE[dtype])) // cols
    rows = max(1, int(2 ** rng.uniform(0, np.log2(max(2, most)))))
    return {"op": op, "rows": min(rows, max(1, most)), "cols": cols, "dtype": dtype,
            "p": rng.choice([0.0, 0.05, 0.1, 0.2, 0.3, 0.5, 0.9])}


def work(case):
    n, cols, rows = case["rows"] * case["cols"], case["cols"], case["rows"]
    size = STREAMS[case["op"]] * n * SIZE[case["dtype"]]
    if "norm" in case["op"]:
        size += 8 * rows + (12 if case["op"].endswith("bwd") else 8) * cols  # statistics; weights (and gradients)
    return {"bytes": size, "flops": FLOPS[case["op"]] * n}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, dtype = case["rows"], case["cols"], DTYPES[case["dtype"]]

    def normal(scale, *shape):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale)

    def feature():  # rows of different level and spread, as activations have
        x = normal(1.0, rows, cols)
        x.mul_(normal(0.5, rows, 1).exp_()).add_(normal(0.3, rows, 1))
        return x.to(dtype)

    s = {"op": case["op"], "p": case["p"], "seed": int(torch.randint(1 << 62, (), device="cuda", generator=gen)),
         "offset": seed * 7 + 1, "out": None}
    if case["op"] in ("layer_norm", "dropout_add_norm"):
        s["x"] = feature()
        s["weight"] = normal(0.2, cols).add_(1.0)
        s["bias"] = normal(0.2, cols)
    elif case["op"].endswith("norm_bwd"):
        z = feature()
        zf = z.float()
        s["mean"] = zf.mean(1)
        s["rstd"] = 1.0 / torch.sqrt((zf - s["mean"][:, None]).square_().mean(1) + EPS)
        s["z"] = z
        s["dy"] = normal(0.1, rows, cols).to(dtype)
        s["weight"] = normal(0.2, cols).add_(1.0)
    else:
        s["x"] = feature() if case["op"] == "dropout" else normal(0.1, rows, cols).to(dtype)
    if case["op"] == "dropout_add_norm":
        s["residual"] = feature()
    elif case["op"] == "dropout_add_norm_bwd":
        s["dz"] = normal(0.1, rows, cols).to(dtype)
    return s


def _philox(groups, offset, seed):
    """The four 32-bit words of each counter, as int64 tensors.  A 32 x 32-bit product is formed from two
    32 x 16-bit ones, which fit 63 bits."""
    mask = 0xFFFFFFFF

    def mul(m, x):
        low = x * (m & 0xFFFF)
        mid = x * (m >> 16) + (low >> 16)
        return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)

    c0, c1 = groups & mask, groups >> 32
    c2 = torch.full_like(groups, offset & mask)
    c3 = torch.full_like(groups, (offset >> 32) & mask)
    k0, k1 = seed & mask, (seed >> 32) & mask
    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return c0, c1, c2, c3


def _threshold(p):
    return 65536 if p >= 1 else min(65535, int(p * 65536 + 0.5))


def _keep_scale(s, shape):
    """0 or the scale of a kept value, f32, and whether it is kept."""
    n = shape[0] * shape[1]
    words = _philox(torch.arange((n + 7) // 8, device="cuda", dtype=torch.int64), s["offset"], s["seed"])
    lanes = torch.stack([(w >> half & 0xFFFF).to(torch.int32) for w in words for half in (0, 16)], 1)
    t = _threshold(s["p"])
    return (lanes.view(-1)[:n] >= t).view(shape), 65536.0 / (65536 - t) if t < 65536 else 0.0


def _dropout(s, x):
    if s["p"] == 0:
        return x
    keep, scale = _keep_scale(s, x.shape)
    return torch.where(keep, x * scale, torch.zeros((), device=x.device))


def _layer_norm(s, z):
    mean = z.mean(1, keepdim=True)
    d = z - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    return d * rstd * s["weight"] + s["bias"], mean[:, 0], rstd[:, 0]


def _layer_norm_bwd(s):
    dy, h = s["dy"].float(), (s["z"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["weight"]
    dz = (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)) * s["rstd"][:, None]
    return dz, (dy * h).sum(0), dy.sum(0)


def _plain(s):
    op = s["op"]
    if op in ("dropout", "dropout_bwd"):
        return _dropout(s, s["x"].float()).to(s["x"].dtype)
    if op == "layer_norm":
        y, mean, rstd = _layer_norm(s, s["x"].float())
        return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}
    if op == "dropout_add_norm":
        z = (s["residual"].float() + _dropout(s, s["x"].float())).to(s["x"].dtype)  # stored, and normalised as stored
        y, mean, rstd = _layer_norm(s, z.float())
        return {"y": y.to(z.dtype), "z": z, "mean": mean, "rstd": rstd}
    dz, dweight, dbias = _layer_norm_bwd(s)
    if op == "layer_norm_bwd":
        return {"dx": dz.to(s["z"].dtype), "dweight": dweight, "dbias": dbias}
    dz = dz + s["dz"].float()
    return {"dx": _dropout(s, dz).to(s["z"].dtype), "dresidual": dz.to(s["z"].dtype), "dweight": dweight,
            "dbias": dbias}


def run(state):
    s = state
    if not own:
        return _plain(s)
    from vauss_b200 import ops
    op = s["op"]
    if op == "dropout":
        s["out"] = y = ops.dropout(s["x"], s["p"], s["seed"], s["offset"], out=s["out"])
        return y
    if op == "dropout_bwd":
        s["out"] = dx = ops.dropout_bwd(s["x"], s["p"], s["seed"], s["offset"], out=s["out"])
        return dx
    if op == "layer_norm":
        s["out"] = o = ops.layer_norm(s["x"], s["weight"], s["bias"], EPS, out=s["out"])
        return {"y": o.y, "mean": o.mean, "rstd": o.rstd}
    if op == "dropout_add_norm":
        s["out"] = o = ops.dropout_add_norm(s["x"], s["residual"], s["weight"], s["bias"], s["p"], s["seed"],
                                            s["offset"], EPS, out=s["out"])
        return {"y": o.y, "z": o.z, "mean": o.mean, "rstd": o.rstd}
    if op == "layer_norm_bwd":
        s["out"] = g = ops.layer_norm_bwd(s["dy"], s["z"], s["weight"], s["mean"], s["rstd"], out=s["out"])
        return {"dx": g.dx, "dweight": g.dweight, "dbias": g.dbias}
    s["out"] = g = ops.dropout_add_norm_bwd(s["dy"], s["dz"], s["z"], s["weight"], s["mean"], s["rstd"], s["p"],
                                            s["seed"], s["offset"], out=s["out"])
    return {"dx": g.dx, "dresidual": g.dresidual, "dweight": g.dweight, "dbias": g.dbias}


def _exact_mask(s, rows, cols):
    """The scale factor of every element (0 where it is dropped), from the generator in unsigned 64-bit numpy."""
    t = _threshold(s["p"])
    if t == 0:
        return torch.ones(rows, cols, dtype=torch.float64)
    n = rows * cols
    low = np.uint64(0xFFFFFFFF)
    ctr = [np.arange(-(-n // 8), dtype=np.uint64), None, None, None]
    ctr[1] = ctr[0] >> np.uint64(32)
    ctr[0] = ctr[0] & low
    ctr[2] = np.full_like(ctr[0], s["offset"] % 2**32)
    ctr[3] = np.full_like(ctr[0], s["offset"] // 2**32 % 2**32)
    for r in range(10):
        key = [np.uint64((s["seed"] + r * 0x9E3779B9) % 2**32), np.uint64((s["seed"] // 2**32 + r * 0xBB67AE85) % 2**32)]
        a, b = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(b >> np.uint64(32)) ^ ctr[1] ^ key[0], b & low, (a >> np.uint64(32)) ^ ctr[3] ^ key[1], a & low]
    numbers = np.empty((ctr[0].size, 8), np.uint16)
    for j in range(8):
        numbers[:, j] = (ctr[j // 2] >> np.uint64(16 * (j % 2))).astype(np.uint16)
    kept = torch.from_numpy(numbers.reshape(-1)[:n].astype(np.int32) >= t).view(rows, cols)
    return kept.to(torch.float64) * (65536.0 / (65536 - t))


def exact(case, seed):
    s = prepare(case, seed)
    op, rows, cols = case["op"], case["rows"], case["cols"]
    d = {k: v.double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    factor = _exact_mask(s, rows, cols).cuda() if op not in ("layer_norm", "layer_norm_bwd") else None
    if op in ("dropout", "dropout_bwd"):
        return d["x"] * factor
    if op in ("layer_norm", "dropout_add_norm"):
        x = d["x"]
        if op == "dropout_add_norm":  # z is normalised as it is stored, in the inputs' type
            z = d["residual"] + x * factor
            x = z.to(s["x"].dtype).double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = (var + EPS).rsqrt()
        y = torch.addcmul(d["bias"], (x - mean[:, None]).mul_(rstd[:, None]), d["weight"])
        return {"y": y, "mean": mean, "rstd": rstd} | ({"z": z} if op == "dropout_add_norm" else {})
    h = (d["z"] - d["mean"][:, None]).mul_(d["rstd"][:, None])
    dweight, dbias = torch.einsum("rc,rc->c", d["dy"], h), d["dy"].sum(0)
    g = d["dy"] * d["weight"]
    along = torch.einsum("rc,rc->r", g, h) / cols
    t = (g - g.mean(1, keepdim=True)).sub_(h.mul_(along[:, None])).mul_(d["rstd"][:, None])
    if op == "layer_norm_bwd":
        return {"dx": t, "dweight": dweight, "dbias": dbias}
    t.add_(d["dz"])
    return {"dx": t * factor, "dresidual": t, "dweight": dweight, "dbias": dbias}
