"""A learned head over splats: a residual network that turns a feature vector
each splat carries into an offset of its base colour (no counterpart in the
reference).

The blocks are the usual ones, h <- h + dropout(relu(norm(h) W1) W2).  Between
the matrix products (plain library products through torch) stand the row
operators of ``ops``: ``dropout`` of the features where it is asked for,
``layer_norm`` at the entry, ``dropout_add_norm`` between blocks, which sums,
drops and normalises in one pass, and their gradients.
Weights and the optimizer are f32; rows are f32, f16 or bf16.  The gradient of a
loss over an image is far below f16's range, so an f16 head scales what enters
its backward by a power of two and takes it out of the results again.

``python -m vauss_b200.feature_head`` fits the head to a scene whose splats are
lit differently in the views than in their own colours, and prints the loss.
"""
from __future__ import annotations

import torch

from . import ops


class FeatureHead:
    """forward(features) -> colour offsets [N, 3]; backward(gradient of those) -> gradient of the features, with the
    parameters' gradients in ``grads``.  One forward is kept for one backward.  ``p`` drops the blocks' branches, ``p_in``
    the features."""

    def __init__(self, width: int, hidden: int, blocks: int, p: float, device, dtype=torch.bfloat16, seed: int = 0,
                 p_in: float = 0.0):
        assert width > 0 and hidden > 0 and blocks >= 0 and 0.0 <= p <= 1.0 and 0.0 <= p_in <= 1.0
        gen = torch.Generator(device=device).manual_seed(seed)
        self.blocks, self.p, self.p_in, self.dtype, self.seed, self.step = blocks, p, p_in, dtype, seed, 0
        self.params: dict[str, torch.Tensor] = {}

        def weight(name, rows, cols, gain):
            self.params[name] = torch.randn(rows, cols, device=device, generator=gen) * (gain / rows ** 0.5)

        for k in range(blocks + 1):
            self.params[f"norm{k}.weight"] = torch.ones(width, device=device)
            self.params[f"norm{k}.bias"] = torch.zeros(width, device=device)
        for k in range(blocks):
            weight(f"block{k}.w1", width, hidden, 2 ** 0.5)
            weight(f"block{k}.w2", hidden, width, 0.5)
        weight("out", width, 3, 0.1)
        self.grads = {k: torch.zeros_like(v) for k, v in self.params.items()}
        self._saved = None

    def _w(self, name: str) -> torch.Tensor:
        return self.params[name].to(self.dtype)

    def forward(self, features: torch.Tensor, train: bool = True) -> torch.Tensor:
        """features [N, width] in the head's type.  ``train`` draws a new mask per call and block."""
        assert features.dtype == self.dtype, f"features are {features.dtype}, the head is {self.dtype}"
        p, p_in = (self.p, self.p_in) if train else (0.0, 0.0)
        if train:
            self.step += 1
        w = self.params
        offset_in = (1 << 63) + self.step  # apart from the blocks'
        if p_in:
            features = ops.dropout(features.contiguous(), p_in, self.seed, offset_in)
        first = ops.layer_norm(features, w["norm0.weight"], w["norm0.bias"])
        h, y, kept = features, first.y, []
        for k in range(self.blocks):
            a = torch.relu(y @ self._w(f"block{k}.w1"))
            r = a @ self._w(f"block{k}.w2")
            offset = self.step * max(self.blocks, 1) + k
            o = ops.dropout_add_norm(r, h, w[f"norm{k + 1}.weight"], w[f"norm{k + 1}.bias"], p, self.seed, offset)
            kept.append((y, a, o, offset))
            h, y = o.z, o.y
        self._saved = (features, first, kept, y, p, p_in, offset_in)
        return (y @ self._w("out")).float()

    def backward(self, dout: torch.Tensor) -> torch.Tensor:
        """The features' gradient, in the head's type (f32 for an f16 head, whose range small ones would leave)."""
        features, first, kept, y, p, p_in, offset_in = self._saved
        g, w = self.grads, self.params
        scale = _f16_scale(dout) if self.dtype == torch.float16 else None
        dout = (dout if scale is None else dout * scale).to(self.dtype)

        def product(a, b):  # over the rows: in f32 where the sum could leave the type's range
            return a @ b if scale is None else torch.mm(a, b, out_dtype=torch.float32)

        def leave(name, value):
            g[name].copy_(value if scale is None else value / scale)

        leave("out", product(y.t(), dout))
        dy, dz = dout @ self._w("out").t(), None
        for k in reversed(range(self.blocks)):
            y_in, a, o, offset = kept[k]
            d = ops.dropout_add_norm_bwd(dy, dz, o.z, w[f"norm{k + 1}.weight"], o.mean, o.rstd, p, self.seed, offset)
            leave(f"norm{k + 1}.weight", d.dweight)
            leave(f"norm{k + 1}.bias", d.dbias)
            dz = d.dresidual
            leave(f"block{k}.w2", product(a.t(), d.dx))
            da = (d.dx @ self._w(f"block{k}.w2").t()).mul_(a > 0)
            leave(f"block{k}.w1", product(y_in.t(), da))
            dy = da @ self._w(f"block{k}.w1").t()
        d = ops.layer_norm_bwd(dy, features, w["norm0.weight"], first.mean, first.rstd)
        leave("norm0.weight", d.dweight)
        leave("norm0.bias", d.dbias)
        if scale is None:
            dx = d.dx if dz is None else d.dx + dz
        else:
            dx = (d.dx.float() if dz is None else d.dx.float() + dz.float()) / scale
        return ops.dropout_bwd(dx, p_in, self.seed, offset_in, out=dx) if p_in else dx


def _f16_scale(dout: torch.Tensor) -> torch.Tensor:
    """The power of two (on the device) that brings the largest value to 8 to 16: room above for the rows' rstd, of up
    to 1 / sqrt(eps) = 316, and 17 binary places below for values of f16's full precision."""
    if dout.numel() == 0:
        return torch.ones((), device=dout.device)
    places = torch.floor(4.0 - torch.log2(dout.detach().float().abs().amax())).clamp(-60, 60)  # 60 for zeros
    return torch.where(places.isfinite(), torch.exp2(places), 1.0)


def lit_views(n_views: int = 4, device="cuda:0"):
    """The tiny scene, and the images of the same splats lit from one side: (splats, cameras, packed ground truth)."""
    import numpy as np

    from . import scenes
    from .trainer import Splats
    sp, _, cams = scenes.config_tiny()
    lit = scenes.SplatSet(sp.transforms, sp.sh.copy(), sp.raw_opac)
    lit.sh[:, 0, :] += (0.8 * np.tanh(2.0 * sp.transforms[:, :1]) * np.float32([1.0, 0.2, -0.8])).astype(np.float32)
    cfg = ops.render_cfg(0, mip=True)
    shown, splats = Splats.from_numpy(lit, device), Splats.from_numpy(sp, device)
    views = []
    for cam in cams[:n_views]:
        img = ops.render(cam, cfg, shown.transforms, shown.sh_coeffs, shown.raw_opacities).out_img[..., :3]
        views.append((cam, torch.from_numpy(scenes.pack_rgba8(img.cpu().numpy()).view(np.int32)).to(device)))
    return splats, views


def fit(steps: int = 60, width: int = 64, hidden: int = 128, blocks: int = 2, p: float = 0.1, lr: float = 3e-3,
        device="cuda:0", dtype=torch.bfloat16, p_in: float = 0.0) -> list[float]:
    """Trains a head (and nothing else) on ``lit_views``; returns the loss of every step."""
    splats, views = lit_views(device=device)
    cfg = ops.render_cfg(0, mip=True)
    gen = torch.Generator(device=device).manual_seed(1)
    mix = torch.randn(3, width, device=device, generator=gen)
    features = torch.sin(3.0 * splats.transforms[:, :3] @ mix).to(dtype)  # what a splat's place tells
    head = FeatureHead(width, hidden, blocks, p, device, dtype, p_in=p_in)
    opt = torch.optim.Adam(head.params.values(), lr=lr)
    n = splats.num_splats
    base, frame, losses = splats.sh_coeffs[:, 0, :], ops.Frame(ops.context(splats.transforms.device)), []
    for it in range(steps):
        cam, gt = views[it % len(views)]
        sh = (base + head.forward(features)).unsqueeze(1).contiguous()
        out = ops.render(cam, cfg, splats.transforms, sh, splats.raw_opacities, frame=frame)
        loss = ops.image_loss(out.out_img, gt, 0.8, -0.2)
        vc = ops.rasterize_bwd(frame, out.out_img, loss.dl_dpred)
        rows = torch.zeros(n, 14, device=device)  # transforms 10 | SH 3 | opacity 1
        ops.vjp_dense(frame, cfg, splats.transforms, sh, splats.raw_opacities, vc, rows,
                      torch.zeros(n, device=device))
        head.backward(rows[:, 10:13])
        for k, v in head.params.items():
            v.grad = head.grads[k]
        opt.step()
        losses.append(loss.loss.clone())
    ops.check_device(device)
    return torch.stack(losses).tolist()


def main() -> None:
    losses = fit()
    print(f"loss {losses[0]:.4f} -> {sum(losses[-4:]) / 4:.4f} in {len(losses)} steps")


if __name__ == "__main__":
    main()
