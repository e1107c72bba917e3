"""The head over splats against the same network in 64 bits under autograd, and
its fit to a scene through the renderer and its gradient.

Tolerance of the comparison: rows and weights are f32, the products of up to 48
terms run in f32 (allow_tf32 is off by default), so every intermediate is
within about 48 * 2^-24 = 3e-6 of its size per layer; eight layers forward and
back stay below 1e-4 of the largest value of each gradient."""
import numpy as np
import pytest
import torch

from tests.test_gpu_rows import keep_mask
from vauss_b200 import feature_head, ops

pytestmark = pytest.mark.gpu

REL = 1e-4


def _norm(x, w, b):
    m = x.mean(-1, keepdim=True)
    return (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + 1e-5) * w + b


@pytest.mark.parametrize("n,width,p", [(501, 48, 0.25), (64, 33, 0.0), (1, 16, 0.5)])
def test_gradients_match_autograd(cuda, n, width, p):
    head = feature_head.FeatureHead(width, 40, 2, p, cuda, torch.float32, seed=5)
    gen = torch.Generator().manual_seed(n)
    for k, v in head.params.items():  # no weight left at its special value
        v.add_((torch.randn(v.shape, generator=gen) * 0.05).to(cuda))
    x = torch.randn(n, width, generator=gen)
    c = torch.randn(n, 3, generator=gen)
    out = head.forward(x.to(cuda))
    dx = head.backward(c.to(cuda))

    w = {k: v.detach().cpu().double().requires_grad_() for k, v in head.params.items()}
    f = x.double().requires_grad_()
    h, y = f, _norm(f, w["norm0.weight"], w["norm0.bias"])
    for k in range(2):
        r = torch.relu(y @ w[f"block{k}.w1"]) @ w[f"block{k}.w2"]
        keep, scale = keep_mask(r.numel(), p, 5, 1 * 2 + k)
        h = h + r * keep.view(r.shape) * scale
        y = _norm(h, w[f"norm{k + 1}.weight"], w[f"norm{k + 1}.bias"])
    want = y @ w["out"]
    want.backward(c.double())

    def close(got, ref, what):
        err = float((got.detach().cpu().double() - ref).abs().max())
        assert err <= REL * max(1.0, float(ref.abs().max())), f"{what}: {err}"

    close(out, want.detach(), "out")
    close(dx, f.grad, "features")
    for k in head.params:
        close(head.grads[k], w[k].grad, k)


def test_masks_differ_by_step_and_block(cuda):
    head = feature_head.FeatureHead(32, 32, 2, 0.5, cuda, torch.float32)
    x = torch.randn(200, 32, device=cuda)
    a, b = head.forward(x), head.forward(x)
    assert not torch.equal(a, b)
    e = head.forward(x, train=False)
    assert torch.equal(e, head.forward(x, train=False))


def test_fit_lowers_the_loss(cuda):
    losses = feature_head.fit(steps=40)
    assert all(np.isfinite(losses))
    # 0.8 L1 - 0.2 SSIM is -0.2 for equal images
    assert np.mean(losses[-4:]) + 0.2 < 0.6 * (np.mean(losses[:4]) + 0.2)


def test_refuses_other_types(cuda):
    head = feature_head.FeatureHead(16, 16, 1, 0.1, cuda)
    with pytest.raises(AssertionError):
        head.forward(torch.zeros(4, 16, device=cuda))
    with pytest.raises(AssertionError):
        feature_head.FeatureHead(16, 16, 1, 1.5, cuda)


@pytest.mark.parametrize("size", [1e-9, 1e-7, 1.0, 1e5])
def test_f16_gradients_of_any_size(cuda, size):
    """Gradients of a loss over an image are of the order of 1e-7 and less, f16's smallest value is 6e-8.

    Tolerance, on the whole of each gradient (root of the sum of squares): about 14 values in a row are rounded to f16
    (14 * 2^-11 = 0.7 %), and the rounding turns the sign of about 3e-4 of the activations that the relu sees, which
    changes two layers' gradients by the root of that, 1.7 % each: 5 % covers them."""
    n, width, p = 501, 48, 0.25
    head = feature_head.FeatureHead(width, 40, 2, p, cuda, torch.float16, seed=5)
    gen = torch.Generator().manual_seed(n)
    x = torch.randn(n, width, generator=gen).half()
    c = torch.randn(n, 3, generator=gen) * size
    head.forward(x.to(cuda))
    dx = head.backward(c.to(cuda))

    w = {k: v.detach().cpu().double().requires_grad_() for k, v in head.params.items()}
    f = x.double().requires_grad_()
    h, y = f, _norm(f, w["norm0.weight"], w["norm0.bias"])
    for k in range(2):
        r = torch.relu(y @ w[f"block{k}.w1"]) @ w[f"block{k}.w2"]
        keep, scale = keep_mask(r.numel(), p, 5, 1 * 2 + k)
        h = h + r * keep.view(r.shape) * scale
        y = _norm(h, w[f"norm{k + 1}.weight"], w[f"norm{k + 1}.bias"])
    (y @ w["out"]).backward(c.double())
    for name, got, ref in [("features", dx, f.grad)] + [(k, head.grads[k], w[k].grad) for k in head.params]:
        err = float((got.detach().cpu().double() - ref).norm() / ref.norm())
        assert err <= 0.05, f"{name}: {err}"


def test_f16_gradients_of_nothing(cuda):
    head = feature_head.FeatureHead(16, 16, 1, 0.1, cuda, torch.float16)
    for n, value in ((5, 0.0), (0, 0.0)):
        head.forward(torch.ones(n, 16, device=cuda, dtype=torch.float16))
        assert torch.equal(head.backward(torch.full((n, 3), value, device=cuda)), torch.zeros(n, 16, device=cuda))
        assert all(bool((v == 0).all()) for v in head.grads.values())


def test_f16_fit_lowers_the_loss(cuda):
    losses = feature_head.fit(steps=40, dtype=torch.float16)
    assert all(np.isfinite(losses))
    assert np.mean(losses[-4:]) + 0.2 < 0.6 * (np.mean(losses[:4]) + 0.2)


@pytest.mark.parametrize("blocks", [0, 2])
def test_dropped_features(cuda, blocks):
    """Dropout of the features before the first norm, forward and gradient, against autograd; none outside training."""
    n, width, p_in = 301, 40, 0.3
    head = feature_head.FeatureHead(width, 40, blocks, 0.25, cuda, torch.float32, seed=5, p_in=p_in)
    gen = torch.Generator().manual_seed(n)
    x, c = torch.randn(n, width, generator=gen), torch.randn(n, 3, generator=gen)
    # columns of a wider buffer
    out = head.forward(torch.cat((x, x), 1).to(cuda)[:, :width])
    dx = head.backward(c.to(cuda))
    w = {k: v.detach().cpu().double().requires_grad_() for k, v in head.params.items()}
    f = x.double().requires_grad_()
    keep, scale = keep_mask(f.numel(), p_in, 5, 2**63 + 1)
    h = f * keep.view(f.shape) * scale
    y = _norm(h, w["norm0.weight"], w["norm0.bias"])
    for k in range(blocks):
        r = torch.relu(y @ w[f"block{k}.w1"]) @ w[f"block{k}.w2"]
        keep, scale = keep_mask(r.numel(), 0.25, 5, 1 * 2 + k)
        h = h + r * keep.view(r.shape) * scale
        y = _norm(h, w[f"norm{k + 1}.weight"], w[f"norm{k + 1}.bias"])
    want = y @ w["out"]
    want.backward(c.double())
    for what, got, ref in [("out", out, want.detach()), ("features", dx, f.grad)] + \
            [(k, head.grads[k], w[k].grad) for k in head.params]:
        err = float((got.detach().cpu().double() - ref).abs().max())
        assert err <= REL * max(1.0, float(ref.abs().max())), f"{what}: {err}"
    plain = feature_head.FeatureHead(width, 40, blocks, 0.25, cuda, torch.float32, seed=5)
    assert torch.equal(head.forward(x.to(cuda), train=False), plain.forward(x.to(cuda), train=False))


def test_fit_with_dropped_features(cuda):
    losses = feature_head.fit(steps=40, p_in=0.02)
    assert all(np.isfinite(losses))
    assert np.mean(losses[-4:]) + 0.2 < 0.6 * (np.mean(losses[:4]) + 0.2)
