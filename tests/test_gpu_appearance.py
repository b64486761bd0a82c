"""AppearanceHead on rendered views: the layer norm, gated feed-forward and
dropout operators together, forward and backward, as a training program runs
them."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from helpers import BG, small_scene  # noqa: E402
from msplat_amd import camera, device  # noqa: E402


@pytest.fixture(scope="module")
def views():
    """Three views of a small scene and photos of them: each with a gain a
    channel, a gamma and a vignette of its own."""
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    scene = small_scene(n=4000, width=160, height=112)
    g = device.DeviceGaussians.from_arrays(scene.params(), scene.sh_degree)
    renders, photos = [], []
    for i in range(3):
        cam = camera.pinhole(160, 112, 70.0, camera.look_at([5.0 - i, 1.0 + i, 2.0]))
        r = device.render(g, camera.prepare_cam(cam), scene.sh_degree, BG).clamp(0, 1)
        gain = torch.tensor([[0.7, 0.9, 1.1], [1.2, 1.0, 0.8], [0.9, 0.6, 0.9]][i], device="cuda")
        u = torch.linspace(-1, 1, 160, device="cuda")
        photos.append((r ** (0.8 + 0.2 * i)) * gain * (1 - 0.2 * u.square())[:, None])
        renders.append(r)
    device.sync()
    return renders, photos


def _head(**kw):
    from msplat_amd.appearance import AppearanceHead
    return AppearanceHead(3, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_head_learns_the_photos_colours(views, dtype):
    renders, photos = views
    head = _head(dtype=dtype)
    assert torch.equal(head(renders[0], 0), renders[0])   # starts as the identity
    losses = head.fit(renders, photos, steps=240)
    start, end = sum(losses[:3]), sum(losses[-3:])
    assert end < start / 5, (start, end)
    # each photo's code is its own: another code's colours are further off
    def off(render, photo, code):
        return float((head(renders[render], code) - photos[photo]).abs().mean())
    for i in range(3):
        assert off(i, i, i) < 0.5 * off(i, i, (i + 1) % 3)


def test_training_repeats_bit_for_bit(views):
    renders, photos = views
    runs = []
    for _ in range(2):
        head = _head()
        head.fit(renders, photos, steps=12)
        runs.append([p.detach().clone() for p in head.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_gradients_match_plain_operations(views):
    """One training step's gradients in float32 against the same step in
    float64 with plain operations: a chain of two blocks, sums over 17920
    pixels; its relative error is that of a few hundred roundings."""
    import nn_oracle as orc
    renders, photos = views
    head = _head(dtype=torch.float32)
    head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
    loss = (head(renders[1], 1, training=True) - photos[1]).square().mean()
    got = torch.autograd.grad(loss, head.parameters())
    leaves = [p.detach().double().cpu().requires_grad_() for p in head.parameters()]
    embed, codes, nw, nb, out = leaves[:5]
    rgb, photo = renders[1].double().cpu(), photos[1].double().cpu()
    u = torch.linspace(-1, 1, 160).double().expand(112, 160)
    v = torch.linspace(-1, 1, 112).double()[:, None].expand(112, 160)
    x = torch.cat((rgb, torch.stack((u, v), 2)), 2).reshape(-1, 5) @ embed.t() + codes[1]

    def norm(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return d * (d.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w + b

    for i in range(2):
        w, b, wg, wu, wd = leaves[5 + 5 * i:10 + 5 * i]
        keep = orc.keep_mask(x.shape[0], x.shape[1], 0.05, i, 0)
        x = x + torch.where(keep, orc.gated_ffn(norm(x, w, b), wg, wu, wd, "silu") / 0.95, 0.0)
    want = torch.autograd.grad(((rgb + (norm(x, nw, nb) @ out.t()).reshape(112, 160, 3) - photo).square().mean()), leaves)
    for g, v in zip(got, want):
        assert float((g.double().cpu() - v).norm()) <= 1000 * orc.U * float(v.norm()) + 1e-30


def test_refusals(views):
    renders, photos = views
    with pytest.raises(ValueError, match="num_photos"):
        _head(blocks=0)
    head = _head()
    with pytest.raises(ValueError, match="shape"):
        head(renders[0][..., :2], 0)
    with pytest.raises(ValueError, match="photos"):
        head.fit(renders, photos[:2], steps=1)
