"""AppearanceHead with root-mean-square norms and linear layers: the operators in a
run, as a training program and a viewer use them."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import nn_oracle as orc  # noqa: E402
from test_gpu_appearance import _head, views  # noqa: E402,F401


def _plain(head, rgb, photo, leaves, training):
    """The head's formula in 64 bits."""
    embed, codes, nw, out = leaves[:4]
    h, w = rgb.shape[:2]
    u = torch.linspace(-1, 1, w).double().expand(h, w)
    v = torch.linspace(-1, 1, h).double()[:, None].expand(h, w)
    x = torch.cat((rgb, torch.stack((u, v), 2)), 2).reshape(-1, 5) @ embed.t() + codes[photo]

    def norm(x, w):
        return x * (x.square().mean(1, keepdim=True) + 1e-5).rsqrt() * w

    for i in range(len(head.blocks)):
        w_, wg, wu, wd = leaves[4 + 4 * i:8 + 4 * i]
        f = orc.gated_ffn(norm(x, w_), wg, wu, wd, "silu")
        if training:
            f = torch.where(orc.keep_mask(x.shape[0], x.shape[1], head.dropout, i, head.step), f / (1 - head.dropout), 0.0)
        x = x + f
    return rgb + (norm(x, nw) @ out.t()).reshape(h, w, 3)


@pytest.mark.parametrize("dropout", [0.0, 0.05])
def test_gradients_match_plain_operations(views, dropout):
    """As test_gpu_appearance's: a chain of two blocks in float32, sums over 17920
    pixels; its relative error is that of a few hundred roundings."""
    renders, photos = views
    head = _head(dtype=torch.float32, norm="rms", dropout=dropout)
    assert torch.equal(head(renders[0], 0), renders[0])   # starts as the identity
    head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
    got_y = head(renders[1], 1, training=True)
    got = torch.autograd.grad((got_y - photos[1]).square().mean(), head.parameters())
    leaves = [p.detach().double().cpu().requires_grad_() for p in head.parameters()]
    rgb, photo = renders[1].double().cpu(), photos[1].double().cpu()
    y = _plain(head, rgb, 1, leaves, dropout > 0)
    assert float((got_y.detach().double().cpu() - y.detach()).norm()) <= 1000 * orc.U * float(y.detach().norm())
    want = torch.autograd.grad((y - photo).square().mean(), leaves)
    for g, v in zip(got, want):
        assert float((g.double().cpu() - v).norm()) <= 1000 * orc.U * float(v.norm()) + 1e-30


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_checkpoints_in_8_bits(views, dtype, norm):
    """The forward is the same; a gradient is off by the checkpoints' rounding, at
    most 1/16 of each kept number at every one of seven places, in bfloat16 by that
    type's as well: less than half of itself in the mean square."""
    renders, photos = views
    outputs, grads = [], []
    for checkpoint in (None, "mx8"):
        head = _head(dtype=dtype, norm=norm, checkpoint=checkpoint)
        head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
        y = head(renders[1], 1, training=True)
        outputs.append(y.detach())
        grads.append(torch.autograd.grad((y - photos[1]).square().mean(), head.parameters()))
    assert torch.equal(*outputs)
    for a, b in zip(*grads):
        assert torch.isfinite(b).all() and float((a - b).norm()) <= 0.5 * float(a.norm())


def test_training_runs_and_repeats(views):
    renders, photos = views
    runs = []
    for _ in range(2):
        head = _head(norm="rms", checkpoint="mx8")
        losses = head.fit(renders, photos, steps=6)
        assert len(losses) == 6 and all(v == v for v in losses)
        runs.append([p.detach().clone() for p in head.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_viewer_in_float16_and_refusals(views):
    renders, _ = views
    head = _head(norm="rms")
    head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
    with torch.no_grad():
        y = head(renders[0], 2)
        head.dtype = torch.float16
        half = head(renders[0], 2)
    assert float((y - half).abs().max()) < 0.1   # bfloat16's own error
    with pytest.raises(ValueError, match="norm"):
        _head(norm="batch")
    with pytest.raises(ValueError, match="checkpoint"):
        _head(checkpoint="int4")


def test_norm_product_and_gradients_in_a_row(views):
    """A norm writes 8 bits, a product takes them with weights in 8 bits, and a training
    step's backward takes what the forward kept: each result as if by itself."""
    from msplat_amd import nn
    import more_oracle as more
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(3000, 96, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = (torch.randn(160, 96, generator=g, device="cuda") / 96 ** 0.5).bfloat16()
    n, total, rstd = nn.rms_norm_forward(x, None, r, mx8=True)
    y = nn.linear_forward(n, nn.mx8_pack(w), None, None, "gelu")
    values = nn.mx8_unpack(n, torch.float32), nn.mx8_unpack(nn.mx8_pack(w), torch.float32)
    want, _, bound, _ = more.linear(*values, None, None, "gelu", torch.bfloat16)
    more.near(y, want, bound, "y")
    kept = nn.linear_forward(nn.mx8_unpack(n), w, activation="gelu", keep=True)[1]
    dn, dw, _ = nn.linear_backward(y, n, w, nn.mx8_pack(kept), "gelu")
    (want_dn, want_dw, _), (e_dn, e_dw, _) = more.linear_grad(y, nn.mx8_unpack(n), w, nn.mx8_unpack(nn.mx8_pack(kept), torch.float32),
                                                             "gelu", torch.bfloat16)
    more.near(dn, want_dn, e_dn, "dn")
    more.near(dw, want_dw, e_dw, "dw")
    dx, _ = nn.rms_norm_backward(dn, nn.mx8_pack(total), None, rstd, x)
    (want_dx, _), (e_dx, _) = more.rms_norm_grad(dn, nn.mx8_unpack(nn.mx8_pack(total), torch.float32),
                                                 torch.ones(96, dtype=torch.bfloat16, device="cuda"), rstd, x)
    more.near(dx.cpu(), want_dx, e_dx, "dx")
