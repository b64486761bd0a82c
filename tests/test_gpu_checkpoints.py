"""Checkpoints in 8 bits against the formulas with packed numbers in their places."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import more_oracle as more  # noqa: E402
import nn_oracle as orc  # noqa: E402
from test_gpu_appearance import _head, views  # noqa: E402,F401
from test_gpu_nn import _normal, nn  # noqa: E402,F401


def _packed(t):
    return more.mx8(t.detach().float().reshape(-1, t.shape[-1]))[0].reshape(t.shape)


class _At(torch.autograd.Function):
    """f(t, *others), with its gradients those at `kept` in t's place."""

    @staticmethod
    def forward(ctx, f, kept, t, *others):
        ctx.f = f
        ctx.save_for_backward(kept, *others)
        return f(t, *others)

    @staticmethod
    def backward(ctx, dy):
        with torch.enable_grad():
            leaves = [t.detach().requires_grad_() for t in ctx.saved_tensors]
            return (None, None, *torch.autograd.grad(ctx.f(*leaves), leaves, dy))


class _Norm(torch.autograd.Function):
    """t rstd w, with the gradients' t packed and the forward's rstd."""

    @staticmethod
    def forward(ctx, t, w):
        rstd = (t.square().mean(1, keepdim=True) + 1e-5).rsqrt()
        ctx.save_for_backward(_packed(t), w, rstd)
        return t * rstd * w

    @staticmethod
    def backward(ctx, dy):
        t, w, rstd = ctx.saved_tensors
        n, g = t * rstd, dy * w
        return rstd * (g - n * (g * n).mean(1, keepdim=True)), (dy * n).sum(0)


def _formula(head, rgb, photo, leaves):
    """The head with root-mean-square norms in 64 bits: the five numbers of a pixel are
    kept as they are, all else packed."""
    embed, codes, nw, out = leaves[:4]
    h, w = rgb.shape[:2]
    u = torch.linspace(-1, 1, w).double().expand(h, w)
    v = torch.linspace(-1, 1, h).double()[:, None].expand(h, w)
    x = torch.cat((rgb, torch.stack((u, v), 2)), 2).reshape(-1, 5) @ embed.t() + codes[photo]
    for i in range(len(head.blocks)):
        w_, wg, wu, wd = leaves[4 + 4 * i:8 + 4 * i]
        n = _Norm.apply(x, w_)
        f = _At.apply(lambda t, *ws: orc.gated_ffn(t, *ws, "silu"), _packed(n), n, wg, wu, wd)
        if head.dropout > 0:
            f = torch.where(orc.keep_mask(x.shape[0], x.shape[1], head.dropout, i, head.step), f / (1 - head.dropout), 0.0)
        x = x + f
    n = _Norm.apply(x, nw)
    return rgb + _At.apply(lambda t, o: t @ o.t(), _packed(n), n, out).reshape(h, w, 3)


@pytest.mark.parametrize("dropout", [0.0, 0.05])
def test_a_heads_gradients_are_those_at_the_packed_numbers(views, dropout):
    """In float32 a kept number is off by a few hundred roundings of 2^-24, 6e-5 of itself at
    most, so that 2 * 6e-5 * 16 = 2e-3 of them at most fall on another side of the
    middle between two numbers in 8 bits, which lie 1/16 to 1/8 of themselves apart: in
    the mean square 1/8 sqrt(2e-3) = 0.0056 of a gradient at each of six packed places,
    0.014 in all.  A scale or a term that is wrong is off by far more."""
    renders, photos = views
    head = _head(dtype=torch.float32, norm="rms", checkpoint="mx8", dropout=dropout)
    head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
    y = head(renders[1], 1, training=True)
    got = torch.autograd.grad((y - photos[1]).square().mean(), head.parameters())
    leaves = [p.detach().double().cpu().requires_grad_() for p in head.parameters()]
    want = torch.autograd.grad((_formula(head, renders[1].double().cpu(), 1, leaves) - photos[1].double().cpu()).square().mean(),
                               leaves)
    for i, (g, v) in enumerate(zip(got, want)):
        error = float((g.double().cpu() - v).norm()) / float(v.norm())
        print(f"parameter {i}: {error:.2e}")
        assert error <= 0.014, i


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_a_heads_gradients_are_a_few_percent_off(views, dtype, norm):
    """Against those without checkpoints, at the same forward: a kept number is off by half a
    step of 1/8 of its power of two at most, 1/8 / sqrt(12) = 0.036 of it in the mean
    square, and errors of different pixels are independent: with seven places that are
    kept sqrt(7) 0.036 = 0.095 of a gradient."""
    renders, photos = views
    grads = []
    for checkpoint in (None, "mx8"):
        head = _head(dtype=dtype, norm=norm, checkpoint=checkpoint)
        head.out.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1), std=0.1)
        loss = (head(renders[1], 1, training=True) - photos[1]).square().mean()
        grads.append(torch.autograd.grad(loss, head.parameters()))
    for i, (a, b) in enumerate(zip(*grads)):
        error = float((a - b).norm()) / float(a.norm())
        print(f"parameter {i}: {error:.3f}")
        assert error <= 0.095, i


def test_replays_see_new_inputs(nn):
    """A captured norm, its packed sum and its backward: inputs that differ from each other and
    from replay to replay."""
    x, r, dy = (_normal(s, 300, 100, dtype=torch.bfloat16) for s in (16, 17, 18))
    w = 1 + _normal(19, 100, dtype=torch.bfloat16, scale=0.1)

    def step():
        y, total, rstd = nn.rms_norm_forward(x, w, r)
        m, _, _ = nn.rms_norm_forward(total, w, mx8=True)
        return (y, total, rstd, nn.mx8_unpack(m), *nn.rms_norm_backward(dy, nn.mx8_pack(total), w, rstd, y))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (20, 21, 22):
        for i, t in enumerate((x, r, dy)):
            t.copy_(_normal(seed + 10 * i, 300, 100, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(p, q) for p, q in zip(got, step()))
