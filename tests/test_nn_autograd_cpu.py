"""What the differentiable operators of msplat_amd.nn do around their kernels,
without a GPU: plain operations on the CPU stand in for the passes."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from msplat_amd import nn


def _linear_forward(x, weight, bias=None, residual=None, activation=None, out_dtype=None, keep=False):
    z = x @ weight.t()
    z = z if bias is None else z + bias
    y = z if activation is None else torch.nn.functional.silu(z)
    y = (y if residual is None else y + residual.view(y.shape)).to(out_dtype or x.dtype)
    return (y, z) if keep else y


def _rms_norm_forward(x, weight=None, residual=None, eps=1e-5, mx8=False):
    total = x if residual is None else x + residual.view(x.shape)
    rstd = (total.square().mean(-1) + eps).rsqrt()
    y = total * rstd[..., None]
    return y if weight is None else y * weight, total, rstd


def _mx8_pack(x):
    return nn.Mx8._empty(x.shape, x, x.dtype)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(nn, "mx8_pack", _mx8_pack)
    monkeypatch.setattr(nn, "gated_ffn_forward", lambda x, *_: x.clone())
    monkeypatch.setattr(nn, "linear_forward", _linear_forward)
    monkeypatch.setattr(nn, "rms_norm_forward", _rms_norm_forward)


@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_is_refused(plain, grad):
    """No operator has a forward-mode derivative: with a tangent each is an error, with
    and without gradients, and never a result whose tangent is lost."""
    w = torch.ones(4, 4)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        x = forward_ad.make_dual(torch.ones(3, 4), torch.ones(3, 4))
        for call in (lambda: nn.linear(x, w), lambda: nn.linear(w, w, x[0]), lambda: nn.rms_norm(x),
                     lambda: nn.rms_norm(w[:3], None, x)):
            with pytest.raises(NotImplementedError):
                call()


class _NoGradient(torch.autograd.Function):
    @staticmethod
    def forward(ctx, t):
        return t.clone()

    @staticmethod
    def backward(ctx, dy):
        return None


def test_a_norm_that_no_gradient_reaches(plain):
    """Whatever follows may have no gradient for either result: then no input has one."""
    x, r, w = (torch.ones(*s, requires_grad=True) for s in ((3, 4), (3, 4), (4,)))
    y, total = nn.rms_norm(x, w, r)
    grads = torch.autograd.grad((_NoGradient.apply(y) + _NoGradient.apply(total)).sum(), (x, w, r), allow_unused=True)
    assert grads == (None, None, None)
    y = nn.rms_norm(x, w)
    assert torch.autograd.grad(_NoGradient.apply(y).sum(), (x, w), allow_unused=True) == (None, None)


def _kept(call):
    """The tensors that an operator keeps for its backward, and its result."""
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        y = call()
    return kept, y


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_checkpoints_are_never_larger_than_what_they_stand_for(plain, dtype):
    """A row in 8 bits has whole blocks of 32 columns and scales for 128: narrow
    matrices, and some a little wider than a block, are smaller as they are."""
    for dim in (1, 3, 5, 8, 9, 16, 17, 18, 19, 32, 33, 34, 35, 64, 129, 132, 200):
        x = torch.ones(7, dim, dtype=dtype, requires_grad=True)
        w = torch.ones(dim, dim, dtype=dtype, requires_grad=True)
        for call in (lambda c: nn.linear(x, w, activation="silu", checkpoint=c), lambda c: nn.rms_norm(x, checkpoint=c),
                     lambda c: nn.gated_ffn(x, w, w, w, checkpoint=c)):
            size = [sum(t.nbytes for t in _kept(lambda: call(c))[0]) for c in (None, "mx8")]
            packed, plain_size = 32 * -(-dim // 32) + 4 * -(-dim // 128), dim * x.element_size()
            assert size[1] <= size[0]
            assert (size[1] < size[0]) is (packed < plain_size)


def _ids(tensors):
    return {t.data_ptr() for t in tensors if t is not None}


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_only_what_wanted_gradients_take_is_kept(plain, monkeypatch, checkpoint):
    """A frozen weight leaves x out, no activation z, and without any operand that
    requires a gradient nothing is kept, packed or written for one."""
    packed, kept_z = [], []
    monkeypatch.setattr(nn, "mx8_pack", lambda t: packed.append(t) or _mx8_pack(t))
    monkeypatch.setattr(nn, "linear_forward",
                        lambda *a: kept_z.append(len(a) > 6 and a[6]) or _linear_forward(*a))
    x, w, b, r = torch.ones(7, 64), torch.ones(64, 64), torch.ones(64), torch.ones(7, 64)

    def leaf(t, needs):
        return t.clone().requires_grad_(needs)

    for needs in range(16):
        for act in (None, "silu"):
            ops = [leaf(t, bool(needs >> i & 1)) for i, t in enumerate((x, w, b, r))]
            packed.clear(), kept_z.clear()
            kept, y = _kept(lambda: nn.linear(*ops, act, checkpoint=checkpoint))
            takes_x, takes_z = bool(needs & 2), act is not None and bool(needs & 7)
            assert y.requires_grad is bool(needs) and kept_z == [takes_z]
            assert len(packed) == (takes_x + takes_z if checkpoint else 0)
            assert (ops[0].data_ptr() in _ids(kept + packed)) is takes_x
            assert bool(kept) is bool(needs & 7)
    for needs in range(8):
        ops = [leaf(t, bool(needs >> i & 1)) for i, t in enumerate((x, b, r))]
        packed.clear()
        kept, _ = _kept(lambda: nn.rms_norm(*ops, checkpoint=checkpoint))
        assert len(packed) == (1 if checkpoint and needs else 0) and bool(kept) is bool(needs)
        ops = [leaf(t, bool(needs >> i & 1)) for i, t in enumerate((x, w, w))]
        packed.clear()
        kept, _ = _kept(lambda: nn.gated_ffn(*ops, w, checkpoint=checkpoint))
        assert len(packed) == (1 if checkpoint and needs else 0) and bool(kept) is bool(needs)
    packed.clear()
    with torch.no_grad():
        x.requires_grad_(), w.requires_grad_()
        for call in (lambda: nn.linear(x, w, None, None, "silu", None, checkpoint), lambda: nn.rms_norm(x, checkpoint=checkpoint),
                     lambda: nn.gated_ffn(x, w, w, w, checkpoint=checkpoint)):
            assert not _kept(call)[0] and not packed


def test_the_backward_is_asked_for_what_is_wanted(plain, monkeypatch):
    asked = []
    monkeypatch.setattr(nn, "linear_backward", lambda dy, x, w, z, act, wanted: asked.append((x is None, tuple(wanted))) or
                        tuple(t if k else None for t, k in zip((dy @ w, torch.zeros_like(w), dy.sum(0)), wanted)))
    for needs in range(1, 8):
        ops = [t.clone().requires_grad_(bool(needs >> i & 1))
               for i, t in enumerate((torch.ones(7, 64), torch.ones(64, 64), torch.ones(64)))]
        nn.linear(*ops, None, "silu").sum().backward()
        wanted = tuple(bool(needs >> i & 1) for i in range(3))
        assert asked.pop() == (not wanted[1], wanted) and not asked
        assert tuple(t.grad is not None for t in ops) == wanted


def _rms_norm_backward(dy, total, weight, rstd, dtotal=None, wanted=(True, True)):
    dx = dy * 3.0 if dtotal is None else dy * 3.0 + dtotal
    return dx if wanted[0] else None, None


@pytest.mark.parametrize("shape", [(3, 4), (1, 3, 4)])
def test_gradients_share_no_memory(plain, monkeypatch, shape):
    """The gradients of leaves are theirs alone: neither another's nor the one that the
    caller gave backward, so that a second backward pass adds to each once."""
    monkeypatch.setattr(nn, "linear_backward", lambda dy, x, w, z, act, wanted: (dy @ w if wanted[0] else None, None, None))
    monkeypatch.setattr(nn, "rms_norm_backward", _rms_norm_backward)

    def leaves():
        return torch.ones(3, 4, requires_grad=True), torch.ones(shape, requires_grad=True)

    def check(call, want):
        x, r = leaves()
        given = torch.ones(3, 4)
        for times in (1, 2, 3):
            call(x, r).backward(given)
            assert (given == 1).all()
            for t, g in zip((x, r), want):
                assert t.grad is None if g is None else (t.grad == times * g).all(), (times, t.grad, g)
        grads = {t.grad.data_ptr() for t in (x, r, given) if t.grad is not None}
        assert given.data_ptr() not in grads and len(grads) == sum(g is not None for g in want)

    w = torch.eye(4)
    check(lambda x, r: nn.linear(x, w, None, r), (1, 1))
    check(lambda x, r: nn.linear(w[:3], w, None, r), (None, 1))
    check(lambda x, r: nn.rms_norm(x, None, r)[0], (3, 3))
    check(lambda x, r: nn.rms_norm(x, None, r)[1], (1, 1))
    check(lambda x, r: nn.rms_norm(w[:3], None, r)[1], (None, 1))
    check(lambda x, r: sum(nn.rms_norm(x, None, r)), (4, 4))


def test_rows_in_8_bits_are_refused_by_name(monkeypatch):
    """Where a tensor is taken, an Mx8 is a ValueError that says so."""
    monkeypatch.setattr(nn, "_library", lambda t: None)
    x = torch.zeros(4, 8)
    m = nn.Mx8._empty(x.shape, x, x.dtype)
    for call in (lambda: nn.mx8_pack(m), lambda: nn.rms_norm(m), lambda: nn.rms_norm_backward(m, x, None, x[0]),
                 lambda: nn.linear_backward(x, x, m), lambda: nn.linear_backward(m, x, x), lambda: nn.layer_norm(m),
                 lambda: nn.gated_ffn(m, x, x, x), lambda: nn.dropout_add(m, None, 0.5, 1, 2),
                 lambda: nn.rms_norm(x, None, m), lambda: nn.rms_norm(x, m), lambda: nn.linear(x, x, None, m),
                 lambda: nn.linear(x, x, m)):
        with pytest.raises(ValueError, match="Mx8"):
            call()


def test_dropouts_residual_of_another_shape(monkeypatch):
    """As many rows in other axes, which the forward pass takes: its gradient has its shape."""
    monkeypatch.setattr(nn, "dropout_add_forward", lambda x, r, p, seed, offset: x + r.view(x.shape))
    x, given = torch.ones(2, 3, 4), torch.ones(2, 3, 4)
    r = torch.ones(6, 4, requires_grad=True)
    for times in (1, 2):
        nn.dropout_add(x, r, 0.5, 1, 2).backward(given)
        assert r.grad.shape == r.shape and (r.grad == times).all() and (given == 1).all()
