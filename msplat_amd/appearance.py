"""AppearanceHead: per-photo colour correction of rendered views.

Photos of one scene differ in exposure, white balance and vignetting, which a
scene of gaussians cannot represent.  The head learns a code for each photo and
a small network over the pixels of a rendered view that turns the view's
colours into the photo's:

    x = E [rgb, u, v] + code[photo]
    x = x + dropout(ffn(norm(x)))        for each block
    rgb' = rgb + O norm(x)

with the layer norm, gated feed-forward and dropout operators of
msplat_amd.nn.  With norm="rms" the norms are root-mean-square norms, which take
the residual's addition along where nothing is dropped, and the products with E and O
are linear layers of msplat_amd.nn too, so that no pass over the pixels is torch's but
the assembly of [rgb, u, v].  It has no counterpart in the reference.

    head = AppearanceHead(len(photos))
    head.fit(renders, photos, steps=500)     # e.g. renders of GaussianTrainer's cameras
    with torch.no_grad():
        corrected = head(render, photo=3)

Views are (H, W, 3) float32, numpy arrays (as GaussianTrainer.render gives them)
or tensors.  The head is fitted to finished renders: the scene's own training
does not see it.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import nn


class AppearanceHead:
    """dim features a pixel, `blocks` blocks of `hidden` units.  Parameters and
    their optimiser are float32; features and products have the type `dtype`.
    norm: "layer", or "rms" (see above).  checkpoint "mx8" keeps what the backward of
    feed-forward blocks, rms norms and linear layers takes of every pixel in 8 bits (the
    five numbers of the pixel itself as they are), about half of bfloat16's memory for
    gradients less than one percent off (sums over a view's pixels: 0.1 to 0.6%).

    float16 is for correcting views with a head trained in another type
    (head.dtype = torch.float16): a pixel's share of a view's mean loss is
    below its smallest numbers, and scaled up for them the sums over a view's
    pixels pass its largest, so training in it is refused."""

    def __init__(self, num_photos: int, dim: int = 32, hidden: int = 128, blocks: int = 2, dropout: float = 0.05,
                 activation: str = "silu", dtype=torch.bfloat16, seed: int = 0, device: str = "cuda",
                 norm: str = "layer", checkpoint: Optional[str] = None):
        if num_photos < 1 or blocks < 1:
            raise ValueError("num_photos and blocks must be at least 1")
        if norm not in ("layer", "rms"):
            raise ValueError(f"norm {norm!r} is neither 'layer' nor 'rms'")
        if checkpoint not in (None, "mx8"):
            raise ValueError(f"checkpoint {checkpoint!r} is neither None nor 'mx8'")
        self.norm, self.checkpoint = norm, checkpoint
        self.dropout, self.activation, self.dtype, self.seed = dropout, activation, dtype, seed
        self.step = 0
        g = torch.Generator().manual_seed(seed)

        def param(*shape, scale):
            return (scale * torch.randn(shape, generator=g)).to(device).requires_grad_()

        self.embed = param(dim, 5, scale=5 ** -0.5)
        self.codes = param(num_photos, dim, scale=0.1)
        self.blocks = []
        for _ in range(blocks):
            norms = dict(weight=torch.ones(dim, device=device, requires_grad=True))
            if norm == "layer":
                norms["bias"] = torch.zeros(dim, device=device, requires_grad=True)
            self.blocks.append(dict(norms, w_gate=param(hidden, dim, scale=dim ** -0.5),
                                    w_up=param(hidden, dim, scale=dim ** -0.5),
                                    w_down=param(dim, hidden, scale=hidden ** -0.5)))
        self.norm_weight = torch.ones(dim, device=device, requires_grad=True)
        self.norm_bias = torch.zeros(dim, device=device, requires_grad=True) if norm == "layer" else None
        self.out = torch.zeros(3, dim, device=device, requires_grad=True)   # starts as the identity

    def parameters(self) -> List[torch.Tensor]:
        norm = [self.norm_weight] if self.norm_bias is None else [self.norm_weight, self.norm_bias]
        return [self.embed, self.codes, *norm, self.out, *(p for b in self.blocks for p in b.values())]

    def __call__(self, rgb, photo: int, training: bool = False):
        """The (H, W, 3) float32 view in the colours of photo number `photo`, a
        tensor on the head's GPU; differentiable, so without torch.no_grad() it
        keeps what its gradient takes of every pixel."""
        if training and self.dtype is torch.float16:
            raise ValueError("a head is trained in bfloat16 or float32, not float16")
        rgb = self._view(rgb)
        if rgb.dim() != 3 or rgb.shape[2] != 3:
            raise ValueError(f"rgb has shape {tuple(rgb.shape)}, not (H, W, 3)")
        h, w = rgb.shape[:2]
        u = torch.linspace(-1.0, 1.0, w, device=rgb.device).expand(h, w)
        v = torch.linspace(-1.0, 1.0, h, device=rgb.device)[:, None].expand(h, w)
        pixels = torch.cat((rgb, torch.stack((u, v), 2)), 2).reshape(h * w, 5)
        p = self.dropout if training else 0.0
        if self.norm == "rms":
            return self._rms(rgb, pixels, photo, p)
        x = (pixels @ self.embed.t() + self.codes[photo]).to(self.dtype)
        for i, b in enumerate(self.blocks):
            q = {k: t.to(self.dtype) for k, t in b.items()}
            n = nn.layer_norm(x, q["weight"], q["bias"])
            f = nn.gated_ffn(n, q["w_gate"], q["w_up"], q["w_down"], self.activation, self.checkpoint)
            x = nn.dropout_add(f, x, p, seed=(self.seed << 8) + i, offset=self.step)
        n = nn.layer_norm(x, self.norm_weight.to(self.dtype), self.norm_bias.to(self.dtype))
        return rgb + (n.float() @ self.out.t()).reshape(h, w, 3)

    def _rms(self, rgb, pixels, photo, p):
        keep = self.checkpoint
        x = nn.linear(pixels, self.embed, self.codes[photo], out_dtype=self.dtype, checkpoint=keep)
        f = None   # what the last block adds to x
        for i, b in enumerate([*self.blocks, dict(weight=self.norm_weight)]):
            q = {k: t.to(self.dtype) for k, t in b.items()}
            if f is not None and p > 0.0:
                x = nn.dropout_add(f, x, p, seed=(self.seed << 8) + i - 1, offset=self.step)
                f = None
            if f is None:
                n = nn.rms_norm(x, q["weight"], checkpoint=keep)
            else:
                n, x = nn.rms_norm(f, q["weight"], x, checkpoint=keep)
            if "w_gate" in q:
                f = nn.gated_ffn(n, q["w_gate"], q["w_up"], q["w_down"], self.activation, keep)
        h, w = rgb.shape[:2]
        y = nn.linear(n, self.out.to(self.dtype), residual=rgb.reshape(h * w, 3), out_dtype=torch.float32,
                      checkpoint=keep)
        return y.reshape(h, w, 3)

    def _view(self, view):
        return torch.as_tensor(view, dtype=torch.float32, device=self.embed.device)

    def fit(self, renders: Sequence, photos: Sequence, steps: int,
            lr: float = 3e-3, optimiser: Optional[torch.optim.Optimizer] = None) -> List[float]:
        """`steps` steps of the L1 loss between corrected renders and photos,
        cycling through them (a later call goes on where this one stops); the
        loss of every step.  Without `optimiser` a call starts a new Adam: give
        one over parameters() to keep its moments from call to call."""
        if len(renders) != len(photos) or not renders:
            raise ValueError("as many photos as renders are needed, and at least one")
        renders, photos = [self._view(t).detach() for t in renders], [self._view(t) for t in photos]
        optimiser = optimiser or torch.optim.Adam(self.parameters(), lr=lr)
        losses = []
        for _ in range(steps):
            i = self.step % len(renders)
            loss = (self(renders[i], i, training=True) - photos[i]).abs().mean()
            optimiser.zero_grad(set_to_none=True)
            loss.backward()
            optimiser.step()
            self.step += 1
            losses.append(loss.detach())
        return torch.stack(losses).tolist() if losses else []
