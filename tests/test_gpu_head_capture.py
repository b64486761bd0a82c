"""A training step of the head's operators through autograd, captured into a graph and
replayed with the program's own work in between."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from test_gpu_nn import _normal, nn  # noqa: E402,F401


@pytest.mark.parametrize("checkpoint", [None, "mx8"])
def test_a_captured_training_step(nn, checkpoint):
    rows = 700
    x0 = _normal(1, rows, 5)
    target = _normal(2, rows, 3)
    shapes = [(32, 5), (32,), (32,), (128, 32), (128, 32), (32, 128), (32,), (3, 32)]
    leaves = [_normal(10 + i, *s, scale=s[-1] ** -0.5).requires_grad_() for i, s in enumerate(shapes)]

    def step():
        embed, code, w0, wg, wu, wd, w1, out = (t if i < 2 else t.bfloat16() for i, t in enumerate(leaves))
        x = nn.linear(x0, embed, code, None, "silu", torch.bfloat16, checkpoint)
        f = nn.gated_ffn(nn.rms_norm(x, w0, checkpoint=checkpoint), wg, wu, wd, "gelu", checkpoint)
        n, _ = nn.rms_norm(f, w1, x, checkpoint=checkpoint)
        y = nn.linear(n, out, None, x0[:, :3], out_dtype=torch.float32, checkpoint=checkpoint)
        return [y.detach(), *torch.autograd.grad(y, leaves, y - target)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(4):
        x0.copy_(_normal(80 + k, rows, 5))
        target.copy_(_normal(90 + k, rows, 3))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(p, q) for p, q in zip(got, step())), k
        with torch.no_grad():   # an optimiser's step between the replays
            for t, g in zip(leaves, got[1:]):
                t.sub_(g, alpha=1e-4)
