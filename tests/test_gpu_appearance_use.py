"""AppearanceHead as a program calls it: numpy views, several fits."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from msplat_amd.appearance import AppearanceHead  # noqa: E402


@pytest.fixture(scope="module")
def views():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    rng = np.random.default_rng(1)
    renders = [rng.random((20 + i, 30, 3), dtype=np.float32) for i in range(2)]
    return renders, [(0.8 * r).astype(np.float32) for r in renders]


def _parameters(head):
    return [p.detach().clone() for p in head.parameters()]


def test_numpy_views_are_those_of_tensors(views):
    renders, photos = views
    heads = [AppearanceHead(2) for _ in range(2)]
    heads[0].fit(renders, photos, steps=6)
    heads[1].fit([torch.from_numpy(r).cuda() for r in renders], [torch.from_numpy(p).cuda() for p in photos], steps=6)
    assert all(torch.equal(p, q) for p, q in zip(*map(_parameters, heads)))
    with torch.no_grad():
        assert torch.equal(heads[0](renders[0], 1), heads[1](torch.from_numpy(renders[0]).cuda(), 1))


def test_an_optimiser_goes_on_from_fit_to_fit(views):
    renders, photos = views
    whole, parts = AppearanceHead(2), AppearanceHead(2)
    whole.fit(renders, photos, steps=7)
    adam = torch.optim.Adam(parts.parameters(), lr=3e-3)
    for steps in (3, 4):
        parts.fit(renders, photos, steps, optimiser=adam)
    assert all(torch.equal(p, q) for p, q in zip(*map(_parameters, (whole, parts))))
