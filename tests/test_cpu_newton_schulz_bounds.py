"""The bounds of the Newton-Schulz GPU tests refuse what they must: zeros, a step too few, missing rows and columns, coarser products."""
import pytest
import torch
from newton_schulz_bounds import FAST, allowed, distances, emulated, exact, matrix, within

SHAPES = [(16, 16), (33, 65), (40, 24), (128, 1024), (1024, 128), (64, 2048), (70, 4097), (200, 600), (300, 200)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind,steps", [("rank", 1), ("rank", 2), ("low", 2), ("noise", 5), ("low", 5), ("rank", 5)])
def test_bounds_bind(shape, kind, steps):
    u = matrix(shape, kind)
    co = (FAST,) * steps
    want, bounds = allowed(u, co)
    assert bounds[0] <= 5e-3                                       # what five steps of right kernels were measured at: 1e-3 to 2e-3
    good = emulated(u, co)
    assert within(good, want, bounds) and within(want, want, bounds)
    assert not within(emulated(u, co, dtype=torch.bfloat16), want, bounds)
    assert not within(torch.zeros_like(want), want, bounds)
    assert not within(good * 1.01, want, bounds)
    assert not within(torch.full_like(want, float("nan")), want, bounds)
    if steps > 1:
        assert not within(exact(u, co[1:]), want, bounds)
    for cut in (lambda t: t[-1].zero_(), lambda t: t[:, -1].zero_(), lambda t: t[0].zero_(), lambda t: t[:, 0].zero_()):
        bad = good.clone()
        cut(bad)
        assert not within(bad, want, bounds)
    # a product left out, in one step only
    left_out = exact(u, co[:-1] + ((FAST[0], FAST[1], 0.0),))
    assert not within(left_out, want, bounds)


def test_distances():
    want = torch.ones(4, 9, dtype=torch.float64)
    got = want.clone()
    got[2, 3] += 0.5
    assert distances(got, want) == pytest.approx((0.5 / 6, 0.5 * 2 / 6, 0.5 * 3 / 6))
