"""GradArena.norm / clip_ with the factor that an averaging exchange leaves for the step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = {"xyz": (1001, 3), "opacity": (1001, 1), "rotation": (1001, 4)}
U = 2.0 ** -24


def make(seed):
    from gsplat_host.optim import GradArena
    params = {k: torch.zeros(s, device="cuda") for k, s in SHAPES.items()}
    arena = GradArena(params)
    g = torch.Generator().manual_seed(seed)
    for v in arena.views.values():
        v.copy_(torch.randn(v.shape, generator=g))
    return arena


def norm64(arena, p):
    flat = torch.cat([v.double().reshape(-1) for v in arena.views.values()]).abs()
    return float(flat.max() if p == math.inf else flat.sum() if p == 1.0 else flat.square().sum().sqrt())


@pytest.mark.parametrize("world", (1, 2, 3, 8))
@pytest.mark.parametrize("p", (2.0, 1.0, math.inf))
def test_the_mean_is_bounded_not_the_sum(world, p):
    """``flat`` holds a sum over ranks, the step applies 1 / world: it is the product of both whose norm is bounded.
    Norm: its own rounding, the factor's and the product's.  Elements: the bound's quotient and the factor are rounded too."""
    arena = make(world)
    scale = 1.0 / world
    before = {k: v.double() for k, v in arena.views.items()}
    mean = norm64(arena, p) * scale
    got = float(arena.norm(p, grad_scale=scale))
    assert abs(got - mean) <= 4 * U * mean
    bound = 0.4 * mean
    assert abs(float(arena.clip_(bound, p, grad_scale=scale)) - mean) <= 4 * U * mean
    # min(1, max_norm / (grad_scale (norm + 1e-6))); the gradients stay sums
    factor = bound / (scale * (mean / scale + 1e-6))
    for k, v in arena.views.items():
        assert bool(((v.double() - before[k] * factor).abs() <= 5 * U * before[k].abs()).all()), k
    assert abs(norm64(arena, p) * scale - bound) <= 1e-5 * bound
    within = {k: v.clone() for k, v in arena.views.items()}
    arena.clip_(2.0 * bound, p, grad_scale=scale)
    assert all(torch.equal(within[k], v) for k, v in arena.views.items())
    arena.clip_(math.inf, p, grad_scale=scale)
    assert all(torch.equal(within[k], v) for k, v in arena.views.items())


def test_clipping_and_step_agree_with_the_clipped_step():
    """Eight ranks' sum, clipped in the arena and stepped with 1 / 8, against the step that does both.  The 1e-6 of the rule
    stands beside the sum's norm in the one and the mean's in the other: 7e-6 over a sum's norm of 89, 8e-8; the two
    factors' own roundings make 4 U of it.  First moments are 0.1 g from zero: the same relative difference and three more
    roundings."""
    from gsplat_host.optim import GaussianAdam
    arena = make(5)
    norm = norm64(arena, 2.0)
    assert 80.0 < norm < 100.0
    a, b = (GaussianAdam({k: torch.zeros(s, device="cuda") for k, s in SHAPES.items()}, dict.fromkeys(SHAPES, 0.1)) for _ in range(2))
    a.step(arena.views, grad_scale=0.125, max_norm=1.0)
    arena.clip_(1.0, grad_scale=0.125)
    b.step(arena.views, grad_scale=0.125)
    for k in SHAPES:
        x, y = a.exp_avg[k].double(), b.exp_avg[k].double()
        assert bool(((x - y).abs() <= (9e-8 + 10 * U) * x.abs()).all()), k


def test_factors_that_are_refused():
    arena = make(2)
    before = arena.flat.clone()
    for bad in (0.0, -0.5, math.nan, math.inf):
        with pytest.raises(ValueError, match="grad_scale"):
            arena.norm(grad_scale=bad)
        with pytest.raises(ValueError, match="grad_scale"):
            arena.clip_(1.0, grad_scale=bad)
    assert torch.equal(arena.flat, before)
