"""Norm and clipping of a GradArena's gradients: only its tensors count, whatever has happened to the padding between them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPES = {"xyz": (333, 3), "opacity": (333, 1), "f_rest": (333, 0, 3), "rotation": (335, 1)}      # each but one needs padding


def make(seed):
    from gsplat_host.optim import GradArena
    params = {k: torch.zeros(s, device="cuda") for k, s in SHAPES.items()}
    arena = GradArena(params)
    g = torch.Generator().manual_seed(seed)
    fill(arena, g)
    return arena, params


def fill(arena, g):
    for v in arena.views.values():
        v.copy_(torch.randn(v.shape, generator=g))


def norm64(arena, p=2.0):
    flat = torch.cat([v.double().reshape(-1) for v in arena.views.values()]).abs()
    return float(flat.max() if p == math.inf else flat.sum() if p == 1.0 else flat.square().sum().sqrt())


@pytest.mark.parametrize("bad", (math.nan, math.inf, -math.inf))
@pytest.mark.parametrize("p", (2.0, 1.0, math.inf))
def test_a_step_that_is_not_finite_is_forgotten(bad, p):
    """Clipping by a NaN norm makes every gradient NaN; zero_grad clears the gradients, and the next norm is theirs alone."""
    from gsplat_host.optim import GaussianAdam
    arena, params = make(1)
    opt = GaussianAdam(params, dict.fromkeys(params, 0.1))
    arena.attach(opt.params)
    arena.views["xyz"][17, 1] = bad
    norm = float(arena.clip_(1.0, p))
    assert math.isnan(norm) if math.isnan(bad) else norm == math.inf
    opt.zero_grad(set_to_none=False)
    assert float(arena.norm(p)) == 0.0
    fill(arena, torch.Generator().manual_seed(2))
    before = {k: v.clone() for k, v in arena.views.items()}
    want = norm64(arena, p)
    for got in (arena.norm(p), arena.clip_(0.5 * want, p)):
        assert abs(float(got) - want) <= 2.0 ** -23 * want
    factor = 0.5 * want / (want + 1e-6)
    for k, v in arena.views.items():
        assert bool(((v.double() - before[k].double() * factor).abs() <= 2.5 * 2.0 ** -24 * before[k].double().abs()).all()), k


def test_the_padding_is_left_as_it_is():
    arena, _ = make(3)
    inside = torch.zeros_like(arena.flat, dtype=torch.bool)
    for k, o in arena.offsets.items():
        inside[o:o + math.prod(SHAPES[k])] = True
    arena.flat[~inside] = 5.0
    want = norm64(arena)
    assert abs(float(arena.norm()) - want) <= 2.0 ** -23 * want
    assert abs(float(arena.clip_(0.1)) - want) <= 2.0 ** -23 * want
    assert bool((arena.flat[~inside] == 5.0).all())
