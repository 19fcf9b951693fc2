"""densify_and_prune's screen-size rule after an append: the recorded radii are zeros then, and a bound below zero is exceeded
by a zero, in the one pass as in its two steps."""
import pytest
import torch

from gsplat_host.model import GaussianParams
from gsplat_host.optim import GaussianAdam
from gsplat_host.synthetic import make_cloud


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("screen,left", [(-1.0, False), (1e-9, True), (12.0, True)])
def test_zero_radii_against_the_bound(device, screen, left):
    P = 200
    m = GaussianParams(make_cloud(P, sh_degree=0, seed=3), max_sh_degree=0, device=device)
    m.training_setup(GaussianAdam.for_model(m))
    m.xyz_gradient_accum, m.denom = torch.full((P, 1), 0.001, device=device), torch.ones((P, 1), device=device)
    m.max_radii2D = torch.full((P,), 30.0, device=device)
    m.densify_and_prune(0.0005, 0.0, 1e6, screen, generator=torch.Generator().manual_seed(1))
    assert (m._xyz.shape[0] > 0) == left
