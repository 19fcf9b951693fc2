"""GaussianAdam.refine on the CPU: appending and pruning in one call leaves what the two calls leave, and nothing else.
(On the GPU the rows are moved by kernels: test_gpu_rows.py.)"""
import pytest
import torch

from gsplat_host.optim import GaussianAdam

SHAPES = {"xyz": (40, 3), "f_rest": (40, 0, 3), "opacity": (40, 1)}


def make():
    g = torch.Generator().manual_seed(2)
    opt = GaussianAdam({k: torch.randn(*s, generator=g) for k, s in SHAPES.items()}, dict.fromkeys(SHAPES, 0.1))
    for k, s in SHAPES.items():
        opt.exp_avg[k], opt.exp_avg_sq[k] = torch.randn(*s, generator=g), torch.rand(*s, generator=g)
    opt.step_count = 9
    return opt


@pytest.mark.parametrize("extra", (None, 0, 7))
def test_refine_is_append_and_prune(extra):
    a, b = make(), make()
    g = torch.Generator().manual_seed(3)
    born = None if extra is None else {k: torch.randn(extra, *s[1:], generator=g) for k, s in SHAPES.items()}
    keep = torch.rand(40 + (extra or 0), generator=g) < 0.6
    if born is not None:
        b.cat_tensors(born)
    b.prune(keep)
    out = a.refine(keep, born)
    assert a.step_count == 9
    for k in SHAPES:
        assert out[k] is a.params[k] and out[k].is_leaf and out[k].requires_grad and out[k].shape[0] == int(keep.sum())
        assert torch.equal(a.params[k], b.params[k]) and torch.equal(a.exp_avg[k], b.exp_avg[k])
        assert torch.equal(a.exp_avg_sq[k], b.exp_avg_sq[k])


def test_refine_asks_for_every_tensor():
    with pytest.raises(ValueError, match="name every tensor"):
        make().refine(torch.ones(41, dtype=torch.bool), {"xyz": torch.zeros(1, 3)})
