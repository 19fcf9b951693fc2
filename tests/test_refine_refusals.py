"""A refine that is refused on the CPU leaves parameters and moments as they were, as it does on the GPU."""
import pytest
import torch

from gsplat_host.optim import GaussianAdam

SHAPES = {"xyz": (40, 3), "f_rest": (40, 0, 3), "opacity": (40, 1)}


def test_nothing_is_appended_by_a_refused_call():
    opt = GaussianAdam({k: torch.randn(*s) for k, s in SHAPES.items()}, dict.fromkeys(SHAPES, 0.1))
    held = [dict(d) for d in (opt.params, opt.exp_avg, opt.exp_avg_sq)]
    good = {k: torch.zeros(4, *s[1:]) for k, s in SHAPES.items()}
    keep = torch.ones(44, dtype=torch.bool)
    for k, e in [(keep[:43], good), (keep[:40], good), (keep, None), (keep, {**good, "opacity": torch.zeros(5, 1)}),
                 (keep, {**good, "xyz": torch.zeros(4, 2)}), (keep.view(1, -1), good), (keep.float(), good)]:
        with pytest.raises((ValueError, TypeError)):
            opt.refine(k, e)
        assert all(a[n] is b[n] for a, b in zip(held, (opt.params, opt.exp_avg, opt.exp_avg_sq)) for n in SHAPES)
    opt.refine(keep, good)
    assert opt.params["xyz"].shape[0] == 44


def test_rows_on_another_device_are_refused_first():
    opt = GaussianAdam({k: torch.randn(*s) for k, s in SHAPES.items()}, dict.fromkeys(SHAPES, 0.1))
    held = [dict(d) for d in (opt.params, opt.exp_avg, opt.exp_avg_sq)]
    born = {k: torch.zeros(4, *s[1:], device="meta" if k == "opacity" else "cpu") for k, s in SHAPES.items()}
    with pytest.raises(ValueError, match="on meta"):
        opt.refine(torch.ones(44, dtype=torch.bool), born)
    assert all(a[n] is b[n] for a, b in zip(held, (opt.params, opt.exp_avg, opt.exp_avg_sq)) for n in SHAPES)
