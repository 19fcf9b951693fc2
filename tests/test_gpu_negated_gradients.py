"""A gradient that is a negated view (what complex arithmetic leaves behind) counts with its sign."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def make(n):
    from gsplat_host.optim import GaussianAdam
    g = torch.Generator().manual_seed(n)
    return GaussianAdam({"opacity": torch.randn(n, 1, generator=g).cuda()}, {"opacity": 0.05})


@pytest.mark.parametrize("n", (1, 5003))
@pytest.mark.parametrize("max_norm", (None, 0.25, math.inf))
def test_a_step_on_a_negated_view(n, max_norm):
    z = torch.randn(n, 1, dtype=torch.complex64, generator=torch.Generator().manual_seed(1)).cuda()
    views = [torch._neg_view(z.real.contiguous()), z.conj().imag]
    for view in views:
        assert view.is_neg()
        a, b = make(n), make(n)
        kw = {} if max_norm is None else {"max_norm": max_norm}
        got = a.step({"opacity": view}, **kw)
        want = b.step({"opacity": view.resolve_neg().contiguous()}, **kw)
        assert (got is None and want is None) or torch.equal(got, want)
        assert torch.equal(a.params["opacity"], b.params["opacity"]) and torch.equal(a.exp_avg["opacity"], b.exp_avg["opacity"])
        assert torch.equal(a.exp_avg_sq["opacity"], b.exp_avg_sq["opacity"])


def test_norm_and_clipping_of_a_negated_view():
    from gsplat_host.optim import clip_grads_, grad_norm
    x = torch.randn(3001, generator=torch.Generator().manual_seed(3)).cuda()
    view, other = torch._neg_view(x.clone()), (-x).clone()
    assert torch.equal(grad_norm(view), grad_norm(other)) and torch.equal(clip_grads_(view, 0.5), clip_grads_(other, 0.5))
    assert torch.equal(view, other) and torch.equal(-view, -other)
