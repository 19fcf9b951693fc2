"""Clipping of 16-bit gradients, bit for bit: the factor is torch's in its last bit too.

A bf16 significand has 128 values, an fp16 one 1024, so a factor like 0.37 puts whole classes of elements on rounding ties
(175 * 0.37 = 64.75): one last bit of the factor moves all elements of such a class the same way.  The rule is
``max_norm / (norm + 1e-6)`` as torch evaluates it on a float32 norm, the product in float32, one rounding to the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = (torch.bfloat16, torch.float16)
FACTORS = (0.37, 0.3, 0.25 + 2.0 ** -9)


def every_significand(dtype, seed):
    """Each significand in eight binades with both signs, and random elements behind them."""
    bits = 7 if dtype == torch.bfloat16 else 10
    one = 1.0 + torch.arange(2 ** bits, dtype=torch.float32) / 2 ** bits
    grid = (one[:, None] * 2.0 ** torch.arange(-3, 5)).reshape(-1)
    rest = torch.randn(20_011, generator=torch.Generator().manual_seed(seed)) * 3.0
    return torch.cat((grid, -grid, rest)).to(dtype).cuda()


def torchs_factor(norm, bound):
    return (bound / (norm + 1e-6)).clamp(max=1.0)


def by_torch(before, bound, norm):
    """clip_grads_with_norm_ on float32 copies, rounded once."""
    params = []
    for g in before:
        p = torch.nn.Parameter(torch.zeros_like(g, dtype=torch.float32))
        p.grad = g.float()
        params.append(p)
    torch.nn.utils.clip_grads_with_norm_(params, bound, norm)
    return [p.grad.to(g.dtype) for p, g in zip(params, before)]


def bits(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("factor", FACTORS)
@pytest.mark.parametrize("p", (2.0, 1.0, math.inf))
def test_the_factor_is_torchs(dtype, factor, p):
    from gsplat_host.optim import clip_grads_, grad_norm
    for k in range(40):
        source = every_significand(dtype, k) * (1.0 + k / 64)         # another norm each time
        grads = [source.clone(), source[:501].clone()]
        before = [g.clone() for g in grads]
        bound = float(grad_norm(grads, p)) * factor
        norm = clip_grads_(grads, bound, p)
        c = torchs_factor(norm, bound)
        for got, b, t in zip(grads, before, by_torch(before, bound, norm)):
            assert torch.equal(bits(got), bits((b.float() * c).to(dtype))), k
            assert torch.equal(bits(got), bits(t)), k


@pytest.mark.parametrize("dtype", HALVES)
def test_passes_in_a_row(dtype):
    """What the second pass measures is what the first one wrote: both norms and all elements stay torch's."""
    from gsplat_host.optim import clip_grads_
    for k in range(20):
        grads = [every_significand(dtype, 100 + k), every_significand(dtype, 200 + k)[:777]]
        plain = [g.clone() for g in grads]
        bound = None
        for _ in range(3):
            flat = torch.cat([g.double() for g in plain])
            norm = flat.square().sum().sqrt().float()
            bound = float(norm) * 0.37 if bound is None else bound * 0.9999
            c = torchs_factor(norm, bound)
            plain = [(g.float() * c).to(dtype) for g in plain]
            assert torch.equal(clip_grads_(grads, bound), norm)
            for a, b in zip(grads, plain):
                assert torch.equal(bits(a), bits(b)), k


def test_mixed_lists_and_strides():
    """16-bit tensors among float32 ones, back to back in a buffer, and one with gaps."""
    from gsplat_host.optim import clip_grads_, grad_norm
    for k in range(40):
        pool = every_significand(torch.bfloat16, k)
        halves = [pool[1:900], pool[900:4001], every_significand(torch.float16, k).view(-1)[::2]]
        full = torch.randn(5000, generator=torch.Generator().manual_seed(k)).cuda()
        before = [t.clone() for t in halves + [full]]
        bound = float(grad_norm(halves + [full])) * FACTORS[k % 3]
        norm = clip_grads_([halves[0], full] + halves[1:], bound)
        c = torchs_factor(norm, bound)
        for got, b in zip(halves, before):
            assert torch.equal(bits(got.contiguous()), bits((b.float() * c).to(b.dtype))), k
        # float32 elements: the factor rounded once from 64 bits, and the product
        want = before[3].double() * (bound / (math.sqrt(sum(float(b.double().square().sum()) for b in before)) + 1e-6))
        assert bool(((full.double() - want).abs() <= 2.5 * 2.0 ** -24 * want.abs()).all())


def test_where_the_float32_norm_ends():
    """Norms up to the largest float32 by torch's rule (its reciprocal is a subnormal number there), beyond it from 64 bits."""
    from gsplat_host.optim import clip_grads_, grad_norm
    source = every_significand(torch.bfloat16, 3)
    for scale in (2.0 ** 118, 2.0 ** 117, 2.0 ** -120):
        grads = (source.float() * scale).to(torch.bfloat16)
        norm = grad_norm(grads)
        assert math.isfinite(float(norm))
        for bound in (1.0, 2.0 ** 100, float(norm) * 0.37):
            got = grads.clone()
            clip_grads_(got, bound)
            assert torch.equal(bits(got), bits((grads.float() * torchs_factor(norm, bound)).to(torch.bfloat16))), (scale, bound)
    huge = torch.full((1000,), 3e38, dtype=torch.bfloat16, device="cuda")
    before = huge.double()
    assert float(clip_grads_(huge, 1e38)) == math.inf
    norm = float(before.square().sum().sqrt())
    want = before * (1e38 / norm)                            # 3.2e36: the element's own rounding, factor and product
    assert bool(((huge.double() - want).abs() <= want * (2.0 ** -8 + 3 * 2.0 ** -24)).all())


@pytest.mark.parametrize("dtype", HALVES)
def test_within_the_bound_nothing_changes(dtype):
    from gsplat_host.optim import clip_grads_, grad_norm
    g = every_significand(dtype, 9)
    before, norm = g.clone(), float(grad_norm(g))
    for bound in (norm * (1 + 1e-6) + 2e-6, 1e39, math.inf):
        clip_grads_(g, bound)
        assert torch.equal(bits(g), bits(before))
