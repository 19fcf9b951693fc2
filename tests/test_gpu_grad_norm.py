"""Gradient norm over many tensors, clipping, and the Adam step that clips, against the formulas in 64 bits.

Tolerances, u = 2^-24 (half a unit in fp32's last place, relative):
* norm: the sums are in 64 bits (n 2^-53 relative, below 2^-25 for the sizes here), rounded once to fp32: u + 2^-25.
* clipped gradients: the factor is rounded to fp32 (u), the product is (u), and the result to its own type (half its
  epsilon, and half its smallest subnormal absolutely): 2.5 u + eps / 2.  A factor below 2^-126 (gradients 10^38 times
  their bound) is a subnormal number, whose rounding is off by up to 2^-150 absolutely and not by u of it: |g| 2^-150 on
  top (2e-40 is 1.5e5 steps of 2^-149, so up to 3.3e-6 of it).
* step: see test_clipped_step_against_64_bits.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = (torch.float32, torch.float16, torch.bfloat16)
NORMS = (2.0, 1.0, math.inf)
CHUNK = 32768                                     # bytes a workgroup takes at a time


def norm64(tensors, p):
    flat = [t.detach().double().reshape(-1) for t in tensors if t.numel()]
    if not flat:
        return 0.0
    flat = torch.cat(flat).abs()
    return float(flat.max() if p == math.inf else flat.sum() if p == 1.0 else flat.square().sum().sqrt())


def factor64(norm, bound):
    return min(1.0, bound / (norm + 1e-6))


def values(n, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))
    return (t * (1.0 if dtype == torch.float16 else 1e-3)).to(dtype).cuda()


def check_norm(got, tensors, p):
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    want = norm64(tensors, p)
    assert abs(float(got) - want) <= (U + 2.0 ** -25) * want, (float(got), want)


def check_clipped(got, before, factor):
    if not before.numel():
        return
    want = before.double() * factor
    info = torch.finfo(before.dtype)
    allowed = want.abs() * (2.5 * U + info.eps / 2) + info.smallest_normal * info.eps / 2 + before.double().abs() * 2.0 ** -150
    over = (got.double() - want).abs() - allowed
    assert float(over.max()) <= 0.0, float(over.max())


def shifted(t, offset, guard=37):
    """A copy of the 1-D ``t`` that starts ``offset`` elements behind a 256-byte boundary, inside a guarded buffer."""
    buf = torch.full((t.numel() + offset + guard,), 7.0, dtype=t.dtype, device="cuda")
    view = buf[offset:offset + t.numel()]
    view.copy_(t)
    return buf, view


SIZES = (0, 1, 2, 3, 7, 8, 9, 63, 64, 65, 1000, 4095, CHUNK // 4 - 1, CHUNK // 4, CHUNK // 4 + 1, CHUNK // 2 + 3, 100_003)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", (0, 1, 3, 5))
def test_sizes_and_alignments(dtype, offset):
    from gsplat_host.optim import clip_grads_, grad_norm
    for i, n in enumerate(SIZES):
        for p in NORMS:
            buf, g = shifted(values(n, dtype, i), offset)
            before = g.clone()
            check_norm(grad_norm(g, p), [before], p)
            bound = 0.3 * norm64([before], p)
            check_norm(clip_grads_([g], bound, p), [before], p)
            check_clipped(g, before, factor64(norm64([before], p), bound))
            assert bool((buf[:offset] == 7).all()) and bool((buf[offset + n:] == 7).all()), (n, offset, p)


@pytest.mark.parametrize("count", (1, 6, 119, 120, 121, 250, 601))
@pytest.mark.parametrize("p", NORMS)
def test_lists_of_unlike_tensors(count, p):
    """Types mixed, empty tensors and None among them, carved back to back out of one buffer of each type."""
    from gsplat_host.optim import clip_grads_, grad_norm
    rng = np.random.default_rng(count)
    sizes = [int(10 ** rng.uniform(0, 4.3)) if rng.random() > 0.1 else 0 for _ in range(count)]
    pools = {t: values(sum(sizes), t, count + k) for k, t in enumerate(TYPES)}
    at, tensors = dict.fromkeys(TYPES, 0), []
    for k, n in enumerate(sizes):
        t = TYPES[(k * 7 + count) % 3]
        tensors.append(pools[t][at[t]:at[t] + n])
        at[t] += n
    before = [t.clone() for t in tensors]
    rest = {t: pools[t][at[t]:].clone() for t in TYPES}
    check_norm(grad_norm(tensors, p), before, p)
    check_norm(grad_norm({str(k): t for k, t in enumerate(tensors)} | {"none": None}, p), before, p)
    bound = 0.01 * norm64(before, p)
    check_norm(clip_grads_([None] + tensors, bound, p), before, p)
    for got, b in zip(tensors, before):
        check_clipped(got, b, factor64(norm64(before, p), bound))
    for t in TYPES:
        assert torch.equal(pools[t][at[t]:], rest[t])


@pytest.mark.parametrize("p", NORMS)
def test_within_the_bound_nothing_changes(p):
    from gsplat_host.optim import clip_grads_
    for dtype in TYPES:
        g = values(50_001, dtype, 4)
        before = g.clone()
        n = norm64([g], p)
        for bound in (n * 1.01 + 2e-6, math.inf):
            check_norm(clip_grads_(g, bound, p), [before], p)
            assert torch.equal(g, before)


def test_a_zero_bound_gives_zeros_and_zero_gradients_stay():
    from gsplat_host.optim import clip_grads_, grad_norm
    g = values(10_000, torch.float32, 1)
    clip_grads_(g, 0.0)
    assert float(g.abs().max()) == 0.0
    for p in NORMS:
        assert float(grad_norm(g, p)) == 0.0 and float(clip_grads_(g, 1.0, p)) == 0.0 and float(g.abs().max()) == 0.0
        empty = torch.empty((0, 3), device="cuda")
        assert float(grad_norm([empty], p)) == 0.0 and float(clip_grads_([empty, empty], 1.0, p)) == 0.0


def test_strides_and_orders():
    from gsplat_host.optim import clip_grads_, grad_norm
    base = values(24 * 35 * 11, torch.float32, 3).reshape(24, 35, 11)
    makers = (lambda b: b.permute(2, 0, 1), lambda b: b[:, 3:30], lambda b: b[..., ::2], lambda b: b[:, :, 4],
              lambda b: b.transpose(0, 1)[1:], lambda b: b[5], lambda b: b[::3, ::5, ::7])
    for make in makers:
        for p in NORMS:
            whole = base.clone()
            mark = torch.zeros_like(whole)
            make(mark).fill_(1.0)
            t = make(whole)
            before, all_before = t.clone(), whole.clone()
            check_norm(grad_norm([t], p), [before], p)
            bound = 0.5 * norm64([before], p)
            clip_grads_([t], bound, p)
            check_clipped(t, before, factor64(norm64([before], p), bound))
            assert torch.equal(whole[mark == 0], all_before[mark == 0])          # what lies between the elements
    expanded = values(50, torch.float32, 9).reshape(50, 1).expand(50, 20)
    check_norm(grad_norm(expanded), [expanded.contiguous()], 2.0)                 # read as its elements are seen ...
    with pytest.raises(ValueError, match="may share memory"):
        clip_grads_(expanded, 1.0)                                                # ... but not written
    twice = values(500, torch.float32, 2)
    check_norm(grad_norm([twice, twice]), [twice, twice], 2.0)
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grads_([twice, twice[10:20]], 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite(dtype):
    from gsplat_host.optim import clip_grads_, grad_norm
    for at in (0, 1, 4097, 20_000, 29_998):
        for bad in (math.nan, math.inf, -math.inf):
            for p in NORMS:
                g = values(29_999, dtype, 5)
                g[at] = bad
                other = values(77, torch.float32, 6)
                got = float(grad_norm([other, g], p))
                assert math.isnan(got) if math.isnan(bad) else got == math.inf
                kept = g.clone()
                assert torch.equal(torch.isnan(clip_grads_([g], math.inf, p)), torch.tensor(math.isnan(bad), device="cuda"))
                assert torch.equal(g.nan_to_num(1.5, 2.5, 3.5), kept.nan_to_num(1.5, 2.5, 3.5))
                clip_grads_([other, g], 1.0, p)
                if math.isnan(bad):
                    assert bool(g.isnan().all()) and bool(other.isnan().all())
                else:
                    assert bool(g[at].isnan()) and int((g != 0).sum()) == 1 and float(other.abs().max()) == 0.0
    two = torch.tensor([math.inf, math.nan, math.inf, -math.inf], device="cuda", dtype=dtype)
    assert all(math.isnan(float(grad_norm(two.roll(k), p))) for p in NORMS for k in range(4))


def test_the_whole_range_of_fp32():
    from gsplat_host.optim import clip_grads_, grad_norm
    huge = torch.full((1000,), 3e38, device="cuda")
    assert float(grad_norm(huge)) == math.inf and abs(float(grad_norm(huge, math.inf)) / 3e38 - 1) < 1e-6
    before = huge.clone()
    clip_grads_(huge, 2.0)                                  # the fp32 norm overflows, the factor does not
    check_clipped(huge, before, factor64(norm64([before], 2.0), 2.0))
    tiny = torch.full((1000,), 1e-42, device="cuda")        # subnormal: the squares vanish in 32 bits
    for p in NORMS:
        want = norm64([tiny], p)
        assert abs(float(grad_norm(tiny, p)) - want) <= (U + 2.0 ** -25) * want + 2.0 ** -150
    big_h = torch.full((4097,), 65504.0, device="cuda", dtype=torch.float16)
    check_norm(grad_norm(big_h), [big_h], 2.0)


def test_equal_calls_give_equal_bits():
    from gsplat_host.optim import grad_norm
    tensors = [values(n, t, k) for k, (n, t) in enumerate([(2_000_003, torch.float32), (11, torch.float16), (777_777, torch.bfloat16)])]
    for p in NORMS:
        first = grad_norm(tensors, p)
        assert all(torch.equal(first, grad_norm(tensors, p)) for _ in range(5))


def test_past_32_bits():
    """2^31 + 101 elements, 4.3 GB: the elements that count lie at both ends."""
    from gsplat_host.optim import clip_grads_
    n = 2 ** 31 + 101
    g = torch.zeros(n, dtype=torch.float16, device="cuda")
    g[0], g[2 ** 31 - 1], g[2 ** 31], g[n - 1] = 3.0, 4.0, 12.0, 84.0
    assert float(clip_grads_(g, 42.5)) == 85.0
    c = factor64(85.0, 42.5)
    for at, x in ((0, 3.0), (2 ** 31 - 1, 4.0), (2 ** 31, 12.0), (n - 1, 84.0)):
        assert abs(float(g[at]) - x * c) <= x * c * (2.0 ** -11 + 3 * U)
    assert int(torch.count_nonzero(g)) == 4


def test_another_stream_and_replayed_graphs():
    """Calls on a side stream; two graphs that share the pool of captured memory, replayed with other work between."""
    from gsplat_host.optim import clip_grads_, grad_norm
    a, b = values(300_001, torch.float32, 1), values(50_000, torch.bfloat16, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        n = grad_norm([a, b])
    torch.cuda.current_stream().wait_stream(side)
    check_norm(n, [a, b], 2.0)
    side.synchronize()
    source = [t.clone() for t in (a, b)]
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        n1 = clip_grads_([a], 0.5)
    with torch.cuda.graph(g2, pool=g1.pool()):
        n2 = clip_grads_([b, a], 0.25, 1.0)
    for k in range(4):
        a.copy_(source[0] * (k + 1))
        b.copy_(source[1])
        start_a, start_b = a.clone(), b.clone()
        g1.replay()
        torch.cuda.synchronize()
        check_norm(n1, [start_a], 2.0)
        check_clipped(a, start_a, factor64(norm64([start_a], 2.0), 0.5))
        mid = a.clone()
        grad_norm([mid, b], math.inf)                                   # eager work in between
        g2.replay()
        torch.cuda.synchronize()
        check_norm(n2, [mid, start_b], 1.0)
        c = factor64(norm64([mid, start_b], 1.0), 0.25)
        check_clipped(a, mid, c)
        check_clipped(b, start_b, c)


def test_autograd_sees_the_write():
    from gsplat_host.optim import clip_grads_
    x = torch.ones(1000, device="cuda", requires_grad=True)
    y = x * 2.0
    z = (y * y).sum()                                                   # saves y
    clip_grads_(y.detach(), 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()


# ---- the step ----------------------------------------------------------------------------------------------------

SHAPES = {"xyz": (5003, 3), "f_dc": (5003, 1, 3), "f_rest": (5003, 15, 3), "opacity": (5003, 1), "scaling": (5003, 3),
          "rotation": (5003, 4)}
LRS = {"xyz": 0.00016, "f_dc": 0.0025, "f_rest": 0.0025 / 20.0, "opacity": 0.05, "scaling": 0.005, "rotation": 0.001}


def make(seed, shapes=SHAPES, moments=True):
    from gsplat_host.optim import GaussianAdam
    g = torch.Generator().manual_seed(seed)
    opt = GaussianAdam({k: torch.randn(*s, generator=g).cuda() for k, s in shapes.items()}, {k: LRS[k] for k in shapes})
    if moments:
        for k, s in shapes.items():
            opt.exp_avg[k] = (torch.randn(*s, generator=g) * 1e-3).cuda()
            opt.exp_avg_sq[k] = (torch.rand(*s, generator=g) * 1e-5).cuda()
        opt.step_count = 41
    return opt


def state_of(opt):
    return {k: (opt.params[k].clone(), opt.exp_avg[k].clone(), opt.exp_avg_sq[k].clone()) for k in opt.params}


def same(a, b):
    return all(torch.equal(x, y) for k in a for x, y in zip(a[k], b[k]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", NORMS)
@pytest.mark.parametrize("grad_scale", (1.0, 0.125))
def test_clipped_step_is_the_step_on_the_clipped_gradient(dtype, p, grad_scale):
    """Bit for bit: the unclipped step with the factor in its grad_scale, the gradient converted first."""
    grads = {k: values(math.prod(s), dtype, j).view(s) for j, (k, s) in enumerate(SHAPES.items())}
    full = {k: g.float() for k, g in grads.items()}
    n = norm64(grads.values(), p) * grad_scale
    for bound in (0.2 * n, 1.5 * n, math.inf, 0.0):
        a, b = make(3), make(3)
        c = np.float32(factor64(n, bound))
        b.step(full, grad_scale=float(np.float32(grad_scale) * c))
        got = a.step(grads, grad_scale, max_norm=bound, norm_type=p)
        assert abs(float(got) - n) <= (U + 2.0 ** -25) * n
        assert same(state_of(a), state_of(b)) and a.step_count == 42
    kept = {k: values(math.prod(s), dtype, j).view(s) for j, (k, s) in enumerate(SHAPES.items())}
    assert all(torch.equal(kept[k], grads[k]) for k in grads)                    # the gradients are only read


def test_clipped_step_against_64_bits():
    """g' = g s: s and the product rounded (2 u).  m + w (g' - m): three roundings and w's own, each of at most |m| + |g'|
    (6 u of that with g's 2).  v: relative, all terms positive: 2 x 2 u (g') + 3 u (w, two products) + u (sum) = 8 u.
    p - step m / (sqrt(v) c + eps): step, c, the division, the product: 7 u of the update with v's 4 u, m's error through
    the quotient, and u of p."""
    opt = make(8)
    grads = {k: values(math.prod(s), torch.float32, j).view(s) for j, (k, s) in enumerate(SHAPES.items())}
    n = norm64(grads.values(), 2.0)
    s = factor64(n, 0.3 * n)
    before = state_of(opt)
    opt.step(grads, max_norm=0.3 * n)
    t = opt.step_count
    for k in SHAPES:
        p0, m0, v0 = (x.double() for x in before[k])
        g = grads[k].double() * s
        m, v = 0.9 * m0 + (1 - 0.9) * g, 0.999 * v0 + (1 - 0.999) * g * g
        denom = (v / (1 - 0.999 ** t)).sqrt() + 1e-15
        rate = LRS[k] / (1 - 0.9 ** t)
        m_err = 6 * U * (m0.abs() + g.abs())
        assert bool(((opt.exp_avg[k].double() - m).abs() <= m_err).all()), k
        assert bool(((opt.exp_avg_sq[k].double() - v).abs() <= 8 * U * v + 1e-44).all()), k
        p_err = 1.5 * U * (p0.abs() + rate * (m / denom).abs()) + rate * (m_err + 12 * U * m.abs()) / denom
        assert bool(((opt.params[k].double() - (p0 - rate * m / denom)).abs() <= p_err).all()), k


def test_small_and_odd_sizes_and_missing_gradients():
    for n in (1, 2, 3, 5, 1023, 3079, 6151):
        shapes = {"xyz": (n, 3), "f_rest": (n, 0, 3), "opacity": (n, 1)}
        for offset in (0, 1):
            a, b = make(n, shapes), make(n, shapes)
            flat = values(4 * n + offset, torch.bfloat16, n)[offset:]
            grads = {"xyz": flat[:3 * n].view(n, 3), "f_rest": torch.empty((n, 0, 3), device="cuda"), "opacity": flat[3 * n:].view(n, 1)}
            norm = norm64(grads.values(), 2.0)
            got = a.step(grads, max_norm=0.5 * norm)
            b.step({k: g.float() for k, g in grads.items()}, grad_scale=float(np.float32(factor64(norm, 0.5 * norm))))
            assert same(state_of(a), state_of(b)) and abs(float(got) - norm) <= 2 * U * norm
    opt = make(1)
    before = state_of(opt)
    assert float(opt.step({k: None for k in SHAPES}, max_norm=1.0)) == 0.0 and same(state_of(opt), before)
    only = {k: None for k in SHAPES} | {"opacity": values(5003, torch.float32, 3).view(5003, 1)}
    opt.step(only, max_norm=1e-3)
    after = state_of(opt)
    assert not torch.equal(after["opacity"][0], before["opacity"][0])
    assert all(torch.equal(after[k][0], before[k][0]) for k in SHAPES if k != "opacity")
    with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
        opt.step({k: torch.zeros(s, dtype=torch.float64, device="cuda") for k, s in SHAPES.items()}, max_norm=1.0)
    with pytest.raises(ValueError, match="elements"):
        opt.step({k: torch.zeros(3, device="cuda") for k in SHAPES}, max_norm=1.0)


@pytest.mark.parametrize("bad", (math.nan, math.inf))
def test_a_step_that_is_not_finite(bad):
    grads = {k: values(math.prod(s), torch.float32, j).view(s) for j, (k, s) in enumerate(SHAPES.items())}
    grads["opacity"][77] = bad
    opt = make(5)
    before = state_of(opt)
    norm = opt.step(grads, max_norm=1.0, skip_nonfinite=True)
    assert not math.isfinite(float(norm)) and same(state_of(opt), before) and opt.step_count == 42
    opt.step(grads, max_norm=1.0)
    assert bool(opt.params["opacity"][77].isnan())
    huge = {k: torch.full(s, 3e38, device="cuda") for k, s in SHAPES.items()}      # finite, though the fp32 norm is not
    opt = make(5)
    assert float(opt.step(huge, max_norm=1.0, skip_nonfinite=True)) == math.inf
    assert all(bool(torch.isfinite(p).all()) for p in opt.params.values()) and not same(state_of(opt), before)


def test_a_captured_step():
    grads = {k: values(math.prod(s), torch.float32, j).view(s) for j, (k, s) in enumerate(SHAPES.items())}
    source = {k: g.clone() for k, g in grads.items()}
    a, b = make(2), make(2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = a.step(grads, max_norm=0.1)
    for k in range(4):                                                  # the captured step keeps its count: so does b's
        for name in grads:
            grads[name].copy_(source[name] * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        b.step_count = 41
        want = b.step(grads, max_norm=0.1)
        assert torch.equal(norm, want) and same(state_of(a), state_of(b)), k


def test_training_with_clipping_end_to_end():
    """render -> loss -> arena -> norm, clip or clipped step: the three ways give the same parameters."""
    from gsplat_host.cameras import orbit_camera
    from gsplat_host.loss import photometric_loss
    from gsplat_host.model import GaussianParams
    from gsplat_host.optim import GaussianAdam, GradArena, grad_norm
    from gsplat_host.render import PipelineParams, render
    from gsplat_host.synthetic import make_cloud
    dev = torch.device("cuda")
    cam, bg = orbit_camera(160, 96, device=dev), torch.zeros(3, device=dev)
    gt = torch.rand(3, 96, 160, generator=torch.Generator().manual_seed(2)).to(dev)
    model = GaussianParams(make_cloud(3000, sh_degree=3, seed=4), device=dev)
    opt = GaussianAdam.for_model(model)
    arena = GradArena(opt.params)
    arena.attach(opt.params)
    photometric_loss(render(cam, model, PipelineParams(fused_activations=True), bg)["render"], gt).backward()
    grads = [p.grad for p in opt.params.values()]
    norm = norm64(grads, 2.0)
    assert norm > 0 and abs(float(arena.norm()) - norm) <= 2 * U * norm and abs(float(grad_norm(grads)) - norm) <= 2 * U * norm
    clone = {k: p.detach().clone() for k, p in opt.params.items()}
    other = GaussianAdam(clone, dict(opt.lrs))
    got = other.step({k: p.grad for k, p in opt.params.items()}, max_norm=norm / 7)
    clipped = arena.clip_(norm / 7)
    assert abs(float(got) - norm) <= 2 * U * norm and abs(float(clipped) - norm) <= 2 * U * norm
    opt.step()
    for k in clone:
        # the same factor on the same gradients, once inside the step: the same bits
        assert torch.equal(clone[k], opt.params[k].detach()) and torch.equal(other.exp_avg[k], opt.exp_avg[k])
    assert float(arena.norm()) <= norm / 7 * (1 + 1e-5)


def test_lists_whose_partial_results_are_joined_first():
    """601 tensors of several chunks each: more partial results than a clipping wave joins by itself."""
    from gsplat_host.optim import clip_grads_, grad_norm
    pool = values(601 * 81_921, torch.bfloat16, 3)
    tensors = list(pool.split(81_921))
    before = pool.clone()
    for p in NORMS:
        check_norm(grad_norm(tensors, p), [before], p)
    bound = 0.2 * norm64([before], 2.0)
    check_norm(clip_grads_(tensors, bound), [before], 2.0)
    check_clipped(pool, before, factor64(norm64([before], 2.0), bound))


def test_gradients_beyond_the_last_level_cache():
    """Over 256 MiB, which are scaled past the caches: all three types, at odd alignments and of odd sizes."""
    from gsplat_host.optim import clip_grads_
    sizes = [(40_000_003, torch.float32), (1, torch.float16), (30_000_001, torch.bfloat16), (25_165_827, torch.float16), (77, torch.float32)]
    pools = [values(n + 3, t, k) for k, (n, t) in enumerate(sizes)]
    tensors = [p[1 + k % 2:1 + k % 2 + n] for k, (p, (n, _)) in enumerate(zip(pools, sizes))]
    assert sum(t.numel() * t.element_size() for t in tensors) > 256 << 20
    before = [p.clone() for p in pools]
    inside = [b[1 + k % 2:1 + k % 2 + n] for k, (b, (n, _)) in enumerate(zip(before, sizes))]
    norm = norm64(inside, 2.0)
    check_norm(clip_grads_(tensors, 0.4 * norm), inside, 2.0)
    for k, (t, b, p, whole) in enumerate(zip(tensors, inside, pools, before)):
        check_clipped(t, b, factor64(norm, 0.4 * norm))
        at = 1 + k % 2
        assert torch.equal(p[:at], whole[:at]) and torch.equal(p[at + t.numel():], whole[at + t.numel():])


@pytest.mark.parametrize("dtype,n", [(torch.float32, 67_108_867), (torch.bfloat16, 134_217_731)])
def test_a_step_over_gradients_beyond_the_last_level_cache(dtype, n):
    """Just over 256 MiB of gradients, which the step then reads past the caches: the same bits all the same."""
    shapes = {"f_rest": (n - 5,), "opacity": (5,)}
    a, b = make(6, shapes, moments=False), make(6, shapes, moments=False)
    grads = {k: values(math.prod(s), dtype, j) for j, (k, s) in enumerate(shapes.items())}
    norm = norm64(grads.values(), 2.0)
    got = a.step(grads, max_norm=0.3 * norm)
    b.step({k: g.float() for k, g in grads.items()}, grad_scale=float(np.float32(factor64(norm, 0.3 * norm))))
    assert abs(float(got) - norm) <= (U + 2.0 ** -25) * norm and same(state_of(a), state_of(b))
