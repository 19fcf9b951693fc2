"""Rows of many tensors moved at once, against torch's concatenation and indexing: copies, so bit for bit."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

# row shapes whose bytes are multiples of 16, 8, 4, 2, 1 and of nothing, short and long
KINDS = [((3,), torch.float32), ((15, 3), torch.float32), ((), torch.float32), ((4,), torch.float32), ((2,), torch.float32),
         ((0, 3), torch.float32), ((7,), torch.float16), ((1,), torch.bfloat16), ((5,), torch.uint8), ((), torch.bool),
         ((3,), torch.int64), ((33,), torch.float64), ((257,), torch.int16), ((1000,), torch.float32), ((4099,), torch.uint8)]


def data(n, shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    raw = torch.randint(0, 256, (n * math.prod(shape) * dtype.itemsize,), dtype=torch.uint8, generator=g, device="cuda")
    return (raw > 127).view(n, *shape) if dtype == torch.bool else raw.view(dtype).view(n, *shape)


def bits(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


def same(a, b):
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(bits(a), bits(b))


def tensors(n, seed=0, kinds=KINDS):
    return [data(n, s, d, seed + k) for k, (s, d) in enumerate(kinds)]


def pick(t, index):
    """t[index], zeros where the index is outside."""
    inside = (index >= 0) & (index < t.shape[0])
    out = torch.zeros((index.numel(),) + t.shape[1:], dtype=t.dtype, device=t.device)
    at = inside.nonzero().view(-1)
    out[at] = t[index.long()[at]]
    return out


@pytest.mark.parametrize("dtype", (torch.int32, torch.int64))
@pytest.mark.parametrize("n,picked", [(1, 1), (1, 9), (2, 3), (7, 5), (64, 64), (257, 1), (1000, 4099), (5003, 5003), (20_011, 3001)])
def test_select(n, picked, dtype):
    from gsplat_host.rows import select_rows
    old = tensors(n)
    g = torch.Generator(device="cuda").manual_seed(picked)
    orders = {"any order, repeats": torch.randint(0, n, (picked,), generator=g, device="cuda"),
              "ascending": torch.randint(0, n, (picked,), generator=g, device="cuda").sort().values,
              "one row": torch.full((picked,), n - 1, device="cuda"),
              "a run": torch.arange(picked, device="cuda") % n,
              "backwards": (n - 1 - torch.arange(picked, device="cuda")) % n}
    for name, index in orders.items():
        new = select_rows(old, index.to(dtype))
        assert len(new) == len(old)
        for t, o, kind in zip(old, new, KINDS):
            assert same(o, t[index]), (name, kind)


@pytest.mark.parametrize("dtype", (torch.int32, torch.int64))
def test_an_index_outside_the_rows_gives_zeros(dtype):
    from gsplat_host.rows import select_rows
    n = 300
    old = tensors(n)
    bad = [-1, -2, n, n + 1, 2 ** 31 - 1, -2 ** 31] + ([2 ** 32, 2 ** 32 + 5, -2 ** 32, 2 ** 63 - 1, -2 ** 63] if dtype == torch.int64 else [])
    index = torch.tensor([0, n - 1] + [x for b in bad for x in (b, 5)] + bad, dtype=dtype, device="cuda")
    for t, o, kind in zip(old, select_rows(old, index), KINDS):
        assert same(o, pick(t, index)), kind
    for o in select_rows([t[:0] for t in old], index):                          # no row at all
        assert not bool(bits(o).any())
    for t, o in zip(old, select_rows(old, index[:0])):
        assert o.shape == (0,) + t.shape[1:] and o.dtype == t.dtype


def masks(total):
    g = torch.Generator(device="cuda").manual_seed(total)
    r = torch.rand((total,), generator=g, device="cuda")
    yield "most", r < 0.9
    yield "few", r < 0.02
    yield "all", torch.ones((total,), dtype=torch.bool, device="cuda")
    yield "none", torch.zeros((total,), dtype=torch.bool, device="cuda")
    yield "runs", (torch.arange(total, device="cuda") // 37) % 3 > 0
    yield "last", torch.arange(total, device="cuda") == total - 1
    yield "not first", torch.arange(total, device="cuda") > 0


@pytest.mark.parametrize("n,extra", [(0, 0), (1, 0), (0, 5), (3, 2), (16, 0), (17, 1), (4095, 0), (4096, 1), (4097, 300), (12_289, 4097), (70_001, 999)])
def test_compact(n, extra):
    from gsplat_host.rows import compact_rows
    old = tensors(n)
    more = [None if k % 3 == 2 else data(extra, s, d, 100 + k) for k, (s, d) in enumerate(KINDS)]
    for name, keep in masks(n + extra):
        new, index = compact_rows(old, keep, more)
        assert index.dtype == torch.int32 and torch.equal(index.long(), keep.nonzero().view(-1)), name
        for t, e, o, kind in zip(old, more, new, KINDS):
            whole = torch.cat((t, torch.zeros((extra,) + t.shape[1:], dtype=t.dtype, device="cuda") if e is None else e))
            assert same(o, whole[keep]), (name, kind)
        if not extra:
            for o, again in zip(new, compact_rows(old, keep)[0]):
                assert same(o, again)


def test_many_tensors_and_many_flags():
    from gsplat_host.rows import compact_rows, select_rows
    n = 1001
    old = [data(n, (k % 5 + 1,), torch.float32, k) for k in range(113)]          # several launches
    index = torch.arange(n - 1, -1, -1, device="cuda")
    for t, o in zip(old, select_rows(old, index)):
        assert same(o, t[index])
    big = 9_000_001                                                              # several tiles to a workgroup
    ids = torch.arange(big, dtype=torch.int32, device="cuda")
    for name, keep in masks(big):
        (out,), index = compact_rows([ids], keep)
        assert torch.equal(out, ids[keep]) and torch.equal(index, out), name


def test_strides_and_alignments():
    from gsplat_host.rows import compact_rows, select_rows
    n = 777
    base = data(n + 3, (15, 3), torch.float32, 1)
    g = torch.Generator(device="cuda").manual_seed(2)
    index = torch.randint(0, n, (2 * 900,), generator=g, device="cuda")[::2]     # a strided index
    keep_buffer = torch.rand((n + 64,), generator=g, device="cuda") < 0.6
    flat = data(4 * n + 16, (), torch.uint8, 3)
    half = data(3 * n + 16, (), torch.float16, 4)
    old = [base[3:], base[3:].transpose(1, 2), base[:n, ::2], base[:n].permute(0, 2, 1)[:, 1:], data(3, (n,), torch.float32, 9).t(),
           data(1, (4,), torch.float32, 8).expand(n, 4)]
    old += [flat[o:o + 4 * n].view(n, 4) for o in (1, 2, 3, 4)] + [half[o:o + 3 * n].view(n, 3) for o in (1, 2, 3)]
    for t, o in zip(old, select_rows(old, index)):
        assert same(o, t[index])
    for offset in (0, 1, 3, 15, 16, 17):                                         # flags at any address
        keep = keep_buffer[offset:offset + n]
        new, at = compact_rows(old, keep)
        assert torch.equal(at.long(), keep.nonzero().view(-1))
        for t, o in zip(old, new):
            assert same(o, t[keep])
    strided = keep_buffer[:n + n % 2].view(-1, 1).expand(-1, 2)[:n, 0]
    assert same(compact_rows(old[:1], strided)[0][0], old[0][strided])


@pytest.mark.parametrize("offset", (0, 1, 2, 3))
def test_row_lengths(offset):
    """Rows of 1 to 40 bytes at every alignment, with first and last rows next to one another and apart."""
    from gsplat_host.rows import compact_rows, select_rows
    n = 203
    for length in range(1, 41):
        t = data(n * length + 4, (), torch.uint8, length)[offset:offset + n * length].view(n, length)
        e = data(17 * length + 4, (), torch.uint8, 99 + length)[offset:offset + 17 * length].view(17, length)
        g = torch.Generator(device="cuda").manual_seed(length)
        index = torch.randint(0, n, (1009,), generator=g, device="cuda")
        index[::7], index[1::7], index[2::7] = n - 1, 0, n - 2
        index[500:700] = torch.arange(200, device="cuda")
        index[3::50] = -1
        assert same(select_rows([t], index)[0], pick(t, index)), length
        keep = torch.rand((n + 17,), generator=g, device="cuda") < 0.8
        keep[n - 2:n + 2] = True                                 # across the seam of the two buffers
        for more in (e, None):
            out, = compact_rows([t], keep, [more])[0]
            assert same(out, torch.cat((t, torch.zeros_like(e) if more is None else more))[keep]), (length, more is None)


def test_views_that_only_look_conjugated_or_negated():
    from gsplat_host.rows import select_rows
    z = torch.randn(50, 3, dtype=torch.complex64, device="cuda")
    index = torch.tensor([4, 49, 0, 4], device="cuda")
    for t in (z, z.conj(), z.conj().imag, z.imag, z.resolve_conj().real):
        out, = select_rows([t], index)
        assert torch.equal(out, t[index]) and not out.is_conj() and not out.is_neg()


def test_compaction_refuses_to_be_captured():
    from gsplat_host.rows import compact_rows
    t, keep = torch.zeros((40, 3), device="cuda"), torch.ones(40, dtype=torch.bool, device="cuda")
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.capture_begin()
        with pytest.raises(RuntimeError, match="cannot be captured"):
            compact_rows([t], keep)
        t.add_(1.0)                                              # a graph of something
        graph.capture_end()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(compact_rows([t], keep)[0][0], t)


def test_two_threads_on_streams_of_their_own():
    """Both compact and clip at once: nothing is shared between their calls."""
    import threading
    from gsplat_host.optim import clip_grads_
    from gsplat_host.rows import compact_rows
    problems = []

    def work(seed):
        try:
            g = torch.Generator(device="cuda").manual_seed(seed)
            with torch.cuda.stream(torch.cuda.Stream()):
                for k in range(30):
                    n = 1000 + 977 * k + seed
                    t, keep = torch.rand((n, 5), generator=g, device="cuda"), torch.rand((n,), generator=g, device="cuda") < 0.5
                    (out,), index = compact_rows([t], keep)
                    want = t[keep]
                    norm = clip_grads_([t], 1.0)
                    kept = t[keep]
                    if not (same(out, want) and torch.equal(index.long(), keep.nonzero().view(-1))
                            and torch.allclose(kept * norm, want, rtol=1e-5, atol=0)):   # factor, product and this one: 4 x 2^-24
                        problems.append((seed, k))
                torch.cuda.current_stream().synchronize()
        except Exception as e:                                   # reported by the main thread
            problems.append((seed, repr(e)))

    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2, 3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not problems, problems


def test_past_32_bits():
    """A tensor of 4.4 GB: rows that lie, and land, behind 2^32 bytes."""
    from gsplat_host.rows import compact_rows, select_rows
    n, w = 1_100_000, 1000
    big = torch.zeros((n, w), dtype=torch.float32, device="cuda")
    marks = torch.tensor([0, 5, 1_073_741, 1_073_742, 1_090_001, n - 1], device="cuda")
    big[marks] = torch.arange(1.0, 7.0, device="cuda")[:, None] + torch.arange(w, device="cuda") / 4096.0
    out, = select_rows([big], torch.cat((marks, marks.flip(0))))
    assert torch.equal(out, torch.cat((big[marks], big[marks.flip(0)])))
    keep = torch.ones((n,), dtype=torch.bool, device="cuda")
    keep[7] = keep[1_073_000] = False
    (out,), index = compact_rows([big], keep)
    assert out.shape == (n - 2, w)
    for j in (0, 5, 7, 1_072_999, 1_073_739, 1_073_740, 1_089_999, n - 3):
        assert torch.equal(out[j], big[int(index[j])])
    assert abs(float(out.sum(dtype=torch.float64)) - float(big.sum(dtype=torch.float64))) < 1e-6


def test_refusals():
    from gsplat_host.rows import compact_rows, select_rows
    a, b = torch.zeros((4, 3), device="cuda"), torch.zeros((5, 3), device="cuda")
    index, keep = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.ones(4, dtype=torch.bool, device="cuda")
    for fn, arg in ((select_rows, index), (compact_rows, keep)):
        with pytest.raises(ValueError, match="first dimension"):
            fn([a, b], arg)
        with pytest.raises(ValueError, match="first dimension"):
            fn([torch.zeros((), device="cuda")], arg)
        with pytest.raises(ValueError, match="on the GPU"):
            fn([a, a.cpu()], arg)
        with pytest.raises(ValueError, match="is on cpu"):
            fn([a], arg.cpu())
        with pytest.raises(TypeError):
            fn([a], arg.float())
        with pytest.raises(TypeError):
            fn([a], arg.view(1, -1))
    for bad, more in ((torch.ones(3, dtype=torch.bool), None), (torch.ones(5, dtype=torch.bool), None), (torch.ones(3, dtype=torch.bool), [None])):
        with pytest.raises(ValueError, match="entries for 4 rows"):
            compact_rows([a], bad.cuda(), more)
    five = torch.ones(5, dtype=torch.bool, device="cuda")
    for more in ([torch.zeros((2, 3), device="cuda")], [torch.zeros((1, 4), device="cuda")], [torch.zeros((1, 3))],
                 [torch.zeros((1, 3), device="cuda", dtype=torch.float64)]):
        with pytest.raises(ValueError, match="do not fit"):
            compact_rows([a], five, more)
    with pytest.raises(ValueError, match="appended entries"):
        compact_rows([a], five, [None, None])


def test_another_stream_and_a_replayed_graph():
    from gsplat_host.rows import compact_rows, select_rows
    n = 30_011
    old = [data(n, s, torch.float32, k) for k, s in enumerate([(3,), (15, 3), (1,), (4,)])]
    g = torch.Generator(device="cuda").manual_seed(4)
    keep = torch.rand((n,), generator=g, device="cuda") < 0.7
    index = torch.randint(-1, n, (9001,), generator=g, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        new, at = compact_rows(old, keep)
        forked = select_rows(old, at[:5000])
    side.synchronize()
    for t, o, f in zip(old, new, forked):
        assert same(o, t[keep]) and same(f, t[keep][:5000])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = select_rows(old, index)
    for k in range(3):
        index.copy_(torch.randint(-1, n, (9001,), generator=g, device="cuda"))
        old[1].copy_(data(n, (15, 3), torch.float32, 50 + k))
        graph.replay()
        torch.cuda.synchronize()
        for t, o in zip(old, out):
            assert same(o, pick(t, index))


# ---- the model's own paths -------------------------------------------------------------------------------------

def model(P, deg, seed):
    from gsplat_host.model import GaussianParams
    from gsplat_host.optim import GaussianAdam
    from gsplat_host.synthetic import make_cloud
    m = GaussianParams(make_cloud(P, sh_degree=deg, seed=seed), max_sh_degree=deg, device="cuda")
    opt = GaussianAdam.for_model(m)
    m.training_setup(opt, percent_dense=0.01)
    g = torch.Generator().manual_seed(seed)
    for k, p in opt.params.items():
        opt.exp_avg[k] = torch.randn(p.shape, generator=g).cuda()
        opt.exp_avg_sq[k] = torch.rand(p.shape, generator=g).cuda()
    opt.step_count = 7
    m.xyz_gradient_accum = (torch.rand((P, 1), generator=g) * 0.001).cuda()
    m.denom = torch.ones((P, 1), device="cuda")
    m.denom[:5] = 0.0
    m.max_radii2D = (torch.rand((P,), generator=g) * 30).cuda()
    with torch.no_grad():
        m._opacity[10:40] = -8.0
    return m, opt


def state(m, opt):
    out = {k: (p.detach(), opt.exp_avg[k], opt.exp_avg_sq[k]) for k, p in opt.params.items()}
    out["stats"] = (m.xyz_gradient_accum, m.denom, m.max_radii2D)
    return out


def by_torch(m, opt, gone, born=None):
    """cat_tensors and prune as concatenations and masks, tensor by tensor."""
    keep, out = ~gone, {}
    for k, p in opt.params.items():
        ts = [p.detach(), opt.exp_avg[k], opt.exp_avg_sq[k]]
        if born is not None:
            ts = [torch.cat((ts[0], born[k]))] + [torch.cat((t, torch.zeros_like(born[k]))) for t in ts[1:]]
        out[k] = tuple(t[keep] for t in ts)
    return out


@pytest.mark.parametrize("P,deg", [(1, 0), (50, 0), (5003, 3), (20_000, 1)])
def test_prune_and_refine_are_what_concatenation_and_masks_give(P, deg):
    g = torch.Generator(device="cuda").manual_seed(P)
    for extra in (None, 0, 1, P // 3 + 1):
        m, opt = model(P, deg, 2)
        total = P + (extra or 0)
        gone = torch.rand((total,), generator=g, device="cuda") < 0.3
        born = None if extra is None else {k: torch.randn((extra,) + p.shape[1:], generator=g, device="cuda") for k, p in opt.params.items()}
        want = by_torch(m, opt, gone, born)
        got = opt.prune(~gone) if extra is None else opt.refine(~gone, born)
        assert opt.step_count == 7
        for k in want:
            assert got[k] is opt.params[k] and got[k].is_leaf and got[k].requires_grad
            for a, b in zip(want[k], (got[k].detach(), opt.exp_avg[k], opt.exp_avg_sq[k])):
                assert same(a, b), (k, extra)
    m, opt = model(300, 1, 3)
    with pytest.raises(ValueError, match="name every tensor"):
        opt.refine(torch.ones(301, dtype=torch.bool, device="cuda"), {"xyz": torch.zeros((1, 3), device="cuda")})


@pytest.mark.parametrize("grad,screen", [(0.0005, None), (0.0005, 12.0), (10.0, 12.0), (10.0, None),
                                         (math.nan, 12.0), (math.nan, None)])
def test_densify_and_prune_equals_its_steps(grad, screen):
    """The one pass against copies, children, densification_postfix and prune_points one after the other; with
    grad = 10 only the never seen are restless (0.001 / 0 here), and with NaN nothing is and it only prunes."""
    from gsplat_host.model import quaternion_to_matrix
    P, extent, min_opacity = 5003, 22.0, 0.005
    a, opt_a = model(P, 2, 5)
    b, opt_b = model(P, 2, 5)
    with torch.no_grad():
        ratio = (b.xyz_gradient_accum / b.denom).view(-1).nan_to_num(0.0)
        scale = b.get_scaling
        large = scale.amax(dim=1) > b.percent_dense * extent
        copy, parent = ((ratio >= grad) & ~large).nonzero().view(-1), ((ratio >= grad) & large).nonzero().view(-1)
        family = parent.repeat(2)
        spread = scale[family]
        offsets = torch.randn(spread.shape, generator=torch.Generator().manual_seed(1)).cuda() * spread
        world = torch.einsum("nij,nj->ni", quaternion_to_matrix(b._rotation[family]), offsets)
        both = torch.cat((copy, family))
        if both.numel():
            b.densification_postfix(torch.cat((b._xyz[copy], b._xyz[family] + world)), b._features_dc[both], b._features_rest[both],
                                    b._opacity[both], torch.cat((b._scaling[copy], torch.log(spread / 1.6))), b._rotation[both])
        gone = torch.zeros((b._xyz.shape[0],), dtype=torch.bool, device="cuda")
        gone[parent] = True
        gone |= b.get_opacity.reshape(-1) < min_opacity
        if screen:
            gone |= b.get_scaling.amax(dim=1) > 0.1 * extent
            gone |= b.max_radii2D > screen
        want, keep = by_torch(b, opt_b, gone), ~gone
        want["stats"] = (b.xyz_gradient_accum[keep], b.denom[keep], b.max_radii2D[keep])
    a.densify_and_prune(grad, min_opacity, extent, screen, generator=torch.Generator().manual_seed(1))
    got = state(a, opt_a)
    assert a._xyz is opt_a.params["xyz"] and 0 < a._xyz.shape[0] != P and (copy.numel() > 0) == (not math.isnan(grad))
    for k in want:
        for x, y in zip(want[k], got[k]):
            assert same(x, y), k
