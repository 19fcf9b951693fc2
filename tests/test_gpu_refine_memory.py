"""Peak memory of refinement: the tensors are moved group by group, so that the old moments go as the new ones come."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TAILS = {"xyz": (3,), "f_dc": (1, 3), "f_rest": (15, 3), "opacity": (1,), "scaling": (3,), "rotation": (4,)}


def make(n):
    from gsplat_host.optim import GaussianAdam
    g = torch.Generator(device="cuda").manual_seed(1)
    new = lambda: {k: torch.randn((n, *s), generator=g, device="cuda") for k, s in TAILS.items()}
    opt = GaussianAdam(new(), dict.fromkeys(TAILS, 0.1))
    opt.exp_avg, opt.exp_avg_sq = new(), new()
    return opt


def peak_of(call):
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    call()
    return torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("extra", (None, 0, 30_000))
def test_refinement_needs_a_third_more_not_twice(extra):
    n = 300_000
    opt = make(n)
    caller = dict(opt.params)                                # a model holds the old parameters until it takes the new ones
    state = 3 * sum(t.numel() * 4 for t in caller.values())
    keep = torch.ones(n + (extra or 0), dtype=torch.bool, device="cuda")
    keep[::50] = False
    born = None if extra is None else {k: torch.randn((extra, *s), device="cuda") for k, s in TAILS.items()}
    want = {}
    for k in TAILS:                                          # on the host: nothing of it counts here
        whole = [t[k].detach().cpu() for t in (opt.params, opt.exp_avg, opt.exp_avg_sq)]
        if born is not None:
            whole = [torch.cat((t, born[k].cpu() if i == 0 else torch.zeros(born[k].shape))) for i, t in enumerate(whole)]
        want[k] = [t[keep.cpu()] for t in whole]
    peak = peak_of(lambda: opt.prune(keep) if extra is None else opt.refine(keep, born))
    # new parameters beside the old, one moment's new tensors while its old ones live (10 % more rows at most), the index
    # (4 bytes a row of 708), the allocator's rounding
    assert peak <= state * (0.5 if extra else 0.4), peak / state
    for k in TAILS:
        for a, b in zip(want[k], (opt.params[k], opt.exp_avg[k], opt.exp_avg_sq[k])):
            assert torch.equal(a, b.detach().cpu())


def test_a_refused_refinement_changes_nothing():
    opt = make(50)
    held = [dict(d) for d in (opt.params, opt.exp_avg, opt.exp_avg_sq)]
    good = {k: torch.zeros((4, *s), device="cuda") for k, s in TAILS.items()}
    keep = torch.ones(54, dtype=torch.bool, device="cuda")
    bad = [(keep[:53], good), (keep[:49], None), (keep, None), (keep, {**good, "rotation": torch.zeros((4, 3), device="cuda")}),
           (keep, {**good, "xyz": torch.zeros((5, 3), device="cuda")}), (keep, {**good, "opacity": torch.zeros((4, 1))}),
           (keep.view(1, -1), good)]
    for k, e in bad:
        with pytest.raises((ValueError, TypeError)):
            opt.refine(k, e)
        assert all(a[n] is b[n] for a, b in zip(held, (opt.params, opt.exp_avg, opt.exp_avg_sq)) for n in TAILS)


@pytest.mark.parametrize("moved", (0, 1))
def test_memory_that_ends_half_way(moved, monkeypatch):
    """The second moments, or the parameters, cannot be moved: parameters as before, moments of their sizes, all zeros."""
    from gsplat_host import rows
    opt = make(500)
    held, again = dict(opt.params), rows._again
    left = [moved]

    def until_full(*args):
        if not left[0]:
            raise torch.cuda.OutOfMemoryError("no memory")
        left[0] -= 1
        return again(*args)

    keep = torch.arange(500, device="cuda") % 3 > 0
    born = {k: torch.zeros((167, *s), device="cuda") for k, s in TAILS.items()}
    with monkeypatch.context() as m:
        m.setattr(rows, "_again", until_full)
        with pytest.raises(torch.cuda.OutOfMemoryError):                 # as many new rows as removed ones
            opt.refine(torch.cat((keep, torch.ones(167, dtype=torch.bool, device="cuda"))), born)
    assert all(opt.params[k] is held[k] for k in TAILS)
    for moments in (opt.exp_avg, opt.exp_avg_sq):
        assert all(moments[k].shape == held[k].shape and not bool(moments[k].any()) for k in TAILS)
    opt.prune(keep)
    opt.step({k: torch.ones_like(p) for k, p in opt.params.items()}, max_norm=1.0)
