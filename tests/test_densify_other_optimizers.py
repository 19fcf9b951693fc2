"""densify_and_prune with an optimiser that has ``prune`` / ``cat_tensors`` / ``replace_tensor`` only, and with subclasses that
do more in those steps: what GaussianAdam's one pass gives, by the two steps."""
import pytest
import torch

from gsplat_host.model import GaussianParams
from gsplat_host.optim import GaussianAdam
from gsplat_host.synthetic import make_cloud

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


class ThreeSteps:
    """Not a GaussianAdam: the interface densification asked for before there was ``refine``."""

    def __init__(self, inner):
        self._inner = inner

    def prune(self, keep):
        return self._inner.prune(keep)

    def cat_tensors(self, extension):
        return self._inner.cat_tensors(extension)

    def replace_tensor(self, name, tensor):
        return self._inner.replace_tensor(name, tensor)


class Tagged(GaussianAdam):
    """Keeps a number for each row beside the tensors."""

    def cat_tensors(self, extension):
        rows = next(iter(extension.values())).shape[0]
        self.tags = torch.cat((self.tags, self.tags.new_full((rows,), -1)))
        return super().cat_tensors(extension)

    def prune(self, keep):
        self.tags = self.tags[keep]
        return super().prune(keep)


class Watched(GaussianParams):
    """Does more when rows are appended and removed, and has its own opacity."""

    def densification_postfix(self, new_xyz, *more):
        self.ages = torch.cat((self.ages, self.ages.new_zeros(new_xyz.shape[0])))
        super().densification_postfix(new_xyz, *more)

    def prune_points(self, mask):
        self.ages = self.ages[~mask]
        super().prune_points(mask)


class Fainter(GaussianParams):
    @property
    def get_opacity(self):
        return 0.01 * torch.sigmoid(self._opacity)


def make(device, model=GaussianParams, optimizer=GaussianAdam):
    P = 400
    m = model(make_cloud(P, sh_degree=1, seed=3), max_sh_degree=1, device=device)
    base = GaussianAdam.for_model(m)
    opt = optimizer(base.params, base.lrs)
    m.training_setup(opt, percent_dense=0.01)
    g = torch.Generator().manual_seed(6)
    for k, p in opt.params.items():
        opt.exp_avg[k], opt.exp_avg_sq[k] = torch.randn(p.shape, generator=g).to(device), torch.rand(p.shape, generator=g).to(device)
    m.xyz_gradient_accum = (torch.rand((P, 1), generator=g) * 0.001).to(device)
    m.denom = torch.ones((P, 1), device=device)
    m.max_radii2D = (torch.rand((P,), generator=g) * 30).to(device)
    with torch.no_grad():
        m._opacity[10:40] = -8.0
    return m, opt


def densify(m, grad=0.0005, screen=12.0):
    m.densify_and_prune(grad, 0.005, 22.0, screen, generator=torch.Generator().manual_seed(1))


def state(m, opt):
    out = [t.detach() for k in opt.params for t in (opt.params[k], opt.exp_avg[k], opt.exp_avg_sq[k])]
    return out + [getattr(m, a).detach() for _, a in m.GROUPS] + [m.xyz_gradient_accum, m.denom, m.max_radii2D]


def same(a, b):
    return len(a) == len(b) and all(x.shape == y.shape and torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("grad", (0.0005, 1.0))              # 1.0: nothing is restless, it only prunes
def test_an_optimizer_without_refine(device, grad):
    a, opt_a = make(device)
    b, opt_b = make(device)
    b.optimizer = ThreeSteps(opt_b)
    densify(a, grad)
    densify(b, grad)
    assert same(state(a, opt_a), state(b, opt_b)) and a._xyz.shape[0] != 400


@pytest.mark.parametrize("device", DEVICES)
def test_an_optimizer_that_does_more_in_its_steps(device):
    a, opt_a = make(device)
    b, opt_b = make(device, optimizer=Tagged)
    opt_b.tags = torch.arange(400, device=device)
    densify(a)
    densify(b)
    assert same(state(a, opt_a), state(b, opt_b)) and opt_b.tags.shape[0] == b._xyz.shape[0]
    old = opt_b.tags >= 0
    assert 0 < int(old.sum()) < old.numel() and bool((opt_b.tags[old].diff() > 0).all())
    keep = torch.ones(opt_b.tags.shape[0] + 2, dtype=torch.bool, device=device)
    keep[0] = False
    opt_b.refine(keep, {k: torch.zeros((2,) + p.shape[1:], device=device) for k, p in opt_b.params.items()})
    assert opt_b.tags.shape[0] == opt_b.params["xyz"].shape[0] and bool((opt_b.tags[-2:] == -1).all())


@pytest.mark.parametrize("device", DEVICES)
def test_a_model_that_does_more_in_its_steps(device):
    a, opt_a = make(device)
    b, opt_b = make(device, model=Watched)
    b.ages = torch.arange(1.0, 401.0, device=device)
    densify(a)
    densify(b)
    assert same(state(a, opt_a), state(b, opt_b)) and b.ages.shape[0] == b._xyz.shape[0] and int((b.ages == 0).sum()) > 0


@pytest.mark.parametrize("device", DEVICES)
def test_a_model_with_its_own_opacity(device):
    """No opacity above 0.01, so with 0.005 as the least everything whose logit is negative goes, new rows included."""
    m, opt = make(device, model=Fainter)
    densify(m, screen=None)
    assert m._xyz.shape[0] > 0 and float(m.get_opacity.detach().min()) >= 0.005 and opt.params["xyz"].shape[0] == m._xyz.shape[0]
