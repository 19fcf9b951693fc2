"""Clipping refuses a tensor without gaps that shares elements with one that has gaps: which tensors do, without a GPU; the
refusal itself, with one."""
import itertools

import pytest
import torch

from gsplat_host import optim


def addresses(t):
    """Addresses of every byte of ``t``'s elements."""
    at = {t.data_ptr()}
    for d in range(t.dim()):
        at = {a + i * t.stride(d) * t.element_size() for a in at for i in range(t.size(d))}
    return {a + b for a in at for b in range(t.element_size())} if t.numel() else set()


def test_a_stretch_of_memory_against_a_tensor_with_gaps():
    base = torch.zeros(600, dtype=torch.uint8)
    at = base.data_ptr()
    gapped = [base[:96].view(8, 12)[:, 2:7], base[::3], base[5:500].view(5, 9, 11)[1:, ::2, 3:9], base[:480].view(4, 10, 12).permute(2, 0, 1)[::5],
              base[:96].view(torch.float32).view(4, 6)[:, 1::2], base[:96].view(torch.int16).view(6, 8)[::2, :1], base[:0].view(0, 3)[:, ::2],
              base.as_strided((3, 1, 4), (100, 7, 2)), base[7:8].expand(1)]
    for t in gapped:
        have = addresses(t)
        for begin, length in itertools.product(range(0, 600, 1), (1, 2, 3, 4, 7, 30)):
            span = range(at + begin, at + begin + length)
            assert optim._touches(t, span.start, span.stop) == any(a in have for a in span), (t.shape, t.stride(), begin, length)


def test_which_lists_share():
    base = torch.zeros(40, 8)
    half = torch.zeros(40, 8, dtype=torch.bfloat16)
    rows, left, right = base[3], base[::2], base[:, 4:]
    assert not optim._any_stretch_touches([rows, base[1:2]], [left])                     # rows between those of another
    assert optim._any_stretch_touches([rows, base[2]], [left])
    assert optim._any_stretch_touches([base], [right]) and not optim._any_stretch_touches([half], [left, right])
    assert not optim._any_stretch_touches([base[7, :4], base[8, :4]], [right])
    assert optim._any_stretch_touches([base[7, :4], base[8, :5]], [right])
    assert not optim._any_stretch_touches([], [right]) and not optim._any_stretch_touches([base[:0]], [right])
    many = [base[i] for i in range(1, 40, 2)]
    assert not optim._any_stretch_touches(many, [left]) and optim._any_stretch_touches(many + [base[20, 3:4]], [left])


@pytest.mark.gpu
def test_clipping_refuses_them():
    buf = torch.randn(64, 12, generator=torch.Generator().manual_seed(1)).cuda()
    before = buf.clone()
    for bad in ([buf, buf[:, ::2]], [buf[:, 3:5], buf[7]], [buf[::3], torch.ones(5, device="cuda"), buf[6, 11:]]):
        with pytest.raises(ValueError, match="share"):
            optim.clip_grads_(bad, 0.1)
        assert torch.equal(buf, before)
    norm = float(before.double().square().sum().sqrt())
    got = float(optim.clip_grads_([buf[:, :5], buf[:, 5:]], 0.1))                         # side by side
    assert abs(got - norm) <= 2.0 ** -23 * norm
    factor = 0.1 / (norm + 1e-6)
    assert bool(((buf.double() - before.double() * factor).abs() <= 2.5 * 2.0 ** -24 * before.double().abs()).all())
    mid = buf.clone()
    optim.clip_grads_([buf[::2], buf[1], buf[33]], 0.0)                                  # rows between
    assert not bool(buf[::2].any()) and not bool(buf[1].any()) and not bool(buf[33].any()) and torch.equal(buf[3], mid[3])
