"""Rows of more than 2^30 units of one byte: the lengths at which the kernels' divisor is largest."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", (2 ** 30 + 1, 2 ** 31 - 1))
def test_long_rows(length):
    from gsplat_host.rows import select_rows
    g = torch.Generator(device="cuda").manual_seed(length)
    t = torch.randint(0, 256, (2 * length,), dtype=torch.uint8, generator=g, device="cuda").view(2, length)
    out, = select_rows([t], torch.tensor([1, -1, 0, 1], device="cuda"))
    assert torch.equal(out[0], t[1]) and torch.equal(out[2], t[0]) and torch.equal(out[3], t[1])
    assert int(torch.count_nonzero(out[1])) == 0
