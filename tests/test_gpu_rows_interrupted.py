"""A compaction that ends early, between its count's launch and its arrival: the count has landed before the call returns, so
that it cannot land in a later call's word."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Stop(Exception):
    pass


@pytest.mark.parametrize("where", ("_Move", "_await_count"))
def test_the_count_has_landed_when_the_error_arrives(where, monkeypatch):
    from gsplat_host import rows
    n = 50_021
    t = torch.randn(n, 3, generator=torch.Generator().manual_seed(4)).cuda()
    keep = torch.rand(n, generator=torch.Generator().manual_seed(5)).cuda() < 0.5
    want = t[keep]
    rows.compact_rows([t], keep)                             # the word exists
    _, word = rows._landing(t.device)
    work = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    last = word.value

    def stop(*_):
        raise Stop

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(20):                                  # some milliseconds before the count
            work = work @ work * 1e-4
        with monkeypatch.context() as m:
            m.setattr(rows, where, stop)
            with pytest.raises(Stop):
                rows.compact_rows([t], keep)
        assert side.query()
    assert word.value != last and word.value & 0xFFFFFFFF == want.shape[0]
    (out,), _ = rows.compact_rows([t], keep)                 # on another stream than the abandoned one
    assert torch.equal(out, want)
