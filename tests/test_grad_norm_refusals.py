"""What the gradient norm, clipping and the clipped step refuse, before anything is launched: no GPU needed."""
import ctypes as C
import math

import pytest
import torch

import diff_gaussian_rasterization as dgr
from gsplat_host import optim

lib = dgr._lib
F32, F16, BF16 = 0, 1, 2
MAX, ONE, TWO = 0, 1, 2
SCRATCH = 0x100000                                    # never dereferenced: the checks fail first
NORM = C.c_void_p(0x200000)


def words(*tensors):
    return (C.c_uint64 * (3 * max(1, len(tensors))))(*[w for t in tensors for w in t])


def last():
    return lib.gsr_last_error().decode()


def call(fn, tensors, norm_type=TWO, norm=NORM, scratch=SCRATCH, nbytes=1 << 20, count=None, bound=()):
    n = len(tensors) if count is None else count
    return fn(n, words(*tensors) if tensors else None, norm_type, *bound, norm, scratch, nbytes, None)


@pytest.mark.parametrize("fn,bound", [(lib.gsr_grad_norm, ()), (lib.gsr_clip_grads, (1.0,))])
def test_library_checks(fn, bound):
    ok = (0x1000, 16, F32)
    assert call(fn, [], count=-1, bound=bound) == -1 and "-1 tensors" in last()
    assert call(fn, [], count=3, bound=bound) == -1 and "null tensor list" in last()
    for bad in (-1, 3, 7):
        assert call(fn, [ok], norm_type=bad, bound=bound) == -1 and "norm type" in last()
    assert call(fn, [ok], norm=None, bound=bound) == -1 and "null pointer for the norm" in last()
    assert call(fn, [ok, (0x2000, 4, 3)], bound=bound) == -1 and "tensor 1 has unknown type" in last()
    assert call(fn, [ok, (0, 4, F16)], bound=bound) == -1 and "null pointer in tensor 1" in last()
    assert call(fn, [(0x1002, 4, F32)], bound=bound) == -1 and "not aligned" in last()
    assert call(fn, [(0x1001, 4, BF16)], bound=bound) == -1 and "not aligned" in last()
    assert call(fn, [(0x1000, 1 << 45, F32)], bound=bound) == -1 and "elements" in last()
    assert call(fn, [(0x1000 + (i << 46), 1 << 44, F32) for i in range(2)], bound=bound) == -1 and "chunks" in last()
    assert call(fn, [ok], nbytes=16, bound=bound) == -3 and "scratch too small" in last()
    assert call(fn, [ok], scratch=SCRATCH + 16, bound=bound) == -3 and "256-byte aligned" in last()
    assert call(fn, [ok], scratch=None, bound=bound) == -3


def test_scratch_grows_with_the_list():
    sizes = [lib.gsr_grad_norm_bytes(n) for n in (0, 1, 120, 121, 10_000)]
    assert sizes == sorted(sizes) and all(s % 256 == 0 and s > 0 for s in sizes) and sizes[-1] > sizes[0]
    assert lib.gsr_grad_norm_bytes(-5) == sizes[0]


@pytest.mark.parametrize("tensors", [
    [(0x1000, 16, F32), (0x1000, 16, F32)],                       # the same tensor twice
    [(0x1000, 16, F32), (0x103c, 4, F32)],                        # the last element of one is the first of another
    [(0x5000, 4, F32), (0x1000, 100, BF16), (0x1080, 1, F16)],    # one inside another, not in order
    [(0x1000, 1000, F32)] + [(0x8000 + 64 * i, 16, F32) for i in range(200)] + [(0x1f00, 1, F32)],
])
def test_clipping_refuses_tensors_that_share_memory(tensors):
    assert call(lib.gsr_clip_grads, tensors, bound=(1.0,)) == -1 and "share memory" in last()


@pytest.mark.parametrize("bound", [-1.0, -math.inf, math.nan])
def test_bounds_below_zero_are_refused(bound):
    assert call(lib.gsr_clip_grads, [(0x1000, 16, F32)], bound=(bound,)) == -1 and "bound" in last()
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grads_([torch.ones(3)], bound)


def adam(count=1, tensors=None, types=None, step=1, norm_type=TWO, bound=1.0, norm=NORM, scratch=SCRATCH, nbytes=1 << 20):
    arr = (optim._AdamTensor * 8)(*(tensors if tensors is not None else [(0x1000, 0x2000, 0x3000, 0x4000, 16, 0.1, 0)]))
    kinds = None if types is None else (C.c_int * 8)(*types)
    return lib.gsr_adam_step_clipped(count, arr, kinds, 0.9, 0.999, 1e-15, step, 1.0, norm_type, bound, 0, norm, scratch, nbytes, None)


def test_the_clipped_step_checks_its_arguments():
    assert adam(count=9) == -1 and "9 tensors" in last()
    assert adam(count=-1) == -1
    assert adam(step=0) == -1 and "step counts from 1" in last()
    assert adam(bound=-0.5) == -1 and "bound" in last()
    assert adam(bound=math.nan) == -1
    assert adam(norm_type=9) == -1 and "norm type" in last()
    assert adam(norm=None) == -1
    assert adam(types=[5]) == -1 and "unknown type" in last()
    for hole in range(4):
        t = [0x1000, 0x2000, 0x3000, 0x4000, 16, 0.1, 0]
        t[hole] = None
        assert adam(tensors=[tuple(t)]) == -1 and "null pointer in tensor 0" in last(), hole
    assert adam(nbytes=8) == -3 and adam(scratch=SCRATCH + 8) == -3


def test_python_refuses_what_the_kernels_do_not_read():
    for fn in (optim.grad_norm, lambda g, p=2.0: optim.clip_grads_(g, 1.0, p)):
        with pytest.raises(ValueError, match="on the GPU"):
            fn([torch.ones(3)])
        with pytest.raises(ValueError, match="on the GPU"):
            fn(torch.ones(3))
        for dtype in (torch.float64, torch.int32, torch.complex64, torch.bool):
            with pytest.raises(TypeError, match="float32, float16 or bfloat16"):
                fn({"a": torch.ones(3).to(dtype)})
        for empty in ([], {}, [None, None], iter(())):
            with pytest.raises(ValueError, match="no gradients"):
                fn(empty)
        with pytest.raises(ValueError, match="dense"):
            fn([torch.eye(3).to_sparse()])
    for p in (0.0, 3.0, -1.0, math.nan, -math.inf, 0.5):
        with pytest.raises(ValueError, match="norm_type"):
            optim._norm_code(p)
    assert [optim._norm_code(p) for p in (1, 2, math.inf, 2.0, "inf")] == [1, 2, 0, 2, 0]


def test_a_refused_step_is_not_counted():
    opt = optim.GaussianAdam({"a": torch.zeros(4)}, {"a": 0.1})
    for kw in ({"max_norm": -1.0}, {"max_norm": math.nan}, {"max_norm": 1.0, "norm_type": 3.0}, {"skip_nonfinite": True}, {}):
        with pytest.raises(ValueError):
            opt.step({"a": torch.zeros(4)}, **kw)
    assert opt.step_count == 0


def test_which_strides_fill_memory_and_which_share_it():
    base = torch.arange(24.0).reshape(2, 3, 4)
    fills, shares = optim._fills_its_memory, optim._shares_elements
    for t in (base, base.permute(2, 0, 1), base.transpose(0, 1), base[1], base[:, :1, :1].squeeze(), base[:0], torch.ones(())):
        assert not shares(t)
    assert fills(base.permute(2, 0, 1)) and fills(base.transpose(1, 2)) and fills(base[1]) and fills(torch.ones(()))
    assert fills(base.as_strided((4, 1, 6), (1, 99, 4)))          # a dimension of size 1 may have any stride
    for t in (base[:, :2], base[..., ::2], base[:, :, 1], base.as_strided((2, 3), (12, 4))):
        assert not fills(t) and not shares(t)
    for t in (torch.ones(1).expand(5), torch.ones(3, 1).expand(3, 4), base.as_strided((5, 4), (3, 1)), base.as_strided((3, 3), (2, 2))):
        assert not fills(t) and shares(t)
