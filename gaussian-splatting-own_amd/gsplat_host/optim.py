"""Optimiser step and data-parallel gradient exchange of the reference's training loop.

The reference steps ``torch.optim.Adam`` over six parameter tensors with one
learning rate each and ``eps = 1e-15`` (``scene/gaussian_model.py:154-163``,
``train.py:126-128``) and decays the position learning rate log-linearly
(``:164-175``, ``utils/general_utils.py:29-62``).  Here the update of all six
tensors is ONE fused HIP launch (``gsr_adam_step``; with the gradients' norm bounded first two,
``gsr_adam_step_clipped``), and, when several ranks
each render their own view of a replicated model, their gradients meet in one
flat buffer that is summed over the ranks (reduce-scatter + all-gather over RCCL) before the step.  There is no
CPU path for the update: the parameters must live on the GPU.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from bisect import bisect_left, bisect_right
from dataclasses import dataclass
from itertools import chain
from typing import Dict, Iterable, List, Optional, Union

import torch
import torch.distributed as dist

import diff_gaussian_rasterization as _dgr

_lib = _dgr._lib
MAX_TENSORS = 8


class _AdamTensor(C.Structure):
    _fields_ = [("param", C.c_void_p), ("grad", C.c_void_p), ("exp_avg", C.c_void_p), ("exp_avg_sq", C.c_void_p),
                ("n", C.c_size_t), ("lr", C.c_float), ("vec4", C.c_int)]


_lib.gsr_adam_step.argtypes = [C.c_int, C.POINTER(_AdamTensor), C.c_double, C.c_double, C.c_double, C.c_int, C.c_float,
                               C.c_void_p]
_lib.gsr_grad_norm_bytes.restype = C.c_size_t
_lib.gsr_grad_norm_bytes.argtypes = [C.c_int]
_lib.gsr_grad_norm.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
_lib.gsr_clip_grads.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_double, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
_lib.gsr_adam_step_clipped.argtypes = [C.c_int, C.c_void_p, C.c_void_p, C.c_double, C.c_double, C.c_double,
                                       C.c_int, C.c_float, C.c_int, C.c_double, C.c_int, C.c_void_p, C.c_void_p, C.c_size_t,
                                       C.c_void_p]
_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}         # GSR_F32, GSR_F16, GSR_BF16 of gsr.h
_NORMS = {math.inf: 0, 1.0: 1, 2.0: 2}                                   # GSR_NORM_MAX, GSR_NORM_1, GSR_NORM_2
Grads = Union[torch.Tensor, Iterable[Optional[torch.Tensor]], Dict[str, Optional[torch.Tensor]]]


def expon_lr(step: int, lr_init: float, lr_final: float, lr_delay_steps: int = 0, lr_delay_mult: float = 1.0,
             max_steps: int = 1_000_000) -> float:
    """Log-linear learning-rate decay with an optional eased-in start (utils/general_utils.py:29-62)."""
    if step < 0 or (lr_init == 0.0 and lr_final == 0.0):
        return 0.0
    if lr_delay_steps > 0:
        delay = lr_delay_mult + (1 - lr_delay_mult) * math.sin(0.5 * math.pi * min(max(step / lr_delay_steps, 0), 1))
    else:
        delay = 1.0
    t = min(max(step / max_steps, 0), 1)
    return delay * math.exp(math.log(lr_init) * (1 - t) + math.log(lr_final) * t)


@dataclass
class OptimizationParams:
    """The optimiser-related fields of arguments/__init__.py:71-90."""
    position_lr_init: float = 0.00016
    position_lr_final: float = 0.0000016
    position_lr_delay_mult: float = 0.01
    position_lr_max_steps: int = 30_000
    feature_lr: float = 0.0025
    opacity_lr: float = 0.05
    scaling_lr: float = 0.005
    rotation_lr: float = 0.001


EXCHANGES = ("scatter_gather", "direct", "all_reduce")


def _sum_flat_over_ranks(flat: torch.Tensor, group, method: str) -> None:
    """In place: ``flat`` (1-D fp32, the same length on every rank) becomes its sum over the ranks of ``group``.

    ``scatter_gather`` (the default): reduce-scatter, then all-gather.  Rank r ends the first step with the sum of
    slice r of every rank's buffer and the second hands the slices round: each rank sends and receives 2 (n-1)/n
    of the buffer, spread over its links to all n-1 peers, where one ring would push the same bytes through one
    link (8 GPUs joined point to point by 7 xGMI links each; 236 MB of gradients at a million Gaussians).
    ``direct``: the same two steps spelled out with point-to-point traffic only, an all-to-all of the slices,
    a local sum, an all-gather: no ring even if the library would build one for a reduce-scatter.
    ``all_reduce``: one collective, the library's choice of algorithm.
    The first two need the length to be a multiple of the number of ranks (a GradArena pads for that); otherwise
    the call falls back to ``all_reduce``.  ``gloo`` only ever sees host tensors."""
    if method not in EXCHANGES:
        raise ValueError(f"exchange method must be one of {EXCHANGES}")
    world = dist.get_world_size(group)
    if world <= 1:
        return
    work = flat
    on_host = dist.get_backend(group) == "gloo" and flat.is_cuda
    if on_host:
        work = flat.cpu()
    n = work.numel()
    if method == "all_reduce" or n % world != 0:
        dist.all_reduce(work, op=dist.ReduceOp.SUM, group=group)
    else:
        piece = n // world
        if method == "scatter_gather":
            mine = torch.empty((piece,), dtype=work.dtype, device=work.device)
            dist.reduce_scatter_tensor(mine, work, op=dist.ReduceOp.SUM, group=group)
        else:
            theirs = torch.empty_like(work)                         # slice `rank` of every rank's buffer
            dist.all_to_all_single(theirs, work, group=group)
            mine = theirs.view(world, piece).sum(dim=0)
        dist.all_gather_into_tensor(work, mine, group=group)
    if on_host:
        flat.copy_(work)


class GradArena:
    """One flat fp32 buffer holding the gradients of all parameter tensors back to back (each
    start 16-byte aligned, the whole padded to a multiple of 1024 floats so that it splits evenly over
    any power-of-two number of ranks), with a view per tensor.  Backward passes write into the views, the
    data-parallel exchange works on ``flat`` as a whole, and the optimiser reads the views."""

    def __init__(self, params: Dict[str, torch.Tensor]):
        self.offsets, total = {}, 0
        for name, p in params.items():
            self.offsets[name] = total
            total += (p.numel() + 3) // 4 * 4
        first = next(iter(params.values()))
        self.flat = torch.zeros(((total + 1023) // 1024 * 1024,), dtype=torch.float32, device=first.device)
        self.views = {name: self.flat[o:o + params[name].numel()].view_as(params[name])
                      for name, o in self.offsets.items()}

    def attach(self, params: Dict[str, torch.Tensor]) -> None:
        """Makes every parameter's ``.grad`` the arena view, so autograd accumulates in place."""
        for name, p in params.items():
            p.grad = self.views[name]

    def zero_(self) -> None:
        self.flat.zero_()

    # The norm is over the views, not over ``flat``: clipping by a NaN norm would leave NaNs in the padding, which clearing
    # the gradients alone does not reach, and every later norm would be NaN.
    def norm(self, norm_type: float = 2.0, grad_scale: float = 1.0) -> torch.Tensor:
        """``grad_norm`` of ``grad_scale`` times all gradients (the padding between them does not count).  After
        ``all_reduce`` every rank holds the same gradients and finds the same norm, without a collective of its own;
        they are SUMS over the ranks then, and ``grad_scale`` is the factor that ``all_reduce`` returned."""
        scale = _positive_scale(grad_scale)
        norm = grad_norm(self.views, norm_type)
        return norm if scale == 1.0 else norm.mul_(scale)

    def clip_(self, max_norm: float, norm_type: float = 2.0, grad_scale: float = 1.0) -> torch.Tensor:
        """``clip_grads_`` of all gradients (the padding is left as it is) for a step with ``grad_scale``: the norm that is
        bounded, and returned, is that of ``grad_scale`` times the gradients, which are themselves scaled by
        ``min(1, max_norm / (grad_scale (norm + 1e-6)))`` and stay without that factor.  After an averaging
        ``all_reduce``, pass what it returned here and to the step: without it the sum over the ranks is bounded and not
        the mean.  ``GaussianAdam.step(max_norm=..., grad_scale=...)`` does both at once."""
        scale = _positive_scale(grad_scale)
        norm = clip_grads_(self.views, max_norm / scale, norm_type)
        return norm if scale == 1.0 else norm.mul_(scale)

    def all_reduce(self, group=None, average: bool = True, method: str = "scatter_gather") -> float:
        """Sums the gradients over the ranks of ``group`` (``method``: see _sum_flat_over_ranks; two collectives on
        the one flat buffer by default) and returns the factor the
        optimiser step still has to apply: 1 / world size when every rank back-propagated its own
        un-normalised loss (``average``, the default: sum -> mean over ranks), 1.0 when the losses were
        already scaled so that their sum over ranks IS the wanted gradient (``average=False``: what
        ``multiview_step`` does, it divides every view's loss by the global view count).
        Without an initialised process group this is a no-op with factor 1."""
        if not (dist.is_available() and dist.is_initialized()):
            return 1.0
        world = dist.get_world_size(group)
        _sum_flat_over_ranks(self.flat, group, method)
        return 1.0 / world if average else 1.0


def all_reduce_gradients(params: Dict[str, torch.Tensor], group=None, average: bool = True,
                         method: str = "all_reduce") -> float:
    """Sums ``param.grad`` of every tensor over the ranks and returns the factor left for the optimiser step to
    apply: 1 / world size, or 1.0 with ``average=False`` (losses already normalised over all ranks' views, as
    ``multiview_step`` does; see GradArena.all_reduce).  ``method="all_reduce"``: one collective per tensor, all in
    flight together (the 45-coefficient SH gradient is 3/4 of the bytes; coalescing the small ones buys nothing
    next to it).  ``"scatter_gather"`` / ``"direct"``: the gradients are packed into one flat buffer, exchanged as
    GradArena does, and unpacked (two extra copies of the gradients; gradients that already sit in a GradArena
    skip them: use its ``all_reduce``)."""
    if not (dist.is_available() and dist.is_initialized()):
        return 1.0
    world = dist.get_world_size(group)
    if world > 1 and method != "all_reduce":
        have = {k: p for k, p in params.items() if p.grad is not None}
        if have:
            arena = GradArena({k: p.grad for k, p in have.items()})
            for k, p in have.items():
                arena.views[k].copy_(p.grad)
            _sum_flat_over_ranks(arena.flat, group, method)
            for k, p in have.items():
                p.grad.copy_(arena.views[k])
    elif world > 1:
        host_side = dist.get_backend(group) == "gloo"
        pending = []
        for p in params.values():
            if p.grad is None:
                continue
            if host_side and p.grad.is_cuda:
                h = p.grad.cpu()                            # gloo only ever sees host tensors
                dist.all_reduce(h, op=dist.ReduceOp.SUM, group=group)
                p.grad.copy_(h)
            else:
                pending.append(dist.all_reduce(p.grad, op=dist.ReduceOp.SUM, group=group, async_op=True))
        for w in pending:
            w.wait()
    return 1.0 / world if average else 1.0


def _norm_code(norm_type: float) -> int:
    code = _NORMS.get(float(norm_type))
    if code is None:
        raise ValueError(f"norm_type must be 1, 2 or infinity, got {norm_type}")
    return code


def _positive_scale(grad_scale: float) -> float:
    grad_scale = float(grad_scale)
    if not 0.0 < grad_scale < math.inf:
        raise ValueError(f"grad_scale must be positive and finite, got {grad_scale}")
    return grad_scale


class _GradList:
    """The tensors of ``grads``, checked (on one GPU, of a type the kernels read), and their descriptors.

    Attribute by attribute, because a loop over the tensors takes twice as long: 0.3 us a tensor."""

    def __init__(self, grads: Grads):
        if isinstance(grads, torch.Tensor):
            grads = (grads,)
        elif isinstance(grads, dict):
            grads = grads.values()
        self.tensors = out = [g for g in grads if g is not None]
        if not out:
            raise ValueError("no gradients given")
        dtypes = [g.dtype for g in out]
        kinds = set(dtypes)
        if not _TYPES.keys() >= kinds:
            raise TypeError(f"gradients must be float32, float16 or bfloat16, got {sorted(map(str, kinds - _TYPES.keys()))}")
        devices = {g.get_device() for g in out}
        try:
            self.packed = all([g.is_contiguous() for g in out])
            pointers = [g.data_ptr() for g in out]
        except RuntimeError:                       # neither has an answer for sparse layouts
            pointers = None
        if pointers is None or -1 in devices:
            raise ValueError(f"gradients must be dense tensors on the GPU, got {[(str(g.layout), str(g.device)) for g in out][:8]}")
        if len(devices) > 1:
            raise ValueError(f"gradients are on GPUs {sorted(devices)}: one call works on one GPU")
        self.device = out[0].device
        self.words = words = [0] * (3 * len(out))  # a GsrGrad each
        words[0::3] = pointers
        words[1::3] = [g.numel() for g in out]
        words[2::3] = [_TYPES[d] for d in dtypes]

    def run(self, what: str, fn, code: int, *bound: float) -> torch.Tensor:
        """One norm or clipping call, on the current stream of the tensors' GPU."""
        dev, n = self.device, len(self.tensors)
        with _dgr._on_device(dev.index):
            nb = _lib.gsr_grad_norm_bytes(n)
            scratch = torch.empty((nb,), dtype=torch.uint8, device=dev)
            norm = torch.empty((), dtype=torch.float32, device=dev)
            _dgr._run(what, fn, n, struct.pack(f"{3 * n}Q", *self.words), code, *bound, norm.data_ptr(), scratch.data_ptr(), nb,
                      _dgr._raw_stream(dev.index))
        return norm


def _fills_its_memory(t: torch.Tensor) -> bool:
    """Whether the elements, in whatever order of dimensions, fill one stretch of memory without gaps."""
    if t.is_contiguous():
        return True
    order = sorted(range(t.dim()), key=lambda d: (t.stride(d), t.size(d)), reverse=True)
    return t.permute(order).is_contiguous()


def _shares_elements(t: torch.Tensor) -> bool:
    """Whether two elements may lie at one address (an expanded tensor, or one of overlapping windows)."""
    reach = 0
    for stride, size in sorted((t.stride(d), t.size(d)) for d in range(t.dim()) if t.size(d) > 1):
        if stride <= reach:
            return True
        reach += (size - 1) * stride
    return False


def _dims(t: torch.Tensor) -> List[tuple]:
    """(stride in bytes, size) of ``t``'s dimensions, the longest stride first; those of one element left out."""
    return sorted(((t.stride(d) * t.element_size(), t.size(d)) for d in range(t.dim()) if t.size(d) > 1), reverse=True)


def _touches(t: torch.Tensor, begin: int, end: int) -> bool:
    """Whether any byte of ``t``'s elements, no two of which share memory, lies in [begin, end).

    Such elements lie in the order of their indices, longest stride first, so those that begin before an address are
    counted dimension by dimension."""
    dims = _dims(t)

    def begin_before(address: int) -> int:
        offset, count = address - t.data_ptr(), 0
        if offset <= 0 or not t.numel():
            return 0
        inner = t.numel()
        for stride, size in dims:
            inner //= size
            whole = min(offset // stride, size)              # of them begin and end their inner dimensions before it
            count += whole * inner
            if whole == size:
                return count
            offset -= whole * stride
        return count + (offset > 0)

    return begin < end and begin_before(end) > begin_before(begin - t.element_size() + 1)


def _any_stretch_touches(packed: Iterable[torch.Tensor], gapped: Iterable[torch.Tensor]) -> bool:
    """Whether one of ``packed``, each of which fills a stretch of memory, shares an element with one of ``gapped``.
    (Two of ``packed`` that overlap are the library's to refuse.)"""
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in packed if t.numel())
    begins, ends = [b for b, _ in spans], [e for _, e in spans]
    for t in gapped:
        last = t.data_ptr() + sum(stride * (size - 1) for stride, size in _dims(t)) + t.element_size()
        near = spans[bisect_right(ends, t.data_ptr()):bisect_left(begins, last)]
        if any(_touches(t, b, e) for b, e in near):
            return True
    return False


def grad_norm(grads: Grads, norm_type: float = 2.0) -> torch.Tensor:
    """The norm of all gradients together, as a float32 scalar on their GPU; nothing waits for it.

    ``grads``: a tensor, an iterable or a dictionary of tensors (entries that are None are left out), float32, float16
    and bfloat16 mixed as they come, of any shape and strides.  ``norm_type``: 2 (root of the sum of squares), 1 (sum
    of magnitudes) or infinity (the largest magnitude).  Sums are held in 64 bits; a NaN anywhere gives NaN.
    A tensor that is given twice counts twice.  No gradient flows through the norm."""
    code, listed = _norm_code(norm_type), _GradList(grads)
    if not listed.packed:
        listed = _GradList([g if _fills_its_memory(g) else g.detach().contiguous() for g in listed.tensors])
    return listed.run("grad_norm", _lib.gsr_grad_norm, code)


def clip_grads_(grads: Grads, max_norm: float, norm_type: float = 2.0) -> torch.Tensor:
    """Scales all gradients in place by ``min(1, max_norm / (norm + 1e-6))`` (the rule of
    ``torch.nn.utils.clip_grad_norm_``) and returns the norm they had, a float32 scalar on their GPU.

    Arguments as ``grad_norm``'s; two tensors that share memory, or one that shares it with itself (expanded), are
    refused, with one exception: two tensors that BOTH have gaps between their elements are not compared, and an element
    that they share counts twice and is scaled once.
    The product is formed in float32 and rounded to the gradient's type.  The factor of float32 gradients is formed in 64
    bits and rounded once; float16 and bfloat16 ones take torch's, ``(norm + 1e-6).reciprocal() * max_norm`` in float32
    throughout, and with it torch's roundings, element by element.  A NaN norm makes every
    element NaN and an infinite one the finite elements 0, as there: look at the returned norm, or step with
    ``GaussianAdam.step(max_norm=..., skip_nonfinite=True)`` instead.
    An infinite ``max_norm`` scales nothing."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0, got {max_norm}")
    code, listed = _norm_code(norm_type), _GradList(grads)
    tensors = listed.tensors
    if listed.packed:
        norm = listed.run("clip_grads", _lib.gsr_clip_grads, code, max_norm)
    else:
        # a tensor with gaps between its elements is scaled as a copy without them and copied back
        staged = [None if _fills_its_memory(g) else g.detach().contiguous() for g in tensors]
        for g, copy in zip(tensors, staged):
            if copy is not None and _shares_elements(g):
                raise ValueError(f"a gradient of shape {tuple(g.shape)} and strides {g.stride()} has elements that may share memory")
        if _any_stretch_touches([g for g, copy in zip(tensors, staged) if copy is None],
                                [g for g, copy in zip(tensors, staged) if copy is not None]):
            raise ValueError("two gradients of the list share memory: one that fills its memory, and one with gaps")
        listed = _GradList([g if copy is None else copy for g, copy in zip(tensors, staged)])
        norm = listed.run("clip_grads", _lib.gsr_clip_grads, code, max_norm)
        for g, copy in zip(tensors, staged):
            if copy is not None:
                g.detach().copy_(copy)
    torch.autograd.graph.increment_version(tensors)          # written behind autograd's back
    return norm


class GaussianAdam:
    """torch.optim.Adam as the reference configures it (scene/gaussian_model.py:154-163), fused.

    ``params``: name -> tensor, in the reference's group names (xyz, f_dc, f_rest, opacity, scaling,
    rotation); ``lrs``: name -> learning rate.  State (exp_avg, exp_avg_sq, step) is what
    torch.optim.Adam keeps per parameter; ``state_dict`` / ``load_state_dict`` exchange it in that
    optimiser's layout."""

    def __init__(self, params: Dict[str, torch.Tensor], lrs: Dict[str, float], betas=(0.9, 0.999),
                 eps: float = 1e-15):
        if len(params) > MAX_TENSORS:
            raise ValueError(f"at most {MAX_TENSORS} tensors per fused step")
        for name, p in params.items():
            if p.dtype != torch.float32 or not p.is_contiguous():
                raise ValueError(f"{name}: parameters must be contiguous float32 tensors")
        self.params, self.lrs = dict(params), dict(lrs)
        self.betas, self.eps = betas, eps
        self.step_count = 0
        self.exp_avg = {k: torch.zeros_like(p) for k, p in params.items()}
        self.exp_avg_sq = {k: torch.zeros_like(p) for k, p in params.items()}

    @classmethod
    def for_model(cls, model, opt: Optional[OptimizationParams] = None, spatial_lr_scale: float = 1.0):
        """The six groups of training_setup (scene/gaussian_model.py:154-161)."""
        opt = opt or OptimizationParams()
        params = {"xyz": model._xyz, "f_dc": model._features_dc, "f_rest": model._features_rest,
                  "opacity": model._opacity, "scaling": model._scaling, "rotation": model._rotation}
        lrs = {"xyz": opt.position_lr_init * spatial_lr_scale, "f_dc": opt.feature_lr, "f_rest": opt.feature_lr / 20.0,
               "opacity": opt.opacity_lr, "scaling": opt.scaling_lr, "rotation": opt.rotation_lr}
        o = cls(params, lrs)
        o.schedule = (opt.position_lr_init * spatial_lr_scale, opt.position_lr_final * spatial_lr_scale,
                      opt.position_lr_delay_mult, opt.position_lr_max_steps)
        return o

    def update_learning_rate(self, iteration: int) -> float:
        """scene/gaussian_model.py:169-175: only the position group is scheduled."""
        lr_init, lr_final, mult, max_steps = self.schedule
        lr = expon_lr(iteration, lr_init, lr_final, lr_delay_mult=mult, max_steps=max_steps)
        self.lrs["xyz"] = lr
        return lr

    # ---- the optimiser surgery of densification (scene/gaussian_model.py:258-327): the number of Gaussians
    # changes between steps, the moments of the survivors stay ------------------------------------------------
    @torch.no_grad()
    def replace_tensor(self, name: str, tensor: torch.Tensor) -> torch.nn.Parameter:
        """replace_tensor_to_optimizer (:258-271): a new value for one tensor, its moments start again at zero,
        the step count stays (torch.optim.Adam keeps ``state["step"]`` there too)."""
        p = torch.nn.Parameter(tensor.detach().contiguous().requires_grad_(True))
        self.params[name] = p
        self.exp_avg[name] = torch.zeros_like(p)
        self.exp_avg_sq[name] = torch.zeros_like(p)
        return p

    @torch.no_grad()
    def prune(self, keep: torch.Tensor) -> Dict[str, torch.nn.Parameter]:
        """_prune_optimizer (:273-289): keeps the rows selected by the boolean mask ``keep`` of every tensor and
        of both moments; returns the new parameters by group name."""
        if self._moves_rows_on_the_gpu(keep):
            return self._move_rows(keep, None)
        for name, p in self.params.items():
            self.exp_avg[name] = self.exp_avg[name][keep].contiguous()
            self.exp_avg_sq[name] = self.exp_avg_sq[name][keep].contiguous()
            self.params[name] = torch.nn.Parameter(p.detach()[keep].contiguous().requires_grad_(True))
        return dict(self.params)

    def _moves_rows_on_the_gpu(self, keep: torch.Tensor) -> bool:
        """Whether ``keep`` and every tensor are what ``compact_rows`` moves: one bool per row, on one GPU."""
        state = [t for group in (self.params, self.exp_avg, self.exp_avg_sq) for t in group.values()]
        return (len(state) > 0 and keep.dtype == torch.bool and keep.dim() == 1 and keep.is_cuda
                and all(t.device == keep.device and t.dim() > 0 and t.shape[0] == keep.shape[0] for t in state))

    @torch.no_grad()
    def refine(self, keep: torch.Tensor, extension: Optional[Dict[str, torch.Tensor]] = None) -> Dict[str, torch.nn.Parameter]:
        """``cat_tensors(extension)`` and then ``prune(keep)``, in one pass: ``keep`` has one bool per row, the old
        ones first and the appended ones behind them.  On the GPU the parameters and each of the moments are moved by a
        launch each and the concatenations are never built (``gsplat_host.rows.compact_rows``).  Arguments that do not fit
        are refused before anything changes.  Where memory ends between two of the launches the parameters stay as they
        are and their moments start again at zero."""
        if extension is not None and set(extension) != set(self.params):
            raise ValueError(f"extension must name every tensor: {sorted(self.params)}")
        own_steps = type(self).prune is GaussianAdam.prune and type(self).cat_tensors is GaussianAdam.cat_tensors
        if keep.is_cuda and own_steps:
            return self._move_rows(keep, extension)
        extra = 0
        for n, p in self.params.items():           # nothing has been appended when a call is refused
            if extension is not None:
                extra = next(iter(extension.values())).shape[0]
                if extension[n].shape != (extra, *p.shape[1:]) or extension[n].device != p.device:
                    raise ValueError(f"{n}: appended rows of shape {tuple(extension[n].shape)} on {extension[n].device} do not "
                                     f"fit {extra} rows of a tensor of shape {tuple(p.shape)} on {p.device}")
            if keep.dtype != torch.bool or keep.shape != (p.shape[0] + extra,):
                raise ValueError(f"keep must have a bool for each of {p.shape[0]} + {extra} rows, got {keep.dtype} of shape "
                                 f"{tuple(keep.shape)}")
        if extension is not None:                  # a subclass may do more in these
            self.cat_tensors(extension)
        return self.prune(keep)

    def _move_rows(self, keep: torch.Tensor, extension: Optional[Dict[str, torch.Tensor]]) -> Dict[str, torch.nn.Parameter]:
        """``refine`` on the GPU."""
        from . import rows
        names = list(self.params)
        new, nothing = [None] * len(names), [None] * len(names)
        if extension is not None:
            new = [extension[n].detach().to(self.params[n].dtype) for n in names]
        groups = (self.exp_avg, self.exp_avg_sq, self.params)
        _, _, _, _, extra = rows._checked_compaction([g[n].detach() for g in groups for n in names], keep,
                                                     None if extension is None else nothing + nothing + new)
        # group by group, so that the old moments go as the new ones come: a third of the state on top of it at the peak
        # and not all of it (the old parameters are the caller's until it takes the new ones)
        moved, index = rows.compact_rows([self.exp_avg[n] for n in names], keep, nothing)
        self.exp_avg.update(zip(names, moved))
        try:
            moved = rows._again([self.exp_avg_sq[n] for n in names], index, nothing, extra)
            self.exp_avg_sq.update(zip(names, moved))
            moved = rows._again([self.params[n].detach() for n in names], index, new, extra)
        except BaseException:
            # the old moments are gone and the parameters are as they were: their moments start again
            moved = index = None
            for moments in (self.exp_avg, self.exp_avg_sq):
                moments.clear()
                moments.update((n, torch.zeros_like(p)) for n, p in self.params.items())
            raise
        self.params.update([(n, torch.nn.Parameter(t.requires_grad_(True))) for n, t in zip(names, moved)])
        return dict(self.params)

    @torch.no_grad()
    def cat_tensors(self, extension: Dict[str, torch.Tensor]) -> Dict[str, torch.nn.Parameter]:
        """cat_tensors_to_optimizer (:307-327): appends rows to every tensor; the new rows' moments are zero."""
        if set(extension) != set(self.params):
            raise ValueError(f"extension must name every tensor: {sorted(self.params)}")
        for name, p in self.params.items():
            ext = extension[name].detach().to(p.dtype)
            self.exp_avg[name] = torch.cat((self.exp_avg[name], torch.zeros_like(ext)), dim=0)
            self.exp_avg_sq[name] = torch.cat((self.exp_avg_sq[name], torch.zeros_like(ext)), dim=0)
            self.params[name] = torch.nn.Parameter(torch.cat((p.detach(), ext), dim=0).contiguous().requires_grad_(True))
        return dict(self.params)

    # ---- checkpoints: torch.optim.Adam's own layout (what the reference saves, scene/gaussian_model.py:73) ----
    def state_dict(self) -> dict:
        """The dictionary ``torch.optim.Adam(...).state_dict()`` returns for the reference's six groups
        (scene/gaussian_model.py:154-163): per parameter ``step`` / ``exp_avg`` / ``exp_avg_sq``, per group the
        hyper-parameters, ``name`` and the parameter's index."""
        names = list(self.params)
        state = {}
        if self.step_count > 0:
            for i, n in enumerate(names):
                state[i] = {"step": torch.tensor(float(self.step_count)), "exp_avg": self.exp_avg[n],
                            "exp_avg_sq": self.exp_avg_sq[n]}
        groups = [{"lr": float(self.lrs[n]), "name": n, "betas": tuple(self.betas), "eps": self.eps, "weight_decay": 0,
                   "amsgrad": False, "maximize": False, "foreach": None, "capturable": False, "differentiable": False,
                   "fused": None, "params": [i]} for i, n in enumerate(names)]
        return {"state": state, "param_groups": groups}

    @torch.no_grad()
    def load_state_dict(self, sd: dict) -> None:
        """Takes the moments, the step count and the learning rates from a ``torch.optim.Adam`` state dictionary
        whose groups carry the reference's names (or come in the same order)."""
        groups = sd["param_groups"]
        if len(groups) != len(self.params):
            raise ValueError(f"{len(groups)} parameter groups for {len(self.params)} tensors")
        steps = set()
        for i, (g, own) in enumerate(zip(groups, list(self.params))):
            name = g.get("name", own)
            if name not in self.params:
                raise ValueError(f"unknown parameter group {name!r}")
            if len(g["params"]) != 1:
                raise ValueError("one tensor per group, as the reference sets them up")
            p = self.params[name]
            self.lrs[name] = float(g["lr"])
            st = sd["state"].get(g["params"][0])
            if st is None:
                self.exp_avg[name], self.exp_avg_sq[name] = torch.zeros_like(p), torch.zeros_like(p)
                continue
            for key, store in (("exp_avg", self.exp_avg), ("exp_avg_sq", self.exp_avg_sq)):
                t = st[key]
                if tuple(t.shape) != tuple(p.shape):
                    raise ValueError(f"{name}.{key}: shape {tuple(t.shape)} does not match the parameter's {tuple(p.shape)}")
                store[name] = t.detach().to(device=p.device, dtype=torch.float32).contiguous().clone()
            steps.add(int(float(st["step"])))
        if len(steps) > 1:
            raise ValueError(f"the groups were stepped {sorted(steps)} times: one fused step cannot continue that")
        self.step_count = steps.pop() if steps else 0
        if groups and "betas" in groups[0]:
            self.betas, self.eps = tuple(groups[0]["betas"]), float(groups[0]["eps"])

    @torch.no_grad()
    def step(self, grads: Optional[Dict[str, torch.Tensor]] = None, grad_scale: float = 1.0,
             max_norm: Optional[float] = None, norm_type: float = 2.0, skip_nonfinite: bool = False) -> Optional[torch.Tensor]:
        """One Adam update of every tensor that has a gradient (``grads[name]`` or ``param.grad``).

        With ``max_norm`` the norm of all gradients of the step, after ``grad_scale``, is bounded first, as
        ``clip_grads_`` would (``norm_type`` as there), in the same two launches and without touching the gradients,
        which may then be float32, float16 or bfloat16; the step returns the norm, a float32 scalar on the GPU.
        ``max_norm=math.inf`` only measures.  ``skip_nonfinite`` (with ``max_norm``): a step whose norm is infinite or
        NaN (in the 64 bits it is summed in, so only where an element is) leaves parameters and moments as they are;
        ``step_count`` counts it.  A step captured into a graph repeats the bias corrections of the count it was captured
        with."""
        for name, p in self.params.items():
            if not p.is_cuda:
                raise ValueError(f"{name}: the fused update runs on the GPU only, the parameter is on {p.device}")
        if max_norm is None:
            if skip_nonfinite:
                raise ValueError("skip_nonfinite needs max_norm: a step without it does not look at the gradients first")
        else:
            max_norm, code = float(max_norm), _norm_code(norm_type)
            if not max_norm >= 0.0:
                raise ValueError(f"max_norm must be at least 0, got {max_norm}")
        rows: List[tuple] = []                     # the fields of a GsrAdamTensor each
        types: List[int] = []
        dev = next(iter(self.params.values())).device if self.params else torch.device("cuda", torch.cuda.current_device())
        keep: List[torch.Tensor] = []
        for name, p in self.params.items():
            g = grads[name] if grads is not None else p.grad
            if g is None:
                continue
            n = p.numel()
            if g.numel() != n:
                raise ValueError(f"{name}: gradient has {g.numel()} elements, parameter {n}")
            if n == 0:
                continue
            if g.is_neg():                         # a negated view's memory holds the opposite of its values
                g = g.resolve_neg()
            if max_norm is None:
                g = _dgr._f32(g, f"grad of {name}")
            else:
                kind = _TYPES.get(g.dtype)
                if kind is None:
                    raise TypeError(f"grad of {name} must be float32, float16 or bfloat16, got {g.dtype}")
                if g.device != dev or p.device != dev:
                    raise ValueError(f"{name}: parameter and gradient must be on {dev}, they are on {p.device} and {g.device}")
                types.append(kind)
                g = g.contiguous()
            keep.append(g)
            rows.append((p.data_ptr(), g.data_ptr(), self.exp_avg[name].data_ptr(), self.exp_avg_sq[name].data_ptr(), n,
                         float(self.lrs[name]), 0))
        self.step_count += 1
        if max_norm is None:
            _dgr._run("adam_step", _lib.gsr_adam_step, len(rows), (_AdamTensor * MAX_TENSORS)(*rows), float(self.betas[0]),
                      float(self.betas[1]), float(self.eps), int(self.step_count), float(grad_scale), _dgr._stream())
            return None
        with _dgr._on_device(dev.index):
            count = len(rows)
            nb = _lib.gsr_grad_norm_bytes(count)
            scratch = torch.empty((nb,), dtype=torch.uint8, device=dev)
            norm = torch.empty((), dtype=torch.float32, device=dev)
            _dgr._run("adam_step", _lib.gsr_adam_step_clipped, count, struct.pack("5Qfi" * count, *chain.from_iterable(rows)),
                      struct.pack(f"{count}i", *types), float(self.betas[0]), float(self.betas[1]), float(self.eps),
                      int(self.step_count), float(grad_scale), code, max_norm, int(bool(skip_nonfinite)), norm.data_ptr(),
                      scratch.data_ptr(), nb, _dgr._raw_stream(dev.index))
        return norm

    def zero_grad(self, set_to_none: bool = True) -> None:
        """train.py:128."""
        for p in self.params.values():
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()
