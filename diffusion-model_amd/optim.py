"""`Adam`: torch.optim.Adam's update (the optimizer of the reference's training loops,
first-iteration/main.py:51,82-84; third-iteration/main.py:61) as one HIP launch per 88 tensors, and the global gradient
norm with clipping by it: `clip_grad_norm_` / `grad_norm` in front of any optimizer, or `Adam(..., max_grad_norm=...)` /
`adam_step_(..., max_norm=...)`, which scale the gradients as the update reads them instead of writing them first.

Same constructor arguments, same per-parameter state (`step`, `exp_avg`, `exp_avg_sq`) and the same
`state_dict()` layout as torch.optim.Adam, so optimizer checkpoints move both ways.  Parameters must be
contiguous fp32 tensors on the GPU; there is no CPU fallback.
"""
import ctypes as C
import math
from array import array
from itertools import chain
from operator import attrgetter

import torch

from ._lib import call, lib, on_gpu, stream_of

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # DDPM_F32, DDPM_BF16, DDPM_F16
_NORMS = {2.0: 0, math.inf: 1}                                        # DDPM_NORM_2, DDPM_NORM_MAX
_ptr, _numel, _contiguous, _gpu = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _grad = attrgetter("dtype"), attrgetter("grad")


def _array(code, values):
    """(address, owner) of a C array of `values`."""
    a = array(code, values)
    return C.c_void_p(a.buffer_info()[0]), a


def _one_gpu(what, tensors):
    """Index of the GPU that all of them are on."""
    gpus = set(map(_gpu, tensors))
    if len(gpus) != 1 or -1 in gpus:
        raise RuntimeError(f"{what} (HIP): all tensors must be on one GPU, got {sorted(str(t.device) for t in tensors)[:4]}")
    return gpus.pop()


def _distinct(what, pointers, sizes):
    """Tensors that a kernel writes must not be given twice; empty ones may share a pointer."""
    if len(set(pointers)) < len(pointers):
        real = [p for p, n in zip(pointers, sizes) if n]
        if len(set(real)) < len(real):
            raise ValueError(f"{what} (HIP): the same tensor is given twice")


class _Norm:
    """The gradients of one call as the C arrays of the norm and clipping entry points, and the norm itself:
    `state` holds [norm, factor] on the device. They must be contiguous, and different ones where `written` says that they will be
    scaled in place; where the caller has their pointers and sizes already it hands them in."""

    def __init__(self, what, grads, max_norm, norm_type, pointers=None, sizes=None, written=False):
        if norm_type not in _NORMS:
            raise NotImplementedError(f"{what} (HIP): norm_type must be 2 or inf, got {norm_type}")
        if not max_norm >= 0.0:
            raise ValueError(f"Invalid max_norm: {max_norm}")
        self.device = _one_gpu(what, grads)
        types = list(map(_TYPES.get, map(_dtype, grads)))
        if None in types:
            raise RuntimeError(f"{what} (HIP): gradients must be float32, bfloat16 or float16, got {sorted(map(str, set(map(_dtype, grads))))}")
        self.n = len(grads)
        if pointers is None:
            pointers, sizes = list(map(_ptr, grads)), list(map(_numel, grads))
        if written:
            _distinct(what, pointers, sizes)
        (self.pointers, a), (self.numel, b), (self.types, c) = _array("Q", pointers), _array("q", sizes), _array("i", types)
        self._owners = (a, b, c)
        with on_gpu(self.device):
            workspace = torch.empty(lib().ddpm_grad_norm_workspace_doubles(self.n), dtype=torch.float64, device="cuda")
            self.state = torch.empty(2, dtype=torch.float32, device="cuda")
            call("ddpm_grad_norm", self.n, self.pointers, self.numel, self.types, _NORMS[norm_type], float(max_norm),
                 C.c_void_p(workspace.data_ptr()), C.c_void_p(self.state.data_ptr()), stream_of(self.device))

    def factor(self):
        return C.c_void_p(self.state.data_ptr() + 4)


def _gradients(what, parameters):
    """(gradients, the same contiguous)"""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [g for g in map(_grad, parameters) if g is not None]
    try:
        dense = all(map(_contiguous, grads))                    # raises for a sparse one, which spares the others a question
    except (RuntimeError, NotImplementedError):
        dense = False
    if dense:
        return grads, grads
    if any(g.layout != torch.strided for g in grads):
        raise RuntimeError(f"{what} does not support sparse gradients")
    return grads, [g.contiguous() for g in grads]


@torch.no_grad()
def grad_norm(parameters, norm_type=2.0):
    """Norm of all gradients of `parameters` together (a 0-dim fp32 tensor on their GPU): the 2-norm, summed in float64
    in a fixed order, or with norm_type=inf the largest magnitude. The gradients stay as they are; one that several parameters
    share counts for each of them."""
    _, grads = _gradients("grad_norm", parameters)
    return _Norm("grad_norm", grads, math.inf, float(norm_type)).state[0] if grads else torch.tensor(0.0)


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ over fp32, bf16 and fp16 gradients on one GPU: scales all of them in place by
    min(1, max_norm / (norm + 1e-6)) and returns the norm before (0-dim fp32, on the device; nothing waits for it unless
    error_if_nonfinite is set). A norm that is not a number makes every gradient NaN, as there. Norms other than 2 and inf, and a
    gradient given twice, are refused; `foreach` chooses between torch's implementations, and here there is one."""
    grads, dense = _gradients("clip_grad_norm_", parameters)
    if not grads:
        return torch.tensor(0.0)
    norm = _Norm("clip_grad_norm_", dense, max_norm, float(norm_type), written=True)
    if error_if_nonfinite and not math.isfinite(norm.state[0].item()):
        raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot be clipped.")
    with on_gpu(norm.device):
        call("ddpm_clip_grads", norm.n, norm.pointers, norm.numel, norm.types, norm.factor(), stream_of(norm.device))
        if dense is not grads:
            for g, d in zip(grads, dense):
                if g is not d:
                    g.copy_(d)
    torch.autograd.graph.increment_version(grads)
    return norm.state[0]


def _update(lists, pointers, sizes, step, lr, beta1, beta2, eps, weight_decay, factor):
    """Launches the update of checked lists (parameters, gradients, exp_avg, exp_avg_sq) on the current GPU and stream."""
    arrays = [_array("Q", x) for x in pointers]
    numel = _array("q", sizes)
    args = (len(sizes), *(a[0] for a in arrays), numel[0], float(lr), float(beta1), float(beta2), float(eps), float(weight_decay), step)
    stream = stream_of(torch.cuda.current_device())
    if factor is None:
        call("ddpm_adam_step", *args, stream)
    else:
        call("ddpm_adam_step_clipped", *args, factor, stream)
    # the kernel wrote the tensors behind autograd's back: record the in-place change, as any in-place
    # torch op would (saved-tensor checks and caches keyed on the version counter rely on it)
    torch.autograd.graph.increment_version(list(chain(lists[0], lists[2], lists[3])))


@torch.no_grad()
def adam_step_(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, max_norm=None):
    """One Adam update of lists of contiguous fp32 tensors on one GPU, in place; `step` counts from 1, this update
    included. With max_norm the gradients count as if clip_grad_norm_(max_norm) had scaled them first; they themselves stay
    as they are, and their norm is returned (0-dim fp32 on the device; None without max_norm)."""
    lists = [list(x) for x in (params, grads, exp_avgs, exp_avg_sqs)]
    if len(set(map(len, lists))) != 1:
        raise ValueError(f"adam_step_: lists of different lengths {[len(x) for x in lists]}")
    if step < 1:
        raise ValueError(f"Invalid step: {step}")
    if not lists[0]:
        return None
    every = list(chain(*lists))
    gpu = _one_gpu("adam_step_", every)
    if set(map(_dtype, every)) != {torch.float32} or not all(map(_contiguous, every)):
        raise RuntimeError("adam_step_ (HIP): all tensors must be contiguous fp32")
    sizes = list(map(_numel, lists[0]))
    if any(list(map(_numel, x)) != sizes for x in lists[1:]):
        raise RuntimeError("adam_step_ (HIP): gradients and moments must match their parameters in size")
    pointers = [list(map(_ptr, x)) for x in lists]
    _distinct("adam_step_", pointers[0] + pointers[2] + pointers[3], sizes * 3)
    with on_gpu(gpu):
        norm = _Norm("adam_step_", lists[1], max_norm, 2.0, pointers[1], sizes) if max_norm is not None else None
        _update(lists, pointers, sizes, int(step), lr, *betas, eps, weight_decay, norm and norm.factor())
    return norm and norm.state[0]


class Adam(torch.optim.Optimizer):
    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False, *, maximize=False,
                 max_grad_norm=None):
        if not 0.0 <= lr:
            raise ValueError(f"Invalid learning rate: {lr}")
        if not 0.0 <= eps:
            raise ValueError(f"Invalid epsilon value: {eps}")
        if not 0.0 <= betas[0] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 0: {betas[0]}")
        if not 0.0 <= betas[1] < 1.0:
            raise ValueError(f"Invalid beta parameter at index 1: {betas[1]}")
        if not 0.0 <= weight_decay:
            raise ValueError(f"Invalid weight_decay value: {weight_decay}")
        if amsgrad or maximize:
            raise NotImplementedError("amsgrad / maximize are not part of the reference's optimizer and are not implemented")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError(f"Invalid max_grad_norm: {max_grad_norm}")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=False, maximize=False))
        # of the optimizer, not of its groups: the norm is that of all gradients together, and a state_dict keeps torch's keys
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None        # norm of the gradients of the last step (0-dim, on the device) with max_grad_norm

    # torch's optimizers take their groups and state along when copied or pickled, and nothing else
    def __getstate__(self):
        return {**super().__getstate__(), "max_grad_norm": self.max_grad_norm, "grad_norm": self.grad_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self.__dict__.setdefault("max_grad_norm", None)         # pickled before there was one
        self.__dict__.setdefault("grad_norm", None)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, entries = [], {}                                  # entries: of each parameter, so far, where some are listed twice
        listed = [id(p) for group in self.param_groups for p in group["params"]]
        repeated = len(set(listed)) < len(listed)
        for group in self.param_groups:
            by_step = {}
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.is_sparse:
                    raise RuntimeError("Adam does not support sparse gradients")
                if not (p.is_cuda and p.dtype == torch.float32 and p.is_contiguous()):
                    raise RuntimeError("Adam (HIP): parameters must be contiguous fp32 tensors on the GPU")
                if g.dtype != torch.float32 or g.device != p.device or g.shape != p.shape:
                    raise RuntimeError("Adam (HIP): gradient must match its parameter in dtype, device and shape")
                if not g.is_contiguous():
                    g = g.contiguous()
                st = self.state[p]
                if len(st) == 0:
                    st["step"] = torch.tensor(0.0, dtype=torch.float32)
                    st["exp_avg"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                    st["exp_avg_sq"] = torch.zeros_like(p, memory_format=torch.preserve_format)
                # a parameter that a group lists twice takes two steps, one launch behind the other: in one they would race
                step = int(st["step"].item()) + 1
                if repeated:
                    step += entries.get(p, 0)
                    entries[p] = entries.get(p, 0) + 1
                by_step.setdefault(step, []).append((p, g, st["exp_avg"], st["exp_avg_sq"]))
            work += [(group, step, items) for step, items in sorted(by_step.items())]
        norm = None
        if self.max_grad_norm is not None and work:
            norm = _Norm("Adam", list({t[0]: t[1] for _, _, items in work for t in items}.values()), self.max_grad_norm, 2.0)
            self.grad_norm = norm.state[0]
        for group, step, items in work:
            with on_gpu(items[0][0].get_device()):
                lists = [list(x) for x in zip(*items)]
                _update(lists, [list(map(_ptr, x)) for x in lists], list(map(_numel, lists[0])), step, group["lr"], *group["betas"], group["eps"], group["weight_decay"],
                        norm and norm.factor())
            for p, *_ in items:
                self.state[p]["step"] += 1
        return loss
