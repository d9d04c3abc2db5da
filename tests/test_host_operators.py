"""Refusals of the clipping, rotary and span attention operators: they come before any GPU call, so they are checked here, on a
machine without a GPU, through the C ABI and through the Python functions."""
import ctypes as C
import math

import pytest
import torch

from diffusion_model_amd import _lib, optim


def _aligned(n=256):
    buf = (C.c_char * (n + 64))()
    base = C.addressof(buf)
    return buf, base + (-base) % 64


@pytest.mark.parametrize("change", [dict(n=-1), dict(types=[3]), dict(types=[-1]), dict(numel=[-1]), dict(numel=[(1 << 36) + 1]), dict(ptr=0),
                                    dict(off=2), dict(kind=2), dict(kind=-1), dict(max_norm=-1.0), dict(max_norm=math.nan), dict(ws=False),
                                    dict(state=False), dict(lists=False)])
def test_grad_norm_refuses(change):
    a = dict(n=1, types=[0], numel=[4], ptr=1, off=0, kind=0, max_norm=1.0, ws=True, state=True, lists=True)
    a.update(change)
    keep, base = _aligned()
    ok = C.c_void_p(base)
    lists = ((C.c_void_p * 1)(base + a["off"] if a["ptr"] else 0), (C.c_int64 * 1)(*a["numel"]), (C.c_int32 * 1)(*a["types"])) if a["lists"] else (None,) * 3
    L = _lib.lib()
    assert L.ddpm_grad_norm(a["n"], *lists, a["kind"], a["max_norm"], ok if a["ws"] else None, ok if a["state"] else None, None) == -1
    assert L.ddpm_last_error()
    if not {"kind", "max_norm", "ws"} & set(change):
        assert L.ddpm_clip_grads(a["n"], *lists, ok if a["state"] else None, None) == -1


def test_clipped_adam_refuses_a_missing_factor_and_bad_scalars():
    L = _lib.lib()
    keep, base = _aligned()
    p, n = (C.c_void_p * 1)(base), (C.c_int64 * 1)(4)
    good = [1, p, p, p, p, n, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, C.c_void_p(base), None]
    for at, bad in ((12, None), (0, -1), (6, -1.0), (7, 1.0), (8, 1.0), (9, -1.0), (10, -1.0), (11, 0), (5, (C.c_int64 * 1)(-1)), (1, (C.c_void_p * 1)(0))):
        args = list(good)
        args[at] = bad
        assert L.ddpm_adam_step_clipped(*args) == -1, at


def test_clipping_functions_refuse_before_the_gpu():
    p = torch.nn.Parameter(torch.zeros(4))
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0           # no gradient: nothing to do
    assert float(optim.grad_norm([p])) == 0.0
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="on one GPU"):
        optim.clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        optim.clip_grad_norm_([p], math.nan)
    with pytest.raises(NotImplementedError, match="norm_type"):
        optim.clip_grad_norm_([p], 1.0, norm_type=1)
    with pytest.raises(ValueError, match="max_grad_norm"):
        optim.Adam([p], max_grad_norm=-1.0)
    t = [torch.zeros(4)]
    with pytest.raises(RuntimeError, match="on one GPU"):
        optim.adam_step_(t, t, t, t, 1)
    with pytest.raises(ValueError, match="different lengths"):
        optim.adam_step_(t, [], t, t, 1)
    with pytest.raises(ValueError, match="step"):
        optim.adam_step_(t, t, t, t, 0)
    assert optim.adam_step_([], [], [], [], 1, max_norm=1.0) is None
