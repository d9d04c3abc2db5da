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


def _rotary_args(at, **change):
    a = _lib.RotaryArgs()
    a.type, a.batch, a.tokens, a.dim, a.axes, a.tensors, a.base, a.position_type = 0, 1, 2, 16, 2, 2, 1e4, 3
    a.axis_dim[:2] = (8, 8)
    a.heads[:] = (1, 1)
    a.positions = at
    a.x[:], a.out[:] = (at, at + 16), (at + 32, at + 48)
    for k, v in change.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [dict(type=3), dict(position_type=1), dict(batch=-1), dict(tokens=-1), dict(dim=0), dict(dim=514), dict(dim=8),
                                    dict(axes=0), dict(axes=5), dict(axis_dim=(0, 7)), dict(axis_dim=(0, 0)), dict(axis_dim=(1, 10)),
                                    dict(tensors=0), dict(tensors=3), dict(base=1.0), dict(base=math.inf), dict(base=math.nan), dict(positions=None),
                                    dict(x=(1, None)), dict(out=(0, None)), dict(heads=(1, 0)), dict(heads=(0, 70000))])
def test_rotary_refuses(change):
    keep, base = _aligned()
    assert _lib.lib().ddpm_rotary(C.byref(_rotary_args(base, **change)), None) == -1
    assert _lib.lib().ddpm_last_error()


def test_rotary_refuses_overlap_null_and_misaligned():
    keep, base = _aligned()
    L = _lib.lib()
    assert L.ddpm_rotary(None, None) == -1
    assert L.ddpm_rotary(C.byref(_rotary_args(base, out=(0, base))), None) == -1
    assert L.ddpm_rotary(C.byref(_rotary_args(base, x=(0, base + 2))), None) == -1
    assert L.ddpm_rotary(C.byref(_rotary_args(base, batch=0)), None) == 0          # nothing to do


def test_rotary_function_refuses():
    from diffusion_model_amd.embedding import grid_positions, rotary
    q, k, pos = torch.zeros(2, 6, 4, 16), torch.zeros(2, 6, 2, 16), grid_positions(2, 3, device="cpu")
    assert pos.tolist() == [[0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]
    for args, error in (((q[0], k, pos, (8, 8)), ValueError), ((q, k.double(), pos, (8, 8)), TypeError), ((q.double(), None, pos, (8, 8)), TypeError),
                        ((q, k[:, :5], pos, (8, 8)), ValueError), ((q, k, pos, (8, 10)), ValueError), ((q, k, pos, (7, 8)), ValueError),
                        ((q, k, pos, ()), ValueError), ((q, k, pos, (16,)), ValueError), ((q, k, pos[:5], (8, 8)), ValueError),
                        ((q, k, pos.double(), (8, 8)), TypeError), ((q, k, pos.float().requires_grad_(True), (8, 8)), TypeError),
                        ((q, k, pos, (8, 8)), RuntimeError), ((torch.zeros(1, 6, 1, 514), None, pos, (8, 8)), ValueError)):
        with pytest.raises(error):
            rotary(*args)
    with pytest.raises(ValueError):
        grid_positions()
    with pytest.raises(ValueError):
        grid_positions(3, 0, device="cpu")


def _span_args(at, **change):
    a = _lib.SpanAttentionArgs()
    a.type, a.batch, a.nq, a.nk, a.heads, a.kv_heads, a.dim, a.scale = 0, 1, 4, 4, 2, 1, 8, 0.5
    for name in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, name, at)
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv"):
        getattr(a, name + "_stride")[:] = (64, 16, 8)
    for k, v in change.items():
        if isinstance(v, tuple):
            getattr(a, k)[v[0]] = v[1]
        else:
            setattr(a, k, v)
    return a


@pytest.mark.parametrize("change", [dict(type=3), dict(type=-1), dict(batch=-1), dict(heads=65536, kv_heads=65536), dict(nq=-1), dict(nk=-1), dict(nk=(1 << 30) + 1),
                                    dict(heads=0), dict(heads=3, kv_heads=2), dict(kv_heads=0), dict(dim=0), dict(dim=10), dict(dim=132), dict(softcap=-1.0),
                                    dict(softcap=1e-31), dict(softcap=1e-3, scale=1e28), dict(softcap=math.nan), dict(scale=math.inf), dict(scale=math.nan), dict(q_stride=(1, 17)), dict(k_stride=(0, 2)),
                                    dict(v_stride=(2, 1)), dict(out_stride=(1, 3)), dict(type=1, dim=12), dict(type=1, q_stride=(1, 12))])
def test_span_attention_refuses_sizes(change):
    keep, base = _aligned()
    L, a, ws = _lib.lib(), _span_args(base, **change), C.c_void_p(base)
    assert L.ddpm_span_attention_fwd(C.byref(a), ws, None) == -1
    assert L.ddpm_span_attention_bwd(C.byref(a), ws, None) == -1
    assert L.ddpm_span_attention_fwd_workspace(C.byref(a)) < 0 and L.ddpm_span_attention_bwd_workspace(C.byref(a)) < 0
    assert L.ddpm_last_error()


def test_span_attention_refuses_pointers():
    keep, base = _aligned()
    L, ws = _lib.lib(), C.c_void_p(base)
    for name in ("q", "k", "v", "out"):
        for bad in (None, base + 4):
            a = _span_args(base, **{name: bad})
            assert L.ddpm_span_attention_fwd(C.byref(a), ws, None) == -1, name
            assert L.ddpm_span_attention_bwd(C.byref(a), ws, None) == -1, name
    for name in ("lse", "dout", "dq", "dk", "dv"):
        assert L.ddpm_span_attention_bwd(C.byref(_span_args(base, **{name: None})), ws, None) == -1, name
    assert L.ddpm_span_attention_bwd(C.byref(_span_args(base, dout_stride=(1, 2))), ws, None) == -1
    assert L.ddpm_span_attention_bwd(C.byref(_span_args(base)), None, None) == -1
    assert L.ddpm_span_attention_bwd(C.byref(_span_args(base)), C.c_void_p(base + 4), None) == -1
    few = _span_args(base, nq=1, nk=100000)
    assert L.ddpm_span_attention_fwd_workspace(C.byref(few)) > 0
    assert L.ddpm_span_attention_fwd(C.byref(few), None, None) == -1          # a split call needs its workspace
    for f in (L.ddpm_span_attention_fwd, L.ddpm_span_attention_bwd):
        assert f(None, ws, None) == -1
        assert f(C.byref(_span_args(base, batch=0)), ws, None) == 0           # nothing to do


def test_span_attention_function_refuses():
    from diffusion_model_amd.attention import span_attention
    q, k = torch.zeros(2, 6, 4, 16), torch.zeros(2, 9, 2, 16)
    ok = dict(slopes=torch.zeros(4), spans=torch.zeros(2, 6, 2, dtype=torch.int32), positions=torch.zeros(6, dtype=torch.int32))
    for args, how, error in (((q[0], k, k), {}, ValueError), ((q, k, k.half()), {}, TypeError), ((q.double(), k.double(), k.double()), {}, TypeError),
                             ((q, k, k[:, :8]), {}, ValueError), ((q, k[:1], k[:1]), {}, ValueError), ((q[:, :, :3], k, k), {}, ValueError),
                             ((torch.zeros(2, 6, 4, 136), torch.zeros(2, 9, 2, 136), torch.zeros(2, 9, 2, 136)), {}, ValueError),
                             ((q, k, k), dict(softcap=-1.0), ValueError), ((q, k, k), dict(softcap=1e-31), ValueError),
                             ((q, k, k), dict(softcap=1e-3, scale=1e28), ValueError), ((q, k, k), dict(softcap=math.nan), ValueError),
                             ((q, k, k), dict(scale=math.inf), ValueError), ((q, k, k), dict(slopes=torch.zeros(2)), ValueError),
                             ((q, k, k), dict(slopes=torch.zeros(4).double()), ValueError),
                             ((q, k, k), dict(slopes=torch.zeros(4).requires_grad_(True)), NotImplementedError),
                             ((q, k, k), dict(spans=torch.zeros(2, 6, 2)), ValueError), ((q, k, k), dict(spans=torch.zeros(3, 6, 2).int()), ValueError),
                             ((q, k, k), dict(spans=torch.zeros(6, 2).int()), ValueError), ((q, k, k), dict(positions=torch.zeros(2, 5).int()), ValueError),
                             ((q, k, k), dict(positions=torch.zeros(6)), ValueError), ((q, k, k), ok, RuntimeError)):
        with pytest.raises(error):
            span_attention(*args, **how)


def test_key_spans():
    from diffusion_model_amd.attention import key_spans
    ids = torch.tensor([[5, 5, 2, 2, 2, 5], [1, 1, 1, 1, 1, 1]])
    assert key_spans(6, documents=ids).tolist() == [[[0, 2], [0, 2], [2, 5], [2, 5], [2, 5], [5, 6]], [[0, 6]] * 6]
    assert key_spans(6, documents=ids[0], causal=True).tolist() == [[[0, 1], [0, 2], [2, 3], [2, 4], [2, 5], [5, 6]]]
    assert key_spans(6, documents=ids[0], prefix=2).tolist() == [[[0, 2], [0, 2], [2, 4], [2, 4], [2, 5], [5, 6]]]
    assert key_spans(4, prefix=torch.tensor([0, 3, 9])).tolist() == [[[0, 1], [0, 2], [0, 3], [0, 4]], [[0, 3]] * 3 + [[0, 4]], [[0, 4]] * 4]
    assert key_spans(4, lengths=torch.tensor([0, 3])).tolist() == [[[0, 0]] * 4, [[0, 3]] * 3 + [[0, 0]]]
    assert key_spans(4, window=(1, 0), device="cpu").tolist() == [[[0, 1], [0, 2], [1, 3], [2, 4]]]
    assert key_spans(2, 5, causal=True, device="cpu").tolist() == [[[0, 4], [0, 5]]]
    assert key_spans(2, 5, documents=ids[0, :5]).tolist() == [[[2, 5], [2, 5]]]
    assert key_spans(3, 1, documents=ids[0, :1]).tolist() == [[[0, 0], [0, 0], [0, 1]]]
    assert key_spans(0, device="cpu").shape == (1, 0, 2) and key_spans(0, documents=ids[:, :0]).shape == (2, 0, 2)
    assert key_spans(4, device="cpu").dtype == torch.int32
    for bad in (dict(documents=ids[:, :5]), dict(documents=ids[None])):
        with pytest.raises(ValueError):
            key_spans(6, **bad)
    with pytest.raises(ValueError):
        key_spans(-1)


def test_reference_gradient_against_differences():
    """The float64 reference that the GPU tests compare with, against central differences of itself: step 1e-5, so that truncation
    (1e-10) and cancellation (1e-11) stay below 1e-7."""
    import os
    import sys
    sys.path.insert(0, os.path.dirname(__file__))
    from span_reference import reference
    g = torch.Generator().manual_seed(0)
    q, k, v, dout = (torch.randn(1, n, h, 4, generator=g, dtype=torch.float64) for n, h in ((6, 4), (9, 2), (9, 2), (6, 4)))
    how = dict(softcap=3.0, slopes=torch.rand(4, generator=g), causal=True, spans=torch.tensor([[[0, 9], [2, 5], [0, 0], [1, 9], [3, 3], [0, 7]]]).int())
    want = reference(q, k, v, dout, **how)
    for x, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        e = torch.randn(x.shape, generator=g, dtype=torch.float64)
        at = [(reference(*(y + s * e if y is x else y for y in (q, k, v)), **how)["out"][0] * dout).sum() for s in (1e-5, -1e-5)]
        assert abs(float((at[0] - at[1]) / 2e-5 - (want[name][0] * e).sum())) < 1e-7
    assert (want["out"][0][:, [2, 4]] == 0).all() and (want["dq"][0][:, [2, 4]] == 0).all()


@pytest.mark.parametrize("layout", ["coo", "csr"])
def test_clip_refuses_sparse_gradients(layout):
    p = torch.nn.Parameter(torch.zeros(3, 4))
    q = torch.nn.Parameter(torch.zeros(3))
    dense = torch.eye(3, 4)
    q.grad = torch.ones(3)
    p.grad = dense.to_sparse()
    if layout == "csr":
        p = torch.nn.Parameter(torch.zeros(3, 4).to_sparse_csr())
        p.grad = dense.to_sparse_csr()
    for f in (lambda: optim.clip_grad_norm_([q, p], 1.0), lambda: optim.grad_norm([q, p])):
        with pytest.raises(RuntimeError, match="sparse"):
            f()
