"""Global gradient norm, clipping by it and the Adam step that takes the factor, against the formulas in float64.

Tolerances count roundings of half a step each: the norm is one fp32 rounding of a float64 result (2^-24; 2^-23 leaves room
for the float64 sum); the factor adds the rounding of its sum and its quotient, the scaled gradient that of the product:
4 * 2^-24 in fp32, and one rounding of the gradient's own type on top (bf16 2^-8, fp16 2^-11, or half its smallest step)."""
import math

import pytest
import torch

from diffusion_model_amd import optim
from gpu_util import P, call, stream

pytestmark = pytest.mark.gpu

# sizes around the kernels' chunks (8192 elements, 2048 for Adam) and loads, empty tensors, one large one
SIZES = [1, 0, 3, 2047, 2048, 2049, 8191, 8192, 8193, 3 * 8192 + 5, 64 * 64 * 9, 1 << 20]
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def _params(sizes, types, scale=1.0, seed=0, offset=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        t = types[i % len(types)]
        base = torch.empty(n + offset, dtype=t, device="cuda")
        p = torch.nn.Parameter(torch.zeros(n, dtype=t, device="cuda"))
        p.grad = base[offset:].copy_((torch.randn(n, generator=g) * scale).to(t))
        out.append(p)
    return out


def _norm64(params):
    return math.sqrt(sum(float(p.grad.double().square().sum()) for p in params))


def _check_scaled(params, before, coef):
    for p, b in zip(params, before):
        want = b.double() * coef
        tiny = {FP32: 2.0 ** -150, BF16: 2.0 ** -134, FP16: 2.0 ** -25}[b.dtype]
        own = 0.0 if b.dtype == FP32 else torch.finfo(b.dtype).eps / 2
        assert p.grad.dtype == b.dtype
        assert ((p.grad.double() - want).abs() <= want.abs() * (4 * 2.0 ** -24 + own) + tiny).all(), b.dtype


@pytest.mark.parametrize("types", [(FP32,), (BF16,), (FP16,), (FP32, BF16, FP16)])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_and_clip(types, offset):
    params = _params(SIZES, types, offset=offset)
    before = [p.grad.clone() for p in params]
    want = _norm64(params)
    assert float(optim.grad_norm(params)) == pytest.approx(want, rel=2.0 ** -23)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))
    versions = [p.grad._version for p in params]
    got = optim.clip_grad_norm_(params, 1.5)
    assert got.shape == () and got.dtype == FP32 and got.is_cuda
    assert float(got) == pytest.approx(want, rel=2.0 ** -23)
    assert all(p.grad._version > v for p, v in zip(params, versions))
    _check_scaled(params, before, 1.5 / (want + 1e-6))


def test_norm_within_the_bound_leaves_every_bit():
    params = _params(SIZES, (FP32, BF16))
    before = [p.grad.clone() for p in params]
    optim.clip_grad_norm_(params, _norm64(params) * 1.01)
    optim.clip_grad_norm_(params, math.inf)
    assert all(torch.equal(p.grad, b) for p, b in zip(params, before))


@pytest.mark.parametrize("count", [1, 175, 176, 177, 700])
def test_lists_longer_than_one_launch(count):
    params = _params([1 + i % 7 for i in range(count)], (FP32, FP16), seed=count)
    before = [p.grad.clone() for p in params]
    want = _norm64(params)
    assert float(optim.clip_grad_norm_(iter(params), 0.25)) == pytest.approx(want, rel=2.0 ** -23)
    _check_scaled(params, before, min(1.0, 0.25 / (want + 1e-6)))


def test_maximum_norm_and_nonfinite_values():
    params = _params(SIZES, (FP32, BF16))
    params[-1].grad[12345] = -77.5
    assert float(optim.grad_norm(params, math.inf)) == 77.5
    assert float(optim.clip_grad_norm_(params, 1.0, norm_type=math.inf)) == 77.5
    for bad in (math.inf, -math.inf, math.nan):
        for where in (0, 4, len(params) - 1):
            params = _params(SIZES, (FP32,))
            params[where].grad[params[where].numel() // 2] = bad
            for kind in (2.0, math.inf):
                n = float(optim.grad_norm(params, kind))
                assert math.isnan(n) if math.isnan(bad) else n == math.inf
            with pytest.raises(RuntimeError, match="non-finite"):
                optim.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
            ours = [p.grad.clone() for p in params]
            optim.clip_grad_norm_(params, 1.0)
            for p, g in zip(params, ours):                      # as torch: 0 * inf, or NaN everywhere
                want = g * (0.0 if not math.isnan(bad) else math.nan)
                assert torch.equal(p.grad.isnan(), want.isnan()) and torch.equal(p.grad.nan_to_num(), want.nan_to_num())


def test_squares_beyond_fp32():
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = torch.full((100,), 1e25, device="cuda")
    assert float(optim.grad_norm([p])) == pytest.approx(1e26, rel=1e-6)
    p.grad = torch.full((100,), 1e-30, device="cuda")
    assert float(optim.grad_norm([p])) == pytest.approx(1e-29, rel=1e-6)


def test_same_bits_every_time_and_no_gradient():
    params = _params(SIZES, (FP32,))
    first = optim.grad_norm(params)
    assert all(torch.equal(first, optim.grad_norm(params)) for _ in range(5))
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(3, device="cuda"))], 1.0)) == 0.0
    empty = _params([0, 0], (FP32,))
    assert float(optim.clip_grad_norm_(empty, 1.0)) == 0.0
    single = _params([9], (FP32,))[0]
    want = single.grad.double().norm()
    assert float(optim.clip_grad_norm_(single, 0.5)) == pytest.approx(float(want), rel=2.0 ** -23)


def test_gradients_in_another_memory_order():
    p = torch.nn.Parameter(torch.zeros(8, 16, 3, 3, device="cuda"))
    g = torch.randn(8, 16, 3, 3, device="cuda")
    p.grad = g.clone(memory_format=torch.channels_last)
    norm = float(g.double().norm())
    optim.clip_grad_norm_([p], 1.0)
    assert p.grad.is_contiguous(memory_format=torch.channels_last)
    assert (p.grad.double() - g.double() / (norm + 1e-6)).abs().max() <= g.abs().max() * 4 * 2.0 ** -24


@pytest.mark.parametrize("max_norm", [0.5, 1e9])
@pytest.mark.parametrize("weight_decay", [0.0, 0.01])
def test_clipped_adam_step_is_clip_then_step(max_norm, weight_decay):
    """Bit for bit what clipping the gradients first and then stepping gives; the gradients themselves stay."""
    sizes = SIZES + [5] * 90                                     # two launches
    a, b = _params(sizes, (FP32,), seed=3), _params(sizes, (FP32,), seed=3)
    state = [[torch.rand(n, device="cuda") * s for n in sizes] for s in (0.1, 0.01)]
    other = [[t.clone() for t in x] for x in state]
    grads = [p.grad.clone() for p in a]
    for step in (1, 7):
        want = optim.clip_grad_norm_(b, max_norm)
        assert optim.adam_step_(b, [p.grad for p in b], *other, step, lr=1e-2, weight_decay=weight_decay) is None
        got = optim.adam_step_(a, grads, *state, step, lr=1e-2, weight_decay=weight_decay, max_norm=max_norm)
        assert torch.equal(got, want)
        for p, g in zip(b, grads):
            p.grad.copy_(g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert all(torch.equal(s, t) for x, y in zip(state, other) for s, t in zip(x, y))
    assert all(torch.equal(p.grad, g) for p, g in zip(a, grads))


def test_adam_class_clips_over_all_groups():
    a, b = _params([5000, 33], (FP32,), seed=5), _params([5000, 33], (FP32,), seed=5)
    ours = optim.Adam([dict(params=a[:1], lr=1e-2), dict(params=a[1:], lr=1e-3)], max_grad_norm=0.7)
    theirs = optim.Adam([dict(params=b[:1], lr=1e-2), dict(params=b[1:], lr=1e-3)])
    for _ in range(3):
        keep = [p.grad.clone() for p in b]
        norm = optim.clip_grad_norm_(b, 0.7)
        theirs.step()
        ours.step()
        assert torch.equal(ours.grad_norm, norm)
        for p, g in zip(b, keep):
            p.grad.copy_(g)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    assert set(ours.state_dict()["param_groups"][0]) == set(theirs.state_dict()["param_groups"][0])


def test_replayed_graph_and_side_stream():
    params = _params(SIZES, (FP32, BF16), seed=9)
    source = [p.grad.clone() for p in params]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                                # a first call outside the capture, on another stream
        eager = optim.clip_grad_norm_(params, 1.0)
    torch.cuda.current_stream().wait_stream(side)
    want = [p.grad.clone() for p in params]
    assert float(eager) > 1.0
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(params, 1.0)
    for k in range(4):
        for p, s in zip(params, source):
            p.grad.copy_(s)
        if k % 2:
            torch.cuda.synchronize()
            optim.grad_norm(params)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, eager)
        assert all(torch.equal(p.grad, w) for p, w in zip(params, want))


def test_the_entry_point_alone_on_fp32_tensors():
    """Through the C ABI: state = [norm, factor]."""
    import ctypes as C
    from diffusion_model_amd import _lib
    g = torch.randn(10000, device="cuda")
    ws = torch.empty(_lib.lib().ddpm_grad_norm_workspace_doubles(1), dtype=torch.float64, device="cuda")
    state = torch.empty(2, device="cuda")
    args = (1, (C.c_void_p * 1)(g.data_ptr()), (C.c_int64 * 1)(g.numel()), (C.c_int32 * 1)(0))
    call("ddpm_grad_norm", *args, 0, 2.0, P(ws), P(state), stream())
    norm = float(g.double().norm())
    assert float(state[0]) == pytest.approx(norm, rel=2.0 ** -23)
    assert float(state[1]) == pytest.approx(2.0 / (norm + 1e-6), rel=4 * 2.0 ** -24)
    call("ddpm_grad_norm", 0, None, None, None, 0, 2.0, P(ws), P(state), stream())
    assert state.tolist() == [0.0, 1.0]


def test_functions_refuse_on_the_gpu():
    """Host-side checks that need tensors on a GPU to get that far; nothing is launched."""
    p, = _params([16], (FP32,))
    twin = torch.nn.Parameter(torch.zeros(16, device="cuda"))
    twin.grad = p.grad
    with pytest.raises(ValueError, match="twice"):
        optim.clip_grad_norm_([p, twin], 1.0)
    wide = torch.nn.Parameter(torch.zeros(4, dtype=torch.float64, device="cuda"))
    wide.grad = torch.ones_like(wide)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        optim.clip_grad_norm_([wide], 1.0)
    t, u, v, w = (torch.zeros(16, device="cuda") for _ in range(4))
    with pytest.raises(ValueError, match="twice"):
        optim.adam_step_([t], [u], [v], [t], 1)
    with pytest.raises(RuntimeError, match="size"):
        optim.adam_step_([t], [u[:4]], [v], [w], 1)
    with pytest.raises(RuntimeError, match="fp32"):
        optim.adam_step_([t.half()], [u], [v], [w], 1)
    with pytest.raises(RuntimeError, match="contiguous"):
        optim.adam_step_([t], [torch.zeros(16, 2, device="cuda")[:, 0]], [v], [w], 1)
