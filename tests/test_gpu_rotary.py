"""Rotary positions with several axes against complex rotations in float64.

Tolerance: the reduced angle is rounded once (2^-25 of a half turn, 2^-23.3 radian) and its sine and cosine to one unit (2^-24), so each
is off by less than 2^-22.6; with the roundings of two products and their sum an output is off by less than
(|x1| + |x2|) 2^-22, and by half a step of its own type when that has 16 bits (bf16 2^-8, fp16 2^-11, or half fp16's smallest step)."""
import pytest
import torch

from diffusion_model_amd.embedding import grid_positions, rotary

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def _turned(x, positions, axes, interleaved, sign=1, base=10000.0):
    """Result in float64, and (|x1| + |x2|) of each element."""
    y, size, o = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64, device=x.device), 0
    p = positions.double() if positions.dim() == 3 else positions.double()[None]
    for a, d in enumerate(axes):
        i = torch.arange(d // 2, device=x.device)
        one = o + (2 * i if interleaved else i)
        two = one + (1 if interleaved else d // 2)
        th = sign * p[..., a, None] * float(base) ** (-2.0 * i.double() / d)
        z = torch.complex(x[..., one].double(), x[..., two].double()) * torch.polar(torch.ones_like(th), th)[:, :, None]
        y[..., one], y[..., two] = z.real, z.imag
        size[..., one] = size[..., two] = x[..., one].double().abs() + x[..., two].double().abs()
        o += d
    return y, size


def _check(got, want, size):
    own = 0.0 if got.dtype == FP32 else torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == FP16 else 2.0 ** -134
    err = (got.double() - want).abs()
    assert (err <= size * 2.0 ** -22 + want.abs() * own * 1.001 + tiny).all(), f"{err.max().item():.3e}"


def _x(shape, dtype, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("axes,dim", [((64,), 64), ((32, 32), 64), ((32, 48, 48), 128), ((2,), 2), ((6, 10), 20), ((42, 14, 28), 104),
                                      ((2, 2, 2, 2), 9), ((16,), 80), ((100, 156), 256), ((512,), 512)])
def test_forward_and_gradient(dtype, interleaved, axes, dim):
    b, n, h, hk = 2, 37, 3, 2
    pos = torch.randint(-500, 500, (b, n, len(axes)), generator=torch.Generator().manual_seed(1)).int().cuda()
    q, k = _x((b, n, h, dim), dtype, 2).requires_grad_(True), _x((b, n, hk, dim), dtype, 3).requires_grad_(True)
    gq, gk = _x((b, n, h, dim), dtype, 4), _x((b, n, hk, dim), dtype, 5)
    yq, yk = rotary(q, k, pos, axes, interleaved=interleaved)
    assert yq.shape == q.shape and yk.shape == k.shape and yq.dtype == dtype and yq.is_contiguous()
    _check(yq.detach(), *_turned(q.detach(), pos, axes, interleaved))
    _check(yk.detach(), *_turned(k.detach(), pos, axes, interleaved))
    assert torch.equal(yq.detach()[..., sum(axes):], q.detach()[..., sum(axes):])
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    _check(dq, *_turned(gq, pos, axes, interleaved, -1))
    _check(dk, *_turned(gk, pos, axes, interleaved, -1))


def test_gradient_against_differences():
    """The map is linear: <rotary(x + e) - rotary(x), g> = <e, gradient>, in float64 sums of fp32 results; 600 terms of size
    |g| |e| 2^-21 at most."""
    pos = grid_positions(5, 6)
    x, e, g = (_x((1, 30, 2, 10), FP32, s) for s in (1, 2, 3))
    x.requires_grad_(True)
    y = rotary(x, None, pos, (4, 6))
    dx, = torch.autograd.grad(y, x, g)
    moved = rotary((x + e).detach(), None, pos, (4, 6))
    left = ((moved.double() - y.detach().double()) * g.double()).sum()
    right = (((x + e).detach().double() - x.detach().double()) * dx.double()).sum()
    assert abs(float(left - right)) <= float((g.double().abs() * (x.detach().double().abs() + e.double().abs() + 1)).sum()) * 2.0 ** -20


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, FP32])
@pytest.mark.parametrize("shared", [False, True])
def test_position_types_and_far_positions(dtype, shared):
    pos = torch.tensor([[0, 1], [-1, 10 ** 7], [123456, 16777215], [999999, -10 ** 7]])
    pos = (pos if shared else torch.stack([pos, pos.flip(0), pos + 1])).to(dtype).cuda()
    if dtype == FP32:
        pos = pos + 0.25 * (pos.abs() < 1000)                   # fractions
    x = _x((3, 4, 2, 32), FP32)
    y = rotary(x, None, pos, (16, 16))
    _check(y, *_turned(x, pos, (16, 16), False))
    _check(rotary(x, None, pos, (16, 16), base=500.0), *_turned(x, pos, (16, 16), False, base=500.0))


@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("batch,tokens,heads", [(1, 1, 1), (16, 1, 40), (1, 4097, 1), (3, 300, 65), (1, 1, 300)])
def test_sizes(dtype, batch, tokens, heads):
    pos = torch.randint(0, 4096, (batch, tokens, 1), generator=torch.Generator().manual_seed(0)).cuda()
    x = _x((batch, tokens, heads, 64), dtype)
    _check(rotary(x, None, pos, (64,)), *_turned(x, pos, (64,), False))


def test_strides():
    """A fused projection's slices, a head-first tensor, an expanded one, a slice whose channels are not neighbours, and one
    off a 16-byte boundary."""
    pos = grid_positions(4, 5)
    fused = _x((2, 20, 6 * 32), BF16)
    q, k = fused[..., :128].view(2, 20, 4, 32), fused[..., 128:].view(2, 20, 2, 32)
    yq, yk = rotary(q, k, pos, (16, 16))
    _check(yq, *_turned(q, pos, (16, 16), False))
    _check(yk, *_turned(k, pos, (16, 16), False))
    base = _x((2, 4, 20, 32), FP32)
    odd = _x((2 * 20 * 4 * 32 + 1,), FP32)[1:].view(2, 20, 4, 32)
    for x in (base.transpose(1, 2), base[:1, :1].transpose(1, 2).expand(2, 20, 4, 32), _x((2, 20, 4, 64), FP32)[..., ::2], odd,
              _x((2, 20, 4, 33), FP32)[..., :32]):
        before = x.clone()
        for il in (False, True):
            _check(rotary(x, None, pos, (16, 16), interleaved=il), *_turned(x, pos, (16, 16), il))
        assert torch.equal(x, before)


def test_nothing_to_turn():
    pos = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    assert rotary(_x((2, 0, 3, 8), FP32), None, pos, (8,)).shape == (2, 0, 3, 8)
    assert rotary(_x((0, 4, 3, 8), FP32), None, torch.zeros(4, 1, dtype=torch.int32, device="cuda"), (8,)).shape == (0, 4, 3, 8)


def test_special_values_pass_behind_the_axes():
    x = _x((1, 3, 2, 16), BF16)
    x[..., 8:] = torch.tensor([float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e38, -1e38, 1.0], device="cuda")
    y = rotary(x, None, torch.arange(3, device="cuda")[:, None], (8,))
    assert torch.equal(y[..., 8:].view(torch.int16), x[..., 8:].view(torch.int16))
    assert torch.equal(y[:, 0].view(torch.int16), x[:, 0].view(torch.int16))      # position 0 turns nothing


def test_one_gradient_missing():
    pos = grid_positions(3, 3)
    q, k = _x((1, 9, 2, 8), FP32).requires_grad_(True), _x((1, 9, 1, 8), FP32, 1).requires_grad_(True)
    yq, yk = rotary(q, k, pos, (4, 4))
    dk, = torch.autograd.grad(yk.sum(), k)
    _check(dk, *_turned(torch.ones_like(k), pos, (4, 4), False, -1))
    yq, yk = rotary(q.detach(), k, pos, (4, 4))
    assert not yq.requires_grad or yk.requires_grad
    yk.sum().backward()
    assert torch.equal(k.grad, dk)


def test_replayed_graph_and_side_stream():
    pos = grid_positions(8, 8)
    x, k = _x((2, 64, 4, 32), BF16), _x((2, 64, 2, 32), BF16, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotary(x, k, pos, (16, 16))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y, z = rotary(x, k, pos, (16, 16))
    for i in range(4):
        x.copy_(_x((2, 64, 4, 32), BF16, 10 + i))
        want = rotary(x, k, pos, (16, 16))
        if i % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])
