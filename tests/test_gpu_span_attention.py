"""Span attention and its gradient against float64 (tests/span_reference.py derives the bounds)."""
import math

import pytest
import torch

from diffusion_model_amd.attention import key_spans, span_attention
from span_reference import check, reference

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [FP32, BF16, FP16]


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _inputs(b, nq, nk, heads, kv, dim, dtype, seed=0):
    return (_rand((b, nq, heads, dim), dtype, seed, 1.5), _rand((b, nk, kv, dim), dtype, seed + 1, 1.5), _rand((b, nk, kv, dim), dtype, seed + 2),
            _rand((b, nq, heads, dim), dtype, seed + 3))


def _slopes(heads):
    return (2.0 ** (-8.0 * torch.arange(1, heads + 1) / heads)).cuda()


def _check_all(q, k, v, dout, **how):
    want = reference(q, k, v, dout, **how)
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out, lse = span_attention(*leaves, return_lse=True, **how)
    assert out.dtype == q.dtype and lse.dtype == FP32 and not lse.requires_grad
    grads = torch.autograd.grad(out, leaves, dout)
    check(lse, want, "lse")
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        assert got.dtype == q.dtype
        check(got, want, name)
    with torch.no_grad():                                       # the call without a gradient gives the same bits
        assert torch.equal(span_attention(*leaves, **how), out)
    return out.detach(), grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 49, 64, 65, 127, 128, 129, 200, 385])
def test_lengths(dtype, n):
    _check_all(*_inputs(2, n, n, 3, 3, 32, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 96, 104, 128])
def test_head_sizes(dtype, dim):
    _check_all(*_inputs(1, 70, 130, 2, 1, dim, dtype), softcap=20.0, slopes=_slopes(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 4, 20, 33, 127])
def test_head_sizes_that_need_a_copy(dtype, dim):
    _check_all(*_inputs(1, 33, 40, 2, 2, dim, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 4), (4, 2), (6, 2), (5, 1), (8, 1)])
@pytest.mark.parametrize("nq,nk", [(150, 150), (5, 300), (200, 70)])
def test_shared_heads(dtype, heads, kv, nq, nk):
    _check_all(*_inputs(2, nq, nk, heads, kv, 48, dtype), causal=nq <= nk, slopes=_slopes(heads))


def _masks(b, n):
    g = torch.Generator().manual_seed(n)
    ids = torch.sort(torch.randint(0, max(2, n // 20), (b, n), generator=g), 1).values.cuda()
    lengths = torch.randint(1, n + 1, (b,), generator=g).cuda()
    lengths[0] = 0
    return {
        "documents": key_spans(n, documents=ids), "causal documents": key_spans(n, documents=ids, causal=True),
        "prefix of documents": key_spans(n, documents=ids, prefix=3), "prefix": key_spans(n, prefix=lengths // 2), "shared prefix": key_spans(n, prefix=5, device="cuda"),
        "lengths": key_spans(n, lengths=lengths), "causal lengths": key_spans(n, lengths=lengths, causal=True), "window": key_spans(n, window=(7, 2), device="cuda"),
        "nothing": torch.zeros(1, n, 2, dtype=torch.int32, device="cuda"),
        "anything": torch.randint(-20, n + 20, (b, n, 2), generator=g).int().cuda(),
        "beyond": torch.tensor([-2 ** 31, 2 ** 31 - 1], dtype=torch.int32, device="cuda").expand(b, n, 2),
    }


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [60, 301])
@pytest.mark.parametrize("mask", ["documents", "causal documents", "prefix of documents", "prefix", "shared prefix", "lengths", "causal lengths", "window",
                                  "nothing", "anything", "beyond"])
def test_masks(dtype, n, mask):
    spans = _masks(3, n)[mask]
    out, grads = _check_all(*_inputs(3, n, n, 2, 1, 32, dtype), spans=spans)
    empty = (spans[..., 1].clamp(max=n) <= spans[..., 0].clamp(min=0)).expand(3, n)
    assert (out[empty] == 0).all() and (grads[0][empty] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_positions(dtype, causal):
    pos = torch.randint(-30, 160, (2, 90), generator=torch.Generator().manual_seed(0)).int().cuda()
    q, k, v, dout = _inputs(2, 90, 140, 4, 2, 64, dtype)
    _check_all(q, k, v, dout, positions=pos, causal=causal, slopes=_slopes(4), softcap=5.0)
    _check_all(q, k, v, dout, positions=pos[:1], causal=causal, spans=key_spans(90, 140, window=(60, 10), device="cuda"))
    far = torch.full((1, 90), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    assert torch.equal(span_attention(q, k, v, positions=far, causal=True), span_attention(q, k, v))
    assert (span_attention(q, k, v, positions=-far - 1, causal=True) == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,softcap", [(1.0, 0.0), (0.0, 0.0), (-0.3, 0.0), (1.0, 2.0), (0.01, 100.0)])
def test_scales_and_caps(dtype, scale, softcap):
    _check_all(*_inputs(1, 100, 100, 2, 2, 32, dtype), scale=scale, softcap=softcap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,nq,nk,heads,kv,dim", [(1, 1, 1, 1, 1, 64), (1, 1, 5000, 8, 8, 128), (3, 1, 4097, 8, 2, 80), (2, 5, 3000, 6, 1, 64),
                                                      (1, 40, 2500, 4, 1, 32), (40, 1, 700, 4, 4, 64), (1, 1, 20000, 16, 1, 96)])
def test_few_rows_against_many_keys(dtype, batch, nq, nk, heads, kv, dim):
    """Single tokens and a few: rows of a group together, keys split over workgroups, lengths from none to all."""
    q, k, v, _ = _inputs(batch, nq, nk, heads, kv, dim, dtype)
    n = torch.randint(0, nk + 1, (batch,), generator=torch.Generator().manual_seed(0)).int().cuda()
    n[0] = nk
    pos = (n[:, None] - nq + torch.arange(nq, device="cuda")).int()
    spans = torch.stack([torch.zeros_like(pos), (pos + 1).clamp(0, nk)], -1)
    for how in (dict(spans=spans, positions=pos, slopes=_slopes(heads)), dict(causal=True, softcap=30.0), dict(causal=True, positions=pos)):
        out, lse = span_attention(q, k, v, return_lse=True, **how)
        want = reference(q, k, v, **how)
        check(out, want, "out")
        check(lse, want, "lse")


@pytest.mark.parametrize("dtype", TYPES)
def test_batches_of_more_entries_than_a_grid_holds(dtype):
    b = 65535 + 9                                               # such as the frames of every pixel
    q, k, v, dout = _inputs(b, 2, 3, 2, 1, 8, dtype)
    g = torch.Generator().manual_seed(0)
    ends = torch.sort(torch.randint(0, 4, (b, 2, 2), generator=g), -1).values.int().cuda()
    positions = torch.randint(0, 9, (b, 2), generator=g).int().cuda()
    _check_all(q, k, v, dout, spans=ends, positions=positions, slopes=_slopes(2))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale,softcap,size", [(1e-3, 50.0, 50.0), (2e-5, 50.0, 350.0), (-2e-7, 1.0, 500.0), (1.0, 1e-4, 2e-3), (1.0, 1e-9, 0.0), (1e-30, 1e20, 100.0),
                                                (1e-3, 50.0, 24.0), (2e-5, 50.0, 170.0), (-2e-7, 1.0, 240.0), (1.0, 1e-4, 1.1e-3), (1.0, 1e-3, 3.4e-3)])
def test_scores_of_any_size_beside_the_cap(dtype, scale, softcap, size):
    """Scores of about a third or a seventh of the cap (or none), made from very large and very small products."""
    q, k, v, dout = _inputs(1, 70, 90, 2, 1, 32, dtype)
    _check_all(q * size, k * size, v, dout, scale=scale, softcap=softcap)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,nk,heads,kv,dim", [(40, 1500, 4, 1, 64), (700, 700, 2, 2, 32), (1100, 600, 3, 1, 128), (2100, 90, 2, 1, 96), (1, 2000, 2, 2, 40)])
def test_gradients_whose_work_is_dealt_out(dtype, nq, nk, heads, kv, dim):
    """Few blocks of rows (or keys) against many of the other: several workgroups share a block, and their sums are added up."""
    q, k, v, dout = _inputs(1, nq, nk, heads, kv, dim, dtype)
    g = torch.Generator().manual_seed(0)
    ends = torch.sort(torch.randint(-50, nk + 50, (1, nq, 2), generator=g), -1).values.int().cuda()
    _check_all(q, k, v, dout, softcap=15.0, slopes=_slopes(heads))
    _check_all(q, k, v, dout, spans=ends, causal=nq > nk)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_what_padding_holds_does_not_matter(dtype, bad):
    """NaN and infinities in keys that no row sees and in rows that see no key: outputs and gradients as with noughts there."""
    n, lengths = 200, torch.tensor([200, 70, 0, 129], device="cuda")
    spans = key_spans(n, lengths=lengths)
    good = _inputs(4, n, n, 4, 2, 64, dtype)
    dead = torch.arange(n, device="cuda")[None] >= lengths[:, None]
    results = []
    for fill in (0.0, bad):
        leaves = [x.clone() for x in good]
        for x in leaves:
            x[dead] = fill
        for x in leaves[:3]:
            x.requires_grad_(True)
        out = span_attention(*leaves[:3], spans=spans, causal=True)
        results.append([out.detach(), *torch.autograd.grad(out, leaves[:3], leaves[3])])
    for x, y in zip(*results):
        assert torch.equal(x, y) and x.isfinite().all()
        assert (x[dead] == 0).all()
    few = span_attention(*(x[:, -3:] if i == 0 else x for i, x in enumerate(leaves[:3])), spans=torch.tensor([[[0, 200]] * 3, [[0, 70]] * 3, [[0, 0]] * 3, [[0, 129]] * 3]).int().cuda())
    assert few[[0, 1, 2]][2].eq(0).all()


def test_not_a_number_stays_visible():
    q, k, v, _ = _inputs(1, 8, 40, 1, 1, 32, BF16)
    v[0, 3, 0, 5] = math.nan
    out = span_attention(q, k, v)
    assert out[..., 5].isnan().all() and out[..., :5].isfinite().all()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_strides(dtype):
    """Slices of a fused projection, head-first tensors, expanded keys, channel strides, odd offsets, one token of many."""
    b, n, h, d = 2, 77, 4, 32
    fused = _rand((b, n, 3 * h * d), dtype, 1)
    q, k, v = (x.view(b, n, h, d) for x in fused.chunk(3, -1))
    dout = _rand((b, h, n, d), dtype, 2).transpose(1, 2)
    _check_all(q, k, v, dout, causal=True)
    first = [_rand((b, h, n, d), dtype, s).transpose(1, 2) for s in (3, 4, 5)]
    _check_all(*first, dout)
    one = _rand((1, 1, 1, d), dtype, 6).expand(b, n, h, d)
    _check_all(q, one, v, dout)
    _check_all(q, k, v, _rand((1, 1, 1, 1), dtype, 7).expand(b, n, h, d))
    wide = _rand((b, n, h, 2 * d), dtype, 8)
    _check_all(wide[..., ::2], wide[..., 1::2], wide[..., 3:3 + d], dout)
    _check_all(q[:, 5:6], k[:, :9], v[:, :9], dout[:, 5:6])
    _check_all(q[1:], k[1:], v[1:], dout[1:])


def test_keys_beyond_32_bit_offsets():
    """Rows of a buffer whose last keys lie past 2^31 elements."""
    nk, heads = 270000, 64
    buffer = torch.empty(1, nk, heads, 128, dtype=BF16, device="cuda")
    k, v = _rand((1, nk, 1, 128), BF16, 1), _rand((1, nk, 1, 128), BF16, 2)
    buffer[:, :, 62:63], buffer[:, :, 63:64] = k, v
    assert buffer[:, nk - 1:, 63].storage_offset() > 2 ** 31
    q = _rand((1, 1, 2, 128), BF16, 3)
    spans = torch.tensor([[[nk - 3000, nk]]], dtype=torch.int32, device="cuda")
    want = span_attention(q, k[:, -3000:], v[:, -3000:])
    for how in (dict(spans=spans),):
        got = span_attention(q, buffer[:, :, 62:63], buffer[:, :, 63:64], **how)
        ref = reference(q, k[:, -3000:], v[:, -3000:])
        check(got, ref, "out")
        check(want, ref, "out")


@pytest.mark.parametrize("dtype", TYPES)
def test_nothing(dtype):
    q, k, v, dout = _inputs(2, 6, 0, 2, 1, 16, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out, lse = span_attention(*leaves, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    assert (dq == 0).all() and dk.shape == k.shape and dv.shape == v.shape
    q, k, v, dout = _inputs(2, 0, 6, 2, 1, 16, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out = span_attention(*leaves)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    assert out.shape == q.shape and (dk == 0).all() and (dv == 0).all()
    q, k, v, _ = _inputs(0, 5, 6, 2, 1, 16, dtype)
    assert span_attention(q, k, v).shape == (0, 5, 2, 16)


@pytest.mark.parametrize("dtype", TYPES)
def test_same_bits_every_time(dtype):
    q, k, v, dout = _inputs(2, 300, 300, 4, 1, 64, dtype)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    first = None
    for _ in range(3):
        out = span_attention(*leaves, softcap=10.0, causal=True)
        now = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
        assert first is None or all(torch.equal(x, y) for x, y in zip(first, now))
        first = now
    few = span_attention(q[:, :1].detach(), k.detach(), v.detach())
    assert torch.equal(few, span_attention(q[:, :1].detach(), k.detach(), v.detach()))


@pytest.mark.parametrize("size", [1e-6, 1e3])
def test_fp16_gradients_of_any_size(size):
    """Score gradients far below and above fp16's normal numbers: as exact as others (relative to their own size)."""
    q, k, v, _ = _inputs(1, 260, 260, 2, 1, 64, FP16)
    dout = _rand((1, 260, 2, 64), FP32, 9, size).to(FP16)
    _check_all(q, k, v, dout, softcap=20.0)
    _check_all(q, k, v * 100, dout / 8)


def test_gradient_against_differences():
    """Central differences with step 2^-6 along a random direction of all three inputs: rounding adds (2^-19 / 2^-6) and the third
    derivative about 3 * 2^-12 of the sum of |g|; both stay below 2^-10 of it."""
    how = dict(softcap=4.0, slopes=_slopes(2), causal=True, spans=key_spans(40, documents=torch.arange(40, device="cuda") // 13))
    x = [t.double() for t in _inputs(1, 40, 40, 2, 1, 16, FP32)]
    e = [_rand(t.shape, FP32, 20 + i, 0.5).double() for i, t in enumerate(x[:3])]
    leaves = [t.float().requires_grad_(True) for t in x[:3]]
    out = span_attention(*leaves, **how)
    grads = torch.autograd.grad(out, leaves, x[3].float())
    at = lambda s: span_attention(*((t + s * d).float() for t, d in zip(x[:3], e)), **how).double()      # noqa: E731
    left = ((at(2.0 ** -6) - at(-2.0 ** -6)) * x[3]).sum() * 2.0 ** 5
    right = sum((g.double() * d).sum() for g, d in zip(grads, e))
    assert abs(float(left - right)) <= float(x[3].abs().sum()) * 2.0 ** -10


def test_replayed_graph_and_side_stream():
    """Forward and gradient captured together, and a split call for one token; every replay against the eager result."""
    q, k, v, dout = _inputs(2, 130, 130, 4, 2, 64, BF16)
    one, many = _rand((1, 1, 4, 64), BF16, 5), _rand((1, 5000, 2, 64), BF16, 6)
    side = torch.cuda.Stream()

    def step():
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        out = span_attention(*leaves, causal=True, softcap=9.0)
        return [out.detach(), *torch.autograd.grad(out, leaves, dout), span_attention(one, many, many)]

    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(on_side, step()))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        for n, x in enumerate((q, k, v, dout, one, many)):
            x.copy_(_rand(x.shape, BF16, 100 + 10 * i + n))
        want = step()
        if i % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), i


def test_key_spans_of_rows_behind_the_keys():
    """5 new rows behind 7 earlier keys, causal: row i stands at 7 + i."""
    assert key_spans(5, 12, causal=True, device="cuda").tolist() == [[[0, 8 + i] for i in range(5)]]


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_attention_loss_backward_clipped_step(dtype):
    """One training step of an attention block over the pixels of packed images as a user writes it: fused projection, rotary
    positions on two axes, span attention over documents, backward, clipped Adam. Projection and loss in fp32. Against the
    same step in float64, with the updated weights' distance measured in units of the learning rate: an element of Adam's first step
    moves by lr * g / (|g| + eps), so where |g| is above eps and above the gradient's own error its sign decides."""
    from diffusion_model_amd.embedding import grid_positions, rotary
    from diffusion_model_amd import optim
    g = torch.Generator().manual_seed(4)
    sizes, heads, kv, dim, width = [(8, 8), (5, 7), (1, 1), (9, 4)], 4, 2, 32, 48
    pos = torch.cat([grid_positions(*s) for s in sizes])
    ids = torch.cat([torch.full((h * w,), i) for i, (h, w) in enumerate(sizes)]).cuda()
    n = len(ids)
    x = torch.randn(1, n, width, generator=g).cuda()
    w0 = (torch.randn((heads + 2 * kv) * dim, width, generator=g) * 0.2).cuda()
    target = torch.randn(1, n, heads, dim, generator=g).cuda()
    w = torch.nn.Parameter(w0.clone())
    fused = (x @ w.t()).to(dtype).view(1, n, heads + 2 * kv, dim)
    q, k, v = fused.split([heads, kv, kv], 2)
    q, k = rotary(q, k, pos, (16, 16))
    out = span_attention(q, k, v, spans=key_spans(n, documents=ids), softcap=30.0)
    loss = ((out.float() - target) ** 2).sum()
    loss.backward()
    gradient = w.grad.clone()
    opt = optim.Adam([w], lr=1e-2, max_grad_norm=0.5)
    opt.step()

    wd = w0.double().requires_grad_(True)
    q, k, v = (x.double() @ wd.t()).view(1, n, heads + 2 * kv, dim).split([heads, kv, kv], 2)
    th = torch.cat([pos[:, a, None].double() * 10000.0 ** (-2.0 * torch.arange(8, device="cuda").double() / 16) for a in (0, 1)], 1)
    c, s = (f(th)[None, :, None] for f in (torch.cos, torch.sin))
    one = torch.tensor([*range(8), *range(16, 24)], device="cuda")

    def turn(y):
        a, b = y[..., one], y[..., one + 8]
        z = torch.cat([a * c - b * s, b * c + a * s], -1)
        return z[..., torch.argsort(torch.cat([one, one + 8]))]

    t = turn(q).transpose(1, 2) @ turn(k).transpose(1, 2).repeat_interleave(2, 1).transpose(2, 3).contiguous() / dim ** 0.5
    t = torch.where(ids[:, None] == ids[None], 30 * torch.tanh(t / 30), -math.inf)
    o = (torch.softmax(t, -1) @ v.transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2)
    want, = torch.autograd.grad(((o - target.double()) ** 2).sum(), wd)
    # roundings of the 16-bit tensors on the way (projection, turned q and k, weights, out, score gradients, gradients of each):
    # at most ten in a row, each half a step of independent sign; in fp32 the sums' own roundings, some 2^-18
    tol = {FP32: 2.0 ** -18, BF16: 10 * 2.0 ** -8, FP16: 10 * 2.0 ** -11}[dtype]
    assert float((gradient.double() - want).norm()) <= tol * float(want.norm())
    assert float(opt.grad_norm) == pytest.approx(float(gradient.double().norm()), rel=2.0 ** -23)
    moved = w0.double() - w.detach().double()
    coef = 0.5 / (float(gradient.double().norm()) + 1e-6)
    step = 1e-2 * gradient.double() * coef / ((gradient.double() * coef).abs() + 1e-8)
    # 16 roundings of Adam's own on the step, and the rounding of the weight it is taken from
    assert ((moved - step).abs() <= 16 * 2.0 ** -24 * step.abs() + w0.double().abs() * 2.0 ** -23).all()
