"""Span attention where memory holds NaN and infinities at keys that no row sees and in rows that see none, anywhere in a sequence:
outputs and gradients are, bit for bit, those with noughts there, and those meet the bounds of span_reference.py."""
import math

import pytest
import torch

from diffusion_model_amd.attention import span_attention
from span_reference import check, reference

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [FP32, BF16, FP16]


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _padded(lengths, room, causal=False):
    """Documents of these lengths, each in `room` tokens, of which the last ones see nothing and are seen by none."""
    rows = []
    for d, n in enumerate(lengths):
        rows += [(d * room, d * room + (i + 1 if causal else n)) if i < n else (0, 0) for i in range(room)]
    return torch.tensor([rows], dtype=torch.int32)


def _spans(kind, n):
    g = torch.Generator().manual_seed(n)
    if kind == "padded":                                        # gaps inside a block of rows and a tile of keys
        return _padded([7, 16, 1, 11] * (n // 64), 16)
    if kind == "padded causal":
        return _padded([7, 16, 1, 11] * (n // 64), 16, causal=True)
    if kind == "wide":                                          # gaps of several tiles, next to keys of all rows
        return _padded([40, 3] * (n // 400), 200)
    if kind == "two ends":                                      # every row sees keys at one of the two ends, not in order
        side = torch.randint(0, 2, (1, n, 1), generator=g)
        return torch.where(side == 0, torch.tensor([5, 20]), torch.tensor([n - 30, n - 4])).int()
    first = torch.randint(0, n, (1, n, 1), generator=g)         # scattered: a few keys each, rows that see none among them
    return torch.cat([first, first + torch.randint(0, 3, (1, n, 1), generator=g)], -1).clamp(max=n).int() // 4 * 4


def _seen(spans, keys):
    j = torch.arange(keys)
    s = spans.cpu()
    see = (j >= s[..., :1]) & (j < s[..., 1:])
    return see.any(1), see.any(2)                               # keys that some row sees, rows that see some key


def _run(x, dout, **how):
    leaves = [t.clone().requires_grad_(True) for t in x]
    out, lse = span_attention(*leaves, return_lse=True, **how)
    return [out.detach(), lse, *torch.autograd.grad(out, leaves, dout)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 72, 128])
@pytest.mark.parametrize("kind,n", [("padded", 192), ("padded causal", 192), ("wide", 800), ("two ends", 500), ("scattered", 260)])
def test_what_unseen_keys_hold_does_not_matter(dtype, dim, kind, n):
    spans = _spans(kind, n)
    keys, rows = _seen(spans, n)
    assert not keys.all()
    spans = spans.cuda()
    q, k, v, dout = (_rand((1, n, h, dim), dtype, s) for s, h in enumerate((4, 2, 2, 4)))
    for x in (k, v):
        x[:, ~keys[0]] = 0
    for x in (q, dout):
        x[:, ~rows[0]] = 0
    how = dict(spans=spans, softcap=9.0, slopes=torch.full((4,), 0.01, device="cuda"))
    clean = _run((q, k, v), dout, **how)
    want = reference(q, k, v, dout, **how)
    for name, got in zip(("out", "lse", "dq", "dk", "dv"), clean):
        check(got, want, name)
    for bad in (math.nan, math.inf):
        y = [x.clone() for x in (q, k, v, dout)]
        for i, x in enumerate(y):
            x[:, ~(keys if i in (1, 2) else rows)[0]] = bad
        for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), clean, _run(y[:3], y[3], **how)):
            assert torch.equal(a, b), (name, bad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(4, 4), (6, 2)])
def test_few_rows_against_many_keys(dtype, heads, kv):
    """Keys split over workgroups, heads of a group as rows of one; queries finite, rows of every batch entry that sees keys compared."""
    n, dim = 3000, 64
    spans = torch.tensor([[[0, 100], [2000, 2900], [90, 130]], [[0, 0], [10, 11], [2999, 3000]], [[0, 0]] * 3, [[500, 700], [700, 900], [0, 3000]]],
                         dtype=torch.int32)
    keys, rows = _seen(spans, n)
    q, k, v = _rand((4, 3, heads, dim), dtype, 1), _rand((4, n, kv, dim), dtype, 2), _rand((4, n, kv, dim), dtype, 3)
    k[~keys] = 0
    v[~keys] = 0
    how = dict(spans=spans.cuda(), return_lse=True)
    clean = span_attention(q, k, v, **how)
    want = reference(q, k, v, spans=spans.cuda())
    check(clean[0], want, "out")
    check(clean[1], want, "lse")
    for bad in (math.nan, -math.inf):
        k[~keys] = bad
        v[~keys] = bad
        assert all(torch.equal(a, b) for a, b in zip(clean, span_attention(q, k, v, **how))), bad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nq,nk", [(40, 40), (3, 3000)])
def test_rows_that_see_none_are_nought_whatever_the_others_see(dtype, nq, nk):
    spans = torch.tensor([[[0, nk] if i % 2 else [0, 0] for i in range(nq)]], dtype=torch.int32, device="cuda")
    q, k, v, dout = _rand((1, nq, 2, 32), dtype, 1), _rand((1, nk, 2, 32), dtype, 2), _rand((1, nk, 2, 32), dtype, 3), _rand((1, nq, 2, 32), dtype, 4)
    k[0, 5, 0, 3] = math.nan
    v[0, 7, 1, 2] = math.inf
    out, lse, dq, _, _ = _run((q, k, v), dout, spans=spans)
    assert (out[:, ::2] == 0).all() and (dq[:, ::2] == 0).all() and (lse[..., ::2] == -math.inf).all()
    assert out[:, 1::2, 0].isnan().all() and not out[:, 1::2, 1, 2].isfinite().any()


def test_replayed_graph_finds_the_gaps_of_the_spans_it_meets():
    """Padded documents with a bias, forward and gradient, captured once; spans and inputs change between replays, and NaN stands at
    what is not seen."""
    n = 192
    q, k, v, dout = (_rand((1, n, h, 64), BF16, s) for s, h in enumerate((4, 2, 2, 4)))
    spans = _spans("padded", n).cuda()
    slopes = torch.full((4,), 0.01, device="cuda")
    step = lambda: _run((q, k, v), dout, spans=spans, slopes=slopes)          # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = step()
    for i, kind in enumerate(("scattered", "padded causal", "two ends", "padded")):
        spans.copy_(_spans(kind, n))
        keys, rows = _seen(spans, n)
        for m, x in enumerate((q, k, v, dout)):
            x.copy_(_rand(x.shape, BF16, 10 * i + m))
            x[:, ~(keys if m in (1, 2) else rows)[0]] = math.nan
        want = step()
        if i % 2:
            torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) and x.isnan().sum() == 0 for x, y in zip(got, want)), kind
