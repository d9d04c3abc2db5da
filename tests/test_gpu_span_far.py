"""Span attention with a bias by distance where rows stand far from all keys that they see. A row's weights do not change when its
position moves to the nearest such key (all its distances shrink by the same number), so outputs and gradients have to meet the bounds that
span_reference.py derives for the moved positions, whose biases are small; lse those and half a step of itself on top."""
import pytest
import torch

from diffusion_model_amd import _lib
from diffusion_model_amd.attention import span_attention
from gpu_util import P, call, stream
from span_reference import check, reference

pytestmark = pytest.mark.gpu
FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [FP32, BF16, FP16]


def _rand(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).cuda()


def _case(dtype, b, nq, nk, heads, kv, dim, far, causal, spans):
    """Inputs; positions `far` from the keys, and moved to the nearest seen one; how far they moved."""
    q, k, v, dout = (_rand((b, n, h, dim), dtype, s, 1.5) for s, (n, h) in enumerate(((nq, heads), (nk, kv), (nk, kv), (nq, heads))))
    g = torch.Generator().manual_seed(7)
    pos = far + torch.randint(0, 50, (b, nq), generator=g)
    pos[:, ::5] = torch.randint(0, nk, pos[:, ::5].shape, generator=g)      # some stand among the keys
    ends = torch.sort(torch.randint(0, nk + 1, (b, nq, 2), generator=g), -1).values if spans else torch.tensor([0, nk]).expand(b, nq, 2)
    first, last = ends[..., 0], ends[..., 1]
    if causal:
        last = torch.minimum(last, pos + 1)
    near = torch.where(first < last, torch.minimum(torch.maximum(pos, first), last - 1), pos)
    how = dict(spans=ends.int().cuda().contiguous() if spans else None, causal=causal)
    return (q, k, v, dout), how, pos.int().cuda(), near.int().cuda(), (pos - near).abs().double().cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("far", [10 ** 6, -10 ** 6, 2 ** 30 - 60, -2 ** 30, 2 ** 24 - 20])
@pytest.mark.parametrize("causal,spans,softcap", [(False, False, 0.0), (False, True, 20.0), (True, True, 0.0)])
def test_rows_far_from_their_keys(dtype, far, causal, spans, softcap):
    (q, k, v, dout), how, pos, near, way = _case(dtype, 2, 70, 140, 4, 2, 64, far, causal, spans)
    slopes = torch.tensor([0.5, 0.1, 1e-3, 0.0], device="cuda")
    want = reference(q, k, v, dout, positions=near, slopes=slopes, softcap=softcap, **how)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    out, lse = span_attention(*leaves, positions=pos, slopes=slopes, softcap=softcap, return_lse=True, **how)
    grads = torch.autograd.grad(out, leaves, dout)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads)):
        check(got, want, name)
    value, bound = want["lse"]
    shift = slopes.double()[None, :, None] * way[:, None]
    # the distance, its product and the difference are rounded
    check(lse, {"lse": (value - shift, bound + 3 * 2.0 ** -24 * (shift + value.nan_to_num(neginf=0.0).abs()))}, "lse")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("far", [10 ** 6, -10 ** 6])
def test_few_rows_against_many_keys(dtype, far):
    (q, k, v, _), how, pos, near, way = _case(dtype, 2, 3, 4000, 4, 2, 64, far, False, True)
    slopes = torch.tensor([0.5, 0.1, 1e-3, 0.0], device="cuda")
    want = reference(q, k, v, positions=near, slopes=slopes, **how)
    out, lse = span_attention(q, k, v, positions=pos, slopes=slopes, return_lse=True, **how)
    check(out, want, "out")
    value, bound = want["lse"]
    shift = slopes.double()[None, :, None] * way[:, None]
    check(lse, {"lse": (value - shift, bound + 3 * 2.0 ** -24 * (shift + value.nan_to_num(neginf=0.0).abs()))}, "lse")


def test_far_windows_without_positions():
    """Rows stand at their index; the keys that their spans show them are 60000 further on."""
    nq, nk = 200, 60200
    q, k, v = _rand((1, nq, 2, 32), BF16, 1, 1.5), _rand((1, nk, 2, 32), BF16, 2, 1.5), _rand((1, nk, 2, 32), BF16, 3)
    first = torch.arange(nq)[None] + 59900
    spans = torch.stack([first, first + 100], -1).int().cuda()
    slopes = torch.tensor([1.0, 0.25], device="cuda")
    standing = torch.arange(nq, device="cuda")[None].int()
    want = reference(q, k, v, positions=spans[..., 0], spans=spans, slopes=slopes)
    check(span_attention(q, k, v, spans=spans, slopes=slopes, positions=standing), want, "out")


@pytest.mark.parametrize("near", [True, False])
def test_the_entry_points_with_and_without_the_near_statistic(near):
    """Without lse_near the backward call takes its weights from lse: at distances of 5000 and slopes of 0.05 off by 2^-24 of 250 at most,
    which span_reference.py's bounds have for biases of that size."""
    (q, k, v, dout), how, pos, moved, _ = _case(FP32, 2, 70, 140, 4, 2, 64, 5000, False, True)
    slopes = torch.full((4,), 0.05, device="cuda")
    want = reference(q, k, v, dout, positions=pos, slopes=slopes, **how)
    a = _lib.SpanAttentionArgs()
    a.type, a.batch, a.nq, a.nk, a.heads, a.kv_heads, a.dim, a.scale = 0, 2, 70, 140, 4, 2, 64, 64 ** -0.5
    a.slopes, a.spans, a.positions, a.span_batch_stride, a.position_batch_stride = slopes.data_ptr(), how["spans"].data_ptr(), pos.data_ptr(), 140, 70
    made = {n: torch.full_like(x, float("nan")) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    lse, stat = (torch.empty(2, 4, 70, device="cuda") for _ in range(2))
    for name, x in dict(q=q, k=k, v=v, dout=dout, **made).items():
        setattr(a, name, x.data_ptr())
        getattr(a, name + "_stride")[:] = x.stride()[:3]
    a.lse, a.lse_near = lse.data_ptr(), stat.data_ptr() if near else None
    import ctypes as C
    for entry in ("ddpm_span_attention_fwd", "ddpm_span_attention_bwd"):
        size = getattr(_lib.lib(), entry + "_workspace")(C.byref(a))
        workspace = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
        call(entry, C.byref(a), P(workspace), stream())
    check(lse, want, "lse")
    for name, x in made.items():
        check(x, want, name)
