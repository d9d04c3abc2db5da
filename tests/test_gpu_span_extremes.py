"""Span attention whose scores are as large as their types and its arguments allow."""
import math

import pytest
import torch

from diffusion_model_amd.attention import span_attention

pytestmark = pytest.mark.gpu


FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("nq,nk", [(5, 9), (40, 200), (1, 5000)])
@pytest.mark.parametrize("dtype,size", [(FP32, 2.0 ** 55), (BF16, 2.0 ** 55), (FP32, 2.0 ** 40), (BF16, 2.0 ** 18), (FP16, 2.0 ** 14), (FP32, 2.0 ** 12)])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size_have_a_largest(dtype, nq, nk, size, sign):
    """Scores sign (1 + j / 256) size^2 2^-2.5 32 / 8 of the j-th key, all powers of two but j's factor: neighbours are 2^14 and more apart,
    so that the whole weight is the largest one's (several have it where bf16 rounds j's factor), and its value comes out as it is."""
    j = torch.arange(nk) % 200
    first = 0 if sign < 0 else min(nk - 1, 199)
    k = (sign * (1 + j / 256.0) * size)[None, :, None, None].expand(1, nk, 1, 32).to(dtype).cuda()
    assert (k[0, :, 0, 0].double().cpu() == sign * (1 + j / 256.0) * size).all() or dtype == BF16
    top = k[0, :, 0, 0].double().cpu() * size
    hit = (top == top.max()).nonzero()[:, 0]
    assert first in hit
    q = torch.full((1, nq, 2, 32), size / 8, dtype=dtype, device="cuda")
    v = torch.randn(1, nk, 1, 32, generator=torch.Generator().manual_seed(0)).to(dtype)
    out, lse = span_attention(q, k, v.cuda(), return_lse=True)
    want = v[0, hit, 0].double().mean(0)
    h = {FP32: 0.0, BF16: 2.0 ** -8, FP16: 2.0 ** -11}[dtype]
    tol = (len(hit) + 8) * 2.0 ** -24 * v[0, hit, 0].double().abs().mean(0) + 2 * h * v[0, hit, 0].double().abs().mean(0)
    assert ((out[0].double().cpu() - want).abs() <= tol).all()
    value = float(top.max()) / 8 * 32 * 32 ** -0.5
    assert ((lse.double() - value).abs() <= abs(value) * 2.0 ** -21 + math.log(len(hit))).all()


def test_a_saturated_cap_of_the_largest_size():
    q, k = torch.full((1, 3, 1, 32), 1e17, device="cuda"), torch.full((1, 70, 1, 32), -1e17, device="cuda")
    v = torch.randn(1, 70, 1, 32, generator=torch.Generator().manual_seed(0)).cuda()
    out = span_attention(q, k, v, softcap=9e29)
    assert (out - v.mean(1, keepdim=True)).abs().max() <= 80 * 2.0 ** -24 * v.abs().max()
