"""The kernels over lists of tensors at the places where a list is cut: tensors that end inside a chunk or a load, on and off 16-byte
boundaries, empty ones in between, lists of one launch and of several. Adam's step against torch.optim.Adam's formula in float64."""
import math

import pytest
import torch

from diffusion_model_amd import optim

pytestmark = pytest.mark.gpu


def _list(sizes, offset, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    room = sum(-(-(n + offset) // 4) * 4 for n in sizes) + 4
    flat, out, at = torch.full((room,), math.nan, device="cuda"), [], 0
    for n in sizes:
        out.append(flat[at + offset:at + offset + n].normal_(generator=g))
        at += -(-(n + offset) // 4) * 4
    return flat, out


@pytest.mark.parametrize("offset", [0, 1, 2])
@pytest.mark.parametrize("sizes", [[2047] * 90, [0, 1, 2, 3, 4, 5, 1023, 1024, 1025, 0, 2044, 2045, 2046, 2048, 2051, 4095, 6144, 0],
                                   [(7 * i) % 23 for i in range(500)], [0] * 88 + [5], [12345]])
def test_adam_step(offset, sizes):
    """Roundings of half a step: m and v one product and one sum each (m: of a difference), v's square two; the step a square root, two
    quotients and a sum, below 8 of them; the weight its own."""
    (pf, p), (gf, g), (mf, m), (vf, v) = (_list(sizes, offset, s) for s in range(4))
    for x in v:
        x.abs_()
    was = [[x.double() for x in y] for y in (p, g, m, v)]
    spare = [f.isnan() for f in (pf, gf, mf, vf)]
    optim.adam_step_(p, g, m, v, 3, lr=1e-2)
    for f, s in zip((pf, gf, mf, vf), spare):
        assert torch.equal(f.isnan(), s)                         # nothing beside the tensors was written
    u = 2.0 ** -24
    for i in range(len(sizes)):
        p0, g0, m0, v0 = (x[i] for x in was)
        m1 = m0 + (1 - 0.9) * (g0 - m0)
        v1 = 0.999 * v0 + (1 - 0.999) * g0 * g0
        step = 1e-2 / (1 - 0.9 ** 3) * m1 / (v1.sqrt() / math.sqrt(1 - 0.999 ** 3) + 1e-8)
        em = 4 * u * (m0.abs() + 0.1 * (g0 - m0).abs())
        assert ((m[i].double() - m1).abs() <= em).all()
        assert ((v[i].double() - v1).abs() <= 5 * u * v1).all()
        es = 16 * u * step.abs() + em * 1e-2 / (1 - 0.9 ** 3) / (v1.sqrt() / math.sqrt(1 - 0.999 ** 3) + 1e-8)
        assert ((p[i].double() - (p0 - step)).abs() <= es + u * (p0.abs() + step.abs())).all()


@pytest.mark.parametrize("sizes", [[2047] * 180, [(7 * i) % 23 for i in range(500)], [0] * 176 + [5], [0] * 64 + [8191, 0, 8193] + [0] * 64])
def test_norm_and_clipping(sizes):
    params = []
    for i, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
        p.grad = torch.full((n,), 1.0 + i % 5, device="cuda")
        params.append(p)
    norm = math.sqrt(sum(n * (1.0 + i % 5) ** 2 for i, n in enumerate(sizes)))
    assert float(optim.clip_grad_norm_(params, 0.5)) == pytest.approx(norm, rel=2.0 ** -23)
    for i, p in enumerate(params):
        assert ((p.grad.double() - (1.0 + i % 5) * 0.5 / (norm + 1e-6)).abs() <= 4 * 2.0 ** -24 * 5 * 0.5 / norm).all()
