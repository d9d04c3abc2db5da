"""Span attention in float64, with a bound for each output of what its roundings can add up to.

A rounding is off by half a step: u = 2^-24 relative in fp32; h for the 16-bit types (bf16 2^-8, fp16 2^-11), 0 in fp32.
  scores   t = scale q.k: (dim + 3) u sum |scale q k|; the cap adds 2^-21 of itself (exponential, quotient and product of its
           tanh), the bias and the subtraction of the maximum 4 u of their size
  weights  relative: the error of their score and that of the sum they are divided by: rho = 2 max error of the row + 8 u
  out      (rho + h + n u) sum p |v| + h |out|                 n: length of the sum; h: weights rounded to 16 bits, then the result
  D        (dim u + h) sum |dout out| + sum |dout| err(out)
  ds       rho |ds| + scale p (dim u sum |dout v| + err(D)) g + scale p |dp - D| err(g) + h |ds|; fp16 adds 2^-36 of the largest |ds|
  dq, dk, dv as sums of these, each with n u of its terms and h of itself."""
import math

import torch

U = 2.0 ** -24


def visible(q, k, spans=None, positions=None, causal=False):
    b, nq, nk, dev = q.shape[0], q.shape[1], k.shape[1], q.device
    j = torch.arange(nk, device=dev)
    pos = (torch.arange(nq, device=dev) + nk - nq)[None] if positions is None else positions.reshape(-1, nq).long()
    see = torch.ones(b, nq, nk, dtype=torch.bool, device=dev)
    if spans is not None:
        see &= (j >= spans[..., :1]) & (j < spans[..., 1:])
    if causal:
        see &= j <= pos[..., None]
    return see[:, None], (pos[..., None] - j).abs().double()[:, None]


def reference(q, k, v, dout=None, scale=None, softcap=0.0, slopes=None, spans=None, positions=None, causal=False):
    """{"out": (value, bound), "lse": ..., "dq": ..., "dk": ..., "dv": ...}, in the layouts of the operator."""
    h = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float64: 0.0}[q.dtype]
    half = q.dtype == torch.float16
    b, nq, heads, dim = q.shape
    nk, kvh = k.shape[1], k.shape[2]
    g = heads // kvh
    scale = dim ** -0.5 if scale is None else scale
    see, dist = visible(q, k, spans, positions, causal)
    heads_first = lambda x: x.double().transpose(1, 2).contiguous()                     # noqa: E731
    qd = heads_first(q)
    kd, vd = (heads_first(x).repeat_interleave(g, 1) for x in (k, v))
    t = scale * qd @ kd.transpose(2, 3).contiguous()
    err = (dim + 3) * U * abs(scale) * (qd.abs() @ kd.abs().transpose(2, 3).contiguous())
    w, dg, eg = t, torch.ones_like(t), torch.zeros_like(t)
    if softcap:
        th = torch.tanh(t / softcap)
        w = softcap * th
        err = err + softcap * 2.0 ** -21
        dg, eg = 1 - th * th, 2 * err / softcap
    err = err + 4 * U * w.abs()
    if slopes is not None:
        bias = slopes.double()[None, :, None, None] * dist
        w = w - bias
        err = err + 4 * U * bias.abs()
    w = torch.where(see, w, -math.inf)
    any_ = see.any(-1, keepdim=True)
    top = torch.where(any_, w.amax(-1, keepdim=True), 0.0) if nk else torch.zeros(b, heads, nq, 1, dtype=torch.float64, device=q.device)
    err = err + 4 * U * top.abs()
    e = torch.exp(w - top)
    s = e.sum(-1, keepdim=True)
    p = e / torch.where(s == 0, 1.0, s)
    seen_err = torch.where(see, err, 0.0)
    worst = seen_err.amax(-1, keepdim=True) if nk else torch.zeros_like(top)
    rho = 2 * worst + 8 * U
    out = p @ vd
    e_out = (rho + h + nk * U) * (p @ vd.abs()) + h * out.abs()
    lse = torch.where(any_, top + torch.log(torch.where(any_, s, 1.0)), -math.inf)[..., 0]
    e_lse = (worst + (nk + 8) * U + 4 * U * top.abs())[..., 0]
    back = lambda x: x.transpose(1, 2)                                                  # noqa: E731
    got = {"out": (back(out), back(e_out)), "lse": (lse, e_lse)}
    if dout is None:
        return got
    do = heads_first(dout)
    delta = (do * out).sum(-1, keepdim=True)
    e_delta = (dim * U + h) * (do * out).abs().sum(-1, keepdim=True) + (do.abs() * e_out).sum(-1, keepdim=True)
    dp = do @ vd.transpose(2, 3).contiguous()
    e_dp = dim * U * (do.abs() @ vd.abs().transpose(2, 3).contiguous())
    ds = scale * p * (dp - delta) * dg
    e_ds = (rho + h + 8 * U) * ds.abs() + abs(scale) * p * ((e_dp + e_delta) * dg + (dp - delta).abs() * eg)
    # An exponential or a product below 2^-126, the smallest normal float, is nought: p may lack all of so small a weight, ds that times
    # its other factors and, as a product, another 2^-126; each of the n terms of a sum may lack as much.
    tiny = torch.where(see, 2.0 ** -126, 0.0)
    e_p = (rho + h) * p + tiny
    e_ds = e_ds + tiny * (1 + abs(scale) * (dp - delta).abs() * dg)
    if half:
        e_ds = torch.where(see, e_ds + 2.0 ** -36 * ds.abs().amax((2, 3), keepdim=True), 0.0)
    share = lambda x: x.reshape(b, kvh, g, nk, dim).sum(2).transpose(1, 2)              # noqa: E731
    dq = ds @ kd
    got["dq"] = back(dq), back(e_ds @ kd.abs() + nk * U * (ds.abs() @ kd.abs()) + h * dq.abs())
    dst, pt = ds.transpose(2, 3).contiguous(), p.transpose(2, 3).contiguous()
    dk, dv = share(dst @ qd), share(pt @ do)
    n = nq * g * U
    got["dk"] = dk, share(e_ds.transpose(2, 3).contiguous() @ qd.abs()) + n * share(dst.abs() @ qd.abs()) + h * dk.abs()
    got["dv"] = dv, share(e_p.transpose(2, 3).contiguous() @ do.abs()) + n * share(pt @ do.abs()) + h * dv.abs()
    for name, terms in (("dq", nk), ("dk", nq * g), ("dv", nq * g)):
        got[name] = got[name][0], got[name][1] + terms * 2.0 ** -126
    if half:                                                    # the smallest steps of the type
        for name in ("out", "dq", "dk", "dv"):
            got[name] = got[name][0], got[name][1] + 2.0 ** -25
    return got


def check(got, want, name):
    value, bound = want[name]
    got = got.double()
    assert got.shape == value.shape, name
    assert torch.equal(got.isfinite(), value.isfinite()), f"{name}: not finite in other places"
    fine = value.isfinite()
    err, bound = (got - value)[fine].abs(), bound[fine] + 1e-38
    assert err.numel() == 0 or (err <= bound).all(), f"{name}: off by {(err / bound).max().item():.2f} times the bound, {err.max().item():.2e} at most"
