"""Span attention without a GPU: workspace sizes, refusals and key spans."""
import ctypes as C

import pytest

from diffusion_model_amd import _lib


def _args(at, **sizes):
    a = _lib.SpanAttentionArgs()
    a.batch, a.nq, a.nk, a.heads, a.kv_heads, a.dim, a.scale = 1, 8192, 8192, 8, 8, 128, 0.1
    for name in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        setattr(a, name, at)
    for k, v in sizes.items():
        setattr(a, k, v)
    for name, n, h in (("q", a.nq, a.heads), ("out", a.nq, a.heads), ("k", a.nk, a.kv_heads), ("v", a.nk, a.kv_heads)):
        for prefix in ("", "d"):
            getattr(a, prefix + name + "_stride")[:] = (n * h * a.dim, h * a.dim, a.dim)
    return a


@pytest.mark.parametrize("kind", [0, 1, 2])
@pytest.mark.parametrize("sizes", [dict(), dict(nq=1, nk=65536), dict(nq=300, nk=4096, heads=4, kv_heads=1, dim=64), dict(nq=4096, nk=300, heads=4, kv_heads=1),
                                   dict(batch=3, nq=2125, nk=2125, dim=64), dict(batch=65535 + 7, nq=900, nk=90, heads=2, kv_heads=1, dim=32)])
def test_workspaces_follow_from_sizes_and_type_alone(kind, sizes):
    """As the header says: one workspace for all calls of a shape, whatever masks and biases they have."""
    a = _args(4096, type=kind, **sizes)
    for size in (_lib.lib().ddpm_span_attention_fwd_workspace, _lib.lib().ddpm_span_attention_bwd_workspace):
        plain = size(C.byref(a))
        assert plain >= 0
        for given in (("spans",), ("slopes",), ("positions",), ("out_low",), ("spans", "slopes", "positions", "out_low")):
            b = _args(4096, type=kind, causal=1, softcap=5.0, **sizes)
            for name in given:
                setattr(b, name, 4096)
            assert size(C.byref(b)) == plain, given
