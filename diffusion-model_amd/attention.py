"""Span attention: several heads, keys and values shared by groups of query heads, scores capped by a tanh, a bias by
distance, and masks in which every row sees one span of keys (documents packed into a sequence, prefixes, padded lengths,
windows, causal order), with its gradient. It stands beside the UNet's own self-attention (second-iteration/unet.py:39-61: one
head, every pixel sees every pixel) for networks over tokens of images, video and text."""
import torch

from ._lib import SpanAttentionArgs, call, lib, on_gpu, packer, refuse_tangents, stream_of

_TYPES = {torch.float32: (0, 4), torch.bfloat16: (1, 8), torch.float16: (2, 8)}      # DDPM_* code, elements of 16 bytes
MAX_DIM = 128


def key_spans(rows, keys=None, *, documents=None, prefix=None, lengths=None, window=None, causal=False, device=None):
    """Spans [first, last) of keys that each of `rows` rows sees, int32 [batch or 1][rows][2], for span_attention. Row i stands at
    position i + keys - rows; every condition given narrows what it sees:
      documents  [batch][keys] or [keys], any integers: a document is a run of equal ones; rows see their own document
      causal     no key behind the row's position
      prefix     an int or [batch]: causal, but all see the first `prefix` keys (of their document)
      lengths    [batch]: keys from lengths[b] on hold nothing, and rows that stand there see nothing
      window     (left, right): keys at most that far before and behind the row's position"""
    keys = rows if keys is None else keys
    if rows < 0 or keys < 0:
        raise ValueError(f"key_spans: {rows} rows, {keys} keys")
    if device is None:
        given = [t.device for t in (documents, prefix, lengths) if isinstance(t, torch.Tensor)]
        device = given[0] if given else "cuda"
    at = torch.arange(rows, device=device)[None] + (keys - rows)
    first, last = torch.zeros_like(at), torch.full_like(at, keys)
    if documents is not None:
        d = documents.to(device)
        d = d[None] if d.dim() == 1 else d
        if d.dim() != 2 or d.shape[1] != keys:
            raise ValueError(f"key_spans: documents are [batch][{keys}], got {tuple(documents.shape)}")
        j = torch.arange(keys, device=device).expand_as(d)
        new = torch.ones_like(d, dtype=torch.bool)
        new[:, 1:] = d[:, 1:] != d[:, :-1]
        begin = torch.where(new, j, 0).cummax(1).values if keys else j
        stop = torch.where(new, j, keys).roll(-1, 1) if keys else j
        if keys:
            stop[:, -1] = keys
            stop = stop.flip(1).cummin(1).values.flip(1)
        own = at.clamp(0, max(keys - 1, 0)).expand(d.shape[0], rows)
        inside = (at >= 0) & (at < keys)
        first = begin.gather(1, own)
        last = torch.where(inside, stop.gather(1, own), first)
    if prefix is not None:
        p = prefix.to(device).reshape(-1, 1) if isinstance(prefix, torch.Tensor) else torch.tensor([[prefix]], device=device)
        last = torch.minimum(last, torch.maximum(at + 1, first + p))
    if causal:
        last = torch.minimum(last, at + 1)
    if window is not None:
        left, right = window
        first = torch.maximum(first, at - left)
        last = torch.minimum(last, at + right + 1)
    if lengths is not None:
        n = lengths.to(device).reshape(-1, 1)
        last = torch.where(at < n, torch.minimum(last, n), 0)
    first, last = torch.broadcast_tensors(first, torch.maximum(last, first))
    return torch.stack([first, last], -1).to(torch.int32)


def _fit(x, width):
    """x, or a copy, with neighbouring channels on 16-byte boundaries and 64 rows within 2 GiB; and its strides."""
    batch, rows, heads, dim = x.shape
    if x.is_contiguous() and x.data_ptr() % 16 == 0:
        return x, (rows * heads * dim, heads * dim, dim)
    strides = [s if n > 1 else 0 for n, s in zip(x.shape, x.stride())]
    if (x.stride(3) != 1 or x.data_ptr() % 16 or any(s % width for s in strides[:3])
            or strides[1] * x.element_size() >= 1 << 25):
        return x.clone(memory_format=torch.contiguous_format), (rows * heads * dim, heads * dim, dim)
    return x, strides[:3]


def _address(x):
    return 0 if x is None else x.data_ptr()


_pack = packer(SpanAttentionArgs)
_NO_GRADIENT = (0,) * 16


def _run(entry, q, k, v, out, low, lse, near, how, gradient=_NO_GRADIENT):
    """q, k, v, out: (tensor, strides). Runs on the current GPU, the tensors' own."""
    scale, softcap, slopes, spans, positions, causal = how
    x, y = q[0], k[0]
    batch, rows, heads, dim = x.shape
    _, keys, kv_heads, _ = y.shape
    a = _pack(_TYPES[x.dtype][0], batch, rows, keys, heads, kv_heads, dim, causal, scale, softcap, _address(slopes), _address(spans),
              _address(positions), spans.stride(0) if spans is not None and spans.shape[0] > 1 else 0,
              positions.stride(0) if positions is not None and positions.shape[0] > 1 else 0, x.data_ptr(), y.data_ptr(), v[0].data_ptr(),
              out[0].data_ptr(), _address(low), _address(lse), *q[1], *k[1], *v[1], *out[1], *gradient, _address(near))
    size = getattr(lib(), entry + "_workspace")(a)
    workspace = x.new_empty(size, dtype=torch.uint8) if size > 0 else None
    call(entry, a, _address(workspace), stream_of(x.get_device()))


def _forward(q, k, v, how, with_lse, training=False):
    width = _TYPES[q.dtype][1]
    q, k, v = _fit(q, width), _fit(k, width), _fit(v, width)
    x = q[0]
    batch, rows, heads, dim = x.shape
    with on_gpu(x.get_device()):
        out = torch.empty_like(x, memory_format=torch.contiguous_format)
        lse = x.new_empty((batch, heads, rows), dtype=torch.float32) if with_lse else None
        low = torch.empty_like(out) if training and x.dtype != torch.float32 else None
        near = torch.empty_like(lse) if training and how[2] is not None else None       # without a bias it is lse
        _run("ddpm_span_attention_fwd", q, k, v, _fit(out, width), low, lse, near, how)
    return x, k[0], v[0], out, low, lse, near


class _SpanAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, softcap, slopes, spans, positions, causal):
        q, k, v, out, low, lse, near = _forward(q, k, v, (scale, softcap, slopes, spans, positions, causal), True, True)
        ctx.save_for_backward(q, k, v, out, low, lse, near, slopes, spans, positions)
        ctx.how = scale, softcap, causal
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _):
        if dout is None:
            return (None,) * 9
        q, k, v, out, low, lse, near, slopes, spans, positions = ctx.saved_tensors
        scale, softcap, causal = ctx.how
        width = _TYPES[q.dtype][1]
        with on_gpu(q.get_device()):
            dout, ds = _fit(dout, width)
            dq, dk, dv = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
            (_, qs), (_, ks) = _fit(dq, width), _fit(dk, width)
            gradient = dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), *ds, *qs, *ks, *ks
            _run("ddpm_span_attention_bwd", _fit(q, width), _fit(k, width), _fit(v, width), _fit(out, width), low, lse, near,
                 (scale, softcap, slopes, spans, positions, causal), gradient)
        return dq, dk, dv, None, None, None, None, None, None


def span_attention(q, k, v, *, scale=None, softcap=0.0, slopes=None, spans=None, positions=None, causal=False, return_lse=False):
    """softmax(w) v over the keys that each row sees, w = softcap tanh(scale q.k / softcap) - slope |position - j|.

    q: [batch][rows][heads][dim]; k, v: [batch][keys][kv_heads][dim] with heads a multiple of kv_heads (query head h uses
    key/value head h // (heads / kv_heads)); float32, bfloat16 or float16, dim at most 128, any strides (16-byte aligned
    ones are used in place, others through a copy).
      scale      of q.k; dim ** -0.5 when not given          softcap    0: no cap
      slopes     float32 [heads], or None: no bias           causal     row i sees no key behind its position
      spans      int32 [batch or 1][rows][2]: the keys [first, last) of each row (key_spans makes them), or None: all
      positions  int32 [rows] or [batch or 1][rows], within 2^30 of 0; row i stands at i + keys - rows when not given
    A row that sees no key comes out as noughts. Single tokens against long keys (rows = 1, one span each) are split over
    the GPU. Returns out [batch][rows][heads][dim], with return_lse also the log-sum-exp of w, float32
    [batch][heads][rows] (-inf for a row that sees none), which has no gradient; q, k and v have one, whose weights exp(w - lse)
    are off by up to 2^-21 |w| of themselves: scores in the millions leave it few right digits, from some 10^8 on none."""
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != 4:
            raise ValueError(f"span_attention: {name} is [batch][tokens][heads][dim], got {tuple(x.shape)}")
        if x.dtype not in _TYPES or x.dtype != q.dtype:
            raise TypeError(f"span_attention: q, k and v are of one type, float32, bfloat16 or float16, got {q.dtype} and {x.dtype}")
    batch, rows, heads, dim = q.shape
    if k.shape != v.shape or k.shape[0] != batch or k.shape[3] != dim or k.shape[2] < 1 or heads < 1 or heads % k.shape[2]:
        raise ValueError(f"span_attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f"span_attention: at most {MAX_DIM} channels a head, got {dim}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not abs(scale) < 1e30:
        raise ValueError(f"span_attention: scale must be finite, got {scale}")
    if softcap and not (1e-30 < softcap < 1e30 and abs(scale) / softcap < 1e30):
        raise ValueError(f"span_attention: softcap is 0 or a positive number that the scale does not dwarf, got {softcap} with scale {scale}")
    if slopes is not None:
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,):
            raise ValueError(f"span_attention: slopes are float32 [{heads}], got {slopes.dtype} {tuple(slopes.shape)}")
        if slopes.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("span_attention: slopes have no gradient")
        slopes = slopes.contiguous()
    if spans is not None:
        if spans.dtype != torch.int32 or tuple(spans.shape) not in ((batch, rows, 2), (1, rows, 2)):
            raise ValueError(f"span_attention: spans are int32 [{batch} or 1][{rows}][2], got {spans.dtype} {tuple(spans.shape)}")
        spans = spans.contiguous()
    if positions is not None:
        positions = positions[None] if positions.dim() == 1 else positions
        if positions.dtype != torch.int32 or tuple(positions.shape) not in ((batch, rows), (1, rows)):
            raise ValueError(f"span_attention: positions are int32 [{batch} or 1][{rows}], got {positions.dtype} {tuple(positions.shape)}")
        positions = positions.contiguous()
    refuse_tangents("span_attention", (q, k, v, slopes))
    if not all(x.is_cuda and x.device == q.device for x in (q, k, v, slopes, spans, positions) if x is not None):
        raise RuntimeError("span_attention runs on the MI355X only: all tensors must be on one GPU")
    spare = -dim % _TYPES[q.dtype][1]
    if spare:                                                   # noughts fill the last 16 bytes of a head
        q, k, v = (torch.nn.functional.pad(x, (0, spare)) for x in (q, k, v))
    if torch.is_grad_enabled() and any(x.requires_grad for x in (q, k, v)):
        out, lse = _SpanAttention.apply(q, k, v, scale, float(softcap), slopes, spans, positions, bool(causal))
    else:
        _, _, _, out, _, lse, _ = _forward(q, k, v, (scale, float(softcap), slopes, spans, positions, bool(causal)), return_lse)
    if spare:
        out = out[..., :dim].contiguous()
    return (out, lse) if return_lse else out
