"""Sinusoidal timestep embedding module (interface of first-iteration/embeddings.py:6-20), and rotary positions with
several axes (time, height, width) for the tokens of images and video."""
import ctypes as C

import torch
import torch.nn as nn

from ._lib import RotaryArgs, call, on_gpu, packer, refuse_tangents, stream_of


class SinusoidalTimeEmbedding(nn.Module):
    def __init__(self, embedding_dim):
        super().__init__()
        self.embedding_dim = embedding_dim

    def forward(self, timesteps):
        if not timesteps.is_cuda:
            raise RuntimeError("SinusoidalTimeEmbedding runs on the MI355X only: move `timesteps` to the GPU")
        if timesteps.dtype not in (torch.int64, torch.float32):
            timesteps = timesteps.to(torch.float32 if timesteps.is_floating_point() else torch.int64)
        t = timesteps.contiguous()
        half = self.embedding_dim // 2
        out = torch.empty((t.shape[0], 2 * half), device=t.device, dtype=torch.float32)
        call("ddpm_sinusoidal_embedding", C.c_void_p(t.data_ptr()), int(t.dtype == torch.float32), t.shape[0],
             self.embedding_dim, C.c_void_p(out.data_ptr()), C.c_void_p(torch.cuda.current_stream().cuda_stream))
        return out


_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}                  # DDPM_F32, DDPM_BF16, DDPM_F16
_POSITION_TYPES = {torch.float32: 0, torch.int32: 3, torch.int64: 4}              # DDPM_F32, DDPM_I32, DDPM_I64


def grid_positions(*sizes, device="cuda"):
    """Positions of the tokens of a grid, row by row: int32 [prod(sizes)][len(sizes)]. grid_positions(height, width) for
    images, grid_positions(time, height, width) for video."""
    if not sizes or any(int(n) < 1 for n in sizes):
        raise ValueError(f"grid_positions: sizes must be positive, got {sizes}")
    axes = [torch.arange(int(n), dtype=torch.int32, device=device) for n in sizes]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).reshape(-1, len(sizes))


_pack = packer(RotaryArgs)
_ptr = torch.Tensor.data_ptr


def _turn(tensors, positions, axes, base, interleaved, inverse):
    tensors = [x if x.stride(3) == 1 else x.contiguous() for x in tensors]
    first = tensors[0]
    batch, tokens, _, dim = first.shape
    gpu = first.get_device()
    with on_gpu(gpu):
        outs = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in tensors]
        spare = 2 - len(tensors)                                # no k
        strides = [n for s in (tensors, outs) for n in (*(n for x in s for n in x.stride()[:3]), *(0,) * 3 * spare)]
        heads, *pointers = ((*values, *(0,) * spare) for values in ([x.shape[2] for x in tensors], map(_ptr, tensors), map(_ptr, outs)))
        a = _pack(_TYPES[first.dtype], batch, tokens, dim, len(axes), *axes, *(0,) * (4 - len(axes)), bool(interleaved), inverse,
                  _POSITION_TYPES[positions.dtype], len(tensors), *heads, base, _ptr(positions),
                  positions.stride(0) if positions.dim() == 3 and positions.shape[0] > 1 else 0, *pointers[0], *pointers[1], *strides)
        call("ddpm_rotary", a, stream_of(gpu))
    return outs


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, axes, base, interleaved, *tensors):
        ctx.save_for_backward(positions)
        ctx.how = axes, base, interleaved
        ctx.set_materialize_grads(False)
        return tuple(_turn(tensors, positions, axes, base, interleaved, False))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        given = [g for g in grads if g is not None]
        turned = iter(_turn(given, *ctx.saved_tensors, *ctx.how, True) if given else ())
        return (None,) * 4 + tuple(None if g is None else next(turned) for g in grads)


def rotary(q, k, positions, axes, base=10000.0, interleaved=False):
    """Rotary positions of queries [batch][tokens][heads][dim] and keys (own head count, or None), as new tensors; one launch,
    with a gradient for q and k. Axis a owns axes[a] channels (even), consecutive from channel 0; its pair i is turned by
    positions[..., a] * base^(-2 i / axes[a]); further channels pass. Pairs are (i, axes[a]/2 + i), or with interleaved
    (2 i, 2 i + 1). positions: [tokens][len(axes)], or [batch or 1][tokens][len(axes)]; int32, int64 or float32, angles are
    formed in float64, off by 2^-51 radian for each unit of the position. q and k: float32, bfloat16 or float16, any strides.
    Returns (q, k), or q alone when k is None."""
    tensors = (q,) if k is None else (q, k)
    axes = tuple(int(d) for d in axes)
    for x in tensors:
        if x.dim() != 4:
            raise ValueError(f"rotary: q and k are [batch][tokens][heads][dim], got {tuple(x.shape)}")
        if x.dtype not in _TYPES or x.dtype != q.dtype:
            raise TypeError(f"rotary: q and k are of one type, float32, bfloat16 or float16, got {q.dtype} and {x.dtype}")
        if x.shape[:2] != q.shape[:2] or x.shape[3] != q.shape[3]:
            raise ValueError(f"rotary: q {tuple(q.shape)} and k {tuple(x.shape)} differ in more than their heads")
    if not 1 <= len(axes) <= 4 or any(d < 2 or d % 2 for d in axes) or sum(axes) > q.shape[3]:
        raise ValueError(f"rotary: axes are 1 to 4 even channel counts of together at most {q.shape[3]}, got {axes}")
    if q.shape[3] > 512:
        raise ValueError(f"rotary: at most 512 channels, got {q.shape[3]}")
    if positions.dtype not in _POSITION_TYPES or positions.requires_grad and torch.is_grad_enabled():
        raise TypeError(f"rotary: positions are int32, int64 or float32 without a gradient, got {positions.dtype}")
    batch, tokens = q.shape[:2]
    if tuple(positions.shape) not in ((tokens, len(axes)), (batch, tokens, len(axes)), (1, tokens, len(axes))):
        raise ValueError(f"rotary: positions are [tokens][axes] or [batch][tokens][axes] for {(batch, tokens, len(axes))}, got {tuple(positions.shape)}")
    refuse_tangents("rotary", (*tensors, positions))
    if not all(x.is_cuda and x.device == q.device for x in (*tensors, positions)):
        raise RuntimeError("rotary runs on the MI355X only: q, k and positions must be on one GPU")
    positions = positions.contiguous()
    if torch.is_grad_enabled() and any(x.requires_grad for x in tensors):
        out = _Rotary.apply(positions, axes, float(base), interleaved, *tensors)
    else:
        out = tuple(_turn(tensors, positions, axes, float(base), interleaved, False))
    return out[0] if k is None else out
