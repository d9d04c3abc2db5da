// Rotary positions with several axes (time, height, width): channel pair i of the d channels that axis a owns is turned by
//   theta = position[token][a] * base^(-2 i / d),   (x1, x2) -> (x1 cos - x2 sin, x2 cos + x1 sin);
// the gradient is the same turn by -theta. It stands beside the sinusoidal timestep embedding (embed.hip).
//
// Bound by HBM (x read once, y written once). A thread owns 16 bytes of channels of one token and loops over heads of q and
// k, so that angles are formed once per token and channel (interleaved: twice a pair, which costs nothing beside memory) and not once per
// head; 65536 tokens of 16 + 4 bf16 heads of 128
// channels and their gradient (1.34 GB) take 284 us, 4.7 TB/s, 95 % of a large copy's rate. Angles are formed in float64, in
// turns, and reduced there, off by 2^-51 of the position: a product in fp32 would be off by a whole radian at position 10^7; the sine and cosine
// of the reduced angle are fp32 like everything else.
#include <cmath>

#include "common.h"

using ddpm::as_stream;

namespace {

constexpr int kMaxAxes = DDPM_ROTARY_MAX_AXES;
constexpr int kMaxPairs = DDPM_ROTARY_MAX_DIM / 2;

struct Tensor {
    const void* x;
    void* out;
    int64_t xb, xn, xh, ob, on, oh;      // strides in elements: batch, token, head
};

struct RotaryDev {
    Tensor t[2];
    int heads0, heads;                   // heads of the first tensor, of both
    int heads_per_block;
    int tokens, dim, axes, interleaved;
    int64_t total;                       // batch * tokens
    float sign;
    const void* positions;
    int position_type;
    int64_t position_batch;              // stride, 0 = shared by the batch
    int end[kMaxAxes];                   // first channel behind each axis
    double turns[kMaxPairs];             // base^(-2 i / d) / (2 pi) of every pair, axis after axis
};

__device__ __forceinline__ double position_of(const RotaryDev& a, int64_t at) {
    if (a.position_type == DDPM_I32) return static_cast<const int32_t*>(a.positions)[at];
    if (a.position_type == DDPM_I64) return static_cast<double>(static_cast<const int64_t*>(a.positions)[at]);
    return static_cast<const float*>(a.positions)[at];
}

// W channels of 16-bit or 32-bit values per thread: 16 bytes, or one channel where sizes, strides or pointers do not allow it.
// PARTNER: the channels' partners are W neighbours too (every half axis a multiple of W) and come with one load; otherwise
// one at a time, from the line that is in the L1 by then, or, interleaved, from the thread's own channels. 65536 tokens of 16 + 4 heads of 128
// channels, forward, bf16 (fp32): 142 us (248) with partners, 142 (251) interleaved, 197 (267) with halves of 18, 22 and 24 channels,
// 302 (347) one channel a thread, with every head two bytes (four) off its boundary.
template <typename T, int W, bool PARTNER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryDev a) {
    typedef T V __attribute__((ext_vector_type(W)));
    const int per_token = a.dim / W;
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t token = id / per_token;
    if (token >= a.total) return;
    const int c0 = static_cast<int>(id - token * per_token) * W;
    const int64_t b = token / a.tokens, n = token - b * a.tokens;

    // y[c] = x[c] cosine[c] + x[partner[c]] sine[c]
    float cosine[W], sine[W];
    int partner[W];
    const int64_t where = b * a.position_batch + n * a.axes;
    int axis = 0, begin = 0;
#pragma unroll
    for (int e = 0; e < W; ++e) {
        const int c = c0 + e;
        while (axis < a.axes && c >= a.end[axis]) begin = a.end[axis++];
        cosine[e] = 1.f;
        sine[e] = 0.f;
        partner[e] = c;
        if (axis < a.axes) {
            const int half = (a.end[axis] - begin) >> 1, k = c - begin;
            const bool second = a.interleaved ? (k & 1) : k >= half;
            const int pair = a.interleaved ? k >> 1 : (second ? k - half : k);
            partner[e] = a.interleaved ? (second ? c - 1 : c + 1) : (second ? c - half : c + half);
            double r = position_of(a, where + axis) * a.turns[(begin >> 1) + pair];
            r -= rint(r);
            float s, co;
            sincospif(static_cast<float>(2.0 * r), &s, &co);
            cosine[e] = co;
            sine[e] = second ? a.sign * s : -a.sign * s;
        }
    }

    const int first = blockIdx.y * a.heads_per_block;
    const int last = min(first + a.heads_per_block, a.heads);
#pragma unroll 4
    for (int h = first; h < last; ++h) {
        const Tensor& t = a.t[h < a.heads0 ? 0 : 1];
        const int head = h < a.heads0 ? h : h - a.heads0;
        const T* __restrict__ x = static_cast<const T*>(t.x) + b * t.xb + n * t.xn + head * t.xh;
        T* __restrict__ out = static_cast<T*>(t.out) + b * t.ob + n * t.on + head * t.oh;
        const V own = *reinterpret_cast<const V*>(x + c0);
        V other;
        if (PARTNER) {
            other = *reinterpret_cast<const V*>(x + partner[0]);
        } else if (W > 1 && a.interleaved) {
#pragma unroll
            for (int e = 0; e < W; ++e) other[e] = own[e ^ 1];
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e) other[e] = x[partner[e]];
        }
        V y;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float v = static_cast<float>(own[e]);
            // channels behind the last axis pass as they are, NaN and infinities among them
            const float turned = fmaf(static_cast<float>(other[e]), sine[e], v * cosine[e]);
            y[e] = partner[e] == c0 + e ? own[e] : static_cast<T>(turned);
        }
        *reinterpret_cast<V*>(out + c0) = y;
    }
}

template <typename T>
void launch(RotaryDev& a, bool wide, bool partner, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    const int per_token = wide ? a.dim / W : a.dim;
    const int64_t blocks = (a.total * per_token + 255) / 256;
    // Heads of a thread: all of them where the tokens fill the chip (8 workgroups per compute unit), fewer where they do not.
    int64_t split = (2048 + blocks - 1) / blocks;
    if (split > a.heads) split = a.heads;
    a.heads_per_block = static_cast<int>((a.heads + split - 1) / split);
    const dim3 grid(static_cast<unsigned>(blocks), (a.heads + a.heads_per_block - 1) / a.heads_per_block);
    if (!wide)
        rotary_kernel<T, 1, false><<<grid, 256, 0, stream>>>(a);
    else if (partner)
        rotary_kernel<T, W, true><<<grid, 256, 0, stream>>>(a);
    else
        rotary_kernel<T, W, false><<<grid, 256, 0, stream>>>(a);
}

}  // namespace

extern "C" int ddpm_rotary(const ddpm_rotary_args* args, void* stream) {
    DDPM_REQUIRE(args);
    const ddpm_rotary_args& r = *args;
    DDPM_REQUIRE(r.type == DDPM_F32 || r.type == DDPM_BF16 || r.type == DDPM_F16);
    DDPM_REQUIRE(r.position_type == DDPM_I32 || r.position_type == DDPM_I64 || r.position_type == DDPM_F32);
    DDPM_REQUIRE(r.batch >= 0 && r.tokens >= 0 && r.tensors >= 1 && r.tensors <= 2);
    DDPM_REQUIRE(r.dim >= 2 && r.dim <= DDPM_ROTARY_MAX_DIM && r.axes >= 1 && r.axes <= kMaxAxes);
    DDPM_REQUIRE(r.base > 1.0 && std::isfinite(r.base));
    RotaryDev a = {};
    const int size = r.type == DDPM_F32 ? 4 : 2, width = 16 / size;
    bool wide = r.dim % width == 0, partner = !r.interleaved;
    int end = 0;
    for (int i = 0; i < r.axes; ++i) {
        const int d = r.axis_dim[i];
        DDPM_REQUIRE(d >= 2 && d % 2 == 0 && d <= r.dim - end);
        for (int k = 0; k < d / 2; ++k) a.turns[end / 2 + k] = std::pow(r.base, -2.0 * k / d) / (2.0 * M_PI);
        if ((d / 2) % width) partner = false;
        end += d;
        a.end[i] = end;
    }
    if (r.batch == 0 || r.tokens == 0) return DDPM_OK;
    DDPM_REQUIRE(r.positions);
    for (int i = 0; i < r.tensors; ++i) {
        DDPM_REQUIRE(r.x[i] && r.out[i] && r.x[i] != r.out[i] && r.heads[i] >= 1);
        const int64_t* xs = r.x_stride[i];
        const int64_t* os = r.out_stride[i];
        a.t[i] = {r.x[i], r.out[i], xs[0], xs[1], xs[2], os[0], os[1], os[2]};
        DDPM_REQUIRE(((reinterpret_cast<uintptr_t>(r.x[i]) | reinterpret_cast<uintptr_t>(r.out[i])) & (size - 1)) == 0);
        if (!ddpm::aligned16(r.x[i]) || !ddpm::aligned16(r.out[i])) wide = false;
        for (int s = 0; s < 3; ++s)
            if (xs[s] % width || os[s] % width) wide = false;
    }
    a.heads0 = r.heads[0];
    DDPM_REQUIRE(r.tensors == 1 || r.heads[1] <= INT32_MAX - r.heads[0]);
    a.heads = r.heads[0] + (r.tensors == 2 ? r.heads[1] : 0);
    DDPM_REQUIRE(a.heads <= 65535);
    a.tokens = r.tokens;
    a.dim = r.dim;
    a.axes = r.axes;
    a.interleaved = r.interleaved != 0;
    a.total = static_cast<int64_t>(r.batch) * r.tokens;
    DDPM_REQUIRE(a.total <= ((int64_t(1) << 32) - 256) / r.dim * (wide ? width : 1));      // threads of a launch within 2^32
    a.sign = r.inverse ? -1.f : 1.f;
    a.positions = r.positions;
    a.position_type = r.position_type;
    a.position_batch = r.position_batch_stride;
    if (r.type == DDPM_F32)
        launch<float>(a, wide, partner, as_stream(stream));
    else if (r.type == DDPM_BF16)
        launch<__bf16>(a, wide, partner, as_stream(stream));
    else
        launch<_Float16>(a, wide, partner, as_stream(stream));
    return ddpm::check_launch("rotary_kernel");
}
