// Adam update of a list of tensors in one or a few launches (the optimizer.step() that follows every
// backward of the training loop, first-iteration/main.py:51,84: torch.optim.Adam with its defaults).
// HBM-bound: 16 bytes read and 12 written per parameter element.  The tensor list travels in the kernel
// arguments, so the call allocates nothing and copies nothing.
// A device scalar may scale every gradient as it is read (ddpm_adam_step_clipped with the factor of ddpm_grad_norm): the
// clipped gradients are never written, which saves a pass of 8 bytes per element and a launch.
#include <cmath>

#include "tensor_list.h"

namespace {

constexpr int kTensorsPerLaunch = 88;     // 44 bytes of kernel arguments each, below 4 KiB together
constexpr int64_t kChunk = 2048;          // elements: two 16-byte loads of each of the four arrays per thread in flight
constexpr int kMaxBlocks = 4096;

struct AdamBatch {
    ddpm::ChunkMap<kTensorsPerLaunch> map;
    float* p[kTensorsPerLaunch];
    const float* g[kTensorsPerLaunch];
    float* m[kTensorsPerLaunch];
    float* v[kTensorsPerLaunch];
    int64_t n[kTensorsPerLaunch];
};

struct AdamScalars {
    float b1, b2, one_minus_b1, one_minus_b2, step_size, bc2_sqrt, eps, weight_decay;
};

// the arithmetic of torch.optim.Adam: m.lerp_(g, 1-b1); v.mul_(b2).addcmul_(g, g, 1-b2);
// p.addcdiv_(m, sqrt(v)/sqrt(1-b2^t) + eps, -lr/(1-b1^t))
__device__ __forceinline__ void adam_elem(float& p, float g, float& m, float& v, const AdamScalars& s) {
    if (s.weight_decay != 0.f) g = fmaf(s.weight_decay, p, g);
    m = fmaf(s.one_minus_b1, g - m, m);
    v = fmaf(s.one_minus_b2 * g, g, v * s.b2);
    const float denom = sqrtf(v) / s.bc2_sqrt + s.eps;
    p = fmaf(-s.step_size, m / denom, p);
}

using f32x4 = __attribute__((ext_vector_type(4))) float;

template <bool CLIP>
__global__ __launch_bounds__(256) void adam_kernel(const AdamBatch b, const AdamScalars s, const float* __restrict__ factor) {
    const float f = CLIP ? factor[0] : 1.f;
    for (int c = blockIdx.x; c < b.map.chunks; c += gridDim.x) {
        const int t = ddpm::tensor_of_chunk(b.map, c);
        const int64_t begin = static_cast<int64_t>(c - b.map.first[t]) * kChunk;
        const int64_t end = begin + kChunk < b.n[t] ? begin + kChunk : b.n[t];
        float* __restrict__ p = b.p[t];
        const float* __restrict__ g = b.g[t];
        float* __restrict__ m = b.m[t];
        float* __restrict__ v = b.v[t];
        const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m) |
                           reinterpret_cast<uintptr_t>(v)) & 15) == 0;
        // All loads of a thread are in flight before the first store, behind a tensor's end and off 16-byte boundaries too: 400 tensors of 2047
        // elements take 16.3 us, 300 of 1 to 8192 12.6; elements one by one, and tensors searched for by halves, made that 22.4 and 17.1.
        const int n = static_cast<int>(end - begin);
        if (vec) {
            constexpr int kLoads = static_cast<int>(kChunk) / 1024;
            f32x4 pv[kLoads], gv[kLoads], mv[kLoads], vv[kLoads];
            const int count = n >> 2;
            const int64_t first = begin >> 2;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = threadIdx.x + i * 256;
                pv[i] = gv[i] = mv[i] = vv[i] = f32x4{};
                if (at >= count) continue;
                pv[i] = reinterpret_cast<const f32x4*>(p)[first + at];
                gv[i] = reinterpret_cast<const f32x4*>(g)[first + at];
                mv[i] = reinterpret_cast<const f32x4*>(m)[first + at];
                vv[i] = reinterpret_cast<const f32x4*>(v)[first + at];
            }
            const int64_t last = begin + 4 * count + threadIdx.x;        // up to three elements more
            float pe = 0.f, ge = 0.f, me = 0.f, ve = 0.f;
            if (last < end) {
                pe = p[last];
                ge = g[last];
                me = m[last];
                ve = v[last];
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = threadIdx.x + i * 256;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float px = pv[i][e], mx = mv[i][e], vx = vv[i][e];
                    adam_elem(px, CLIP ? gv[i][e] * f : gv[i][e], mx, vx, s);
                    pv[i][e] = px;
                    mv[i][e] = mx;
                    vv[i][e] = vx;
                }
                if (at >= count) continue;
                reinterpret_cast<f32x4*>(p)[first + at] = pv[i];
                reinterpret_cast<f32x4*>(m)[first + at] = mv[i];
                reinterpret_cast<f32x4*>(v)[first + at] = vv[i];
            }
            if (last < end) {
                adam_elem(pe, CLIP ? ge * f : ge, me, ve, s);
                p[last] = pe;
                m[last] = me;
                v[last] = ve;
            }
        } else {
            constexpr int kSingle = static_cast<int>(kChunk) / 256;
            float ps[kSingle], gs[kSingle], ms[kSingle], vs[kSingle];
#pragma unroll
            for (int i = 0; i < kSingle; ++i) {
                const int64_t at = begin + threadIdx.x + i * 256;
                ps[i] = gs[i] = ms[i] = vs[i] = 0.f;
                if (at >= end) continue;
                ps[i] = p[at];
                gs[i] = g[at];
                ms[i] = m[at];
                vs[i] = v[at];
            }
#pragma unroll
            for (int i = 0; i < kSingle; ++i) {
                const int64_t at = begin + threadIdx.x + i * 256;
                adam_elem(ps[i], CLIP ? gs[i] * f : gs[i], ms[i], vs[i], s);
                if (at >= end) continue;
                p[at] = ps[i];
                m[at] = ms[i];
                v[at] = vs[i];
            }
        }
    }
}

int adam_step(int ntensors, float* const* params, const float* const* grads, float* const* exp_avg, float* const* exp_avg_sq,
              const int64_t* numel, double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
              const float* factor, void* stream) {
    DDPM_REQUIRE(ntensors >= 0 && step >= 1 && lr >= 0.0 && eps >= 0.0);
    DDPM_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && weight_decay >= 0.0);
    if (ntensors == 0) return 0;
    DDPM_REQUIRE(params && grads && exp_avg && exp_avg_sq && numel);
    // the scalars as torch.optim.Adam forms them: in double, rounded to float where they meet the tensors
    const double bc1 = 1.0 - std::pow(beta1, static_cast<double>(step));
    const double bc2 = 1.0 - std::pow(beta2, static_cast<double>(step));
    AdamScalars s;
    s.b1 = static_cast<float>(beta1);
    s.b2 = static_cast<float>(beta2);
    s.one_minus_b1 = static_cast<float>(1.0 - beta1);
    s.one_minus_b2 = static_cast<float>(1.0 - beta2);
    s.step_size = static_cast<float>(lr / bc1);
    s.bc2_sqrt = static_cast<float>(std::sqrt(bc2));
    s.eps = static_cast<float>(eps);
    s.weight_decay = static_cast<float>(weight_decay);
    hipStream_t st = ddpm::as_stream(stream);
    for (int i = 0; i < ntensors; ++i) {
        DDPM_REQUIRE(numel[i] >= 0 && numel[i] <= ddpm::kLongestTensor);
        DDPM_REQUIRE(numel[i] == 0 || (params[i] && grads[i] && exp_avg[i] && exp_avg_sq[i]));
    }
    DDPM_REQUIRE(ddpm::chunks_fit(ntensors, numel, kTensorsPerLaunch, kChunk));
    for (int t0 = 0; t0 < ntensors; t0 += kTensorsPerLaunch) {
        AdamBatch b;
        const int cnt = ntensors - t0 < kTensorsPerLaunch ? ntensors - t0 : kTensorsPerLaunch;
        ddpm::map_chunks(b.map, numel + t0, cnt, kChunk);
        for (int i = 0; i < cnt; ++i) {
            b.p[i] = params[t0 + i];
            b.g[i] = grads[t0 + i];
            b.m[i] = exp_avg[t0 + i];
            b.v[i] = exp_avg_sq[t0 + i];
            b.n[i] = numel[t0 + i];
        }
        if (b.map.chunks == 0) continue;
        const int blocks = b.map.chunks < kMaxBlocks ? b.map.chunks : kMaxBlocks;
        if (factor)
            adam_kernel<true><<<blocks, 256, 0, st>>>(b, s, factor);
        else
            adam_kernel<false><<<blocks, 256, 0, st>>>(b, s, nullptr);
    }
    return ddpm::check_launch("adam_kernel");
}

}  // namespace

extern "C" int ddpm_adam_step(int ntensors, float* const* params, const float* const* grads, float* const* exp_avg,
                              float* const* exp_avg_sq, const int64_t* numel, double lr, double beta1, double beta2, double eps,
                              double weight_decay, int64_t step, void* stream) {
    return adam_step(ntensors, params, grads, exp_avg, exp_avg_sq, numel, lr, beta1, beta2, eps, weight_decay, step, nullptr, stream);
}

extern "C" int ddpm_adam_step_clipped(int ntensors, float* const* params, const float* const* grads, float* const* exp_avg,
                                      float* const* exp_avg_sq, const int64_t* numel, double lr, double beta1, double beta2,
                                      double eps, double weight_decay, int64_t step, const float* factor, void* stream) {
    DDPM_REQUIRE(factor);
    return adam_step(ntensors, params, grads, exp_avg, exp_avg_sq, numel, lr, beta1, beta2, eps, weight_decay, step, factor, stream);
}
