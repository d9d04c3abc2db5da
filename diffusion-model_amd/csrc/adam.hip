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
    const int chunks = b.map.first[b.map.count];
    for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
        const int t = ddpm::tensor_of_chunk(b.map, c);
        const int64_t begin = static_cast<int64_t>(c - b.map.first[t]) * kChunk;
        const int64_t end = begin + kChunk < b.n[t] ? begin + kChunk : b.n[t];
        float* __restrict__ p = b.p[t];
        const float* __restrict__ g = b.g[t];
        float* __restrict__ m = b.m[t];
        float* __restrict__ v = b.v[t];
        const bool vec = ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(m) |
                           reinterpret_cast<uintptr_t>(v)) & 15) == 0;
        if (vec && end - begin == kChunk) {
            constexpr int kLoads = static_cast<int>(kChunk) / 1024;
            f32x4 pv[kLoads], gv[kLoads], mv[kLoads], vv[kLoads];
            const int64_t at = (begin >> 2) + threadIdx.x;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                pv[i] = reinterpret_cast<const f32x4*>(p)[at + i * 256];
                gv[i] = reinterpret_cast<const f32x4*>(g)[at + i * 256];
                mv[i] = reinterpret_cast<const f32x4*>(m)[at + i * 256];
                vv[i] = reinterpret_cast<const f32x4*>(v)[at + i * 256];
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float pe = pv[i][e], me = mv[i][e], ve = vv[i][e];
                    adam_elem(pe, CLIP ? gv[i][e] * f : gv[i][e], me, ve, s);
                    pv[i][e] = pe;
                    mv[i][e] = me;
                    vv[i][e] = ve;
                }
                reinterpret_cast<f32x4*>(p)[at + i * 256] = pv[i];
                reinterpret_cast<f32x4*>(m)[at + i * 256] = mv[i];
                reinterpret_cast<f32x4*>(v)[at + i * 256] = vv[i];
            }
        } else {
            for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
                float pe = p[i], me = m[i], ve = v[i];
                adam_elem(pe, CLIP ? g[i] * f : g[i], me, ve, s);
                p[i] = pe;
                m[i] = me;
                v[i] = ve;
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
        int32_t chunks = 0;
        b.map.count = cnt;
        b.map.first[0] = 0;
        for (int i = 0; i < cnt; ++i) {
            b.p[i] = params[t0 + i];
            b.g[i] = grads[t0 + i];
            b.m[i] = exp_avg[t0 + i];
            b.v[i] = exp_avg_sq[t0 + i];
            b.n[i] = numel[t0 + i];
            chunks += static_cast<int32_t>((numel[t0 + i] + kChunk - 1) / kChunk);
            b.map.first[i + 1] = chunks;
        }
        if (chunks == 0) continue;
        const int blocks = chunks < kMaxBlocks ? chunks : kMaxBlocks;
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
