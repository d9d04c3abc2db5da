// Norm of all gradients together and clipping by it: what a training loop puts between loss.backward() and
// optimizer.step() (first-iteration/main.py:83-84) when single batches can throw the weights far off.
//   norm = sqrt(sum over all tensors of g^2)  (or max |g|),  c = min(1, max_norm / (norm + 1e-6)),  g <- c g
// Bound by HBM: the norm reads every gradient once, clipping reads and writes it once more; the Adam step that takes c
// (adam.hip) needs no clipping pass at all. Squares are summed in float64 (exact products of fp32 numbers, no overflow at
// 1e19, and at two elements per clock and compute unit far below the float64 rate), per thread, per workgroup and over
// the workgroups in a fixed order: the same gradients give the same bits.
#include <cmath>
#include <type_traits>

#include "tensor_list.h"

using ddpm::as_stream;

namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 176;             // 20 bytes of kernel arguments each, below 4 KiB together
constexpr int64_t kChunk = 8192;          // elements: 8 (fp32) or 4 (16-bit) loads of 16 bytes per thread in flight
constexpr int kMaxBlocks = 2048;          // 8 workgroups per compute unit; also the partial results a launch leaves

// Lengths and types share a word. With the types as bytes, the compiler took the address of a byte, kernel arguments + t, as the base of the
// scalar load of p[t] as well, and 7 t as its offset: scalar loads drop the low two bits of each.
struct List {
    ddpm::ChunkMap<kTensors> map;
    void* p[kTensors];
    int64_t length_type[kTensors];        // 4 n + type
};

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Wide;
template <>
struct Wide<float> {
    typedef f32x4 type;
};
template <>
struct Wide<__bf16> {
    typedef bf16x8 type;
};
template <>
struct Wide<_Float16> {
    typedef f16x8 type;
};

// max that keeps a NaN once it has met one, as torch's maximum does
__device__ __forceinline__ double keep_max(double m, double a) { return (a > m || a != a) ? a : m; }

template <bool MAXIMUM>
__device__ __forceinline__ double join(double a, double b) {
    return MAXIMUM ? keep_max(a, b) : a + b;
}

template <bool MAXIMUM>
__device__ __forceinline__ double take(double acc, float g) {
    const double d = g;
    return MAXIMUM ? keep_max(acc, fabs(d)) : fma(d, d, acc);
}

// The elements of a chunk [p, p + n) on their way through a thread's registers: all of its loads are in flight before the first is
// used, behind a tensor's end too. A last chunk of 8191 elements taken one by one took longer than the rest of a launch:
// 26.5 us for the norm of 133 tensors of 62 MB and 26.2 us for their clipping, 17.5 and 21.9 us so. 133 ragged tensors of 59 MB take 13.7 and
// 18.9 us with their bases on 16-byte boundaries, 13.8 and 19.2 with none of them.
template <typename T>
struct Chunk {
    typedef typename Wide<T>::type V;
    static constexpr int W = 16 / sizeof(T), kLoads = static_cast<int>(kChunk) / (kThreads * W), kSingle = 8;

    // f(element) -> new value; stored where STORE. Noughts stand for elements behind the end.
    template <bool STORE, typename F>
    static __device__ __forceinline__ void each(T* __restrict__ p, int n, F f) {
        int done = 0;
        if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
            const int vectors = n / W;
            V v[kLoads];
            V* q = reinterpret_cast<V*>(p);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = i * kThreads + threadIdx.x;
                v[i] = V{};
                if (at < vectors) v[i] = q[at];
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int at = i * kThreads + threadIdx.x;
#pragma unroll
                for (int e = 0; e < W; ++e) v[i][e] = f(v[i][e]);
                if (STORE && at < vectors) q[at] = v[i];
            }
            done = vectors * W;
        }
        for (int first = done + threadIdx.x; first < n; first += kSingle * kThreads) {
            T x[kSingle];
#pragma unroll
            for (int i = 0; i < kSingle; ++i) {
                const int at = first + i * kThreads;
                x[i] = at < n ? p[at] : static_cast<T>(0.f);
            }
#pragma unroll
            for (int i = 0; i < kSingle; ++i) {
                const int at = first + i * kThreads;
                x[i] = f(x[i]);
                if (STORE && at < n) p[at] = x[i];
            }
        }
    }
};

// f<T>(first element, elements) of every chunk of this workgroup
template <typename F>
__device__ __forceinline__ void each_chunk(const List& l, F f) {
    for (int c = blockIdx.x; c < l.map.chunks; c += gridDim.x) {
        const int t = ddpm::tensor_of_chunk(l.map, c);
        const int64_t begin = static_cast<int64_t>(c - l.map.first[t]) * kChunk;
        const int64_t left = (l.length_type[t] >> 2) - begin;
        const int n = static_cast<int>(kChunk < left ? kChunk : left), type = static_cast<int>(l.length_type[t] & 3);
        if (type == DDPM_F32)
            f(static_cast<float*>(l.p[t]) + begin, n);
        else if (type == DDPM_BF16)
            f(static_cast<__bf16*>(l.p[t]) + begin, n);
        else
            f(static_cast<_Float16*>(l.p[t]) + begin, n);
    }
}

// v of every thread of the workgroup, joined in a fixed order; valid in thread 0
template <int THREADS, bool MAXIMUM>
__device__ __forceinline__ double join_block(double v) {
    __shared__ double sh[THREADS / 64];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = join<MAXIMUM>(v, __shfl_down(v, d));
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < THREADS / 64; ++w) v = join<MAXIMUM>(v, sh[w]);
    return v;
}

template <bool MAXIMUM>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(const List l, double* __restrict__ partial) {
    double acc = 0.0;
    each_chunk(l, [&](auto* p, int n) __attribute__((always_inline)) {
        using T = std::remove_reference_t<decltype(*p)>;
        Chunk<T>::template each<false>(p, n, [&](T g) __attribute__((always_inline)) {
            acc = take<MAXIMUM>(acc, static_cast<float>(g));
            return g;
        });
    });
    acc = join_block<kThreads, MAXIMUM>(acc);
    if (threadIdx.x == 0) partial[blockIdx.x] = acc;
}

// state[0] = norm, state[1] = factor that brings it to max_norm. A norm that is not a number makes the factor one too.
template <bool MAXIMUM>
__global__ __launch_bounds__(1024) void grad_norm_finish_kernel(const double* __restrict__ partial, int n, float max_norm,
                                                                float* __restrict__ state) {
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += 1024) acc = join<MAXIMUM>(acc, partial[i]);
    acc = join_block<1024, MAXIMUM>(acc);
    if (threadIdx.x == 0) {
        const float norm = static_cast<float>(MAXIMUM ? acc : sqrt(acc));
        const float c = max_norm / (norm + 1e-6f);
        state[0] = norm;
        state[1] = c > 1.f ? 1.f : c;
    }
}

__global__ __launch_bounds__(kThreads) void grad_clip_kernel(const List l, const float* __restrict__ factor) {
    const float f = factor[0];
    if (f == 1.f) return;      // inside the bound: every product would be the gradient itself
    each_chunk(l, [&](auto* p, int n) __attribute__((always_inline)) {
        using T = std::remove_reference_t<decltype(*p)>;
        Chunk<T>::template each<true>(p, n, [&](T g) __attribute__((always_inline)) { return static_cast<T>(static_cast<float>(g) * f); });
    });
}

bool known_type(int t) { return t == DDPM_F32 || t == DDPM_BF16 || t == DDPM_F16; }

// no launch's chunks pass 32 bits
static_assert(kTensors * (ddpm::kLongestTensor / kChunk) + kMaxBlocks <= INT32_MAX, "chunks of a launch");

int check_list(int ntensors, const void* const* grads, const int64_t* numel, const int32_t* types) {
    for (int i = 0; i < ntensors; ++i) {
        DDPM_REQUIRE(known_type(types[i]));
        DDPM_REQUIRE(numel[i] >= 0 && numel[i] <= ddpm::kLongestTensor && (numel[i] == 0 || grads[i]));
        DDPM_REQUIRE((reinterpret_cast<uintptr_t>(grads[i]) & (types[i] == DDPM_F32 ? 3 : 1)) == 0);
    }
    return DDPM_OK;
}

// tensors t0, t0 + 1, ... of the list, as many as one launch takes
void fill(List& l, int t0, int ntensors, const void* const* grads, const int64_t* numel, const int32_t* types) {
    const int cnt = ntensors - t0 < kTensors ? ntensors - t0 : kTensors;
    ddpm::map_chunks(l.map, numel + t0, cnt, kChunk);
    for (int i = 0; i < cnt; ++i) {
        l.p[i] = const_cast<void*>(grads[t0 + i]);
        l.length_type[i] = 4 * numel[t0 + i] + types[t0 + i];
    }
}

int blocks_of(const List& l) { return l.map.chunks < kMaxBlocks ? l.map.chunks : kMaxBlocks; }

}  // namespace

extern "C" int64_t ddpm_grad_norm_workspace_doubles(int ntensors) {
    return ntensors <= 0 ? 1 : static_cast<int64_t>((ntensors + kTensors - 1) / kTensors) * kMaxBlocks;
}

extern "C" int ddpm_grad_norm(int ntensors, const void* const* grads, const int64_t* numel, const int32_t* types, int kind,
                              float max_norm, double* workspace, float* state, void* stream) {
    DDPM_REQUIRE(ntensors >= 0 && state && workspace && (kind == DDPM_NORM_2 || kind == DDPM_NORM_MAX));
    DDPM_REQUIRE(max_norm >= 0.f);
    DDPM_REQUIRE(ntensors == 0 || (grads && numel && types));
    if (int rc = check_list(ntensors, grads, numel, types)) return rc;
    int partials = 0;
    for (int t0 = 0; t0 < ntensors; t0 += kTensors) {
        List l;
        fill(l, t0, ntensors, grads, numel, types);
        const int blocks = blocks_of(l);
        if (blocks == 0) continue;
        if (kind == DDPM_NORM_2)
            grad_norm_kernel<false><<<blocks, kThreads, 0, as_stream(stream)>>>(l, workspace + partials);
        else
            grad_norm_kernel<true><<<blocks, kThreads, 0, as_stream(stream)>>>(l, workspace + partials);
        partials += blocks;
    }
    if (kind == DDPM_NORM_2)
        grad_norm_finish_kernel<false><<<1, 1024, 0, as_stream(stream)>>>(workspace, partials, max_norm, state);
    else
        grad_norm_finish_kernel<true><<<1, 1024, 0, as_stream(stream)>>>(workspace, partials, max_norm, state);
    return ddpm::check_launch("grad_norm_kernel");
}

extern "C" int ddpm_clip_grads(int ntensors, void* const* grads, const int64_t* numel, const int32_t* types, const float* factor,
                               void* stream) {
    DDPM_REQUIRE(ntensors >= 0 && factor);
    DDPM_REQUIRE(ntensors == 0 || (grads && numel && types));
    if (int rc = check_list(ntensors, grads, numel, types)) return rc;
    for (int t0 = 0; t0 < ntensors; t0 += kTensors) {
        List l;
        fill(l, t0, ntensors, grads, numel, types);
        if (const int blocks = blocks_of(l); blocks > 0)
            grad_clip_kernel<<<blocks, kThreads, 0, as_stream(stream)>>>(l, factor);
    }
    return ddpm::check_launch("grad_clip_kernel");
}
