// A list of tensors as the work of one launch: the list travels in the kernel arguments (nothing is allocated or copied),
// every tensor is cut into chunks of a fixed number of elements, and a workgroup takes chunks first, first + gridDim.x, ...
// of the whole list. A launch over many small tensors and a few large ones is then as even as one over a single buffer.
#pragma once
#include "common.h"

namespace ddpm {

// first[t] = number of chunks before tensor t; first[count] = chunks in all. Tensors without elements own no chunk.
template <int N>
struct ChunkMap {
    int32_t count;
    int32_t first[N + 1];
};

// the tensor that owns `chunk` (uniform over the workgroup)
template <int N>
__device__ __forceinline__ int tensor_of_chunk(const ChunkMap<N>& m, int chunk) {
    int lo = 0, hi = m.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (m.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Longest tensor of a list, in elements.
constexpr int64_t kLongestTensor = int64_t(1) << 36;

// Does the number of chunks of every launch over `per_launch` tensors stay within 32 bits, a grid's step past the last one included? For
// checked lengths.
inline bool chunks_fit(int ntensors, const int64_t* numel, int per_launch, int64_t chunk) {
    int64_t chunks = 0;
    for (int i = 0; i < ntensors; ++i) {
        if (i % per_launch == 0) chunks = 0;
        chunks += (numel[i] + chunk - 1) / chunk;
        if (chunks > INT32_MAX - 65536) return false;
    }
    return true;
}

}  // namespace ddpm
