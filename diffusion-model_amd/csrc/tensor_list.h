// A list of tensors as the work of one launch: the list travels in the kernel arguments (nothing is allocated or copied),
// every tensor is cut into chunks of a fixed number of elements, and a workgroup takes chunks first, first + gridDim.x, ...
// of the whole list. A launch over many small tensors and a few large ones is then as even as one over a single buffer.
#pragma once
#include "common.h"

namespace ddpm {

// first[t] = number of chunks before tensor t, INT32_MAX behind the last tensor. Tensors without elements own no chunk.
template <int N>
struct ChunkMap {
    int32_t chunks;                      // in all
    int32_t first[N];
};

// the map of tensors of these lengths, `count` of them
template <int N>
void map_chunks(ChunkMap<N>& m, const int64_t* numel, int count, int64_t chunk) {
    m.chunks = 0;
    for (int i = 0; i < N; ++i) {
        m.first[i] = i < count ? m.chunks : INT32_MAX;
        if (i < count) m.chunks += static_cast<int32_t>((numel[i] + chunk - 1) / chunk);
    }
}

// The tensor that owns `chunk` (uniform over the workgroup): the last one that begins at it or before. A wave looks at all of them at once; a
// search by halves waits for up to eight scalar loads, one behind the other.
template <int N>
__device__ __forceinline__ int tensor_of_chunk(const ChunkMap<N>& m, int chunk) {
    int before = 0;
#pragma unroll
    for (int i = 0; i < N; i += 64) {
        const int t = i + static_cast<int>(threadIdx.x & 63);
        before += __popcll(__ballot(t < N && m.first[t] <= chunk));
    }
    return before - 1;
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
