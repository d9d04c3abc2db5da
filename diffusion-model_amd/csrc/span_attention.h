// Parts shared by the forward and backward kernels of span attention: how rows of a tensor meet the matrix instructions,
// how tiles reach LDS, what a row sees, and how a score comes from a product.
//
// Everything is built from two products of a 32-row tile in LDS:
//   dot:    X[row][col] = sum over channels of tile[row] and the lane's own row (held in registers),
//   spread: Y[channel][col] += sum over tile rows of tile[row][channel] * weight[row][col],
// with one column per lane (col = lane % 32). In the layout of the 32x32 results a lane holds 16 rows of its column,
// register r of lane half h being row 8 (r / 4) + 4 h + r % 4, so the weights made from a dot's result are already where spread
// wants its second operand: the sum over rows may run in any order, and the first operand is read from LDS in the order the
// registers have. No score ever moves between lanes; a column's maximum and sum need one exchange between the lane halves.
//   forward:  scores = dot(K, q), out += spread(V, p)                    columns are queries
//   dq:       scores = dot(K, q), dp = dot(V, dout), dq += spread(K, ds)  columns are queries
//   dk, dv:   scores = dot(Q, k), dp = dot(dOut, v), dv += spread(dOut, p), dk += spread(Q, ds)   columns are keys
#pragma once
#include "common.h"

namespace span {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;            // 4 waves
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Running maximum before the first key: finite, so that its difference from -infinity (a masked score) is one, and below any finite score but
// fp32's lowest ones, so that a row's first score takes its place.
constexpr float kNoMax = -3e38f;
constexpr int kMaxTile = 64;             // rows of a tile, at most

struct Strides {
    int64_t batch, row, head;
};

struct Dev {
    int nq, nk, heads, group, dim;       // group: query heads per key/value head
    int causal;
    float scale, softcap;
    const float* slopes;
    const int32_t* spans;
    const int32_t* positions;
    int64_t span_batch, position_batch;
    const void *q, *k, *v;
    void *out, *out_low;
    float *lse, *lse_near;
    Strides sq, sk, sv, so;
    const void* dout;
    void *dq, *dk, *dv;
    Strides sdo, sdq, sdk, sdv;
};

// ---- what a row sees -----------------------------------------------------------------------------------------------
// The bias counts from the nearest key that the row sees: -slope |pos - j| with pos moved there differs from the one with the row's position by
// the same number for all of them, which the softmax does not notice. Far from all its keys (a million positions at a slope of 0.5) the
// full bias would take the scores' last bits: one step of fp32 is 0.06 there.
struct Row {
    int lo, hi, pos;                     // keys [lo, hi); lo = INT_MAX, hi = 0: none; position, moved to the nearest key
};

__device__ __forceinline__ int position_of(const Dev& a, int b, int i) {
    return a.positions ? a.positions[b * a.position_batch + i] : i + a.nk - a.nq;
}

__device__ __forceinline__ Row row_of(const Dev& a, int b, int i) {
    Row r;
    r.pos = position_of(a, b, i);
    r.lo = 0;
    r.hi = a.nk;
    if (a.spans) {
        const int32_t* s = a.spans + b * a.span_batch + 2 * static_cast<int64_t>(i);
        r.lo = max(s[0], 0);
        r.hi = min(s[1], a.nk);
    }
    if (a.causal && r.pos < r.hi) r.hi = r.pos + 1;
    if (r.hi <= r.lo) {
        r.lo = INT32_MAX;
        r.hi = 0;
    } else {
        r.pos = min(max(r.pos, r.lo), r.hi - 1);
    }
    return r;
}

// what the move left out of the bias of all keys: lse = lse_near - it
__device__ __forceinline__ float left_out(const Dev& a, int b, int i, const Row& row, int head) {
    if (!a.slopes || row.hi == 0) return 0.f;
    const int at = position_of(a, b, i);
    const unsigned way = at < row.pos ? static_cast<unsigned>(row.pos) - static_cast<unsigned>(at) : static_cast<unsigned>(at) - static_cast<unsigned>(row.pos);
    return a.slopes[head] * static_cast<float>(way);
}

__device__ __forceinline__ Row no_row() { return {INT32_MAX, 0, 0}; }

// smallest lo and largest hi of the wave
__device__ __forceinline__ void join_rows(int& lo, int& hi) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        lo = min(lo, __shfl_xor(lo, d));
        hi = max(hi, __shfl_xor(hi, d));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
}

// the other lane half's value of this column
__device__ __forceinline__ float other_half(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
    return __builtin_bit_cast(float, (threadIdx.x & 32) ? r[0] : r[1]);
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- tiles in LDS ------------------------------------------------------------------------------------------------------
// Rows of DP channels without gaps (loads from memory to LDS write 1 KiB of neighbouring lanes), their 16-byte chunks exchanged
// by row: chunk c of a row lies at c ^ swizzle(row). In units of 64 bytes the four rows of a transposing read then fall into the
// four different quarters of the 256 bytes of banks, and 16 rows read at one chunk (dot) into 16 different chunks of them.
// With 8 channels of padding instead, both kinds of reads met conflicts.
template <typename T, int DP>
__device__ __forceinline__ constexpr int swizzle(int row) {
    constexpr int chunks = DP * static_cast<int>(sizeof(T)) / 16;
    if (sizeof(T) == 4) return row & 7;
    return ((row >> 2) & 3) | (chunks == 16 ? (row & 3) << 2 : chunks == 8 ? ((row >> 1) & 1) << 2 : 0);
}

// Byte offset in a tile whose chunk is `delta` bytes (a constant) from that of `at`: an exclusive or as far as the exchange
// reaches, which is the largest power of two in the row's length at most, and a sum above.
template <typename T, int DP>
__device__ __forceinline__ int chunk_from(int at, int delta) {
    constexpr int bytes = DP * static_cast<int>(sizeof(T)), power = bytes & -bytes;
    return (at ^ (delta & (power - 1))) + (delta & ~(power - 1));
}

// The offsets of a product differ by constants from one, but an exclusive or is no offset that an instruction has room for: left
// alone (FRESH false), the compiler computes all of them ahead of the loop and keeps them in registers, 16 and more. Where those are
// wanted for something else they are computed as they are used.
template <bool FRESH>
__device__ __forceinline__ int offset(int at) {
    if (FRESH) asm volatile("" : "+v"(at));
    return at;
}

template <typename V, typename T>
__device__ __forceinline__ V read_at(const T* tile, int at) {
    return *reinterpret_cast<const V*>(reinterpret_cast<const char*>(tile) + at);
}

// ---- matrix products of a type ---------------------------------------------------------------------------------------
template <typename T>
struct Ops {                             // bf16, fp16
    typedef T Frag __attribute__((ext_vector_type(8)));
    static constexpr int W = 8;          // elements of 16 bytes
    static constexpr int kStep = 16;     // channels of one step of dot
    static constexpr int kTile = kMaxTile;   // rows in LDS at a time
    // How far scores may pass the maximum that weights are relative to before sums are rescaled, in powers of two. Any number
    // serves fp32's and bf16's exponents; fp16 has room for one beside kShift. With 0 some row of a wave has a new maximum in most tiles.
    static constexpr float kSlack = __is_same(T, _Float16) ? 1.f : 8.f;
    // Weights are scaled by 2^kShift before they are rounded to T: fp16 has no more than 2^-24 at its small end, and a row of
    // thousands of keys has many weights below its normal numbers; bf16 has fp32's range.
    static constexpr int kShift = __is_same(T, _Float16) ? 14 : 0;
    struct Weights {
        Frag f[2];
    };

    static __device__ __forceinline__ f32x16 mfma(Frag a, Frag b, f32x16 c) {
        if constexpr (__is_same(T, _Float16))
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
        else
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Weights pack(const f32x16& p) {
        Weights w;
#pragma unroll
        for (int r = 0; r < 16; ++r) w.f[r >> 3][r & 7] = static_cast<T>(p[r]);
        return w;
    }
    // what pack() left of p
    static __device__ __forceinline__ Weights rest(const f32x16& p, const Weights& w) {
        Weights low;
#pragma unroll
        for (int r = 0; r < 16; ++r) low.f[r >> 3][r & 7] = static_cast<T>(p[r] - static_cast<float>(w.f[r >> 3][r & 7]));
        return low;
    }
    // acc[db] += over 32 tile rows; `tile` points at the first of them. With `low` the weights are w + low.
    template <int DP, bool FRESH = false>
    static __device__ __forceinline__ void spread(f32x16* acc, const T* tile, const Weights& w, const Weights* low = nullptr) {
        // The transposing read gives lane l of 16 the column l of a 4 x 16 block whose rows four lanes each point at: rows
        // 4 h ... 4 h + 3 (and 8 further) are the ones whose weights this lane half holds.
        const int lane = threadIdx.x & 63, l16 = lane & 15, row = 4 * (lane >> 5) + (l16 >> 2);
        const int chunk = 2 * ((lane >> 4) & 1) + ((l16 >> 1) & 1);
        const int at = offset<FRESH>(2 * row * DP + 16 * (chunk ^ swizzle<T, DP>(row)) + 8 * (l16 & 1));
        const auto four = [&](int rows, int db) __attribute__((always_inline)) {       // rows: a multiple of 8; 8 exchanges by 2
            const char* x = reinterpret_cast<const char*>(tile) + chunk_from<T, DP>(at, (64 * db) ^ (rows & 8 ? 32 : 0)) + 2 * rows * DP;
            return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)x);
        };
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) {
                const auto xy = __builtin_shufflevector(four(16 * t, db), four(16 * t + 8, db), 0, 1, 2, 3, 4, 5, 6, 7);
                acc[db] = mfma(__builtin_bit_cast(Frag, xy), w.f[t], acc[db]);
                if (low) acc[db] = mfma(__builtin_bit_cast(Frag, xy), low->f[t], acc[db]);
            }
    }
    static __device__ __forceinline__ f32x16 mul(Frag a, Frag b, f32x16 c) { return mfma(a, b, c); }
};

template <>
struct Ops<float> {
    typedef f32x4 Frag;
    static constexpr int W = 4;
    static constexpr int kStep = 8;
    static constexpr int kTile = 32;
    static constexpr int kShift = 0;
    static constexpr float kSlack = 8.f;
    typedef f32x16 Weights;

    static __device__ __forceinline__ f32x16 mul(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Weights pack(const f32x16& p) { return p; }
    template <int DP, bool FRESH = false>
    static __device__ __forceinline__ void spread(f32x16* acc, const float* tile, const Weights& w) {
        const int lane = threadIdx.x & 63, half = lane >> 5;
        const int at = offset<FRESH>(16 * half * DP + 16 * (((lane >> 2) & 7) ^ (4 * half)) + 4 * (lane & 3));
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int x = (at ^ (16 * (r & 3))) + 4 * (8 * (r >> 2) + (r & 3)) * DP;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(read_at<float>(tile, x + 128 * db), w[r], acc[db], 0, 0, 0);
        }
    }
};

// the lane's own row: channels kStep s + W h ... of step s, nought behind dim
template <typename T, int DP>
struct OwnRow {
    static constexpr int kSteps = DP / Ops<T>::kStep;
    typename Ops<T>::Frag f[kSteps];

    __device__ __forceinline__ void load(const T* row, int dim) {       // row == nullptr: noughts
        const int c0 = Ops<T>::W * ((threadIdx.x >> 5) & 1);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = c0 + Ops<T>::kStep * s;
            f[s] = typename Ops<T>::Frag{};
            if (row && c < dim) f[s] = *reinterpret_cast<const typename Ops<T>::Frag*>(row + c);
        }
    }
    __device__ __forceinline__ void negate() {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) f[s] = -f[s];
    }
    // product with 32 tile rows; like it with the own rows, 32 of a wave, in LDS too
    template <bool FRESH = false>
    __device__ __forceinline__ f32x16 dot(const T* tile) const {
        const int lane = threadIdx.x & 63, row = lane & 31;
        const int at = offset<FRESH>(static_cast<int>(sizeof(T)) * row * DP + 16 * (swizzle<T, DP>(row) ^ (lane >> 5)));
        f32x16 acc = {};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) acc = Ops<T>::mul(read_at<typename Ops<T>::Frag>(tile, chunk_from<T, DP>(at, 32 * s)), f[s], acc);
        return acc;
    }
};

template <typename T, int DP, bool FRESH = false>
__device__ __forceinline__ f32x16 dot_from_lds(const T* tile, const T* own) {
    const int lane = threadIdx.x & 63, row = lane & 31;
    const int at = offset<FRESH>(static_cast<int>(sizeof(T)) * row * DP + 16 * (swizzle<T, DP>(row) ^ (lane >> 5)));
    f32x16 acc = {};
#pragma unroll
    for (int s = 0; s < DP / Ops<T>::kStep; ++s) {
        acc = Ops<T>::mul(read_at<typename Ops<T>::Frag>(tile, chunk_from<T, DP>(at, 32 * s)),
                          read_at<typename Ops<T>::Frag>(own, chunk_from<T, DP>(at, 32 * s)), acc);
    }
    return acc;
}

// Rows of a tensor on their way to tiles in LDS. A tile's loads have one 64-bit address, which the wave keeps in scalar registers, and
// 32-bit unsigned offsets of the lanes, which do not change from tile to tile (the host sees to it that kMaxTile rows span less than
// 2 GiB; no tile has more than twice as many).
// Rows outside [lo, hi) read the nearest row inside: they are masked, and what memory holds behind a sequence is not looked
// at. Chunks behind dim read the row's first one: their products with the noughts of an OwnRow are nought, and channels there
// are not written. The loads have arrived behind the next arrived().
template <typename T, int DP, int ROWS = Ops<T>::kTile>
struct Fetch {
    static constexpr int W = Ops<T>::W, kChunks = DP / W, kRows = ROWS, kPieces = kRows * kChunks / 64, kWaves = kThreads / 64;
    static constexpr int kLoads = (kPieces + kWaves - 1) / kWaves;      // pieces of 1 KiB, in turn for the waves
    static_assert(kRows * kChunks % 64 == 0, "whole pieces");
    const char* base;
    int64_t row_bytes;
    int lo, hi;
    unsigned offset[kLoads];

    static __device__ __forceinline__ int piece(int i) { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) + i * kWaves; }
    static __device__ __forceinline__ int row_in_tile(int i) { return (piece(i) * 64 + static_cast<int>(threadIdx.x & 63)) / kChunks; }
    static __device__ __forceinline__ unsigned column(int i, int dim) {
        const int row = row_in_tile(i), c = W * ((piece(i) * 64 + static_cast<int>(threadIdx.x & 63) - row * kChunks) ^ swizzle<T, DP>(row));
        return (c < dim ? c : 0) * sizeof(T);
    }
    __device__ __forceinline__ void start(const T* tensor, int64_t row_stride, int lo_, int hi_, int dim) {
        base = reinterpret_cast<const char*>(tensor);
        row_bytes = row_stride * static_cast<int64_t>(sizeof(T));
        lo = lo_;
        hi = hi_;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) offset[i] = static_cast<unsigned>(row_in_tile(i)) * static_cast<unsigned>(row_bytes) + column(i, dim);
    }
    __device__ __forceinline__ void load(T* tile, int row0, int dim) const {
        const char* at = base + row0 * row_bytes;
        const bool inside = row0 >= lo && row0 + kRows <= hi;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            if (kPieces % kWaves && piece(i) >= kPieces) break;
            unsigned o = offset[i];
            if (!inside) o = static_cast<unsigned>(max(min(row_in_tile(i), hi - 1 - row0), lo - row0)) * static_cast<unsigned>(row_bytes) + column(i, dim);
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(at + o),
                                             (__attribute__((address_space(3))) unsigned*)(tile + piece(i) * 64 * W), 16, 0, 0);
        }
    }
};

// 64 lanes' words of 4 bytes from memory to LDS, like a Fetch.
__device__ __forceinline__ void fetch_words(void* to, const void* from) {
    const unsigned lane = 4 * (threadIdx.x & 63);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) unsigned*)(static_cast<const char*>(from) + lane),
                                     (__attribute__((address_space(3))) unsigned*)to, 4, 0, 0);
}

// Barrier behind which every wave's fetches are in LDS. __syncthreads() alone does not wait for them: they count as loads from
// memory, which a workgroup's fence leaves in flight.
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Waits until matrix instructions have written x. The compiler inserts these waits itself, but its search for the instruction that
// wrote a register, going back over a join of branches, may follow the long way round to it alone and find that enough time has
// passed: a read behind `products; branch around something; join` has met the registers of before. Between products and the
// next branch the wait is therefore written out: 18 states behind the fp32 instruction, 12 behind the 16-bit ones.
template <typename T>
__device__ __forceinline__ void settle(f32x16& x) {
    if constexpr (sizeof(T) == 4)
        asm volatile("s_nop 15\n\ts_nop 1" : "+v"(x));
    else
        asm volatile("s_nop 11" : "+v"(x));
}
template <typename T>
__device__ __forceinline__ void settle(f32x16& x, f32x16& y) {
    if constexpr (sizeof(T) == 4)
        asm volatile("s_nop 15\n\ts_nop 1" : "+v"(x), "+v"(y));
    else
        asm volatile("s_nop 11" : "+v"(x), "+v"(y));
}

// ---- keys that no row sees ---------------------------------------------------------------------------------------------
// A masked key has weight nought, but nought times what its row of v (for dq, of k) holds is nought for finite numbers alone. Keys outside
// of all that a workgroup's rows see are not fetched; the ones in between that none of them sees, as behind each of several padded
// documents, are made noughts in LDS. Where the rows see neighbouring or overlapping spans, one after the other, there are none, which
// takes some comparisons of a lane; elsewhere a search, and in a tile with such keys a barrier: 8192 rows, 16 + 4 heads of 128, bf16, in
// documents of 340 padded to 352 take 64 us (forward) and 329 (with the gradient) for the 61 and 321 without, of 352 the same as without.
struct Gaps {
    static constexpr int kRows = kThreads / 2;
    int lo[kRows], hi[kRows];            // of the workgroup's rows
    int from[kRows], to[kRows];          // gaps

    // before a barrier: the rows of this wave, whose lane halves hold the same
    __device__ __forceinline__ void tell(const Row& row) {
        if ((threadIdx.x & 32) == 0) {
            const int x = (threadIdx.x >> 6) * 32 + (threadIdx.x & 31);
            lo[x] = row.lo;
            hi[x] = row.hi;
        }
    }
    // behind it, for all of the workgroup: how many gaps there are below key `top`. Every wave searches by itself.
    __device__ __forceinline__ int find(int top) {
        // A gap begins at the end of a span that is in no span, and ends where the next one begins. Most ends are in the next row's span, or are
        // its end too; those that are not are looked at one by one. A row that sees none has lo = INT_MAX, hi = 0.
        const int lane = threadIdx.x & 63;
        int l[2], h[2];
        unsigned long long ends[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int x = lane + 64 * i;
            l[i] = lo[x];
            h[i] = hi[x];
            ends[i] = __ballot(h[i] != 0 && h[i] < top && !(x + 1 < kRows && lo[x + 1] <= h[i] && hi[x + 1] >= h[i]));
        }
        int n = 0;
        while (ends[0] | ends[1]) {
            const int end = ends[0] ? __builtin_amdgcn_readlane(h[0], __builtin_ctzll(ends[0])) : __builtin_amdgcn_readlane(h[1], __builtin_ctzll(ends[1]));
            bool inside = false;
            int next = INT32_MAX;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                ends[i] &= ~__ballot(h[i] == end);
                inside |= l[i] <= end && h[i] > end;
                if (l[i] > end) next = min(next, l[i]);
            }
            if (__any(inside)) continue;
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) next = min(next, __shfl_xor(next, d));
            if (threadIdx.x == 0) {
                from[n] = end;
                to[n] = next;
            }
            ++n;
        }
        if (n > 0) __syncthreads();
        return n;
    }
    // nought into the rows of two tiles of keys j0 ... that are in a gap; `n` is the same for the workgroup
    template <typename T, int DP, int TILE>
    __device__ __forceinline__ void clear(int n, int j0, T* x, T* y) const {
        constexpr int kChunks = DP / Ops<T>::W;
        typedef typename Ops<T>::Frag Frag;
        bool any = false;
        for (int g = 0; g < n; ++g) {
            const int first = max(from[g] - j0, 0), last = min(to[g] - j0, TILE);
            if (first >= last) continue;
            any = true;
            for (int c = first * kChunks + static_cast<int>(threadIdx.x); c < last * kChunks; c += kThreads)
                reinterpret_cast<Frag*>(x)[c] = reinterpret_cast<Frag*>(y)[c] = Frag{};
        }
        if (any) __syncthreads();
    }
};

// ---- scores ------------------------------------------------------------------------------------------------------------
// From x = |scale| / scale q.k to log2(e) w. Where there is neither cap nor bias that is a product with a constant, which goes into the
// exponential's argument as exp2(x * mul - maximum), one operation for both; elsewhere log2(e) w is formed first, and mul is 1 there.
struct Score {
    float pre, cap, inv, mul;            // inv: 1 / (cap log2 e), turns the result back into the tanh
    bool capped, plain;
    float near16, near32;                // products below this, relative to the cap, go into the polynomials of apply

    __device__ __forceinline__ Score(const Dev& a) {
        capped = a.softcap > 0.f;
        plain = !capped && !a.slopes;
        cap = a.softcap * kLog2e;
        inv = capped ? 1.f / cap : 0.f;
        // at scale 0 a number that makes every score nought and still keeps -infinity (a masked key) what it is
        pre = fmaxf(fabsf(capped ? a.scale / a.softcap : a.scale * kLog2e), 1e-37f);
        mul = plain ? pre : 1.f;
        // their constants hold pre^6 and pre^10, which must not leave fp32's range: a scale of 1 / 128 and a cap of 50 do so for fp32
        near16 = pre >= 1e-5f && pre <= 10.f && cap * pre <= 1e20f ? 0.5f : 0.f;
        near32 = pre >= 1e-3f && near16 != 0.f ? 0.75f : 0.f;
    }
    // x into log2(e) u, where not plain
    template <typename T>
    __device__ __forceinline__ void apply(f32x16& s) const {
        if (plain) return;
        if (!capped) {
            s *= pre;
            return;
        }
        // cap tanh x = cap x (1 + x^2 (...)) where all of the wave's scores are small beside the cap, as most are: fitted for the smallest
        // largest relative error, 6.4e-7 below x = 0.5 (less than a thousandth of a 16-bit weight's rounding), 3.3e-8 below 0.75 for
        // fp32. With the constants multiplied out for s itself it costs 5 operations (fp32: 7) for the 11 (an exponential and a
        // reciprocal take four each) of 1 - 2 / (e^2x + 1).
        constexpr bool exact = __is_same(T, float);
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) most = fmaxf(most, fabsf(s[r]));
        if (__all(most * pre < (exact ? near32 : near16))) {
            const float c0 = cap * pre, y = pre * pre, c1 = (exact ? -3.333306838e-01f : -3.332815933e-01f) * c0 * y;
            const float c2 = (exact ? 1.332652116e-01f : 1.320535960e-01f) * c0 * y * y;
            const float c3 = (exact ? -5.339025798e-02f : -4.475064100e-02f) * c0 * y * y * y;
            const float c4 = 1.966491225e-02f * c0 * y * y * y * y, c5 = -4.769489293e-03f * c0 * y * y * y * y * y;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float z = s[r] * s[r];
                float p = exact ? fmaf(z, fmaf(z, c5, c4), c3) : c3;
                p = fmaf(z, fmaf(z, fmaf(z, p, c2), c1), c0);
                s[r] *= p;
            }
            return;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float x = s[r] * pre;
            if constexpr (exact) {
                s[r] = cap * tanhf(x);
            } else {
                const float e = exp2_(x * (2.f * kLog2e));
                s[r] = fmaf(-2.f * cap, __builtin_amdgcn_rcpf(e + 1.f), cap);
            }
        }
    }
    // d u / d t
    __device__ __forceinline__ float slope(float u) const {
        const float t = u * inv;
        return fmaf(-t, t, 1.f);
    }
};

// Four channels of a row of out, and what their rounding left, for D in the backward call: D from a rounded out would be off by as
// much as the rounding of all score gradients together. fp32 leaves nothing worth keeping.
template <typename T>
__device__ __forceinline__ void write_out(const Dev& a, int64_t at, const float (&o)[4]) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 high, low;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        high[e] = static_cast<T>(o[e]);
        low[e] = static_cast<T>(o[e] - static_cast<float>(high[e]));
    }
    *reinterpret_cast<T4*>(static_cast<T*>(a.out) + at) = high;
    if (sizeof(T) == 2 && a.out_low) *reinterpret_cast<T4*>(static_cast<T*>(a.out_low) + at) = low;
}

// The block of rows (or keys) x, of gridDim.x, and the pair of head and batch entry that a workgroup takes. Workgroups start in the order
// of their index and go to the 8 XCDs in turn. Where the pairs are a multiple of 8, pairs run fastest: an XCD, with its L2, keeps to
// an eighth of the pairs, and all of them start with their first blocks, which the caller makes the longest ones, so that short ones fill
// up the end. Otherwise neighbouring blocks of one pair go to one XCD.
struct Place {
    int x, head, batch;
};
__device__ __forceinline__ Place place_of() {
    const unsigned pairs = gridDim.y * gridDim.z;
    if (pairs % 8 == 0) {
        const unsigned id = blockIdx.x + gridDim.x * (blockIdx.y + gridDim.y * blockIdx.z), pair = id % pairs;
        return {static_cast<int>(id / pairs), static_cast<int>(pair % gridDim.y), static_cast<int>(pair / gridDim.y)};
    }
    const dim3 id = ddpm::xcd_block();
    return {static_cast<int>(id.x), static_cast<int>(id.y), static_cast<int>(id.z)};
}

// tile row of register r of this lane half
__device__ __forceinline__ int reg_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// span_attention_fwd.hip
bool check_args(const ddpm_span_attention_args& a);
bool fits_tile(const ddpm_span_attention_args& a, const int64_t* stride);      // rows of a tile within 32-bit offsets
Dev dev_args(const ddpm_span_attention_args& a);
// The grid holds 65535 entries of a batch; a longer one takes several launches, one behind the other, in the same workspace:
// entries [first, first + kMaxBatch) of a.
constexpr int kMaxBatch = 65535;
ddpm_span_attention_args entries_from(const ddpm_span_attention_args& a, int first);

// f(head size as a compile-time constant): dim rounded up to a multiple of 32
template <typename F>
void for_dim(int dim, F&& f) {
    if (dim <= 32)
        f(std::integral_constant<int, 32>{});
    else if (dim <= 64)
        f(std::integral_constant<int, 64>{});
    else if (dim <= 96)
        f(std::integral_constant<int, 96>{});
    else
        f(std::integral_constant<int, 128>{});
}

}  // namespace span
