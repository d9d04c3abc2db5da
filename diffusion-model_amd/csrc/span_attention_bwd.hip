// Span attention, gradient (the mathematics and the two products are in span_attention.h):
//   D_i = sum_c dout_ic out_ic,  p_ij = exp(w_ij - lse_i),  dp_ij = dout_i . v_j,  ds_ij = scale (du/dt)_ij p_ij (dp_ij - D_i)
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
// in two kernels, each of which recomputes the scores: dq walks over keys with rows in registers, dk and dv over rows with keys in
// registers. That is 7 products (for 16-bit types 8, as score gradients enter dq in two parts) for the 5 of a single kernel, whose dq
// would be added up with atomics in an order that changes from call to call, and in fp32 memory that must be cleared before and
// converted behind. The gradient of a key/value head is summed over the query heads that share it inside its workgroup.
#include <algorithm>

#include "span_attention.h"

using ddpm::as_stream;

namespace {

using namespace span;

constexpr int kRows = 128;               // rows (dq) or keys (dk, dv) of a workgroup, 32 a wave

// What 32 rows see together: keys [lo, hi) are seen by some of them, [all_lo, all_hi) by all (all_lo = INT_MAX when one sees none).
struct Seen {
    int lo, hi, all_lo, all_hi;
};

// What the dq kernel leaves for the other one, in groups of 32 rows.
struct Work {
    Seen* seen;                          // [batch][groups]
    int* spans;                          // [batch][groups][lo of 32 rows | hi]
    int* positions;                      // [batch][groups][32, and 32 unused]
    float* stats;                        // [batch][heads][groups][-lse in units of log 2 plus kShift | D]
    float* largest;                      // fp16: largest |ds| of a group: [batch][heads][q_parts][groups]
    float* q_sums;                       // split dq kernel: [q_parts][batch][nq][heads][dim]
    float* sums;                         // split dk/dv kernel: [dk | dv][parts][batch][nk][kv_heads][dim]
    int groups, q_parts, parts;
};

// fp16 has five bits of exponent, and score gradients are as small as a loss makes them: they are scaled by a power of two
// that brings the largest to 2^13 ... 2^14 before they are rounded, and the sums are scaled back. Limits keep both factors finite.
__device__ __forceinline__ float gain_for(float largest) {
    int e = static_cast<int>((__builtin_bit_cast(unsigned, largest) >> 23) & 255) - 127;
    e = max(-100, min(100, 13 - e));
    return __builtin_bit_cast(float, static_cast<unsigned>(127 + e) << 23);
}
__device__ __forceinline__ float inverse_gain(float gain) {
    return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(unsigned, gain));
}

// lse in units of log 2, such that exp2(score - it) is nought for a row whose weights are all nought
__device__ __forceinline__ float stat_of(float lse) { return lse == -INFINITY ? -kNoMax : lse * kLog2e; }

template <typename T, int DP>
__device__ __forceinline__ void write_row(T* out, const f32x16* acc, float f, int dim) {      // acc has settled
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int half = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * db + 8 * g + 4 * half;
            T4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(acc[db][4 * g + e] * f);
            if (d < dim) *reinterpret_cast<T4*>(out + d) = o;
        }
}

// dq. A workgroup of 4 waves takes 128 rows of one head, 32 a wave, and walks over the keys that any of them sees; where there are few
// rows and many keys several workgroups take a tile in turn each (SPLIT), and a last kernel adds up their sums. It also leaves what the
// other kernel has to know of the rows. Up to 32 channels there is room for three waves on a SIMD: 32 x 1024 rows and keys, 4 heads, fp32 take
// 555 us (the whole gradient) with them, 566 with two. fp32 above 64 channels has one wave: 4 x 1024 rows, 8 heads of 128 take 546 us so, and
// 855 with two, whose registers spill; at 96 channels both take 426.
template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(kThreads, DP <= 32 ? 3 : sizeof(T) * DP <= 256 ? 2 : 1) void dq_kernel(const Dev a, const Work work) {
    constexpr int kTile = Ops<T>::kTile, kBlocks = kTile / 32;
    constexpr bool kGain = __is_same(T, _Float16);
    __shared__ __attribute__((aligned(1024))) T k_even[kTile * DP], k_odd[kTile * DP], v_even[kTile * DP], v_odd[kTile * DP];
    __shared__ int bounds[2][4];
    __shared__ Gaps gaps;

    const Place id = place_of();
    const int parts = SPLIT ? work.q_parts : 1, part = SPLIT ? id.x % parts : 0;
    const int block = (gridDim.x - 1 - id.x) / parts, head = id.head, b = id.batch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int i = block * kRows + wave * 32 + (lane & 31);
    const bool real = i < a.nq;
    const int kv = head / a.group;
    const Row row = real ? row_of(a, b, i) : no_row();
    int wlo = row.lo, whi = row.hi;
    join_rows(wlo, whi);
    const int64_t group = static_cast<int64_t>(b) * work.groups + block * 4 + wave;
    if (head == 0 && part == 0) {
        int alo = row.lo, ahi = row.hi;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            alo = max(alo, __shfl_xor(alo, d));
            ahi = min(ahi, __shfl_xor(ahi, d));
        }
        if (lane == 0) work.seen[group] = {wlo, whi, alo, ahi};
        work.spans[64 * group + lane] = half ? row.hi : row.lo;
        work.positions[64 * group + lane] = row.pos;
    }
    if (lane == 0) {
        bounds[0][wave] = wlo;
        bounds[1][wave] = whi;
    }
    const bool apart = a.spans && a.nq > 1;              // without spans a row sees all keys from the first on
    if (apart) gaps.tell(row);
    const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.nq + i;
    OwnRow<T, DP> q, dout;
    q.load(real ? static_cast<const T*>(a.q) + b * a.sq.batch + i * a.sq.row + head * a.sq.head : nullptr, a.dim);
    dout.load(real ? static_cast<const T*>(a.dout) + b * a.sdo.batch + i * a.sdo.row + head * a.sdo.head : nullptr, a.dim);
    if (a.scale < 0.f) q.negate();       // Score counts on a factor that is positive
    float delta = 0.f, stat = -kNoMax;
    {
        const int64_t mine = b * a.so.batch + i * a.so.row + head * a.so.head;
        OwnRow<T, DP> out, low;
        out.load(real ? static_cast<const T*>(a.out) + mine : nullptr, a.dim);
        low.load(real && sizeof(T) == 2 && a.out_low ? static_cast<const T*>(a.out_low) + mine : nullptr, a.dim);
#pragma unroll
        for (int s = 0; s < OwnRow<T, DP>::kSteps; ++s)
#pragma unroll
            for (int e = 0; e < Ops<T>::W; ++e)
                delta = fmaf(static_cast<float>(dout.f[s][e]), static_cast<float>(out.f[s][e]) + static_cast<float>(low.f[s][e]), delta);
        delta += other_half(delta);
    }
    if (real) stat = stat_of(a.lse_near ? a.lse_near[at] : a.lse[at] + left_out(a, b, i, row, head));
    if (part == 0)
        work.stats[64 * ((static_cast<int64_t>(b) * a.heads + head) * work.groups + block * 4 + wave) + lane] = half ? delta : Ops<T>::kShift - stat;
    __syncthreads();
    const int lo = min(min(bounds[0][0], bounds[0][1]), min(bounds[0][2], bounds[0][3]));
    const int hi = max(max(bounds[1][0], bounds[1][1]), max(bounds[1][2], bounds[1][3]));
    const int unseen = apart ? gaps.find(hi) : 0;
    const int first = lo < hi ? lo / kTile + part : 0, last = lo < hi ? (hi + kTile - 1) / kTile : 0;      // every parts-th tile

    const Score score(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
    f32x16 acc[DP / 32] = {};
    float gain = gain_for(0.f), largest = 0.f;
    Fetch<T, DP> ks, vs;
    ks.start(static_cast<const T*>(a.k) + b * a.sk.batch + kv * a.sk.head, a.sk.row, lo, hi, a.dim);
    vs.start(static_cast<const T*>(a.v) + b * a.sv.batch + kv * a.sv.head, a.sv.row, lo, hi, a.dim);
    if (first < last) {
        ks.load(k_even, first * kTile, a.dim);
        vs.load(v_even, first * kTile, a.dim);
    }
    const auto step = [&](int t, T* k_now, T* v_now, T* k_next, T* v_next) __attribute__((always_inline)) {
        arrived();                       // tile t is here, tile t - 1 is done with
        const int j0 = t * kTile;
        if (t + parts < last) {
            ks.load(k_next, j0 + parts * kTile, a.dim);
            vs.load(v_next, j0 + parts * kTile, a.dim);
        }
        if (unseen) gaps.template clear<T, DP, kTile>(unseen, j0, k_now, v_now);
        if (j0 + kTile <= wlo || j0 >= whi) return;
        const bool whole = __all(row.lo <= j0 && row.hi >= j0 + kTile);
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) {
            f32x16 s = q.dot(k_now + kb * 32 * DP);
            f32x16 ds = dout.dot(v_now + kb * 32 * DP);
            settle<T>(s, ds);
            score.apply<T>(s);
            // s becomes p, dp becomes ds, in place; what is the same for the whole wave stands outside of the loops over elements
            ds -= delta;
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] *= score.slope(s[e]);
            }
            if (a.slopes) {
                const float here = static_cast<float>(row.pos - (j0 + 4 * half));
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = fmaf(-slope, fabsf(here - static_cast<float>(32 * kb + reg_row(e, 0))), s[e]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) ds[e] *= exp2_(fmaf(s[e], score.mul, -stat));
            if (!whole) {                // one comparison: a row that sees none has lo = INT_MAX, hi = 0, and both sides wrap
                const int from = j0 + 4 * half - row.lo;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int c = 32 * kb + reg_row(e, 0);
                    if (static_cast<unsigned>(from + c) >= static_cast<unsigned>(row.hi - row.lo)) ds[e] = 0.f;
                }
            }
            if constexpr (kGain) {
                float m = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(m, fabsf(ds[e]));
                m = fmaxf(m, other_half(m));
                largest = fmaxf(largest, m);
                if (__any(m * gain >= 32768.f)) {
                    const float next = fminf(gain, gain_for(m)), f = next * inverse_gain(gain);
                    gain = next;
#pragma unroll
                    for (int db = 0; db < DP / 32; ++db) acc[db] *= f;
                }
                ds *= gain;
            }
            // A score gradient enters as two 16-bit numbers. With one, dq would be off by its rounding, the rounding of dq and
            // what the forward call's rounded weights leave in D: 2.5e-3 of dq in bf16 where rounding dq alone leaves 1.66e-3,
            // and 1.8e-3 so, for a quarter of this kernel's time (8192 rows and keys, 16 + 4 heads of 128: 806 us with one, 1004 to 1031 with two).
            const auto w = Ops<T>::pack(ds);
            if constexpr (sizeof(T) == 2) {
                const auto low = Ops<T>::rest(ds, w);
                // A wave with products to start goes before one that works on scores: 961 us for the 1004 of that call, 99 for 96
                // with documents of 512; at 64 channels, and in the other two kernels, it makes no difference or costs.
                if (DP > 64) __builtin_amdgcn_s_setprio(1);
                Ops<T>::template spread<DP>(acc, k_now + kb * 32 * DP, w, &low);
                if (DP > 64) __builtin_amdgcn_s_setprio(0);
            } else {
                Ops<T>::template spread<DP>(acc, k_now + kb * 32 * DP, w);
            }
        }
    };
    for (int t = first; t < last; t += 2 * parts) {  // both buffers written out, as in the forward kernel
        step(t, k_even, v_even, k_odd, v_odd);
        if (t + parts < last) step(t + parts, k_odd, v_odd, k_even, v_even);
    }
    if constexpr (kGain) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
        if (lane == 0) work.largest[((static_cast<int64_t>(b) * a.heads + head) * parts + part) * work.groups + block * 4 + wave] = largest;
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) settle<T>(acc[db]);
    if (!real) return;
    if (row.hi == 0) {                   // sees none, whatever the others see
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
    }
    const float f = kGain ? inverse_gain(gain) * a.scale : a.scale;
    if (SPLIT)
        write_row<float, DP>(work.q_sums + (((static_cast<int64_t>(part) * gridDim.z + b) * a.nq + i) * a.heads + head) * a.dim, acc, f, a.dim);
    else
        write_row<T, DP>(static_cast<T*>(a.dq) + b * a.sdq.batch + i * a.sdq.row + head * a.sdq.head, acc, f, a.dim);
}

// The tiles of kTile rows that see any of the keys [begin, end), for one query head after the other. What a tile sees comes through
// scalar loads: a vector load behind the fetches of a tile could only arrive after them.
// Of `parts` parts (a power of two) that share the tiles of these keys, part p takes those whose number plus the head's leaves p.
template <int GROUPS>                    // groups of 32 rows in a tile
struct Tiles {
    typedef const __attribute__((address_space(4))) Seen* Scalar;
    const Seen* seen;
    int groups, tiles, heads, begin, end, part, parts;
    int base;                            // 64 tiles from `base` on are in `mask`
    unsigned long long mask;
    // the current one
    int head, tile;
    Seen now[GROUPS];

    __device__ __forceinline__ void look() {
        const int t = base + (threadIdx.x & 63);
        bool any = false;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            if (t * GROUPS + g < groups) any |= seen[t * GROUPS + g].lo < end && seen[t * GROUPS + g].hi > begin;
        mask = __ballot(any && ((t + head) & (parts - 1)) == part);
    }
    __device__ __forceinline__ void start() {
        base = head = 0;
        look();
    }
    // moves to the next tile; false behind the last one
    __device__ __forceinline__ bool next() {
        while (mask == 0) {
            base += 64;
            if (base >= tiles) {
                base = 0;
                if (++head >= heads) return false;
            }
            look();
        }
        tile = base + __builtin_ctzll(mask);
        mask &= mask - 1;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const Scalar s = (Scalar)(seen + tile * GROUPS + g);
            now[g] = {s->lo, s->hi, s->all_lo, s->all_hi};
        }
        return true;
    }
};

// dk and dv. A workgroup of 4 waves takes 128 keys, 32 a wave, and walks over the rows that see any of them, for every query head
// that shares them. For 16-bit types of more than 64 channels v stays in LDS and is read for each product, which leaves a wave
// room beside another on its SIMD (256 registers); with k and v both in registers it would have some 390 and the SIMD for itself, and
// the matrix unit would wait while it works on scores: 623 TFLOP/s at 128 channels, 828 so. Where there are few keys and many rows
// the rows are dealt out to several workgroups (SPLIT), whose sums a last kernel adds up.
template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 || DP <= 64 ? 2 : 1) void dkv_kernel(const Dev a, const Work work) {
    constexpr bool kLdsV = sizeof(T) == 2 && DP > 64, kFresh = kLdsV && DP > 96;
    constexpr int kTile = kLdsV ? 32 : Ops<T>::kTile, kBlocks = kTile / 32;
    __shared__ __attribute__((aligned(1024))) T v_rows[kLdsV ? kRows * DP : 1];
    constexpr bool kGain = __is_same(T, _Float16);
    constexpr float kUnshift = 1.f / (1 << Ops<T>::kShift);
    __shared__ __attribute__((aligned(1024))) T q_even[kTile * DP], q_odd[kTile * DP], do_even[kTile * DP], do_odd[kTile * DP];
    __shared__ __attribute__((aligned(256))) float stats_even[64 * kBlocks], stats_odd[64 * kBlocks];
    __shared__ __attribute__((aligned(256))) int spans_even[64 * kBlocks], spans_odd[64 * kBlocks], pos_even[64 * kBlocks], pos_odd[64 * kBlocks];
    __shared__ float wave_max[4];

    const Place id = place_of();
    const int kv = id.head, b = id.batch;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int part = SPLIT ? id.x & (work.parts - 1) : 0;
    const int begin = (SPLIT ? id.x / work.parts : id.x) * kRows, w0 = begin + wave * 32, j = w0 + (lane & 31);   // keys of the workgroup, the wave, the lane
    const bool real = j < a.nk;
    OwnRow<T, DP> k, v;
    k.load(real ? static_cast<const T*>(a.k) + b * a.sk.batch + j * a.sk.row + kv * a.sk.head : nullptr, a.dim);
    if constexpr (kLdsV) {
        Fetch<T, DP, kRows> vs;
        vs.start(static_cast<const T*>(a.v) + b * a.sv.batch + kv * a.sv.head, a.sv.row, 0, a.nk, a.dim);
        vs.load(v_rows, begin, a.dim);
    } else {
        v.load(real ? static_cast<const T*>(a.v) + b * a.sv.batch + j * a.sv.row + kv * a.sv.head : nullptr, a.dim);
    }

    if (a.scale < 0.f) k.negate();       // used in scores alone
    float gain = 1.f;
    if constexpr (kGain) {
        const int each = work.groups * work.q_parts;                   // of a head
        const float* largest = work.largest + (static_cast<int64_t>(b) * a.heads + kv * a.group) * each;
        float m = 0.f;
        for (int64_t x = threadIdx.x; x < static_cast<int64_t>(a.group) * each; x += kThreads) m = fmaxf(m, largest[x]);
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
        if (lane == 0) wave_max[wave] = m;
        __syncthreads();
        gain = gain_for(fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3])));
    }

    const Score score(a);
    f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    Tiles<kBlocks> tiles;
    tiles.seen = work.seen + static_cast<int64_t>(b) * work.groups;
    tiles.groups = work.groups;
    tiles.tiles = (a.nq + kTile - 1) / kTile;
    tiles.heads = a.group;
    tiles.begin = begin;
    tiles.end = min(begin + kRows, a.nk);
    tiles.part = part;
    tiles.parts = SPLIT ? work.parts : 1;
    tiles.start();

    Fetch<T, DP, kTile> qs, dos;
    qs.start(static_cast<const T*>(a.q), a.sq.row, 0, a.nq, a.dim);
    dos.start(static_cast<const T*>(a.dout), a.sdo.row, 0, a.nq, a.dim);
    // starts the loads of the tile that `tiles` stands at, and of what the other kernel left about its rows
    const auto load = [&](T* q_to, T* do_to, float* stats_to, int* spans_to, int* pos_to) __attribute__((always_inline)) {
        const int head = kv * a.group + tiles.head;
        qs.base = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.sq.batch + head * a.sq.head);
        dos.base = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + b * a.sdo.batch + head * a.sdo.head);
        qs.load(q_to, tiles.tile * kTile, a.dim);
        dos.load(do_to, tiles.tile * kTile, a.dim);
        const int group = tiles.tile * kBlocks + wave;
        if (wave < kBlocks) {
            fetch_words(stats_to + 64 * wave, work.stats + 64 * ((static_cast<int64_t>(b) * a.heads + head) * work.groups + group));
            fetch_words(spans_to + 64 * wave, work.spans + 64 * (static_cast<int64_t>(b) * work.groups + group));
            if (a.slopes) fetch_words(pos_to + 64 * wave, work.positions + 64 * (static_cast<int64_t>(b) * work.groups + group));
        }
    };

    if constexpr (kLdsV)
        if (a.dim < DP) {                // noughts behind dim, as in an OwnRow: both sides of this product come from LDS
            arrived();
            constexpr int W = Ops<T>::W, kChunks = DP / W;
            for (int x = threadIdx.x; x < kRows * kChunks; x += kThreads)
                if (W * ((x % kChunks) ^ swizzle<T, DP>(x / kChunks)) >= a.dim) reinterpret_cast<typename Ops<T>::Frag*>(v_rows)[x] = {};
        }
    bool more = tiles.next();
    if (more) load(q_even, do_even, stats_even, spans_even, pos_even);
    const auto step = [&](T* q_now, T* do_now, const float* stats_now, const int* spans_now, const int* pos_now, T* q_next, T* do_next,
                          float* stats_next, int* spans_next, int* pos_next) __attribute__((always_inline)) {
        arrived();                       // this tile is here, the one before is done with
        const int head = kv * a.group + tiles.head;
        Seen now[kBlocks];
        bool all = true;                 // does every row see some key?
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            now[g] = tiles.now[g];
            all &= now[g].all_lo != INT32_MAX;
        }
        const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
        more = tiles.next();
        if (more) load(q_next, do_next, stats_next, spans_next, pos_next);
        if (!all) {                      // what q and dout hold in a row that sees none does not matter: noughts
            constexpr int kChunks = DP / Ops<T>::W;
            for (int x = threadIdx.x; x < kTile * kChunks; x += kThreads)
                if (spans_now[64 * (x / kChunks / 32) + 32 + x / kChunks % 32] == 0)
                    reinterpret_cast<typename Ops<T>::Frag*>(q_now)[x] = reinterpret_cast<typename Ops<T>::Frag*>(do_now)[x] = {};
            __syncthreads();
        }
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            if (now[g].lo >= w0 + 32 || now[g].hi <= w0) continue;
            const bool whole = now[g].all_lo <= w0 && now[g].all_hi >= w0 + 32;
            f32x16 s = k.template dot<kFresh>(q_now + g * 32 * DP);
            if (kFresh) __builtin_amdgcn_sched_barrier(0);
            f32x16 ds;
            if constexpr (kLdsV)
                ds = dot_from_lds<T, DP, kFresh>(do_now + g * 32 * DP, v_rows + wave * 32 * DP);
            else
                ds = v.dot(do_now + g * 32 * DP);
            settle<T>(s, ds);
            score.apply<T>(s);
            // s becomes p, dp becomes ds, in place; what is the same for the whole wave stands outside of the loops over elements
            const int rows0 = 64 * g + 4 * half;                       // and 8 x further: four rows
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 deltas = *reinterpret_cast<const f32x4*>(stats_now + rows0 + 32 + 8 * x);
#pragma unroll
                for (int e = 0; e < 4; ++e) ds[4 * x + e] -= deltas[e];
            }
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] *= score.slope(s[e]);
            }
            if (a.slopes) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[e] = fmaf(-slope, fabsf(static_cast<float>(pos_now[64 * g + reg_row(e, half)] - j)), s[e]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 stats = *reinterpret_cast<const f32x4*>(stats_now + rows0 + 8 * x);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * x + e] = exp2_(fmaf(s[4 * x + e], score.mul, stats[e]));
                    ds[4 * x + e] *= s[4 * x + e];
                }
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 64 * g + reg_row(e, half);
                    if (j < spans_now[at] || j >= spans_now[at + 32]) s[e] = ds[e] = 0.f;
                }
            }
            if constexpr (kGain) ds *= gain * kUnshift;
            // 16-bit types round weights and score gradients once: dk and dv are off by 2.4e-3 of themselves (bf16), 1.4 times what rounding
            // them alone leaves; a second part, as in dq, would cost two more products.
            Ops<T>::template spread<DP, kFresh>(dv, do_now + g * 32 * DP, Ops<T>::pack(s));
            if (kFresh) __builtin_amdgcn_sched_barrier(0);
            Ops<T>::template spread<DP, kFresh>(dk, q_now + g * 32 * DP, Ops<T>::pack(ds));
        }
    };
    while (more) {                       // both buffers written out, as in the forward kernel
        step(q_even, do_even, stats_even, spans_even, pos_even, q_odd, do_odd, stats_odd, spans_odd, pos_odd);
        if (more) step(q_odd, do_odd, stats_odd, spans_odd, pos_odd, q_even, do_even, stats_even, spans_even, pos_even);
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) settle<T>(dk[db], dv[db]);
    if (!real) return;
    const float fk = kGain ? inverse_gain(gain) * a.scale : a.scale;
    if (SPLIT) {
        const int64_t keys = static_cast<int64_t>(gridDim.z) * a.nk * gridDim.y, at = (static_cast<int64_t>(b) * a.nk + j) * gridDim.y + kv;
        write_row<float, DP>(work.sums + (part * keys + at) * a.dim, dk, fk, a.dim);
        write_row<float, DP>(work.sums + ((work.parts + part) * keys + at) * a.dim, dv, kUnshift, a.dim);
    } else {
        write_row<T, DP>(static_cast<T*>(a.dk) + b * a.sdk.batch + j * a.sdk.row + kv * a.sdk.head, dk, fk, a.dim);
        write_row<T, DP>(static_cast<T*>(a.dv) + b * a.sdv.batch + j * a.sdv.row + kv * a.sdv.head, dv, kUnshift, a.dim);
    }
}

// Adds up the parts of a gradient, four channels a thread, in the parts' order: sums [parts][batch][n][heads][dim] -> out.
template <typename T>
__global__ __launch_bounds__(256) void add_parts_kernel(const float* sums, const int parts, const int64_t rows, const int n, const int heads,
                                                        const int dim, T* out, const Strides s) {
    const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int quads = dim / 4;
    const int64_t row = id / quads;
    if (row >= rows) return;
    const int c = 4 * static_cast<int>(id - row * quads);
    f32x4 sum = {};
    for (int p = 0; p < parts; ++p) sum += *reinterpret_cast<const f32x4*>(sums + (p * rows + row) * dim + c);
    const int head = static_cast<int>(row % heads);
    const int64_t bn = row / heads, b = bn / n, i = bn % n;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(sum[e]);
    *reinterpret_cast<T4*>(out + b * s.batch + i * s.row + head * s.head + c) = o;
}

template <typename T>
void add_parts(const float* sums, int parts, int64_t batch, int n, int heads, int dim, void* out, const Strides& s, hipStream_t stream) {
    const int64_t rows = batch * n * heads;
    add_parts_kernel<T><<<static_cast<unsigned>((rows * (dim / 4) + 255) / 256), 256, 0, stream>>>(sums, parts, rows, n, heads, dim,
                                                                                                 static_cast<T*>(out), s);
}

// Workgroups that share the tiles of a block of rows or keys: a power of two up to 8 that brings the call to `wanted` workgroups, with
// `least` tiles each at least.
int parts_for(int64_t blocks, int64_t wanted, int64_t tiles, int least) {
    int parts = 1;
    while (parts < 8 && blocks * parts < wanted && tiles / (2 * parts) >= least) parts *= 2;
    return parts;
}

// Two workgroups a compute unit fill the chip; spans load them unevenly, and then four are better. dk and dv of 8192 packed tokens in
// documents of 340, 4 key/value heads shared by 16, are 256 blocks: 1056 us with a workgroup each, 542 with two, 304 with four,
// 285 with eight; where all rows see all keys 1692 us with one, 1178 with two, 1192 with four.
int parts_of(const ddpm_span_attention_args& a, bool spans) {
    const int64_t blocks = (static_cast<int64_t>(a.nk) + kRows - 1) / kRows * a.kv_heads * a.batch;
    return parts_for(blocks, spans ? 1024 : 512, (static_cast<int64_t>(a.nq) + 31) / 32 * (a.heads / a.kv_heads), 8);
}
int q_parts_of(const ddpm_span_attention_args& a) {
    const int64_t blocks = (static_cast<int64_t>(a.nq) + kRows - 1) / kRows * a.heads * a.batch;
    return parts_for(blocks, 512, (static_cast<int64_t>(a.nk) + 63) / 64, 4);
}

int groups_of(int nq) { return (nq + kRows - 1) / kRows * 4; }

// Places the parts of Work in a workspace, and returns its size: that of a call with spans, which has the more parts, so that one workspace
// serves all calls of the same sizes and type.
int64_t place(const ddpm_span_attention_args& a, void* workspace, Work* w) {
    w->groups = groups_of(a.nq);
    const int64_t rows = static_cast<int64_t>(a.batch) * w->groups, heads = rows * a.heads;
    char* at = static_cast<char*>(workspace);
    w->stats = reinterpret_cast<float*>(at);
    at += heads * 256;
    w->spans = reinterpret_cast<int*>(at);
    at += rows * 256;
    w->positions = reinterpret_cast<int*>(at);
    at += rows * 256;
    w->seen = reinterpret_cast<Seen*>(at);
    at += rows * sizeof(Seen);
    w->largest = reinterpret_cast<float*>(at);
    w->q_parts = q_parts_of(a);
    if (a.type == DDPM_F16) at += (heads * w->q_parts * 4 + 15) / 16 * 16;
    w->q_sums = reinterpret_cast<float*>(at);
    if (w->q_parts > 1) at += static_cast<int64_t>(w->q_parts) * a.batch * a.nq * a.heads * a.dim * 4;
    w->sums = reinterpret_cast<float*>(at);
    w->parts = parts_of(a, a.spans != nullptr);
    if (const int most = parts_of(a, true); most > 1) at += static_cast<int64_t>(most) * 2 * a.batch * a.nk * a.kv_heads * a.dim * 4;
    return at - static_cast<char*>(workspace);
}

template <typename T>
void launch(const ddpm_span_attention_args& a, void* workspace, hipStream_t stream) {
    const Dev d = dev_args(a);
    Work work;
    place(a, workspace, &work);
    for_dim(a.dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        const dim3 rows(work.groups / 4 * work.q_parts, a.heads, a.batch), keys((a.nk + kRows - 1) / kRows * work.parts, a.kv_heads, a.batch);
        if (a.nq > 0 && work.q_parts == 1) dq_kernel<T, DP, false><<<rows, kThreads, 0, stream>>>(d, work);
        if (a.nq > 0 && work.q_parts > 1) dq_kernel<T, DP, true><<<rows, kThreads, 0, stream>>>(d, work);
        if (a.nk > 0 && work.parts == 1) dkv_kernel<T, DP, false><<<keys, kThreads, 0, stream>>>(d, work);
        if (a.nk > 0 && work.parts > 1) dkv_kernel<T, DP, true><<<keys, kThreads, 0, stream>>>(d, work);
    });
    if (a.nq > 0 && work.q_parts > 1) add_parts<T>(work.q_sums, work.q_parts, a.batch, a.nq, a.heads, a.dim, a.dq, d.sdq, stream);
    if (a.nk > 0 && work.parts > 1) {
        add_parts<T>(work.sums, work.parts, a.batch, a.nk, a.kv_heads, a.dim, a.dk, d.sdk, stream);
        add_parts<T>(work.sums + static_cast<int64_t>(work.parts) * a.batch * a.nk * a.kv_heads * a.dim, work.parts, a.batch, a.nk, a.kv_heads, a.dim,
                     a.dv, d.sdv, stream);
    }
}

bool check_bwd(const ddpm_span_attention_args& a) {
    if (!check_args(a)) return false;
    const int w = a.type == DDPM_F32 ? 4 : 8;
    for (const int64_t* s : {a.dout_stride, a.dq_stride, a.dk_stride, a.dv_stride})
        if (s[0] % w || s[1] % w || s[2] % w) return false;
    return fits_tile(a, a.q_stride) && fits_tile(a, a.dout_stride);
}

}  // namespace

extern "C" int64_t ddpm_span_attention_bwd_workspace(const ddpm_span_attention_args* a) {
    if (!a || !check_bwd(*a)) return ddpm::fail_invalid("span attention sizes, type or strides");
    Work work;
    int64_t bytes = place(entries_from(*a, 0), nullptr, &work);
    if (a->batch > kMaxBatch)            // the last launches, of fewer entries, may deal out their work
        bytes = std::max(bytes, place(entries_from(*a, a->batch / kMaxBatch * kMaxBatch), nullptr, &work));
    return bytes;
}

extern "C" int ddpm_span_attention_bwd(const ddpm_span_attention_args* a, void* workspace, void* stream) {
    DDPM_REQUIRE(a && check_bwd(*a));
    if (a->batch == 0) return DDPM_OK;
    DDPM_REQUIRE(a->nq == 0 || (a->q && a->out && a->lse && a->dout && a->dq));
    DDPM_REQUIRE(a->nk == 0 || (a->k && a->v && a->dk && a->dv));
    for (const void* p : {a->q, a->k, a->v, static_cast<const void*>(a->out), static_cast<const void*>(a->out_low), a->dout, static_cast<const void*>(a->dq),
                          static_cast<const void*>(a->dk), static_cast<const void*>(a->dv), static_cast<const void*>(workspace)})
        DDPM_REQUIRE(ddpm::aligned16(p));
    DDPM_REQUIRE(a->nq == 0 || workspace);                // dk and dv of no rows are noughts, and need none
    for (int64_t first = 0; first < a->batch; first += kMaxBatch) {
        const ddpm_span_attention_args part = entries_from(*a, static_cast<int>(first));
        if (a->type == DDPM_F32)
            launch<float>(part, workspace, as_stream(stream));
        else if (a->type == DDPM_BF16)
            launch<__bf16>(part, workspace, as_stream(stream));
        else
            launch<_Float16>(part, workspace, as_stream(stream));
    }
    return ddpm::check_launch("span attention backward");
}
