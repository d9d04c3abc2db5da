// Span attention, gradient (the mathematics and the two products are in span_attention.h):
//   D_i = sum_c dout_ic out_ic,  p_ij = exp(w_ij - lse_i),  dp_ij = dout_i . v_j,  ds_ij = scale (du/dt)_ij p_ij (dp_ij - D_i)
//   dq_i = sum_j ds_ij k_j,  dk_j = sum_i ds_ij q_i,  dv_j = sum_i p_ij dout_i
// in two kernels, each of which recomputes the scores: dq walks over keys with rows in registers, dk and dv over rows with keys in
// registers. That is 7 products for the 5 of a single kernel, whose dq would be added up with atomics in an order that changes
// from call to call, and in fp32 memory that must be cleared before and converted behind. The gradient of a key/value head is
// summed over the query heads that share it inside its workgroup.
#include "span_attention.h"

using ddpm::as_stream;

namespace {

using namespace span;

constexpr int kRows = 128;               // rows (dq) or keys (dk, dv) of a workgroup, 32 a wave

// What 32 rows see together: keys [lo, hi) are seen by some of them, [all_lo, all_hi) by all (all_lo = INT_MAX when one sees none).
struct Seen {
    int lo, hi, all_lo, all_hi;
};

struct Work {
    float* delta;                        // D: [batch][heads][nq]
    Seen* seen;                          // [batch][groups], groups of 32 rows
    float* largest;                      // fp16: largest |ds| of the rows of a group: [batch][heads][groups]
    int groups;
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
__device__ __forceinline__ void write_row(T* out, const f32x16* acc, float f, int dim) {
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

template <typename T, int DP>
__global__ __launch_bounds__(kThreads, sizeof(T) * DP <= 256 ? 2 : 1) void dq_kernel(const Dev a, const Work work) {
    constexpr int kTile = Ops<T>::kTile, kBlocks = kTile / 32;
    constexpr bool kGain = __is_same(T, _Float16);
    __shared__ __attribute__((aligned(1024))) T k_even[kTile * DP], k_odd[kTile * DP], v_even[kTile * DP], v_odd[kTile * DP];
    __shared__ int bounds[2][4];

    const dim3 id = ddpm::xcd_block();
    const int block = gridDim.x - 1 - id.x, head = id.y, b = id.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int i = block * kRows + wave * 32 + (lane & 31);
    const bool real = i < a.nq;
    const int kv = head / a.group;
    const Row row = real ? row_of(a, b, i) : no_row();
    int wlo = row.lo, whi = row.hi;
    join_rows(wlo, whi);
    if (head == 0) {
        int alo = row.lo, ahi = row.hi;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            alo = max(alo, __shfl_xor(alo, d));
            ahi = min(ahi, __shfl_xor(ahi, d));
        }
        if (lane == 0) work.seen[static_cast<int64_t>(b) * work.groups + block * 4 + wave] = {wlo, whi, alo, ahi};
    }
    if (lane == 0) {
        bounds[0][wave] = wlo;
        bounds[1][wave] = whi;
    }
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
    if (real) {
        stat = stat_of(a.lse[at]);
        if (half == 0) work.delta[at] = delta;
    }
    __syncthreads();
    const int lo = min(min(bounds[0][0], bounds[0][1]), min(bounds[0][2], bounds[0][3]));
    const int hi = max(max(bounds[1][0], bounds[1][1]), max(bounds[1][2], bounds[1][3]));
    const int first = lo < hi ? lo / kTile : 0, last = lo < hi ? (hi + kTile - 1) / kTile : 0;

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
    const auto step = [&](int t, const T* k_now, const T* v_now, T* k_next, T* v_next) __attribute__((always_inline)) {
        arrived();                       // tile t is here, tile t - 1 is done with
        const int j0 = t * kTile;
        if (t + 1 < last) {
            ks.load(k_next, j0 + kTile, a.dim);
            vs.load(v_next, j0 + kTile, a.dim);
        }
        if (j0 + kTile <= wlo || j0 >= whi) return;
        const bool whole = __all(row.lo <= j0 && row.hi >= j0 + kTile);
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) {
            f32x16 s = q.dot(k_now + kb * 32 * DP);
            const f32x16 dp = dout.dot(v_now + kb * 32 * DP);
            score.apply<T>(s);
            f32x16 ds = s;               // log2(e) w, then p, then ds; the uniform cases stand outside of the loops over elements
            if (a.slopes) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    ds[e] = fmaf(-slope, fabsf(static_cast<float>(row.pos - (j0 + 32 * kb + reg_row(e, half)))), ds[e]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) ds[e] = exp2_(fmaf(ds[e], score.mul, -stat)) * (dp[e] - delta);
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] *= score.slope(s[e]);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = j0 + 32 * kb + reg_row(e, half);
                    if (j < row.lo || j >= row.hi) ds[e] = 0.f;
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
            Ops<T>::template spread<DP>(acc, k_now + kb * 32 * DP, Ops<T>::pack(ds));
        }
    };
    for (int t = first; t < last; t += 2) {          // both buffers written out, as in the forward kernel
        step(t, k_even, v_even, k_odd, v_odd);
        if (t + 1 < last) step(t + 1, k_odd, v_odd, k_even, v_even);
    }
    if constexpr (kGain) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) largest = fmaxf(largest, __shfl_xor(largest, d));
        if (lane == 0) work.largest[(static_cast<int64_t>(b) * a.heads + head) * work.groups + block * 4 + wave] = largest;
    }
    if (real)
        write_row<T, DP>(static_cast<T*>(a.dq) + b * a.sdq.batch + i * a.sdq.row + head * a.sdq.head, acc, kGain ? inverse_gain(gain) * a.scale : a.scale, a.dim);
}

// The tiles of kTile rows that see any of the keys [begin, end), for one query head after the other. A lane holds what one of 64
// tiles sees, so that going on needs no memory (a load behind the fetches of a tile could only arrive after them).
template <int GROUPS>                    // groups of 32 rows in a tile
struct Tiles {
    const Seen* seen;
    int groups, tiles, heads, begin, end;
    int base;                            // 64 tiles from `base` on are in `mask` and `mine`
    unsigned long long mask;
    Seen mine[GROUPS];
    // the current one
    int head, tile;
    Seen now[GROUPS];

    __device__ __forceinline__ void look() {
        const int t = base + (threadIdx.x & 63);
        bool any = false;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            mine[g] = {INT32_MAX, 0, INT32_MAX, 0};
            if (t * GROUPS + g < groups) mine[g] = seen[t * GROUPS + g];
            any |= mine[g].lo < end && mine[g].hi > begin;
        }
        mask = __ballot(any);
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
        const int lane = __builtin_ctzll(mask);
        mask &= mask - 1;
        tile = base + lane;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            now[g].lo = __builtin_amdgcn_readlane(mine[g].lo, lane);
            now[g].hi = __builtin_amdgcn_readlane(mine[g].hi, lane);
            now[g].all_lo = __builtin_amdgcn_readlane(mine[g].all_lo, lane);
            now[g].all_hi = __builtin_amdgcn_readlane(mine[g].all_hi, lane);
        }
        return true;
    }
};

template <typename T, int DP>
__global__ __launch_bounds__(kThreads, DP <= 64 ? 2 : 1) void dkv_kernel(const Dev a, const Work work) {
    constexpr int kTile = Ops<T>::kTile, kBlocks = kTile / 32;
    constexpr bool kGain = __is_same(T, _Float16);
    constexpr float kUnshift = 1.f / (1 << Ops<T>::kShift);
    __shared__ __attribute__((aligned(1024))) T q_even[kTile * DP], q_odd[kTile * DP], do_even[kTile * DP], do_odd[kTile * DP];
    __shared__ __attribute__((aligned(16))) float stat_tile[2][kTile], delta_tile[2][kTile];
    __shared__ __attribute__((aligned(16))) int lo_tile[2][kTile], hi_tile[2][kTile], pos_tile[2][kTile];
    __shared__ float wave_max[4];

    const dim3 id = ddpm::xcd_block();
    const int kv = id.y, b = id.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int begin = id.x * kRows, w0 = begin + wave * 32, j = w0 + (lane & 31);   // keys of the workgroup, the wave, the lane
    const bool real = j < a.nk;
    OwnRow<T, DP> k, v;
    k.load(real ? static_cast<const T*>(a.k) + b * a.sk.batch + j * a.sk.row + kv * a.sk.head : nullptr, a.dim);
    v.load(real ? static_cast<const T*>(a.v) + b * a.sv.batch + j * a.sv.row + kv * a.sv.head : nullptr, a.dim);

    if (a.scale < 0.f) k.negate();       // used in scores alone
    float gain = 1.f;
    if constexpr (kGain) {
        const float* largest = work.largest + (static_cast<int64_t>(b) * a.heads + kv * a.group) * work.groups;
        float m = 0.f;
        for (int64_t x = threadIdx.x; x < static_cast<int64_t>(a.group) * work.groups; x += kThreads) m = fmaxf(m, largest[x]);
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
    tiles.start();

    // Of the tile that `tiles` stands at: what its rows see, their lse and their D, into registers and then (write_rows) into LDS, and
    // the loads of its q and dout, in this order, so that the registers do not have to wait for the tile.
    Row row = no_row();
    float stat = 0.f, delta = 0.f, next_slope = 0.f;
    Fetch<T, DP> qs, dos;
    qs.start(static_cast<const T*>(a.q), a.sq.row, 0, a.nq, a.dim);
    dos.start(static_cast<const T*>(a.dout), a.sdo.row, 0, a.nq, a.dim);
    const auto load = [&](T* q_to, T* do_to) __attribute__((always_inline)) {
        const int head = kv * a.group + tiles.head, i0 = tiles.tile * kTile;
        if (a.slopes) next_slope = a.slopes[head] * kLog2e;
        if (threadIdx.x < kTile) {
            const int i = i0 + threadIdx.x;
            row = no_row();
            stat = -kNoMax;
            delta = 0.f;
            if (i < a.nq) {
                const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.nq + i;
                row = row_of(a, b, i);
                stat = a.lse[at];
                delta = work.delta[at];
            }
        }
        qs.base = reinterpret_cast<const char*>(static_cast<const T*>(a.q) + b * a.sq.batch + head * a.sq.head);
        dos.base = reinterpret_cast<const char*>(static_cast<const T*>(a.dout) + b * a.sdo.batch + head * a.sdo.head);
        qs.load(q_to, i0, a.dim);
        dos.load(do_to, i0, a.dim);
    };
    const auto write_rows = [&](int to) __attribute__((always_inline)) {
        if (threadIdx.x < kTile) {
            lo_tile[to][threadIdx.x] = row.lo;
            hi_tile[to][threadIdx.x] = row.hi;
            pos_tile[to][threadIdx.x] = row.pos;
            stat_tile[to][threadIdx.x] = Ops<T>::kShift - stat_of(stat);
            delta_tile[to][threadIdx.x] = delta;
        }
    };

    bool more = tiles.next();
    if (more) {
        load(q_even, do_even);
        write_rows(0);
    }
    const auto step = [&](int in, T* q_now, T* do_now, T* q_next, T* do_next) __attribute__((always_inline)) {
        arrived();                       // this tile is here, the one before is done with
        const float slope = next_slope;
        Seen now[kBlocks];
        bool all = true;                 // does every row see some key?
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            now[g] = tiles.now[g];
            all &= now[g].all_lo != INT32_MAX;
        }
        more = tiles.next();
        if (more) load(q_next, do_next);
        if (!all) {                      // what q and dout hold in a row that sees none does not matter: noughts
            constexpr int kChunks = DP / Ops<T>::W;
            for (int x = threadIdx.x; x < kTile * kChunks; x += kThreads)
                if (hi_tile[in][x / kChunks] == 0)
                    reinterpret_cast<typename Ops<T>::Frag*>(q_now)[x] = reinterpret_cast<typename Ops<T>::Frag*>(do_now)[x] = {};
            __syncthreads();
        }
#pragma unroll
        for (int g = 0; g < kBlocks; ++g) {
            if (now[g].lo >= w0 + 32 || now[g].hi <= w0) continue;
            const bool whole = now[g].all_lo <= w0 && now[g].all_hi >= w0 + 32;
            f32x16 s = k.dot(q_now + g * 32 * DP);
            const f32x16 dp = v.dot(do_now + g * 32 * DP);
            score.apply<T>(s);
            f32x16 p = s, ds;            // log2(e) w, then p; the uniform cases stand outside of the loops over elements
            if (a.slopes) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    p[e] = fmaf(-slope, fabsf(static_cast<float>(pos_tile[in][32 * g + reg_row(e, half)] - j)), p[e]);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const f32x4 stats = *reinterpret_cast<const f32x4*>(stat_tile[in] + 32 * g + 8 * x + 4 * half);       // of four rows
                const f32x4 deltas = *reinterpret_cast<const f32x4*>(delta_tile[in] + 32 * g + 8 * x + 4 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[4 * x + e] = exp2_(fmaf(p[4 * x + e], score.mul, stats[e]));
                    ds[4 * x + e] = p[4 * x + e] * (dp[4 * x + e] - deltas[e]);
                }
            }
            if (score.capped) {
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] *= score.slope(s[e]);
            }
            if (!whole) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 32 * g + reg_row(e, half);
                    if (j < lo_tile[in][at] || j >= hi_tile[in][at]) p[e] = ds[e] = 0.f;
                }
            }
            if constexpr (kGain) ds *= gain * kUnshift;
            Ops<T>::template spread<DP>(dv, do_now + g * 32 * DP, Ops<T>::pack(p));
            Ops<T>::template spread<DP>(dk, q_now + g * 32 * DP, Ops<T>::pack(ds));
        }
        if (more) write_rows(in ^ 1);
    };
    while (more) {                       // both buffers written out, as in the forward kernel
        step(0, q_even, do_even, q_odd, do_odd);
        if (more) step(1, q_odd, do_odd, q_even, do_even);
    }
    if (!real) return;
    write_row<T, DP>(static_cast<T*>(a.dk) + b * a.sdk.batch + j * a.sdk.row + kv * a.sdk.head, dk, kGain ? inverse_gain(gain) * a.scale : a.scale, a.dim);
    write_row<T, DP>(static_cast<T*>(a.dv) + b * a.sdv.batch + j * a.sdv.row + kv * a.sdv.head, dv, kUnshift, a.dim);
}

int groups_of(int nq) { return (nq + kRows - 1) / kRows * 4; }

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

template <typename T>
void launch(const ddpm_span_attention_args& a, void* workspace, hipStream_t stream) {
    const Dev d = dev_args(a);
    Work work = {};
    work.groups = groups_of(a.nq);
    char* at = static_cast<char*>(workspace);
    work.seen = reinterpret_cast<Seen*>(at);
    at += static_cast<int64_t>(a.batch) * work.groups * sizeof(Seen);
    work.delta = reinterpret_cast<float*>(at);
    at += round16(static_cast<int64_t>(a.batch) * a.heads * a.nq * 4);
    work.largest = reinterpret_cast<float*>(at);
    for_dim(a.dim, [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        if (a.nq > 0) dq_kernel<T, DP><<<dim3(work.groups / 4, a.heads, a.batch), kThreads, 0, stream>>>(d, work);
        if (a.nk > 0) dkv_kernel<T, DP><<<dim3((a.nk + kRows - 1) / kRows, a.kv_heads, a.batch), kThreads, 0, stream>>>(d, work);
    });
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
    const int64_t groups = groups_of(a->nq);
    return static_cast<int64_t>(a->batch) * groups * static_cast<int64_t>(sizeof(Seen)) +
           round16(static_cast<int64_t>(a->batch) * a->heads * a->nq * 4) +
           (a->type == DDPM_F16 ? round16(static_cast<int64_t>(a->batch) * a->heads * groups * 4) : 0);
}

extern "C" int ddpm_span_attention_bwd(const ddpm_span_attention_args* a, void* workspace, void* stream) {
    DDPM_REQUIRE(a && check_bwd(*a));
    if (a->batch == 0) return DDPM_OK;
    DDPM_REQUIRE(a->nq == 0 || (a->q && a->out && a->lse && a->dout && a->dq));
    DDPM_REQUIRE(a->nk == 0 || (a->k && a->v && a->dk && a->dv));
    for (const void* p : {a->q, a->k, a->v, static_cast<const void*>(a->out), static_cast<const void*>(a->out_low), a->dout, static_cast<const void*>(a->dq),
                          static_cast<const void*>(a->dk), static_cast<const void*>(a->dv), static_cast<const void*>(workspace)})
        DDPM_REQUIRE(ddpm::aligned16(p));
    DDPM_REQUIRE(a->nq == 0 || workspace);
    if (a->type == DDPM_F32)
        launch<float>(*a, workspace, as_stream(stream));
    else if (a->type == DDPM_BF16)
        launch<__bf16>(*a, workspace, as_stream(stream));
    else
        launch<_Float16>(*a, workspace, as_stream(stream));
    return ddpm::check_launch("span attention backward");
}
