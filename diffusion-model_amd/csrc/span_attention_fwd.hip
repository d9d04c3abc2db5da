// Span attention, forward (the mathematics and the two products are in span_attention.h).
//
// A workgroup of 4 waves takes 128 rows of one head, 32 a wave, and walks over the keys that any of them sees, a tile of 64
// (fp32: 32) at a time: k and v go straight into LDS, the next tile's while this one is worked on, and a
// running maximum and sum turn the scores into weights in one pass. With few rows (single tokens) the query heads that share
// a key/value head are rows of one workgroup, and the keys are split over workgroups whose parts a second kernel joins.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "span_attention.h"

using ddpm::as_stream;

namespace span {

bool fits_tile(const ddpm_span_attention_args& a, const int64_t* stride) {
    return stride[1] >= 0 && stride[1] < (int64_t(1) << 31) / kMaxTile / (a.type == DDPM_F32 ? 4 : 2);
}

bool check_args(const ddpm_span_attention_args& a) {
    const int w = a.type == DDPM_F32 ? 4 : 8;
    const auto fits = [&](const int64_t* s) { return s[0] % w == 0 && s[1] % w == 0 && s[2] % w == 0; };
    return (a.type == DDPM_F32 || a.type == DDPM_BF16 || a.type == DDPM_F16) && a.batch >= 0 && a.nq >= 0 && a.nk >= 0 &&
           a.heads >= 1 && a.heads <= 65535 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0 && a.dim >= w &&
           a.dim <= DDPM_SPAN_ATTENTION_MAX_DIM && a.dim % w == 0 && a.nq <= (1 << 30) && a.nk <= (1 << 30) &&
           a.scale >= -1e30f && a.scale <= 1e30f && (a.softcap == 0.f || (a.softcap >= 1e-30f && a.softcap <= 1e30f &&
           std::abs(a.scale) / static_cast<double>(a.softcap) <= 1e30)) && fits(a.q_stride) && fits(a.k_stride) && fits(a.v_stride) &&
           fits(a.out_stride) && fits_tile(a, a.k_stride) && fits_tile(a, a.v_stride);
}

Dev dev_args(const ddpm_span_attention_args& a) {
    const auto strides = [](const int64_t* s) { return Strides{s[0], s[1], s[2]}; };
    Dev d = {};
    d.nq = a.nq;
    d.nk = a.nk;
    d.heads = a.heads;
    d.group = a.heads / a.kv_heads;
    d.dim = a.dim;
    d.causal = a.causal != 0;
    d.scale = a.scale;
    d.softcap = a.softcap;
    d.slopes = a.slopes;
    d.spans = a.spans;
    d.positions = a.positions;
    d.span_batch = a.span_batch_stride;
    d.position_batch = a.position_batch_stride;
    d.q = a.q;
    d.k = a.k;
    d.v = a.v;
    d.out = a.out;
    d.out_low = a.out_low;
    d.lse = a.lse;
    d.lse_near = a.lse_near;
    d.sq = strides(a.q_stride);
    d.sk = strides(a.k_stride);
    d.sv = strides(a.v_stride);
    d.so = strides(a.out_stride);
    d.dout = a.dout;
    d.dq = a.dq;
    d.dk = a.dk;
    d.dv = a.dv;
    d.sdo = strides(a.dout_stride);
    d.sdq = strides(a.dq_stride);
    d.sdk = strides(a.dk_stride);
    d.sdv = strides(a.dv_stride);
    return d;
}

ddpm_span_attention_args entries_from(const ddpm_span_attention_args& a, int first) {
    ddpm_span_attention_args r = a;
    const int64_t size = a.type == DDPM_F32 ? 4 : 2;
    const auto move = [&](auto*& p, int64_t bytes) {
        if (p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(p) + first * bytes);
    };
    r.batch = std::min(a.batch - first, kMaxBatch);
    move(r.spans, a.span_batch_stride * 4);
    move(r.positions, a.position_batch_stride * 4);
    move(r.q, a.q_stride[0] * size);
    move(r.k, a.k_stride[0] * size);
    move(r.v, a.v_stride[0] * size);
    move(r.out, a.out_stride[0] * size);
    move(r.out_low, a.out_stride[0] * size);
    move(r.lse, static_cast<int64_t>(a.heads) * a.nq * 4);
    move(r.lse_near, static_cast<int64_t>(a.heads) * a.nq * 4);
    move(r.dout, a.dout_stride[0] * size);
    move(r.dq, a.dq_stride[0] * size);
    move(r.dk, a.dk_stride[0] * size);
    move(r.dv, a.dv_stride[0] * size);
    return r;
}

}  // namespace span

namespace {

using namespace span;

constexpr int kRows = 128;               // rows of a workgroup
constexpr int kMaxSplits = 128;          // parts of the keys

// How the rows and keys of a call are spread over workgroups.
struct Plan {
    int pack;                            // query heads that are rows of one workgroup
    int blocks;                          // workgroups along the rows
    int splits;                          // parts of the keys
};

Plan plan_of(const ddpm_span_attention_args& a) {
    Plan p;
    const int group = a.heads / a.kv_heads, tile = a.type == DDPM_F32 ? 32 : 64;
    // Rows of one head that do not fill a workgroup share it with the other heads of their group: k and v are read once for all.
    p.pack = a.nq < kRows ? group : 1;
    p.blocks = static_cast<int>((static_cast<int64_t>(a.nq) * p.pack + kRows - 1) / kRows);
    const int64_t all = static_cast<int64_t>(p.blocks) * (a.heads / p.pack) * a.batch, tiles = (a.nk + tile - 1) / tile;
    // Two workgroups a compute unit, each with 4 tiles at least, so that joining stays small beside reading.
    p.splits = all > 0 && all < 512 ? static_cast<int>(std::min<int64_t>((512 + all - 1) / all, tiles / 4)) : 1;
    p.splits = std::max(1, std::min(p.splits, kMaxSplits));
    return p;
}

__device__ __forceinline__ void write_lse(const Dev& a, int64_t at, float lse, int b, int i, const Row& row, int head) {
    if (a.lse_near) a.lse_near[at] = lse;
    if (a.lse) a.lse[at] = lse - left_out(a, b, i, row, head);
}

struct Parts {                           // of a split call: per part and row the sum before division, its maximum and weight sum
    float* out;                          // [splits][batch][heads][nq][dim]
    float* stat;                         // [splits][batch][heads][nq][2]
    int splits;
    int64_t rows;                        // batch * heads * nq
};

template <typename T, int DP, bool SPLIT>
__global__ __launch_bounds__(kThreads, 2) void fwd_kernel(const Dev a, const int pack, const Parts parts) {
    constexpr int kTile = Ops<T>::kTile, kBlocks = kTile / 32;
    __shared__ __attribute__((aligned(1024))) T k_even[kTile * DP], k_odd[kTile * DP], v_even[kTile * DP], v_odd[kTile * DP];
    __shared__ int bounds[2][4];
    __shared__ Gaps gaps;

    // x: row blocks (the last first: under causal order they have most to do), and with SPLIT the parts of the keys beside them
    const Place id = place_of();
    const int part = SPLIT ? id.x % parts.splits : 0;
    const int block = SPLIT ? id.x / parts.splits : gridDim.x - 1 - id.x;
    const int b = id.batch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int r = block * kRows + wave * 32 + (lane & 31);          // row of this lane's column
    const bool real = r < a.nq * pack;
    const int i = real ? r / pack : 0;
    const int head = id.head * pack + (real ? r % pack : 0);
    const int kv = (id.head * pack) / a.group;

    const Row row = real ? row_of(a, b, i) : no_row();
    int wlo = row.lo, whi = row.hi;
    join_rows(wlo, whi);
    if (lane == 0) {
        bounds[0][wave] = wlo;
        bounds[1][wave] = whi;
    }
    const bool apart = a.spans && a.nq > 1;              // without spans a row sees all keys from the first on
    if (apart) gaps.tell(row);
    OwnRow<T, DP> q;
    q.load(real ? static_cast<const T*>(a.q) + b * a.sq.batch + i * a.sq.row + head * a.sq.head : nullptr, a.dim);
    if (a.scale < 0.f) q.negate();       // Score counts on a factor that is positive
    __syncthreads();
    const int lo = min(min(bounds[0][0], bounds[0][1]), min(bounds[0][2], bounds[0][3]));
    const int hi = max(max(bounds[1][0], bounds[1][1]), max(bounds[1][2], bounds[1][3]));
    const int unseen = apart ? gaps.find(hi) : 0;

    int first = lo < hi ? lo / kTile : 0, last = lo < hi ? (hi + kTile - 1) / kTile : 0;   // tiles
    if (SPLIT) {
        const int n = last - first, begin = first;
        first = begin + static_cast<int>(static_cast<int64_t>(n) * part / parts.splits);
        last = begin + static_cast<int>(static_cast<int64_t>(n) * (part + 1) / parts.splits);
    }

    Score score(a);
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;

    f32x16 acc[DP / 32] = {};
    float top = kNoMax, sum = 0.f;       // of this column: maximum of all its scores, sum of this lane half's weights
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
        if (t + 1 < last) {
            ks.load(k_next, j0 + kTile, a.dim);
            vs.load(v_next, j0 + kTile, a.dim);
        }
        if (unseen) gaps.template clear<T, DP, kTile>(unseen, j0, k_now, v_now);
        if (j0 + kTile <= wlo || j0 >= whi) return;                 // nothing here for this wave's rows
        f32x16 s[kBlocks];
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) s[kb] = q.dot(k_now + kb * 32 * DP);
        if constexpr (kBlocks == 2)
            settle<T>(s[0], s[1]);
        else
            settle<T>(s[0]);
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) score.apply<T>(s[kb]);
        if (a.slopes) {
#pragma unroll
            for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    s[kb][e] = fmaf(-slope, fabsf(static_cast<float>(row.pos - (j0 + 32 * kb + reg_row(e, half)))), s[kb][e]);
        }
        if (!__all(row.lo <= j0 && row.hi >= j0 + kTile)) {
#pragma unroll
            for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = j0 + 32 * kb + reg_row(e, half);
                    if (j < row.lo || j >= row.hi) s[kb][e] = -INFINITY;
                }
        }
        float m = s[0][0];
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb)
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, s[kb][e]);
        m = fmaxf(m, other_half(m)) * score.mul;
        if (__any(m > top + Ops<T>::kSlack)) {
            m = fmaxf(m, top);
            const float f = exp2_(top - m);
            top = m;
            sum *= f;
#pragma unroll
            for (int db = 0; db < DP / 32; ++db) acc[db] *= f;
            // A score enters its exponential as a product that is not rounded, and `top` is one that is: past 2^20 what the rounding left
            // would be a factor of its own, and overflow. From there on scores are rounded first.
            if (score.plain && __any(fabsf(top) > 1048576.f && top != kNoMax)) {
#pragma unroll
                for (int kb = 0; kb < kBlocks; ++kb) s[kb] *= score.mul;
                score.plain = false;
                score.mul = 1.f;
            }
        }
        const float shift = Ops<T>::kShift - top;
#pragma unroll
        for (int kb = 0; kb < kBlocks; ++kb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[kb][e] = exp2_(fmaf(s[kb][e], score.mul, shift));
                sum += s[kb][e];
            }
            // 16-bit types round weights for the matrix instructions, their sum stays fp32: out is off by 2.2e-3 of itself (bf16, 16384 keys),
            // where rounding it alone leaves 1.65e-3. A second part of each weight would double this product.
            Ops<T>::template spread<DP>(acc, v_now + kb * 32 * DP, Ops<T>::pack(s[kb]));
        }
    };
    // The two buffers are variables of their own, and the loop is written out for both: with one indexed by t the compiler has to
    // assume that a read of this tile may meet the loads of the next, and waits for them at once.
    for (int t = first; t < last; t += 2) {
        step(t, k_even, v_even, k_odd, v_odd);
        if (t + 1 < last) step(t + 1, k_odd, v_odd, k_even, v_even);
    }

#pragma unroll
    for (int db = 0; db < DP / 32; ++db) settle<T>(acc[db]);
    sum += other_half(sum);
    if (!real) return;
    const int64_t at = (static_cast<int64_t>(b) * a.heads + head) * a.nq + i;
    if (SPLIT) {
        float* out = parts.out + (part * parts.rows + at) * a.dim;
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * db + 8 * g + 4 * half;
                if (d < a.dim) *reinterpret_cast<f32x4*>(out + d) = f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
            }
        if (half == 0) {
            parts.stat[2 * (part * parts.rows + at)] = top - Ops<T>::kShift;
            parts.stat[2 * (part * parts.rows + at) + 1] = sum;
        }
        return;
    }
    if (half == 0) write_lse(a, at, sum == 0.f ? -INFINITY : (top - Ops<T>::kShift + log2f(sum)) * kLn2, b, i, row, head);
    // no weight, no output: nought times a sum of noughts would be NaN where another row sees a value that is not finite
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (sum == 0.f) {
#pragma unroll
        for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
    }
    const int64_t out = b * a.so.batch + i * a.so.row + head * a.so.head;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * db + 8 * g + 4 * half;
            const float o[4] = {acc[db][4 * g] * inv, acc[db][4 * g + 1] * inv, acc[db][4 * g + 2] * inv, acc[db][4 * g + 3] * inv};
            if (d < a.dim) write_out<T>(a, out + d, o);
        }
}

// Joins the parts of a split call, a workgroup per row: the parts' maxima and sums at once, then 8 groups of 32 lanes add up every
// eighth part, 4 channels a lane (lanes behind dim idle), and the groups are added in order. 128 parts of 32 rows take 5 us; a
// wave per row that walked over the parts took 95.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Dev a, const Parts parts) {
    __shared__ float factor[kMaxSplits];
    __shared__ float wave_top[4], wave_sum[4];
    __shared__ f32x4 group_acc[8][32];
    const int64_t at = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, p = threadIdx.x;
    float top = kNoMax, sum = 0.f;
    if (p < parts.splits) {
        top = parts.stat[2 * (p * parts.rows + at)];
        sum = parts.stat[2 * (p * parts.rows + at) + 1];
    }
    float all = top;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) all = fmaxf(all, __shfl_xor(all, d));
    if (lane == 0) wave_top[wave] = all;
    __syncthreads();
    all = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    const float f = exp2_(top - all);
    if (p < parts.splits) factor[p] = f;
    sum *= f;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
    if (lane == 0) wave_sum[wave] = sum;
    __syncthreads();
    sum = (wave_sum[0] + wave_sum[1]) + (wave_sum[2] + wave_sum[3]);

    const int group = threadIdx.x >> 5, c = 4 * (threadIdx.x & 31);
    f32x4 acc = {};
    if (c < a.dim) {
#pragma unroll 4
        for (int s = group; s < parts.splits; s += 8) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(parts.out + (s * parts.rows + at) * a.dim + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = fmaf(x[e], factor[s], acc[e]);
        }
    }
    group_acc[group][threadIdx.x & 31] = acc;
    __syncthreads();
    if (group > 0) return;
    const int i = static_cast<int>(at % a.nq);
    const int64_t bh = at / a.nq;
    const int head = static_cast<int>(bh % a.heads);
    const int64_t b = bh / a.heads;
    if ((a.lse || a.lse_near) && threadIdx.x == 0)
        write_lse(a, at, sum == 0.f ? -INFINITY : (all + log2f(sum)) * kLn2, static_cast<int>(b), i, row_of(a, static_cast<int>(b), i), head);
    if (c >= a.dim) return;
#pragma unroll
    for (int g = 1; g < 8; ++g) acc += group_acc[g][threadIdx.x];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (sum == 0.f) acc = f32x4{};
    const float o[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    write_out<T>(a, b * a.so.batch + i * a.so.row + head * a.so.head + c, o);
}

template <typename T>
void launch(const ddpm_span_attention_args& a, const Plan& plan, void* workspace, hipStream_t stream) {
    const Dev d = dev_args(a);
    Parts parts = {};
    parts.splits = plan.splits;
    parts.rows = static_cast<int64_t>(a.batch) * a.heads * a.nq;
    parts.out = static_cast<float*>(workspace);
    parts.stat = parts.out + parts.splits * parts.rows * a.dim;
    const dim3 grid(plan.blocks * plan.splits, a.heads / plan.pack, a.batch);
    for_dim(a.dim, [&](auto dp) {
        if (plan.splits > 1)
            fwd_kernel<T, decltype(dp)::value, true><<<grid, kThreads, 0, stream>>>(d, plan.pack, parts);
        else
            fwd_kernel<T, decltype(dp)::value, false><<<grid, kThreads, 0, stream>>>(d, plan.pack, parts);
    });
    if (plan.splits > 1) join_kernel<T><<<static_cast<unsigned>(parts.rows), 256, 0, stream>>>(d, parts);
}

}  // namespace

extern "C" int64_t ddpm_span_attention_fwd_workspace(const ddpm_span_attention_args* a) {
    if (!a || !span::check_args(*a)) return ddpm::fail_invalid("span attention sizes, type or strides");
    if (a->batch == 0 || a->nq == 0) return 0;
    const Plan plan = plan_of(*a);       // a batch that takes several launches is not split
    return plan.splits == 1 ? 0 : static_cast<int64_t>(plan.splits) * a->batch * a->heads * a->nq * (a->dim + 2) * 4;
}

extern "C" int ddpm_span_attention_fwd(const ddpm_span_attention_args* a, void* workspace, void* stream) {
    DDPM_REQUIRE(a && span::check_args(*a));
    if (a->batch == 0 || a->nq == 0) return DDPM_OK;
    DDPM_REQUIRE(a->q && a->out && (a->nk == 0 || (a->k && a->v)));
    DDPM_REQUIRE(ddpm::aligned16(a->q) && ddpm::aligned16(a->k) && ddpm::aligned16(a->v) && ddpm::aligned16(a->out) && ddpm::aligned16(a->out_low));
    const Plan plan = plan_of(*a);
    DDPM_REQUIRE(plan.splits == 1 || (workspace && ddpm::aligned16(workspace)));
    for (int64_t first = 0; first < a->batch; first += span::kMaxBatch) {
        const ddpm_span_attention_args part = span::entries_from(*a, static_cast<int>(first));
        if (a->type == DDPM_F32)
            launch<float>(part, plan, workspace, as_stream(stream));
        else if (a->type == DDPM_BF16)
            launch<__bf16>(part, plan, workspace, as_stream(stream));
        else
            launch<_Float16>(part, plan, workspace, as_stream(stream));
    }
    return ddpm::check_launch("span attention forward");
}
