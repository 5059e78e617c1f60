// Low-rank adapters of many requests beside a projection that all rows share
// (rfxq_lora_add): for the rows r of group g
//   v = A_g x[r] (rank_g values),  out[r] = y[r] + scale_g B_g v
// and out[r] = y[r] for rows in no group. Two launches: rfxq_lora_down_*
// leaves v (f32) in the workspace, in ranges of K where rows are few, and
// rfxq_lora_up_* adds the ranges in order, so results do not change from call
// to call.
//
// Both read their operands straight into the matrix instructions' registers:
// lane (l, q) of a wave holds 8 neighbouring values of row l, from 8 q on, of a
// 32-wide step (the order within a step is free, as long as both operands keep
// it). Activations and adapters of one half type multiply exactly. f32 values (x,
// and v always) beside half-typed adapters are split for each step into pieces of
// the adapters' type, scaled by a power of two per row and step so that the row's
// largest lies in [2^14, 2^15): 2 pieces of f16 (2^-22 of a value, 2^-39 of the
// largest for values below 2^-17 of it), 3 of bf16 (exact; for bf16 results too: where y
// and the adapter cancel, what 2 of them lose, 2^-15 of v, is more than the result's
// rounding). f32 matrix instructions take 256 cycles for what 2 or 3 half-typed ones
// and four multiply-adds take about 50 for; they are left for f32 adapters.
#pragma once
#include "common.hpp"
#include "grouped.hpp"
#include "rows.hpp"

struct LoraArgs {
    const void* x;
    const void* a;  // [groups][rank][k]
    const void* b;  // [groups][n][rank]
    const int32_t* ranks;
    const float* scales;
    const int32_t* offsets;
    const int32_t* order;
    const void* y;
    void* out;
    float* v;  // [splits][rows][ldv]
    uint64_t ldx, ldy, ldo;
    uint32_t rows, x_rows, k, n;
    uint32_t rank, ldv, groups, splits;
    uint32_t k_split, tiles, across, pad;
};

// 4 neighbouring values of a row as they lie in memory, at any element.
template <typename T>
struct FourOf {
    typedef T type __attribute__((ext_vector_type(4)));
    typedef T any __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};
template <typename T>
using Four = typename FourOf<T>::type;

template <typename T>
RFXQ_DEV Four<T> ld_four(const T* p) {
    return *(const RFXQ_GLOBAL typename FourOf<T>::any*)p;
}
template <typename T>
RFXQ_DEV Four<T> ld_four(const T* p, uint32_t have) {
    if (have >= 4u) return ld_four(p);
    Four<T> r = {};
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++)
        if (i < have) r[i] = ((const RFXQ_GLOBAL T*)p)[i];
    return r;
}
template <typename T>
RFXQ_DEV void st_four(T* p, uint32_t have, f4v_t v) {
    const Four<T> r = __builtin_convertvector(v, Four<T>);
    if (have >= 4u) {
        *(RFXQ_GLOBAL typename FourOf<T>::any*)p = r;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            if (i < have) ((RFXQ_GLOBAL T*)p)[i] = r[i];
    }
}

// The first `have` of 8 values, then zeros.
template <typename T>
RFXQ_DEV Eight<T> first_of(Eight<T> r, uint32_t have) {
    if constexpr (__is_same(T, float)) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) r.v[i >> 2][i & 3u] = i < have ? r.v[i >> 2][i & 3u] : 0.0f;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) r.v[i] &= have > 2u * i + 1u ? 0xFFFFFFFFu : have > 2u * i ? 0xFFFFu : 0u;
    }
    return r;
}

// the rank of a tile's group (`extra` of find_tile: its value of ranks)
RFXQ_DEV uint32_t lora_rank(const LoraArgs& a, const RowTile& t) {
    if (!t.any) return 0;
    return a.ranks ? min((uint32_t)max(t.extra, 0), a.rank) : a.rank;
}

// Place p's row; a load without a condition (without an order it reads the first offset).
RFXQ_DEV int64_t lora_row(const LoraArgs& a, uint32_t p) {
    const int32_t i = ((const RFXQ_GLOBAL int32_t*)(a.order ? a.order : a.offsets))[a.order ? p : 0u];
    const int32_t r = a.order ? i : (int32_t)p;
    return r >= 0 && (uint32_t)r < a.x_rows ? (int64_t)r : -1;
}

// The state of a workgroup of rfxq_lora_down_*, and its passes over up to 64 rows of A.
template <typename TX, typename TW, uint32_t MT>
struct LoraDown {
    int64_t row[MT];  // -1: a place without a row
    RowTile t;
    uint32_t rank, split, wave, lane, k0, k1;

    // RT 16-row operands from row r0 of A. The number is known at compile time: the
    // products of a step and what reads them stay free of branches (mfma_settle).
    template <uint32_t RT>
    __device__ __forceinline__ void pass(const LoraArgs& a, uint32_t r0, f4v_t (*part)[MT][4][64]) const {
        const uint32_t l = lane & 15u, q = lane >> 4;
        f4v_t acc[MT][RT] = {};
        const TW* w[RT];
#pragma unroll
        for (uint32_t f = 0; f < RT; f++) {
            // rows past the rank read the last one; their results are dropped below
            w[f] = static_cast<const TW*>(a.a) + ((uint64_t)t.group * a.rank + min(r0 + 16u * f + l, rank - 1u)) * a.k + 8u * q;
        }
        k_range<TX, TW, MT, RT>(
            w,
            [&](const TX*(&x)[MT]) {
#pragma unroll
                for (uint32_t m = 0; m < MT; m++)  // places without a row read the first one: what comes of it is not used
                    x[m] = static_cast<const TX*>(a.x) + (row[m] < 0 ? 0 : (uint64_t)row[m] * a.ldx) + 8u * q;
            },
            k0, k1, acc);
        __syncthreads();
        if (wave) {
#pragma unroll
            for (uint32_t m = 0; m < MT; m++)
#pragma unroll
                for (uint32_t f = 0; f < RT; f++) part[wave - 1u][m][f][lane] = acc[m][f];
        }
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (uint32_t m = 0; m < MT; m++) {
                const uint32_t p = t.beg + 16u * m + l;
                if (p >= t.end) break;
                float* v = a.v + ((uint64_t)split * a.rows + p) * a.ldv + r0 + 4u * q;
#pragma unroll
                for (uint32_t f = 0; f < RT; f++) {
                    if (r0 + 16u * f >= rank) break;
                    f4v_t s = ((acc[m][f] + part[0][m][f][lane]) + part[1][m][f][lane]) + part[2][m][f][lane];
#pragma unroll
                    for (uint32_t i = 0; i < 4u; i++)
                        if (r0 + 16u * f + 4u * q + i >= rank) s[i] = 0.0f;
                    *(RFXQ_GLOBAL f4v_t*)(v + 16u * f) = s;
                }
            }
        }
    }
};

// v: 16 MT rows of one group, one range of K; the workgroup's 4 waves take
// quarters of it (whole steps of 64) and add them in LDS. x bounds it where rows are many
// (4096 rows of 4096 f32 values, ranks to 64: 19.8 us, 3.4 TB/s), A where they are few (256
// rows, 64 adapters, bf16: 9.5 us).
template <typename TX, typename TW, uint32_t MT>
RFXQ_DEV void lora_down(const LoraArgs& a) {
    __shared__ f4v_t part[3][MT][4][64];
    LoraDown<TX, TW, MT> d;
    d.split = blockIdx.x / a.tiles;
    d.t = find_tile(a.offsets, a.groups, a.rows, 16u * MT, blockIdx.x % a.tiles, a.ranks);
    if (!d.t.any) return;
    d.rank = lora_rank(a, d.t);
    d.lane = threadIdx.x & 63u;
    d.wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
#pragma unroll
    for (uint32_t m = 0; m < MT; m++) {
        const uint32_t p = d.t.beg + 16u * m + (d.lane & 15u);
        const int64_t found = lora_row(a, min(p, d.t.end - 1u));
        d.row[m] = p < d.t.end ? found : -1;
    }
    const uint32_t quarter = (a.k_split / 4u + 63u) & ~63u;
    const uint32_t end = min(a.k, (d.split + 1u) * a.k_split);
    d.k0 = min(d.split * a.k_split + d.wave * quarter, end);
    d.k1 = min(d.k0 + quarter, end);
    for (uint32_t r0 = 0; r0 < d.rank; r0 += 64u) {
        const uint32_t left = d.rank - r0;
        if (left <= 16u)
            d.template pass<1>(a, r0, part);
        else if (left <= 32u)
            d.template pass<2>(a, r0, part);
        else
            d.template pass<4>(a, r0, part);
    }
}

// out: 16 MT rows, strips of 16 NF columns: a.across workgroups share a tile's strips,
// a wave takes every (4 across)th. v, added up and in pieces, lies in LDS for
// all of them; B's values and y of the next strip are loaded during a strip.
//
// y, out and B bound it: 4096 rows of 4096 f32 values 32 us, 4.6 TB/s; 256 rows, 64
// adapters of ranks to 64, 14336 values, bf16: 28 us, 4.5 TB/s of whole lines of B and y
// (939 of 940 thousand requests are of 128 bytes).
//
// VEC: rank is a multiple of 8 and n of 4. Then no load has a condition: what does not
// exist reads the row's first values and is left out where it is used, so loads
// stay in flight until then. (Loads under a condition are waited for at its end.)
//
// LDS: f32 adapters: v [16 MT][ldv + 4]. Others: the pieces [NP][16 MT][ldl + 8]
// (halves, ldl = rank in whole steps of 32), then 2^e [16 MT][ldl / 32].
template <typename TX, typename TW, uint32_t MT, uint32_t NF, bool VEC>
RFXQ_DEV void lora_up(const LoraArgs& a) {
    constexpr bool F32 = __is_same(TW, float);
    constexpr uint32_t BM = 16u * MT, NP = __is_same(TW, __bf16) ? 3u : 2u;
    extern __shared__ uint32_t lds[];
    RowTile t = find_tile(a.offsets, a.groups, a.rows, BM, blockIdx.x / a.across, a.ranks);
    if (!t.any) {  // rows in no group
        if (a.y == a.out) return;
        const int32_t o = a.offsets[a.groups];
        t.beg = (o < 0 ? 0u : (uint32_t)o) + t.beg * BM;
        if (t.beg >= a.rows) return;
        t.end = min(t.beg + BM, a.rows);
        t.group = a.groups;
    }
    const uint32_t rank = lora_rank(a, t), lane = threadIdx.x & 63u;
    if (rank == 0 && a.y == a.out) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t l = lane & 15u, q = lane >> 4, strips = (a.n + 16u * NF - 1u) / (16u * NF);
    const uint32_t group = min(t.group, a.groups - 1u);
    const uint32_t steps = (rank + 31u) / 32u, ldl = (a.rank + 31u) & ~31u;
    struct Strip {
        Eight<TW> w[2][NF];  // the first 64 of the rank
        Four<TX> y[MT][NF];
    };
    const TW* matrix = static_cast<const TW*>(a.b) + (uint64_t)group * a.n * a.rank;
    const auto load_w = [&](Eight<TW>(&w)[NF], uint32_t n0, uint32_t r) {
        const uint32_t at = r + 8u * q;
#pragma unroll
        for (uint32_t f = 0; f < NF; f++) {
            const TW* row = matrix + (uint64_t)min(n0 + 16u * f + l, a.n - 1u) * a.rank;
            if constexpr (VEC)
                w[f] = ld_eight(row + (at < rank ? at : 0u));
            else
                w[f] = ld_eight(row + at, rank > at ? rank - at : 0u);
        }
    };
    const auto load_ws = [&](Strip& s, uint32_t n0) {
        if (rank) load_w(s.w[0], n0, 0);
        if (rank > 32u) load_w(s.w[1], n0, 32u);
    };
    const uint32_t first = (blockIdx.x % a.across) * 4u + wave, by = 4u * a.across;
    Strip s[2];
    if (first < strips) load_ws(s[0], 16u * NF * first);  // on their way while the rows are looked up
    const TX* y[MT];
    TX* o[MT];
    bool there[MT];
#pragma unroll
    for (uint32_t m = 0; m < MT; m++) {
        const uint32_t p = t.beg + 16u * m + l;
        const int64_t found = lora_row(a, min(p, t.end - 1u)), row = p < t.end ? found : -1;
        there[m] = row >= 0;
        y[m] = static_cast<const TX*>(a.y) + (row < 0 ? 0 : (uint64_t)row * a.ldy);
        o[m] = static_cast<TX*>(a.out) + (row < 0 ? 0 : (uint64_t)row * a.ldo);
    }
    const auto load_ys = [&](Strip& s, uint32_t n0) {
#pragma unroll
        for (uint32_t m = 0; m < MT; m++)
#pragma unroll
            for (uint32_t f = 0; f < NF; f++) {
                const uint32_t n = n0 + 16u * f + 4u * q;
                if constexpr (VEC)
                    s.y[m][f] = ld_four(y[m] + (n < a.n ? n : 0u));
                else
                    s.y[m][f] = ld_four(y[m] + n, n >= a.n ? 0u : a.n - n);
            }
    };
    const auto load = [&](Strip& s, uint32_t n0) {
        load_ws(s, n0);
        load_ys(s, n0);
    };
    if (first < strips) load_ys(s[0], 16u * NF * first);

    // v into LDS: a lane's 8 values of a row and step, the ranges of K added in
    // order; v is written, with zeros, up to the next whole 16
    for (uint32_t j = wave; j < MT * steps; j += 4u) {
        const uint32_t m = j % MT, r = 32u * (j / MT) + 8u * q, p = t.beg + 16u * m + l;
        Eight<float> sum = {};
        if (p < t.end && r < rank) {
            const float* v = a.v + (uint64_t)p * a.ldv + r;
#pragma unroll 4
            for (uint32_t i = 0; i < a.splits; i++) {
                const float* vs = v + (uint64_t)i * a.rows * a.ldv;
                sum.v[0] += *(const RFXQ_GLOBAL f4v_t*)vs;
                sum.v[1] += *(const RFXQ_GLOBAL f4v_t*)(vs + 4);
            }
        }
        if constexpr (F32) {
            f4v_t* to = reinterpret_cast<f4v_t*>(lds + (16u * m + l) * (ldl + 4u) + r);
            to[0] = sum.v[0];
            to[1] = sum.v[1];
        } else {
            const uint32_t top = top_over_q(top_of_eight(sum));
            const StepScale step = step_scale(top);
            u4_t out[NP];
            split_eight<TW, NP>(sum, step.up, top, out);
#pragma unroll
            for (uint32_t n = 0; n < NP; n++)
                *reinterpret_cast<u4_t*>(reinterpret_cast<uint16_t*>(lds) + (n * BM + 16u * m + l) * (ldl + 8u) + r) = out[n];
            if (q == 0)
                reinterpret_cast<float*>(lds + NP * BM * (ldl + 8u) / 2u)[(16u * m + l) * (ldl / 32u) + j / MT] = step.back;
        }
    }
    __syncthreads();
    const float scale = t.group < a.groups && a.scales ? a.scales[t.group] : 1.0f;

    const auto multiply = [&](const Eight<TW>(&loaded)[NF], uint32_t step, f4v_t(&acc)[MT][NF]) {
        Eight<TW> w[NF];
#pragma unroll
        for (uint32_t f = 0; f < NF; f++) w[f] = loaded[f];
        if (VEC && 32u * (step + 1u) > rank) {
            const uint32_t at = 32u * step + 8u * q;
#pragma unroll
            for (uint32_t f = 0; f < NF; f++) w[f] = first_of(loaded[f], rank > at ? rank - at : 0u);
        }
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) {
            if constexpr (F32) {
                Eight<float> v;
                const f4v_t* at = reinterpret_cast<const f4v_t*>(lds + (16u * m + l) * (ldl + 4u) + 32u * step + 8u * q);
                v.v[0] = at[0];
                v.v[1] = at[1];
#pragma unroll
                for (uint32_t f = 0; f < NF; f++)
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++)
                        acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[f].at(j), v.at(j), acc[m][f], 0, 0, 0);
            } else {
                u4_t v[NP];
#pragma unroll
                for (uint32_t n = 0; n < NP; n++)
                    v[n] = *reinterpret_cast<const u4_t*>(reinterpret_cast<const uint16_t*>(lds) +
                                                          (n * BM + 16u * m + l) * (ldl + 8u) + 32u * step + 8u * q);
                const float back = reinterpret_cast<const float*>(lds + NP * BM * (ldl + 8u) / 2u)[(16u * m + l) * (ldl / 32u) + step];
#pragma unroll
                for (uint32_t f = 0; f < NF; f++) {
                    f4v_t d = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t n = 0; n < NP; n++) d = mfma32<TW>(w[f].v, v[NP - 1u - n], d);
                    acc[m][f] += d * back;
                }
            }
        }
    };
    const auto finish = [&](const Strip& s, uint32_t n0) {
        f4v_t acc[MT][NF] = {};
        if (rank) multiply(s.w[0], 0, acc);
        if (rank > 32u) multiply(s.w[1], 1, acc);
        for (uint32_t step = 2; step < steps; step++) {
            Eight<TW> w[NF];
            load_w(w, n0, 32u * step);
            multiply(w, step, acc);
        }
        if constexpr (F32) mfma_settle();
#pragma unroll
        for (uint32_t m = 0; m < MT; m++)
#pragma unroll
            for (uint32_t f = 0; f < NF; f++) {
                const uint32_t n = n0 + 16u * f + 4u * q;
                f4v_t r = __builtin_convertvector(s.y[m][f], f4v_t);
                if (rank) r += scale * acc[m][f];
                if constexpr (VEC) {
                    if (there[m] && n < a.n) st_four(o[m] + n, 4u, r);
                } else {
                    st_four(o[m] + n, !there[m] || n >= a.n ? 0u : a.n - n, r);
                }
            }
    };
    for (uint32_t i = first; i < strips; i += 2u * by) {
        if (i + by < strips) load(s[1], 16u * NF * (i + by));
        finish(s[0], 16u * NF * i);
        if (i + by >= strips) break;
        if (i + 2u * by < strips) load(s[0], 16u * NF * (i + 2u * by));
        finish(s[1], 16u * NF * (i + by));
    }
}

#define RFXQ_LORA(name, TX, TW)                                                                                            \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_down_##name(LoraArgs a) { lora_down<TX, TW, 1>(a); }      \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_down_##name##_32(LoraArgs a) { lora_down<TX, TW, 2>(a); } \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_up_##name(LoraArgs a) { lora_up<TX, TW, 1, 2, true>(a); } \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_up_##name##_32(LoraArgs a) {                             \
        lora_up<TX, TW, 2, 2, true>(a);                                                                                    \
    }                                                                                                                      \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_up_##name##_any(LoraArgs a) { lora_up<TX, TW, 1, 2, false>(a); }
RFXQ_LORA(f32_f32, float, float)
RFXQ_LORA(f32_f16, float, half_t)
RFXQ_LORA(f32_bf16, float, __bf16)
RFXQ_LORA(f16_f16, half_t, half_t)
RFXQ_LORA(bf16_bf16, __bf16, __bf16)
