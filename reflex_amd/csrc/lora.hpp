// Low-rank adapters of many requests beside a projection that all rows share
// (rfxq_lora_add): for the rows r of group g
//   v = A_g x[r] (rank_g values),  out[r] = y[r] + scale_g B_g v
// and out[r] = y[r] for rows in no group. Two launches: rfxq_lora_down_*
// leaves v (f32) in the workspace, in ranges of K where rows are few, and
// rfxq_lora_up_* adds the ranges in order, so results do not change from call
// to call.
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
    uint32_t k_split, tiles, tiles_n, vec;  // vec: 1 rows of x, 2 of A, 4 of B start at whole 16 bytes
};

template <typename T>
RFXQ_DEV float to_f32(T v) { return (float)v; }

// 4 values at p, of which the first `have` are there: the others are 0.
template <typename T>
RFXQ_DEV f4v_t ld_four(const T* p, uint32_t have, bool vec) {
    typedef T t4_t __attribute__((ext_vector_type(4)));
    f4v_t r = {0, 0, 0, 0};
    if (vec && have >= 4u) {
        const t4_t t = *(const RFXQ_GLOBAL t4_t*)p;
#pragma unroll
        for (int i = 0; i < 4; i++) r[i] = (float)t[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            if (i < have) r[i] = (float)((const RFXQ_GLOBAL T*)p)[i];
    }
    return r;
}

RFXQ_DEV uint32_t lora_rank(const LoraArgs& a, uint32_t g) {
    if (g >= a.groups) return 0;
    if (!a.ranks) return a.rank;
    const int32_t r = a.ranks[g];
    return r < 0 ? 0u : (uint32_t)r < a.rank ? (uint32_t)r : a.rank;
}

RFXQ_DEV int64_t lora_row(const LoraArgs& a, uint32_t p) {
    const int32_t r = a.order ? a.order[p] : (int32_t)p;
    return r >= 0 && (uint32_t)r < a.x_rows ? (int64_t)r : -1;
}

constexpr uint32_t kLoraRows = 16, kLoraCols = 256;

// v: 16 rows of one group, one range of K; the workgroup's 4 waves take
// quarters of it and add them in LDS.
template <typename TX, typename TW>
RFXQ_DEV void lora_down(const LoraArgs& a) {
    __shared__ f4v_t part[3][4][64];
    const uint32_t split = blockIdx.x / a.tiles;
    const RowTile t = find_tile(a.offsets, a.groups, a.rows, kLoraRows, blockIdx.x % a.tiles);
    if (!t.any) return;
    const uint32_t rank = lora_rank(a, t.group), wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    const uint32_t l = lane & 15u, q = lane >> 4;
    const uint32_t p = t.beg + l;
    const int64_t row = p < t.end ? lora_row(a, p) : -1;
    const TX* x = static_cast<const TX*>(a.x) + (row < 0 ? 0 : (uint64_t)row * a.ldx);
    const uint32_t quarter = (a.k_split / 4u + 15u) & ~15u;
    const uint32_t k_end = min(a.k, (split + 1u) * a.k_split);
    const uint32_t k0 = split * a.k_split + wave * quarter, k1 = min(k_end, k0 + quarter);
    for (uint32_t r0 = 0; r0 < rank; r0 += 64u) {
        f4v_t acc[4] = {};
        const TW* w[4];
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++)
            w[f] = static_cast<const TW*>(a.a) + ((uint64_t)t.group * a.rank + min(r0 + 16u * f + l, a.rank - 1u)) * a.k;
        for (uint32_t k = k0 + 4u * q; k < k0 + quarter; k += 16u) {
            const uint32_t have = k < k1 ? k1 - k : 0u;
            const f4v_t xv = ld_four(x + k, row < 0 ? 0u : have, a.vec & 1u);
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) {
                if (r0 + 16u * f >= rank) break;
                const f4v_t wv = ld_four(w[f] + k, r0 + 16u * f + l < rank ? have : 0u, a.vec & 2u);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[j], xv[j], acc[f], 0, 0, 0);
            }
        }
        __syncthreads();
        if (wave) {
#pragma unroll
            for (int f = 0; f < 4; f++) part[wave - 1u][f][lane] = acc[f];
        }
        __syncthreads();
        if (wave == 0 && p < t.end) {
            float* v = a.v + ((uint64_t)split * a.rows + p) * a.ldv + r0 + 4u * q;
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) {
                if (r0 + 16u * f >= rank) break;
                const f4v_t s = ((acc[f] + part[0][f][lane]) + part[1][f][lane]) + part[2][f][lane];
                *(RFXQ_GLOBAL f4v_t*)(v + 16u * f) = s;  // rows rank.. of the last 16 are 0
            }
        }
    }
}

// out: 16 rows x 256 columns, a wave 64 columns.
template <typename TX, typename TW>
RFXQ_DEV void lora_up(const LoraArgs& a) {
    const uint32_t tn = blockIdx.x % a.tiles_n;
    RowTile t = find_tile(a.offsets, a.groups, a.rows, kLoraRows, blockIdx.x / a.tiles_n);
    if (!t.any) {  // rows in no group
        if (a.y == a.out) return;
        const int32_t o = a.offsets[a.groups];
        t.beg = (o < 0 ? 0u : (uint32_t)o) + t.beg * kLoraRows;
        if (t.beg >= a.rows) return;
        t.end = min(t.beg + kLoraRows, a.rows);
        t.group = a.groups;
    }
    const uint32_t rank = lora_rank(a, t.group), wave = threadIdx.x >> 6, lane = threadIdx.x & 63u;
    if (rank == 0 && a.y == a.out) return;
    const uint32_t l = lane & 15u, q = lane >> 4, p = t.beg + l, n0 = tn * kLoraCols + wave * 64u;
    const int64_t row = p < t.end ? lora_row(a, p) : -1;
    f4v_t acc[4] = {};
    const float* v = a.v + (uint64_t)min(p, t.end - 1u) * a.ldv;
    const TW* w[4];
    uint32_t cols = 0;
#pragma unroll
    for (uint32_t f = 0; f < 4u; f++) {
        const uint32_t n = n0 + (l >> 2) * 16u + 4u * f + (l & 3u);
        cols |= n < a.n ? 1u << f : 0u;
        w[f] = static_cast<const TW*>(a.b) + ((uint64_t)min(t.group, a.groups - 1u) * a.n + min(n, a.n - 1u)) * a.rank;
    }
    for (uint32_t r = 4u * q; r < ((rank + 15u) & ~15u); r += 16u) {
        f4v_t vv = {0, 0, 0, 0};
        for (uint32_t s = 0; s < a.splits; s++) vv += *(const RFXQ_GLOBAL f4v_t*)(v + (uint64_t)s * a.rows * a.ldv + r);
        const uint32_t have = r < rank ? rank - r : 0u;
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++) {
            const f4v_t wv = ld_four(w[f] + r, cols >> f & 1u ? have : 0u, a.vec & 4u);
#pragma unroll
            for (int j = 0; j < 4; j++) acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[j], vv[j], acc[f], 0, 0, 0);
        }
    }
    if (row < 0) return;
    const float scale = t.group < a.groups && a.scales ? a.scales[t.group] : 1.0f;
    const TX* y = static_cast<const TX*>(a.y) + (uint64_t)row * a.ldy;
    TX* o = static_cast<TX*>(a.out) + (uint64_t)row * a.ldo;
#pragma unroll
    for (uint32_t f = 0; f < 4u; f++)
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t n = n0 + 16u * q + 4u * f + i;
            if (n < a.n) o[n] = rank ? (TX)((float)y[n] + scale * acc[f][i]) : y[n];
        }
}

#define RFXQ_LORA(name, TX, TW)                                                                                    \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_down_##name(LoraArgs a) { lora_down<TX, TW>(a); } \
    extern "C" __global__ __launch_bounds__(256) void rfxq_lora_up_##name(LoraArgs a) { lora_up<TX, TW>(a); }
RFXQ_LORA(f32_f32, float, float)
RFXQ_LORA(f32_f16, float, half_t)
RFXQ_LORA(f32_bf16, float, __bf16)
RFXQ_LORA(f16_f16, half_t, half_t)
RFXQ_LORA(bf16_bf16, __bf16, __bf16)
