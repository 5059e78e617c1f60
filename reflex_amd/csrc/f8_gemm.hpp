// Products in 8-bit floating point (e4m3) with f32 scales, one for each 128 of an
// activation row and one for each 128 x 128 block of weights:
//   y[m][n] = sum_b sx[m][b] sw[n / 128][b] sum_{k in block b} x[m][k] w[n][k]
// The inner sum is 16 x 16 results of matrix instructions, started at zero; the outer sum
// is f32 multiply-adds, one for each result and block.
//
// Two ways to the inner sum:
//   half results  v_mfma_f32_16x16x128_f8f6f4, the whole block in one instruction of 32
//                 cycles. It adds the products in eights (8 neighbouring codes of a lane),
//                 cutting each to multiples of 2^-13 of the eight's largest
//                 (its power of two; measured: 2^-14 of 1 is lost beside it), and the eights in f32. A
//                 product of that size carries the roundings of its own codes, 2^-4 each,
//                 and the result is rounded to 2^-12 or 2^-9: 1.5e-5 of a result for
//                 normal values, under either.
//   f32 results   the codes are widened to f16, which holds all of them, and multiplied by
//                 v_mfma_f32_16x16x32_f16: products exact, sums f32, at half the rate.
// Kernels that memory bounds (few rows) use the second for all, and the exact entry points only it.
//
// Both operands lie in memory with K along their rows. Which of the 128 values a lane
// brings does not matter as long as both operands agree: a lane takes 16 bytes of
// the first 64 and 16 of the second.
#pragma once
#include "common.hpp"
#include "tiles.hpp"

typedef int v8i_t __attribute__((ext_vector_type(8)));
typedef u4_t u4a1_t __attribute__((aligned(1)));

struct F8Args {
    const uint8_t* x;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    void* y;
    const int32_t* offsets;  // grouped rows (rfxq_group_rows); NULL: all rows are one group's
    const int32_t* x_index;
    const int32_t* y_index;
    uint64_t ldx, ldxs, ldy, w_stride, ws_stride;
    uint32_t rows, x_rows, y_rows, x_div;
    uint32_t k, n, groups, y_type;  // y_type: 0 f32, 1 f16, 2 bf16
    uint32_t tiles_m, tiles_n, sm, sn;
    uint32_t first_m, first_n;  // the launch's first tile
};

constexpr uint32_t kBlock = 128;

// A lane's 32 codes of a 16 x 128 operand.
template <bool EXACT>
struct Operand {
    v8i_t v;
    __device__ __forceinline__ void take(u4_t a, u4_t b) {
        v = v8i_t{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
    }
};
template <>
struct Operand<true> {
    h8_t v[4];
    __device__ __forceinline__ void take(u4_t a, u4_t b) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) {
            const uint32_t c = i < 4u ? a[i] : b[i - 4u];
            const h2_t lo = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, false);
            const h2_t hi = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.0f, true);
            v[i >> 1][4 * (i & 1u)] = lo[0];
            v[i >> 1][4 * (i & 1u) + 1] = lo[1];
            v[i >> 1][4 * (i & 1u) + 2] = hi[0];
            v[i >> 1][4 * (i & 1u) + 3] = hi[1];
        }
    }
};

// one block's products of 16 x 16 results, from zero
RFXQ_DEV f4v_t multiply(const Operand<false>& a, const Operand<false>& b) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, f4v_t{0, 0, 0, 0}, 0, 0, 0, 0, 0, 0);
}
RFXQ_DEV f4v_t multiply(const Operand<true>& a, const Operand<true>& b) {
    f4v_t d = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[i], b.v[i], d, 0, 0, 0);
    return d;
}

// 16 codes at any byte
RFXQ_DEV u4_t ld_codes(const uint8_t* p) { return *(const RFXQ_GLOBAL u4a1_t*)p; }
// The last, partial block of a row of k >= 16 codes: 16 codes from `at` on are read from min(at, k - 16) on, so that no
// load has a condition (those are waited for one by one), and moved down by as many bytes, zeros behind
// them: by whole dwords, then by bytes.
RFXQ_DEV u4_t cut_codes(u4_t v, uint32_t by) {
    if (by & 8u) v = u4_t{v.z, v.w, 0, 0};
    if (by & 4u) v = u4_t{v.y, v.z, v.w, 0};
    const u4_t r = {alignbyte(v.y, v.x, by & 3u), alignbyte(v.z, v.y, by & 3u), alignbyte(v.w, v.z, by & 3u),
                    alignbyte(0, v.w, by & 3u)};
    return by < 16u ? r : u4_t{0, 0, 0, 0};
}
// A row of k < 16 codes: one by one.
RFXQ_DEV u4_t ld_short(const uint8_t* row, uint32_t k, uint32_t at) {
    u4_t r = {0, 0, 0, 0};
    const uint32_t have = at ? 0u : k;
#pragma unroll 1
    for (uint32_t i = 0; i < have; i++) {
        const uint32_t c = (uint32_t)((const RFXQ_GLOBAL uint8_t*)row)[i] << (8u * (i & 3u));
#pragma unroll
        for (uint32_t d = 0; d < 4u; d++) r[d] |= i >> 2 == d ? c : 0u;
    }
    return r;
}

// The tile of this workgroup; false: there is none.
RFXQ_DEV bool f8_place(const F8Args& a, uint32_t& tm, uint32_t& tn) {
    const bool there = tile_place(a, blockIdx.x, tm, tn);
    tm += a.first_m;
    tn += a.first_n;
    return there;
}
// The rows of a tile: a search among the groups, or counted.
template <bool GROUPED>
RFXQ_DEV RowTile f8_tile(const F8Args& a, uint32_t bm, uint32_t tm) {
    if constexpr (GROUPED) return find_tile(a.offsets, a.groups, a.rows, bm, tm);
    return {0, tm * bm, min(tm * bm + bm, a.rows), 0, true};
}
// Place p's row of x and of y; -1: there is none (it is not computed).
template <bool GROUPED>
RFXQ_DEV int64_t f8_src(const F8Args& a, uint32_t p) {
    if constexpr (GROUPED) return src_row(a, p);
    return (int64_t)p;
}
template <bool GROUPED>
RFXQ_DEV int64_t f8_dst(const F8Args& a, uint32_t p) {
    if constexpr (GROUPED) return dst_row(a, p);
    return (int64_t)p;
}

// 4 F neighbouring results of one row from column n on, each rounded once.
template <typename T, uint32_t F>
RFXQ_DEV void st_results(T* y, uint32_t have, const f4v_t (&v)[F]) {
    typedef T t4_t __attribute__((ext_vector_type(4)));
    typedef T t4a_t __attribute__((ext_vector_type(4), aligned(__alignof__(T))));
    if (have >= 4u * F) {
#pragma unroll
        for (uint32_t f = 0; f < F; f++) {
            t4_t r;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++) r[i] = (T)v[f][i];
            *(RFXQ_GLOBAL t4a_t*)(y + 4u * f) = r;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u * F; i++)
            if (i < have) ((RFXQ_GLOBAL T*)y)[i] = (T)v[i >> 2][i & 3u];
    }
}
template <uint32_t F>
RFXQ_DEV void f8_out(const F8Args& a, int64_t row, uint32_t n, const f4v_t (&v)[F]) {
    const uint32_t have = a.n > n ? a.n - n : 0u;
    const uint64_t at = (uint64_t)row * a.ldy + n;
    if (a.y_type == 0)
        st_results(static_cast<float*>(a.y) + at, have, v);
    else if (a.y_type == 1)
        st_results(static_cast<half_t*>(a.y) + at, have, v);
    else
        st_results(static_cast<__bf16*>(a.y) + at, have, v);
}

// ---------------------------------------------------------------- any alignment

// 32 MF x 32 NF tiles (in one block of columns: a scale of the weights' a step), operands through
// registers to one of two LDS buffers, a barrier a step, the loads of AHEAD steps in flight during the
// products. KG groups of four waves of 16 MF x 16 NF results take a block of K each of a step's KG,
// and add their parts in LDS. Rows and columns past the tile read others, whose results are not
// stored; the last, partial block has zeros behind the end of both operands, a block past it
// zeros and the scale 0. Bound by loads of 16 bytes at any byte (100 x K x 4099, f32: K = 4096 18 us, 4100 21, 4098
// 25, 4099 28): 333 x 1235 x 1531 f32 9.4 us in 32 x 64 tiles (264 of them), 1000 x 4099 x 4099 half
// results 83 us, 16 x 4099 x 14336 f32 24.5 us (2.4 TB/s). Two steps ahead pay for 64 x 128 tiles (333 x 4099 x
// 4099 half: 34 us, one 37), not for 32 x 64 (11.4, one 9.4). Tried: whole dwords and the fifth that a lane needs by a load
// of its own or from the next lane (10.5 and 11.1), four groups of waves (15).
template <uint32_t MF, uint32_t NF, uint32_t KG, uint32_t AHEAD, bool EXACT, bool GROUPED>
RFXQ_DEV void f8_any(const F8Args& a) {
    constexpr uint32_t BM = 32u * MF, BN = 32u * NF, ROWS = 32, NX = BM / ROWS, NW = BN / ROWS;
    __shared__ u4_t xs[2][KG][BM * 8u], ws[2][KG][BN * 8u];
    uint32_t tm, tn;
    if (!f8_place(a, tm, tn)) return;
    const RowTile t = f8_tile<GROUPED>(a, BM, tm);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), kg = wave >> 2;
    const uint32_t tid = threadIdx.x & 255u, lane = tid & 63u, l = lane & 15u, q = lane >> 4;
    const uint32_t n0 = tn * BN, c = tid & 7u, row0 = (wave >> 1 & 1u) * 16u * MF, col0 = (wave & 1u) * 16u * NF;
    const uint32_t full = a.k / kBlock, tail = a.k % kBlock, blocks = full + (tail ? 1u : 0u);
    const uint8_t* w = a.w + (uint64_t)t.group * a.w_stride;
    const float* sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)(n0 / kBlock) * blocks;
    const uint8_t *xp[NX], *wp[NW];
    const float* sx[MF];
#pragma unroll
    for (uint32_t i = 0; i < NX; i++) {
        const int64_t s = f8_src<GROUPED>(a, min(t.beg + (tid >> 3) + ROWS * i, t.end - 1u));
        xp[i] = a.x + (s < 0 ? 0 : (uint64_t)s * a.ldx);
    }
#pragma unroll
    for (uint32_t m = 0; m < MF; m++) {
        const int64_t s = f8_src<GROUPED>(a, min(t.beg + row0 + 16u * m + l, t.end - 1u));
        sx[m] = a.xs + (s < 0 ? 0 : (uint64_t)s * a.ldxs);
    }
#pragma unroll
    for (uint32_t i = 0; i < NW; i++)
        wp[i] = w + (uint64_t)min(n0 + col_of<NF>((tid >> 3) + ROWS * i), a.n - 1u) * a.k;
    f4v_t acc[MF][NF] = {};
    struct Block {
        u4_t x[NX], w[NW];
        float sx[MF], sw;
    } r[AHEAD];
    // no condition round loads: those under one are waited for at its end. Blocks past the last read its end.
    const auto load = [&](Block& to, uint32_t b) {
        const uint32_t k = min(b * kBlock + 16u * c, a.k - 16u), at = min(b, blocks - 1u);
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) to.w[i] = ld_codes(wp[i] + k);
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) to.x[i] = ld_codes(xp[i] + k);
        to.sw = ((const RFXQ_GLOBAL float*)sw)[at];
#pragma unroll
        for (uint32_t m = 0; m < MF; m++) to.sx[m] = ((const RFXQ_GLOBAL float*)sx[m])[at];
    };
    const auto step = [&](uint32_t b, Block& now, uint32_t buffer, auto more) {
        u4_t *xl = xs[buffer][kg], *wl = ws[buffer][kg];
        if (b + kg >= full) {  // a partial block, or one behind it
            const uint32_t k = (b + kg) * kBlock + 16u * c, by = k - min(k, a.k - 16u);
#pragma unroll
            for (uint32_t i = 0; i < NW; i++) now.w[i] = cut_codes(now.w[i], by);
#pragma unroll
            for (uint32_t i = 0; i < NX; i++) now.x[i] = cut_codes(now.x[i], by);
        }
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) xl[lds_piece((tid >> 3) + ROWS * i, c)] = now.x[i];
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) wl[lds_piece((tid >> 3) + ROWS * i, c)] = now.w[i];
        float scale[MF];
#pragma unroll
        for (uint32_t m = 0; m < MF; m++) scale[m] = b + kg < blocks ? now.sx[m] * now.sw : 0.0f;
        lds_barrier();
        if constexpr (decltype(more)::value) load(now, b + AHEAD * KG + kg);
        Operand<EXACT> wf[NF];
#pragma unroll
        for (uint32_t f = 0; f < NF; f++)
            wf[f].take(wl[lds_piece(col0 + 16u * f + l, q)], wl[lds_piece(col0 + 16u * f + l, 4u + q)]);
#pragma unroll
        for (uint32_t m = 0; m < MF; m++) {
            Operand<EXACT> xf;
            xf.take(xl[lds_piece(row0 + 16u * m + l, q)], xl[lds_piece(row0 + 16u * m + l, 4u + q)]);
            f4v_t d[NF];
#pragma unroll
            for (uint32_t f = 0; f < NF; f++) d[f] = multiply(wf[f], xf);
#pragma unroll
            for (uint32_t f = 0; f < NF; f++) acc[m][f] += d[f] * scale[m];
        }
    };
    if (a.k >= 16u) {
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; i++) load(r[i], KG * i + kg);
        for (uint32_t b = 0;; b += 2u * KG) {
            step(b, r[0], 0, Count<1>{});
            if (b + KG >= blocks) break;
            step(b + KG, r[AHEAD - 1u], 1, Count<1>{});
            if (b + 2u * KG >= blocks) break;
        }
    } else {
        const uint32_t k = kg * kBlock + 16u * c;
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) r[0].w[i] = ld_short(wp[i], a.k, k);
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) r[0].x[i] = ld_short(xp[i], a.k, k);
        r[0].sw = *(const RFXQ_GLOBAL float*)sw;
#pragma unroll
        for (uint32_t m = 0; m < MF; m++) r[0].sx[m] = *(const RFXQ_GLOBAL float*)sx[m];
        step(0, r[0], 0, Count<0>{});
    }
    if constexpr (KG > 1) {
        static_assert(KG == 2 && sizeof ws >= 4u * MF * NF * 64u * sizeof(f4v_t));
        __syncthreads();
        f4v_t* part = reinterpret_cast<f4v_t*>(ws) + (wave & 3u) * MF * NF * 64u + lane;
        if (kg) {
#pragma unroll
            for (uint32_t i = 0; i < MF * NF; i++) part[64u * i] = acc[i / NF][i % NF];
        }
        __syncthreads();
        if (kg) return;
#pragma unroll
        for (uint32_t i = 0; i < MF * NF; i++) acc[i / NF][i % NF] += part[64u * i];
    }
#pragma unroll
    for (uint32_t m = 0; m < MF; m++) {
        const uint32_t p = t.beg + row0 + 16u * m + l;
        if (p >= t.end) continue;
        const int64_t src = f8_src<GROUPED>(a, p), dst = f8_dst<GROUPED>(a, p);
        if (src >= 0 && dst >= 0) f8_out(a, dst, n0 + col0 + 4u * NF * q, acc[m]);
    }
}

#define RFXQ_F8_ANY(MF, NF, KG, AHEAD, WAVES, name, EXACT)                                                          \
    extern "C" __global__ __launch_bounds__(256 * KG, WAVES) void rfxq_f8_any##MF##_##KG##_##name(F8Args a) {       \
        f8_any<MF, NF, KG, AHEAD, EXACT, false>(a);                                                                 \
    }                                                                                                               \
    extern "C" __global__ __launch_bounds__(256 * KG, WAVES) void rfxq_f8_any##MF##_##KG##_##name##_grouped(F8Args a) { \
        f8_any<MF, NF, KG, AHEAD, EXACT, true>(a);                                                                  \
    }
RFXQ_F8_ANY(1, 2, 2, 1, 4, half, false)
RFXQ_F8_ANY(1, 2, 2, 1, 4, f32, true)
RFXQ_F8_ANY(2, 4, 1, 1, 3, half, false)
RFXQ_F8_ANY(2, 4, 2, 2, 2, half, false)
RFXQ_F8_ANY(2, 4, 2, 2, 2, f32, true)

// ---------------------------------------------------------------- few rows, any alignment

// 16 x 16 results a workgroup: both operands from memory straight into registers, a block
// of K in every 8th for each of its 8 waves, which add their parts in LDS. Two blocks are
// multiplied while the next two are on their way. A matrix instruction's operand has
// 16 rows' pieces side by side, which memory pipes take at 16 bytes a cycle (whole lines: 63):
// f8_few.hpp is for rows that start at 16 bytes. 1 x 4099 x 4099: 11.8 us (32 x 64 tiles: 22).
template <bool GROUPED>
RFXQ_DEV void f8_few(const F8Args& a) {
    constexpr uint32_t D = 2, WK = 8;
    __shared__ f4v_t part[WK][64];
    uint32_t tm, tn;
    if (!f8_place(a, tm, tn)) return;
    const RowTile t = f8_tile<GROUPED>(a, 16, tm);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4, n0 = tn * 16u;
    const uint32_t full = a.k / kBlock, tail = a.k % kBlock, blocks = full + (tail ? 1u : 0u);
    const float* sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)(n0 / kBlock) * blocks;
    // columns past the last read it again; their results are not stored
    const uint8_t* w = a.w + (uint64_t)t.group * a.w_stride + (uint64_t)min(n0 + l, a.n - 1u) * a.k;
    struct Block {
        u4_t w[2], x[2];
        float sx, sw;
    } s[2][D];
    const auto load_w = [&](Block& r, uint32_t b) {
        r.w[0] = ld_codes(w + (uint64_t)b * kBlock + 16u * q);
        r.w[1] = ld_codes(w + (uint64_t)b * kBlock + 64u + 16u * q);
        r.sw = ((const RFXQ_GLOBAL float*)sw)[b];
    };
#pragma unroll
    for (uint32_t i = 0; i < D; i++)  // on their way while the rows are looked up
        if (wave + WK * i < full) load_w(s[0][i], wave + WK * i);
    const int64_t src = f8_src<GROUPED>(a, min(t.beg + l, t.end - 1u));
    const uint8_t* x = a.x + (src < 0 ? 0 : (uint64_t)src * a.ldx);
    const float* sx = a.xs + (src < 0 ? 0 : (uint64_t)src * a.ldxs);
    const auto load_x = [&](Block& r, uint32_t b) {
        r.x[0] = ld_codes(x + (uint64_t)b * kBlock + 16u * q);
        r.x[1] = ld_codes(x + (uint64_t)b * kBlock + 64u + 16u * q);
        r.sx = ((const RFXQ_GLOBAL float*)sx)[b];
    };
    f4v_t acc = {0, 0, 0, 0};
    const auto products = [&](const Block& r) {
        Operand<true> wf, xf;
        wf.take(r.w[0], r.w[1]);
        xf.take(r.x[0], r.x[1]);
        acc += multiply(wf, xf) * (r.sx * r.sw);
    };
#pragma unroll
    for (uint32_t i = 0; i < D; i++)
        if (wave + WK * i < full) load_x(s[0][i], wave + WK * i);
    for (uint32_t b = wave; b < full; b += 2u * D * WK) {
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t at = b + D * WK * h;
#pragma unroll
            for (uint32_t i = 0; i < D; i++) {
                const uint32_t next = at + WK * (D + i);
                if (next < full) {
                    load_w(s[h ^ 1u][i], next);
                    load_x(s[h ^ 1u][i], next);
                }
            }
#pragma unroll
            for (uint32_t i = 0; i < D; i++)
                if (at + WK * i < full) products(s[h][i]);
        }
    }
    if (tail && wave == full % WK) {
        Block& r = s[0][0];
        const uint32_t k = full * kBlock + 16u * q;
        if (a.k >= 16u) {
            const uint32_t from[2] = {min(k, a.k - 16u), min(k + 64u, a.k - 16u)};
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                r.w[h] = ld_codes(w + from[h]);
                r.x[h] = ld_codes(x + from[h]);
            }
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                r.w[h] = cut_codes(r.w[h], k + 64u * h - from[h]);
                r.x[h] = cut_codes(r.x[h], k + 64u * h - from[h]);
            }
        } else {
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) {
                r.w[h] = ld_short(w, a.k, k + 64u * h);
                r.x[h] = ld_short(x, a.k, k + 64u * h);
            }
        }
        r.sw = sw[full];
        r.sx = sx[full];
        products(r);
    }
    part[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    f4v_t sum[1] = {part[0][lane]};
#pragma unroll
    for (uint32_t v = 1; v < WK; v++) sum[0] += part[v][lane];
    const uint32_t p = t.beg + l;
    if (p >= t.end || src < 0) return;
    const int64_t dst = f8_dst<GROUPED>(a, p);
    if (dst >= 0) f8_out(a, dst, n0 + 4u * q, sum);
}

extern "C" __global__ __launch_bounds__(512) void rfxq_f8_few(F8Args a) { f8_few<false>(a); }
extern "C" __global__ __launch_bounds__(512) void rfxq_f8_few_grouped(F8Args a) { f8_few<true>(a); }
