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
// Kernels that memory bounds (few rows) use the second for all.
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
// the first `have` of them, one by one, then zeros
RFXQ_DEV u4_t ld_codes(const uint8_t* p, uint32_t have) {
    if (have >= 16u) return ld_codes(p);
    u4_t r = {0, 0, 0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 16u; i++)
        if (i < have) r[i >> 2] |= (uint32_t)((const RFXQ_GLOBAL uint8_t*)p)[i] << (8u * (i & 3u));
    return r;
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

// 64 x 128 tiles (one block of weights' scales a step), 4 waves of 32 x 64, operands
// through registers to LDS, the next block's loads in flight during the products. Rows and
// columns past the tile read others, whose results are not stored; the last,
// partial block is loaded byte by byte with zeros behind the end of both operands.
template <bool EXACT, bool GROUPED>
RFXQ_DEV void f8_any(const F8Args& a) {
    constexpr uint32_t BM = 64, BN = 128, NX = BM * 8u / 256u, NW = BN * 8u / 256u;
    __shared__ u4_t xs[BM * 8u], ws[BN * 8u];
    uint32_t tm, tn;
    if (!tile_place(a, blockIdx.x, tm, tn)) return;
    const RowTile t = f8_tile<GROUPED>(a, BM, tm);
    if (!t.any) return;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63u, l = lane & 15u, q = lane >> 4;
    const uint32_t n0 = tn * BN, c = tid & 7u, row0 = (wave >> 1) * 32u, col0 = (wave & 1u) * 64u;
    const uint32_t full = a.k / kBlock, tail = a.k % kBlock, blocks = full + (tail ? 1u : 0u);
    const uint8_t* w = a.w + (uint64_t)t.group * a.w_stride;
    const float* sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)tn * blocks;
    const uint8_t *xp[NX], *wp[NW];
    const float* sx[2];
#pragma unroll
    for (uint32_t i = 0; i < NX; i++) {
        const int64_t s = f8_src<GROUPED>(a, min(t.beg + (tid >> 3) + 32u * i, t.end - 1u));
        xp[i] = a.x + (s < 0 ? 0 : (uint64_t)s * a.ldx) + 16u * c;
    }
#pragma unroll
    for (uint32_t m = 0; m < 2u; m++) {
        const int64_t s = f8_src<GROUPED>(a, min(t.beg + row0 + 16u * m + l, t.end - 1u));
        sx[m] = a.xs + (s < 0 ? 0 : (uint64_t)s * a.ldxs);
    }
#pragma unroll
    for (uint32_t i = 0; i < NW; i++)
        wp[i] = w + (uint64_t)min(n0 + col_of((tid >> 3) + 32u * i), a.n - 1u) * a.k + 16u * c;
    f4v_t acc[2][4] = {};
    u4_t xv[NX], wv[NW];
    float xsc[2], wsc;
    const auto load = [&](uint32_t b) {
        const uint32_t k = b * kBlock;
        if (b < full) {
#pragma unroll
            for (uint32_t i = 0; i < NW; i++) wv[i] = ld_codes(wp[i] + k);
#pragma unroll
            for (uint32_t i = 0; i < NX; i++) xv[i] = ld_codes(xp[i] + k);
        } else if (b < blocks) {
            const uint32_t have = tail > 16u * c ? tail - 16u * c : 0u;
#pragma unroll
            for (uint32_t i = 0; i < NW; i++) wv[i] = ld_codes(wp[i] + k, have);
#pragma unroll
            for (uint32_t i = 0; i < NX; i++) xv[i] = ld_codes(xp[i] + k, have);
        }
        const uint32_t at = min(b, blocks - 1u);
        wsc = ((const RFXQ_GLOBAL float*)sw)[at];
#pragma unroll
        for (uint32_t m = 0; m < 2u; m++) xsc[m] = ((const RFXQ_GLOBAL float*)sx[m])[at];
    };
    load(0);
    for (uint32_t b = 0; b < blocks; b++) {
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) xs[lds_piece((tid >> 3) + 32u * i, c)] = xv[i];
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) ws[lds_piece((tid >> 3) + 32u * i, c)] = wv[i];
        __syncthreads();
        float scale[2];
#pragma unroll
        for (uint32_t m = 0; m < 2u; m++) scale[m] = xsc[m] * wsc;
        load(b + 1u);
        Operand<EXACT> wf[4];
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++)
            wf[f].take(ws[lds_piece(col0 + 16u * f + l, q)], ws[lds_piece(col0 + 16u * f + l, 4u + q)]);
#pragma unroll
        for (uint32_t m = 0; m < 2u; m++) {
            Operand<EXACT> xf;
            xf.take(xs[lds_piece(row0 + 16u * m + l, q)], xs[lds_piece(row0 + 16u * m + l, 4u + q)]);
            f4v_t d[4];
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) d[f] = multiply(wf[f], xf);
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) acc[m][f] += d[f] * scale[m];
        }
    }
#pragma unroll
    for (uint32_t m = 0; m < 2u; m++) {
        const uint32_t p = t.beg + row0 + 16u * m + l;
        if (p >= t.end) continue;
        const int64_t src = f8_src<GROUPED>(a, p), dst = f8_dst<GROUPED>(a, p);
        if (src >= 0 && dst >= 0) f8_out(a, dst, n0 + col0 + 16u * q, acc[m]);
    }
}

#define RFXQ_F8_ANY(name, EXACT)                                                                                            \
    extern "C" __global__ __launch_bounds__(256, 3) void rfxq_f8_any_##name(F8Args a) { f8_any<EXACT, false>(a); }          \
    extern "C" __global__ __launch_bounds__(256, 3) void rfxq_f8_any_##name##_grouped(F8Args a) { f8_any<EXACT, true>(a); }
RFXQ_F8_ANY(half, false)
RFXQ_F8_ANY(f32, true)

// ---------------------------------------------------------------- few rows

// Up to 16 MT rows of a tile: what the weights weigh is all that counts, so they go
// from memory straight into registers, each once, as the matrix instructions' 16-row
// operands. A workgroup's WK waves take every WKth block of K each (neighbouring
// blocks are on their way together) for all of its 16 MT x 16 NT results and add
// their parts in LDS. Two blocks are multiplied while the next two are on their way.
template <uint32_t MT, uint32_t NT, uint32_t WK, bool GROUPED>
RFXQ_DEV void f8_few(const F8Args& a) {
    constexpr uint32_t D = 2;
    __shared__ f4v_t part[WK][MT * NT][64];
    uint32_t tm, tn;
    if (!tile_place(a, blockIdx.x, tm, tn)) return;
    const RowTile t = f8_tile<GROUPED>(a, 16u * MT, tm);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4, n0 = tn * 16u * NT;
    const uint32_t full = a.k / kBlock, tail = a.k % kBlock, blocks = full + (tail ? 1u : 0u);
    const float* sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)(n0 / kBlock) * blocks;
    const uint8_t *w[NT], *x[MT];
    const float* sx[MT];
#pragma unroll
    for (uint32_t f = 0; f < NT; f++)  // columns past the last read it again; their results are not stored
        w[f] = a.w + (uint64_t)t.group * a.w_stride + (uint64_t)min(n0 + 16u * f + l, a.n - 1u) * a.k + 16u * q;
    struct Block {
        u4_t w[NT][2], x[MT][2];
        float sx[MT], sw;
    } s[2][D];
    const auto load_w = [&](Block& r, uint32_t b) {
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) {
            r.w[f][0] = ld_codes(w[f] + (uint64_t)b * kBlock);
            r.w[f][1] = ld_codes(w[f] + (uint64_t)b * kBlock + 64u);
        }
        r.sw = ((const RFXQ_GLOBAL float*)sw)[b];
    };
    const auto load_x = [&](Block& r, uint32_t b) {
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) {
            r.x[m][0] = ld_codes(x[m] + (uint64_t)b * kBlock);
            r.x[m][1] = ld_codes(x[m] + (uint64_t)b * kBlock + 64u);
            r.sx[m] = ((const RFXQ_GLOBAL float*)sx[m])[b];
        }
    };
    f4v_t acc[MT][NT] = {};
    const auto products = [&](const Block& r) {
        Operand<true> wf[NT];
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) wf[f].take(r.w[f][0], r.w[f][1]);
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) {
            Operand<true> xf;
            xf.take(r.x[m][0], r.x[m][1]);
            const float scale = r.sx[m] * r.sw;
            f4v_t d[NT];
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) d[f] = multiply(wf[f], xf);
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) acc[m][f] += d[f] * scale;
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < D; i++)  // on their way while the rows are looked up
        if (wave + WK * i < full) load_w(s[0][i], wave + WK * i);
#pragma unroll
    for (uint32_t m = 0; m < MT; m++) {
        const int64_t src = f8_src<GROUPED>(a, min(t.beg + 16u * m + l, t.end - 1u));
        x[m] = a.x + (src < 0 ? 0 : (uint64_t)src * a.ldx) + 16u * q;
        sx[m] = a.xs + (src < 0 ? 0 : (uint64_t)src * a.ldxs);
    }
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
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t k = 64u * h + 16u * q, have = tail > k ? tail - k : 0u;
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) r.w[f][h] = ld_codes(w[f] + (uint64_t)full * kBlock + 64u * h, have);
#pragma unroll
            for (uint32_t m = 0; m < MT; m++) r.x[m][h] = ld_codes(x[m] + (uint64_t)full * kBlock + 64u * h, have);
        }
        r.sw = sw[full];
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) r.sx[m] = sx[m][full];
        products(r);
    }
#pragma unroll
    for (uint32_t m = 0; m < MT; m++)
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) part[wave][m * NT + f][lane] = acc[m][f];
    __syncthreads();
    for (uint32_t i = wave; i < MT * NT; i += WK) {
        f4v_t sum[1] = {part[0][i][lane]};
#pragma unroll
        for (uint32_t v = 1; v < WK; v++) sum[0] += part[v][i][lane];
        const uint32_t p = t.beg + 16u * (i / NT) + l;
        if (p >= t.end) continue;
        const int64_t src = f8_src<GROUPED>(a, p), dst = f8_dst<GROUPED>(a, p);
        if (src >= 0 && dst >= 0) f8_out(a, dst, n0 + 16u * (i % NT) + 4u * q, sum);
    }
}

#define RFXQ_F8_FEW(MT, NT, WK)                                                                                             \
    extern "C" __global__ __launch_bounds__(64 * WK) void rfxq_f8_few_##MT##_##NT##_##WK(F8Args a) {                        \
        f8_few<MT, NT, WK, false>(a);                                                                                       \
    }                                                                                                                       \
    extern "C" __global__ __launch_bounds__(64 * WK) void rfxq_f8_few_##MT##_##NT##_##WK##_grouped(F8Args a) {              \
        f8_few<MT, NT, WK, true>(a);                                                                                        \
    }
RFXQ_F8_FEW(1, 1, 8)
