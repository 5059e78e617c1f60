// Products of grouped rows with a stack of F16 or BF16 matrices
// (rfxq_grouped_gemm): y[dst_p][n] = sum_k x[src_p][k] W_g[n][k] for the rows p
// of group g, f32 accumulation, one rounding to the type of y.
//
// f32 activations keep their accuracy: a first launch splits each value into
// pieces of the weights' type that add up to it, and the products run over the
// pieces (the same weights, f32 accumulation).
// Rows are scaled by a power of two first, so that a row's largest value lies
// in [2^14, 2^15) (the matrix instructions take subnormal bf16 operands as 0):
//   f16:  hi = RN16(x), lo = RN16(x - hi): 22 bits or more of every value above
//         2^-17 of the row's largest, 2^-39 of the largest of every other
//   bf16: three truncations of 8 bits each: exact for every value above 2^-100
//         of the row's largest
// Products of the pieces cost 2 (f16) or 3 (bf16) times the matrix
// instructions; one rounding of x to the weights' type would cost 2^-12 or 2^-9
// of every value, which f32 outputs show.
#pragma once
#include "common.hpp"
#include "rows.hpp"

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef u4_t u4a2_t __attribute__((aligned(2)));

template <typename T>
RFXQ_DEV f4v_t mfma32(u4_t a, u4_t b, f4v_t c) {
    if constexpr (__is_same(T, half_t))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

struct GroupedArgs {
    const uint16_t* x;  // rows of halves (pieces: plane p of `plane` elements)
    const uint16_t* w;
    void* y;
    const int32_t* offsets;
    const int32_t* x_index;
    const int32_t* y_index;
    const int32_t* x_exp;  // pieces: the results are taken times 2^x_exp[src], or NULL
    uint64_t ldx, ldy, plane, w_stride;
    uint32_t rows, x_rows, y_rows, x_div;
    uint32_t k, n, groups, pieces;
    uint32_t y_f32, tiles_m, tiles_n, sm, sn, pad;
};

// 16 zero bytes that lanes past a row's end copy from
__device__ const u4_t rfxq_zero16 = {0, 0, 0, 0};

// Row p's source and destination; -1 where an index is out of range (such a row
// is not computed).
RFXQ_DEV int64_t src_row(const GroupedArgs& a, uint32_t p) {
    if (!a.x_index) return p < a.x_rows ? (int64_t)p : -1;
    const int32_t i = a.x_index[p];
    if (i < 0) return -1;
    const uint32_t s = (uint32_t)i / a.x_div;
    return s < a.x_rows ? (int64_t)s : -1;
}
RFXQ_DEV int64_t dst_row(const GroupedArgs& a, uint32_t p) {
    const int32_t i = a.y_index ? a.y_index[p] : (int32_t)p;
    return i >= 0 && (uint32_t)i < a.y_rows ? (int64_t)i : -1;
}

// Workgroup b's place in the grid of tiles: workgroups go round-robin to the 8
// XCDs, and each XCD takes blocks of sm x sn neighbouring tiles, whose rows
// and columns meet in its L2.
RFXQ_DEV bool tile_place(const GroupedArgs& a, uint32_t b, uint32_t& tm, uint32_t& tn) {
    const uint32_t j = b >> 3, per = a.sm * a.sn;
    const uint32_t block = (j / per) * 8u + (b & 7u), r = j % per, across = (a.tiles_n + a.sn - 1u) / a.sn;
    tm = (block / across) * a.sm + r % a.sm;
    tn = (block % across) * a.sn + r / a.sm;
    return tm < a.tiles_m && tn < a.tiles_n;
}

// 8 halves at p, of which the first `have` are there: the others are 0.
RFXQ_DEV u4_t ld_halves(const uint16_t* p, uint32_t have) {
    if (have >= 8u) return *(const RFXQ_GLOBAL u4a2_t*)p;
    uint16_t v[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) v[i] = i < have ? ((const RFXQ_GLOBAL uint16_t*)p)[i] : (uint16_t)0;
    u4_t r;
#pragma unroll
    for (uint32_t i = 0; i < 4u; i++) r[i] = (uint32_t)v[2 * i] | (uint32_t)v[2 * i + 1] << 16;
    return r;
}

// 16 neighbouring results of one row, of which the first `have` are there.
template <typename T>
RFXQ_DEV void st_row(const GroupedArgs& a, int64_t row, uint32_t n, const f4v_t (&v)[4]) {
    const uint32_t have = a.n > n ? a.n - n : 0u;
    const uint64_t at = (uint64_t)row * a.ldy + n;
    if (a.y_f32) {
        float* y = static_cast<float*>(a.y) + at;
        if (have >= 16u && (reinterpret_cast<uintptr_t>(y) & 15u) == 0u) {
#pragma unroll
            for (int i = 0; i < 4; i++) *(RFXQ_GLOBAL f4v_t*)(y + 4 * i) = v[i];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 16u; i++)
                if (i < have) stf(y + i, v[i >> 2][i & 3u]);
        }
        return;
    }
    uint16_t* y = static_cast<uint16_t*>(a.y) + at;
    u4_t r[2];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const T lo = (T)v[i >> 1][2 * (i & 1)], hi = (T)v[i >> 1][2 * (i & 1) + 1];
        r[i >> 2][i & 3] = (uint32_t)__builtin_bit_cast(uint16_t, lo) | (uint32_t)__builtin_bit_cast(uint16_t, hi) << 16;
    }
    if (have >= 16u && (reinterpret_cast<uintptr_t>(y) & 15u) == 0u) {
        *(RFXQ_GLOBAL u4_t*)y = r[0];
        *(RFXQ_GLOBAL u4_t*)(y + 8) = r[1];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16u; i++)
            if (i < have) ((RFXQ_GLOBAL uint16_t*)y)[i] = (uint16_t)(r[i >> 3][(i >> 1) & 3] >> (16u * (i & 1u)));
    }
}

// Place of 16-byte piece c (of 8) of LDS row r: rows of 128 bytes, pieces
// xor'ed with the row so that 8 rows' pieces of one column lie in 8 banks' groups.
RFXQ_DEV uint32_t lds_piece(uint32_t r, uint32_t c) { return r * 8u + (c ^ (r & 7u)); }

// The column of a tile that LDS row j of the weights holds. A lane's results
// are rows 4q..4q+3 of each 16-row operand (q = lane / 16): with this order the
// four operands of a wave's 64 columns give it 16 neighbouring ones.
RFXQ_DEV uint32_t col_of(uint32_t j) { return (j & ~63u) + ((j >> 2) & 3u) * 16u + ((j >> 4) & 3u) * 4u + (j & 3u); }

// The wave's 16 MF x 64 tile of one 64-wide step of K, both operands in LDS.
template <typename T, int MF>
RFXQ_DEV void tile_step(const u4_t* xs, const u4_t* ws, uint32_t xr, uint32_t wr, f4v_t (&acc)[MF][4]) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4;
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) {
        u4_t wf[4], xf[MF];
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++) wf[f] = ws[lds_piece(wr + 16u * f + l, 4u * h + q)];
#pragma unroll
        for (uint32_t m = 0; m < (uint32_t)MF; m++) xf[m] = xs[lds_piece(xr + 16u * m + l, 4u * h + q)];
#pragma unroll
        for (uint32_t m = 0; m < (uint32_t)MF; m++)
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) acc[m][f] = mfma32<T>(wf[f], xf[m], acc[m][f]);
    }
}

template <typename T, int MF>
RFXQ_DEV void tile_out(const GroupedArgs& a, const RowTile& t, uint32_t m0, uint32_t n0, const f4v_t (&acc)[MF][4]) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4;
#pragma unroll
    for (uint32_t m = 0; m < (uint32_t)MF; m++) {
        const uint32_t p = t.beg + m0 + 16u * m + l;
        if (p >= t.end) continue;
        const int64_t src = src_row(a, p), dst = dst_row(a, p);
        if (src < 0 || dst < 0) continue;
        f4v_t v[4];
        const int e = a.x_exp ? a.x_exp[src] : 0;
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[f][i] = a.x_exp ? __builtin_ldexpf(acc[m][f][i], e) : acc[m][f][i];
        st_row<T>(a, dst, n0 + 16u * q, v);
    }
}

// Any alignment and any K: operands through registers, element by element at
// a row's end. 64 x 128 tiles, 4 waves of 32 x 64.
template <typename T>
RFXQ_DEV void grouped_any(const GroupedArgs& a) {
    constexpr uint32_t BM = 64, BN = 128, NX = BM * 8u / 256u, NW = BN * 8u / 256u;
    __shared__ u4_t xs[BM * 8u], ws[BN * 8u];
    uint32_t tm, tn;
    if (!tile_place(a, blockIdx.x, tm, tn)) return;
    const RowTile t = find_tile(a.offsets, a.groups, a.rows, BM, tm);
    if (!t.any) return;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, n0 = tn * BN;
    const uint16_t* w = a.w + (uint64_t)t.group * a.w_stride;
    const uint16_t* xp[NX];
    const uint16_t* wp[NW];
#pragma unroll
    for (uint32_t i = 0; i < NX; i++) {
        const uint32_t p = t.beg + (tid >> 3) + 32u * i;
        const int64_t s = p < t.end ? src_row(a, p) : -1;
        xp[i] = s < 0 ? nullptr : a.x + (uint64_t)s * a.ldx;
    }
#pragma unroll
    for (uint32_t i = 0; i < NW; i++) {
        const uint32_t n = n0 + col_of((tid >> 3) + 32u * i);
        wp[i] = n < a.n ? w + (uint64_t)n * a.k : nullptr;
    }
    f4v_t acc[2][4] = {};
    const uint32_t steps = (a.k + 63u) / 64u * a.pieces, c = tid & 7u;
    u4_t xv[NX], wv[NW];
    const auto load = [&](uint32_t s) {
        const uint32_t k = s / a.pieces * 64u + 8u * c, have = k < a.k ? a.k - k : 0u;
        const uint64_t at = (uint64_t)(s % a.pieces) * a.plane + k;
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) xv[i] = xp[i] && have ? ld_halves(xp[i] + at, have) : u4_t{0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) wv[i] = wp[i] && have ? ld_halves(wp[i] + k, have) : u4_t{0, 0, 0, 0};
    };
    load(0);
    for (uint32_t s = 0; s < steps; s++) {
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) xs[lds_piece((tid >> 3) + 32u * i, c)] = xv[i];
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) ws[lds_piece((tid >> 3) + 32u * i, c)] = wv[i];
        __syncthreads();
        if (s + 1u < steps) load(s + 1u);
        tile_step<T, 2>(xs, ws, (wave >> 1) * 32u, (wave & 1u) * 64u, acc);
    }
    tile_out<T, 2>(a, t, (wave >> 1) * 32u, n0 + (wave & 1u) * 64u, acc);
}

extern "C" __global__ __launch_bounds__(256) void rfxq_grouped_any_f16(GroupedArgs a) { grouped_any<half_t>(a); }
extern "C" __global__ __launch_bounds__(256) void rfxq_grouped_any_bf16(GroupedArgs a) { grouped_any<__bf16>(a); }

// ---------------------------------------------------------------- f32 activations as pieces

struct SplitArgs {
    const float* x;
    uint16_t* out;    // [pieces][rows][ldo]
    int32_t* exp;     // the rows' exponents
    uint64_t ldx, plane;
    uint32_t rows, k, ldo, pad;
};

// A wave per row; columns k..ldo-1 are 0.
template <bool F16>
RFXQ_DEV void split_rows(const SplitArgs& a) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t r = blockIdx.x * 4u + (threadIdx.x >> 6); r < a.rows; r += gridDim.x * 4u) {
        const float* x = a.x + (uint64_t)r * a.ldx;
        uint16_t* o = a.out + (uint64_t)r * a.ldo;
        float top = 0.0f;  // of the finite values: infinities and NaN stay what they are
        for (uint32_t i = lane; i < a.k; i += 64u) {
            const float v = __builtin_fabsf(x[i]);
            top = v < __builtin_inff() ? fmaxf(top, v) : top;
        }
        top = wave_max(top);
        const int e = top > 0.0f ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;  // top / 2^e in [2^14, 2^15)
        if (lane == 0) a.exp[r] = e;
        for (uint32_t i = lane; i < a.ldo; i += 64u) {
            const float s = i < a.k ? __builtin_ldexpf(x[i], -e) : 0.0f;
            const bool fine = __builtin_fabsf(s) < __builtin_inff();
            if (F16) {
                const half_t hi = (half_t)s;
                const half_t lo = fine ? (half_t)(s - (float)hi) : (half_t)0.0f;
                o[i] = __builtin_bit_cast(uint16_t, hi);
                o[a.plane + i] = __builtin_bit_cast(uint16_t, lo);
            } else {
                const uint32_t h = __builtin_bit_cast(uint32_t, s) & 0xFFFF0000u;
                const float left = fine ? s - as_f32(h) : 0.0f;
                const uint32_t m = __builtin_bit_cast(uint32_t, left) & 0xFFFF0000u;
                const float last = left - as_f32(m);
                // a NaN keeps a set fraction bit
                o[i] = (uint16_t)(h >> 16 | (s != s ? 0x40u : 0u));
                o[a.plane + i] = (uint16_t)(m >> 16);
                o[2u * a.plane + i] = (uint16_t)(__builtin_bit_cast(uint32_t, last) >> 16);
            }
        }
    }
}

extern "C" __global__ __launch_bounds__(256) void rfxq_split_f16(SplitArgs a) { split_rows<true>(a); }
extern "C" __global__ __launch_bounds__(256) void rfxq_split_bf16(SplitArgs a) { split_rows<false>(a); }
