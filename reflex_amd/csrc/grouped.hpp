// Products of grouped rows with a stack of F16 or BF16 matrices
// (rfxq_grouped_gemm): y[dst_p][n] = sum_k x[src_p][k] W_g[n][k] for the rows p
// of group g, f32 accumulation, one rounding to the type of y.
//
// f32 activations keep 22 (f16) or all (bf16) of their bits: they are split into pieces of the
// weights' type that add up to them and multiply the same weights (where a wave has one
// operand of weights, they go through f32 matrix instructions as they are). A
// row's 32 or 64 values of a step are scaled by a power of two first, so that the
// largest lies in [2^14, 2^15) (the matrix instructions take subnormal bf16
// operands as 0), and the step's sum is scaled back as it is added:
//   f16:  x = RN16(x) + RN16(the rest): 22 bits or more of every value above
//         2^-17 of the step's largest, 2^-39 of the largest of every other
//   bf16: three truncations of 8 bits each: exact
// Products of the pieces cost 2 (f16) or 3 (bf16) times the matrix
// instructions; one rounding of x to the weights' type would cost 2^-12 or 2^-9
// of every value, which f32 outputs show.
#pragma once
#include "common.hpp"
#include "rows.hpp"
#include "tiles.hpp"


template <typename T>
RFXQ_DEV f4v_t mfma32(u4_t a, u4_t b, f4v_t c) {
    if constexpr (__is_same(T, half_t))
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, a), __builtin_bit_cast(h8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, a), __builtin_bit_cast(b8_t, b), c, 0, 0, 0);
}

struct GroupedArgs {
    const void* x;
    const uint16_t* w;
    void* y;
    const int32_t* offsets;
    const int32_t* x_index;
    const int32_t* y_index;
    uint64_t ldx, ldy, w_stride;
    uint32_t rows, x_rows, y_rows, x_div;
    uint32_t k, n, groups, y_f32;
    uint32_t tiles_m, tiles_n, sm, sn;
};

// the largest of the four lanes (l, 0..3)
RFXQ_DEV uint32_t top_over_q(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)r[0], (uint32_t)r[1]);
    const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return max((uint32_t)s[0], (uint32_t)s[1]);
}

// The scale of a row's values of a step, from the largest of their sizes: 2^e
// and 2^-e with that one times 2^-e in [2^14, 2^15), kept so that both are f32
// values. Steps with infinities or NaN are not scaled up: what is finite there
// does not show.
struct StepScale {
    float up, back;
};
RFXQ_DEV StepScale step_scale(uint32_t top) {
    const int e = max((int)(top >> 23) - 127 - 14, -126);
    return {as_f32((uint32_t)(127 - e) << 23), as_f32((uint32_t)(127 + e) << 23)};
}

// 8 f32 values of a step as pieces of T that add up to them times `scale`.
// Infinities and NaN (anywhere in the wave: `top`) are whole in the first piece.
template <typename T, uint32_t NP>
RFXQ_DEV void split_eight(const Eight<float>& x, float scale, uint32_t top, u4_t (&out)[NP]) {
    float v[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) v[i] = x.at(i) * scale;
    const auto pieces = [&](bool all_finite) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
            for (uint32_t n = 0; n < NP; n++) {
                float pa, pb;
                if constexpr (__is_same(T, half_t)) {
                    const h2_t h = {(half_t)a, (half_t)b};
                    out[n][i] = h2_bits(h);
                    pa = (float)h[0];
                    pb = (float)h[1];
                } else {  // truncated: the upper halves of the bits (a NaN keeps a set fraction bit there)
                    uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
                    if (!all_finite) {
                        ua |= a != a ? 0x400000u : 0u;
                        ub |= b != b ? 0x400000u : 0u;
                    }
                    out[n][i] = ua >> 16 | (ub & 0xFFFF0000u);
                    pa = as_f32(ua & 0xFFFF0000u);
                    pb = as_f32(ub & 0xFFFF0000u);
                }
                if (n + 1u < NP) {
                    a = all_finite || __builtin_fabsf(a) < __builtin_inff() ? a - pa : 0.0f;
                    b = all_finite || __builtin_fabsf(b) < __builtin_inff() ? b - pb : 0.0f;
                }
            }
        }
    };
    if (__builtin_amdgcn_ballot_w64(top >= kInfBits))
        pieces(false);
    else
        pieces(true);
}

// 16 neighbouring results of one row, of which the first `have` are there. Whole
// vectors at any element (2331 pairs over 11 experts, 1531 x 1235, f32: 49 us, 57 with
// single stores where a row does not start at 16 bytes).
template <typename T>
RFXQ_DEV void st_row(const GroupedArgs& a, int64_t row, uint32_t n, const f4v_t (&v)[4]) {
    const uint32_t have = a.n > n ? a.n - n : 0u;
    const uint64_t at = (uint64_t)row * a.ldy + n;
    if (a.y_f32) {
        float* y = static_cast<float*>(a.y) + at;
        if (have >= 16u) {
#pragma unroll
            for (int i = 0; i < 4; i++) *(RFXQ_GLOBAL f4a4_t*)(y + 4 * i) = v[i];
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
    if (have >= 16u) {
        *(RFXQ_GLOBAL u4a2_t*)y = r[0];
        *(RFXQ_GLOBAL u4a2_t*)(y + 8) = r[1];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 16u; i++)
            if (i < have) ((RFXQ_GLOBAL uint16_t*)y)[i] = (uint16_t)(r[i >> 3][(i >> 1) & 3] >> (16u * (i & 1u)));
    }
}

// 4 neighbouring results of one row.
template <typename T>
RFXQ_DEV void st_four(const GroupedArgs& a, int64_t row, uint32_t n, f4v_t v) {
    const uint32_t have = a.n > n ? a.n - n : 0u;
    const uint64_t at = (uint64_t)row * a.ldy + n;
    if (a.y_f32) {
        float* y = static_cast<float*>(a.y) + at;
        if (have >= 4u) {
            *(RFXQ_GLOBAL f4a4_t*)y = v;
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++)
                if (i < have) stf(y + i, v[i]);
        }
        return;
    }
    typedef T t4_t __attribute__((ext_vector_type(4)));
    typedef T t4a2_t __attribute__((ext_vector_type(4), aligned(2)));
    T* y = static_cast<T*>(a.y) + at;
    t4_t r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = (T)v[i];
    if (have >= 4u) {
        *(RFXQ_GLOBAL t4a2_t*)y = r;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++)
            if (i < have) ((RFXQ_GLOBAL T*)y)[i] = r[i];
    }
}

// The wave's 16 MF x 64 tile of one 64-wide step of K, both operands in LDS
// (the activations' pieces XS apart, the last ones first).
template <typename T, int MF, uint32_t PIECES, uint32_t XS>
RFXQ_DEV void tile_step(const u4_t* xs, const u4_t* ws, uint32_t xr, uint32_t wr, f4v_t (&acc)[MF][4]) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4;
#pragma unroll
    for (uint32_t h = 0; h < 2u; h++) {
        u4_t wf[4];
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++) wf[f] = ws[lds_piece(wr + 16u * f + l, 4u * h + q)];
#pragma unroll
        for (uint32_t j = 0; j < PIECES; j++) {
            u4_t xf[MF];
#pragma unroll
            for (uint32_t m = 0; m < (uint32_t)MF; m++)
                xf[m] = xs[(PIECES - 1u - j) * XS + lds_piece(xr + 16u * m + l, 4u * h + q)];
#pragma unroll
            for (uint32_t m = 0; m < (uint32_t)MF; m++)
#pragma unroll
                for (uint32_t f = 0; f < 4u; f++) acc[m][f] = mfma32<T>(wf[f], xf[m], acc[m][f]);
        }
    }
}

// 16-row operand m holds the tile's rows m0 + STEP m and on.
template <typename T, int MF, uint32_t STEP = 16>
RFXQ_DEV void tile_out(const GroupedArgs& a, const RowTile& t, uint32_t m0, uint32_t n0, const f4v_t (&acc)[MF][4]) {
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4;
    mfma_settle();
#pragma unroll
    for (uint32_t m = 0; m < (uint32_t)MF; m++) {
        const uint32_t p = t.beg + m0 + STEP * m + l;
        if (p >= t.end) continue;
        const int64_t src = src_row(a, p), dst = dst_row(a, p);
        if (src < 0 || dst < 0) continue;
        st_row<T>(a, dst, n0 + 16u * q, acc[m]);
    }
}

// Any alignment and any K: operands through registers, the next step's loads in
// flight during the products. 64 x 128 tiles, 4 waves of 32 x 64. Loads of
// whole steps have no condition: rows and columns past the tile read others,
// whose results are not stored. The last, partial step is loaded element by
// element, with zeros behind the end of both operands.
// Memory bounds it at 32 rows a group (4096 pairs over 128 experts, 768 x 2048
// bf16: 99 us, 410 MB at 4.2 TB/s, matrix pipes 14% busy), 4 workgroups a CU.
// TX float: split into pieces on the way to LDS, all against one tile of weights
// (2331 pairs over 11 experts, 1531 x 1235 bf16: 49 us, 564 tiles, pipes 28% busy; the
// pieces written by a launch of their own, read again: 30% more).
template <typename TX, typename T>
RFXQ_DEV void grouped_any(const GroupedArgs& a) {
    constexpr bool F32 = __is_same(TX, float);
    constexpr uint32_t P = !F32 ? 1u : __is_same(T, half_t) ? 2u : 3u;
    constexpr uint32_t BM = 64, BN = 128, NX = BM * 8u / 256u, NW = BN * 8u / 256u;
    __shared__ u4_t xs[P][BM * 8u], ws[BN * 8u];
    __shared__ float back[F32 ? BM : 1u];  // of the step's rows
    uint32_t tm, tn;
    if (!tile_place(a, blockIdx.x, tm, tn)) return;
    const RowTile t = find_tile(a.offsets, a.groups, a.rows, BM, tm);
    if (!t.any) return;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, n0 = tn * BN, c = tid & 7u, l = tid & 15u;
    const T* w = reinterpret_cast<const T*>(a.w) + (uint64_t)t.group * a.w_stride;
    const TX* xp[NX];
    const T* wp[NW];
#pragma unroll
    for (uint32_t i = 0; i < NX; i++) {
        const int64_t s = src_row(a, min(t.beg + (tid >> 3) + 32u * i, t.end - 1u));
        xp[i] = static_cast<const TX*>(a.x) + (s < 0 ? 0 : (uint64_t)s * a.ldx) + 8u * c;
    }
#pragma unroll
    for (uint32_t i = 0; i < NW; i++)
        wp[i] = w + (uint64_t)min(n0 + col_of<>((tid >> 3) + 32u * i), a.n - 1u) * a.k + 8u * c;
    f4v_t acc[2][4] = {};
    const uint32_t full = a.k / 64u, tail = a.k % 64u, steps = full + (tail ? 1u : 0u);
    const uint32_t row0 = (wave >> 1) * 32u, col0 = (wave & 1u) * 64u;
    Eight<TX> xv[NX];
    Eight<T> wv[NW];
    const auto load = [&](uint32_t s) {
        const uint32_t k = s * 64u;
        if (s < full) {
#pragma unroll
            for (uint32_t i = 0; i < NW; i++) wv[i] = ld_eight(wp[i] + k);
#pragma unroll
            for (uint32_t i = 0; i < NX; i++) xv[i] = ld_eight(xp[i] + k);
        } else if (s < steps) {
            const uint32_t have = tail > 8u * c ? tail - 8u * c : 0u;
#pragma unroll
            for (uint32_t i = 0; i < NW; i++) wv[i] = ld_eight(wp[i] + k, have);
#pragma unroll
            for (uint32_t i = 0; i < NX; i++) xv[i] = ld_eight(xp[i] + k, have);
        }
    };
    load(0);
    for (uint32_t s = 0; s < steps; s++) {
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) {
            const uint32_t r = (tid >> 3) + 32u * i;
            if constexpr (F32) {
                const uint32_t top = top_over_8(top_of_eight(xv[i]));
                const StepScale scale = step_scale(top);
                u4_t p[P];
                split_eight<T, P>(xv[i], scale.up, top, p);
#pragma unroll
                for (uint32_t j = 0; j < P; j++) xs[j][lds_piece(r, c)] = p[j];
                if (c == 0) back[r] = scale.back;
            } else {
                xs[0][lds_piece(r, c)] = xv[i].v;
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) ws[lds_piece((tid >> 3) + 32u * i, c)] = wv[i].v;
        __syncthreads();
        load(s + 1u);
        if constexpr (F32) {
            f4v_t d[2][4] = {};
            tile_step<T, 2, P, BM * 8u>(xs[0], ws, row0, col0, d);
#pragma unroll
            for (uint32_t m = 0; m < 2u; m++) {
                const float scale = back[row0 + 16u * m + l];
#pragma unroll
                for (uint32_t f = 0; f < 4u; f++) acc[m][f] += d[m][f] * scale;
            }
        } else {
            tile_step<T, 2, 1, 0>(xs[0], ws, row0, col0, acc);
        }
    }
    tile_out<T, 2>(a, t, row0, n0 + col0, acc);
}

extern "C" __global__ __launch_bounds__(256, 4) void rfxq_grouped_any_f16(GroupedArgs a) { grouped_any<half_t, half_t>(a); }
extern "C" __global__ __launch_bounds__(256, 4) void rfxq_grouped_any_bf16(GroupedArgs a) { grouped_any<__bf16, __bf16>(a); }
extern "C" __global__ __launch_bounds__(256, 3) void rfxq_grouped_any_f32_f16(GroupedArgs a) { grouped_any<float, half_t>(a); }
extern "C" __global__ __launch_bounds__(256, 3) void rfxq_grouped_any_f32_bf16(GroupedArgs a) { grouped_any<float, __bf16>(a); }

// ---------------------------------------------------------------- tiles filled by asynchronous copies

// BM x BN tiles of WM x WN waves (each BM / WM rows x 64 columns), 64-wide
// steps of K in STAGES buffers: copies global -> LDS are issued STAGES - 1 steps
// ahead of the products, without registers between. Rows of x and W start at
// whole 16 bytes; what lies past a row's end or the tile's last row is copied
// from past the buffer's end, which fills it with zeros. Offsets within x and
// within one matrix stay below 4 GiB (the host's rule). 64 x 128, 3 buffers: one
// or two workgroups a CU reach memory's rate (8 x 4096 x 14336, 32 rows each, bf16:
// 186 us, 5.0 TB/s; 247 through registers). In two of the loop's three steps the
// compiler has the first LDS read wait for every copy in flight (it cannot tell the
// buffers that they go to from the one it reads): there the copies are one step ahead only.
template <typename T, int BM, int BN, int WM, int WN, int STAGES>
struct GroupedTile {
    static constexpr uint32_t THREADS = 64u * WM * WN, MF = BM / WM / 16;
    static constexpr uint32_t NX = BM * 8u / THREADS, NW = BN * 8u / THREADS, LOADS = NX + NW;
    static constexpr uint32_t PAST = 0xFFFFFFF0u;
    static_assert(BN == 64 * WN && NX >= 1 && NW >= 1 && LOADS < 64);

    RowTile t;
    rsrc_t xr, wr;
    uint32_t xo[NX], wo[NW];  // lanes' byte offsets at k = 0
    uint32_t lane, wave, piece, n0, k, steps;
    uint32_t at = 0;  // of the next step to copy

    __device__ __forceinline__ void issue(u4_t* xs, u4_t* ws) {
        // past the end: as many copies, so that waits count the same
        const bool there = at + 64u <= k || at + 8u * piece < k;
        const uint32_t by = at < k ? 2u * at : 0u;
#pragma unroll
        for (uint32_t i = 0; i < NX; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, RFXQ_LDSP(xs + (wave * NX + i) * 64u), 16, there ? xo[i] : PAST, by,
                                                     0, 0);
#pragma unroll
        for (uint32_t i = 0; i < NW; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(wr, RFXQ_LDSP(ws + (wave * NW + i) * 64u), 16, there ? wo[i] : PAST, by,
                                                     0, 0);
        at += 64u;
    }

    // the tile, and where its rows are; false: there is none
    __device__ __forceinline__ bool begin(const GroupedArgs& a) {
        uint32_t tm, tn;
        if (!tile_place(a, blockIdx.x, tm, tn)) return false;
        t = find_tile(a.offsets, a.groups, a.rows, BM, tm);
        if (!t.any) return false;
        lane = threadIdx.x & 63u;
        n0 = tn * BN;
        wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        piece = (lane & 7u) ^ (lane >> 3);
        k = a.k;
        const uint64_t xbytes = ((uint64_t)(a.x_rows - 1u) * a.ldx + a.k) * 2u;
        xr = make_rsrc(a.x, (uint32_t)xbytes);
        wr = make_rsrc(a.w + (uint64_t)t.group * a.w_stride, (uint32_t)(2u * a.w_stride));
#pragma unroll
        for (uint32_t i = 0; i < NX; i++) {
            const uint32_t p = t.beg + (wave * NX + i) * 8u + (lane >> 3);
            const int64_t s = p < t.end ? src_row(a, p) : -1;
            xo[i] = s < 0 ? PAST : (uint32_t)((uint64_t)s * a.ldx * 2u) + 16u * piece;
        }
#pragma unroll
        for (uint32_t i = 0; i < NW; i++) {
            const uint32_t n = n0 + col_of<>((wave * NW + i) * 8u + (lane >> 3));
            wo[i] = n < a.n ? n * a.k * 2u + 16u * piece : PAST;
        }
        steps = (a.k + 63u) / 64u;
        return true;
    }

    __device__ __forceinline__ void run(const GroupedArgs& a) {
        static_assert(STAGES == 3);
        __shared__ u4_t xs0[BM * 8], xs1[BM * 8], xs2[BM * 8], ws0[BN * 8], ws1[BN * 8], ws2[BN * 8];
        if (!begin(a)) return;
        f4v_t acc[MF][4] = {};
        const uint32_t row0 = (wave / WN) * (BM / WM), col0 = (wave % WN) * 64u;
        issue(xs0, ws0);
        issue(xs1, ws1);
        const auto step = [&](const u4_t* xs, const u4_t* ws, u4_t* nx, u4_t* nw) {
            __builtin_amdgcn_s_waitcnt(0x0F70 | (LOADS & 15u) | (LOADS >> 4) << 14);  // all but the next step's copies
            lds_barrier();
            issue(nx, nw);
            tile_step<T, MF, 1, 0>(xs, ws, row0, col0, acc);
        };
        for (uint32_t s = 0; s < steps; s += 3u) {
            step(xs0, ws0, xs2, ws2);
            if (s + 1u < steps) step(xs1, ws1, xs0, ws0);
            if (s + 2u < steps) step(xs2, ws2, xs1, ws1);
        }
        __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy outlives the workgroup
        tile_out<T, MF>(a, t, row0, n0 + col0, acc);
    }

    // 256 x 256 tiles, 8 waves. The waves of a SIMD (w and w + 4) take turns: while
    // one multiplies 32 of K from its registers, the other reads its next operands
    // from LDS. A turn ends with a barrier, the upper waves are a turn behind.
    // Reads of a step end with the upper waves' fourth turn, so the copies into its
    // buffer begin in the first turn of the next step; they are waited for at the
    // end of that step's last turn (the upper waves' last reading turn).
    // The lower and the upper waves take every other 16 rows of the tile, and leave
    // out those behind the group's last row: FULL has none.
    // 8192 rows over 8 matrices of 14336 x 4096 f16: 0.90 to 0.94 ms, 1.02 to 1.07
    // PFLOP/s, matrix pipes 58% busy (64 x 128 tiles: 1.46 ms); without copies 0.66 ms,
    // with all of them from L2 0.77: their traffic and the clock it costs bound it.
    template <bool FULL>
    __device__ __forceinline__ void turns(u4_t* xs0, u4_t* xs1, u4_t* ws0, u4_t* ws1, f4v_t (&acc)[MF][4]) {
        const uint32_t upper = wave >> 2, l = lane & 15u, q = lane >> 4, row0 = upper * 16u, col0 = (wave & 3u) * 64u;
        const uint32_t rows = t.end - t.beg, some = rows > row0 ? (rows - row0 + 31u) / 32u : 0u;
        u4_t wf[4], xf[MF];
        const auto turn_over = [] {
            __builtin_amdgcn_sched_barrier(0);
            lds_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        const auto read = [&](const u4_t* xs, const u4_t* ws, uint32_t h) {
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) wf[f] = ws[lds_piece(col0 + 16u * f + l, 4u * h + q)];
#pragma unroll
            for (uint32_t m = 0; m < MF; m++)
                if (FULL || m < some) xf[m] = xs[lds_piece(row0 + 32u * m + l, 4u * h + q)];
        };
        const auto multiply = [&] {
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (uint32_t m = 0; m < MF; m++)
                if (FULL || m < some) {
#pragma unroll
                    for (uint32_t f = 0; f < 4u; f++) acc[m][f] = mfma32<T>(wf[f], xf[m], acc[m][f]);
                }
            __builtin_amdgcn_s_setprio(0);
        };
        const auto step = [&](const u4_t* xs, const u4_t* ws, u4_t* nx, u4_t* nw) {
            read(xs, ws, 0);
            issue(nx, nw);
            turn_over();
            multiply();
            turn_over();
            read(xs, ws, 1);
            if (upper) __builtin_amdgcn_s_waitcnt(0x0F70);
            turn_over();
            multiply();
            if (!upper) __builtin_amdgcn_s_waitcnt(0x0F70);
            turn_over();
        };
        issue(xs0, ws0);
        __builtin_amdgcn_s_waitcnt(0x0F70);
        turn_over();
        if (upper) turn_over();
        for (uint32_t s = 0; s < steps; s += 2u) {
            step(xs0, ws0, xs1, ws1);
            if (s + 1u < steps) step(xs1, ws1, xs0, ws0);
        }
        if (!upper) turn_over();
        __builtin_amdgcn_s_waitcnt(0x0F70);  // no copy outlives the workgroup
    }
    __device__ __forceinline__ void run_turns(const GroupedArgs& a) {
        static_assert(WM * WN == 8 && WN == 4 && STAGES == 2);
        __shared__ u4_t xs0[BM * 8], xs1[BM * 8], ws0[BN * 8], ws1[BN * 8];
        if (!begin(a)) return;
        f4v_t acc[MF][4] = {};
        if (t.end - t.beg == BM)
            turns<true>(xs0, xs1, ws0, ws1, acc);
        else
            turns<false>(xs0, xs1, ws0, ws1, acc);
        tile_out<T, MF, 32>(a, t, (wave >> 2) * 16u, n0 + (wave & 3u) * 64u, acc);
    }
};

#define RFXQ_GROUPED_TILE(name, T, BM, BN, WM, WN, STAGES, RUN)                                      \
    extern "C" __global__ __launch_bounds__(64 * WM * WN) void rfxq_grouped_##name(GroupedArgs a) { \
        GroupedTile<T, BM, BN, WM, WN, STAGES> t;                                                    \
        t.RUN(a);                                                                                    \
    }
RFXQ_GROUPED_TILE(64_f16, half_t, 64, 128, 2, 2, 3, run)
RFXQ_GROUPED_TILE(64_bf16, __bf16, 64, 128, 2, 2, 3, run)
RFXQ_GROUPED_TILE(256_f16, half_t, 256, 256, 2, 4, 2, run_turns)
RFXQ_GROUPED_TILE(256_bf16, __bf16, 256, 256, 2, 4, 2, run_turns)

// ---------------------------------------------------------------- ranges of K, a wave each

// 16 MT rows times 16 RT columns over [k0, k1) of K, a wave by itself: both operands
// from memory straight into registers, 64 of K (whole 128-byte lines of half-typed
// rows) a step. w, and x as rows() gives it, point to the lane's first values, 8
// (lane / 16) on from k = 0. The numbers of operands are known at compile time: the
// products of a step and what reads them stay free of branches (mfma_settle). Other
// waves hide the loads: with steps in flight ahead a wave needs the registers of two
// (rfxq_lora_down, 4096 rows of 4096 values, rank 64: 58.0 us with rfxq_lora_up, 56.4 without).
template <typename TX, typename TW, uint32_t MT, uint32_t RT, typename Rows>
RFXQ_DEV void k_range(const TW* const (&w)[RT], const Rows& rows, uint32_t k0, uint32_t k1, f4v_t (&acc)[MT][RT]) {
    const uint32_t full = (k1 - k0) / 64u, tail = (k1 - k0) % 64u;
    Eight<TX> xv[MT][2];
    Eight<TW> wv[RT][2];
    const TX* x[MT];
    const auto load_w = [&](uint32_t k) {
#pragma unroll
        for (uint32_t f = 0; f < RT; f++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) wv[f][h] = ld_eight(w[f] + k + 32u * h);
    };
    const auto load_x = [&](uint32_t k) {
#pragma unroll
        for (uint32_t m = 0; m < MT; m++)
#pragma unroll
            for (uint32_t h = 0; h < 2u; h++) xv[m][h] = ld_eight(x[m] + k + 32u * h);
    };
    const auto multiply = [&](uint32_t h) {
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) {
            if constexpr (__is_same(TW, float)) {
#pragma unroll
                for (uint32_t f = 0; f < RT; f++)
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++)
                        acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[f][h].at(j), xv[m][h].at(j), acc[m][f], 0, 0, 0);
            } else if constexpr (__is_same(TX, TW)) {
#pragma unroll
                for (uint32_t f = 0; f < RT; f++) acc[m][f] = mfma32<TW>(wv[f][h].v, xv[m][h].v, acc[m][f]);
            } else {
                constexpr uint32_t NP = __is_same(TW, half_t) ? 2u : 3u;
                const uint32_t top = top_over_q(top_of_eight(xv[m][h]));
                const StepScale scale = step_scale(top);
                const float back = scale.back;
                u4_t xp[NP];
                split_eight<TW, NP>(xv[m][h], scale.up, top, xp);
#pragma unroll
                for (uint32_t f = 0; f < RT; f++) {
                    f4v_t d = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t n = 0; n < NP; n++) d = mfma32<TW>(wv[f][h].v, xp[NP - 1u - n], d);
                    acc[m][f] += d * back;
                }
            }
        }
    };
    if (full) load_w(k0);  // on their way while the rows are looked up
    rows(x);
    for (uint32_t i = 0; i < full; i++) {
        if (i) load_w(k0 + 64u * i);
        load_x(k0 + 64u * i);
        multiply(0);
        multiply(1);
    }
    mfma_settle();
    if (tail) {
        const uint32_t q = (threadIdx.x & 63u) >> 4;
#pragma unroll
        for (uint32_t h = 0; h < 2u; h++) {
            const uint32_t k = k0 + 64u * full + 32u * h, have = tail > 32u * h + 8u * q ? tail - 32u * h - 8u * q : 0u;
#pragma unroll
            for (uint32_t f = 0; f < RT; f++) wv[f][h] = ld_eight(w[f] + k, have);
#pragma unroll
            for (uint32_t m = 0; m < MT; m++) xv[m][h] = ld_eight(x[m] + k, have);
        }
        multiply(0);
        multiply(1);
        mfma_settle();
    }
}

// f32 activations where 64 x 128 tiles leave CUs without work or are mostly empty: 32 x 64,
// the workgroup's waves take quarters of K and add them in LDS, any alignment. A
// tile's time there is that of its steps, a quarter as many here (8 groups of 64
// rows, N x K 1024 x 4096: 38 us against 95; a CU's loads bound it: the same with
// steps copied ahead).
template <typename TX, typename TW>
RFXQ_DEV void grouped_quarters(const GroupedArgs& a) {
    constexpr uint32_t MT = 2, RT = 4;
    __shared__ f4v_t part[4][MT][RT][64];
    uint32_t tm, tn;
    if (!tile_place(a, blockIdx.x, tm, tn)) return;
    const RowTile t = find_tile(a.offsets, a.groups, a.rows, 16u * MT, tm);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4, n0 = tn * 16u * RT;
    const TW* w[RT];
#pragma unroll
    for (uint32_t f = 0; f < RT; f++)  // columns past the last read it again; their results are not stored
        w[f] = reinterpret_cast<const TW*>(a.w) + (uint64_t)t.group * a.w_stride + (uint64_t)min(n0 + 16u * f + l, a.n - 1u) * a.k +
               8u * q;
    const uint32_t quarter = ((a.k + 3u) / 4u + 63u) & ~63u, k0 = min(wave * quarter, a.k);
    int64_t src[MT];
    f4v_t acc[MT][RT] = {};
    k_range<TX, TW, MT, RT>(
        w,
        [&](const TX*(&x)[MT]) {
#pragma unroll
            for (uint32_t m = 0; m < MT; m++) {
                const uint32_t p = t.beg + 16u * m + l;
                const int64_t found = src_row(a, min(p, t.end - 1u));
                src[m] = p < t.end ? found : -1;
                x[m] = static_cast<const TX*>(a.x) + (src[m] < 0 ? 0 : (uint64_t)src[m] * a.ldx) + 8u * q;
            }
        },
        k0, min(k0 + quarter, a.k), acc);
#pragma unroll
    for (uint32_t m = 0; m < MT; m++)
#pragma unroll
        for (uint32_t f = 0; f < RT; f++) part[wave][m][f][lane] = acc[m][f];
    __syncthreads();
#pragma unroll
    for (uint32_t m = 0; m < MT; m++) {  // a wave stores 16 of the columns
        const f4v_t s = ((part[0][m][wave][lane] + part[1][m][wave][lane]) + part[2][m][wave][lane]) + part[3][m][wave][lane];
        if (src[m] < 0) continue;
        const int64_t dst = dst_row(a, t.beg + 16u * m + l);
        if (dst >= 0) st_four<TW>(a, dst, n0 + 16u * wave + 4u * q, s);
    }
}

#define RFXQ_GROUPED_QUARTERS(name, TX, TW) \
    extern "C" __global__ __launch_bounds__(256) void rfxq_grouped_quarters_##name(GroupedArgs a) { grouped_quarters<TX, TW>(a); }
RFXQ_GROUPED_QUARTERS(f32_f16, float, half_t)
RFXQ_GROUPED_QUARTERS(f32_bf16, float, __bf16)

// ---------------------------------------------------------------- few rows a group

// Decode: what a group's matrix weighs is all that counts, so its rows go from
// memory straight into the matrix instructions' registers, each once, as their
// 16-row operand; up to 16 activation rows are the other one. A wave takes 16 NT
// columns and all of K (WK = 1) or, where that makes too few waves, a quarter of K
// (WK = 4, the workgroup's waves add their parts in LDS). Loads run a block of 128 of K
// ahead of the products, any alignment. A token over 8 of 128 experts, 768 x 2048 bf16:
// 7.6 us, 3.3 TB/s, three trips to memory one after the other.
// f32 activations: in pieces where a wave has two operands of weights for them (128
// experts, 32 tokens over 8 of them, 2048 x 768 f16: 54 us, 5.9 TB/s of weights; 61 with
// f32 matrix instructions, 256 cycles for 8 x 4 of K and an operand, which the memory
// reads no longer hid), as they are where it has one (60 x 1024 x 4096: 111 against 127 us).
template <typename TX, typename TW, uint32_t NT, uint32_t WK>
RFXQ_DEV void grouped_few(const GroupedArgs& a) {
    constexpr bool F32 = __is_same(TX, float);
    __shared__ f4v_t part[WK > 1 ? (WK - 1) * NT * 64u : 1u];
    constexpr uint32_t COLS = 16u * NT * 4u / WK;  // a workgroup's
    const uint32_t tn = blockIdx.x % a.tiles_n;
    const RowTile t = find_tile(a.offsets, a.groups, a.rows, 16, blockIdx.x / a.tiles_n);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4;
    const uint32_t n0 = tn * COLS + (WK == 1 ? wave * 16u * NT : 0u);
    const uint32_t blocks = (a.k + 127u) / 128u, each = (blocks + WK - 1u) / WK;
    const uint32_t b0 = WK == 1 ? 0u : min(wave * each, blocks), b1 = WK == 1 ? blocks : min(b0 + each, blocks);
    const uint32_t p = t.beg + l;
    const TW* w[NT];
#pragma unroll
    for (uint32_t f = 0; f < NT; f++)
        w[f] = reinterpret_cast<const TW*>(a.w) + (uint64_t)t.group * a.w_stride + (uint64_t)min(n0 + 16u * f + l, a.n - 1u) * a.k;
    f4v_t acc[NT] = {};
    Eight<TW> wv[2][4][NT];
    Eight<TX> xv[2][4];
    // blocks of 128 that are whole, without conditions; then the last values of K
    const auto load_w = [&](uint32_t s, uint32_t b, uint32_t i) {
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) wv[s][i][f] = ld_eight(w[f] + 128u * b + 32u * i + 8u * q);
    };
    const uint32_t whole = min(b1, a.k / 128u);
    if (b0 < whole) {  // on their way while the rows are looked up
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) load_w(0, b0, i);
    }
    const int64_t found = src_row(a, min(p, t.end - 1u)), src = p < t.end ? found : -1;
    const TX* x = static_cast<const TX*>(a.x) + (src < 0 ? 0 : (uint64_t)src * a.ldx);
    const auto load_x = [&](uint32_t s, uint32_t b, uint32_t i) { xv[s][i] = ld_eight(x + 128u * b + 32u * i + 8u * q); };
    const auto load = [&](uint32_t s, uint32_t b) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            load_w(s, b, i);
            load_x(s, b, i);
        }
    };
    const auto load_tail = [&](uint32_t b) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            const uint32_t k = 128u * b + 32u * i + 8u * q, have = a.k > k ? a.k - k : 0u;
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) wv[0][i][f] = ld_eight(w[f] + k, have);
            xv[0][i] = ld_eight(x + k, have);
        }
    };
    const auto multiply = [&](uint32_t s) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) {
            if constexpr (F32 && WK > 1) {
#pragma unroll
                for (uint32_t f = 0; f < NT; f++)
#pragma unroll
                    for (uint32_t j = 0; j < 8u; j++)
                        acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(wv[s][i][f].at(j), xv[s][i].at(j), acc[f], 0, 0, 0);
            } else if constexpr (F32) {
                constexpr uint32_t NP = __is_same(TW, half_t) ? 2u : 3u;
                const uint32_t top = top_over_q(top_of_eight(xv[s][i]));
                const StepScale scale = step_scale(top);
                const float back = scale.back;
                u4_t xp[NP];
                split_eight<TW, NP>(xv[s][i], scale.up, top, xp);
#pragma unroll
                for (uint32_t f = 0; f < NT; f++) {
                    f4v_t d = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t n = 0; n < NP; n++) d = mfma32<TW>(wv[s][i][f].v, xp[NP - 1u - n], d);
                    acc[f] += d * back;
                }
            } else {
#pragma unroll
                for (uint32_t f = 0; f < NT; f++) acc[f] = mfma32<TW>(wv[s][i][f].v, xv[s][i].v, acc[f]);
            }
        }
    };
    if (b0 < whole) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; i++) load_x(0, b0, i);
    }
    for (uint32_t b = b0; b < whole; b += 2u) {
        if (b + 1u < whole) load(1, b + 1u);
        multiply(0);
        if (b + 2u < whole) load(0, b + 2u);
        if (b + 1u < whole) multiply(1);
    }
    if (whole < b1 && b0 < b1) {
        load_tail(b1 - 1u);
        multiply(0);
    }
    mfma_settle();
    if constexpr (WK > 1) {
        if (wave) {
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) part[((wave - 1u) * NT + f) * 64u + lane] = acc[f];
        }
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (uint32_t v = 0; v + 1u < WK; v++)
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) acc[f] += part[(v * NT + f) * 64u + lane];
    }
    if (src < 0) return;
    const int64_t dst = dst_row(a, p);
    if (dst < 0) return;
#pragma unroll
    for (uint32_t f = 0; f < NT; f++) st_four<TW>(a, dst, n0 + 16u * f + 4u * q, acc[f]);
}

#define RFXQ_GROUPED_FEW(name, TX, TW)                                                                                  \
    extern "C" __global__ __launch_bounds__(256) void rfxq_grouped_few_##name(GroupedArgs a) { grouped_few<TX, TW, 2, 1>(a); } \
    extern "C" __global__ __launch_bounds__(256) void rfxq_grouped_few4_##name(GroupedArgs a) { grouped_few<TX, TW, 1, 4>(a); }
RFXQ_GROUPED_FEW(f16, half_t, half_t)
RFXQ_GROUPED_FEW(bf16, __bf16, __bf16)
RFXQ_GROUPED_FEW(f32_f16, float, half_t)
RFXQ_GROUPED_FEW(f32_bf16, float, __bf16)
