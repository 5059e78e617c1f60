// Tiles of rfxq_gemm_f8 and rfxq_grouped_gemm_f8 filled by asynchronous copies
// (f8_gemm.hpp has the formula, and the kernels of the rest).
//
// What bounds them, a CU: the instruction of 16 x 16 x 128 takes 33 cycles, 35 with its four
// multiply-adds beside it and two waves a SIMD (4.1 PFLOP/s in all at 2.1 GHz); LDS
// gives 239 bytes a cycle to 8 waves (124 to 4), copies bring 63. A 256 x 256 tile takes 2240
// cycles of instructions for a block of K, 800 of LDS (192 KB) and 1040 of copies (64 KB): large tiles are bound by
// the instructions and by what holds their issue up, small ones by their operands' LDS reads, by the copies' writes
// there and by the barrier of a step.
#pragma once
#include "f8_gemm.hpp"

// dma16 to LDS address `lds` with an offset that all lanes share, and unseen by the compiler's wait counting: it
// takes LDS reads of one buffer to depend on copies into another and waits for
// them. Whoever calls it waits with wait_copies, and has no other load from memory in
// flight that the compiler would wait for. The buffer's end is checked for each dword, the shared offset
// included: dwords behind it are zeros.
RFXQ_DEV void copy16(rsrc_t r, uint32_t lds, uint32_t off, uint32_t by) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(r), "s"(by)
                 : "memory", "m0");
}
// all of the wave's copies but the last N have landed
template <uint32_t N>
RFXQ_DEV void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// acc += d * scale, here: the compiler would keep the products of a whole step in registers
// and add them after it.
RFXQ_DEV void add_scaled(f4v_t& acc, f4v_t d, float scale) {
#pragma unroll
    for (uint32_t e = 0; e < 4u; e++) acc[e] = __builtin_fmaf(d[e], scale, acc[e]);
    asm volatile("" : "+v"(acc));
}

// What both kinds of tiles share: the tile, and copies of steps of DEPTH blocks of K, [block]
// [row] of 128 bytes. Copies go global -> LDS without registers between. Rows of x
// and W start at whole 16 bytes; what lies past a row's end or the tile's last
// row is copied from past the buffer's end, which fills it with zeros. Offsets within x and
// within one matrix stay below 4 GiB (the host's rule).
template <bool GROUPED, uint32_t BM, uint32_t BN, uint32_t DEPTH>
struct F8Tile {
    static constexpr uint32_t WAVES = 8, NX = BM * DEPTH * 8u / (64u * WAVES), NW = BN * DEPTH * 8u / (64u * WAVES);
    static constexpr uint32_t PAST = 0xFFFFFFF0u;
    static_assert(NX >= 1 && NW >= 1 && BM * DEPTH % 64u == 0 && NX % DEPTH == 0 && NW % DEPTH == 0);

    RowTile t;
    rsrc_t xr, wr;
    uint32_t xo[NX / DEPTH], wo[NW / DEPTH];  // lanes' byte offsets at k = 0
    uint32_t lane, wave, piece, tn, n0, k, blocks;
    uint32_t at = 0;  // of the next step to copy
    const float* sw;  // the tile's first block of columns

    // The wave's copies [from, to) of a step: of each NX (NW), NX / DEPTH in each block.
    __device__ __forceinline__ void issue_x(uint32_t xs, uint32_t from, uint32_t to) {
        issue<NX, BM>(xr, xo, xs, from, to);
    }
    __device__ __forceinline__ void issue_w(uint32_t ws, uint32_t from, uint32_t to) {
        issue<NW, BN>(wr, wo, ws, from, to);
    }
    template <uint32_t COUNT, uint32_t ROWS>
    __device__ __forceinline__ void issue(rsrc_t r, const uint32_t (&o)[COUNT / DEPTH], uint32_t lds, uint32_t from,
                                          uint32_t to) {
        constexpr uint32_t EACH = COUNT / DEPTH;
#pragma unroll
        for (uint32_t i = from; i < to; i++) {
            const uint32_t b = i / EACH, j = i % EACH, k0 = at + kBlock * b;
            // past the end: as many copies, of zeros, so that waits count the same
            const bool there = k0 + kBlock <= k || k0 + 16u * piece < k;
            copy16(r, lds + 128u * ROWS * b + 1024u * (wave * EACH + j), there ? o[j] : PAST, k0 < k ? k0 : 0u);
        }
    }

    // the tile, and where its rows are; false: there is none
    __device__ __forceinline__ bool begin(const F8Args& a) {
        uint32_t tm;
        if (!f8_place(a, tm, tn)) return false;
        t = f8_tile<GROUPED>(a, BM, tm);
        if (!t.any) return false;
        lane = threadIdx.x & 63u;
        n0 = tn * BN;
        wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
        piece = (lane & 7u) ^ (lane >> 3);
        k = a.k;
        blocks = (k + kBlock - 1u) / kBlock;
        xr = make_rsrc(a.x, (uint32_t)((uint64_t)(a.x_rows - 1u) * a.ldx + k));
        wr = make_rsrc(a.w + (uint64_t)t.group * a.w_stride, (uint32_t)a.w_stride);
        sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)(n0 / kBlock) * blocks;
#pragma unroll
        for (uint32_t j = 0; j < NX / DEPTH; j++) {
            const uint32_t p = t.beg + (wave * (NX / DEPTH) + j) * 8u + (lane >> 3);
            const int64_t s = p < t.end ? f8_src<GROUPED>(a, p) : -1;
            xo[j] = s < 0 ? PAST : (uint32_t)((uint64_t)s * a.ldx) + 16u * piece;
        }
#pragma unroll
        for (uint32_t j = 0; j < NW / DEPTH; j++) {
            const uint32_t n = n0 + col_of<>((wave * (NW / DEPTH) + j) * 8u + (lane >> 3));
            wo[j] = n < a.n ? n * k + 16u * piece : PAST;
        }
        return true;
    }

    // Scales of the tile's rows for blocks [b0, b0 + COUNT), [block][row], with those of
    // its columns where they are one block's (BN = 128). Blocks past the last
    // have zeros: an infinite scale would make NaN of their products.
    template <uint32_t COUNT>
    __device__ __forceinline__ void stage_scales(const F8Args& a, float* ss, uint32_t b0) {
        constexpr uint32_t PER = COUNT / 4u;
#pragma unroll 1
        for (uint32_t j = threadIdx.x; j < BM * PER; j += 64u * WAVES) {
            const uint32_t r = j / PER, b = 4u * (j % PER);
            const int64_t src = f8_src<GROUPED>(a, min(t.beg + r, t.end - 1u));
            const float* p = a.xs + (src < 0 ? 0 : (uint64_t)src * a.ldxs);
            float v[4];
#pragma unroll
            for (uint32_t e = 0; e < 4u; e++) {
                const uint32_t at_block = min(b0 + b + e, blocks - 1u);
                v[e] = ((const RFXQ_GLOBAL float*)p)[at_block];
                if constexpr (BN == kBlock) v[e] *= ((const RFXQ_GLOBAL float*)sw)[at_block];
                if (b0 + b + e >= blocks) v[e] = 0.0f;
            }
#pragma unroll
            for (uint32_t e = 0; e < 4u; e++) ss[(b + e) * BM + r] = v[e];
        }
    }

    // One row of 16 columns from n on.
    __device__ __forceinline__ void out_row(const F8Args& a, uint32_t row, uint32_t n, const f4v_t (&acc)[4]) {
        const uint32_t p = t.beg + row;
        if (p >= t.end) return;
        const int64_t src = f8_src<GROUPED>(a, p), dst = f8_dst<GROUPED>(a, p);
        if (src >= 0 && dst >= 0) f8_out(a, dst, n, acc);
    }
};

// ---------------------------------------------------------------- 64 x 128 and 128 x 128

// 8 waves: four of 16 MF x 64 results take the even blocks of K, four the odd ones,
// and they add their parts in LDS. Buffers of two blocks, copies STAGES - 1 steps ahead, a
// barrier a step. 512 x 14336 x 4096, half results: 40 us in 64 x 128 tiles, one a CU (1.5 PFLOP/s, a
// third of the instructions' rate; 33 bytes of copies a cycle and CU); 1000 x 4096 x 4096 in 128 x 128: 23 us. f32
// results 64 and 38 us: their codes are widened, their instructions run at half the rate. Tried: operands
// read from LDS a step ahead (no gain), 64 x 64 tiles of four blocks a step (256 x 4096 x 4096: 12.7 us, 64 x 128
// 13.4; f32 16.7 and 22.4, but two rounds of them 28.6), weights straight to registers (4096 x 4096 x 14336:
// 354 us), a ring of six buffers of one block filled by four waves that only copy (45 us for 40: lines take
// 400 cycles and are there in time; the operands' 64 KB of LDS reads a block, and a barrier for each, are not).
template <uint32_t MF, uint32_t STAGES, bool EXACT, bool GROUPED>
RFXQ_DEV void f8_mid(const F8Args& a) {
    constexpr uint32_t BM = 32u * MF, BN = 128, D = 2, CHUNK = 32;  // CHUNK: blocks whose scales are in LDS
    typedef F8Tile<GROUPED, BM, BN, D> Tile;
    constexpr uint32_t COPIES = Tile::NX + Tile::NW;
    __shared__ u4_t xs0[BM * D * 8], xs1[BM * D * 8], xs2[STAGES > 2 ? BM * D * 8 : 1];
    __shared__ u4_t ws0[BN * D * 8], ws1[BN * D * 8], ws2[STAGES > 2 ? BN * D * 8 : 1];
    __shared__ float ss[CHUNK * BM];
    Tile t;
    if (!t.begin(a)) return;
    const uint32_t lane = t.lane, l = lane & 15u, q = lane >> 4, half = t.wave >> 2;
    const uint32_t row0 = (t.wave >> 1 & 1u) * 16u * MF, col0 = (t.wave & 1u) * 64u, steps = (t.blocks + D - 1u) / D;
    const uint32_t x0 = half * BM * 8u + lds_piece(row0 + l, q), x1 = half * BM * 8u + lds_piece(row0 + l, 4u + q);
    const uint32_t w0 = half * BN * 8u + lds_piece(col0 + l, q), w1 = half * BN * 8u + lds_piece(col0 + l, 4u + q);
    f4v_t acc[MF][4] = {};
    const auto issue = [&](const u4_t* xs, const u4_t* ws) {
        t.issue_x(lds_addr(xs), 0, Tile::NX);
        t.issue_w(lds_addr(ws), 0, Tile::NW);
        t.at += kBlock * D;
    };
    const auto step = [&](uint32_t s, const u4_t* xs, const u4_t* ws, const u4_t* nx, const u4_t* nw) {
        wait_copies<COPIES * (STAGES - 2u)>();  // but the next steps'
        if (D * s % CHUNK == 0 && s) {
            lds_barrier();
            t.template stage_scales<CHUNK>(a, ss, D * s);
        }
        __builtin_amdgcn_sched_barrier(0);
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const float* sc = ss + (D * s % CHUNK + half) * BM + row0 + l;
        Operand<EXACT> wf[4], xf[2];
        float scale[2];
        u4_t xv[2][2];
        const auto read_x = [&](uint32_t m) {
            xv[m & 1u][0] = xs[x0 + 128u * m];
            xv[m & 1u][1] = xs[x1 + 128u * m];
            scale[m & 1u] = sc[16u * m];
        };
        read_x(0);
#pragma unroll
        for (uint32_t f = 0; f < 4u; f++) wf[f].take(ws[w0 + 128u * f], ws[w1 + 128u * f]);
        f4v_t d[4];
        float sm[2];
#pragma unroll
        for (uint32_t i = 0; i < 4u * MF + 2u; i++) {
            const uint32_t m = i >> 2;
            if (i < 4u * MF && (i & 3u) == 0) {
                xf[m & 1u].take(xv[m & 1u][0], xv[m & 1u][1]);
                sm[m & 1u] = scale[m & 1u];
                if (m + 1u < MF) read_x(m + 1u);
            }
            if (i < 4u * MF) d[i & 3u] = multiply(wf[i & 3u], xf[m & 1u]);
            __builtin_amdgcn_sched_barrier(0);
            // copies one by one: their issue holds a wave up
            if (i < Tile::NX) t.issue_x(lds_addr(nx), i, i + 1u);
            if (i >= Tile::NX && i < COPIES) t.issue_w(lds_addr(nw), i - Tile::NX, i - Tile::NX + 1u);
            if (i >= 2u) {
                const uint32_t j = i - 2u;
                add_scaled(acc[j >> 2][j & 3u], d[j & 3u], sm[(j >> 2) & 1u]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        static_assert(COPIES <= 4u * MF);
        t.at += kBlock * D;
    };
    issue(xs0, ws0);
    if constexpr (STAGES == 3) issue(xs1, ws1);
    t.template stage_scales<CHUNK>(a, ss, 0);
    if constexpr (STAGES == 3) {
        for (uint32_t s = 0; s < steps; s += 3u) {
            step(s, xs0, ws0, xs2, ws2);
            if (s + 1u < steps) step(s + 1u, xs1, ws1, xs0, ws0);
            if (s + 2u < steps) step(s + 2u, xs2, ws2, xs1, ws1);
        }
    } else {
        for (uint32_t s = 0; s < steps; s += 2u) {
            step(s, xs0, ws0, xs1, ws1);
            if (s + 1u < steps) step(s + 1u, xs1, ws1, xs0, ws0);
        }
    }
    wait_copies<0>();
    lds_barrier();  // nothing is read or copied any more: the buffers hold the parts
    f4v_t* part = reinterpret_cast<f4v_t*>(xs0);
    static_assert(sizeof xs0 >= 4u * 64u * (MF / 2u) * 4u * sizeof(f4v_t));
    // the even blocks' waves store the first half of the rows, the odd ones' the second: each passes the other on
    f4v_t* mine = part + (t.wave & 3u) * (MF / 2u) * 256u + lane;
    const auto pass = [&](auto first) {
#pragma unroll
        for (uint32_t m = 0; m < MF / 2u; m++)
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) mine[(4u * m + f) * 64u] = acc[decltype(first)::value + m][f];
    };
    const auto add = [&](auto first) {
        constexpr uint32_t F = decltype(first)::value;
#pragma unroll
        for (uint32_t m = 0; m < MF / 2u; m++) {
#pragma unroll
            for (uint32_t f = 0; f < 4u; f++) {
                const f4v_t other = mine[(4u * m + f) * 64u];
                acc[F + m][f] = F ? other + acc[F + m][f] : acc[F + m][f] + other;  // even blocks + odd ones
            }
            t.out_row(a, row0 + 16u * (F + m) + l, t.n0 + col0 + 16u * q, acc[F + m]);
        }
    };
    if (half) pass(Count<0>{});
    lds_barrier();
    if (!half) add(Count<0>{});
    lds_barrier();
    if (!half) pass(Count<MF / 2u>{});
    lds_barrier();
    if (half) add(Count<MF / 2u>{});
}

#define RFXQ_F8_MID(BM, STAGES, name, EXACT)                                                                        \
    extern "C" __global__ __launch_bounds__(512) void rfxq_f8_##BM##_##name(F8Args a) {                             \
        f8_mid<BM / 32, STAGES, EXACT, false>(a);                                                                   \
    }                                                                                                               \
    extern "C" __global__ __launch_bounds__(512) void rfxq_f8_##BM##_##name##_grouped(F8Args a) {                   \
        f8_mid<BM / 32, STAGES, EXACT, true>(a);                                                                    \
    }
RFXQ_F8_MID(64, 3, half, false)
RFXQ_F8_MID(64, 3, f32, true)
RFXQ_F8_MID(128, 2, half, false)
RFXQ_F8_MID(128, 2, f32, true)

// ---------------------------------------------------------------- 128 x 256 and 256 x 256, half results

// 8 waves of 16 MF x 64. A step is a block of K: its weights are in registers from its start, its
// activations come from LDS two 16-row operands ahead of their products; at MF - 2
// of them all reads of the step are done and the next step's copies have landed (the one
// barrier). 4096 x 4096 x 14336: 217 us, 2.2 PFLOP/s (128 x 256: 237; a library's product with one
// scale a tensor: 200); instructions 59% busy at 8192^3, 3.5 rounds of tiles over the CUs done as 4.
// 128 x 256 has three stages, for 256 x 256 two fill the LDS. Tried: two workgroups of 128 x 128 a CU
// (283 us), operands that two waves take in turns (311), 192 x 256 tiles.
template <uint32_t MF, uint32_t STAGES, bool GROUPED>
RFXQ_DEV void f8_large(const F8Args& a) {
    constexpr uint32_t BM = 32u * MF, BN = 256;
    typedef F8Tile<GROUPED, BM, BN, 1> Tile;
    __shared__ u4_t xs0[BM * 8], xs1[BM * 8], xs2[STAGES > 2 ? BM * 8 : 1];
    __shared__ u4_t ws0[BN * 8], ws1[BN * 8], ws2[STAGES > 2 ? BN * 8 : 1];
    __shared__ float ss[2][BM][4];  // of four blocks, and of the next four
    Tile t;
    if (!t.begin(a)) return;
    const uint32_t lane = t.lane, l = lane & 15u, q = lane >> 4, steps = t.blocks;
    const uint32_t row0 = (t.wave >> 2) * 16u * MF, col0 = (t.wave & 3u) * 64u;
    f4v_t acc[MF][4] = {};
    // columns past the last: any scale
    const uint64_t first_w =
        reinterpret_cast<uint64_t>(t.sw + (t.n0 + col0 < a.n ? (uint64_t)(col0 / kBlock) * steps : 0u));
    const __attribute__((address_space(4))) float* s_w = (const __attribute__((address_space(4))) float*)(
        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)first_w) |
        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(first_w >> 32)) << 32);
    float s_next = s_w[0];
    Operand<false> wf[4];
    u4_t xv[3][2];
    float sx[3];
    // pieces of a lane's rows: every 16th row has the same ones
    const uint32_t p0 = lds_piece(row0 + l, q), p1 = lds_piece(row0 + l, 4u + q), pr = row0 + l;
    const uint32_t w0 = lds_piece(col0 + l, q), w1 = lds_piece(col0 + l, 4u + q);
    const auto read_x = [&](const u4_t* xs, uint32_t b, uint32_t m, uint32_t to) {
        xv[to][0] = xs[p0 + 128u * m];
        xv[to][1] = xs[p1 + 128u * m];
        sx[to] = ss[b >> 2 & 1u][pr + 16u * m][b & 3u];
    };
    // scales of four blocks, a row a lane; rows past the tile's last are not used
    const rsrc_t sr = make_rsrc(a.xs, (uint32_t)(4u * ((uint64_t)(a.x_rows - 1u) * a.ldxs + steps)));
    uint32_t so = Tile::PAST;
    if (t.wave < BM / 64u) {
        const int64_t src = f8_src<GROUPED>(a, min(t.t.beg + t.wave * 64u + lane, t.t.end - 1u));
        so = src < 0 ? Tile::PAST : (uint32_t)((uint64_t)src * a.ldxs * 4u);
    }
    const auto copy_scales = [&](uint32_t c) {
        const bool there = 4u * c < steps;
        if (t.wave < BM / 64u)
            copy16(sr, lds_addr(ss) + 16u * ((c & 1u) * BM + 64u * t.wave), there ? so : Tile::PAST, there ? 16u * c : 0u);
    };
    const auto read_w = [&](const u4_t* ws, uint32_t f) { wf[f].take(ws[w0 + 128u * f], ws[w1 + 128u * f]); };
    const auto step = [&](uint32_t s, const u4_t* xs, const u4_t* xn, const u4_t* wn, const u4_t* xc, const u4_t* wc,
                          auto first) {
        constexpr uint32_t r0 = decltype(first)::value, LAST = 4u * MF, SYNC = 4u * (MF - 2u);
        constexpr uint32_t COPIES = Tile::NX + Tile::NW;  // r0: where the first rows are
        static_assert(2u * COPIES <= LAST);
        const float s_col = s_next;
        Operand<false> xf;
        f4v_t d[4];
        float scale[2];
#pragma unroll
        for (uint32_t i = 0; i < LAST + 2u; i++) {
            const uint32_t m = i >> 2;
            if (i < LAST && (i & 3u) == 0) {
                scale[m & 1u] = sx[(r0 + m) % 3u] * s_col;
                xf.take(xv[(r0 + m) % 3u][0], xv[(r0 + m) % 3u][1]);
                if (i == SYNC) {
                    wait_copies<STAGES == 3 ? (SYNC / 2u < COPIES ? SYNC / 2u : COPIES) : 0u>();
                    __builtin_amdgcn_sched_barrier(0);
                    lds_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                    s_next = s_w[min(s + 1u, steps - 1u)];
                }
                if (i < SYNC)
                    read_x(xs, s, m + 2u, (r0 + m + 2u) % 3u);
                else
                    read_x(xn, s + 1u, m + 2u - MF, (r0 + m + 2u) % 3u);
            }
            // copies one by one: their issue holds a wave up
            if constexpr (STAGES == 3) {
                constexpr uint32_t NX = Tile::NX;
                if ((i & 1u) == 0 && i < 2u * NX) t.issue_x(lds_addr(xc), i / 2u, i / 2u + 1u);
                if ((i & 1u) == 0 && i >= 2u * NX && i < 2u * COPIES)
                    t.issue_w(lds_addr(wc), i / 2u - NX, i / 2u - NX + 1u);
                if (i + 2u == 2u * COPIES) t.at += kBlock;
            } else {
                if (i < 2u * Tile::NW && (i & 1u) == 0) {
                    t.issue_w(lds_addr(wc), i / 2u, i / 2u + 1u);
                    if (i / 2u + 1u == Tile::NW) t.at += kBlock;
                }
                if (i >= SYNC && i < SYNC + 2u * Tile::NX && (i & 1u) == 0)
                    t.issue_x(lds_addr(xc), (i - SYNC) / 2u, (i - SYNC) / 2u + 1u);
            }
            if (i == LAST - 1u && (s & 3u) == 0) copy_scales(s / 4u + 1u);
            if (i < LAST) d[i & 3u] = multiply(wf[i & 3u], xf);
            __builtin_amdgcn_sched_barrier(0);
            if (i >= LAST - 4u && i < LAST) read_w(wn, i + 4u - LAST);  // behind its last product of the step
            if (i >= 2u) {
                const uint32_t j = i - 2u;
                add_scaled(acc[j >> 2][j & 3u], d[j & 3u], scale[(j >> 2) & 1u]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    t.issue_x(lds_addr(xs0), 0, Tile::NX);
    t.issue_w(lds_addr(ws0), 0, Tile::NW);
    t.at += kBlock;
    copy_scales(0);
    t.issue_x(lds_addr(xs1), 0, Tile::NX);
    if constexpr (STAGES == 3) {
        t.issue_w(lds_addr(ws1), 0, Tile::NW);
        t.at += kBlock;
    }
    wait_copies<STAGES == 3 ? Tile::NX + Tile::NW : Tile::NX>();
    lds_barrier();
#pragma unroll
    for (uint32_t f = 0; f < 4u; f++) read_w(ws0, f);
    read_x(xs0, 0, 0, 0);
    read_x(xs0, 0, 1, 1);
    for (uint32_t s = 0; s < steps; s += 6u) {
        if constexpr (STAGES == 3) {
            step(s, xs0, xs1, ws1, xs2, ws2, Count<0>{});
            if (s + 1u < steps) step(s + 1u, xs1, xs2, ws2, xs0, ws0, Count<MF % 3u>{});
            if (s + 2u < steps) step(s + 2u, xs2, xs0, ws0, xs1, ws1, Count<2u * MF % 3u>{});
            if (s + 3u < steps) step(s + 3u, xs0, xs1, ws1, xs2, ws2, Count<0>{});
            if (s + 4u < steps) step(s + 4u, xs1, xs2, ws2, xs0, ws0, Count<MF % 3u>{});
            if (s + 5u < steps) step(s + 5u, xs2, xs0, ws0, xs1, ws1, Count<2u * MF % 3u>{});
        } else {
            step(s, xs0, xs1, ws1, xs0, ws1, Count<0>{});
            if (s + 1u < steps) step(s + 1u, xs1, xs0, ws0, xs1, ws0, Count<MF % 3u>{});
            if (s + 2u < steps) step(s + 2u, xs0, xs1, ws1, xs0, ws1, Count<2u * MF % 3u>{});
            if (s + 3u < steps) step(s + 3u, xs1, xs0, ws0, xs1, ws0, Count<0>{});
            if (s + 4u < steps) step(s + 4u, xs0, xs1, ws1, xs0, ws1, Count<MF % 3u>{});
            if (s + 5u < steps) step(s + 5u, xs1, xs0, ws0, xs1, ws0, Count<2u * MF % 3u>{});
        }
    }
    wait_copies<0>();  // no copy outlives the workgroup
#pragma unroll
    for (uint32_t m = 0; m < MF; m++) t.out_row(a, row0 + 16u * m + l, t.n0 + col0 + 16u * q, acc[m]);
}

#define RFXQ_F8_LARGE(BM, STAGES)                                                                                   \
    extern "C" __global__ __launch_bounds__(512) void rfxq_f8_##BM##_wide(F8Args a) {                               \
        f8_large<BM / 32, STAGES, false>(a);                                                                        \
    }                                                                                                               \
    extern "C" __global__ __launch_bounds__(512) void rfxq_f8_##BM##_wide_grouped(F8Args a) {                       \
        f8_large<BM / 32, STAGES, true>(a);                                                                         \
    }
RFXQ_F8_LARGE(256, 2)
RFXQ_F8_LARGE(128, 3)
