// Few rows of rfxq_gemm_f8 and rfxq_grouped_gemm_f8 (f8_gemm.hpp has the formula).
#pragma once
#include "f8_tile.hpp"

// Up to 16 MT rows of a tile, 16 NT columns: the weights' bytes are all that counts.
// A workgroup's WAVES waves take every WAVES-th block of K each (neighbouring blocks are on
// their way together) for all of its results and add their parts in LDS.
// Each wave copies its own operands into its own R places in LDS, R blocks ahead, and waits
// for nobody. Whole lines by copies: 63 bytes a cycle and CU, where loads in the order of an instruction's
// operands take 16. 1 x 4096 x 14336: 11.4 us, 5.2 TB/s of weights (a large copy: 4.87);
// 1 x 4096 x 4096: 6.3; 32 tokens over 8 of 128 experts, 2048 x 768: 31 us for the 118 MB of the 75 experts
// that have rows, 3.8 TB/s (26 where a call finds part of them in the memory-side cache). More columns a workgroup read x less often, fewer make more
// workgroups; the host's table has what each measured. 32 x 64 and 64 x 64 tiles are for 33 to some 256 rows,
// whose copies and products bound: 128 x 14336 x 4096 21 us for half results and 23 for f32 ones, 256 rows 29 and 35. (The
// smaller tiles gain less by the instruction of 128, 64 rows in 32 x 32 16.4 us for 17.0, and have
// exact products for all results.)
template <uint32_t MT, uint32_t NT, uint32_t R, uint32_t WAVES, bool EXACT, bool GROUPED>
RFXQ_DEV void f8_stream(const F8Args& a) {
    constexpr uint32_t CHUNK = 64;  // blocks whose scales are in LDS
    constexpr uint32_t PER = MT + NT, COPIES = 2u * PER, PAST = 0xFFFFFFF0u;
    __shared__ u4_t ring[WAVES][R][PER][128];
    __shared__ float ss[CHUNK][16 * MT];
    static_assert(sizeof ring >= WAVES * MT * NT * 64u * sizeof(f4v_t));
    uint32_t tm, tn;
    if (!f8_place(a, tm, tn)) return;
    const RowTile t = f8_tile<GROUPED>(a, 16u * MT, tm);
    if (!t.any) return;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63u, l = lane & 15u, q = lane >> 4, n0 = tn * 16u * NT;
    const uint32_t blocks = (a.k + kBlock - 1u) / kBlock, piece = (lane & 7u) ^ (lane >> 3);
    const rsrc_t xr = make_rsrc(a.x, (uint32_t)((uint64_t)(a.x_rows - 1u) * a.ldx + a.k));
    const rsrc_t wr = make_rsrc(a.w + (uint64_t)t.group * a.w_stride, (uint32_t)a.w_stride);
    const float* sw = a.ws + (uint64_t)t.group * a.ws_stride + (uint64_t)(n0 / kBlock) * blocks;
    uint32_t wo[2 * NT], xo[2 * MT];  // lanes' byte offsets at k = 0: 8 rows a copy
#pragma unroll
    for (uint32_t j = 0; j < 2u * NT; j++) {
        const uint32_t n = n0 + 8u * j + (lane >> 3);
        wo[j] = n < a.n ? n * a.k + 16u * piece : PAST;
    }
    const auto copy_w = [&](uint32_t to, uint32_t b) {
        const bool there = (b + 1u) * kBlock <= a.k || (b < blocks && b * kBlock + 16u * piece < a.k);
#pragma unroll
        for (uint32_t j = 0; j < 2u * NT; j++)
            copy16(wr, lds_addr(ring) + 16u * (((wave * R + to) * PER) * 128u + 64u * j), there ? wo[j] : PAST,
                   b < blocks ? b * kBlock : 0u);
    };
    const auto copy_x = [&](uint32_t to, uint32_t b) {
        const bool there = (b + 1u) * kBlock <= a.k || (b < blocks && b * kBlock + 16u * piece < a.k);
#pragma unroll
        for (uint32_t j = 0; j < 2u * MT; j++)
            copy16(xr, lds_addr(ring) + 16u * (((wave * R + to) * PER + NT) * 128u + 64u * j), there ? xo[j] : PAST,
                   b < blocks ? b * kBlock : 0u);
    };
#pragma unroll
    for (uint32_t j = 0; j < 2u * MT; j++) {
        const uint32_t p = t.beg + 8u * j + (lane >> 3);
        const int64_t s = p < t.end ? f8_src<GROUPED>(a, p) : -1;
        xo[j] = s < 0 ? PAST : (uint32_t)((uint64_t)s * a.ldx) + 16u * piece;
    }
    const auto stage_scales = [&](uint32_t b0) {
        const uint32_t count = min(CHUNK, blocks - b0);
        for (uint32_t j = threadIdx.x; j < count * 16u * MT; j += 64u * WAVES) {
            const uint32_t r = j / count, b = j % count;
            const int64_t src = f8_src<GROUPED>(a, min(t.beg + r, t.end - 1u));
            ss[b][r] = ((const RFXQ_GLOBAL float*)a.xs)[(src < 0 ? 0 : (uint64_t)src * a.ldxs) + b0 + b] *
                       ((const RFXQ_GLOBAL float*)sw)[b0 + b];
        }
    };
    stage_scales(0);
#pragma unroll
    for (uint32_t i = 0; i < R; i++) {
        copy_w(i, wave + WAVES * i);
        copy_x(i, wave + WAVES * i);
    }
    lds_barrier();
    f4v_t acc[MT][NT] = {};
    const uint32_t p0 = lds_piece(l, q), p1 = lds_piece(l, 4u + q);
    const auto block = [&](uint32_t at, uint32_t b) {
        wait_copies<COPIES*(R - 1u)>();
        u4_t raw[PER][2];
        float scale[MT];
#pragma unroll
        for (uint32_t j = 0; j < PER; j++) {
            raw[j][0] = ring[wave][at][j][p0];
            raw[j][1] = ring[wave][at][j][p1];
        }
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) scale[m] = ss[b % CHUNK][16u * m + l];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before they are copied over
        __builtin_amdgcn_sched_barrier(0);
        copy_w(at, b + WAVES * R);
        copy_x(at, b + WAVES * R);
        Operand<EXACT> wf[NT];
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) wf[f].take(raw[f][0], raw[f][1]);
#pragma unroll
        for (uint32_t m = 0; m < MT; m++) {
            Operand<EXACT> xf;
            xf.take(raw[NT + m][0], raw[NT + m][1]);
            f4v_t d[NT];
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) d[f] = multiply(wf[f], xf);
#pragma unroll
            for (uint32_t f = 0; f < NT; f++) acc[m][f] += d[f] * scale[m];
        }
    };
    for (uint32_t b0 = 0; b0 < blocks; b0 += CHUNK) {
        if (b0) {
            lds_barrier();
            stage_scales(b0);
            lds_barrier();
        }
        static_assert(CHUNK % (WAVES * R) == 0);
        for (uint32_t b = b0 + wave; b < min(b0 + CHUNK, blocks); b += WAVES * R) {
            block(0, b);
#pragma unroll
            for (uint32_t i = 1; i < R; i++)
                if (b + WAVES * i < blocks) block(i, b + WAVES * i);
        }
    }
    wait_copies<0>();
    __syncthreads();
    f4v_t* part = reinterpret_cast<f4v_t*>(ring);
#pragma unroll
    for (uint32_t m = 0; m < MT; m++)
#pragma unroll
        for (uint32_t f = 0; f < NT; f++) part[(wave * MT * NT + m * NT + f) * 64u + lane] = acc[m][f];
    __syncthreads();
    for (uint32_t i = wave; i < MT * NT; i += WAVES) {
        f4v_t sum[1] = {part[i * 64u + lane]};
#pragma unroll
        for (uint32_t v = 1; v < WAVES; v++) sum[0] += part[(v * MT * NT + i) * 64u + lane];
        const uint32_t p = t.beg + 16u * (i / NT) + l;
        if (p >= t.end) continue;
        const int64_t src = f8_src<GROUPED>(a, p), dst = f8_dst<GROUPED>(a, p);
        if (src >= 0 && dst >= 0) f8_out(a, dst, n0 + 16u * (i % NT) + 4u * q, sum);
    }
}

// the last four for one matrix: grouped rows, of which tiles end early, took 1.1 to 1.7 times as long with them
#define RFXQ_F8_STREAM(MT, NT, R, WAVES)                                                                            \
    extern "C" __global__ __launch_bounds__(64 * WAVES) void rfxq_f8_stream_##MT##_##NT##_##R##_##WAVES(F8Args a) {     \
        f8_stream<MT, NT, R, WAVES, true, false>(a);                                                                \
    }                                                                                                               \
    extern "C" __global__                                                                                           \
        __launch_bounds__(64 * WAVES) void rfxq_f8_stream_##MT##_##NT##_##R##_##WAVES##_grouped(F8Args a) {         \
        f8_stream<MT, NT, R, WAVES, true, true>(a);                                                                 \
    }
#define RFXQ_F8_STREAM1(MT, NT, name, EXACT)                                                                        \
    extern "C" __global__ __launch_bounds__(512) void rfxq_f8_stream_##MT##_##NT##_##name(F8Args a) {               \
        f8_stream<MT, NT, 1, 8, EXACT, false>(a);                                                                   \
    }
RFXQ_F8_STREAM(1, 1, 2, 8)
RFXQ_F8_STREAM(1, 2, 1, 8)
RFXQ_F8_STREAM(2, 2, 1, 8)
RFXQ_F8_STREAM(1, 4, 1, 4)
RFXQ_F8_STREAM1(2, 4, half, false)
RFXQ_F8_STREAM1(2, 4, f32, true)
RFXQ_F8_STREAM1(4, 4, half, false)
RFXQ_F8_STREAM1(4, 4, f32, true)
