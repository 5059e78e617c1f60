// What half.hip and f8.hip share: the search for the tile a workgroup computes, the places
// of tiles, rows and LDS pieces, vectors of a row's values. `Args`: the arguments of either's kernels.
#pragma once
#include "common.hpp"

// Inclusive sum over the wave's lanes: within 16-lane rows by row shifts, then
// the rows' last lanes carried over (row_bcast 15 and 31).
RFXQ_DEV uint32_t wave_scan(uint32_t v) {
#define RFXQ_SCAN(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, (ctrl), (rows), 0xF, false)
    RFXQ_SCAN(0x111, 0xF);
    RFXQ_SCAN(0x112, 0xF);
    RFXQ_SCAN(0x114, 0xF);
    RFXQ_SCAN(0x118, 0xF);
    RFXQ_SCAN(0x142, 0xA);
    RFXQ_SCAN(0x143, 0xC);
#undef RFXQ_SCAN
    return v;
}

// The rows [beg, end) of one tile of at most `bm` rows, all of one group; where
// there is none (any = false), `beg` is the tile's number behind the last one.
struct RowTile {
    uint32_t group, beg, end;
    int32_t extra;
    bool any;
};

template <uint32_t N>
struct Count {
    static constexpr uint32_t value = N;
};

// Tile t of the grouped rows: the groups' tiles counted in order, each group
// starting a tile of its own. Every wave searches by itself (no LDS, no
// barrier), a group a lane: the offsets of up to 256 groups are one trip to memory,
// which every kernel here waits for before it knows what to read (with neighbouring
// groups in a lane it is two and more: a token over 8 of 128 experts, 768 x 2048, 8.4 us
// against 7.5).
// Offsets are taken as they are found: clamped to [0, rows], and a group
// whose end lies before its start has no tiles, so that no value there leads
// outside the arrays. `extra`: a value per group, returned for the tile's.
RFXQ_DEV RowTile find_tile(const int32_t* offsets, uint32_t groups, uint32_t rows, uint32_t bm, uint32_t t,
                           const int32_t* extra = nullptr) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t before = 0;  // tiles of the groups looked at
    RowTile r = {0, 0, 0, 0, false};
    const auto look = [&](auto n, uint32_t g0) {
        constexpr uint32_t N = decltype(n)::value;
        int32_t b[N], e[N], x[N];
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            const uint32_t g = g0 + 64u * i + lane;
            b[i] = ((const RFXQ_GLOBAL int32_t*)offsets)[min(g, groups)];
            e[i] = ((const RFXQ_GLOBAL int32_t*)offsets)[min(g + 1u, groups)];
            x[i] = extra ? ((const RFXQ_GLOBAL int32_t*)extra)[min(g, groups - 1u)] : 0;
        }
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            const uint32_t bi = min((uint32_t)max(b[i], 0), rows), ei = min((uint32_t)max(e[i], 0), rows);
            const uint32_t mine = ei > bi ? (ei - bi + bm - 1u) / bm : 0u;
            const uint32_t upto = before + wave_scan(mine);
            const uint64_t has = __builtin_amdgcn_ballot_w64(upto > t);
            if (has) {
                const int l = __builtin_ctzll(has);
                const uint32_t left = t - (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), l);
                if (left >= (uint32_t)__builtin_amdgcn_readlane((int)mine, l)) return;  // a sum that wrapped
                const uint32_t end = (uint32_t)__builtin_amdgcn_readlane((int)ei, l);
                r.group = g0 + 64u * i + (uint32_t)l;
                r.beg = (uint32_t)__builtin_amdgcn_readlane((int)bi, l) + left * bm;
                r.end = min(r.beg + bm, end);
                r.extra = __builtin_amdgcn_readlane(x[i], l);
                r.any = true;
                return;
            }
            before = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        }
    };
    if (groups <= 64u)
        look(Count<1>{}, 0);
    else
        for (uint32_t g0 = 0; g0 < groups && !r.any; g0 += 256u) look(Count<4>{}, g0);
    if (!r.any) r.beg = t - before;
    return r;
}

// Between a run of matrix instructions that ends at a branch and the first reads
// of their results. The compiler's own wait states have come out short there: a
// result read as the first instruction behind a branch was read too early.
// 32 wait states, more than the longest of the instructions used here needs.
RFXQ_DEV void mfma_settle() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Row p's source and destination; -1 where an index is out of range (such a row
// is not computed). The load has no condition (without an index it reads the first
// offset), so that nothing waits for it where it is issued.
template <typename Args>
RFXQ_DEV int64_t src_row(const Args& a, uint32_t p) {
    const int32_t i = ((const RFXQ_GLOBAL int32_t*)(a.x_index ? a.x_index : a.offsets))[a.x_index ? p : 0u];
    const uint32_t s = a.x_index ? (uint32_t)i / a.x_div : p;
    return (i >= 0 || !a.x_index) && s < a.x_rows ? (int64_t)s : -1;
}
template <typename Args>
RFXQ_DEV int64_t dst_row(const Args& a, uint32_t p) {
    const int32_t i = a.y_index ? a.y_index[p] : (int32_t)p;
    return i >= 0 && (uint32_t)i < a.y_rows ? (int64_t)i : -1;
}

// Vectors that may start at any element.
typedef u4_t u4a2_t __attribute__((aligned(2)));
typedef float f4a4_t __attribute__((ext_vector_type(4), aligned(4)));

typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));

// 8 neighbouring values of a row as they lie in memory.
template <typename T>
struct Eight {
    u4_t v;
    __device__ __forceinline__ float at(uint32_t j) const {
        if constexpr (__is_same(T, half_t))
            return (float)__builtin_bit_cast(h8_t, v)[j];
        else
            return (float)__builtin_bit_cast(b8_t, v)[j];
    }
};
template <>
struct Eight<float> {
    f4v_t v[2];
    __device__ __forceinline__ float at(uint32_t j) const { return v[j >> 2][j & 3u]; }
};

// The 8 values at p.
template <typename T>
RFXQ_DEV Eight<T> ld_eight(const T* p) {
    Eight<T> r;
    if constexpr (__is_same(T, float)) {
        r.v[0] = *(const RFXQ_GLOBAL f4a4_t*)p;
        r.v[1] = *(const RFXQ_GLOBAL f4a4_t*)(p + 4);
    } else {
        r.v = *(const RFXQ_GLOBAL u4a2_t*)p;
    }
    return r;
}
// The first `have` of the 8 values at p, one by one, then zeros.
template <typename T>
RFXQ_DEV Eight<T> ld_eight(const T* p, uint32_t have) {
    if (have >= 8u) return ld_eight(p);
    T t[8];
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) t[i] = i < have ? ((const RFXQ_GLOBAL T*)p)[i] : (T)0.0f;
    Eight<T> r;
    __builtin_memcpy(&r, t, sizeof t);
    return r;
}

// The largest of 8 values' sizes, as bits: sizes order like their bits, and
// infinities and NaN lie above every finite one.
constexpr uint32_t kInfBits = 0x7F800000u;
RFXQ_DEV uint32_t top_of_eight(const Eight<float>& x) {
    uint32_t t = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) t = max(t, __builtin_bit_cast(uint32_t, x.at(i)) & 0x7FFFFFFFu);
    return t;
}
#define RFXQ_DPP_U32(v, ctrl) (uint32_t) __builtin_amdgcn_update_dpp(0, (int)(v), (ctrl), 0xF, 0xF, false)
// the largest of 8 neighbouring lanes
RFXQ_DEV uint32_t top_over_8(uint32_t v) {
    v = max(v, RFXQ_DPP_U32(v, 0xB1));
    v = max(v, RFXQ_DPP_U32(v, 0x4E));
    return max(v, RFXQ_DPP_U32(v, 0x141));
}

// Workgroup b's place in the grid of tiles: workgroups go round-robin to the 8
// XCDs, and each XCD takes blocks of sm x sn neighbouring tiles, whose rows
// and columns meet in its L2.
template <typename Args>
RFXQ_DEV bool tile_place(const Args& a, uint32_t b, uint32_t& tm, uint32_t& tn) {
    const uint32_t j = b >> 3, per = a.sm * a.sn;
    const uint32_t block = (j / per) * 8u + (b & 7u), r = j % per, across = (a.tiles_n + a.sn - 1u) / a.sn;
    tm = (block / across) * a.sm + r % a.sm;
    tn = (block % across) * a.sn + r / a.sm;
    return tm < a.tiles_m && tn < a.tiles_n;
}

// Place of 16-byte piece c (of 8) of LDS row r: rows of 128 bytes, pieces
// xor'ed with the row so that 8 rows' pieces of one column lie in 8 banks' groups.
RFXQ_DEV uint32_t lds_piece(uint32_t r, uint32_t c) { return r * 8u + (c ^ (r & 7u)); }

// The column of a tile that LDS row j of the weights holds. A lane's results
// are rows 4q..4q+3 of each 16-row operand (q = lane / 16): with this order the
// F operands of a wave's 16 F columns give it 4 F neighbouring ones.
template <uint32_t F = 4>
RFXQ_DEV uint32_t col_of(uint32_t j) {
    return (j & ~(16u * F - 1u)) + ((j >> 2) & 3u) * 4u * F + ((j >> 4) & (F - 1u)) * 4u + (j & 3u);
}
