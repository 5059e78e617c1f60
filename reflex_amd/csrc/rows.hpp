// Rows grouped by an id (rfxq_group_rows), and the search of the products that
// work on such groups for the tile a workgroup computes.
//
// key_i = id_i, or `groups` for an id outside [0, groups);
//   offsets[g] = #{ i : key_i < g }, g = 0..groups
//   order      = the rows i sorted by (key_i, i)
// a stable counting sort: the place of row i is
//   offsets[key_i] + #{ j < i : key_j = key_i }.
#pragma once
#include "common.hpp"

constexpr uint32_t kMaxGroups = 1024;

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

struct GroupRowsArgs {
    const int32_t* ids;
    int32_t* offsets;
    int32_t* order;
    uint32_t* counts;  // rfxq_group_count's: [workgroups][groups + 1], or NULL
    uint32_t n, groups, rounds, pad;
};

constexpr uint32_t kGroupThreads = 1024, kGroupWaves = kGroupThreads / 64u, kGroupRounds = 4;

RFXQ_DEV uint32_t group_key(const GroupRowsArgs& a, uint32_t i) {
    const uint32_t id = (uint32_t)((const RFXQ_GLOBAL int32_t*)a.ids)[i];
    return id < a.groups ? id : a.groups;
}

// The rows of each key in [begin, end) added to LDS counters, 8 ids a thread in
// flight.
RFXQ_DEV void count_keys(const GroupRowsArgs& a, uint32_t begin, uint32_t end, uint32_t* cnt) {
    uint32_t i = begin + threadIdx.x;
    for (; i + 7u * kGroupThreads < end; i += 8u * kGroupThreads) {
        uint32_t key[8];
#pragma unroll
        for (uint32_t j = 0; j < 8u; j++) key[j] = group_key(a, i + j * kGroupThreads);
#pragma unroll
        for (uint32_t j = 0; j < 8u; j++) atomicAdd(cnt + key[j], 1u);
    }
    for (; i < end; i += kGroupThreads) atomicAdd(cnt + group_key(a, i), 1u);
}

// Many rows: each workgroup's rows by key, for rfxq_group_rows. Dynamic LDS:
// groups + 1 counters.
extern "C" __global__ __launch_bounds__(1024) void rfxq_group_count(GroupRowsArgs a) {
    extern __shared__ uint32_t lds[];
    const uint32_t keys = a.groups + 1u, chunk = kGroupThreads * a.rounds, begin = blockIdx.x * chunk;
    for (uint32_t k = threadIdx.x; k < keys; k += kGroupThreads) lds[k] = 0;
    __syncthreads();
    count_keys(a, begin, min(begin + chunk, a.n), lds);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < keys; k += kGroupThreads) a.counts[(uint64_t)blockIdx.x * keys + k] = lds[k];
}

// Workgroup b places rows [b c, (b + 1) c), c = 1024 rounds. It needs each key's
// rows before its own and in all: up to some ten thousand rows it counts
// them itself (one launch, no scratch memory; the ids come from L2, the LDS
// atomics bound it: 15.6 us for 131072 rows, 128 groups), for more it adds up what
// rfxq_group_count left (9.7 us: 2.6 there, 7.2 here, trips to memory and barriers).
//
// Dynamic LDS: before[groups + 1], rest[groups + 1] (rows before the
// workgroup's own; the others), then wcnt[16][groups + 1] (16 bits: a wave's own rows).
extern "C" __global__ __launch_bounds__(1024) void rfxq_group_rows(GroupRowsArgs a) {
    extern __shared__ uint32_t lds[];
    const uint32_t keys = a.groups + 1u, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    uint32_t* before = lds;
    uint32_t* rest = lds + keys;
    uint16_t* wcnt = reinterpret_cast<uint16_t*>(lds + 2u * keys);
    __shared__ uint32_t part[kGroupWaves];
    const uint32_t chunk = kGroupThreads * a.rounds, begin = blockIdx.x * chunk;
    // a wave takes 64 neighbouring rows a round; their ids are on their way meanwhile
    int32_t id[kGroupRounds] = {};
    if (a.n) {
#pragma unroll
        for (uint32_t r = 0; r < kGroupRounds; r++)
            id[r] = ((const RFXQ_GLOBAL int32_t*)a.ids)[min(begin + (wave * a.rounds + r) * 64u + lane, a.n - 1u)];
    }
    const uint32_t words = 2u * keys + (kGroupWaves * keys + 1u) / 2u;
    for (uint32_t i = tid; i < words; i += kGroupThreads) lds[i] = 0;
    __syncthreads();

    if (a.counts) {
        // the threads of one key take every `parts`th workgroup's counts
        const uint32_t parts = max(kGroupThreads / keys, 1u);
        for (uint32_t j = tid; j < parts * keys; j += kGroupThreads) {
            const uint32_t k = j % keys;
            uint32_t ahead = 0, behind = 0;
            for (uint32_t w = j / keys; w < gridDim.x; w += 8u * parts) {
                uint32_t c[8];  // loads without a condition: all on their way at once
#pragma unroll
                for (uint32_t u = 0; u < 8u; u++)
                    c[u] = ((const RFXQ_GLOBAL uint32_t*)a.counts)[(uint64_t)min(w + u * parts, gridDim.x - 1u) * keys + k];
#pragma unroll
                for (uint32_t u = 0; u < 8u; u++) {
                    const uint32_t at = w + u * parts, n = at < gridDim.x ? c[u] : 0u;
                    ahead += at < blockIdx.x ? n : 0u;
                    behind += at < blockIdx.x ? 0u : n;
                }
            }
            atomicAdd(before + k, ahead);
            atomicAdd(rest + k, behind);
        }
    } else {
        count_keys(a, 0, begin, before);
        count_keys(a, begin, a.n, rest);
    }
    __syncthreads();

    // exclusive sums over the groups' counts, a thread per group
    const uint32_t all = tid < a.groups ? before[tid] + rest[tid] : 0u;
    const uint32_t incl = wave_scan(all);
    if (lane == 63u) part[wave] = incl;
    __syncthreads();
    uint32_t base = 0, total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kGroupWaves; w++) {
        base += w < wave ? part[w] : 0u;
        total += part[w];
    }
    base += incl - all;
    if (blockIdx.x == 0) {
        if (tid < a.groups) a.offsets[tid] = (int32_t)base;
        if (tid == 0) a.offsets[a.groups] = (int32_t)total;
    }
    if (tid < a.groups) before[tid] += base;
    if (tid == 0) before[a.groups] += total;

    // the own rows: lanes of one key find each other by ballots over the key's bits
    const uint32_t bits = 32u - (uint32_t)__builtin_clz(a.groups);
    const uint64_t below = ((uint64_t)1 << lane) - 1u;
    uint32_t key[kGroupRounds], rank[kGroupRounds];
#pragma unroll
    for (uint32_t r = 0; r < kGroupRounds; r++) {
        if (r >= a.rounds) break;
        const uint32_t i = begin + (wave * a.rounds + r) * 64u + lane;
        const bool own = i < a.n;
        key[r] = own ? min((uint32_t)id[r], a.groups) : 0u;
        uint64_t same = __builtin_amdgcn_ballot_w64(own);
        for (uint32_t b = 0; b < bits; b++) {
            const uint64_t set = __builtin_amdgcn_ballot_w64((key[r] >> b) & 1u);
            same &= (key[r] >> b) & 1u ? set : ~set;
        }
        if (own) {
            volatile uint16_t* c = &wcnt[wave * keys + key[r]];
            const uint32_t had = *c, ahead = (uint32_t)__builtin_popcountll(same & below);
            rank[r] = had + ahead;
            __builtin_amdgcn_wave_barrier();
            if (ahead == 0u) *c = (uint16_t)(had + (uint32_t)__builtin_popcountll(same));
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (uint32_t k = tid; k < keys; k += kGroupThreads) {  // each wave's first place of a key
        uint32_t run = 0;
#pragma unroll
        for (uint32_t w = 0; w < kGroupWaves; w++) {
            const uint32_t v = wcnt[w * keys + k];
            wcnt[w * keys + k] = (uint16_t)run;
            run += v;
        }
    }
    __syncthreads();
#pragma unroll
    for (uint32_t r = 0; r < kGroupRounds; r++) {
        if (r >= a.rounds) break;
        const uint32_t i = begin + (wave * a.rounds + r) * 64u + lane;
        if (i < a.n) a.order[before[key[r]] + wcnt[wave * keys + key[r]] + rank[r]] = (int32_t)i;
    }
}

// A token's pairs in increasing expert order, as rfxq_moe_combine adds them
// up: ids and weights [tokens][k] in selection order -> pair numbers and
// weights. A pair's place is the number of those before it (equal ids by their
// place, so that the places are a permutation for any ids).
extern "C" __global__ __launch_bounds__(256) void rfxq_moe_order(const int32_t* __restrict__ ids,
                                                                const float* __restrict__ w, int32_t* __restrict__ pair,
                                                                float* __restrict__ pair_w, uint32_t pairs, uint32_t k) {
    for (uint32_t p = blockIdx.x * 256u + threadIdx.x; p < pairs; p += gridDim.x * 256u) {
        const uint32_t first = p - p % k;
        const int32_t mine = ids[p];
        uint32_t at = first;
        for (uint32_t j = first; j < first + k; j++) at += ids[j] < mine || (ids[j] == mine && j < p) ? 1u : 0u;
        pair[at] = (int32_t)p;
        pair_w[at] = w[p];
    }
}
