// Host side of the entry points on grouped rows: rfxq_group_rows,
// rfxq_grouped_gemm and rfxq_lora_add (kernels: rows.hpp, grouped.hpp,
// lora.hpp). Included by rfxq.cpp, whose errors, contexts, launches and
// workspaces it uses.
#pragma once

namespace {

constexpr uint32_t kMaxGroups = 1024;         // rows.hpp
constexpr uint32_t kMaxGroupRows = 1u << 24;  // rows of rfxq_group_rows
constexpr uint32_t kMaxRank = 512;            // v of a 16-row tile in LDS
constexpr uint32_t kGroupThreads = 1024;      // of its workgroups, 1 to 4 rows each

// Mirrors of the device structs.
struct GroupRowsArgs {
    const int32_t* ids;
    int32_t* offsets;
    int32_t* order;
    uint32_t* counts;
    uint32_t n, groups, rounds, pad;
};
static_assert(sizeof(GroupRowsArgs) == 48, "GroupRowsArgs layout");

struct GroupedArgs {
    const void* x;
    const void* w;
    void* y;
    const int32_t* offsets;
    const int32_t* x_index;
    const int32_t* y_index;
    uint64_t ldx, ldy, w_stride;
    uint32_t rows, x_rows, y_rows, x_div;
    uint32_t k, n, groups, y_f32;
    uint32_t tiles_m, tiles_n, sm, sn;
};
static_assert(sizeof(GroupedArgs) == 120, "GroupedArgs layout");

struct LoraArgs {
    const void* x;
    const void* a;
    const void* b;
    const int32_t* ranks;
    const float* scales;
    const int32_t* offsets;
    const int32_t* order;
    const void* y;
    void* out;
    float* v;
    uint64_t ldx, ldy, ldo;
    uint32_t rows, x_rows, k, n;
    uint32_t rank, ldv, groups, splits;
    uint32_t k_split, tiles, across, pad;
};
static_assert(sizeof(LoraArgs) == 152, "LoraArgs layout");

bool float_type(uint32_t ty) { return ty == RFXQ_TYPE_F32 || ty == RFXQ_TYPE_F16 || ty == RFXQ_TYPE_BF16; }
bool half_type(uint32_t ty) { return ty == RFXQ_TYPE_F16 || ty == RFXQ_TYPE_BF16; }
uint32_t elem_bytes(uint32_t ty) { return ty == RFXQ_TYPE_F32 ? 4u : 2u; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16u == 0; }

// A stack of float matrices: [in, out] or [in, out, count].
int check_stack(const rfxq_weight* w, bool f32_too, const char* what) {
    if (!w) return fail(RFXQ_ERR_INVALID_INPUT, "%s: weight is NULL", what);
    if (!half_type(w->ggml_type) && !(f32_too && w->ggml_type == RFXQ_TYPE_F32))
        return fail(RFXQ_ERR_GGUF, "%s: ggml_type=%u (%sF16 or BF16 stacks)", what, w->ggml_type,
                    f32_too ? "F32, " : "");
    if (w->in_features == 0 || w->out_features == 0)
        return fail(RFXQ_ERR_OTHER, "%s: shape [%u, %u]", what, w->in_features, w->out_features);
    if (w->expert_count > kMaxGroups)
        return fail(RFXQ_ERR_OTHER, "%s: expert_count=%u (at most %u)", what, w->expert_count, kMaxGroups);
    const unsigned __int128 need = (unsigned __int128)std::max(w->expert_count, 1u) * w->out_features *
                                   w->in_features * elem_bytes(w->ggml_type);
    if (w->len < need)
        return fail(RFXQ_ERR_OTHER, "%s: weight of %llu bytes, shape [%u, %u, %u] needs %llu", what,
                    (unsigned long long)w->len, w->in_features, w->out_features, std::max(w->expert_count, 1u),
                    (unsigned long long)need);
    if (std::max(w->in_features, w->out_features) > 0x7FFFFFFFu)  // sums of these and a tile's size do not wrap
        return fail(RFXQ_ERR_OTHER, "%s: shape [%u, %u] (each below 2^31)", what, w->in_features, w->out_features);
    if (!w->data) return fail(RFXQ_ERR_INVALID_INPUT, "%s: weight data is NULL", what);
    if (reinterpret_cast<uintptr_t>(w->data) % elem_bytes(w->ggml_type))
        return fail(RFXQ_ERR_OTHER, "%s: weight data at %p is not %u-byte aligned", what, w->data,
                    elem_bytes(w->ggml_type));
    return RFXQ_OK;
}

int check_rows(const rfxq_rows* r, uint32_t columns, const char* what, const char* name) {
    if (!r) return fail(RFXQ_ERR_INVALID_INPUT, "%s: %s is NULL", what, name);
    if (!float_type(r->type)) return fail(RFXQ_ERR_GGUF, "%s: %s of type %u (F32, F16 or BF16)", what, name, r->type);
    if (r->rows == 0) return RFXQ_OK;
    if (!r->data) return fail(RFXQ_ERR_INVALID_INPUT, "%s: %s data is NULL", what, name);
    // as many bytes as an address space holds: products of these do not wrap
    if (r->rows > 0x7FFFFFFFu || (unsigned __int128)r->rows * r->stride >> 47)
        return fail(RFXQ_ERR_OTHER, "%s: %u rows of %s, stride=%llu", what, r->rows, name, (unsigned long long)r->stride);
    if (r->stride < columns)
        return fail(RFXQ_ERR_OTHER, "%s: %s stride=%llu (at least %u columns)", what, name,
                    (unsigned long long)r->stride, columns);
    if (reinterpret_cast<uintptr_t>(r->data) % elem_bytes(r->type))
        return fail(RFXQ_ERR_OTHER, "%s: %s at %p is not %u-byte aligned", what, name, r->data, elem_bytes(r->type));
    return RFXQ_OK;
}

// bytes from a matrix's first element to its last
uint64_t rows_span(const rfxq_rows* r, uint32_t columns) {
    return r->rows ? ((uint64_t)(r->rows - 1u) * r->stride + columns) * elem_bytes(r->type) : 0;
}

// caller's workspace, or the library's own
int take_workspace(Ctx* c, void* ws, uint64_t have, uint64_t need, hipStream_t stream, const char* what, void** out) {
    if (!ws) return need ? ctx_workspace(c, need, out, stream) : RFXQ_OK;
    if (have < need)
        return fail(RFXQ_ERR_INVALID_INPUT, "%s: workspace of %llu bytes, needs %llu", what, (unsigned long long)have,
                    (unsigned long long)need);
    if (need && !aligned16(ws)) return fail(RFXQ_ERR_OTHER, "%s: workspace is not 16-byte aligned", what);
    *out = ws;
    return RFXQ_OK;
}

// Row tiles that `rows` rows in `groups` groups can need: every group may end
// inside one.
uint32_t max_tiles(uint32_t rows, uint32_t groups, uint32_t bm) { return rows / bm + std::min(rows, groups); }

// ------------------------------------------------------------------ grouping

struct GroupPlan {
    uint32_t rounds, grid;
    uint64_t counts;  // bytes of the workgroups' counts, 0: each counts all rows
};
GroupPlan group_plan(uint32_t n, uint32_t groups) {
    GroupPlan p;
    // One launch, in which every workgroup counts all ids, or a launch of counts before
    // it (us, 128 groups: 7.6 against 8.8 at 32768 rows, 10.2 against 8.8 at 65536, 15.6
    // against 9.7 at 131072; 1024 groups, whose counts are longer to add up: 14.6 against
    // 16.5 at 131072, 43 against 21 at 300000). 2 rows a thread there (131072: 9.6 with
    // 1, 11.1 with 4), 4 from 262144 on (a million: 17 against 27).
    const bool many = n > (groups > 256u ? 131072u : 32768u);
    p.rounds = !many ? 1u : n <= 262144u ? 2u : 4u;
    p.grid = std::max(1u, (n + kGroupThreads * p.rounds - 1u) / (kGroupThreads * p.rounds));
    p.counts = many ? align256(4ull * p.grid * (groups + 1u)) : 0u;
    return p;
}

// ------------------------------------------------------------------ grouped GEMM

constexpr uint64_t kMaxOffset = 0xFFFFFFF0ull;  // bytes a buffer's 32-bit offsets reach

// The kernel of a grouped product, by the mean rows of the groups that can have any and
// the tiles that makes, measured (us) over groups 1..128, rows of 1..2048, N and K of
// 64..14336:
//   few4      16 x 16, K in quarters, weights straight from memory: where its tiles are
//             at most 3 a CU. There a tile's own time is all: smaller ones on more CUs win
//             (f16, 8 groups of 16 rows, N x K 1024 x 4096: 18 against 32 with 64 x 128
//             tiles; 8 x 64 rows, 320 x 1000: 6.4 against 9.4; 16 a CU lose, 115
//             against 51 at 32 x 32 x 1024 x 4096). Rows that do not start at 16 bytes: 2
//             a CU (8 x 64 x 320 x 3149 at 2.5: 48 against 41)
//   few rows  for decode, where every weight is read once: few4 up to 4 rows (64 against
//             72 on 128 x 768 x 2048 at 4 rows), long K up to 6 (60 x 1024 x 4096 at 6: 96
//             against 114; 60 x 4096 x 1024: 104 against 96); with short K, up to 2
//             rows, all of K in a wave (51 against 54 at 2 rows, 66 against 61 at 4), for
//             f32 activations up to 8 where a CU has a tile of 128 columns, for long K six
//             (quarters in its place: 128 x 2048 x 768 at 8 105 against 91, 128 x 320 x 1000
//             33 against 27; 60 x 1024 x 4096 104 against 109)
//   quarters  32 x 64, K in quarters, f32 activations: few tiles (8 x 64 x 1024 x 4096: 38
//             against 95; 8 x 64 x 2048 x 768: 17 against 23; from 4 a CU on 36
//             against 32), and up to 16 rows, long K up to 32 (128 x 768 x 2048 at 16: 96
//             against 110; 60 x 1024 x 4096 at 20: 115 against 132; short K 60 x 2816 x 704
//             at 6: 56 against 50)
//   large     256 x 256: from where its steps pay (8 x 14336 x 4096: 327 against
//             324 at 128 rows, 358 against 395 at 200) and its tiles fill over half of
//             the CUs (8 x 4096 x 4096, 256 rows, 128 tiles: 111 against 111; 64 tiles,
//             8 x 512 x 1024 x 4096: 85 against 53)
//   pipelined 64 x 128 copied ahead into three buffers: up to 2 tiles a CU, where each
//             workgroup has to hide its own latency (8 x 4096 x 14336 at 32 rows: 186
//             against 247; 8 x 512 x 1024 x 4096: 53 against 57); beyond, faster
//             without (8 x 192 x 4096 x 4096: 105 against 88)
//   tiles     64 x 128 through registers: the rest
struct GroupedVariant {
    uint32_t kernel;  // RFXQ_GROUPED_*
    uint32_t bm, bn, threads;
};
GroupedVariant grouped_variant(uint64_t cus, bool f32, uint32_t rows, uint32_t groups, uint32_t k, uint32_t n, bool aligned,
                               bool copies) {
    const uint32_t used = std::min(rows, groups), mean = rows / used;
    const auto tiles = [&](uint32_t bm, uint32_t bn) {
        return (uint64_t)used * ((mean + bm - 1u) / bm) * (((uint64_t)n + bn - 1u) / bn);
    };
    const GroupedVariant few4 = {RFXQ_GROUPED_FEW4, 16, 16, 256}, few = {RFXQ_GROUPED_FEW, 16, 128, 256};
    if (tiles(16, 16) <= (aligned ? 3u : 2u) * cus) return few4;
    if (aligned && f32 && mean <= 8u && tiles(16, 128) >= (k < 2048u ? 1u : 6u) * cus) return few;
    if (aligned && !f32 && k < 1024u && mean <= 2u && tiles(16, 128) >= 2u * cus) return few;
    if (aligned && !f32 && k >= 1024u && mean <= (k >= 2048u ? 6u : 4u)) return few4;
    if (f32 && ((aligned && mean <= (k >= 2048u ? 32u : k >= 1024u ? 16u : 0u)) || tiles(32, 64) <= 3u * cus))
        return {RFXQ_GROUPED_QUARTERS, 32, 64, 256};
    if (copies && mean > 160u && 8u * tiles(256, 256) >= 5u * cus) return {RFXQ_GROUPED_LARGE, 256, 256, 512};
    if (copies && tiles(64, 128) <= 2u * cus) return {RFXQ_GROUPED_COPIED, 64, 128, 256};
    return {RFXQ_GROUPED_TILES, 64, 128, 256};
}
// the kernel for `rows` (> 0) places of checked x and w (x->rows > 0)
GroupedVariant grouped_variant(uint64_t cus, const rfxq_rows* x, const rfxq_weight* w, uint32_t rows) {
    const uint32_t k = w->in_features, n = w->out_features;
    const bool f32 = x->type == RFXQ_TYPE_F32;
    const bool aligned = aligned16(x->data) && x->stride % (f32 ? 4u : 8u) == 0 && aligned16(w->data) && k % 8u == 0;
    // asynchronous copies: half types, rows at whole 16 bytes, 32-bit offsets
    const bool copies = aligned && !f32 && rows_span(x, k) < kMaxOffset && 2ull * k * n < kMaxOffset;
    return grouped_variant(cus, f32, rows, std::max(w->expert_count, 1u), k, n, aligned, copies);
}
hipFunction_t grouped_function(const HalfKernels& h, uint32_t kernel, bool f32, uint32_t w_type) {
    const uint32_t t = w_type == RFXQ_TYPE_F16 ? 0u : 1u, xt = f32 ? 0u : 1u;
    switch (kernel) {
        case RFXQ_GROUPED_FEW4: return h.few4[xt][t];
        case RFXQ_GROUPED_FEW: return h.few[xt][t];
        case RFXQ_GROUPED_QUARTERS: return h.quarters[t];
        case RFXQ_GROUPED_LARGE: return h.t256[t];
        case RFXQ_GROUPED_COPIED: return h.t64[t];
        default: return h.any[xt][t];
    }
}

// ------------------------------------------------------------------ adapters

// whole vectors in every row of b and out (lora.hpp)
bool lora_vec(uint32_t rank, uint32_t n) { return rank % 8u == 0 && n % 4u == 0; }

// 32-row tiles from 17 rows a group on. The ranges of K of rfxq_lora_down: until
// the workgroups fill the CUs twice (16-row tiles) or once (32: 4096 rows of 4096 60.6 us, twice
// 65.2), of at least 256 values each.
struct LoraPlan {
    uint32_t ldv, bm, tiles, splits, k_split;
    uint64_t total;
};
LoraPlan lora_plan(uint32_t k, uint32_t n, uint32_t rank, uint32_t groups, uint32_t rows, uint32_t cus) {
    LoraPlan p;
    p.ldv = (rank + 15u) & ~15u;
    p.bm = rows / std::min(rows, groups) > 16u && rank <= 256u && lora_vec(rank, n) ? 32u : 16u;
    p.tiles = max_tiles(rows, groups, p.bm);
    const uint32_t want = ((p.bm == 32u ? 1u : 2u) * cus + p.tiles - 1u) / p.tiles, most = (k + 255u) / 256u;
    p.splits = std::max(1u, std::min({want, most, 32u}));
    p.k_split = ((k + p.splits - 1u) / p.splits + 127u) & ~127u;
    p.splits = (k + p.k_split - 1u) / p.k_split;
    p.total = align256(4ull * p.splits * rows * p.ldv);
    return p;
}

}  // namespace

extern "C" {

uint64_t rfxq_group_rows_workspace_size(uint32_t n, uint32_t groups) {
    if (n > kMaxGroupRows || groups == 0 || groups > kMaxGroups) return 0;
    return group_plan(n, groups).counts;
}

int rfxq_group_rows(const int32_t* ids, uint32_t n, uint32_t groups, int32_t* offsets, int32_t* order, void* workspace,
                    uint64_t workspace_bytes, hipStream_t stream) {
    if (groups == 0 || groups > kMaxGroups)
        return fail(RFXQ_ERR_OTHER, "group_rows: groups=%u (1..=%u)", groups, kMaxGroups);
    if (n > kMaxGroupRows) return fail(RFXQ_ERR_OTHER, "group_rows: n=%u (at most %u)", n, kMaxGroupRows);
    if (!offsets || (n && (!ids || !order))) return fail(RFXQ_ERR_INVALID_INPUT, "group_rows: NULL pointer");
    if ((reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(order)) % 4u)
        return fail(RFXQ_ERR_OTHER, "group_rows: a pointer is not 4-byte aligned");
    if (overlap(ids, 4ull * n, order, 4ull * n) || overlap(ids, 4ull * n, offsets, 4ull * (groups + 1u)) ||
        overlap(order, 4ull * n, offsets, 4ull * (groups + 1u)))
        return fail(RFXQ_ERR_INVALID_INPUT, "group_rows: ids, offsets and order overlap");
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    const GroupPlan p = group_plan(n, groups);
    void* ws = nullptr;
    if (p.counts)
        if (int rc = take_workspace(c, workspace, workspace_bytes, p.counts, stream, "group_rows", &ws)) return rc;
    GroupRowsArgs a = {ids, offsets, order, static_cast<uint32_t*>(ws), n, groups, p.rounds, 0};
    const uint32_t keys = groups + 1u, lds = 8u * keys + 4u * ((16u * keys + 1u) / 2u);
    if (p.counts)
        if (int rc = launch(c->half.group_count, p.grid, 4u * keys, stream, &a, sizeof a, "rfxq_group_count launch",
                            kGroupThreads))
            return rc;
    if (int rc = launch(c->half.group_rows, p.grid, lds, stream, &a, sizeof a, "rfxq_group_rows launch", kGroupThreads))
        return rc;
    return ok();
}

int rfxq_grouped_gemm_policy(const rfxq_rows* x, const rfxq_weight* w, uint32_t rows, rfxq_grouped_policy* out) {
    if (!out) return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm_policy: NULL output");
    if (int rc = check_stack(w, false, "grouped_gemm_policy")) return rc;
    if (int rc = check_rows(x, w->in_features, "grouped_gemm_policy", "x")) return rc;
    if (rows == 0 || rows > 0x7FFFFFFFu || x->rows == 0)
        return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm_policy: rows=%u of %u", rows, x->rows);
    const Ctx* c = loaded_ctx();
    const GroupedVariant v = grouped_variant(c ? (uint64_t)c->cus : 256u, x, w, rows);
    *out = {v.kernel, v.bm, v.bn};
    return ok();
}

int rfxq_grouped_gemm(const rfxq_rows* x, const rfxq_weight* w, const int32_t* offsets, uint32_t rows,
                      const int32_t* x_index, uint32_t x_div, const int32_t* y_index, const rfxq_rows* y,
                      hipStream_t stream) {
    if (int rc = check_stack(w, false, "grouped_gemm")) return rc;
    if (int rc = check_rows(x, w->in_features, "grouped_gemm", "x")) return rc;
    if (int rc = check_rows(y, w->out_features, "grouped_gemm", "y")) return rc;
    const uint32_t ty = w->ggml_type, k = w->in_features, n = w->out_features;
    if (x->type != RFXQ_TYPE_F32 && x->type != ty)
        return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: x of type %u with weights of type %u (F32 or the weights')",
                    x->type, ty);
    if (y->type != RFXQ_TYPE_F32 && y->type != ty)
        return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: y of type %u with weights of type %u (F32 or the weights')",
                    y->type, ty);
    if (rows > 0x7FFFFFFFu) return fail(RFXQ_ERR_OTHER, "grouped_gemm: rows=%u", rows);
    if (x_div == 0) return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: x_div=0");
    if (!x_index && x_div != 1) return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: x_div=%u without x_index", x_div);
    if (rows == 0 || x->rows == 0 || y->rows == 0) return ok();
    if (!offsets) return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: offsets is NULL");
    if (overlap(x->data, rows_span(x, k), y->data, rows_span(y, n)))
        return fail(RFXQ_ERR_INVALID_INPUT, "grouped_gemm: x and y overlap");
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    const uint32_t groups = std::max(w->expert_count, 1u);
    GroupedArgs a;
    std::memset(&a, 0, sizeof a);
    a.x = x->data;
    a.w = w->data;
    a.y = y->data;
    a.offsets = offsets;
    a.x_index = x_index;
    a.y_index = y_index;
    a.ldx = x->stride;
    a.ldy = y->stride;
    a.w_stride = (uint64_t)k * n;
    a.rows = rows;
    a.x_rows = x->rows;
    a.y_rows = y->rows;
    a.x_div = x_div;
    a.k = k;
    a.n = n;
    a.groups = groups;
    a.y_f32 = y->type == RFXQ_TYPE_F32 ? 1u : 0u;
    const GroupedVariant v = grouped_variant((uint64_t)c->cus, x, w, rows);
    const bool few = v.kernel == RFXQ_GROUPED_FEW4 || v.kernel == RFXQ_GROUPED_FEW;
    a.tiles_m = max_tiles(rows, groups, v.bm);
    a.tiles_n = (n + v.bn - 1u) / v.bn;
    // XCD blocks of up to 4 row tiles and 4 column tiles, evenly cut, small enough that every XCD has several
    // (47 x 12 tiles: 12% less time with 2 row tiles than with 4)
    const uint32_t across = (a.tiles_n + 3u) / 4u;
    const uint64_t each = (uint64_t)a.tiles_m * across / 64u;
    a.sm = each >= 4u ? 4u : each >= 2u ? 2u : 1u;
    a.sn = (a.tiles_n + across - 1u) / across;
    const uint64_t blocks = (uint64_t)((a.tiles_m + a.sm - 1u) / a.sm) * ((a.tiles_n + a.sn - 1u) / a.sn);
    const uint64_t grid = few ? (uint64_t)a.tiles_m * a.tiles_n : (blocks + 7u) / 8u * 8u * a.sm * a.sn;
    if (grid * v.threads > 0xFFFFFFFFull)  // a launch's threads
        return fail(RFXQ_ERR_OTHER, "grouped_gemm: %u rows x %u columns need %llu workgroups", rows, n,
                    (unsigned long long)grid);
    if (int rc = launch(grouped_function(c->half, v.kernel, x->type == RFXQ_TYPE_F32, ty), (uint32_t)grid, 0, stream, &a,
                        sizeof a, "rfxq_grouped launch", v.threads))
        return rc;
    return ok();
}

uint64_t rfxq_lora_add_workspace_size(const rfxq_weight* a, uint32_t rows) {
    if (!a || rows == 0 || a->in_features == 0 || a->out_features == 0) return 0;
    const Ctx* c = loaded_ctx();
    // What any number of rows up to `rows` needs: there are at least rows / 32 tiles,
    // so the ranges are fewer than 64 CUs / rows + 1 (fewer rows can take more
    // ranges, and more memory, than the most rows do).
    const uint64_t ldv = (a->out_features + 15ull) & ~15ull, cus = c ? (uint64_t)c->cus : 256u;
    return align256(4u * ldv * std::min<uint64_t>(32ull * rows, 64u * cus + rows));
}

int rfxq_lora_add(const rfxq_rows* x, const rfxq_weight* a, const rfxq_weight* b, const int32_t* ranks,
                  const float* scales, const int32_t* offsets, const int32_t* order, const rfxq_rows* y,
                  const rfxq_rows* out, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
    if (int rc = check_stack(a, true, "lora_add a")) return rc;
    if (int rc = check_stack(b, true, "lora_add b")) return rc;
    const uint32_t k = a->in_features, rank = a->out_features, n = b->out_features;
    if (b->in_features != rank || b->expert_count != a->expert_count || b->ggml_type != a->ggml_type)
        return fail(RFXQ_ERR_OTHER, "lora_add: a [%u, %u, %u] of type %u and b [%u, %u, %u] of type %u", k, rank,
                    a->expert_count, a->ggml_type, b->in_features, n, b->expert_count, b->ggml_type);
    if (rank > kMaxRank) return fail(RFXQ_ERR_OTHER, "lora_add: rank=%u (at most %u)", rank, kMaxRank);
    if (int rc = check_rows(x, k, "lora_add", "x")) return rc;
    if (int rc = check_rows(y, n, "lora_add", "y")) return rc;
    if (int rc = check_rows(out, n, "lora_add", "out")) return rc;
    if (x->rows != y->rows || x->rows != out->rows)
        return fail(RFXQ_ERR_OTHER, "lora_add: %u rows of x, %u of y, %u of out", x->rows, y->rows, out->rows);
    if (x->type != y->type || x->type != out->type || (x->type != RFXQ_TYPE_F32 && x->type != a->ggml_type))
        return fail(RFXQ_ERR_INVALID_INPUT,
                    "lora_add: x of type %u, y %u, out %u with adapters of type %u (one type, F32 or the adapters')",
                    x->type, y->type, out->type, a->ggml_type);
    const uint32_t rows = x->rows, groups = std::max(a->expert_count, 1u);
    if (rows == 0) return ok();
    if (!offsets) return fail(RFXQ_ERR_INVALID_INPUT, "lora_add: offsets is NULL");
    const uint64_t sx = rows_span(x, k), sy = rows_span(y, n), so = rows_span(out, n);
    if (overlap(x->data, sx, out->data, so)) return fail(RFXQ_ERR_INVALID_INPUT, "lora_add: x and out overlap");
    if (!(y->data == out->data && y->stride == out->stride) && overlap(y->data, sy, out->data, so))
        return fail(RFXQ_ERR_INVALID_INPUT, "lora_add: y and out overlap without being the same rows");
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    const LoraPlan p = lora_plan(k, n, rank, groups, rows, (uint32_t)c->cus);
    // a tile's strips of 32 columns are shared by as many workgroups as give 8 a CU (4096 rows of 4096
    // columns, rank 64: 61.7 us; 4 a CU: 66, 2: 68)
    const uint32_t across = std::max(1u, std::min((8u * (uint32_t)c->cus + p.tiles - 1u) / p.tiles, (n + 127u) / 128u));
    const uint64_t up = (uint64_t)(p.tiles + 1u) * across;
    if (up * 256u > 0xFFFFFFFFull || (uint64_t)p.tiles * p.splits * 256u > 0xFFFFFFFFull)
        return fail(RFXQ_ERR_OTHER, "lora_add: %u rows need %llu workgroups", rows, (unsigned long long)up);
    void* ws = nullptr;
    if (int rc = take_workspace(c, workspace, workspace_bytes, p.total, stream, "lora_add", &ws)) return rc;
    LoraArgs l;
    std::memset(&l, 0, sizeof l);
    l.x = x->data;
    l.a = a->data;
    l.b = b->data;
    l.ranks = ranks;
    l.scales = scales;
    l.offsets = offsets;
    l.order = order;
    l.y = y->data;
    l.out = out->data;
    l.v = static_cast<float*>(ws);
    l.ldx = x->stride;
    l.ldy = y->stride;
    l.ldo = out->stride;
    l.rows = l.x_rows = rows;
    l.k = k;
    l.n = n;
    l.rank = rank;
    l.ldv = p.ldv;
    l.groups = groups;
    l.splits = p.splits;
    l.k_split = p.k_split;
    l.tiles = p.tiles;
    l.across = across;
    const uint32_t t = x->type == RFXQ_TYPE_F32 ? (a->ggml_type == RFXQ_TYPE_F32 ? 0u : a->ggml_type == RFXQ_TYPE_F16 ? 1u : 2u)
                       : x->type == RFXQ_TYPE_F16 ? 3u : 4u;
    const uint32_t wide = p.bm == 32u ? 1u : 0u, form = lora_vec(rank, n) ? wide : 2u, ldl = (rank + 31u) & ~31u;
    const uint32_t pieces = a->ggml_type == RFXQ_TYPE_BF16 ? 3u : 2u;
    const uint32_t lds = a->ggml_type == RFXQ_TYPE_F32 ? 4u * p.bm * (ldl + 4u)
                                                       : 2u * pieces * p.bm * (ldl + 8u) + 4u * p.bm * (ldl / 32u);
    if (int rc = launch(c->half.lora_down[t][wide], p.tiles * p.splits, 0, stream, &l, sizeof l, "rfxq_lora_down launch"))
        return rc;
    if (int rc = launch(c->half.lora_up[t][form], (uint32_t)up, lds, stream, &l, sizeof l, "rfxq_lora_up launch")) return rc;
    return ok();
}

}  // extern "C"

namespace {

bool half_layer(const rfxq_weight* gate, const rfxq_weight* up, const rfxq_weight* down) {
    return gate && up && down && half_type(gate->ggml_type) && half_type(up->ggml_type) && half_type(down->ggml_type);
}

// What rfxq_moe_ffn_grouped(_device) refuse of a layer with such stacks, before any
// routing. Of its own: gate and up may be of two half types, and x and the stacks
// start at any element.
int check_moe_half(const float* x, uint32_t rows, uint32_t hidden, uint32_t expert_count, uint32_t top_k,
                   const rfxq_weight* gate, const rfxq_weight* up, const rfxq_weight* down, const float* out) {
    if (gate->expert_count != expert_count || up->expert_count != expert_count || down->expert_count != expert_count)
        return fail(RFXQ_ERR_OTHER, "moe_ffn_grouped: expert tensors must have expert_count=%u", expert_count);
    if (gate->in_features != hidden || up->in_features != hidden || down->out_features != hidden ||
        gate->out_features != up->out_features || down->in_features != gate->out_features)
        return fail(RFXQ_ERR_OTHER, "moe_ffn_grouped: shapes gate [%u,%u] up [%u,%u] down [%u,%u] hidden %u",
                    gate->in_features, gate->out_features, up->in_features, up->out_features, down->in_features,
                    down->out_features, hidden);
    if (expert_count == 0 || expert_count > kRouteMaxE)
        return fail(RFXQ_ERR_OTHER, "moe_ffn_grouped: expert_count=%u (1..=%u)", expert_count, kRouteMaxE);
    if (top_k == 0 || top_k > expert_count || top_k > 64u)
        return fail(RFXQ_ERR_OTHER, "route_top_k: k (%u) must be in 1..=%u (logits.len())", top_k,
                    std::min(expert_count, 64u));
    if (int rc = check_stack(gate, false, "moe_ffn_grouped gate")) return rc;
    if (int rc = check_stack(up, false, "moe_ffn_grouped up")) return rc;
    if (int rc = check_stack(down, false, "moe_ffn_grouped down")) return rc;
    const uint64_t P64 = (uint64_t)rows * top_k;
    if (P64 > kMaxGroupRows)
        return fail(RFXQ_ERR_OTHER, "moe_ffn_grouped: %llu routed pairs (at most %u)", (unsigned long long)P64,
                    kMaxGroupRows);
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % 4u)
        return fail(RFXQ_ERR_OTHER, "moe_ffn_grouped: x or out not 4-byte aligned");
    if (overlap(x, 4ull * rows * hidden, out, 4ull * rows * hidden))
        return fail(RFXQ_ERR_INVALID_INPUT, "moe_ffn_grouped: x and out overlap");
    return RFXQ_OK;
}

// rfxq_moe_ffn_grouped(_device) over F16 or BF16 stacks: the routing (from the
// device's logits, or the host's, copied up), rfxq_group_rows, three grouped
// products of f32 activations and the combine in increasing expert order.
int moe_half(const float* x, uint32_t rows, uint32_t hidden, const float* router_logits, const uint32_t* host_idx,
             const float* host_w, uint32_t expert_count, uint32_t top_k, int normalize, float weight_scale,
             const rfxq_weight* gate, const rfxq_weight* up, const rfxq_weight* down, float* out, hipStream_t stream) {
    if (!x || !out) return fail(RFXQ_ERR_INVALID_INPUT, "moe_ffn_grouped: NULL argument");
    if (rows == 0) return ok();
    if (int rc = check_moe_half(x, rows, hidden, expert_count, top_k, gate, up, down, out)) return rc;
    const uint32_t P = rows * top_k, ffn = gate->out_features;
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    const uint64_t pairs = align256(4ull * P), wide = align256(4ull * P * ffn);
    const uint64_t o_w = pairs, o_order = o_w + pairs, o_pair = o_order + pairs, o_pair_w = o_pair + pairs;
    const uint64_t o_off = o_pair_w + pairs, o_cnt = o_off + align256(4ull * (expert_count + 1u));
    const uint64_t cnt = rfxq_group_rows_workspace_size(P, expert_count);
    const uint64_t o_gate = o_cnt + cnt, o_up = o_gate + wide, o_s = o_up + wide, o_down = o_s + wide;
    void* ws;
    if (int rc = ctx_workspace(c, o_down + align256(4ull * P * hidden), &ws, stream)) return rc;
    uint8_t* base = static_cast<uint8_t*>(ws);
    int32_t* idx = reinterpret_cast<int32_t*>(base);
    float* w = reinterpret_cast<float*>(base + o_w);
    int32_t* order = reinterpret_cast<int32_t*>(base + o_order);
    int32_t* pair = reinterpret_cast<int32_t*>(base + o_pair);
    float* pair_w = reinterpret_cast<float*>(base + o_pair_w);
    int32_t* offsets = reinterpret_cast<int32_t*>(base + o_off);
    float* g = reinterpret_cast<float*>(base + o_gate);
    float* u = reinterpret_cast<float*>(base + o_up);
    float* inner = reinterpret_cast<float*>(base + o_s);
    float* d = reinterpret_cast<float*>(base + o_down);
    if (router_logits) {
        if (int rc = moe_route_launch(c, router_logits, rows, expert_count, top_k, normalize, weight_scale, idx, w, nullptr,
                                      0, nullptr, nullptr, nullptr, stream))
            return rc;
    } else {
        if (int rc = stage_upload(c, idx, host_idx, 4ull * P, stream)) return rc;
        if (int rc = stage_upload(c, w, host_w, 4ull * P, stream)) return rc;
    }
    if (int rc = rfxq_group_rows(idx, P, expert_count, offsets, order, cnt ? base + o_cnt : nullptr, cnt, stream)) return rc;
    const rfxq_rows xr = {const_cast<float*>(x), RFXQ_TYPE_F32, rows, hidden};
    const rfxq_rows gr = {g, RFXQ_TYPE_F32, P, ffn}, ur = {u, RFXQ_TYPE_F32, P, ffn}, sr = {inner, RFXQ_TYPE_F32, P, ffn};
    const rfxq_rows dr = {d, RFXQ_TYPE_F32, P, hidden};
    if (int rc = rfxq_grouped_gemm(&xr, gate, offsets, P, order, top_k, nullptr, &gr, stream)) return rc;
    if (int rc = rfxq_grouped_gemm(&xr, up, offsets, P, order, top_k, nullptr, &ur, stream)) return rc;
    if (int rc = rfxq_silu_and_mul(g, u, inner, (uint64_t)P * ffn, stream)) return rc;
    if (int rc = rfxq_grouped_gemm(&sr, down, offsets, P, nullptr, 1, order, &dr, stream)) return rc;
    struct {
        const int32_t* ids;
        const float* w;
        int32_t* pair;
        float* pair_w;
        uint32_t pairs, k;
    } a = {idx, w, pair, pair_w, P, top_k};
    if (int rc = launch(c->half.moe_order, std::min((P + 255u) / 256u, 16384u), 0, stream, &a, sizeof a,
                        "rfxq_moe_order launch"))
        return rc;
    if (int rc = launch_combine(c, d, pair, pair_w, out, rows, top_k, hidden, stream)) return rc;
    return ok();
}

}  // namespace
