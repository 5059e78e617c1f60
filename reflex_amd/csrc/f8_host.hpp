// Host side of the entry points in 8-bit floating point: rfxq_quantize_f8,
// rfxq_silu_and_mul_f8, rfxq_add_rmsnorm_f8 (kernels: f8_rows.hpp), rfxq_gemm_f8 and
// rfxq_grouped_gemm_f8 (f8_gemm.hpp). Included by rfxq.cpp behind half_host.hpp, whose
// checks of rows it uses.
#pragma once

namespace {

constexpr uint32_t kF8Block = 128;  // f8_rows.hpp

// Mirrors of the device structs.
struct F8RowsArgs {
    const void* x;
    const void* x2;
    const float* weight;
    void* sum;
    void* y;
    uint8_t* out;
    float* scales;
    uint64_t ldx, ldx2, ldsum, ldy, ldo, lds;
    uint32_t rows, k, groups;
    float eps;
    uint32_t by_rows, by_groups;
};
static_assert(sizeof(F8RowsArgs) == 128, "F8RowsArgs layout");

struct F8Args {
    const uint8_t* x;
    const float* xs;
    const uint8_t* w;
    const float* ws;
    void* y;
    const int32_t* offsets;
    const int32_t* x_index;
    const int32_t* y_index;
    uint64_t ldx, ldxs, ldy, w_stride, ws_stride;
    uint32_t rows, x_rows, y_rows, x_div;
    uint32_t k, n, groups, y_type;
    uint32_t tiles_m, tiles_n, sm, sn;
    uint32_t first_m, first_n;
};
static_assert(sizeof(F8Args) == 160, "F8Args layout");

uint32_t f8_groups(uint32_t k) { return (k + kF8Block - 1u) / kF8Block; }
uint32_t float_index(uint32_t ty) { return ty == RFXQ_TYPE_F32 ? 0u : ty == RFXQ_TYPE_F16 ? 1u : 2u; }

int check_f8_rows(const rfxq_f8_rows* r, uint32_t columns, const char* what, const char* name) {
    if (!r) return fail(RFXQ_ERR_INVALID_INPUT, "%s: %s is NULL", what, name);
    if (r->rows == 0) return RFXQ_OK;
    if (!r->data || !r->scales) return fail(RFXQ_ERR_INVALID_INPUT, "%s: %s data or scales is NULL", what, name);
    // as many bytes as an address space holds: products of these do not wrap
    if (r->rows > 0x7FFFFFFFu || (unsigned __int128)r->rows * r->stride >> 47 ||
        (unsigned __int128)r->rows * r->scale_stride >> 45)
        return fail(RFXQ_ERR_OTHER, "%s: %u rows of %s, stride=%llu, scale_stride=%llu", what, r->rows, name,
                    (unsigned long long)r->stride, (unsigned long long)r->scale_stride);
    if (r->stride < columns || r->scale_stride < f8_groups(columns))
        return fail(RFXQ_ERR_OTHER, "%s: %s stride=%llu, scale_stride=%llu (at least %u columns, %u scales)", what, name,
                    (unsigned long long)r->stride, (unsigned long long)r->scale_stride, columns, f8_groups(columns));
    if (reinterpret_cast<uintptr_t>(r->scales) % 4u)
        return fail(RFXQ_ERR_OTHER, "%s: %s scales at %p are not 4-byte aligned", what, name, (void*)r->scales);
    return RFXQ_OK;
}

int check_f8_weight(const rfxq_f8_weight* w, const char* what) {
    if (!w) return fail(RFXQ_ERR_INVALID_INPUT, "%s: weight is NULL", what);
    const uint32_t k = w->in_features, n = w->out_features;
    if (k == 0 || n == 0 || k > 0x7FFFFFFFu || n > 0x7FFFFFFFu)
        return fail(RFXQ_ERR_OTHER, "%s: shape [%u, %u] (each 1..2^31 - 1)", what, k, n);
    if (w->expert_count > kMaxGroups)
        return fail(RFXQ_ERR_OTHER, "%s: expert_count=%u (at most %u)", what, w->expert_count, kMaxGroups);
    const uint32_t count = std::max(w->expert_count, 1u);
    const unsigned __int128 need = (unsigned __int128)count * k * n;
    const unsigned __int128 scales = (unsigned __int128)count * f8_groups(k) * f8_groups(n) * 4u;
    if (w->len < need || w->scales_len < scales)
        return fail(RFXQ_ERR_OTHER, "%s: weight of %llu bytes and %llu of scales, shape [%u, %u, %u] needs %llu and %llu",
                    what, (unsigned long long)w->len, (unsigned long long)w->scales_len, k, n, count,
                    (unsigned long long)need, (unsigned long long)scales);
    if (!w->data || !w->scales) return fail(RFXQ_ERR_INVALID_INPUT, "%s: weight data or scales is NULL", what);
    if (reinterpret_cast<uintptr_t>(w->scales) % 4u)
        return fail(RFXQ_ERR_OTHER, "%s: weight scales at %p are not 4-byte aligned", what, (const void*)w->scales);
    return RFXQ_OK;
}

// A piece of memory from its first byte to its last.
struct Span {
    const void* p;
    uint64_t bytes;
    const char* name;
};
Span span_of(const rfxq_rows* r, uint32_t columns, const char* name) { return {r->data, rows_span(r, columns), name}; }
Span codes_of(const rfxq_f8_rows* r, uint32_t columns, const char* name) {
    return {r->data, r->rows ? (uint64_t)(r->rows - 1u) * r->stride + columns : 0u, name};
}
Span scales_of(const rfxq_f8_rows* r, uint32_t columns, const char* name) {
    return {r->scales, r->rows ? 4u * ((uint64_t)(r->rows - 1u) * r->scale_stride + f8_groups(columns)) : 0u, name};
}
int check_apart(const Span& a, const Span& b, const char* what) {
    if (a.p && b.p && overlap(a.p, a.bytes, b.p, b.bytes))
        return fail(RFXQ_ERR_INVALID_INPUT, "%s: %s and %s overlap", what, a.name, b.name);
    return RFXQ_OK;
}

// What rfxq_quantize_f8 and rfxq_silu_and_mul_f8 share: a group of 128 for 16 lanes.
int f8_rows_launch(const hipFunction_t* fns, const rfxq_rows* x, const rfxq_rows* up, uint32_t k, const rfxq_f8_rows* out,
                   hipStream_t stream, const char* what) {
    F8RowsArgs a;
    std::memset(&a, 0, sizeof a);
    a.x = x->data;
    a.ldx = x->stride;
    if (up) {
        a.x2 = up->data;
        a.ldx2 = up->stride;
    }
    a.out = static_cast<uint8_t*>(out->data);
    a.scales = out->scales;
    a.ldo = out->stride;
    a.lds = out->scale_stride;
    a.rows = x->rows;
    a.k = k;
    a.groups = f8_groups(k);
    const uint64_t grid = std::min<uint64_t>(((uint64_t)a.rows * a.groups + 15u) / 16u, 1u << 20);
    a.by_rows = (uint32_t)(grid * 16u / a.groups);
    a.by_groups = (uint32_t)(grid * 16u % a.groups);
    return launch(fns[float_index(x->type)], (uint32_t)grid, 0, stream, &a, sizeof a, what);
}

// The kernels of a product: place in kF8ProductNames, its tile, and what it takes (us), measured
// over rows of 1..8192, N and K of 768..14336: `start` once, and for every round of tiles over
// the CUs `tile` and `block` for each 128 of K. Kernels whose workgroups share a CU take rounds as they
// come, those that fill it (`whole`) whole ones. Rows that start at 16 bytes:
//   stream 16 x 16  64 tiles: 4.3 (1 x 4096 x 1024), 256: 6.3 (1 x 4096 x 4096), 11.9 (1 x 14336 x 4096)
//   stream 16 x 32  1 x 4096 x 14336: 11.5 (16 x 16: 15), 32 x 4096 x 4096: 6.4 (32 x 32: 7.5)
//   stream 32 x 32  64 x 4096 x 4096: 7.6 (16 x 32: 8.7, 64 x 128: 13), 128 rows: 11.0 (64 x 128: 13)
//   stream 16 x 64  32 tokens over 8 of 128 experts, 2048 x 768: 31 (16 x 32: 56, 64 x 128: 44);
//                   32 x 4096 x 14336: 12.8 (16 x 32: 14.3)
//   stream 32 x 64  128 x 4096 x 4096: 8.7, f32 results 9.2 (32 x 32: 11.1), 128 x 14336 x 4096: 20.9, 22.4 (28.1);
//                   32 x 4096 x 14336: 17.3 (16 x 32: 14.3, 32 x 32: 18.8)
//   stream 64 x 64  256 x 4096 x 4096: 12.0 (64 x 128: 13.3), 256 x 14336 x 4096: 29.0 (36.7), 64 x 4096 x 14336: 16.3
//                   (14.9); f32 results of 200 x 4096 x 4096: 13.2 (32 x 32: 18.3, 64 x 128: 22.2), 256 x
//                   14336 x 4096: 35 (65); 300 x 4096 x 4096: 23.8 (64 x 128: 22.8)
//   64 x 128        256 x 4096 x 4096: 13 (32 x 32: 19), 512 x 14336 x 4096: 39 (128 x 128: 65); f32 results 68
//   128 x 128       1000 x 4096 x 4096: 23 (64 x 128: 26, 128 x 256: 28); f32 38 (64 x 128: 47)
//   128 x 256       2048 x 4096 x 4096: 36 (128 x 128: 46, 256 x 256: 46)
//   256 x 256       4096 x 4096 x 14336: 217 (128 x 256: 237)
// and rows at any byte:
//   few 16 x 16     1 x 4099 x 4099: 11.8 (32 x 64: 22), 16 rows: 22 (22), 40 x 1235 x 1531: 7.0 (7.8)
//   32 x 64         333 x 1235 x 1531: 9.4 (64 x 128: 15.2), 16 x 4099 x 14336: 24.5 (35; few: 80)
//   64 x 128        1000 x 4099 x 4099, half results: 83 with 4 waves, 93 with 8 (32 x 64: 110); 333 rows: 43,
//                   34 (48); f32, 8 waves: 333 rows 39 (32 x 64: 49)
struct F8Variant {
    uint32_t product, kernel;  // kernel: RFXQ_F8_*
    uint32_t bm, bn, threads;
    float start, tile, block;
    bool whole;
};
constexpr F8Variant kF8Stream[] = {{6, RFXQ_F8_STREAM, 16, 16, 512, 2.8f, 1.3f, 0.069f, false},
                                   {7, RFXQ_F8_STREAM, 16, 32, 512, 2.8f, 0.9f, 0.085f, false},
                                   {8, RFXQ_F8_STREAM, 32, 32, 512, 2.8f, 1.0f, 0.1175f, false},
                                   {9, RFXQ_F8_STREAM, 16, 64, 256, 2.8f, 0.6f, 0.2f, false}};
// the first two of each: one matrix
constexpr F8Variant kF8Half[] = {{16, RFXQ_F8_STREAM, 32, 64, 512, 2.3f, 1.5f, 0.153f, true},
                                 {18, RFXQ_F8_STREAM, 64, 64, 512, 2.0f, 2.9f, 0.2125f, true},
                                 {10, RFXQ_F8_COPIED, 64, 128, 512, 0, 3.5f, 0.31f, true},
                                 {12, RFXQ_F8_COPIED, 128, 128, 512, 0, 4.0f, 0.59f, true},
                                 {14, RFXQ_F8_LARGE, 128, 256, 512, 0, 4.5f, 0.95f, true},
                                 {15, RFXQ_F8_LARGE, 256, 256, 512, 0, 6.0f, 1.6f, true}};
constexpr F8Variant kF8F32[] = {{17, RFXQ_F8_STREAM, 32, 64, 512, 2.3f, 1.5f, 0.166f, true},
                                {19, RFXQ_F8_STREAM, 64, 64, 512, 2.0f, 3.3f, 0.258f, true},
                                {11, RFXQ_F8_COPIED, 64, 128, 512, 0, 4.0f, 0.55f, true},
                                {13, RFXQ_F8_COPIED, 128, 128, 512, 0, 4.0f, 0.95f, true}};
// one row's operand has one line where 16 have 16
constexpr F8Variant kF8Few[2] = {{5, RFXQ_F8_FEW, 16, 16, 512, 3.0f, 0, 0.27f, false},
                                 {5, RFXQ_F8_FEW, 16, 16, 512, 3.0f, 0, 0.55f, false}};
constexpr F8Variant kF8AnyHalf[] = {{0, RFXQ_F8_ANY, 32, 64, 512, 3.5f, 1.2f, 0.45f, false},
                                    {2, RFXQ_F8_ANY, 64, 128, 256, 2.0f, 2.0f, 1.2f, false},
                                    {3, RFXQ_F8_ANY, 64, 128, 512, 0, 5.0f, 0.87f, true}};
constexpr F8Variant kF8AnyF32[] = {{1, RFXQ_F8_ANY, 32, 64, 512, 3.5f, 1.2f, 0.45f, false},
                                   {4, RFXQ_F8_ANY, 64, 128, 512, 0, 7.1f, 0.97f, true}};

// rows of tiles: grouped rows end inside a tile, half a tile on average
double f8_tile_rows(uint32_t rows, uint32_t groups, bool grouped, uint32_t bm) {
    const double used = std::min(rows, groups);
    return grouped ? used * std::max(1.0, rows / used / bm + 0.5) : std::ceil((double)rows / bm);
}

// `exact`: exact products (f32 results have them); `copies`: rows start at 16 bytes and offsets fit 32 bits
F8Variant f8_variant(uint32_t cus, uint32_t rows, uint32_t groups, bool grouped, uint32_t k, uint32_t n, bool exact,
                     bool copies) {
    const F8Variant* best = nullptr;
    double least = 0;
    const auto look = [&](const F8Variant& v) {
        const bool one = v.kernel == RFXQ_F8_STREAM && v.whole;  // for one matrix
        if (one && grouped) return;
        double rounds = f8_tile_rows(rows, groups, grouped, v.bm) * std::ceil((double)n / v.bn) / cus;
        rounds = v.whole ? std::ceil(rounds) : std::max(rounds, 1.0);
        if (v.bm == 16u && v.bn == 64u && rounds < 1.5) return;  // four waves: measured where they are many
        // the weights' bytes bound: tiles of 16 rows have more of them in flight
        if (copies && !grouped && rows <= 32u && v.bm > 16u) return;
        double t = v.start + rounds * (v.tile + (double)f8_groups(k) * v.block);
        if (one) t = std::max(t, (double)k * n / 3.6e6);  // weights at 3.6 TB/s (64 x 4096 x 14336: 16.3)
        if (!best || t < least) {
            best = &v;
            least = t;
        }
    };
    if (copies) {
        for (const F8Variant& v : kF8Stream) look(v);
        if (exact)
            for (const F8Variant& v : kF8F32) look(v);
        else
            for (const F8Variant& v : kF8Half) look(v);
    } else {
        look(kF8Few[rows > std::min(rows, groups) ? 1 : 0]);
        if (exact)
            for (const F8Variant& v : kF8AnyF32) look(v);
        else
            for (const F8Variant& v : kF8AnyHalf) look(v);
    }
    return *best;
}
// How a product of `rows` (> 0) places of checked x and w runs: its kernel, its tiles, their blocks for an XCD, and the
// tiles of a launch.
struct F8Plan {
    F8Variant v;
    uint32_t tiles_m, tiles_n, sm, sn;
    uint32_t most_m, most_n;
    uint64_t grid(uint32_t m, uint32_t n) const {  // workgroups for m x n tiles
        return ((uint64_t)((m + sm - 1u) / sm) * ((n + sn - 1u) / sn) + 7u) / 8u * 8u * sm * sn;
    }
};
F8Plan f8_plan(uint32_t cus, const rfxq_f8_rows* x, const rfxq_f8_weight* w, uint32_t rows, bool grouped, bool exact) {
    const uint32_t k = w->in_features, n = w->out_features, groups = grouped ? std::max(w->expert_count, 1u) : 1u;
    const bool copies = aligned16(x->data) && x->stride % 16u == 0 && aligned16(w->data) && k % 16u == 0 &&
                        codes_of(x, k, "").bytes < kMaxOffset && scales_of(x, k, "").bytes < kMaxOffset &&
                        (uint64_t)k * n < kMaxOffset;
    F8Plan p;
    const F8Variant v = p.v = f8_variant(cus, rows, groups, grouped, k, n, exact, copies);
    p.tiles_m = grouped ? max_tiles(rows, groups, v.bm) : (rows + v.bm - 1u) / v.bm;
    p.tiles_n = (n + v.bn - 1u) / v.bn;
    // XCD blocks of sm x sn tiles: the tallest of those whose fullest XCD has the fewest tiles, or, of
    // workgroups that fill a CU, rounds of them. Of those, dense ones of up to four rows of tiles (4096 x 4096 x 14336:
    // 217 us, of two 230, of one 243), fewer where four leave blocks half empty (700 x 4096 x 14336, f32 results: three 100
    // us, four 127); grouped ones of as many as a group has, up to three (4096 tokens over 8 of 128 experts, 2048 x 768:
    // 91 us, of four 102, of one 101; 128 tokens over 2 of 8, 4096 x 4096, f32 results: of one 42, of three 52). The
    // others two (64 x 4096 x 14336: 19 us, of one 22, of four 30; 333 x 1235 x 1531 the same).
    const uint32_t across = (p.tiles_n + 3u) / 4u;
    p.sn = (p.tiles_n + across - 1u) / across;
    const double tiles = f8_tile_rows(rows, groups, grouped, v.bm) / std::min(rows, groups);
    const uint32_t most = std::min(!v.whole ? 2u : grouped ? 3u : 4u, grouped ? (uint32_t)std::min(std::ceil(tiles), 3.0) : 4u);
    uint64_t least = ~0ull;
    for (uint32_t s = std::min(most, p.tiles_m); s; s--) {
        const uint64_t each = ((uint64_t)((p.tiles_m + s - 1u) / s) * across + 7u) / 8u * s * p.sn;
        const uint64_t take = v.whole ? (each * 8u + cus - 1u) / cus : each;
        if (take < least) {
            least = take;
            p.sm = s;
        }
    }
    // a launch has fewer than 2^32 threads: 134 million rows of 16 x 16 tiles are two
    p.most_m = p.tiles_m;
    p.most_n = p.tiles_n;
    while (p.grid(p.most_m, p.most_n) * v.threads > 0xFFFFFFFFull) {
        uint32_t& longer = p.most_m > p.most_n ? p.most_m : p.most_n;
        longer = (longer + 1u) / 2u;
    }
    return p;
}

int f8_product(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const int32_t* offsets, uint32_t rows,
               const int32_t* x_index, uint32_t x_div, const int32_t* y_index, const rfxq_rows* y, bool exact,
               hipStream_t stream, const char* what) {
    const uint32_t k = w->in_features, n = w->out_features, groups = std::max(w->expert_count, 1u);
    const Span sy = span_of(y, n, "y");
    const Span inputs[] = {codes_of(x, k, "x"), scales_of(x, k, "x's scales"), {w->data, (uint64_t)groups * k * n, "weight"},
                           {w->scales, 4ull * groups * f8_groups(k) * f8_groups(n), "weight's scales"}};
    for (const Span& in : inputs)
        if (int rc = check_apart(in, sy, what)) return rc;
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    F8Args a;
    std::memset(&a, 0, sizeof a);
    a.x = static_cast<const uint8_t*>(x->data);
    a.xs = x->scales;
    a.w = static_cast<const uint8_t*>(w->data);
    a.ws = w->scales;
    a.y = y->data;
    a.offsets = offsets;
    a.x_index = x_index;
    a.y_index = y_index;
    a.ldx = x->stride;
    a.ldxs = x->scale_stride;
    a.ldy = y->stride;
    a.w_stride = (uint64_t)k * n;
    a.ws_stride = (uint64_t)f8_groups(k) * f8_groups(n);
    a.rows = rows;
    a.x_rows = x->rows;
    a.y_rows = y->rows;
    a.x_div = x_div;
    a.k = k;
    a.n = n;
    a.groups = groups;
    a.y_type = float_index(y->type);
    const F8Plan p = f8_plan((uint32_t)c->cus, x, w, rows, offsets != nullptr, exact || a.y_type == 0);
    a.sm = p.sm;
    a.sn = p.sn;
    for (a.first_m = 0; a.first_m < p.tiles_m; a.first_m += a.tiles_m) {
        a.tiles_m = std::min(p.most_m, p.tiles_m - a.first_m);
        for (a.first_n = 0; a.first_n < p.tiles_n; a.first_n += a.tiles_n) {
            a.tiles_n = std::min(p.most_n, p.tiles_n - a.first_n);
            if (int rc = launch(c->f8.product[p.v.product][offsets ? 1 : 0], (uint32_t)p.grid(a.tiles_m, a.tiles_n), 0, stream, &a,
                                sizeof a, "rfxq_f8 product launch", p.v.threads))
                return rc;
        }
    }
    return RFXQ_OK;
}

int f8_gemm(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const rfxq_rows* y, bool exact, hipStream_t stream,
            const char* what) {
    if (int rc = check_f8_weight(w, what)) return rc;
    if (w->expert_count > 1u)
        return fail(RFXQ_ERR_OTHER, "%s: a stack of %u matrices (rfxq_grouped_gemm_f8 takes stacks)", what, w->expert_count);
    if (int rc = check_f8_rows(x, w->in_features, what, "x")) return rc;
    if (int rc = check_rows(y, w->out_features, what, "y")) return rc;
    if (x->rows != y->rows) return fail(RFXQ_ERR_OTHER, "%s: %u rows of x, %u of y", what, x->rows, y->rows);
    if (x->rows == 0) return ok();
    if (int rc = f8_product(x, w, nullptr, x->rows, nullptr, 1, nullptr, y, exact, stream, what)) return rc;
    return ok();
}

int f8_grouped(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const int32_t* offsets, uint32_t rows,
               const int32_t* x_index, uint32_t x_div, const int32_t* y_index, const rfxq_rows* y, bool exact,
               hipStream_t stream, const char* what) {
    if (int rc = check_f8_weight(w, what)) return rc;
    if (int rc = check_f8_rows(x, w->in_features, what, "x")) return rc;
    if (int rc = check_rows(y, w->out_features, what, "y")) return rc;
    if (rows > 0x7FFFFFFFu) return fail(RFXQ_ERR_OTHER, "%s: rows=%u", what, rows);
    if (x_div == 0) return fail(RFXQ_ERR_INVALID_INPUT, "%s: x_div=0", what);
    if (!x_index && x_div != 1) return fail(RFXQ_ERR_INVALID_INPUT, "%s: x_div=%u without x_index", what, x_div);
    if (rows == 0 || x->rows == 0 || y->rows == 0) return ok();
    if (!offsets) return fail(RFXQ_ERR_INVALID_INPUT, "%s: offsets is NULL", what);
    if (int rc = f8_product(x, w, offsets, rows, x_index, x_div, y_index, y, exact, stream, what)) return rc;
    return ok();
}

// what the test hooks report of
int f8_plan_for(const rfxq_f8_rows* x, const rfxq_f8_weight* w, uint32_t rows, int grouped, uint32_t y_type, const char* what,
                F8Plan* p) {
    if (int rc = check_f8_weight(w, what)) return rc;
    if (int rc = check_f8_rows(x, w->in_features, what, "x")) return rc;
    if (rows == 0 || rows > 0x7FFFFFFFu || x->rows == 0)
        return fail(RFXQ_ERR_INVALID_INPUT, "%s: rows=%u of %u", what, rows, x->rows);
    if (!float_type(y_type)) return fail(RFXQ_ERR_GGUF, "%s: y of type %u (F32, F16 or BF16)", what, y_type);
    const Ctx* c = loaded_ctx();
    *p = f8_plan(c ? (uint32_t)c->cus : 256u, x, w, rows, grouped != 0, y_type == RFXQ_TYPE_F32);
    return RFXQ_OK;
}

}  // namespace

extern "C" {

int rfxq_quantize_f8(const rfxq_rows* x, uint32_t k, const rfxq_f8_rows* out, hipStream_t stream) {
    if (k == 0 || k > 0x7FFFFFFFu) return fail(RFXQ_ERR_OTHER, "quantize_f8: k=%u", k);
    if (int rc = check_rows(x, k, "quantize_f8", "x")) return rc;
    if (int rc = check_f8_rows(out, k, "quantize_f8", "out")) return rc;
    if (x->rows != out->rows) return fail(RFXQ_ERR_OTHER, "quantize_f8: %u rows of x, %u of out", x->rows, out->rows);
    if (x->rows == 0) return ok();
    const Span sx = span_of(x, k, "x"), sc = codes_of(out, k, "out"), ss = scales_of(out, k, "out's scales");
    for (auto& [a, b] : {std::pair{sx, sc}, std::pair{sx, ss}, std::pair{sc, ss}})
        if (int rc = check_apart(a, b, "quantize_f8")) return rc;
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    if (int rc = f8_rows_launch(c->f8.quantize, x, nullptr, k, out, stream, "rfxq_f8_quantize launch")) return rc;
    return ok();
}

int rfxq_silu_and_mul_f8(const rfxq_rows* gate, const rfxq_rows* up, uint32_t k, const rfxq_f8_rows* out,
                         hipStream_t stream) {
    if (k == 0 || k > 0x7FFFFFFFu) return fail(RFXQ_ERR_OTHER, "silu_and_mul_f8: k=%u", k);
    if (int rc = check_rows(gate, k, "silu_and_mul_f8", "gate")) return rc;
    if (int rc = check_rows(up, k, "silu_and_mul_f8", "up")) return rc;
    if (int rc = check_f8_rows(out, k, "silu_and_mul_f8", "out")) return rc;
    if (gate->type != up->type)
        return fail(RFXQ_ERR_INVALID_INPUT, "silu_and_mul_f8: gate of type %u, up %u", gate->type, up->type);
    if (gate->rows != up->rows || gate->rows != out->rows)
        return fail(RFXQ_ERR_OTHER, "silu_and_mul_f8: %u rows of gate, %u of up, %u of out", gate->rows, up->rows, out->rows);
    if (gate->rows == 0) return ok();
    const Span sg = span_of(gate, k, "gate"), su = span_of(up, k, "up"), sc = codes_of(out, k, "out");
    const Span ss = scales_of(out, k, "out's scales");
    for (auto& [a, b] :
         {std::pair{sg, sc}, std::pair{su, sc}, std::pair{sg, ss}, std::pair{su, ss}, std::pair{sc, ss}})
        if (int rc = check_apart(a, b, "silu_and_mul_f8")) return rc;
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    if (int rc = f8_rows_launch(c->f8.silu, gate, up, k, out, stream, "rfxq_f8_silu launch")) return rc;
    return ok();
}

int rfxq_add_rmsnorm_f8(const rfxq_rows* x, const rfxq_rows* residual, const float* weight, uint32_t k, float eps,
                        const rfxq_rows* sum, const rfxq_f8_rows* out, const rfxq_rows* y, hipStream_t stream) {
    const char* const what = "add_rmsnorm_f8";
    if (k == 0 || k > 0x7FFFFFFFu) return fail(RFXQ_ERR_OTHER, "add_rmsnorm_f8: k=%u", k);
    if (!(eps >= 0.0f) || std::isinf(eps)) return fail(RFXQ_ERR_INVALID_INPUT, "add_rmsnorm_f8: eps=%g", (double)eps);
    if (int rc = check_rows(x, k, what, "x")) return rc;
    if (residual)
        if (int rc = check_rows(residual, k, what, "residual")) return rc;
    if (sum)
        if (int rc = check_rows(sum, k, what, "sum")) return rc;
    if (y)
        if (int rc = check_rows(y, k, what, "y")) return rc;
    if (int rc = check_f8_rows(out, k, what, "out")) return rc;
    const rfxq_rows* const rows[] = {residual, sum, y};
    for (const rfxq_rows* r : rows) {
        if (!r) continue;
        if (r->type != x->type)
            return fail(RFXQ_ERR_INVALID_INPUT, "add_rmsnorm_f8: rows of types %u and %u (one type)", x->type, r->type);
        if (r->rows != x->rows) return fail(RFXQ_ERR_OTHER, "add_rmsnorm_f8: %u and %u rows", x->rows, r->rows);
    }
    if (out->rows != x->rows) return fail(RFXQ_ERR_OTHER, "add_rmsnorm_f8: %u rows of x, %u of out", x->rows, out->rows);
    if (x->rows == 0) return ok();
    if (!weight || reinterpret_cast<uintptr_t>(weight) % 4u)
        return fail(RFXQ_ERR_INVALID_INPUT, "add_rmsnorm_f8: weight is NULL or not 4-byte aligned");
    const Span none = {nullptr, 0, ""};
    const Span in[] = {span_of(x, k, "x"), residual ? span_of(residual, k, "residual") : none,
                       {weight, 4ull * k, "weight"}};
    const Span results[] = {codes_of(out, k, "out"), scales_of(out, k, "out's scales"),
                            sum ? span_of(sum, k, "sum") : none, y ? span_of(y, k, "y") : none};
    for (size_t i = 0; i < 4; i++) {
        for (size_t j = 0; j < 3; j++) {
            const rfxq_rows* r = j == 0 ? x : j == 1 ? residual : nullptr;
            if (i == 2 && r && sum && sum->data == r->data && sum->stride == r->stride) continue;  // in place
            if (int rc = check_apart(in[j], results[i], what)) return rc;
        }
        for (size_t j = 0; j < i; j++)
            if (int rc = check_apart(results[j], results[i], what)) return rc;
    }
    Ctx* c;
    if (int rc = current_ctx(&c)) return rc;
    F8RowsArgs a;
    std::memset(&a, 0, sizeof a);
    a.x = x->data;
    a.ldx = x->stride;
    if (residual) {
        a.x2 = residual->data;
        a.ldx2 = residual->stride;
    }
    a.weight = weight;
    if (sum) {
        a.sum = sum->data;
        a.ldsum = sum->stride;
    }
    if (y) {
        a.y = y->data;
        a.ldy = y->stride;
    }
    a.out = static_cast<uint8_t*>(out->data);
    a.scales = out->scales;
    a.ldo = out->stride;
    a.lds = out->scale_stride;
    a.rows = x->rows;
    a.k = k;
    a.groups = f8_groups(k);
    a.eps = eps;
    const uint32_t form = k <= 8192u ? 0u : k <= 32768u ? 1u : 2u, each = form == 1u ? 32u : 8u;
    const uint32_t threads = std::min(1024u, ((k + each - 1u) / each + 63u) / 64u * 64u);
    if (int rc = launch(c->f8.norm[float_index(x->type)][form], std::min(a.rows, 1u << 20), 0, stream, &a, sizeof a,
                        "rfxq_f8_norm launch", threads))
        return rc;
    return ok();
}

int rfxq_gemm_f8(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const rfxq_rows* y, hipStream_t stream) {
    return f8_gemm(x, w, y, false, stream, "gemm_f8");
}

int rfxq_gemm_f8_exact(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const rfxq_rows* y, hipStream_t stream) {
    return f8_gemm(x, w, y, true, stream, "gemm_f8_exact");
}

int rfxq_grouped_gemm_f8(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const int32_t* offsets, uint32_t rows,
                         const int32_t* x_index, uint32_t x_div, const int32_t* y_index, const rfxq_rows* y,
                         hipStream_t stream) {
    return f8_grouped(x, w, offsets, rows, x_index, x_div, y_index, y, false, stream, "grouped_gemm_f8");
}

int rfxq_grouped_gemm_f8_exact(const rfxq_f8_rows* x, const rfxq_f8_weight* w, const int32_t* offsets, uint32_t rows,
                               const int32_t* x_index, uint32_t x_div, const int32_t* y_index, const rfxq_rows* y,
                               hipStream_t stream) {
    return f8_grouped(x, w, offsets, rows, x_index, x_div, y_index, y, true, stream, "grouped_gemm_f8_exact");
}

int rfxq_gemm_f8_policy(const rfxq_f8_rows* x, const rfxq_f8_weight* w, uint32_t rows, int grouped, uint32_t y_type,
                        rfxq_f8_policy* out) {
    if (!out) return fail(RFXQ_ERR_INVALID_INPUT, "gemm_f8_policy: NULL output");
    F8Plan p;
    if (int rc = f8_plan_for(x, w, rows, grouped, y_type, "gemm_f8_policy", &p)) return rc;
    *out = {p.v.kernel, p.v.bm, p.v.bn};
    return ok();
}

int rfxq_gemm_f8_launch(const rfxq_f8_rows* x, const rfxq_f8_weight* w, uint32_t rows, int grouped, uint32_t y_type,
                        rfxq_f8_launch* out) {
    if (!out) return fail(RFXQ_ERR_INVALID_INPUT, "gemm_f8_launch: NULL output");
    F8Plan p;
    if (int rc = f8_plan_for(x, w, rows, grouped, y_type, "gemm_f8_launch", &p)) return rc;
    const auto times = [](uint32_t all, uint32_t most) { return (all + most - 1u) / most; };
    *out = {p.v.threads, times(p.tiles_m, p.most_m) * times(p.tiles_n, p.most_n)};
    return ok();
}

}  // extern "C"
