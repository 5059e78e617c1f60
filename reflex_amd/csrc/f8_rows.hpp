// Rows in 8-bit floating point (e4m3: 4 bits of exponent, 3 of fraction, no
// infinities, largest 448) with an f32 scale for each 128 of a row, written by what
// produces them: plain rows, SiLU(gate) * up, and the RMS norm with the residual's
// addition. Of a group's 128 values v
//   amax = max |v|,  scale = max(amax / 448, 2^-120),  code = RN_e4m3(v / scale)
// with amax / 448 a product by f32's 1 / 448, as tensor libraries divide by a number (a step of f32 off the quotient
// at most; the quotient itself would make one code in 100000 of f16 rows another than theirs, next to ties, and those
// are what rows are compared with), and v / scale an f32 quotient (SiLU's within 2^-22).
// A group with a value that is not finite has NaN for its scale. The smallest scale
// keeps 1 / scale an f32 value; groups of zeros have it.
//
// 16 lanes (a DPP row) hold a group, 8 values each: amax is four lane moves, and the
// group's codes one 128-byte line. All three kernels are bound by memory: each input
// is read once, each output written once (a large copy runs at 4.87 TB/s, reads and writes
// together; few rows cost what a launch does: an empty one 1.7 us in a graph). In a graph, on three sets of
// operands in turn:
//   quantize  4096 x 4096 bf16    10.4 us, 4.9 TB/s;  1 x 4096: 2.1 us
//   SiLU      4096 x 14336 bf16   55 us, 5.4 TB/s;    256 x 768 f32: 2.3 us
//   norm      4096 x 4096 bf16    25.2 us, 4.7 TB/s;  1 x 4096 f32: 2.9 us, 32 x 4096: 3.1 us
#pragma once
#include "common.hpp"
#include "tiles.hpp"

constexpr uint32_t kF8Block = 128;
constexpr float kF8Top = 448.0f, kF8Least = 0x1p-120f;
typedef u2_t u2a1_t __attribute__((aligned(1)));

struct F8RowsArgs {
    const void* x;
    const void* x2;       // SiLU: up; norm: the residual, or NULL
    const float* weight;  // norm
    void* sum;            // norm: x + residual, or NULL
    void* y;              // norm: the values before they are quantized, or NULL
    uint8_t* out;
    float* scales;
    uint64_t ldx, ldx2, ldsum, ldy, ldo, lds;
    uint32_t rows, k, groups;  // groups = ceil(k / 128)
    float eps;
    uint32_t by_rows, by_groups;  // the launch's groups, in rows and groups (quantize, SiLU)
};

// v / s rounded once, for 8 values and the group's scale s, as f32 division has it, where that changes a code
// (SiLU's v are within 2^-20 themselves and do with a reciprocal). Two operations a value, where division takes
// eleven and another reciprocal (4096 x 4096 bf16 10.4 us, by division 13.0, by one reciprocal 9.95; the norm 25.1, 26.4,
// 25.1; SiLU of 4096 x 14336 bf16 would take 60 and 69 for 55):
//   near + rest is 1 / s to 2^-44 of it, near below it so that rest >= 0 keeps the sign of zeros;
//   RN(v near + v rest) is RN(v / s), unless a midpoint of two f32 values lies within 2^-44 of v / s.
// A code depends on that only where RN may or may not give a midpoint m of two codes: at m + h / 2 and m - h / 2, with h f32's
// step there (below a power of two m - h / 4). m has 5 bits, so that v and m s are multiples of h s0 / 16, s0 the power of two
// below s, and v comes that near to (m +- h / 2) s only if 8 s / s0 is next to a whole number: less than 26 of its steps away,
// and not on it, since a quotient is no midpoint. Such scales take the division itself, and so do large ones, whose
// `rest` has no bits left. Rows of at most 11 bits (HALF: f16 and bf16 as they are) meet such scales often, where amax is a
// multiple of 7, but no such v: with v and m N of so few bits, N the whole number, v would have to be m N s0 / 8, and lies 16
// or more sixteenths of a step from m s then, for a half step's 8 to 15 (16 would be a scale just below a power of
// two, but 448 times one has that for its scale). Groups that are not `fine` have zeros, and NaN of what is not finite
// (infinite s: the division's).
template <bool HALF>
RFXQ_DEV void over_scale(const float (&v)[8], float s, bool fine, float (&q)[8]) {
    const uint32_t off = __builtin_bit_cast(uint32_t, s) & 0xFFFFFu;
    if (!HALF && min(off - 1u, 0x100000u - off) < 64u || s > 0x1p96f) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) q[i] = v[i] / s;
    } else {
        const float r = __builtin_amdgcn_rcpf(s), up = __builtin_fmaf(__builtin_fmaf(-s, r, 1.0f), r, r);
        const float below = as_f32(__builtin_bit_cast(uint32_t, up) - 1u), e = __builtin_fmaf(-s, below, 1.0f);
        const float near = fine ? below : 0.0f, rest = fine ? below * __builtin_fmaf(e, e, e) : 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) q[i] = __builtin_fmaf(v[i], near, v[i] * rest);
    }
}

// 8 values starting at v of the group that the 16 lanes of this DPP row hold, as codes
// and the group's scale.
template <bool EXACT, bool HALF = false>
RFXQ_DEV u2_t to_f8(const float (&v)[8], float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8u; i++) top = max(top, __builtin_bit_cast(uint32_t, v[i]) & 0x7FFFFFFFu);
    top = top_over_8(top);
    top = max(top, RFXQ_DPP_U32(top, 0x140));
    const bool fine = top < kInfBits;
    const float s = fmaxf(as_f32(top) * (1.0f / kF8Top), kF8Least);
    scale = fine ? s : __builtin_nanf("");
    float q[8];
    if constexpr (EXACT) {
        over_scale<HALF>(v, s, fine, q);
    } else {
        const float r = fine ? __builtin_amdgcn_rcpf(s) : 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++) q[i] = v[i] * r;
    }
    u2_t codes;
#pragma unroll
    for (uint32_t i = 0; i < 2u; i++) {
        int c = __builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i], q[4 * i + 1], 0, false);
        codes[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[4 * i + 2], q[4 * i + 3], c, true);
    }
    return codes;
}

// The first `have` of 8 codes, at any byte.
RFXQ_DEV void st_codes(uint8_t* p, u2_t codes, uint32_t have) {
    if (have >= 8u) {
        *(RFXQ_GLOBAL u2a1_t*)p = codes;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++)
            if (i < have) ((RFXQ_GLOBAL uint8_t*)p)[i] = (uint8_t)(codes[i >> 2] >> (8u * (i & 3u)));
    }
}

// The first `have` of 8 values, rounded to T.
template <typename T>
RFXQ_DEV void st_eight(T* p, const float (&v)[8], uint32_t have) {
    if (have >= 8u) {
        if constexpr (__is_same(T, float)) {
            *(RFXQ_GLOBAL f4a4_t*)p = f4v_t{v[0], v[1], v[2], v[3]};
            *(RFXQ_GLOBAL f4a4_t*)(p + 4) = f4v_t{v[4], v[5], v[6], v[7]};
        } else {
            u4_t r;
#pragma unroll
            for (uint32_t i = 0; i < 4u; i++)
                r[i] = (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * i]) |
                       (uint32_t)__builtin_bit_cast(uint16_t, (T)v[2 * i + 1]) << 16;
            *(RFXQ_GLOBAL u4a2_t*)p = r;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8u; i++)
            if (i < have) ((RFXQ_GLOBAL T*)p)[i] = (T)v[i];
    }
}

// g / (1 + exp(-g)) * u. exp by 2^(t + r) with t = RN(-g log2 e) and r what the rounding and log2 e's
// own bits left, so that far values keep f32's bits; no product of it overflows within its bounds, beyond which
// it is 0 beside 1, or the gate far.
constexpr float kLog2e = 1.44269504088896340736f, kLog2eRest = 1.92596299112661746887e-8f, kSiluFar = -87.0f;
RFXQ_DEV float silu_mul(float g, float u) {
    const float n = __builtin_amdgcn_fmed3f(-g, -128.0f, 128.0f), t = n * kLog2e;
    const float r = __builtin_fmaf(n, kLog2e, -t) + n * kLog2eRest, e = __builtin_amdgcn_exp2f(t);
    return g * __builtin_amdgcn_rcpf(1.0f + __builtin_fmaf(e, r * 0.69314718055994530942f, e)) * u;
}
// The same for g below kSiluFar, where it is g exp(g) u and exp(g), or exp(-g), may leave f32's range: an ordinary value
// beside a large u down to g = -197. exp(g) is f 2^i with f near 1, and half of i goes to g, half to the product, so that
// what counts of neither leaves it (below -256 all of it is 0; 0 g makes NaN of an infinite g).
RFXQ_DEV float silu_mul_far(float g, float u) {
    const float n = fmaxf(g, -256.0f), whole = rintf(n * kLog2e);
    const float f = __builtin_amdgcn_exp2f(__builtin_fmaf(n, kLog2eRest, __builtin_fmaf(n, kLog2e, -whole)));
    const int i = (int)whole, half = i / 2;
    return __builtin_fmaf(0.0f, g, ldexpf(ldexpf(n * f, half) * u, i - half));
}

// Plain rows, and SiLU(gate) * up: a group is 16 lanes' work, whichever row it is of, so that
// short rows leave no lane idle; a workgroup for every 16 groups, up to 2^20 of them. Two
// groups a thread, their loads in flight together: SiLU of 4096 x 14336 bf16 50.4 us (one: 52.0), but
// 4096 x 4096 16.9 (15.4) and 256 x 768 2.9 (2.4).
template <typename T, bool SILU>
RFXQ_DEV void f8_rows(const F8RowsArgs& a) {
    const uint32_t first = (blockIdx.x * 256u + threadIdx.x) >> 4, c = (threadIdx.x & 15u) * 8u;
    uint32_t row = first / a.groups, group = first % a.groups;
    while (row < a.rows) {
        const uint32_t k = group * kF8Block + c, have = k < a.k ? a.k - k : 0u;
        const Eight<T> x = ld_eight(static_cast<const T*>(a.x) + (uint64_t)row * a.ldx + k, have);
        float v[8], scale;
        if constexpr (SILU) {
            const Eight<T> up = ld_eight(static_cast<const T*>(a.x2) + (uint64_t)row * a.ldx2 + k, have);
#pragma unroll
            for (uint32_t j = 0; j < 8u; j++) v[j] = silu_mul(x.at(j), up.at(j));
            float least = x.at(0);
#pragma unroll
            for (uint32_t j = 1; j < 8u; j++) least = fminf(least, x.at(j));
            if (least < kSiluFar) {
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++)
                    if (x.at(j) < kSiluFar) v[j] = silu_mul_far(x.at(j), up.at(j));
            }
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 8u; j++) v[j] = x.at(j);
        }
        const u2_t codes = to_f8<!SILU, !__is_same(T, float)>(v, scale);
        st_codes(a.out + (uint64_t)row * a.ldo + k, codes, have);
        if (c == 0) stf(a.scales + (uint64_t)row * a.lds + group, scale);
        group += a.by_groups;
        const uint32_t over = group >= a.groups ? 1u : 0u;
        group -= over ? a.groups : 0u;
        row += a.by_rows + over;
    }
}

#define RFXQ_F8_ROWS(name, T)                                                                                             \
    extern "C" __global__ __launch_bounds__(256) void rfxq_f8_quantize_##name(F8RowsArgs a) { f8_rows<T, false>(a); }     \
    extern "C" __global__ __launch_bounds__(256) void rfxq_f8_silu_##name(F8RowsArgs a) { f8_rows<T, true>(a); }
RFXQ_F8_ROWS(f32, float)
RFXQ_F8_ROWS(f16, half_t)
RFXQ_F8_ROWS(bf16, __bf16)

// t = x + residual, y = t / sqrt(mean t^2 + eps) * weight: a row a workgroup, its values
// in registers between the two, in f32 throughout (the sum that is stored is rounded, the
// norm's is not). N = 1: 8 values a thread, up to 8192 columns; N = 4: up to 32768 (1 x 14336
// f32: 5.3 us, one CU's three reads); N = 0: rows of any length, read twice; a thread reads
// its values for the second time before it writes over them.
template <typename T, uint32_t N>
RFXQ_DEV void f8_norm(const F8RowsArgs& a) {
    __shared__ float part[16];
    const uint32_t tid = threadIdx.x, waves = blockDim.x >> 6, by = blockDim.x * 8u;
    for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(a.x) + (uint64_t)row * a.ldx;
        const T* r = static_cast<const T*>(a.x2) + (uint64_t)row * a.ldx2;
        const auto load = [&](uint32_t k, float(&v)[8]) {
            const uint32_t have = k < a.k ? a.k - k : 0u;
            const Eight<T> p = ld_eight(x + k, have);
            if (a.x2) {
                const Eight<T> q = ld_eight(r + k, have);
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++) v[j] = p.at(j) + q.at(j);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++) v[j] = p.at(j);
            }
        };
        float t[N ? N : 1u][8], sum = 0.0f;
        if constexpr (N > 0) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++) load((tid + blockDim.x * i) * 8u, t[i]);
#pragma unroll
            for (uint32_t i = 0; i < N; i++)
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++) sum = __builtin_fmaf(t[i][j], t[i][j], sum);
        } else {
            for (uint32_t k = tid * 8u; k < a.k; k += by) {
                load(k, t[0]);
#pragma unroll
                for (uint32_t j = 0; j < 8u; j++) sum = __builtin_fmaf(t[0][j], t[0][j], sum);
            }
        }
        sum = group_sum<64>(sum);
        __syncthreads();  // the last row's parts have been read
        if ((tid & 63u) == 0) part[tid >> 6] = sum;
        __syncthreads();
        float all = 0.0f;
        for (uint32_t w = 0; w < waves; w++) all += part[w];
        const float rinv = 1.0f / sqrtf(all / (float)a.k + a.eps);
        const auto write = [&](uint32_t k, const float(&v)[8]) {
            const uint32_t have = k < a.k ? a.k - k : 0u;
            if (a.sum) st_eight(static_cast<T*>(a.sum) + (uint64_t)row * a.ldsum + k, v, have);
            const Eight<float> w = ld_eight(a.weight + k, have);
            float y[8], scale;
#pragma unroll
            for (uint32_t j = 0; j < 8u; j++) y[j] = v[j] * rinv * w.at(j);
            if (a.y) st_eight(static_cast<T*>(a.y) + (uint64_t)row * a.ldy + k, y, have);
            const u2_t codes = to_f8<true>(y, scale);
            st_codes(a.out + (uint64_t)row * a.ldo + k, codes, have);
            if ((tid & 15u) == 0 && have) stf(a.scales + (uint64_t)row * a.lds + k / kF8Block, scale);
        };
        if constexpr (N > 0) {
#pragma unroll
            for (uint32_t i = 0; i < N; i++) write((tid + blockDim.x * i) * 8u, t[i]);
        } else {
            // whole groups of 16 lanes: the lanes behind the row's end hold zeros
            for (uint32_t k = tid * 8u; k < (a.k + kF8Block - 1u) / kF8Block * kF8Block; k += by) {
                load(k, t[0]);
                write(k, t[0]);
            }
        }
    }
}

#define RFXQ_F8_NORM(name, T)                                                                                         \
    extern "C" __global__ __launch_bounds__(1024) void rfxq_f8_norm_##name##_1(F8RowsArgs a) { f8_norm<T, 1>(a); }    \
    extern "C" __global__ __launch_bounds__(1024) void rfxq_f8_norm_##name##_4(F8RowsArgs a) { f8_norm<T, 4>(a); }    \
    extern "C" __global__ __launch_bounds__(1024) void rfxq_f8_norm_##name##_any(F8RowsArgs a) { f8_norm<T, 0>(a); }
RFXQ_F8_NORM(f32, float)
RFXQ_F8_NORM(f16, half_t)
RFXQ_F8_NORM(bf16, __bf16)
