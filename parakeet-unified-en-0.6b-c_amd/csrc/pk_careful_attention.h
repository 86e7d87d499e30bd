// pk_careful_attention.h - what the attention with rules (several new tokens a sequence,
// caps, biases, ranges) needs whatever its tiles are: which rows and tokens, the
// score's last steps, and one row taken by itself with plain arithmetic.
#pragma once

#include "pk_decode.h"

#include <cfloat>

namespace pkgpu {
namespace decode {

struct RuleArgs {
    float cap_in, cap_exp, cap2; // x = raw cap_in, e^2x = 2^(raw cap_exp), cap * log2(e); cap2 = 0: no cap
    const float* slopes;
    const int *first, *until;    // of each query row
    const int* starts;           // [B + 1], or NULL: row b is sequence b's
    int rows, max_new;
    int by_row;                  // the workspace's rows are q's, not (sequence, new token)s
    int per_seq;                 // row tiles of every sequence, 0: by its rows
};

// Sequence b's new tokens: rows row .. row + count - 1, whatever `starts` holds.
struct NewTokens { int row, count; };
__device__ inline NewTokens new_tokens(const RuleArgs& r, int b)
{
    if (!r.starts) return {b, b < r.rows ? 1 : 0};
    const int s = min(max(r.starts[b], 0), r.rows), e = min(max(r.starts[b + 1], s), r.rows);
    return {s, min(e - s, r.max_new)};
}

// Whether row `row` is one of some sequence's new tokens.
__device__ inline bool is_new_token(const RuleArgs& r, int B, int row)
{
    for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + (threadIdx.x & 63);
        bool mine = false;
        if (b < B) {
            const NewTokens n = new_tokens(r, b);
            mine = row >= n.row && row - n.row < n.count;
        }
        if (__any(mine)) return true;
    }
    return false;
}

// The tokens [lo, hi) that new token i of a sequence of `len` tokens sees, and its
// position p (negative where a sequence has more new tokens than tokens).
struct RowRange { int lo, hi, p; };
__device__ inline RowRange range_of(const RuleArgs& r, int len, int count, int i, int row, int window)
{
    RowRange s;
    s.p = len - count + i;
    s.lo = r.first ? max(r.first[row], 0) : 0;
    if (window > 0) s.lo = max(s.lo, s.p - window + 1);
    s.hi = s.p + 1;
    if (r.until) s.hi = max(s.hi, r.until[row]);
    s.hi = max(min(s.hi, len), 0);
    return s;
}

// cap tanh(raw scale / cap) in powers of two, with tanh x = 1 - 2 / (e^2x + 1): off by some
// units of 2^-24 of the cap.  Where f32 outputs want units of the value, small arguments
// take the quotient that the continued fraction x / (1 + x^2 / (3 + x^2 / (5 + ...)))
// gives, cut off behind 13: within 2^-40 below 1/2.
template <int T>
__device__ inline float capped(const RuleArgs& r, float raw)
{
    const float e = __builtin_amdgcn_exp2f(__fmul_rn(raw, r.cap_exp));
    float y = __builtin_fmaf(__fmul_rn(-2.0f, r.cap2), __builtin_amdgcn_rcpf(__fadd_rn(e, 1.0f)), r.cap2);
    if constexpr (T == F32) {
        const float x = __fmul_rn(raw, r.cap_in), z = __fmul_rn(x, x);
        const float a = __builtin_fmaf(__builtin_fmaf(z + 378.0f, z, 17325.0f), z, 135135.0f);
        const float b = __builtin_fmaf(__builtin_fmaf(__builtin_fmaf(28.0f, z, 3150.0f), z, 62370.0f), z, 135135.0f);
        const float small = __fmul_rn(__fmul_rn(x, r.cap2), __fmul_rn(a, __builtin_amdgcn_rcpf(b)));
        y = fabsf(x) < 0.5f ? small : y;
    }
    return y;
}

// A head's slope in powers of two, 0 without slopes.  One that the factor would make infinite
// stays at the largest float, so that its token at distance 0 is not 0 times infinity.
__device__ inline float slope_of(const RuleArgs& r, int head)
{
    if (!r.slopes) return 0.0f;
    const float s = r.slopes[head], t = s * 1.4426950408889634f;
    return fabsf(s) <= FLT_MAX && fabsf(t) > FLT_MAX ? copysignf(FLT_MAX, s) : t;
}

// A score in powers of two: raw = q . k, `ahead` the query's position less the key's.
template <int T>
__device__ inline float ruled_score(const RuleArgs& r, float raw, float scale2, float slope2, int ahead)
{
    float s = r.cap2 != 0.0f ? capped<T>(r, raw) : __fmul_rn(raw, scale2);
    if (r.slopes) s = __builtin_fmaf(-slope2, fabsf((float)ahead), s);
    return s;
}

// One key-value head of a sequence.
struct CacheView {
    const char *k, *v;
    const float *k_scale, *v_scale;
    const int* pages;
    int n_pages, page_shift, kv_heads, kvh;
    // the cache row of token t, -1: absent
    __device__ long long row(int t) const
    {
        const int id = pages[t >> page_shift];
        if ((uint32_t)id >= (uint32_t)n_pages) return -1;
        return (((long long)id * kv_heads + kvh) << page_shift) + (t & ((1 << page_shift) - 1));
    }
};

// Elements 8 part.. of a cache row; 4-bit ones with their unit, 8-bit ones without their scale.
template <int CACHE, int DIM>
__device__ inline void row_part(const char* base, const float* scales, long long row, int part, float* x)
{
    if constexpr (CACHE == E2M1)
        values_e2m1(reinterpret_cast<const uint32_t*>(base)[row * (DIM / 8) + part],
                    reinterpret_cast<const uint8_t*>(scales)[row * (DIM / kGroup) + part / (kGroup / 8)], x);
    else
        load8<CACHE>(base + (row * DIM + 8 * part) * size_of(CACHE), x);
}

// One query row over the tokens [s.lo, s.hi) by one wave, in fp32 throughout and without
// matrix instructions: a token that is not seen enters nothing, an infinite value that
// is seen enters as what it is, and weights are 2^-40 of the usual, so that sums of
// the largest values over 2^30 tokens stay finite.  It is there for what the tiles
// cannot hold apart, not for speed: lanes take a token each for the scores and 8
// elements each for the values.  One NaN in the first tokens, which all rows see, 32 heads over 8
// of 128 in bf16: 4096 tokens 26 ms (0.16 without it), 8192 103 (0.55), 500 behind 2500 others 3.8
// (0.06), 16 sequences of 4000 with 5 new tokens, a NaN in one, 0.87 (0.06).  Rows of another
// sequence set it off as well where a page in a tile of many rows is absent, whose place is staged
// from slot 0.  Writes out and lse, or with out NULL the chunk's share.
template <int CACHE, int T, int DIM>
__device__ void careful_row(const CacheView& c, const RuleArgs& r, const char* q, RowRange s, float scale2, float slope2,
                            char* out, float* lse, float* part, float* ml)
{
    constexpr int LANES = DIM / 8, SUBS = 64 / LANES;
    const int lane = threadIdx.x & 63;
    auto score = [&](int t, long long row) {
        if (row < 0) return -__builtin_inff();
        float sum = 0.0f;
#pragma unroll 1
        for (int i = 0; i < LANES; ++i) {
            float x[8], y[8];
            load8<T>(q + 8 * i * size_of(T), x);
            row_part<CACHE, DIM>(c.k, c.k_scale, row, i, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) sum = __builtin_fmaf(x[j], y[j], sum);
        }
        if constexpr (row_scaled(CACHE)) sum = __fmul_rn(sum, c.k_scale[row]);
        return ruled_score<T>(r, sum, scale2, slope2, s.p - t);
    };
    float m = -FLT_MAX;
#pragma unroll 1
    for (int t = s.lo + lane; t < s.hi; t += 64) m = fmaxf(m, score(t, c.row(t)));
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    m = __fadd_rn(m, 40.0f);
    float l = 0.0f, o[8] = {};
    const int sub = lane / LANES, mine = lane % LANES;
#pragma unroll 1
    for (int t0 = s.lo; t0 < s.hi; t0 += 64) {
        const int t = t0 + lane;
        const long long row = t < s.hi ? c.row(t) : -1;
        const float p = row < 0 ? 0.0f : __builtin_amdgcn_exp2f(score(t, row) - m);
        l = __fadd_rn(l, p);
#pragma unroll 1
        for (int j = 0; j < 64; j += SUBS) {
            const long long at = __shfl(row, j + sub);
            const float w = __shfl(p, j + sub);
            if (at < 0) continue;
            float x[8];
            row_part<CACHE, DIM>(c.v, c.v_scale, at, mine, x);
            const float f = row_scaled(CACHE) ? c.v_scale[at] : 1.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = row_scaled(CACHE) ? __fmul_rn(x[i], f) : x[i];
                o[i] = fabsf(v) <= FLT_MAX ? __builtin_fmaf(w, v, o[i]) : __fadd_rn(o[i], v);
            }
        }
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) l = __fadd_rn(l, __shfl_xor(l, d));
#pragma unroll
    for (int d = 32; d >= LANES; d >>= 1)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = __fadd_rn(o[i], __shfl_xor(o[i], d));
    if (out) {
        const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = l == 0.0f ? 0.0f : __fmul_rn(o[i], inv);
        if (sub == 0) store8<T>(out + 8 * mine * size_of(T), o);
        if (lse && lane == 0)
            *lse = l == 0.0f ? -__builtin_inff() : __fmul_rn(__fadd_rn(m, __builtin_amdgcn_logf(l)), 0.69314718055994531f);
    } else {
        if (sub == 0) store8<F32>(part + 8 * mine, o);
        if (lane == 0) { ml[0] = m; ml[1] = l; }
    }
}

}  // namespace decode
}  // namespace pkgpu
