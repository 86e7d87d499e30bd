// pk_paged_attention.h - attention of one new token per sequence over a paged
// key-value cache: the kernel, instantiated per cache type by
// pk_paged_attention_*.hip.
//
//   s_t = scale * k_scale_t * (q . k_t),   o = sum_t p_t v_scale_t v_t,
//   p_t = 2^(s_t log2e - m) / l,  l = sum_t 2^(s_t log2e - m)
//
// One workgroup takes up to 16 query heads that share a key-value head of one
// sequence, and one chunk of its tokens; its waves take tiles of 32 tokens in
// turn, each with a running maximum and sum of its own, joined through LDS at
// the end.  Sequences of several chunks leave (m, l, o) per chunk in the
// workspace, and a second launch joins those in chunk order.
//
// Both products run on 16x16x32 matrix instructions with the operands swapped
// round so that nothing is exchanged between lanes:
//   S^T [16 tokens][16 heads] = K [16 tokens][dim] Q^T: lane l holds 4 scores
//     of head l % 16 (tokens 4 (l / 16) + r);
//   O^T [16 of dim][16 heads] += V^T [16 of dim][32 tokens] P^T: its second
//     operand wants, of lane l, 8 tokens of head l % 16: the 4 + 4 that the two
//     16-token halves of the tile left there.
// So k index 8 g + i of the second product stands for token 4 g + i (i < 4) or
// 16 + 4 g + i - 4, and the first product's k index for whichever elements of
// the head a lane has loaded as one 16-byte piece; the sums do not care.  V^T
// comes from rows by byte permutes in registers: a lane loads the same
// head_dim / 16 elements of its 8 tokens and transposes them 4 x 4.
//
// Arithmetic: int8 and e4m3 codes are exact in bf16 and f16, and so are the
// caches' 16-bit elements in their own type.  Queries enter with all their bits:
// f16 and bf16 ones in their own type, f32 ones as a sum of 3 bf16 terms (8 bits
// each, cut off: rounded, a query near the largest float would become infinite).  So
// scores have fp32 accuracy.
// p v_scale enters the second product in 2 bf16 terms for 16-bit outputs (16
// bits of it; one term would add as much error as the output's own rounding,
// and the matrix instructions have the time) and 3 for f32 (24).  An F16 cache
// takes f16 queries and p in 2 f16 terms (22 bits), raised by 2^7 so that a p down to
// 2^-10 of the running maximum keeps all of them and one down to 2^-21 its first 11.
// Maxima, sums and outputs are fp32 throughout.
//
// Bytes of K and V are the bound, once for each 16 query heads of a key-value head:
// the workgroups of further 16s fetch them again (32 sequences of 3000 tokens over 1
// head of 128 in bf16 21.8 us with 16 query heads, 23.5 with 32, 37.3 with 64).
// Registers hold what is in flight: 8 waves a workgroup, one or two workgroups a CU,
// each wave with a tile's keys and values (8 KB of int8 at 128) on the way.  96
// sequences of 3000 tokens, 8 heads of 128: 111 us in int8 (5.5 TB/s), 205 us in bf16
// (5.75 TB/s).
//
// The running maximum m only moves when a score passes it by more than 8
// (powers of two, where p and its sums lose nothing), so most tiles need no
// exchange between lanes at all.
//
// Values of the largest magnitudes: sums of up to 2^8 p v over 2^30 tokens can
// pass the largest float where their mean does not; and where v or k is infinite,
// a second term of p or q that is 0 or of the other sign makes NaN of it.  A wave
// whose sums have passed 2^100 or become NaN takes its tiles once more, with
// infinities and NaN left out of all products but the first term's, and with m raised
// by 40: p stays below 2^-32, all its sums below 2^126, and the 8 waves' and 256
// chunks' sums below that still (their tokens are 2^30 together).  Exponents of p then
// hold up to 48 + what they held, 2^-19 off.  Every other wave's sums are below 2^100,
// so what they join to is finite.  Sums of F16 values stay below 2^61: there m is not
// raised.
//
// A tile's keys and values stay in registers and are loaded one tile ahead: the
// next keys once this tile's scores are formed, the next values once they
// are added.  Bound by the cache's bytes.
#pragma once

#include "pk_decode.h"

#include <cfloat>
#include <type_traits>

namespace pkgpu {
namespace decode {

struct PagedArgs {
    const char *k, *v;
    const float *k_scale, *v_scale;
    const char* q;
    size_t ldq;                  // bytes
    const int* pages;
    size_t ld_pages;
    const int* lens;
    char* out;
    size_t ldo;                  // bytes
    float* lse;
    float* part;                 // [B][heads][splits][dim], then
    float* ml;                   // [B][heads][splits][2]
    float scale2;                // scale * log2(e)
    int B, max_len, window;
    int kv_heads, group, head_tiles;
    int n_pages, page_shift;
    int chunk, splits;
    int longest_first;
};

// Tokens a sequence's new token sees, from `first` on; chunks start at `base`.
struct Span { int first, base, len, chunks; };
__device__ __host__ inline Span span_of(int len, int max_len, int window, int chunk)
{
    Span s;
    s.len = len < 0 ? 0 : len > max_len ? max_len : len;
    s.first = window > 0 && s.len > window ? s.len - window : 0;
    s.base = s.first & ~31;
    s.chunks = s.len > s.first ? (s.len - s.base + chunk - 1) / chunk : 0;
    return s;
}

// Waves of a workgroup, all of one chunk.  8 keep one CU's share of the memory
// busy by themselves; which sequences are split all the same, cuts() says.  The
// kernels with most registers (heads of 256, queries in 3 terms) run one wave a
// SIMD: 64 sequences of 2000 tokens, 2 heads of 256 in int8, f32 queries 34.8 us;
// 8 waves, which spill, 44.
constexpr int waves_of(int cache, int t, int dim) { return t == F32 && dim == 256 ? 4 : 8; }

// The sequence with nth sequences before it in order of falling length (ties
// by index), counted by every workgroup for itself: lens of the launch's up to
// kSortedMax sequences in LDS, a thread a sequence.
constexpr int kSortedMax = 256;
__device__ inline int nth_longest(const PagedArgs& a, int nth, int* lens, int wave)
{
    const int i = threadIdx.x;
    const int quads = (a.B + 3) / 4;
    int mine = i < a.B ? a.lens[i] : -1;
    mine = mine < 0 ? (i < a.B ? 0 : -1) : mine > a.max_len ? a.max_len : mine;
    if (i < 4 * quads) lens[i] = mine;
    __syncthreads();
    int rank = 0;
    if (64 * wave < a.B) {
#pragma unroll 1
        for (int q = 0; q < quads; ++q) {
            const i32x4 l = reinterpret_cast<const i32x4*>(lens)[q];
#pragma unroll
            for (int j = 0; j < 4; ++j) rank += l[j] > mine || (l[j] == mine && 4 * q + j < i);
        }
        if (i < a.B && rank == nth) lens[kSortedMax] = i;
    }
    __syncthreads();
    const int b = __builtin_amdgcn_readfirstlane(lens[kSortedMax]);
    __syncthreads();                           // the array is free again
    return b;
}

// Terms of the query and of p: see above.
// Whether the scores are formed in f16: its own caches, and f16 queries over
// codes, which f16 holds exactly too.
constexpr bool keys_f16(int cache, int t) { return cache == F16 || t == F16; }
constexpr int q_terms(int cache, int t) { return t == F32 ? 3 : 1; }
constexpr int p_terms(int t) { return t == F32 ? 3 : 2; }

template <bool IN_F16>
__device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c)
{
    if constexpr (IN_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 4 codes to 4 bf16 or f16, exactly.
template <int CACHE, bool IN_F16>
__device__ inline u32x2 codes_16(uint32_t w)
{
    if constexpr (CACHE == I8) {
        const uint32_t a = __float_as_uint((float)(int)(signed char)w);
        const uint32_t b = __float_as_uint((float)(int)(signed char)(w >> 8));
        const uint32_t c = __float_as_uint((float)(int)(signed char)(w >> 16));
        const uint32_t d = __float_as_uint((float)(int)(signed char)(w >> 24));
        if constexpr (IN_F16)
            return (u32x2){__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(a), __uint_as_float(b))),
                           __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(c), __uint_as_float(d)))};
        else
            return (u32x2){__builtin_amdgcn_perm(b, a, 0x07060302u), __builtin_amdgcn_perm(d, c, 0x07060302u)};
    } else if constexpr (IN_F16) {
        const f16x2 l = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false);
        const f16x2 h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true);
        return (u32x2){__builtin_bit_cast(uint32_t, l), __builtin_bit_cast(uint32_t, h)};
    } else {
        const bf16x2 l = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false);
        const bf16x2 h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
        return (u32x2){__builtin_bit_cast(uint32_t, l), __builtin_bit_cast(uint32_t, h)};
    }
}

// 8 elements with infinities and NaN as zeros.
template <bool IN_F16>
__device__ inline u32x4 finite_of(u32x4 f)
{
    constexpr uint32_t EXP = IN_F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
    for (int d = 0; d < 4; ++d)
        f[d] &= ((f[d] & EXP) != EXP ? 0xffffu : 0u) | ((f[d] >> 16 & EXP) != EXP ? 0xffff0000u : 0u);
    return f;
}
// x as the sum of 3 bf16 terms, exactly: 8 bits of it each.
__device__ inline void cut_pair(float x, float y, uint32_t* t)
{
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        t[i] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
        x = __fsub_rn(x, bf16_lo(t[i]));
        y = __fsub_rn(y, bf16_hi(t[i]));
    }
}
// x as TERMS terms of the matrix type, the first the largest.
template <bool IN_F16, int TERMS>
__device__ inline void split_pair(float x, float y, uint32_t* t)
{
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        t[i] = IN_F16 ? pack_f16(x, y) : pack_bf16(x, y);
        if (i + 1 == TERMS) break;
        const f16x2 h = __builtin_bit_cast(f16x2, t[i]);
        x = __fsub_rn(x, IN_F16 ? (float)h[0] : bf16_lo(t[i]));
        y = __fsub_rn(y, IN_F16 ? (float)h[1] : bf16_hi(t[i]));
    }
}

template <int CACHE, int T, int DIM>
__global__ void __launch_bounds__(64 * waves_of(CACHE, T, DIM), waves_of(CACHE, T, DIM) / 4) paged_attention(PagedArgs a)
{
    constexpr int NW = waves_of(CACHE, T, DIM);
    constexpr int S = size_of(CACHE);
    constexpr bool CODED = CACHE == I8 || CACHE == E4M3;
    constexpr int KL = DIM * S / 64;           // 16-byte pieces of a key a lane holds
    constexpr int STEPS = DIM / 32;            // matrix instructions along a head
    constexpr int VB = DIM * S / 16;           // bytes of a value a lane holds
    constexpr int VW = VB / 4;
    constexpr int E = DIM / 16;                // elements of those, accumulators
    constexpr int QT = q_terms(CACHE, T), PT = p_terms(T);
    constexpr float BIAS = CACHE == F16 ? 7.0f : 0.0f;
    constexpr bool KF = keys_f16(CACHE, T), VF = CACHE == F16;  // types of the two products

    union Shared {
        int lens[kSortedMax + 4];
        u32x4 q[STEPS][QT][64];
        f32x4 buf[NW - 1][E][64];
    };
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;

    // Workgroups go round the 8 L2s.  Chunks slowest, and the pairs of a chunk
    // rotated by its index, so that neither a chunk index (the last ones of ragged
    // sequences are mostly empty) nor a long sequence stays on one of them.
    const uint32_t pairs = (uint32_t)a.B * a.kv_heads * a.head_tiles;
    const int split = blockIdx.x / pairs;
    uint32_t x = (blockIdx.x + split) % pairs;
    const int htile = x % (uint32_t)a.head_tiles;
    x /= (uint32_t)a.head_tiles;
    const int kvh = x % (uint32_t)a.kv_heads;
    int b = x / (uint32_t)a.kv_heads;
    if (a.longest_first) b = nth_longest(a, b, sh.lens, wave);

    const int* const pages = a.pages + (size_t)b * a.ld_pages;
    const int page_mask = (1 << a.page_shift) - 1;
    const int len = a.lens[b];
    // entries of the first two tiles, before the length is here (no window: the
    // chunk's tokens do not depend on it; table rows hold max_len tokens)
    int early[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const long long tt = (long long)split * a.chunk + 32 * (wave + i * NW) + 16 * u;
            early[i][u] = a.window == 0 && tt < a.max_len ? pages[tt >> a.page_shift] : -1;
        }

    const int in_group = htile * 16 + n;
    const bool head_ok = in_group < a.group;
    const int heads = a.kv_heads * a.group;
    const int head = kvh * a.group + in_group;

    // queries: step c takes elements el(c, i) = i + 8 g + 32 c of a 16-bit cache's
    // rows, i + 16 g + 8 (c % 2) + 64 (c / 2) of an 8-bit one's; every wave reads
    // the same ones, in the order they are multiplied, from LDS
    constexpr int QS = (STEPS + NW - 1) / NW;  // steps a wave stages
    float qv[QS][8] = {};
#pragma unroll
    for (int i = 0; i < QS; ++i) {
        const int c = wave + i * NW;
        const int el = S == 2 ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c % 2);
        if (c < STEPS && head_ok)
            load8<T>(a.q + (size_t)b * a.ldq + ((size_t)head * DIM + el) * size_of(T), qv[i]);
    }

    const Span sp = span_of(len, a.max_len, a.window, a.chunk);
    if (split > 0 && split >= sp.chunks) return;
    const int begin = sp.base + split * a.chunk;
    const int end = sp.chunks ? min(sp.len, begin + a.chunk) : begin;

    // the two 16-token halves of the tile at token t: first cache row, presence
    struct Halves { size_t row[2]; bool ok[2]; };
    auto half = [&](Halves& h, int u, int tt, int id) {
        id = __builtin_amdgcn_readfirstlane(tt < end ? id : -1);     // the wave's: rows' addresses stay scalar
        h.ok[u] = (uint32_t)id < (uint32_t)a.n_pages;
        h.row[u] = (((size_t)(h.ok[u] ? id : 0) * a.kv_heads + kvh) << a.page_shift) + (tt & page_mask);
    };
    auto halves = [&](int t) {
        Halves h;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int tt = t + 16 * u;
            half(h, u, tt, tt < end ? pages[tt >> a.page_shift] : -1);
        }
        return h;
    };

    u32x4 kr[2][KL];
    uint32_t vr[2][4][VW];
    f32x4 ks[2], vs[2];
    // scalar base + this lane's offset + a constant
    const uint32_t k_off = n * (DIM * S) + 16 * g;
    const uint32_t v_off = 4 * g * (DIM * S) + n * (VB > 16 ? 16 : VB);
    const uint32_t s_off = 16 * g;
    auto load_k = [&](const Halves& h) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* base = a.k + h.row[u] * (DIM * S);
#pragma unroll
            for (int j = 0; j < KL; ++j) kr[u][j] = *reinterpret_cast<const u32x4*>(base + k_off + 64 * j);
            if constexpr (CODED)
                ks[u] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(a.k_scale + h.row[u]) + s_off);
        }
    };
    auto load_v = [&](const Halves& h) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const char* base = a.v + h.row[u] * (DIM * S);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const char* p = base + v_off + i * (DIM * S);
                if constexpr (VB == 4) {
                    vr[u][i][0] = *reinterpret_cast<const uint32_t*>(p);
                } else if constexpr (VB == 8) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(p);
                    vr[u][i][0] = w[0]; vr[u][i][1] = w[1];
                } else {
#pragma unroll
                    for (int j = 0; j < VB / 16; ++j) {
                        const u32x4 w = *reinterpret_cast<const u32x4*>(p + 256 * j);
#pragma unroll
                        for (int d = 0; d < 4; ++d) vr[u][i][4 * j + d] = w[d];
                    }
                }
            }
            if constexpr (CODED)
                vs[u] = *reinterpret_cast<const f32x4*>(reinterpret_cast<const char*>(a.v_scale + h.row[u]) + s_off);
        }
    };

    float m = -FLT_MAX, l = 0.0f;
    f32x4 acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};

    int t = begin + 32 * wave;
    Halves cur{}, next{};
    if (t < end) {
        if (a.window == 0) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                half(cur, u, t + 16 * u, early[0][u]);
                half(next, u, t + 32 * NW + 16 * u, early[1][u]);
            }
        } else {
            cur = halves(t);
            next = halves(t + 32 * NW);
        }
        load_k(cur);
        load_v(cur);
    }
#pragma unroll
    for (int i = 0; i < QS; ++i) {
        const int c = wave + i * NW;
        if (c >= STEPS) break;
        u32x4 f[QT];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            uint32_t w[QT];
            if constexpr (QT == 3) cut_pair(qv[i][2 * d], qv[i][2 * d + 1], w);
            else split_pair<KF, QT>(qv[i][2 * d], qv[i][2 * d + 1], w);
#pragma unroll
            for (int j = 0; j < QT; ++j) f[j][d] = w[j];
        }
#pragma unroll
        for (int j = 0; j < QT; ++j) sh.q[c][j][lane] = f[j];
    }
    __syncthreads();
    // One tile.  The last one of a wave is a copy of its own without loads: loads
    // on a condition would have every wait for this tile's values wait for the
    // next one's keys too.  So are tiles that are taken once more.
    auto tile = [&](auto last, auto again) {
        constexpr bool MORE = !decltype(last)::value, AGAIN = decltype(again)::value;
        Halves after{};
        if constexpr (MORE) after = halves(t + 64 * NW);

        // scores
        f32x4 s[2] = {(f32x4){0.0f, 0.0f, 0.0f, 0.0f}, (f32x4){0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            u32x4 qf[QT];
#pragma unroll
            for (int j = 0; j < QT; ++j) qf[j] = sh.q[c][j][lane];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 f;
                if constexpr (CODED) {
                    const u32x2 lo = codes_16<CACHE, KF>(kr[u][c / 2][2 * (c % 2)]);
                    const u32x2 hi = codes_16<CACHE, KF>(kr[u][c / 2][2 * (c % 2) + 1]);
                    f = (u32x4){lo[0], lo[1], hi[0], hi[1]};
                } else {
                    f = kr[u][c];
                }
#pragma unroll
                for (int j = QT - 1; j >= 0; --j)
                    s[u] = mfma<KF>(AGAIN && !CODED && j > 0 ? finite_of<KF>(f) : f, qf[j], s[u]);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                s[u][r] = __fmul_rn(s[u][r], CODED ? __fmul_rn(ks[u][r], a.scale2) : a.scale2);
        if constexpr (MORE) load_k(next);

        const bool whole = t >= sp.first && t + 32 <= end && cur.ok[0] && cur.ok[1];
        if (!whole) {
            // masked tokens: no score, and no value either (0 * NaN is NaN)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int tok = t + 16 * u + 4 * g + r;
                    const bool in = cur.ok[u] && tok >= sp.first && tok < end;
                    if (!in) {
                        s[u][r] = -__builtin_inff();
                        if constexpr (CODED) vs[u][r] = 0.0f;
#pragma unroll
                        for (int d = 0; d < VW; ++d) vr[u][r][d] = 0;
                    }
                }
        }

        float top = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                          fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        if constexpr (AGAIN && !VF) top = __fadd_rn(top, 40.0f);
        if (__any(top > m + 8.0f)) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float mn = fmaxf(m, top);
            const float f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l = __fmul_rn(l, f);
#pragma unroll
            for (int e = 0; e < E; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[e][r] = __fmul_rn(acc[e][r], f);
        }

        u32x4 p[PT];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = __builtin_amdgcn_exp2f(s[u][r] - m + BIAS);
                l = __fadd_rn(l, e);
                w[r] = CODED ? __fmul_rn(e, vs[u][r]) : e;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t pt[PT];
                split_pair<VF, PT>(w[2 * h], w[2 * h + 1], pt);
#pragma unroll
                for (int j = 0; j < PT; ++j) p[j][2 * u + h] = pt[j];
            }
        }

        // O^T += V^T P^T
        if constexpr (CODED) {
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                uint32_t y[2][4];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t a0 = vr[u][0][w], a1 = vr[u][1][w], a2 = vr[u][2][w], a3 = vr[u][3][w];
                    const uint32_t l01 = __builtin_amdgcn_perm(a1, a0, 0x05010400u);
                    const uint32_t h01 = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
                    const uint32_t l23 = __builtin_amdgcn_perm(a3, a2, 0x05010400u);
                    const uint32_t h23 = __builtin_amdgcn_perm(a3, a2, 0x07030602u);
                    y[u][0] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
                    y[u][1] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
                    y[u][2] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
                    y[u][3] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const u32x2 lo = codes_16<CACHE, VF>(y[0][i]), hi = codes_16<CACHE, VF>(y[1][i]);
                    const u32x4 f = (u32x4){lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                    for (int j = PT - 1; j >= 0; --j) acc[4 * w + i] = mfma<VF>(f, p[j], acc[4 * w + i]);
                }
            }
        } else {
#pragma unroll
            for (int w = 0; w < VW; ++w) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t sel = i ? 0x07060302u : 0x05040100u;
                    u32x4 f;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        f[2 * u] = __builtin_amdgcn_perm(vr[u][1][w], vr[u][0][w], sel);
                        f[2 * u + 1] = __builtin_amdgcn_perm(vr[u][3][w], vr[u][2][w], sel);
                    }
#pragma unroll
                    for (int j = PT - 1; j >= 0; --j)
                        acc[2 * w + i] = mfma<VF>(AGAIN && j > 0 ? finite_of<VF>(f) : f, p[j], acc[2 * w + i]);
                }
            }
        }
        if constexpr (MORE) load_v(next);
        cur = next;
        next = after;
        t += 32 * NW;
    };
    if (t < end) {
        while (t + 32 * NW < end) tile(std::false_type{}, std::false_type{});
        tile(std::true_type{}, std::false_type{});
        float size[4] = {};
#pragma unroll
        for (int e = 0; e < E; ++e)
#pragma unroll
            for (int r = 0; r < 4; ++r) size[r] = __fadd_rn(size[r], fabsf(acc[e][r]));
        const float sum = __fadd_rn(__fadd_rn(size[0], size[1]), __fadd_rn(size[2], size[3]));
        if (__any(!(sum < 0x1p100f))) {
            m = -FLT_MAX;
            l = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (t = begin + 32 * wave; t < end;) {
                cur = halves(t);
                load_k(cur);
                load_v(cur);
                tile(std::true_type{}, std::true_type{});
            }
        }
    }

    // join the waves: the same registers of the same lanes, in wave order
    l = __fadd_rn(l, __shfl_xor(l, 16));
    l = __fadd_rn(l, __shfl_xor(l, 32));
    __shared__ float ml[NW][2][16];
    if (g == 0) { ml[wave][0][n] = m; ml[wave][1][n] = l; }
    __syncthreads();                           // and nobody reads queries any more
    float mx = ml[0][0][n];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, ml[w][0][n]);
    const float f = __builtin_amdgcn_exp2f(m - mx);
#pragma unroll
    for (int e = 0; e < E; ++e) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[e][r] = __fmul_rn(acc[e][r], f);
        if (wave > 0) sh.buf[wave - 1][e][lane] = acc[e];
    }
    __syncthreads();
    if (wave > 0) return;
    float lt = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w)
        lt = __fadd_rn(lt, __fmul_rn(ml[w][1][n], __builtin_amdgcn_exp2f(ml[w][0][n] - mx)));
#pragma unroll 1                   // the loop above, not this one, sets the registers
    for (int w = 0; w < NW - 1; ++w)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const f32x4 o = sh.buf[w][e][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[e][r] = __fadd_rn(acc[e][r], o[r]);
        }
    if (!head_ok) return;

    // element e of row 4 g + r stands for el = (4 g + r) E + e of the head (or,
    // where a lane holds 32 bytes, 128 (e / 8) + 8 (4 g + r) + e % 8)
    const bool direct = sp.chunks <= 1;
    const float inv = lt == 0.0f ? 0.0f : __fdiv_rn(1.0f, lt);
    constexpr int RUN = VB > 16 ? 8 : E;       // consecutive elements
    const size_t row = (size_t)b * heads + head;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int h = 0; h < E / RUN; ++h) {
            const int el = VB > 16 ? 128 * h + 8 * (4 * g + r) : (4 * g + r) * E;
            float o[RUN];
#pragma unroll
            for (int i = 0; i < RUN; ++i) o[i] = acc[h * RUN + i][r];
            if (direct) {
#pragma unroll
                for (int i = 0; i < RUN; ++i) o[i] = lt == 0.0f ? 0.0f : __fmul_rn(o[i], inv);
                char* p = a.out + (size_t)b * a.ldo + ((size_t)head * DIM + el) * size_of(T);
                if constexpr (RUN >= 8) {
#pragma unroll
                    for (int i = 0; i < RUN; i += 8) store8<T>(p + i * size_of(T), o + i);
                } else if constexpr (T == F32) {
                    *reinterpret_cast<f32x4*>(p) = (f32x4){o[0], o[1], o[2], o[3]};
                } else {
                    *reinterpret_cast<u32x2*>(p) = T == F16 ? (u32x2){pack_f16(o[0], o[1]), pack_f16(o[2], o[3])}
                                                            : (u32x2){pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
                }
            } else {
                float* p = a.part + (row * a.splits + split) * DIM + el;
#pragma unroll
                for (int i = 0; i < RUN; i += 4)
                    *reinterpret_cast<f32x4*>(p + i) = (f32x4){o[i], o[i + 1], o[i + 2], o[i + 3]};
            }
        }
    }
    if (g == 0) {
        if (direct) {
            if (a.lse) a.lse[row] = lt == 0.0f ? -__builtin_inff()
                                               : __fmul_rn(__fadd_rn(mx - BIAS, __builtin_amdgcn_logf(lt)),
                                                           0.69314718055994531f);
        } else {
            a.ml[(row * a.splits + split) * 2] = mx - BIAS;
            a.ml[(row * a.splits + split) * 2 + 1] = lt;
        }
    }
}

hipError_t launch_paged_f16(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_paged_bf16(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_paged_i8(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_paged_e4m3(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);

template <int CACHE, int T>
hipError_t launch_paged(int dim, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    const dim3 block(64 * waves_of(CACHE, T, dim));
    return dim == 64    ? launch(paged_attention<CACHE, T, 64>, grid, block, 0, s, a)
           : dim == 128 ? launch(paged_attention<CACHE, T, 128>, grid, block, 0, s, a)
                        : launch(paged_attention<CACHE, T, 256>, grid, block, 0, s, a);
}

}  // namespace decode
}  // namespace pkgpu
