// pk_rope.hip - rotary positions: of rows (pk_gpu_rope_dev), and of a step's queries and
// keys with the keys' and values' way into the cache (pk_gpu_rope_kv_write_dev).
//
//   a' = (a cos t - b sin t) scale,   b' = (b cos t + a sin t) scale,   t = p freq_i
//
// A workgroup takes up to 4 tokens.  It forms cos and sin of their angles once, one angle a
// thread, into LDS (fp64 for the product and the reduction, so that far positions keep
// their bits); a thread then keeps those of its elements in registers over all heads.
// Bound by the rows' bytes, each read and written once: 8191 tokens of 32 + 8 + 8 heads
// of 128 in bf16, keys and values into int8 codes, 32 us, 5.8 TB/s (passes over the same rows, some
// of which the card's large cache then holds: a copy of 1 GiB makes 5.15); 4001 rows of 16 heads of
// 64 in f32 8.6, 3.8.
#include "pk_kv_rows.h"

#include <cmath>

namespace pkgpu {
namespace decode {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;          // of a workgroup where there are many
constexpr int kMostDim = 1024;

struct RopeArgs {
    const float* freqs;
    float scale;
    int rot, interleaved;
    const int* pos;
    int n, tokens;                  // all, and of a workgroup
    const char* x;                  // rows that are turned
    char* y;
    size_t ldx, ldy;                // elements
    int heads, dim;
    int wide;                       // 8 elements at a time
    // keys and values and the cache that takes them
    const char *rk, *rv;
    size_t ldk, ldv;
    void *k, *v;
    float *k_scale, *v_scale;
    const int* slots;
    int kv_heads, page_shift, n_slots;
};

struct Turn { float c, s; };

// cos and sin of p freq, times scale.  The angle is reduced in fp64; what its rounding
// to fp32 leaves enters by the first order (its square is below 2^-46).
__device__ inline Turn turn_of(int p, float freq, float scale)
{
    const double t = (double)p * (double)freq;
    const double k = __builtin_rint(t * 0.15915494309189535);       // 1 / (2 pi)
    double r = __builtin_fma(-k, 6.283185307179586, t);             // 2 pi, its nearest double and the rest
    r = __builtin_fma(-k, 2.4492935982947064e-16, r);
    const float f = (float)r, d = (float)(r - (double)f);
    float s, c;
    sincosf(f, &s, &c);
    return {__fmul_rn(__builtin_fmaf(-s, d, c), scale), __fmul_rn(__builtin_fmaf(c, d, s), scale)};
}

__device__ inline float first_of(float a, float b, Turn t) { return __builtin_fmaf(a, t.c, -__fmul_rn(b, t.s)); }
__device__ inline float second_of(float a, float b, Turn t) { return __builtin_fmaf(b, t.c, __fmul_rn(a, t.s)); }

// The workgroup's angles: turns[token][pair].
__device__ inline void make_turns(const RopeArgs& a, int token0, int tokens, Turn* turns)
{
    const int half = a.rot / 2;
    for (int i = threadIdx.x; i < tokens * half; i += kThreads) {
        const int t = i / half;
        turns[i] = turn_of(a.pos[token0 + t], a.freqs[i - t * half], a.scale);
    }
    __syncthreads();
}

// The heads of the workgroup's rows.  A thread has one place of a head (8 pairs of
// the half layout, 4 of the interleaved one, 8 elements that stay; one pair or element
// where rows are not wide) and goes over tokens and heads; it reads both elements of its
// pairs before it writes them, so rows may be turned in place.
template <int T>
__device__ inline void turn_rows(const RopeArgs& a, int token0, int tokens, const Turn* turns)
{
    constexpr int S = size_of(T);
    const int half = a.rot / 2, per = a.wide ? 8 : 1;
    const int turning = a.wide ? (a.interleaved ? a.rot / 8 : a.rot / 16) : half;
    const int rest = a.x == a.y ? 0 : (a.dim - a.rot) / per;
    const int places = turning + rest;
    const int lanes = places < kThreads ? places : kThreads, step = kThreads / lanes;
    const int head0 = threadIdx.x / lanes;
    if (head0 >= step) return;
    for (int u = threadIdx.x - head0 * lanes; u < places; u += lanes) {
        const bool turns_here = u < turning;
        // first element of the place, and of its partners
        const int e = turns_here ? (a.interleaved && !a.wide ? 2 * u : per * u) : a.rot + per * (u - turning);
        const int o = a.interleaved ? e + 1 : e + half;
        for (int t = 0; t < tokens; ++t) {
            const char* const x = a.x + (size_t)(token0 + t) * a.ldx * S;
            char* const y = a.y + (size_t)(token0 + t) * a.ldy * S;
            const Turn* const of = turns + t * half;
            if (!a.wide) {
                const Turn w = turns_here ? of[u] : Turn{1.0f, 0.0f};
                for (int h = head0; h < a.heads; h += step) {
                    const size_t at = (size_t)h * a.dim;
                    const float p = load1<T>(x, at + e);
                    if (!turns_here) {
                        store1<T>(y, at + e, p);
                        continue;
                    }
                    const float q = load1<T>(x, at + o);
                    store1<T>(y, at + e, first_of(p, q, w));
                    store1<T>(y, at + o, second_of(p, q, w));
                }
                continue;
            }
            Turn w[8];
            if (turns_here) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    w[i] = a.interleaved ? of[e / 2 + i / 2] : of[e + i];
            }
            for (int h = head0; h < a.heads; h += step) {
                const size_t at = (size_t)h * a.dim;
                float p[8];
                load8<T>(x + (at + e) * S, p);
                if (turns_here && a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float q = p[i];
                        p[i] = first_of(q, p[i + 1], w[i]);
                        p[i + 1] = second_of(q, p[i + 1], w[i]);
                    }
                } else if (turns_here) {
                    float q[8];
                    load8<T>(x + (at + o) * S, q);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float b = q[i];
                        q[i] = second_of(p[i], b, w[i]);
                        p[i] = first_of(p[i], b, w[i]);
                    }
                    store8<T>(y + (at + o) * S, q);
                }
                store8<T>(y + (at + e) * S, p);
            }
        }
    }
}

struct Part { int token0, tokens; };
__device__ inline Part part_of(const RopeArgs& a)
{
    const int token0 = blockIdx.x * a.tokens;
    return {token0, min(a.tokens, a.n - token0)};
}

template <int T>
__global__ void __launch_bounds__(kThreads) rope_rows(RopeArgs a)
{
    extern __shared__ Turn turns[];
    const Part p = part_of(a);
    make_turns(a, p.token0, p.tokens, turns);
    turn_rows<T>(a, p.token0, p.tokens, turns);
}

// Keys and values as pk_kv_cache.hip writes them, 8 elements of a row a lane; a lane
// of the half layout reads its elements' partners too.
template <int CACHE, int T, int DIM>
__global__ void __launch_bounds__(kThreads) rope_kv_write(RopeArgs a)
{
    constexpr int LANES = DIM / 8, S = size_of(T), ROWS = kThreads / LANES;
    extern __shared__ Turn turns[];
    const Part w = part_of(a);
    make_turns(a, w.token0, w.tokens, turns);
    const int part = threadIdx.x % LANES, half = a.rot / 2, e0 = 8 * part;
    for (int r = threadIdx.x / LANES; r < a.kv_heads * w.tokens; r += ROWS) {      // whole lane groups leave together
        const int t = r / a.kv_heads, head = r - t * a.kv_heads, token = w.token0 + t;
        const long long row = cache_row(a.slots[token], head, a.kv_heads, a.page_shift, a.n_slots);
        const size_t at = (size_t)head * DIM;
        const char* const xk = a.rk + (size_t)token * a.ldk * S;
        const Turn* const of = turns + t * half;
        float k[8], v[8];
        load8<T>(xk + (at + e0) * S, k);
        load8<T>(a.rv + ((size_t)token * a.ldv + at + e0) * S, v);
        if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 8; i += 2)
                if (e0 + i < a.rot) {
                    const Turn f = of[(e0 + i) / 2];
                    const float x = k[i];
                    k[i] = first_of(x, k[i + 1], f);
                    k[i + 1] = second_of(x, k[i + 1], f);
                }
        } else if (e0 < a.rot) {
            float o[8];
            if (half % 8 == 0) {
                load8<T>(xk + (at + (e0 < half ? e0 + half : e0 - half)) * S, o);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = e0 + i;
                    o[i] = e < a.rot ? load1<T>(xk, at + (e < half ? e + half : e - half)) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = e0 + i;
                if (e < half) k[i] = first_of(k[i], o[i], of[e]);
                else if (e < a.rot) k[i] = second_of(o[i], k[i], of[e - half]);
            }
        }
        write_part<CACHE, DIM>(a.k, a.k_scale, row, part, k);
        write_part<CACHE, DIM>(a.v, a.v_scale, row, part, v);
    }
    if (a.heads) turn_rows<T>(a, w.token0, w.tokens, turns);
}

struct Launch { long long workgroups; size_t lds; };
// 4 tokens a workgroup from 416 such workgroups on, else one: an angle a thread at 128
// turning elements, and less of it to wait for before rows move.  Measured (us, 4 and
// one; 32 + 8 + 8 heads of 128 in bf16 and into bf16):
//   1500 tokens  12.6 11.6      1800  13.1 13.6      8191  43.6 62.4
Launch launch_of(RopeArgs* a)
{
    a->tokens = a->n >= 416 * kTokens ? kTokens : 1;
    return {((long long)a->n + a->tokens - 1) / a->tokens, (size_t)a->tokens * (a->rot / 2) * sizeof(Turn)};
}

int check_rope(const pk_gpu_rope* r, const char* who, int dtype, int heads, int dim, int n)
{
    if (!r) return rt::error(PK_GPU_EINVAL, "%s: NULL rope", who);
    if (!is_float(dtype)) return rt::error(PK_GPU_EINVAL, "%s: rows of type %d (F32, F16 or BF16)", who, dtype);
    if (n < 0 || heads < 0) return rt::error(PK_GPU_EINVAL, "%s: n = %d, heads = %d", who, n, heads);
    if (r->rot_dim < 2 || r->rot_dim % 2 || r->rot_dim > dim)
        return rt::error(PK_GPU_EINVAL, "%s: rot_dim = %d of a head of %d (even, 2 at least)", who, r->rot_dim, dim);
    if (!(std::fabs(r->scale) <= 3.4e38f)) return rt::error(PK_GPU_EINVAL, "%s: scale = %g", who, r->scale);
    if (!r->freqs) return rt::error(PK_GPU_EINVAL, "%s: NULL frequencies", who);
    if (!aligned(r->freqs, 4)) return rt::error(PK_GPU_EINVAL, "%s: frequencies are not aligned to a float", who);
    return PK_GPU_OK;
}

// whether 8 elements may go at a time
bool wide_rows(const RopeArgs& a, int es)
{
    return a.dim % 8 == 0 && a.rot % (a.interleaved ? 8 : 16) == 0 && aligned16(a.x) && aligned16(a.y) &&
           a.ldx * es % 16 == 0 && a.ldy * es % 16 == 0;
}

RopeArgs rope_args(const pk_gpu_rope* r, const int* pos, int n, const void* x, int ldx, int heads, int dim, void* y, int ldy)
{
    RopeArgs a{};
    a.freqs = r->freqs;
    a.scale = r->scale;
    a.rot = r->rot_dim;
    a.interleaved = r->interleaved != 0;
    a.pos = pos;
    a.n = n;
    a.x = static_cast<const char*>(x);
    a.y = static_cast<char*>(y);
    a.ldx = ldx;
    a.ldy = ldy;
    a.heads = heads;
    a.dim = dim;
    return a;
}

template <int CACHE, int T>
hipError_t launch_dim(dim3 grid, size_t lds, const RopeArgs& a, hipStream_t s)
{
    const dim3 block(kThreads);
    return a.dim == 64    ? launch(rope_kv_write<CACHE, T, 64>, grid, block, lds, s, a)
           : a.dim == 128 ? launch(rope_kv_write<CACHE, T, 128>, grid, block, lds, s, a)
                          : launch(rope_kv_write<CACHE, T, 256>, grid, block, lds, s, a);
}
template <int CACHE>
hipError_t launch_rows(int t, dim3 grid, size_t lds, const RopeArgs& a, hipStream_t s)
{
    return t == F32   ? launch_dim<CACHE, F32>(grid, lds, a, s)
           : t == F16 ? launch_dim<CACHE, F16>(grid, lds, a, s)
                      : launch_dim<CACHE, BF16>(grid, lds, a, s);
}

}  // namespace
}  // namespace decode
}  // namespace pkgpu

extern "C" {

using namespace pkgpu::decode;
namespace rt = pkgpu::rt;

int pk_gpu_rope_freqs(int rot_dim, double base, int scaling, double factor, double trained, double slow, double fast,
                      float* freqs)
{
    const char* who = "rope frequencies";
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > kMostDim)
        return rt::error(PK_GPU_EINVAL, "%s: rot_dim = %d (even, 2 to %d)", who, rot_dim, kMostDim);
    if (!(base > 0.0) || !std::isfinite(base)) return rt::error(PK_GPU_EINVAL, "%s: base = %g", who, base);
    if (scaling < PK_GPU_ROPE_PLAIN || scaling > PK_GPU_ROPE_PARTS)
        return rt::error(PK_GPU_EINVAL, "%s: scaling = %d", who, scaling);
    if (scaling != PK_GPU_ROPE_PLAIN && (!(factor > 0.0) || !std::isfinite(factor)))
        return rt::error(PK_GPU_EINVAL, "%s: factor = %g", who, factor);
    if (scaling == PK_GPU_ROPE_BASE && rot_dim < 4)
        return rt::error(PK_GPU_EINVAL, "%s: rot_dim = %d has one frequency, which no base changes", who, rot_dim);
    if (scaling == PK_GPU_ROPE_PARTS &&
        (!(trained > 0.0) || !(slow >= 0.0) || !(fast > slow) || !std::isfinite(trained) || !std::isfinite(fast)))
        return rt::error(PK_GPU_EINVAL, "%s: trained = %g, slow = %g, fast = %g", who, trained, slow, fast);
    if (!freqs) return rt::error(PK_GPU_EINVAL, "%s: NULL freqs", who);
    if (scaling == PK_GPU_ROPE_BASE) base *= std::pow(factor, (double)rot_dim / (rot_dim - 2));
    auto freq = [&](int i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == PK_GPU_ROPE_LINEAR) f /= factor;
        if (scaling == PK_GPU_ROPE_PARTS) {
            double keep = (trained * f / 6.283185307179586 - slow) / (fast - slow);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f = f * keep + f / factor * (1.0 - keep);
        }
        return (float)f;
    };
    for (int i = 0; i < rot_dim / 2; ++i)
        if (!std::isfinite(base) || !std::isfinite(freq(i)))
            return rt::error(PK_GPU_EINVAL, "%s: base = %g, factor = %g give frequencies that floats do not hold", who, base,
                             factor);
    for (int i = 0; i < rot_dim / 2; ++i) freqs[i] = freq(i);
    return PK_GPU_OK;
}

int pk_gpu_rope_dev(const pk_gpu_rope* rope, int dtype, const void* dx, int ldx, int heads, int head_dim,
                    const int* dpos, int n, void* dy, int ldy, void* stream)
{
    const char* who = "rope";
    if (head_dim < 2 || head_dim > kMostDim)
        return rt::error(PK_GPU_ENOTSUP, "%s: head_dim = %d (2 to %d)", who, head_dim, kMostDim);
    int rc = check_rope(rope, who, dtype, heads, head_dim, n);
    if (rc) return rc;
    const long long wide = (long long)heads * head_dim;
    if (wide > 0x7fffffff || ldx < wide || ldy < wide)
        return rt::error(PK_GPU_EINVAL, "%s: rows of %lld elements, ldx = %d, ldy = %d", who, wide, ldx, ldy);
    if (n && heads && (!dx || !dy || !dpos)) return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    const int es = size_of(dtype);
    if (!aligned(dx, es) || !aligned(dy, es) || !aligned(dpos, 4))
        return rt::error(PK_GPU_EINVAL, "%s: rows or positions are not aligned to their elements", who);
    if (dx && dx == dy && ldx != ldy)
        return rt::error(PK_GPU_EINVAL, "%s: in place with ldx = %d, ldy = %d", who, ldx, ldy);
    RopeArgs a = rope_args(rope, dpos, n, dx, ldx, heads, head_dim, dy, ldy);
    a.wide = wide_rows(a, es);
    const Launch l = launch_of(&a);
    if (!launchable(l.workgroups, kThreads)) return rt::error(PK_GPU_EINVAL, "%s: %d rows exceed the grid", who, n);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!n || !heads) return PK_GPU_OK;
    const dim3 grid((uint32_t)l.workgroups), block(kThreads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == F32   ? launch(rope_rows<F32>, grid, block, l.lds, s, a)
                         : dtype == F16 ? launch(rope_rows<F16>, grid, block, l.lds, s, a)
                                        : launch(rope_rows<BF16>, grid, block, l.lds, s, a);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

int pk_gpu_rope_kv_write_dev(const pk_gpu_rope* rope, const pk_gpu_kv_cache* cache, int dtype, const void* dq, int ldq,
                             int heads, void* dqo, int ldqo, const void* dk, int ldk, const void* dv, int ldv,
                             const int* dpos, const int* dslots, int n, void* stream)
{
    const char* who = "rope kv write";
    int rc = check_cache(cache, who);
    if (!rc) rc = check_rope(rope, who, dtype, heads, cache->head_dim, n);
    if (rc) return rc;
    const int dim = cache->head_dim;
    const long long wide = (long long)cache->heads * dim, qwide = (long long)heads * dim;
    if (ldk < wide || ldv < wide)
        return rt::error(PK_GPU_EINVAL, "%s: rows of %lld elements, ldk = %d, ldv = %d", who, wide, ldk, ldv);
    if (heads && (qwide > 0x7fffffff || ldq < qwide || ldqo < qwide))
        return rt::error(PK_GPU_EINVAL, "%s: queries of %lld elements, ldq = %d, ldqo = %d", who, qwide, ldq, ldqo);
    if ((long long)n * cache->heads > 0x7fffffff)
        return rt::error(PK_GPU_EINVAL, "%s: %d tokens of %d heads exceed 2^31 rows", who, n, cache->heads);
    if (n && (!dk || !dv || !dpos || !dslots || (heads && (!dq || !dqo))))
        return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    const int es = size_of(dtype);
    if (!aligned16(dk) || !aligned16(dv) || (size_t)ldk * es % 16 || (size_t)ldv * es % 16 ||
        (heads && (!aligned16(dq) || !aligned16(dqo) || (size_t)ldq * es % 16 || (size_t)ldqo * es % 16)))
        return rt::error(PK_GPU_EINVAL, "%s: rows must be 16-byte aligned", who);
    if (!aligned(dslots, 4) || !aligned(dpos, 4))
        return rt::error(PK_GPU_EINVAL, "%s: slots or positions are not aligned to an int", who);
    if (heads && dq && dq == dqo && ldq != ldqo)
        return rt::error(PK_GPU_EINVAL, "%s: in place with ldq = %d, ldqo = %d", who, ldq, ldqo);
    RopeArgs a = rope_args(rope, dpos, n, dq, ldq, heads, dim, dqo, ldqo);
    a.wide = wide_rows(a, es);
    a.rk = static_cast<const char*>(dk);
    a.rv = static_cast<const char*>(dv);
    a.ldk = ldk;
    a.ldv = ldv;
    a.k = cache->k;
    a.v = cache->v;
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.slots = dslots;
    a.kv_heads = cache->heads;
    a.page_shift = __builtin_ctz(cache->page_size);
    a.n_slots = cache->n_pages * cache->page_size;
    const Launch l = launch_of(&a);
    if (!launchable(l.workgroups, kThreads)) return rt::error(PK_GPU_EINVAL, "%s: %d tokens exceed the grid", who, n);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!n) return PK_GPU_OK;
    const dim3 grid((uint32_t)l.workgroups);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = cache->dtype == I8     ? launch_rows<I8>(dtype, grid, l.lds, a, s)
                         : cache->dtype == E4M3 ? launch_rows<E4M3>(dtype, grid, l.lds, a, s)
                         : cache->dtype == E2M1 ? launch_rows<E2M1>(dtype, grid, l.lds, a, s)
                         : cache->dtype == F16  ? launch_rows<F16>(dtype, grid, l.lds, a, s)
                                                : launch_rows<BF16>(dtype, grid, l.lds, a, s);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

}  // extern "C"
