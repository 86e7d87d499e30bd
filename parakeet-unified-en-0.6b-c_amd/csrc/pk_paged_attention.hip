// pk_paged_attention.hip - host side of the attention over a paged cache, and
// the kernel that joins a sequence's chunks.
#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {
namespace {

constexpr int kMaxSplits = 256;     // the join's threads: one a chunk

struct JoinArgs {
    const float *part, *ml;
    const int* lens;
    char* out;
    size_t ldo;
    float* lse;
    int heads, splits, chunk, max_len, window;
};

// One workgroup joins the chunks of one head: out = sum_c 2^(m_c - m) o_c /
// sum_c 2^(m_c - m) l_c.  DIM / 4 lanes cover the head, the other lanes take
// every PARTS-th chunk; sums run in a fixed order.  All that it reads first,
// the length, the chunks' (m, l) and EARLY chunks' outputs of a thread, is asked
// for at once: the workspace holds them whether the sequence has them or not.
template <int T, int DIM>
__global__ void __launch_bounds__(256) paged_join(JoinArgs a)
{
    constexpr int LANES = DIM / 4, PARTS = 256 / LANES, EARLY = 4;
    __shared__ float red[2][4];
    __shared__ float wgt[kMaxSplits];
    __shared__ f32x4 sum[PARTS][LANES];
    const int b = blockIdx.x / (uint32_t)a.heads, head = blockIdx.x % (uint32_t)a.heads;
    const size_t row = (size_t)b * a.heads + head;
    const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
    const int part = i / LANES, d4 = i % LANES;
    const int len = a.lens[b];
    const float* ml = a.ml + row * a.splits * 2;
    float m = -FLT_MAX, l = 0.0f;
    if (i < a.splits) { m = ml[2 * i]; l = ml[2 * i + 1]; }
    const float* src = a.part + row * a.splits * DIM + 4 * d4;
    f32x4 v[EARLY];
#pragma unroll
    for (int e = 0; e < EARLY; ++e)
        if (part + e * PARTS < a.splits) v[e] = *reinterpret_cast<const f32x4*>(src + (size_t)(part + e * PARTS) * DIM);
    const int chunks = span_of(len, a.max_len, a.window, a.chunk).chunks;
    if (chunks <= 1) return;                        // written by the first launch
    if (i >= chunks) { m = -FLT_MAX; l = 0.0f; }
    float mx = m;
#pragma unroll
    for (int d = 32; d; d >>= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
    if (lane == 0) red[0][wave] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float w = i < chunks ? __builtin_amdgcn_exp2f(m - mx) : 0.0f;
    wgt[i] = w;
    float lt = __fmul_rn(l, w);
#pragma unroll
    for (int d = 32; d; d >>= 1) lt = __fadd_rn(lt, __shfl_xor(lt, d));
    if (lane == 0) red[1][wave] = lt;
    __syncthreads();
    lt = __fadd_rn(__fadd_rn(red[1][0], red[1][1]), __fadd_rn(red[1][2], red[1][3]));
    f32x4 o = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < EARLY; ++e) {
        const int c = part + e * PARTS;
        if (c < chunks)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = __fmaf_rn(v[e][r], wgt[c], o[r]);
    }
#pragma unroll 4
    for (int c = part + EARLY * PARTS; c < chunks; c += PARTS) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(src + (size_t)c * DIM);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = __fmaf_rn(x[r], wgt[c], o[r]);
    }
    sum[part][d4] = o;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int p = 1; p < PARTS; ++p)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = __fadd_rn(o[r], sum[p][d4][r]);
    const float inv = lt == 0.0f ? 0.0f : __fdiv_rn(1.0f, lt);
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = lt == 0.0f ? 0.0f : __fmul_rn(o[r], inv);
    char* p = a.out + (size_t)b * a.ldo + ((size_t)head * DIM + 4 * d4) * size_of(T);
    if constexpr (T == F32) *reinterpret_cast<f32x4*>(p) = o;
    else
        *reinterpret_cast<u32x2*>(p) = T == F16 ? (u32x2){pack_f16(o[0], o[1]), pack_f16(o[2], o[3])}
                                                : (u32x2){pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
    if (d4 == 0 && a.lse)
        a.lse[row] = lt == 0.0f ? -__builtin_inff()
                                : __fmul_rn(__fadd_rn(mx, __builtin_amdgcn_logf(lt)), 0.69314718055994531f);
}

template <int T>
hipError_t launch_join(int dim, const JoinArgs& a, uint32_t rows, hipStream_t s)
{
    return dim == 64    ? launch(paged_join<T, 64>, dim3(rows), dim3(256), 0, s, a)
           : dim == 128 ? launch(paged_join<T, 128>, dim3(rows), dim3(256), 0, s, a)
                        : launch(paged_join<T, 256>, dim3(rows), dim3(256), 0, s, a);
}

// 16 query heads of a key-value head a workgroup.
int head_tiles(int group) { return (group + 15) / 16; }

struct Plan { int chunk, splits; };

// Tokens that the longest sequence's chunks cover: a window's begin up to 31 before it.
long long span_at_most(int max_len, int window)
{
    const long long seen = window > 0 ? (long long)window + 31 : max_len;
    const long long span = seen < max_len ? seen : max_len;
    return span < 1 ? 1 : span;
}

constexpr int kRound = 256;         // 8 waves' tiles

// Chunks that a sequence is cut into, before they are made whole rounds.  Up to 3
// rounds one workgroup takes the whole: a round costs about 2 us, the second
// launch that joins chunks 4 to 5 us.  Longer ones are cut until there is a
// workgroup for each of the 256 CUs, and up to two where chunks keep 384 KB of
// cache.  Measured (us; one chunk, 256, 512 workgroups):
//   1 sequence of 100003 tokens, 8 heads of 128 in bf16     1059, 76, 78
//   4 ragged ones up to 30000, 2 heads of 256 in bf16        615, 36, 29
//   8 ragged ones up to 4000, 8 heads of 128 in int8           34, 16, 19.5
//   32 ragged ones up to 2000, the same (256 unsplit)           22, 22, 27
//   160 windows of 1024 over a head of 256 (160 unsplit)       21, 21, 30
long long cuts(const pk_gpu_kv_cache* c, long long pairs, long long span)
{
    const long long rounds = (span + kRound - 1) / kRound;
    if (rounds <= 3) return 1;
    const long long fill = 256 / pairs, two = 512 / pairs, large = span * 2 * c->head_dim * size_of(c->dtype) / (384 << 10);
    long long n = two < large ? two : large;
    if (n < fill) n = fill;
    if (n > rounds) n = rounds;
    if (n > kMaxSplits) n = kMaxSplits;
    return n < 1 ? 1 : n;
}

long long pairs_of(const pk_gpu_kv_cache* c, int B, int heads)
{
    return (long long)B * c->heads * head_tiles(heads / c->heads);
}

Plan plan(const pk_gpu_kv_cache* c, int B, int heads, int max_len, int window)
{
    const long long span = span_at_most(max_len, window), rounds = (span + kRound - 1) / kRound;
    const long long n = cuts(c, pairs_of(c, B > 0 ? B : 1, heads), span);
    const long long chunk = (rounds + n - 1) / n * kRound;
    return {(int)chunk, (int)((span + chunk - 1) / chunk)};
}

int check_attention(const pk_gpu_kv_cache* c, int B, int heads, int max_len, int window)
{
    const char* who = "paged attention";
    const int rc = check_cache(c, who);
    if (rc) return rc;
    if (B < 0 || max_len < 0 || window < 0)
        return rt::error(PK_GPU_EINVAL, "%s: B = %d, max_len = %d, window = %d", who, B, max_len, window);
    if (max_len > 1 << 30)      // token indices of a round ahead stay below 2^31
        return rt::error(PK_GPU_EINVAL, "%s: max_len = %d is above 2^30", who, max_len);
    if (heads < 1 || heads % c->heads)
        return rt::error(PK_GPU_EINVAL, "%s: %d query heads over %d key-value heads", who, heads, c->heads);
    const Plan p = plan(c, B, heads, max_len, window);
    // 8 waves a workgroup at most; the join has 256 threads a head, of up to 16 * 256 heads
    if (!launchable(pairs_of(c, B, heads) * p.splits, 512) || (long long)B * heads > 0x7fffffff)
        return rt::error(PK_GPU_EINVAL, "%s: %d sequences of %d heads exceed the grid", who, B, heads);
    return PK_GPU_OK;
}

size_t ws_floats_of(const pk_gpu_kv_cache* c, int B, int heads, const Plan& p)
{
    return p.splits <= 1 ? 0 : (size_t)B * heads * p.splits * (c->head_dim + 2);
}

// What any call with up to B sequences, up to max_len tokens and a window up to this
// one takes: cuts() does not fall as the span grows, and chunks are never more.
// Above 256 pairs there are none.
size_t ws_floats_up_to(const pk_gpu_kv_cache* c, int B, int heads, int max_len, int window)
{
    const long long span = span_at_most(max_len, window);
    size_t most = 0;
    for (int b = 1; b <= B && pairs_of(c, b, heads) <= 256; ++b) {
        const size_t n = cuts(c, pairs_of(c, b, heads), span);
        if (n > 1 && b * n > most) most = b * n;
    }
    return most * heads * (c->head_dim + 2);
}

}  // namespace
}  // namespace decode
}  // namespace pkgpu

extern "C" {

using namespace pkgpu::decode;

size_t pk_gpu_paged_attention_ws_floats(const pk_gpu_kv_cache* cache, int B, int heads, int max_len, int window)
{
    if (check_attention(cache, B, heads, max_len, window) != PK_GPU_OK || B == 0) return 0;
    return ws_floats_up_to(cache, B, heads, max_len, window);
}

int pk_gpu_paged_attention_dev(const pk_gpu_kv_cache* cache, int dtype, const void* dq, int ldq, int heads,
                               const int* dpages, int ld_pages, const int* dlens, int B, int max_len,
                               float scale, int window, void* dout, int ldo, float* dlse, float* dws,
                               size_t ws_floats, void* stream)
{
    namespace rt = pkgpu::rt;
    const char* who = "paged attention";
    int rc = check_attention(cache, B, heads, max_len, window);
    if (rc) return rc;
    if (!is_float(dtype))
        return rt::error(PK_GPU_EINVAL, "%s: queries of type %d (F32, F16 or BF16)", who, dtype);
    if ((cache->dtype == F16 && dtype != F16) || (cache->dtype == BF16 && dtype == F16))
        return rt::error(PK_GPU_ENOTSUP, "%s: queries of type %d over a cache of type %d (F16 caches take F16, "
                         "BF16 caches BF16 or F32)", who, dtype, cache->dtype);
    const long long wide = (long long)heads * cache->head_dim;
    if (ldq < wide || ldo < wide)
        return rt::error(PK_GPU_EINVAL, "%s: rows of %lld elements, ldq = %d, ldo = %d", who, wide, ldq, ldo);
    if (ld_pages < 0 || ((long long)ld_pages << __builtin_ctz(cache->page_size)) < max_len)
        return rt::error(PK_GPU_EINVAL, "%s: %d pages a sequence do not hold max_len = %d tokens", who, ld_pages,
                         max_len);
    if (B && (!dq || !dout || !dlens || (max_len && !dpages)))
        return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    const size_t es = size_of(dtype);
    if (!aligned16(dq) || !aligned16(dout) || (size_t)ldq * es % 16 || (size_t)ldo * es % 16)
        return rt::error(PK_GPU_EINVAL, "%s: query and output rows must be 16-byte aligned", who);
    if (!aligned(dpages, 4) || !aligned(dlens, 4) || !aligned(dlse, 4))
        return rt::error(PK_GPU_EINVAL, "%s: pages, lengths or lse are not aligned to their elements", who);
    const long long pairs = pairs_of(cache, B, heads);
    const Plan p = plan(cache, B, heads, max_len, window);
    const size_t need = ws_floats_of(cache, B, heads, p);
    if (need && (!dws || ws_floats < need || !aligned16(dws)))
        return rt::error(PK_GPU_EINVAL, "%s: needs a 16-byte aligned workspace of %zu floats "
                         "(pk_gpu_paged_attention_ws_floats)", who, need);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!B) return PK_GPU_OK;
    PagedArgs a{};
    a.k = static_cast<const char*>(cache->k);
    a.v = static_cast<const char*>(cache->v);
    a.k_scale = cache->k_scale;
    a.v_scale = cache->v_scale;
    a.q = static_cast<const char*>(dq);
    a.ldq = (size_t)ldq * es;
    a.pages = dpages;
    a.ld_pages = ld_pages;
    a.lens = dlens;
    a.out = static_cast<char*>(dout);
    a.ldo = (size_t)ldo * es;
    a.lse = dlse;
    a.part = dws;
    a.ml = dws ? dws + (size_t)B * heads * p.splits * cache->head_dim : nullptr;
    a.scale2 = scale * 1.4426950408889634f;
    a.B = B;
    a.max_len = max_len;
    a.window = window;
    a.kv_heads = cache->heads;
    a.group = heads / cache->heads;
    a.head_tiles = head_tiles(a.group);
    a.n_pages = cache->n_pages;
    a.page_shift = __builtin_ctz(cache->page_size);
    a.chunk = p.chunk;
    a.splits = p.splits;
    // Where there are more workgroups than the 512 that run at a time, the longest
    // sequences go first: 96 ragged sequences of up to 6000 tokens and 8 heads 122
    // us against 139 in order, the same number of equal ones 114 against 111; of
    // short sequences the counting costs more (256 of up to 1000: 87 against 67).
    a.longest_first = B > 1 && B <= kSortedMax && pairs * p.splits > 512 && max_len / 16 >= B &&
                      (window == 0 || window / 16 >= B);
    const dim3 grid((uint32_t)(pairs * p.splits));
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int dim = cache->head_dim;
    hipError_t e = cache->dtype == F16    ? launch_paged_f16(dtype, dim, a, grid, s)
                   : cache->dtype == BF16 ? launch_paged_bf16(dtype, dim, a, grid, s)
                   : cache->dtype == I8   ? launch_paged_i8(dtype, dim, a, grid, s)
                                          : launch_paged_e4m3(dtype, dim, a, grid, s);
    if (e == hipSuccess && p.splits > 1) {
        JoinArgs j{};
        j.part = a.part;
        j.ml = a.ml;
        j.lens = dlens;
        j.out = a.out;
        j.ldo = a.ldo;
        j.lse = dlse;
        j.heads = heads;
        j.splits = p.splits;
        j.chunk = p.chunk;
        j.max_len = max_len;
        j.window = window;
        const uint32_t rows = (uint32_t)((long long)B * heads);
        e = dtype == F32   ? launch_join<F32>(dim, j, rows, s)
            : dtype == F16 ? launch_join<F16>(dim, j, rows, s)
                           : launch_join<BF16>(dim, j, rows, s);
    }
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

}  // extern "C"
