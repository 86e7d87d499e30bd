// pk_prompt_attention.hip - host side of the attention of several new tokens per sequence
// over a paged cache, with rules for scores and for what a token sees.
#include "pk_prompt_attention.h"

#include <climits>
#include <cmath>

namespace pkgpu {
namespace decode {
namespace {

constexpr const char* kWho = "prompt attention";

// A call's sizes, as its workspace is made for.
struct Sizes { int B, heads, max_new, max_len, window; };

// a * b of sizes, at most the largest number: bounds of a call may be far from what it holds, and
// products of four of them pass 64 bits.
long long times(long long a, long long b)
{
    long long r;
    return __builtin_mul_overflow(a, b, &r) ? LLONG_MAX : r;
}

// Tokens that a workgroup's columns see at most, from a multiple of 32 on.
long long span_of_rows(const Sizes& z)
{
    const long long seen = z.window > 0 ? (long long)z.window + z.max_new + 30 : z.max_len;
    const long long span = seen < z.max_len ? seen : z.max_len;
    return span < 1 ? 1 : span;
}

int check_sizes(const pk_gpu_kv_cache* c, const Sizes& z)
{
    const int rc = check_cache(c, kWho);
    if (rc) return rc;
    if (z.B < 0 || z.max_new < 0 || z.max_len < 0 || z.window < 0)
        return rt::error(PK_GPU_EINVAL, "%s: B = %d, max_new = %d, max_len = %d, window = %d", kWho, z.B, z.max_new,
                         z.max_len, z.window);
    if (z.max_len > 1 << 30 || z.max_new > 1 << 30)
        return rt::error(PK_GPU_EINVAL, "%s: max_new = %d or max_len = %d is above 2^30", kWho, z.max_new, z.max_len);
    if (z.heads < 1 || z.heads % c->heads)
        return rt::error(PK_GPU_EINVAL, "%s: %d query heads over %d key-value heads", kWho, z.heads, c->heads);
    return PK_GPU_OK;
}

// Calls of few rows, (new token, head) pairs of a key-value head, go 16 a workgroup over
// the tiles of the one-token attention, the others kPromptRows a workgroup.
//
// 16 rows, or fewer, read the cache once that way, and faster.  Where sequences have up to 32,
// the second 16 of them read it again, from L2; that still is less than what 128 rows lose, but
// where sequences are short and there is more than one workgroup of these for a CU. f32
// queries (3 terms) and 4 bits (a conversion, for few rows) lose more by them, and hold out up to 48
// rows while there are not two for a CU.  Measured (us, few and many; 32 heads over 8 of
// 128, queries and cache in bf16; f32 queries; bf16 over int8; over 4 bits):
//   60 x 8 of 300                  29.6 17.3    36.2 36.8    30.4 17.7    18.2 14.5
//   60 x 6 of 1000                 66.6 48.1    73.8 86.9    50.7 38.3    29.5 28.3
//   60 x 6 of up to 1000           35.2 40.2    39.1 84.1    32.3 43.8    20.5 37.9
//   100 x 8 of 2000                191  211     204  311     148  177     82.6 138
//   16 x 8 of 4000                 65.3 77.0    68.0 106     49.5 64.3    28.4 52.3
//   16 x 12 of 4000                94.0 78.8    98.3 116     69.6 72.5    42.3 58.5
//
// Of more rows still go that way the calls of at most as many such workgroups as CUs, if
// short: 16 rows start sooner than 128, and keys that need no way through LDS sooner still
// where that way is a conversion, of which 4 bits need most.  Measured (the same; 8 heads of 128
// on as many key-value heads):
//   1 x 256 of 256 tokens           8.7 10.8     9.0 18.3     9.0 13.4     8.1 11.2
//   1 x 417 of 417                 10.1 14.2    10.6 21.8    10.8 16.7     8.8 15.3
//   1 x 128 of 4000                19.4 17.9    20.3 25.2    19.3 20.8    16.2 17.9
//   1 x 1024 of 1024               23.1 24.9    24.7 32.0    22.0 27.5    14.4 25.2
//   1 x 1400 of 1400               34.6 35.1    38.8 47.4    32.3 42.7    20.9 36.8
//   1 x 500 of 3000                42.1 26.3    44.5 32.9    28.1 29.9    21.9 27.4
//   8 x 256 of 256                 27.3 11.8    31.9 18.6    27.5 13.8
// Above 512 such workgroups (16-bit caches: 256) batches and groups gain by 128 rows, and so calls of
// all kinds go that way.  Single long prompts with a head for each key-value head lose by it up to
// 1400 tokens, over 4 bits beyond, and the rule does not tell them from the others (f32 queries; bf16
// over int8; over 4 bits; few and many, the same heads, in brackets workgroups of 16 rows):
//   1 x 1100 of 1100 (552)                      31.7 41.2    26.9 36.2    17.2 31.4
//   1 x 1400 of 1400 (704)                      38.8 47.8    32.6 42.7    20.9 36.9
//   1 x 2000 of 2000 (1000)                     64.2 62.8    54.6 52.0    31.7 46.7
//   4 x 300 of 600 (608)                        30.4 28.4    26.7 21.6    17.4 19.6
//   8 x 160 of 160 (640)                        21.0 15.1    17.6 11.0    12.3  9.2
//   1 x 500 of 500, 32 heads over 8 (1000)      33.4 25.9    27.9 19.5    17.7 18.1
bool few_rows(const pk_gpu_kv_cache* c, const Sizes& z, int dtype)
{
    const long long each = (long long)z.max_new * (z.heads / c->heads), pairs = times(times((each + 15) / 16, z.B), c->heads);
    const long long heads = (long long)z.B * c->heads, span = span_of_rows(z);
    const bool narrow = dtype != F32 && (c->dtype == F16 || c->dtype == BF16), four = c->dtype == E2M1;
    const bool wide = dtype == F32 || four;
    return each <= 16 || (each <= 32 && (heads < 256 || span >= (wide ? 512 : 1536))) ||
           (each > 32 && each <= 48 && wide && heads < 512) ||
           (pairs <= (narrow ? 256 : 512) && times(pairs, span) <= (narrow ? 160 << 10 : four && dtype != F32 ? 1 << 20 : 512 << 10));
}

// Chunks of a call of many rows, where its tiles are fewer than the CUs: up to `slots`
// workgroups, as many as run at a time (the CUs, or two on each), of 512 tokens at least, or
// 256 where tiles are few.  Measured (us; 32 heads over 8 of 128 in bf16; chunks of 512
// and of 256 tokens at least):
//   64 new of 4000 tokens, 16 tiles     24.9 21.5
//   128 of 1500, 32                     30.1 23.8
//   512 of 1000, 128                    25.9 38.7
constexpr int kMostSlots = 768;     // of prompt_slots, whatever the types
long long prompt_cuts(long long pairs, long long span, int slots)
{
    if (pairs >= 256) return 1;
    const long long n = slots / pairs, most = span / (pairs <= 64 ? 256 : 512);
    const long long cut = n < most ? n : most;
    return cut < 1 ? 1 : cut > 64 ? 64 : cut;
}
// Tiles of a call's rows, whatever the sequences they are of.
long long split_pairs(const pk_gpu_kv_cache* c, long long rows, int group)
{
    return ((rows * group + kPromptRows - 1) / kPromptRows) * c->heads;
}

// Sides of a workgroup's rows.  Two make it faster by itself, one gets more work out of a full
// card: so two for launches that are one round of workgroups, or two of long ones; and for more of packed
// documents (`first`), whose longest one a launch waits for.  Where tiles are few and tokens many, more
// chunks do as much, and few tokens are not worth the join.  Measured (us, one side and two; 32 heads over 8;
// heads of 128 in bf16, of 128 over int8, of 64 in bf16):
//   16 x 16 of 200 tokens, 128 tiles  11.4 12.1
//   300 of 6000, 80                   51.2 54.5    60.7 67.5    40.5 40.3
//   700 of 9000, 176                  139  148     188  205     (2 chunks and 1)
//   500 of 500, 128                   15.9 15.9    21.1 19.2    12.6 11.8
//   800 of 3000, 200                  74.6 55.5    90.0 74.1    60.0 62.8
//   1000 of 8000, 256                 153  139     243  184     120  98.3
//   2000 of 2000, 504                 51.1 50.3    72.1 64.0    36.5 33.3
//   4 x 400 of 400, 416               19.4 25.2    23.9 29.4    13.5 14.2
//   4096 of 4096, 1024                136  168     178  214     88.2 97.2
// f32 queries over heads of 128 354 and 342 in bf16, 88.2 and 51.8 for 1000 over int8.
// With documents the limit for heads of 64 is two rounds of what runs at a time.  Documents of 300, 900
// and 3000 tokens on average, 16 heads over 4, three draws each (heads of 64 in f16, of 128 in bf16):
//   3000 tokens, 379 tiles       23.1 20.4   36.6 30.7   50.2 45.1     32.4 29.4   41.2 36.6   53.6 46.2
//   5000, 629                    28.1 25.6   41.9 36.4   69.3 60.0     34.2 42.2   53.5 58.1   83.3 82.8
//   9000, 1129                   39.4 38.4   59.3 55.1   97.3 92.0     58.1 71.4   102  117    190  204
//   16000, 2004                  56.7 60.9   112  110    180  172      86.6 116    179  205    350  384
//   32000, 4004                  94.9 107    206  204    468  470      162  231    290  359    943  1076
// and with documents of 300 and 3000, heads of 64, bf16 over int8 and f32 over bf16:
//   5000, 629                    34.4 33.0   127  112                  40.9 42.8   117  111
//   9000, 1129                   47.4 51.1   204  200                  59.5 69.4   175  173
int prompt_sides(const pk_gpu_kv_cache* c, int dtype, long long pairs, long long split, long long span, bool packed)
{
    const int dim = c->head_dim;
    if (!has_sides(c->dtype, dtype, dim, 2)) return 1;
    if (!has_sides(c->dtype, dtype, dim, 1)) return 2;
    const long long rounds = 2ll * prompt_slots(c->dtype, dtype, dim, 2);
    const long long most = dim == 64 ? (packed && rounds > 512 ? rounds : 512) : span >= 1024 ? 512 : 256;
    if (pairs > most || span < 384) return 1;
    return pairs >= 192 || prompt_cuts(split, span, prompt_slots(c->dtype, dtype, dim, 1)) == 1 ? 2 : 1;
}

// How a call is laid out: workgroups of one chunk, chunks, rows of the workspace.
struct Layout {
    bool few;
    int per_seq, sides;
    long long pairs, outs;
    Plan plan;
};
Layout layout_of(const pk_gpu_kv_cache* c, const Sizes& z, int rows, int dtype, bool packed)
{
    const int group = z.heads / c->heads;
    const long long each = (long long)z.max_new * group, span = span_of_rows(z);
    Layout l{};
    l.few = few_rows(c, z, dtype);
    if (l.few) {
        l.pairs = times(times((each + 15) / 16, z.B), c->heads);
        l.outs = times(times(z.B, z.max_new), z.heads);
        l.plan = plan_of(c->dtype, c->head_dim, l.pairs > 0 ? l.pairs : 1, span);
    } else {
        const int bm = kPromptRows;
        // tiles of every sequence, or of all rows with one that is not whole for each sequence
        const long long per = (each + bm - 1) / bm, all = (long long)rows * group / bm + z.B;
        l.per_seq = times(per, z.B) <= all ? (int)per : 0;
        l.pairs = times(l.per_seq ? per * z.B : all, c->heads);
        l.outs = (long long)rows * z.heads;
        const long long split = split_pairs(c, rows, group);
        l.sides = prompt_sides(c, dtype, l.pairs, split, span, packed);
        const long long n = prompt_cuts(split, span, prompt_slots(c->dtype, dtype, c->head_dim, l.sides));
        const int keys = prompt_keys(c->dtype, c->head_dim);
        const long long chunk = ((span + n - 1) / n + keys - 1) / keys * keys;
        // a tile of rows begins anywhere in its chunk's first tile of tokens
        l.plan = {(int)chunk, (int)(n == 1 ? 1 : (span + keys - 1 + chunk - 1) / chunk)};
        if (n == 1) l.plan.chunk = 1 << 30;
    }
    return l;
}

// Floats that any call with these sizes at most takes, few rows or many.  Few: see
// ws_floats_up_to of the one-token attention; above 256 pairs no sequence is split.
// Many: chunks fall as the rows' tiles grow, and there is one more than prompt_cuts at most.
size_t most_floats(const pk_gpu_kv_cache* c, const Sizes& z, int rows)
{
    const int group = z.heads / c->heads;
    const long long span = span_of_rows(z);
    size_t most = 0;
    for (long long b = 1; b <= z.B && b * c->heads <= 256; ++b)
        for (long long t = 1; t * b * c->heads <= 256; ++t) {
            // the most new tokens of so many tiles
            const long long n = 16 * t / group < z.max_new ? 16 * t / group : z.max_new;
            if (n < 1) continue;
            const size_t cut = cuts(c->dtype, c->head_dim, t * b * c->heads, span);
            if (cut > 1 && b * n * cut > most) most = b * n * cut;
        }
    for (long long t = 1; t * c->heads < 256; ++t) {
        const long long n = kPromptRows * t / group < rows ? kPromptRows * t / group : rows;
        const size_t cut = prompt_cuts(t * c->heads, span, kMostSlots);
        if (n >= 1 && cut > 1 && n * (cut + 1) > most) most = n * (cut + 1);
    }
    return most * z.heads * (c->head_dim + 2);
}

hipError_t launch_prompts(int cache, int t, int dim, int sides, const PagedArgs& a, uint32_t workgroups, uint32_t rows, hipStream_t s)
{
    const dim3 grid(workgroups);
    const hipError_t e = cache == F16    ? launch_prompt_f16(t, dim, sides, a, grid, s)
                         : cache == BF16 ? launch_prompt_bf16(t, dim, sides, a, grid, s)
                         : cache == I8   ? launch_prompt_i8(t, dim, sides, a, grid, s)
                         : cache == E2M1 ? launch_prompt_e2m1(t, dim, sides, a, grid, s)
                                         : launch_prompt_e4m3(t, dim, sides, a, grid, s);
    return e == hipSuccess && a.splits > 1 ? launch_joins(t, dim, true, a, rows, s) : e;
}

}  // namespace
}  // namespace decode
}  // namespace pkgpu

extern "C" {

using namespace pkgpu::decode;
namespace rt = pkgpu::rt;

size_t pk_gpu_prompt_attention_ws_floats(const pk_gpu_kv_cache* cache, int B, int rows, int heads, int max_new, int max_len,
                                         int window)
{
    const Sizes z{B, heads, max_new < rows ? max_new : rows, max_len, window < max_len ? window : 0};
    if (check_sizes(cache, z) != PK_GPU_OK) return 0;
    return most_floats(cache, z, rows);
}

int pk_gpu_prompt_attention_dev(const pk_gpu_kv_cache* cache, int dtype, const void* dq, int ldq, int heads,
                                const int* dpages, int ld_pages, const int* dlens, const int* dstarts, int B, int rows,
                                int max_new, int max_len, const pk_gpu_attention_rules* rules, void* dout, int ldo,
                                float* dlse, float* dws, size_t ws_floats, void* stream)
{
    if (!rules) return rt::error(PK_GPU_EINVAL, "%s: NULL rules", kWho);
    Sizes z{B, heads, max_new, max_len, rules->window};
    int rc = check_sizes(cache, z);
    if (rc) return rc;
    if (rows < 0) return rt::error(PK_GPU_EINVAL, "%s: rows = %d", kWho, rows);
    if (!is_float(dtype)) return rt::error(PK_GPU_EINVAL, "%s: queries of type %d (F32, F16 or BF16)", kWho, dtype);
    if ((cache->dtype == F16 && dtype != F16) || (cache->dtype == BF16 && dtype == F16))
        return rt::error(PK_GPU_ENOTSUP, "%s: queries of type %d over a cache of type %d (F16 caches take F16, "
                         "BF16 caches BF16 or F32)", kWho, dtype, cache->dtype);
    // times what turns them into powers of two they stay below the largest float; a quotient below
    // the normal ones has lost bits, which times the cap are bits of the score
    const float most = 0x1p120f, least = 0x1p-126f;
    const double of_cap = rules->cap > 0.0f ? std::fabs((double)rules->scale / rules->cap) : 0.0;
    if (!(std::fabs(rules->scale) <= most) || !(rules->cap >= 0.0f) || !(rules->cap <= most) || of_cap > most ||
        (rules->scale != 0.0f && rules->cap > 0.0f && of_cap < least))
        return rt::error(PK_GPU_EINVAL, "%s: scale = %g, cap = %g", kWho, rules->scale, rules->cap);
    const long long wide = (long long)heads * cache->head_dim;
    if (ldq < wide || ldo < wide)
        return rt::error(PK_GPU_EINVAL, "%s: rows of %lld elements, ldq = %d, ldo = %d", kWho, wide, ldq, ldo);
    if (ld_pages < 0 || ((long long)ld_pages << __builtin_ctz(cache->page_size)) < max_len)
        return rt::error(PK_GPU_EINVAL, "%s: %d pages a sequence do not hold max_len = %d tokens", kWho, ld_pages, max_len);
    const bool some = B && rows && max_new;
    if (some && (!dq || !dout || !dlens || (max_len && !dpages)))
        return rt::error(PK_GPU_EINVAL, "%s: NULL operand", kWho);
    const size_t es = size_of(dtype);
    if (!aligned16(dq) || !aligned16(dout) || (size_t)ldq * es % 16 || (size_t)ldo * es % 16)
        return rt::error(PK_GPU_EINVAL, "%s: query and output rows must be 16-byte aligned", kWho);
    if (!aligned(dpages, 4) || !aligned(dlens, 4) || !aligned(dlse, 4) || !aligned(dstarts, 4) || !aligned(rules->slopes, 4) ||
        !aligned(rules->first, 4) || !aligned(rules->until, 4))
        return rt::error(PK_GPU_EINVAL, "%s: pages, lengths, starts, lse or a rule's array are not aligned to their elements",
                         kWho);
    // no row has more, and a window that wide hides nothing
    if (z.max_new > rows) z.max_new = rows;
    if (!dstarts && z.max_new > 1) z.max_new = 1;
    if (z.window >= max_len) z.window = 0;
    const Layout l = layout_of(cache, z, rows, dtype, rules->first != nullptr);
    const Plan& p = l.plan;
    if (!launchable(times(l.pairs, p.splits), 512) || l.outs > 0x7fffffff || (p.splits > 1 && !launchable(l.outs, 256)))
        return rt::error(PK_GPU_EINVAL, "%s: %d sequences of %d new tokens and %d heads exceed the grid", kWho, B, z.max_new,
                         heads);
    const size_t need = p.splits <= 1 ? 0 : (size_t)l.outs * p.splits * (cache->head_dim + 2);
    if (need && (!dws || ws_floats < need || !aligned16(dws)))
        return rt::error(PK_GPU_EINVAL, "%s: needs a 16-byte aligned workspace of %zu floats "
                         "(pk_gpu_prompt_attention_ws_floats)", kWho, need);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!some) return PK_GPU_OK;
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
    a.ml = need ? dws + (size_t)l.outs * p.splits * cache->head_dim : nullptr;
    a.scale2 = rules->scale * 1.4426950408889634f;
    a.B = B;
    a.max_len = max_len;
    a.window = z.window;
    a.kv_heads = cache->heads;
    a.group = heads / cache->heads;
    a.head_tiles = (int)(l.pairs / (l.few ? (long long)B * cache->heads : cache->heads));
    a.n_pages = cache->n_pages;
    a.page_shift = __builtin_ctz(cache->page_size);
    a.chunk = p.chunk;
    a.splits = p.splits;
    a.rules.cap2 = rules->cap * 1.4426950408889634f;
    a.rules.cap_in = rules->cap > 0.0f ? rules->scale / rules->cap : 0.0f;
    a.rules.cap_exp = rules->cap > 0.0f ? rules->scale / rules->cap * 2.8853900817779268f : 0.0f;     // 2 log2(e)
    a.rules.slopes = rules->slopes;
    a.rules.first = rules->first;
    a.rules.until = rules->until;
    a.rules.starts = dstarts;
    a.rules.rows = rows;
    a.rules.max_new = z.max_new;
    a.rules.by_row = !l.few;
    a.rules.per_seq = l.per_seq;
    // Where there are more workgroups of whole sequences than CUs, the longest sequences go
    // first (see the one-token call) if they are long for what counting them costs: 33 of 3000
    // tokens, 8 new ones, 32 heads over 8 of 128 in bf16, ragged 50 us, 63 in order, all
    // equal 119 against 115; 60 of 1000, 5 new ones, 37 against 34 and 74 against 67.
    a.longest_first = l.few && p.splits == 1 && l.pairs > 256 && B > 1 && B <= kSortedMax && max_len / 32 >= B && z.window == 0;
    const hipError_t e = l.few ? launch_attention(cache->dtype, dtype, cache->head_dim, true, a, (uint32_t)(l.pairs * p.splits),
                                                  (uint32_t)l.outs, static_cast<hipStream_t>(stream))
                               : launch_prompts(cache->dtype, dtype, cache->head_dim, l.sides, a, (uint32_t)(l.pairs * p.splits),
                                                (uint32_t)l.outs, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, kWho);
}

}  // extern "C"
