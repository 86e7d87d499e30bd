// pk_kv_cache.hip - writing the key-value cache of a decoder and reading it
// back (pk_gpu_kv_write_dev, pk_gpu_kv_read_dev).
//
// A cache row is one token's key (or value) of one head: head_dim elements at
// ((page * heads + head) * page_size + offset) * head_dim.  8-bit caches hold
// codes with one fp32 scale a row (pk_decode.h gives the formula); the row's
// largest magnitude is exact whatever the order it is found in, so codes and
// scales do not depend on the launch.
//
// Both kernels move 8 elements of K and of V a thread, head_dim / 8 lanes a
// row, so that a wave's loads and stores are whole rows; the maximum is
// reduced inside that lane group and nothing goes through LDS.
#include "pk_decode.h"

namespace pkgpu {
namespace decode {
namespace {

struct RowsArgs {
    void *k, *v;                    // the cache
    float *k_scale, *v_scale;
    char *rk, *rv;                  // the rows, ldk and ldv elements apart
    size_t ldk, ldv;
    const int* slots;
    uint32_t rows;                  // n * heads
    uint32_t heads;
    int page_shift, page_size, n_slots;
};

// Threads of a workgroup: a launch of many rows takes 1024 (20011 tokens of 8
// heads of 128 from int8 to bf16: 25.6 us against 27.5 of 256), one of few 256, on
// more CUs.
constexpr int kMostThreads = 1024;

// Index of the cache row that row r = token * heads + head names, or -1.
__device__ inline long long cache_row(const RowsArgs& a, uint32_t token, uint32_t head)
{
    const int slot = a.slots[token];
    if (slot < 0 || slot >= a.n_slots) return -1;
    const uint32_t page = (uint32_t)slot >> a.page_shift, off = (uint32_t)slot & (a.page_size - 1);
    return ((long long)page * a.heads + head) * a.page_size + off;
}

__device__ inline uint32_t max_bits(const float* x)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        m = b > m ? b : m;
    }
    return m;
}

// One row's 8 elements of this lane into the cache at element `at`.
template <int CACHE, int DIM>
__device__ inline void write_part(void* cache, float* scales, long long row, int part, float* x)
{
    if constexpr (CACHE == I8 || CACHE == E4M3) {
        const RowCode c = row_code(max_over<DIM / 8>(max_bits(x)), top_of(CACHE));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = coded(x[i], c);
        if (row >= 0 && part == 0) scales[row] = c.scale;
    }
    if (row >= 0)
        store8<CACHE>(static_cast<char*>(cache) + ((size_t)row * DIM + 8 * part) * size_of(CACHE), x);
}

template <int CACHE, int ROWS, int DIM>
__global__ void __launch_bounds__(kMostThreads) kv_write(RowsArgs a)
{
    constexpr int LANES = DIM / 8;
    const uint32_t r = blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES;
    const int part = threadIdx.x % LANES;
    if (r >= a.rows) return;                       // whole lane groups leave together
    const uint32_t token = r / a.heads, head = r - token * a.heads;
    const long long row = cache_row(a, token, head);
    const size_t at = (size_t)head * DIM + 8 * part;
    float k[8], v[8];
    // the rows' loads do not wait for the slot: padding rows are read too
    load8<ROWS>(a.rk + (token * a.ldk + at) * size_of(ROWS), k);
    load8<ROWS>(a.rv + (token * a.ldv + at) * size_of(ROWS), v);
    write_part<CACHE, DIM>(a.k, a.k_scale, row, part, k);
    write_part<CACHE, DIM>(a.v, a.v_scale, row, part, v);
}

template <int CACHE, int ROWS, int DIM>
__global__ void __launch_bounds__(kMostThreads) kv_read(RowsArgs a)
{
    constexpr int LANES = DIM / 8;
    const uint32_t r = blockIdx.x * (blockDim.x / LANES) + threadIdx.x / LANES;
    const int part = threadIdx.x % LANES;
    if (r >= a.rows) return;
    const uint32_t token = r / a.heads, head = r - token * a.heads;
    const long long row = cache_row(a, token, head);
    if (row < 0) return;
    const size_t from = ((size_t)row * DIM + 8 * part) * size_of(CACHE);
    float k[8], v[8];
    load8<CACHE>(static_cast<const char*>(a.k) + from, k);
    load8<CACHE>(static_cast<const char*>(a.v) + from, v);
    if constexpr (CACHE == I8 || CACHE == E4M3) {
        const float sk = a.k_scale[row], sv = a.v_scale[row];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            k[i] = __fmul_rn(k[i], sk);
            v[i] = __fmul_rn(v[i], sv);
        }
    }
    const size_t at = (size_t)head * DIM + 8 * part;
    store8<ROWS>(a.rk + (token * a.ldk + at) * size_of(ROWS), k);
    store8<ROWS>(a.rv + (token * a.ldv + at) * size_of(ROWS), v);
}

struct Launch { int threads; long long workgroups; };
Launch launch_of(long long rows, int dim)
{
    const int lanes = dim / 8, threads = rows / 1024 * lanes >= 256 ? kMostThreads : 256;
    const int per = threads / lanes;
    return {threads, (rows + per - 1) / per};
}

template <int CACHE, int ROWS>
hipError_t launch_dim(bool write, int dim, const RowsArgs& a, hipStream_t s)
{
    const Launch l = launch_of(a.rows, dim);
    const dim3 grid((uint32_t)l.workgroups), block(l.threads);
#define PK_ROWS_DIM(D) launch(write ? kv_write<CACHE, ROWS, D> : kv_read<CACHE, ROWS, D>, grid, block, 0, s, a)
    return dim == 64 ? PK_ROWS_DIM(64) : dim == 128 ? PK_ROWS_DIM(128) : PK_ROWS_DIM(256);
#undef PK_ROWS_DIM
}

template <int CACHE>
hipError_t launch_rows(bool write, int rows_type, int dim, const RowsArgs& a, hipStream_t s)
{
    return rows_type == F32 ? launch_dim<CACHE, F32>(write, dim, a, s)
         : rows_type == F16 ? launch_dim<CACHE, F16>(write, dim, a, s)
                            : launch_dim<CACHE, BF16>(write, dim, a, s);
}

int kv_call(bool write, const pk_gpu_kv_cache* c, int dtype, const void* dk, int ldk, const void* dv,
            int ldv, const int* dslots, int n, void* stream)
{
    const char* who = write ? "kv write" : "kv read";
    int rc = check_cache(c, who);
    if (rc) return rc;
    if (!is_float(dtype)) return rt::error(PK_GPU_EINVAL, "%s: rows of type %d (F32, F16 or BF16)", who, dtype);
    if (n < 0) return rt::error(PK_GPU_EINVAL, "%s: n = %d", who, n);
    const long long wide = (long long)c->heads * c->head_dim;
    if (ldk < wide || ldv < wide)
        return rt::error(PK_GPU_EINVAL, "%s: rows of %lld elements, ldk = %d, ldv = %d", who, wide, ldk, ldv);
    if ((long long)n * c->heads > 0x7fffffff)
        return rt::error(PK_GPU_EINVAL, "%s: %d tokens of %d heads exceed 2^31 rows", who, n, c->heads);
    const Launch l = launch_of((long long)n * c->heads, c->head_dim);
    if (!launchable(l.workgroups, l.threads))
        return rt::error(PK_GPU_EINVAL, "%s: %d tokens of %d heads of %d exceed the grid", who, n, c->heads, c->head_dim);
    if (n && (!dk || !dv || !dslots)) return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    const int es = size_of(dtype);
    if (!aligned16(dk) || !aligned16(dv) || (size_t)ldk * es % 16 || (size_t)ldv * es % 16)
        return rt::error(PK_GPU_EINVAL, "%s: rows must be 16-byte aligned", who);
    if (!aligned(dslots, 4)) return rt::error(PK_GPU_EINVAL, "%s: slots are not aligned to an int", who);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!n) return PK_GPU_OK;
    RowsArgs a{};
    a.k = c->k; a.v = c->v;
    a.k_scale = c->k_scale; a.v_scale = c->v_scale;
    a.rk = static_cast<char*>(const_cast<void*>(dk));
    a.rv = static_cast<char*>(const_cast<void*>(dv));
    a.ldk = ldk; a.ldv = ldv;
    a.slots = dslots;
    a.rows = (uint32_t)n * c->heads;
    a.heads = c->heads;
    a.page_size = c->page_size;
    a.page_shift = __builtin_ctz(c->page_size);
    a.n_slots = c->n_pages * c->page_size;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = c->dtype == I8   ? launch_rows<I8>(write, dtype, c->head_dim, a, s)
                       : c->dtype == E4M3 ? launch_rows<E4M3>(write, dtype, c->head_dim, a, s)
                       : c->dtype == F16  ? launch_rows<F16>(write, dtype, c->head_dim, a, s)
                                          : launch_rows<BF16>(write, dtype, c->head_dim, a, s);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

}  // namespace

int check_cache(const pk_gpu_kv_cache* c, const char* who)
{
    if (!c) return rt::error(PK_GPU_EINVAL, "%s: NULL cache", who);
    if (c->dtype != F16 && c->dtype != BF16 && c->dtype != I8 && c->dtype != E4M3)
        return rt::error(PK_GPU_EINVAL, "%s: a cache of type %d (F16, BF16, I8 or E4M3)", who, c->dtype);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return rt::error(PK_GPU_ENOTSUP, "%s: head_dim = %d (64, 128 or 256)", who, c->head_dim);
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1)))
        return rt::error(PK_GPU_ENOTSUP, "%s: page_size = %d (a power of two from 16 on)", who, c->page_size);
    if (c->n_pages < 1 || c->heads < 1)
        return rt::error(PK_GPU_EINVAL, "%s: %d pages of %d heads", who, c->n_pages, c->heads);
    if ((long long)c->n_pages * c->page_size > 0x7fffffff)
        return rt::error(PK_GPU_EINVAL, "%s: %d pages of %d exceed 2^31 slots", who, c->n_pages, c->page_size);
    if ((long long)c->heads * c->head_dim > 0x7fffffff)
        return rt::error(PK_GPU_EINVAL, "%s: %d heads of %d exceed 2^31 elements", who, c->heads, c->head_dim);
    const bool coded = c->dtype == I8 || c->dtype == E4M3;
    if (!c->k || !c->v || (coded && (!c->k_scale || !c->v_scale)))
        return rt::error(PK_GPU_EINVAL, "%s: the cache's k, v or their scales are NULL", who);
    if (!aligned16(c->k) || !aligned16(c->v) || (coded && (!aligned16(c->k_scale) || !aligned16(c->v_scale))))
        return rt::error(PK_GPU_EINVAL, "%s: the cache's arrays must be 16-byte aligned", who);
    return PK_GPU_OK;
}

}  // namespace decode
}  // namespace pkgpu

extern "C" {

int pk_gpu_kv_write_dev(const pk_gpu_kv_cache* cache, int dtype, const void* dk, int ldk,
                        const void* dv, int ldv, const int* dslots, int n, void* stream)
{
    return pkgpu::decode::kv_call(true, cache, dtype, dk, ldk, dv, ldv, dslots, n, stream);
}

int pk_gpu_kv_read_dev(const pk_gpu_kv_cache* cache, int dtype, const int* dslots, int n, void* dk,
                       int ldk, void* dv, int ldv, void* stream)
{
    return pkgpu::decode::kv_call(false, cache, dtype, dk, ldk, dv, ldv, dslots, n, stream);
}

}  // extern "C"
