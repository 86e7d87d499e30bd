// pk_rms_norm.hip - root-mean-square norm with the residual's addition and an
// output in 8 bits with row scales (pk_gpu_rms_norm_dev).
//
//   h = T(x + res)                         stored if asked for
//   r = fl32(1 / sqrt(mean(h^2) + eps))    squares, mean, root in fp64
//   y = fl(fl(h r) gamma)                  fp32
//   out = y rounded to its type, or codes and a scale (pk_decode.h)
//
// The norm is of the stored sum, so that what a later layer reads and what was
// normalised here are the same numbers.  h^2 is exact in fp64 and a thread
// adds up to D / 1024 + 32 of them: the sum's error is below 2^-43 up to D = 2^20 (2^-32
// for the longest rows), so r does not depend on the order of the additions but
// once in 2^18 rows or so: codes are reproducible across launch shapes.  The fp64 work is two instructions an element.
//
// A row stays in registers between its statistics and its output: TPR threads
// (a wave, or a workgroup of 4 or 16) hold CH pieces of 8 consecutive elements
// each.  Pieces are read and written whole whatever their alignment (rows of odd
// D begin anywhere): 8192 rows of 2047 in bf16 31 us, 46 by single elements.
// Rows above 16384 are read again for each pass.  Sums and
// maxima over a wave go by mirrors of lane groups in the vector unit (33 rows of
// 1024: 3.1 us; 4.7 through LDS).  Bound by the rows' bytes, for few rows by the
// launch and one load's latency.
#include "pk_decode.h"

namespace pkgpu {
namespace decode {
namespace {

struct NormArgs {
    const char *x, *res;
    char* sum;
    const float* gamma;
    char* out;
    float* scales;
    size_t ldx, ldr, lds, ldo;      // bytes
    double eps;
    int rows, D;
};

constexpr int kNormThreads = 256;

__device__ inline float norm_factor(double sum, int D, double eps)
{
    return (float)(1.0 / __dsqrt_rn(sum / (double)D + eps));
}

// 8 elements of a row, from element i on, as they lie in memory; at the `edge`,
// a constant of the unrolled loops, the row's last piece may have n < 8 of them.
// (Loads on a condition make every wait longer, so there is a kernel without
// them for D % 8 == 0.)  Rows are aligned to their elements only.
template <int T>
struct Piece {
    static constexpr int WORDS = size_of(T) / 2;
    u32x4 w[WORDS];
    __device__ inline __attribute__((always_inline)) void load(const char* p, int i, int n, bool edge)
    {
        p += (size_t)i * size_of(T);
        if (!edge || n >= 8) {
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = reinterpret_cast<const u32x4_any*>(p)[k];
        } else {
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                e[j] = j >= n ? 0u : T == F32 ? reinterpret_cast<const uint32_t*>(p)[j]
                                              : reinterpret_cast<const uint16_t*>(p)[j];
#pragma unroll
            for (int j = 0; j < 4 * WORDS; ++j) w[j / 4][j % 4] = T == F32 ? e[j] : e[2 * (j % 4)] | e[2 * (j % 4) + 1] << 16;
        }
    }
    __device__ void values(float* x) const { load8<T>(w, x); }
};

template <int T>
__device__ inline __attribute__((always_inline)) void store_piece(char* p, int i, int n, const float* x, bool edge)
{
    p += (size_t)i * size_of(T);
    if (!edge || n >= 8) {
        u32x4 w[T == F32 ? 2 : 1];
        store8<T>(w, x);
        if constexpr (T == I8) {
            *reinterpret_cast<u32x2_any*>(p) = (u32x2){w[0][0], w[0][1]};
        } else {
#pragma unroll
            for (int k = 0; k < (T == F32 ? 2 : 1); ++k) reinterpret_cast<u32x4_any*>(p)[k] = w[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (j < n) {
                if constexpr (T == I8) reinterpret_cast<signed char*>(p)[j] = (signed char)(int)__builtin_rintf(x[j]);
                else store1<T>(p, j, x[j]);
            }
    }
}

// one element of h, for the rows that are read again
template <int T>
__device__ inline float sum_at(const NormArgs& a, size_t row, size_t i)
{
    float h = load1<T>(a.x + row * a.ldx, i);
    if (a.res) h = as_type<T>(__fadd_rn(h, load1<T>(a.res + row * a.ldr, i)));
    return h;
}

constexpr int norm_threads(int tpr) { return tpr > kNormThreads ? tpr : kNormThreads; }

template <int T, int OUT, int TPR, int CH, bool EDGE>
__global__ void __launch_bounds__(norm_threads(TPR)) rms_norm(NormArgs a)
{
    constexpr int RPB = norm_threads(TPR) / TPR;         // rows a workgroup has at a time
    constexpr int WAVES = norm_threads(TPR) / 64;
    __shared__ double red_sum[2][WAVES];
    __shared__ uint32_t red_max[2][WAVES];
    constexpr int W = 8;
    // only rows of more than CH / 2 * TPR pieces come here (launch_norm), so the first
    // CH / 2 of a thread's are whole ones
    const auto at_edge = [](int c) { return EDGE && (CH == 1 || c >= CH / 2); };
    const int t = threadIdx.x % TPR, wave = threadIdx.x / 64;
    // the next row's pieces are on their way while this one is summed
    Piece<T> nx[CH], nr[CH];
    auto ask = [&](long long row) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = (c * TPR + t) * W;
            if (row < a.rows && i < a.D) {
                nx[c].load(a.x + row * a.ldx, i, a.D - i, at_edge(c));
                if (a.res) nr[c].load(a.res + row * a.ldr, i, a.D - i, at_edge(c));
            }
        }
    };
    const long long stride = (long long)gridDim.x * RPB;
    ask((long long)blockIdx.x * RPB + threadIdx.x / TPR);
    float gm[CH][W];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int i = (c * TPR + t) * W;
#pragma unroll
        for (int j = 0; j < W; ++j) gm[c][j] = 1.0f;
        if (a.gamma && i < a.D) {
            Piece<F32> g;
            g.load(reinterpret_cast<const char*>(a.gamma), i, a.D - i, at_edge(c));
            g.values(gm[c]);
        }
    }
    int turn = 0;
    for (long long r0 = (long long)blockIdx.x * RPB; r0 < a.rows; r0 += stride, turn ^= 1) {
        const long long row = r0 + threadIdx.x / TPR;
        const bool live = row < a.rows;
        float h[CH][W];
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = (c * TPR + t) * W;
#pragma unroll
            for (int j = 0; j < W; ++j) h[c][j] = 0.0f;
            if (live && i < a.D) {
                nx[c].values(h[c]);
                if (a.res) {
                    float v[W];
                    nr[c].values(v);
#pragma unroll
                    for (int j = 0; j < W; ++j) h[c][j] = as_type<T>(__fadd_rn(h[c][j], v[j]));
                }
            }
        }
        ask(row + stride);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = (c * TPR + t) * W;
            if (a.sum && live && i < a.D) store_piece<T>(a.sum + row * a.lds, i, a.D - i, h[c], at_edge(c));
#pragma unroll
            for (int j = 0; j < W; ++j) sum = __fma_rn((double)h[c][j], (double)h[c][j], sum);
        }
        sum = sum_over_wave(sum);
        if constexpr (TPR > 64) {
            if (threadIdx.x % 64 == 0) red_sum[turn][wave] = sum;
            __syncthreads();
            sum = red_sum[turn][0];
#pragma unroll
            for (int w = 1; w < WAVES; ++w) sum = sum + red_sum[turn][w];
        }
        const float r = norm_factor(sum, a.D, a.eps);
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                h[c][j] = __fmul_rn(__fmul_rn(h[c][j], r), gm[c][j]);
                if constexpr (OUT == I8) {
                    const uint32_t b = __float_as_uint(h[c][j]) & 0x7fffffffu;
                    if ((c * TPR + t) * W < a.D) top = b > top ? b : top;
                }
            }
        if constexpr (OUT == I8) {
            top = max_over<64>(top);
            if constexpr (TPR > 64) {
                if (threadIdx.x % 64 == 0) red_max[turn][wave] = top;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < WAVES; ++w) top = red_max[turn][w] > top ? red_max[turn][w] : top;
            }
            const RowCode code = row_code(top, top_of(I8));
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int j = 0; j < W; ++j) h[c][j] = coded(h[c][j], code);
            if (live && t == 0) a.scales[row] = code.scale;
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int i = (c * TPR + t) * W;
            if (live && i < a.D) store_piece<OUT>(a.out + row * a.ldo, i, a.D - i, h[c], at_edge(c));
        }
    }
}

// Rows longer than the registers hold, any alignment: each pass reads the row
// again (from the stored sum, if there is one; each thread its own elements, one at
// a time, which any D and alignment take alike).  No row of this framework is
// that long; 1024 of 16392 in bf16 with residual and sum 48 us
// against 25 of 16384, of 50000 185 us.  Indices are 64 bits: one step behind the
// longest rows' last 1024 elements is past 2^31.
template <int T, int OUT>
__global__ void __launch_bounds__(1024) rms_norm_long(NormArgs a)
{
    __shared__ double red_sum[16];
    __shared__ uint32_t red_max[16];
    const int wave = threadIdx.x / 64;
    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
        double sum = 0.0;
        for (long long i = threadIdx.x; i < a.D; i += 1024) {
            const float h = sum_at<T>(a, row, i);
            if (a.sum) store1<T>(a.sum + row * a.lds, i, h);
            sum = __fma_rn((double)h, (double)h, sum);
        }
        sum = sum_over_wave(sum);
        __syncthreads();                                  // the last row's readers are done
        if (threadIdx.x % 64 == 0) red_sum[wave] = sum;
        __syncthreads();
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < 16; ++w) sum = sum + red_sum[w];
        const float r = norm_factor(sum, a.D, a.eps);
        auto value = [&](long long i) {
            const float h = a.sum ? load1<T>(a.sum + row * a.lds, i) : sum_at<T>(a, row, i);
            return __fmul_rn(__fmul_rn(h, r), a.gamma ? a.gamma[i] : 1.0f);
        };
        RowCode code{};
        if constexpr (OUT == I8) {
            uint32_t top = 0;
            for (long long i = threadIdx.x; i < a.D; i += 1024) {
                const uint32_t b = __float_as_uint(value(i)) & 0x7fffffffu;
                top = b > top ? b : top;
            }
            top = max_over<64>(top);
            if (threadIdx.x % 64 == 0) red_max[wave] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 16; ++w) top = red_max[w] > top ? red_max[w] : top;
            code = row_code(top, top_of(I8));
            if (threadIdx.x == 0) a.scales[row] = code.scale;
        }
        for (long long i = threadIdx.x; i < a.D; i += 1024) {
            float y = value(i);
            if constexpr (OUT == I8) y = coded(y, code);
            store_piece<OUT>(a.out + row * a.ldo, (int)i, 1, &y, true);
        }
    }
}

// A wave a row while its pieces fit 4 a lane, else a workgroup.  1024 workgroups,
// each with the next row on its way (8192 rows of 4096 in bf16 with residual and
// sum: 50.5 us, 5.3 TB/s; 2048 workgroups 57, 512 59, 4096 without the next row 62).
template <int T, int OUT, bool EDGE>
hipError_t launch_norm(const NormArgs& a, hipStream_t s)
{
    const auto grid = [&](int rows_each) {
        const long long n = ((long long)a.rows + rows_each - 1) / rows_each;
        return dim3((uint32_t)(n < 1024 ? n : 1024));
    };
    const dim3 block(kNormThreads);
    const int pieces = a.D / 8 + (a.D % 8 != 0);
    if (pieces <= 64) return launch(rms_norm<T, OUT, 64, 1, EDGE>, grid(4), block, 0, s, a);
    if (pieces <= 128) return launch(rms_norm<T, OUT, 64, 2, EDGE>, grid(4), block, 0, s, a);
    if (pieces <= 256) return launch(rms_norm<T, OUT, 64, 4, EDGE>, grid(4), block, 0, s, a);
    if (pieces <= 512) return launch(rms_norm<T, OUT, 256, 2, EDGE>, grid(1), block, 0, s, a);
    if (pieces <= 1024) return launch(rms_norm<T, OUT, 256, 4, EDGE>, grid(1), block, 0, s, a);
    if (pieces <= 2048) return launch(rms_norm<T, OUT, 1024, 2, EDGE>, grid(1), dim3(1024), 0, s, a);
    return launch(rms_norm_long<T, OUT>, grid(1), dim3(1024), 0, s, a);
}

template <int T, int OUT>
hipError_t launch_edge(const NormArgs& a, hipStream_t s)
{
    return a.D % 8 ? launch_norm<T, OUT, true>(a, s) : launch_norm<T, OUT, false>(a, s);
}

template <int T>
hipError_t launch_out(int out, const NormArgs& a, hipStream_t s)
{
    return out == I8    ? launch_edge<T, I8>(a, s)
           : out == F32 ? launch_edge<T, F32>(a, s)
           : out == F16 ? launch_edge<T, F16>(a, s)
                        : launch_edge<T, BF16>(a, s);
}

}  // namespace
}  // namespace decode
}  // namespace pkgpu

extern "C" int pk_gpu_rms_norm_dev(int dtype, const void* dx, int ldx, const void* dres, int ldr, void* dsum,
                                   int lds, const float* dgamma, float eps, int out_dtype, void* dout, int ldo,
                                   float* dscales, int rows, int D, void* stream)
{
    using namespace pkgpu::decode;
    namespace rt = pkgpu::rt;
    const char* who = "rms norm";
    if (!is_float(dtype)) return rt::error(PK_GPU_EINVAL, "%s: rows of type %d (F32, F16 or BF16)", who, dtype);
    if (!is_float(out_dtype) && out_dtype != I8)
        return rt::error(PK_GPU_EINVAL, "%s: output of type %d (F32, F16, BF16 or I8)", who, out_dtype);
    if (rows < 0 || D < 1) return rt::error(PK_GPU_EINVAL, "%s: rows = %d, D = %d", who, rows, D);
    if (!(eps >= 0.0f)) return rt::error(PK_GPU_EINVAL, "%s: eps = %g", who, (double)eps);
    if (ldx < D || ldo < D || (dres && ldr < D) || (dsum && lds < D))
        return rt::error(PK_GPU_EINVAL, "%s: a leading dimension of %d, %d, %d, %d is below D = %d", who, ldx, ldr,
                         lds, ldo, D);
    if (rows && (!dx || !dout || (out_dtype == I8 && !dscales)))
        return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    const int es = size_of(dtype), os = size_of(out_dtype);
    const auto off = [](const void* p, size_t bytes) { return !aligned(p, bytes); };
    if (off(dx, es) || off(dres, es) || off(dsum, es) || off(dout, os) || off(dgamma, 4) || off(dscales, 4))
        return rt::error(PK_GPU_EINVAL, "%s: an operand is not aligned to its elements", who);
    // one thread reads and writes an element in place; other overlaps would race
    if (rows && ((dout == dx && (os != es || ldo != ldx)) || (dout == dres && dres && (os != es || ldo != ldr)) ||
        (dsum && ((dsum == dx && lds != ldx) || (dsum == dres && lds != ldr) || dsum == dout))))
        return rt::error(PK_GPU_EINVAL, "%s: out or sum in place needs the input's type and leading dimension, and "
                         "sum may not be out", who);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!rows) return PK_GPU_OK;
    NormArgs a{};
    a.x = static_cast<const char*>(dx);
    a.res = static_cast<const char*>(dres);
    a.sum = static_cast<char*>(dsum);
    a.gamma = dgamma;
    a.out = static_cast<char*>(dout);
    a.scales = dscales;
    a.ldx = (size_t)ldx * es;
    a.ldr = (size_t)ldr * es;
    a.lds = (size_t)lds * es;
    a.ldo = (size_t)ldo * os;
    a.eps = (double)eps;
    a.rows = rows;
    a.D = D;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == F32   ? launch_out<F32>(out_dtype, a, s)
                         : dtype == F16 ? launch_out<F16>(out_dtype, a, s)
                                        : launch_out<BF16>(out_dtype, a, s);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}
