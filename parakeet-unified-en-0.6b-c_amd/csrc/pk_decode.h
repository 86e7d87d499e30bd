// pk_decode.h - what the decoder operators share (pk_rms_norm.hip,
// pk_kv_cache.hip, pk_paged_attention*.hip, pk_w8a8.hip): element types, the
// conversion of a row to 8-bit codes, and the host side of a call.
//
// Codes of a row (a cache row, or a normalised row): with a = max |x|,
// top = 127 (int8) or 448 (e4m3),
//   scale = fl(a / top) (at most kTopScale), inv = fl(top / a),
//   code = round(fl(x * inv)),
// rounded to the nearest int8 or e4m3 value, ties to even.  One division a
// row and one product an element: x * inv is off the true quotient by at
// most 2 roundings (2^-23 relative), against half a step (2^-8 of the
// largest code) of the code's own rounding.  |x * inv| <= top * (1 + 2^-23),
// which rounds to top, so no clamp is needed.  A row with a < 2^-100 gets
// scale 0 and codes 0 (inv of smaller rows could overflow); a row that holds
// an infinity or a NaN gets scale NaN and codes 0, so all of it reads back as
// NaN rather than as finite values of a wrong size.
//
// 4-bit rows (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) are cut into
// groups of 32 elements; with a = max |x| of a group its unit u is the smallest
// power of two with a <= 7 u, so that no element is off by more than half a step (7 u
// goes to 6 u), and code = x / u rounded to nearest, ties to even: exact steps all
// of them, done by the matrix cores' own conversion.  u is stored as one byte,
// its exponent + 127, at most 2^125 (6 u stays finite); a < 2^-100 gives zeros with
// byte 0, a group with an infinity or a NaN byte 255, which reads back as NaN.
// code * u is exact in bf16.
#pragma once

#include "pk_gpu.h"
#include "pk_gpu_internal.h"

#include <hip/hip_runtime.h>

#include <cstdint>

namespace pkgpu {
namespace decode {

using f32x4 = __attribute__((ext_vector_type(4))) float;
using u32x2 = __attribute__((ext_vector_type(2))) uint32_t;
using u32x4 = __attribute__((ext_vector_type(4))) uint32_t;
using i32x4 = __attribute__((ext_vector_type(4))) int;
using bf16x2 = __attribute__((ext_vector_type(2))) __bf16;
using f16x2 = __attribute__((ext_vector_type(2))) _Float16;
using bf16x8 = __attribute__((ext_vector_type(8))) __bf16;
using f16x8 = __attribute__((ext_vector_type(8))) _Float16;
using f32x2 = __attribute__((ext_vector_type(2))) float;

// The same vectors at an address that is only aligned to their elements: the
// compiler keeps them one access (global memory takes any alignment on this
// target), which may touch one cache line more.
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// element types as template parameters
constexpr int F32 = PK_GPU_F32, F16 = PK_GPU_F16, BF16 = PK_GPU_BF16, I8 = PK_GPU_I8, E4M3 = PK_GPU_E4M3,
              E2M1 = PK_GPU_E2M1;
constexpr int size_of(int t) { return t == F32 ? 4 : t == F16 || t == BF16 ? 2 : 1; }     // not of E2M1
constexpr int bytes_of(int t, int elements) { return t == E2M1 ? elements / 2 : elements * size_of(t); }
constexpr int kGroup = 32;                 // elements of an e2m1 row that share a unit
// whether a cache holds codes with an fp32 scale for each row
constexpr bool row_scaled(int t) { return t == I8 || t == E4M3; }
constexpr float top_of(int t) { return t == I8 ? 127.0f : 448.0f; }
constexpr float kTinyRow = 0x1p-100f;
// The largest scale s whose 127 s is finite: fl(a / 127) of an a within an ulp
// of the largest float rounds up to one whose product would be infinite.
constexpr float kTopScale = 0x1.020406p+121f;

// ---- device: values of one type as fp32, and back (rounded to nearest) -----

__device__ inline float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ inline float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ inline uint32_t pack_bf16(float a, float b)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2));
}
__device__ inline uint32_t pack_f16(float a, float b)
{
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2));
}

template <int T>
__device__ inline float load1(const void* p, size_t i)
{
    if constexpr (T == F32) return static_cast<const float*>(p)[i];
    else if constexpr (T == F16) return (float)static_cast<const _Float16*>(p)[i];
    else return __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}
template <int T>
__device__ inline void store1(void* p, size_t i, float x)
{
    if constexpr (T == F32) static_cast<float*>(p)[i] = x;
    else if constexpr (T == F16) static_cast<_Float16*>(p)[i] = (_Float16)x;
    else static_cast<uint16_t*>(p)[i] = (uint16_t)pack_bf16(x, x);
}
// x rounded to T and back
template <int T>
__device__ inline float as_type(float x)
{
    if constexpr (T == F32) return x;
    else if constexpr (T == F16) return (float)(_Float16)x;
    else return bf16_lo(pack_bf16(x, x));
}

// 8 consecutive elements at a 16-byte (8-bit types: 8-byte) aligned address
template <int T>
__device__ inline void load8(const void* p, float* x)
{
    if constexpr (T == F32) {
        const f32x4 a = static_cast<const f32x4*>(p)[0], b = static_cast<const f32x4*>(p)[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
    } else if constexpr (T == F16) {
        const f16x8 a = *static_cast<const f16x8*>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
    } else if constexpr (T == BF16) {
        const u32x4 a = *static_cast<const u32x4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[2 * i] = bf16_lo(a[i]); x[2 * i + 1] = bf16_hi(a[i]); }
    } else {
        const u32x2 a = *static_cast<const u32x2*>(p);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (T == I8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * i + j] = (float)(int)(signed char)(a[i] >> (8 * j));
            } else {
                const f32x2 l = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], false);
                const f32x2 h = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], true);
                x[4 * i] = l[0]; x[4 * i + 1] = l[1]; x[4 * i + 2] = h[0]; x[4 * i + 3] = h[1];
            }
        }
    }
}

// 8 values to T (8-bit types: x already multiplied by inv)
template <int T>
__device__ inline void store8(void* p, const float* x)
{
    if constexpr (T == F32) {
        static_cast<f32x4*>(p)[0] = (f32x4){x[0], x[1], x[2], x[3]};
        static_cast<f32x4*>(p)[1] = (f32x4){x[4], x[5], x[6], x[7]};
    } else if constexpr (T == F16 || T == BF16) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[i] = T == F16 ? pack_f16(x[2 * i], x[2 * i + 1]) : pack_bf16(x[2 * i], x[2 * i + 1]);
        *static_cast<u32x4*>(p) = w;
    } else {
        u32x2 w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (T == I8) {
                uint32_t u = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    u |= ((uint32_t)(int)__builtin_rintf(x[4 * i + j]) & 0xffu) << (8 * j);
                w[i] = u;
            } else {
                int u = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
                w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], u, true);
            }
        }
        *static_cast<u32x2*>(p) = w;
    }
}

// The row's scale and multiplier from the bits of max |x| (as unsigned: NaN >
// infinity > every finite value).
struct RowCode { float scale, inv; };
__device__ inline RowCode row_code(uint32_t amax_bits, float top)
{
    if (amax_bits >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.0f};
    const float a = __uint_as_float(amax_bits);
    if (a < kTinyRow) return {0.0f, 0.0f};
    return {fminf(__fdiv_rn(a, top), kTopScale), __fdiv_rn(top, a)};
}
// The unit of a group of 4-bit codes from the bits of its max |x|: its byte. A
// unit's bits as a float are byte << 23 (the conversions take 0 for 2^-127 and
// infinity for NaN).
__device__ inline uint32_t group_byte(uint32_t amax_bits)
{
    if (amax_bits >= 0x7f800000u) return 255;
    if (__uint_as_float(amax_bits) < kTinyRow) return 0;
    const uint32_t e = (amax_bits >> 23) - 2 + ((amax_bits & 0x7fffffu) > 0x600000u);
    return e < 252 ? e : 252;
}
// 8 elements of a group as codes; zeros where it has none.
__device__ inline uint32_t codes_e2m1(const float* x, uint32_t byte)
{
    const bool none = byte == 0 || byte == 255;
    const float unit = __uint_as_float(byte << 23);
    uint32_t w = 0;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = none ? 0.0f : x[i];
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[0], y[1], unit, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[2], y[3], unit, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[4], y[5], unit, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, y[6], y[7], unit, 3);
}
__device__ inline void values_e2m1(uint32_t w, uint32_t byte, float* x)
{
    const float unit = __uint_as_float(byte << 23);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, unit, 3);
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
}
// x * inv, 0 where the row has no codes (x may be NaN or infinite there)
__device__ inline float coded(float x, RowCode c) { return c.inv == 0.0f ? 0.0f : __fmul_rn(x, c.inv); }

// x of the lane's partner among 2, 4, 8 or 16 lanes (STEP 1, 2, 4, 8) where the
// lanes of each half group hold the same value already: mirrors of the group, so
// a few cycles in the vector unit instead of a trip through LDS.
template <int STEP>
__device__ inline uint32_t mirrored(uint32_t x)
{
    constexpr int CTRL = STEP == 1 ? 0xB1 : STEP == 2 ? 0x4E : STEP == 4 ? 0x141 : 0x140;
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xF, 0xF, true);
}
template <int STEP>
__device__ inline uint32_t partner(uint32_t x)
{
    if constexpr (STEP < 16) return mirrored<STEP>(x);
    else return __shfl_xor(x, STEP);
}
// The largest over aligned groups of LANES lanes.
template <int LANES, int STEP = 1>
__device__ inline uint32_t max_over(uint32_t x)
{
    if constexpr (STEP < LANES) {
        const uint32_t o = partner<STEP>(x);
        return max_over<LANES, 2 * STEP>(o > x ? o : x);
    } else {
        return x;
    }
}
// The sum over the wave, the same on every lane (a + b = b + a).
template <int STEP = 1>
__device__ inline double sum_over_wave(double x)
{
    if constexpr (STEP < 64) {
        const uint32_t lo = partner<STEP>((uint32_t)__double2loint(x)), hi = partner<STEP>((uint32_t)__double2hiint(x));
        return sum_over_wave<2 * STEP>(x + __hiloint2double((int)hi, (int)lo));
    } else {
        return x;
    }
}

// ---- host ------------------------------------------------------------------

// One entry point's time on the library's device: initialises the library if
// needed and makes its device current until the call returns, whichever device
// the calling thread had.  Unlike rt::bind it creates no stream, so a thread's
// first call may be one that is captured.
class OnDevice {
    int prev_ = -1;
public:
    int rc;
    OnDevice()
    {
        int cur = -1, dev = 0;
        if (hipGetDevice(&cur) != hipSuccess) cur = -1;
        rc = rt::enter(&dev);
        int now = -1;
        if (rc) return;
        (void)hipGetDevice(&now);
        if (now != dev) {
            const hipError_t e = hipSetDevice(dev);
            if (e != hipSuccess) rc = rt::hip_error(e, "hipSetDevice");
        }
        prev_ = cur >= 0 && cur != dev ? cur : -1;
    }
    ~OnDevice() { if (prev_ >= 0) (void)hipSetDevice(prev_); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

// Launch fn and return its own status: an error that an earlier HIP call of
// the thread left behind is not this call's.
template <typename Args>
inline hipError_t launch(void (*fn)(Args), dim3 grid, dim3 block, size_t lds, hipStream_t s, Args a)
{
    void* p[] = {&a};
    return hipLaunchKernel(reinterpret_cast<const void*>(fn), grid, block, p, lds, s);
}

// Whether a launch of so many workgroups is one that HIP takes: below 2^32 threads.
inline bool launchable(long long workgroups, int threads)
{
    return workgroups <= 0x7fffffff && workgroups * threads < 1ll << 32;
}

inline bool is_float(int t) { return t == F32 || t == F16 || t == BF16; }
inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
inline bool aligned16(const void* p) { return aligned(p, 16); }
// PK_GPU_OK, or the error of a cache description
int check_cache(const pk_gpu_kv_cache* c, const char* who);

}  // namespace decode
}  // namespace pkgpu
