// pk_w8a8.hip - int8 rows times int8 weights with bias, activation and residual
// in the epilogue (pk_gpu_gemm_w8a8_dev), for rows that pk_gpu_rms_norm_dev
// wrote with one scale each.
//
//   acc_ij = sum_k a_ik b_kj                     int32, exact (K <= 131071)
//   v      = fl(fl32(acc) * fl(sa_i sb_j)) (+ bias_j)
//   C_ij   = epilogue(v), rounded once to C's type
//
// v_mfma_i32_16x16x64_i8 with the weights as its first operand: a lane then
// holds 4 consecutive columns of one row of C.  Both operands want 16
// consecutive k of one row (column) per lane.  Activations are stored that way;
// weights [K][N] are not, so a panel holds them re-laid out once, in the order
// lanes read them: [N / 16][K / 64][lane][16 bytes], zero past N and K (K to a
// multiple of 128).  A lane's 16 bytes of lane l, block (nb, kb): column
// 16 nb + l % 16, k from 64 kb + 16 (l / 16).
//
// Tiled kernel: a workgroup's tile of A and of the panel goes from memory to LDS
// past the registers, 128 of K at a time in 2 or 4 stages; half a stage is read
// into registers while the half before it is multiplied, with one barrier a
// stage.  At full size (8192 x 8192 x 8192) 2.1 PFLOP/s, where the library's int8
// product reaches 2.07 on the same card: the clock falls to 1.74 GHz under it, and
// the matrix cores are busy for 60 % of the cycles.  Below, bound by what the caches
// bring to a CU, and by one tile a CU whose epilogue nothing hides.
// Few-row kernel: nothing is shared between waves but the sums, so there is no
// staging: a workgroup takes 16 columns and its 16 waves every 16th block of K,
// A straight from the caches, and the waves' int32 sums are added in LDS.  Bound
// by the launch and one load's latency (33 x 4096 x 1024: 4.8 us), for longer
// rows by what the caches bring to a CU (1 x 4096 x 4096: 5.9 us, 2.9 TB/s).
#include "pk_decode.h"

#include <type_traits>

namespace pkgpu {
namespace decode {
namespace {

struct W8Args {
    const int8_t* A;
    const float* sa;
    const char* panel;
    const float* sb;                // per column, or null: sb1
    const float* bias;
    const char* res;
    char* C;
    size_t lda, ldr, ldc;           // bytes
    float sb1;
    int M, N, K, kb;                // kb: blocks of 64 of K in the panel
    int epi;
    int mt, nt;                     // tiles
};

struct PanelArgs {
    const int8_t* B;
    u32x4* panel;
    long long blocks;
    int ldb, K, N, kb;
};

int blocks_of_k(int K) { return (K + 127) / 128 * 2; }
long long panel_blocks(int K, int N) { return (N + 15ll) / 16 * blocks_of_k(K); }

__global__ void __launch_bounds__(256) w8_panel(PanelArgs p)
{
    const int kb = p.kb, K = p.K, N = p.N;
    const long long blk = (long long)blockIdx.x * 4 + threadIdx.x / 64;
    if (blk >= p.blocks) return;
    const int lane = threadIdx.x & 63;
    const long long nb = blk / kb;
    const long long n = nb * 16 + (lane & 15);
    const int k0 = (int)(blk - nb * kb) * 64 + 16 * (lane >> 4);
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        uint32_t v = 0;
        if (n < N && k0 + i < K) v = (uint8_t)p.B[(size_t)(k0 + i) * p.ldb + n];
        w[i / 4] |= v << (8 * (i % 4));
    }
    p.panel[blk * 64 + lane] = w;
}

__device__ inline i32x4 mfma_i8(u32x4 b, u32x4 a, i32x4 c)
{
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c,
                                                 0, 0, 0);
}

// v / (1 + e^-v) as v times the hardware's reciprocal (within 2^-23), e^-v =
// 2^t with t = -v log2(e).  For f32 outputs e^-v takes the product's rounding
// t' in, 2^t (1 + ln2 t'), and the whole is within 2^-21 of its value; for
// 16-bit ones t is off by up to 2^-24 |t|, so the value by 2^-21 + 2^-24 |v|.
// (The fp32 GEMMs' Swish follows the reference's polynomial, whose e^-v is off
// by up to 2.4e-6.)  Below v = -87.3 e^-v's reciprocal leaves the normal range and
// the result is -0, off by at most 2^-119.  The IEEE division took 12 of this
// epilogue's 35 instructions an element.
template <int T>
__device__ inline float swish(float v)
{
    float e;
    if constexpr (T == F32) {
        const float x = fminf(fmaxf(-v, -100.0f), 100.0f);
        const float t = __fmul_rn(x, 0x1.715476p+0f);
        const float lo = __fmaf_rn(x, 0x1.4ae0cp-26f, __fmaf_rn(x, 0x1.715476p+0f, -t));
        e = __fmul_rn(__builtin_amdgcn_exp2f(t), __fmaf_rn(lo, 0x1.62e43p-1f, 1.0f));
    } else {
        e = __builtin_amdgcn_exp2f(__fmul_rn(v, -0x1.715476p+0f));
    }
    return __fmul_rn(v, __builtin_amdgcn_rcpf(__fadd_rn(1.0f, e)));
}

template <int T, int EPI>
__device__ inline float finish(float v, float res)
{
    if constexpr (EPI == PK_GPU_EPI_SWISH) return swish<T>(v);
    else if constexpr (EPI == PK_GPU_EPI_HALF_RESIDUAL) return __fadd_rn(res, __fmul_rn(0.5f, v));
    else if constexpr (EPI == PK_GPU_EPI_RESIDUAL) return __fadd_rn(res, v);
    else if constexpr (EPI == PK_GPU_EPI_RELU) return v > 0.0f ? v : 0.0f;
    else return v;
}

// What the 4 columns from j on are multiplied with and biased by.
struct Columns { float s[4], b[4]; };
__device__ inline Columns columns_of(const W8Args& a, int j)
{
    Columns c;
#pragma unroll
    for (int e = 0; e < 4; ++e) { c.s[e] = a.sb1; c.b[e] = 0.0f; }
    if (j + 4 <= a.N) {
        if (a.sb) {
            const f32x4 s = *reinterpret_cast<const f32x4_any*>(a.sb + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) c.s[e] = s[e];
        }
        if (a.bias) {
            const f32x4 b = *reinterpret_cast<const f32x4_any*>(a.bias + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) c.b[e] = b[e];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < a.N) {
                if (a.sb) c.s[e] = a.sb[j + e];
                if (a.bias) c.b[e] = a.bias[j + e];
            }
    }
    return c;
}

// 4 sums of row i (scale sa), columns j .. j + 3, to C
template <int T, int EPI>
__device__ inline void store_c(const W8Args& a, int i, float sa, int j, const Columns& col, i32x4 acc)
{
    if (i >= a.M || j >= a.N) return;
    constexpr bool residual = EPI == PK_GPU_EPI_RESIDUAL || EPI == PK_GPU_EPI_HALF_RESIDUAL;
    const char* r = a.res + (size_t)i * a.ldr;
    char* c = a.C + (size_t)i * a.ldc;
    float v[4], old[4] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[e] = __fmul_rn((float)acc[e], __fmul_rn(sa, col.s[e]));
        if (a.bias) v[e] = __fadd_rn(v[e], col.b[e]);
    }
    if (j + 4 <= a.N) {                // whole accesses at any alignment
        if constexpr (residual) {
            if constexpr (T == F32) {
                const f32x4 o = *reinterpret_cast<const f32x4_any*>(r + (size_t)j * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) old[e] = o[e];
            } else {
                const u32x2 o = *reinterpret_cast<const u32x2_any*>(r + (size_t)j * 2);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t w = o[e];       // a bit cast of o[e] itself takes o[0]'s bits
                    const f16x2 h = __builtin_bit_cast(f16x2, w);
                    old[2 * e] = T == F16 ? (float)h[0] : bf16_lo(w);
                    old[2 * e + 1] = T == F16 ? (float)h[1] : bf16_hi(w);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = finish<T, EPI>(v[e], old[e]);
        if constexpr (T == F32)
            *reinterpret_cast<f32x4_any*>(c + (size_t)j * 4) = (f32x4){v[0], v[1], v[2], v[3]};
        else
            *reinterpret_cast<u32x2_any*>(c + (size_t)j * 2) =
                T == F16 ? (u32x2){pack_f16(v[0], v[1]), pack_f16(v[2], v[3])}
                         : (u32x2){pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (j + e < a.N) {
            if constexpr (residual) old[e] = load1<T>(r, j + e);
            store1<T>(c, j + e, finish<T, EPI>(v[e], old[e]));
        }
}

// 16 bytes a lane from base + off to LDS at lds + 16 * lane, past the registers.
// The caller counts and waits (wait_loads): the compiler does not see it.
__device__ inline void load_to_lds(uint32_t lds, const char* base, uint32_t off)
{
    __asm__ volatile("s_mov_b32 m0, %0\n\t"
                     "s_nop 0\n\t"
                     "global_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}
// Until LEFT of them are outstanding, and no LDS read is.
template <int LEFT>
__device__ inline void wait_loads()
{
    __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
}

// WM x WN waves of MB x NB blocks of 16 x 16; STAGES of 128 of K in LDS.
//
// A stage's block of 16 rows of A is 2 pieces of 8 rows x 128 bytes, so that
// every load takes whole cache lines; slot c of row r holds the row's 16-byte
// chunk c ^ (r % 8), so that the 8 rows a quarter wave reads of one chunk are in
// different banks.  A stage's block of 16 columns is 2 pieces of the panel, for
// its two halves of K.
template <int T, int EPI, int WM, int WN, int MB, int NB, int STAGES>
__global__ void __launch_bounds__(64 * WM * WN, WM * WN / 4) w8_tiled(W8Args a)
{
    constexpr int NW = WM * WN, AB = WM * MB, BB = WN * NB;    // blocks of a tile
    constexpr int PIECES = 2 * (AB + BB);                      // 1 KB pieces of a stage
    static_assert(PIECES % NW == 0);
    constexpr int P = PIECES / NW;                             // pieces a wave loads
    __shared__ u32x4 lds[STAGES][PIECES][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // Consecutive workgroups go round the 8 L2s: each L2 gets a run of the tiles
    // in an order that goes down 8 of them before it moves right, so that the
    // tiles it has at a time share rows and columns.
    const uint32_t tiles = (uint32_t)a.mt * a.nt, per = tiles / 8, rest = tiles % 8;
    const uint32_t l2 = blockIdx.x % 8, at = blockIdx.x / 8;
    const uint32_t id = l2 * per + (l2 < rest ? l2 : rest) + at;
    const uint32_t band = id / (8u * a.nt), first = band * 8, rows = min(8u, a.mt - first);
    const int mt = first + (id - band * 8 * a.nt) % rows, nt = (id - band * 8 * a.nt) / rows;

    // piece q < 2 AB: rows 8 q on of the tile's; then the panel's
    const char* base[P];
    uint32_t off[P];
    const uint32_t klast = (uint32_t)(a.K - 1) / 16 * 16;
    const uint32_t k0 = 16 * ((lane & 7) ^ (lane >> 3));
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int q = wave * P + i;
        if (q < 2 * AB) {
            int m0 = mt * AB * 16 + 8 * q;
            m0 = m0 < a.M ? m0 : a.M - 1;
            const int m = m0 + (lane >> 3) < a.M ? lane >> 3 : a.M - 1 - m0;
            base[i] = reinterpret_cast<const char*>(a.A) + (size_t)m0 * a.lda;
            off[i] = (uint32_t)m * (uint32_t)a.lda;
        } else {
            const int nblocks = (a.N + 15) / 16;
            int nb = nt * BB + (q - 2 * AB) / 2;
            nb = nb < nblocks ? nb : nblocks - 1;
            base[i] = a.panel + ((size_t)nb * a.kb + q % 2) * 1024;
            off[i] = 16 * lane;
        }
    }
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)(char*)&lds[0][0][0];
    auto load = [&](int s) {
        const uint32_t k = 128 * s + k0;
        const uint32_t ka = k < klast ? k : klast;     // past K the panel is zero: any of the row's bytes will do
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int q = wave * P + i;
            load_to_lds(lds0 + ((s % STAGES) * PIECES + q) * 1024, base[i], q < 2 * AB ? off[i] + ka : off[i] + 2048 * s);
        }
    };
    struct Frags { u32x4 a[MB], b[NB]; };
    const int row = lane & 15;
    auto read = [&](int s, int half, Frags& f) {
        const int slot = row * 8 + ((4 * half + (lane >> 4)) ^ (row & 7));
#pragma unroll
        for (int j = 0; j < NB; ++j) f.b[j] = lds[s % STAGES][2 * (AB + wn * NB + j) + half][lane];
#pragma unroll
        for (int i = 0; i < MB; ++i) f.a[i] = lds[s % STAGES][2 * (wm * MB + i)][slot];
    };
    i32x4 acc[MB][NB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = (i32x4){0, 0, 0, 0};
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[i][j] = mfma_i8(f.b[j], f.a[i], acc[i][j]);
    };

    const int steps = a.kb / 2;
    // Each half of a step is read while the half before it is multiplied.  At the
    // second half of step s all waves' reads of stage s are back before the
    // barrier, so stage s + STAGES may overwrite it behind it.  The last steps are
    // copies without loads: on a condition, the wait for one half's operands
    // would be one for the next half's too.
    auto step = [&](int s, Frags& f0, Frags& f1, auto loads, auto left) {
        read(s, 1, f1);
        multiply(f0);
        wait_loads<decltype(left)::value * P>();
        __builtin_amdgcn_s_barrier();
        if constexpr (decltype(loads)::value) load(s + STAGES);
        read(s + 1, 0, f0);
        multiply(f1);
    };
    const std::integral_constant<int, 0> all;          // stages that may still be on their way
    const std::integral_constant<int, STAGES - 2> ahead;
    Frags f0, f1;
    if (steps >= STAGES) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) load(i);
        wait_loads<(STAGES - 1) * P>();
    } else {
        for (int i = 0; i < steps; ++i) load(i);
        wait_loads<0>();
    }
    __builtin_amdgcn_s_barrier();
    read(0, 0, f0);
    int s = 0;
    for (; s + STAGES < steps; ++s) step(s, f0, f1, std::true_type{}, ahead);
    for (; s + 1 < steps; ++s) step(s, f0, f1, std::false_type{}, all);
    read(s, 1, f1);
    multiply(f0);
    multiply(f1);

    Columns col[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) col[j] = columns_of(a, (nt * BB + wn * NB + j) * 16 + 4 * (lane >> 4));
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = (mt * AB + wm * MB + i) * 16 + row;
        const float sa = a.sa[m < a.M ? m : a.M - 1];
#pragma unroll
        for (int j = 0; j < NB; ++j)
            store_c<T, EPI>(a, m, sa, (nt * BB + wn * NB + j) * 16 + 4 * (lane >> 4), col[j], acc[i][j]);
    }
}

constexpr int kFewWaves = 16;

// MB blocks of 16 rows from block MB * blockIdx.y on, 16 columns.
template <int T, int EPI, int MB>
__global__ void __launch_bounds__(64 * kFewWaves) w8_few(W8Args a)
{
    __shared__ i32x4 sums[kFewWaves][MB][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nb = blockIdx.x, m0 = 16 * MB * blockIdx.y;
    const char* rows[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int m = m0 + 16 * i + (lane & 15);
        rows[i] = reinterpret_cast<const char*>(a.A) + (size_t)(m < a.M ? m : a.M - 1) * a.lda;
    }
    const char* w = a.panel + ((size_t)nb * a.kb * 64 + lane) * 16;
    i32x4 acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = (i32x4){0, 0, 0, 0};
#pragma unroll 4
    for (int kb = wave; kb < a.kb; kb += kFewWaves) {
        const u32x4 fb = *reinterpret_cast<const u32x4*>(w + (size_t)kb * 1024);
        const int k = 64 * kb + 16 * (lane >> 4);
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const u32x4 fa = *reinterpret_cast<const u32x4*>(rows[i] + (k < a.K ? k : 0));
            acc[i] = mfma_i8(fb, fa, acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave >= MB) return;
    i32x4 sum = sums[0][wave][lane];
#pragma unroll
    for (int v = 1; v < kFewWaves; ++v) sum += sums[v][wave][lane];
    const int row = m0 + 16 * wave + (lane & 15), j = 16 * nb + 4 * (lane >> 4);
    store_c<T, EPI>(a, row, a.sa[row < a.M ? row : a.M - 1], j, columns_of(a, j), sum);
}

// The kernel that a product goes to, and its launch.
enum Kernel { FEW, TILE_64, TILE_128_DEEP, TILE_128, TILE_256 };
struct Choice { Kernel kernel; int bm, bn; long long workgroups; int threads; };

long long tiles_of(int M, int N, int bm, int bn)
{
    return ((long long)M + bm - 1) / bm * (((long long)N + bn - 1) / bn);
}

Choice choose(int M, int N)
{
    const auto of = [&](Kernel k, int bm, int bn, int threads) {
        return Choice{k, bm, bn, tiles_of(M, N, bm, bn), threads};
    };
    // Few rows, or too few 64 x 64 tiles to be worth staging (us; this kernel,
    // 64 x 64 tiles): 33 x 4096 x 4096 9.8, 11.2; 64 x 4096 x 4096 12.5, 11.5; 64 x
    // 1024 x 4096 5.8, 10.1; 128 x 1024 x 4096 8.0, 10.0; 256 x 1024 x 4096 12.3, 11.4;
    // 17 x 16384 x 4096 17.8, 14.7.
    const long long small = tiles_of(M, N, 64, 64);
    if (M <= 16 || small < 48 || (small < 128 && M <= 48)) {
        // as many blocks of rows a workgroup as leave 256 workgroups (33 x 1024 x
        // 4096: 5.6 us in 64 x 3 workgroups, 8.0 in 64).  4 never do: fewer than 48
        // tiles of 64 x 64 are at most 4 * 47 of 64 x 16, and M <= 48 has 3.
        const int blocks = (M + 15) / 16;
        int mb = blocks < 3 ? blocks : 3;
        while (mb > 1 && tiles_of(M, N, 16 * mb, 16) < 256) --mb;
        return of(FEW, 16 * mb, 16, 64 * kFewWaves);
    }
    // The largest tile of which there are enough for the 256 CUs; 128 x 128 with
    // two workgroups a CU (2 stages each) where there are more tiles than CUs, with
    // 4 stages where there are not.  Measured (us; 256 x 256, 128 x 128 in 2 and in
    // 4 stages, 64 x 64), bf16 output:
    //   8192 x 4096 x 8192   276, 306, 348, 477
    //   4001 x 4096 x 1024    30, 30.5, 37, 47
    //   2000 x 4096 x 1024    26, 17.6, 20.4, 25
    //   4001 x 1024 x 4096    63, 29, 26.7, 36
    //    512 x 4096 x 4096    61, 27, 23.7, 18.8
    //    128 x 4096 x 1024    23, 9.2, 9.3, 5.9
    if (tiles_of(M, N, 256, 256) >= 200) return of(TILE_256, 256, 256, 512);
    const long long mid = tiles_of(M, N, 128, 128);
    if (mid > 256) return of(TILE_128, 128, 128, 512);
    if (mid >= 200) return of(TILE_128_DEEP, 128, 128, 512);
    return of(TILE_64, 64, 64, 512);
}

template <int T, int EPI, int WM, int WN, int MB, int NB, int STAGES>
hipError_t launch_tiled(W8Args a, const Choice& c, hipStream_t s)
{
    static_assert(WM * WN == 8);
    a.mt = (a.M + c.bm - 1) / c.bm;
    a.nt = (a.N + c.bn - 1) / c.bn;
    return launch(w8_tiled<T, EPI, WM, WN, MB, NB, STAGES>, dim3((uint32_t)c.workgroups), dim3(c.threads), 0, s, a);
}

template <int T, int EPI>
hipError_t launch_w8(const W8Args& a, const Choice& c, hipStream_t s)
{
    switch (c.kernel) {
    case TILE_256: return launch_tiled<T, EPI, 2, 4, 8, 4, 2>(a, c, s);
    case TILE_128: return launch_tiled<T, EPI, 2, 4, 4, 2, 2>(a, c, s);
    case TILE_128_DEEP: return launch_tiled<T, EPI, 2, 4, 4, 2, 4>(a, c, s);
    case TILE_64: return launch_tiled<T, EPI, 2, 4, 2, 1, 4>(a, c, s);
    case FEW: break;
    }
    const dim3 grid((a.N + 15) / 16, (a.M + c.bm - 1) / c.bm), block(c.threads);
    return c.bm == 16   ? launch(w8_few<T, EPI, 1>, grid, block, 0, s, a)
           : c.bm == 32 ? launch(w8_few<T, EPI, 2>, grid, block, 0, s, a)
                        : launch(w8_few<T, EPI, 3>, grid, block, 0, s, a);
}

template <int T>
hipError_t launch_epi(const W8Args& a, const Choice& c, hipStream_t s)
{
    switch (a.epi) {
    case PK_GPU_EPI_SWISH: return launch_w8<T, PK_GPU_EPI_SWISH>(a, c, s);
    case PK_GPU_EPI_HALF_RESIDUAL: return launch_w8<T, PK_GPU_EPI_HALF_RESIDUAL>(a, c, s);
    case PK_GPU_EPI_RESIDUAL: return launch_w8<T, PK_GPU_EPI_RESIDUAL>(a, c, s);
    case PK_GPU_EPI_RELU: return launch_w8<T, PK_GPU_EPI_RELU>(a, c, s);
    default: return launch_w8<T, PK_GPU_EPI_NONE>(a, c, s);
    }
}

}  // namespace
}  // namespace decode
}  // namespace pkgpu

extern "C" {

using namespace pkgpu::decode;

size_t pk_gpu_w8_panel_bytes(int K, int N)
{
    if (K < 1 || N < 1 || K > 131071 || N > 1 << 30) return 0;
    const long long blocks = panel_blocks(K, N);
    return launchable((blocks + 3) / 4, 256) ? (size_t)blocks * 1024 : 0;
}

int pk_gpu_w8_panel_dev(int K, int N, const int8_t* dB, int ldb, void* dpanel, void* stream)
{
    namespace rt = pkgpu::rt;
    const char* who = "w8 panel";
    if (K < 1 || N < 1 || K > 131071 || N > 1 << 30)
        return rt::error(PK_GPU_EINVAL, "%s: K = %d (1..131071), N = %d (1..2^30)", who, K, N);
    if (ldb < N) return rt::error(PK_GPU_EINVAL, "%s: ldb = %d < N = %d", who, ldb, N);
    if (!dB || !dpanel) return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    if (!aligned16(dpanel)) return rt::error(PK_GPU_EINVAL, "%s: the panel must be 16-byte aligned", who);
    const long long blocks = panel_blocks(K, N);
    if (!launchable((blocks + 3) / 4, 256)) return rt::error(PK_GPU_EINVAL, "%s: %d x %d exceeds the grid", who, K, N);
    OnDevice on;
    if (on.rc) return on.rc;
    const PanelArgs p{dB, static_cast<u32x4*>(dpanel), blocks, ldb, K, N, blocks_of_k(K)};
    const hipError_t e = launch(w8_panel, dim3((uint32_t)((blocks + 3) / 4)), dim3(256), 0,
                                static_cast<hipStream_t>(stream), p);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

int pk_gpu_gemm_w8a8_dev(int M, int N, int K, const int8_t* dA, int lda, const float* dA_scales,
                         const void* dpanel, float B_scale, const float* dB_scales, const float* dbias,
                         int epilogue, const void* dres, int ldr, int dtype, void* dC, int ldc, void* stream)
{
    namespace rt = pkgpu::rt;
    const char* who = "w8a8 gemm";
    if (M < 0 || N < 0 || M > 1 << 30 || N > 1 << 30 || K < 1 || K > 131071)
        return rt::error(PK_GPU_EINVAL, "%s: M = %d, N = %d (0..2^30), K = %d (1..131071)", who, M, N, K);
    if (!is_float(dtype)) return rt::error(PK_GPU_EINVAL, "%s: output of type %d (F32, F16 or BF16)", who, dtype);
    if (epilogue < PK_GPU_EPI_NONE || epilogue > PK_GPU_EPI_RELU)
        return rt::error(PK_GPU_EINVAL, "%s: epilogue %d is not one of PK_GPU_EPI_*", who, epilogue);
    if (lda < K || lda % 16 || lda > 1 << 27)          // 16 rows within 32 bits
        return rt::error(PK_GPU_EINVAL, "%s: lda = %d (a multiple of 16 from K = %d to 2^27)", who, lda, K);
    const bool residual = epilogue == PK_GPU_EPI_RESIDUAL || epilogue == PK_GPU_EPI_HALF_RESIDUAL;
    if (ldc < N || (residual && ldr < N))
        return rt::error(PK_GPU_EINVAL, "%s: ldc = %d, ldr = %d below N = %d", who, ldc, ldr, N);
    if (M && N && (!dA || !dA_scales || !dpanel || !dC || (residual && !dres)))
        return rt::error(PK_GPU_EINVAL, "%s: NULL operand", who);
    if (!aligned16(dA) || !aligned16(dpanel))
        return rt::error(PK_GPU_EINVAL, "%s: A and the panel must be 16-byte aligned", who);
    const int es = size_of(dtype);
    const auto off = [](const void* p, size_t bytes) { return !aligned(p, bytes); };
    if (off(dC, es) || (residual && off(dres, es)) || off(dA_scales, 4) || off(dB_scales, 4) || off(dbias, 4))
        return rt::error(PK_GPU_EINVAL, "%s: an operand is not aligned to its elements", who);
    if (residual && dres == dC && ldr != ldc)
        return rt::error(PK_GPU_EINVAL, "%s: a residual in place needs C's leading dimension", who);
    const Choice c = M && N ? choose(M, N) : Choice{};
    if (!launchable(c.workgroups, c.threads)) return rt::error(PK_GPU_EINVAL, "%s: %d x %d exceeds the grid", who, M, N);
    OnDevice on;
    if (on.rc) return on.rc;
    if (!M || !N) return PK_GPU_OK;
    W8Args a{};
    a.A = dA;
    a.lda = lda;
    a.sa = dA_scales;
    a.panel = static_cast<const char*>(dpanel);
    a.sb = dB_scales;
    a.sb1 = B_scale;
    a.bias = dbias;
    a.res = residual ? static_cast<const char*>(dres) : nullptr;
    a.ldr = residual ? (size_t)ldr * es : 0;
    a.C = static_cast<char*>(dC);
    a.ldc = (size_t)ldc * es;
    a.M = M; a.N = N; a.K = K;
    a.kb = blocks_of_k(K);
    a.epi = epilogue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const hipError_t e = dtype == F32   ? launch_epi<F32>(a, c, s)
                         : dtype == F16 ? launch_epi<F16>(a, c, s)
                                        : launch_epi<BF16>(a, c, s);
    return e == hipSuccess ? PK_GPU_OK : rt::hip_error(e, who);
}

}  // extern "C"
