// pk_prompt_attention.h - attention of many new tokens per sequence over a paged
// key-value cache: the kernel, instantiated per cache type by pk_prompt_attention_*.hip.
#pragma once

#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;

// Tokens of a tile: as many as leave the registers of two workgroups a CU whole (one
// at heads of 256, and there half as many where codes wait in registers too).
constexpr int prompt_keys(int cache, int t, int dim)
{
    return dim == 64 ? 128 : dim == 128 ? 64 : cache == F16 || cache == BF16 || (cache == E2M1 && t == BF16) ? 64 : 32;
}

constexpr int prompt_p_terms(int cache, int t) { return t == F32 ? 3 : t == F16 && cache != F16 ? 2 : 1; }
// column blocks of 32 rows a wave takes, and workgroups a CU
constexpr int prompt_blocks(int cache, int t, int dim) { return 1; }
constexpr int prompt_occupancy(int cache, int t, int dim) { return dim == 256 || t == F32 ? 1 : 2; }

template <bool IN_F16>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (IN_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16 bytes a lane from base + off to LDS at lds + 16 * lane, past the registers.  The
// compiler does not see it: whoever reads waits for vmcnt(0) first.
__device__ inline void cache_to_lds(uint32_t lds, const char* base, uint32_t off)
{
    __asm__ volatile("s_mov_b32 m0, %0\n\t"
                     "s_nop 0\n\t"
                     "global_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// The sequence and row tile of the launch's tau-th row tile: tiles of BM rows, sequence by
// sequence, the last tiles (whose rows see most) first.  False behind the last.
struct RowTile { int b, tile; };
template <int BM>
__device__ inline bool row_tile(const PagedArgs& a, int tau, RowTile* out)
{
    const int lane = threadIdx.x & 63;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int b = b0 + lane;
        int n = b < a.B ? (int)(((long long)new_tokens(a.rules, b).count * a.group + BM - 1) / BM) : 0;
        int upto = n;
        if (a.B > 1) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(upto, d);
                upto += lane >= d ? o : 0;
            }
        } else {
            upto = __builtin_amdgcn_readfirstlane(n);
        }
        const unsigned long long mine = __ballot(upto > tau);
        if (mine) {
            const int l = __builtin_ctzll(mine);
            out->b = b0 + l;
            out->tile = __builtin_amdgcn_readlane(upto, l) - 1 - tau;
            return true;
        }
        tau -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

template <int CACHE, int T, int DIM, int NQ>
__global__ void __launch_bounds__(256, prompt_occupancy(CACHE, T, DIM)) prompt_attention(PagedArgs a)
{
    constexpr int BM = 128 * NQ;
    constexpr int RB = bytes_of(CACHE, DIM);
    constexpr bool CODED = row_scaled(CACHE), SIXTEEN = CACHE == F16 || CACHE == BF16;
    constexpr bool KF = keys_f16(CACHE, T), VF = CACHE == F16;
    constexpr int QT = q_terms(CACHE, T), PT = prompt_p_terms(CACHE, T);
    constexpr float BIAS = VF ? 7.0f : 0.0f;
    constexpr int PR = DIM / 8;                // 16-byte pieces of a row in LDS
    constexpr int STEPS = DIM / 16, DB = DIM / 32;
    constexpr int KT = prompt_keys(CACHE, T, DIM), NU = KT / 32, NB = KT / 16;   // a tile's tokens, blocks of 32 and of 16

    __shared__ u32x4 tiles[2][2][KT * PR];  // [stage][keys, values][row][piece]
    __shared__ float scales[CODED ? 2 : 1][2][KT];
    __shared__ int spans[2][4];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 31, g = lane >> 5;

    const uint32_t per_split = (uint32_t)a.head_tiles * a.kv_heads;
    const int split = blockIdx.x / per_split;
    const uint32_t in_split = blockIdx.x - split * per_split;
    const int kvh = in_split % (uint32_t)a.kv_heads;
    RowTile rt;
    if (!row_tile<BM>(a, in_split / (uint32_t)a.kv_heads, &rt)) return;
    const int b = __builtin_amdgcn_readfirstlane(rt.b);
    const NewTokens news = new_tokens(a.rules, b);
    const int* const pages = a.pages + (size_t)b * a.ld_pages;
    const int len = min(max(a.lens[b], 0), a.max_len);
    const int heads = a.kv_heads * a.group;

    // this lane's rows, one a block
    bool ok[NQ];
    int token[NQ], head[NQ];
    RowRange see[NQ];
    float slope2[NQ];
    uint32_t lo0 = 0x7fffffffu, hi0 = 0, lo1 = 0, hi1 = 0x7fffffffu;    // any row's, and all rows', of the wave
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        const uint32_t r = (uint32_t)__builtin_amdgcn_readfirstlane(rt.tile) * BM + (wave * NQ + j) * 32 + n;
        const int i = r / (uint32_t)a.group;
        ok[j] = i < news.count;
        head[j] = kvh * a.group + (int)(r - (uint32_t)i * a.group);
        token[j] = news.row + (ok[j] ? i : 0);
        see[j] = range_of(a.rules, len, news.count, ok[j] ? i : 0, token[j], a.window);
        slope2[j] = a.rules.slopes ? a.rules.slopes[head[j]] * 1.4426950408889634f : 0.0f;
        if (ok[j]) {
            if (see[j].lo < see[j].hi) {
                lo0 = min(lo0, (uint32_t)see[j].lo);
                hi0 = max(hi0, (uint32_t)see[j].hi);
            }
            lo1 = max(lo1, (uint32_t)see[j].lo);
            hi1 = min(hi1, (uint32_t)see[j].hi);
        }
    }
    lo0 = 0x7fffffffu - max_over<32>(0x7fffffffu - lo0);
    hi0 = max_over<32>(hi0);
    lo1 = max_over<32>(lo1);
    hi1 = 0x7fffffffu - max_over<32>(0x7fffffffu - hi1);
    const int wave_lo = __builtin_amdgcn_readfirstlane(lo0), wave_hi = __builtin_amdgcn_readfirstlane(hi0);
    const int all_lo = __builtin_amdgcn_readfirstlane(lo1), all_hi = __builtin_amdgcn_readfirstlane(hi1);
    if (lane == 0) { spans[0][wave] = wave_lo; spans[1][wave] = wave_hi; }
    __syncthreads();
    int first = min(min(spans[0][0], spans[0][1]), min(spans[0][2], spans[0][3]));
    int last = max(max(spans[1][0], spans[1][1]), max(spans[1][2], spans[1][3]));
    first = __builtin_amdgcn_readfirstlane(last ? first : 0);
    last = __builtin_amdgcn_readfirstlane(last);
    const int base = first & ~(KT - 1);
    const long long from = base + (long long)split * a.chunk;
    const int begin = from < last ? (int)from : last;
    const int end = min((long long)last, from + a.chunk);

    // queries: lane (n, g) holds elements 16 c + 8 g .. of row n
    u32x4 qf[NQ][QT][STEPS];
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int c = 0; c < STEPS; ++c) {
            const char* p = a.q + (size_t)token[j] * a.ldq + ((size_t)head[j] * DIM + 16 * c + 8 * g) * size_of(T);
            if constexpr (T == F32) {
                float x[8];
                load8<T>(p, x);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    uint32_t w[3];
                    cut_pair(x[2 * d], x[2 * d + 1], w);
#pragma unroll
                    for (int i = 0; i < 3; ++i) qf[j][i][c][d] = w[i];
                }
            } else if constexpr (QT == 2) {
                float x[8];
                load8<T>(p, x);
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    uint32_t w[2];
                    split_pair<false, 2>(x[2 * d], x[2 * d + 1], w);
                    qf[j][0][c][d] = w[0];
                    qf[j][1][c][d] = w[1];
                }
            } else {
                qf[j][0][c] = *reinterpret_cast<const u32x4*>(p);
            }
        }

    // ---- staging ----
    // The tile's blocks of 16 tokens lie in one page each.  Rows outside of [begin or first, end) are
    // copies of the nearest row inside, so that what lies there enters nothing, and an
    // absent page's are slot 0's: both are masked.
    const int lo_row = max(first, begin), page_mask = (1 << a.page_shift) - 1;
    // All are worked out at once, one a lane, from pages that were asked for a tile before.
    struct Blocks { size_t mine, off[NB]; uint32_t present; };      // bytes into the cache's arrays
    const size_t page_bytes = ((size_t)a.kv_heads << a.page_shift) * RB, head_bytes = ((size_t)kvh << a.page_shift) * RB;
    auto block_at = [&](int t0, int j) { return 16 * min(max((t0 >> 4) + j, lo_row >> 4), (end - 1) >> 4); };
    auto pages_of = [&](int t0) { return pages[block_at(t0, lane % NB) >> a.page_shift]; };
    auto blocks = [&](int t0, int ids) {
        const bool there = (uint32_t)ids < (uint32_t)a.n_pages;
        const size_t off = (there ? (uint32_t)ids * page_bytes + head_bytes : 0) +
                           (uint32_t)(block_at(t0, lane % NB) & page_mask) * (uint32_t)RB;
        Blocks s;
        s.mine = off;
        s.present = (uint32_t)__ballot(there) & ((1u << NB) - 1);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            s.off[j] = (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), j) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)off, j);
        return s;
    };
    auto inside = [&](int t0) { return t0 >= lo_row && t0 + KT <= end; };
    const uint32_t lds0 = (uint32_t)(size_t)(__attribute__((address_space(3))) char*)(char*)&tiles[0][0][0];
    // slot of a row's piece
    auto slot_k = [](int row, int piece) { return PR == 8 ? piece ^ ((row >> 1) & 7) : piece ^ (row & 15); };
    auto slot_v = [](int row, int piece) { return PR == 8 ? piece ^ (4 * ((row >> 1) & 1)) : piece ^ (4 * (row & 3)); };

    // loads in registers on their way to LDS, of the caches that hold codes
    constexpr int CP = RB / 16;                // 16-byte pieces of a row in the cache
    constexpr int LOADS = SIXTEEN ? 1 : (KT * CP + 255) / 256;
    u32x4 raw[2][LOADS];
    uint32_t unit[2][LOADS];
    // a thread's row scale: keys' of waves 0 (and 1), values' of the others; rows of short tiles are taken twice
    float row_scale = 0.0f;
    const int scale_side = KT > 64 ? wave >> 1 : wave & 1;
    constexpr int RPC = SIXTEEN ? 64 / PR : 1;     // rows of a wave's 1 KB
    // a tile at t0, all of it within the rows that count (WHOLE) or not, on its way to a stage
    auto pick = [](const Blocks& s, int blk) {
        return (size_t)(uint32_t)__shfl((int)(s.mine >> 32), blk) << 32 | (uint32_t)__shfl((int)s.mine, blk);
    };
    auto fetch_as = [&](auto whole, const Blocks& s, int t0, int stage) {
        constexpr bool WHOLE = decltype(whole)::value;
        if constexpr (SIXTEEN) {
#pragma unroll
            for (int i = 0; i < KT / RPC / 4; ++i) {
                // its block: i, i / 2, or 2 i and 2 i + 1 for two waves each
                const int blk = PR == 16 ? i : PR == 32 ? i / 2 : 2 * i + (wave >> 1);
                const size_t off = PR == 8 ? (wave >= 2 ? s.off[(2 * i + 1) % NB] : s.off[2 * i % NB]) : s.off[blk % NB];
                const int row = (4 * i + wave) * RPC + lane / PR;
                int t = row % 16;
                if constexpr (!WHOLE) {
                    const int at = block_at(t0, blk);
                    t = min(max(at + t, lo_row), end - 1) - at;
                }
                const uint32_t lds = lds0 + (stage * 2 * KT * PR + (4 * i + wave) * 64) * 16;
                cache_to_lds(lds, a.k + off, t * RB + 16 * slot_k(row, lane % PR));
                cache_to_lds(lds + KT * PR * 16, a.v + off, t * RB + 16 * slot_v(row, lane % PR));
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = threadIdx.x + 256 * i, row = p / CP % KT;
                // a wave's rows are of one block, or of several whose rows are picked by lane
                const int blk = row / 16;
                const size_t off = pick(s, blk);
                int t = row % 16;
                if constexpr (!WHOLE) {
                    const int at = block_at(t0, blk);
                    t = min(max(at + t, lo_row), end - 1) - at;
                }
                const size_t b = off + t * RB + 16 * (p % CP);
                raw[0][i] = *reinterpret_cast<const u32x4*>(a.k + b);
                raw[1][i] = *reinterpret_cast<const u32x4*>(a.v + b);
                if constexpr (CACHE == E2M1) {     // a byte for each 16
                    unit[0][i] = reinterpret_cast<const uint8_t*>(a.k_scale)[b / 16];
                    unit[1][i] = reinterpret_cast<const uint8_t*>(a.v_scale)[b / 16];
                }
            }
            if constexpr (CODED) {
                const int row = lane % KT + (KT > 64 ? 64 * (wave & 1) : 0), blk = row / 16;
                const size_t off = pick(s, blk);
                int t = row % 16;
                if constexpr (!WHOLE) {
                    const int at = block_at(t0, blk);
                    t = min(max(at + t, lo_row), end - 1) - at;
                }
                const size_t r = off / RB + t;
                row_scale = (scale_side ? a.v_scale : a.k_scale)[r];
            }
        }
    };
    auto fetch = [&](const Blocks& s, int t0, int stage) {
        if (inside(t0)) fetch_as(std::true_type{}, s, t0, stage);
        else fetch_as(std::false_type{}, s, t0, stage);
    };
    auto put = [&](int stage) {
        if constexpr (!SIXTEEN) {
            u32x4* const k = tiles[stage][0];
            u32x4* const v = tiles[stage][1];
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = threadIdx.x + 256 * i, row = p / CP;
                if (LOADS * 256 > KT * CP && row >= KT) break;
                if constexpr (CACHE == E2M1) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        k[row * PR + slot_k(row, 4 * (p % CP) + d)] = bf16_of_e2m1(raw[0][i][d], unit[0][i]);
                        v[row * PR + slot_v(row, 4 * (p % CP) + d)] = bf16_of_e2m1(raw[1][i][d], unit[1][i]);
                    }
                } else if constexpr (CODED) {
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const u32x2 k0 = codes_16<CACHE, KF>(raw[0][i][2 * d]), k1 = codes_16<CACHE, KF>(raw[0][i][2 * d + 1]);
                        const u32x2 v0 = codes_16<CACHE, VF>(raw[1][i][2 * d]), v1 = codes_16<CACHE, VF>(raw[1][i][2 * d + 1]);
                        k[row * PR + slot_k(row, 2 * (p % CP) + d)] = (u32x4){k0[0], k0[1], k1[0], k1[1]};
                        v[row * PR + slot_v(row, 2 * (p % CP) + d)] = (u32x4){v0[0], v0[1], v1[0], v1[1]};
                    }
                }
            }
            if constexpr (CODED)
                scales[stage][scale_side][lane % KT + (KT > 64 ? 64 * (wave & 1) : 0)] = row_scale;
        }
    };

    float m[NQ], l[NQ];
    f32x16 acc[NQ][DB];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        m[j] = -FLT_MAX;
        l[j] = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[j][d][i] = 0.0f;
    }
    const bool plain = a.rules.cap2 == 0.0f && !a.rules.slopes && a.scale2 > 0.0f;
    // this lane's part of a transposed read: row lane / 4 % 4 of 4, elements 4 (lane % 4).. of 16
    const int vrow = (lane >> 2) & 3;
    uint32_t v_off[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        const int piece = 4 * d + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        v_off[d] = (4 * g + vrow) * (PR * 16) + 16 * slot_v(vrow, piece) + 8 * (lane & 1);
    }

    // Accumulators of more than half the registers stay in the matrix cores' half.
    auto pin = [&] {
        if constexpr (DIM == 256)
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int d = 0; d < DB; ++d) __asm__ volatile("" : "+a"(acc[j][d]));
    };
    auto compute = [&](int t0, auto at, uint32_t present) {
        pin();
        constexpr int stage = decltype(at)::value;
        const u32x4* const k = tiles[stage][0];
        f32x16 s[NU][NQ];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[u][j][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
                const int row = 32 * u + n;
                const u32x4 f = k[row * PR + slot_k(row, 2 * c + g)];
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int i = QT - 1; i >= 0; --i) s[u][j] = mfma32<KF>(f, qf[j][i][c], s[u][j]);
            }
        }
        // register i of block u is token 32 u + 8 (i / 4) + 4 g + i % 4
        float scale = a.scale2;
        if constexpr (CODED) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const f32x4 ks = *reinterpret_cast<const f32x4*>(&scales[stage][0][32 * u + 2 * i + 4 * g]);
#pragma unroll
                    for (int j = 0; j < NQ; ++j)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[u][j][i + r] = __fmul_rn(s[u][j][i + r], ks[r]);
                }
        }
        if (!plain) {
            scale = 1.0f;
            if (a.rules.cap2 != 0.0f) {
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[u][j][i] = capped<T>(a.rules, s[u][j][i]);
            } else {
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[u][j][i] = __fmul_rn(s[u][j][i], a.scale2);
            }
            if (a.rules.slopes) {
#pragma unroll
                for (int j = 0; j < NQ; ++j) {
                    const float ahead = (float)(see[j].p - t0 - 4 * g);
#pragma unroll
                    for (int u = 0; u < NU; ++u)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            s[u][j][i] = __builtin_fmaf(-slope2[j], fabsf(__fsub_rn(ahead, (float)(32 * u + 8 * (i / 4) + i % 4))),
                                                        s[u][j][i]);
                }
            }
        }
        const bool whole = present == (1u << NB) - 1 && t0 >= max(all_lo, begin) && t0 + KT <= min(all_hi, end);
        if (!whole) {
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                const int from = max(see[j].lo, begin) - t0 - 4 * g, to = min(see[j].hi, end) - t0 - 4 * g;
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int t = 32 * u + 8 * (i / 4) + i % 4;
                        const bool in = t >= from && t < to && (present >> ((32 * u + 2 * i) / 16) & 1);
                        s[u][j][i] = in ? s[u][j][i] : -__builtin_inff();
                    }
            }
        }
        u32x4 pf[NQ][PT][NB];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
            float top = s[0][j][0];
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[u][j][i]);
            top = __fmul_rn(top, scale);
            if (__any(top > m[j] + 8.0f)) {
                top = fmaxf(top, __shfl_xor(top, 32));
                const float mn = fmaxf(m[j], top), f = __builtin_amdgcn_exp2f(m[j] - mn);
                m[j] = mn;
                l[j] = __fmul_rn(l[j], f);
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[j][d][i] = __fmul_rn(acc[j][d][i], f);
            }
            __builtin_amdgcn_s_setprio(1);
            pin();
            const float off = BIAS - m[j];
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float w[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][j][i + r], scale, off));
                        l[j] = __fadd_rn(l[j], w[r]);
                    }
                    if constexpr (CODED) {
                        const float* const vs = &scales[stage][1][32 * u + 8 * (i / 4) + 4 * g + i % 4];
                        w[0] = __fmul_rn(w[0], vs[0]);
                        w[1] = __fmul_rn(w[1], vs[1]);
                    }
                    uint32_t t[PT];
                    split_pair<VF, PT>(w[0], w[1], t);
#pragma unroll
                    for (int x = 0; x < PT; ++x) pf[j][x][2 * u + i / 8][i % 8 / 2] = t[x];
                }
        }
        // k index 8 g + i of step c is token 16 c + 8 (i / 4) + 4 g + i % 4
        const uint32_t vbase = lds0 + (stage * 2 + 1) * KT * PR * 16;
#pragma unroll
        for (int c = 0; c < NB; ++c) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                u32x4 f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4*)(size_t)(vbase + v_off[d] + (16 * c + 8 * h) * PR * 16));
                    const u32x2 w = __builtin_bit_cast(u32x2, x);
                    f[2 * h] = w[0];
                    f[2 * h + 1] = w[1];
                }
#pragma unroll
                for (int j = 0; j < NQ; ++j)
#pragma unroll
                    for (int x = PT - 1; x >= 0; --x) acc[j][d] = mfma32<VF>(f, pf[j][x][c], acc[j][d]);
            }
        }
    };

    auto arrived = [] {
        __builtin_amdgcn_s_setprio(0);
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);        // vmcnt and lgkmcnt 0, and the compiler knows it
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");         // nothing of the new stage is read before
    };
    // Two tiles a turn, so that their stages are constants.
    if (begin < end) {
        int t = begin & ~(KT - 1), ids = pages_of(t + KT);
        const Blocks s = blocks(t, pages_of(t));
        fetch(s, t, 0);
        put(0);
        uint32_t present = s.present;
        arrived();
        auto step = [&](auto at) {
            constexpr int stage = decltype(at)::value;
            const bool more = t + KT < end;
            uint32_t next = 0;
            if (more) {
                const Blocks s1 = blocks(t + KT, ids);
                ids = pages_of(t + 2 * KT);
                next = s1.present;
                fetch(s1, t + KT, stage ^ 1);
            }
            if (t < wave_hi && t + KT > wave_lo) compute(t, at, present);
            if (!more) return false;
            put(stage ^ 1);
            arrived();
            present = next;
            t += KT;
            return true;
        };
#pragma unroll 1
        while (step(std::integral_constant<int, 0>{}) && step(std::integral_constant<int, 1>{})) {}
    }

    // sums that have left the range, or a NaN: the workgroup's rows again, one by one
    bool careful = false;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        float size = 0.0f;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) size = __fadd_rn(size, fabsf(acc[j][d][i]));
        careful |= !(size < 0x1p100f);
        l[j] = __fadd_rn(l[j], __shfl_xor(l[j], 32));
    }
    careful = __any(careful);
    if (careful) {
        const CacheView view{a.k, a.v, a.k_scale, a.v_scale, pages, a.n_pages, a.page_shift, a.kv_heads, kvh};
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
#pragma unroll 1
            for (int c = 0; c < 32; ++c) {
                if (!__builtin_amdgcn_readlane((int)ok[j], c)) break;          // rows behind the last
                const int h = __builtin_amdgcn_readlane(head[j], c), q = __builtin_amdgcn_readlane(token[j], c);
                const RowRange r{max(__builtin_amdgcn_readlane(see[j].lo, c), begin),
                                 min(__builtin_amdgcn_readlane(see[j].hi, c), end), __builtin_amdgcn_readlane(see[j].p, c)};
                const float slope = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(slope2[j]), c));
                const size_t at = (size_t)q * heads + h;
                careful_row<CACHE, T, DIM>(view, a.rules, a.q + (size_t)q * a.ldq + (size_t)h * DIM * size_of(T), r, a.scale2,
                                           slope, a.splits == 1 ? a.out + (size_t)q * a.ldo + (size_t)h * DIM * size_of(T) : nullptr,
                                           a.lse ? a.lse + (size_t)q * heads + h : nullptr,
                                           a.part + (at * a.splits + split) * DIM, a.ml + (at * a.splits + split) * 2);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
        if (!ok[j]) continue;
        const size_t row = (size_t)token[j] * heads + head[j];
        const bool direct = a.splits == 1;
        const float inv = l[j] == 0.0f ? 0.0f : __fdiv_rn(1.0f, l[j]);
        char* const out = a.out + (size_t)token[j] * a.ldo + (size_t)head[j] * DIM * size_of(T);
        float* const part = a.part + (row * a.splits + split) * DIM;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int el = 32 * d + 2 * i + 4 * g;
                f32x4 o = (f32x4){acc[j][d][i], acc[j][d][i + 1], acc[j][d][i + 2], acc[j][d][i + 3]};
                if (direct) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[r] = l[j] == 0.0f ? 0.0f : __fmul_rn(o[r], inv);
                    if constexpr (T == F32) *reinterpret_cast<f32x4*>(out + 4 * el) = o;
                    else
                        *reinterpret_cast<u32x2*>(out + 2 * el) = T == F16 ? (u32x2){pack_f16(o[0], o[1]), pack_f16(o[2], o[3])}
                                                                           : (u32x2){pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
                } else if (l[j] != 0.0f) {
                    *reinterpret_cast<f32x4*>(part + el) = o;
                }
            }
        if (g == 0) {
            if (!direct) {
                a.ml[(row * a.splits + split) * 2] = m[j] - BIAS;
                a.ml[(row * a.splits + split) * 2 + 1] = l[j];
            } else if (a.lse) {
                a.lse[(size_t)token[j] * heads + head[j]] =
                    l[j] == 0.0f ? -__builtin_inff()
                                 : __fmul_rn(__fadd_rn(m[j] - BIAS, __builtin_amdgcn_logf(l[j])), 0.69314718055994531f);
            }
        }
    }
}

// Row tiles of BM packed rows.
constexpr int prompt_rows(int cache, int t, int dim) { return 128 * prompt_blocks(cache, t, dim); }

hipError_t launch_prompt_f16(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_bf16(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_i8(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_e4m3(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_e2m1(int t, int dim, const PagedArgs& a, dim3 grid, hipStream_t s);

template <int CACHE, int T, int DIM>
hipError_t launch_prompt_as(const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return launch(prompt_attention<CACHE, T, DIM, prompt_blocks(CACHE, T, DIM)>, grid, dim3(256), 0, s, a);
}
template <int CACHE, int T>
hipError_t launch_prompt(int dim, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return dim == 64    ? launch_prompt_as<CACHE, T, 64>(a, grid, s)
           : dim == 128 ? launch_prompt_as<CACHE, T, 128>(a, grid, s)
                        : launch_prompt_as<CACHE, T, 256>(a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
