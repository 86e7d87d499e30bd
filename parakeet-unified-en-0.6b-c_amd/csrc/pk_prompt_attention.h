// pk_prompt_attention.h - attention of many new tokens per sequence over a paged
// key-value cache: the kernel, instantiated per cache type by pk_prompt_attention_*.hip.
//
// For each row, a (new token, query head) pair, over the tokens [lo, hi) that it sees,
//   s_t = cap tanh(scale q.k_t / cap) - slope |p - t|,  o = sum_t e^(s_t) v_t / sum_t e^(s_t)
// in one pass: a running maximum m, l = sum 2^(s - m) and acc = sum 2^(s - m) v, with s in
// powers of two.  m moves, and acc and l are scaled, only once a score is 8 above it, which
// most tiles of tokens spare; weights stay below 2^8 (times 2^BIAS over f16 values).
//
// A workgroup holds kPromptRows rows of one key-value head, the rows of its query heads
// next to each other, so a group's heads share what it stages: tiles of prompt_keys
// tokens, keys and values, in 16 bits, two stages in LDS.  16-bit caches go there past the
// registers, codes through a conversion; a tile's loads are out while the one before is
// multiplied.  Row scales of 8-bit codes are taken on scores and weights.
//   S^T = K Q^T: a lane gets scores of one row, so the row's statistics are its registers'
//     but for one or three exchanges, and its scores are, in order, the second operand of
//   O^T = V^T P^T: weights go from register to register, never through LDS.  V^T comes from
//     LDS by transposing reads.
// With two sides two waves have the same 32 rows and half of each tile's tokens each, so a
// workgroup is through its tokens sooner: launches that do not fill the card many times over are
// as long as their longest workgroup.  Their sums are joined in LDS at the end.
// Pieces of 16 bytes are XORed with their row, such that the 16 lanes that read at a time
// meet all banks.
//
// Roundings.  The first product is exact but for fp32 sums: codes and 16-bit elements are
// held as they are, and so are bf16 and f16 queries, in their own type (f16 ones over 4 bits as
// 2 bf16 terms); f32 ones are 3 bf16 terms (24 bits).  Weights are rounded for the second
// product: into one term for bf16 queries (8 bits) and for f16 over f16 (11, scaled by 2^7 so that
// weights above 2^-21 are normal numbers), as the output is itself.  Each weight w is off by half a
// step relative to it, so the output by half a step of sum w |v| / l at the worst: as much as its
// own rounding where values have one sign, more where they cancel, less where many tokens' errors
// are independent; l sums the unrounded.  f16 queries over codes take 2 terms (16 bits), f32 3.
// More terms are more products: 4096 tokens of 32 heads of 128 take 141 us with one for
// each, 341 with f32's 3 by 3.
//
// What bounds it: 8192 tokens of 32 heads over 8 of 128 in bf16 take 504 to 511 us, 1080 of the
// 1267 TFLOP/s that a product of two 8192 x 8192 matrices reaches here; both are held by the
// clock, which matrix instructions bring down to some 1.8 GHz.  Blocks of 32x32 halve the
// reads of LDS for a row against 16x16.  Heads of 256 do not leave the registers for them:
// each wave reads a tile for 16 rows, which keeps LDS busier than the matrix cores (4096
// tokens of 16 heads in bf16 149 us, 920 TFLOP/s; 4 bits, through a conversion, 161).
// Heads of 64 do half the products per score, so the exponentials and their like count as
// much as they (168 us, 820 TFLOP/s), and a cap adds 2 transcendental instructions to one (128:
// 141 us, 174 capped).
#pragma once

#include "pk_paged_attention.h"

namespace pkgpu {
namespace decode {

using f32x16 = __attribute__((ext_vector_type(16))) float;
using s16x4 = __attribute__((ext_vector_type(4))) short;

constexpr int prompt_p_terms(int cache, int t) { return t == F32 ? 3 : t == F16 && cache != F16 ? 2 : 1; }
// Rows of a wave, its matrix instructions' (32x32x16 or 16x16x32), waves of a workgroup, and
// its rows.  With two sides (heads of 64 and 128) two waves have the same rows and half of each
// tile's tokens each, and join their sums at the end.
constexpr int prompt_block(int dim) { return dim == 256 ? 16 : 32; }
constexpr int prompt_waves(int dim, int sides) { return dim == 256 ? 8 : 4 * sides; }
constexpr int kPromptRows = 128;
// Tokens of a tile: 64, whose two stages take 32 to 128 KB.  4-bit heads of 64 would leave half
// the threads without a piece to convert (4096 tokens of 64 heads 184 us, of 128 tokens 167).
constexpr int prompt_keys(int cache, int dim) { return dim == 64 && cache == E2M1 ? 128 : 64; }
// Which of them there are (prompt_sides in pk_prompt_attention.hip says which a call takes): heads
// of 256 have no registers for two, 4-bit heads of 64 spill with two at the occupancy that
// pays, and f32 queries in 3 terms over heads of 128 are better by two always (one spills).
constexpr bool has_sides(int cache, int t, int dim, int sides)
{
    return dim == 256 || (dim == 64 && cache == E2M1)      ? sides == 1
           : dim == 128 && t == F32 && cache != E2M1 ? sides == 2 : true;
}
// Waves of a SIMD, and so workgroups that run at a time: as many as the registers take.
// Heads of 64 leave room for three (bf16 over int8 214 against 236) or four by two sides.
constexpr int prompt_occupancy(int cache, int t, int dim, int sides)
{
    return dim != 64 || t == F32 || cache == E2M1 ? 2 : sides == 2 ? 4 : 3;
}
constexpr int prompt_slots(int cache, int t, int dim, int sides)
{
    return 256 * 4 * prompt_occupancy(cache, t, dim, sides) / prompt_waves(dim, sides);
}

template <bool IN_F16>
__device__ inline f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c)
{
    if constexpr (IN_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Words d ^ turn of x.
__device__ inline u32x4 turned_words(u32x4 x, int turn)
{
    x = turn & 1 ? (u32x4){x[1], x[0], x[3], x[2]} : x;
    return turn & 2 ? (u32x4){x[2], x[3], x[0], x[1]} : x;
}

// 16 bytes a lane from base + off to LDS at lds + 16 * lane, past the registers.  The
// compiler does not see it: whoever reads waits for vmcnt(0) first.
__device__ inline void cache_to_lds(uint32_t lds, const char* base, uint32_t off)
{
    __asm__ volatile("s_mov_b32 m0, %0\n\t"
                     "s_nop 0\n\t"
                     "global_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory", "m0");
}

// The sequence and row tile of the launch's tau-th row tile, false where there is none: tiles of BM
// rows, sequence by sequence, so that workgroups that run together read the same tokens, a
// sequence's last ones (whose rows see most) first.  Either every sequence has per_seq of them, or
// as many as its rows take: for up to 64 sequences a sum over the lanes; beyond, sequence b has
// those from floor(S_b / BM) + b on, with S_b the rows before it, which is never fewer than they
// take and can be searched 64 sequences at a time.  Measured (us): 4000 sequences of up to 100
// rows 233 searched, 577 summed; 8 of up to 2000, where a workgroup without rows may
// cost another round, 209 summed and 207 to 223 searched.
struct RowTile { int b, tile; };
template <int BM>
__device__ inline bool row_tile(const PagedArgs& a, uint32_t tau, RowTile* out)
{
    const int lane = threadIdx.x & 63;
    auto tiles_of = [&](int b) { return (int)(((long long)new_tokens(a.rules, b).count * a.group + BM - 1) / BM); };
    uint32_t nth;
    if (a.rules.per_seq) {
        out->b = tau / (uint32_t)a.rules.per_seq;
        nth = tau - (uint32_t)out->b * a.rules.per_seq;
    } else if (a.B <= 64) {
        const int mine = lane < a.B ? tiles_of(lane) : 0;
        uint32_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_up(upto, d);
            upto += lane >= d ? o : 0;
        }
        const unsigned long long behind = __ballot(upto > tau);
        if (!behind) return false;
        out->b = __builtin_ctzll(behind);
        out->tile = __builtin_amdgcn_readlane((int)upto, out->b) - 1 - (int)tau;
        return true;
    } else {
        auto tiles_before = [&](int b) {
            const int s = a.rules.starts ? min(max(a.rules.starts[b], 0), a.rules.rows) : min(b, a.rules.rows);
            return (uint32_t)((unsigned long long)s * (uint32_t)a.group / BM) + (uint32_t)b;
        };
        int lo = 0, n = a.B;
        uint32_t before;
        do {
            const int step = (n + 63) / 64, at = lane * step;
            const uint32_t t = at < n ? tiles_before(lo + at) : 0xffffffffu;
            const unsigned long long upto = __ballot(t <= tau);
            if (!upto) return false;
            const int l = 63 - __builtin_clzll(upto);
            before = __builtin_amdgcn_readlane((int)t, l);
            lo += l * step;
            n = min(step, n - l * step);
        } while (n > 1);
        out->b = lo;
        nth = tau - before;
    }
    const int n = tiles_of(out->b);
    out->tile = n - 1 - (int)nth;
    return nth < (uint32_t)n;
}

template <int CACHE, int T, int DIM, int SIDES>
__global__ void __launch_bounds__(64 * prompt_waves(DIM, SIDES), prompt_occupancy(CACHE, T, DIM, SIDES)) prompt_attention(PagedArgs a)
{
    constexpr int R = prompt_block(DIM), W = prompt_waves(DIM, SIDES), THREADS = 64 * W;
    constexpr int WR = W / SIDES, BM = kPromptRows;
    static_assert(BM == R * WR, "rows of a workgroup");
    constexpr int NR = R * R / 64;             // registers of a block of sums
    using Sums = __attribute__((ext_vector_type(NR))) float;
    constexpr int RB = bytes_of(CACHE, DIM);
    constexpr bool CODED = row_scaled(CACHE), SIXTEEN = CACHE == F16 || CACHE == BF16;
    constexpr bool KF = keys_f16(CACHE, T), VF = CACHE == F16;
    constexpr int QT = q_terms(CACHE, T), PT = prompt_p_terms(CACHE, T);
    constexpr float BIAS = VF ? 7.0f : 0.0f;
    constexpr int PR = DIM / 8;                // 16-byte pieces of a row in LDS
    constexpr int KS = 512 / R;                // of a matrix instruction's sum
    constexpr int STEPS = DIM / KS, DB = DIM / R;
    constexpr int KT = prompt_keys(CACHE, DIM), NB = KT / 16;
    constexpr int KW = KT / SIDES, NU = KW / R, NS = KW / KS;      // tokens of a wave's part of a tile

    __shared__ u32x4 tiles[2][2][KT * PR];     // [stage][keys, values][row][piece]
    __shared__ float scales[CODED ? 2 : 1][2][KT];
    __shared__ int spans[2][W];

    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane % R, g = lane / R;
    const int side = SIDES == 1 ? 0 : wave / WR, in_side = SIDES == 1 ? wave : wave % WR;

    const uint32_t per_split = (uint32_t)a.head_tiles * a.kv_heads;
    const int split = blockIdx.x / per_split;
    const uint32_t in_split = blockIdx.x - split * per_split;
    const int kvh = in_split % (uint32_t)a.kv_heads;
    RowTile rt;
    if (!row_tile<BM>(a, in_split / (uint32_t)a.kv_heads, &rt)) return;
    const int b = rt.b;
    const NewTokens news = new_tokens(a.rules, b);
    const int* const pages = a.pages + (size_t)b * a.ld_pages;
    const int len = min(max(a.lens[b], 0), a.max_len);
    const int heads = a.kv_heads * a.group;

    // this lane's row
    const uint32_t r = (uint32_t)rt.tile * BM + in_side * R + n;
    const int nth = r / (uint32_t)a.group;
    const bool ok = nth < news.count;
    const int head = kvh * a.group + (int)(r - (uint32_t)nth * a.group);
    const int token = news.row + (ok ? nth : 0);
    const RowRange see = range_of(a.rules, len, news.count, ok ? nth : 0, token, a.window);
    const float slope2 = slope_of(a.rules, head);
    // tokens that any row of the wave sees, and that all do
    const bool sees = ok && see.lo < see.hi;
    const int wave_lo = (int)(0x7fffffffu - max_over<R>(sees ? 0x7fffffffu - (uint32_t)see.lo : 0u));
    const int wave_hi = (int)max_over<R>(sees ? (uint32_t)see.hi : 0u);
    const int all_lo = __builtin_amdgcn_readfirstlane((int)max_over<R>(ok ? (uint32_t)see.lo : 0u));
    const int all_hi = __builtin_amdgcn_readfirstlane((int)(0x7fffffffu - max_over<R>(ok ? 0x7fffffffu - (uint32_t)see.hi : 0u)));
    if (lane == 0) { spans[0][wave] = wave_lo; spans[1][wave] = wave_hi; }
    __syncthreads();
    int first = spans[0][0], last = spans[1][0];
#pragma unroll
    for (int w = 1; w < W; ++w) { first = min(first, spans[0][w]); last = max(last, spans[1][w]); }
    first = __builtin_amdgcn_readfirstlane(last ? first : 0);
    last = __builtin_amdgcn_readfirstlane(last);
    const int mine_lo = __builtin_amdgcn_readfirstlane(wave_lo), mine_hi = __builtin_amdgcn_readfirstlane(wave_hi);
    const int base = first & ~(KT - 1);
    const long long from = base + (long long)split * a.chunk;
    const int begin = from < last ? (int)from : last;
    const int end = min((long long)last, from + a.chunk);

    // queries: lane (n, g) holds elements KS c + 8 g .. of row n
    u32x4 qf[QT][STEPS];
#pragma unroll
    for (int c = 0; c < STEPS; ++c) {
        const char* p = a.q + (size_t)token * a.ldq + ((size_t)head * DIM + KS * c + 8 * g) * size_of(T);
        if constexpr (QT == 1) {
            qf[0][c] = *reinterpret_cast<const u32x4*>(p);
        } else {
            float x[8];
            load8<T>(p, x);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint32_t w[QT];
                if constexpr (QT == 3) cut_pair(x[2 * d], x[2 * d + 1], w);
                else split_pair<false, QT>(x[2 * d], x[2 * d + 1], w);
#pragma unroll
                for (int i = 0; i < QT; ++i) qf[i][c][d] = w[i];
            }
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
                           (size_t)(uint32_t)(block_at(t0, lane % NB) & page_mask) * RB;     // a page may pass 4 GiB
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
    auto slot_v = [](int row, int piece) { return R == 16  ? piece ^ (2 * (row & 7))
                                              : PR == 8 ? piece ^ (4 * ((row >> 1) & 1)) : piece ^ (4 * (row & 3)); };

    // loads in registers on their way to LDS, of the caches that hold codes
    constexpr int CP = RB / 16;                // 16-byte pieces of a row in the cache
    constexpr int LOADS = SIXTEEN ? 1 : (KT * CP + THREADS - 1) / THREADS;
    u32x4 raw[2][LOADS];
    uint32_t unit[2][LOADS];
    // row scales, one a lane: keys' of wave 0 (tiles of 128: and 1), values' of the next ones
    float row_scale = 0.0f;
    constexpr int SW = KT / 64;                // waves a side
    const int scale_side = wave / SW, scale_row = 64 * (wave % SW) + lane;
    constexpr int RPC = SIXTEEN ? 64 / PR : 1;     // rows of a wave's 1 KB
    constexpr int PER = PR / 4;                // such of a block
    auto pick = [](const Blocks& s, int blk) {
        return (size_t)(uint32_t)__shfl((int)(s.mine >> 32), blk) << 32 | (uint32_t)__shfl((int)s.mine, blk);
    };
    auto fetch_as = [&](auto whole, const Blocks& s, int t0, int stage) {
        constexpr bool WHOLE = decltype(whole)::value;
        if constexpr (SIXTEEN) {
#pragma unroll
            for (int i = 0; i < KT / RPC / W; ++i) {
                // its block: one for all waves, or W / PER for PER waves each
                constexpr int MANY = W > PER ? W / PER : 1;
                const int blk = W > PER ? MANY * i + wave / PER : W * i / PER;
                const size_t off = W > PER ? (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(s.mine >> 32), blk) << 32 |
                                             (uint32_t)__builtin_amdgcn_readlane((int)s.mine, blk)
                                           : s.off[W * i / PER];
                const int row = (W * i + wave) * RPC + lane / PR;
                int t = row % 16;
                if constexpr (!WHOLE) {
                    const int at = block_at(t0, blk);
                    t = min(max(at + t, lo_row), end - 1) - at;
                }
                const uint32_t lds = lds0 + (stage * 2 * KT * PR + (W * i + wave) * 64) * 16;
                cache_to_lds(lds, a.k + off, t * RB + 16 * slot_k(row, lane % PR));
                cache_to_lds(lds + KT * PR * 16, a.v + off, t * RB + 16 * slot_v(row, lane % PR));
            }
        } else {
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int p = threadIdx.x + THREADS * i, row = p / CP % KT;
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
                const int blk = scale_row / 16;
                const size_t off = pick(s, blk);
                int t = scale_row % 16;
                if constexpr (!WHOLE) {
                    const int at = block_at(t0, blk);
                    t = min(max(at + t, lo_row), end - 1) - at;
                }
                if (wave < 2 * SW) row_scale = (scale_side ? a.v_scale : a.k_scale)[off / RB + t];
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
                const int p = threadIdx.x + THREADS * i, row = p / CP;
                if (LOADS * THREADS > KT * CP && row >= KT) break;
                if constexpr (CACHE == E2M1) {
                    // A lane's 4 pieces lie next to each other, so lanes write theirs in orders of
                    // their own, d ^ turn, that put 16 lanes' into different banks.
                    const int far = PR == 32 ? p % CP >> 2 : 0;
                    const int turn_k = 2 * far, turn_v = PR == 32 ? far : row & 3;
                    const u32x4 xk = turned_words(raw[0][i], turn_k), xv = turned_words(raw[1][i], turn_v);
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        k[row * PR + slot_k(row, 4 * (p % CP) + (d ^ turn_k))] = bf16_of_e2m1(xk[d], unit[0][i]);
                        v[row * PR + slot_v(row, 4 * (p % CP) + (d ^ turn_v))] = bf16_of_e2m1(xv[d], unit[1][i]);
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
                if (wave < 2 * SW) scales[stage][scale_side][scale_row] = row_scale;
        }
    };

    float m = -FLT_MAX, l = 0.0f;
    Sums acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < NR; ++i) acc[d][i] = 0.0f;
    const bool plain = a.rules.cap2 == 0.0f && !a.rules.slopes && a.scale2 > 0.0f;
    auto multiply = [](auto in_f16, u32x4 x, u32x4 y, Sums z) {
        if constexpr (R == 32) return mfma32<decltype(in_f16)::value>(x, y, z);
        else return mfma<decltype(in_f16)::value>(x, y, z);
    };
    const std::integral_constant<bool, KF> keys_type;
    const std::integral_constant<bool, VF> values_type;
    // this lane's part of a transposed read, of 4 rows by 16 elements for 16 lanes: row
    // lane / 4 % 4, elements 4 (lane % 4)..
    const int vrow = 4 * g + ((lane >> 2) & 3);
    uint32_t v_off[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) {
        const int piece = R / 8 * d + (R == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1);
        v_off[d] = vrow * (PR * 16) + 16 * slot_v(vrow, piece) + 8 * (lane & 1);
    }

    auto compute = [&](int t0, auto at, uint32_t present) {
        t0 += KW * side;
        if constexpr (SIDES > 1) present = present >> (KW / 16 * side) & ((1u << KW / 16) - 1);
        constexpr int stage = decltype(at)::value;
        const u32x4* const k = tiles[stage][0];
        Sums s[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
#pragma unroll
            for (int i = 0; i < NR; ++i) s[u][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < STEPS; ++c) {
                const int row = KW * side + R * u + n;
                const u32x4 f = k[row * PR + slot_k(row, KS / 8 * c + g)];
#pragma unroll
                for (int i = QT - 1; i >= 0; --i) s[u] = multiply(keys_type, f, qf[i][c], s[u]);
            }
        }
        // in this order: reads of keys AHEAD steps before their product (0x100: LDS reads, 8: products)
        constexpr int AHEAD = QT == 1 && NU * STEPS >= 8 ? 8 : 4;
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int i = 0; i < NU * STEPS - AHEAD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, QT, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * QT, 0);
        // register i of block u is token R u + 8 (i / 4) + 4 g + i % 4
        float scale = a.scale2;
        if constexpr (CODED) {
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < NR; i += 4) {
                    const f32x4 ks = *reinterpret_cast<const f32x4*>(&scales[stage][0][KW * side + R * u + 2 * i + 4 * g]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) s[u][i + r] = __fmul_rn(s[u][i + r], ks[r]);
                }
        }
        if (!plain) {
            scale = 1.0f;
            if (a.rules.cap2 != 0.0f) {
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int i = 0; i < NR; ++i) s[u][i] = capped<T>(a.rules, s[u][i]);
            } else {
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int i = 0; i < NR; ++i) s[u][i] = __fmul_rn(s[u][i], a.scale2);
            }
            if (a.rules.slopes) {
                const float ahead = (float)(see.p - t0 - 4 * g);
#pragma unroll
                for (int u = 0; u < NU; ++u)
#pragma unroll
                    for (int i = 0; i < NR; ++i)
                        s[u][i] = __builtin_fmaf(-slope2, fabsf(__fsub_rn(ahead, (float)(R * u + 8 * (i / 4) + i % 4))), s[u][i]);
            }
        }
        const bool whole = present == (1u << KW / 16) - 1 && t0 >= max(all_lo, begin) && t0 + KW <= min(all_hi, end);
        if (!whole) {
            const int from = max(see.lo, begin) - t0 - 4 * g, to = min(see.hi, end) - t0 - 4 * g;
#pragma unroll
            for (int u = 0; u < NU; ++u)
#pragma unroll
                for (int i = 0; i < NR; ++i) {
                    const int t = R * u + 8 * (i / 4) + i % 4;
                    const bool in = t >= from && t < to && (present >> ((R * u + 8 * (i / 4)) / 16) & 1);
                    s[u][i] = in ? s[u][i] : -__builtin_inff();
                }
        }
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < NR; ++i) top = fmaxf(top, s[u][i]);
        top = __fmul_rn(top, scale);
        if (__any(top > m + 8.0f)) {
#pragma unroll
            for (int d = 32; d >= R; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
            const float mn = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l = __fmul_rn(l, f);
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < NR; ++i) acc[d][i] = __fmul_rn(acc[d][i], f);
        }
        __builtin_amdgcn_s_setprio(1);
        const float off = BIAS - m;
        u32x4 pf[PT][NS];
#pragma unroll
        for (int u = 0; u < NU; ++u)
#pragma unroll
            for (int i = 0; i < NR; i += 2) {
                float w[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    w[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i + r], scale, off));
                    l = __fadd_rn(l, w[r]);
                }
                if constexpr (CODED) {
                    const float* const vs = &scales[stage][1][KW * side + R * u + 8 * (i / 4) + 4 * g + i % 4];
                    w[0] = __fmul_rn(w[0], vs[0]);
                    w[1] = __fmul_rn(w[1], vs[1]);
                }
                uint32_t t[PT];
                split_pair<VF, PT>(w[0], w[1], t);
#pragma unroll
                for (int x = 0; x < PT; ++x) {
                    if constexpr (R == 32) pf[x][2 * u + i / 8][i % 8 / 2] = t[x];
                    else pf[x][u / 2][2 * (u % 2) + i / 2] = t[x];
                }
            }
        // k index 8 g + i of step c is token KS c + KS / 2 (i / 4) + 4 g + i % 4
        const uint32_t vbase = lds0 + ((stage * 2 + 1) * KT + KW * side) * PR * 16;
#pragma unroll
        for (int c = 0; c < NS; ++c) {
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                u32x4 f;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4*)(size_t)(vbase + v_off[d] + (KS * c + KS / 2 * h) * PR * 16));
                    const u32x2 w = __builtin_bit_cast(u32x2, x);
                    f[2 * h] = w[0];
                    f[2 * h + 1] = w[1];
                }
#pragma unroll
                for (int x = PT - 1; x >= 0; --x) acc[d] = multiply(values_type, f, pf[x][c], acc[d]);
            }
        }
        // values, two reads each, 4 products ahead
        __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
        for (int i = 0; i < NS * DB - 4; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, PT, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4 * PT, 0);
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
            if (t + KW * side < mine_hi && t + KW * side + KW > mine_lo) compute(t, at, present);
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

    // sums that have left the range, or a NaN: the wave's rows again, one by one
#pragma unroll
    for (int d = 32; d >= R; d >>= 1) l = __fadd_rn(l, __shfl_xor(l, d));
    float size = 0.0f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < NR; ++i) size = __fadd_rn(size, fabsf(acc[d][i]));
    if constexpr (SIDES > 1) {
        // the two sides of a block of rows: one leaves its sums in LDS, the other adds them
        static_assert(SIDES == 2 && WR * 64 * DB * NR * 4 <= sizeof(tiles), "sums of half the waves fit");
        __shared__ float others[WR][3][64];
        __syncthreads();                           // the tiles are read
        float* const sums = reinterpret_cast<float*>(&tiles[0][0][0]) + in_side * (64 * DB * NR) + lane;
        if (side) {
            others[in_side][0][lane] = m;
            others[in_side][1][lane] = l;
            others[in_side][2][lane] = size;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < NR; ++i) sums[64 * (NR * d + i)] = acc[d][i];
        }
        __syncthreads();
        if (side) return;
        const float m1 = others[in_side][0][lane], mn = fmaxf(m, m1);
        const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(m1 - mn);
        size = __fadd_rn(size, others[in_side][2][lane]);
        l = __fadd_rn(__fmul_rn(l, f0), __fmul_rn(others[in_side][1][lane], f1));
        m = mn;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int i = 0; i < NR; ++i) acc[d][i] = __fadd_rn(__fmul_rn(acc[d][i], f0), __fmul_rn(sums[64 * (NR * d + i)], f1));
    }
    if (__any(!(size < 0x1p100f))) {
        const CacheView view{a.k, a.v, a.k_scale, a.v_scale, pages, a.n_pages, a.page_shift, a.kv_heads, kvh};
#pragma unroll 1
        for (int c = 0; c < R; ++c) {
            if (!__builtin_amdgcn_readlane((int)ok, c)) break;             // rows behind the last
            const int h = __builtin_amdgcn_readlane(head, c), q = __builtin_amdgcn_readlane(token, c);
            const RowRange r{max(__builtin_amdgcn_readlane(see.lo, c), begin), min(__builtin_amdgcn_readlane(see.hi, c), end),
                             __builtin_amdgcn_readlane(see.p, c)};
            const float slope = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(slope2), c));
            const size_t at = (size_t)q * heads + h;
            careful_row<CACHE, T, DIM>(view, a.rules, a.q + (size_t)q * a.ldq + (size_t)h * DIM * size_of(T), r, a.scale2, slope,
                                       a.splits == 1 ? a.out + (size_t)q * a.ldo + (size_t)h * DIM * size_of(T) : nullptr,
                                       a.lse ? a.lse + at : nullptr, a.part + (at * a.splits + split) * DIM,
                                       a.ml + (at * a.splits + split) * 2);
        }
        return;
    }
    if (!ok) return;
    const size_t row = (size_t)token * heads + head;
    const bool direct = a.splits == 1;
    const float inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
    char* const out = a.out + (size_t)token * a.ldo + (size_t)head * DIM * size_of(T);
    float* const part = a.part + (row * a.splits + split) * DIM;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < NR; i += 4) {
            const int el = R * d + 2 * i + 4 * g;
            f32x4 o = (f32x4){acc[d][i], acc[d][i + 1], acc[d][i + 2], acc[d][i + 3]};
            if (direct) {
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = l == 0.0f ? 0.0f : __fmul_rn(o[r], inv);
                if constexpr (T == F32) *reinterpret_cast<f32x4*>(out + 4 * el) = o;
                else
                    *reinterpret_cast<u32x2*>(out + 2 * el) = T == F16 ? (u32x2){pack_f16(o[0], o[1]), pack_f16(o[2], o[3])}
                                                                       : (u32x2){pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3])};
            } else if (l != 0.0f) {
                *reinterpret_cast<f32x4*>(part + el) = o;
            }
        }
    if (g == 0) {
        if (!direct) {
            a.ml[(row * a.splits + split) * 2] = l == 0.0f ? -__builtin_inff() : m - BIAS;     // without outputs
            a.ml[(row * a.splits + split) * 2 + 1] = l;
        } else if (a.lse) {
            a.lse[row] = l == 0.0f ? -__builtin_inff()
                                   : __fmul_rn(__fadd_rn(m - BIAS, __builtin_amdgcn_logf(l)), 0.69314718055994531f);
        }
    }
}

hipError_t launch_prompt_f16(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_bf16(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_i8(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_e4m3(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s);
hipError_t launch_prompt_e2m1(int t, int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s);

template <int CACHE, int T, int DIM>
hipError_t launch_prompt_as(int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    const dim3 block(64 * prompt_waves(DIM, sides));
    if constexpr (has_sides(CACHE, T, DIM, 2))
        if (sides == 2) return launch(prompt_attention<CACHE, T, DIM, 2>, grid, block, 0, s, a);
    if constexpr (has_sides(CACHE, T, DIM, 1)) return launch(prompt_attention<CACHE, T, DIM, 1>, grid, block, 0, s, a);
    else return hipErrorInvalidValue;
}
template <int CACHE, int T>
hipError_t launch_prompt(int dim, int sides, const PagedArgs& a, dim3 grid, hipStream_t s)
{
    return dim == 64    ? launch_prompt_as<CACHE, T, 64>(sides, a, grid, s)
           : dim == 128 ? launch_prompt_as<CACHE, T, 128>(sides, a, grid, s)
                        : launch_prompt_as<CACHE, T, 256>(sides, a, grid, s);
}

}  // namespace decode
}  // namespace pkgpu
