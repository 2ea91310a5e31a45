// Softmax cross entropy of query rows over a whole catalogue of item rows, and its gradients, without the logits ever being in memory.
//
//   z_rv = s <x_r, e_v> + b_v      lse_r = log sum_v exp z_rv      loss_r = lse_r - z_{r, t_r}      p_rv = exp(z_rv - lse_r)
//   dx_r = s g_r (sum_v p_rv e_v - e_{t_r})      de_v = s sum_r g_r (p_rv - [v = t_r]) x_r      db_v = sum_r g_r (p_rv - [v = t_r])
//
// A row's target stands apart from its other classes throughout, so that a row that has learnt its target (p_t close to 1) keeps its digits:
// with lse' and p' over the classes but the target,  x = lse' - z_t,  loss = log(1 + e^x),  1 - p_t = 1 / (1 + e^-x),
//   dx_r = s g_r (1 - p_t) (sum_{v /= t} p'_v e_v - e_t)        and the target's weight in de is  -g_r (1 - p_t).
//
// Two passes of ONE kernel shape.  A wave keeps 32 "stationary" rows as matrix operands in registers and walks over tiles of "streaming" rows in LDS:
//   S^T = streaming . stationary^T     (a lane holds one stationary row, its 16 registers 16 streaming rows)
//   W   = f(S^T)                       in registers
//   O^T += streaming^T . W             (W is already laid out as the second product's operand; the tile is read transposed from LDS)
// Pass 1: stationary = queries, streaming = catalogue, f = exp with a running maximum: gives lse' and sum_v p'_v e_v, all that dx needs, at once.
// Pass 2: stationary = catalogue, streaming = queries, f = the finished probabilities, the targets' put in: gives de (and db).
// 8 N V d operations in all against 6 N V d with stored logits (4 bytes each way per logit): the recomputed product is cheaper than their traffic.
//
// float32 rows: each value is split into two float16 terms, x 2^e = hi + lo, with one power of two for a whole operand that puts its largest value in
// [2^14, 2^15): 22 bits wherever a value is above 2^-18 of the largest, an absolute error of 2^-40 of it below.  A product then is
// hi hi + hi lo + lo hi on the float16 matrix instructions with float32 sums (the missing lo lo term is below 2^-22): three times the work of a
// 16-bit product, five times faster than the float32 matrix instructions.
#include <algorithm>

#include "head_common.h"
#include "knn_internal.h"   // lds_dma16_v, lds_addr

namespace hwer {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr double kLn2d = 0.6931471805599453;
constexpr float kLowest = -INFINITY;
// The weights are rounded to the rows' 16-bit type for the second product.  bfloat16 has float32's range.  float16 ends at 2^16 above, and below 2^-14
// its steps stay at 2^-24, so float16 weights carry a power of two that uses the range up: pass 1, whose weights may exceed the maximum they are
// taken against by 2^kStale before it is renewed, 2^11 (weights are kept to 2^-36 of a row's largest); pass 2, whose weights are at most 1, 2^15
// (kept to 2^-40).
constexpr float kStale = 4.f;
template <typename E> struct CeType;
template <> struct CeType<f16_t> {
    static constexpr float offset[2] = {11.f, 15.f};
    typedef f16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <> struct CeType<bf16_t> {
    static constexpr float offset[2] = {0.f, 0.f};
    typedef bf16x8 x8;
    static __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};

// device-side scalars of a call (in its workspace)
struct CeScalars {
    int shift_s;                                 // float32 rows: -(eq + ee), -eq as a factor and -ee: they undo the operands' powers of two 2^eq and 2^ee
    float unscale_q, unscale_e;
    float fac_e, fac_b;                          // factors of de (float32 rows: and unscale_q, alone, as both together may leave float32's range) and db
    float g_top;                                 // largest |upstream gradient| of a row
    int counted;                                 // counted rows, of more than kCountedByRow
};

// A sum over the rows: one workgroup walks over up to kSumRows of them, more are summed in kSumParts parts first (1 M rows' losses by one workgroup 0.3 ms).
constexpr int64_t kSumRows = 16384;
constexpr int kSumParts = 256;
struct CeSums {
    double loss[kSumParts];
    float top[kSumParts];
    int counted[kSumParts];
};

struct CePass {
    const short *stat, *stat_lo, *strm, *strm_lo;      // 16-bit terms; rows of DP values (lo: second term of float32 rows)
    int64_t ld_stat, ld_strm, n_stat, n_strm;
    const float* bias;           // per catalogue row
    float scale;
    const CeScalars* sc;
    int subs_per_split, n_splits, stat_blocks;      // a split takes so many times 32 streaming rows
    float *m, *l, *o;            // pass 1: (split, n_stat) maxima and sums, (split, n_stat, DP) weighted sums; pass 2: l, o likewise when split
    const int64_t* target;       // per query its target
    int* counts;                 // pass 1: counted rows of each 32 queries
    const float* loss_rows;      // pass 2, nullable: the queries' losses, reduced by one more workgroup
    const CeSums* sums;          // (nullable: those of more than kSumRows queries are summed in parts)
    float* loss;
    int reduction;
    float* zt;                   // pass 1: per query its target's logit, in the unit of m
    const float* rowp;           // pass 2: four arrays of ld_rowp, per query: what is taken off its logits, factor of its weights, its target's weight, its
    int64_t ld_rowp;             // target (int bits) or -1; rows n_strm .. ld_rowp - 1 have weights of zero
    void* out;                   // pass 2, one split: de in the rows' type, and db
    float* out_b;
    int64_t ld_out;
    int d, out_vec;
};

enum { kLse = 0, kMean = 1, kTable = 2 };

// times 32 streaming rows in an LDS tile: 8 - 32 KB, so that two workgroups (rows of 256: one) fit a CU with four tiles each
template <int TERMS, int DP> constexpr int ce_sub() { return TERMS * DP <= 128 || (TERMS == 1 && DP == 256) ? 2 : 1; }

// Waves of a SIMD that registers are shared out for.  An MFMA occupies its own wave for all its passes, so a wave never overlaps its products with its
// exponentials: only another wave's do.  Rows of 256 need all registers of a SIMD for one wave (128 accumulators, 64 or 128 of stationary rows).
// Tried at 4 096 x 1.25 M x 128 bfloat16: two groups of 4 waves a CU held one phase apart by barriers 4.85 ms, against 5.00 ms of waves that run freely; the
// larger workgroups cost 10 - 25 % at every smaller size, so waves run freely.  (Priority for either phase of a wave: no difference.)  Under this load the card
// runs at 1.8 - 1.9 GHz.
template <int TERMS, int DP> constexpr int ce_waves() { return DP == 256 ? 1 : 2; }

// LDS image: rows of DP / 8 chunks of 16 bytes, chunk c of row r at c ^ ce_swz(r).  The banks serve 256 bytes a cycle: 16 lanes of a fragment read (16 rows,
// one chunk) or 32 of a transposed read (4 rows, four neighbouring chunks).  With this image either touches 16 different 16-byte slots; a swizzle of
// 8 rows, enough for 128 bytes a cycle, spent half of the LDS cycles on conflicts.
template <int DP>
__device__ __forceinline__ int ce_swz(int r) {
    if constexpr (DP == 64) return ((r & 2) << 1) | ((r >> 2) & 3);      // two rows to 256 bytes
    else return ((r & 3) << 2) | ((r >> 2) & 3);
}

// WT: 16-bit terms of a weight.  Two for float32 rows; and where a sum has few terms (kFewTerms), whose roundings do not average out.  In longer sums of 16-bit
// rows one, but two for targets' weights in pass 2, each of which may be the better part of its class's gradient: 2-norm errors of de are those of one rounding
// to the type then (1 037 x 50 021 x 250 float16 2.40e-4, with one term for all 2.94e-4; 4 096 x 1.25 M x 128 bfloat16 1.67e-3 and 2.00e-3).  That costs
// 1 - 3 % where targets are spread over the catalogue, up to 10 % where the first hundreds of classes are most queries' targets (4 096 x 26 744 x 128 bfloat16 160
// and 175 us); in the phases of the product itself, under a branch for each matrix instruction, 184.
constexpr int kFewTerms = 128;

// Sum or mean of the rows' losses, and how many rows count; with no row counted the mean is 0.  One workgroup, 64-bit sums in a fixed order.
template <int T>
__device__ __forceinline__ void ce_reduce_loss(const float* loss_rows, const int64_t* target, const CeSums* sums, int64_t n, int reduction, float* loss, float* counted) {
    __shared__ double s_sum[T / 64];
    __shared__ int s_cnt[T / 64];
    double sum = 0.0;
    int cnt = 0;      // n < 2^31
    if (sums) {
        for (int i = threadIdx.x; i < kSumParts; i += T) sum += sums->loss[i], cnt += sums->counted[i];
    } else {
        for (int64_t r = threadIdx.x; r < n; r += T) {
            sum += double(loss_rows[r]);
            cnt += target[r] != -1;
        }
    }
    sum = wave_sum_f64(sum);
    cnt = wave_sum_i32(cnt);
    if ((threadIdx.x & 63) == 0) {
        s_sum[threadIdx.x >> 6] = sum;
        s_cnt[threadIdx.x >> 6] = cnt;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < T / 64; ++i) sum += s_sum[i], cnt += s_cnt[i];
        if (loss) *loss = float(reduction == 1 ? sum / double(max(cnt, 1)) : sum);
        if (counted) *counted = float(cnt);
    }
}

// ... one part of them
__global__ __launch_bounds__(256) void ce_loss_parts_kernel(const float* loss_rows, const int64_t* target, int64_t n, CeSums* sums) {
    __shared__ double s_sum[4];
    __shared__ int s_cnt[4];
    double sum = 0.0;
    int cnt = 0;
    for (int64_t r = int64_t(blockIdx.x) * 256 + threadIdx.x; r < n; r += kSumParts * 256) {
        sum += double(loss_rows[r]);
        cnt += target[r] != -1;
    }
    sum = wave_sum_f64(sum);
    cnt = wave_sum_i32(cnt);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = sum, s_cnt[threadIdx.x >> 6] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        sums->loss[blockIdx.x] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        sums->counted[blockIdx.x] = (s_cnt[0] + s_cnt[1]) + (s_cnt[2] + s_cnt[3]);
    }
}

// f(0 .. N - 1) with compile-time numbers
template <int I, int N, class F>
__device__ __forceinline__ void ce_static_for(F f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>());
        ce_static_for<I + 1, N>(f);
    }
}

template <typename E, int TERMS, int WT, int DP, int MODE, bool BIAS, bool ROWG>
__global__ __launch_bounds__(256, (ce_waves<TERMS, DP>())) void ce_pass_kernel(CePass a) {
    typedef CeType<E> X;
    constexpr int WAVES = 4;
    constexpr int KC = DP / 16, DB = DP / 32, SB = ce_sub<TERMS, DP>(), TS = 32 * SB, ROWB = DP * 2, PLANE = TS * ROWB;
    // Tiles in LDS: the last one, whose last 32 rows the second product still reads, the one at work, the next,
    // and the one after that: a tile is fetched while two are worked on.
    constexpr int RING = 4;
    // The factor carries a query's own upstream gradient, and the part of its lse that float32 cannot hold beside |lse| ~ 40 (2^-19 of a weight):
    // of no account in 16-bit gradients, so plain 16-bit passes save the multiplication, but for tiles with a row beyond FAR.
    constexpr bool MUL = MODE == kTable && (ROWG || BIAS || TERMS == 2);
    constexpr float OFF = X::offset[MODE == kTable];
    __shared__ __align__(16) char s_tile[RING][TERMS][PLANE];
    __shared__ __align__(16) float s_par[RING][MODE == kTable ? 4 : 1][TS];      // pass 1: bias; pass 2: CePass::rowp
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l31 = lane & 31;
    if constexpr (MODE == kTable) {
        if (blockIdx.x + 1 == gridDim.x && a.loss) return ce_reduce_loss<256>(a.loss_rows, a.target, a.sums, a.n_strm, a.reduction, a.loss, nullptr);
    }
    // consecutive numbers stay on one XCD (workgroup id mod 8), and consecutive numbers share a split: the tiles they stream meet in that XCD's L2
    const int total = a.stat_blocks * a.n_splits, per = (total + 7) / 8;
    const int id = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
    if (int(blockIdx.x >> 3) >= per || id >= total) return;
    const int split = id / a.stat_blocks, sblock = id % a.stat_blocks;
    const int64_t row0 = int64_t(sblock) * (32 * WAVES) + wave * 32, my = row0 + l31;
    const int64_t myc = my < a.n_stat ? my : a.n_stat - 1;

    s16x8 xf[TERMS][KC];
#pragma unroll
    for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int k = 0; k < KC; ++k) xf[t][k] = *reinterpret_cast<const s16x8*>((t ? a.stat_lo : a.stat) + myc * a.ld_stat + 16 * k + 8 * half);
    f32x16 o[MODE == kLse ? 1 : DB];
#pragma unroll
    for (int i = 0; i < (MODE == kLse ? 1 : DB); ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    const float scl = fmaxf(TERMS == 2 ? ldexpf(a.scale, a.sc->shift_s) : a.scale, 1.2e-38f), c = fmaxf(scl * kLog2e, 1.2e-38f);      // (never 0: 0 * -inf)
    const float thr = BIAS ? kStale * kLn2 : kStale / c;
    float m = kLowest, renew = kLowest, l = 0.f, l_low = 0.f;      // l_low: what l is too large by
    const int64_t target = MODE != kTable && my < a.n_stat ? a.target[my] : -1;
    if (MODE != kTable && split == 0) {      // (-1 once per row: both halves of a wave hold the same rows)
        const int cnt = __builtin_popcountll(__ballot(half == 0 && target != -1));
        if (lane == 0) a.counts[WAVES * sblock + wave] = cnt;
    }
    float zt = 0.f;
    bool has_zt = false;
    const float my_bias = (BIAS && MODE == kTable) ? a.bias[myc] : 0.f;

    // this split's streaming rows: `subs` times 32 from strm0 on, in tiles of SB times 32
    const int64_t strm0 = int64_t(split) * a.subs_per_split * 32;
    const int subs = int(max(int64_t(0), min(int64_t(a.subs_per_split), (a.n_strm - strm0 + 31) / 32))), tiles = (subs + SB - 1) / SB;
    constexpr int RPI = 1024 / ROWB, PER_WAVE = PLANE / (1024 * WAVES);      // rows of a DMA instruction (1 KB); instructions of a wave, tile and term
    uint32_t piece_at[PER_WAVE];      // byte of this lane's 16 in a tile's memory
#pragma unroll
    for (int i = 0; i < PER_WAVE; ++i) {
        const int r = (wave * PER_WAVE + i) * RPI + lane / (ROWB / 16);
        piece_at[i] = uint32_t(r) * uint32_t(a.ld_strm * 2) + 16 * ((lane % (ROWB / 16)) ^ ce_swz<DP>(r));
    }
    auto fetch = [&](int tile, int slot) __attribute__((always_inline)) {
        const int64_t first_row = strm0 + int64_t(tile) * TS;
        const bool whole = first_row + TS <= a.n_strm;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            const short* base = (t ? a.strm_lo : a.strm) + first_row * a.ld_strm;
#pragma unroll
            for (int i = 0; i < PER_WAVE; ++i) {
                const int piece = wave * PER_WAVE + i;
                const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(&s_tile[slot][t][piece * 1024]));
                if (whole) {
                    lds_dma16(base, piece_at[i], to);
                } else {      // rows past the end repeat the last one; their weights are zero
                    const int r = piece * RPI + lane / (ROWB / 16), in = int(min(int64_t(r), a.n_strm - 1 - first_row));
                    lds_dma16_v(base + int64_t(in) * a.ld_strm + 8 * ((lane % (ROWB / 16)) ^ ce_swz<DP>(r)), to);
                }
            }
        }
    };
    // ... and the rows' parameters: wave i of the first four brings array i
    auto fetch_params = [&](int tile, int slot) __attribute__((always_inline)) {
        if (MODE == kTable ? wave < 4 : (BIAS && wave == 0)) {
            const int64_t first_row = strm0 + int64_t(tile) * TS;
            if (TS >= 64 || lane < TS) {
#pragma unroll
                for (int i = 0; i < (TS + 63) / 64; ++i) {
                    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(&s_par[slot][MODE == kTable ? wave : 0][i * 64]));
                    // (a bias is the caller's: rows past the end repeat the last one)
                    if (MODE == kTable) lds_dma4(a.rowp + wave * a.ld_rowp + first_row, uint32_t(i * 64 + lane) * 4, to);
                    else lds_dma4(a.bias + first_row, uint32_t(min(int64_t(i * 64 + lane), a.n_strm - 1 - first_row)) * 4, to);
                }
            }
        }
    };
    // This wave's share of tile `tile`, and of its parameters, has arrived (before a barrier: everyone's has).  What was fetched after it, the next tile's rows,
    // may be under way.
    auto arrived = [&](int tile) __attribute__((always_inline)) {
        if (tile + 1 < tiles) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(TERMS * PER_WAVE) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    if (tiles) {
        __builtin_amdgcn_s_waitcnt(0);      // (nothing of the above is counted below)
        fetch_params(0, 0);
        fetch(0, 0);
        if (tiles > 1) fetch(1, 1);
        arrived(0);
    }
    __syncthreads();

    // LDS addresses of this lane's pieces of the next fragments (bytes; they move on with the tiles), the rest of an address is a constant
    constexpr int SWZ = DP == 64 ? 8 : 16;      // chunks that are exchanged among each other
    constexpr int SLOT = TERMS * PLANE;
    // Chunk 2 k + half, or 4 k + cl, of a lane's row is at the address of k = 0 with 32 k, or 64 k, exclusive-or'd in; held for each k where registers allow.
    constexpr bool HELD = DP < 256;
    uint32_t fr_at[HELD ? SWZ / 2 : 1], tr_at[HELD ? SWZ / 4 : 1];
    fr_at[0] = lds_addr(s_tile) + l31 * ROWB + 16 * (half ^ ce_swz<DP>(l31));
    {
        const int r = 4 * half + ((lane & 15) >> 2), cl = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        tr_at[0] = lds_addr(s_tile) + r * ROWB + 8 * (lane & 1) + 16 * (cl ^ ce_swz<DP>(r));
    }
#pragma unroll
    for (int k = 1; k < (HELD ? SWZ / 2 : 1); ++k) fr_at[k] = fr_at[0] ^ (32 * k);
#pragma unroll
    for (int k = 1; k < (HELD ? SWZ / 4 : 1); ++k) tr_at[k] = tr_at[0] ^ (64 * k);

    f32x16 s;
    s16x8 ph[2], pl[2];      // weights of the last 32 streaming rows, as the second product's operand
    // A product phase is N2 + N1 steps, each with a fragment (two with two terms) from LDS: the second product of 32 rows (O^T += rows^T . weights), then the
    // first of the next 32 (S^T = rows . stationary^T).  Fragments are read DEPTH steps ahead, the first of them before the phase begins.
    constexpr int N2 = MODE == kLse ? 0 : 2 * DB, N1 = KC, DEPTH = TERMS * DP >= 256 ? 4 : 8, PRE = N2 < 2 ? N2 : 2;
    s16x8 ring[DEPTH][TERMS];
    typedef const __attribute__((address_space(3))) s16x8* lds8_t;
    typedef __attribute__((address_space(3))) s16x4* lds4_t;
    auto read_transposed = [&](int t, int row, auto i_) __attribute__((always_inline)) {      // 16 streaming rows x 32 columns
        constexpr int i = decltype(i_)::value;
        const uint32_t p = HELD ? tr_at[i % (SWZ / 4) * HELD] : tr_at[0] ^ (64 * (i % (SWZ / 4)));
        const int off = t * PLANE + row * ROWB + 16 * SWZ * (i / (SWZ / 4));
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4_t>(p + off));
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds4_t>((p ^ 32) + (off + 8 * ROWB)));      // (8 rows on, the swizzle differs by 2)
        return s16x8(__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto read = [&](auto u_, auto sb2_, auto sb1_) __attribute__((always_inline)) {
        constexpr int u = decltype(u_)::value, sb2 = decltype(sb2_)::value, sb1 = decltype(sb1_)::value;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            if constexpr (u < N2) {
                ring[u % DEPTH][t] = read_transposed(t, sb2 * 32 + 16 * (u / DB), std::integral_constant<int, u % DB>());
            } else {
                constexpr int k = u - N2;
                ring[u % DEPTH][t] = *reinterpret_cast<lds8_t>((HELD ? fr_at[k % (SWZ / 2) * HELD] : fr_at[0] ^ (32 * (k % (SWZ / 2)))) + (t * PLANE + sb1 * 32 * ROWB + 16 * SWZ * (k / (SWZ / 2))));
            }
        }
    };
    auto multiply = [&](auto u_) __attribute__((always_inline)) {
        constexpr int u = decltype(u_)::value;
        const s16x8 hi = ring[u % DEPTH][0], lo = ring[u % DEPTH][TERMS - 1];
        if constexpr (u < N2) {
            constexpr int k = u / DB, i = u % DB;
            o[i] = X::mfma(hi, ph[k], o[i]);
            if constexpr (TERMS == 2) o[i] = X::mfma(lo, ph[k], o[i]);
            if constexpr (WT == 2) o[i] = X::mfma(hi, pl[k], o[i]);
        } else {
            constexpr int k = u - N2;
            if constexpr (k == 0) {
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = 0.f;
            }
            s = X::mfma(hi, xf[0][k], s);
            if constexpr (TERMS == 2) {
                // (in the same order of the operands in both passes: a logit has the same bits in either)
                s = MODE == kTable ? X::mfma(hi, xf[1][k], s) : X::mfma(lo, xf[0][k], s);
                s = MODE == kTable ? X::mfma(lo, xf[0][k], s) : X::mfma(hi, xf[1][k], s);
            }
        }
    };
    auto steps = [&](auto from_, auto to_, auto sb2, auto sb1) __attribute__((always_inline)) {      // steps from .. to - 1, their first reads done up to `from + PRE`
        constexpr int from = decltype(from_)::value, to = decltype(to_)::value;
        ce_static_for<from, to>([&](auto u) __attribute__((always_inline)) {
            multiply(u);
            constexpr int v = decltype(u)::value + DEPTH;
            if constexpr (v < to) read(std::integral_constant<int, v>(), sb2, sb1);
            __builtin_amdgcn_sched_barrier(0);      // the compiler would put every read right before its use
        });
    };
    // What the weights of 32 streaming rows take besides S (registers 4 q + j: row 8 q + 4 half + j of the 32), read before their phase where registers allow
    constexpr bool HAS_X = MODE == kTable || BIAS, EARLY = HAS_X && TERMS * DP <= 256;
    float px[HAS_X ? 16 : 1], pm[MUL ? 16 : 1];
    auto read_params = [&](int slot, int sb) __attribute__((always_inline)) {
        if constexpr (HAS_X) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float4 v = *reinterpret_cast<const float4*>(&s_par[slot][0][sb * 32 + 4 * half + 8 * q]);
                px[4 * q] = v.x, px[4 * q + 1] = v.y, px[4 * q + 2] = v.z, px[4 * q + 3] = v.w;
                if constexpr (MUL) {
                    const float4 u = *reinterpret_cast<const float4*>(&s_par[slot][1][sb * 32 + 4 * half + 8 * q]);
                    pm[4 * q] = u.x, pm[4 * q + 1] = u.y, pm[4 * q + 2] = u.z, pm[4 * q + 3] = u.w;
                }
            }
        }
    };
    // The sum of a lane's weights, over up to millions of rows: 16 at a time as a tree, added with the last addition's rounding error (one after the other, 1.2
    // million equal weights lost 5.5e-3 of their sum).
    auto add_weights = [&](const float (&w)[16]) __attribute__((always_inline)) {
        const float a0 = (w[0] + w[1]) + (w[2] + w[3]), a1 = (w[4] + w[5]) + (w[6] + w[7]), a2 = (w[8] + w[9]) + (w[10] + w[11]), a3 = (w[12] + w[13]) + (w[14] + w[15]);
        const float add = ((a0 + a1) + (a2 + a3)) - l_low, sum = l + add;
        l_low = (sum - l) - add;
        l = sum;
    };
    // S -> weights.  row: the first of the 32; reads: the first fragment reads of the product phase, issued before the exponentials
    float sub = BIAS ? 0.f : OFF;      // what exponents are taken against (without a maximum yet: 0)
    // Without a bias that is OFF - m c rounded, next to which an exponent's 2^-24 count where it is large: `far` rows' weights are put right by `fix`
    // (pass 1, per lane), or the row's factor (pass 2).
    constexpr float FAR = 256.f;
    float fix = 1.f;
    bool far = false;
    auto weights = [&](int slot, int sb, int64_t row, int my_target, uint32_t hits, auto reads) __attribute__((always_inline)) {
        if constexpr (HAS_X && !EARLY) read_params(slot, sb);
        float w[16];
        typename X::x8 low[MODE == kTable && WT == 1 ? 2 : 1];      // what rounding leaves of targets' weights
        if constexpr (MODE == kTable) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = BIAS ? fmaf(fmaf(s[j], scl, my_bias) - px[j], kLog2e, OFF) : fmaf(s[j], c, -px[j]);
            reads();
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                w[j] = __builtin_amdgcn_exp2f(w[j]);
                if constexpr (MUL) w[j] *= pm[j];
            }
            if (!MUL && far) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 u = *reinterpret_cast<const float4*>(&s_par[slot][1][sb * 32 + 4 * half + 8 * q]);
                    w[4 * q] *= u.x, w[4 * q + 1] *= u.y, w[4 * q + 2] *= u.z, w[4 * q + 3] *= u.w;
                }
            }
            if (hits) {      // (popular classes are hit in every tile: four rows' targets and weights at a time, not one after the other)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    if constexpr (WT == 1)
#pragma unroll
                        for (int j = 0; j < 4; ++j) low[q / 2][4 * (q % 2) + j] = E(0.f);
                    if (!(hits >> (8 * q) & 255)) continue;
                    const int r = sb * 32 + 8 * q + 4 * half;
                    const float4 t = *reinterpret_cast<const float4*>(&s_par[slot][3][r]), v = *reinterpret_cast<const float4*>(&s_par[slot][2][r]);
                    const float ts[4] = {t.x, t.y, t.z, t.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const bool mine = __float_as_int(ts[j]) == int(my);
                        w[4 * q + j] = mine ? vs[j] : w[4 * q + j];
                        if constexpr (WT == 1) low[q / 2][4 * (q % 2) + j] = E(mine ? vs[j] - float(E(vs[j])) : 0.f);
                    }
                }
            }
            if (BIAS) add_weights(w);
        } else {
            if (row + 32 > a.n_strm) {      // rows past the end
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (row + 4 * half + 8 * (j >> 2) + (j & 3) >= a.n_strm) s[j] = kLowest;
            }
            if (BIAS) {
#pragma unroll
                for (int j = 0; j < 16; ++j) s[j] = fmaf(s[j], scl, px[j]);
            }
            if (hits) {      // a target in this tile, and perhaps among these 32 rows: its logit is noted, and it is left out
                const int at = my_target - sb * 32;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (at == 8 * (j >> 2) + 4 * half + (j & 3)) {
                        zt = s[j];
                        has_zt = true;
                        s[j] = kLowest;
                    }
            }
            float mx = fmaxf(fmaxf(s[0], s[1]), s[2]);      // (pairs of them are one instruction)
#pragma unroll
            for (int j = 3; j < 15; j += 2) mx = fmaxf(fmaxf(mx, s[j]), s[j + 1]);
            mx = fmaxf(mx, s[15]);
            mx = fmaxf(mx, __uint_as_float(lane_xor32<32>(__float_as_uint(mx))));
            if (__any(mx > renew)) {
                const float mn = mx > renew ? fmaxf(m, mx) : m;      // (row by row: a row's result does not depend on the rows beside it)
                // (m = -inf: nothing so far, l and o are 0; differences first: a bias of float32's lowest value must not overflow)
                const float f = m == kLowest ? 1.f : __builtin_amdgcn_exp2f((m - mn) * (BIAS ? kLog2e : c));
                m = mn;
                renew = m == kLowest ? kLowest : m + thr;
                if (renew - m > 1.01f * thr) renew = m;      // (float32's steps at m are larger: the weights' range would not hold)
                sub = m == kLowest ? (BIAS ? 0.f : OFF) : (BIAS ? m : fmaf(-m, c, OFF));
                if (!BIAS) {
                    const bool mine = fabsf(sub) > FAR && m != kLowest;
                    fix = mine ? __builtin_amdgcn_exp2f(OFF - fmaf(m, c, sub)) : 1.f;
                    far = __any(mine);
                }
                l *= f, l_low *= f;
                if constexpr (MODE == kMean) {
#pragma unroll
                    for (int i = 0; i < DB; ++i)
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[i][j] *= f;
                }
            }
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = BIAS ? fmaf(s[j] - sub, kLog2e, OFF) : fmaf(s[j], c, sub);
            reads();
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j] = __builtin_amdgcn_exp2f(w[j]);
            if (!BIAS && far) {
#pragma unroll
                for (int j = 0; j < 16; ++j) w[j] *= fix;
            }
            add_weights(w);
        }
        if constexpr (MODE != kLse) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                typename X::x8 hi, lo;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    hi[j] = E(w[8 * k + j]);
                    if (WT == 2) lo[j] = E(w[8 * k + j] - float(hi[j]));
                }
                ph[k] = __builtin_bit_cast(s16x8, hi);
                if (WT == 2) pl[k] = __builtin_bit_cast(s16x8, lo);
            }
            // Targets' weights have a second term in one-term products too: ONE rounding would be the error of the gradient of a class that is seldom a target.  Its
            // product is made by itself, for 16 rows with a target among them.
            if constexpr (MODE == kTable && WT == 1) {
                if (hits) {
                    ce_static_for<0, 2>([&](auto k_) __attribute__((always_inline)) {
                        constexpr int k = decltype(k_)::value;
                        if (!(hits >> (16 * k) & 65535)) return;
                        ce_static_for<0, DB>([&](auto i_) __attribute__((always_inline)) {
                            constexpr int i = decltype(i_)::value;
                            o[i] = X::mfma(read_transposed(0, sb * 32 + 16 * k, i_), __builtin_bit_cast(s16x8, low[k]), o[i]);
                        });
                    });
                }
            }
        }
    };

    // first(0), weights(0), second(0) first(1), weights(1), ...; one barrier a tile, before its last 32 rows' products: the next tile is there then
    typedef std::integral_constant<int, 0> zero_t;
    if (tiles) {
        ce_static_for<N2, N2 + (DEPTH < N1 ? DEPTH : N1)>([&](auto u) __attribute__((always_inline)) { read(u, zero_t(), zero_t()); });
        steps(std::integral_constant<int, N2>(), std::integral_constant<int, N2 + N1>(), zero_t(), zero_t());
        if (EARLY) read_params(0, 0);
    }
    int slot = 0, at = 0;      // at: number of the 32 rows at work
    for (int tile = 0; tile < tiles; ++tile) {
        const int next = (slot + 1) % RING;
        const int64_t row = strm0 + int64_t(tile) * TS, from_tile = target - row;
        const int my_target = MODE != kTable && from_tile >= 0 && from_tile < TS ? int(from_tile) : -1;
        uint64_t hits = __any(my_target >= 0) ? ~uint64_t(0) : 0;
        if (MODE == kTable) {      // which of the tile's queries have their target among this wave's rows?
            const int t = (TS >= 64 || lane < TS) ? __float_as_int(s_par[slot][MODE == kTable ? 3 : 0][lane & (TS - 1)]) : -1;
            static_assert(TS <= 64, "a lane a row");
            hits = __ballot(t >= row0 && t < row0 + 32);
            if (!MUL) {
                const float off = (TS >= 64 || lane < TS) ? fabsf(s_par[slot][0][lane & (TS - 1)]) : 0.f;
                far = __any(off > FAR && off < INFINITY);
            }
        }
        ce_static_for<0, SB>([&](auto sb_) __attribute__((always_inline)) {
            constexpr int sb = decltype(sb_)::value, sb1 = sb == SB - 1 ? 0 : sb + 1;
            if (at >= subs) return;      // (uniform: the last tile may be shorter)
            if (sb == 0 && tile + 1 < tiles) {      // (the slot that is filled held the tile before the last: all waves have passed the last one's barrier)
                fetch_params(tile + 1, next);
                if (tile + 2 < tiles) fetch(tile + 2, (slot + 2) % RING);
            }
            weights(slot, sb, row + sb * 32, my_target, uint32_t(hits >> (32 * sb)), [&]() __attribute__((always_inline)) {
                __builtin_amdgcn_sched_barrier(0);
                ce_static_for<0, PRE>([&](auto u) __attribute__((always_inline)) { read(u, sb_, std::integral_constant<int, sb1>()); });
                __builtin_amdgcn_sched_barrier(0);
            });
            if (sb == SB - 1) {
                if (tile + 1 < tiles) arrived(tile + 1);
                __builtin_amdgcn_sched_barrier(0);
                asm volatile("" ::: "memory");
                __builtin_amdgcn_s_barrier();      // (waits for the waves only, not for memory)
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);
                const int move = (next - slot) * SLOT;
#pragma unroll
                for (int k = 0; k < (HELD ? SWZ / 2 : 1); ++k) fr_at[k] += move;
            }
            // (Behind the last 32 rows the first product reads what is there, and its result is not used.)
            ce_static_for<PRE, DEPTH>([&](auto u) __attribute__((always_inline)) { read(u, sb_, std::integral_constant<int, sb1>()); });
            steps(zero_t(), std::integral_constant<int, N2 + N1>(), sb_, std::integral_constant<int, sb1>());
            if constexpr (EARLY) read_params(sb == SB - 1 ? next : slot, sb1);
            ++at;
        });
        const int move = (next - slot) * SLOT;
#pragma unroll
        for (int k = 0; k < (HELD ? SWZ / 4 : 1); ++k) tr_at[k] += move;
        slot = next;
    }

    l += __uint_as_float(lane_xor32<32>(__float_as_uint(l)));
    if (my >= a.n_stat) return;
    if (MODE != kTable && has_zt) a.zt[my] = zt;
    const bool direct = MODE == kTable && a.n_splits == 1;
    if (!direct) {
        const int64_t at = int64_t(split) * a.n_stat + my;
        if (half == 0) {
            if (MODE != kTable) a.m[at] = m;
            if (MODE != kTable || BIAS) a.l[at] = l;
        }
        if constexpr (MODE != kLse) {
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4*>(a.o + at * DP + 32 * i + 8 * q + 4 * half) = float4{o[i][4 * q], o[i][4 * q + 1], o[i][4 * q + 2], o[i][4 * q + 3]};
        }
        return;
    }
    if constexpr (MODE == kTable) {
        typedef typename std::conditional<TERMS == 2, float, E>::type OUT;
        const float f = a.sc->fac_e, un = TERMS == 2 ? a.sc->unscale_q : 1.f;
        OUT* out = static_cast<OUT*>(a.out) + my * a.ld_out;
        if (BIAS && half == 0 && a.out_b) a.out_b[my] = l * a.sc->fac_b;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int col = 32 * i + 8 * q + 4 * half;
                typedef OUT out4 __attribute__((ext_vector_type(4)));
                const out4 v = {OUT(o[i][4 * q] * f * un), OUT(o[i][4 * q + 1] * f * un), OUT(o[i][4 * q + 2] * f * un), OUT(o[i][4 * q + 3] * f * un)};
                if (a.out_vec) {
                    if (col < a.d) *reinterpret_cast<out4*>(out + col) = v;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col + j < a.d) out[col + j] = v[j];
                }
            }
    }
}

// ---------------------------------------------------------------------------------------------------------------- operands
// Rows that the passes cannot read in place (width not 64 / 128 / 256, rows not on 16 bytes, float32, a table some of whose rows may be taken out) are laid
// out once per call.  Queries that do not count and classes that are taken out become rows of zeros there: their weights are zero, and zero times what an
// unused row holds (infinity, NaN) would be NaN in every other row's gradient.
struct CePack {
    const void* src[2];
    short *hi[2], *lo[2];
    int64_t rows[2], ld[2];
    int d, dp;
    float* tops;             // (2, kTopBlocks) partial maxima of |value|, n_tops of them
    int n_tops;
    CeScalars* sc;
    const int64_t* target;
    const float* bias;
    __device__ __forceinline__ bool used(int w, int64_t r) const {
        if (w == 0) return target[r] >= 0 && target[r] < rows[1];
        return !bias || bias[r] != -INFINITY;
    }
};
constexpr int kTopBlocks = 512;

// 16-bit rows: copied with zeros behind them.  blockIdx.y: which operand.
__global__ __launch_bounds__(256) void ce_pack16_kernel(CePack a) {
    const int w = blockIdx.y, chunks = a.dp / 8;
    if (!a.hi[w]) return;
    const int shift = 31 - __clz(chunks);      // chunks of a row: 8, 16 or 32
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < a.rows[w] * chunks; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i >> shift;
        const int c = int(i & (chunks - 1)) * 8;
        const short* p = static_cast<const short*>(a.src[w]) + r * a.ld[w];
        const int d = a.used(w, r) ? a.d : 0;
        s16x8 v;
        if (c + 8 <= d) __builtin_memcpy(&v, p + c, 16);      // (at any alignment: 50 021 x 250 float16 with 1 037 queries 11.5 us, 17 element by element)
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c + j < d ? p[c + j] : short(0);
        *reinterpret_cast<s16x8*>(a.hi[w] + r * a.dp + c) = v;
    }
}

// 8 float32 values of a row from column c, zeros past its end
__device__ __forceinline__ void ce_load8(const CePack& a, int w, int64_t r, int c, float (&v)[8]) {
    const float* p = static_cast<const float*>(a.src[w]) + r * a.ld[w] + c;
    const int d = a.used(w, r) ? a.d : 0;
    if (c + 8 <= d) {
        __builtin_memcpy(v, p, 32);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < d ? p[j] : 0.f;
    }
}

__global__ __launch_bounds__(256) void ce_top_kernel(CePack a) {
    __shared__ float s[4];
    const int w = blockIdx.y, chunks = a.dp / 8, shift = 31 - __clz(chunks);
    float top = 0.f;
#pragma unroll 4
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < a.rows[w] * chunks; i += int64_t(gridDim.x) * 256) {
        float v[8];
        ce_load8(a, w, i >> shift, int(i & (chunks - 1)) * 8, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fabsf(v[j]) < INFINITY ? fmaxf(top, fabsf(v[j])) : top;      // (of the finite ones: a row with others spoils no other row)
    }
    top = wave_max_f32(top);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) a.tops[w * kTopBlocks + blockIdx.x] = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
}

// exponent that puts `top` into [2^14, 2^15), as far as 2^126 does
__device__ __forceinline__ int ce_exponent(float top) {
    if (!(top > 0.f) || !(top < INFINITY)) return 0;
    return min(126, 14 - ilogbf(top));
}

__global__ __launch_bounds__(256) void ce_split_kernel(CePack a) {
    __shared__ float s[2];
    const int w = blockIdx.y, lane = threadIdx.x & 63;
    if (threadIdx.x < 128) {      // a wave per operand
        float top = 0.f;
        for (int i = lane; i < a.n_tops; i += 64) top = fmaxf(top, a.tops[(threadIdx.x >> 6) * kTopBlocks + i]);
        top = wave_max_f32(top);
        if (lane == 0) s[threadIdx.x >> 6] = top;
    }
    __syncthreads();
    const int eq = ce_exponent(s[0]), ee = ce_exponent(s[1]);
    if (blockIdx.x == 0 && w == 0 && threadIdx.x == 0) {
        a.sc->shift_s = -eq - ee;
        a.sc->unscale_q = ldexpf(1.f, -eq);
        a.sc->unscale_e = ldexpf(1.f, -ee);
    }
    const float f = ldexpf(1.f, w ? ee : eq);
    const int chunks = a.dp / 8, shift = 31 - __clz(chunks);
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < a.rows[w] * chunks; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i >> shift;
        const int c = int(i & (chunks - 1)) * 8;
        float v[8];
        ce_load8(a, w, r, c, v);
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi[j] = f16_t(v[j] * f);
            lo[j] = f16_t(v[j] * f - float(hi[j]));
        }
        *reinterpret_cast<f16x8*>(a.hi[w] + r * a.dp + c) = hi;
        *reinterpret_cast<f16x8*>(a.lo[w] + r * a.dp + c) = lo;
    }
}

// ---------------------------------------------------------------------------------------------------------------- rows
struct CeRows {
    const void* e;
    int64_t lde;
    const float* bias;
    const int64_t* target;
    int64_t n, v;
    int d, dp, n_splits;
    float scale;
    const float *m, *l, *o;       // partials of pass 1 (o nullable)
    CeScalars* sc;
    const float* zt;              // targets' logits (unit of m)
    float* loss_rows;
    float4* state;                // per row {lse, its low part, 1 - p_t, -}: with a bias in natural units, without in powers of two
    float* mean;                  // (n, d) sum_{v /= t} p'_v e_v, nullable
    // backward
    const float *counted, *grad;  // number of counted rows; upstream gradient (1, or n values when per_row), nullable = 1
    int reduction, per_row;       // 0 none, 1 mean, 2 sum
    void* dq;
    int64_t lddq;
    float* rowp;                  // CePass::rowp
    int64_t ld_rowp;
    const int* counts;            // counted rows (partial)
    int n_counts;
    float off, off2;              // powers of two that the weights of pass 1 / 2 carry
    const short* q;               // queries that pass 1 reads in place, nullable: copied for pass 2, rows that do not count as zeros (as CePack lays them out)
    int64_t ldq;
    short* q_copy;
};
constexpr int kCUs = 256, kMaxSplits = 512;      // splits of a streaming side
// Every row adds up to so many counts of 32 rows by itself (8 192 rows: 4 loads a lane); more are added once, by a launch of their own
constexpr int kCountedByRow = 256;

// What a row's state {lse, its low part, 1 - p_t} means to pass 2 (CePass::rowp); rel: its gradient relative to the largest.  Rows from n on: weights of zero.
template <bool BIAS>
__device__ __forceinline__ void ce_put_rowp(const CeRows& a, int64_t r, bool on, float lse, float low, float miss, float rel, int64_t t) {
    const bool some = on && lse != kLowest;
    const float px = BIAS ? lse : lse - a.off2;
    if (!BIAS && some) {      // (what that subtraction leaves)
        const float back = px - lse;
        low += (lse - (px - back)) - (a.off2 + back);
    }
    a.rowp[r] = some ? px : INFINITY;
    a.rowp[a.ld_rowp + r] = on ? rel * __builtin_amdgcn_exp2f(BIAS ? -low * kLog2e : -low) : 0.f;
    a.rowp[2 * a.ld_rowp + r] = -rel * miss * __builtin_amdgcn_exp2f(a.off2);
    a.rowp[3 * a.ld_rowp + r] = __int_as_float(on ? int(t) : -1);
}

__device__ __forceinline__ void ce_copy_query(const CeRows& a, int64_t r, bool on, int t) {      // thread t of at least dp / 8
    if (a.q && 8 * t < a.dp)
        *reinterpret_cast<s16x8*>(a.q_copy + r * a.dp + 8 * t) = on ? *reinterpret_cast<const s16x8*>(a.q + r * a.ldq + 8 * t) : s16x8{0, 0, 0, 0, 0, 0, 0, 0};
}

// Joins the splits of pass 1: loss_r, lse_r, 1 - p_t and sum_{v /= t} p'_v e_v.  TR threads a row (a wave, or 256 where there are many splits); DP / 4 of
// them hold 4 columns each, the groups of them share the splits.  GRADS: dx and pass 2's parameters at once (the loss's own gradient is 1).
template <typename E, bool F32, bool BIAS, int TR, bool GRADS>
__global__ __launch_bounds__(256) void ce_rows_kernel(CeRows a) {
    __shared__ float s_m[TR > 64 ? kMaxSplits : 1], s_red[8];
    __shared__ float4 s_o[TR > 64 ? 256 : 1];
    const int lane = threadIdx.x & 63, t_in = threadIdx.x % TR;
    const int64_t r = int64_t(blockIdx.x) * (256 / TR) + threadIdx.x / TR;
    if (r >= a.n) {      // (whole rows: with TR = 256 the whole workgroup)
        if (GRADS && r < a.ld_rowp && t_in == 0) ce_put_rowp<BIAS>(a, r, false, 0.f, 0.f, 0.f, 0.f, -1);
        return;
    }
    const float unit = BIAS ? kLog2e : fmaxf((F32 ? ldexpf(a.scale, a.sc->shift_s) : a.scale) * kLog2e, 1.2e-38f);      // from the maxima's unit to powers of two (as in the pass)
    float top = kLowest;
    for (int s = t_in; s < a.n_splits; s += TR) top = fmaxf(top, a.m[int64_t(s) * a.n + r]);
    top = wave_max_f32(top);
    if constexpr (TR > 64) {
        if (lane == 0) s_red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    }
    auto factor = [&](int s) {      // (a split without classes has l = 0, or NaN from NaN rows)
        const float m = a.m[int64_t(s) * a.n + r];
        return m == kLowest ? 1.f : __builtin_amdgcn_exp2f((m - top) * unit);
    };
    float sum = 0.f;
    for (int s = t_in; s < a.n_splits; s += TR) {
        const float f = factor(s);
        if constexpr (TR > 64) s_m[s] = f;
        sum += a.l[int64_t(s) * a.n + r] * f;
    }
    sum = lanes_sum<64>(sum);
    if constexpr (TR > 64) {
        if (lane == 0) s_red[4 + (threadIdx.x >> 6)] = sum;
        __syncthreads();
        sum = (s_red[4] + s_red[5]) + (s_red[6] + s_red[7]);
    }
    // in powers of two, 64 bits: the other classes' lse (all of them where no target counts) and the target's logit
    const int64_t t = a.target[r];
    const bool on = t >= 0 && t < a.v, there = on && !(BIAS && a.bias[t] == -INFINITY);      // (a target that is taken out has no row and no gradient)
    const double rest = sum == 0.f ? -double(INFINITY) : double(top) * double(unit) + log2(double(sum)) - double(a.off);
    double lse = rest, miss = 0.0, loss = 0.0;
    if (on) {
        const double z = double(a.zt[r]) * double(unit), x = rest - z;
        const bool none = sum == 0.f && z == -double(INFINITY);      // every class masked
        loss = none ? double(INFINITY) : x > 64.0 ? x * kLn2d : log1p(exp2(x));
        miss = none ? 1.0 : 1.0 / (1.0 + exp2(-x));
        // (a target far below adds nothing, and from its logit, float32's lowest value perhaps, the sum of the others would be lost)
        if (!none && x <= 64.0) lse = z + loss / kLn2d;
    } else if (t != -1) {
        loss = NAN;      // no such class: nothing to learn from, and seen in the loss
    }
    if (BIAS) lse /= double(unit);      // (the inverse of the factor that the passes' exponents have)
    const float hi = float(lse), low = hi == kLowest ? 0.f : float(lse - double(hi));
    float g = 1.f;
    if constexpr (GRADS) {
        if (a.reduction == 1) {
            int cnt = a.sc->counted;
            if (a.n_counts <= kCountedByRow) {
                cnt = 0;
                for (int i = lane; i < a.n_counts; i += 64) cnt += a.counts[i];
                cnt = wave_sum_i32(cnt);
            }
            g = 1.f / float(max(cnt, 1));
        }
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            const float unoff = __builtin_amdgcn_exp2f(-a.off2);
            a.sc->fac_e = a.scale * g * unoff;
            a.sc->fac_b = g * unoff;
        }
    }
    if (t_in == 0) {
        a.loss_rows[r] = float(loss);
        if constexpr (GRADS) ce_put_rowp<BIAS>(a, r, on, hi, low, float(miss), on ? 1.f : 0.f, there ? t : -1);
        else a.state[r] = {hi, low, float(miss), 0.f};
    }
    if (!GRADS && !a.mean) return;
    if constexpr (GRADS && !F32) ce_copy_query(a, r, on, t_in);
    const int per = a.dp / 4, groups = TR / per, c4 = t_in & (per - 1), grp = t_in / per;
    float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = grp; s < a.n_splits; s += groups) {
        const float f = TR > 64 ? s_m[s] : factor(s);
        const float4 x = *reinterpret_cast<const float4*>(a.o + (int64_t(s) * a.n + r) * a.dp + 4 * c4);
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y), v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
    }
    if constexpr (TR > 64) {
        s_o[threadIdx.x] = v;
        __syncthreads();
        if (grp) return;
        for (int k = 1; k < groups; ++k) {
            const float4 x = s_o[k * per + c4];
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
    } else {
        for (int k = per; k < 64; k <<= 1) {      // groups lie side by side in the wave
            v.x += __shfl_xor(v.x, k, kWave), v.y += __shfl_xor(v.y, k, kWave), v.z += __shfl_xor(v.z, k, kWave), v.w += __shfl_xor(v.w, k, kWave);
        }
        if (grp) return;
    }
    const float f = sum == 0.f ? 0.f : 1.f / sum, un = F32 ? a.sc->unscale_e : 1.f;      // (one after the other: both may leave float32's range)
    const float mean[4] = {v.x * f * un, v.y * f * un, v.z * f * un, v.w * f * un};
    const E* e = static_cast<const E*>(a.e) + (there ? t : 0) * a.lde;
    const float fq = a.scale * g * float(miss);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int c = 4 * c4 + j;
        if (c >= a.d) break;
        if constexpr (GRADS) static_cast<E*>(a.dq)[r * a.lddq + c] = E(on ? fq * (mean[j] - (there ? float(e[c]) : 0.f)) : 0.f);
        else a.mean[r * a.d + c] = mean[j];
    }
}

__global__ __launch_bounds__(1024) void ce_count_kernel(const int* counts, int n_counts, CeScalars* sc) {
    __shared__ int s[16];
    int cnt = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < n_counts; i += 1024) cnt += counts[i];
    cnt = wave_sum_i32(cnt);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) cnt += s[i];
        sc->counted = cnt;
    }
}

__global__ __launch_bounds__(1024) void ce_loss_kernel(const float* loss_rows, const int64_t* target, const CeSums* sums, int64_t n, int reduction, float* loss, float* counted) {
    ce_reduce_loss<1024>(loss_rows, target, sums, n, reduction, loss, counted);
}

// Largest |upstream gradient| of the rows that count (another row's may be anything): of all by one workgroup, or a part of them by each of kSumParts ones, and
// then of the parts.  (0 without rows.)
__global__ __launch_bounds__(1024) void ce_grad_top_kernel(const float* grad, const int64_t* target, int64_t n, int64_t v, CeScalars* sc, CeSums* sums, bool of_parts) {
    __shared__ float s[16];
    float top = 0.f;
    if (!of_parts)
        for (int64_t r = int64_t(blockIdx.x) * 1024 + threadIdx.x; r < n; r += int64_t(gridDim.x) * 1024) top = fmaxf(top, target[r] >= 0 && target[r] < v ? fabsf(grad[r]) : 0.f);
    else if (threadIdx.x < kSumParts) top = sums->top[threadIdx.x];
    top = wave_max_f32(top);
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        if (gridDim.x > 1) sums->top[blockIdx.x] = top;
        else sc->g_top = top;
    }
}

// Backward by itself: dx, and what pass 2 needs of every query (CePass::rowp).  One wave per row.
template <typename E, bool F32, bool BIAS>
__global__ __launch_bounds__(256) void ce_dq_kernel(CeRows a) {
    const int lane = threadIdx.x & 63;
    const int64_t r = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    // the gradient of a counted row, or with one per row what they are relative to
    const float g = a.per_row ? a.sc->g_top : (a.grad ? a.grad[0] : 1.f) / (a.reduction == 1 ? fmaxf(a.counted[0], 1.f) : 1.f);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        const float unoff = __builtin_amdgcn_exp2f(-a.off2);
        a.sc->fac_e = a.scale * g * unoff;
        a.sc->fac_b = g * unoff;
    }
    if (r >= a.n) {
        if (a.rowp && r < a.ld_rowp && lane == 0) ce_put_rowp<BIAS>(a, r, false, 0.f, 0.f, 0.f, 0.f, -1);
        return;
    }
    const int64_t t = a.target[r];
    const bool on = t >= 0 && t < a.v, there = on && !(BIAS && a.bias[t] == -INFINITY);
    const float4 st = a.state[r];
    const float gr = a.per_row ? a.grad[r] : g;
    if (a.rowp && lane == 0) ce_put_rowp<BIAS>(a, r, on, st.x, st.y, st.z, !on ? 0.f : a.per_row ? (g > 0.f ? gr / g : gr) : 1.f, there ? t : -1);
    if (!F32 && a.rowp) ce_copy_query(a, r, on, lane);
    if (a.dq) {
        E* dq = static_cast<E*>(a.dq) + r * a.lddq;
        const E* e = static_cast<const E*>(a.e) + (there ? t : 0) * a.lde;
        const float f = a.scale * gr * st.z;
        for (int c = lane; c < a.d; c += 64) dq[c] = E(on ? f * (a.mean[r * a.d + c] - (there ? float(e[c]) : 0.f)) : 0.f);
    }
}

// Joins the splits of pass 2
template <typename E>
__global__ __launch_bounds__(256) void ce_de_kernel(const float* __restrict__ o, const float* __restrict__ l, int n_splits, int64_t v, int d, int dp,
                                                   const CeScalars* sc, E* __restrict__ de, int64_t ldde, float* __restrict__ db) {
    const int per = dp / 4, shift = 31 - __clz(per);
    const float fe = sc->fac_e, fb = sc->fac_b, un = std::is_same<E, float>::value ? sc->unscale_q : 1.f;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < v * per; i += int64_t(gridDim.x) * 256) {
        const int64_t r = i >> shift;
        const int c = int(i & (per - 1)) * 4;
        if (c < d) {
            float4 s = *reinterpret_cast<const float4*>(o + r * dp + c);
#pragma unroll 4
            for (int k = 1; k < n_splits; ++k) {
                const float4 t = *reinterpret_cast<const float4*>(o + (int64_t(k) * v + r) * dp + c);
                s.x += t.x, s.y += t.y, s.z += t.z, s.w += t.w;
            }
            E* out = de + r * ldde + c;
            out[0] = E(s.x * fe * un);
            if (c + 1 < d) out[1] = E(s.y * fe * un);
            if (c + 2 < d) out[2] = E(s.z * fe * un);
            if (c + 3 < d) out[3] = E(s.w * fe * un);
        }
        if (db && c == 0) {
            float s = l[r];
            for (int k = 1; k < n_splits; ++k) s += l[int64_t(k) * v + r];
            db[r] = s * fb;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
constexpr int kCeMaxDim = 256;
// Classes are 32-bit numbers; a wave for each query has to stay below a launch's 2^32 threads
constexpr int64_t kCeMaxRows = (int64_t(1) << 26) - 256;
static bool ce_rows_fit(int64_t n, int64_t v) { return n >= 0 && n <= kCeMaxRows && v >= 1 && v <= (int64_t(1) << 31) - 256; }
static int ce_width(int64_t d) { return d >= 1 && d <= kCeMaxDim ? int(d) : 0; }      // 0: refused by CeCall::check
static int ce_padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

static bool ce_direct(const void* p, int64_t ld, int d, int dtype) {
    return dtype != HWER_F32 && d == ce_padded(d) && aligned_to(p, ld * 2, 16) && ld < (1 << 23);      // (a tile's bytes are addressed in 32 bits)
}

// Splits of the streaming side, in 32s of its rows.  A call takes as long as its fullest CU (which holds two workgroups, or one of the widest rows): rounds of
// workgroups times (a split's 32s + about 4 for its start and end); and each split leaves sums behind that are written and read again, about 3 MB in the
// time of 32 rows (with 2: 8 192 x 4 000 x 128 bfloat16 101 us, 89 so, 89 with 6; 2 000 x 3 000 x 100 float32 77, 74 and 70; 100 000 x 129 x 128 the same).
// A split is no longer than its products' sums can bear: the matrix instructions add to one float32 sum twice for 32 rows (float32 rows: six times), and with
// terms of one direction (equal rows) N additions leave up to N 2^-25 of it.  float32 rows: 1 536 additions, 4.6e-5; 16-bit rows: 8 192, 2.4e-4, half a rounding
// of float16.  As long as the splits' sums fit into kSplitBytes: 65 536 x 1.2 M float32 rows of 64 are 147 splits, 2.5 GB.
// Tried for pass 2: one workgroup for each place on the CUs with an equal share of all blocks' work.  No last round that is not full (1 037 x 50 021 x 250
// float16 256 -> 241 us), but no workgroup takes over from a slower one either, and the loop over blocks costs registers: 4 096 x 1.25 M x 128 bfloat16
// 4.90 -> 5.00 ms, x 400 k x 64 0.97 -> 1.04, x 400 k x 256 4.0 -> 4.7.
struct CeSplit {
    int blocks, splits, subs;
};
constexpr int kRows = 128;      // stationary rows of a workgroup
constexpr int64_t kSplitBytes = int64_t(8) << 30;
static CeSplit ce_split(int64_t n_stat, int64_t n_strm, int d, int dtype) {
    const int dp = ce_padded(d);
    const int64_t blocks = cdiv64(n_stat, kRows), subs = std::max<int64_t>(1, cdiv64(n_strm, 32)), slots = (dp == 256 ? 1 : 2) * kCUs;
    const int64_t most = std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, kSplitBytes / (std::max<int64_t>(blocks, 1) * kRows * dp * 4)));
    const int64_t least = std::min(most, cdiv64(subs, dtype == HWER_F32 ? 256 : 4096));
    double best = INFINITY;
    int64_t per = cdiv64(subs, least);
    for (int64_t s = least; s <= std::min<int64_t>(subs, kMaxSplits) && (s == least || blocks * s <= 8 * slots); ++s) {
        const int64_t p = cdiv64(subs, s), n = cdiv64(subs, p);
        const double cost = double(cdiv64(blocks * n, slots) * (p + 4)) + (n > 1 ? double(blocks * kRows * dp * 8) * double(n) / 3e6 : 0.0);
        if (cost < best) best = cost, per = p;
    }
    return {int(blocks), int(cdiv64(subs, per)), int(per)};
}

// queries with parameters for pass 2, whole tiles of at most 128 from any 32nd query on
static int64_t ce_rowp_ld(int64_t n) { return cdiv64(n, 32) * 32 + 128; }

static size_t up(size_t b) { return (b + 255) & ~size_t(255); }

// Where a call's workspace keeps what.  The head (scalars, laid-out operands) serves both passes of a call.
struct CeLayout {
    size_t sums, tops, q_hi, q_lo, e_hi, e_lo, loss_rows, counts, rowp, head, zt, m, l, o, fwd_end, l2, o2, bwd_end;
    CeSplit f, b;      // of pass 1 and 2
    size_t bytes(bool want_mean) const { return std::max<size_t>(256, want_mean ? std::max(fwd_end, bwd_end) : fwd_end); }
};
static CeLayout ce_layout(int64_t n, int64_t v, int d, int dtype, bool q_direct, bool e_direct, bool want_mean) {
    const size_t dp = ce_padded(d);
    CeLayout y{};
    const CeSplit f = y.f = ce_split(n, v, d, dtype), b = y.b = ce_split(v, n, d, dtype);
    size_t at = 256;      // CeScalars
    y.sums = at, at += n > kSumRows ? up(sizeof(CeSums)) : 0;
    y.tops = at, at += dtype == HWER_F32 ? 2 * kTopBlocks * 4 : 0;
    y.q_hi = at, at += q_direct && !want_mean ? 0 : up(size_t(n) * dp * 2);
    y.q_lo = at, at += dtype == HWER_F32 ? up(size_t(n) * dp * 2) : 0;
    y.e_hi = at, at += e_direct ? 0 : up(size_t(v) * dp * 2);
    y.e_lo = at, at += dtype == HWER_F32 ? up(size_t(v) * dp * 2) : 0;
    y.counts = at, at += up(size_t(f.blocks) * 16);
    y.loss_rows = at, at += want_mean ? up(size_t(n) * 4) : 0;
    y.rowp = at, at += want_mean ? up(size_t(ce_rowp_ld(n)) * 16) : 0;
    y.head = at;
    y.zt = at, at += up(size_t(n) * 4);
    y.m = at, at += up(size_t(f.splits) * n * 4);
    y.l = at, at += up(size_t(f.splits) * n * 4);
    y.o = at, at += want_mean ? up(size_t(f.splits) * n * dp * 4) : 0;
    y.fwd_end = at;
    at = y.head;
    y.l2 = at, at += b.splits > 1 ? up(size_t(b.splits) * v * 4) : 0;
    y.o2 = at, at += b.splits > 1 ? up(size_t(b.splits) * v * dp * 4) : 0;
    y.bwd_end = at;
    return y;
}

// One call: checked operands, and the steps that the entries below are made of.
struct CeCall {
    const void *q, *e;
    int64_t ldq, lde;
    const float* bias;
    const int64_t* target;
    int64_t n, v;
    int d, dtype;
    float scale;
    int reduction;
    unsigned char* ws;
    hipStream_t st;
    bool q_direct, e_direct;
    int dp;
    CeLayout y;

    template <typename T> T* at(size_t off) const { return reinterpret_cast<T*>(ws + off); }
    const short* q_hi() const { return q_direct ? static_cast<const short*>(q) : at<short>(y.q_hi); }
    const short* e_hi() const { return e_direct ? static_cast<const short*>(e) : at<short>(y.e_hi); }
    const short* q_lo() const { return dtype == HWER_F32 ? at<short>(y.q_lo) : nullptr; }
    const short* e_lo() const { return dtype == HWER_F32 ? at<short>(y.e_lo) : nullptr; }
    int64_t q_ld() const { return q_direct ? ldq : dp; }
    int64_t e_ld() const { return e_direct ? lde : dp; }

    int check(const char* what, void* workspace, size_t bytes, bool want_mean, void* stream) {
        if (!known_dtype(dtype)) return fail(HWER_EINVAL, "%s: unknown element type %d", what, dtype);
        if (d < 1) return fail(HWER_EINVAL, "%s: rows of 1..%d elements are supported", what, kCeMaxDim);
        if (!ce_rows_fit(n, v))
            return fail(HWER_EINVAL, "%s: %lld rows (at most %lld), %lld classes (at most 2^31 - 256)", what, (long long)n, (long long)kCeMaxRows, (long long)v);
        if (!(scale > 0.f) || !(scale < INFINITY)) return fail(HWER_EINVAL, "%s: scale must be positive and finite", what);
        if (n && (!q || !target)) return fail(HWER_EINVAL, "%s: null queries or targets", what);
        if (!e || ldq < d || lde < d) return fail(HWER_EINVAL, "%s: null table or a row stride below d", what);
        q_direct = ce_direct(q, ldq, d, dtype), e_direct = !bias && ce_direct(e, lde, d, dtype), dp = ce_padded(d);
        y = ce_layout(n, v, d, dtype, q_direct, e_direct, want_mean);
        const size_t need = y.bytes(want_mean);
        if (!workspace || bytes < need) return fail(HWER_EWORKSPACE, "%s: workspace of %zu bytes needed", what, need);
        if (!aligned_to(workspace, 0, 256)) return fail(HWER_EINVAL, "%s: the workspace must be 256-byte aligned", what);
        ws = static_cast<unsigned char*>(workspace), st = as_stream(stream);
        return HWER_OK;
    }

    CeSums* sums() const { return n > kSumRows ? at<CeSums>(y.sums) : nullptr; }      // (nullptr: one workgroup does it)
    // before a workgroup reduces the rows' losses
    void sum_losses(const float* loss_rows) const {
        if (sums()) ce_loss_parts_kernel<<<dim3(kSumParts), dim3(256), 0, st>>>(loss_rows, target, n, sums());
    }
    void grad_top(const float* grad) const {
        CeScalars* sc = at<CeScalars>(0);
        ce_grad_top_kernel<<<dim3(sums() ? kSumParts : 1), dim3(1024), 0, st>>>(grad, target, n, v, sc, sums(), false);
        if (sums()) ce_grad_top_kernel<<<dim3(1), dim3(1024), 0, st>>>(grad, target, n, v, sc, sums(), true);
    }

    // lays out what the passes cannot read in place
    int prepare() const {
        CePack p{{q, e}, {nullptr, nullptr}, {nullptr, nullptr}, {n, v}, {ldq, lde}, d, dp, at<float>(y.tops), 0, at<CeScalars>(0), target, bias};
        if (!q_direct) p.hi[0] = at<short>(y.q_hi);
        if (!e_direct) p.hi[1] = at<short>(y.e_hi);
        const dim3 grid(unsigned(std::max<int64_t>(1, std::min<int64_t>(cdiv64(std::max(n, v) * (dp / 8), 256), kMaxStreamBlocks))), 2);
        if (dtype == HWER_F32) {
            p.lo[0] = at<short>(y.q_lo), p.lo[1] = at<short>(y.e_lo);
            p.n_tops = int(std::max<int64_t>(1, std::min<int64_t>(kTopBlocks, cdiv64(std::max(n, v) * (dp / 8), 256))));
            ce_top_kernel<<<dim3(p.n_tops, 2), dim3(256), 0, st>>>(p);
            ce_split_kernel<<<grid, dim3(256), 0, st>>>(p);
        } else if (p.hi[0] || p.hi[1]) {
            ce_pack16_kernel<<<grid, dim3(256), 0, st>>>(p);
        }
        return check_launch("catalogue_ce(operands)");
    }

    int pass1(bool mean, CeRows& r) const {
        const CeSplit& s = y.f;
        CePass p{};
        p.stat = q_hi(), p.stat_lo = q_lo(), p.strm = e_hi(), p.strm_lo = e_lo();
        p.ld_stat = q_ld(), p.ld_strm = e_ld(), p.n_stat = n, p.n_strm = v;
        p.bias = bias, p.scale = scale, p.sc = at<CeScalars>(0);
        p.subs_per_split = s.subs, p.n_splits = s.splits, p.stat_blocks = s.blocks;
        p.m = at<float>(y.m), p.l = at<float>(y.l), p.o = at<float>(y.o);
        p.target = target, p.zt = at<float>(y.zt), p.counts = at<int>(y.counts), p.d = d;
        mean ? ce_pass_any<kMean>(p, dp, dtype, false, st) : ce_pass_any<kLse>(p, dp, dtype, false, st);
        r = rows();
        r.n_splits = s.splits, r.m = p.m, r.l = p.l, r.o = p.o, r.zt = p.zt, r.counts = p.counts, r.n_counts = 4 * s.blocks;
        return check_launch("catalogue_ce(pass)");
    }

    CeRows rows() const {
        CeRows r{};
        r.e = e, r.lde = lde, r.bias = bias, r.target = target, r.n = n, r.v = v, r.d = d, r.dp = dp, r.scale = scale, r.sc = at<CeScalars>(0);
        if (q_direct) r.q = static_cast<const short*>(q), r.ldq = ldq, r.q_copy = at<short>(y.q_hi);
        r.reduction = reduction, r.ld_rowp = ce_rowp_ld(n), r.off = ce_offset(dtype, 0), r.off2 = ce_offset(dtype, 1);
        return r;
    }

    int pass2(void* de, int64_t ldde, float* dbias, bool rowg, const float* loss_rows, float* loss) const {
        const CeSplit& s = y.b;
        CePass p{};
        p.stat = e_hi(), p.stat_lo = e_lo(), p.strm = at<short>(y.q_hi), p.strm_lo = q_lo();      // (queries: laid out, or copied by the rows' kernel)
        p.ld_stat = e_ld(), p.ld_strm = dp, p.n_stat = v, p.n_strm = n;
        p.bias = bias, p.scale = scale, p.sc = at<CeScalars>(0);
        p.subs_per_split = s.subs, p.n_splits = s.splits, p.stat_blocks = s.blocks;
        p.l = at<float>(y.l2), p.o = at<float>(y.o2);
        p.rowp = at<float>(y.rowp), p.ld_rowp = ce_rowp_ld(n), p.out = de, p.out_b = dbias, p.ld_out = ldde, p.d = d;
        p.out_vec = d % 4 == 0 && aligned_to(de, ldde * dtype_bytes(dtype), 4 * dtype_bytes(dtype));
        p.target = target, p.loss_rows = loss_rows, p.sums = sums(), p.loss = loss, p.reduction = reduction;
        if (loss) sum_losses(loss_rows);
        ce_pass_any<kTable>(p, dp, dtype, rowg, st);
        if (int rc = check_launch("catalogue_ce(table pass)")) return rc;
        if (s.splits > 1) {
            const dim3 grid(unsigned(std::min<int64_t>(cdiv64(v * (dp / 4), 256), 4 * kMaxStreamBlocks)));
            if (dtype == HWER_F32) ce_de_kernel<float><<<grid, dim3(256), 0, st>>>(p.o, p.l, s.splits, v, d, dp, p.sc, static_cast<float*>(de), ldde, dbias);
            else if (dtype == HWER_F16) ce_de_kernel<f16_t><<<grid, dim3(256), 0, st>>>(p.o, p.l, s.splits, v, d, dp, p.sc, static_cast<f16_t*>(de), ldde, dbias);
            else ce_de_kernel<bf16_t><<<grid, dim3(256), 0, st>>>(p.o, p.l, s.splits, v, d, dp, p.sc, static_cast<bf16_t*>(de), ldde, dbias);
        }
        return check_launch("catalogue_ce(table)");
    }

    template <typename E, int TERMS, int WT, int DP, int MODE>
    static void ce_pass_launch(const CePass& a, bool rowg, hipStream_t st) {
        const bool more = MODE == kTable && a.loss;      // one more workgroup reduces the losses
        const dim3 grid(unsigned((int64_t(a.stat_blocks) * a.n_splits + 7) / 8 * 8 + more)), block(256);
        if constexpr (MODE == kTable) {
            if (a.bias) rowg ? ce_pass_kernel<E, TERMS, WT, DP, MODE, true, true><<<grid, block, 0, st>>>(a) : ce_pass_kernel<E, TERMS, WT, DP, MODE, true, false><<<grid, block, 0, st>>>(a);
            else rowg ? ce_pass_kernel<E, TERMS, WT, DP, MODE, false, true><<<grid, block, 0, st>>>(a) : ce_pass_kernel<E, TERMS, WT, DP, MODE, false, false><<<grid, block, 0, st>>>(a);
        } else {
            if (a.bias) ce_pass_kernel<E, TERMS, WT, DP, MODE, true, false><<<grid, block, 0, st>>>(a);
            else ce_pass_kernel<E, TERMS, WT, DP, MODE, false, false><<<grid, block, 0, st>>>(a);
        }
    }
    template <typename E, int TERMS, int WT, int MODE>
    static void ce_pass_width(const CePass& a, int dp, bool rowg, hipStream_t st) {
        if (dp == 64) ce_pass_launch<E, TERMS, WT, 64, MODE>(a, rowg, st);
        else if (dp == 128) ce_pass_launch<E, TERMS, WT, 128, MODE>(a, rowg, st);
        else ce_pass_launch<E, TERMS, WT, 256, MODE>(a, rowg, st);
    }
    template <int MODE>
    static void ce_pass_any(const CePass& a, int dp, int dtype, bool rowg, hipStream_t st) {
        const bool two = MODE != kLse && a.n_strm <= kFewTerms;
        constexpr int W2 = MODE == kLse ? 1 : 2;
        if (dtype == HWER_F32) ce_pass_width<f16_t, 2, W2, MODE>(a, dp, rowg, st);
        else if (dtype == HWER_F16) two ? ce_pass_width<f16_t, 1, W2, MODE>(a, dp, rowg, st) : ce_pass_width<f16_t, 1, 1, MODE>(a, dp, rowg, st);
        else two ? ce_pass_width<bf16_t, 1, W2, MODE>(a, dp, rowg, st) : ce_pass_width<bf16_t, 1, 1, MODE>(a, dp, rowg, st);
    }
    static float ce_offset(int dtype, int pass) { return dtype == HWER_BF16 ? CeType<bf16_t>::offset[pass] : CeType<f16_t>::offset[pass]; }

    template <bool GRADS>
    int join(const CeRows& r) const {
        if (GRADS && reduction == 1 && r.n_counts > kCountedByRow) ce_count_kernel<<<dim3(1), dim3(1024), 0, st>>>(r.counts, r.n_counts, r.sc);
        if (dtype == HWER_F32) join_typed<float, true, GRADS>(r);
        else if (dtype == HWER_F16) join_typed<f16_t, false, GRADS>(r);
        else join_typed<bf16_t, false, GRADS>(r);
        return check_launch("catalogue_ce(rows)");
    }
    template <typename E, bool F32, bool GRADS>
    void join_typed(const CeRows& r) const {
        // a wave per row walks over a few splits in less than a microsecond; hundreds of them (few rows, long catalogue) took 230 us at 466
        const bool wave = r.n_splits <= 16;
        const int64_t rows = GRADS ? ce_rowp_ld(n) : n;
        const dim3 grid(unsigned(wave ? cdiv64(rows, 4) : rows)), block(256);
        if (bias) wave ? ce_rows_kernel<E, F32, true, 64, GRADS><<<grid, block, 0, st>>>(r) : ce_rows_kernel<E, F32, true, 256, GRADS><<<grid, block, 0, st>>>(r);
        else wave ? ce_rows_kernel<E, F32, false, 64, GRADS><<<grid, block, 0, st>>>(r) : ce_rows_kernel<E, F32, false, 256, GRADS><<<grid, block, 0, st>>>(r);
    }
    template <typename E, bool F32>
    void dq_typed(const CeRows& r) const {
        const dim3 grid(unsigned(cdiv64(ce_rowp_ld(n), 4))), block(256);      // (without rows it leaves the factors of zeros)
        bias ? ce_dq_kernel<E, F32, true><<<grid, block, 0, st>>>(r) : ce_dq_kernel<E, F32, false><<<grid, block, 0, st>>>(r);
    }
    int backward_rows(const CeRows& r) const {
        if (dtype == HWER_F32) dq_typed<float, true>(r);
        else if (dtype == HWER_F16) dq_typed<f16_t, false>(r);
        else dq_typed<bf16_t, false>(r);
        return check_launch("catalogue_ce(row gradients)");
    }
};

}  // namespace hwer

using namespace hwer;

extern "C" {

int hwer_catalogue_ce_max_dim(void) { return kCeMaxDim; }

int hwer_catalogue_ce_reads_in_place(const void* rows, int64_t ld, int64_t d, int dtype) { return ce_width(d) && ce_direct(rows, ld, int(d), dtype) ? 1 : 0; }

size_t hwer_catalogue_ce_workspace_bytes(int64_t n, int64_t v, int64_t d, int dtype, int q_in_place, int e_in_place, int want_gradients) {
    if (!known_dtype(dtype) || !ce_width(d) || !ce_rows_fit(n, v)) return 0;      // (what the calls refuse)
    return ce_layout(n, v, int(d), dtype, q_in_place != 0, e_in_place != 0, want_gradients != 0).bytes(want_gradients != 0);
}

int hwer_catalogue_ce(const void* q, int64_t ldq, const void* e, int64_t lde, const float* bias, const int64_t* target, int64_t n, int64_t v, int64_t d, int dtype,
                      float scale, int reduction, float* loss_rows, float* state, float* loss, float* counted, float* mean, void* workspace, size_t workspace_bytes,
                      void* stream) {
    CeCall c{q, e, ldq, lde, bias, target, n, v, ce_width(d), dtype, scale, reduction};
    if (int rc = c.check("catalogue_ce", workspace, workspace_bytes, mean != nullptr, stream)) return rc;
    if (reduction < 0 || reduction > 2) return fail(HWER_EINVAL, "catalogue_ce: unknown reduction %d", reduction);
    if (!counted || (reduction && !loss) || (n && (!loss_rows || !state))) return fail(HWER_EINVAL, "catalogue_ce: null output");
    if (!aligned_to(state, 0, 16)) return fail(HWER_EINVAL, "catalogue_ce: state must be 16-byte aligned");
    if (n) {
        CeRows r;
        if (int rc = c.prepare()) return rc;
        if (int rc = c.pass1(mean != nullptr, r)) return rc;
        r.loss_rows = loss_rows, r.state = reinterpret_cast<float4*>(state), r.mean = mean;
        if (int rc = c.join<false>(r)) return rc;
    }
    c.sum_losses(loss_rows);
    ce_loss_kernel<<<dim3(1), dim3(1024), 0, c.st>>>(loss_rows, target, c.sums(), n, reduction, loss, counted);
    return check_launch("catalogue_ce");
}

int hwer_catalogue_ce_backward(const void* q, int64_t ldq, const void* e, int64_t lde, const float* bias, const int64_t* target, int64_t n, int64_t v, int64_t d,
                               int dtype, float scale, int reduction, const float* grad, const float* state, const float* counted, const float* mean, void* dq,
                               int64_t lddq, void* de, int64_t ldde, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    CeCall c{q, e, ldq, lde, bias, target, n, v, ce_width(d), dtype, scale, reduction};
    if (int rc = c.check("catalogue_ce_backward", workspace, workspace_bytes, true, stream)) return rc;
    if (reduction < 0 || reduction > 2 || (reduction == 0 && n && !grad)) return fail(HWER_EINVAL, "catalogue_ce_backward: unknown reduction %d, or rows' losses without their gradients", reduction);
    if (!counted || (n && (!state || (dq && !mean)))) return fail(HWER_EINVAL, "catalogue_ce_backward: what the forward call left is missing");
    if (!aligned_to(state, 0, 16)) return fail(HWER_EINVAL, "catalogue_ce_backward: state must be 16-byte aligned");
    if ((dq && lddq < d) || (de && ldde < d)) return fail(HWER_EINVAL, "catalogue_ce_backward: a row stride is below d");
    if (dbias && (!bias || !de)) return fail(HWER_EINVAL, "catalogue_ce_backward: dbias needs the bias, and comes with the table's gradient");
    if (de || dtype == HWER_F32)
        if (int rc = c.prepare()) return rc;
    CeRows r = c.rows();
    r.state = reinterpret_cast<float4*>(const_cast<float*>(state)), r.mean = const_cast<float*>(mean), r.counted = counted, r.grad = grad, r.per_row = reduction == 0;
    r.dq = dq, r.lddq = lddq, r.rowp = de ? c.at<float>(c.y.rowp) : nullptr;
    if (reduction == 0) c.grad_top(grad);
    if (int rc = c.backward_rows(r)) return rc;
    return de ? c.pass2(de, ldde, dbias, reduction == 0, nullptr, nullptr) : HWER_OK;
}

int hwer_catalogue_ce_grads(const void* q, int64_t ldq, const void* e, int64_t lde, const float* bias, const int64_t* target, int64_t n, int64_t v, int64_t d, int dtype,
                            float scale, int reduction, float* loss, void* dq, int64_t lddq, void* de, int64_t ldde, float* dbias, void* workspace,
                            size_t workspace_bytes, void* stream) {
    CeCall c{q, e, ldq, lde, bias, target, n, v, ce_width(d), dtype, scale, reduction};
    if (int rc = c.check("catalogue_ce_grads", workspace, workspace_bytes, true, stream)) return rc;
    if (reduction < 1 || reduction > 2) return fail(HWER_EINVAL, "catalogue_ce_grads: reduction %d: 1 (mean) or 2 (sum)", reduction);
    if (!loss || !de || (n && !dq) || lddq < d || ldde < d) return fail(HWER_EINVAL, "catalogue_ce_grads: null output or a row stride below d");
    if (dbias && !bias) return fail(HWER_EINVAL, "catalogue_ce_grads: a gradient of a bias that is not there");
    if (int rc = c.prepare()) return rc;
    float* loss_rows = c.at<float>(c.y.loss_rows);
    CeRows r = c.rows();
    if (n) {
        if (int rc = c.pass1(true, r)) return rc;
        r.loss_rows = loss_rows, r.dq = dq, r.lddq = lddq, r.rowp = c.at<float>(c.y.rowp);
        if (int rc = c.join<true>(r)) return rc;
    } else {
        r.per_row = 1;      // no rows: the factors of a sum over nothing
        c.grad_top(nullptr);
        if (int rc = c.backward_rows(r)) return rc;
    }
    return c.pass2(de, ldde, dbias, false, loss_rows, loss);
}

}  // extern "C"
