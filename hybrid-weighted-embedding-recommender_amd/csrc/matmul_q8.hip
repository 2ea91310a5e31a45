// Product of 8-bit rows:  out[m][n] = (sum_k A[m][k] B[n][k]) sa[m] sb[n] (+ bias[n]),  int8 codes with one float32 scale for each row of either side
// (a token's on the left, a channel's or catalogue row's on the right).  Sums are exact 32-bit integers (K <= 131 071: K * 128 * 128 < 2^31), so
// they depend on no order and no split; one rounding per product with a scale and one to the output's type follow.
//
//   matmul_q8_tile   both sides long: tiles of C on the 8-bit matrix instructions, operands staged in LDS by DMA
//   matmul_q8_few    one side short (<= 32 rows): the long side streams from memory once (1 x 8 192 x 8 192: 12.7 us, 5.3 TB/s; 1 x 400 k x 512: 31 us,
//                    6.5 TB/s, part of it from the last-level cache)
#include <algorithm>

#include "head_common.h"
#include "knn_internal.h"   // lds_dma16_v, lds_addr

namespace hwer {

typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i16_t __attribute__((ext_vector_type(16)));

struct QmmArgs {
    const int8_t *a, *b;      // rows of the output / columns of the output
    const float *sa, *sb, *bias;
    void* out;
    int64_t m, n, lda, ldb, ldo;
    int k;
};

// what a DMA lane reads where a row or a K chunk does not exist
__device__ const uint32_t kZero16[4] = {0u, 0u, 0u, 0u};

// 16 bytes at any address: the whole 4-byte words that hold them, shifted once they are there.  16-byte loads that are not on 4 bytes run at half the
// rate of others (1 x 8 192 rows of 8 190: 31 us against 23.5; but tiles, whose loads are covered by products: 2 000 x 8 192 x 8 190 155 us with such
// loads, 186 with these).
__device__ __forceinline__ i4_t bytes16(const int8_t* p) {
    i4_t v;
    __builtin_memcpy(&v, p, 16);
    return v;
}
struct Words5 {
    uint32_t d[5];
    int off;
    __device__ __forceinline__ void load(const int8_t* p) {
        off = int(reinterpret_cast<uintptr_t>(p) & 3);
        const int8_t* w = p - off;
        __builtin_memcpy(d, __builtin_assume_aligned(w, 4), 16);
        d[4] = *reinterpret_cast<const uint32_t*>(w + ((off + 15) & ~3));      // (the last word with a byte of the 16)
    }
    __device__ __forceinline__ void load(const int8_t* p, int n) {      // the first n (any number) of them, no word read that holds none
        off = int(reinterpret_cast<uintptr_t>(p) & 3);
        const int last = n > 0 ? (off + std::min(n, 16) - 1) & ~3 : 0;
#pragma unroll
        for (int i = 0; i < 5; ++i) d[i] = n > 0 ? *reinterpret_cast<const uint32_t*>(p - off + std::min(4 * i, last)) : 0u;
    }
    __device__ __forceinline__ i4_t get() const {
        i4_t v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = int(__builtin_amdgcn_alignbyte(d[i + 1], d[i], off));
        return v;
    }
    __device__ __forceinline__ i4_t get(int n) const {      // zeros after n bytes
        i4_t v = get();
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = n >= 4 * i + 4 ? v[i] : n <= 4 * i ? 0 : v[i] & int((1u << (8 * (n - 4 * i))) - 1u);
        return v;
    }
};

// 16 bytes of a row at byte k, zeros past the row's end.  ALIGNED: K, the row strides and the pointers are multiples of 16.
template <bool ALIGNED>
__device__ __forceinline__ i4_t load16(const int8_t* row, int k, int K) {
    if constexpr (ALIGNED) {
        return k < K ? *reinterpret_cast<const i4_t*>(row + k) : i4_t{0, 0, 0, 0};
    } else {
        Words5 w;
        w.load(row + k, K - k);
        return w.get(K - k);
    }
}

template <typename O>
__device__ __forceinline__ O finish(int acc, float sa, float sb, float bias) {
    return O(float(acc) * sa * sb + bias);
}

// ---------------------------------------------------------------------------------------------------------------- both sides long
// A workgroup of WM x WN waves makes a tile of C; a wave XM x XN blocks of 32 x 32.  Operands go through LDS in steps of 128 bytes of K, by DMA, the
// next step's while this one's is multiplied (STAGES = 2).
constexpr int kTK = 128;

// LDS image of an operand: 128 bytes (8 chunks of 16) a row, chunk c of row r at c ^ ((r / 2) & 7).  The banks serve 256 bytes a cycle, two rows: the 16 lanes
// of a ds_read_b128 that are served together read 16 rows' same chunk from 16 different 16-byte slots.  (r & 7 instead: two of them from each slot.)
template <bool ALIGNED, int ROWS, int WAVES>
__device__ __forceinline__ void stage(const int8_t* base, int64_t ld, int64_t row0, int64_t rows, int k0, int K, int8_t* lds, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < ROWS / (8 * WAVES); ++i) {      // 8 rows (1 KB) at a time
        const int r8 = (wave * (ROWS / (8 * WAVES)) + i) * 8, r = r8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        const bool in = row0 + r < rows;
        const int8_t* row = base + (in ? row0 + r : 0) * ld;
        if constexpr (ALIGNED) {
            const void* p = in && k0 + 16 * c < K ? static_cast<const void*>(row + k0 + 16 * c) : static_cast<const void*>(kZero16);
            lds_dma16_v(p, __builtin_amdgcn_readfirstlane(lds_addr(lds + r8 * kTK)));
        } else {
            const i4_t v = !in ? i4_t{0, 0, 0, 0} : k0 + kTK <= K ? bytes16(row + k0 + 16 * c) : load16<false>(row, k0 + 16 * c, K);
            *reinterpret_cast<i4_t*>(lds + r8 * kTK + lane * 16) = v;
        }
    }
}

template <typename O, bool ALIGNED, int WM, int WN, int XM, int XN, int STAGES>
__global__ __launch_bounds__(64 * WM * WN, (STAGES == 1 ? 4 : 2)) void matmul_q8_tile_kernel(QmmArgs g, int tiles_m, int tiles_n, int rows, int vec) {
    constexpr int WAVES = WM * WN, TM = 32 * XM * WM, TN = 32 * XN * WN, STAGE = (TM + TN) * kTK;
    constexpr int OROW = TN * int(sizeof(O)) + 16, OUT = 32 * WM * OROW;      // output rows on their way out: 32 of each wave's at a time
    __shared__ __align__(16) int8_t s_buf[STAGES * STAGE > OUT ? STAGES * STAGE : OUT];
    __shared__ __align__(16) float s_scale[TN], s_bias[TN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, l31 = lane & 31;
    // tiles of one XCD (workgroup id mod 8) are neighbours: bands of `rows` rows of tiles, walked along the columns
    const int total = tiles_m * tiles_n, per = (total + 7) / 8;
    const int id = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
    if (int(blockIdx.x >> 3) >= per || id >= total) return;
    const int band = id / (rows * tiles_n), in_band = id % (rows * tiles_n), bh = min(rows, tiles_m - rows * band);
    const int tm = band * rows + in_band % bh, tn = in_band / bh;
    const int64_t m0 = int64_t(tm) * TM, n0 = int64_t(tn) * TN;
    const int wm = (wave % WM) * 32 * XM, wn = (wave / WM) * 32 * XN;
    i16_t acc[XM][XN];
#pragma unroll
    for (int x = 0; x < XM; ++x)
#pragma unroll
        for (int y = 0; y < XN; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[x][y][i] = 0;
    const int steps = (g.k + kTK - 1) / kTK;
    // Whole steps of aligned operands: this lane's bytes of a panel as 32-bit offsets from a scalar address, rows past the end read as the last one (their
    // results are not written).  The general form's addresses cost a third of the vector instructions of a long product.
    constexpr int NA = TM / (8 * WAVES), NB = TN / (8 * WAVES);
    uint32_t at_a[ALIGNED ? NA : 1], at_b[ALIGNED ? NB : 1];
    if constexpr (ALIGNED) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int r = (wave * NA + i) * 8 + (lane >> 3);
            at_a[i] = uint32_t(std::min<int64_t>(r, g.m - 1 - m0)) * uint32_t(g.lda) + 16 * ((lane & 7) ^ ((r >> 1) & 7));
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int r = (wave * NB + i) * 8 + (lane >> 3);
            at_b[i] = uint32_t(std::min<int64_t>(r, g.n - 1 - n0)) * uint32_t(g.ldb) + 16 * ((lane & 7) ^ ((r >> 1) & 7));
        }
    }
    auto put = [&](int s, int buf) __attribute__((always_inline)) {
        if constexpr (ALIGNED) {
            if ((s + 1) * kTK <= g.k) {
                const int8_t *pa = g.a + m0 * g.lda + s * kTK, *pb = g.b + n0 * g.ldb + s * kTK;
                const uint32_t to = lds_addr(s_buf) + buf * STAGE;
#pragma unroll
                for (int i = 0; i < NA; ++i) lds_dma16(pa, at_a[i], __builtin_amdgcn_readfirstlane(to + (wave * NA + i) * 8 * kTK));
#pragma unroll
                for (int i = 0; i < NB; ++i) lds_dma16(pb, at_b[i], __builtin_amdgcn_readfirstlane(to + (TM + (wave * NB + i) * 8) * kTK));
                return;
            }
        }
        stage<ALIGNED, TM, WAVES>(g.a, g.lda, m0, g.m, s * kTK, g.k, s_buf + buf * STAGE, wave, lane);
        stage<ALIGNED, TN, WAVES>(g.b, g.ldb, n0, g.n, s * kTK, g.k, s_buf + buf * STAGE + TM * kTK, wave, lane);
    };
    // (older than the loads that are counted below, written to LDS after them: TN <= threads)
    const int64_t my_n = std::min<int64_t>(n0 + threadIdx.x % TN, g.n - 1);
    const float my_scale = g.sb[my_n], my_bias = g.bias ? g.bias[my_n] : 0.f;
    float row_scale[XM];
#pragma unroll
    for (int x = 0; x < XM; ++x) row_scale[x] = g.sa[std::min<int64_t>(m0 + wm + 32 * x + l31, g.m - 1)];
    constexpr int KC = kTK / 32;
    i4_t fa[2][XM], fb[2][XN];
    auto read = [&](int buf, int kc) __attribute__((always_inline)) {
        const int8_t *pa = s_buf + buf * STAGE, *pb = pa + TM * kTK;
        const int c = 2 * kc + half;
#pragma unroll
        for (int y = 0; y < XN; ++y) {
            const int r = wn + 32 * y + l31;
            fb[kc & 1][y] = *reinterpret_cast<const i4_t*>(pb + r * kTK + 16 * (c ^ ((r >> 1) & 7)));
        }
#pragma unroll
        for (int x = 0; x < XM; ++x) {
            const int r = wm + 32 * x + l31;
            fa[kc & 1][x] = *reinterpret_cast<const i4_t*>(pa + r * kTK + 16 * (c ^ ((r >> 1) & 7)));
        }
    };
    auto multiply = [&](int kc) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < XM; ++x)
#pragma unroll
            for (int y = 0; y < XN; ++y) acc[x][y] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[kc & 1][y], fa[kc & 1][x], acc[x][y], 0, 0, 0);
    };
    // What this wave has asked for is there - all of it, or all but the newest `LEFT` steps' loads - and everyone is here.
    auto meet = [&](auto left) __attribute__((always_inline)) {
        constexpr int LEFT = ALIGNED ? decltype(left)::value * (NA + NB) : 0;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LEFT) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    typedef std::integral_constant<int, 0> all_t;
    if constexpr (!ALIGNED && STAGES > 1) {
        // Any alignment: through registers, a step's loads under way while the last one is multiplied
        i4_t va[NA], vb[NB];
        const int8_t *pa[NA], *pb[NB];
#pragma unroll
        for (int i = 0; i < NA; ++i) pa[i] = g.a + std::min<int64_t>(m0 + (wave * NA + i) * 8 + (lane >> 3), g.m - 1) * g.lda + 16 * (lane & 7);
#pragma unroll
        for (int i = 0; i < NB; ++i) pb[i] = g.b + std::min<int64_t>(n0 + (wave * NB + i) * 8 + (lane >> 3), g.n - 1) * g.ldb + 16 * (lane & 7);
        auto load = [&](int s) __attribute__((always_inline)) {
            if ((s + 1) * kTK <= g.k) {
#pragma unroll
                for (int i = 0; i < NA; ++i) va[i] = bytes16(pa[i] + s * kTK);
#pragma unroll
                for (int i = 0; i < NB; ++i) vb[i] = bytes16(pb[i] + s * kTK);
            } else {
                const int n = g.k - 16 * (lane & 7);
#pragma unroll
                for (int i = 0; i < NA; ++i) va[i] = load16<false>(pa[i], s * kTK, n);
#pragma unroll
                for (int i = 0; i < NB; ++i) vb[i] = load16<false>(pb[i], s * kTK, n);
            }
        };
        auto store = [&](int buf) __attribute__((always_inline)) {
            int8_t* to = s_buf + buf * STAGE;
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int r = (wave * NA + i) * 8 + (lane >> 3);
                *reinterpret_cast<i4_t*>(to + r * kTK + 16 * ((lane & 7) ^ ((r >> 1) & 7))) = va[i];
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int r = (wave * NB + i) * 8 + (lane >> 3);
                *reinterpret_cast<i4_t*>(to + (TM + r) * kTK + 16 * ((lane & 7) ^ ((r >> 1) & 7))) = vb[i];
            }
        };
        if (steps) {
            load(0);
            store(0);
        }
        for (int s = 0; s < steps; ++s) {
            meet(all_t());      // step s is there, and everyone is done with the other buffer
            if (s + 1 < steps) load(s + 1);
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                read(s & 1, kc);
                multiply(kc);
            }
            if (s + 1 < steps) store((s + 1) & 1);
        }
    } else if constexpr (STAGES == 1) {
        if (steps) put(0, 0);
        for (int s = 0; s < steps; ++s) {
            if (s) {
                meet(all_t());      // everyone is done with the last step
                put(s, 0);
            }
            meet(all_t());
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                read(0, kc);
                multiply(kc);
            }
        }
    } else if (steps) {
        // Fragments are read one quarter of a step ahead.  The last quarter's are in registers when the waves meet: the buffer is free for the step STAGES on,
        // whose loads have STAGES - 1 steps to arrive, and the next step's first fragments are read beside the last products.
        typedef std::integral_constant<int, STAGES - 2> later_t;
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
            if (s < steps) put(s, s);
        if (STAGES <= steps) meet(std::integral_constant<int, STAGES - 1>());
        else meet(all_t());
        read(0, 0);
        int buf = 0;
        for (int s = 0; s < steps; ++s) {
            const int next = buf == STAGES - 1 ? 0 : buf + 1;
#pragma unroll
            for (int kc = 0; kc < KC; ++kc) {
                if (kc + 1 < KC) {
                    read(buf, kc + 1);
                } else if (s + 1 < steps) {
                    if (s + STAGES - 1 < steps) meet(later_t());
                    else meet(all_t());
                    if (s + STAGES < steps) put(s + STAGES, buf);
                    read(next, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                multiply(kc);
                __builtin_amdgcn_sched_barrier(0);
            }
            buf = next;
        }
    }
    if (int(threadIdx.x) < TN) s_scale[threadIdx.x] = my_scale, s_bias[threadIdx.x] = my_bias;
    // C fragment: column (lane & 31) = row m of the output, register rows = 4 consecutive n at a time.  Written through LDS, 32 rows of each wave at a time, so
    // that lanes write neighbouring bytes of a whole row of the tile: parts of memory lines cost as much as whole ones.
    // (Waves meet here with their LDS work done, not their stores: those of the last rows may be under way while the next ones are made.)
    auto meet_lds = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    constexpr int PIECE = 16 / int(sizeof(O)), LPR = TN / PIECE, RPI = 64 / LPR;      // elements of 16 bytes, lanes of a row, rows of an instruction
    const int cols = int(std::min<int64_t>(TN, g.n - n0));
#pragma unroll
    for (int x = 0; x < XM; ++x) {
        meet_lds();
#pragma unroll
        for (int y = 0; y < XN; ++y)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                typedef O o4 __attribute__((ext_vector_type(4)));
                const int c = wn + 32 * y + 8 * q + 4 * half;
                const float4 sb = *reinterpret_cast<const float4*>(s_scale + c);
                const float4 bi = *reinterpret_cast<const float4*>(s_bias + c);
                const float sa = row_scale[x];
                const o4 v = {finish<O>(acc[x][y][4 * q], sa, sb.x, bi.x), finish<O>(acc[x][y][4 * q + 1], sa, sb.y, bi.y),
                              finish<O>(acc[x][y][4 * q + 2], sa, sb.z, bi.z), finish<O>(acc[x][y][4 * q + 3], sa, sb.w, bi.w)};
                *reinterpret_cast<o4*>(s_buf + ((wave % WM) * 32 + l31) * OROW + c * int(sizeof(O))) = v;
            }
        meet_lds();
        constexpr int RPW = 32 * WM / WAVES;      // rows of a wave
#pragma unroll
        for (int i = 0; i < RPW / RPI; ++i) {
            const int r = wave * RPW + i * RPI + lane / LPR, c = (lane % LPR) * PIECE;
            const int64_t m = m0 + (r / 32) * 32 * XM + 32 * x + r % 32;
            if (m >= g.m || c >= cols) continue;
            const i4_t v = *reinterpret_cast<const i4_t*>(s_buf + r * OROW + c * int(sizeof(O)));
            O* out = static_cast<O*>(g.out) + m * g.ldo + n0 + c;
            if (vec) *reinterpret_cast<i4_t*>(out) = v;      // whole 16-byte pieces (n and the row stride are multiples of a piece)
            else if (c + PIECE <= cols) __builtin_memcpy(out, &v, 16);
            else
                for (int k = 0; k < cols - c; ++k) out[k] = *reinterpret_cast<const O*>(s_buf + r * OROW + (c + k) * int(sizeof(O)));
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- one side short
// `few` (at most 16 FT rows) against `many`: 16 rows of `many` belong to KS waves, each with its part of K; a workgroup of 4 waves takes 64 / KS rows.
// 16x16x64 matrix instruction: the register rows are rows of `many`, the columns rows of `few`.  A lane reads 32 consecutive bytes of a row per step,
// 4 lanes a whole 128-byte line.
struct QmmFewArgs {
    const int8_t *few, *many;
    const float *s_few, *s_many, *bias;
    void* out;
    int64_t n_many, ld_few, ld_many, o_few, o_many;     // output strides along either side
    int n_few, k, bias_many, vec;                              // bias_many: the bias belongs to `many`'s rows
};

template <typename O, int FT, bool ALIGNED, int KS>
__global__ __launch_bounds__(256) void matmul_q8_few_kernel(QmmFewArgs g) {
    static_assert(KS == 1 || KS == 4, "a workgroup's waves have a block of rows each, or all the same");
    __shared__ int s_part[KS - 1 ? KS - 1 : 1][FT * 4][64];
    const int lane = threadIdx.x & 63, wave = KS == 1 ? 0 : threadIdx.x >> 6, l15 = lane & 15, quad = lane >> 4;
    const int64_t r0 = (KS == 1 ? int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6) : int64_t(blockIdx.x)) * 16;
    const int64_t mr = std::min<int64_t>(r0 + l15, g.n_many - 1);       // rows past the end are read as the last one and not written
    const int8_t* many = g.many + mr * g.ld_many;
    const int8_t* few[FT];
#pragma unroll
    for (int f = 0; f < FT; ++f) few[f] = g.few + int64_t(std::min(16 * f + l15, g.n_few - 1)) * g.ld_few;
    i4_t acc[FT];
#pragma unroll
    for (int f = 0; f < FT; ++f) acc[f] = i4_t{0, 0, 0, 0};
    const int steps = (g.k + 127) / 128, per = (steps + KS - 1) / KS;
    const int s1 = std::min(steps, (wave + 1) * per);
    auto load = [&](i4_t (&v)[2 * FT + 2], int s, auto get) __attribute__((always_inline)) {
        const int k = s * 128 + quad * 32;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v[h] = get(many, k + 16 * h);
#pragma unroll
            for (int f = 0; f < FT; ++f) v[2 * f + 2 + h] = get(few[f], k + 16 * h);
        }
    };
    auto multiply = [&](const i4_t (&v)[2 * FT + 2]) __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int f = 0; f < FT; ++f) acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(v[h], v[2 * f + 2 + h], acc[f], 0, 0, 0);
    };
    auto plain = [](const int8_t* row, int k) __attribute__((always_inline)) {
        if constexpr (ALIGNED) return *reinterpret_cast<const i4_t*>(row + k);
        Words5 w;
        w.load(row + k);
        return w.get();
    };
    const int whole = std::min(s1, g.k / 128);
    int s = wave * per;
    // Whole steps, with no end to look for: the loads of AHEAD steps under way at once
    constexpr int AHEAD = KS == 1 ? 2 : 4;
    i4_t v[AHEAD][2 * FT + 2];
    for (; s + AHEAD <= whole; s += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) load(v[u], s + u, plain);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) multiply(v[u]);
    }
    for (; s < whole; ++s) {
        load(v[0], s, plain);
        multiply(v[0]);
    }
    if (s < s1) {      // the last, partial one
        load(v[0], s, [&](const int8_t* row, int k) __attribute__((always_inline)) { return load16<ALIGNED>(row, k, g.k); });
        multiply(v[0]);
    }
    if constexpr (KS > 1) {
        if (wave > 0) {
#pragma unroll
            for (int f = 0; f < FT; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) s_part[wave - 1][4 * f + i][lane] = acc[f][i];
        }
        __syncthreads();
        if (wave > 0) return;
#pragma unroll
        for (int f = 0; f < FT; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int w = 0; w < KS - 1; ++w) acc[f][i] += s_part[w][4 * f + i][lane];
    }
    const int64_t r = r0 + 4 * quad;
    if (r >= g.n_many) return;
    const int rows = int(std::min<int64_t>(4, g.n_many - r));
    float sm[4], bm[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        sm[i] = g.s_many[r + std::min(i, rows - 1)];
        bm[i] = g.bias && g.bias_many ? g.bias[r + std::min(i, rows - 1)] : 0.f;
    }
#pragma unroll
    for (int f = 0; f < FT; ++f) {
        const int row = 16 * f + l15;
        if (row >= g.n_few) continue;
        const float sf = g.s_few[row], bf = g.bias && !g.bias_many ? g.bias[row] : 0.f;
        typedef O o4 __attribute__((ext_vector_type(4)));
        o4 v;
        // the left side's scale first, whichever side is the short one
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = g.bias_many ? finish<O>(acc[f][i], sf, sm[i], bm[i]) : finish<O>(acc[f][i], sm[i], sf, bf);
        O* out = static_cast<O*>(g.out) + row * g.o_few + r * g.o_many;
        if (g.vec && rows == 4) {
            *reinterpret_cast<o4*>(out) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < rows) out[i * g.o_many] = v[i];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
// 64 x 8 192 x 8 192: 42 us streamed, 21 us as tiles of 64 x 64; 32 x 8 192 x 8 192: 24 us and 21, but with short sides on both ends (24 x 356 x 2 490)
// 9 and 25
constexpr int kFewRows = 32;
// 1 x 1.6 M x 64: 27 us with a wave's own rows, 76 with K split over a workgroup's waves; 1 x 400 k x 512: 31 and 33; x 50 k x 1 024: 11.1 and 10.2;
// 24 x 356 x 2 490: 20 and 9
constexpr int kFewWholeK = 512;

// A launch has fewer than 2^32 threads: 256 for 64 or 16 rows against a few, or for 128 x 128 of the output, 512 for 128 x 256
static bool matmul_q8_fits(int64_t m, int64_t n, int64_t k) {
    if (m > (int64_t(1) << 31) - 256 || n > (int64_t(1) << 31) - 256) return false;
    if (std::min(m, n) <= kFewRows) return cdiv64(std::max(m, n), k <= kFewWholeK ? 64 : 16) < (int64_t(1) << 24);
    return cdiv64(m, 128) * std::max(cdiv64(n, 128), 2 * cdiv64(n, 256)) < (int64_t(1) << 24) - 8;
}

template <typename O, bool ALIGNED>
static void matmul_q8_launch(const QmmArgs& g, hipStream_t st) {
    if (std::min(g.m, g.n) <= kFewRows) {
        const bool left = g.m <= g.n;      // which side is short
        QmmFewArgs f{left ? g.a : g.b, left ? g.b : g.a, left ? g.sa : g.sb, left ? g.sb : g.sa, g.bias, g.out, left ? g.n : g.m, left ? g.lda : g.ldb,
                     left ? g.ldb : g.lda, left ? g.ldo : 1, left ? 1 : g.ldo, int(left ? g.m : g.n), g.k, left ? 1 : 0, 0};
        f.vec = left && aligned_to(g.out, g.ldo * int64_t(sizeof(O)), 4 * sizeof(O));
        auto launch = [&](auto ft, auto ks) {
            matmul_q8_few_kernel<O, decltype(ft)::value, ALIGNED, decltype(ks)::value><<<dim3(unsigned(cdiv64(f.n_many, 64 / decltype(ks)::value))), dim3(256), 0, st>>>(f);
        };
        typedef std::integral_constant<int, 1> one_t;
        typedef std::integral_constant<int, 2> two_t;
        typedef std::integral_constant<int, 4> four_t;
        if (g.k <= kFewWholeK) f.n_few <= 16 ? launch(one_t(), one_t()) : launch(two_t(), one_t());
        else f.n_few <= 16 ? launch(one_t(), four_t()) : launch(two_t(), four_t());
        return;
    }
    const int vec = (g.n * int64_t(sizeof(O))) % 16 == 0 && aligned_to(g.out, g.ldo * int64_t(sizeof(O)), 16);
    auto tiles = [&](int tm, int tn) { return cdiv64(g.m, tm) * cdiv64(g.n, tn); };
    auto grid = [&](int tm, int tn) { return dim3(unsigned((tiles(tm, tn) + 7) / 8 * 8)); };
    auto go = [&](auto kernel, int tm, int tn, int threads, int band) {
        kernel<<<grid(tm, tn), dim3(threads), 0, st>>>(g, int(cdiv64(g.m, tm)), int(cdiv64(g.n, tn)), band, vec);
    };
    // Few K steps: the output's traffic counts, one buffer and many workgroups a CU.  With few tiles smaller ones (943 x 1 682 x 64 bfloat16: 5.4 us, 6.8 as
    // 128 x 128).  Rows of the output seldom begin on a memory line, so parts of one line come from two tiles: float32 tiles are wider and their bands are
    // narrower, so that these meet sooner (4 096 x 26 744 x 256: 104 us, 120 as 128 x 128 in bands of 8 rows; bfloat16: 72 both ways, x 128: 61 and 60,
    // with rows on 128 bytes 54 and 49).
    constexpr bool wide = sizeof(O) == 4;
    if (g.k <= 2 * kTK && tiles(128, 128) < 1024) go(matmul_q8_tile_kernel<O, ALIGNED, 2, 2, 1, 2, 1>, 64, 128, 256, 4);
    else if (g.k <= 2 * kTK) go(matmul_q8_tile_kernel<O, ALIGNED, 2, wide ? 4 : 2, 2, 2, 1>, 128, wide ? 256 : 128, wide ? 512 : 256, wide ? 2 : 8);
    // Many: the largest tile of which there are enough for the CUs; the smallest has four buffers, as little work covers its loads.
    else if (tiles(256, 256) >= 192) go(matmul_q8_tile_kernel<O, ALIGNED, 2, 4, 4, 2, 2>, 256, 256, 512, 8);
    else if (tiles(128, 128) >= 192) go(matmul_q8_tile_kernel<O, ALIGNED, 2, 2, 2, 2, 2>, 128, 128, 256, 8);
    else go(matmul_q8_tile_kernel<O, ALIGNED, 2, 2, 1, 1, 4>, 64, 64, 256, 8);
}

}  // namespace hwer

using namespace hwer;

extern "C" int hwer_matmul_q8(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* b, int64_t ldb, const float* b_scale, const float* bias,
                              int64_t m, int64_t n, int64_t k, void* out, int64_t ldo, int out_dtype, void* stream) {
    if (!known_dtype(out_dtype)) return fail(HWER_EINVAL, "matmul_q8: unknown output type %d", out_dtype);
    if (m < 0 || n < 0 || k < 0 || k > 131071) return fail(HWER_EINVAL, "matmul_q8: m=%lld, n=%lld, k=%lld (k <= 131071: sums stay in 32 bits)", (long long)m, (long long)n, (long long)k);
    if (m == 0 || n == 0) return HWER_OK;
    if (!matmul_q8_fits(m, n, k))
        return fail(HWER_EINVAL, "matmul_q8: m=%lld, n=%lld: too many tiles for one call", (long long)m, (long long)n);
    if ((k && (!a || !b)) || !a_scale || !b_scale || !out) return fail(HWER_EINVAL, "matmul_q8: null operand");
    if (lda < k || ldb < k || ldo < n) return fail(HWER_EINVAL, "matmul_q8: a row stride is below the row's length");
    const QmmArgs g{a, b, a_scale, b_scale, bias, out, m, n, lda, ldb, ldo, int(k)};
    hipStream_t st = as_stream(stream);
    const bool al = k % 16 == 0 && aligned_to(a, lda, 16) && aligned_to(b, ldb, 16) && std::max(lda, ldb) < (1 << 23);      // (a panel's bytes in 32 bits)
    if (out_dtype == HWER_F32) al ? matmul_q8_launch<float, true>(g, st) : matmul_q8_launch<float, false>(g, st);
    else if (out_dtype == HWER_F16) al ? matmul_q8_launch<f16_t, true>(g, st) : matmul_q8_launch<f16_t, false>(g, st);
    else al ? matmul_q8_launch<bf16_t, true>(g, st) : matmul_q8_launch<bf16_t, false>(g, st);
    return check_launch("matmul_q8");
}
