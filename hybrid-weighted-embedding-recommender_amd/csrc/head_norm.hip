// Row kernels of the learned head: root-mean-square norm with the residual's addition, its gradients, and rows in 8 bits with a scale.
//
//   h = round_T(x + residual)                 r = 1 / sqrt(mean_j h_j^2 + eps)          y_j = round_T(h_j r w_j)
//   dx_j = r (w_j dy_j - h_j r^2 mean_i(h_i w_i dy_i)) + dh_j                              dw_j = sum_rows dy_j h_j r
//   v_j = h_j w_j      q_j = round_half_even(127 v_j / max|v|)      scale = max|v| r / 127  (r = 1 without the norm)
// The norm is taken of the ROUNDED sum h, so that the backward pass, which has h only, is the gradient of what the forward pass computed.
// The codes do not depend on r: they are quotients of two exact values, rounded once, and equal in every implementation that rounds right.
//
// All three are bound by memory: a row is read once, held in registers (raw, 16 bytes per load), reduced over the lanes that hold it and
// written once.  T lanes hold a row (16, a wave, 4 waves, 16 waves) with VPT vectors each; a workgroup keeps its share of the weights in
// registers and walks over rows.
#include <algorithm>

#include "head_common.h"

namespace hwer {

constexpr int kNormBlock = 256;     // threads of a workgroup unless one row takes more

template <typename E, int N>
struct alignas(sizeof(E) * N) Pack {
    E e[N];
};

// v / top rounded to a code: the float32 quotient decides unless it is close to a border between two codes (its error is below 127 * 2^-21),
// then the quotient in 64 bits does, where h * w is exact for every type (24 + 24 bits); so it does where 127 / top leaves float32's range
__device__ __forceinline__ int q8_code(float v, float inv, double exact_v, double top) {
    const float t = v * inv;
    float c = rintf(t);
    if (inv > 1e32f || fabsf(fabsf(t - c) - 0.5f) < 1e-4f) c = float(rint(127.0 * exact_v / top));
    return int(c);
}

// ---------------------------------------------------------------------------------------------------------------- forward
struct NormFwdArgs {
    const void *x, *res, *w;
    void *y, *h;            // y: T rows (Q8 = false) or int8 codes
    float* scale;
    int64_t rows, ldx, ldr, ldy, ldh;
    int d;
    float eps;
    int norm;               // 0: r = 1 (codes only)
};

// sum over the T threads of a row; T > 64: over the waves of the workgroup through `slots` (two alternating sets: one barrier per row)
template <int T>
__device__ __forceinline__ float row_sum(float v, float* slots, int flip) {
    v = lanes_sum<(T < 64 ? T : 64)>(v);
    if constexpr (T > 64) {
        float* s = slots + flip * (T / 64);
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = s[0];
#pragma unroll
        for (int i = 1; i < T / 64; ++i) v += s[i];
    }
    return v;
}

template <typename E, typename W, int T, int VPT, int VW, bool Q8>
__global__ __launch_bounds__(T > kNormBlock ? T : kNormBlock) void norm_fwd_kernel(NormFwdArgs a) {
    constexpr int B = T > kNormBlock ? T : kNormBlock, R = B / T;     // R rows at a time
    __shared__ float s_sum[2 * (T > 64 ? T / 64 : 1)];
    __shared__ double s_top[2 * (T > 64 ? T / 64 : 1)];
    typedef Pack<E, VW> PE;
    const int t = threadIdx.x % T, sub = threadIdx.x / T;
    const E* xp = static_cast<const E*>(a.x);
    const E* rp = static_cast<const E*>(a.res);
    const W* wp = static_cast<const W*>(a.w);
    float w[VPT * VW];
#pragma unroll
    for (int p = 0; p < VPT; ++p)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const int c = (p * T + t) * VW + j;
            w[p * VW + j] = (wp && c < a.d) ? float(wp[c]) : 1.f;
        }
    const float inv_d = 1.f / float(a.d);
    int flip = 0;
    // every thread of the workgroup makes the same number of turns: the barriers of row_sum are met by all
    for (int64_t base = int64_t(blockIdx.x) * R; base < a.rows; base += int64_t(gridDim.x) * R, flip ^= 1) {
        const int64_t r = base + sub;
        const bool on = r < a.rows;
        PE h[VPT];
        float ss = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; ++p) {
            const int c = (p * T + t) * VW;
            const bool in = on && c < a.d;        // VW > 1 only where d is a multiple of VW
#pragma unroll
            for (int j = 0; j < VW; ++j) h[p].e[j] = E(0.f);
            if (in) {
                h[p] = *reinterpret_cast<const PE*>(xp + r * a.ldx + c);
                if (rp) {
                    const PE q = *reinterpret_cast<const PE*>(rp + r * a.ldr + c);
#pragma unroll
                    for (int j = 0; j < VW; ++j) h[p].e[j] = E(float(h[p].e[j]) + float(q.e[j]));
                    *reinterpret_cast<PE*>(static_cast<E*>(a.h) + r * a.ldh + c) = h[p];
                }
            }
#pragma unroll
            for (int j = 0; j < VW; ++j) ss = fmaf(float(h[p].e[j]), float(h[p].e[j]), ss);
        }
        float rstd = 1.f;
        if (a.norm) rstd = 1.f / sqrtf(row_sum<T>(ss, s_sum, flip) * inv_d + a.eps);
        if constexpr (!Q8) {
#pragma unroll
            for (int p = 0; p < VPT; ++p) {
                const int c = (p * T + t) * VW;
                if (on && c < a.d) {
                    PE o;
#pragma unroll
                    for (int j = 0; j < VW; ++j) o.e[j] = E(float(h[p].e[j]) * rstd * w[p * VW + j]);
                    *reinterpret_cast<PE*>(static_cast<E*>(a.y) + r * a.ldy + c) = o;
                }
            }
        } else {
            double top = 0.0;
            float bad = 0.f;      // becomes NaN with any NaN or infinity among the products
#pragma unroll
            for (int p = 0; p < VPT; ++p)
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const bool in = (p * T + t) * VW + j < a.d;
                    const double v = in ? double(float(h[p].e[j])) * double(w[p * VW + j]) : 0.0;
                    top = fmax(top, fabs(v));
                    bad = fmaf(float(v), 0.f, bad);
                }
            if (!(bad == 0.f)) top = INFINITY;
            top = lanes_max<(T < 64 ? T : 64)>(top);
            if constexpr (T > 64) {
                double* s = s_top + flip * (T / 64);
                if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top;
                __syncthreads();
                top = s[0];
#pragma unroll
                for (int i = 1; i < T / 64; ++i) top = fmax(top, s[i]);
            }
            const bool fine = top > 0.0 && top < double(INFINITY);
            const float inv = fine ? 127.f / float(top) : 0.f;
            if (on && t == 0) a.scale[r] = top < double(INFINITY) ? float(top) * rstd / 127.f : NAN;   // a row with a NaN or an infinity: codes 0, scale NaN
#pragma unroll
            for (int p = 0; p < VPT; ++p) {
                const int c = (p * T + t) * VW;
                if (on && c < a.d) {
                    Pack<int8_t, VW> o;
#pragma unroll
                    for (int j = 0; j < VW; ++j) {
                        const float hv = float(h[p].e[j]), wv = w[p * VW + j];
                        o.e[j] = fine ? int8_t(q8_code(hv * wv, inv, double(hv) * double(wv), top)) : int8_t(0);
                    }
                    *reinterpret_cast<Pack<int8_t, VW>*>(static_cast<int8_t*>(a.y) + r * a.ldy + c) = o;
                }
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------- backward
struct NormBwdArgs {
    const void *dy, *h, *w, *dh;
    void* dx;
    float* dw_part;         // (gridDim.x, d) partial sums, nullable
    int64_t rows, lddy, ldh, lddh, lddx;
    int d;
    float eps;
};

template <typename E, typename W, int T, int VPT, int VW>
__global__ __launch_bounds__(T > kNormBlock ? T : kNormBlock) void norm_bwd_kernel(NormBwdArgs a) {
    constexpr int B = T > kNormBlock ? T : kNormBlock, R = B / T;
    __shared__ float s_sum[4 * (T > 64 ? T / 64 : 1)];
    __shared__ float s_dw[R > 1 ? B * VPT * VW : 1];
    typedef Pack<E, VW> PE;
    const int t = threadIdx.x % T, sub = threadIdx.x / T;
    const W* wp = static_cast<const W*>(a.w);
    float w[VPT * VW], dw[VPT * VW];
#pragma unroll
    for (int p = 0; p < VPT; ++p)
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            const int c = (p * T + t) * VW + j;
            w[p * VW + j] = (wp && c < a.d) ? float(wp[c]) : 1.f;
            dw[p * VW + j] = 0.f;
        }
    const float inv_d = 1.f / float(a.d);
    int flip = 0;
    for (int64_t base = int64_t(blockIdx.x) * R; base < a.rows; base += int64_t(gridDim.x) * R, flip ^= 1) {
        const int64_t r = base + sub;
        const bool on = r < a.rows;
        PE h[VPT], g[VPT];
        float ss = 0.f, sc = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; ++p) {
            const int c = (p * T + t) * VW;
#pragma unroll
            for (int j = 0; j < VW; ++j) h[p].e[j] = g[p].e[j] = E(0.f);
            if (on && c < a.d) {
                h[p] = *reinterpret_cast<const PE*>(static_cast<const E*>(a.h) + r * a.ldh + c);
                g[p] = *reinterpret_cast<const PE*>(static_cast<const E*>(a.dy) + r * a.lddy + c);
            }
        }
#pragma unroll
        for (int p = 0; p < VPT; ++p)
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float hv = float(h[p].e[j]);
                ss = fmaf(hv, hv, ss);
                sc = fmaf(hv * w[p * VW + j], float(g[p].e[j]), sc);
            }
        ss = lanes_sum<(T < 64 ? T : 64)>(ss);
        sc = lanes_sum<(T < 64 ? T : 64)>(sc);
        if constexpr (T > 64) {
            float* s = s_sum + flip * 2 * (T / 64);
            if ((threadIdx.x & 63) == 0) {
                s[threadIdx.x >> 6] = ss;
                s[T / 64 + (threadIdx.x >> 6)] = sc;
            }
            __syncthreads();
            ss = s[0];
            sc = s[T / 64];
#pragma unroll
            for (int i = 1; i < T / 64; ++i) ss += s[i], sc += s[T / 64 + i];
        }
        const float rstd = 1.f / sqrtf(ss * inv_d + a.eps);
        const float back = (sc * inv_d) * rstd * rstd;
#pragma unroll
        for (int p = 0; p < VPT; ++p) {
            const int c = (p * T + t) * VW;
            if (on && c < a.d) {
                PE o, add;
                if (a.dh) add = *reinterpret_cast<const PE*>(static_cast<const E*>(a.dh) + r * a.lddh + c);
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const float hv = float(h[p].e[j]), gv = float(g[p].e[j]);
                    float v = rstd * (w[p * VW + j] * gv - hv * back);
                    if (a.dh) v += float(add.e[j]);
                    o.e[j] = E(v);
                    dw[p * VW + j] = fmaf(gv, hv * rstd, dw[p * VW + j]);
                }
                *reinterpret_cast<PE*>(static_cast<E*>(a.dx) + r * a.lddx + c) = o;
            }
        }
    }
    if (!a.dw_part) return;
    float* out = a.dw_part + int64_t(blockIdx.x) * a.d;
    if constexpr (R > 1) {      // the workgroup's R groups of rows, added in order
#pragma unroll
        for (int i = 0; i < VPT * VW; ++i) s_dw[i * B + threadIdx.x] = dw[i];
        __syncthreads();
        if (sub == 0) {
#pragma unroll
            for (int i = 0; i < VPT * VW; ++i) {
                float v = s_dw[i * B + t];
#pragma unroll
                for (int k = 1; k < R; ++k) v += s_dw[i * B + k * T + t];
                dw[i] = v;
            }
        }
    }
    if (sub == 0) {
#pragma unroll
        for (int p = 0; p < VPT; ++p)
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const int c = (p * T + t) * VW + j;
                if (c < a.d) out[c] = dw[p * VW + j];
            }
    }
}

// dw[c] = sum over the partials in a fixed order: a workgroup takes 32 columns, 32 threads of each column walk over the partials
template <typename W>
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n_part, int d, W* __restrict__ dw) {
    __shared__ float s[32][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), k = threadIdx.x >> 5;
    float v = 0.f;
    if (c < d)
        for (int i = k; i < n_part; i += 32) v += part[int64_t(i) * d + c];
    s[k][threadIdx.x & 31] = v;
    __syncthreads();
    if (k == 0 && c < d) {
        v = s[0][threadIdx.x];
        for (int i = 1; i < 32; ++i) v += s[i][threadIdx.x];
        dw[c] = W(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------- rows too wide for registers
constexpr int kWideThreads = 1024;

template <typename E, typename W, bool Q8>
__global__ __launch_bounds__(kWideThreads) void norm_fwd_wide_kernel(NormFwdArgs a) {
    __shared__ float s_sum[2 * (kWideThreads / 64)];
    __shared__ double s_top[kWideThreads / 64];
    const int t = threadIdx.x;
    const W* wp = static_cast<const W*>(a.w);
    int flip = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
        const E* x = static_cast<const E*>(a.x) + r * a.ldx;
        const E* q = a.res ? static_cast<const E*>(a.res) + r * a.ldr : nullptr;
        // the sum is formed again from the inputs in each pass: `h` may share memory with nothing, but is written once only
        auto value = [&](int c) { return q ? float(E(float(x[c]) + float(q[c]))) : float(x[c]); };
        float ss = 0.f;
        double top = 0.0;
        float bad = 0.f;
        for (int c = t; c < a.d; c += kWideThreads) {
            const float hv = value(c);
            ss = fmaf(hv, hv, ss);
            if (Q8) {
                const double v = double(hv) * double(wp ? float(wp[c]) : 1.f);
                top = fmax(top, fabs(v));
                bad = fmaf(float(v), 0.f, bad);
            }
        }
        float rstd = 1.f;
        if (a.norm) rstd = 1.f / sqrtf(row_sum<kWideThreads>(ss, s_sum, flip) / float(a.d) + a.eps);
        float inv = 0.f;
        bool fine = false;
        if (Q8) {
            if (!(bad == 0.f)) top = INFINITY;
            top = lanes_max<64>(top);
            __syncthreads();
            if ((t & 63) == 0) s_top[t >> 6] = top;
            __syncthreads();
            top = s_top[0];
            for (int i = 1; i < kWideThreads / 64; ++i) top = fmax(top, s_top[i]);
            fine = top > 0.0 && top < double(INFINITY);
            inv = fine ? 127.f / float(top) : 0.f;
            if (t == 0) a.scale[r] = top < double(INFINITY) ? float(top) * rstd / 127.f : NAN;
        }
        for (int c = t; c < a.d; c += kWideThreads) {
            const float hv = value(c), wv = wp ? float(wp[c]) : 1.f;
            if (a.res) static_cast<E*>(a.h)[r * a.ldh + c] = E(hv);
            if (Q8) static_cast<int8_t*>(a.y)[r * a.ldy + c] = fine ? int8_t(q8_code(hv * wv, inv, double(hv) * double(wv), top)) : int8_t(0);
            else static_cast<E*>(a.y)[r * a.ldy + c] = E(hv * rstd * wv);
        }
    }
}

// dx of a row, and the row's r into `rstd`; dw is then summed down the columns by norm_dw_wide_kernel
template <typename E, typename W>
__global__ __launch_bounds__(kWideThreads) void norm_bwd_wide_kernel(NormBwdArgs a, float* __restrict__ rstd_out) {
    __shared__ float s_sum[4 * (kWideThreads / 64)];
    const int t = threadIdx.x;
    const W* wp = static_cast<const W*>(a.w);
    int flip = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
        const E* h = static_cast<const E*>(a.h) + r * a.ldh;
        const E* g = static_cast<const E*>(a.dy) + r * a.lddy;
        float ss = 0.f, sc = 0.f;
        for (int c = t; c < a.d; c += kWideThreads) {
            const float hv = float(h[c]);
            ss = fmaf(hv, hv, ss);
            sc = fmaf(hv * (wp ? float(wp[c]) : 1.f), float(g[c]), sc);
        }
        ss = row_sum<kWideThreads>(ss, s_sum, flip);
        sc = row_sum<kWideThreads>(sc, s_sum + 2 * (kWideThreads / 64), flip);
        const float rstd = 1.f / sqrtf(ss / float(a.d) + a.eps);
        const float back = (sc / float(a.d)) * rstd * rstd;
        for (int c = t; c < a.d; c += kWideThreads) {
            float v = rstd * ((wp ? float(wp[c]) : 1.f) * float(g[c]) - float(h[c]) * back);
            if (a.dh) v += float(static_cast<const E*>(a.dh)[r * a.lddh + c]);
            static_cast<E*>(a.dx)[r * a.lddx + c] = E(v);
        }
        if (rstd_out && t == 0) rstd_out[r] = rstd;
    }
}

template <typename E>
__global__ __launch_bounds__(1024) void norm_dw_wide_kernel(NormBwdArgs a, const float* __restrict__ rstd, int rows_per_part) {
    __shared__ float s[16][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), k = threadIdx.x >> 6;
    const int64_t r0 = int64_t(blockIdx.y) * rows_per_part, r1 = r0 + rows_per_part < a.rows ? r0 + rows_per_part : a.rows;
    float v = 0.f;
    if (c < a.d)
        for (int64_t r = r0 + k; r < r1; r += 16)
            v = fmaf(float(static_cast<const E*>(a.dy)[r * a.lddy + c]), float(static_cast<const E*>(a.h)[r * a.ldh + c]) * rstd[r], v);
    s[k][threadIdx.x & 63] = v;
    __syncthreads();
    if (k == 0 && c < a.d) {
        for (int i = 1; i < 16; ++i) v += s[i][threadIdx.x];
        a.dw_part[int64_t(blockIdx.y) * a.d + c] = v;
    }
}

// ---------------------------------------------------------------------------------------------------------------- host
// How a row of d elements is held: T lanes with VPT vectors of VW elements.  The narrowest T whose lanes hold the row; T * VPT * VW >= d.
// A workgroup of 1 024 threads has 128 registers a thread: 16 elements each (32 spill in the backward kernel).
constexpr bool norm_fits(int t, int vpt, int vw) { return t < 1024 || vpt * vw <= 16; }
struct NormPlan {
    int t, vpt;      // t = 0: the wide kernels
};
static NormPlan norm_plan(int d, int vw) {
    static const NormPlan plans[] = {{16, 1}, {16, 2}, {64, 1}, {64, 2}, {64, 4}, {256, 2}, {256, 4}, {1024, 2}, {1024, 4}};
    for (const NormPlan& p : plans)
        if (int64_t(p.t) * p.vpt * vw >= d && norm_fits(p.t, p.vpt, vw)) return p;
    return {0, 0};
}

// workgroups of a launch: enough to fill the chip several times over, few enough that the weights are read once per many rows
static int norm_grid(int64_t rows, int t) {
    const int r = t >= kNormBlock ? 1 : kNormBlock / t;
    return int(std::min<int64_t>(cdiv64(rows, r), kMaxStreamBlocks));
}
// ... of a backward launch: each leaves a partial sum of the weights' gradient behind
static int norm_bwd_grid(int64_t rows, int t) {
    const int r = t >= kNormBlock ? 1 : kNormBlock / t;
    return int(std::min<int64_t>(cdiv64(rows, r), 1024));
}
constexpr int kWideDwParts = 32;

template <typename E, typename W, bool Q8, int VW>
static void norm_fwd_launch(const NormFwdArgs& a, hipStream_t st) {
    const NormPlan p = norm_plan(a.d, VW);
    const int grid = norm_grid(a.rows, p.t ? p.t : kWideThreads);
#define HWER_NORM_FWD(T, V) \
    if constexpr (norm_fits(T, V, VW))          \
        if (p.t == T && p.vpt == V) return norm_fwd_kernel<E, W, T, V, VW, Q8><<<dim3(grid), dim3(T > kNormBlock ? T : kNormBlock), 0, st>>>(a)
    HWER_NORM_FWD(16, 1); HWER_NORM_FWD(16, 2); HWER_NORM_FWD(64, 1); HWER_NORM_FWD(64, 2); HWER_NORM_FWD(64, 4);
    HWER_NORM_FWD(256, 2); HWER_NORM_FWD(256, 4); HWER_NORM_FWD(1024, 2); HWER_NORM_FWD(1024, 4);
#undef HWER_NORM_FWD
    norm_fwd_wide_kernel<E, W, Q8><<<dim3(grid), dim3(kWideThreads), 0, st>>>(a);
}

template <typename E, typename W>
static void norm_fwd_typed(const NormFwdArgs& a, bool q8, hipStream_t st) {
    constexpr int VW = 16 / int(sizeof(E));
    const int64_t e = int64_t(sizeof(E));
    // wide loads where every row of every operand starts on 16 bytes (codes: on VW bytes) and ends with a whole vector; single elements otherwise
    const bool vec = a.d % VW == 0 && aligned_to(a.x, a.ldx * e, 16) && (!a.res || (aligned_to(a.res, a.ldr * e, 16) && aligned_to(a.h, a.ldh * e, 16))) &&
                     (q8 ? aligned_to(a.y, a.ldy, VW) : aligned_to(a.y, a.ldy * e, 16));
    if (q8) vec ? norm_fwd_launch<E, W, true, VW>(a, st) : norm_fwd_launch<E, W, true, 1>(a, st);
    else vec ? norm_fwd_launch<E, W, false, VW>(a, st) : norm_fwd_launch<E, W, false, 1>(a, st);
}

static int norm_fwd_any(const NormFwdArgs& a, int dtype, int w_dtype, bool q8, const char* what, void* stream) {
    hipStream_t st = as_stream(stream);
    const bool w32 = !a.w || w_dtype == HWER_F32;
    if (dtype == HWER_F32) norm_fwd_typed<float, float>(a, q8, st);
    else if (dtype == HWER_F16) w32 ? norm_fwd_typed<f16_t, float>(a, q8, st) : norm_fwd_typed<f16_t, f16_t>(a, q8, st);
    else w32 ? norm_fwd_typed<bf16_t, float>(a, q8, st) : norm_fwd_typed<bf16_t, bf16_t>(a, q8, st);
    return check_launch(what);
}

static int norm_check(const char* what, const void* x, int64_t ldx, const void* w, int w_dtype, int64_t rows, int d, int dtype, float eps) {
    if (!known_dtype(dtype)) return fail(HWER_EINVAL, "%s: unknown element type %d", what, dtype);
    if (w && w_dtype != HWER_F32 && w_dtype != dtype) return fail(HWER_EINVAL, "%s: the weights are float32 or of the rows' type", what);
    if (rows < 0 || d < 1) return fail(HWER_EINVAL, "%s: rows=%lld, d=%d", what, (long long)rows, d);
    if (rows && (!x || ldx < d)) return fail(HWER_EINVAL, "%s: null rows or a row stride below d", what);
    if (!(eps >= 0.f) || !(eps < INFINITY)) return fail(HWER_EINVAL, "%s: eps must be finite and not negative", what);
    return HWER_OK;
}

}  // namespace hwer

using namespace hwer;

extern "C" {

int hwer_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int weight_dtype, int64_t rows, int d, int dtype,
                  float eps, void* y, int64_t ldy, void* h, int64_t ldh, void* stream) {
    if (int rc = norm_check("rms_norm", x, ldx, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (rows == 0) return HWER_OK;
    if (!y || ldy < d || (residual && (!h || ldr < d || ldh < d))) return fail(HWER_EINVAL, "rms_norm: null output or a row stride below d");
    const NormFwdArgs a{x, residual, weight, y, h, nullptr, rows, ldx, ldr, ldy, ldh, d, eps, 1};
    return norm_fwd_any(a, dtype, weight_dtype, false, "rms_norm", stream);
}

int hwer_rms_norm_q8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int weight_dtype, int64_t rows, int d, int dtype,
                     int norm, float eps, int8_t* q, int64_t ldq, float* scale, void* h, int64_t ldh, void* stream) {
    if (int rc = norm_check("rms_norm_q8", x, ldx, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (rows == 0) return HWER_OK;
    if (!q || !scale || ldq < d || (residual && (!h || ldr < d || ldh < d))) return fail(HWER_EINVAL, "rms_norm_q8: null output or a row stride below d");
    const NormFwdArgs a{x, residual, weight, q, h, scale, rows, ldx, ldr, ldq, ldh, d, eps, norm ? 1 : 0};
    return norm_fwd_any(a, dtype, weight_dtype, true, "rms_norm_q8", stream);
}

size_t hwer_rms_norm_backward_workspace_bytes(int64_t rows, int d) {
    if (rows <= 0 || d < 1) return 16;
    // partial sums of dweight (at most 1 024 workgroups; rows too wide for registers: kWideDwParts and one r per row)
    return size_t(std::max<int64_t>(std::min<int64_t>(rows, 1024), kWideDwParts)) * d * 4 + size_t(rows) * 4;
}

int hwer_rms_norm_backward(const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* weight, int weight_dtype, const void* dh, int64_t lddh,
                           int64_t rows, int d, int dtype, float eps, void* dx, int64_t lddx, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = norm_check("rms_norm_backward", h, ldh, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (dweight && !weight) return fail(HWER_EINVAL, "rms_norm_backward: a gradient of weights that are not there");
    if (rows && (!dy || !dx || lddy < d || lddx < d || (dh && lddh < d))) return fail(HWER_EINVAL, "rms_norm_backward: null rows or a row stride below d");
    if (dweight && (!workspace || workspace_bytes < hwer_rms_norm_backward_workspace_bytes(rows, d)))
        return fail(HWER_EWORKSPACE, "rms_norm_backward: workspace of %zu bytes needed", hwer_rms_norm_backward_workspace_bytes(rows, d));
    hipStream_t st = as_stream(stream);
    NormBwdArgs a{dy, h, weight, dh, dx, dweight ? static_cast<float*>(workspace) : nullptr, rows, lddy, ldh, lddh, lddx, d, eps};
    int parts = 0;
    auto run = [&](auto e, auto wt) {
        typedef decltype(e) E;
        typedef decltype(wt) W;
        constexpr int VW = 16 / int(sizeof(E));
        const int64_t s = int64_t(sizeof(E));
        const bool vec = d % VW == 0 && aligned_to(dy, lddy * s, 16) && aligned_to(h, ldh * s, 16) && aligned_to(dx, lddx * s, 16) && (!dh || aligned_to(dh, lddh * s, 16));
        const NormPlan p = norm_plan(d, vec ? VW : 1);
        if (p.t == 0) {
            float* rstd = a.dw_part ? a.dw_part + int64_t(kWideDwParts) * d : nullptr;
            const int grid = norm_grid(rows, kWideThreads);
            norm_bwd_wide_kernel<E, W><<<dim3(grid), dim3(kWideThreads), 0, st>>>(a, rstd);
            if (a.dw_part) {
                parts = int(std::min<int64_t>(kWideDwParts, rows));
                norm_dw_wide_kernel<E><<<dim3((d + 63) / 64, parts), dim3(1024), 0, st>>>(a, rstd, int(cdiv64(rows, parts)));
            }
            return;
        }
        parts = norm_bwd_grid(rows, p.t);
#define HWER_NORM_BWD(T, V, VWX)                                                                                                            \
    if constexpr (norm_fits(T, V, VWX))                                                                                                     \
        if (p.t == T && p.vpt == V) return norm_bwd_kernel<E, W, T, V, VWX><<<dim3(parts), dim3(T > kNormBlock ? T : kNormBlock), 0, st>>>(a)
#define HWER_NORM_BWD_ALL(VWX)                                                                                                              \
    HWER_NORM_BWD(16, 1, VWX); HWER_NORM_BWD(16, 2, VWX); HWER_NORM_BWD(64, 1, VWX); HWER_NORM_BWD(64, 2, VWX); HWER_NORM_BWD(64, 4, VWX); \
    HWER_NORM_BWD(256, 2, VWX); HWER_NORM_BWD(256, 4, VWX); HWER_NORM_BWD(1024, 2, VWX); HWER_NORM_BWD(1024, 4, VWX)
        if (vec) {
            HWER_NORM_BWD_ALL(VW);
        } else {
            HWER_NORM_BWD_ALL(1);
        }
#undef HWER_NORM_BWD_ALL
#undef HWER_NORM_BWD
    };
    const bool w32 = !weight || weight_dtype == HWER_F32;
    if (rows) {
        if (dtype == HWER_F32) run(float(), float());
        else if (dtype == HWER_F16) w32 ? run(f16_t(), float()) : run(f16_t(), f16_t());
        else w32 ? run(bf16_t(), float()) : run(bf16_t(), bf16_t());
        if (int rc = check_launch("rms_norm_backward")) return rc;
    }
    if (dweight) {      // no rows: a sum over nothing, zeros
        const dim3 grid((d + 31) / 32);
        if (w32) norm_dw_kernel<float><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, d, static_cast<float*>(dweight));
        else if (dtype == HWER_F16) norm_dw_kernel<f16_t><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, d, static_cast<f16_t*>(dweight));
        else norm_dw_kernel<bf16_t><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, d, static_cast<bf16_t*>(dweight));
    }
    return check_launch("rms_norm_backward(dweight)");
}

}  // extern "C"
