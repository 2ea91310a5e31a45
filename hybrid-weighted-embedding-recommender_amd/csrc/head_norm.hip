// Row kernels of the learned head: root-mean-square norm with the residual's addition, its gradients, and rows in 8 bits with a scale.
//
//   h = round_T(x + residual)                 r = 1 / sqrt(mean_j h_j^2 + eps)          y_j = round_T(h_j r w_j)
//   dx_j = r (w_j dy_j - h_j r^2 mean_i(h_i w_i dy_i)) + dh_j                              dw_j = sum_rows dy_j h_j r
//   v_j = h_j w_j      q_j = round_half_even(127 v_j / max|v|)      scale = max|v| r / 127  (r = 1 without the norm)
// The norm is taken of the ROUNDED sum h, so that the backward pass, which has h only, is the gradient of what the forward pass computed.
// The codes do not depend on r: they are quotients of two exact values, rounded once, and equal in every implementation that rounds right.
//
// All three are bound by memory: a row is read once, held in registers (raw, 16 bytes per load), reduced over the lanes that hold it and
// written once.  T lanes hold a row (16, or 1 to 16 waves: NormPlan) with VPT vectors each; a workgroup keeps its share of the weights in
// registers and walks over rows.
#include <algorithm>

#include "head_common.h"

namespace hwer {

// threads of a workgroup: 256 with rows of their own for each wave or part of one, or those of one row
constexpr int norm_block(int t) { return t <= 64 ? 256 : t; }

// N elements of a row from column c, and back: one access of 16 bytes (codes: N bytes) at any alignment; at the row's end element by element, zeros past it
template <typename E, int N>
struct Pack {
    E e[N];
};
template <typename E, int N>
__device__ __forceinline__ Pack<E, N> load_pack(const E* row, int c, int d) {
    Pack<E, N> v;
    if (c + N <= d) {
        __builtin_memcpy(&v, row + c, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) v.e[j] = c + j < d ? row[c + j] : E(0.f);
    }
    return v;
}
template <typename E, int N>
__device__ __forceinline__ void store_pack(E* row, int c, int d, const Pack<E, N>& v) {
    if (c + N <= d) {
        __builtin_memcpy(row + c, &v, sizeof(v));
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c + j < d) row[c + j] = v.e[j];
    }
}

// A code is round_half_even(127 v / top) of exact values.  The float32 quotient t = fl(v) (127 / fl(top)) is off by at most 4 * 2^-24 |t|, which leaves two
// codes open next to the border between them - seldom for products of float32 weights, often for 16-bit rows, whose quotients can BE borders.  Then the
// sign of 127 v - border * top decides: both products next to their rounding errors (one fma each), the products' difference, which has no error (they
// are within a factor of two), and the errors' difference, which has few bits.  That is exact where v and top are float32 values.  Products of float32
// weights have low parts, whose own roundings leave 2^-45.7 of the product: closer than 2^-44 to a border a code is done once more, in 64 bits.
__device__ __forceinline__ bool q8_open(float t, float c) { return fabsf(fabsf(t - c) - 0.5f) <= 3e-7f * fabsf(t); }
// v = vh + ve, top = th + te; 127 and the border over 128, which keeps the products in range
__device__ __forceinline__ float q8_settle(float t, float c, float vh, float ve, float th, float te, bool& unsure) {
    const float side = t > c ? 1.f : -1.f, border = c + 0.5f * side, k = 127.f / 128.f, l = border * (1.f / 128.f);
    const float p = k * vh, q = l * th;
    const float d = ((p - q) + (fmaf(k, vh, -p) - fmaf(l, th, -q)) + (k * ve - l * te)) * side;
    unsure = unsure || ((ve != 0.f || te != 0.f) && fabsf(d) <= 0x1p-44f * fabsf(p));
    return d > 0.f ? c + side : d < 0.f ? c : rintf(border);      // (on the border: the even one)
}
// the same in 64 bits, which hold the 48 of a product: 127 v and border * top have 56, and their errors 3
__device__ __forceinline__ int q8_exact(float h, float w, double top) {
    const double v = double(h) * double(w), t = 127.0 * v / top, c = rint(t);
    if (!(fabs(fabs(t - c) - 0.5) <= 1e-13 * fabs(t))) return int(c);
    const double side = t > c ? 1.0 : -1.0, border = c + 0.5 * side, p = 127.0 * v, q = border * top;
    const double d = ((p - q) + (fma(127.0, v, -p) - fma(border, top, -q))) * side;
    return int(d > 0.0 ? c + side : d < 0.0 ? c : rint(border));
}
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }      // ordered like |v|, infinities and NaN above all else
constexpr uint32_t kInfBits = 0x7f800000u, kTinyBits = 0x0da24260u;      // 1e-30: below it 127 / top and the products' errors leave float32's range

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

// Waves of a SIMD that registers are shared out for: as they come, but codes of 16-bit rows with float32 weights held by 8 waves would take 130 registers, and a
// CU one workgroup.
template <typename E, typename W, int T, bool Q8>
constexpr int norm_fwd_waves() {
    return Q8 && T == 512 && sizeof(E) < sizeof(W) ? 4 : 1;
}

template <typename E, typename W, int T, int VPT, int VW, bool Q8>
__global__ __launch_bounds__(norm_block(T), (norm_fwd_waves<E, W, T, Q8>())) void norm_fwd_kernel(NormFwdArgs a) {
    constexpr int B = norm_block(T), R = B / T;     // R rows at a time
    __shared__ float s_sum[2 * (T > 64 ? T / 64 : 1)];
    __shared__ uint32_t s_top[2 * (T > 64 ? T / 64 : 1)];
    __shared__ double s_exact[T > 64 ? T / 64 : 1];
    __shared__ float s_low[T > 64 ? T / 64 : 1];
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
        const int own = on ? a.d : 0;      // columns of this thread's row that exist
        const int64_t rc = on ? r : 0;
        PE h[VPT];
        float ss = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; ++p) h[p] = load_pack<E, VW>(xp + rc * a.ldx, (p * T + t) * VW, own);
        if (rp) {
#pragma unroll
            for (int p = 0; p < VPT; ++p) {
                const PE q = load_pack<E, VW>(rp + rc * a.ldr, (p * T + t) * VW, own);
#pragma unroll
                for (int j = 0; j < VW; ++j) h[p].e[j] = E(float(h[p].e[j]) + float(q.e[j]));
                store_pack<E, VW>(static_cast<E*>(a.h) + rc * a.ldh, (p * T + t) * VW, own, h[p]);
            }
        }
#pragma unroll
        for (int p = 0; p < VPT; ++p)
#pragma unroll
            for (int j = 0; j < VW; ++j) ss = fmaf(float(h[p].e[j]), float(h[p].e[j]), ss);
        float rstd = 1.f;
        if (a.norm) rstd = 1.f / sqrtf(row_sum<T>(ss, s_sum, flip) * inv_d + a.eps);
        if constexpr (!Q8) {
#pragma unroll
            for (int p = 0; p < VPT; ++p) {
                PE o;
#pragma unroll
                for (int j = 0; j < VW; ++j) o.e[j] = E(float(h[p].e[j]) * rstd * w[p * VW + j]);
                store_pack<E, VW>(static_cast<E*>(a.y) + rc * a.ldy, (p * T + t) * VW, own, o);
            }
        } else {
            // the largest product, rounded: rounding keeps the order, so the exact one is among those that round to it
            uint32_t top_bits = 0;
#pragma unroll
            for (int p = 0; p < VPT; ++p)
#pragma unroll
                for (int j = 0; j < VW; ++j)      // (past the row's end h is 0 and w 1)
                    top_bits = max(top_bits, abs_bits(float(h[p].e[j]) * w[p * VW + j]));
            top_bits = lanes_max_u32<(T < 64 ? T : 64)>(top_bits);
            if constexpr (T > 64) {
                uint32_t* s = s_top + flip * (T / 64);
                if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = top_bits;
                __syncthreads();
                top_bits = s[0];
#pragma unroll
                for (int i = 1; i < T / 64; ++i) top_bits = max(top_bits, s[i]);
            }
            const bool fine = top_bits > 0 && top_bits < kInfBits;
            const float top = __uint_as_float(top_bits), inv = fine ? 127.f / top : 0.f;
            if (on && t == 0) a.scale[r] = fine ? top * rstd / 127.f : top_bits == 0 ? 0.f : NAN;      // (zeros: 0, without eps too; a NaN or an infinity: NaN)
            const bool tiny = fine && top_bits < kTinyBits;
            bool unsure = false;      // is a code of this lane too close to a border for float32?
            int8_t* q = static_cast<int8_t*>(a.y) + rc * a.ldy;
            constexpr bool PAIR = std::is_same<W, float>::value;      // weights of 24 bits: products have a low part (16-bit rows and weights: exact)
            float te = 0.f;      // low part of the largest product, needed where a code is open
            bool settle = true;      // is any code of the row open: looked at for each again then (without low parts that is all there is to it)
            if constexpr (PAIR) {
                if (wp) {
                    bool some = false;
#pragma unroll
                    for (int p = 0; p < VPT; ++p)
#pragma unroll
                        for (int j = 0; j < VW; ++j) {
                            const float v = float(h[p].e[j]) * w[p * VW + j] * inv;
                            some = some || q8_open(v, rintf(v));
                        }
                    // the same for all that hold the row (a wave may hold several)
                    if constexpr (T > 64) settle = __syncthreads_or(some);
                    else settle = __any(some);
                    if (settle) {
                        te = -INFINITY;
#pragma unroll
                        for (int p = 0; p < VPT; ++p)
#pragma unroll
                            for (int j = 0; j < VW; ++j) {
                                const float hv = fabsf(float(h[p].e[j])), wv = fabsf(w[p * VW + j]);
                                if (abs_bits(hv * wv) == top_bits) te = fmaxf(te, fmaf(hv, wv, -top));
                            }
                        te = lanes_max_f32<(T < 64 ? T : 64)>(te);
                        if constexpr (T > 64) {
                            if ((threadIdx.x & 63) == 0) s_low[threadIdx.x >> 6] = te;
                            __syncthreads();
                            te = s_low[0];
#pragma unroll
                            for (int i = 1; i < T / 64; ++i) te = fmaxf(te, s_low[i]);
                        }
                    }
                }
            }
            if (!settle) {
#pragma unroll
                for (int p = 0; p < VPT; ++p) {
                    Pack<int8_t, VW> out;
#pragma unroll
                    for (int j = 0; j < VW; ++j) out.e[j] = fine ? int8_t(int(rintf(float(h[p].e[j]) * w[p * VW + j] * inv))) : int8_t(0);
                    store_pack<int8_t, VW>(q, (p * T + t) * VW, own, out);
                }
            } else {
#pragma unroll
            for (int p = 0; p < VPT; ++p) {
                Pack<int8_t, VW> out;
#pragma unroll
                for (int j = 0; j < VW; ++j) {
                    const float hv = float(h[p].e[j]), wv = w[p * VW + j], v = hv * wv, quo = v * inv;
                    float c = rintf(quo);
                    if (q8_open(quo, c)) c = q8_settle(quo, c, v, PAIR ? fmaf(hv, wv, -v) : 0.f, top, te, unsure);
                    out.e[j] = fine ? int8_t(int(c)) : int8_t(0);
                }
                store_pack<int8_t, VW>(q, (p * T + t) * VW, own, out);
            }
            }
            // Once more from memory, in 64 bits: rows of nothing but tiny products, and a lane's elements with a code that is still open
            bool again;
            if constexpr (T > 64) again = tiny;
            else again = __any(tiny);
            const bool mine = tiny || (PAIR && unsure && fine);
            if (again || mine) {
                const E* hp = rp ? static_cast<const E*>(a.h) + rc * a.ldh : xp + rc * a.ldx;
                double exact = double(top) + double(te);
                if (again) {
                    double v = 0.0;
#pragma unroll 1
                    for (int i = 0; i < VPT * VW; ++i) {
                        const int c = (i / VW * T + t) * VW + i % VW;
                        if (tiny && c < own) v = fmax(v, fabs(double(float(hp[c])) * double(wp ? float(wp[c]) : 1.f)));
                    }
                    v = lanes_max<(T < 64 ? T : 64)>(v);
                    if constexpr (T > 64) {
                        __syncthreads();
                        if ((threadIdx.x & 63) == 0) s_exact[threadIdx.x >> 6] = v;
                        __syncthreads();
                        v = s_exact[0];
#pragma unroll 1
                        for (int i = 1; i < T / 64; ++i) v = fmax(v, s_exact[i]);
                    }
                    if (tiny) exact = v;
                }
#pragma unroll 1
                for (int i = 0; i < VPT * VW; ++i) {
                    const int c = (i / VW * T + t) * VW + i % VW;
                    if (mine && c < own) q[c] = int8_t(q8_exact(float(hp[c]), wp ? float(wp[c]) : 1.f, exact));
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
__global__ __launch_bounds__(norm_block(T)) void norm_bwd_kernel(NormBwdArgs a) {
    constexpr int B = norm_block(T), R = B / T;
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
        const int own = on ? a.d : 0;
        const int64_t rc = on ? r : 0;
        PE h[VPT], g[VPT];
        float ss = 0.f, sc = 0.f;
#pragma unroll
        for (int p = 0; p < VPT; ++p) {
            h[p] = load_pack<E, VW>(static_cast<const E*>(a.h) + rc * a.ldh, (p * T + t) * VW, own);
            g[p] = load_pack<E, VW>(static_cast<const E*>(a.dy) + rc * a.lddy, (p * T + t) * VW, own);
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
            PE o, add;
            if (a.dh) add = load_pack<E, VW>(static_cast<const E*>(a.dh) + rc * a.lddh, c, own);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float hv = float(h[p].e[j]), gv = float(g[p].e[j]);
                float v = rstd * (w[p * VW + j] * gv - hv * back);
                if (a.dh) v += float(add.e[j]);
                o.e[j] = E(v);
                dw[p * VW + j] = on ? fmaf(gv, hv * rstd, dw[p * VW + j]) : dw[p * VW + j];
            }
            store_pack<E, VW>(static_cast<E*>(a.dx) + rc * a.lddx, c, own, o);
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

// dw[c] = sum over the partials in a fixed order: a workgroup takes 16 columns, 64 threads of each column walk over the partials.  (32 columns and 32
// threads: half the workgroups and twice the loads in a row, 10.8 us against 4 at 1 024 partials of 1 024.)
template <typename W>
__global__ __launch_bounds__(1024) void norm_dw_kernel(const float* __restrict__ part, int n_part, int d, W* __restrict__ dw) {
    __shared__ float s[64][17];
    const int c = blockIdx.x * 16 + (threadIdx.x & 15), k = threadIdx.x >> 4;
    float v = 0.f;
    if (c < d) {
#pragma unroll 8
        for (int i = k; i < n_part; i += 64) v += part[int64_t(i) * d + c];
    }
    s[k][threadIdx.x & 15] = v;
    __syncthreads();
    if (k < 8) {
#pragma unroll
        for (int i = 1; i < 8; ++i) v += s[k + 8 * i][threadIdx.x & 15];
        s[k][threadIdx.x & 15] = v;
    }
    __syncthreads();
    if (k == 0 && c < d) {
#pragma unroll
        for (int i = 1; i < 8; ++i) v += s[i][threadIdx.x];
        dw[c] = W(v);
    }
}

// ---------------------------------------------------------------------------------------------------------------- rows too wide for registers
// Read twice, 16 bytes a lane, the second time from the caches while few rows are under way.
constexpr int kWideThreads = 1024;

template <typename W, int N>
__device__ __forceinline__ Pack<W, N> load_weights(const W* w, int c, int d) {      // (none: ones)
    if (w) return load_pack<W, N>(w, c, d);
    Pack<W, N> v;
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = W(1.f);
    return v;
}

template <typename E, typename W, bool Q8>
__global__ __launch_bounds__(kWideThreads) void norm_fwd_wide_kernel(NormFwdArgs a) {
    __shared__ float s_sum[2 * (kWideThreads / 64)];
    __shared__ double s_top[kWideThreads / 64];
    constexpr int VW = 16 / int(sizeof(E));
    typedef Pack<E, VW> PE;
    typedef Pack<W, VW> PW;
    const int t = threadIdx.x;
    const W* wp = static_cast<const W*>(a.w);
    int flip = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
        const E* x = static_cast<const E*>(a.x) + r * a.ldx;
        const E* q = a.res ? static_cast<const E*>(a.res) + r * a.ldr : nullptr;
        // the sum is formed again from the inputs in each pass: `h` may share memory with nothing, but is written once only
        auto load = [&](int c) {
            PE h = load_pack<E, VW>(x, c, a.d);
            if (q) {
                const PE p = load_pack<E, VW>(q, c, a.d);
#pragma unroll
                for (int j = 0; j < VW; ++j) h.e[j] = E(float(h.e[j]) + float(p.e[j]));
            }
            return h;
        };
        float ss = 0.f;
        double top = 0.0;
        float bad = 0.f;
        for (int c = t * VW; c < a.d; c += kWideThreads * VW) {      // (past the row's end h is 0)
            const PE h = load(c);
            const PW w = Q8 ? load_weights<W, VW>(wp, c, a.d) : PW();
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float hv = float(h.e[j]);
                ss = fmaf(hv, hv, ss);
                if (Q8) {
                    top = fmax(top, fabs(double(hv) * double(float(w.e[j]))));
                    bad = fmaf(hv * float(w.e[j]), 0.f, bad);      // becomes NaN with any NaN or infinity
                }
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
            if (t == 0) a.scale[r] = fine ? float(top) * rstd / 127.f : top == 0.0 ? 0.f : NAN;
        }
        for (int c = t * VW; c < a.d; c += kWideThreads * VW) {
            const PE h = load(c);
            const PW w = load_weights<W, VW>(wp, c, a.d);
            if (a.res) store_pack<E, VW>(static_cast<E*>(a.h) + r * a.ldh, c, a.d, h);
            PE y;
            Pack<int8_t, VW> code;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float hv = float(h.e[j]), wv = float(w.e[j]);
                if (Q8) {
                    const float quo = hv * wv * inv, near = rintf(quo);
                    const bool open = top < 1e-30 || q8_open(quo, near);
                    code.e[j] = !fine ? int8_t(0) : int8_t(open ? q8_exact(hv, wv, top) : int(near));
                } else {
                    y.e[j] = E(hv * rstd * wv);
                }
            }
            if constexpr (Q8) store_pack<int8_t, VW>(static_cast<int8_t*>(a.y) + r * a.ldy, c, a.d, code);
            else store_pack<E, VW>(static_cast<E*>(a.y) + r * a.ldy, c, a.d, y);
        }
    }
}

// dx of a row, and the row's r into `rstd`; dw is then summed down the columns by norm_dw_wide_kernel
template <typename E, typename W>
__global__ __launch_bounds__(kWideThreads) void norm_bwd_wide_kernel(NormBwdArgs a, float* __restrict__ rstd_out) {
    __shared__ float s_sum[4 * (kWideThreads / 64)];
    constexpr int VW = 16 / int(sizeof(E));
    typedef Pack<E, VW> PE;
    typedef Pack<W, VW> PW;
    const int t = threadIdx.x;
    const W* wp = static_cast<const W*>(a.w);
    int flip = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, flip ^= 1) {
        const E* h = static_cast<const E*>(a.h) + r * a.ldh;
        const E* g = static_cast<const E*>(a.dy) + r * a.lddy;
        float ss = 0.f, sc = 0.f;
        for (int c = t * VW; c < a.d; c += kWideThreads * VW) {
            const PE hp = load_pack<E, VW>(h, c, a.d), gp = load_pack<E, VW>(g, c, a.d);
            const PW w = load_weights<W, VW>(wp, c, a.d);
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                const float hv = float(hp.e[j]);
                ss = fmaf(hv, hv, ss);
                sc = fmaf(hv * float(w.e[j]), float(gp.e[j]), sc);
            }
        }
        ss = row_sum<kWideThreads>(ss, s_sum, flip);
        sc = row_sum<kWideThreads>(sc, s_sum + 2 * (kWideThreads / 64), flip);
        const float rstd = 1.f / sqrtf(ss / float(a.d) + a.eps);
        const float back = (sc / float(a.d)) * rstd * rstd;
        for (int c = t * VW; c < a.d; c += kWideThreads * VW) {
            const PE hp = load_pack<E, VW>(h, c, a.d), gp = load_pack<E, VW>(g, c, a.d);
            const PW w = load_weights<W, VW>(wp, c, a.d);
            PE add;
            if (a.dh) add = load_pack<E, VW>(static_cast<const E*>(a.dh) + r * a.lddh, c, a.d);
            PE dx;
#pragma unroll
            for (int j = 0; j < VW; ++j) {
                float v = rstd * (float(w.e[j]) * float(gp.e[j]) - float(hp.e[j]) * back);
                if (a.dh) v += float(add.e[j]);
                dx.e[j] = E(v);
            }
            store_pack<E, VW>(static_cast<E*>(a.dx) + r * a.lddx, c, a.d, dx);
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
// How a row of d elements is held: T lanes with VPT vectors of VW elements, T * VPT * VW >= d.
struct NormPlan {
    int t, vpt;      // t = 0: the wide kernels
};
#define HWER_NORM_PLANS(X) X(16, 1) X(64, 1) X(64, 2) X(256, 1) X(512, 1) X(1024, 1) X(1024, 2)
// Codes take two reductions and more work an element: 16 elements a lane, so that fewer waves meet.  32 768 x 2 048 bfloat16 with float32 weights 119 us, 136
// with 8 elements, 176 with 32; 8 192 x 8 192 126, 155 and 175; 16 384 x 2 048 float32 (4, 8, 16 elements) 87, 89 and 82.
#define HWER_NORM_CODE_PLANS_16(X) X(16, 1) X(64, 1) X(64, 2) X(128, 2) X(256, 2) X(512, 2) X(1024, 2)
#define HWER_NORM_CODE_PLANS_32(X) X(16, 1) X(64, 1) X(64, 2) X(64, 4) X(128, 4) X(256, 4) X(512, 4)
// Gradients of wide 16-bit rows: 16 384 x 4 096 bfloat16 105 us, 116 with 8 elements a lane (32 768 x 2 048 150 and 107: too few waves with two a row)
#define HWER_NORM_BWD_PLANS_16(X) X(16, 1) X(64, 1) X(64, 2) X(256, 1) X(256, 2) X(512, 2) X(1024, 2)
#define HWER_NORM_TRY(T, V) \
    if (int64_t(T) * V * vw >= d) return {T, V};
static NormPlan norm_plan(int d, int vw) {
    HWER_NORM_PLANS(HWER_NORM_TRY)
    return {0, 0};
}
static NormPlan norm_code_plan(int d, int vw) {
    if (vw == 8) {
        HWER_NORM_CODE_PLANS_16(HWER_NORM_TRY)
    } else {
        HWER_NORM_CODE_PLANS_32(HWER_NORM_TRY)
    }
    return {0, 0};
}
static NormPlan norm_bwd_plan(int d, int vw) {
    if (vw == 8) {
        HWER_NORM_BWD_PLANS_16(HWER_NORM_TRY)
        return {0, 0};
    }
    return norm_plan(d, vw);
}
#undef HWER_NORM_TRY

// workgroups of a launch: enough to fill the chip several times over, few enough that the weights are read once per many rows
static int norm_grid(int64_t rows, int t) {
    const int r = norm_block(t) / t;
    return int(std::min<int64_t>(cdiv64(rows, r), kMaxStreamBlocks));
}
// ... of a backward launch: each leaves a partial sum of the weights' gradient behind
static int norm_bwd_grid(int64_t rows, int t) {
    const int r = norm_block(t) / t;
    return int(std::min<int64_t>(cdiv64(rows, r), 1024));
}
constexpr int kWideDwParts = 32;
// Columns are 32-bit numbers, which the wide kernels run past a row's end by up to kWideThreads * 8
constexpr int64_t kNormMaxDim = (int64_t(1) << 31) - (int64_t(1) << 14);

template <typename E, typename W, bool Q8>
static void norm_fwd_launch(const NormFwdArgs& a, hipStream_t st) {
    constexpr int VW = 16 / int(sizeof(E));
    NormPlan p = Q8 ? norm_code_plan(a.d, VW) : norm_plan(a.d, VW);
    // Two waves that a row nearly fills, instead of one with twice the elements: 16 384 x 1 024 bfloat16 25 us, 30 as one wave; but 65 536 x 300 float32 87, 54
    // as one wave.
    if (!Q8 && a.d > 112 * VW && a.d <= 128 * VW) p = {128, 1};
    const int grid = norm_grid(a.rows, p.t ? p.t : kWideThreads);
#define HWER_NORM_FWD(T, V) \
    if (p.t == T && p.vpt == V) return norm_fwd_kernel<E, W, T, V, VW, Q8><<<dim3(grid), dim3(norm_block(T)), 0, st>>>(a);
    if constexpr (!Q8) {
        HWER_NORM_PLANS(HWER_NORM_FWD)
        HWER_NORM_FWD(128, 1)
    } else if constexpr (VW == 8) {
        HWER_NORM_CODE_PLANS_16(HWER_NORM_FWD)
    } else {
        HWER_NORM_CODE_PLANS_32(HWER_NORM_FWD)
    }
#undef HWER_NORM_FWD
    norm_fwd_wide_kernel<E, W, Q8><<<dim3(grid), dim3(kWideThreads), 0, st>>>(a);
}
template <typename E, typename W>
static void norm_fwd_typed(const NormFwdArgs& a, bool q8, hipStream_t st) {
    q8 ? norm_fwd_launch<E, W, true>(a, st) : norm_fwd_launch<E, W, false>(a, st);
}

static int norm_fwd_any(const NormFwdArgs& a, int dtype, int w_dtype, bool q8, const char* what, void* stream) {
    hipStream_t st = as_stream(stream);
    const bool w32 = a.w && w_dtype == HWER_F32;      // (without weights products are the rows' own values: no low parts)
    if (dtype == HWER_F32) norm_fwd_typed<float, float>(a, q8, st);
    else if (dtype == HWER_F16) w32 ? norm_fwd_typed<f16_t, float>(a, q8, st) : norm_fwd_typed<f16_t, f16_t>(a, q8, st);
    else w32 ? norm_fwd_typed<bf16_t, float>(a, q8, st) : norm_fwd_typed<bf16_t, bf16_t>(a, q8, st);
    return check_launch(what);
}

static int norm_check(const char* what, const void* x, int64_t ldx, const void* w, int w_dtype, int64_t rows, int64_t d, int dtype, float eps) {
    if (!known_dtype(dtype)) return fail(HWER_EINVAL, "%s: unknown element type %d", what, dtype);
    if (w && w_dtype != HWER_F32 && w_dtype != dtype) return fail(HWER_EINVAL, "%s: the weights are float32 or of the rows' type", what);
    if (rows < 0 || d < 1 || d > kNormMaxDim) return fail(HWER_EINVAL, "%s: rows=%lld, d=%lld (d <= %lld)", what, (long long)rows, (long long)d, (long long)kNormMaxDim);
    if (rows && (!x || ldx < d)) return fail(HWER_EINVAL, "%s: null rows or a row stride below d", what);
    if (!(eps >= 0.f) || !(eps < INFINITY)) return fail(HWER_EINVAL, "%s: eps must be finite and not negative", what);
    return HWER_OK;
}

}  // namespace hwer

using namespace hwer;

extern "C" {

int hwer_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int weight_dtype, int64_t rows, int64_t d, int dtype,
                  float eps, void* y, int64_t ldy, void* h, int64_t ldh, void* stream) {
    if (int rc = norm_check("rms_norm", x, ldx, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (rows == 0) return HWER_OK;
    if (!y || ldy < d || (residual && (!h || ldr < d || ldh < d))) return fail(HWER_EINVAL, "rms_norm: null output or a row stride below d");
    const NormFwdArgs a{x, residual, weight, y, h, nullptr, rows, ldx, ldr, ldy, ldh, int(d), eps, 1};
    return norm_fwd_any(a, dtype, weight_dtype, false, "rms_norm", stream);
}

int hwer_rms_norm_q8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int weight_dtype, int64_t rows, int64_t d, int dtype,
                     int norm, float eps, int8_t* q, int64_t ldq, float* scale, void* h, int64_t ldh, void* stream) {
    if (int rc = norm_check("rms_norm_q8", x, ldx, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (rows == 0) return HWER_OK;
    if (!q || !scale || ldq < d || (residual && (!h || ldr < d || ldh < d))) return fail(HWER_EINVAL, "rms_norm_q8: null output or a row stride below d");
    const NormFwdArgs a{x, residual, weight, q, h, scale, rows, ldx, ldr, ldq, ldh, int(d), eps, norm ? 1 : 0};
    return norm_fwd_any(a, dtype, weight_dtype, true, "rms_norm_q8", stream);
}

size_t hwer_rms_norm_backward_workspace_bytes(int64_t rows, int64_t d) {
    if (rows <= 0 || d < 1 || d > kNormMaxDim) return 16;
    // partial sums of dweight (at most 1 024 workgroups; rows too wide for registers: kWideDwParts and one r per row)
    return size_t(std::max<int64_t>(std::min<int64_t>(rows, 1024), kWideDwParts)) * d * 4 + size_t(rows) * 4;
}

int hwer_rms_norm_backward(const void* dy, int64_t lddy, const void* h, int64_t ldh, const void* weight, int weight_dtype, const void* dh, int64_t lddh,
                           int64_t rows, int64_t d, int dtype, float eps, void* dx, int64_t lddx, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = norm_check("rms_norm_backward", h, ldh, weight, weight_dtype, rows, d, dtype, eps)) return rc;
    if (dweight && !weight) return fail(HWER_EINVAL, "rms_norm_backward: a gradient of weights that are not there");
    if (rows && (!dy || !dx || lddy < d || lddx < d || (dh && lddh < d))) return fail(HWER_EINVAL, "rms_norm_backward: null rows or a row stride below d");
    if (dweight && (!workspace || workspace_bytes < hwer_rms_norm_backward_workspace_bytes(rows, d)))
        return fail(HWER_EWORKSPACE, "rms_norm_backward: workspace of %zu bytes needed", hwer_rms_norm_backward_workspace_bytes(rows, d));
    if (dweight && !aligned_to(workspace, 0, 16)) return fail(HWER_EINVAL, "rms_norm_backward: the workspace must be 16-byte aligned");
    hipStream_t st = as_stream(stream);
    NormBwdArgs a{dy, h, weight, dh, dx, dweight ? static_cast<float*>(workspace) : nullptr, rows, lddy, ldh, lddh, lddx, int(d), eps};
    int parts = 0;
    auto run = [&](auto e, auto wt) {
        typedef decltype(e) E;
        typedef decltype(wt) W;
        constexpr int VW = 16 / int(sizeof(E));
        const NormPlan p = norm_bwd_plan(a.d, VW);
        if (p.t == 0) {
            float* rstd = a.dw_part ? a.dw_part + int64_t(kWideDwParts) * d : nullptr;
            const int grid = norm_grid(rows, kWideThreads);
            norm_bwd_wide_kernel<E, W><<<dim3(grid), dim3(kWideThreads), 0, st>>>(a, rstd);
            if (a.dw_part) {
                parts = int(std::min<int64_t>(kWideDwParts, cdiv64(rows, 64)));      // (16 waves share a part's rows: 152 x 20 000 bfloat16 5.3 us, 18.6 as 32 parts)
                norm_dw_wide_kernel<E><<<dim3((a.d + 63) / 64, parts), dim3(1024), 0, st>>>(a, rstd, int(cdiv64(rows, parts)));
            }
            return;
        }
        parts = norm_bwd_grid(rows, p.t);
#define HWER_NORM_BWD(T, V) \
        if (p.t == T && p.vpt == V) return norm_bwd_kernel<E, W, T, V, VW><<<dim3(parts), dim3(norm_block(T)), 0, st>>>(a);
        if constexpr (VW == 8) {
            HWER_NORM_BWD_PLANS_16(HWER_NORM_BWD)
        } else {
            HWER_NORM_PLANS(HWER_NORM_BWD)
        }
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
        const dim3 grid((a.d + 15) / 16);
        if (w32) norm_dw_kernel<float><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, a.d, static_cast<float*>(dweight));
        else if (dtype == HWER_F16) norm_dw_kernel<f16_t><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, a.d, static_cast<f16_t*>(dweight));
        else norm_dw_kernel<bf16_t><<<grid, dim3(1024), 0, st>>>(a.dw_part, parts, a.d, static_cast<bf16_t*>(dweight));
    }
    return check_launch("rms_norm_backward(dweight)");
}

}  // extern "C"
