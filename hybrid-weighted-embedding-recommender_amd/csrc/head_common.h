// Element types, lane reductions and host checks shared by the learned head's kernels (head_norm.hip, matmul_q8.hip, catalogue_ce.hip).
#pragma once
#include "hwer_common.h"

namespace hwer {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;   // conversions from float round to nearest even (v_cvt_pk_bf16_f32)

__host__ __device__ static inline bool known_dtype(int t) { return t == HWER_F32 || t == HWER_F16 || t == HWER_BF16; }
__host__ __device__ static inline int dtype_bytes(int t) { return t == HWER_F32 ? 4 : 2; }

static inline bool aligned_to(const void* p, int64_t row_bytes, int bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes == 0 && row_bytes % bytes == 0;
}

// sum / maximum over groups of T consecutive lanes (T = 16 or 64), result in every lane of the group: VALU exchanges, butterfly order
template <int T>
__device__ __forceinline__ float lanes_sum(float v) {
    v += __uint_as_float(lane_xor32<1>(__float_as_uint(v)));
    v += __uint_as_float(lane_xor32<2>(__float_as_uint(v)));
    v += __uint_as_float(lane_xor32<4>(__float_as_uint(v)));
    v += __uint_as_float(lane_xor32<8>(__float_as_uint(v)));
    if constexpr (T > 16) {
        v += __uint_as_float(lane_xor32<16>(__float_as_uint(v)));
        v += __uint_as_float(lane_xor32<32>(__float_as_uint(v)));
    }
    return v;
}
template <int T>
__device__ __forceinline__ uint32_t lanes_max_u32(uint32_t v) {
    v = max(v, lane_xor32<1>(v));
    v = max(v, lane_xor32<2>(v));
    v = max(v, lane_xor32<4>(v));
    v = max(v, lane_xor32<8>(v));
    if constexpr (T > 16) {
        v = max(v, lane_xor32<16>(v));
        v = max(v, lane_xor32<32>(v));
    }
    return v;
}
template <int T>
__device__ __forceinline__ float lanes_max_f32(float v) {
    v = fmaxf(v, __uint_as_float(lane_xor32<1>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor32<2>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor32<4>(__float_as_uint(v))));
    v = fmaxf(v, __uint_as_float(lane_xor32<8>(__float_as_uint(v))));
    if constexpr (T > 16) {
        v = fmaxf(v, __uint_as_float(lane_xor32<16>(__float_as_uint(v))));
        v = fmaxf(v, __uint_as_float(lane_xor32<32>(__float_as_uint(v))));
    }
    return v;
}
template <int T>
__device__ __forceinline__ double lanes_max(double v) {
    auto step = [](double a, uint64_t b) { return fmax(a, __longlong_as_double((long long)b)); };
    v = step(v, lane_xor64<1>((uint64_t)__double_as_longlong(v)));
    v = step(v, lane_xor64<2>((uint64_t)__double_as_longlong(v)));
    v = step(v, lane_xor64<4>((uint64_t)__double_as_longlong(v)));
    v = step(v, lane_xor64<8>((uint64_t)__double_as_longlong(v)));
    if constexpr (T > 16) {
        v = step(v, lane_xor64<16>((uint64_t)__double_as_longlong(v)));
        v = step(v, lane_xor64<32>((uint64_t)__double_as_longlong(v)));
    }
    return v;
}

}  // namespace hwer
