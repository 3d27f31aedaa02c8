// Definitions shared by the row operators (rms_norm.hip, linear.hip, prior_balance.hip).
#pragma once
#include "mpc_internal.h"

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

inline int mpc_type_bytes(int type) {
    return type == MPC_TYPE_F32 ? 4 : type == MPC_TYPE_F16 || type == MPC_TYPE_BF16 ? 2 : type == MPC_TYPE_E4M3 ? 1 : 0;
}

// Most threads of a launch: HIP takes fewer than 2^32, and where there are more it runs what their number leaves modulo 2^32,
// without an error.
constexpr int64_t MPC_LAUNCH_THREADS = 1ll << 31;

#if defined(__HIPCC__)
constexpr float E4M3_MAX = 448.0f;

// Two floats as e4m3 (nearest, ties to even; the caller has scaled them to at most 448 up to rounding, which 464, the first
// value that would round past the largest, is far from), in the low or the high half of `old`.
template <bool HIGH>
__device__ __forceinline__ int e4m3_pack2(float a, float b, int old) {
    return __builtin_amdgcn_cvt_pk_fp8_f32(a, b, old, HIGH);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const unsigned o = __shfl_xor(v, off, 64);
        v = v > o ? v : o;
    }
    return v;
}
#endif
