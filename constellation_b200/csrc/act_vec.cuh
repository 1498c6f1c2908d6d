// Activation vectors: up to 8 consecutive elements of a row as fp32, for the row kernels whose
// tensors may be fp16, bf16 or fp32 (dtype codes of the C ABI: 1, 2, 3).  VEC = 8 moves 16
// bytes at a time (two 16-byte accesses for fp32) and needs 16-byte aligned rows; VEC = 1 is
// the form for rows that no vector access may touch.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cst {

template <int VEC>
__device__ __forceinline__ void load_act(const void* base, int dtype, int64_t i, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        if (dtype == 3) v[0] = static_cast<const float*>(base)[i];
        else if (dtype == 2) v[0] = __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
        else v[0] = __half2float(static_cast<const __half*>(base)[i]);
    } else if (dtype == 3) {
        const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
        const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (dtype == 2) {
                v[2 * k] = __uint_as_float(w[k] << 16);
                v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                v[2 * k] = f.x;
                v[2 * k + 1] = f.y;
            }
        }
    }
}

template <int VEC>
__device__ __forceinline__ void store_act(void* base, int dtype, int64_t i, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        if (dtype == 3) static_cast<float*>(base)[i] = v[0];
        else if (dtype == 2) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v[0]);
        else static_cast<__half*>(base)[i] = __float2half_rn(v[0]);
    } else if (dtype == 3) {
        *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(static_cast<float*>(base) + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (dtype == 2) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * k], v[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t*>(&b);
            } else {
                const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
                w[k] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Whether every row of a tensor of `esize`-byte elements starts 16-byte aligned.
inline bool rows_aligned16(const void* p, int64_t ld, int esize) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * esize) % 16 == 0;
}

inline int act_size(int dtype) { return dtype == 3 ? 4 : dtype == 4 ? 1 : 2; }

}  // namespace cst
