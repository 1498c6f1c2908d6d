// Activation vectors: 8 consecutive elements of a row as fp32, for the row kernels whose tensors may
// be fp16, bf16 or fp32 (dtype codes of the C ABI: 1, 2, 3).  A dtype that is a constant costs
// nothing; at run time it is one uniform branch a vector.
//
// Aligned rows move 16 bytes at a time.  For rows that start anywhere, a kernel lays its vectors along the
// row that it writes, so that its stores are whole, and reads with load8_any: the one or two aligned 16-byte
// pieces around the vector, shifted together -- a quarter of the instructions of eight loads.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace cst {

__device__ __forceinline__ void unpack8(const uint4& u, int dtype, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    if (dtype == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            v[2 * k] = __uint_as_float(w[k] << 16);
            v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
            v[2 * k] = f.x;
            v[2 * k + 1] = f.y;
        }
    }
}

__device__ __forceinline__ void unpack4(const uint4& u, float* v) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
}

__device__ __forceinline__ float load1(const void* base, int dtype, int64_t i) {
    if (dtype == 3) return static_cast<const float*>(base)[i];
    if (dtype == 2) return __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]);
    return __half2float(static_cast<const __half*>(base)[i]);
}

__device__ __forceinline__ void store1(void* base, int dtype, int64_t i, float v) {
    if (dtype == 3) static_cast<float*>(base)[i] = v;
    else if (dtype == 2) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v);
    else static_cast<__half*>(base)[i] = __float2half_rn(v);
}

// Elements i .. i + 7; the address is 16-byte aligned.
__device__ __forceinline__ void load8(const void* base, int dtype, int64_t i, float (&v)[8]) {
    if (dtype == 3) {
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const float*>(base) + i);
        unpack4(p[0], v);
        unpack4(p[1], v + 4);
    } else {
        unpack8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(base) + i), dtype, v);
    }
}

__device__ __forceinline__ uint4 pack8(int dtype, const float (&v)[8]) {
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
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void store8(void* base, int dtype, int64_t i, const float (&v)[8]) {
    if (dtype == 3) {
        float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
        p[0] = make_float4(v[0], v[1], v[2], v[3]);
        p[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(base) + i) = pack8(dtype, v);
    }
}

// The aligned 16-byte pieces around the 16 bytes at p, which it is cut from once they are there.
struct Around {
    uint4 lo, hi;
    uint32_t off;
    __device__ __forceinline__ uint4 piece() const {
        if (off == 0) return lo;  // mostly of a whole warp
        const bool two = off & 8u, one = off & 4u;
        const uint32_t a0 = two ? lo.z : lo.x, a1 = two ? lo.w : lo.y, a2 = two ? hi.x : lo.z, a3 = two ? hi.y : lo.w,
                       a4 = two ? hi.z : hi.x, a5 = two ? hi.w : hi.y;
        const uint32_t b0 = one ? a1 : a0, b1 = one ? a2 : a1, b2 = one ? a3 : a2, b3 = one ? a4 : a3, b4 = one ? a5 : a4;
        const uint32_t s = (off & 3u) * 8u;
        return make_uint4(__funnelshift_r(b0, b1, s), __funnelshift_r(b1, b2, s), __funnelshift_r(b2, b3, s),
                          __funnelshift_r(b3, b4, s));
    }
};
__device__ __forceinline__ Around load_around(const void* p) {
    Around a;
    a.off = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) - a.off);
    a.lo = q[0];
    a.hi = a.off ? q[1] : make_uint4(0, 0, 0, 0);
    return a;
}

// Whether the pieces around elements c .. c + 7 of a row of 16-bit elements lie in the row.
__device__ __forceinline__ bool inner8(int c, int H) { return c >= 8 && c + 16 <= H; }

// 16 bytes from any address; the aligned 16-byte pieces that hold them have to be readable.
__device__ __forceinline__ uint4 load16_any(const uint8_t* p) { return load_around(p).piece(); }

// Elements c .. c + 7 of a row of H elements at `row` (its first element's index), zero outside [0, H).
__device__ __forceinline__ void load8_any(const void* base, int dtype, int64_t row, int c, int H, float (&v)[8]) {
    if (inner8(c, H)) {
        const uint8_t* p = static_cast<const uint8_t*>(base) + (row + c) * (dtype == 3 ? 4 : 2);
        if (dtype == 3) {
            unpack4(load16_any(p), v);
            unpack4(load16_any(p + 16), v + 4);
        } else {
            unpack8(load16_any(p), dtype, v);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = unsigned(c + k) < unsigned(H) ? load1(base, dtype, row + c + k) : 0.0f;
    }
}

// Elements c .. c + 7, of which those in [0, H) are written.
__device__ __forceinline__ void store8_any(void* base, int dtype, int64_t row, int c, int H, const float (&v)[8]) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(base) + (row + c) * (dtype == 3 ? 4 : 2);
    if (c >= 0 && c + 8 <= H && p % 16 == 0) {
        store8(base, dtype, row + c, v);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (unsigned(c + k) < unsigned(H)) store1(base, dtype, row + c + k, v[k]);
    }
}

// How many elements before `row` the nearest 16-byte boundary lies (0 .. 7; 0 .. 3 for fp32).
__device__ __forceinline__ int lead_in(const void* base, int dtype, int64_t row) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(base) + row * (dtype == 3 ? 4 : 2);
    return int(p & 15u) >> (dtype == 3 ? 2 : 1);
}

// Whether every row of a tensor of `esize`-byte elements starts 16-byte aligned.
inline bool rows_aligned16(const void* p, int64_t ld, int esize) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && (ld * esize) % 16 == 0;
}

inline int act_size(int dtype) { return dtype == 3 ? 4 : dtype == 4 ? 1 : 2; }

}  // namespace cst
