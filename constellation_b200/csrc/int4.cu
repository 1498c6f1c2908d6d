// Products with 4-bit weights, grouped by expert.  With q[e, n, k] in 0..15 and one scale (and
// one zero point, 8 if there is none) for `group` consecutive k,
//     y[r, n] = sum_G scale[e, n, G] * sum_{k in G} (q[e, n, k] - zero[e, n, G]) * x[r, k]
// for the rows r in [offsets[e], offsets[e + 1]) of expert e; rows behind offsets[E] are zero.
// x in e4m3 carries one fp32 scale for 128 columns of a row.  With `swiglu` the first half of
// the N weight rows is "up", the second "gate", and y = silu(gate) * up, [R, N / 2].
// q - zero is exact in 16 bits and so is e4m3 in fp16, so every product is exact and only the
// fp32 sums and the one final cast round.
//
// Layout of one weight (written once by pack_kernel): blocks of 64 weight rows, each a run of
// chunks of 128 k; a chunk is 4096 bytes of q in the order the matrix instructions take them,
// then the 64 rows' scales [128 / group][64], then their zero points [128 / group][64].
// Inside the 4096 bytes: [row tile of 16][half of 64 k][lane][word j of 4]; lane (g, c) holds
// rows g and g + 8 and the 16 consecutive k from 16 c of its half, word j the four from 4 j:
// bits 4 i + 16 e .. of a word hold row g + 8 (i & 1), k = 16 c + 4 j + 2 (i >> 1) + e.
// With swiglu a block is 32 "up" rows and the 32 "gate" rows that go with them.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/constellation_b200.h"
#include "act_vec.cuh"
#include "cst_common.cuh"
#include "kernels.h"

namespace cst {

namespace {

constexpr int kRows = 64;    // weight rows of a block
constexpr int kChunk = 128;  // k of a chunk
constexpr int kQBytes = kRows * kChunk / 2;

struct Geom {
    int E, N, K, group, scale_dtype, has_zero, swiglu;
    int out_n;       // columns of the result
    int blocks;      // blocks of weight rows
    int chunks;      // chunks of k
    int groups;      // scales of a weight row
    int chunk_bytes;
    int zero_at;     // byte offset of the zero points in a chunk
    __host__ __device__ int64_t expert_bytes() const { return int64_t(blocks) * chunks * chunk_bytes; }
};

Geom make_geom(const cst_int4_weight& w) {
    Geom g{w.n_experts, w.n, w.k, w.group, w.scale_dtype, w.has_zero, w.swiglu};
    g.out_n = w.swiglu ? w.n / 2 : w.n;
    const int per = w.swiglu ? kRows / 2 : kRows;
    g.blocks = (g.out_n + per - 1) / per;
    g.chunks = (w.k + kChunk - 1) / kChunk;
    g.groups = w.k / w.group;
    const int scales = kChunk / w.group * kRows;
    g.zero_at = kQBytes + scales * act_size(w.scale_dtype);
    g.chunk_bytes = g.zero_at + (w.has_zero ? scales : 0);
    return g;
}

// weight row behind row r of block b, or -1 for padding
__device__ __forceinline__ int source_row(const Geom& g, int b, int r) {
    if (!g.swiglu) {
        const int n = b * kRows + r;
        return n < g.N ? n : -1;
    }
    const int n = b * (kRows / 2) + (r & 31);
    return n < g.out_n ? n + (r >= 32 ? g.out_n : 0) : -1;
}

// One CTA per (chunk, block, expert).  Padding (rows past N, k past K) gets q = 8 and scale 0,
// zero point 8, so it adds exactly nothing.
__global__ void __launch_bounds__(256) pack_kernel(Geom g, const uint8_t* q, const void* scale, const uint8_t* zero,
                                                   uint8_t* out) {
    const int chunk = blockIdx.x, b = blockIdx.y, e = blockIdx.z;
    uint8_t* dst = out + e * g.expert_bytes() + (int64_t(b) * g.chunks + chunk) * g.chunk_bytes;
    for (int w = threadIdx.x; w < kQBytes / 4; w += blockDim.x) {
        const int j = w & 3, lane = (w >> 2) & 31, half = (w >> 7) & 1, tile = w >> 8;
        uint32_t word = 0;
        for (int i = 0; i < 4; ++i) {
            const int n = source_row(g, b, tile * 16 + (lane >> 2) + 8 * (i & 1));
            for (int el = 0; el < 2; ++el) {
                const int k = chunk * kChunk + half * 64 + (lane & 3) * 16 + 4 * j + 2 * (i >> 1) + el;
                uint32_t v = 8;
                if (n >= 0 && k < g.K) {
                    const uint8_t two = q[((int64_t(e) * g.N + n) * g.K + k) >> 1];
                    v = (k & 1) ? two >> 4 : two & 15;
                }
                word |= v << (4 * i + 16 * el);
            }
        }
        reinterpret_cast<uint32_t*>(dst)[w] = word;
    }
    for (int s = threadIdx.x; s < kChunk / g.group * kRows; s += blockDim.x) {
        const int n = source_row(g, b, s % kRows), G = chunk * (kChunk / g.group) + s / kRows;
        const bool in = n >= 0 && G < g.groups;
        const int64_t at = (int64_t(e) * g.N + n) * g.groups + G;
        if (g.scale_dtype == CST_DTYPE_FP32)
            reinterpret_cast<uint32_t*>(dst + kQBytes)[s] = in ? static_cast<const uint32_t*>(scale)[at] : 0u;
        else
            reinterpret_cast<uint16_t*>(dst + kQBytes)[s] = in ? static_cast<const uint16_t*>(scale)[at] : uint16_t(0);
        if (g.has_zero) dst[g.zero_at + s] = in ? (zero[at] & 15) : 8;
    }
}

struct Int4Args {
    Geom g;
    const uint8_t* data;
    const void* x;
    int x_dtype;
    int64_t ld_x;
    const float* x_scale;
    int64_t ld_xs;
    const int32_t* offsets;  // null: every row belongs to expert 0
    int R;
    void* out;
    int out_dtype;
    int64_t ld_out;
};

__device__ __forceinline__ float scale_at(const uint8_t* chunk, int dtype, int s) {
    const uint8_t* p = chunk + kQBytes;
    if (dtype == 3) return reinterpret_cast<const float*>(p)[s];
    if (dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[s]);
    return __half2float(reinterpret_cast<const __half*>(p)[s]);
}

__device__ __forceinline__ float x_at(const Int4Args& a, int64_t r, int k) {
    const int64_t i = r * a.ld_x + k;
    if (a.x_dtype == 4) return e4m3_to_f32(static_cast<const uint8_t*>(a.x)[i]);
    float v[1];
    load_act<1>(a.x, a.x_dtype, i, v);
    return v[0];
}

// One CTA per (block of weight rows, row of x): 4 threads a weight row, each a quarter of k.
__global__ void __launch_bounds__(256) int4_simple_kernel(Int4Args a) {
    __shared__ float s_y[kRows];
    chain_wait();
    chain_release();
    const Geom& g = a.g;
    const int b = blockIdx.x, n = threadIdx.x >> 2, quarter = threadIdx.x & 3;
    const int per = g.swiglu ? kRows / 2 : kRows;
    for (int r = blockIdx.y; r < a.R; r += gridDim.y) {
        int e = a.offsets ? -1 : 0;
        for (int i = 0; a.offsets && i < g.E; ++i)
            if (r >= a.offsets[i] && r < a.offsets[i + 1]) e = i;
        float y = 0.0f;
        for (int chunk = 0; e >= 0 && chunk < g.chunks; ++chunk) {
            const uint8_t* src = a.data + e * g.expert_bytes() + (int64_t(b) * g.chunks + chunk) * g.chunk_bytes;
            const float xs = a.x_scale ? a.x_scale[r * a.ld_xs + chunk] : 1.0f;
            for (int k0 = quarter; k0 < kChunk; k0 += 4) {
                const int k = chunk * kChunk + k0;
                if (k >= g.K) break;
                const int half = k0 >> 6, c = (k0 >> 4) & 3, j = (k0 >> 2) & 3, el = k0 & 1;
                const int i = ((n >> 3) & 1) + (k0 & 2);
                const int lane = (n & 7) * 4 + c, tile = n >> 4;
                const uint32_t word = reinterpret_cast<const uint32_t*>(src)[((tile * 2 + half) * 32 + lane) * 4 + j];
                const int s = (k0 / g.group) * kRows + n;
                const int q = int((word >> (4 * i + 16 * el)) & 15u) - (g.has_zero ? src[g.zero_at + s] : 8);
                y = fmaf(scale_at(src, g.scale_dtype, s) * xs * float(q), x_at(a, r, k), y);
            }
        }
        y += __shfl_xor_sync(0xffffffffu, y, 1);
        y += __shfl_xor_sync(0xffffffffu, y, 2);
        if (quarter == 0) s_y[n] = y;
        __syncthreads();
        if (threadIdx.x < per && b * per + int(threadIdx.x) < g.out_n) {
            float v[1] = {s_y[threadIdx.x]};
            if (g.swiglu) {
                const float gate = s_y[threadIdx.x + 32];
                v[0] *= gate / (1.0f + __expf(-gate));
            }
            store_act<1>(a.out, a.out_dtype, r * a.ld_out + b * per + threadIdx.x, v);
        }
        __syncthreads();
    }
}

int check_weight(const cst_int4_weight* w) {
    if (!w) return set_last_error(CST_ERR_INVALID_ARG, "null weight");
    if (w->n_experts < 1 || w->n_experts > CST_INT4_MAX_EXPERTS || w->n < 1 || w->k < 1 || w->n > (1 << 20) ||
        w->k > (1 << 20))
        return set_last_error(CST_ERR_INVALID_ARG, "weight shape [%d, %d, %d] outside [1, %d] x [1, 2^20] x [1, 2^20]",
                              w->n_experts, w->n, w->k, CST_INT4_MAX_EXPERTS);
    if ((w->group != 32 && w->group != 64 && w->group != 128) || w->k % w->group)
        return set_last_error(CST_ERR_INVALID_ARG, "group must be 32, 64 or 128 and divide k=%d, got %d", w->k,
                              w->group);
    if (w->scale_dtype < CST_DTYPE_FP16 || w->scale_dtype > CST_DTYPE_FP32)
        return set_last_error(CST_ERR_INVALID_ARG, "invalid scale dtype %d", w->scale_dtype);
    if (w->swiglu && w->n % 2)
        return set_last_error(CST_ERR_INVALID_ARG, "swiglu needs an even n (up rows, then gate rows), got %d", w->n);
    return CST_OK;
}

}  // namespace

}  // namespace cst

using namespace cst;

extern "C" int cst_int4_bytes(const cst_int4_weight* w, int64_t* bytes) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (!bytes) return set_last_error(CST_ERR_INVALID_ARG, "null bytes");
    *bytes = make_geom(*w).expert_bytes() * w->n_experts;
    return CST_OK;
}

extern "C" int cst_int4_pack(const cst_int4_weight* w, const uint8_t* q, const void* scale, const uint8_t* zero,
                             void* data, void* stream) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (!q || !scale || !data || (w->has_zero && !zero))
        return set_last_error(CST_ERR_INVALID_ARG, "null q, scale, zero or data");
    if (reinterpret_cast<uintptr_t>(data) & 15u) return set_last_error(CST_ERR_INVALID_ARG, "data must be 16-byte aligned");
    const Geom g = make_geom(*w);
    pack_kernel<<<dim3(g.chunks, g.blocks, g.E), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        g, q, scale, zero, static_cast<uint8_t*>(data));
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "int4_pack launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}

extern "C" int cst_grouped_int4(const cst_int4_weight* w, const void* data, const void* x, int32_t x_dtype,
                                int64_t ld_x, const float* x_scale, int64_t ld_x_scale, const int32_t* offsets,
                                int32_t R, void* out, int32_t out_dtype, int64_t ld_out, void* stream) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    const Geom g = make_geom(*w);
    if (x_dtype != CST_DTYPE_FP16 && x_dtype != CST_DTYPE_BF16 && x_dtype != CST_DTYPE_E4M3)
        return set_last_error(CST_ERR_INVALID_ARG, "x must be fp16, bf16 or e4m3, got dtype %d", x_dtype);
    if (out_dtype < CST_DTYPE_FP16 || out_dtype > CST_DTYPE_FP32)
        return set_last_error(CST_ERR_INVALID_ARG, "invalid out dtype %d", out_dtype);
    if ((x_dtype == CST_DTYPE_E4M3) != (x_scale != nullptr) && R > 0)
        return set_last_error(CST_ERR_INVALID_ARG, "x_scale goes with e4m3 rows, and only with them");
    if (!offsets && w->n_experts != 1)
        return set_last_error(CST_ERR_INVALID_ARG, "offsets are needed for %d experts", w->n_experts);
    if (R < 0 || ld_x < w->k || ld_out < g.out_n || (x_scale && ld_x_scale < (w->k + 127) / 128))
        return set_last_error(CST_ERR_INVALID_ARG, "R=%d must be >= 0 and no row stride below the row", R);
    if (R == 0) return CST_OK;
    if (!data || !x || !out) return set_last_error(CST_ERR_INVALID_ARG, "null data, x or out");
    const Int4Args a{g, static_cast<const uint8_t*>(data), x, x_dtype, ld_x, x_scale, ld_x_scale, offsets, R, out,
                     out_dtype, ld_out};
    const cudaError_t e = launch_chained(int4_simple_kernel, dim3(g.blocks, R < 65535 ? R : 65535), dim3(256), 0,
                                         static_cast<cudaStream_t>(stream), a);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "grouped_int4 launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}
