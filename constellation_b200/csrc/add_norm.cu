// Residual add + RMSNorm, and its form whose result leaves in 8 bits:
//     h[t, c]   = x[t, c] + residual[t, c]                                  (fp32)
//     sum[t, c] = h[t, c], rounded once to the residual's type
//     y[t, c]   = h[t, c] * rsqrt(mean_c(h[t, :]^2) + eps) * weight[c]      (fp32)
//     out[t, c] = y, rounded once; or, in e4m3 with one scale per 128 columns,
//     scale[t, b] = max_{c in b} |y[t, c]| / 448 (1 where a block is all zero),
//     out[t, c]   = e4m3(y[t, c] / scale[t, c / 128])
// The norm is taken of the unrounded h, and the row stays in registers between the sum of
// squares and the result, so each element is read once and written once: the kernel is bound
// by HBM, (2 + 2 + 2 + 1) bytes an element for bf16 to e4m3.
#include <cfloat>
#include <cstdint>

#include "../../include/constellation_b200.h"
#include "act_vec.cuh"
#include "cst_common.cuh"
#include "kernels.h"

namespace cst {

namespace {

struct AddNormArgs {
    const void* x;
    int x_dtype;
    int64_t ld_x;
    const void* res;  // null: no residual
    int res_dtype;
    int64_t ld_res;
    int T, H;
    const float* weight;  // null: ones
    float eps;
    void* sum;  // [T, H] in res_dtype, or null
    int64_t ld_sum;
    void* out;
    int out_dtype;  // 1, 2, 3, or 4 = e4m3 with `scale`
    int64_t ld_out;
    float* scale;  // [T, ceil(H / 128)]
    int warps_per_row;
};

constexpr int kMaxNormWidth = 32768;  // 1024 threads x 32 elements in registers

// A row is held by `warps_per_row` warps, V vectors of VEC elements a thread; a block holds
// blockDim / 32 / warps_per_row rows.
template <int VEC, int V>
__global__ void __launch_bounds__(1024) add_norm_kernel(AddNormArgs a) {
    __shared__ float s_part[32];
    __shared__ float s_max[VEC == 1 ? 32 * V : 1];  // VEC 1: maxima of 32 consecutive elements
    chain_wait();
    chain_release();
    const int W = a.warps_per_row, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int local = warp / W, first_warp = local * W;
    const int64_t row = int64_t(blockIdx.x) * (int(blockDim.x >> 5) / W) + local;
    const bool live = row < a.T;
    const int tid = threadIdx.x - first_warp * 32, step = W * 32;

    float h[V][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (tid + v * step) * VEC;
        const bool in = live && c < a.H;
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[v][k] = 0.0f;
        if (in) load_act<VEC>(a.x, a.x_dtype, row * a.ld_x + c, h[v]);
    }
    if (a.res) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (tid + v * step) * VEC;
            if (!(live && c < a.H)) continue;
            float r[VEC];
            load_act<VEC>(a.res, a.res_dtype, row * a.ld_res + c, r);
#pragma unroll
            for (int k = 0; k < VEC; ++k) h[v][k] += r[k];
            if (a.sum) store_act<VEC>(a.sum, a.res_dtype, row * a.ld_sum + c, h[v]);
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < VEC; ++k) ss = fmaf(h[v][k], h[v][k], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (W > 1) {
        if (lane == 0) s_part[warp] = ss;
        __syncthreads();
        ss = 0.0f;
        for (int w = 0; w < W; ++w) ss += s_part[first_warp + w];  // fixed order
    }
    const float r = rsqrtf(ss / float(a.H) + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (tid + v * step) * VEC;
        if (c >= a.H) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) h[v][k] = h[v][k] * r * (a.weight ? __ldg(a.weight + c + k) : 1.0f);
    }
    if (a.out_dtype != 4) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (tid + v * step) * VEC;
            if (live && c < a.H) store_act<VEC>(a.out, a.out_dtype, row * a.ld_out + c, h[v]);
        }
        return;
    }
    // e4m3: the maximum of each 128 columns, 16 threads (VEC 8) or 4 warps' steps (VEC 1)
    float most[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        most[v] = 0.0f;
#pragma unroll
        for (int k = 0; k < VEC; ++k) most[v] = fmaxf(most[v], fabsf(h[v][k]));
#pragma unroll
        for (int o = VEC == 8 ? 8 : 16; o > 0; o >>= 1)
            most[v] = fmaxf(most[v], __shfl_xor_sync(0xffffffffu, most[v], o));
    }
    if constexpr (VEC == 1) {
        // 32-column piece j of the row at s_max[first_warp * V + j]
        if (lane == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) s_max[first_warp * V + v * W + (warp - first_warp)] = most[v];
        }
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int j = v * W + (warp - first_warp), j0 = j & ~3;
            for (int i = j0; i < j0 + 4 && i < W * V; ++i) most[v] = fmaxf(most[v], s_max[first_warp * V + i]);
        }
    }
    const int blocks = (a.H + 127) / 128;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = (tid + v * step) * VEC;
        if (!live || c >= a.H) continue;
        // a block of zeros takes scale 1; the smallest normal keeps 1 / s finite
        const float s = most[v] == 0.0f ? 1.0f : fmaxf(most[v] / 448.0f, FLT_MIN);
        const float inv = 1.0f / s;
        if (c % 128 == 0) a.scale[row * blocks + c / 128] = s;
        uint8_t* o = static_cast<uint8_t*>(a.out) + row * a.ld_out + c;
        if constexpr (VEC == 1) {
            *o = e4m3_rn(h[v][0] * inv);
        } else {
            uint32_t q[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) q[k] = e4m3x2_rn(h[v][2 * k] * inv, h[v][2 * k + 1] * inv);
            *reinterpret_cast<uint2*>(o) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
        }
    }
}

template <int VEC, int V>
cudaError_t launch(AddNormArgs a, cudaStream_t stream) {
    int W = 1;
    while (W * 32 * V * VEC < a.H) W *= 2;
    a.warps_per_row = W;
    const int warps = W < 8 ? 8 : W, rows = warps / W;
    return launch_chained(add_norm_kernel<VEC, V>, dim3((a.T + rows - 1) / rows), dim3(warps * 32), 0, stream, a);
}

}  // namespace

}  // namespace cst

using namespace cst;

extern "C" int cst_add_rmsnorm(const void* x, int32_t x_dtype, int64_t ld_x, const void* residual,
                               int32_t residual_dtype, int64_t ld_residual, int32_t T, int32_t H, const float* weight,
                               float eps, void* sum, int64_t ld_sum, void* out, int32_t out_dtype, int64_t ld_out,
                               float* scale, void* stream) {
    clear_last_error();
    auto act = [](int d) { return d >= CST_DTYPE_FP16 && d <= CST_DTYPE_FP32; };
    if (!act(x_dtype) || (residual && !act(residual_dtype)) || !(act(out_dtype) || out_dtype == CST_DTYPE_E4M3))
        return set_last_error(CST_ERR_INVALID_ARG, "invalid dtype (x %d, residual %d, out %d)", x_dtype,
                              residual_dtype, out_dtype);
    if (T < 0 || H < 1 || H > kMaxNormWidth)
        return set_last_error(CST_ERR_INVALID_ARG, "T=%d must be >= 0 and H=%d in [1, %d]", T, H, kMaxNormWidth);
    if (ld_x < H || ld_out < H || (residual && ld_residual < H) || (residual && sum && ld_sum < H))
        return set_last_error(CST_ERR_INVALID_ARG, "a row stride is below H=%d", H);
    if (!residual && sum)
        return set_last_error(CST_ERR_INVALID_ARG, "sum without a residual");
    if (T == 0) return CST_OK;
    if (!x || !out || (out_dtype == CST_DTYPE_E4M3 && !scale))
        return set_last_error(CST_ERR_INVALID_ARG, "null x, out or scale");
    AddNormArgs a{x, x_dtype, ld_x, residual, residual_dtype, ld_residual, T, H, weight, eps, sum, ld_sum, out,
                  out_dtype, ld_out, scale, 0};
    const bool vec = H % 8 == 0 && rows_aligned16(x, ld_x, act_size(x_dtype)) &&
                     (!residual || rows_aligned16(residual, ld_residual, act_size(residual_dtype))) &&
                     (!sum || rows_aligned16(sum, ld_sum, act_size(residual_dtype))) &&
                     (out_dtype == CST_DTYPE_E4M3
                          ? (reinterpret_cast<uintptr_t>(out) % 8 == 0 && ld_out % 8 == 0)
                          : rows_aligned16(out, ld_out, act_size(out_dtype)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = vec ? launch<8, 4>(a, s) : launch<1, 32>(a, s);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "add_rmsnorm launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}
