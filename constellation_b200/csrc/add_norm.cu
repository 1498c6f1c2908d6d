// Residual add + RMSNorm, and its form whose result leaves in 8 bits:
//     h[t, c]   = x[t, c] + residual[t, c]                                  (fp32)
//     sum[t, c] = h[t, c], rounded once to the residual's type
//     y[t, c]   = h[t, c] * rsqrt(mean_c(h[t, :]^2) + eps) * weight[c]      (fp32)
//     out[t, c] = y, rounded once; or, in e4m3 with one scale per 128 columns,
//     scale[t, b] = max_{c in b} |y[t, c]| / 448 (1 where a block is all zero),
//     out[t, c]   = e4m3(y[t, c] / scale[t, c / 128])
// The norm is taken of the unrounded h, and the row stays in registers between the sum of
// squares and the result, so each element is read once and written once: the kernel is bound
// by HBM, (2 + 2 + 2 + 1) bytes an element for bf16 to e4m3.  4096 x 7168 bf16 rows: to e4m3 39 us (5.3 TB/s),
// to bf16 38.6 us (6.1 TB/s); one row: 3.1 us, a launch and two trips to memory.
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

// A block of zeros takes scale 1; the smallest normal keeps 1 / s finite.
__device__ __forceinline__ float block_scale(float most) {
    return most == 0.0f ? 1.0f : fmaxf(most * (1.0f / 448.0f), FLT_MIN);
}

// 1 / s but for a unit or two of the last place, which only moves a value that lies between two of e4m3's.
__device__ __forceinline__ float quick_inverse(float s) { return __fdividef(1.0f, s); }

// A row is held by `warps_per_row` warps, V vectors of 8 elements a thread; a block holds
// blockDim / 32 / warps_per_row rows.  DT: the type of x, residual, sum and a 16- or 32-bit out when they
// all have it, 0 otherwise.  F8: the e4m3 form.  ANY: rows that start anywhere; the vectors then begin
// up to 7 columns before the row, on the 16-byte boundaries of the tensor that is written, and what is read
// is cut from two aligned pieces, which costs some 20 operations for 16 bytes: 4000 x 7001 bf16 to e4m3 110 us
// (1.8 TB/s), bound by them; 333 x 5001 fp16 6.2 us.
template <int V, int THREADS, int DT, bool F8, bool ANY>
__global__ void __launch_bounds__(THREADS) add_norm_kernel(AddNormArgs a) {
    __shared__ float s_part[32];
    __shared__ int s_most[F8 && ANY ? kMaxNormWidth / 128 : 1];  // ANY: a row's block maxima, as bits (one row a block)
    chain_wait();
    chain_release();
    const int W = a.warps_per_row, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int local = warp / W, first_warp = local * W;
    const int64_t row = int64_t(blockIdx.x) * (int(blockDim.x >> 5) / W) + local;
    const bool live = row < a.T;
    const int tid = threadIdx.x - first_warp * 32, step = W * 32;
    const int xt = DT ? DT : a.x_dtype, rt = DT ? DT : a.res_dtype, ot = DT ? DT : a.out_dtype;
    int lead = 0;
    if constexpr (ANY) {
        if (live) {
            lead = a.sum ? lead_in(a.sum, rt, row * a.ld_sum)
                   : F8  ? int((reinterpret_cast<uintptr_t>(a.out) + row * a.ld_out) & 7u)
                         : lead_in(a.out, ot, row * a.ld_out);
        }
        if constexpr (F8) {
            for (int i = threadIdx.x; i < (a.H + 127) / 128; i += blockDim.x) s_most[i] = 0;
        }
    }
    auto column = [&](int v) { return (tid + v * step) * 8 - lead; };
    // a vector may lie outside the row altogether: beyond its end
    auto within = [&](int c) { return live && c < a.H; };

    float h[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = column(v);
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] = 0.0f;
        if (!within(c)) continue;
        if constexpr (ANY) load8_any(a.x, xt, row * a.ld_x, c, a.H, h[v]);
        else load8(a.x, xt, row * a.ld_x + c, h[v]);
    }
    if (a.res) {
        // all loads before the first store, which the compiler has to take for one into the residual
        float r[V][8];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = column(v);
            if (!within(c)) continue;
            if constexpr (ANY) load8_any(a.res, rt, row * a.ld_res, c, a.H, r[v]);
            else load8(a.res, rt, row * a.ld_res + c, r[v]);
        }
        // in place, a neighbour's wide read must not meet a store of this row
        if constexpr (ANY) __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = column(v);
            if (!within(c)) continue;
#pragma unroll
            for (int k = 0; k < 8; ++k) h[v][k] += r[v][k];
            if (!a.sum) continue;
            if constexpr (ANY) store8_any(a.sum, rt, row * a.ld_sum, c, a.H, h[v]);
            else store8(a.sum, rt, row * a.ld_sum + c, h[v]);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = fmaf(h[v][k], h[v][k], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (W > 1 || ANY) {
        if (lane == 0) s_part[warp] = ss;
        __syncthreads();
        ss = 0.0f;
        for (int w = 0; w < W; ++w) ss += s_part[first_warp + w];  // fixed order
    }
    const float r = rsqrtf(ss / float(a.H) + a.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = column(v);
        float w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = 1.0f;
        if (a.weight && c < a.H) {
            if constexpr (ANY) load8_any(a.weight, CST_DTYPE_FP32, 0, c, a.H, w);
            else load8(a.weight, CST_DTYPE_FP32, c, w);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) h[v][k] = h[v][k] * r * w[k];
        if constexpr (!F8) {
            if (!within(c)) continue;
            if constexpr (ANY) store8_any(a.out, ot, row * a.ld_out, c, a.H, h[v]);
            else store8(a.out, ot, row * a.ld_out + c, h[v]);
        }
    }
    if constexpr (F8) {
        const int blocks = (a.H + 127) / 128;
        uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.ld_out;
        if constexpr (!ANY) {
            // the maximum of 128 columns: 16 threads
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = column(v);
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(h[v][k]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (!within(c)) continue;
                const float s = block_scale(most), inv = quick_inverse(s);
                if (c % 128 == 0) a.scale[row * blocks + c / 128] = s;
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = e4m3x2_rn(h[v][2 * k] * inv, h[v][2 * k + 1] * inv);
                *reinterpret_cast<uint2*>(out + c) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
            }
        } else {
            // a vector may belong to two blocks; the maximum does not depend on the order it is taken in
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = column(v);
                if (!within(c)) continue;
                const int b0 = max(c, 0) >> 7, edge = (b0 + 1) << 7;
                float most0 = 0.0f, most1 = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {  // columns outside the row are zero
                    const float m = fabsf(h[v][k]);
                    most0 = fmaxf(most0, c + k < edge ? m : 0.0f);
                    most1 = fmaxf(most1, c + k < edge ? 0.0f : m);
                }
                atomicMax(&s_most[b0], __float_as_int(most0));
                if (c + 8 > edge && edge < a.H) atomicMax(&s_most[b0 + 1], __float_as_int(most1));
            }
            __syncthreads();
            if (live)
                for (int i = tid; i < blocks; i += step) a.scale[row * blocks + i] = block_scale(__int_as_float(s_most[i]));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = column(v);
                if (!within(c)) continue;
                const int b0 = max(c, 0) >> 7, edge = (b0 + 1) << 7;
                const float inv0 = quick_inverse(block_scale(__int_as_float(s_most[b0])));
                const float inv1 = c + 8 > edge && edge < a.H ? quick_inverse(block_scale(__int_as_float(s_most[b0 + 1]))) : inv0;
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    q[k] = e4m3x2_rn(h[v][2 * k] * (c + 2 * k >= edge ? inv1 : inv0),
                                     h[v][2 * k + 1] * (c + 2 * k + 1 >= edge ? inv1 : inv0));
                const uint2 both = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
                if (c >= 0 && c + 8 <= a.H && (reinterpret_cast<uintptr_t>(out + c) & 7u) == 0) {
                    *reinterpret_cast<uint2*>(out + c) = both;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        if (unsigned(c + k) < unsigned(a.H))
                            out[c + k] = uint8_t((k < 4 ? both.x >> (8 * k) : both.y >> (8 * (k - 4))) & 255u);
                }
            }
        }
    }
}

// Many aligned rows of one 16-bit type: a block goes from row to row and has the next row's loads in flight
// while it finishes one, which a block a row has not: 4096 x 7168 bf16 to e4m3 39 us (57 us that way), 2048 x 16384
// 50 us (69), to bf16 43 us (6.2 TB/s).
template <int V, int THREADS, int DT, bool F8>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) add_norm_stream_kernel(AddNormArgs a) {
    __shared__ float s_part[2][32];
    chain_wait();
    chain_release();
    const int W = a.warps_per_row, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int local = warp / W, first_warp = local * W, rows = int(blockDim.x >> 5) / W;
    const int tid = threadIdx.x - first_warp * 32, step = W * 32;
    const int blocks = (a.H + 127) / 128;
    uint4 x[V], r[V];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (tid + v * step) * 8;
            const bool in = row < a.T && c < a.H;
            x[v] = r[v] = make_uint4(0, 0, 0, 0);
            if (in) x[v] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.ld_x + c);
            if (in && a.res) r[v] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.res) + row * a.ld_res + c);
        }
    };
    int64_t row = int64_t(blockIdx.x) * rows + local;
    load(row);
    // every warp of the block makes the same number of turns
    for (int64_t first = int64_t(blockIdx.x) * rows, turn = 0; first < a.T; first += int64_t(gridDim.x) * rows, ++turn) {
        const int64_t next = row + int64_t(gridDim.x) * rows;
        const bool live = row < a.T;
        float h[V][8], ss = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float e[8];
            unpack8(x[v], DT, h[v]);
            unpack8(r[v], DT, e);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                h[v][k] += e[k];
                ss = fmaf(h[v][k], h[v][k], ss);
            }
        }
        load(next);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (W > 1) {
            if (lane == 0) s_part[turn & 1][warp] = ss;
            __syncthreads();
            ss = 0.0f;
            for (int w = 0; w < W; ++w) ss += s_part[turn & 1][first_warp + w];  // fixed order
        }
        const float inv_rms = rsqrtf(ss / float(a.H) + a.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = (tid + v * step) * 8;
            const bool in = live && c < a.H;
            if (in && a.sum) store8(a.sum, DT, row * a.ld_sum + c, h[v]);
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = 1.0f;
            if (a.weight && c < a.H) load8(a.weight, CST_DTYPE_FP32, c, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) h[v][k] = h[v][k] * inv_rms * w[k];
            if constexpr (!F8) {
                if (in) store8(a.out, DT, row * a.ld_out + c, h[v]);
            } else {
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(h[v][k]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (!in) continue;
                const float s = block_scale(most), inv = quick_inverse(s);
                if (c % 128 == 0) a.scale[row * blocks + c / 128] = s;
                uint32_t q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = e4m3x2_rn(h[v][2 * k] * inv, h[v][2 * k + 1] * inv);
                *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.out) + row * a.ld_out + c) =
                    make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
            }
        }
        row = next;
    }
}

template <int V, int THREADS, int DT>
cudaError_t launch_stream(AddNormArgs a, int sms, cudaStream_t stream) {
    const int W = (a.H + 32 * V * 8 - 1) / (32 * V * 8);
    a.warps_per_row = W;
    const int rows = W >= 8 ? 1 : 8 / W, threads = rows * W * 32;
    const int64_t ctas = (int64_t(a.T) + rows - 1) / rows, fit = int64_t(sms) * (1024 / threads > 1 ? 1024 / threads : 1);
    auto kernel = a.out_dtype == CST_DTYPE_E4M3 ? add_norm_stream_kernel<V, THREADS, DT, true>
                                                : add_norm_stream_kernel<V, THREADS, DT, false>;
    return launch_chained(kernel, dim3(unsigned(ctas < fit ? ctas : fit)), dim3(threads), 0, stream, a);
}

template <int V, int THREADS, int DT, bool ANY>
cudaError_t launch(AddNormArgs a, cudaStream_t stream) {
    const int W = (a.H + (ANY ? 7 : 0) + 32 * V * 8 - 1) / (32 * V * 8);  // ANY: up to 7 columns before the row
    a.warps_per_row = W;
    const int rows = ANY || W >= 8 ? 1 : 8 / W;
    auto kernel = a.out_dtype == CST_DTYPE_E4M3 ? add_norm_kernel<V, THREADS, DT, true, ANY>
                                                : add_norm_kernel<V, THREADS, DT, false, ANY>;
    return launch_chained(kernel, dim3((a.T + rows - 1) / rows), dim3(rows * W * 32), 0, stream, a);
}

template <int DT>
cudaError_t launch_aligned(const AddNormArgs& a, int sms, cudaStream_t s) {
    // Few rows: as many threads a row as it has vectors.  Many: 2 vectors a thread, whose loads are all in
    // flight at once.
    if (a.H > 16384) return launch<4, 1024, DT, false>(a, s);  // holds more than 64 registers a thread: spills
    if (a.H > 8192) {
        if constexpr (DT == CST_DTYPE_BF16 || DT == CST_DTYPE_FP16) {
            if (a.T > 2 * sms) return launch_stream<2, 1024, DT>(a, sms, s);
        }
        return launch<2, 1024, DT, false>(a, s);
    }
    if (a.T <= 4 * sms) return launch<1, 1024, DT, false>(a, s);
    if constexpr (DT == CST_DTYPE_BF16 || DT == CST_DTYPE_FP16) {
        if (a.H <= 256) return launch_stream<1, 256, DT>(a, sms, s);
        return launch_stream<2, 512, DT>(a, sms, s);
    }
    return launch<2, 512, DT, false>(a, s);
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
    if (T < 0 || T > (1 << 30) || H < 1 || H > kMaxNormWidth)
        return set_last_error(CST_ERR_INVALID_ARG, "T=%d must be in [0, 2^30] and H=%d in [1, %d]", T, H, kMaxNormWidth);
    if (ld_x < H || ld_out < H || (residual && ld_residual < H) || (residual && sum && ld_sum < H))
        return set_last_error(CST_ERR_INVALID_ARG, "a row stride is below H=%d", H);
    if (!residual && sum)
        return set_last_error(CST_ERR_INVALID_ARG, "sum without a residual");
    if (T == 0) return CST_OK;
    if (!x || !out || (out_dtype == CST_DTYPE_E4M3 && !scale))
        return set_last_error(CST_ERR_INVALID_ARG, "null x, out or scale");
    AddNormArgs a{x, x_dtype, ld_x, residual, residual_dtype, ld_residual, T, H, weight, eps, sum, ld_sum, out,
                  out_dtype, ld_out, scale, 0};
    const bool f8 = out_dtype == CST_DTYPE_E4M3;
    const bool aligned = H % 8 == 0 && (reinterpret_cast<uintptr_t>(weight) & 15u) == 0 &&
                         rows_aligned16(x, ld_x, act_size(x_dtype)) &&
                         (!residual || rows_aligned16(residual, ld_residual, act_size(residual_dtype))) &&
                         (!sum || rows_aligned16(sum, ld_sum, act_size(residual_dtype))) &&
                         (f8 ? (reinterpret_cast<uintptr_t>(out) % 8 == 0 && ld_out % 8 == 0)
                             : rows_aligned16(out, ld_out, act_size(out_dtype)));
    const bool same = (!residual || residual_dtype == x_dtype) && (f8 || out_dtype == x_dtype);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int sms = current_sms();
    const cudaError_t e = !aligned && H > 16377 ? launch<5, 1024, 0, true>(a, s)
                          : !aligned && H > 8185 ? launch<2, 1024, 0, true>(a, s)
                          : !aligned && same && x_dtype == CST_DTYPE_BF16 ? launch<2, 512, 2, true>(a, s)
                          : !aligned && same && x_dtype == CST_DTYPE_FP16 ? launch<2, 512, 1, true>(a, s)
                          : !aligned ? launch<2, 512, 0, true>(a, s)
                          : !same  ? launch_aligned<0>(a, sms, s)
                          : x_dtype == CST_DTYPE_BF16 ? launch_aligned<2>(a, sms, s)
                          : x_dtype == CST_DTYPE_FP16 ? launch_aligned<1>(a, sms, s)
                                                      : launch_aligned<3>(a, sms, s);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "add_rmsnorm launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}
