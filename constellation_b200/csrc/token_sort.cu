// Tokens sorted by expert and back.  A token t has K routes (t, k) to experts; with the routes of
// the experts held here numbered in the order (expert, t, k),
//     row_of[t, k]  = that number, or -1 where the expert is not held here
//     route_of[row] = t * K + k, -1 for the rows behind the last expert's
//     offsets[e]    = first row of expert e; offsets[E] = rows in use
//     sort:          rows[row_of[t, k]] = x[t]; rows behind offsets[E] are zero
//     unsort:        out[t] = sum_k weight[t, k] * rows[row_of[t, k]] (+ residual[t])
//     unsort's gradients for g = d out:
//                    d rows[row_of[t, k]] = weight[t, k] * g[t]; zero behind offsets[E]
//                    d weight[t, k]       = <g[t], rows[row_of[t, k]]>, 0 for an absent route
// (sort's gradient is unsort without weights.)  Sums run in fp32 in the order of k with one
// rounding at the end; no atomics, so results repeat bit for bit.
#include <cooperative_groups.h>
#include <cstdint>

#include "../../include/constellation_b200.h"
#include "act_vec.cuh"
#include "cst_common.cuh"
#include "kernels.h"

namespace cst {

namespace cg = cooperative_groups;

namespace {

// ---- order ------------------------------------------------------------------------------
// A stable counting sort by one cluster: every warp owns a contiguous run of routes and a
// histogram of its own in shared memory; the CTAs read one another's totals over distributed
// shared memory, so there is one launch and no workspace.

constexpr int kSortWarps = 16;
constexpr int kSortMaxCluster = 8;
constexpr int kSortMaxExperts = 1024;

struct OrderArgs {
    const void* idx;
    int idx64;
    int n;  // routes
    int E, first;
    int32_t* row_of;
    int32_t* route_of;
    int32_t* offsets;
};

__device__ __forceinline__ int local_expert(const OrderArgs& a, int i) {
    const int64_t v = a.idx64 ? static_cast<const int64_t*>(a.idx)[i] : static_cast<const int32_t*>(a.idx)[i];
    const int64_t e = v - a.first;
    return (v >= 0 && e >= 0 && e < a.E) ? int(e) : a.E;
}

__global__ void __launch_bounds__(kSortWarps * 32) order_kernel(OrderArgs a) {
    extern __shared__ int32_t s_hist[];  // [kSortWarps][E + 1], then totals [E + 1], then bases [E + 2]
    __shared__ int32_t s_warp[kSortWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), ranks = int(cluster.num_blocks());
    const int B = a.E + 1;
    int32_t* s_total = s_hist + kSortWarps * B;
    int32_t* s_base = s_total + B;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < kSortWarps * B; i += blockDim.x) s_hist[i] = 0;
    chain_wait();
    chain_release();
    __syncthreads();
    // this warp's routes [lo, hi)
    const int runs = ranks * kSortWarps, run = rank * kSortWarps + warp;
    const int per = (a.n + runs - 1) / runs;
    const int lo = int(min(int64_t(run) * per, int64_t(a.n))), hi = int(min(int64_t(lo) + per, int64_t(a.n)));
    int32_t* mine = s_hist + warp * B;
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < hi ? local_expert(a, i) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
        __syncwarp();
    }
    __syncthreads();
    // per expert: exclusive prefix over the warps, and this CTA's total
    for (int e = threadIdx.x; e < B; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < kSortWarps; ++w) {
            const int c = s_hist[w * B + e];
            s_hist[w * B + e] = sum;
            sum += c;
        }
        s_total[e] = sum;
    }
    cluster.sync();
    // all CTAs' totals of every expert, scanned over the experts (chunks of blockDim experts)
    int carry = 0;
    for (int e0 = 0; e0 < B; e0 += blockDim.x) {
        const int e = e0 + int(threadIdx.x);
        int all = 0, before = 0;
        if (e < B) {
            for (int r = 0; r < ranks; ++r) {
                const int c = *cluster.map_shared_rank(s_total + e, r);
                if (r < rank) before += c;
                all += c;
            }
        }
        int inc = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        int base = carry;
        for (int w = 0; w < warp; ++w) base += s_warp[w];
        for (int w = 0; w < kSortWarps; ++w) carry += s_warp[w];
        const int first = base + inc - all;
        if (e < B) {
            s_base[e] = first + before;
            if (rank == 0) a.offsets[e] = first;  // e == E: the rows in use
        }
        __syncthreads();
    }
    cluster.sync();  // no CTA leaves while another still reads its totals
    for (int i0 = lo; i0 < hi; i0 += 32) {
        const int i = i0 + lane;
        const int e = i < hi ? local_expert(a, i) : -1;
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        if (e >= 0) {
            const int row = s_base[e] + mine[e] + __popc(peers & ((1u << lane) - 1u));
            a.row_of[i] = e == a.E ? -1 : row;
            a.route_of[row] = e == a.E ? -1 : i;
        }
        __syncwarp();
        if (e >= 0 && lane == __ffs(peers) - 1) mine[e] += __popc(peers);
        __syncwarp();
    }
}

// ---- rows -------------------------------------------------------------------------------

struct CopyArgs {
    const uint8_t* x;  // [T] rows of `bytes`, ld_x bytes apart
    int64_t bytes, ld_x;
    const uint8_t* scale;  // second plane (row scales), or null
    int64_t sbytes, ld_scale;
    int T, K;
    const int32_t* row_of;
    const int32_t* rows_used;
    uint8_t* rows;   // [T * K] rows of `bytes`, packed
    uint8_t* srows;  // [T * K] rows of `sbytes`, packed
};

template <typename U>
__device__ __forceinline__ void spread(const uint8_t* src, uint8_t* rows, int64_t bytes, const int32_t* row, int K,
                                       int R) {
    const U* s = reinterpret_cast<const U*>(src);
    const int64_t n = bytes / int64_t(sizeof(U));
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) {
        const U v = s[i];
        for (int k = 0; k < K; ++k) {
            const int r = __ldg(row + k);
            if (unsigned(r) < unsigned(R)) reinterpret_cast<U*>(rows + r * bytes)[i] = v;
        }
    }
}

template <typename U>
__device__ __forceinline__ void clear(uint8_t* dst, int64_t bytes) {
    const int64_t n = bytes / int64_t(sizeof(U));
    U z{};
    for (int64_t i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<U*>(dst)[i] = z;
}

// Blocks of tokens first, then the rows behind the last expert's.
template <typename U, typename S>
__global__ void __launch_bounds__(256) sort_rows_kernel(CopyArgs a) {
    chain_wait();
    chain_release();
    const int R = a.T * a.K;
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        const int32_t* row = a.row_of + int64_t(t) * a.K;
        spread<U>(a.x + t * a.ld_x, a.rows, a.bytes, row, a.K, R);
        if (a.scale) spread<S>(a.scale + t * a.ld_scale, a.srows, a.sbytes, row, a.K, R);
    }
    const int used = max(0, min(*a.rows_used, R));
    for (int64_t r = used + int64_t(blockIdx.x); r < R; r += gridDim.x) {
        clear<U>(a.rows + r * a.bytes, a.bytes);
        if (a.scale) clear<S>(a.srows + r * a.sbytes, a.sbytes);
    }
}

// ---- back to the tokens -----------------------------------------------------------------

struct UnsortArgs {
    const void* rows;
    int dtype;
    int64_t ld;
    const int32_t* row_of;
    const float* weight;  // [T, K] or null (ones)
    int T, K, H;
    const void* res;
    int res_dtype;
    int64_t ld_res;
    void* out;
    int out_dtype;
};

template <int VEC>
__global__ void __launch_bounds__(256) unsort_kernel(UnsortArgs a) {
    chain_wait();
    chain_release();
    const int t = blockIdx.x, R = a.T * a.K;
    const int32_t* row = a.row_of + int64_t(t) * a.K;
    const float* weight = a.weight ? a.weight + int64_t(t) * a.K : nullptr;
    for (int c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC; c < a.H; c += gridDim.y * blockDim.x * VEC) {
        float acc[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        for (int k = 0; k < a.K; ++k) {
            const int r = __ldg(row + k);
            if (unsigned(r) >= unsigned(R)) continue;
            const float w = weight ? __ldg(weight + k) : 1.0f;
            float v[VEC];
            load_act<VEC>(a.rows, a.dtype, r * a.ld + c, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w, v[i], acc[i]);
        }
        if (a.res) {
            float v[VEC];
            load_act<VEC>(a.res, a.res_dtype, t * a.ld_res + c, v);
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[i] += v[i];
        }
        store_act<VEC>(a.out, a.out_dtype, int64_t(t) * a.H + c, acc);
    }
}

struct UnsortGradArgs {
    const void* g;
    int g_dtype;
    int64_t ld_g;
    const void* rows;  // null: no weight gradient
    int dtype;         // of rows and d_rows
    int64_t ld;
    const int32_t* row_of;
    const float* weight;
    const int32_t* rows_used;
    int T, K, H;
    void* d_rows;     // [T * K, H] packed, or null
    float* d_weight;  // [T, K], or null
};

template <int VEC>
__global__ void __launch_bounds__(256) unsort_grad_kernel(UnsortGradArgs a) {
    __shared__ float s_part[8];
    chain_wait();
    chain_release();
    const int R = a.T * a.K;
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        for (int k = 0; k < a.K; ++k) {
            const int r = __ldg(a.row_of + int64_t(t) * a.K + k);
            const bool here = unsigned(r) < unsigned(R);
            const float w = a.weight ? __ldg(a.weight + int64_t(t) * a.K + k) : 1.0f;
            float dot = 0.0f;
            if (here) {
                for (int c = threadIdx.x * VEC; c < a.H; c += blockDim.x * VEC) {
                    float g[VEC], v[VEC];
                    load_act<VEC>(a.g, a.g_dtype, t * a.ld_g + c, g);
                    if (a.d_weight) {
                        load_act<VEC>(a.rows, a.dtype, r * a.ld + c, v);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) dot = fmaf(g[i], v[i], dot);
                    }
                    if (a.d_rows) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[i] = w * g[i];
                        store_act<VEC>(a.d_rows, a.dtype, int64_t(r) * a.H + c, v);
                    }
                }
            }
            if (a.d_weight) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = dot;
                __syncthreads();
                if (threadIdx.x == 0) {
                    float sum = 0.0f;
                    for (int i = 0; i < 8; ++i) sum += s_part[i];
                    a.d_weight[int64_t(t) * a.K + k] = here ? sum : 0.0f;
                }
                __syncthreads();
            }
        }
    }
    if (!a.d_rows) return;
    const int used = max(0, min(*a.rows_used, R));
    float zero[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) zero[i] = 0.0f;
    for (int64_t r = used + int64_t(blockIdx.x); r < R; r += gridDim.x)
        for (int c = threadIdx.x * VEC; c < a.H; c += blockDim.x * VEC)
            store_act<VEC>(a.d_rows, a.dtype, r * a.H + c, zero);
}

cudaError_t launch_order(const OrderArgs& a, cudaStream_t stream) {
    const size_t smem = size_t(kSortWarps + 2) * (a.E + 1) * 4;
    cudaError_t e = cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
    const int ranks = a.n > 4096 ? kSortMaxCluster : 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ranks);
    cfg.blockDim = dim3(kSortWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, order_kernel, a);
}

bool act_dtype(int d) { return d >= CST_DTYPE_FP16 && d <= CST_DTYPE_FP32; }

// The largest power of two up to 16 that divides all of a plane's addresses and strides.
int copy_unit(const void* a, const void* b, int64_t bytes, int64_t ld) {
    const uint64_t all = reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | uint64_t(bytes) |
                         uint64_t(ld) | 16u;
    return int(all & (~all + 1));
}

template <typename U>
cudaError_t launch_sort_rows(const CopyArgs& a, int sunit, int grid, cudaStream_t s) {
    if (sunit >= 16) return launch_chained(sort_rows_kernel<U, uint4>, dim3(grid), dim3(256), 0, s, a);
    return launch_chained(sort_rows_kernel<U, uint32_t>, dim3(grid), dim3(256), 0, s, a);
}

int check_routes(const char* what, int64_t T, int64_t K) {
    if (T < 0 || K < 1 || K > CST_SORT_MAX_TOP_K || T * K > (int64_t(1) << 30))
        return set_last_error(CST_ERR_INVALID_ARG, "%s: T=%lld must be >= 0, K=%lld in [1, %d] and T * K at most 2^30",
                              what, (long long)T, (long long)K, CST_SORT_MAX_TOP_K);
    return CST_OK;
}

int launched(const char* what, cudaError_t e) {
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "%s launch failed: %s", what, cudaGetErrorString(e));
    return CST_OK;
}

}  // namespace

}  // namespace cst

using namespace cst;

extern "C" int cst_sort_routes(const void* topk_idx, int32_t idx_bytes, int32_t T, int32_t K, int32_t n_experts,
                               int32_t first_expert, int32_t* row_of, int32_t* route_of, int32_t* offsets,
                               void* stream) {
    clear_last_error();
    if (const int rc = check_routes("sort_routes", T, K)) return rc;
    if (idx_bytes != 4 && idx_bytes != 8)
        return set_last_error(CST_ERR_INVALID_ARG, "idx_bytes must be 4 or 8, got %d", idx_bytes);
    if (n_experts < 1 || n_experts > kSortMaxExperts || first_expert < 0)
        return set_last_error(CST_ERR_INVALID_ARG, "n_experts=%d must be in [1, %d] and first_expert=%d >= 0",
                              n_experts, kSortMaxExperts, first_expert);
    if (!offsets || (T > 0 && (!topk_idx || !row_of || !route_of)))
        return set_last_error(CST_ERR_INVALID_ARG, "null index or output");
    const OrderArgs a{topk_idx, idx_bytes == 8, T * K, n_experts, first_expert, row_of, route_of, offsets};
    return launched("sort_routes", launch_order(a, static_cast<cudaStream_t>(stream)));
}

extern "C" int cst_sort_rows(const void* x, int64_t row_bytes, int64_t ld_bytes, const float* scale, int32_t n_scale,
                             int64_t ld_scale, int32_t T, int32_t K, const int32_t* row_of, const int32_t* rows_used,
                             void* rows, float* rows_scale, void* stream) {
    clear_last_error();
    if (const int rc = check_routes("sort_rows", T, K)) return rc;
    if (row_bytes < 1 || ld_bytes < row_bytes || (scale && (n_scale < 1 || ld_scale < n_scale)))
        return set_last_error(CST_ERR_INVALID_ARG, "row sizes must be positive and strides at least as long");
    if (T == 0) return CST_OK;
    if (!x || !row_of || !rows_used || !rows || (scale && !rows_scale))
        return set_last_error(CST_ERR_INVALID_ARG, "null x, order or rows");
    const CopyArgs a{static_cast<const uint8_t*>(x), row_bytes, ld_bytes, reinterpret_cast<const uint8_t*>(scale),
                     int64_t(n_scale) * 4, ld_scale * 4, T, K, row_of, rows_used, static_cast<uint8_t*>(rows),
                     reinterpret_cast<uint8_t*>(rows_scale)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int unit = copy_unit(x, rows, row_bytes, ld_bytes);
    const int sunit = scale ? copy_unit(scale, rows_scale, a.sbytes, a.ld_scale) : 4;
    const int grid = T;
    cudaError_t e;
    switch (unit) {
        case 16: e = launch_sort_rows<uint4>(a, sunit, grid, s); break;
        case 8: e = launch_sort_rows<uint2>(a, sunit, grid, s); break;
        case 4: e = launch_sort_rows<uint32_t>(a, sunit, grid, s); break;
        case 2: e = launch_sort_rows<uint16_t>(a, sunit, grid, s); break;
        default: e = launch_sort_rows<uint8_t>(a, sunit, grid, s); break;
    }
    return launched("sort_rows", e);
}

extern "C" int cst_unsort_rows(const void* rows, int32_t rows_dtype, int64_t ld_rows, const int32_t* row_of,
                               const float* weight, int32_t T, int32_t K, int32_t H, const void* residual,
                               int32_t residual_dtype, int64_t ld_residual, void* out, int32_t out_dtype,
                               void* stream) {
    clear_last_error();
    if (const int rc = check_routes("unsort_rows", T, K)) return rc;
    if (!act_dtype(rows_dtype) || !act_dtype(out_dtype) || (residual && !act_dtype(residual_dtype)))
        return set_last_error(CST_ERR_INVALID_ARG, "invalid dtype (rows %d, residual %d, out %d)", rows_dtype,
                              residual_dtype, out_dtype);
    if (H < 1 || ld_rows < H || (residual && ld_residual < H))
        return set_last_error(CST_ERR_INVALID_ARG, "H=%d must be positive and no row stride below it", H);
    if (T == 0) return CST_OK;
    if (!rows || !row_of || !out) return set_last_error(CST_ERR_INVALID_ARG, "null rows, order or out");
    const UnsortArgs a{rows, rows_dtype, ld_rows, row_of, weight, T, K, H, residual, residual_dtype, ld_residual, out,
                       out_dtype};
    const bool vec = H % 8 == 0 && rows_aligned16(rows, ld_rows, act_size(rows_dtype)) &&
                     rows_aligned16(out, H, act_size(out_dtype)) &&
                     (!residual || rows_aligned16(residual, ld_residual, act_size(residual_dtype)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int V = vec ? 8 : 1;
    const dim3 grid(T, (H + 256 * V - 1) / (256 * V));
    return launched("unsort_rows", vec ? launch_chained(unsort_kernel<8>, grid, dim3(256), 0, s, a)
                                       : launch_chained(unsort_kernel<1>, grid, dim3(256), 0, s, a));
}

extern "C" int cst_unsort_rows_grad(const void* grad, int32_t grad_dtype, int64_t ld_grad, const void* rows,
                                    int32_t rows_dtype, int64_t ld_rows, const int32_t* row_of, const float* weight,
                                    const int32_t* rows_used, int32_t T, int32_t K, int32_t H, void* d_rows,
                                    float* d_weight, void* stream) {
    clear_last_error();
    if (const int rc = check_routes("unsort_rows_grad", T, K)) return rc;
    if (!act_dtype(grad_dtype) || !act_dtype(rows_dtype))
        return set_last_error(CST_ERR_INVALID_ARG, "invalid dtype (grad %d, rows %d)", grad_dtype, rows_dtype);
    if (H < 1 || ld_grad < H || (d_weight && ld_rows < H))
        return set_last_error(CST_ERR_INVALID_ARG, "H=%d must be positive and no row stride below it", H);
    if (T == 0 || (!d_rows && !d_weight)) return CST_OK;
    if (!grad || !row_of || !rows_used || (d_weight && !rows))
        return set_last_error(CST_ERR_INVALID_ARG, "null grad, rows or order");
    const UnsortGradArgs a{grad, grad_dtype, ld_grad, rows, rows_dtype, ld_rows, row_of, weight, rows_used, T, K, H,
                           d_rows, d_weight};
    const bool vec = H % 8 == 0 && rows_aligned16(grad, ld_grad, act_size(grad_dtype)) &&
                     (!d_weight || rows_aligned16(rows, ld_rows, act_size(rows_dtype))) &&
                     (!d_rows || rows_aligned16(d_rows, H, act_size(rows_dtype)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launched("unsort_rows_grad", vec ? launch_chained(unsort_grad_kernel<8>, dim3(T), dim3(256), 0, s, a)
                                            : launch_chained(unsort_grad_kernel<1>, dim3(T), dim3(256), 0, s, a));
}
