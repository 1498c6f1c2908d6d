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
// shared memory, so there is one launch and no workspace.  A run is taken 256 routes at a time, whose
// loads are all in flight at once: the wait for memory, not the counting, is what a run costs.  Up to 2048 routes
// 5 us, 16384 8 us, 131072 25 us (of which the launch alone is 2).

constexpr int kSortMaxWarps = 32, kSortMinWarps = 8;
constexpr int kSortHeld = 8;  // routes of a lane at a time
constexpr int kSortMaxCluster = 8;
constexpr int kSortMaxExperts = 1024;

struct OrderArgs {
    const void* idx;
    int idx64;
    int n;  // routes
    int E, first;
    int bits;  // of a number up to E, and one more, which only -1 has
    int32_t* row_of;
    int32_t* route_of;
    int32_t* offsets;
};

__device__ __forceinline__ int local_expert(const OrderArgs& a, int i) {
    const int64_t v = a.idx64 ? static_cast<const int64_t*>(a.idx)[i] : static_cast<const int32_t*>(a.idx)[i];
    const int64_t e = v - a.first;
    return (v >= 0 && e >= 0 && e < a.E) ? int(e) : a.E;
}

// The lanes whose expert is this lane's, from one vote a bit of the expert's number (-1 has all of them set).
__device__ __forceinline__ unsigned same_expert(int e, int bits) {
    unsigned peers = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = (e >> b) & 1;
        const unsigned vote = __ballot_sync(0xffffffffu, set);
        peers &= set ? vote : ~vote;
    }
    return peers;
}

__global__ void __launch_bounds__(kSortMaxWarps * 32) order_kernel(OrderArgs a) {
    extern __shared__ int32_t s_hist[];  // [warps][E + 1], then totals [E + 1], then bases [E + 1]
    __shared__ int32_t s_warp[kSortMaxWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = int(cluster.block_rank()), ranks = int(cluster.num_blocks());
    const int B = a.E + 1, warps = blockDim.x >> 5;
    int32_t* s_total = s_hist + warps * B;
    int32_t* s_base = s_total + B;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int i = threadIdx.x; i < warps * B; i += blockDim.x) s_hist[i] = 0;
    chain_wait();
    chain_release();
    __syncthreads();
    // this warp's routes [lo, hi)
    const int runs = ranks * warps, run = rank * warps + warp;
    const int per = (a.n + runs - 1) / runs;
    const int lo = int(min(int64_t(run) * per, int64_t(a.n))), hi = int(min(int64_t(lo) + per, int64_t(a.n)));
    int32_t* mine = s_hist + warp * B;
    int held[kSortHeld];
    auto load = [&](int i0) {
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j) {
            const int i = i0 + j * 32 + lane;
            held[j] = i < hi ? local_expert(a, i) : -1;
        }
    };
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortHeld) {
        load(i0);
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j) {
            if (i0 + j * 32 >= hi) break;
            if (held[j] >= 0) atomicAdd(&mine[held[j]], 1);  // whole numbers: the order does not matter
        }
    }
    __syncthreads();
    // per expert: exclusive prefix over the warps, and this CTA's total
    for (int e = threadIdx.x; e < B; e += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < warps; ++w) {
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
        for (int w = 0; w < warps; ++w) carry += s_warp[w];
        const int first = base + inc - all;
        if (e < B) {
            s_base[e] = first + before;
            if (rank == 0) a.offsets[e] = first;  // e == E: the rows in use
        }
        __syncthreads();
    }
    cluster.sync();  // no CTA leaves while another still reads its totals
    for (int i0 = lo; i0 < hi; i0 += 32 * kSortHeld) {
        if (hi - lo > 32 * kSortHeld) load(i0);  // a short run is still held
#pragma unroll
        for (int j = 0; j < kSortHeld; ++j) {
            if (i0 + j * 32 >= hi) break;
            const int i = i0 + j * 32 + lane, e = held[j];
            const unsigned peers = same_expert(e, a.bits);
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
}

// ---- rows -------------------------------------------------------------------------------

struct CopyArgs {
    const uint8_t* x;  // [T] rows of `bytes`, ld_x bytes apart
    int64_t bytes, ld_x;
    const uint32_t* scale;  // [T] rows of n_scale words, ld_scale words apart, or null
    int n_scale;
    int64_t ld_scale;
    int T, K;
    const int32_t* row_of;
    const int32_t* rows_used;
    uint8_t* rows;    // [T * K] rows of `bytes`, packed
    uint32_t* srows;  // [T * K] rows of n_scale words, packed
};

// Bytes [at, at + 16) of a row of `bytes`, of which those in the row are written; dst + at is 16-byte aligned.
__device__ __forceinline__ void store16_any(uint8_t* dst, int64_t at, int64_t bytes, const uint4& u) {
    if (at >= 0 && at + 16 <= bytes) {
        *reinterpret_cast<uint4*>(dst + at) = u;
    } else {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (uint64_t(at + k) < uint64_t(bytes)) dst[at + k] = uint8_t(w[k >> 2] >> (8 * (k & 3)));
    }
}

// ANY: rows that start anywhere.  Each copy of a row then lies on 16-byte boundaries of its own, and its
// pieces are read shifted from the one source row, which the CTA's first copy brought into L1.
template <bool ANY>
__device__ __forceinline__ void copy_row(const uint8_t* src, uint8_t* dst, int64_t bytes) {
    const int64_t lead = ANY ? int64_t(reinterpret_cast<uintptr_t>(dst) & 15u) : 0;
    for (int64_t at = int64_t(threadIdx.x) * 16 - lead; at < bytes; at += int64_t(blockDim.x) * 16) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (src == nullptr) {
        } else if (!ANY) {
            u = *reinterpret_cast<const uint4*>(src + at);
        } else if (at >= 16 && at + 32 <= bytes) {
            u = load16_any(src + at);
        } else {
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (uint64_t(at + k) < uint64_t(bytes)) w[k >> 2] |= uint32_t(src[at + k]) << (8 * (k & 3));
            u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (!ANY) *reinterpret_cast<uint4*>(dst + at) = u;
        else store16_any(dst, at, bytes, u);
    }
}

__device__ __forceinline__ void clear_tail(const CopyArgs& a, int used, bool any) {
    const int R = a.T * a.K;
    for (int64_t r = max(0, min(used, R)) + int64_t(blockIdx.x); r < R; r += gridDim.x) {
        if (any) copy_row<true>(nullptr, a.rows + r * a.bytes, a.bytes);
        else copy_row<false>(nullptr, a.rows + r * a.bytes, a.bytes);
        if (a.scale)
            for (int c = threadIdx.x; c < a.n_scale; c += blockDim.x) a.srows[r * a.n_scale + c] = 0u;
    }
}

// Rows of whole 16-byte pieces: a thread reads one piece of a token and stores it K times.  Pieces are numbered
// through all tokens, so that narrow rows fill a CTA; every CTA also clears its share of the rows behind the
// last expert's.  Bound by HBM's writes: 2048 tokens of 7168 bf16 to 8 rows each 43 us (6.1 TB/s).
__global__ void __launch_bounds__(256) sort_pieces_kernel(CopyArgs a, int pieces) {
    chain_wait();
    chain_release();
    const int R = a.T * a.K;
    const int64_t all = int64_t(a.T) * pieces, step = int64_t(gridDim.x) * blockDim.x;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += step) {
        const int t = int(i / pieces);
        const int64_t at = (i - int64_t(t) * pieces) * 16;
        const uint4 u = *reinterpret_cast<const uint4*>(a.x + t * a.ld_x + at);
        const int32_t* row = a.row_of + int64_t(t) * a.K;
#pragma unroll 8
        for (int k = 0; k < a.K; ++k) {
            const int r = __ldg(row + k);
            if (unsigned(r) < unsigned(R)) *reinterpret_cast<uint4*>(a.rows + r * a.bytes + at) = u;
        }
    }
    if (a.scale) {
        const int64_t words = int64_t(a.T) * a.n_scale;
        for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < words; i += step) {
            const int t = int(i / a.n_scale), c = int(i - int64_t(t) * a.n_scale);
            const uint32_t v = a.scale[t * a.ld_scale + c];
            for (int k = 0; k < a.K; ++k) {
                const int r = __ldg(a.row_of + int64_t(t) * a.K + k);
                if (unsigned(r) < unsigned(R)) a.srows[int64_t(r) * a.n_scale + c] = v;
            }
        }
    }
    clear_tail(a, *a.rows_used, false);
}

// Rows of any length and place: one CTA a token.  2048 tokens of 5001 bf16 to 8 rows each 60 us (3.1 TB/s), bound by
// the shifting.
__global__ void __launch_bounds__(256) sort_rows_kernel(CopyArgs a) {
    chain_wait();
    chain_release();
    const int R = a.T * a.K;
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        const int32_t* row = a.row_of + int64_t(t) * a.K;
        for (int k = 0; k < a.K; ++k) {
            const int r = __ldg(row + k);
            if (unsigned(r) >= unsigned(R)) continue;
            copy_row<true>(a.x + t * a.ld_x, a.rows + r * a.bytes, a.bytes);
            if (a.scale)
                for (int c = threadIdx.x; c < a.n_scale; c += blockDim.x)
                    a.srows[int64_t(r) * a.n_scale + c] = a.scale[t * a.ld_scale + c];
        }
    }
    clear_tail(a, *a.rows_used, true);
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

// A thread takes 8 columns of a token and loads them of up to 8 of its rows before it adds any, so a sum costs
// one wait for memory.  DT: the rows' type where it is 16 bits, 0 otherwise.  Vectors are numbered through
// all tokens, so that narrow rows fill a CTA.  Bound by HBM: 4096 tokens of 8 rows of 7168 bf16 111 us (5.3 TB/s),
// 64 tokens 3.2 us.  ANY is bound by the shifting of what lies across 16 bytes: 2048 tokens of 5001 columns 69 us
// (3.0 TB/s; 91 us when pieces on a boundary were shifted too).  With all 8 rows loaded ahead it needed 111 registers
// and was slower.
template <int DT, bool ANY>
__global__ void __launch_bounds__(256) unsort_kernel(UnsortArgs a, int vectors) {
    constexpr int kAhead = 8;
    chain_wait();
    chain_release();
    const int R = a.T * a.K;
    const int64_t all = int64_t(a.T) * vectors;
    for (int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += int64_t(gridDim.x) * blockDim.x) {
        const int t = int(i / vectors), at = int(i - int64_t(t) * vectors) * 8;
        const int64_t out_row = int64_t(t) * a.H;
        const int c = ANY ? at - lead_in(a.out, a.out_dtype, out_row) : at;
        if (ANY && c >= a.H) continue;
        const int32_t* row = a.row_of + int64_t(t) * a.K;
        const float* weight = a.weight ? a.weight + int64_t(t) * a.K : nullptr;
        float acc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = 0.0f;
        for (int k0 = 0; k0 < a.K; k0 += kAhead) {
            if constexpr (DT != 0 && !ANY) {
                uint4 u[kAhead];
                float w[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    const int r = k0 + k < a.K ? __ldg(row + k0 + k) : -1;
                    const bool here = unsigned(r) < unsigned(R);
                    u[k] = here ? *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.rows) + r * a.ld + c)
                                : make_uint4(0, 0, 0, 0);
                    w[k] = !here ? 0.0f : weight ? __ldg(weight + k0 + k) : 1.0f;  // an absent route's weight is not used
                }
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    float v[8];
                    unpack8(u[k], DT, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w[k], v[j], acc[j]);
                }
            } else {
#pragma unroll 4
                for (int k = k0; k < min(k0 + kAhead, a.K); ++k) {
                    const int r = __ldg(row + k);
                    if (unsigned(r) >= unsigned(R)) continue;
                    const float w = weight ? __ldg(weight + k) : 1.0f;
                    float v[8];
                    if constexpr (ANY) load8_any(a.rows, a.dtype, r * a.ld, c, a.H, v);
                    else load8(a.rows, a.dtype, r * a.ld + c, v);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, v[j], acc[j]);
                }
            }
        }
        if (a.res) {
            float v[8];
            if constexpr (ANY) load8_any(a.res, a.res_dtype, t * a.ld_res, c, a.H, v);
            else load8(a.res, a.res_dtype, t * a.ld_res + c, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += v[j];
        }
        if constexpr (ANY) store8_any(a.out, a.out_dtype, out_row, c, a.H, acc);
        else store8(a.out, a.out_dtype, out_row + c, acc);
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

// One CTA a token, kAhead of its routes at a time: a thread loads 8 columns of the gradient and of these routes'
// rows together, stores the rows' gradients and keeps a partial dot product for each.  DT: the type of g, rows and
// d_rows where all have it, 0 otherwise.  Bound by HBM: 4096 tokens of 8 rows of 7168 bf16 184 us (5.4 TB/s).  ANY:
// 2048 tokens of 5001 columns 146 us (2.4 TB/s; 184 us with one route after the other).
template <int DT, bool ANY>
__global__ void __launch_bounds__(256) unsort_grad_kernel(UnsortGradArgs a) {
    constexpr int kAhead = 8;
    __shared__ float s_part[8][kAhead];
    chain_wait();
    chain_release();
    const int R = a.T * a.K, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int gt = DT ? DT : a.g_dtype, dt = DT ? DT : a.dtype;
    for (int t = blockIdx.x; t < a.T; t += gridDim.x) {
        for (int k0 = 0; k0 < a.K; k0 += kAhead) {
            int r[kAhead];
            float w[kAhead], dot[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int at = k0 + k < a.K ? __ldg(a.row_of + int64_t(t) * a.K + k0 + k) : -1;
                r[k] = unsigned(at) < unsigned(R) ? at : -1;
                w[k] = r[k] >= 0 && a.weight ? __ldg(a.weight + int64_t(t) * a.K + k0 + k) : 1.0f;
                dot[k] = 0.0f;
            }
            if constexpr (!ANY) {
                for (int c = threadIdx.x * 8; c < a.H; c += blockDim.x * 8) {
                    float g[8];
                    load8(a.g, gt, t * a.ld_g + c, g);
                    if constexpr (DT == 1 || DT == 2) {
                        uint4 u[kAhead];
                        if (a.d_weight) {
#pragma unroll
                            for (int k = 0; k < kAhead; ++k)
                                if (r[k] >= 0)
                                    u[k] = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.rows) + r[k] * a.ld + c);
                        }
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) {
                            if (r[k] < 0) continue;
                            float v[8];
                            if (a.d_weight) {
                                unpack8(u[k], DT, v);
#pragma unroll
                                for (int j = 0; j < 8; ++j) dot[k] = fmaf(g[j], v[j], dot[k]);
                            }
                            if (a.d_rows) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] = w[k] * g[j];
                                store8(a.d_rows, DT, int64_t(r[k]) * a.H + c, v);
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < kAhead; ++k) {
                            if (r[k] < 0) continue;
                            float v[8];
                            if (a.d_weight) {
                                load8(a.rows, dt, r[k] * a.ld + c, v);
#pragma unroll
                                for (int j = 0; j < 8; ++j) dot[k] = fmaf(g[j], v[j], dot[k]);
                            }
                            if (a.d_rows) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] = w[k] * g[j];
                                store8(a.d_rows, dt, int64_t(r[k]) * a.H + c, v);
                            }
                        }
                    }
                }
            } else {
                // each route's vectors lie on the 16-byte boundaries of the row that is written; kTake of them are
                // loaded together
                constexpr int kTake = 4;
#pragma unroll
                for (int h = 0; h < kAhead; h += kTake) {
                    if (k0 + h >= a.K) break;
                    int lead[kTake];
#pragma unroll
                    for (int k = 0; k < kTake; ++k)
                        lead[k] = a.d_rows && r[h + k] >= 0 ? lead_in(a.d_rows, dt, int64_t(r[h + k]) * a.H) : 0;
                    for (int i = threadIdx.x * 8; i < a.H + 7; i += blockDim.x * 8) {
                        Around ug[kTake], uv[kTake];
                        if constexpr (DT != 0) {
#pragma unroll
                            for (int k = 0; k < kTake; ++k) {
                                const int c = i - lead[k];
                                if (r[h + k] < 0 || !inner8(c, a.H)) continue;
                                ug[k] = load_around(static_cast<const uint16_t*>(a.g) + t * a.ld_g + c);
                                if (a.d_weight)
                                    uv[k] = load_around(static_cast<const uint16_t*>(a.rows) + r[h + k] * a.ld + c);
                            }
                        }
#pragma unroll
                        for (int k = 0; k < kTake; ++k) {
                            const int c = i - lead[k];
                            if (r[h + k] < 0 || c >= a.H) continue;
                            const bool whole = DT != 0 && inner8(c, a.H);
                            float g[8], v[8];
                            if (whole) unpack8(ug[k].piece(), DT, g);
                            else load8_any(a.g, gt, t * a.ld_g, c, a.H, g);
                            if (a.d_weight) {
                                if (whole) unpack8(uv[k].piece(), DT, v);
                                else load8_any(a.rows, dt, r[h + k] * a.ld, c, a.H, v);
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (unsigned(c + j) < unsigned(a.H)) dot[h + k] = fmaf(g[j], v[j], dot[h + k]);
                            }
                            if (a.d_rows) {
#pragma unroll
                                for (int j = 0; j < 8; ++j) v[j] = w[h + k] * g[j];
                                store8_any(a.d_rows, dt, int64_t(r[h + k]) * a.H, c, a.H, v);
                            }
                        }
                    }
                }
            }
            if (!a.d_weight) continue;
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
                if (lane == 0) s_part[warp][k] = dot[k];
            }
            __syncthreads();
            if (threadIdx.x < kAhead && k0 + int(threadIdx.x) < a.K) {
                float sum = 0.0f;
                for (int i = 0; i < int(blockDim.x >> 5); ++i) sum += s_part[i][threadIdx.x];  // fixed order
                a.d_weight[int64_t(t) * a.K + k0 + threadIdx.x] = sum;  // 0 for an absent route
            }
            __syncthreads();
        }
    }
    if (!a.d_rows) return;
    const int used = max(0, min(*a.rows_used, R));
    const int64_t bytes = int64_t(a.H) * (dt == 3 ? 4 : 2);
    for (int64_t r = used + int64_t(blockIdx.x); r < R; r += gridDim.x)
        copy_row<ANY>(nullptr, static_cast<uint8_t*>(a.d_rows) + r * bytes, bytes);
}

cudaError_t launch_order(const OrderArgs& a, cudaStream_t stream) {
    // A cluster counts 2048 routes a turn and costs about 1 us more than one CTA: 4096 routes 9.5 -> 6.6 us.
    const int ranks = a.n > 1024 ? kSortMaxCluster : 1;
    int warps = kSortMaxWarps;
    while (warps > kSortMinWarps && int64_t(warps / 2) * ranks * 32 * 2 >= a.n) warps /= 2;  // two routes a lane or fewer
    const size_t smem = size_t(warps + 2) * (a.E + 1) * 4;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(order_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ranks);
    cfg.blockDim = dim3(warps * 32);
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
    int bits = 1;
    while ((n_experts >> (bits - 1)) != 0) ++bits;
    const OrderArgs a{topk_idx, idx_bytes == 8, T * K, n_experts, first_expert, bits, row_of, route_of, offsets};
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
    const CopyArgs a{static_cast<const uint8_t*>(x), row_bytes, ld_bytes, reinterpret_cast<const uint32_t*>(scale),
                     n_scale, ld_scale, T, K, row_of, rows_used, static_cast<uint8_t*>(rows),
                     reinterpret_cast<uint32_t*>(rows_scale)};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool aligned = row_bytes % 16 == 0 && rows_aligned16(x, ld_bytes, 1) && rows_aligned16(rows, row_bytes, 1);
    const int64_t pieces = (row_bytes + 15) / 16;
    if (pieces > INT32_MAX) return set_last_error(CST_ERR_INVALID_ARG, "row_bytes=%lld is too long", (long long)row_bytes);
    cudaError_t e;
    if (aligned) {
        const int64_t ctas = (T * pieces + 255) / 256;
        e = launch_chained(sort_pieces_kernel, dim3(unsigned(ctas < INT32_MAX ? ctas : INT32_MAX)), dim3(256), 0, s, a,
                           int(pieces));
    } else {
        // as many threads as a row has pieces, up to 256
        const int threads = pieces >= 256 ? 256 : int((pieces + 31) / 32 * 32);
        e = launch_chained(sort_rows_kernel, dim3(T), dim3(threads), 0, s, a);
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
    if (H < 1 || H > (1 << 30) || ld_rows < H || (residual && ld_residual < H))
        return set_last_error(CST_ERR_INVALID_ARG, "H=%d must be in [1, 2^30] and no row stride below it", H);
    if (T == 0) return CST_OK;
    if (!rows || !row_of || !out) return set_last_error(CST_ERR_INVALID_ARG, "null rows, order or out");
    const UnsortArgs a{rows, rows_dtype, ld_rows, row_of, weight, T, K, H, residual, residual_dtype, ld_residual, out,
                       out_dtype};
    const bool vec = H % 8 == 0 && rows_aligned16(rows, ld_rows, act_size(rows_dtype)) &&
                     rows_aligned16(out, H, act_size(out_dtype)) &&
                     (!residual || rows_aligned16(residual, ld_residual, act_size(residual_dtype)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int vectors = (H + 7) / 8 + (vec ? 0 : 1);  // anywhere: up to 7 columns before the row
    const int64_t ctas = (int64_t(T) * vectors + 255) / 256;
    auto kernel = !vec ? unsort_kernel<0, true>
                  : rows_dtype == CST_DTYPE_BF16 ? unsort_kernel<2, false>
                  : rows_dtype == CST_DTYPE_FP16 ? unsort_kernel<1, false>
                                                 : unsort_kernel<0, false>;
    return launched("unsort_rows", launch_chained(kernel, dim3(unsigned(ctas < INT32_MAX ? ctas : INT32_MAX)), dim3(256), 0,
                                                  s, a, vectors));
}

extern "C" int cst_unsort_rows_grad(const void* grad, int32_t grad_dtype, int64_t ld_grad, const void* rows,
                                    int32_t rows_dtype, int64_t ld_rows, const int32_t* row_of, const float* weight,
                                    const int32_t* rows_used, int32_t T, int32_t K, int32_t H, void* d_rows,
                                    float* d_weight, void* stream) {
    clear_last_error();
    if (const int rc = check_routes("unsort_rows_grad", T, K)) return rc;
    if (!act_dtype(grad_dtype) || !act_dtype(rows_dtype))
        return set_last_error(CST_ERR_INVALID_ARG, "invalid dtype (grad %d, rows %d)", grad_dtype, rows_dtype);
    if (H < 1 || H > (1 << 30) || ld_grad < H || (d_weight && ld_rows < H))
        return set_last_error(CST_ERR_INVALID_ARG, "H=%d must be in [1, 2^30] and no row stride below it", H);
    if (T == 0 || (!d_rows && !d_weight)) return CST_OK;
    if (!grad || !row_of || !rows_used || (d_weight && !rows))
        return set_last_error(CST_ERR_INVALID_ARG, "null grad, rows or order");
    const UnsortGradArgs a{grad, grad_dtype, ld_grad, rows, rows_dtype, ld_rows, row_of, weight, rows_used, T, K, H,
                           d_rows, d_weight};
    const bool vec = H % 8 == 0 && rows_aligned16(grad, ld_grad, act_size(grad_dtype)) &&
                     (!d_weight || rows_aligned16(rows, ld_rows, act_size(rows_dtype))) &&
                     (!d_rows || rows_aligned16(d_rows, H, act_size(rows_dtype)));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool same = grad_dtype == rows_dtype;
    auto kernel = !vec && same && rows_dtype == CST_DTYPE_BF16 ? unsort_grad_kernel<2, true>
                  : !vec && same && rows_dtype == CST_DTYPE_FP16 ? unsort_grad_kernel<1, true>
                  : !vec ? unsort_grad_kernel<0, true>
                  : !same ? unsort_grad_kernel<0, false>
                  : rows_dtype == CST_DTYPE_BF16 ? unsort_grad_kernel<2, false>
                  : rows_dtype == CST_DTYPE_FP16 ? unsort_grad_kernel<1, false>
                                                 : unsort_grad_kernel<3, false>;
    // as many threads as a row has vectors, up to 256
    const int threads = H >= 2048 ? 256 : (H + 7) / 8 < 32 ? 32 : ((H + 7) / 8 + 31) / 32 * 32;
    return launched("unsort_rows_grad", launch_chained(kernel, dim3(T), dim3(threads), 0, s, a));
}
