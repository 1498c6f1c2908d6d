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
// rows g and g + 8 and the 8 consecutive k from 8 c of both 32s of its half, a word 4 of them:
// bits 4 i + 16 e .. of a word hold row g + 8 (i & 1), k = 32 (j >> 1) + 8 c + 4 (j & 1) + 2 (i >> 1) + e,
// and the word is rotated left by 3, which puts them where dequantising wants them.
// With swiglu a block is 32 "up" rows and the 32 "gate" rows that go with them.
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "../../include/constellation_b200.h"
#include "act_vec.cuh"
#include "cst_common.cuh"
#include "kernels.h"

namespace cst {

namespace {

constexpr int kRows = 64;    // weight rows of a block
constexpr int kChunk = 128;  // k of a chunk
constexpr int kQBytes = kRows * kChunk / 2;
constexpr int kErrBytes = 256;  // behind the experts: the device error word of the products' bounded waits

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
    const int chunk = blockIdx.x, b = blockIdx.y, e = blockIdx.z;  // e counts from the first expert of the call
    uint8_t* dst = out + e * g.expert_bytes() + (int64_t(b) * g.chunks + chunk) * g.chunk_bytes;
    for (int w = threadIdx.x; w < kQBytes / 4; w += blockDim.x) {
        const int j = w & 3, lane = (w >> 2) & 31, half = (w >> 7) & 1, tile = w >> 8;
        uint32_t word = 0;
        for (int i = 0; i < 4; ++i) {
            const int n = source_row(g, b, tile * 16 + (lane >> 2) + 8 * (i & 1));
            for (int el = 0; el < 2; ++el) {
                const int k = chunk * kChunk + half * 64 + 32 * (j >> 1) + (lane & 3) * 8 + 4 * (j & 1) + 2 * (i >> 1) + el;
                uint32_t v = 8;
                if (n >= 0 && k < g.K) {
                    const uint8_t two = q[((int64_t(e) * g.N + n) * g.K + k) >> 1];
                    v = (k & 1) ? two >> 4 : two & 15;
                }
                word |= v << (4 * i + 16 * el);
            }
        }
        reinterpret_cast<uint32_t*>(dst)[w] = (word << 3) | (word >> 29);
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
    const uint8_t* x;
    int64_t ld_x;  // bytes
    const float* x_scale;
    int64_t ld_xs;
    const int32_t* offsets;  // null: every row belongs to expert 0
    int R;
    void* out;
    int out_dtype;
    int64_t ld_out;
    int* err;
    int tile;         // rows of x of an item: 8, 16 or 32
    int ranks;        // CTAs of a cluster, which split k
    int stages;       // ring depth
    int stage_bytes;  // weights, then x, then x scales
    int x_at, xs_at;  // offsets in a stage
};

constexpr int kSlices = 4;                       // chunks of a stage = k slices of the consumer warps
constexpr int kRowTiles = 2;                     // tiles of 16 weight rows of a warp
constexpr int kConsumers = kSlices * 4 / kRowTiles;
constexpr int kThreads = (kConsumers + 1) * 32;  // and the producer warp
constexpr int kMaxStages = 12;

enum class XType { bf16, f16, e4m3 };

// Bytes of one row of x in a stage.  8 lanes of a 16-byte (16-bit x) or 16 of an 8-byte (e4m3)
// shared-memory read take 64 (32) bytes of a row each: rows 64 (32) bytes apart mod 128 keep
// them on different banks.
template <XType X>
__host__ __device__ constexpr int x_pitch() {
    return X == XType::e4m3 ? kSlices * kChunk + 32 : kSlices * kChunk * 2 + 64;
}

__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
    return d;
}

template <XType X>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (X == XType::bf16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Eight k of x for two matrix instructions: words 0, 1 go with the first, 2, 3 with the second.
template <XType X>
__device__ __forceinline__ void load_x(const uint8_t* p, uint32_t (&v)[4]) {
    if constexpr (X == XType::e4m3) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        const uint32_t w[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w[i]), __NV_E4M3);
            v[i] = uint32_t(h.x) | (uint32_t(h.y) << 16);
        }
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    }
}

__device__ __forceinline__ float scale_at(const uint8_t* scales, int dtype, int s) {
    if (dtype == 3) return reinterpret_cast<const float*>(scales)[s];
    if (dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(scales)[s]);
    return __half2float(reinterpret_cast<const __half*>(scales)[s]);
}

// The 8 weights of a word as 16 + q in the product's type, exactly: q goes to the top four bits of
// the mantissa of 2^4, bits 3..6 for bf16 and 6..9 for fp16.
template <XType X>
__device__ __forceinline__ void widen(uint32_t w, uint32_t (&a)[4]) {
    if constexpr (X == XType::bf16) {
        a[0] = lop_and_or(w, 0x00780078u, 0x41804180u);
        a[1] = lop_and_or(w >> 4, 0x00780078u, 0x41804180u);
        a[2] = lop_and_or(w >> 8, 0x00780078u, 0x41804180u);
        a[3] = lop_and_or(__funnelshift_r(w, w, 12), 0x00780078u, 0x41804180u);
    } else {
        a[0] = lop_and_or(w << 3, 0x03c003c0u, 0x4c004c00u);
        a[1] = lop_and_or(w >> 1, 0x03c003c0u, 0x4c004c00u);
        a[2] = lop_and_or(w >> 5, 0x03c003c0u, 0x4c004c00u);
        a[3] = lop_and_or(__funnelshift_r(w, w, 9), 0x03c003c0u, 0x4c004c00u);
    }
}

// One warp: kRowTiles tiles of 16 weight rows times one chunk of k for NT tiles of 8 rows of x.
// GROUPS: scales of a weight row in the chunk.  sum (q - z) x = sum (16 + q) x - (16 + z) sum x: the
// second sum comes from a matrix instruction with ones, one for all row tiles, so a weight costs
// one shift and one logic operation a pair and no subtraction.
template <XType X, int GROUPS, int NT>
__device__ __forceinline__ void chunk_product(const Geom& g, const uint8_t* chunk, const uint8_t* x, const float* xs,
                                              int row_tile, int lane, float (&acc)[kRowTiles][NT][4]) {
    const int gid = lane >> 2, c = lane & 3, n = row_tile * 16 + gid;
    constexpr int kX = X == XType::e4m3 ? 1 : 2;
    constexpr uint32_t kOne = X == XType::bf16 ? 0x3f803f80u : 0x3c003c00u;
    const uint32_t ones[4] = {kOne, kOne, kOne, kOne};
    float part[kRowTiles][NT][4], sum[NT][4];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        uint4 q4[kRowTiles];
#pragma unroll
        for (int r = 0; r < kRowTiles; ++r)
            q4[r] = *reinterpret_cast<const uint4*>(chunk + (((row_tile + r) * 2 + half) * 32 + lane) * 16);
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {  // 32 k
            const int piece = half * 2 + jj;
            if (piece % (4 / GROUPS) == 0) {
#pragma unroll
                for (int t = 0; t < NT; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        sum[t][i] = 0.0f;
#pragma unroll
                        for (int r = 0; r < kRowTiles; ++r) part[r][t][i] = 0.0f;
                    }
                }
            }
            uint32_t b[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                load_x<X>(x + (t * 8 + gid) * x_pitch<X>() + (piece * 32 + c * 8) * kX, b[t]);
                mma<X>(sum[t], ones, b[t][0], b[t][1]);
                mma<X>(sum[t], ones, b[t][2], b[t][3]);
            }
#pragma unroll
            for (int r = 0; r < kRowTiles; ++r) {
                uint32_t a[4];
                widen<X>(jj ? q4[r].z : q4[r].x, a);
#pragma unroll
                for (int t = 0; t < NT; ++t) mma<X>(part[r][t], a, b[t][0], b[t][1]);
                widen<X>(jj ? q4[r].w : q4[r].y, a);
#pragma unroll
                for (int t = 0; t < NT; ++t) mma<X>(part[r][t], a, b[t][2], b[t][3]);
            }
            if (piece % (4 / GROUPS) == 4 / GROUPS - 1) {
                float s0[NT], s1[NT];
                if constexpr (X == XType::e4m3) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        s0[t] = xs[(t * 8 + c * 2) * kSlices];
                        s1[t] = xs[(t * 8 + c * 2 + 1) * kSlices];
                    }
                }
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
                    const int s = piece / (4 / GROUPS) * kRows + n + r * 16;
                    const float lo = scale_at(chunk + kQBytes, g.scale_dtype, s);
                    const float hi = scale_at(chunk + kQBytes, g.scale_dtype, s + 8);
                    float zlo = -24.0f, zhi = -24.0f;
                    if (g.has_zero) {
                        zlo = -16.0f - float(chunk[g.zero_at + s]);
                        zhi = -16.0f - float(chunk[g.zero_at + s + 8]);
                    }
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float p[4] = {fmaf(zlo, sum[t][0], part[r][t][0]), fmaf(zlo, sum[t][1], part[r][t][1]),
                                      fmaf(zhi, sum[t][2], part[r][t][2]), fmaf(zhi, sum[t][3], part[r][t][3])};
                        if constexpr (X == XType::e4m3) {
                            p[0] *= s0[t];
                            p[1] *= s1[t];
                            p[2] *= s0[t];
                            p[3] *= s1[t];
                        }
                        acc[r][t][0] = fmaf(p[0], lo, acc[r][t][0]);
                        acc[r][t][1] = fmaf(p[1], lo, acc[r][t][1]);
                        acc[r][t][2] = fmaf(p[2], hi, acc[r][t][2]);
                        acc[r][t][3] = fmaf(p[3], hi, acc[r][t][3]);
                    }
                }
            }
        }
    }
}

// Arrives on the barrier at the same place of CTA `rank` of the cluster; releases this CTA's
// shared-memory writes to it.
__device__ __forceinline__ void arrive_remote(uint64_t* bar, int rank) {
    asm volatile(
        "{\n"
        ".reg .b32 r;\n"
        "mapa.shared::cluster.u32 r, %0, %1;\n"
        "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [r];\n"
        "}\n" ::"r"(smem_u32(bar)), "r"(rank)
        : "memory");
}

__device__ __forceinline__ float load_remote(const float* p, int rank) {
    float v;
    asm volatile(
        "{\n"
        ".reg .b32 r;\n"
        "mapa.shared::cluster.u32 r, %1, %2;\n"
        "ld.shared::cluster.f32 %0, [r];\n"
        "}\n"
        : "=f"(v)
        : "r"(smem_u32(p)), "r"(rank)
        : "memory");
    return v;
}

__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, int* err) {
    const uint64_t t0 = global_ns();
    for (uint32_t i = 1; i < kSpinLimit; ++i) {
        uint32_t ok;
        asm volatile(
            "{\n"
            ".reg .pred p;\n"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
            "selp.u32 %0, 1, 0, p;\n"
            "}\n"
            : "=r"(ok)
            : "r"(smem_u32(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((i & 255u) == 0u && global_ns() - t0 > kWaitLimitNs) break;
    }
    atomicMax(err, CST_DEV_ERR_TIMEOUT);
    return false;
}

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumers * 32) : "memory"); }

struct Item {
    int expert, row, rows, block;
};

// Item i: the row tile i / blocks and the block of weight rows i % blocks; s_tile[e] = first tile
// of expert e, s_row[e] = its first row.
__device__ __forceinline__ Item find_item(const Int4Args& a, const int* s_tile, const int* s_row, int64_t i) {
    const int tile = int(i / a.g.blocks);
    int lo = 0, hi = a.g.E - 1;  // the last expert whose first tile is <= tile
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_tile[mid] <= tile) lo = mid;
        else hi = mid - 1;
    }
    Item it;
    it.expert = lo;
    it.row = s_row[lo] + (tile - s_tile[lo]) * a.tile;
    it.rows = min(a.tile, s_row[lo + 1] - it.row);
    it.block = int(i - int64_t(tile) * a.g.blocks);
    return it;
}

template <XType X, int GROUPS, bool WIDE>
__global__ void __launch_bounds__(kThreads, WIDE ? 1 : 2) int4_kernel(Int4Args a) {
    extern __shared__ __align__(128) uint8_t s_ring[];
    __shared__ int s_tile[CST_INT4_MAX_EXPERTS + 1], s_row[CST_INT4_MAX_EXPERTS + 1];
    __shared__ int s_scan[kThreads / 32][2];
    __shared__ uint64_t s_full[kMaxStages], s_empty[kMaxStages], s_join[2];
    // behind the ring: the k slices' sums of an item, [slice][row of x][weight row], and for a cluster
    // this CTA's sums of the item and of the one before
    const int values_cap = a.tile * kRows;
    float* s_slice = reinterpret_cast<float*>(s_ring + a.stages * a.stage_bytes);
    float* s_part = s_slice + kSlices * values_cap;
    const Geom& g = a.g;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = a.ranks > 1 ? int(blockIdx.x) % a.ranks : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            // the producer's arrival with the bytes to come; e4m3: its lanes' copies of row scales too
            mbar_init(&s_full[s], X == XType::e4m3 ? 33 : 1);
            mbar_init(&s_empty[s], kConsumers);
        }
        mbar_init(&s_join[0], a.ranks);
        mbar_init(&s_join[1], a.ranks);
        fence_barrier_init();
    }
    if (a.ranks > 1) {  // every CTA's barriers exist before any CTA arrives on them
        asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
    } else {
        __syncthreads();
    }
    chain_wait();
    chain_release();

    // first rows (clamped, made ascending) and first tiles of the experts
    {
        constexpr int kPer = (CST_INT4_MAX_EXPERTS + kThreads) / kThreads;  // experts + 1 over the threads
        int row[kPer], carry = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = int(threadIdx.x) * kPer + i;
            int r = 0;
            if (e <= g.E) r = a.offsets ? max(0, min(a.offsets[e], a.R)) : (e == 0 ? 0 : a.R);
            carry = max(carry, r);
            row[i] = carry;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, carry, o);
            if (lane >= o) carry = max(carry, v);
        }
        if (lane == 31) s_scan[warp][0] = carry;
        int before = __shfl_up_sync(0xffffffffu, carry, 1);
        if (lane == 0) before = 0;
        __syncthreads();
        for (int w = 0; w < warp; ++w) before = max(before, s_scan[w][0]);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = int(threadIdx.x) * kPer + i;
            if (e <= g.E) s_row[e] = max(row[i], before);
        }
        __syncthreads();
        int tiles[kPer], sum = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = int(threadIdx.x) * kPer + i;
            tiles[i] = sum;
            if (e < g.E) sum += (s_row[e + 1] - s_row[e] + a.tile - 1) / a.tile;
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) s_scan[warp][1] = inc;
        __syncthreads();
        int base = inc - sum;
        for (int w = 0; w < warp; ++w) base += s_scan[w][1];
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = int(threadIdx.x) * kPer + i;
            if (e <= g.E) s_tile[e] = base + tiles[i];
        }
        __syncthreads();
    }
    const int64_t items = int64_t(s_tile[g.E]) * g.blocks;
    const int64_t first = blockIdx.x / a.ranks, step = gridDim.x / a.ranks;
    // this CTA's chunks of k, whole stages
    const int all_stages = (g.chunks + kSlices - 1) / kSlices;
    const int per = (all_stages + a.ranks - 1) / a.ranks;
    const int chunk0 = min(rank * per * kSlices, g.chunks), chunk1 = min(chunk0 + per * kSlices, g.chunks);
    constexpr int kX = X == XType::e4m3 ? 1 : 2;

    if (warp == kConsumers) {
        int s = 0, issued = 0;
        uint32_t phase = 0;
        bool alive = true;
        for (int64_t i = first; alive && i < items; i += step) {
            const Item it = find_item(a, s_tile, s_row, i);
            const uint8_t* w = a.data + it.expert * g.expert_bytes() + int64_t(it.block) * g.chunks * g.chunk_bytes;
            const uint8_t* x = a.x + int64_t(it.row + min(lane, it.rows - 1)) * a.ld_x;
            for (int c = chunk0; c < chunk1; c += kSlices) {
                alive = mbar_wait(&s_empty[s], phase ^ 1, a.err);
                if (!alive) break;
                uint8_t* stage = s_ring + s * a.stage_bytes;
                const int n = min(kSlices, chunk1 - c);
                const int want = n * kChunk, have = min(want, g.K - c * kChunk);  // columns of x
                uint8_t* xs = stage + a.x_at + lane * x_pitch<X>();
                if (have < want && lane < it.rows) {
                    // past k x belongs to someone else: zeros, ordered before this and later bulk copies
                    for (int b = have * kX; b < want * kX; b += 16)
                        *reinterpret_cast<uint4*>(xs + b) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive_expect_tx(&s_full[s], n * g.chunk_bytes + it.rows * have * kX);
                    tma_bulk_g2s(stage, w + int64_t(c) * g.chunk_bytes, n * g.chunk_bytes, &s_full[s]);
                }
                __syncwarp();
                if (lane < it.rows) tma_bulk_g2s(xs, x + int64_t(c) * kChunk * kX, have * kX, &s_full[s]);
                if constexpr (X == XType::e4m3) {
                    if (lane < it.rows) {
                        for (int k = 0; k < n; ++k)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(
                                             smem_u32(stage + a.xs_at + (lane * kSlices + k) * 4)),
                                         "l"(a.x_scale + int64_t(it.row + lane) * a.ld_xs + c + k)
                                         : "memory");
                    }
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(smem_u32(&s_full[s]))
                                 : "memory");
                }
                issued = max(issued, s + 1);
                if (++s == a.stages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // no copy is left in flight when the CTA ends, whatever became of the consumers
        for (int j = 0; j < a.stages; ++j)
            if (j < issued) mbar_wait(&s_full[j], j < s ? phase : phase ^ 1, a.err);
    } else {
        const int slice = warp / (4 / kRowTiles), row_tile = warp % (4 / kRowTiles) * kRowTiles;
        int s = 0, turn = 0;
        uint32_t phase = 0;
        bool alive = true;
        // rows of no expert
        {
            const int used = s_row[g.E], lead = s_row[0];
            const int64_t outside = int64_t(lead) + (a.R - used);
            for (int64_t r = blockIdx.x; r < outside; r += gridDim.x) {
                const int64_t row = r < lead ? r : r - lead + used;
                const float zero[1] = {0.0f};
                for (int n = threadIdx.x; n < g.out_n; n += kConsumers * 32)
                    store_act<1>(a.out, a.out_dtype, row * a.ld_out + n, zero);
            }
        }
        for (int64_t i = first; i < items; i += step, ++turn) {
            const Item it = find_item(a, s_tile, s_row, i);
            auto product = [&](auto tiles) {
                constexpr int NT = decltype(tiles)::value;
                float acc[kRowTiles][NT][4];
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        acc[r][t][0] = acc[r][t][1] = acc[r][t][2] = acc[r][t][3] = 0.0f;
                for (int c = chunk0; alive && c < chunk1; c += kSlices) {
                    alive = mbar_wait(&s_full[s], phase, a.err);
                    const uint8_t* stage = s_ring + s * a.stage_bytes;
                    if (alive && c + slice < chunk1)
                        chunk_product<X, GROUPS, NT>(g, stage + slice * g.chunk_bytes,
                                                     stage + a.x_at + slice * kChunk * kX,
                                                     reinterpret_cast<const float*>(stage + a.xs_at) + slice, row_tile,
                                                     lane, acc);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&s_empty[s]);
                    if (++s == a.stages) {
                        s = 0;
                        phase ^= 1;
                    }
                }
                const int n = row_tile * 16 + (lane >> 2), m = (lane & 3) * 2;
#pragma unroll
                for (int r = 0; r < kRowTiles; ++r) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        float* p = s_slice + slice * values_cap + (t * 8 + m) * kRows + n + r * 16;
                        p[0] = acc[r][t][0];
                        p[kRows] = acc[r][t][1];
                        p[8] = acc[r][t][2];
                        p[kRows + 8] = acc[r][t][3];
                    }
                }
            };
            if (it.rows <= 8) product(std::integral_constant<int, 1>{});
            else if (!WIDE || it.rows <= 16) product(std::integral_constant<int, 2>{});
            else if constexpr (WIDE) product(std::integral_constant<int, 4>{});
            consumer_sync();
            // the slices' sums, and over a cluster the CTAs', in fixed order
            const int values = it.rows * kRows;
            auto slices = [&](int v) {
                float y = s_slice[v];
#pragma unroll
                for (int k = 1; k < kSlices; ++k) y += s_slice[k * values_cap + v];
                return y;
            };
            float* part = s_part + (turn & 1) * values_cap;
            int v0 = 0, v1 = values;
            if (a.ranks > 1) {
                for (int v = threadIdx.x; v < values; v += kConsumers * 32) part[v] = slices(v);
                consumer_sync();
                // two barriers in turn: a fast CTA's arrival for the next item cannot count for this one
                if (threadIdx.x < a.ranks) arrive_remote(&s_join[turn & 1], threadIdx.x);
                if (alive) alive = wait_cluster(&s_join[turn & 1], (turn >> 1) & 1, a.err);
                const int share = (it.rows + a.ranks - 1) / a.ranks;  // rows of x that this CTA writes
                v0 = min(rank * share, it.rows) * kRows;
                v1 = min(v0 + share * kRows, values);
            }
            const int per_block = g.swiglu ? kRows / 2 : kRows;
            for (int v = v0 + int(threadIdx.x); v < v1; v += kConsumers * 32) {
                const int n = v % kRows, col = it.block * per_block + n;
                if (n >= per_block || col >= g.out_n) continue;
                float y[1], gate = 0.0f;
                if (a.ranks == 1) {
                    y[0] = slices(v);
                    if (g.swiglu) gate = slices(v + 32);
                } else {
                    y[0] = 0.0f;
                    for (int r = 0; r < a.ranks; ++r) {
                        y[0] += load_remote(part + v, r);
                        if (g.swiglu) gate += load_remote(part + v + 32, r);
                    }
                }
                if (g.swiglu) y[0] *= gate / (1.0f + expf(-gate));
                store_act<1>(a.out, a.out_dtype, int64_t(it.row + v / kRows) * a.ld_out + col, y);
            }
            if (a.ranks == 1) consumer_sync();  // the slices are read before the next item's are written
        }
    }
    // no CTA of a cluster leaves while another may still read its sums or arrive on its barrier
    if (a.ranks > 1) {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
    }
}

// Rows of x of an item.  Taking more rows than an expert has costs shared memory (ring depth); taking
// fewer runs its weights twice, the second time from L2.
int choose_tile(int R, int E) {
    const int mean = (R + E - 1) / E;
    return R <= 8 || mean <= 4 ? 8 : R <= 16 || mean <= 8 ? 16 : 32;
}

// CTAs that share an item's k.  A wave of clusters takes (stages / ranks + a fixed cost) for each of its
// rounds; few items leave SMs idle unless k is split.
int choose_ranks(int64_t items, int all_stages, int sms) {
    int best = 1;
    double least = 0;
    for (int ranks = 1; ranks <= 8; ranks *= 2) {
        const int64_t slots = sms / ranks, rounds = (items + slots - 1) / slots;
        const double cost = double(rounds) * ((all_stages + ranks - 1) / ranks + (ranks == 1 ? 2 : 4));
        if (ranks == 1 || cost < least) {
            least = cost;
            best = ranks;
        }
    }
    return best;
}

template <XType X, int GROUPS, bool WIDE>
cudaError_t launch_int4(Int4Args a, int sms, cudaStream_t stream) {
    constexpr int kShared = WIDE ? 216 * 1024 : 103 * 1024;
    sms *= WIDE ? 1 : 2;
    a.x_at = kSlices * a.g.chunk_bytes;
    a.xs_at = a.x_at + a.tile * x_pitch<X>();
    a.stage_bytes = (a.xs_at + (X == XType::e4m3 ? a.tile * kSlices * 4 : 0) + 127) / 128 * 128;
    const int all_stages = (a.g.chunks + kSlices - 1) / kSlices;
    // experts with rows: at most every expert and every row; tiles of rows beyond one an expert
    const int64_t touched = a.R < a.g.E ? a.R : a.g.E;
    const int64_t most = (touched + a.R / a.tile) * a.g.blocks;
    a.ranks = choose_ranks(a.R <= a.tile ? int64_t(a.g.blocks) * touched : most, all_stages, sms);
    const int sums = (kSlices + (a.ranks > 1 ? 2 : 0)) * a.tile * kRows * 4;
    a.stages = (kShared - sums) / a.stage_bytes;
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    const int64_t clusters = most < sms / a.ranks ? most : sms / a.ranks;
    auto kernel = int4_kernel<X, GROUPS, WIDE>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(clusters * a.ranks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = size_t(a.stages) * a.stage_bytes + sums;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.ranks;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.ranks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <XType X, int GROUPS>
cudaError_t launch_tile(Int4Args a, int sms, cudaStream_t s) {
    a.tile = choose_tile(a.R, a.g.E);
    return a.tile > 16 ? launch_int4<X, GROUPS, true>(a, sms, s) : launch_int4<X, GROUPS, false>(a, sms, s);
}

template <XType X>
cudaError_t launch_groups(const Int4Args& a, int sms, cudaStream_t s) {
    return a.g.group == 128 ? launch_tile<X, 1>(a, sms, s)
           : a.g.group == 64 ? launch_tile<X, 2>(a, sms, s)
                             : launch_tile<X, 4>(a, sms, s);
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
    *bytes = make_geom(*w).expert_bytes() * w->n_experts + kErrBytes;
    return CST_OK;
}

extern "C" int cst_int4_pack(const cst_int4_weight* w, int32_t first, int32_t count, const uint8_t* q,
                             const void* scale, const uint8_t* zero, void* data, void* stream) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (first < 0 || count < 0 || count > w->n_experts - first)
        return set_last_error(CST_ERR_INVALID_ARG, "experts [%d, %d + %d) outside [0, %d)", first, first, count,
                              w->n_experts);
    if (count == 0) return CST_OK;
    if (!q || !scale || !data || (w->has_zero && !zero))
        return set_last_error(CST_ERR_INVALID_ARG, "null q, scale, zero or data");
    if (reinterpret_cast<uintptr_t>(data) & 15u)
        return set_last_error(CST_ERR_INVALID_ARG, "data must be 16-byte aligned");
    const Geom g = make_geom(*w);
    pack_kernel<<<dim3(g.chunks, g.blocks, count), 256, 0, static_cast<cudaStream_t>(stream)>>>(
        g, q, scale, zero, static_cast<uint8_t*>(data) + first * g.expert_bytes());
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "int4_pack launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}

extern "C" int cst_int4_device_error(const cst_int4_weight* w, void* data, void* stream) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (!data) return set_last_error(CST_ERR_INVALID_ARG, "null data");
    const Geom g = make_geom(*w);
    void* word = static_cast<uint8_t*>(data) + g.expert_bytes() * g.E;
    int32_t v = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaMemcpyAsync(&v, word, 4, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, 4, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "int4_device_error failed: %s", cudaGetErrorString(e));
    if (v != CST_DEV_OK)
        return set_last_error(CST_ERR_DEVICE_TIMEOUT, "a bounded wait in a 4-bit product gave up (code %d)", v);
    return CST_OK;
}

extern "C" int cst_grouped_int4(const cst_int4_weight* w, void* data, const void* x, int32_t x_dtype, int64_t ld_x,
                                const float* x_scale, int64_t ld_x_scale, const int32_t* offsets, int32_t R,
                                void* out, int32_t out_dtype, int64_t ld_out, void* stream) {
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
    if (!rows_aligned16(x, ld_x, act_size(x_dtype)) || (reinterpret_cast<uintptr_t>(data) & 15u))
        return set_last_error(CST_ERR_INVALID_ARG, "data and every row of x must be 16-byte aligned");
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "cannot query the SM count: %s", cudaGetErrorString(e));
    Int4Args a{};
    a.g = g;
    a.data = static_cast<const uint8_t*>(data);
    a.x = static_cast<const uint8_t*>(x);
    a.ld_x = ld_x * act_size(x_dtype);
    a.x_scale = x_scale;
    a.ld_xs = ld_x_scale;
    a.offsets = offsets;
    a.R = R;
    a.out = out;
    a.out_dtype = out_dtype;
    a.ld_out = ld_out;
    a.err = reinterpret_cast<int*>(static_cast<uint8_t*>(data) + g.expert_bytes() * g.E);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = x_dtype == CST_DTYPE_BF16   ? launch_groups<XType::bf16>(a, sms, s)
        : x_dtype == CST_DTYPE_FP16 ? launch_groups<XType::f16>(a, sms, s)
                                    : launch_groups<XType::e4m3>(a, sms, s);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "grouped_int4 launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}
