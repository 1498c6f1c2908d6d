// Products with 4-bit weights, grouped by expert.  With q[e, n, k] in 0..15 and one scale (and
// one zero point, 8 if there is none) for `group` consecutive k,
//     y[r, n] = sum_G scale[e, n, G] * sum_{k in G} (q[e, n, k] - zero[e, n, G]) * x[r, k]
// for the rows r in [offsets[e], offsets[e + 1]) of expert e; rows behind offsets[E] are zero.
// x in e4m3 carries one fp32 scale for 128 columns of a row.  With `swiglu` the first half of
// the N weight rows is "up", the second "gate", and y = silu(gate) * up, [R, N / 2].
//
// A byte q of 0..15 is the e4m3 number q * 2^-9: 0..7 are its subnormals and 8..15 its first normals, in
// even steps.  So a pair of logic operations turns 8 packed weights into 8 operands of the 8-bit
// matrix product, and the zero point is one more product of the same x with a constant operand,
//     2^-9 sum (q - z) x = sum (q 2^-9) x + sum (-z 2^-9) x,
// into the same accumulator.  x enters as e4m3 terms with a power of two s that fits the largest |x| of the
// row to 448: two terms for bf16 (8 bits = 4 + 4), x = s (t1 + t2 / 16), three for fp16 (11 bits),
// x = s (t1 + t2 + t3 / 512).  They are x exactly where |x| is above 2^-13 (bf16) or 2^-11 (fp16) of that
// largest; below, what they drop is less than 2^-21 (2^-22) of the largest.  A chunk of 128 columns whose own
// largest lies 5 or more binades below the row's, as they do around an outlier, takes an s of its own, so what
// it drops is at any rate less than 2^-17 (2^-18) of the chunk's largest.  e4m3 rows enter as they are,
// with their scales.  The products are exact and the sums fp32, with one rounding at the end.
//
// Layout of one weight (written once by pack_kernel): blocks of 128 weight rows, each a run of
// chunks of 128 k; a chunk is 8192 bytes of q, then the 128 rows' scales [128 / group][128], then
// their zero points [128 / group][128].  q: [32 k][row][word of 8 k]; byte j of a word holds k = j in its
// lower and k = 4 + j in its upper half.
// With swiglu the rows of a block are 64 "up" rows, each followed by the "gate" row that goes with it.
#include <cfloat>
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

#include "../../include/constellation_b200.h"
#include "act_vec.cuh"
#include "cst_common.cuh"
#include "kernels.h"

namespace cst {

namespace {

constexpr int kRows = 128;   // weight rows of a block
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
    const int n = b * (kRows / 2) + (r >> 1);
    return n < g.out_n ? n + (r & 1 ? g.out_n : 0) : -1;
}

// One CTA per (chunk, block, expert).  Padding (rows past N, k past K) gets q = 8 and scale 0,
// zero point 8, so it adds exactly nothing.
__global__ void __launch_bounds__(256) pack_kernel(Geom g, const uint8_t* q, const void* scale, const uint8_t* zero,
                                                   uint8_t* out) {
    const int chunk = blockIdx.x, b = blockIdx.y, e = blockIdx.z;  // e counts from the first expert of the call
    uint8_t* dst = out + e * g.expert_bytes() + (int64_t(b) * g.chunks + chunk) * g.chunk_bytes;
    for (int w = threadIdx.x; w < kQBytes / 4; w += blockDim.x) {
        // source order: the 16 words of a row one after the other
        const int n = source_row(g, b, w >> 4), k = chunk * kChunk + (w & 15) * 8;
        uint32_t word = 0x88888888u;
        if (n >= 0 && k < g.K) {  // k ends on a multiple of 32
            const uint8_t* src = q + ((int64_t(e) * g.N + n) * g.K + k) / 2;
            word = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t v = i & 1 ? src[i >> 1] >> 4 : src[i >> 1] & 15;
                word |= v << (8 * (i & 3) + 4 * (i >> 2));
            }
        }
        reinterpret_cast<uint32_t*>(dst)[(((w & 15) >> 2) * kRows + (w >> 4)) * 4 + (w & 3)] = word;
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

// ---- the rows of x as e4m3 terms -----------------------------------------------------------

constexpr int kFactBytes = 16;  // of an e4m3 row and chunk: its scale, padded to what a bulk copy takes

// A chunk whose largest lies within these binades of its row's takes the row's power of two.  Rows without outliers then
// have one, which is multiplied once a result; powers of two of chunks are a load and a product for each accumulator.  A
// launch with such rows took 16.5 us instead of 15.8 (8 rows of up and gate [4096, 7168]), 220 instead of 187 (64 experts of
// 8 rows), 115 instead of 99 (254 fp16 rows of down [7168, 2048]) and 335 instead of 256 (groups of 32).
constexpr int kNear = 4;

// The exponent of a power of two for the terms of numbers up to `most`.
__device__ __forceinline__ int terms_exp(float most) { return int(__float_as_uint(pow2_scale_for(most)) >> 23); }

// One CTA a row.  terms: [rows * TERMS][chunks * 128] (of three terms [t1, t3, t2][rows][chunks * 128], so that one
// product takes t1 and t3), columns past k zero.  facts: [chunks][rows] of the power of two of a row's terms in a
// chunk, negative in all of a row that has a chunk with one of its own; for e4m3 (TERMS 1) of x_scale, 16 bytes each.
// A chunk is 8 columns of 16 threads, who find its largest by shuffles.  A row's first 8192 columns (256 threads) stay in
// registers between its maximum and its terms; more are read twice.
template <int TERMS>
__global__ void __launch_bounds__(256) split_x_kernel(const void* x, int x_dtype, int64_t ld, const float* x_scale,
                                                      int64_t ld_xs, int rows, int k, uint8_t* terms, float* facts) {
    __shared__ float s_most[8], s_least[8];
    chain_wait();
    chain_release();
    const int chunks = (k + kChunk - 1) / kChunk, width = chunks * kChunk;
    const int64_t r = blockIdx.x, at = r * ld;
    if constexpr (TERMS == 1) {
        const uint8_t* src = static_cast<const uint8_t*>(x) + at;
        const bool vec = reinterpret_cast<uintptr_t>(src) % 16 == 0;
        for (int c = threadIdx.x * 16; c < width; c += blockDim.x * 16) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c < k) {  // k is a multiple of 32
                if (vec) {
                    v = *reinterpret_cast<const uint4*>(src + c);
                } else {
                    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 16; ++j) w[j >> 2] |= uint32_t(src[c + j]) << (8 * (j & 3));
                    v = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
            *reinterpret_cast<uint4*>(terms + r * width + c) = v;
        }
        for (int c = threadIdx.x; c < chunks; c += blockDim.x)
            facts[(int64_t(c) * rows + r) * (kFactBytes / 4)] = x_scale[r * ld_xs + c];
        return;
    }
    constexpr int kHeld = 4;  // vectors of 8 columns a thread holds
    const bool vec = (reinterpret_cast<uintptr_t>(x) + at * 2) % 16 == 0;
    auto load = [&](int c, float (&v)[8]) {
        if (vec) {
            load8(x, x_dtype, at + c, v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = load1(x, x_dtype, at + c + j);
        }
        // e4m3 has no infinities: one makes its row's results NaN, as a NaN does
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (isinf(v[j])) v[j] = __int_as_float(0x7fffffff);
    };
    const int step = blockDim.x * 8, lane = threadIdx.x & 31, lead = lane * 8, first = threadIdx.x * 8 - lead;
    // the largest of each of the two chunks that a warp has; a NaN is none
    auto largest = [&](const float (&v)[8]) {
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[j]));
        const uint32_t bits = __float_as_uint(m);  // in the order of the numbers, which are not negative
        return make_float2(__uint_as_float(__reduce_max_sync(0xffffffffu, lane < 16 ? bits : 0u)),
                           __uint_as_float(__reduce_max_sync(0xffffffffu, lane < 16 ? 0u : bits)));
    };
    float held[kHeld][8], most = 0.0f, least = FLT_MAX;  // the largest of the row, and the smallest chunk's that is not 0
    auto add = [&](float2 m) {
        most = fmaxf(most, fmaxf(m.x, m.y));
        least = fminf(least, fminf(m.x > 0.0f ? m.x : FLT_MAX, m.y > 0.0f ? m.y : FLT_MAX));
    };
    // loops run over the vectors of whole warps, whose lanes stay together
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) held[i][j] = 0.0f;
        if (first + lead + i * step < k) load(first + lead + i * step, held[i]);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (first + i * step < k) add(largest(held[i]));
    for (int c0 = first + kHeld * step; c0 < k; c0 += step) {
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (c0 + lead < k) load(c0 + lead, v);
        add(largest(v));
    }
    if (lane == 0) {
        s_most[threadIdx.x >> 5] = most;
        s_least[threadIdx.x >> 5] = least;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        if (w >= int(blockDim.x >> 5)) break;
        most = fmaxf(most, s_most[w]);
        least = fminf(least, s_least[w]);
    }
    const int row_exp = terms_exp(most);
    const bool own = most > 0.0f && row_exp - terms_exp(least) > kNear;
    auto store = [&](int c, const float (&x8)[8], float2 both) {
        const float m = lane < 16 ? both.x : both.y;
        int e = row_exp;
        if (own && m > 0.0f) {
            const int near = terms_exp(m);
            if (row_exp - near > kNear) e = near;
        }
        const float scale = __uint_as_float(uint32_t(e) << 23), inv = pow2_recip(scale);
        if (c % kChunk == 0) facts[int64_t(c / kChunk) * rows + r] = own ? -scale : scale;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x8[j] * inv;
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
            // exact: the rest has fewer bits than v; its largest is 16 after the first term, which 16-fold stays
            // below 448, and 1/2 after the second of three, which does so 512-fold
            const float up = TERMS == 2 ? 16.0f : t == 0 ? 1.0f : 512.0f;
            uint32_t q[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                q[j] = e4m3x2_rn(v[2 * j], v[2 * j + 1]);
                const float2 f = e4m3x2_to_f32x2(q[j]);
                v[2 * j] = (v[2 * j] - f.x) * up;
                v[2 * j + 1] = (v[2 * j + 1] - f.y) * up;
            }
            const int64_t at_row = TERMS == 2 ? r * 2 + t : (t == 0 ? 0 : 3 - t) * int64_t(rows) + r;
            *reinterpret_cast<uint2*>(terms + at_row * width + c) = make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16));
        }
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int c = first + lead + i * step;
        if (c - lead >= width) continue;
        const float2 m = own ? largest(held[i]) : make_float2(0.0f, 0.0f);
        if (c < width) store(c, held[i], m);
    }
    for (int c0 = first + kHeld * step; c0 < width; c0 += step) {
        float v[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (c0 + lead < k) load(c0 + lead, v);
        const float2 m = own ? largest(v) : make_float2(0.0f, 0.0f);
        if (c0 + lead < width) store(c0 + lead, v, m);
    }
}

// ---- the product ---------------------------------------------------------------------------
// One persistent CTA per SM walks items (row tile of an expert, block of 128 weight rows); the
// CTAs of a cluster split an item's k.  Per step of up to four chunks of 128 k:
//   warp 0     one lane is the producer: one bulk copy of the packed weights with their scales (8.4 KB a
//              chunk) and one TMA box of x's terms [step][tile * TERMS][128 k], swizzled as the matrix unit
//              reads them (and for e4m3 the rows' scales), into a ring;
//   warps 2..  wideners, two sets of four: each thread owns a weight row, turns its 64 packed bytes into 128 e4m3
//              numbers with 48 logic operations and stores them to tensor memory, where they are the matrix
//              product's A operand (and the row's zero points, if there are any);
//   warp 1     one lane issues the tcgen05 products, a fresh fp32 accumulator for each group;
//   the last   output warps, as many sets: each thread owns a weight row of the accumulators:
//              acc[t] += 2^9 scale * (D1[t] + D2[t] / 16), and at the end of an item the results.
// So each weight byte is read once from HBM and once from shared memory, and never goes back there.
//
// Bound: HBM up to about 8 rows an expert; above, the handing of steps from role to role (a step is 600 to 1500
// cycles, in which no role is busy throughout), which is why a step holds as many chunks as tensor memory has
// room for twice, and the widening (a third of the issue slots).  Up and gate [4096, 7168], groups of 128, bf16
// rows: 32 experts of 1 row 91 us (5.3 TB/s of weights and rows), 64 experts of 8 rows 189 us (5.2 TB/s),
// 32 experts of 32 rows 162 us (371 TFLOP/s).  Down [7168, 2048], groups of 64 with zero points, 254 fp16 rows over
// 32 experts: 96 us (2.7 TB/s).  200 e4m3 rows over 8 experts of [4096, 7168]: 64 us, two and a third rounds
// of items over the SMs taking three.
// Operands of x's own 16-bit type instead of e4m3 terms would need no terms, but 9 to 11 operations for 8
// weights instead of 3: the 32 experts of 1 row took 134 us, of 32 rows 180 us.

constexpr int kMaxStages = 12;
constexpr int kMaxStep = 4;                     // chunks of a step, which the roles hand on at a time
constexpr int kSets = 2;                        // sets of 4 wideners and of 4 output warps, which take the steps in turn
constexpr int kWarpMma = 1, kWarpWiden = 2, kWarpOut = kWarpWiden + 4 * kSets;
constexpr int kThreads = (kWarpOut + 4 * kSets) * 32;
constexpr int kMaxBufs = 4;                     // steps in tensor memory
constexpr int kACols = kChunk / 4;              // columns of A: [128 rows][128 k] of 8 bits
constexpr int kMostColumns = 512 / 2 - kACols - 32;  // accumulator columns of a chunk with which two steps fit

// Columns of tensor memory of an accumulator: [rows][terms], for three terms [2][rows], of which the first
// takes two.  A product is a multiple of 16 wide.
__host__ __device__ constexpr int acc_columns(int terms, int tile) {
    return terms == 3 ? 2 * (tile < 16 ? 16 : tile) : (tile * terms + 15) / 16 * 16;
}

struct Int4Args {
    Geom g;
    const uint8_t* data;
    const float* facts;      // of split_x_kernel
    const int32_t* offsets;  // null: every row belongs to expert 0
    int R;
    void* out;
    int out_dtype;
    int64_t ld_out;
    int* err;
    int tile;         // rows of x of an item: 8, 16 or 32
    int ranks;        // CTAs of a cluster
    int stages;       // ring depth
    int stage_bytes;  // x [step][tile * TERMS][128], then the chunks, then for e4m3 the facts [step][tile]
    int q_at, f_at;   // offsets in a stage
    int step;         // chunks of a step
    int bufs;         // steps in tensor memory: A, behind all of them the zero points, then the accumulators
    int z_at, d_at;   // first columns of the zero points (8 for each group of a step, or 8 in all) and accumulators
    int d_cols;       // acc_columns
};

__device__ __forceinline__ float scale_at(const uint8_t* scales, int dtype, int s) {
    if (dtype == 3) return reinterpret_cast<const float*>(scales)[s];
    if (dtype == 2) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(scales)[s]);
    return __half2float(reinterpret_cast<const __half*>(scales)[s]);
}

// x's terms of rows from y and chunks from z, all 128 columns of them.
__device__ __forceinline__ void tma_box_g2s(void* dst, const CUtensorMap* map, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(0), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// The same of three planes of rows.
__device__ __forceinline__ void tma_planes_g2s(void* dst, const CUtensorMap* map, int y, int z, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %2, %4}], [%5];\n" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(0), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// 32 consecutive 32-bit columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_fill8(uint32_t taddr, uint32_t v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%1,%1,%1,%1,%1,%1,%1};\n" ::"r"(taddr), "r"(v) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

// D[tmem] (+)= A[tmem] x B[smem desc], e4m3 x e4m3 -> fp32, K = 32.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t bdesc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n"
        "}\n" ::"r"(d),
        "r"(a), "l"(bdesc), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}

// True in one lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "elect.sync _|p, 0xffffffff;\n"
        "selp.u32 %0, 1, 0, p;\n"
        "}\n"
        : "=r"(p));
    return p != 0;
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

// A copy of 4 bytes to shared memory, and the wait for all of this thread's.
__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}

// The clock that bounds a wait costs some hundred cycles to read, so it is left to waits that take long.
__device__ __forceinline__ bool lane_wait(uint64_t* bar, uint32_t parity, int* err) {
    for (int i = 0; i < 256; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    return mbar_wait(bar, parity, err);
}

// A wait of a whole warp, with one outcome for all its lanes.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err) {
    return __all_sync(0xffffffffu, lane_wait(bar, parity, err));
}

// A place in a ring of `n` buffers and the parity of its current pass.
struct Ring {
    int i = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int n) {
        if (++i == n) {
            i = 0;
            phase ^= 1;
        }
    }
};

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

// First rows (clamped to [0, R], made ascending) and first tiles of the experts, by all threads.
__device__ __forceinline__ void scan_offsets(const Int4Args& a, int* s_tile, int* s_row, int (*s_scan)[2]) {
    constexpr int kPer = (CST_INT4_MAX_EXPERTS + kThreads) / kThreads;  // experts + 1 over the threads
    static_assert(kPer * kThreads >= CST_INT4_MAX_EXPERTS + 1, "every expert needs a thread");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = a.g.E;
    int row[kPer], most = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = int(threadIdx.x) * kPer + i;
        int r = 0;
        if (e <= E) r = a.offsets ? max(0, min(a.offsets[e], a.R)) : (e == 0 ? 0 : a.R);
        most = max(most, r);
        row[i] = most;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, most, o);
        if (lane >= o) most = max(most, v);
    }
    if (lane == 31) s_scan[warp][0] = most;
    int before = __shfl_up_sync(0xffffffffu, most, 1);
    if (lane == 0) before = 0;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before = max(before, s_scan[w][0]);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = int(threadIdx.x) * kPer + i;
        if (e <= E) s_row[e] = max(row[i], before);
    }
    __syncthreads();
    int tiles[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = int(threadIdx.x) * kPer + i;
        tiles[i] = sum;
        if (e < E) sum += (s_row[e + 1] - s_row[e] + a.tile - 1) / a.tile;
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
        if (e <= E) s_tile[e] = base + tiles[i];
    }
    __syncthreads();
}

// The ring of stages; declared here so that the roles address it as shared memory.
extern __shared__ __align__(1024) uint8_t s_ring[];

struct Shared {
    int tile[CST_INT4_MAX_EXPERTS + 1], row[CST_INT4_MAX_EXPERTS + 1];
    int scan[kThreads / 32][2];
    uint64_t full[kMaxStages], empty[kMaxStages];
    // of a buffer in tensor memory: A written and the last accumulators taken; the products done
    uint64_t ready[kMaxBufs], done[kMaxBufs];
    uint64_t join[2];
    uint32_t tmem;
    bool own[kSets * 4];
};

// The work of one CTA: its items, and its steps of k in each.
struct Span {
    int64_t items, first, step;
    int step0, step1;
};

// One elected lane.  A step is one bulk copy of its chunks and one TMA box of x's terms for all of them.
template <int TERMS>
__device__ __forceinline__ void producer_role(const Int4Args& a, Shared& sh, const CUtensorMap& xmap, const Span& sp) {
    Ring s;
    int issued = 0;
    bool waiting = true;
    const uint32_t x_bytes = uint32_t(a.step * a.tile * TERMS * kChunk);
    for (int64_t i = sp.first; i < sp.items; i += sp.step) {
        const Item it = find_item(a, sh.tile, sh.row, i);
        const uint8_t* w = a.data + it.expert * a.g.expert_bytes() +
                           (int64_t(it.block) * a.g.chunks + int64_t(sp.step0) * a.step) * a.g.chunk_bytes;
        const int x_row = TERMS == 2 ? it.row * 2 : it.row;
        for (int c = sp.step0; c < sp.step1; ++c) {
            if (!lane_wait(&sh.empty[s.i], s.phase ^ 1, a.err)) goto out;
            uint8_t* stage = s_ring + s.i * a.stage_bytes;
            const int n = min(a.step, a.g.chunks - c * a.step);
            const uint32_t w_bytes = uint32_t(n * a.g.chunk_bytes);
            // a TMA box always counts whole: what lies past the rows and chunks arrives as zeros
            mbar_arrive_expect_tx(&sh.full[s.i], w_bytes + x_bytes + (TERMS == 1 ? n * it.rows * kFactBytes : 0));
            tma_bulk_g2s(stage + a.q_at, w, w_bytes, &sh.full[s.i]);
            w += w_bytes;
            if (waiting) {
                chain_wait();
                waiting = false;
            }
            if constexpr (TERMS == 3) tma_planes_g2s(stage, &xmap, x_row, c * a.step, &sh.full[s.i]);
            else tma_box_g2s(stage, &xmap, x_row, c * a.step, &sh.full[s.i]);
            if constexpr (TERMS == 1)
                for (int h = 0; h < n; ++h)
                    tma_bulk_g2s(stage + a.f_at + h * a.tile * kFactBytes,
                                 a.facts + (int64_t(c * a.step + h) * a.R + it.row) * (kFactBytes / 4),
                                 it.rows * kFactBytes, &sh.full[s.i]);
            issued = max(issued, s.i + 1);
            s.next(a.stages);
        }
    }
out:
    if (waiting) chain_wait();  // this grid must not be done before the one that it did not wait for
    // no copy is left in flight when the CTA ends, whatever became of the consumers
    for (int j = 0; j < issued; ++j) lane_wait(&sh.full[j], j < s.i ? s.phase : s.phase ^ 1, a.err);
}

template <int GROUPS>
__device__ __forceinline__ void widen_role(const Int4Args& a, Shared& sh, const Span& sp) {
    const int warp = (int(threadIdx.x) >> 5) - kWarpWiden, lane = threadIdx.x & 31, set = warp >> 2;
    const int quarter = (int(threadIdx.x) >> 5) & 3;  // the lanes of tensor memory this warp may touch
    const int row = quarter * 32 + lane;
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    if (!a.g.has_zero && set == 0) {  // -8 * 2^-9 for every product of this launch; the first arrival below orders it
        tmem_fill8(lanes + a.z_at, 0x88888888u);
        tmem_wait_st();  // here, for a CTA without items has no step that waits, and gives its columns back
    }
    Ring s, b;
    int turn = set;
    for (int64_t i = sp.first; i < sp.items; i += sp.step) {
        for (int c = sp.step0; c < sp.step1; ++c, s.next(a.stages), b.next(a.bufs)) {
            if (turn != 0) {
                --turn;
                continue;
            }
            turn = kSets - 1;
            if (!warp_wait(&sh.full[s.i], s.phase, a.err) || !warp_wait(&sh.done[b.i], b.phase ^ 1, a.err)) return;
            tc_fence_after();
            const uint8_t* chunk = s_ring + s.i * a.stage_bytes + a.q_at + row * 16;
            uint32_t dst = lanes + b.i * a.step * kACols;
            const int n = min(a.step, a.g.chunks - c * a.step);
#pragma unroll 1
            for (int h = 0; h < n; ++h, chunk += a.g.chunk_bytes, dst += kACols) {
                uint32_t v[32];
#pragma unroll
                for (int p = 0; p < 4; ++p) {  // 32 k
                    const uint4 q = *reinterpret_cast<const uint4*>(chunk + p * (kRows * 16));
                    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[p * 8 + j * 2] = w[j] & 0x0f0f0f0fu;
                        v[p * 8 + j * 2 + 1] = (w[j] >> 4) & 0x0f0f0f0fu;
                    }
                }
                tmem_st32(dst, v);
                if (a.g.has_zero) {
#pragma unroll
                    for (int g = 0; g < GROUPS; ++g) {
                        const uint32_t z = chunk[a.g.zero_at + g * kRows - row * 15];  // of this row
                        tmem_fill8(lanes + a.z_at + ((b.i * a.step + h) * GROUPS + g) * 8, (z | 0x80u) * 0x01010101u);
                    }
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.ready[b.i]);
                mbar_arrive(&sh.empty[s.i]);
            }
        }
    }
}

// One elected lane.  The operands of an instruction come from uniform registers: under an elected
// lane, with addresses that are sums of a base and constants, a 128 x 16 x 16 product takes 11 cycles to issue;
// through a lane that the compiler does not know to be alone it took 160.
template <int TERMS, int GROUPS, int TILE, bool ZERO>
__device__ __forceinline__ void mma_role(const Int4Args& a, Shared& sh, const Span& sp) {
    constexpr uint32_t kD = acc_columns(TERMS, TILE);       // columns of an accumulator
    constexpr uint32_t kPlane = TILE * kChunk / 16;         // bytes of a term of three, over 16
    constexpr uint32_t kX = TILE * TERMS * kChunk / 16;     // bytes of x of a chunk, over 16
    Ring s, b;
    int used = 0;
    const uint64_t x0 = umma_desc_sw128(smem_u32(s_ring));
    const uint32_t x_step = uint32_t(a.stage_bytes) >> 4;
    for (int64_t i = sp.first; i < sp.items; i += sp.step) {
        const Item it = find_item(a, sh.tile, sh.row, i);
        // three terms: the first and the third side by side, then the second onto the first
        const uint32_t idesc = umma_idesc_e4m3(128, TERMS == 3 ? kD / (TILE < 16 ? 2 : 1) : (it.rows * TERMS + 15) / 16 * 16);
        const uint32_t idesc2 = umma_idesc_e4m3(128, kD / 2);
        for (int c = sp.step0; c < sp.step1; ++c) {
            // A is written, and so the stage with its x is full; the accumulators are free
            if (!lane_wait(&sh.ready[b.i], b.phase, a.err)) goto out;
            tc_fence_after();
            const uint64_t x = x0 + uint64_t(uint32_t(s.i) * x_step);
            const uint32_t w = uint32_t(b.i * a.step) * kACols, d = uint32_t(a.d_at) + uint32_t(b.i * a.step * GROUPS) * kD;
            const uint32_t z = uint32_t(a.z_at) + (ZERO ? uint32_t(b.i * a.step * GROUPS) * 8 : 0);
            const int n = min(a.step, a.g.chunks - c * a.step);
#pragma unroll
            for (int h = 0; h < kMaxStep; ++h) {
                if (h >= n) break;
#pragma unroll
                for (int ks = 0; ks < 4; ++ks) {  // 32 k
                    const uint32_t g = h * GROUPS + ks / (4 / GROUPS);
                    const uint64_t xk = x + h * kX + ks * 2;
                    const uint32_t dg = d + g * kD, wk = w + h * kACols + ks * 8, zk = ZERO ? z + g * 8 : z;
                    tc_mma_ts(dg, wk, xk, idesc, ks % (4 / GROUPS) > 0);
                    tc_mma_ts(dg, zk, xk, idesc, true);
                    if constexpr (TERMS == 3) {
                        if constexpr (TILE < 16) {  // a product is 16 rows wide at least, so the third has its own
                            tc_mma_ts(dg + kD / 2, wk, xk + kPlane, idesc, ks % (4 / GROUPS) > 0);
                            tc_mma_ts(dg + kD / 2, zk, xk + kPlane, idesc, true);
                        }
                        tc_mma_ts(dg, wk, xk + 2 * kPlane, idesc2, true);
                        tc_mma_ts(dg, zk, xk + 2 * kPlane, idesc2, true);
                    }
                }
            }
            tc_commit(&sh.done[b.i]);
            used = max(used, b.i + 1);
            s.next(a.stages);
            b.next(a.bufs);
        }
    }
out:
    // tensor memory and the ring stay until the last products are done
    for (int j = 0; j < used; ++j) lane_wait(&sh.done[j], j < b.i ? b.phase : b.phase ^ 1, a.err);
}

// The columns of N rows (8 or 16) from `d` of this thread's lane of tensor memory; of three terms the second half
// lies `half` columns on.
template <int TERMS, int N>
__device__ __forceinline__ void load_piece(uint32_t d, int half, uint32_t* v) {
    if constexpr (TERMS * N == 8 || TERMS == 3) tmem_ld8(d, v);
    else tmem_ld16(d, v);
    if constexpr (TERMS == 3) tmem_ld8(d + half, v + 8);
    static_assert(TERMS == 1 ? N == 8 || N == 16 : N == 8, "a piece is 8 or 16 columns");
}

// One item: the sums of ROWS rows of x over the steps of this set of output warps, for this thread's weight
// row.  Without OWN a row's terms have one power of two, which its sums then lack; with it each chunk's is a factor.
// `mine`: 8 times 32 floats of this warp alone, kRows apart, for these of a step's chunks and of the next step's, whose
// copies are in flight meanwhile.
template <int TERMS, int GROUPS, int ROWS, bool OWN>
__device__ __forceinline__ bool accumulate(const Int4Args& a, Shared& sh, const Span& sp, const Item& it, int row,
                                           uint32_t lanes, float* mine, Ring& s, Ring& b, int& turn, float (&acc)[ROWS]) {
    // a row's columns; rows whose columns are in registers at a time
    constexpr int kAccs = TERMS == 1 ? 1 : 2, kCols = 16, kFit = kCols / kAccs;
    constexpr int kAt = ROWS < kFit ? ROWS : kFit, kGo = kAt == ROWS && kAt * kAccs < kCols ? kCols / (kAt * kAccs) : 1;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int t = 0; t < ROWS; ++t) acc[t] = 0.0f;
    int half = 0;  // of `mine`
    auto fetch = [&](int c) {  // lane t: of row t
        if (lane < it.rows && c < sp.step1) {
            const float* fact = a.facts + int64_t(c) * a.step * a.R + it.row + lane;
            const int n = min(a.step, a.g.chunks - c * a.step);
#pragma unroll
            for (int h = 0; h < kMaxStep; ++h)
                if (h < n) cp_async4(mine + (half + h) * kRows + lane, fact + int64_t(h) * a.R);
        }
    };
    if constexpr (OWN) fetch(sp.step0 + turn);
    for (int c = sp.step0; c < sp.step1; ++c, s.next(a.stages), b.next(a.bufs)) {
        if (turn != 0) {
            --turn;
            continue;
        }
        turn = kSets - 1;
        const float* facts = mine + half * kRows;
        if constexpr (OWN) {
            cp_async_wait();
            __syncwarp();
            half ^= kMaxStep;
            fetch(c + kSets);
        }
        if (!warp_wait(&sh.done[b.i], b.phase, a.err)) {
            if constexpr (OWN) cp_async_wait();
            return false;
        }
        tc_fence_after();
        const uint8_t* stage = s_ring + s.i * a.stage_bytes;
        const int n = min(a.step, a.g.chunks - c * a.step) * GROUPS;  // accumulators of the step
        uint32_t d = a.d_at + lanes + b.i * a.step * GROUPS * a.d_cols;
        // (chunk, group) pieces, kGo of them at a time while their columns fit in registers
#pragma unroll 1
        for (int p = 0; p < n; p += kGo, d += kGo * a.d_cols) {
            uint32_t v[kGo][kAt * kAccs];
            float scale[kGo];
#pragma unroll
            for (int k = 0; k < kGo; ++k)
                if (k == 0 || p + k < n) load_piece<TERMS, kAt>(d + k * a.d_cols, a.d_cols / 2, v[k]);
#pragma unroll
            for (int k = 0; k < kGo; ++k) {
                const int q = min(p + k, n - 1);
                scale[k] = scale_at(stage + a.q_at + q / GROUPS * a.g.chunk_bytes + kQBytes, a.g.scale_dtype,
                                    q % GROUPS * kRows + row) * 512.0f;
            }
#pragma unroll
            for (int t0 = 0; t0 < ROWS; t0 += kAt) {
                if (t0 > 0) load_piece<TERMS, kAt>(d + (TERMS == 2 ? 2 * t0 : t0), a.d_cols / 2, v[0]);  // then kGo is 1
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < kGo; ++k) tmem_reg_fence(v[k]);
#pragma unroll
                for (int k = 0; k < kGo; ++k) {
                    if (k > 0 && p + k >= n) break;
                    float4 f;
#pragma unroll
                    for (int t = 0; t < kAt; ++t) {
                        float y, w = scale[k];
                        if constexpr (OWN) {
                            if (t % 4 == 0) f = *reinterpret_cast<const float4*>(facts + (p + k) / GROUPS * kRows + t0 + t);
                            w *= t % 4 == 0 ? f.x : t % 4 == 1 ? f.y : t % 4 == 2 ? f.z : f.w;
                        }
                        if constexpr (TERMS == 1) y = __uint_as_float(v[k][t]);
                        if constexpr (TERMS == 2)
                            y = fmaf(__uint_as_float(v[k][2 * t + 1]), 0.0625f, __uint_as_float(v[k][2 * t]));
                        if constexpr (TERMS == 3)
                            y = fmaf(__uint_as_float(v[k][kAt + t]), 1.0f / 512, __uint_as_float(v[k][t]));
                        if constexpr (TERMS == 1)
                            y *= *reinterpret_cast<const float*>(stage + a.f_at + ((p + k) / GROUPS * a.tile + t0 + t) * kFactBytes);
                        acc[t0 + t] = fmaf(y, w, acc[t0 + t]);
                    }
                }
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
            mbar_arrive(&sh.ready[b.i]);
            mbar_arrive(&sh.empty[s.i]);
        }
    }
    return true;
}

// Result of weight row `row` of the block for row t of the tile: with swiglu even rows are "up" and
// their odd neighbours the "gate" that goes with them.
__device__ __forceinline__ void write_out(const Int4Args& a, const Item& it, int row, int t, float y) {
    int col = it.block * kRows + row;
    if (a.g.swiglu) {
        const float gate = __shfl_down_sync(0xffffffffu, y, 1);
        y *= gate / (1.0f + expf(-gate));
        col >>= 1;
    }
    if (col < a.g.out_n && !(a.g.swiglu && (row & 1)))
        store1(a.out, a.out_dtype, int64_t(it.row + t) * a.ld_out + col, y);
}

__device__ __forceinline__ void output_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(kSets * 128) : "memory"); }

// Whether a row has a chunk with a power of two of its own: the output warps' look at the rows while the first products are
// under way.  At all rows of experts, while that is one wait for memory; of more, each thread looks at an item's of this
// CTA's (131072 bf16 rows over 64 experts [256, 128]: 396 us, and 123 us more with a look at all rows).
__device__ __forceinline__ bool any_own(const Int4Args& a, Shared& sh, const Span& sp) {
    const int me = int(threadIdx.x) - kWarpOut * 32, warp = me >> 5, first = sh.row[0], last = sh.row[a.g.E];
    constexpr int kAtOnce = 8;
    bool own = false;
    if (last - first <= kAtOnce * kSets * 128) {
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
            const int r = first + me + i * kSets * 128;
            if (r < last) own |= __ldcg(a.facts + r) < 0.0f;
        }
    } else {
        for (int64_t i = sp.first + me * sp.step; i < sp.items; i += kSets * 128 * sp.step) {
            const Item it = find_item(a, sh.tile, sh.row, i);
#pragma unroll 8
            for (int t = 0; t < it.rows; ++t) own |= __ldcg(a.facts + it.row + t) < 0.0f;
        }
    }
    own = __any_sync(0xffffffffu, own);
    if ((threadIdx.x & 31) == 0) sh.own[warp] = own;
    output_sync();
    own = false;
#pragma unroll
    for (int w = 0; w < kSets * 4; ++w) own |= sh.own[w];
    return own;
}

template <int TERMS, int GROUPS, bool OWN>
__device__ __forceinline__ void out_role(const Int4Args& a, Shared& sh, float* s_part, const Span& sp, int rank) {
    const int lane = threadIdx.x & 31, quarter = (int(threadIdx.x) >> 5) & 3, row = quarter * 32 + lane;
    const int set = ((int(threadIdx.x) >> 5) - kWarpOut) >> 2, size = a.tile * kRows;
    int wait_turns = set;  // steps until this set's next
    const uint32_t lanes = uint32_t(quarter * 32) << 16;
    Ring s, b;
    bool alive = true;
    uint32_t turn = 0;
    for (int64_t i = sp.first; i < sp.items; i += sp.step, ++turn) {
        const Item it = find_item(a, sh.tile, sh.row, i);
        float* part = s_part + (a.ranks > 1 ? (turn & 1) * kSets * size : 0);  // [set][row of x][weight row]
        auto item = [&](auto rows) {
            constexpr int ROWS = decltype(rows)::value;
            float acc[ROWS];
            alive = alive && accumulate<TERMS, GROUPS, ROWS, OWN>(a, sh, sp, it, row, lanes, part + set * size + quarter * 32, s,
                                                                   b, wait_turns, acc);
#pragma unroll
            for (int t = 0; t < ROWS; ++t) part[set * size + t * kRows + row] = acc[t];
        };
        if (it.rows <= 8) item(std::integral_constant<int, 8>{});
        else if (it.rows <= 16) item(std::integral_constant<int, 16>{});
        else item(std::integral_constant<int, 32>{});
        // Lane t has what the sums of row t lack.
        float scale = TERMS > 1 && lane < it.rows ? __ldcg(a.facts + it.row + lane) : 1.0f;
        if constexpr (OWN) scale = scale < 0.0f ? -1.0f : 1.0f;
        int t0 = 0, t1 = it.rows;
        output_sync();
        if (a.ranks > 1) {
            // the CTAs' sums over the cluster, in order; two barriers in turn, so that a fast CTA's arrival
            // for the next item cannot count for this one
            const int me = int(threadIdx.x) - kWarpOut * 32;
            if (me < a.ranks) arrive_remote(&sh.join[turn & 1], me);
            alive = alive && __all_sync(0xffffffffu, wait_cluster(&sh.join[turn & 1], (turn >> 1) & 1, a.err));
            const int share = (it.rows + a.ranks - 1) / a.ranks;  // rows of x that this CTA writes
            t0 = rank * share;
            t1 = min(t0 + share, it.rows);
        }
#pragma unroll 4
        for (int t = t0 + set; t < t1; t += kSets) {
            float y = 0.0f;
            if (a.ranks == 1) {
#pragma unroll
                for (int h = 0; h < kSets; ++h) y += part[h * size + t * kRows + row];
            } else {
                for (int r = 0; r < a.ranks; ++r)
#pragma unroll
                    for (int h = 0; h < kSets; ++h) y += load_remote(part + h * size + t * kRows + row, r);
            }
            if constexpr (TERMS > 1) y *= __shfl_sync(0xffffffffu, scale, t);
            write_out(a, it, row, t, y);
        }
        // the sums are read before the next item's are written
        if (a.ranks == 1) output_sync();
    }
}

template <int TERMS, int GROUPS>
__global__ void __launch_bounds__(kThreads, 1) int4_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ Int4Args a) {
    __shared__ Shared sh;
    // behind the ring: the output sets' sums [row of x][weight row] of an item, for a cluster also of the one
    // before
    float* s_part = reinterpret_cast<float*>(s_ring + a.stages * a.stage_bytes);
    const Geom& g = a.g;
    const int warp = threadIdx.x >> 5;
    const int rank = a.ranks > 1 ? int(blockIdx.x) % a.ranks : 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&sh.full[s], 1);  // the producer's arrival with the bytes to come
            mbar_init(&sh.empty[s], 4 + 4);  // a set of wideners; a set of output warps, after the products
        }
        for (int b = 0; b < a.bufs; ++b) {
            mbar_init(&sh.ready[b], 4 + 4);
            mbar_init(&sh.done[b], 1);
        }
        mbar_init(&sh.join[0], a.ranks);
        mbar_init(&sh.join[1], a.ranks);
        fence_barrier_init();
    }
    if (warp == kWarpMma) {
        tmem_alloc(&sh.tmem, 512);  // all of it, so addresses start at column 0
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (a.ranks > 1) cluster_barrier();  // every CTA's barriers exist before any CTA arrives on them
    // The kernel before this one on the stream is split_x_kernel, which let this one start only after it had
    // waited for everything before it: offsets and weights are there, and `out` is free.  What it writes
    // itself, x's terms and facts, the producer and the output warps read, each after a wait of its own.
    chain_release();
    scan_offsets(a, sh.tile, sh.row, sh.scan);

    Span sp;
    sp.items = int64_t(sh.tile[g.E]) * g.blocks;
    sp.first = blockIdx.x / a.ranks;
    sp.step = gridDim.x / a.ranks;
    const int steps = (g.chunks + a.step - 1) / a.step, per = (steps + a.ranks - 1) / a.ranks;
    sp.step0 = min(rank * per, steps);
    sp.step1 = min(sp.step0 + per, steps);

    if (warp == 0) {
        if (elect_one()) producer_role<TERMS>(a, sh, xmap, sp);
    } else if (warp == kWarpMma) {
        if (elect_one()) {
            if (a.tile == 8) {
                if (g.has_zero) mma_role<TERMS, GROUPS, 8, true>(a, sh, sp);
                else mma_role<TERMS, GROUPS, 8, false>(a, sh, sp);
            } else if (a.tile == 16) {
                if (g.has_zero) mma_role<TERMS, GROUPS, 16, true>(a, sh, sp);
                else mma_role<TERMS, GROUPS, 16, false>(a, sh, sp);
            } else {
                if (g.has_zero) mma_role<TERMS, GROUPS, 32, true>(a, sh, sp);
                else mma_role<TERMS, GROUPS, 32, false>(a, sh, sp);
            }
        }
    } else if (warp < kWarpOut) {
        widen_role<GROUPS>(a, sh, sp);
    } else {
        if ((threadIdx.x & 31) == 0 && warp < kWarpOut + 4)  // no accumulators to take before the first products
            for (int j = 0; j < a.bufs; ++j) mbar_arrive(&sh.ready[j]);
        // rows of no expert
        const int used = sh.row[g.E], lead = sh.row[0];
        const int64_t outside = int64_t(lead) + (a.R - used);
        for (int64_t r = blockIdx.x; r < outside; r += gridDim.x) {
            for (int n = int(threadIdx.x) - kWarpOut * 32; n < g.out_n; n += kSets * 128)
                store1(a.out, a.out_dtype, (r < lead ? r : r - lead + used) * a.ld_out + n, 0.0f);
        }
        if constexpr (TERMS > 1) {
            chain_wait();  // the facts are split_x_kernel's
            if (any_own(a, sh, sp)) out_role<TERMS, GROUPS, true>(a, sh, s_part, sp, rank);
            else out_role<TERMS, GROUPS, false>(a, sh, s_part, sp, rank);
        } else {
            out_role<TERMS, GROUPS, false>(a, sh, s_part, sp, rank);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarpMma) tmem_dealloc(sh.tmem, 512);
    // no CTA of a cluster leaves while another may still read its sums or arrive on its barriers
    if (a.ranks > 1) {
        __syncwarp();
        cluster_barrier();
    }
}

// Rows of x of an item.  A pass over an expert's weights costs the same for 1 row as for a tile of 8, and rows
// that a tile has and the expert has not cost little: the tile holds about twice the mean, unless its
// accumulators would leave tensor memory no second step.
int choose_tile(int R, int E, int columns_a_row) {
    const int mean = (R + E - 1) / E;
    int tile = R <= 8 || mean <= 4 ? 8 : R <= 16 || mean <= 8 ? 16 : 32;
    while (tile > 8 && tile * columns_a_row > kMostColumns) tile /= 2;
    return tile;
}

// CTAs that share an item's k.  A wave of clusters takes (steps / ranks + a fixed cost) for each of its
// rounds; few items leave SMs idle unless k is split.
int choose_ranks(int64_t items, int steps, int sms) {
    int best = 1;
    double least = 0;
    for (int ranks = 1; ranks <= 8; ranks *= 2) {
        const int64_t slots = sms / ranks, rounds = (items + slots - 1) / slots;
        const double cost = double(rounds) * ((steps + ranks - 1) / ranks + (ranks == 1 ? 2 : 4));
        if (ranks == 1 || cost < least) {
            least = cost;
            best = ranks;
        }
    }
    return best;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

int64_t terms_bytes(const Geom& g, int terms, int64_t R) {
    return (R * terms * g.chunks * kChunk + 255) / 256 * 256;
}

template <int TERMS, int GROUPS>
int launch_int4(Int4Args a, void* workspace, int sms, cudaStream_t stream) {
    constexpr int kShared = 216 * 1024;
    a.tile = choose_tile(a.R, a.g.E, (TERMS == 1 ? 1 : 2) * GROUPS);
    a.d_cols = acc_columns(TERMS, a.tile);
    // tensor memory: of a chunk, and once for a constant zero point
    const int cols = kACols + (a.d_cols + (a.g.has_zero ? 8 : 0)) * GROUPS, once = a.g.has_zero ? 0 : 8;
    for (a.step = kMaxStep; a.step > 1 && (512 - once) / (a.step * cols) < 2;) --a.step;
    a.bufs = (512 - once) / (a.step * cols);
    if (a.bufs > kMaxBufs) a.bufs = kMaxBufs;
    a.z_at = a.bufs * a.step * kACols;
    a.d_at = a.z_at + (a.g.has_zero ? a.bufs * a.step * GROUPS * 8 : 8);
    a.q_at = a.step * a.tile * TERMS * kChunk;
    a.f_at = a.q_at + a.step * a.g.chunk_bytes;
    a.stage_bytes = (a.f_at + (TERMS == 1 ? a.step * a.tile * kFactBytes : 0) + 1023) / 1024 * 1024;
    // experts with rows: at most every expert and every row; tiles of rows beyond one an expert
    const int64_t touched = a.R < a.g.E ? a.R : a.g.E;
    const int64_t most = (touched + a.R / a.tile) * a.g.blocks;
    a.ranks = choose_ranks(a.R <= a.tile ? int64_t(a.g.blocks) * touched : most, (a.g.chunks + a.step - 1) / a.step, sms);
    const int sums = (a.ranks > 1 ? 2 : 1) * kSets * a.tile * kRows * 4;
    a.stages = (kShared - sums) / a.stage_bytes;
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    if (a.stages < 2 || a.bufs < 1) return set_last_error(CST_ERR_INVALID_ARG, "no room for a product of this shape");
    const int64_t clusters = most < sms / a.ranks ? most : sms / a.ranks;

    CUtensorMap map;
    const EncodeTiled encode = encode_tiled();
    if (!encode) return set_last_error(CST_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
    // [chunk][row and term][128 columns of the chunk], of three terms [chunk][term][row][128 columns]
    const cuuint64_t chunks = a.g.chunks, width = chunks * kChunk, R = a.R;
    const cuuint32_t tile = a.tile, step = a.step, ones[4] = {1, 1, 1, 1};
    const cuuint64_t dims[4] = {kChunk, TERMS == 3 ? R : R * TERMS, TERMS == 3 ? 3 : chunks, chunks};
    const cuuint64_t strides[3] = {width, TERMS == 3 ? R * width : kChunk, kChunk};
    const cuuint32_t box[4] = {kChunk, TERMS == 3 ? tile : tile * TERMS, TERMS == 3 ? 3 : step, step};
    const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, TERMS == 3 ? 4 : 3, workspace, dims, strides, box, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_last_error(CST_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", int(r));

    auto kernel = int4_kernel<TERMS, GROUPS>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared);
    if (e == cudaSuccess) {
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
        e = cudaLaunchKernelEx(&cfg, kernel, map, a);
    }
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "grouped_int4 launch failed: %s", cudaGetErrorString(e));
    return CST_OK;
}

template <int TERMS>
int launch_terms(Int4Args a, const void* x, int x_dtype, int64_t ld_x, const float* x_scale, int64_t ld_xs,
                 void* workspace, int sms, cudaStream_t s) {
    float* facts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + terms_bytes(a.g, TERMS, a.R));
    a.facts = facts;
    // a thread for 8 columns, up to 256 (131072 rows of k = 128: 138 us, with 256 threads 364)
    const int threads = a.g.chunks >= 16 ? 256 : (a.g.chunks + 1) / 2 * 32;
    const cudaError_t e = launch_chained(split_x_kernel<TERMS>, dim3(unsigned(a.R)), dim3(threads), 0, s, x, x_dtype, ld_x,
                                         x_scale, ld_xs, a.R, a.g.K, static_cast<uint8_t*>(workspace), facts);
    if (e != cudaSuccess) return set_last_error(CST_ERR_CUDA, "split_x launch failed: %s", cudaGetErrorString(e));
    return a.g.group == 128  ? launch_int4<TERMS, 1>(a, workspace, sms, s)
           : a.g.group == 64 ? launch_int4<TERMS, 2>(a, workspace, sms, s)
                             : launch_int4<TERMS, 4>(a, workspace, sms, s);
}

int terms_of(int x_dtype) { return x_dtype == CST_DTYPE_E4M3 ? 1 : x_dtype == CST_DTYPE_BF16 ? 2 : 3; }

int check_x_dtype(int x_dtype) {
    if (x_dtype != CST_DTYPE_FP16 && x_dtype != CST_DTYPE_BF16 && x_dtype != CST_DTYPE_E4M3)
        return set_last_error(CST_ERR_INVALID_ARG, "x must be fp16, bf16 or e4m3, got dtype %d", x_dtype);
    return CST_OK;
}

// Rows in memory: `rows` of `bytes`, `pitch` bytes apart.
struct Extent {
    const void* p;
    int64_t rows, bytes, pitch;
    uint64_t first() const { return reinterpret_cast<uintptr_t>(p); }
    uint64_t end() const { return first() + uint64_t((rows - 1) * pitch + bytes); }
};

// Whether two extents may share a byte; columns of one array that lie side by side share none.
bool overlap(const Extent& a, const Extent& b) {
    if (!a.p || !b.p || a.first() >= b.end() || b.first() >= a.end()) return false;
    if (a.pitch != b.pitch) return true;
    const int64_t shift = b.first() >= a.first() ? int64_t((b.first() - a.first()) % uint64_t(a.pitch))
                                                 : a.pitch - 1 - int64_t((a.first() - b.first() - 1) % uint64_t(a.pitch));
    return shift < a.bytes || shift + b.bytes > a.pitch;
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

extern "C" int cst_int4_workspace(const cst_int4_weight* w, int32_t x_dtype, int32_t R, int64_t* bytes) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (const int rc = check_x_dtype(x_dtype)) return rc;
    if (R < 0 || !bytes) return set_last_error(CST_ERR_INVALID_ARG, "R=%d must be >= 0 and bytes not null", R);
    const Geom g = make_geom(*w);
    const int terms = terms_of(x_dtype);
    *bytes = terms_bytes(g, terms, R) + int64_t(R) * g.chunks * (terms == 1 ? kFactBytes : 4);
    return CST_OK;
}

extern "C" int cst_grouped_int4(const cst_int4_weight* w, void* data, const void* x, int32_t x_dtype, int64_t ld_x,
                                const float* x_scale, int64_t ld_x_scale, const int32_t* offsets, int32_t R,
                                void* workspace, void* out, int32_t out_dtype, int64_t ld_out, void* stream) {
    clear_last_error();
    if (const int rc = check_weight(w)) return rc;
    if (const int rc = check_x_dtype(x_dtype)) return rc;
    const Geom g = make_geom(*w);
    if (out_dtype < CST_DTYPE_FP16 || out_dtype > CST_DTYPE_FP32)
        return set_last_error(CST_ERR_INVALID_ARG, "invalid out dtype %d", out_dtype);
    if ((x_dtype == CST_DTYPE_E4M3) != (x_scale != nullptr) && R > 0)
        return set_last_error(CST_ERR_INVALID_ARG, "x_scale goes with e4m3 rows, and only with them");
    if (!offsets && w->n_experts != 1)
        return set_last_error(CST_ERR_INVALID_ARG, "offsets are needed for %d experts", w->n_experts);
    if (R < 0 || R > (1 << 28) || ld_x < w->k || ld_out < g.out_n || (x_scale && ld_x_scale < (w->k + 127) / 128))
        return set_last_error(CST_ERR_INVALID_ARG, "R=%d must be in [0, 2^28] and no row stride below the row", R);
    if (R == 0) return CST_OK;
    if (!data || !x || !out || !workspace)
        return set_last_error(CST_ERR_INVALID_ARG, "null data, x, workspace or out");
    if (((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(workspace)) & 15u))
        return set_last_error(CST_ERR_INVALID_ARG, "data and workspace must be 16-byte aligned");
    // Rows of `out` are written before the last of these is read: by the product's CTAs while others have not begun,
    // and where they belong to no expert even beside split_x_kernel.
    const int64_t x_size = act_size(x_dtype), out_size = act_size(out_dtype), xs = (w->k + kChunk - 1) / kChunk;
    const Extent written{out, R, g.out_n * out_size, ld_out * out_size};
    int64_t data_bytes = 0, room_bytes = 0;
    cst_int4_bytes(w, &data_bytes);
    cst_int4_workspace(w, x_dtype, R, &room_bytes);
    const struct {
        const char* name;
        Extent at;
    } read[] = {{"x", {x, R, w->k * x_size, ld_x * x_size}},
                {"x_scale", {x_scale, R, xs * 4, ld_x_scale * 4}},
                {"offsets", {offsets, 1, (w->n_experts + 1) * 4, (w->n_experts + 1) * 4}},
                {"the weight", {data, 1, data_bytes, data_bytes}},
                {"the workspace", {workspace, 1, room_bytes, room_bytes}}};
    for (const auto& r : read)
        if (overlap(written, r.at))
            return set_last_error(CST_ERR_INVALID_ARG, "out overlaps %s, which is still read while results are written",
                                  r.name);
    const int sms = current_sms();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Int4Args a{};
    a.g = g;
    a.data = static_cast<const uint8_t*>(data);
    a.offsets = offsets;
    a.R = R;
    a.out = out;
    a.out_dtype = out_dtype;
    a.ld_out = ld_out;
    a.err = reinterpret_cast<int*>(static_cast<uint8_t*>(data) + g.expert_bytes() * g.E);
    auto launch = x_dtype == CST_DTYPE_E4M3 ? launch_terms<1> : x_dtype == CST_DTYPE_BF16 ? launch_terms<2> : launch_terms<3>;
    return launch(a, x, x_dtype, ld_x, x_scale, ld_x_scale, workspace, sms, s);
}
