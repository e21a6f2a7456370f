// Causal attention over a packed token stream, forward and backward, on sm_100a tensor cores.
//
// The stream holds sequences one after another (cu_seqlens); a query attends to the keys of its own
// sequence up to its own position. Query head h reads key/value head h / (heads / kv_heads). With
// s_ij = scale q_i . k_j, p_ij = exp(s_ij - lse_i), lse_i = log sum_{j <= i} exp(s_ij):
//   o_i  = sum_j p_ij v_j
//   dv_j = sum_i p_ij do_i,  ds_ij = p_ij (do_i . v_j - delta_i),  delta_i = o_i . do_i
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i    (dk, dv also over the head's group)
//
// Tiles are 128 x 128 scores; a head is kD = 64 or 128 wide in shared memory (narrower heads are padded
// with zeros by the tensor-map bounds). Scores, statistics and all sums are float32 in tensor memory or
// registers; p and ds are rounded to the inputs' type where they become operands of the second product.
//
//   plan      one small launch: the list of row blocks of all sequences, longest work first, and zeros
//             for the rows that no sequence owns
//   forward   persistent CTAs, two 128-row query tiles each: while one tile's softmax runs, the tensor
//             core works for the other. p overwrites s in tensor memory and is the A operand of p v
//   dkdv      a 128-row key tile per work item, all query tiles and heads that see it; s^T and dp^T
//             are computed transposed so that p^T and ds^T are A operands from tensor memory
//   dq        a 128-row query tile per work item over its key tiles
// dk, dv and dq are each summed by one CTA in a fixed order: no atomics, the same bits every time. That
// costs two of seven products (s and dp are computed twice).
//
// What bounds it: long sequences run into the board's power limit (16384 tokens, 32 heads on 8 of 128, bf16:
// forward 1.62 ms, 1350 TFLOP/s; dkdv 3.1-3.2 ms, 1400 TFLOP/s, both at 1.6 GHz; dq 2.6-2.9 ms, 1140-1270
// TFLOP/s), short ones and narrow heads the chain scores -> softmax -> product of a query tile (8192 tokens of
// ragged prompts, 16 heads on 4 of 64, fp16: 83 us, 530 TFLOP/s), since one tile's softmax takes about 1700
// cycles of which 1024 are the ex2 unit's, and tensor memory holds no third tile of width 128. Work items are not split
// where they are few: with 4 heads on 1 at 8192 tokens dkdv has 64 for 148 SMs, each of up to 256 steps, and takes 380
// us where balanced work would take about 85 (forward: 128 items, 115 us where it would take 50).
//
// Rows beyond a sequence's end inside a tile belong to other sequences: their scores are masked by
// selection, and where a masked (zero) probability would multiply such a row, the row is zeroed in shared
// memory first, so that not even a NaN crosses over. Every wait is bounded, as in the grouped GEMM; after one that
// ran out a CTA still waits for its copies and products in flight before it ends.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace xma {
namespace attn {

using namespace ptx;

constexpr int kTile = 128;            // query or key rows of a tile
constexpr int kThreads = 384;         // load warp, MMA warp, two idle, two groups of four compute warps
constexpr int kTmemCols = 512;
// The accumulator is rescaled when a row's maximum grew by more than 2^kRescaleLog2, and p carries 2^kShiftLog2: together
// they leave a factor of two under fp16's largest number, and p of a key that others outweigh keeps its bits down to 2^-23
// beside the row's largest and has some down to 2^-33 (without the shift 2^-14 and 2^-25, which thousands of such keys
// show). 2^4 and 2^11 cost rescaled tiles: 8192 tokens, 32 heads on 8 of 128, 465 us against 441; 2^6 costs nothing. bf16
// has float32's range and needs no shift.
template <typename T>
constexpr float kRescaleLog2 = std::is_same<T, __half>::value ? 6.f : 8.f;
template <typename T>
constexpr float kShiftLog2 = std::is_same<T, __half>::value ? 9.f : 0.f;
// The same in the backward pass, where p is at most 1: it carries 2^kProbLog2, which the row statistics are kept less of
// and dv and ds are divided by; a factor of four under the largest number is for what the exponent is off by.
template <typename T>
constexpr int kProbLog2 = std::is_same<T, __half>::value ? 14 : 0;
template <typename T>
constexpr float kProbInverse = 1.f / static_cast<float>(1 << kProbLog2<T>);
constexpr int kControlRegs = 88;      // registers of the load and MMA warps' group and of the compute groups:
constexpr int kComputeRegs = 208;     // 128 * 88 + 256 * 208 = 384 * 168
constexpr int kPlanThreads = 1024;
constexpr int kPlanBuckets = 1024;
constexpr int kMaxHeads = 4096;

// One block of rows of one sequence.
struct Block {
    int start;  // first token of the sequence
    int len;    // its tokens
    int index;  // block number inside the sequence
    int pad;    // first entry of the sequence in the padded row statistics
};

struct Params {
    const Block* blocks;
    const int32_t* num_blocks;
    int heads, kv_heads, group, dim;
    int dim_steps;     // ceil(dim / 16): what the products see of a head, zeros up to there
    int64_t pad_rows;  // entries of the padded row statistics per head
    float scale, scale_log2;
    void* out;         // forward: o
    float* lse;        // [heads][pad_rows], log2 units, less kProbLog2; may be NULL in the forward pass
    uint8_t* rest;     // [tokens, heads, rest_row]: what out's rounding took away; NULL when lse is
    int64_t rest_row;  // dim, rounded up to 16
    const float* delta;      // negated
    void* dq;
    void* dk;
    void* dv;
    const uint32_t* absmax;  // backward, fp16: bit patterns of the largest finite |do| and |v|
    int32_t* status;
    int ab_format;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lg2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// ---------------------------------------------------------------------------------------------
// Plan
// ---------------------------------------------------------------------------------------------

// Sequence b of cu_seqlens, clamped into the stream whatever the array holds.
template <typename IntT>
__device__ __forceinline__ void sequence(const IntT* cu, int64_t b, int64_t total, int* start, int* len) {
    const int64_t s = min(max(static_cast<int64_t>(cu[b]), int64_t(0)), total);
    const int64_t e = min(max(static_cast<int64_t>(cu[b + 1]), s), total);
    *start = static_cast<int>(s);
    *len = static_cast<int>(e - s);
}
__device__ __forceinline__ int pad_offset(int start, int64_t b) { return static_cast<int>((start / kTile + b) * kTile); }

struct ZeroRows {
    void* base;
    int64_t row_bytes;  // a multiple of 16
};

// Block 0 (and 1, for the second list) writes a list; the others zero the rows before the first and after
// the last sequence. A list holds every block of `block_rows` rows of every sequence, by falling work:
// kFromEnd = false: a block's index (keys before it), true: the number of blocks after it. Offsets out of order are no
// valid cu_seqlens: sequences would overlap and could be more than a list holds, or than its counters count. They get an
// empty list; in order, the blocks are at most total / block_rows + batch.
template <typename IntT>
__global__ void __launch_bounds__(kPlanThreads)
plan_kernel(const IntT* __restrict__ cu, int64_t batch, int64_t total, int block_rows, Block* list0, int32_t* count0, Block* list1,
            int32_t* count1, uint32_t* absmax, ZeroRows z0, ZeroRows z1, ZeroRows z2, int num_lists) {
    if (static_cast<int>(blockIdx.x) >= num_lists) {
        const int64_t first = min(max(static_cast<int64_t>(cu[0]), int64_t(0)), total);
        const int64_t last = min(max(static_cast<int64_t>(cu[batch]), first), total);
        const int64_t tail = total - last, rows = first + tail;
        const int64_t at = static_cast<int64_t>(blockIdx.x - num_lists) * blockDim.x + threadIdx.x;
        const int64_t step = static_cast<int64_t>(gridDim.x - num_lists) * blockDim.x;
        const ZeroRows zs[3] = {z0, z1, z2};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            if (zs[i].base == nullptr) continue;
            const int64_t per_row = zs[i].row_bytes / 16;
            for (int64_t c = at; c < rows * per_row; c += step) {
                const int64_t r = c / per_row;
                const int64_t row = r < first ? r : last + (r - first);
                reinterpret_cast<uint4*>(zs[i].base)[row * per_row + (c - r * per_row)] = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    const bool from_end = blockIdx.x == 1;
    Block* list = from_end ? list1 : list0;
    __shared__ int bucket[kPlanBuckets];
    __shared__ int warp_sum[32];
    for (int i = threadIdx.x; i < kPlanBuckets; i += blockDim.x) bucket[i] = 0;
    if (threadIdx.x < 2 && absmax != nullptr && !from_end) absmax[threadIdx.x] = 0;
    int32_t* count = from_end ? count1 : count0;
    bool falls = false;
    for (int64_t b = threadIdx.x; b < batch; b += kPlanThreads) falls = falls || cu[b + 1] < cu[b];
    if (__syncthreads_or(falls)) {
        if (threadIdx.x == 0) *count = 0;
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int64_t b = warp; b < batch; b += kPlanThreads / 32) {
        int start, len;
        sequence(cu, b, total, &start, &len);
        const int n = (len + block_rows - 1) / block_rows;
        for (int i = lane; i < n; i += 32) atomicAdd(&bucket[min(from_end ? n - 1 - i : i, kPlanBuckets - 1)], 1);
    }
    __syncthreads();
    // thread t takes bucket kPlanBuckets - 1 - t: an exclusive prefix sum from the largest work down
    const int mine = kPlanBuckets - 1 - static_cast<int>(threadIdx.x);
    const int value = bucket[mine];
    int incl = value;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, off);
        if (lane >= off) incl += o;
    }
    if (lane == 31) warp_sum[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int v = warp_sum[lane];
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, v, off);
            if (lane >= off) v += o;
        }
        warp_sum[lane] = v;
    }
    __syncthreads();
    bucket[mine] = incl - value + (warp > 0 ? warp_sum[warp - 1] : 0);
    if (threadIdx.x == 0) *count = warp_sum[31];
    __syncthreads();
    for (int64_t b = warp; b < batch; b += kPlanThreads / 32) {
        int start, len;
        sequence(cu, b, total, &start, &len);
        const int n = (len + block_rows - 1) / block_rows;
        for (int i = lane; i < n; i += 32) {
            // the order inside a bucket is not fixed; it decides who computes a block, not what
            const int at = atomicAdd(&bucket[min(from_end ? n - 1 - i : i, kPlanBuckets - 1)], 1);
            list[at] = Block{start, len, i, pad_offset(start, b)};
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Shared device pieces
// ---------------------------------------------------------------------------------------------

// A list entry, read by a converged warp and known to be the same in all of it.
__device__ __forceinline__ Block load_block(const Block* at) {
    const int4 v = __ldg(reinterpret_cast<const int4*>(at));
    return Block{warp_uniform(v.x), warp_uniform(v.y), warp_uniform(v.z), warp_uniform(v.w)};
}

// A [128, kD] tile of one head from a [tokens, heads, dim] tensor: kD / 64 boxes of 128 rows x 64 columns
// (128-byte swizzle), 16 KB each.
template <int kD>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, uint32_t bar, int head, int row) {
#pragma unroll
    for (int c = 0; c < kD / 64; ++c) tma_load_3d_cta1(dst + c * (kTile * 128), map, bar, c * 64, head, row);
}

// Rows [first, 128) of a tile become zeros (a warp's work); the tile's rows are 128 bytes per box.
template <int kD>
__device__ __forceinline__ void zero_tile_rows(uint32_t tile, int first, int lane) {
    const int chunks = (kTile - first) * 8;
#pragma unroll
    for (int c = 0; c < kD / 64; ++c)
        for (int i = lane; i < chunks; i += 32)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(tile + c * (kTile * 128) + first * 128 + i * 16), "r"(0) : "memory");
}

// Operand with the reduction along the head dimension (a tile's rows are rows or columns of the product),
// and its step kk of 16 elements.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t tile) { return make_smem_desc(tile, 0, 1024); }
__device__ __forceinline__ constexpr uint64_t k_step(int kk) { return ((kk >> 2) * (kTile * 128) + (kk & 3) * 32) >> 4; }
// Operand with the reduction along the tile's rows (the head dimension is a dimension of the product).
__device__ __forceinline__ uint64_t desc_row_major(uint32_t tile) { return make_smem_desc(tile, kTile * 128, 1024); }
__device__ __forceinline__ constexpr uint64_t row_step(int kk) { return (kk * 2048) >> 4; }

// D[128, 128] = A B^T over the head dimension, `steps` times 16 of it.
template <int kD>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a_tile, uint32_t b_tile, uint32_t idesc, int steps) {
    const uint64_t a = desc_k_major(a_tile), b = desc_k_major(b_tile);
#pragma unroll
    for (int kk = 0; kk < kD / 16; ++kk)
        if (kk < steps) umma_ss_cta1(d, a + k_step(kk), b + k_step(kk), idesc, kk != 0 ? 1u : 0u);
}
// D[128, head] (+)= A B over rows 16 kFirst .. 16 kLast - 1 of B; A in tensor memory, the part for the upper 64
// rows `second` columns on.
template <int kFirst = 0, int kLast = kTile / 16>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t second, uint32_t b_tile, uint32_t idesc, bool accumulate) {
    const uint64_t b = desc_row_major(b_tile);
#pragma unroll
    for (int kk = kFirst; kk < kLast; ++kk)
        umma_ts_cta1(d, a + (kk >> 2) * second + (kk & 3) * 8, b + row_step(kk), idesc, (accumulate || kk != 0) ? 1u : 0u);
}

// p in two operands, for sequences of one key tile: rounded down, and what that took. Few keys do not average p's rounding
// out, and the backward pass meets it again in delta: with one operand o was 1.04 to 1.14 and dq 1.46 to 1.52 times a
// single rounding off on sequences of 120 to 2 tokens, with two 1.0 and 1.42. Longer sequences (700 tokens: 1.23 and 1.47)
// gain less and would pay a product more. The second operand is positive where p is, so that an infinite value makes an
// infinity, as in one product, and no NaN.
template <typename T>
constexpr float kLeast = std::is_same<T, __half>::value ? 0x1p-24f : 0x1p-100f;
template <typename T>
__device__ __forceinline__ uint32_t pack2_down(float a, float b) {
    uint32_t r;
    if (std::is_same<T, __half>::value) asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    else asm("cvt.rz.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
// 32 columns of scores, of which `row` sees `seen`: p times 2^kShiftLog2 beside the row's maximum, as packed operands; the sum
// of p is returned. `neg_m` is the shift less the maximum.
template <typename T>
__device__ __forceinline__ float two_operands(const uint32_t (&s)[32], int seen, float scale_log2, float neg_m, uint32_t* high, uint32_t* low) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float a = 2 * i < seen ? ex2(fmaf(__uint_as_float(s[2 * i]), scale_log2, neg_m)) : 0.f;
        const float b = 2 * i + 1 < seen ? ex2(fmaf(__uint_as_float(s[2 * i + 1]), scale_log2, neg_m)) : 0.f;
        sum += a + b;
        high[i] = pack2_down<T>(a, b);
        const float2 f = unpack2<T>(high[i]);
        low[i] = pack2<T>(fmaxf(a - f.x, fminf(a, kLeast<T>)), fmaxf(b - f.y, fminf(b, kLeast<T>)));
    }
    return sum;
}

// The softmax of such a tile, a row a thread: scores at taddr to operands, the first of 64 keys at columns 64 h .. 64 h + 31,
// the second at the 32 after them; `ready` are the halves' barriers. Returns the row's maximum (log2 units) and sum. A call
// of its own: inlined it costs the long sequences' loops registers.
template <typename T>
__device__ __noinline__ float2 one_tile_probabilities(uint32_t taddr, int row, float scale_log2, uint32_t ready) {
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
        uint32_t s[32];
        tmem_ld32(taddr + c * 32, s);
        tmem_ld_wait();
        tmem_tie32(s);
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (c * 32 + i <= row) m = fmaxf(m, __uint_as_float(s[i]));
    }
    m *= scale_log2;
    const float neg_m = m == -INFINITY ? 0.f : kShiftLog2<T> - m;
#pragma unroll 1
    for (int h = 0; h < 2; ++h) {
        uint32_t s[2][32], high[32], low[32];
        tmem_ld32(taddr + h * 64, s[0]);
        tmem_ld32(taddr + h * 64 + 32, s[1]);
        tmem_ld_wait();
        tmem_tie32(s[0]);
        tmem_tie32(s[1]);
        l += two_operands<T>(s[0], row + 1 - h * 64, scale_log2, neg_m, high, low);
        l += two_operands<T>(s[1], row + 1 - h * 64 - 32, scale_log2, neg_m, high + 16, low + 16);
        tmem_st32(taddr + h * 64, high);
        tmem_st32(taddr + h * 64 + 32, low);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(ready + 8 * h);
    }
    return make_float2(m, l);
}
// The products of half h of such a tile. Rolled up: with the loops written out the kernel's other loops lost 4 % (8192
// tokens 446 us against 426), to the instruction cache as it seems.
__device__ __forceinline__ void one_tile_products(uint32_t d, uint32_t a, uint32_t b_tile, uint32_t idesc, int h) {
    const uint64_t b = desc_row_major(b_tile);
#pragma unroll 1
    for (int part = 0; part < 2; ++part)
#pragma unroll 1
        for (int kk = 0; kk < 4; ++kk)
            umma_ts_cta1(d, a + h * 64 + part * 32 + kk * 8, b + row_step(h * 4 + kk), idesc, (h != 0 || part != 0 || kk != 0) ? 1u : 0u);
}

// What rounding o to T takes away is kept in 8 bits (e5m2, times a power of two that puts the residue of values from
// 2^-16 to 2^12 into its range; beyond it saturates or underflows). delta = o . do is subtracted for every key of a
// row, so an error of o would not average out over the keys; two mantissa bits leave an eighth of it at most.
template <typename T>
constexpr float kRestScale = std::is_same<T, __half>::value ? 32768.f : 4096.f;

// 32 values of o, divided by their row's sum. The sum adds p as it was, the product p as it was rounded (2^-11 off at most),
// so a mean of values next to fp16's largest number could round to infinity; no mean is above the largest value.
template <typename T>
__device__ __forceinline__ void scale_output(uint32_t (&r)[32], float scale) {
    float top[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const float v = __uint_as_float(r[i]) * scale;
        r[i] = __float_as_uint(v);
        if (std::is_same<T, __half>::value) top[i & 3] = fmaxf(top[i & 3], fabsf(v));
    }
    if (std::is_same<T, __half>::value &&
        __any_sync(0xffffffffu, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) > 65504.f)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const float v = __uint_as_float(r[i]);
            if (fabsf(v) < 65600.f) r[i] = __float_as_uint(fminf(fmaxf(v, -65504.f), 65504.f));  // an infinity stays one
        }
    }
}

// 16-byte pieces of one row of kD float32 values in tensor memory, scaled and rounded, to global memory.
template <typename T, int kD, bool kOutput = false>
__device__ __forceinline__ void store_row(uint32_t taddr, T* dst, int dim, float scale, bool valid) {
#pragma unroll
    for (int c = 0; c < kD / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(taddr + c * 32, r);
        tmem_ld_wait();
        tmem_tie32(r);
        if (kOutput) {
            scale_output<T>(r, scale);
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * scale);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (valid && c * 32 + q * 8 < dim) {
                uint4 v;
                v.x = pack2<T>(__uint_as_float(r[q * 8]), __uint_as_float(r[q * 8 + 1]));
                v.y = pack2<T>(__uint_as_float(r[q * 8 + 2]), __uint_as_float(r[q * 8 + 3]));
                v.z = pack2<T>(__uint_as_float(r[q * 8 + 4]), __uint_as_float(r[q * 8 + 5]));
                v.w = pack2<T>(__uint_as_float(r[q * 8 + 6]), __uint_as_float(r[q * 8 + 7]));
                *reinterpret_cast<uint4*>(dst + c * 32 + q * 8) = v;
            }
        }
    }
}

// Byte `at` of a staging tile as a bulk store with 128-byte swizzle reads it (tile 1024-byte aligned).
__device__ __forceinline__ uint32_t swizzled(uint32_t at) { return at ^ ((at >> 7 & 7u) << 4); }
__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// What rounding took from eight values, one byte each.
template <typename T>
__device__ __forceinline__ uint2 rest8(const uint32_t* r) {
    uint32_t two[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = __uint_as_float(r[2 * e]), b = __uint_as_float(r[2 * e + 1]);
        const float2 f = unpack2<T>(pack2<T>(a, b));
        two[e] = __nv_cvt_float2_to_fp8x2(make_float2((a - f.x) * kRestScale<T>, (b - f.y) * kRestScale<T>), __NV_SATFINITE, __NV_E5M2);
    }
    return make_uint2(two[0] | two[1] << 16, two[2] | two[3] << 16);
}

// The output rows of one warp (32 of a tile, one a lane) and, with `save`, what their rounding took away. Full
// groups of rows leave through bulk tensor stores from the warp's 4 KB staging tile: 32 rows written 16 bytes a lane
// straight from registers would take the load/store unit 32 cycles an instruction, some 4000 cycles a work item. Rows
// at a sequence's end go that way, since a tile's store would run into the next sequence.
template <typename T, int kD>
__device__ __forceinline__ void store_output(uint32_t o_addr, uint32_t staging, const CUtensorMap* map_out, const CUtensorMap* map_rest,
                                             T* out, uint8_t* rest, int64_t rest_row, int64_t token, int rows, int heads, int head,
                                             int dim, float scale, int lane) {
    if (rows <= 0) return;
    if (rows < 32) {
        const int64_t row = (token + lane) * heads + head;
        store_row<T, kD, true>(o_addr, out + row * dim, dim, scale, lane < rows);
        if (rest == nullptr) return;
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(o_addr + c * 32, r);
            tmem_ld_wait();
            tmem_tie32(r);
            scale_output<T>(r, scale);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (lane < rows && c * 32 + q * 8 < dim)
                    *reinterpret_cast<uint2*>(rest + row * rest_row + c * 32 + q * 8) = rest8<T>(r + q * 8);
        }
        return;
    }
#pragma unroll 1
    for (int c = 0; c < kD / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(o_addr + c * 32, r);
        if ((c & 1) == 0) {
            if (lane == 0) bulk_wait_read<0>();  // the store that used the tile last has read it
            __syncwarp();
        }
        tmem_ld_wait();
        tmem_tie32(r);
        scale_output<T>(r, scale);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = pack2<T>(__uint_as_float(r[q * 8 + 2 * e]), __uint_as_float(r[q * 8 + 2 * e + 1]));
            st_shared16(staging + swizzled(lane * 128 + ((c & 1) * 4 + q) * 16), w[0], w[1], w[2], w[3]);
        }
        if (c & 1) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0 && (c - 1) * 32 < dim) {
                tma_store_3d(map_out, staging, (c - 1) * 32, head, static_cast<int>(token));
                bulk_commit();
            }
        }
    }
    if (rest == nullptr) return;
    if (lane == 0) bulk_wait_read<0>();
    __syncwarp();
#pragma unroll 1
    for (int c = 0; c < kD / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(o_addr + c * 32, r);
        tmem_ld_wait();
        tmem_tie32(r);
        scale_output<T>(r, scale);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint2 a = rest8<T>(r + h * 16), b = rest8<T>(r + h * 16 + 8);
            st_shared16(staging + swizzled(lane * 128 + c * 32 + h * 16), a.x, a.y, b.x, b.y);
        }
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
        tma_store_3d(map_rest, staging, 0, head, static_cast<int>(token));
        bulk_commit();
    }
}

// The item a CTA takes in its turn-th turn: items lie by falling work, so every other turn runs backwards
// through the CTAs, which evens out what one CTA gets.
__device__ __forceinline__ int64_t work_item(int64_t turn) {
    return turn * gridDim.x + ((turn & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// After a wait that ran out, a CTA waits once more, for what it has in flight (bounded too): copies write shared memory
// and products read it and write tensor memory, all of which another CTA gets next. A load role leaves where its ring
// and its resident tiles stand (the parity of the last turn, 1 if there was none); MMA warps' products are asked for. At
// the end of every CTA instead, without the branch, the loops above came out 2 % slower.
__device__ __forceinline__ uint32_t pack_in_flight(const Ring& ring, uint32_t resident0, uint32_t resident1) {
    return static_cast<uint32_t>(ring.stage) | ring.phase << 8 | resident0 << 9 | resident1 << 10;
}
__device__ __forceinline__ void settle_copies(uint32_t packed, uint32_t full, int stages, uint32_t resident0, uint32_t resident1) {
    Ring ring;
    ring.stage = static_cast<int>(packed & 0xffu);
    ring.phase = packed >> 8 & 1u;
    const uint64_t now = global_timer_ns();
    ring.settle(full, stages, now);
    mbar_settle(resident0, packed >> 9 & 1u, now);
    mbar_settle(resident1, packed >> 10 & 1u, now);
}
__device__ __forceinline__ void settle_products(uint32_t bar) {
    if (elect_one()) umma_commit_cta1(bar);
    __syncwarp();
    mbar_settle(bar, 0, global_timer_ns());
    __syncwarp();
}

// ---------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------

template <int kD>
struct Forward {
    static constexpr uint32_t kTileBytes = kTile * kD * 2;
    static constexpr int kStages = kD == 128 ? 4 : 8;
    static constexpr uint32_t kStaging = 4096;  // of each compute warp
    static constexpr uint32_t kSmem = 1024 + (2 + kStages) * kTileBytes + 8 * kStaging + 256;
    static_assert(kSmem <= 227 * 1024, "shared memory");
    static constexpr uint32_t kO = 256;  // tensor memory: s of the two tiles at 0 and 128, o at 256 and 256 + kD
};

// Work item: 256 query rows (two tiles) of one head. Tile t's last key tile is its diagonal.
// One MMA warp serves both tiles in turn: that keeps their softmaxes half a period apart, where two MMA warps, or
// scores issued further ahead, let them fall into step and wait for the same unit (measured 520 and 441 us against
// 427 and 409 for 8192 tokens). Its operands are computed warp-uniformly: issued from a branch on the lane number
// every product took 100 cycles to issue and 577 us were needed.
template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1)
forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
               const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_out,
               const __grid_constant__ CUtensorMap map_rest, const Params p) {
    using F = Forward<kD>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t q_tile = base, ring = base + 2 * F::kTileBytes;
    constexpr uint32_t kStagingAt = (2 + F::kStages) * F::kTileBytes, kBars = kStagingAt + 8 * F::kStaging;
    const uint32_t bars = base + kBars;
    const uint32_t full = bars, empty = bars + 64;
    const uint32_t q_full = bars + 128, q_empty = bars + 144, s_full = bars + 160, o_full = bars + 176;
    const uint32_t p_ready = bars + 192;  // [tile][half of the keys]
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + kBars + 224);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + kBars + 228);
    const uint32_t settled = bars + 232;
    volatile uint32_t* in_flight = reinterpret_cast<volatile uint32_t*>(gen + kBars + 240);

    const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < F::kStages; ++i) {
            mbar_init(full + 8 * i, 1);
            mbar_init(empty + 8 * i, 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full + 8 * t, 1);
            mbar_init(q_empty + 8 * t, 1);
            mbar_init(s_full + 8 * t, 1);
            mbar_init(p_ready + 16 * t, 4);  // the four warps of a tile
            mbar_init(p_ready + 16 * t + 8, 4);
            mbar_init(o_full + 8 * t, 1);
        }
        mbar_init(settled, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }
    if (warp == 1) {
        tmem_alloc(bars + 228, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    const int64_t items = static_cast<int64_t>(warp_uniform(*p.num_blocks)) * p.heads;

    if (warp < 4) regs_shrink<kControlRegs>();  // in a branch of its own: the compute branch keeps its budget
    if (warp == 0) {
        if (lane == 0) {
            Ring kv;
            uint32_t q_phase[2] = {1u, 1u};
            bool ok = true;
            for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
                const Block b = p.blocks[it / p.heads];
                const int head = static_cast<int>(it % p.heads), kv_head = head / p.group;
                const int row0 = b.index * 2 * kTile;
                const int tiles = b.len > row0 + kTile ? 2 : 1;
                const int n = b.index * 2 + tiles;
                for (int t = 0; ok && t < tiles; ++t) {
                    ok = mbar_wait(q_empty + 8 * t, q_phase[t], abort_flag, p.status, 501);
                    if (!ok) break;
                    q_phase[t] ^= 1u;
                    mbar_expect_tx(q_full + 8 * t, F::kTileBytes);
                    load_tile<kD>(q_tile + t * F::kTileBytes, &map_q, q_full + 8 * t, head, b.start + row0 + t * kTile);
                }
                for (int j = 0; ok && j < 2 * n; ++j) {  // k of tile 0, v of tile 0, k of tile 1, ...
                    ok = mbar_wait(empty + 8 * kv.stage, kv.phase ^ 1u, abort_flag, p.status, 502);
                    if (!ok) break;
                    mbar_expect_tx(full + 8 * kv.stage, F::kTileBytes);
                    load_tile<kD>(ring + kv.stage * F::kTileBytes, (j & 1) ? &map_v : &map_k, full + 8 * kv.stage, kv_head,
                                  b.start + (j >> 1) * kTile);
                    kv.next(F::kStages);
                }
            }
            *in_flight = pack_in_flight(kv, q_phase[0], q_phase[1]);
        }
        __syncwarp();
    } else if (warp == 1) {
        const uint32_t idesc_s = make_idesc(kTile, kTile, false, false, p.ab_format);
        const uint32_t idesc_o = make_idesc(kTile, p.dim_steps * 16, false, true, p.ab_format);
        Ring kv;
        uint32_t q_phase[2] = {0u, 0u}, p_phase[2] = {0u, 0u};
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = load_block(p.blocks + it / p.heads);
            const int row0 = b.index * 2 * kTile;
            const int tiles = b.len > row0 + kTile ? 2 : 1;
            const int n = b.index * 2 + tiles;              // key tiles of the last query tile
            const int first = b.index * 2 + 1;              // key tiles of query tile 0
            // s of key tile 0
            ok = mbar_wait_warp(full + 8 * kv.stage, kv.phase, abort_flag, p.status, 503);
            for (int t = 0; ok && t < tiles; ++t) {
                ok = mbar_wait_warp(q_full + 8 * t, q_phase[t], abort_flag, p.status, 504);
                if (!ok) break;
                q_phase[t] ^= 1u;
                tc_fence_after();
                if (elect_one()) {
                    mma_scores<kD>(tmem + t * kTile, q_tile + t * F::kTileBytes, ring + kv.stage * F::kTileBytes, idesc_s, p.dim_steps);
                    umma_commit_cta1(s_full + 8 * t);
                    if (first + t == 1) umma_commit_cta1(q_empty + 8 * t);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (elect_one()) umma_commit_cta1(empty + 8 * kv.stage);
            kv.next(F::kStages);
            if (b.len <= kTile) {  // p comes in two operands
                const uint32_t v_tile = ring + kv.stage * F::kTileBytes;
                ok = mbar_wait_warp(full + 8 * kv.stage, kv.phase, abort_flag, p.status, 505);
                if (!ok) break;
                if (b.len < kTile) {
                    zero_tile_rows<kD>(v_tile, b.len, lane);
                    fence_proxy_async();
                    __syncwarp();
                }
                for (int h = 0; ok && h < 2; ++h) {
                    ok = mbar_wait_warp(p_ready + 8 * h, p_phase[0], abort_flag, p.status, h == 0 ? 507 : 510);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) {
                        one_tile_products(tmem + F::kO, tmem, v_tile, idesc_o, h);
                        if (h == 1) {
                            umma_commit_cta1(o_full);
                            umma_commit_cta1(empty + 8 * kv.stage);
                        }
                    }
                    __syncwarp();
                }
                p_phase[0] ^= 1u;
                kv.next(F::kStages);
                continue;
            }
            for (int j = 0; ok && j < n; ++j) {
                const uint32_t v_tile = ring + kv.stage * F::kTileBytes;
                const uint32_t v_empty = empty + 8 * kv.stage;
                ok = mbar_wait_warp(full + 8 * kv.stage, kv.phase, abort_flag, p.status, 505);
                if (!ok) break;
                kv.next(F::kStages);
                const int valid = b.len - j * kTile;
                if (valid < kTile) {  // rows of other sequences
                    zero_tile_rows<kD>(v_tile, valid, lane);
                    fence_proxy_async();
                    __syncwarp();
                }
                const uint32_t k_tile = ring + kv.stage * F::kTileBytes;
                const uint32_t k_empty = empty + 8 * kv.stage;
                const bool more = j + 1 < n;
                if (more) ok = mbar_wait_warp(full + 8 * kv.stage, kv.phase, abort_flag, p.status, 506);
                for (int t = 0; ok && t < tiles; ++t) {
                    const int count = first + t;
                    if (j >= count) continue;
                    ok = mbar_wait_warp(p_ready + 16 * t, p_phase[t], abort_flag, p.status, 507);
                    if (!ok) break;
                    tc_fence_after();
                    if (elect_one()) mma_rows<0, 4>(tmem + F::kO + t * kD, tmem + t * kTile, 32, v_tile, idesc_o, j != 0);
                    __syncwarp();
                    ok = mbar_wait_warp(p_ready + 16 * t + 8, p_phase[t], abort_flag, p.status, 510);
                    if (!ok) break;
                    p_phase[t] ^= 1u;
                    tc_fence_after();
                    if (elect_one()) {
                        mma_rows<4, 8>(tmem + F::kO + t * kD, tmem + t * kTile, 32, v_tile, idesc_o, true);
                        if (j + 1 < count) {
                            // overwrites p, which the product just issued reads: the pipe runs them in order
                            mma_scores<kD>(tmem + t * kTile, q_tile + t * F::kTileBytes, k_tile, idesc_s, p.dim_steps);
                            umma_commit_cta1(s_full + 8 * t);
                            if (j + 2 == count) umma_commit_cta1(q_empty + 8 * t);
                        } else {
                            umma_commit_cta1(o_full + 8 * t);
                        }
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (elect_one()) {
                    umma_commit_cta1(v_empty);
                    if (more) umma_commit_cta1(k_empty);
                }
                __syncwarp();
                if (more) kv.next(F::kStages);
            }
        }
    } else if (warp >= 4) {
        regs_grow<kComputeRegs>();
        const int t = (warp >> 2) - 1;               // query tile of this group
        const int row = (warp & 3) * 32 + lane;      // its row, and the tensor-memory lane
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_addr = tmem + lanes + t * kTile, o_addr = tmem + lanes + F::kO + t * kD;
        uint32_t s_phase = 0, o_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = p.blocks[it / p.heads];
            const int head = static_cast<int>(it % p.heads);
            const int row0 = b.index * 2 * kTile;
            if (t == 1 && b.len <= row0 + kTile) continue;
            const int count = b.index * 2 + 1 + t;
            float m = -INFINITY, l = 0.f;  // running maximum (log2 units) that p refers to, and sum of p, shift and all
            const bool one_tile = b.len <= kTile;  // p in two operands
            if (one_tile) {
                ok = mbar_wait(s_full + 8 * t, s_phase, abort_flag, p.status, 508);
                if (!ok) break;
                s_phase ^= 1u;
                tc_fence_after();
                const float2 found = one_tile_probabilities<T>(s_addr, row, p.scale_log2, p_ready + 16 * t);
                m = found.x;
                l = found.y;
            }
            for (int j = one_tile ? count : 0; j < count; ++j) {
                ok = mbar_wait(s_full + 8 * t, s_phase, abort_flag, p.status, 508);
                if (!ok) break;
                s_phase ^= 1u;
                tc_fence_after();
                uint32_t s[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, s[c]);
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_tie32(s[c]);
                if (j == count - 1) {
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (c * 32 + i > row) s[c][i] = 0xff800000u;  // -inf
                }
                float top[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    top[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int i = 1; i < 32; ++i) top[c] = fmaxf(top[c], __uint_as_float(s[c][i]));
                }
                const float tile_max = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale_log2;
                if (j == 0) {
                    m = tile_max;
                } else {
                    // The sum stays exact whatever m is, as long as p does not overflow: the accumulator is
                    // touched only when a maximum grew by so much, which after the first tiles hardly happens.
                    const bool grow = tile_max - m > kRescaleLog2<T>;
                    if (__any_sync(0xffffffffu, grow)) {
                        const float factor = grow ? ex2(m - tile_max) : 1.f;
                        if (grow) m = tile_max;
                        l *= factor;
#pragma unroll
                        for (int c = 0; c < kD / 32; ++c) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + c * 32, o);
                            tmem_ld_wait();
                            tmem_tie32(o);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
                            tmem_st32(o_addr + c * 32, o);
                        }
                    }
                }
                const float neg_m = m == -INFINITY ? 0.f : kShiftLog2<T> - m;  // a row with no finite score so far
                const f32x2 scale2 = make_f32x2(p.scale_log2, p.scale_log2), neg_m2 = make_f32x2(neg_m, neg_m);
                f32x2 sum[2] = {make_f32x2(0.f, 0.f), make_f32x2(0.f, 0.f)};
#pragma unroll
                for (int h = 0; h < 2; ++h) {  // p of 64 keys at a time: their product starts while the others are computed
                    uint32_t packed[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int c = h * 2 + (i >> 4), e = (i & 15) * 2;
                        const f32x2 x = fma_f32x2(make_f32x2(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1])), scale2, neg_m2);
                        float a, d;
                        split_f32x2(x, a, d);
                        a = ex2(a);
                        d = ex2(d);
                        sum[i & 1] = add_f32x2(sum[i & 1], make_f32x2(a, d));
                        packed[i] = pack2<T>(a, d);
                    }
                    tmem_st32(s_addr + h * 32, packed);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_ready + 16 * t + 8 * h);
                }
                float part[2];
                split_f32x2(add_f32x2(sum[0], sum[1]), part[0], part[1]);
                l += part[0] + part[1];
            }
            if (!ok) break;
            ok = mbar_wait(o_full + 8 * t, o_phase, abort_flag, p.status, 509);
            if (!ok) break;
            o_phase ^= 1u;
            tc_fence_after();
            const int r = row0 + t * kTile + row, first = r - lane;
            const bool valid = r < b.len;
            store_output<T, kD>(o_addr, base + kStagingAt + (warp - 4) * F::kStaging, &map_out, &map_rest, static_cast<T*>(p.out),
                                p.rest, p.rest_row, static_cast<int64_t>(b.start) + first, min(32, b.len - first), p.heads, head, p.dim,
                                1.f / l, lane);
            if (p.lse != nullptr && valid) p.lse[head * p.pad_rows + b.pad + r] = m + (lg2(l) - (kShiftLog2<T> + kProbLog2<T>));
            tc_fence_before();
        }
    }
    if (warp >= 4 && lane == 0) bulk_wait_read<0>();  // the staging tiles stay until the last stores have read them
    tc_fence_before();
    __syncthreads();
    if (*abort_flag != 0) {
        if (threadIdx.x == 0) settle_copies(*in_flight, full, F::kStages, q_full, q_full + 8);
        if (warp == 1) settle_products(settled);
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// ---------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------

// Largest finite |x| of eight. A row that holds an infinity or a NaN is lost whatever its factor, and must not take the
// bits of other sequences' gradients with it.
template <typename T>
__device__ __forceinline__ float largest_finite(const uint32_t (&words)[4]) {
    float top = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float2 f = unpack2<T>(words[q]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));  // passes NaNs by
    }
    if (top < INFINITY) return top;
    top = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const float2 f = unpack2<T>(words[q]);
        if (fabsf(f.x) < INFINITY) top = fmaxf(top, fabsf(f.x));
        if (fabsf(f.y) < INFINITY) top = fmaxf(top, fabsf(f.y));
    }
    return top;
}
// Factor (a power of two) that ds carries while it is rounded to T. bf16 has float32's range: 1. fp16 has
// not: |ds| is at most 2 dim max|do| max|v|, and that bound is put at 2^15, just below the largest fp16, so
// that what gradients without loss scaling are made of does not fall under its smallest.
template <typename T>
__device__ __forceinline__ float ds_factor(const Params& p) { return 1.f; }
template <>
__device__ __forceinline__ float ds_factor<__half>(const Params& p) {
    const float bound = 2.f * static_cast<float>(p.dim) * __uint_as_float(p.absmax[0]) * __uint_as_float(p.absmax[1]);
    if (!(bound > 0.f)) return 1.f;
    return exp2f(static_cast<float>(min(max(14 - ilogbf(bound), -100), 100)));
}

// -delta_i = -o_i . do_i for every row of every block and head (negated: the backward kernels add it two at a
// time), o with what its rounding took away; for fp16 also
// max |do| and max |v| of the finite ones (over bit patterns, whose order does not depend on that of the atomics). A CTA takes
// kDeltaRows rows of a block of the plan; groups of kD / 8 lanes take one head of one row each, 16 bytes a lane, four at
// a time. Bound by HBM: 77 us for 16384 tokens x 32 heads of 128 (335 MB, 4.4 TB/s; smaller batches at more occupancy
// gain 5 us there and lose as much on short sequences).
constexpr int kDeltaRows = 16, kDeltaThreads = 256;
template <typename T, int kD>
__global__ void __launch_bounds__(kDeltaThreads, 3)
delta_kernel(const T* __restrict__ o, const uint8_t* __restrict__ rest, const T* __restrict__ d_o, const T* __restrict__ v, int64_t v_token, int64_t v_head,
             float* __restrict__ delta, uint32_t* absmax, const Params p) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kLanes = kD / 8, kSlots = kDeltaThreads / kLanes, kBatch = 4;
    constexpr int kParts = kTile / kDeltaRows;
    if (static_cast<int>(blockIdx.x) / kParts >= *p.num_blocks) return;
    const Block b = p.blocks[blockIdx.x / kParts];
    const int first = b.index * kTile + static_cast<int>(blockIdx.x % kParts) * kDeltaRows;  // row of the sequence
    const int rows = min(kDeltaRows, b.len - first);
    if (rows <= 0) return;
    const int sub = threadIdx.x % kLanes, slot = threadIdx.x / kLanes;
    const bool in_head = sub * 8 < p.dim;
    float most_do = 0.f, most_v = 0.f;
    const int pairs = rows * p.heads;  // (row, head) pairs lie one after another in memory
    const int64_t base = (static_cast<int64_t>(b.start) + first) * p.heads * p.dim + sub * 8;
    const int64_t rest_base = (static_cast<int64_t>(b.start) + first) * p.heads * p.rest_row + sub * 8;
    int r = slot / p.heads, h = slot - r * p.heads;  // pair i0, kept up without dividing
    for (int i0 = slot; i0 - slot < pairs; i0 += kBatch * kSlots) {  // the same trips for every thread: whole warps shuffle
        uint4 x[kBatch], y[kBatch];
        uint2 z[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + u * kSlots;
            x[u] = y[u] = make_uint4(0, 0, 0, 0);
            z[u] = make_uint2(0, 0);
            if (i < pairs && in_head) {
                z[u] = __ldg(reinterpret_cast<const uint2*>(rest + rest_base + static_cast<int64_t>(i) * p.rest_row));
                x[u] = __ldg(reinterpret_cast<const uint4*>(o + base + static_cast<int64_t>(i) * p.dim));
                y[u] = __ldg(reinterpret_cast<const uint4*>(d_o + base + static_cast<int64_t>(i) * p.dim));
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w}, yw[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float2 f = unpack2<T>(xw[q]), g = unpack2<T>(yw[q]);
                const uint32_t two = (q < 2 ? z[u].x : z[u].y) >> ((q & 1) * 16);
                const __half2_raw raw = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xffff), __NV_E5M2);
                const float2 e = __half22float2(*reinterpret_cast<const __half2*>(&raw));
                sum += fmaf(e.x, 1.f / kRestScale<T>, f.x) * g.x + fmaf(e.y, 1.f / kRestScale<T>, f.y) * g.y;
            }
            if (kHalf) most_do = fmaxf(most_do, largest_finite<T>(yw));
#pragma unroll
            for (int w = kLanes / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            if (r < rows && sub == 0) delta[h * p.pad_rows + b.pad + first + r] = -sum;
            for (h += kSlots; h >= p.heads; h -= p.heads) ++r;
        }
    }
    if (kHalf) {
        const int kv_pairs = rows * p.kv_heads;
        for (int i0 = slot; i0 < kv_pairs; i0 += kBatch * kSlots) {
            uint4 x[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kSlots;
                x[u] = make_uint4(0, 0, 0, 0);
                if (i < kv_pairs && in_head) {
                    const int vr = i / p.kv_heads, vh = i - vr * p.kv_heads;
                    x[u] = __ldg(reinterpret_cast<const uint4*>(v + (static_cast<int64_t>(b.start) + first + vr) * v_token + vh * v_head + sub * 8));
                }
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const uint32_t xw[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
                most_v = fmaxf(most_v, largest_finite<T>(xw));
            }
        }
        __shared__ uint32_t most[2];
        if (threadIdx.x < 2) most[threadIdx.x] = 0;
        __syncthreads();
        const uint32_t warp_do = __reduce_max_sync(0xffffffffu, __float_as_uint(most_do));
        const uint32_t warp_v = __reduce_max_sync(0xffffffffu, __float_as_uint(most_v));
        if ((threadIdx.x & 31) == 0) {
            atomicMax(&most[0], warp_do);
            atomicMax(&most[1], warp_v);
        }
        __syncthreads();
        // most CTAs find a larger value there already and leave the one address alone
        if (threadIdx.x < 2 && *static_cast<volatile uint32_t*>(absmax + threadIdx.x) < most[threadIdx.x])
            atomicMax(&absmax[threadIdx.x], most[threadIdx.x]);
    }
}

// Shared memory of the two backward kernels: two resident tiles, a ring of three tiles whose contents live
// through a whole step (they are operands of its first and of its last product), and a ring of two for the
// others. There is no room left for alignment slack: the kernels check that the base is aligned.
template <int kD>
struct Backward {
    static_assert(kD == 64 || kD == 128, "tile widths");
    static constexpr uint32_t kTileBytes = kTile * kD * 2;
    static constexpr int kLong = 3, kShort = 2;
    static constexpr uint32_t kStats = 2 * kTile * 4;  // lse and delta of a query tile (dkdv), beside a short-ring tile
    static constexpr uint32_t kLongAt = 2 * kTileBytes, kShortAt = kLongAt + kLong * kTileBytes;
    static constexpr uint32_t kStatsAt = kShortAt + kShort * kTileBytes;
    static constexpr uint32_t kBars = kStatsAt + kShort * kStats;
    static constexpr uint32_t kSmem = kBars + 256;
    static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ bool base_is_aligned(uint32_t base, int32_t* status) {
    if ((base & 1023u) == 0) return true;
    if (threadIdx.x == 0 && status != nullptr) atomicCAS(status, 0, 530);
    return false;
}

// p (or ds) of 32 neighbouring columns to tensor memory, as 16 packed columns.
template <typename T>
__device__ __forceinline__ void store_packed32(uint32_t taddr, const f32x2* v) {
    uint32_t packed[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        float lo, hi;
        split_f32x2(v[c], lo, hi);
        packed[c] = pack2<T>(lo, hi);
    }
    tmem_st16(taddr, packed);
}
__device__ __forceinline__ f32x2 pair(const uint32_t* r) { return make_f32x2(__uint_as_float(r[0]), __uint_as_float(r[1])); }
// 2^-x
__device__ __forceinline__ f32x2 ex2_neg2(f32x2 x) {
    float lo, hi;
    split_f32x2(x, lo, hi);
    return make_f32x2(ex2(-lo), ex2(-hi));
}
// ds = p (dp - delta), with the factor that fp16 is rounded with (and without the one that p has)
template <typename T>
__device__ __forceinline__ f32x2 ds_pair(f32x2 p, f32x2 dp, f32x2 neg_delta, f32x2 factor) {
    f32x2 d = add_f32x2(dp, neg_delta);
    if (std::is_same<T, __half>::value) d = mul_f32x2(d, factor);  // 1 for bf16
    return mul_f32x2(p, d);
}
// Of 32 columns those before `from` and from `last` on become zeros, whatever they held.
__device__ __forceinline__ void clear_outside(f32x2* v, int from, int last) {
#pragma unroll
    for (int c = 0; c < 16; ++c) {
        float lo, hi;
        split_f32x2(v[c], lo, hi);
        if (2 * c < from || 2 * c >= last) lo = 0.f;
        if (2 * c + 1 < from || 2 * c + 1 >= last) hi = 0.f;
        v[c] = make_f32x2(lo, hi);
    }
}
// Half `part` of the product over 128 rows of B whose A operand store_packed32 wrote: columns 32 part .. 32
// part + 31 of each compute group's 64.
__device__ __forceinline__ void mma_rows_part(int part, uint32_t d, uint32_t a, uint32_t b_tile, uint32_t idesc, bool accumulate) {
    const uint64_t b = desc_row_major(b_tile);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int kk = (i >> 1) * 4 + part * 2 + (i & 1);
        umma_ts_cta1(d, a + (kk >> 2) * 64 + (kk & 3) * 8, b + row_step(kk), idesc, (accumulate || part != 0 || i != 0) ? 1u : 0u);
    }
}

// Work item: 128 key rows of one key/value head, all query tiles at or after them of the group's heads.
// Tensor memory: s^T at 0, dp^T at 128, dv at 256, dk at 256 + kD. Each group of four compute warps takes 64
// of the 128 query columns; p^T (and ds^T) of a half lies at the start of that half's columns. One MMA warp
// issues dv += p^T do and the next s^T, the other dk += ds^T q and the next dp^T: each pair shares a region of
// tensor memory, and while one warp waits for the compute warps the other's products run. Query tiles are
// operands of a step's first and last product, so they need three buffers: with two, a step waited 1400 cycles for
// its tile. 16384 tokens, 32 heads on 8 of 128: 3734 us with two buffers and one MMA warp, 3300 us so
// and 3110 us with probabilities and ds computed two elements an instruction.
template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1)
dkdv_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
            const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Params p) {
    using B = Backward<kD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    if (!base_is_aligned(base, p.status)) return;
    uint8_t* gen = smem_raw;
    const uint32_t k_tile = base, v_tile = base + B::kTileBytes, q_ring = base + B::kLongAt, do_ring = base + B::kShortAt;
    const uint32_t bars = base + B::kBars;
    const uint32_t q_full = bars, q_empty = bars + 24, do_full = bars + 48, do_empty = bars + 64, k_full = bars + 80, k_empty = bars + 88,
                   s_full = bars + 96, dp_full = bars + 104, p_ready = bars + 112, ds_ready = bars + 128, done = bars + 144, v_full = bars + 168, v_empty = bars + 176;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + B::kBars + 160);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + B::kBars + 164);
    const uint32_t settled = bars + 184;  // of each MMA warp
    volatile uint32_t* in_flight = reinterpret_cast<volatile uint32_t*>(gen + B::kBars + 200);  // of each load warp

    const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < B::kLong; ++i) {
            mbar_init(q_full + 8 * i, 1);
            mbar_init(q_empty + 8 * i, 1);
        }
        for (int i = 0; i < B::kShort; ++i) {
            mbar_init(do_full + 8 * i, 1);
            mbar_init(do_empty + 8 * i, 2);  // both MMA warps; the second's commit follows the reads of the statistics
        }
        mbar_init(k_full, 1);
        mbar_init(k_empty, 1);
        mbar_init(v_full, 1);
        mbar_init(v_empty, 1);
        mbar_init(s_full, 1);
        mbar_init(dp_full, 1);
        for (int h = 0; h < 2; ++h) {
            mbar_init(p_ready + 8 * h, 8);
            mbar_init(ds_ready + 8 * h, 8);
        }
        mbar_init(done, 2);
        for (int i = 0; i < 2; ++i) mbar_init(settled + 8 * i, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
        prefetch_tmap(&map_do);
    }
    if (warp == 1) {
        tmem_alloc(bars + 164, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    const uint32_t tm_s = tmem, tm_dp = tmem + kTile, tm_dv = tmem + 2 * kTile, tm_dk = tm_dv + kD;
    const int64_t items = static_cast<int64_t>(warp_uniform(*p.num_blocks)) * p.kv_heads;

    if (warp == 0) {
        // k and the query tiles
        if (lane == 0) {
            Ring q;
            uint32_t k_phase = 1u;
            bool ok = true;
            for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
                const Block b = p.blocks[it / p.kv_heads];
                const int kv_head = static_cast<int>(it % p.kv_heads);
                const int n = (b.len + kTile - 1) / kTile;
                ok = mbar_wait(k_empty, k_phase, abort_flag, p.status, 511);
                if (!ok) break;
                k_phase ^= 1u;
                mbar_expect_tx(k_full, B::kTileBytes);
                load_tile<kD>(k_tile, &map_k, k_full, kv_head, b.start + b.index * kTile);
                for (int g = 0; ok && g < p.group; ++g) {
                    for (int i = b.index; ok && i < n; ++i) {
                        ok = mbar_wait(q_empty + 8 * q.stage, q.phase ^ 1u, abort_flag, p.status, 512);
                        if (!ok) break;
                        mbar_expect_tx(q_full + 8 * q.stage, B::kTileBytes);
                        load_tile<kD>(q_ring + q.stage * B::kTileBytes, &map_q, q_full + 8 * q.stage, kv_head * p.group + g,
                                      b.start + i * kTile);
                        q.next(B::kLong);
                    }
                }
            }
            in_flight[0] = pack_in_flight(q, k_phase, k_phase);
        }
        __syncwarp();
    } else if (warp == 3) {
        // v, and do tiles with the rows' statistics
        if (lane == 0) {
            Ring d;
            uint32_t v_phase = 1u;
            bool ok = true;
            for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
                const Block b = p.blocks[it / p.kv_heads];
                const int kv_head = static_cast<int>(it % p.kv_heads);
                const int n = (b.len + kTile - 1) / kTile;
                ok = mbar_wait(v_empty, v_phase, abort_flag, p.status, 529);
                if (!ok) break;
                v_phase ^= 1u;
                mbar_expect_tx(v_full, B::kTileBytes);
                load_tile<kD>(v_tile, &map_v, v_full, kv_head, b.start + b.index * kTile);
                for (int g = 0; ok && g < p.group; ++g) {
                    const int head = kv_head * p.group + g;
                    for (int i = b.index; ok && i < n; ++i) {
                        ok = mbar_wait(do_empty + 8 * d.stage, d.phase ^ 1u, abort_flag, p.status, 531);
                        if (!ok) break;
                        const uint32_t bar = do_full + 8 * d.stage;
                        mbar_expect_tx(bar, B::kTileBytes + B::kStats);
                        load_tile<kD>(do_ring + d.stage * B::kTileBytes, &map_do, bar, head, b.start + i * kTile);
                        const int64_t at = head * p.pad_rows + b.pad + i * kTile;
                        const uint32_t stats = base + B::kStatsAt + d.stage * B::kStats;
                        bulk_load(stats, p.lse + at, kTile * 4, bar);
                        bulk_load(stats + kTile * 4, p.delta + at, kTile * 4, bar);
                        d.next(B::kShort);
                    }
                }
            }
            in_flight[1] = pack_in_flight(d, v_phase, v_phase);
        }
        __syncwarp();
    } else if (warp == 1) {
        // s^T = k q^T, dv += p^T do
        const uint32_t idesc_s = make_idesc(kTile, kTile, false, false, p.ab_format);
        const uint32_t idesc_d = make_idesc(kTile, p.dim_steps * 16, false, true, p.ab_format);
        Ring q, d;
        uint32_t k_phase = 0, p_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = load_block(p.blocks + it / p.kv_heads);
            const int n = (b.len + kTile - 1) / kTile;
            const int per_head = n - b.index, steps = per_head * p.group;
            ok = mbar_wait_warp(k_full, k_phase, abort_flag, p.status, 513);
            if (!ok) break;
            k_phase ^= 1u;
            ok = mbar_wait_warp(q_full + 8 * q.stage, q.phase, abort_flag, p.status, 514);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                mma_scores<kD>(tm_s, k_tile, q_ring + q.stage * B::kTileBytes, idesc_s, p.dim_steps);
                umma_commit_cta1(s_full);
                if (steps == 1) umma_commit_cta1(k_empty);
            }
            __syncwarp();
            q.next(B::kLong);
            int i = b.index;
            for (int st = 0; st < steps; ++st) {
                const bool more = st + 1 < steps;
                const uint32_t do_tile = do_ring + d.stage * B::kTileBytes, next_q = q_ring + q.stage * B::kTileBytes;
                ok = mbar_wait_warp(do_full + 8 * d.stage, d.phase, abort_flag, p.status, 532);
                if (ok && more) ok = mbar_wait_warp(q_full + 8 * q.stage, q.phase, abort_flag, p.status, 533);
                if (!ok) break;
                const int valid = b.len - i * kTile;
                if (valid < kTile) {  // rows of other sequences, which p = 0 would meet
                    zero_tile_rows<kD>(do_tile, valid, lane);
                    fence_proxy_async();
                    __syncwarp();
                }
                i = i + 1 < n ? i + 1 : b.index;
                ok = mbar_wait_warp(p_ready, p_phase, abort_flag, p.status, 515);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) mma_rows_part(0, tm_dv, tm_s, do_tile, idesc_d, st > 0);
                __syncwarp();
                ok = mbar_wait_warp(p_ready + 8, p_phase, abort_flag, p.status, 534);
                if (!ok) break;
                p_phase ^= 1u;
                tc_fence_after();
                if (elect_one()) {
                    mma_rows_part(1, tm_dv, tm_s, do_tile, idesc_d, true);
                    if (more) {
                        mma_scores<kD>(tm_s, k_tile, next_q, idesc_s, p.dim_steps);
                        umma_commit_cta1(s_full);
                        if (st + 2 == steps) umma_commit_cta1(k_empty);
                    } else {
                        umma_commit_cta1(done);
                    }
                    umma_commit_cta1(do_empty + 8 * d.stage);
                }
                __syncwarp();
                d.next(B::kShort);
                if (more) q.next(B::kLong);
            }
        }
    } else if (warp == 2) {
        // dp^T = v do^T, dk += ds^T q
        const uint32_t idesc_s = make_idesc(kTile, kTile, false, false, p.ab_format);
        const uint32_t idesc_d = make_idesc(kTile, p.dim_steps * 16, false, true, p.ab_format);
        Ring q, d;
        uint32_t v_phase = 0, ds_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = load_block(p.blocks + it / p.kv_heads);
            const int n = (b.len + kTile - 1) / kTile;
            const int per_head = n - b.index, steps = per_head * p.group;
            ok = mbar_wait_warp(v_full, v_phase, abort_flag, p.status, 535);
            if (!ok) break;
            v_phase ^= 1u;
            ok = mbar_wait_warp(do_full + 8 * d.stage, d.phase, abort_flag, p.status, 536);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                mma_scores<kD>(tm_dp, v_tile, do_ring + d.stage * B::kTileBytes, idesc_s, p.dim_steps);
                umma_commit_cta1(dp_full);
                if (steps == 1) umma_commit_cta1(v_empty);
            }
            __syncwarp();
            int i = b.index;
            for (int st = 0; st < steps; ++st) {
                const bool more = st + 1 < steps;
                const uint32_t q_tile = q_ring + q.stage * B::kTileBytes;
                const uint32_t this_empty = do_empty + 8 * d.stage;
                d.next(B::kShort);
                const uint32_t next_do = do_ring + d.stage * B::kTileBytes;
                ok = mbar_wait_warp(q_full + 8 * q.stage, q.phase, abort_flag, p.status, 537);
                if (ok && more) ok = mbar_wait_warp(do_full + 8 * d.stage, d.phase, abort_flag, p.status, 538);
                if (!ok) break;
                ok = mbar_wait_warp(ds_ready, ds_phase, abort_flag, p.status, 516);
                if (!ok) break;
                const int valid = b.len - i * kTile;
                if (valid < kTile) {  // rows of other sequences, which ds = 0 would meet; s^T has read the tile by now
                    zero_tile_rows<kD>(q_tile, valid, lane);
                    fence_proxy_async();
                    __syncwarp();
                }
                i = i + 1 < n ? i + 1 : b.index;
                tc_fence_after();
                if (elect_one()) mma_rows_part(0, tm_dk, tm_dp, q_tile, idesc_d, st > 0);
                __syncwarp();
                ok = mbar_wait_warp(ds_ready + 8, ds_phase, abort_flag, p.status, 539);
                if (!ok) break;
                ds_phase ^= 1u;
                tc_fence_after();
                if (elect_one()) {
                    mma_rows_part(1, tm_dk, tm_dp, q_tile, idesc_d, true);
                    umma_commit_cta1(q_empty + 8 * q.stage);
                    umma_commit_cta1(this_empty);
                    if (more) {
                        mma_scores<kD>(tm_dp, v_tile, next_do, idesc_s, p.dim_steps);
                        umma_commit_cta1(dp_full);
                        if (st + 2 == steps) umma_commit_cta1(v_empty);
                    } else {
                        umma_commit_cta1(done);
                    }
                }
                __syncwarp();
                q.next(B::kLong);
            }
        }
    } else {
        const int half = (warp >> 2) - 1;          // query columns 64 half .. 64 half + 63
        const int row = (warp & 3) * 32 + lane;    // key row
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_addr = tm_s + lanes + half * 64, dp_addr = tm_dp + lanes + half * 64;
        const float factor = ds_factor<T>(p);
        const f32x2 factor2 = make_f32x2(factor * kProbInverse<T>, factor * kProbInverse<T>), neg_scale2 = make_f32x2(-p.scale_log2, -p.scale_log2);
        Ring d;
        uint32_t s_phase = 0, dp_phase = 0, done_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = p.blocks[it / p.kv_heads];
            const int kv_head = static_cast<int>(it % p.kv_heads);
            const int n = (b.len + kTile - 1) / kTile;
            for (int g = 0; ok && g < p.group; ++g) {
                for (int i = b.index; ok && i < n; ++i) {
                    ok = mbar_wait(do_full + 8 * d.stage, d.phase, abort_flag, p.status, 517);
                    if (!ok) break;
                    const float4* lse = reinterpret_cast<const float4*>(gen + B::kStatsAt + d.stage * B::kStats + half * 256);
                    const float4* neg_delta = lse + kTile / 4;
                    ok = mbar_wait(s_full, s_phase, abort_flag, p.status, 518);
                    if (!ok) break;
                    s_phase ^= 1u;
                    tc_fence_after();
                    const int last = b.len - i * kTile - half * 64;        // columns from here on are no queries
                    const int from = i == b.index ? row - half * 64 : 0;   // columns before are not causal
                    const bool edge = last < 64 || i == b.index;
                    // probabilities, two at a time; x = lse - scale s, so that no sign takes an instruction
                    f32x2 pr[32];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t s[32];
                        tmem_ld32(s_addr + c * 32, s);
                        tmem_ld_wait();
                        tmem_tie32(s);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float4 f = lse[c * 8 + e];
                            pr[c * 16 + e * 2] = ex2_neg2(fma_f32x2(pair(s + e * 4), neg_scale2, make_f32x2(f.x, f.y)));
                            pr[c * 16 + e * 2 + 1] = ex2_neg2(fma_f32x2(pair(s + e * 4 + 2), neg_scale2, make_f32x2(f.z, f.w)));
                        }
                        if (edge) clear_outside(pr + c * 16, from - c * 32, last - c * 32);
                        store_packed32<T>(s_addr + c * 16, pr + c * 16);
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready + 8 * c);
                    }

                    ok = mbar_wait(dp_full, dp_phase, abort_flag, p.status, 519);
                    if (!ok) break;
                    dp_phase ^= 1u;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t dp[32];
                        tmem_ld32(dp_addr + c * 32, dp);
                        tmem_ld_wait();
                        tmem_tie32(dp);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float4 f = neg_delta[c * 8 + e];
                            pr[c * 16 + e * 2] = ds_pair<T>(pr[c * 16 + e * 2], pair(dp + e * 4), make_f32x2(f.x, f.y), factor2);
                            pr[c * 16 + e * 2 + 1] = ds_pair<T>(pr[c * 16 + e * 2 + 1], pair(dp + e * 4 + 2), make_f32x2(f.z, f.w), factor2);
                        }
                        // delta of a column outside is no number to rely on; a sequence's first query has one key, whose
                        // score has no gradient: dp - delta would leave a rounding there
                        if (edge) clear_outside(pr + c * 16, (i == 0 && half == 0 ? max(from, 1) : from) - c * 32, last - c * 32);
                        store_packed32<T>(dp_addr + c * 16, pr + c * 16);
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(ds_ready + 8 * c);
                    }
                    d.next(B::kShort);
                }
            }
            if (!ok) break;
            ok = mbar_wait(done, done_phase, abort_flag, p.status, 520);
            if (!ok) break;
            done_phase ^= 1u;
            tc_fence_after();
            const int key = b.index * kTile + row;
            const int64_t at = (static_cast<int64_t>(b.start + key) * p.kv_heads + kv_head) * p.dim;
            if (half == 0) store_row<T, kD>(tm_dv + lanes, static_cast<T*>(p.dv) + at, p.dim, kProbInverse<T>, key < b.len);
            else store_row<T, kD>(tm_dk + lanes, static_cast<T*>(p.dk) + at, p.dim, p.scale / factor, key < b.len);
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag != 0) {
        if (threadIdx.x == 0) settle_copies(in_flight[0], q_full, B::kLong, k_full, k_full);
        if (threadIdx.x == 96) settle_copies(in_flight[1], do_full, B::kShort, v_full, v_full);
        if (warp == 1 || warp == 2) settle_products(settled + 8 * (warp - 1));
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// Work item: 128 query rows of one head over their key tiles. Tensor memory: s at 0 and 128 (two buffers),
// dp (then ds) at 256, dq at 384. The compute groups take 64 key columns each. One MMA warp issues s ahead, the
// other dq += ds k and the next dp. Bound by the compute warps' chain (exponentials, then ds) beside three products
// of 512 cycles: some 2500 cycles a tile (2970 -> 2800 us at 16384 tokens with two elements an instruction). The groups
// a tile apart, three buffers between them, are no faster: the key tiles that fit, which stay from s to dq, run out.
template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1)
dq_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
          const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_do, const Params p) {
    using B = Backward<kD>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t base = smem_u32(smem_raw);
    if (!base_is_aligned(base, p.status)) return;
    uint8_t* gen = smem_raw;
    const uint32_t q_tile = base, do_tile = base + B::kTileBytes, k_ring = base + B::kLongAt, v_ring = base + B::kShortAt;
    const uint32_t bars = base + B::kBars;
    const uint32_t k_full = bars, k_empty = bars + 24, v_full = bars + 48, v_empty = bars + 64, q_full = bars + 80, q_empty = bars + 88,
                   s_full = bars + 96, s_free = bars + 112, dp_full = bars + 128, ds_ready = bars + 136, done = bars + 152, do_full = bars + 168, do_empty = bars + 176;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen + B::kBars + 160);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + B::kBars + 164);
    const uint32_t settled = bars + 184;  // of each MMA warp
    volatile uint32_t* in_flight = reinterpret_cast<volatile uint32_t*>(gen + B::kBars + 200);  // of each load warp

    const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < B::kLong; ++i) {
            mbar_init(k_full + 8 * i, 1);
            mbar_init(k_empty + 8 * i, 1);
        }
        for (int i = 0; i < B::kShort; ++i) {
            mbar_init(v_full + 8 * i, 1);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(s_free + 8 * i, 8);
            mbar_init(ds_ready + 8 * i, 8);
        }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_init(do_full, 1);
        mbar_init(do_empty, 1);
        mbar_init(dp_full, 1);
        mbar_init(done, 1);
        for (int i = 0; i < 2; ++i) mbar_init(settled + 8 * i, 1);
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tmap(&map_q);
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
        prefetch_tmap(&map_do);
    }
    if (warp == 1) {
        tmem_alloc(bars + 164, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    const uint32_t tm_dp = tmem + 2 * kTile, tm_dq = tmem + 3 * kTile;
    const int64_t items = static_cast<int64_t>(warp_uniform(*p.num_blocks)) * p.heads;

    if (warp == 0) {
        // q and the key tiles
        if (lane == 0) {
            Ring k;
            uint32_t q_phase = 1u;
            bool ok = true;
            for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
                const Block b = p.blocks[it / p.heads];
                const int head = static_cast<int>(it % p.heads), kv_head = head / p.group;
                ok = mbar_wait(q_empty, q_phase, abort_flag, p.status, 521);
                if (!ok) break;
                q_phase ^= 1u;
                mbar_expect_tx(q_full, B::kTileBytes);
                load_tile<kD>(q_tile, &map_q, q_full, head, b.start + b.index * kTile);
                for (int j = 0; ok && j <= b.index; ++j) {
                    ok = mbar_wait(k_empty + 8 * k.stage, k.phase ^ 1u, abort_flag, p.status, 522);
                    if (!ok) break;
                    mbar_expect_tx(k_full + 8 * k.stage, B::kTileBytes);
                    load_tile<kD>(k_ring + k.stage * B::kTileBytes, &map_k, k_full + 8 * k.stage, kv_head, b.start + j * kTile);
                    k.next(B::kLong);
                }
            }
            in_flight[0] = pack_in_flight(k, q_phase, q_phase);
        }
        __syncwarp();
    } else if (warp == 3) {
        // do and the value tiles
        if (lane == 0) {
            Ring v;
            uint32_t do_phase = 1u;
            bool ok = true;
            for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
                const Block b = p.blocks[it / p.heads];
                const int head = static_cast<int>(it % p.heads), kv_head = head / p.group;
                ok = mbar_wait(do_empty, do_phase, abort_flag, p.status, 548);
                if (!ok) break;
                do_phase ^= 1u;
                mbar_expect_tx(do_full, B::kTileBytes);
                load_tile<kD>(do_tile, &map_do, do_full, head, b.start + b.index * kTile);
                for (int j = 0; ok && j <= b.index; ++j) {
                    ok = mbar_wait(v_empty + 8 * v.stage, v.phase ^ 1u, abort_flag, p.status, 541);
                    if (!ok) break;
                    mbar_expect_tx(v_full + 8 * v.stage, B::kTileBytes);
                    load_tile<kD>(v_ring + v.stage * B::kTileBytes, &map_v, v_full + 8 * v.stage, kv_head, b.start + j * kTile);
                    v.next(B::kShort);
                }
            }
            in_flight[1] = pack_in_flight(v, do_phase, do_phase);
        }
        __syncwarp();
    } else if (warp == 1) {
        // s = q k^T, up to two tiles ahead of what the compute warps have read
        const uint32_t idesc_s = make_idesc(kTile, kTile, false, false, p.ab_format);
        Ring k, buf;
        uint32_t q_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = load_block(p.blocks + it / p.heads);
            ok = mbar_wait_warp(q_full, q_phase, abort_flag, p.status, 523);
            if (!ok) break;
            q_phase ^= 1u;
            for (int j = 0; j <= b.index; ++j) {
                ok = mbar_wait_warp(k_full + 8 * k.stage, k.phase, abort_flag, p.status, 524);
                if (ok) ok = mbar_wait_warp(s_free + 8 * buf.stage, buf.phase ^ 1u, abort_flag, p.status, 542);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    mma_scores<kD>(tmem + buf.stage * kTile, q_tile, k_ring + k.stage * B::kTileBytes, idesc_s, p.dim_steps);
                    umma_commit_cta1(s_full + 8 * buf.stage);
                    if (j == b.index) umma_commit_cta1(q_empty);
                }
                __syncwarp();
                k.next(B::kLong);
                buf.next(2);
            }
        }
    } else if (warp == 2) {
        // dp = do v^T, dq += ds k
        const uint32_t idesc_s = make_idesc(kTile, kTile, false, false, p.ab_format);
        const uint32_t idesc_d = make_idesc(kTile, p.dim_steps * 16, false, true, p.ab_format);
        Ring k, v;
        uint32_t do_phase = 0, ds_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = load_block(p.blocks + it / p.heads);
            ok = mbar_wait_warp(do_full, do_phase, abort_flag, p.status, 543);
            if (ok) ok = mbar_wait_warp(v_full + 8 * v.stage, v.phase, abort_flag, p.status, 544);
            if (!ok) break;
            do_phase ^= 1u;
            tc_fence_after();
            if (elect_one()) {
                mma_scores<kD>(tm_dp, do_tile, v_ring + v.stage * B::kTileBytes, idesc_s, p.dim_steps);
                umma_commit_cta1(dp_full);
                umma_commit_cta1(v_empty + 8 * v.stage);
                if (b.index == 0) umma_commit_cta1(do_empty);
            }
            __syncwarp();
            v.next(B::kShort);
            for (int j = 0; j <= b.index; ++j) {
                const bool more = j < b.index;
                const uint32_t k_tile = k_ring + k.stage * B::kTileBytes;
                ok = mbar_wait_warp(k_full + 8 * k.stage, k.phase, abort_flag, p.status, 545);
                if (ok && more) ok = mbar_wait_warp(v_full + 8 * v.stage, v.phase, abort_flag, p.status, 546);
                if (ok) ok = mbar_wait_warp(ds_ready, ds_phase, abort_flag, p.status, 525);
                if (!ok) break;
                const int valid = b.len - j * kTile;
                if (valid < kTile) {  // rows of other sequences, which ds = 0 would meet; s has read the tile by now
                    zero_tile_rows<kD>(k_tile, valid, lane);
                    fence_proxy_async();
                    __syncwarp();
                }
                tc_fence_after();
                if (elect_one()) mma_rows_part(0, tm_dq, tm_dp, k_tile, idesc_d, j > 0);
                __syncwarp();
                ok = mbar_wait_warp(ds_ready + 8, ds_phase, abort_flag, p.status, 547);
                if (!ok) break;
                ds_phase ^= 1u;
                tc_fence_after();
                if (elect_one()) {
                    mma_rows_part(1, tm_dq, tm_dp, k_tile, idesc_d, true);
                    umma_commit_cta1(k_empty + 8 * k.stage);
                    if (more) {
                        mma_scores<kD>(tm_dp, do_tile, v_ring + v.stage * B::kTileBytes, idesc_s, p.dim_steps);
                        umma_commit_cta1(dp_full);
                        umma_commit_cta1(v_empty + 8 * v.stage);
                        if (j + 1 == b.index) umma_commit_cta1(do_empty);
                    } else {
                        umma_commit_cta1(done);
                    }
                }
                __syncwarp();
                k.next(B::kLong);
                if (more) v.next(B::kShort);
            }
        }
    } else {
        const int half = (warp >> 2) - 1;          // key columns 64 half .. 64 half + 63
        const int row = (warp & 3) * 32 + lane;    // query row
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t dp_addr = tm_dp + lanes + half * 64;
        const float factor = ds_factor<T>(p);
        const f32x2 factor2 = make_f32x2(factor * kProbInverse<T>, factor * kProbInverse<T>), neg_scale2 = make_f32x2(-p.scale_log2, -p.scale_log2);
        Ring buf;
        uint32_t dp_phase = 0, done_phase = 0;
        bool ok = true;
        for (int64_t turn = 0, it; ok && (it = work_item(turn)) < items; ++turn) {
            const Block b = p.blocks[it / p.heads];
            const int head = static_cast<int>(it % p.heads);
            const int query = b.index * kTile + row;
            const bool valid = query < b.len;
            const int64_t stat = head * p.pad_rows + b.pad + query;
            const float lse = valid ? p.lse[stat] : 0.f, minus = valid ? p.delta[stat] : 0.f;
            const f32x2 lse2 = make_f32x2(lse, lse), neg_delta = make_f32x2(minus, minus);
            for (int j = 0; j <= b.index; ++j) {
                ok = mbar_wait(s_full + 8 * buf.stage, buf.phase, abort_flag, p.status, 526);
                if (!ok) break;
                tc_fence_after();
                const uint32_t s_addr = tmem + lanes + buf.stage * kTile + half * 64;
                uint32_t s[2][32];
                tmem_ld32(s_addr, s[0]);
                tmem_ld32(s_addr + 32, s[1]);
                tmem_ld_wait();
                tmem_tie32(s[0]);
                tmem_tie32(s[1]);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free + 8 * buf.stage);
                buf.next(2);
                f32x2 pr[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) pr[c] = ex2_neg2(fma_f32x2(pair(s[c >> 4] + (c & 15) * 2), neg_scale2, lse2));
                ok = mbar_wait(dp_full, dp_phase, abort_flag, p.status, 527);
                if (!ok) break;
                dp_phase ^= 1u;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t dp[32];
                    tmem_ld32(dp_addr + c * 32, dp);
                    tmem_ld_wait();
                    tmem_tie32(dp);
#pragma unroll
                    for (int i = 0; i < 16; ++i) pr[c * 16 + i] = ds_pair<T>(pr[c * 16 + i], pair(dp + i * 2), neg_delta, factor2);
                    // a sequence's first query has one key, whose score has no gradient
                    if (j == b.index) clear_outside(pr + c * 16, 0, (query == 0 ? 0 : row + 1) - half * 64 - c * 32);
                    store_packed32<T>(dp_addr + c * 16, pr + c * 16);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(ds_ready + 8 * c);
                }
            }
            if (!ok) break;
            ok = mbar_wait(done, done_phase, abort_flag, p.status, 528);
            if (!ok) break;
            done_phase ^= 1u;
            tc_fence_after();
            if (half == 0) {
                T* dst = static_cast<T*>(p.dq) + (static_cast<int64_t>(b.start + query) * p.heads + head) * p.dim;
                store_row<T, kD>(tm_dq + lanes, dst, p.dim, p.scale / factor, valid);
            }
            tc_fence_before();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*abort_flag != 0) {
        if (threadIdx.x == 0) settle_copies(in_flight[0], k_full, B::kLong, q_full, q_full);
        if (threadIdx.x == 96) settle_copies(in_flight[1], v_full, B::kShort, do_full, do_full);
        if (warp == 1 || warp == 2) settle_products(settled + 8 * (warp - 1));
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

// A load role that gives up: copies go through a ring and nobody reads them; what is in flight is settled by the ring's own
// arithmetic. result[0] says that it landed, result[1] that a copy which never started did not (after limit_ns).
constexpr int kSelfTestStages = 3, kSelfTestBytes = 8192;
__global__ void __launch_bounds__(256) settle_selftest_kernel(const uint8_t* src, int fills, uint8_t* dst, int32_t* result, uint64_t limit_ns) {
    __shared__ __align__(128) uint8_t tiles[kSelfTestStages * kSelfTestBytes];
    __shared__ __align__(8) uint64_t bars[kSelfTestStages + 1];
    const uint32_t full = smem_u32(bars);
    if (threadIdx.x == 0) {
        for (int i = 0; i <= kSelfTestStages; ++i) mbar_init(full + 8 * i, 1);
        fence_barrier_init();
        Ring ring;
        for (int i = 0; i < fills; ++i) {
            const uint32_t bar = full + 8 * ring.stage;
            if (!mbar_settle(bar, ring.phase ^ 1u, global_timer_ns(), limit_ns)) break;  // the stage's last copy, in the place of a reader
            mbar_expect_tx(bar, kSelfTestBytes);
            bulk_load(smem_u32(tiles) + ring.stage * kSelfTestBytes, src + static_cast<int64_t>(i) * kSelfTestBytes, kSelfTestBytes, bar);
            ring.next(kSelfTestStages);
        }
        result[0] = ring.settle(full, kSelfTestStages, global_timer_ns(), limit_ns);
        result[1] = mbar_settle(full + 8 * kSelfTestStages, 0, global_timer_ns(), limit_ns);
    }
    __syncthreads();
    const int bytes = min(fills, kSelfTestStages) * kSelfTestBytes;
    for (int i = threadIdx.x; i < bytes; i += blockDim.x) dst[i] = tiles[i];
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// [tokens, heads, dim] with token and head strides in elements; boxes of `rows` tokens x `cols` columns of a head.
static bool stream_map(CUtensorMap* map, int dtype, const void* base, int64_t total, int heads, int dim, int64_t token_stride,
                       int64_t head_stride, int rows = kTile, int cols = 64) {
    const uint64_t size = dtype == kDtypeU8 ? 1 : 2;
    const uint64_t dims[3] = {static_cast<uint64_t>(dim), static_cast<uint64_t>(heads), static_cast<uint64_t>(total)};
    const uint64_t strides[2] = {static_cast<uint64_t>(head_stride) * size, static_cast<uint64_t>(token_stride) * size};
    const uint32_t box[3] = {static_cast<uint32_t>(cols), 1, static_cast<uint32_t>(rows)};
    return make_tmap(map, dtype, base, 3, dims, strides, box);
}

static int64_t list_capacity(int64_t total, int64_t batch, int block_rows) { return total / block_rows + batch; }

struct Workspace {  // counts and maxima, then up to two lists
    int32_t* counts;
    uint32_t* absmax;
    Block* list0;
    Block* list1;
};
static Workspace split_workspace(void* base, int64_t total, int64_t batch) {
    Workspace w;
    w.counts = static_cast<int32_t*>(base);
    w.absmax = reinterpret_cast<uint32_t*>(w.counts + 2);
    w.list0 = reinterpret_cast<Block*>(w.counts + 4);
    w.list1 = w.list0 + list_capacity(total, batch, kTile);
    return w;
}

static int launch_plan(const void* cu, int cu_is_int64, int64_t batch, int64_t total, int block_rows, const Workspace& w, int lists,
                       ZeroRows z0, ZeroRows z1, ZeroRows z2, cudaStream_t stream) {
    constexpr int kZeroBlocks = 32;
    uint32_t* absmax = lists == 2 ? w.absmax : nullptr;
    if (cu_is_int64)
        plan_kernel<int64_t><<<lists + kZeroBlocks, kPlanThreads, 0, stream>>>(
            static_cast<const int64_t*>(cu), batch, total, block_rows, w.list0, w.counts, w.list1, w.counts + 1, absmax, z0, z1, z2, lists);
    else
        plan_kernel<int32_t><<<lists + kZeroBlocks, kPlanThreads, 0, stream>>>(
            static_cast<const int32_t*>(cu), batch, total, block_rows, w.list0, w.counts, w.list1, w.counts + 1, absmax, z0, z1, z2, lists);
    return launch_status();
}

struct Call {
    const void *q, *k, *v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head;
    int dtype;
    const void* cu;
    int cu_is_int64;
    int64_t batch, total;
    int heads, kv_heads, dim;
    float scale;
    void* workspace;
    int32_t* status;
    cudaStream_t stream;
};

static int check_call(const Call& c) {
    if (c.dtype != kDtypeBF16 && c.dtype != kDtypeF16) return XMA_ERR_UNSUPPORTED;
    if (c.batch < 0 || c.total < 0 || c.heads <= 0 || c.kv_heads <= 0 || c.dim <= 0) return XMA_ERR_BAD_ARG;
    if (c.dim % 8 != 0 || c.dim > 128 || c.heads % c.kv_heads != 0 || c.heads > kMaxHeads) return XMA_ERR_UNSUPPORTED;
    if (c.total > (int64_t(1) << 30) || c.batch > (int64_t(1) << 20)) return XMA_ERR_UNSUPPORTED;
    if (!(c.scale > 0.f) || !(c.scale <= 2.3e38f)) return XMA_ERR_BAD_ARG;  // its product with log2(e) is a number too
    if (c.total == 0) return XMA_OK;
    if (!c.q || !c.k || !c.v || !c.cu || !c.workspace) return XMA_ERR_BAD_ARG;
    if (!aligned16(c.q) || !aligned16(c.k) || !aligned16(c.v) || !aligned16(c.workspace)) return XMA_ERR_BAD_ARG;
    const int64_t strides[6] = {c.q_token, c.q_head, c.k_token, c.k_head, c.v_token, c.v_head};
    for (int i = 0; i < 6; ++i)
        if (strides[i] <= 0 || strides[i] % 8 != 0 || strides[i] >= (int64_t(1) << 39)) return XMA_ERR_BAD_ARG;
    return XMA_OK;
}

static Params common_params(const Call& c) {
    Params p{};
    p.heads = c.heads, p.kv_heads = c.kv_heads, p.group = c.heads / c.kv_heads, p.dim = c.dim;
    p.dim_steps = static_cast<int>(ceil_div(c.dim, 16));
    p.rest_row = ceil_div(c.dim, 16) * 16;
    p.pad_rows = (c.total / kTile + c.batch + 1) * kTile;
    p.scale = c.scale;
    p.scale_log2 = c.scale * 1.4426950408889634f;  // log2(e): exp(scale s) = 2^(scale_log2 s)
    p.status = c.status;
    p.ab_format = c.dtype == kDtypeBF16 ? 1 : 0;
    return p;
}

static unsigned grid_for(int64_t items) {
    const int64_t sms = sm_count();
    return static_cast<unsigned>(items < sms ? (items < 1 ? 1 : items) : sms);
}

template <typename T, int kD>
static int run_forward(const Call& c, void* out, float* lse, uint8_t* rest) {
    CUtensorMap mq, mk, mv;
    if (!stream_map(&mq, c.dtype, c.q, c.total, c.heads, c.dim, c.q_token, c.q_head) ||
        !stream_map(&mk, c.dtype, c.k, c.total, c.kv_heads, c.dim, c.k_token, c.k_head) ||
        !stream_map(&mv, c.dtype, c.v, c.total, c.kv_heads, c.dim, c.v_token, c.v_head))
        return XMA_ERR_DRIVER;
    if (!allow_smem<forward_kernel<T, kD>>(Forward<kD>::kSmem)) return XMA_ERR_LAUNCH;
    const Workspace w = split_workspace(c.workspace, c.total, c.batch);
    const ZeroRows zo{out, static_cast<int64_t>(c.heads) * c.dim * 2}, none{nullptr, 0};
    const int status = launch_plan(c.cu, c.cu_is_int64, c.batch, c.total, 2 * kTile, w, 1, zo, none, none, c.stream);
    if (status != XMA_OK) return status;
    Params p = common_params(c);
    p.blocks = w.list0, p.num_blocks = w.counts, p.out = out, p.lse = lse, p.rest = rest;
    CUtensorMap mo, mr = mq;
    if (!stream_map(&mo, c.dtype, out, c.total, c.heads, c.dim, static_cast<int64_t>(c.heads) * c.dim, c.dim, 32)) return XMA_ERR_DRIVER;
    if (rest != nullptr && !stream_map(&mr, kDtypeU8, rest, c.total, c.heads, static_cast<int>(p.rest_row), c.heads * p.rest_row, p.rest_row, 32, 128))
        return XMA_ERR_DRIVER;
    const unsigned grid = grid_for(list_capacity(c.total, c.batch, 2 * kTile) * c.heads);
    forward_kernel<T, kD><<<grid, kThreads, Forward<kD>::kSmem, c.stream>>>(mq, mk, mv, mo, mr, p);
    return launch_status();
}

template <typename T, int kD>
static int run_backward(const Call& c, const void* out, const uint8_t* rest, const void* d_out, const float* lse, float* delta, void* dq, void* dk, void* dv) {
    CUtensorMap mq, mk, mv, mdo;
    const int64_t o_token = static_cast<int64_t>(c.heads) * c.dim;
    if (!stream_map(&mq, c.dtype, c.q, c.total, c.heads, c.dim, c.q_token, c.q_head) ||
        !stream_map(&mk, c.dtype, c.k, c.total, c.kv_heads, c.dim, c.k_token, c.k_head) ||
        !stream_map(&mv, c.dtype, c.v, c.total, c.kv_heads, c.dim, c.v_token, c.v_head) ||
        !stream_map(&mdo, c.dtype, d_out, c.total, c.heads, c.dim, o_token, c.dim))
        return XMA_ERR_DRIVER;
    if (!allow_smem<dkdv_kernel<T, kD>>(Backward<kD>::kSmem) || !allow_smem<dq_kernel<T, kD>>(Backward<kD>::kSmem))
        return XMA_ERR_LAUNCH;
    const Workspace w = split_workspace(c.workspace, c.total, c.batch);
    const int64_t row_q = o_token * 2, row_kv = static_cast<int64_t>(c.kv_heads) * c.dim * 2;
    int status = launch_plan(c.cu, c.cu_is_int64, c.batch, c.total, kTile, w, 2, ZeroRows{dq, row_q}, ZeroRows{dk, row_kv},
                             ZeroRows{dv, row_kv}, c.stream);
    if (status != XMA_OK || c.batch == 0) return status;
    Params p = common_params(c);
    p.lse = const_cast<float*>(lse), p.delta = delta, p.dq = dq, p.dk = dk, p.dv = dv, p.absmax = w.absmax;
    const int64_t blocks = list_capacity(c.total, c.batch, kTile);
    p.blocks = w.list0, p.num_blocks = w.counts;
    delta_kernel<T, kD><<<static_cast<unsigned>(blocks * (kTile / kDeltaRows)), kDeltaThreads, 0, c.stream>>>(
        static_cast<const T*>(out), rest, static_cast<const T*>(d_out), static_cast<const T*>(c.v), c.v_token, c.v_head, delta, w.absmax, p);
    status = launch_status();
    if (status != XMA_OK) return status;
    p.blocks = w.list1, p.num_blocks = w.counts + 1;
    dkdv_kernel<T, kD><<<grid_for(blocks * c.kv_heads), kThreads, Backward<kD>::kSmem, c.stream>>>(mq, mk, mv, mdo, p);
    status = launch_status();
    if (status != XMA_OK) return status;
    p.blocks = w.list0, p.num_blocks = w.counts;
    dq_kernel<T, kD><<<grid_for(blocks * c.heads), kThreads, Backward<kD>::kSmem, c.stream>>>(mq, mk, mv, mdo, p);
    return launch_status();
}

}  // namespace attn
}  // namespace xma

extern "C" {

int64_t xma_attention_workspace_bytes(int64_t total, int64_t batch) {
    if (total < 0 || batch < 0) return 0;
    return 16 + 2 * static_cast<int64_t>(sizeof(xma::attn::Block)) * xma::attn::list_capacity(total, batch, xma::attn::kTile);
}

int64_t xma_attention_stat_rows(int64_t total, int64_t batch) {
    return total < 0 || batch < 0 ? 0 : (total / xma::attn::kTile + batch + 1) * xma::attn::kTile;
}

int xma_selftest_settle(const void* src, int32_t fills, void* dst, int32_t* result, int64_t limit_ns, void* stream) {
    if (!src || !xma::aligned16(src) || !dst || !result || fills < 0 || fills > 64) return XMA_ERR_BAD_ARG;
    if (limit_ns <= 0 || limit_ns > 1000000000ll) return XMA_ERR_BAD_ARG;
    xma::attn::settle_selftest_kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(src), fills, static_cast<uint8_t*>(dst), result, static_cast<uint64_t>(limit_ns));
    return xma::launch_status();
}

int xma_attention_forward(const void* q, const void* k, const void* v, int64_t q_token, int64_t q_head, int64_t k_token,
                          int64_t k_head, int64_t v_token, int64_t v_head, int32_t dtype, const void* cu_seqlens,
                          int32_t cu_is_int64, int64_t batch, int64_t total, int32_t heads, int32_t kv_heads, int32_t dim,
                          float scale, void* out, float* lse, void* out_rest, void* workspace, int32_t* status, void* stream) {
    using namespace xma;
    using namespace xma::attn;
    const Call c{q, k, v, q_token, q_head, k_token, k_head, v_token, v_head, dtype, cu_seqlens, cu_is_int64, batch, total,
                 heads, kv_heads, dim, scale, workspace, status, static_cast<cudaStream_t>(stream)};
    const int rc = check_call(c);
    if (rc != XMA_OK || total == 0) return rc;
    if (!out || !aligned16(out) || !aligned16(out_rest) || (lse == nullptr) != (out_rest == nullptr)) return XMA_ERR_BAD_ARG;
    uint8_t* rest = static_cast<uint8_t*>(out_rest);
    if (dtype == kDtypeBF16)
        return dim <= 64 ? run_forward<__nv_bfloat16, 64>(c, out, lse, rest) : run_forward<__nv_bfloat16, 128>(c, out, lse, rest);
    return dim <= 64 ? run_forward<__half, 64>(c, out, lse, rest) : run_forward<__half, 128>(c, out, lse, rest);
}

int xma_attention_backward(const void* q, const void* k, const void* v, int64_t q_token, int64_t q_head, int64_t k_token,
                           int64_t k_head, int64_t v_token, int64_t v_head, int32_t dtype, const void* cu_seqlens,
                           int32_t cu_is_int64, int64_t batch, int64_t total, int32_t heads, int32_t kv_heads, int32_t dim,
                           float scale, const void* out, const void* out_rest, const void* d_out, const float* lse, float* delta,
                           void* dq, void* dk, void* dv, void* workspace, int32_t* status, void* stream) {
    using namespace xma;
    using namespace xma::attn;
    const Call c{q, k, v, q_token, q_head, k_token, k_head, v_token, v_head, dtype, cu_seqlens, cu_is_int64, batch, total,
                 heads, kv_heads, dim, scale, workspace, status, static_cast<cudaStream_t>(stream)};
    const int rc = check_call(c);
    if (rc != XMA_OK || total == 0) return rc;
    const void* need[] = {out, out_rest, d_out, lse, delta, dq, dk, dv};
    for (int i = 0; i < 8; ++i)
        if (need[i] == nullptr || !aligned16(need[i])) return XMA_ERR_BAD_ARG;
    const uint8_t* rest = static_cast<const uint8_t*>(out_rest);
    if (dtype == kDtypeBF16)
        return dim <= 64 ? run_backward<__nv_bfloat16, 64>(c, out, rest, d_out, lse, delta, dq, dk, dv)
                         : run_backward<__nv_bfloat16, 128>(c, out, rest, d_out, lse, delta, dq, dk, dv);
    return dim <= 64 ? run_backward<__half, 64>(c, out, rest, d_out, lse, delta, dq, dk, dv)
                     : run_backward<__half, 128>(c, out, rest, d_out, lse, delta, dq, dk, dv);
}

}  // extern "C"
