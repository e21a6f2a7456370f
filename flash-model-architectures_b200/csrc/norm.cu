// Root-mean-square norms around a block of a transformer, fused with what joins the block to the
// residual stream. Per row of H elements, in float32, each output rounded once:
//
//   u = post * x * rp,  rp = rsqrt(mean(x^2) + eps)     (u = x without a post norm)
//   s = residual + m * gate * u                          the new residual stream
//   y = weight * s * rs,  rs = rsqrt(mean(s^2) + eps)    the next block's input
//
// Without a residual s = x and only y is written. Backward, with a = weight * dy and the gradient
// d of the stream output:
//
//   ds = rs (a - h mean(a h)) + d,  h = s rs      d_residual = ds
//   d_gate = m ds u,   b = m ds gate post,        dx = rp (b - g mean(b g)),  g = x rp
//   d_weight = sum_rows dy h,                     d_post = sum_rows m ds gate g
//
// sum(b g) follows from three more sums over the row's inputs (ds is linear in a, s and d), so a row
// takes ONE reduction: with c = post * gate * g,
//   sum(c ds) = rs (sum(c a) - mean(a h) rs sum(c s)) + sum(c d).
// No product of two rs, rp or of s and x is formed: of a row of 1e-20 (with an eps that allows it) they are not in
// float32's range, though every h, g and gradient is. Without a post norm g is x, and the sums take it times the power
// of two under rs.
// The backward pass recomputes s from the residual and x where it reads x anyway, so that the rounding of the
// stream does not reach the gradients; for a plain residual add it reads the rounded stream, one tensor less.
//
// The mean of squares adds up (v / H) v, so that it overflows where the mean itself does and no sooner. Below 2^-78 what
// terms lose under float32's smallest normal number begins to show; where eps does not cover that (eps is below 2^-78
// too), such a row's mean is added up again from its values times 2^100, by kernels of their own (kSmallEps: the test alone
// cost the others 1-2 %; 16384 x 4096 with post norm and gate 99 us so, 90 without).
// The ring kernels and the plain forward kernel read and write every tensor once; forward they are bound by HBM, backward
// by issue slots. Rows that the ring does not take are read twice backward, forward above kForwardMaxHidden up to three times.
#include "common.cuh"
#include "ptx.cuh"

namespace xma {
namespace norm {

using namespace ptx;

constexpr int kGateNone = 0;     // no gate
constexpr int kGateChannel = 1;  // [H], a parameter
constexpr int kGateToken = 2;    // [rows], one factor per row
constexpr int kGateFull = 3;     // [rows, H]

constexpr int kForwardThreads = 256;       // plain forward: threads of a CTA with short rows
constexpr int kForwardMaxHidden = 16384;   // plain forward: longer rows are read once per pass
constexpr int kRingThreads = 512;          // ring kernels: threads of a CTA, at most
// Rows of whole vectors, and others: those take one vector a thread (two, backward: 9000 x 4999 bf16 252 us against 271).
constexpr int kRingMaxHidden = 8192, kRingMaxHiddenAny = 4096;
constexpr uint32_t kRingSmem = 220 * 1024;
constexpr int kMaxStages = 6;
// Forward: the ring pays for rows of more than 2048 elements (16384 x 4096 bf16 with a post norm and a gate: 94 us
// against 130 us in the plain kernel, whose CTA-wide sums stall more the more warps share a row; 8191 x 2048 with a
// float32 stream: 43 us against 37 us), with a few chunks for every CTA. Rows that no vector fits load two or four bytes a
// lane, from shared memory sooner than from HBM: 8000 x 3001 bf16 with both 93 us against 126, 16000 x 1111 float32 with a
// residual 58 against 89; 5001 x 1001 float32 (L2, four chunks a CTA) 13 against 11.
constexpr int kRingMinHidden = 2049, kRingMinHiddenAny = 512, kRingMinChunks = 3, kRingMinChunksAny = 8;
constexpr int kPartials = XMA_NORM_PARTIALS;
constexpr float kSmallMean = 0x1p-78f, kSmallScale = 0x1p100f;

struct Params {
    const void* x;
    const void* residual;
    const void* weight;
    const void* post;
    const void* gate;
    int gate_mode;
    bool weight_f32, post_f32, gate_f32;  // parameters in float32 beside 16-bit activations
    int64_t rows;
    int hidden;
    float eps, multiplier;
    void* s_out;
    void* y;
    float* rs;
    float* rp;
    // backward
    const void* dy;
    const void* d_stream;
    const void* s;    // the stream (x for the norm alone); the residual where x is there to compute the stream from
    void* dx;
    void* d_residual;
    void* d_gate;
    float* partials;  // [3][partial_rows][hidden]: weight, post weight, channel gate
    int partial_rows; // as many as there are rows, at most kPartials
    bool want_weight, want_post, want_gate;
    float* row_sums;  // two-kernel backward: [rows][8], what a row's elements need
    int32_t* status;
};

__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 t = unpack2<T>(w[j]);
        f[2 * j] = t.x;
        f[2 * j + 1] = t.y;
    }
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
}

// Eight elements as four pairs.
__device__ __forceinline__ void load8(const float* p, f32x2 (&f)[4]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    f[0] = make_f32x2(a.x, a.y), f[1] = make_f32x2(a.z, a.w), f[2] = make_f32x2(b.x, b.y), f[3] = make_f32x2(b.z, b.w);
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, f32x2 (&f)[4]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 t = unpack2<T>(w[j]);
        f[j] = make_f32x2(t.x, t.y);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const f32x2 (&f)[4]) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) split_f32x2(f[j], v[2 * j], v[2 * j + 1]);
    store8(p, v);
}
__device__ __forceinline__ f32x2 both(float v) { return make_f32x2(v, v); }
__device__ __forceinline__ float total(f32x2 v) {
    float a, b;
    split_f32x2(v, a, b);
    return a + b;
}

// Eight elements of a row: element j of vector `v` of thread `t` (of `group` threads) is column
// column<kVec>(v, t, group, j). Vectorised rows give a thread eight neighbours (one or two 16-byte
// accesses); others give neighbouring threads neighbouring elements, so that any row start and any
// length stays coalesced.
template <bool kVec>
__device__ __forceinline__ int column(int v, int t, int group, int j) {
    return kVec ? (v * group + t) * 8 + j : (v * 8 + j) * group + t;
}
template <bool kVec, typename T>
__device__ __forceinline__ void load_cols(const T* row, int v, int t, int group, int hidden, float (&f)[8]) {
    if (kVec) {
        const int c = column<true>(v, t, group, 0);
        if (c < hidden) {
            load8(row + c, f);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = column<false>(v, t, group, j);
            f[j] = c < hidden ? Elem<T>::to_float(row[c]) : 0.f;
        }
    }
}
template <bool kVec, typename T>
__device__ __forceinline__ void store_cols(T* row, int v, int t, int group, int hidden, const float (&f)[8]) {
    if (kVec) {
        const int c = column<true>(v, t, group, 0);
        if (c < hidden) store8(row + c, f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = column<false>(v, t, group, j);
            if (c < hidden) row[c] = Elem<T>::from_float(f[j]);
        }
    }
}
// A parameter vector, in the activations' type or in float32; ones where there is none.
template <bool kVec, typename T>
__device__ __forceinline__ void load_param(const void* p, bool f32, int v, int t, int group, int hidden, float (&f)[8]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 1.f;
    } else if (f32) {
        load_cols<kVec>(static_cast<const float*>(p), v, t, group, hidden, f);
    } else {
        load_cols<kVec>(static_cast<const T*>(p), v, t, group, hidden, f);
    }
}

__device__ __forceinline__ void group_barrier(int id, int threads) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// Sums kCount values over the `group` threads (whole warps) that share a row; every thread gets the
// sums, added in the same order. `scratch` holds kCount floats per warp of the group; the caller
// alternates between two of them, so that one barrier per call is enough.
template <int kCount>
__device__ __forceinline__ void group_sum(float (&v)[kCount], float* scratch, int t, int group, int barrier) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1)
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], off);
    if (group == 32) return;
    const int warps = group >> 5;
    if ((t & 31) == 0)
#pragma unroll
        for (int i = 0; i < kCount; ++i) scratch[(t >> 5) * kCount + i] = v[i];
    group_barrier(barrier, group);
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = 0.f;
    for (int w = 0; w < warps; ++w)
#pragma unroll
        for (int i = 0; i < kCount; ++i) v[i] += scratch[w * kCount + i];
}

// 1 / sqrt(mean + eps) of a row whose mean was added up again from its values times kSmallScale.
__device__ __forceinline__ float small_rsqrt(float scaled_mean, float eps) {
    return rsqrtf(scaled_mean + eps * kSmallScale * kSmallScale) * kSmallScale;
}
__device__ __forceinline__ bool is_small(float mean, float eps) { return eps < kSmallMean && mean < kSmallMean; }

template <typename T>
__device__ __forceinline__ float token_gate(const Params& p, int64_t row) {
    return p.gate_mode == kGateToken ? Elem<T>::to_float(static_cast<const T*>(p.gate)[row]) : 1.f;
}

// ---------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------

// `group` threads per row hold it in registers (kVpt vectors of eight each); several short rows share a CTA. For few
// rows (4 x 4096: 3.6 us) and rows of up to 2048 elements (8191 x 2048 bf16 with a float32 stream, post norm and
// channel gate: 37 us, 5.4 TB/s); one vector a thread or four are slower (48 and 46 us).
template <typename T, typename R, int kVpt, bool kVec, bool kSmallEps>
__global__ void __launch_bounds__(1024)
forward_kernel(const Params p, int group) {
    __shared__ float scratch[kSmallEps ? 4 : 2][32];
    const int slot = threadIdx.x / group, t = threadIdx.x - slot * group;
    const int slots = blockDim.x / group;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    if (row >= p.rows) return;  // the whole group leaves: its barrier is its own
    const int64_t base = row * p.hidden;
    const int barrier = 1 + slot, my_warps = slot * (group >> 5);
    const float inv_h = 1.f / static_cast<float>(p.hidden);

    float s[kVpt][8];
    // 1 / sqrt(mean(s^2) + eps); `which`: 0 the post norm's, 1 the stream's
    const auto reciprocal_root = [&](int which) {
        float sum[1] = {0.f};
#pragma unroll
        for (int v = 0; v < kVpt; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[0] = fmaf(s[v][j] * inv_h, s[v][j], sum[0]);
        group_sum<1>(sum, &scratch[which][my_warps], t, group, barrier);
        if constexpr (kSmallEps) {
            if (is_small(sum[0], p.eps)) {
                sum[0] = 0.f;
#pragma unroll
                for (int v = 0; v < kVpt; ++v)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum[0] = fmaf(s[v][j] * kSmallScale * inv_h, s[v][j] * kSmallScale, sum[0]);
                group_sum<1>(sum, &scratch[2 + which][my_warps], t, group, barrier);
                return small_rsqrt(sum[0], p.eps);
            }
        }
        return rsqrtf(sum[0] + p.eps);
    };
#pragma unroll
    for (int v = 0; v < kVpt; ++v) load_cols<kVec>(static_cast<const T*>(p.x) + base, v, t, group, p.hidden, s[v]);
    if (p.residual != nullptr) {
        float r[kVpt][8];
#pragma unroll
        for (int v = 0; v < kVpt; ++v)
            load_cols<kVec>(static_cast<const R*>(p.residual) + base, v, t, group, p.hidden, r[v]);
        float scale = p.multiplier * token_gate<T>(p, row);
        if (p.post != nullptr) {
            const float rp = reciprocal_root(0);
            if (t == 0 && p.rp != nullptr) p.rp[row] = rp;
            scale *= rp;
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                float w[8];
                load_param<kVec, T>(p.post, p.post_f32, v, t, group, p.hidden, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[v][j] *= w[j];
            }
        }
        if (p.gate_mode == kGateChannel || p.gate_mode == kGateFull) {
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                float g[8];
                if (p.gate_mode == kGateFull)
                    load_cols<kVec>(static_cast<const T*>(p.gate) + base, v, t, group, p.hidden, g);
                else
                    load_param<kVec, T>(p.gate, p.gate_f32, v, t, group, p.hidden, g);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[v][j] *= g[j];
            }
        }
#pragma unroll
        for (int v = 0; v < kVpt; ++v) {
#pragma unroll
            for (int j = 0; j < 8; ++j) s[v][j] = fmaf(scale, s[v][j], r[v][j]);
            store_cols<kVec>(static_cast<R*>(p.s_out) + base, v, t, group, p.hidden, s[v]);
        }
    }
    const float rs = reciprocal_root(1);
    if (t == 0 && p.rs != nullptr) p.rs[row] = rs;
#pragma unroll
    for (int v = 0; v < kVpt; ++v) {
        float w[8];
        load_param<kVec, T>(p.weight, p.weight_f32, v, t, group, p.hidden, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] *= s[v][j] * rs;
        store_cols<kVec>(static_cast<T*>(p.y) + base, v, t, group, p.hidden, w);
    }
}

template <typename T>
__device__ __forceinline__ float param_at(const void* p, bool f32, int c) {
    if (p == nullptr) return 1.f;
    return f32 ? static_cast<const float*>(p)[c] : Elem<T>::to_float(static_cast<const T*>(p)[c]);
}

// Value of the new stream at one element, from its inputs (scale = multiplier * token gate * rp).
template <typename T, typename R>
__device__ __forceinline__ float stream_at(const Params& p, int64_t base, int c, float scale) {
    float u = Elem<T>::to_float(static_cast<const T*>(p.x)[base + c]);
    if (p.residual == nullptr) return u;
    u *= param_at<T>(p.post, p.post_f32, c);
    if (p.gate_mode == kGateFull) u *= Elem<T>::to_float(static_cast<const T*>(p.gate)[base + c]);
    if (p.gate_mode == kGateChannel) u *= param_at<T>(p.gate, p.gate_f32, c);
    return fmaf(scale, u, Elem<R>::to_float(static_cast<const R*>(p.residual)[base + c]));
}

// Rows too long for registers: one CTA per row, a pass over memory (the row is in L2 by then) for each
// of the sums and one for the outputs.
template <typename T, typename R>
__global__ void __launch_bounds__(1024)
forward_long_kernel(const Params p) {
    __shared__ float scratch[4][32];
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.hidden;
    const int t = threadIdx.x, group = blockDim.x;
    const float inv_h = 1.f / static_cast<float>(p.hidden);
    const auto reciprocal_root = [&](int which, const auto& at) {
        float sum[1] = {0.f};
        for (int c = t; c < p.hidden; c += group) {
            const float v = at(c);
            sum[0] = fmaf(v * inv_h, v, sum[0]);
        }
        group_sum<1>(sum, scratch[which], t, group, 1);
        if (!is_small(sum[0], p.eps)) return rsqrtf(sum[0] + p.eps);
        sum[0] = 0.f;
        for (int c = t; c < p.hidden; c += group) {
            const float v = at(c) * kSmallScale;
            sum[0] = fmaf(v * inv_h, v, sum[0]);
        }
        group_sum<1>(sum, scratch[2 + which], t, group, 1);
        return small_rsqrt(sum[0], p.eps);
    };
    float scale = p.multiplier * token_gate<T>(p, row);
    if (p.residual != nullptr && p.post != nullptr) {
        const float rp = reciprocal_root(0, [&](int c) { return Elem<T>::to_float(static_cast<const T*>(p.x)[base + c]); });
        if (t == 0 && p.rp != nullptr) p.rp[row] = rp;
        scale *= rp;
    }
    const float rs = reciprocal_root(1, [&](int c) { return stream_at<T, R>(p, base, c, scale); });
    if (t == 0 && p.rs != nullptr) p.rs[row] = rs;
    for (int c = t; c < p.hidden; c += group) {
        const float s = stream_at<T, R>(p, base, c, scale);
        if (p.residual != nullptr) static_cast<R*>(p.s_out)[base + c] = Elem<R>::from_float(s);
        static_cast<T*>(p.y)[base + c] = Elem<T>::from_float(param_at<T>(p.weight, p.weight_f32, c) * s * rs);
    }
}

// ---------------------------------------------------------------------------------------------
// Ring kernels: persistent CTAs whose rows come through shared memory
// ---------------------------------------------------------------------------------------------

// `slots` groups of `group` threads share a CTA; a thread keeps its columns (kVpt vectors of eight) and takes
// kRows rows of every chunk of slots * kRows rows. Chunks are copied whole (bulk copies, one per tensor) into a
// ring of stages, so what is in flight does not depend on registers and every row can be read twice. The
// CTA's barriers, which a row sum needs anyway, also say when a stage is free: thread 0 refills it. What a chunk costs
// whatever its size (sums over the CTA, waits, addresses) is some 200 instructions a thread, so a thread takes as
// many rows at once as registers and the ring allow. 16384 x 4096 bf16 with post norm and channel gate: forward 89 us
// (6.1 TB/s, two rows a thread 109), backward 170 us (4.7 TB/s, issue slots half used).
struct RingLayout {
    int slots, group, stages;
    uint32_t stage_bytes;
    uint32_t dy, d_stream, s, x, gate, residual;  // offsets inside a stage
    uint32_t weight, post, channel_gate;          // offsets of the parameters' copies (rows of more than one vector a thread)
    uint32_t ring;                                // offset of stage 0
    uint32_t total;
};
constexpr uint32_t kRingHeader = 128 + 2 * 128 * 4;  // barriers and two scratches of 128 floats

struct RingState {
    uint32_t full;  // barriers
    volatile int* abort_flag;
    float* scratch;
    int stage = 0;
    uint32_t phase = 0, flip = 0;
    __device__ __forceinline__ void next(int stages) {
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    // After a wait that ran out: the copies in flight land, or get the same time once more, before the CTA ends.
    __device__ __forceinline__ void drain(int stages) const {
        const uint64_t begin = global_timer_ns();
        for (int i = 0; i < stages; ++i)
            while (!mbar_try_wait(full + 8 * i, i < stage ? phase ^ 1u : phase) && global_timer_ns() - begin < kWaitLimitNs) {}
    }
};

// Sums of kCount values (a power of two up to 8) over the group's threads, known to each of them; one CTA barrier.
template <int kCount>
__device__ __forceinline__ void ring_sum(float (&v)[kCount], RingState& st, int first_warp, int warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float* scratch = st.scratch + st.flip * 128;
    st.flip ^= 1u;
    // halve the values while lanes are added up: lane bits 16, 8, 4 come to select the value
    int index = 0;
    int off = 16;
#pragma unroll
    for (int n = kCount; n > 1; n >>= 1, off >>= 1) {
        const bool upper = lane & off;
#pragma unroll
        for (int i = 0; i < n / 2; ++i) {
            const float give = upper ? v[i] : v[i + n / 2], keep = upper ? v[i + n / 2] : v[i];
            v[i] = keep + __shfl_xor_sync(0xffffffffu, give, off);
        }
        if (upper) index += n / 2;
    }
#pragma unroll
    for (; off > 0; off >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
    if ((lane & (32 / kCount - 1)) == 0) scratch[warp * kCount + index] = v[0];
    __syncthreads();
    const int count = warps * kCount;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < (16 * kCount + 31) / 32; ++i) {
        const int at = i * 32 + lane;
        if (at < count) sum += scratch[first_warp * kCount + at];
    }
#pragma unroll
    for (int o = 16; o >= kCount; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = __shfl_sync(0xffffffffu, sum, i);
}

// One tensor's share of a chunk, bytes [at, at + bytes), where rows are whole vectors.
__device__ __forceinline__ void ring_copy(uint32_t dst, const void* src, int64_t at, int64_t bytes, uint32_t bar) {
    if (src != nullptr) bulk_load(dst, static_cast<const uint8_t*>(src) + at, static_cast<uint32_t>(bytes), bar);
}
__device__ __forceinline__ int64_t ring_bytes(const void* src, int64_t bytes) { return src != nullptr ? bytes : 0; }

// The same for rows of any length, of a tensor of `total` bytes. Bulk copies take whole pieces of 16 bytes: they start with
// the piece that holds the first byte, so rows lie at & 15 into the tensor's place, and what follows the tensor's last
// whole piece, some elements of two bytes, is copied by the thread itself, before its arrival releases it.
struct RingSpan {
    const uint8_t* src;
    int64_t at, end, from;
    uint32_t bytes;  // of the bulk copy, from `from` on
    __device__ __forceinline__ RingSpan(const void* tensor, int64_t at_, int64_t size, int64_t total)
        : src(static_cast<const uint8_t*>(tensor)), at(at_), end(at_ + size), from(at_ & ~int64_t(15)) {
        bytes = src != nullptr ? static_cast<uint32_t>(max(min((end + 15) & ~int64_t(15), total & ~int64_t(15)) - from, int64_t(0))) : 0u;
    }
    __device__ __forceinline__ void copy_rest(uint8_t* dst) const {
        if (src == nullptr) return;
#pragma unroll 1
        for (int64_t b = max(at, from + bytes); b < end; b += 2)
            *reinterpret_cast<uint16_t*>(dst + (b - from)) = *reinterpret_cast<const uint16_t*>(src + b);
    }
    __device__ __forceinline__ void copy(uint32_t dst, uint32_t bar) const {
        if (bytes > 0) bulk_load(dst, src + from, bytes, bar);
    }
};
// A thread's eight elements of vector v of a row (see `column`); those past the end are zeros where rows have any length,
// and where a vector fits, the caller has seen to it that it lies inside.
template <bool kVec, typename T>
__device__ __forceinline__ void load_cols(const T* row, int v, int t, int group, int hidden, f32x2 (&f)[4]) {
    if (kVec) {
        load8(row + column<true>(v, t, group, 0), f);
    } else {
        float e[8];
        load_cols<false>(row, v, t, group, hidden, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = make_f32x2(e[2 * j], e[2 * j + 1]);
    }
}
// The same from a tensor's place in a stage: `row` is the row's offset in the chunk, `start` the chunk's first element.
template <bool kVec, typename T>
__device__ __forceinline__ void ring_load(const uint8_t* place, int64_t start, int row, int v, int t, int group, int hidden, f32x2 (&f)[4]) {
    if constexpr (kVec) load8(reinterpret_cast<const T*>(place) + (row + column<true>(v, t, group, 0)), f);
    else load_cols<false>(reinterpret_cast<const T*>(place + ((start * sizeof(T)) & 15)) + row, v, t, group, hidden, f);
}
template <bool kVec, typename T>
__device__ __forceinline__ void store_cols(T* row, int v, int t, int group, int hidden, const f32x2 (&f)[4]) {
    if (kVec) {
        store8(row + column<true>(v, t, group, 0), f);
    } else {
        float e[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) split_f32x2(f[j], e[2 * j], e[2 * j + 1]);
        store_cols<false>(row, v, t, group, hidden, e);
    }
}
template <bool kVec, typename T>
__device__ __forceinline__ void load_param(const void* p, bool f32, int v, int t, int group, int hidden, f32x2 (&f)[4]) {
    if (p == nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = both(1.f);
    } else if (f32) {
        load_cols<kVec>(static_cast<const float*>(p), v, t, group, hidden, f);
    } else {
        load_cols<kVec>(static_cast<const T*>(p), v, t, group, hidden, f);
    }
}

// The parameters' copies in shared memory, in their own types.
template <typename T>
__device__ __forceinline__ void copy_param(uint8_t* dst, const void* p, bool f32, int hidden) {
    if (p == nullptr) return;
    for (int c = threadIdx.x; c < hidden; c += blockDim.x) {
        if (f32) reinterpret_cast<float*>(dst)[c] = static_cast<const float*>(p)[c];
        else reinterpret_cast<T*>(dst)[c] = static_cast<const T*>(p)[c];
    }
}

// kDense: every thread's vectors lie inside the row. kVec: rows of whole 16-byte vectors; others take two rows of one vector
// a thread, since the assembler of CUDA 12.9 fails on four rows of 16 bits, which were 10 us faster at 8000 x 3001, and on
// two vectors.
template <typename T, typename R, int kVpt, int kRows, bool kDense, bool kVec, bool kSmallEps>
__global__ void __launch_bounds__(kRingThreads, 1)
forward_ring_kernel(const Params p, const RingLayout lay) {
    extern __shared__ __align__(128) uint8_t smem[];
    RingState st;
    st.full = smem_u32(smem);
    st.abort_flag = reinterpret_cast<volatile int*>(smem + 64);
    st.scratch = reinterpret_cast<float*>(smem + 128);
    const int group = lay.group, warps = group >> 5;
    const int slot = threadIdx.x / group, t = threadIdx.x - slot * group;
    const int first_warp = slot * warps;
    const int per_chunk = lay.slots * kRows;
    const int64_t chunks = (p.rows + per_chunk - 1) / per_chunk;
    const bool full_gate = p.gate_mode == kGateFull, channel_gate = p.gate_mode == kGateChannel;
    const float inv_h = 1.f / static_cast<float>(p.hidden);
    const void* gate_rows = full_gate ? p.gate : nullptr;

    const auto load = [&](int64_t chunk, int stage) {
        if (chunk >= chunks) return;
        const int64_t row0 = chunk * per_chunk;
        const int64_t count = min(static_cast<int64_t>(per_chunk), p.rows - row0) * p.hidden;
        const uint32_t bar = st.full + 8 * stage, place = lay.ring + stage * lay.stage_bytes, dst = smem_u32(smem) + place;
        const int64_t at = row0 * p.hidden, bt = count * static_cast<int64_t>(sizeof(T)), br = count * static_cast<int64_t>(sizeof(R));
        if constexpr (kVec) {
            mbar_expect_tx(bar, static_cast<uint32_t>(bt + ring_bytes(p.residual, br) + ring_bytes(gate_rows, bt)));
            ring_copy(dst + lay.x, p.x, at * sizeof(T), bt, bar);
            ring_copy(dst + lay.residual, p.residual, at * sizeof(R), br, bar);
            ring_copy(dst + lay.gate, gate_rows, at * sizeof(T), bt, bar);
        } else {
            const int64_t all = p.rows * p.hidden;
            const RingSpan x(p.x, at * sizeof(T), bt, all * sizeof(T)), residual(p.residual, at * sizeof(R), br, all * sizeof(R)),
                gate(gate_rows, at * sizeof(T), bt, all * sizeof(T));
            x.copy_rest(smem + place + lay.x);
            residual.copy_rest(smem + place + lay.residual);
            gate.copy_rest(smem + place + lay.gate);
            mbar_expect_tx(bar, x.bytes + residual.bytes + gate.bytes);
            x.copy(dst + lay.x, bar);
            residual.copy(dst + lay.residual, bar);
            gate.copy(dst + lay.gate, bar);
        }
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < lay.stages; ++i) mbar_init(st.full + 8 * i, 1);
        *st.abort_flag = 0;
        fence_barrier_init();
        for (int i = 0; i < lay.stages; ++i) load(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, i);
    }
    // What a column is multiplied with: in registers for one vector a thread, else in shared memory.
    f32x2 w_reg[4], c_reg[4];
    if (kVpt == 1) {
        if (!kVec || t * 8 < p.hidden) {
            load_param<kVec, T>(p.weight, p.weight_f32, 0, t, group, p.hidden, w_reg);
            load_param<kVec, T>(p.post, p.post_f32, 0, t, group, p.hidden, c_reg);
            if (channel_gate) {
                f32x2 g[4];
                load_param<kVec, T>(p.gate, p.gate_f32, 0, t, group, p.hidden, g);
#pragma unroll
                for (int j = 0; j < 4; ++j) c_reg[j] = mul_f32x2(c_reg[j], g[j]);
            }
        }
    } else {
        copy_param<T>(smem + lay.weight, p.weight, p.weight_f32, p.hidden);
        copy_param<T>(smem + lay.post, p.post, p.post_f32, p.hidden);
        if (channel_gate) copy_param<T>(smem + lay.channel_gate, p.gate, p.gate_f32, p.hidden);
    }
    __syncthreads();

    for (int64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int64_t row0 = chunk * per_chunk + slot * kRows;
        if (!mbar_wait(st.full + 8 * st.stage, st.phase, st.abort_flag, p.status, 403)) {
            st.drain(lay.stages);
            break;
        }
        const uint8_t* stage = smem + lay.ring + st.stage * lay.stage_bytes;
        const int64_t start = chunk * per_chunk * p.hidden;  // the chunk's first element
        const auto inside = [&](int v) { return kDense || !kVec || (v * group + t) * 8 < p.hidden; };
        f32x2 s[kRows][kVpt][4];
        float sums[kRows], scale[kRows];
        // kSmallEps: the rows' means become 1 / sqrt(mean + eps); the whole CTA takes the second sum if a row needs it
        const auto small_roots = [&] {
            bool small[kRows], any = false;
#pragma unroll
            for (int r = 0; r < kRows; ++r) any = (small[r] = is_small(sums[r], p.eps)) || any;
            float again[kRows];
            if (lay.slots == 1 ? any : __syncthreads_or(any) != 0) {  // one row group a CTA knows it without asking
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    f32x2 sum = both(0.f);
#pragma unroll
                    for (int v = 0; v < kVpt; ++v)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const f32x2 up = mul_f32x2(s[r][v][j], both(kSmallScale));
                            sum = fma_f32x2(mul_f32x2(up, both(inv_h)), up, sum);
                        }
                    again[r] = total(sum);
                }
                ring_sum<kRows>(again, st, first_warp, warps);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) sums[r] = small[r] ? small_rsqrt(again[r], p.eps) : rsqrtf(sums[r] + p.eps);
        };
        const auto reciprocal_root = [&](int r) { return kSmallEps ? sums[r] : rsqrtf(sums[r] + p.eps); };
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            f32x2 sum = both(0.f);
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                if (inside(v)) ring_load<kVec, T>(stage + lay.x, start, (slot * kRows + r) * p.hidden, v, t, group, p.hidden, s[r][v]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (!inside(v)) s[r][v][j] = both(0.f);
                    sum = fma_f32x2(mul_f32x2(s[r][v][j], both(inv_h)), s[r][v][j], sum);
                }
            }
            sums[r] = total(sum);
            scale[r] = p.residual != nullptr && row0 + r < p.rows ? p.multiplier * token_gate<T>(p, row0 + r) : 1.f;
        }
        if (p.residual != nullptr) {
            if (p.post != nullptr) {
                ring_sum<kRows>(sums, st, first_warp, warps);
                if constexpr (kSmallEps) small_roots();
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    const float rp = reciprocal_root(r);
                    scale[r] *= rp;
                    if (t == 0 && p.rp != nullptr && row0 + r < p.rows) p.rp[row0 + r] = rp;
                }
            }
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                f32x2 f[4];
                if (kVpt > 1 && inside(v)) {
                    load_param<kVec, T>(p.post ? smem + lay.post : nullptr, p.post_f32, v, t, group, p.hidden, f);
                    if (channel_gate) {
                        f32x2 g[4];
                        load_param<kVec, T>(smem + lay.channel_gate, p.gate_f32, v, t, group, p.hidden, g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) f[j] = mul_f32x2(f[j], g[j]);
                    }
                }
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if (!inside(v)) continue;
                    const int off = (slot * kRows + r) * p.hidden;
                    f32x2 res[4];
                    ring_load<kVec, R>(stage + lay.residual, start, off, v, t, group, p.hidden, res);
                    if (full_gate) {
                        f32x2 g[4];
                        ring_load<kVec, T>(stage + lay.gate, start, off, v, t, group, p.hidden, g);
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[r][v][j] = mul_f32x2(s[r][v][j], g[j]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[r][v][j] = fma_f32x2(mul_f32x2(s[r][v][j], kVpt > 1 ? f[j] : c_reg[j]), both(scale[r]), res[j]);
                }
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                f32x2 sum = both(0.f);
#pragma unroll
                for (int v = 0; v < kVpt; ++v)
#pragma unroll
                    for (int j = 0; j < 4; ++j) sum = fma_f32x2(mul_f32x2(s[r][v][j], both(inv_h)), s[r][v][j], sum);
                sums[r] = total(sum);
            }
        }
        ring_sum<kRows>(sums, st, first_warp, warps);
        // every thread has read the stage: it can take the chunk after the ones in flight
        if (threadIdx.x == 0) load(chunk + static_cast<int64_t>(lay.stages) * gridDim.x, st.stage);
        st.next(lay.stages);
        if constexpr (kSmallEps) small_roots();
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row0 + r >= p.rows) continue;
            const float rs = reciprocal_root(r);
            if (t == 0 && p.rs != nullptr) p.rs[row0 + r] = rs;
            const int64_t base = (row0 + r) * p.hidden;
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                if (!inside(v)) continue;
                if (p.residual != nullptr) store_cols<kVec>(static_cast<R*>(p.s_out) + base, v, t, group, p.hidden, s[r][v]);
                f32x2 f[4];
                if (kVpt > 1) load_param<kVec, T>(p.weight ? smem + lay.weight : nullptr, p.weight_f32, v, t, group, p.hidden, f);
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = mul_f32x2(mul_f32x2(s[r][v][j], both(rs)), kVpt > 1 ? f[j] : w_reg[j]);
                store_cols<kVec>(static_cast<T*>(p.y) + base, v, t, group, p.hidden, f);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------

// What the elements of a row need beside their inputs.
struct RowScale {
    float rs, rp;
    float k_s;   // mean(a h), h = rs s
    float k_x;   // mean(b g), g = rp x, with the multiplier and the token gate in it
    float m;     // multiplier * token gate
    float d_token_gate;
};
// What x is multiplied with in the sums: rp, or the power of two under rs where there is no post norm.
__device__ __forceinline__ float sum_scale(const Params& p, float rs, float rp) {
    return p.post != nullptr ? rp : __uint_as_float(min(__float_as_uint(rs) & 0x7f800000u, 0x7e800000u));
}
// That back: g = x rp is `sum_scale` times x times this, 1 or the reciprocal of a power of two.
__device__ __forceinline__ float sum_unscale(const Params& p, float scale) {
    return p.post != nullptr ? 1.f : __uint_as_float(0x7f000000u - __float_as_uint(scale));
}

// sums: (a s), (c a), (c s), (c d); c = post * gate * x * sum_scale
__device__ __forceinline__ RowScale row_scale(const Params& p, const float (&sums)[4], float rs, float rp, float token, float unscale) {
    RowScale r;
    const float inv_h = 1.f / static_cast<float>(p.hidden);
    r.rs = rs;
    r.rp = rp;
    r.k_s = rs * sums[0] * inv_h;
    const float c_ds = (rs * (sums[1] - r.k_s * (rs * sums[2])) + sums[3]) * unscale;
    r.m = p.multiplier * token;
    r.k_x = p.post != nullptr ? r.m * c_ds * inv_h : 0.f;
    r.d_token_gate = p.multiplier * c_ds;
    return r;
}

// The parameters' gradients stay in registers (a thread keeps its columns) until the CTA's last row and leave as
// one partial row per CTA, summed in a fixed order by sum_kernel. kX: a post norm or a gate is there, so x is
// read; kFull: the gate has the shape of x. kCall: what the call is known to have (kCallAny: nothing); a branch per
// vector costs a sixth of the time (16384 x 4096 bf16 with post norm and channel gate: 192 us with them, 159 without).
constexpr int kCallAny = 0, kCallAll = 1, kCallAlone = 2, kCallShared = 3;
template <typename T, typename R, int kVpt, int kRows, bool kX, bool kFull, int kCall, bool kVec>
__global__ void __launch_bounds__(kRingThreads, 1)
backward_ring_kernel(const Params p, const RingLayout lay) {
    constexpr int kSums = kX ? 4 : 1;
    constexpr bool kKnown = kCall != kCallAny;  // every thread's vectors lie inside the row, dy and d_residual are there
    const bool has_dy = kKnown || p.dy != nullptr, has_d_residual = kKnown || p.d_residual != nullptr;
    const bool has_d_stream = kKnown ? kCall != kCallAlone : p.d_stream != nullptr;
    const bool has_dx = kKnown ? kCall == kCallAll : p.dx != nullptr;
    extern __shared__ __align__(128) uint8_t smem[];
    RingState st;
    st.full = smem_u32(smem);
    st.abort_flag = reinterpret_cast<volatile int*>(smem + 64);
    st.scratch = reinterpret_cast<float*>(smem + 128);
    const int group = lay.group, warps = group >> 5;
    const int slot = threadIdx.x / group, t = threadIdx.x - slot * group;
    const int first_warp = slot * warps;
    const int per_chunk = lay.slots * kRows;
    const int64_t chunks = (p.rows + per_chunk - 1) / per_chunk;
    const bool channel_gate = kX && p.gate_mode == kGateChannel;
    const void* gate_rows = kFull ? p.gate : nullptr;

    const auto load = [&](int64_t chunk, int stage) {
        if (chunk >= chunks) return;
        const int64_t row0 = chunk * per_chunk;
        const int64_t count = min(static_cast<int64_t>(per_chunk), p.rows - row0) * p.hidden;
        const uint32_t bar = st.full + 8 * stage, place = lay.ring + stage * lay.stage_bytes, dst = smem_u32(smem) + place;
        const int64_t at = row0 * p.hidden, bt = count * static_cast<int64_t>(sizeof(T)), br = count * static_cast<int64_t>(sizeof(R));
        if constexpr (kVec) {
            mbar_expect_tx(bar, static_cast<uint32_t>(br + ring_bytes(p.dy, bt) + ring_bytes(p.d_stream, br) + ring_bytes(p.x, bt) +
                                                      ring_bytes(gate_rows, bt)));
            ring_copy(dst + lay.s, p.s, at * sizeof(R), br, bar);
            ring_copy(dst + lay.dy, p.dy, at * sizeof(T), bt, bar);
            ring_copy(dst + lay.d_stream, p.d_stream, at * sizeof(R), br, bar);
            ring_copy(dst + lay.x, p.x, at * sizeof(T), bt, bar);
            ring_copy(dst + lay.gate, gate_rows, at * sizeof(T), bt, bar);
        } else {
            const int64_t all = p.rows * p.hidden;
            const RingSpan s(p.s, at * sizeof(R), br, all * sizeof(R)), dy(p.dy, at * sizeof(T), bt, all * sizeof(T)),
                d_stream(p.d_stream, at * sizeof(R), br, all * sizeof(R)), x(p.x, at * sizeof(T), bt, all * sizeof(T)),
                gate(gate_rows, at * sizeof(T), bt, all * sizeof(T));
            s.copy_rest(smem + place + lay.s);
            dy.copy_rest(smem + place + lay.dy);
            d_stream.copy_rest(smem + place + lay.d_stream);
            x.copy_rest(smem + place + lay.x);
            gate.copy_rest(smem + place + lay.gate);
            mbar_expect_tx(bar, s.bytes + dy.bytes + d_stream.bytes + x.bytes + gate.bytes);
            s.copy(dst + lay.s, bar);
            dy.copy(dst + lay.dy, bar);
            d_stream.copy(dst + lay.d_stream, bar);
            x.copy(dst + lay.x, bar);
            gate.copy(dst + lay.gate, bar);
        }
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < lay.stages; ++i) mbar_init(st.full + 8 * i, 1);
        *st.abort_flag = 0;
        fence_barrier_init();
        for (int i = 0; i < lay.stages; ++i) load(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, i);
    }
    // Parameters: in registers for one vector a thread, else in shared memory.
    f32x2 w_reg[4], post_reg[4], gate_reg[4];
    if (kVpt == 1) {
        if (!kVec || t * 8 < p.hidden) {
            load_param<kVec, T>(p.weight, p.weight_f32, 0, t, group, p.hidden, w_reg);
            if (kX) load_param<kVec, T>(p.post, p.post_f32, 0, t, group, p.hidden, post_reg);
            if (kX && !kFull) load_param<kVec, T>(channel_gate ? p.gate : nullptr, p.gate_f32, 0, t, group, p.hidden, gate_reg);
        }
    } else {
        copy_param<T>(smem + lay.weight, p.weight, p.weight_f32, p.hidden);
        copy_param<T>(smem + lay.post, p.post, p.post_f32, p.hidden);
        if (channel_gate) copy_param<T>(smem + lay.channel_gate, p.gate, p.gate_f32, p.hidden);
    }
    const auto weight8 = [&](int v, f32x2 (&f)[4]) {
        if (kVpt > 1) {
            load_param<kVec, T>(p.weight ? smem + lay.weight : nullptr, p.weight_f32, v, t, group, p.hidden, f);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = w_reg[j];
        }
    };
    const auto post8 = [&](int v, f32x2 (&f)[4]) {
        if (kVpt > 1) {
            load_param<kVec, T>(p.post ? smem + lay.post : nullptr, p.post_f32, v, t, group, p.hidden, f);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = post_reg[j];
        }
    };
    const auto gate8 = [&](const uint8_t* place, int64_t start, int row, int v, f32x2 (&f)[4]) {
        if (kFull) {
            ring_load<kVec, T>(place, start, row, v, t, group, p.hidden, f);
        } else if (kVpt > 1) {
            load_param<kVec, T>(channel_gate ? smem + lay.channel_gate : nullptr, p.gate_f32, v, t, group, p.hidden, f);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = gate_reg[j];
        }
    };
    f32x2 acc_w[kVpt][4], acc_p[kVpt][4], acc_g[kVpt][4];
#pragma unroll
    for (int v = 0; v < kVpt; ++v)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc_w[v][j] = acc_p[v][j] = acc_g[v][j] = both(0.f);
    __syncthreads();

    int previous = -1;
    for (int64_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int64_t row0 = chunk * per_chunk + slot * kRows;
        float rs[kRows], scale[kRows], token[kRows];  // scale: rp, where there is a post norm
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const bool valid = row0 + r < p.rows;  // the same in the whole group
            rs[r] = valid ? p.rs[row0 + r] : 0.f;
            scale[r] = kX ? sum_scale(p, rs[r], valid && p.post != nullptr ? p.rp[row0 + r] : 1.f) : 1.f;
            token[r] = valid && kX ? token_gate<T>(p, row0 + r) : 1.f;
        }
        if (!mbar_wait(st.full + 8 * st.stage, st.phase, st.abort_flag, p.status, 402)) {
            st.drain(lay.stages);
            break;
        }
        const uint8_t* stage = smem + lay.ring + st.stage * lay.stage_bytes;
        const int64_t start = chunk * per_chunk * p.hidden;  // the chunk's first element
        const auto outside = [&](int v) { return !kKnown && kVec && (v * group + t) * 8 >= p.hidden; };
        const auto load_t = [&](uint32_t tensor, int row, int v, f32x2 (&f)[4]) {
            ring_load<kVec, T>(stage + tensor, start, row, v, t, group, p.hidden, f);
        };
        const auto load_r = [&](uint32_t tensor, int row, int v, f32x2 (&f)[4]) {
            ring_load<kVec, R>(stage + tensor, start, row, v, t, group, p.hidden, f);
        };
        float sums[kRows * kSums];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int off = (slot * kRows + r) * p.hidden;
            const float m = kX ? p.multiplier * token[r] * sum_unscale(p, scale[r]) : 1.f;
            f32x2 sum[kSums];
#pragma unroll
            for (int i = 0; i < kSums; ++i) sum[i] = both(0.f);
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                if (outside(v)) continue;
                f32x2 a[4], s8[4], f[4], x8[4];
                load_r(lay.s, off, v, s8);
                if (kX) {
                    f32x2 g[4];
                    load_t(lay.x, off, v, x8);
                    post8(v, f);
                    gate8(stage + lay.gate, start, off, v, g);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x8[j] = mul_f32x2(mul_f32x2(x8[j], both(scale[r])), mul_f32x2(f[j], g[j]));
                        s8[j] = fma_f32x2(x8[j], both(m), s8[j]);  // the stream, from the residual
                    }
                }
                if (has_dy) {
                    load_t(lay.dy, off, v, a);
                    weight8(v, f);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[j] = mul_f32x2(a[j], f[j]);
                        sum[0] = fma_f32x2(a[j], s8[j], sum[0]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[j] = both(0.f);
                }
                if (kX) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sum[kSums > 1 ? 1 : 0] = fma_f32x2(x8[j], a[j], sum[kSums > 1 ? 1 : 0]);
                        sum[kSums > 1 ? 2 : 0] = fma_f32x2(x8[j], s8[j], sum[kSums > 1 ? 2 : 0]);
                    }
                    if (has_d_stream) {
                        load_r(lay.d_stream, off, v, f);
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[kSums > 1 ? 3 : 0] = fma_f32x2(x8[j], f[j], sum[kSums > 1 ? 3 : 0]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kSums; ++i) sums[r * kSums + i] = total(sum[i]);
        }
        ring_sum<kRows * kSums>(sums, st, first_warp, warps);
        // every thread is done with the chunk before this one
        if (threadIdx.x == 0 && previous >= 0) load(chunk + static_cast<int64_t>(lay.stages - 1) * gridDim.x, previous);
        previous = st.stage;
        st.next(lay.stages);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            if (row0 + r >= p.rows) continue;
            float four[4] = {sums[r * kSums], 0.f, 0.f, 0.f};
            if (kX) four[1] = sums[r * kSums + kSums - 3], four[2] = sums[r * kSums + kSums - 2], four[3] = sums[r * kSums + kSums - 1];
            const RowScale k = row_scale(p, four, rs[r], kX && p.post != nullptr ? scale[r] : 1.f, token[r], kX ? sum_unscale(p, scale[r]) : 1.f);
            const int64_t base = (row0 + r) * p.hidden;
            const int off = (slot * kRows + r) * p.hidden;
            if (kX && !kFull && p.gate_mode == kGateToken && p.d_gate != nullptr && t == 0)
                static_cast<T*>(p.d_gate)[row0 + r] = Elem<T>::from_float(k.d_token_gate);
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                if (outside(v)) continue;
                f32x2 ds[4], f[4], s8[4], hat[4], u[4], g[4];
                if (has_dy || kX) load_r(lay.s, off, v, s8);
                if (kX) {
                    load_t(lay.x, off, v, hat);
                    post8(v, f);
                    gate8(stage + lay.gate, start, off, v, g);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        hat[j] = mul_f32x2(hat[j], both(k.rp));
                        u[j] = mul_f32x2(hat[j], f[j]);
                        s8[j] = fma_f32x2(mul_f32x2(u[j], g[j]), both(k.m), s8[j]);
                    }
                }
                if (has_d_stream) {
                    load_r(lay.d_stream, off, v, ds);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) ds[j] = both(0.f);
                }
                if (has_dy) {
                    f32x2 d8[4], w8[4];
                    load_t(lay.dy, off, v, d8);
                    weight8(v, w8);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s8[j] = mul_f32x2(s8[j], both(k.rs));
                        acc_w[v][j] = fma_f32x2(d8[j], s8[j], acc_w[v][j]);
                        ds[j] = fma_f32x2(fma_f32x2(s8[j], both(-k.k_s), mul_f32x2(d8[j], w8[j])), both(k.rs), ds[j]);
                    }
                }
                if (has_d_residual) store_cols<kVec>(static_cast<R*>(p.d_residual) + base, v, t, group, p.hidden, ds);
                f32x2 b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) b[j] = mul_f32x2(ds[j], both(k.m));  // gradient of the gated branch, token gate in it
                if (kX) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (kFull) u[j] = mul_f32x2(b[j], u[j]);
                        else acc_g[v][j] = fma_f32x2(b[j], u[j], acc_g[v][j]);
                        b[j] = mul_f32x2(b[j], g[j]);
                        acc_p[v][j] = fma_f32x2(b[j], hat[j], acc_p[v][j]);
                        b[j] = mul_f32x2(fma_f32x2(hat[j], both(-k.k_x), mul_f32x2(b[j], f[j])), both(k.rp));
                    }
                    if (kFull && p.d_gate != nullptr) store_cols<kVec>(static_cast<T*>(p.d_gate) + base, v, t, group, p.hidden, u);
                }
                if (has_dx) store_cols<kVec>(static_cast<T*>(p.dx) + base, v, t, group, p.hidden, b);
            }
        }
    }
    __syncthreads();  // every load has landed and been read: the ring is free

    // The slots' sums, added in slot order, leave as this CTA's partial rows.
    float* buf = reinterpret_cast<float*>(smem + lay.ring);
    const bool want[3] = {p.want_weight, p.want_post, p.want_gate};
#pragma unroll
    for (int which = 0; which < 3; ++which) {
        if (!want[which]) continue;
        f32x2(&acc)[kVpt][4] = which == 0 ? acc_w : which == 1 ? acc_p : acc_g;
        float* out = p.partials + (static_cast<int64_t>(which) * p.partial_rows + blockIdx.x) * p.hidden;
        float* mine = lay.slots == 1 ? out : buf + slot * p.hidden;
#pragma unroll
        for (int v = 0; v < kVpt; ++v) {
            if (kKnown || !kVec || (v * group + t) * 8 < p.hidden) store_cols<kVec>(mine, v, t, group, p.hidden, acc[v]);
        }
        if (lay.slots == 1) continue;
        __syncthreads();
        for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) {
            float sum = 0.f;
            for (int sl = 0; sl < lay.slots; ++sl) sum += buf[sl * p.hidden + c];
            out[c] = sum;
        }
        __syncthreads();
    }
}

// The elements of one position, from global memory (two-kernel backward).
template <typename T, typename R>
struct Element {
    float dy, s, d, x, w, post, gate;  // x: times the row's `scale`
    // m: multiplier * token gate of the row, times what undoes `scale`
    __device__ __forceinline__ Element(const Params& p, int64_t base, int c, float m, float scale) {
        dy = p.dy != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.dy)[base + c]) : 0.f;
        s = Elem<R>::to_float(static_cast<const R*>(p.s)[base + c]);
        d = p.d_stream != nullptr ? Elem<R>::to_float(static_cast<const R*>(p.d_stream)[base + c]) : 0.f;
        x = p.x != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.x)[base + c]) * scale : 0.f;
        w = param_at<T>(p.weight, p.weight_f32, c);
        post = param_at<T>(p.post, p.post_f32, c);
        gate = p.gate_mode == kGateFull      ? Elem<T>::to_float(static_cast<const T*>(p.gate)[base + c])
               : p.gate_mode == kGateChannel ? param_at<T>(p.gate, p.gate_f32, c)
                                             : 1.f;
        if (p.x != nullptr) s = fmaf(x * post * gate, m, s);  // the stream, from the residual
    }
};

// What the ring does not take (longer rows, tensors off a 16-byte boundary), in two kernels: the row sums, from which
// what a row's elements need is worked out once, then the elements (a block of columns times a share of the rows per CTA,
// so that the parameters' gradients are sums in registers; four rows at a time, for loads in flight). Every tensor is
// read twice, two or four bytes a lane, whole vectors or not: 9000 x 4999 bf16 alone 121 + 131 us; 8000 x 3001 bf16 with
// everything took 91 + 119 us here and takes 117 in the ring, 5001 x 1001 float32 19 + 19 and 14. It also takes calls of
// which two stages of two rows a thread do not fit (16384 x 4096 float32 with a post norm: 206 + 269 us, floor 187).
template <typename T, typename R>
__global__ void __launch_bounds__(256)
backward_sums_kernel(const Params p) {
    __shared__ float scratch[8 * 4];
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.hidden;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    const float rp = p.post != nullptr ? p.rp[row] : 1.f, token = token_gate<T>(p, row);
    const float scale = sum_scale(p, p.rs[row], rp), unscale = sum_unscale(p, scale);
    const float m = p.multiplier * token * unscale;
    for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) {
        const Element<T, R> e(p, base, c, m, scale);
        const float a = e.dy * e.w, q = e.x * e.post * e.gate;
        sums[0] += a * e.s;
        sums[1] += q * a;
        sums[2] += q * e.s;
        sums[3] += q * e.d;
    }
    group_sum<4>(sums, scratch, threadIdx.x, blockDim.x, 1);
    if (threadIdx.x == 0) {
        const RowScale k = row_scale(p, sums, p.rs[row], rp, token, unscale);
        float4* out = reinterpret_cast<float4*>(p.row_sums) + row * 2;
        out[0] = make_float4(k.rs, k.k_s, k.rp, k.k_x);
        out[1] = make_float4(k.m, 0.f, 0.f, 0.f);
        if (p.gate_mode == kGateToken && p.d_gate != nullptr) static_cast<T*>(p.d_gate)[row] = Elem<T>::from_float(k.d_token_gate);
    }
}

template <typename T, typename R>
__global__ void __launch_bounds__(256)
backward_elements_kernel(const Params p, int64_t rows_per_cta) {
    constexpr int kBatch = 4;
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * rows_per_cta;
    const int64_t last = min(first + rows_per_cta, p.rows);
    float acc_w = 0.f, acc_p = 0.f, acc_g = 0.f;
    if (c >= p.hidden) return;
    const float w = param_at<T>(p.weight, p.weight_f32, c), post = param_at<T>(p.post, p.post_f32, c);
    const float gate = p.gate_mode == kGateChannel ? param_at<T>(p.gate, p.gate_f32, c) : 1.f;
    for (int64_t row0 = first; row0 < last; row0 += kBatch) {
        float dy[kBatch], s[kBatch], d[kBatch], x[kBatch], g[kBatch];
        float4 k[kBatch];
        float m[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int64_t row = min(row0 + u, last - 1), at = row * p.hidden + c;  // the last row again where there is none
            dy[u] = p.dy != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.dy)[at]) : 0.f;
            s[u] = Elem<R>::to_float(static_cast<const R*>(p.s)[at]);
            d[u] = p.d_stream != nullptr ? Elem<R>::to_float(static_cast<const R*>(p.d_stream)[at]) : 0.f;
            x[u] = p.x != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.x)[at]) : 0.f;
            g[u] = p.gate_mode == kGateFull ? Elem<T>::to_float(static_cast<const T*>(p.gate)[at]) : gate;
            k[u] = reinterpret_cast<const float4*>(p.row_sums)[row * 2];
            m[u] = p.row_sums[row * 8 + 4];
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            if (row0 + u >= last) break;
            const int64_t at = (row0 + u) * p.hidden + c;
            const float rs = k[u].x, k_s = k[u].y, rp = k[u].z, k_x = k[u].w;
            const float g_x = x[u] * rp;
            if (p.x != nullptr) s[u] = fmaf(g_x * post * g[u], m[u], s[u]);
            const float h = s[u] * rs;
            acc_w += dy[u] * h;
            const float ds = fmaf(rs, dy[u] * w - h * k_s, d[u]);
            if (p.d_residual != nullptr) static_cast<R*>(p.d_residual)[at] = Elem<R>::from_float(ds);
            float b = m[u] * ds;
            const float dg = b * g_x * post;
            if (p.gate_mode == kGateFull && p.d_gate != nullptr) static_cast<T*>(p.d_gate)[at] = Elem<T>::from_float(dg);
            acc_g += dg;
            b *= g[u];
            if (p.post != nullptr) {
                acc_p += b * g_x;
                b = rp * (b * post - g_x * k_x);
            }
            if (p.dx != nullptr) static_cast<T*>(p.dx)[at] = Elem<T>::from_float(b);
        }
    }
    const int64_t at = static_cast<int64_t>(blockIdx.y) * p.hidden + c;
    const int64_t plane = static_cast<int64_t>(p.partial_rows) * p.hidden;
    if (p.want_weight) p.partials[at] = acc_w;
    if (p.want_post) p.partials[plane + at] = acc_p;
    if (p.want_gate) p.partials[2 * plane + at] = acc_g;
}

// out[c] = sum of the partial rows, in a fixed order: eight threads take every eighth row of a column.
template <typename T>
__global__ void __launch_bounds__(256)
sum_kernel(const Params p, int count, void* d_weight, void* d_post, void* d_gate) {
    __shared__ float part[8][33];
    const int which = blockIdx.y;
    void* out = which == 0 ? d_weight : which == 1 ? d_post : d_gate;
    if (out == nullptr) return;
    const bool f32 = which == 0 ? p.weight_f32 : which == 1 ? p.post_f32 : p.gate_f32;
    const int c = blockIdx.x * 32 + threadIdx.x;
    const float* src = p.partials + static_cast<int64_t>(which) * p.partial_rows * p.hidden + c;
    float sum = 0.f;
    if (c < p.hidden)
        for (int i = threadIdx.y; i < count; i += 8) sum += src[static_cast<int64_t>(i) * p.hidden];
    part[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y == 0 && c < p.hidden) {
#pragma unroll
        for (int i = 1; i < 8; ++i) sum += part[i][threadIdx.x];
        if (f32) static_cast<float*>(out)[c] = sum;
        else static_cast<T*>(out)[c] = Elem<T>::from_float(sum);
    }
}

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// Threads, stages and offsets of a ring kernel; false when not `min_stages` stages of a chunk fit.
template <typename T, typename R>
static bool ring_layout(const Params& p, bool vec, bool backward, int vpt, int rows, int min_stages, RingLayout* lay) {
    const uint32_t h = static_cast<uint32_t>(p.hidden);
    lay->group = static_cast<int>(ceil_div(ceil_div(h, 8 * vpt), 32) * 32);
    if (lay->group > kRingThreads) return false;
    const uint32_t row_t = h * sizeof(T), row_r = h * sizeof(R);
    uint32_t at = kRingHeader;
    const auto param = [&](bool there, bool f32) {
        const uint32_t here = at;
        if (vpt > 1 && there) at += (h * (f32 ? 4u : static_cast<uint32_t>(sizeof(T))) + 15u) & ~15u;
        return here;
    };
    lay->weight = param(p.weight != nullptr, p.weight_f32);
    lay->post = param(p.post != nullptr, p.post_f32);
    lay->channel_gate = param(p.gate_mode == kGateChannel, p.gate_f32);
    lay->ring = (at + 127u) & ~127u;
    // halve the rows a CTA takes at once until enough stages fit
    for (lay->slots = kRingThreads / lay->group;; lay->slots /= 2) {
        const uint32_t n = static_cast<uint32_t>(lay->slots * rows);
        uint32_t off = 0;
        const auto tensor = [&](bool there, uint32_t row) {
            const uint32_t here = off;
            off += !there ? 0 : vec ? n * row : ((n * row + 15u) & ~15u) + 32u;  // see RingSpan
            return here;
        };
        lay->s = tensor(backward, row_r);
        lay->dy = tensor(backward && p.dy != nullptr, row_t);
        lay->d_stream = tensor(backward && p.d_stream != nullptr, row_r);
        lay->x = tensor(p.x != nullptr, row_t);
        lay->residual = tensor(!backward && p.residual != nullptr, row_r);
        lay->gate = tensor(p.gate_mode == kGateFull, row_t);
        lay->stage_bytes = (off + 127u) & ~127u;
        lay->stages = static_cast<int>((kRingSmem - lay->ring) / lay->stage_bytes);
        if (lay->stages >= min_stages || lay->slots == 1) break;
    }
    if (lay->stages < min_stages) return false;
    if (lay->stages > kMaxStages) lay->stages = kMaxStages;
    uint32_t ring = lay->stage_bytes * static_cast<uint32_t>(lay->stages);
    const uint32_t reduce = backward && lay->slots > 1 ? static_cast<uint32_t>(lay->slots) * h * 4 : 0;
    if (ring < reduce) ring = reduce;
    lay->total = lay->ring + ring;
    return lay->total <= kRingSmem;
}

// Launches a ring kernel on as many CTAs as there are chunks and SMs; *count says how many.
template <auto kKernel>
static int launch_ring(const Params& p, const RingLayout& lay, int rows, int* count, cudaStream_t stream) {
    if (!allow_smem<kKernel>(kRingSmem)) return XMA_ERR_LAUNCH;
    int64_t grid = ceil_div(p.rows, lay.slots * rows);
    const int64_t most = sm_count() < kPartials ? sm_count() : kPartials;
    if (grid > most) grid = most;
    *count = static_cast<int>(grid);
    kKernel<<<static_cast<unsigned>(grid), static_cast<unsigned>(lay.group * lay.slots), lay.total, stream>>>(p, lay);
    return launch_status();
}

// Whether the group's vectors fill a row exactly.
static bool dense(const Params& p, const RingLayout& lay, int vpt) { return p.hidden == lay.group * vpt * 8; }

// Whether rows are whole 16-byte vectors, or at least start on such a boundary with the first one.
struct Layout {
    bool vec, wide;
};

template <typename T, typename R, int kVpt, int kRows, bool kSmallEps>
static int run_forward_ring(const Params& p, const RingLayout& lay, cudaStream_t stream) {
    int count = 0;
    if (dense(p, lay, kVpt)) return launch_ring<forward_ring_kernel<T, R, kVpt, kRows, true, true, kSmallEps>>(p, lay, kRows, &count, stream);
    return launch_ring<forward_ring_kernel<T, R, kVpt, kRows, false, true, kSmallEps>>(p, lay, kRows, &count, stream);
}

template <typename T, typename R, bool kSmallEps>
static int run_forward_of(const Params& p, Layout rows_are, cudaStream_t stream) {
    const bool vec = rows_are.vec;
    if (rows_are.wide && p.hidden >= (vec ? kRingMinHidden : kRingMinHiddenAny) && p.hidden <= (vec ? kRingMaxHidden : kRingMaxHiddenAny)) {
        const int ring_vpt = p.hidden > 4096 ? 2 : 1, rows = vec && ring_vpt == 1 ? 4 : 2;
        RingLayout lay;
        int count = 0;
        if (ring_layout<T, R>(p, vec, false, ring_vpt, rows, 2, &lay) &&
            p.rows >= static_cast<int64_t>(vec ? kRingMinChunks : kRingMinChunksAny) * sm_count() * lay.slots * rows) {
            if (!vec) return launch_ring<forward_ring_kernel<T, R, 1, 2, false, false, kSmallEps>>(p, lay, rows, &count, stream);
            return ring_vpt == 1 ? run_forward_ring<T, R, 1, 4, kSmallEps>(p, lay, stream) : run_forward_ring<T, R, 2, 2, kSmallEps>(p, lay, stream);
        }
    }
    if (p.hidden > kForwardMaxHidden) {
        forward_long_kernel<T, R><<<static_cast<unsigned>(p.rows), 1024, 0, stream>>>(p);
        return launch_status();
    }
    const int vpt = p.hidden > 512 ? 2 : 1;
    const int group = static_cast<int>(ceil_div(ceil_div(p.hidden, 8 * vpt), 32) * 32);
    const int slots = group >= kForwardThreads ? 1 : kForwardThreads / group;
    const unsigned grid = static_cast<unsigned>(ceil_div(p.rows, slots));
    const unsigned threads = static_cast<unsigned>(group * slots);
    if (vpt == 1) {
        if (vec) forward_kernel<T, R, 1, true, kSmallEps><<<grid, threads, 0, stream>>>(p, group);
        else forward_kernel<T, R, 1, false, kSmallEps><<<grid, threads, 0, stream>>>(p, group);
    } else {
        if (vec) forward_kernel<T, R, 2, true, kSmallEps><<<grid, threads, 0, stream>>>(p, group);
        else forward_kernel<T, R, 2, false, kSmallEps><<<grid, threads, 0, stream>>>(p, group);
    }
    return launch_status();
}

template <typename T, typename R>
static int run_forward(const Params& p, Layout rows_are, cudaStream_t stream) {
    return p.eps < kSmallMean ? run_forward_of<T, R, true>(p, rows_are, stream) : run_forward_of<T, R, false>(p, rows_are, stream);
}

template <typename T, typename R, int kVpt, int kRows, bool kX, bool kFull, int kCall, bool kVec = true>
static int launch_backward_ring(const Params& p, const RingLayout& lay, int* count, cudaStream_t stream) {
    return launch_ring<backward_ring_kernel<T, R, kVpt, kRows, kX, kFull, kCall, kVec>>(p, lay, kRows, count, stream);
}

template <typename T, typename R, int kVpt, int kRows>
static int run_backward_ring(const Params& p, const RingLayout& lay, bool vec, int* count, cudaStream_t stream) {
    if constexpr (kVpt == 1) {
        if (!vec && p.x == nullptr) return launch_backward_ring<T, R, kVpt, kRows, false, false, kCallAny, false>(p, lay, count, stream);
        if (!vec)
            return p.gate_mode == kGateFull ? launch_backward_ring<T, R, kVpt, kRows, true, true, kCallAny, false>(p, lay, count, stream)
                                            : launch_backward_ring<T, R, kVpt, kRows, true, false, kCallAny, false>(p, lay, count, stream);
    }
    const bool known = dense(p, lay, kVpt) && p.dy != nullptr && p.d_residual != nullptr;
    const bool all = known && p.d_stream != nullptr && p.dx != nullptr;
    if (p.x == nullptr) {
        if (all) return launch_backward_ring<T, R, kVpt, kRows, false, false, kCallAll>(p, lay, count, stream);
        if (known && p.d_stream == nullptr && p.dx == nullptr)
            return launch_backward_ring<T, R, kVpt, kRows, false, false, kCallAlone>(p, lay, count, stream);
        if (known && p.d_stream != nullptr)
            return launch_backward_ring<T, R, kVpt, kRows, false, false, kCallShared>(p, lay, count, stream);
        return launch_backward_ring<T, R, kVpt, kRows, false, false, kCallAny>(p, lay, count, stream);
    }
    if (p.gate_mode == kGateFull)
        return all ? launch_backward_ring<T, R, kVpt, kRows, true, true, kCallAll>(p, lay, count, stream)
                   : launch_backward_ring<T, R, kVpt, kRows, true, true, kCallAny>(p, lay, count, stream);
    return all ? launch_backward_ring<T, R, kVpt, kRows, true, false, kCallAll>(p, lay, count, stream)
               : launch_backward_ring<T, R, kVpt, kRows, true, false, kCallAny>(p, lay, count, stream);
}

template <typename T, typename R>
static int run_backward(const Params& p, Layout rows_are, void* d_weight, void* d_post, void* d_gate_channel, cudaStream_t stream) {
    int count = 0, status = XMA_OK;
    const int vpt = p.hidden > 4096 ? 2 : 1, rows = vpt == 1 ? 2 : 1;
    RingLayout lay;
    const bool vec = rows_are.vec;
    if (rows_are.wide && p.hidden <= (vec ? kRingMaxHidden : kRingMaxHiddenAny) && ring_layout<T, R>(p, vec, true, vpt, rows, 2, &lay)) {
        status = vpt == 1 ? run_backward_ring<T, R, 1, 2>(p, lay, vec, &count, stream) : run_backward_ring<T, R, 2, 1>(p, lay, vec, &count, stream);
    } else {
        backward_sums_kernel<T, R><<<static_cast<unsigned>(p.rows), 256, 0, stream>>>(p);
        status = launch_status();
        if (status != XMA_OK) return status;
        const int64_t per_cta = ceil_div(p.rows, kPartials);
        count = static_cast<int>(ceil_div(p.rows, per_cta));
        const dim3 grid(static_cast<unsigned>(ceil_div(p.hidden, 256)), static_cast<unsigned>(count));
        backward_elements_kernel<T, R><<<grid, 256, 0, stream>>>(p, per_cta);
        status = launch_status();
    }
    if (status != XMA_OK || (d_weight == nullptr && d_post == nullptr && d_gate_channel == nullptr)) return status;
    const dim3 grid(static_cast<unsigned>(ceil_div(p.hidden, 32)), 3);
    sum_kernel<T><<<grid, dim3(32, 8), 0, stream>>>(p, count, d_weight, d_post, d_gate_channel);
    return launch_status();
}

static Layout layout_of(const Params& p) {
    const void* ptrs[] = {p.x, p.residual, p.weight, p.post, p.gate, p.s_out, p.y, p.dy, p.d_stream, p.s, p.dx, p.d_residual, p.d_gate};
    for (int i = 0; i < static_cast<int>(sizeof(ptrs) / sizeof(ptrs[0])); ++i) {
        const bool token = p.gate_mode == kGateToken && (ptrs[i] == p.gate || ptrs[i] == p.d_gate);
        if (!token && !aligned16(ptrs[i])) return Layout{false, false};
    }
    return Layout{p.hidden % 8 == 0, true};
}

static bool size_ok(int64_t rows, int64_t hidden, int32_t gate_mode) {
    return rows >= 0 && rows <= INT32_MAX && hidden > 0 && hidden <= (1 << 24) && gate_mode >= kGateNone && gate_mode <= kGateFull;
}

}  // namespace norm
}  // namespace xma

extern "C" {

int64_t xma_norm_workspace_floats(int64_t rows, int64_t hidden) {
    if (rows < 0 || hidden < 0) return 0;
    return 3 * (rows < XMA_NORM_PARTIALS ? rows : XMA_NORM_PARTIALS) * hidden + 8 * rows;
}

int xma_norm_forward(const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate,
                     int32_t gate_mode, int32_t dtype, int32_t stream_dtype, int32_t f32_params, int64_t rows, int64_t hidden,
                     float eps, float multiplier, void* stream_out, void* y, float* rstd, float* rstd_post, int32_t* status,
                     void* stream) {
    using namespace xma;
    using namespace xma::norm;
    if (!size_ok(rows, hidden, gate_mode)) return XMA_ERR_BAD_ARG;
    if (rows == 0) return XMA_OK;
    if (!x || !y || (residual && !stream_out) || (gate_mode != kGateNone) != (gate != nullptr)) return XMA_ERR_BAD_ARG;
    if (!residual && (post_weight || gate || stream_dtype != dtype)) return XMA_ERR_BAD_ARG;
    Params p{};
    p.x = x, p.residual = residual, p.weight = weight, p.post = post_weight, p.gate = gate, p.gate_mode = gate_mode;
    p.weight_f32 = f32_params & 1, p.post_f32 = f32_params & 2, p.gate_f32 = f32_params & 4;
    p.rows = rows, p.hidden = static_cast<int>(hidden), p.eps = eps, p.multiplier = multiplier;
    p.s_out = stream_out, p.y = y, p.rs = rstd, p.rp = rstd_post, p.status = status;
    const Layout lay = layout_of(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeBF16) return run_forward<__nv_bfloat16, __nv_bfloat16>(p, lay, st);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeF32) return run_forward<__nv_bfloat16, float>(p, lay, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF16) return run_forward<__half, __half>(p, lay, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF32) return run_forward<__half, float>(p, lay, st);
    if (dtype == kDtypeF32 && stream_dtype == kDtypeF32) return run_forward<float, float>(p, lay, st);
    return XMA_ERR_UNSUPPORTED;
}

int xma_norm_backward(const void* dy, const void* d_stream, const void* stream_or_residual, const void* x, const void* weight,
                      const void* post_weight, const void* gate, int32_t gate_mode, int32_t dtype, int32_t stream_dtype,
                      int32_t f32_params, int64_t rows, int64_t hidden, float multiplier, const float* rstd,
                      const float* rstd_post, void* dx, void* d_residual, void* d_gate, void* d_weight, void* d_post_weight,
                      float* workspace, int32_t* status, void* stream) {
    using namespace xma;
    using namespace xma::norm;
    if (!size_ok(rows, hidden, gate_mode)) return XMA_ERR_BAD_ARG;
    if (rows == 0) return XMA_OK;
    if (!stream_or_residual || !rstd || !workspace || !aligned16(workspace)) return XMA_ERR_BAD_ARG;
    if ((gate_mode != kGateNone) != (gate != nullptr) || ((post_weight || gate) && !x) || (post_weight && !rstd_post))
        return XMA_ERR_BAD_ARG;
    if ((d_weight && !weight) || (d_post_weight && !post_weight) || (d_gate && !gate)) return XMA_ERR_BAD_ARG;
    Params p{};
    p.x = post_weight || gate ? x : nullptr;
    p.weight = weight, p.post = post_weight, p.gate = gate, p.gate_mode = gate_mode;
    p.weight_f32 = f32_params & 1, p.post_f32 = f32_params & 2, p.gate_f32 = f32_params & 4;
    p.rows = rows, p.hidden = static_cast<int>(hidden), p.multiplier = multiplier;
    p.rs = const_cast<float*>(rstd), p.rp = const_cast<float*>(rstd_post);
    p.dy = dy, p.d_stream = d_stream, p.s = stream_or_residual, p.dx = dx, p.d_residual = d_residual;
    p.d_gate = gate_mode == kGateChannel ? nullptr : d_gate;
    p.partial_rows = static_cast<int>(rows < kPartials ? rows : kPartials);
    p.row_sums = workspace;
    p.partials = workspace + 8 * rows;
    void* d_gate_channel = gate_mode == kGateChannel ? d_gate : nullptr;
    p.want_weight = d_weight != nullptr, p.want_post = d_post_weight != nullptr, p.want_gate = d_gate_channel != nullptr;
    p.status = status;
    const Layout lay = layout_of(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeBF16)
        return run_backward<__nv_bfloat16, __nv_bfloat16>(p, lay, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeF32)
        return run_backward<__nv_bfloat16, float>(p, lay, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF16)
        return run_backward<__half, __half>(p, lay, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF32)
        return run_backward<__half, float>(p, lay, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF32 && stream_dtype == kDtypeF32)
        return run_backward<float, float>(p, lay, d_weight, d_post_weight, d_gate_channel, st);
    return XMA_ERR_UNSUPPORTED;
}

}  // extern "C"
