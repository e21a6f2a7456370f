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
//   ds = rs (a - s rs^2 mean(a s)) + d            d_residual = ds
//   d_gate = m ds u,   b = m ds gate post,        dx = rp (b - x rp^2 mean(b x))
//   d_weight = sum_rows dy s rs,                  d_post = sum_rows m ds gate x rp
//
// sum(b x) follows from three more sums over the row's inputs (ds is linear in a, s and d), so a row
// takes ONE reduction: with c = post * gate * x,
//   sum(c ds) = rs sum(c a) - rs^3 mean(a s) sum(c s) + sum(c d).
// The mean of squares adds up (v / H) v, so that it overflows where the mean itself does and no sooner.
// All of it is bound by HBM: every tensor is read and written once.
#include "common.cuh"
#include "ptx.cuh"

namespace xma {
namespace norm {

using namespace ptx;

constexpr int kGateNone = 0;     // no gate
constexpr int kGateChannel = 1;  // [H], a parameter
constexpr int kGateToken = 2;    // [rows], one factor per row
constexpr int kGateFull = 3;     // [rows, H]

constexpr int kMaxThreads = 512;           // threads of a backward CTA that compute (a producer warp comes on top)
constexpr int kForwardThreads = 256;
constexpr int kForwardMaxHidden = 16384;   // longer rows are read once per pass
constexpr int kRingMaxHidden = 8192;       // longer rows take the two-kernel backward
constexpr int kPartials = XMA_NORM_PARTIALS;
constexpr uint32_t kRingSmem = 220 * 1024;
constexpr int kMaxStages = 4;

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
    const void* s;
    void* dx;
    void* d_residual;
    void* d_gate;
    float* partials;  // [3][kPartials][hidden]: weight, post weight, channel gate
    bool want_weight, want_post, want_gate;
    float* row_sums;  // two-kernel backward: [rows][4]
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

template <typename T>
__device__ __forceinline__ float token_gate(const Params& p, int64_t row) {
    return p.gate_mode == kGateToken ? Elem<T>::to_float(static_cast<const T*>(p.gate)[row]) : 1.f;
}

// ---------------------------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------------------------

// `group` threads per row hold it in registers (kVpt vectors of eight each); several short rows share a CTA.
template <typename T, typename R, int kVpt, bool kVec>
__global__ void __launch_bounds__(1024)
forward_kernel(const Params p, int group) {
    __shared__ float scratch[2][32];
    const int slot = threadIdx.x / group, t = threadIdx.x - slot * group;
    const int slots = blockDim.x / group;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * slots + slot;
    if (row >= p.rows) return;  // the whole group leaves: its barrier is its own
    const int64_t base = row * p.hidden;
    float* my_scratch[2] = {&scratch[0][slot * (group >> 5)], &scratch[1][slot * (group >> 5)]};
    const int barrier = 1 + slot;
    const float inv_h = 1.f / static_cast<float>(p.hidden);

    float s[kVpt][8];
#pragma unroll
    for (int v = 0; v < kVpt; ++v) load_cols<kVec>(static_cast<const T*>(p.x) + base, v, t, group, p.hidden, s[v]);
    if (p.residual != nullptr) {
        float r[kVpt][8];
#pragma unroll
        for (int v = 0; v < kVpt; ++v)
            load_cols<kVec>(static_cast<const R*>(p.residual) + base, v, t, group, p.hidden, r[v]);
        float scale = p.multiplier * token_gate<T>(p, row);
        if (p.post != nullptr) {
            float sum[1] = {0.f};
#pragma unroll
            for (int v = 0; v < kVpt; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[0] = fmaf(s[v][j] * inv_h, s[v][j], sum[0]);
            group_sum<1>(sum, my_scratch[0], t, group, barrier);
            const float rp = rsqrtf(sum[0] + p.eps);
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
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < kVpt; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[0] = fmaf(s[v][j] * inv_h, s[v][j], sum[0]);
    group_sum<1>(sum, my_scratch[1], t, group, barrier);
    const float rs = rsqrtf(sum[0] + p.eps);
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
    __shared__ float scratch[2][32];
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.hidden;
    const int t = threadIdx.x, group = blockDim.x;
    const float inv_h = 1.f / static_cast<float>(p.hidden);
    float scale = p.multiplier * token_gate<T>(p, row);
    if (p.residual != nullptr && p.post != nullptr) {
        float sum[1] = {0.f};
        for (int c = t; c < p.hidden; c += group) {
            const float v = Elem<T>::to_float(static_cast<const T*>(p.x)[base + c]);
            sum[0] = fmaf(v * inv_h, v, sum[0]);
        }
        group_sum<1>(sum, scratch[0], t, group, 1);
        const float rp = rsqrtf(sum[0] + p.eps);
        if (t == 0 && p.rp != nullptr) p.rp[row] = rp;
        scale *= rp;
    }
    float sum[1] = {0.f};
    for (int c = t; c < p.hidden; c += group) {
        const float s = stream_at<T, R>(p, base, c, scale);
        sum[0] = fmaf(s * inv_h, s, sum[0]);
    }
    group_sum<1>(sum, scratch[1], t, group, 1);
    const float rs = rsqrtf(sum[0] + p.eps);
    if (t == 0 && p.rs != nullptr) p.rs[row] = rs;
    for (int c = t; c < p.hidden; c += group) {
        const float s = stream_at<T, R>(p, base, c, scale);
        if (p.residual != nullptr) static_cast<R*>(p.s_out)[base + c] = Elem<R>::from_float(s);
        static_cast<T*>(p.y)[base + c] = Elem<T>::from_float(param_at<T>(p.weight, p.weight_f32, c) * s * rs);
    }
}

// ---------------------------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------------------------

// What the elements of a row need beside their inputs.
struct RowScale {
    float rs, rp;
    float k_s;   // rs^2 mean(a s)
    float k_x;   // rp mean(b x), with the multiplier and the token gate in it
    float m;     // multiplier * token gate
    float d_token_gate;
};
// sums: (a s), (c a), (c s), (c d)
__device__ __forceinline__ RowScale row_scale(const Params& p, const float (&sums)[4], float rs, float rp, float token) {
    RowScale r;
    const float inv_h = 1.f / static_cast<float>(p.hidden);
    r.rs = rs;
    r.rp = rp;
    r.k_s = rs * rs * sums[0] * inv_h;
    const float c_ds = rs * sums[1] - rs * r.k_s * sums[2] + sums[3];
    r.m = p.multiplier * token;
    r.k_x = r.m * rp * c_ds * inv_h;
    r.d_token_gate = p.multiplier * rp * c_ds;
    return r;
}

// Shared-memory layout of the ring kernel: parameters, reduction scratch and barriers, then the stages.
struct RingLayout {
    int slots;            // rows a CTA works on at once
    int group;            // threads per row
    int stages;
    uint32_t stage_bytes;
    uint32_t dy, d_stream, s, x, gate;  // offsets inside a stage
    uint32_t post, channel_gate;        // offsets of the parameters (the weight's is 0)
    uint32_t ring;                      // offset of stage 0
    uint32_t total;
};

constexpr uint32_t kRingHeader = 1024;  // barriers and two reduction scratches of 16 warps x 4 floats

// Persistent CTAs walk over the rows; a producer warp copies whole rows (bulk copies) into a ring of
// stages ahead of the warps that compute, so the loads in flight do not depend on registers, and the
// row's second pass reads shared memory. The gradients of the parameters stay in registers (a thread
// keeps its columns) until the CTA's last row and leave as one partial row per CTA, summed in a fixed
// order by sum_kernel.
template <typename T, typename R, int kVpt>
__global__ void __launch_bounds__(kMaxThreads + 32, 1)
backward_ring_kernel(const Params p, const RingLayout lay) {
    extern __shared__ __align__(128) uint8_t smem[];
    const uint32_t base_addr = smem_u32(smem);
    const uint32_t full_bar = base_addr, empty_bar = base_addr + 64;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + 128);
    float* scratch = reinterpret_cast<float*>(smem + 256);  // [2][16 warps][4]
    uint8_t* params_at = smem + kRingHeader;
    uint8_t* ring = smem + lay.ring;
    const int group = lay.group, slots = lay.slots;
    const int compute_threads = group * slots;
    const int64_t chunks = (p.rows + slots - 1) / slots;
    const bool has_x = p.x != nullptr;

    if (threadIdx.x == 0) {
        for (int i = 0; i < lay.stages; ++i) {
            mbar_init(full_bar + 8 * i, 1);
            mbar_init(empty_bar + 8 * i, compute_threads / 32);
        }
        *abort_flag = 0;
        fence_barrier_init();
    }
    // parameters into shared memory, in their own type
    for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) {
        if (p.weight != nullptr) {
            if (p.weight_f32) reinterpret_cast<float*>(params_at)[c] = static_cast<const float*>(p.weight)[c];
            else reinterpret_cast<T*>(params_at)[c] = static_cast<const T*>(p.weight)[c];
        }
        if (p.post != nullptr) {
            if (p.post_f32) reinterpret_cast<float*>(params_at + lay.post)[c] = static_cast<const float*>(p.post)[c];
            else reinterpret_cast<T*>(params_at + lay.post)[c] = static_cast<const T*>(p.post)[c];
        }
        if (p.gate_mode == kGateChannel) {
            if (p.gate_f32) reinterpret_cast<float*>(params_at + lay.channel_gate)[c] = static_cast<const float*>(p.gate)[c];
            else reinterpret_cast<T*>(params_at + lay.channel_gate)[c] = static_cast<const T*>(p.gate)[c];
        }
    }
    __syncthreads();

    if (threadIdx.x >= compute_threads) {
        // ------------------------------ producer warp ------------------------------
        if (threadIdx.x == compute_threads) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int64_t ch = blockIdx.x; ok && ch < chunks; ch += gridDim.x) {
                ok = mbar_wait(empty_bar + 8 * stage, phase ^ 1u, abort_flag, p.status, 401);
                if (!ok) break;
                const int64_t row0 = ch * slots;
                const uint32_t count = static_cast<uint32_t>(min(static_cast<int64_t>(slots), p.rows - row0) * p.hidden);
                const int64_t at = row0 * p.hidden;
                const uint32_t dst = base_addr + lay.ring + stage * lay.stage_bytes;
                const uint32_t bar = full_bar + 8 * stage;
                const uint32_t bytes_t = count * sizeof(T), bytes_r = count * sizeof(R);
                uint32_t expect = bytes_r;
                if (p.dy != nullptr) expect += bytes_t;
                if (p.d_stream != nullptr) expect += bytes_r;
                if (has_x) expect += bytes_t;
                if (p.gate_mode == kGateFull) expect += bytes_t;
                mbar_expect_tx(bar, expect);
                bulk_load(dst + lay.s, static_cast<const R*>(p.s) + at, bytes_r, bar);
                if (p.dy != nullptr) bulk_load(dst + lay.dy, static_cast<const T*>(p.dy) + at, bytes_t, bar);
                if (p.d_stream != nullptr) bulk_load(dst + lay.d_stream, static_cast<const R*>(p.d_stream) + at, bytes_r, bar);
                if (has_x) bulk_load(dst + lay.x, static_cast<const T*>(p.x) + at, bytes_t, bar);
                if (p.gate_mode == kGateFull) bulk_load(dst + lay.gate, static_cast<const T*>(p.gate) + at, bytes_t, bar);
                if (++stage == lay.stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            // Given up: the copies in flight land before the CTA ends (a stage's last load completed the
            // phase before the one that the next load would).
            for (int i = 0; !ok && i < lay.stages; ++i) {
                const uint32_t last = i < stage ? phase : phase ^ 1u;
                const uint64_t begin = global_timer_ns();
                while (!mbar_try_wait(full_bar + 8 * i, last) && global_timer_ns() - begin < kWaitLimitNs) {}
            }
        }
        __syncwarp();
        __syncthreads();  // the one after the compute warps' loop
        return;
    }

    // ------------------------------ compute warps ------------------------------
    const int slot = threadIdx.x / group, t = threadIdx.x - slot * group;
    const int lane = threadIdx.x & 31;
    float* my_scratch = scratch + slot * (group >> 5) * 4;
    float acc_w[kVpt][8], acc_p[kVpt][8], acc_g[kVpt][8];
#pragma unroll
    for (int v = 0; v < kVpt; ++v)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc_w[v][j] = acc_p[v][j] = acc_g[v][j] = 0.f;

    int stage = 0;
    uint32_t phase = 0, flip = 0;
    for (int64_t ch = blockIdx.x; ch < chunks; ch += gridDim.x) {
        const int64_t row = ch * slots + slot;
        const bool valid = row < p.rows;  // uniform in a row's group
        float rs = 0.f, rp = 1.f, token = 1.f;
        if (valid) {
            rs = p.rs[row];
            if (p.post != nullptr) rp = p.rp[row];
            token = token_gate<T>(p, row);
        }
        if (!mbar_wait(full_bar + 8 * stage, phase, abort_flag, p.status, 402)) break;
        const uint8_t* st = ring + stage * lay.stage_bytes;
        const int off = slot * p.hidden;
        const T* dy = reinterpret_cast<const T*>(st + lay.dy) + off;
        const R* dd = reinterpret_cast<const R*>(st + lay.d_stream) + off;
        const R* sr = reinterpret_cast<const R*>(st + lay.s) + off;
        const T* xr = reinterpret_cast<const T*>(st + lay.x) + off;
        const T* gr = reinterpret_cast<const T*>(st + lay.gate) + off;

        float sums[4] = {0.f, 0.f, 0.f, 0.f};
        if (valid) {
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                const int c = (v * group + t) * 8;
                if (c >= p.hidden) continue;
                float a[8], s8[8];
                load8(sr + c, s8);
                if (p.dy != nullptr) {
                    float w[8];
                    load8(dy + c, a);
                    load_param<true, T>(p.weight ? params_at : nullptr, p.weight_f32, v, t, group, p.hidden, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] *= w[j];
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) a[j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) sums[0] += a[j] * s8[j];
                if (has_x) {
                    float x8[8], f[8];
                    load8(xr + c, x8);
                    if (p.post != nullptr) {
                        load_param<true, T>(params_at + lay.post, p.post_f32, v, t, group, p.hidden, f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) x8[j] *= f[j];
                    }
                    if (p.gate_mode == kGateChannel || p.gate_mode == kGateFull) {
                        if (p.gate_mode == kGateFull) load8(gr + c, f);
                        else load_param<true, T>(params_at + lay.channel_gate, p.gate_f32, v, t, group, p.hidden, f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) x8[j] *= f[j];
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        sums[1] += x8[j] * a[j];
                        sums[2] += x8[j] * s8[j];
                    }
                    if (p.d_stream != nullptr) {
                        load8(dd + c, f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) sums[3] += x8[j] * f[j];
                    }
                }
            }
        }
        group_sum<4>(sums, my_scratch + flip * 64, t, group, 1 + slot);
        flip ^= 1u;
        const RowScale k = row_scale(p, sums, rs, rp, token);
        if (valid) {
            const int64_t base = row * p.hidden;
            if (p.gate_mode == kGateToken && p.d_gate != nullptr && t == 0)
                static_cast<T*>(p.d_gate)[row] = Elem<T>::from_float(k.d_token_gate);
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                const int c = (v * group + t) * 8;
                if (c >= p.hidden) continue;
                float ds[8], s8[8], f[8];
                load8(sr + c, s8);
                if (p.dy != nullptr) {
                    float d8[8];
                    load8(dy + c, d8);
                    load_param<true, T>(p.weight ? params_at : nullptr, p.weight_f32, v, t, group, p.hidden, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        acc_w[v][j] += d8[j] * (s8[j] * k.rs);
                        ds[j] = k.rs * (d8[j] * f[j] - s8[j] * k.k_s);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) ds[j] = 0.f;
                }
                if (p.d_stream != nullptr) {
                    load8(dd + c, f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) ds[j] += f[j];
                }
                if (p.d_residual != nullptr) store8(static_cast<R*>(p.d_residual) + base + c, ds);
                if (p.dx == nullptr && !has_x) continue;
                float b[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = k.m * ds[j];  // gradient of the gated branch, token gate in it
                if (has_x) {
                    float x8[8], u[8];
                    load8(xr + c, x8);
#pragma unroll
                    for (int j = 0; j < 8; ++j) u[j] = x8[j] *= k.rp;
                    if (p.post != nullptr) {
                        load_param<true, T>(params_at + lay.post, p.post_f32, v, t, group, p.hidden, f);
#pragma unroll
                        for (int j = 0; j < 8; ++j) u[j] *= f[j];
                    }
                    if (p.gate_mode == kGateChannel || p.gate_mode == kGateFull) {
                        float g[8];
                        if (p.gate_mode == kGateFull) load8(gr + c, g);
                        else load_param<true, T>(params_at + lay.channel_gate, p.gate_f32, v, t, group, p.hidden, g);
#pragma unroll
                        for (int j = 0; j < 8; ++j) u[j] *= b[j];  // d gate
                        if (p.gate_mode == kGateFull) {
                            if (p.d_gate != nullptr) store8(static_cast<T*>(p.d_gate) + base + c, u);
                        } else {
#pragma unroll
                            for (int j = 0; j < 8; ++j) acc_g[v][j] += u[j];
                        }
#pragma unroll
                        for (int j = 0; j < 8; ++j) b[j] *= g[j];
                    }
                    if (p.post != nullptr) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            acc_p[v][j] += b[j] * x8[j];
                            b[j] = k.rp * (b[j] * f[j] - x8[j] * k.k_x);
                        }
                    }
                }
                if (p.dx != nullptr) store8(static_cast<T*>(p.dx) + base + c, b);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty_bar + 8 * stage);
        if (++stage == lay.stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    __syncthreads();  // with the producer: every load has landed and been read, the ring is free

    // The slots' sums, added in slot order, leave as this CTA's partial rows.
    float* buf = reinterpret_cast<float*>(ring);
    const bool want[3] = {p.want_weight, p.want_post, p.want_gate};
#pragma unroll
    for (int which = 0; which < 3; ++which) {
        if (!want[which]) continue;
        float(&acc)[kVpt][8] = which == 0 ? acc_w : which == 1 ? acc_p : acc_g;
        float* out = p.partials + (static_cast<int64_t>(which) * kPartials + blockIdx.x) * p.hidden;
        if (slots == 1) {
#pragma unroll
            for (int v = 0; v < kVpt; ++v) {
                const int c = (v * group + t) * 8;
                if (c < p.hidden) store8(out + c, acc[v]);
            }
            continue;
        }
#pragma unroll
        for (int v = 0; v < kVpt; ++v) {
            const int c = (v * group + t) * 8;
            if (c < p.hidden) store8(buf + slot * p.hidden + c, acc[v]);
        }
        group_barrier(0, compute_threads);
        for (int c = threadIdx.x; c < p.hidden; c += compute_threads) {
            float total = 0.f;
            for (int sl = 0; sl < slots; ++sl) total += buf[sl * p.hidden + c];
            out[c] = total;
        }
        group_barrier(0, compute_threads);
    }
}

// The elements of one position, from global memory (two-kernel backward).
template <typename T, typename R>
struct Element {
    float dy, s, d, x, w, post, gate;
    __device__ __forceinline__ Element(const Params& p, int64_t base, int c) {
        dy = p.dy != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.dy)[base + c]) : 0.f;
        s = Elem<R>::to_float(static_cast<const R*>(p.s)[base + c]);
        d = p.d_stream != nullptr ? Elem<R>::to_float(static_cast<const R*>(p.d_stream)[base + c]) : 0.f;
        x = p.x != nullptr ? Elem<T>::to_float(static_cast<const T*>(p.x)[base + c]) : 0.f;
        w = param_at<T>(p.weight, p.weight_f32, c);
        post = param_at<T>(p.post, p.post_f32, c);
        gate = p.gate_mode == kGateFull      ? Elem<T>::to_float(static_cast<const T*>(p.gate)[base + c])
               : p.gate_mode == kGateChannel ? param_at<T>(p.gate, p.gate_f32, c)
                                             : 1.f;
    }
};

// Any row length and alignment, in two kernels: the row sums, then the elements (a block of columns
// times a share of the rows per CTA, so that the parameters' gradients are sums in registers).
template <typename T, typename R>
__global__ void __launch_bounds__(256)
backward_sums_kernel(const Params p) {
    __shared__ float scratch[8 * 4];
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.hidden;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < p.hidden; c += blockDim.x) {
        const Element<T, R> e(p, base, c);
        const float a = e.dy * e.w, q = e.x * e.post * e.gate;
        sums[0] += a * e.s;
        sums[1] += q * a;
        sums[2] += q * e.s;
        sums[3] += q * e.d;
    }
    group_sum<4>(sums, scratch, threadIdx.x, blockDim.x, 1);
    if (threadIdx.x < 4) p.row_sums[row * 4 + threadIdx.x] = sums[threadIdx.x];
}

template <typename T, typename R>
__global__ void __launch_bounds__(256)
backward_elements_kernel(const Params p, int64_t rows_per_cta) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * rows_per_cta;
    const int64_t last = min(first + rows_per_cta, p.rows);
    float acc_w = 0.f, acc_p = 0.f, acc_g = 0.f;
    if (c >= p.hidden) return;
    for (int64_t row = first; row < last; ++row) {
        const int64_t base = row * p.hidden;
        const Element<T, R> e(p, base, c);
        float sums[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[i] = p.row_sums[row * 4 + i];
        const RowScale k = row_scale(p, sums, p.rs[row], p.post != nullptr ? p.rp[row] : 1.f, token_gate<T>(p, row));
        if (p.gate_mode == kGateToken && p.d_gate != nullptr && c == 0)
            static_cast<T*>(p.d_gate)[row] = Elem<T>::from_float(k.d_token_gate);
        acc_w += e.dy * (e.s * k.rs);
        const float ds = k.rs * (e.dy * e.w - e.s * k.k_s) + e.d;
        if (p.d_residual != nullptr) static_cast<R*>(p.d_residual)[base + c] = Elem<R>::from_float(ds);
        float b = k.m * ds;
        const float hat = e.x * k.rp;
        const float dg = b * hat * e.post;
        if (p.gate_mode == kGateFull && p.d_gate != nullptr) static_cast<T*>(p.d_gate)[base + c] = Elem<T>::from_float(dg);
        acc_g += dg;
        b *= e.gate;
        if (p.post != nullptr) {
            acc_p += b * hat;
            b = k.rp * (b * e.post - hat * k.k_x);
        }
        if (p.dx != nullptr) static_cast<T*>(p.dx)[base + c] = Elem<T>::from_float(b);
    }
    const int64_t at = static_cast<int64_t>(blockIdx.y) * p.hidden + c;
    const int64_t plane = static_cast<int64_t>(kPartials) * p.hidden;
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
    const float* src = p.partials + static_cast<int64_t>(which) * kPartials * p.hidden + c;
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

template <typename T, typename R>
static int run_forward(const Params& p, bool vec, cudaStream_t stream) {
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
        if (vec) forward_kernel<T, R, 1, true><<<grid, threads, 0, stream>>>(p, group);
        else forward_kernel<T, R, 1, false><<<grid, threads, 0, stream>>>(p, group);
    } else {
        if (vec) forward_kernel<T, R, 2, true><<<grid, threads, 0, stream>>>(p, group);
        else forward_kernel<T, R, 2, false><<<grid, threads, 0, stream>>>(p, group);
    }
    return launch_status();
}

// Fills the ring's layout; false when not even one stage of one row fits.
template <typename T, typename R>
static bool ring_layout(const Params& p, int vpt, RingLayout* lay) {
    const uint32_t h = static_cast<uint32_t>(p.hidden);
    lay->group = static_cast<int>(ceil_div(ceil_div(h, 8 * vpt), 32) * 32);
    if (lay->group > kMaxThreads) return false;
    lay->slots = kMaxThreads / lay->group;
    const uint32_t row_t = h * sizeof(T), row_r = h * sizeof(R);
    uint32_t at = p.weight == nullptr ? 0 : h * (p.weight_f32 ? 4 : sizeof(T));
    lay->post = at;
    if (p.post != nullptr) at += h * (p.post_f32 ? 4 : sizeof(T));
    lay->channel_gate = at;
    if (p.gate_mode == kGateChannel) at += h * (p.gate_f32 ? 4 : sizeof(T));
    lay->ring = (kRingHeader + at + 127u) & ~127u;
    // halve the rows a CTA takes at once until two stages fit
    for (;;) {
        const uint32_t n = static_cast<uint32_t>(lay->slots);
        uint32_t off = 0;
        lay->s = off, off += n * row_r;
        lay->dy = off, off += p.dy != nullptr ? n * row_t : 0;
        lay->d_stream = off, off += p.d_stream != nullptr ? n * row_r : 0;
        lay->x = off, off += p.x != nullptr ? n * row_t : 0;
        lay->gate = off, off += p.gate_mode == kGateFull ? n * row_t : 0;
        lay->stage_bytes = (off + 127u) & ~127u;
        lay->stages = static_cast<int>((kRingSmem - lay->ring) / lay->stage_bytes);
        if (lay->stages >= 2 || lay->slots == 1) break;
        lay->slots /= 2;
    }
    if (lay->stages > kMaxStages) lay->stages = kMaxStages;
    if (lay->stages < 1) return false;
    uint32_t ring = lay->stage_bytes * static_cast<uint32_t>(lay->stages);
    const uint32_t reduce = lay->slots > 1 ? static_cast<uint32_t>(lay->slots) * h * 4 : 0;
    if (ring < reduce) ring = reduce;
    lay->total = lay->ring + ring;
    return lay->total <= kRingSmem;
}

template <typename T, typename R, int kVpt>
static int launch_ring(const Params& p, const RingLayout& lay, int* count, cudaStream_t stream) {
    auto kernel = backward_ring_kernel<T, R, kVpt>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRingSmem)) != cudaSuccess) {
        cudaGetLastError();
        return XMA_ERR_LAUNCH;
    }
    int64_t grid = ceil_div(p.rows, lay.slots);
    const int64_t most = sm_count() < kPartials ? sm_count() : kPartials;
    if (grid > most) grid = most;
    *count = static_cast<int>(grid);
    kernel<<<static_cast<unsigned>(grid), static_cast<unsigned>(lay.group * lay.slots + 32), lay.total, stream>>>(p, lay);
    return launch_status();
}

template <typename T, typename R>
static int run_backward(const Params& p, bool vec, void* d_weight, void* d_post, void* d_gate_channel, cudaStream_t stream) {
    int count = 0, status = XMA_OK;
    const int vpt = p.hidden > 512 ? 2 : 1;
    RingLayout lay;
    if (vec && p.hidden <= kRingMaxHidden && ring_layout<T, R>(p, vpt, &lay)) {
        status = vpt == 1 ? launch_ring<T, R, 1>(p, lay, &count, stream) : launch_ring<T, R, 2>(p, lay, &count, stream);
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

static bool all_aligned(const Params& p) {
    const void* ptrs[] = {p.x, p.residual, p.weight, p.post, p.gate, p.s_out, p.y, p.dy, p.d_stream, p.s, p.dx, p.d_residual, p.d_gate};
    for (int i = 0; i < static_cast<int>(sizeof(ptrs) / sizeof(ptrs[0])); ++i) {
        const bool token = p.gate_mode == kGateToken && (ptrs[i] == p.gate || ptrs[i] == p.d_gate);
        if (!token && !aligned16(ptrs[i])) return false;
    }
    return p.hidden % 8 == 0;
}

static bool size_ok(int64_t rows, int64_t hidden, int32_t gate_mode) {
    return rows >= 0 && rows <= INT32_MAX && hidden > 0 && hidden <= (1 << 24) && gate_mode >= kGateNone && gate_mode <= kGateFull;
}

}  // namespace norm
}  // namespace xma

extern "C" {

int64_t xma_norm_workspace_floats(int64_t rows, int64_t hidden) {
    return rows < 0 || hidden < 0 ? 0 : 3 * static_cast<int64_t>(XMA_NORM_PARTIALS) * hidden + 4 * rows;
}

int xma_norm_forward(const void* x, const void* residual, const void* weight, const void* post_weight, const void* gate,
                     int32_t gate_mode, int32_t dtype, int32_t stream_dtype, int32_t f32_params, int64_t rows, int64_t hidden,
                     float eps, float multiplier, void* stream_out, void* y, float* rstd, float* rstd_post, void* stream) {
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
    p.s_out = stream_out, p.y = y, p.rs = rstd, p.rp = rstd_post;
    const bool vec = all_aligned(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeBF16) return run_forward<__nv_bfloat16, __nv_bfloat16>(p, vec, st);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeF32) return run_forward<__nv_bfloat16, float>(p, vec, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF16) return run_forward<__half, __half>(p, vec, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF32) return run_forward<__half, float>(p, vec, st);
    if (dtype == kDtypeF32 && stream_dtype == kDtypeF32) return run_forward<float, float>(p, vec, st);
    return XMA_ERR_UNSUPPORTED;
}

int xma_norm_backward(const void* dy, const void* d_stream, const void* stream_saved, const void* x, const void* weight,
                      const void* post_weight, const void* gate, int32_t gate_mode, int32_t dtype, int32_t stream_dtype,
                      int32_t f32_params, int64_t rows, int64_t hidden, float multiplier, const float* rstd,
                      const float* rstd_post, void* dx, void* d_residual, void* d_gate, void* d_weight, void* d_post_weight,
                      float* workspace, int32_t* status, void* stream) {
    using namespace xma;
    using namespace xma::norm;
    if (!size_ok(rows, hidden, gate_mode)) return XMA_ERR_BAD_ARG;
    if (rows == 0) return XMA_OK;
    if (!stream_saved || !rstd || !workspace || !aligned16(workspace)) return XMA_ERR_BAD_ARG;
    if ((gate_mode != kGateNone) != (gate != nullptr) || ((post_weight || gate) && !x) || (post_weight && !rstd_post))
        return XMA_ERR_BAD_ARG;
    if ((d_weight && !weight) || (d_post_weight && !post_weight) || (d_gate && !gate)) return XMA_ERR_BAD_ARG;
    Params p{};
    p.x = post_weight || gate ? x : nullptr;
    p.weight = weight, p.post = post_weight, p.gate = gate, p.gate_mode = gate_mode;
    p.weight_f32 = f32_params & 1, p.post_f32 = f32_params & 2, p.gate_f32 = f32_params & 4;
    p.rows = rows, p.hidden = static_cast<int>(hidden), p.multiplier = multiplier;
    p.rs = const_cast<float*>(rstd), p.rp = const_cast<float*>(rstd_post);
    p.dy = dy, p.d_stream = d_stream, p.s = stream_saved, p.dx = dx, p.d_residual = d_residual;
    p.d_gate = gate_mode == kGateChannel ? nullptr : d_gate;
    p.partials = workspace;
    p.row_sums = workspace + 3 * static_cast<int64_t>(kPartials) * hidden;
    void* d_gate_channel = gate_mode == kGateChannel ? d_gate : nullptr;
    p.want_weight = d_weight != nullptr, p.want_post = d_post_weight != nullptr, p.want_gate = d_gate_channel != nullptr;
    p.status = status;
    const bool vec = all_aligned(p);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeBF16)
        return run_backward<__nv_bfloat16, __nv_bfloat16>(p, vec, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeBF16 && stream_dtype == kDtypeF32)
        return run_backward<__nv_bfloat16, float>(p, vec, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF16)
        return run_backward<__half, __half>(p, vec, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF16 && stream_dtype == kDtypeF32)
        return run_backward<__half, float>(p, vec, d_weight, d_post_weight, d_gate_channel, st);
    if (dtype == kDtypeF32 && stream_dtype == kDtypeF32)
        return run_backward<float, float>(p, vec, d_weight, d_post_weight, d_gate_channel, st);
    return XMA_ERR_UNSUPPORTED;
}

}  // extern "C"
