// block_norm.cu -- the norms around a transformer block, with its gate, residual and residual scale, in one pass:
//   n = rms(y; eps) * post_w,   r = scale * (resid + gate * n),   z = rms(r; eps) * norm_w
// r is written as the new residual; z as bf16 (with its max |.|, the dynamic scale of an NVFP4 quantiser) and/or as MXFP4
// codes and scales.  Each input is read once and each output written once; DRAM bounds it at prefill sizes.
//
// Two kernels: a row per warp from a few rows per SM on (block_norm_rows_kernel, below), else a row per CTA.  This one:
// persistent CTAs, one row at a time, 8 consecutive elements per thread and chunk.  The rows of y and resid come by
// bulk copies into a ring of two shared-memory stages, so the next row is on its way while this one goes through its
// two or three block-wide barriers (a first version with a CTA per row and loads into registers spent its time
// waiting: 148 us for 8192 x 2816 bf16 with a gate to MXFP4).  NCH chunks per thread: 2 or 4 at many rows (small
// CTAs, several per SM), 1 at few (the shortest path through a row).
//
// The codes stored are those of the float64 z.  With u = 2^-24 a sum of squares is off by at most 17 u of itself (4
// fused steps and a join per chunk, 3 chunk joins, 5 + 4 tree levels), 1 / rms by 10 u, r by 15 u a with a = |scale|
// (|resid| + |gate n|), and z by
//   d = |f w| A (28 u + 16 u k),   A = max a of the chunk,  k = sqrt(sum a^2 / sum r^2),  f = 1 / rms(r),
// without y (r is one product) by 16 u |z|.  Where the codes of z - d and z + d differ (one row in eight at 2816
// elements; one in forty without y), or a sum of squares leaves the range in which the bounds hold, the CTA takes the
// row's sums in float64 and redoes the blocks that need it.
//
// Products are taken as (x f) w, f = 1 / rms(x): |x f| is at most sqrt(H), so what overflows is an overflow of the result,
// while w f may leave fp32 at either end for finite values (w = 2^121 over rows of 2^-14 gave NaN for their zeros).  What
// underflows is off by 2^-150 times the factors behind it (a row whose gate / rms(y) does is redone); a block is redone where
// its maximum is below 2^-60, beside which that does not count as long as 1 / rms(r) and the two weights of an element make
// less than 2^60.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>

#include "common.cuh"
#include "mx.cuh"
#include "sm100.cuh"

namespace nvfp4b {
namespace {

enum Src : int { kNone = 0, kBf16 = 1, kF32 = 2 };
__host__ __device__ constexpr int src_size(Src s) { return s == kF32 ? 4 : s == kBf16 ? 2 : 0; }

constexpr int kNormMaxThreads = 512;
constexpr int kNormMaxSmem = 220 * 1024;
constexpr int kRowWarps = 16;                            // row kernel: warps per CTA, at most

struct NormParams {
    nvfp4b_block_norm_args a;
    int tile_cols;
    float inv_h;
    int chunks16;        // 8-element chunks, rounded up to the 16 of a scale word
    int weight_bytes;    // row kernel: shared memory of the weights
    int in_place;        // an output starts where an input does
    int stages;          // ring depth, 1 or 2
    int y_bytes;         // offset of the resid row in a stage
    int stage_bytes;
    int gate_vec;        // per-feature gate values may be read 16 bytes at a time
    int* err;
};

// Chunk of 8 values as four pairs.
struct V8 {
    float2 p[4];
    __device__ __forceinline__ float at(int i) const { return (i & 1) ? p[i >> 1].y : p[i >> 1].x; }
};

__device__ __forceinline__ V8 unpack8(uint4 q) {
    V8 v;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v.p[j] = make_float2(bf16lo(w[j]), bf16hi(w[j]));
    return v;
}

template <Src S>
__device__ __forceinline__ V8 load8(const void* row, int ch) {
    if constexpr (S == kF32) {
        V8 v;
        const float4 q0 = static_cast<const float4*>(row)[2 * ch], q1 = static_cast<const float4*>(row)[2 * ch + 1];
        v.p[0] = make_float2(q0.x, q0.y);
        v.p[1] = make_float2(q0.z, q0.w);
        v.p[2] = make_float2(q1.x, q1.y);
        v.p[3] = make_float2(q1.z, q1.w);
        return v;
    } else {
        return unpack8(static_cast<const uint4*>(row)[ch]);
    }
}

__device__ __forceinline__ V8 fill8(float x) {
    V8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v.p[j] = make_float2(x, x);
    return v;
}

__device__ __forceinline__ V8 weight8(const void* w, int ch) {
    return w ? unpack8(__ldg(static_cast<const uint4*>(w) + ch)) : fill8(1.f);
}

__device__ __forceinline__ uint4 pack8(const V8& v) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v.p[j].x, v.p[j].y);
        w[j] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Gate of element (row, i): per token, per feature or per element by its strides.
__device__ __forceinline__ float gate_at(const nvfp4b_block_norm_args& a, int row, int i) {
    const long long o = row * a.gate_row_stride + (long long)i * a.gate_col_stride;
    return a.gate_f32 ? __ldg(static_cast<const float*>(a.gate) + o)
                      : __uint_as_float((uint32_t)__ldg(static_cast<const uint16_t*>(a.gate) + o) << 16);
}

// Gates of the 8 elements of a chunk (gate_col_stride = 1).
__device__ __forceinline__ V8 gate8(const NormParams& p, int row, int ch) {
    const nvfp4b_block_norm_args& a = p.a;
    if (p.gate_vec) {
        if (a.gate_f32) return load8<kF32>(static_cast<const float*>(a.gate) + row * a.gate_row_stride, ch);
        return load8<kBf16>(static_cast<const uint16_t*>(a.gate) + row * a.gate_row_stride, ch);
    }
    V8 g;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        g.p[j] = make_float2(gate_at(a, row, ch * 8 + 2 * j), gate_at(a, row, ch * 8 + 2 * j + 1));
    return g;
}

// Whether an element of both is not zero.
__device__ __forceinline__ bool both_nonzero(const V8& a, const V8& b) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= a.at(i) != 0.f && b.at(i) != 0.f;
    return any;
}

// Whether a chunk whose gate * n is zero has an element with y, weight (NULL = ones) and gate all nonzero.
template <Src Y>
__device__ __noinline__ bool lost_product(const NormParams& p, int row, int ch, float g_row, const void* y, const void* w) {
    const V8 n = load8<Y>(y, ch);
    if (g_row == 0.f || !both_nonzero(n, n)) return false;
    const V8 m = w ? unpack8(static_cast<const uint4*>(w)[ch]) : fill8(1.f);
    const V8 g = p.a.gate && p.a.gate_col_stride ? gate8(p, row, ch) : fill8(1.f);
    bool any = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) any |= n.at(i) != 0.f && m.at(i) != 0.f && g.at(i) != 0.f;
    return any;
}

__device__ __forceinline__ float sum_sq(const V8& v) {
    float2 s = __fmul2_rn(v.p[0], v.p[0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) s = __ffma2_rn(v.p[j], v.p[j], s);
    return s.x + s.y;
}

// Block-wide sums, the same bits on every thread.  `red` must not be in use.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : T(0);
#pragma unroll
    for (int o = 8; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return __shfl_sync(0xFFFFFFFFu, v, 0);
}

__device__ __forceinline__ float2 block_sum2(float2 v, float2* red) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, o);
        v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
    }
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : make_float2(0.f, 0.f);
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        v.x += __shfl_xor_sync(0xFFFFFFFFu, v.x, o);
        v.y += __shfl_xor_sync(0xFFFFFFFFu, v.y, o);
    }
    return make_float2(__shfl_sync(0xFFFFFFFFu, v.x, 0), __shfl_sync(0xFFFFFFFFu, v.y, 0));
}

template <typename T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Sum of squares of a lane's chunks, compensated (each addition's rounding error is kept), and over the warp in float64.
struct SumSq {
    float hi = 0.f, lo = 0.f;
    __device__ __forceinline__ void add(const V8& v) {
        const float2 q0 = __ffma2_rn(v.p[1], v.p[1], __fmul2_rn(v.p[0], v.p[0]));
        const float2 q1 = __ffma2_rn(v.p[3], v.p[3], __fmul2_rn(v.p[2], v.p[2]));
        const float2 q = __fadd2_rn(q0, q1);
        const float x = q.x + q.y, s = hi + x, b = s - hi;
        lo += (hi - (s - b)) + (x - b);
        hi = s;
    }
    __device__ __forceinline__ float total() const { return (float)warp_sum((double)hi + (double)lo); }
};

__device__ __forceinline__ float max_abs(const V8& v) {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(v.p[j].x), fabsf(v.p[j].y)));
    return m;
}

__device__ __forceinline__ void store_resid(const nvfp4b_block_norm_args& a, int row, int ch, const V8& r) {
    if (a.resid_out_f32) {
        float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.resid_out) + row * a.ld_resid_out) + 2 * ch;
        o[0] = make_float4(r.p[0].x, r.p[0].y, r.p[1].x, r.p[1].y);
        o[1] = make_float4(r.p[2].x, r.p[2].y, r.p[3].x, r.p[3].y);
    } else {
        reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.resid_out) + row * a.ld_resid_out)[ch] = pack8(r);
    }
}

// Returns the largest magnitude (bf16 bits) of the stored values.
__device__ __forceinline__ uint32_t store_out(const nvfp4b_block_norm_args& a, int row, int ch, const V8& z) {
    const uint4 q = pack8(z);
    reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.ld_out)[ch] = q;
    const uint32_t w = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu),
                                __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
    return max(w & 0xFFFFu, w >> 16);
}

// Padding rows of the last scale tile row, dealt over all threads of the grid.
__device__ __forceinline__ void zero_padding_rows(const NormParams& p) {
    const nvfp4b_block_norm_args& a = p.a;
    const int words = (int)(((long long)a.T + 127) / 128 * 128 - a.T) * p.tile_cols;
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < words; i += gridDim.x * blockDim.x)
        *reinterpret_cast<uint32_t*>(a.scales + mx_scale_offset(a.T + i / p.tile_cols, 4 * (i % p.tile_cols),
                                                                p.tile_cols)) = 0u;
}

// The float64 redo of a row: conversions, at an eighth of the fp32 rate, are what it costs.  The product of two bf16 values
// is exact in fp32, but for underflow and overflow, and then one conversion serves both.  Squares: only a `wild` row holds
// any whose underflow or overflow counts in the sum.  y post_weight: such a product may be all that an element is made of,
// so chunks with one below 2^-130 (16 bits end at 2^-149 from 2^-134 down) of factors that are not 0, or infinite, go the
// long way.
template <Src Y>
__device__ __forceinline__ void weighted64(const V8& y, const V8& w, double (&t)[8]) {
    bool exact = Y == kBf16;
    if constexpr (Y == kBf16) {
        float lo = __int_as_float(0x7F800000), hi = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = fabsf(y.at(i) * w.at(i));
            lo = fminf(lo, q);
            hi = fmaxf(hi, q);
        }
        exact = hi < __int_as_float(0x7F800000);
        if (lo <= 0x1p-130f) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                exact &= fabsf(y.at(i) * w.at(i)) > 0x1p-130f || y.at(i) == 0.f || w.at(i) == 0.f;
        }
    }
    if (exact) {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (double)(y.at(i) * w.at(i));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = (double)y.at(i) * (double)w.at(i);
    }
}

template <Src S>
__device__ __forceinline__ double sum_sq64(const V8& v, bool wild) {
    double q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        q[i] = S == kBf16 && !wild ? (double)(v.at(i) * v.at(i)) : (double)v.at(i) * (double)v.at(i);
    return ((q[0] + q[1]) + (q[2] + q[3])) + ((q[4] + q[5]) + (q[6] + q[7]));
}

// The root of r's mean of squares, to divide by: x times its reciprocal, corrected by the remainder, is the rounded quotient
// (in signs that leave a zero its own).  Without the correction it is an ulp off where the quotient lies on a border, as
// sqrt(H) does for a row's only element.  An infinite root divides to 0: reciprocal 0, no remainder.
struct Rms64 {
    double root, inv;
    __device__ __forceinline__ explicit Rms64(double mean) : root(sqrt(mean)), inv(1.0 / root) {
        if (inv == 0.0) root = 0.0;
    }
    __device__ __forceinline__ double divide(double x) const {
        const double q = x * inv;
        return fma(-fma(q, root, -x), inv, q);
    }
};

// r of a chunk in float64, by the operations of its definition in their order (an exact zero keeps its sign); w = the post
// weights of the chunk, fg = 1 / rms(y), times the gate unless it is per feature.
template <Src Y, Src R>
__device__ __forceinline__ void r64(const NormParams& p, int row, int ch, const void* sy, const void* sr, const V8& w,
                                    double fg, double (&v)[8]) {
    const nvfp4b_block_norm_args& a = p.a;
    const V8 x = a.resid ? load8<R>(sr, ch) : fill8(0.f);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (double)x.at(i);
    if constexpr (Y != kNone) {
        const bool g_col = a.gate && a.gate_col_stride;
        const V8 g = g_col ? gate8(p, row, ch) : fill8(1.f);
        double t[8];
        weighted64<Y>(load8<Y>(sy, ch), w, t);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fma(g_col ? t[i] * (double)g.at(i) : t[i], fg, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= (double)a.scale;
}

// What has to agree in the codes of both ends.  With y the bound is absolute; without, it is relative to each element, so signs
// are not in doubt: those of zeros differ at the lower end, x - x rel, and the upper one keeps them.
template <bool HAS_Y>
constexpr uint32_t kCodeBits = HAS_Y ? 0xFFFFFFFFu : 0x77777777u;

// Whether a mean of squares (+ eps) is in the range where its fp32 value has its relative error bound.
__device__ __forceinline__ bool mean_ok(float m) { return m > 0x1p-80f && m < 0x1p100f; }

template <Src Y, Src R, int NCH, bool MX>
__global__ void __launch_bounds__(kNormMaxThreads, 1) block_norm_kernel(const __grid_constant__ NormParams p) {
    using namespace sm100;
    constexpr bool HAS_Y = Y != kNone;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ float red_y[kNormMaxThreads / 32];
    __shared__ float2 red_r[2][kNormMaxThreads / 32];
    __shared__ double red64[2][kNormMaxThreads / 32];
    __shared__ uint32_t red_max[kNormMaxThreads / 32];
    __shared__ uint64_t full[2];
    __shared__ int timeout;
    const nvfp4b_block_norm_args& a = p.a;
    const int tid = threadIdx.x, threads = blockDim.x, chunks = a.H >> 3;
    const bool want_z = MX || a.out != nullptr;

    auto fetch = [&](int row, int stage) {              // thread 0: the rows of y and resid into a stage
        uint8_t* s = ring + stage * p.stage_bytes;
        const uint32_t yb = (uint32_t)(a.H * src_size(Y)), rb = a.resid ? (uint32_t)(a.H * src_size(R)) : 0u;
        mbar_arrive_expect_tx(&full[stage], yb + rb);
        if constexpr (HAS_Y)
            bulk_load(s, static_cast<const uint8_t*>(a.y) + row * a.ld_y * src_size(Y), yb, &full[stage]);
        if (rb)
            bulk_load(s + p.y_bytes, static_cast<const uint8_t*>(a.resid) + row * a.ld_resid * src_size(R), rb,
                      &full[stage]);
    };
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        timeout = 0;
        fence_mbar_init();
        for (int s = 0; s < p.stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < a.T) fetch((int)row, s);
        }
    }
    __syncthreads();

    uint32_t zmax = 0, phase = 0;
    int stage = 0, odd = 0;
    for (long long lrow = blockIdx.x; lrow < a.T; lrow += gridDim.x) {
        const int row = (int)lrow;
        const uint8_t* sy = ring + stage * p.stage_bytes;
        const uint8_t* sr = sy + p.y_bytes;
        float2 g_row = make_float2(1.f, 1.f);
        if (HAS_Y && a.gate && !a.gate_col_stride) g_row.x = g_row.y = gate_at(a, row, 0);
        mbar_wait(&full[stage], phase, &timeout, kErrTimeoutProducer);   // on expiry the kernel goes on and reports

        V8 r[NCH];
        float top[NCH];                                  // A of the chunk
        float ss = 0.f, sa = 0.f;
        bool wild = false;                               // a sum of squares out of range (the same on every thread)
        float f = 1.f;
        if constexpr (HAS_Y) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = tid + c * threads;
                r[c] = ch < chunks ? load8<Y>(sy, ch) : fill8(0.f);
                ss += sum_sq(r[c]);
            }
            if (a.post_norm) {
                const float m = fmaf(block_sum(ss, red_y), p.inv_h, a.eps);
                wild |= !mean_ok(m);
                f = __frsqrt_rn(m);
            }
            const float2 fg = make_float2(f * g_row.x, f * g_row.y), scale = make_float2(a.scale, a.scale);
            wild |= fabsf(fg.x) < 0x1p-126f && g_row.x != 0.f;
            ss = 0.f;
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = tid + c * threads;
                top[c] = 0.f;
                if (ch >= chunks) continue;
                const V8 w = weight8(a.post_weight, ch);
                const V8 v = a.resid ? load8<R>(sr, ch) : fill8(0.f);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[c].p[j] = __fmul2_rn(__fmul2_rn(r[c].p[j], fg), w.p[j]);
                if (a.gate && a.gate_col_stride) {
                    const V8 g = gate8(p, row, ch);
#pragma unroll
                    for (int j = 0; j < 4; ++j) r[c].p[j] = __fmul2_rn(r[c].p[j], g.p[j]);
                }
                float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = r[c].p[j];
                    r[c].p[j] = __fmul2_rn(__fadd2_rn(v.p[j], t), scale);
                    if constexpr (MX) {
                        const float2 b = make_float2(fabsf(v.p[j].x) + fabsf(t.x), fabsf(v.p[j].y) + fabsf(t.y));
                        top[c] = fmaxf(top[c], fmaxf(b.x, b.y));
                        s2 = __ffma2_rn(b, b, s2);
                    }
                }
                if constexpr (MX) sa += s2.x + s2.y;
                if (want_z) ss += sum_sq(r[c]);
            }
        } else {
            const float2 scale = make_float2(a.scale, a.scale);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = tid + c * threads;
                r[c] = ch < chunks ? load8<R>(sr, ch) : fill8(0.f);
#pragma unroll
                for (int j = 0; j < 4; ++j) r[c].p[j] = __fmul2_rn(r[c].p[j], scale);
                ss += sum_sq(r[c]);
            }
        }

        V8 z[NCH];
        uint32_t code[NCH], byte[NCH];
        uint32_t redo = 0;                               // bit c: the block of chunk c is not proven
        if (want_z) {
            float rel = 0x1p-20f;                        // 16 u, or 28 u + 16 u k
            if (MX && HAS_Y) {
                const float2 s = block_sum2(make_float2(ss, sa), red_r[odd]);
                ss = s.x;
                const float k = fabsf(a.scale) * sqrtf(s.y / ss);
                if (s.y < 0x1p-100f)                     // lost bits; unless scale brings r back, m is eps (or out of
                    rel = fabsf(a.scale) <= 32.f ? 0x1.cp-20f : 1.f;   // range) and k does not enter
                else
                    rel = fmaf(k, 0x1p-20f, 0x1.cp-20f);
                wild |= !(rel < 0x1p-12f);               // also where ss = 0 < sa: r cancelled altogether
            } else {
                ss = block_sum(ss, reinterpret_cast<float*>(red_r[odd]));
            }
            const float m = fmaf(ss, p.inv_h, a.eps);
            wild |= !mean_ok(m);
            f = __frsqrt_rn(m);
            auto lost_zeros = [&](int c, int ch, float wm, const V8& w) {        // chunk c, of a block of zeros
                if constexpr (!HAS_Y) return ch < chunks && both_nonzero(load8<R>(sr, ch), w);
                else if (top[c] > 0.f) return wm > 0.f;
                else return wm > 0.f && lost_product<Y>(p, row, ch, g_row.x, sy, a.post_weight);
            };
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = tid + c * threads;
                const V8 w = ch < chunks ? weight8(a.norm_weight, ch) : fill8(0.f);
                const float2 f2 = make_float2(f, f);
                float zm = 0.f, wm = 0.f;
                float2 all = make_float2(0.f, 0.f);      // NaN if a z is (a NaN weight passes every maximum)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    z[c].p[j] = __fmul2_rn(__fmul2_rn(r[c].p[j], f2), w.p[j]);
                    if constexpr (MX) all = __fadd2_rn(all, z[c].p[j]);
                    zm = fmaxf(zm, fmaxf(fabsf(z[c].p[j].x), fabsf(z[c].p[j].y)));
                    if (MX && HAS_Y) wm = fmaxf(wm, fmaxf(fabsf(w.p[j].x), fabsf(w.p[j].y)));
                }
                if constexpr (MX) {
                    const float d = HAS_Y ? f * fabsf(a.scale) * top[c] * rel : rel;   // per unit of w, or of z
                    float dm = HAS_Y ? wm * d : zm * rel;
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        zm = fmaxf(zm, __shfl_xor_sync(0xFFFFFFFFu, zm, o));
                        dm = fmaxf(dm, __shfl_xor_sync(0xFFFFFFFFu, dm, o));
                    }
                    const uint32_t top_bits = __float_as_uint(zm + dm);
                    byte[c] = mx_byte(top_bits);
                    const float inv = mx_inv_scale(min(byte[c], 252u));
                    const float2 inv2 = make_float2(inv, inv);
                    float2 lo[4], hi[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 q = __fmul2_rn(z[c].p[j], inv2), e = HAS_Y ? w.p[j] : q;
                        const float di = HAS_Y ? d * inv : d;
                        lo[j] = __ffma2_rn(e, make_float2(-di, -di), q);
                        hi[j] = __ffma2_rn(e, make_float2(di, di), q);
                    }
                    code[c] = cvt_e2m1x8(lo[0].x, lo[0].y, lo[1].x, lo[1].y, lo[2].x, lo[2].y, lo[3].x, lo[3].y);
                    const uint32_t up = cvt_e2m1x8(hi[0].x, hi[0].y, hi[1].x, hi[1].y, hi[2].x, hi[2].y, hi[3].x, hi[3].y);
                    const bool doubt = ((code[c] ^ up) & kCodeBits<HAS_Y>) != 0u ||
                                       byte[c] != mx_byte(__float_as_uint(fmaxf(zm - dm, 0.f))) ||
                                       top_bits >= 0x7F000000u ||
                                       (top_bits < 0x21800000u &&                      // below 2^-60, or lost
                                        (top_bits != 0u || lost_zeros(c, ch, wm, w))) ||
                                       !(all.x + all.y == all.x + all.y);
                    redo |= doubt ? 1u << c : 0u;
                    if (!HAS_Y) code[c] = up;
                }
            }
        }
        odd ^= 1;

        const bool again = MX ? __syncthreads_or(wild || redo != 0) != 0 : wild;
        if (again) {                                     // sums of the row in float64; inputs from the stage again
            double fg64 = (double)g_row.x;
            if (HAS_Y && a.post_norm) {
                double s = 0.0;
#pragma unroll 1
                for (int ch = tid; ch < chunks; ch += threads) s += sum_sq64<Y>(load8<Y == kF32 ? kF32 : kBf16>(sy, ch), wild);
                fg64 *= rsqrt(block_sum(s, red64[0]) / a.H + (double)a.eps);
            }
            double s = 0.0;
#pragma unroll 1
            for (int ch = tid; ch < chunks; ch += threads) {
                double v[8];
                r64<Y, R>(p, row, ch, sy, sr, HAS_Y ? weight8(a.post_weight, ch) : V8(), fg64, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fma(v[i], v[i], s);
            }
            const Rms64 rms_r(block_sum(s, red64[1]) / a.H + (double)a.eps);
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const int ch = tid + c * threads;
                uint32_t need = wild ? 1u : (redo >> c) & 1u;
                if constexpr (MX) {                      // the four threads of a block together
                    need |= __shfl_xor_sync(0xFFFFFFFFu, need, 1);
                    need |= __shfl_xor_sync(0xFFFFFFFFu, need, 2);
                }
                if (!__any_sync(0xFFFFFFFFu, need)) continue;
                double v[8], amax = 0.0;
                bool nan = false;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.0;
                if (need && ch < chunks) {
                    r64<Y, R>(p, row, ch, sy, sr, HAS_Y ? weight8(a.post_weight, ch) : V8(), fg64, v);
                    const V8 w = weight8(a.norm_weight, ch);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const double zz = rms_r.divide(v[i]) * (double)w.at(i);
                        if (wild) {
                            ((i & 1) ? r[c].p[i >> 1].y : r[c].p[i >> 1].x) = (float)v[i];
                            ((i & 1) ? z[c].p[i >> 1].y : z[c].p[i >> 1].x) = (float)zz;
                        }
                        v[i] = zz;
                        nan |= zz != zz;
                        amax = fmax(amax, fabs(zz));
                    }
                }
                if constexpr (MX) {
                    if (nan) amax = __longlong_as_double(0x7FF0000000000000ll);    // as an infinity: byte 0xFF
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) amax = fmax(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
                    if (need) {
                        byte[c] = mx_byte64(amax);
                        code[c] = 0u;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            code[c] |= byte[c] == 255u ? 0u : mx_code64(v[i], byte[c]) << (4 * i);
                    }
                }
            }
            __syncthreads();                             // every read of the stage before its refill, and of the row
        }                                                // before the writes (which may be in place)
        if (!MX && !want_z) __syncthreads();
        // Everyone has read the stage: the barrier of the last sum, or of the redo, is behind.
        if (tid == 0 && lrow + (long long)p.stages * gridDim.x < a.T)
            fetch((int)(lrow + (long long)p.stages * gridDim.x), stage);
        if (++stage == p.stages) { stage = 0; phase ^= 1u; }

#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
            const bool ok = ch < chunks;
            if (a.resid_out && ok) store_resid(a, row, ch, r[c]);
            if (a.out && ok) zmax = max(zmax, store_out(a, row, ch, z[c]));
            if constexpr (MX) {
                if (ok) reinterpret_cast<uint32_t*>(a.codes + (size_t)row * (a.H >> 1))[ch] = code[c];
                uint32_t w = ok ? byte[c] << (8 * ((tid & 15) >> 2)) : 0u;
                w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
                w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
                if ((tid & 15) == 0 && (ch >> 4) < p.tile_cols)
                    *reinterpret_cast<uint32_t*>(a.scales + mx_scale_offset(row, ch >> 2, p.tile_cols)) = w;
            }
        }
    }

    if constexpr (MX) zero_padding_rows(p);
    if (a.amax) {
        zmax = __reduce_max_sync(0xFFFFFFFFu, zmax);
        if ((tid & 31) == 0) red_max[tid >> 5] = zmax;
        __syncthreads();
        if (tid < 32) {
            zmax = __reduce_max_sync(0xFFFFFFFFu, tid < (threads >> 5) ? red_max[tid] : 0u) << 16;
            if (tid == 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), zmax);
        }
    }
    if (tid == 0 && timeout != 0) atomicCAS(p.err, 0, timeout);
}

// A row in float64 by a warp.  y and v: the rows of y and resid (valid memory without resid too), in global or shared
// memory.  A chunk's 24 values are loaded before any is used, by no branch apart: written element by element, each
// behind its bounds check, a row of 2816 took 32,000 cycles of exposed latencies instead of about 5,000.
template <Src Y, Src R>
struct Row64 {
    const NormParams& p;
    const void *y, *v;
    const uint4* w_post;
    int row, chunks;
    bool has_v, g_col;
    double fg, scale;

    __device__ __forceinline__ void r8(int ch, double (&r)[8]) const {
        const V8 x = load8<R>(v, ch);
#pragma unroll
        for (int k = 0; k < 8; ++k) r[k] = has_v ? (double)x.at(k) : 0.0;
        if constexpr (Y != kNone) {
            const V8 n = load8<Y>(y, ch), w = unpack8(w_post[ch]);
            double t[8];
            weighted64<Y>(n, w, t);
            if (g_col) {
                const V8 g = gate8(p, row, ch);
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = fma(t[k] * (double)g.at(k), fg, r[k]);
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k) r[k] = fma(t[k], fg, r[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) r[k] *= scale;
    }
    // Sum over the row of the squares of y, or of r.
    template <bool OF_Y>
    __device__ __forceinline__ double sum_sq() const {
        double s = 0.0;
#pragma unroll 1
        for (int ch = threadIdx.x & 31; ch < chunks; ch += 32) {
            double x[8];
            if constexpr (OF_Y) {
                const V8 n = load8<Y == kF32 ? kF32 : kBf16>(y, ch);
#pragma unroll
                for (int k = 0; k < 8; ++k) x[k] = (double)n.at(k);
            } else {
                r8(ch, x);
            }
            s += fma(x[0], x[0], x[1] * x[1]) + fma(x[2], x[2], x[3] * x[3]) +
                 (fma(x[4], x[4], x[5] * x[5]) + fma(x[6], x[6], x[7] * x[7]));
        }
        return warp_sum(s);
    }
    __device__ __forceinline__ Row64(const NormParams& p_, int row_, const void* y_, const void* v_, const uint4* w_post_)
        : p(p_), y(y_), v(v_), w_post(w_post_), row(row_), chunks(p_.a.H >> 3), has_v(p_.a.resid != nullptr),
          scale((double)p_.a.scale) {
        const double h = (double)p.a.H, eps = (double)p.a.eps;
        g_col = Y != kNone && p.a.gate && p.a.gate_col_stride;
        fg = Y != kNone && p.a.gate && !g_col ? (double)gate_at(p.a, row, 0) : 1.0;
        if (Y != kNone && p.a.post_norm) fg *= rsqrt(sum_sq<true>() / h + eps);
    }
};

// The codes and scales of the loop steps (32 chunks each) in `steps`, or for a `wild` row everything (both the same on
// every lane).  Returns the largest bf16 magnitude stored to out.
template <Src Y, Src R, bool MX>
__device__ __noinline__ uint32_t redo_row64(const NormParams& p, int row, uint32_t steps, bool wild, const void* y,
                                            const void* v, const uint4* w_post, const uint4* w_norm) {
    const nvfp4b_block_norm_args& a = p.a;
    const int lane = threadIdx.x & 31;
    const Row64<Y, R> q(p, row, y, v, w_post);
    const Rms64 rms_r(q.template sum_sq<false>() / (double)a.H + (double)a.eps);
    __syncwarp();                                                   // codes and scale words stored before come first
    uint32_t zmax = 0;
    int step = 0;
#pragma unroll 1
    for (int c0 = 0; c0 < p.chunks16; c0 += 32, ++step) {
        if (!wild && !((steps >> step) & 1u)) continue;
        const int ch = c0 + lane;
        const bool ok = ch < q.chunks;
        double z[8], amax = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) z[k] = 0.0;
        if (ok) {
            q.r8(ch, z);
            const V8 w = unpack8(w_norm[ch]);
            V8 s;
#pragma unroll
            for (int j = 0; j < 4; ++j) s.p[j] = make_float2((float)z[2 * j], (float)z[2 * j + 1]);
            if (wild && a.resid_out) store_resid(a, row, ch, s);    // in place: the lane has read its own chunk
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                z[k] = rms_r.divide(z[k]) * (double)w.at(k);
                amax = z[k] != z[k] ? __longlong_as_double(0x7FF0000000000000ll) : fmax(amax, fabs(z[k]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) s.p[j] = make_float2((float)z[2 * j], (float)z[2 * j + 1]);
            if (wild && a.out) zmax = max(zmax, store_out(a, row, ch, s));
        }
        if constexpr (MX) {
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) amax = fmax(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
            const uint32_t byte = mx_byte64(amax);                  // NaN came as an infinity: byte 0xFF
            uint32_t code = 0;
#pragma unroll
            for (int k = 0; k < 8; ++k) code |= byte == 255u ? 0u : mx_code64(z[k], byte) << (4 * k);
            if (ok) reinterpret_cast<uint32_t*>(a.codes + (size_t)row * (a.H >> 1))[ch] = code;
            if ((lane & 3) == 0 && ch < p.chunks16)
                a.scales[mx_scale_offset(row, ch >> 2, p.tile_cols)] = ok ? (uint8_t)byte : (uint8_t)0;
        }
    }
    return zmax;
}

// Many rows: a row per warp.  No block-wide barrier, and the fixed cost of a row (two reductions, the wait for its bulk
// copies) is paid by one warp instead of all warps of a CTA.  Each warp owns one row buffer in shared memory; the weights
// lie there once per CTA; the next row is prefetched into L2 meanwhile.  Pass 1: sum of y^2.  Pass 2: r, written over
// the chunk's own y and resid, and the sums of r^2 and t^2 (t = scale * gate * n).  Pass 3: outputs.  Short code at any
// H, and 16 warps per SM hide each other's latencies (two stages and 8 warps took a third longer at 8192 x 2816).
//
// Bounds: a chunk's sum of squares is off by 4 u of itself, its compensated sum over the row's chunks and the float64
// tree by less than 0.1 u more, 1 / rms by 4.5 u; t by 8.5 u |t|, r by that + u |r|, and z (the rounding of z - d and
// z + d included) by
//   d = f wm E T + Z E (1 + k),   E = 10 u,   k = sqrt(sum t^2 / sum r^2),   wm = max |norm_w|,
// T = max |t| of the lane's chunks, Z = max |z| of the chunk (one d serves its 8 elements); without y by E |z|.  One row
// in sixteen at 2816 elements holds an element that near to a border.  Its redo takes a warp nearly as long as the row
// did, most of it conversions to float64, so the warps of a CTA take their rows from a common count (8192 x 2816 with a
// gate: 55 us, 40% more with a fixed share of the rows for each warp).
template <Src Y, Src R, bool MX>
__global__ void __launch_bounds__(kRowWarps * 32, 1) block_norm_rows_kernel(const __grid_constant__ NormParams p) {
    using namespace sm100;
    constexpr bool HAS_Y = Y != kNone;
    constexpr float kE = 0x1.4p-21f;                                // 10 u
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t full[kRowWarps];
    __shared__ uint32_t red_max[kRowWarps], red_post[kRowWarps];
    __shared__ int taken, timeout;
    const nvfp4b_block_norm_args& a = p.a;
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, warps = blockDim.x >> 5, chunks = a.H >> 3;
    const bool want_z = MX || a.out != nullptr;
    uint4* w_post = reinterpret_cast<uint4*>(smem);                 // bf16, ones where there are none
    uint4* w_norm = w_post + (HAS_Y ? chunks : 0);
    uint8_t* const sy = smem + p.weight_bytes + wid * p.stage_bytes;
    uint8_t* const sr = sy + p.y_bytes;
    // r of a chunk takes the place of its inputs: 32 bytes of the fp32 one, or 16 of either bf16 one
    auto r_lo = [&](int ch) { return reinterpret_cast<float4*>(Y == kF32 ? sy + 32 * ch : R == kF32 ? sr + 32 * ch : sy + 16 * ch); };
    auto r_hi = [&](int ch) { return reinterpret_cast<float4*>(Y == kF32 ? sy + 32 * ch + 16 : R == kF32 ? sr + 32 * ch + 16 : sr + 16 * ch); };

    const uint32_t yb = (uint32_t)(a.H * src_size(Y)), rb = a.resid ? (uint32_t)(a.H * src_size(R)) : 0u;
    auto y_row = [&](long long row) { return static_cast<const uint8_t*>(a.y) + row * a.ld_y * src_size(Y); };
    auto v_row = [&](long long row) { return static_cast<const uint8_t*>(a.resid) + row * a.ld_resid * src_size(R); };
    auto fetch = [&](long long row) {                               // lane 0
        mbar_arrive_expect_tx(&full[wid], yb + rb);
        if constexpr (HAS_Y) bulk_load(sy, y_row(row), yb, &full[wid]);
        if (rb) bulk_load(sr, v_row(row), rb, &full[wid]);
    };
    // the CTA's rows: blockIdx.x + gridDim.x * (0, 1, 2 ...), the first `warps` of them by warp number, then as they come
    const long long first = blockIdx.x + (long long)gridDim.x * wid;
    if (threadIdx.x == 0) {
        timeout = 0;
        taken = warps;
    }
    if (lane == 0) {
        mbar_init(&full[wid], 1);
        fence_mbar_init();
        if (first < a.T) fetch(first);
    }
    const uint4 ones = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
    auto top8 = [](const uint4& q) {                                // largest magnitude of eight bf16
        const uint32_t m = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu),
                                    __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
        return max(m & 0xFFFFu, m >> 16);
    };
    uint32_t wm_bits = 0, post_bits = 0;
    for (int ch = threadIdx.x; ch < chunks; ch += blockDim.x) {
        const uint4 q = a.norm_weight ? __ldg(static_cast<const uint4*>(a.norm_weight) + ch) : ones;
        if constexpr (HAS_Y) {
            const uint4 q1 = a.post_weight ? __ldg(static_cast<const uint4*>(a.post_weight) + ch) : ones;
            w_post[ch] = q1;
            post_bits = max(post_bits, top8(q1));
        }
        w_norm[ch] = q;
        wm_bits = max(wm_bits, top8(q));
    }
    wm_bits = __reduce_max_sync(0xFFFFFFFFu, wm_bits);
    post_bits = __reduce_max_sync(0xFFFFFFFFu, post_bits);
    if (lane == 0) {
        red_max[wid] = wm_bits;
        red_post[wid] = post_bits;
    }
    __syncthreads();
    const float wm = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, lane < warps ? red_max[lane] : 0u) << 16);
    // Blocks of zeros: true ones, or products that underflowed.  Such a product is below 2^-149, so it matters (the least border
    // is 2^-129) only where the factors behind it make more than 2^18: the weights, 1 / rms(r), a gate per feature.  Below, a code
    // of 0 may have the sign of the rounded product and not of the product: looking at every block of zeros took 10% more where
    // half the rows are.
    const uint32_t post_max = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? red_post[lane] : 0u) << 16;
    const float factors =
        HAS_Y && a.gate && a.gate_col_stride ? __int_as_float(0x7F800000) : wm * fmaxf(__uint_as_float(post_max), 1.f);
    __syncthreads();                                                // red_max is used again at the end

    uint32_t zmax = 0, phase = 0;
    for (long long lrow = first, next; lrow < a.T; lrow = next) {
        const int row = (int)lrow;
        next = lane == 0 ? atomicAdd(&taken, 1) : 0;
        next = blockIdx.x + (long long)gridDim.x * __shfl_sync(0xFFFFFFFFu, (int)next, 0);
        const float g_row = HAS_Y && a.gate && !a.gate_col_stride ? gate_at(a, row, 0) : 1.f;
        const bool g_col = HAS_Y && a.gate && a.gate_col_stride;
        mbar_wait(&full[wid], phase, &timeout, kErrTimeoutProducer);   // on expiry the kernel goes on and reports
        phase ^= 1u;
        if (lane == 0 && next < a.T) {
            if constexpr (HAS_Y) l2_prefetch(y_row(next), yb);
            if (rb) l2_prefetch(v_row(next), rb);
        }
        bool wild = false;
        float fgs = 1.f;                                            // scale * gate / rms(y)
        if constexpr (HAS_Y) {
            float f = 1.f;
            if (a.post_norm) {
                SumSq ss;
#pragma unroll 4
                for (int ch = lane; ch < chunks; ch += 32) ss.add(load8<Y>(sy, ch));
                const float m = fmaf(ss.total(), p.inv_h, a.eps);
                wild |= !mean_ok(m);
                f = __frsqrt_rn(m);
            }
            fgs = f * g_row * a.scale;
            wild |= fabsf(fgs) < 0x1p-126f && g_row != 0.f && a.scale != 0.f;
        }
        const float2 scale2 = make_float2(a.scale, a.scale);
        float t_max = 0.f, st = 0.f;
        SumSq ss;
        if constexpr (HAS_Y) {
            const float2 fgs2 = make_float2(fgs, fgs);
#pragma unroll 2
            for (int ch = lane; ch < chunks; ch += 32) {
                const V8 y = load8<Y>(sy, ch), w = unpack8(w_post[ch]), v = a.resid ? load8<R>(sr, ch) : fill8(0.f);
                V8 t, r;
#pragma unroll
                for (int j = 0; j < 4; ++j) t.p[j] = __fmul2_rn(__fmul2_rn(y.p[j], fgs2), w.p[j]);
                if (g_col) {
                    const V8 g = gate8(p, row, ch);
#pragma unroll
                    for (int j = 0; j < 4; ++j) t.p[j] = __fmul2_rn(t.p[j], g.p[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) r.p[j] = __ffma2_rn(v.p[j], scale2, t.p[j]);
                if constexpr (MX) {
                    st += sum_sq(t);
                    t_max = fmaxf(t_max, max_abs(t));
                }
                *r_lo(ch) = make_float4(r.p[0].x, r.p[0].y, r.p[1].x, r.p[1].y);
                *r_hi(ch) = make_float4(r.p[2].x, r.p[2].y, r.p[3].x, r.p[3].y);
                ss.add(r);
            }
        } else {
#pragma unroll 4
            for (int ch = lane; ch < chunks; ch += 32) {
                V8 v = load8<R>(sr, ch);
#pragma unroll
                for (int j = 0; j < 4; ++j) v.p[j] = __fmul2_rn(v.p[j], scale2);
                ss.add(v);
            }
        }
        auto r_chunk = [&](int ch) {
            V8 r;
            if constexpr (HAS_Y) {
                const float4 q0 = *r_lo(ch), q1 = *r_hi(ch);
                r.p[0] = make_float2(q0.x, q0.y);
                r.p[1] = make_float2(q0.z, q0.w);
                r.p[2] = make_float2(q1.x, q1.y);
                r.p[3] = make_float2(q1.z, q1.w);
            } else {
                r = load8<R>(sr, ch);
#pragma unroll
                for (int j = 0; j < 4; ++j) r.p[j] = __fmul2_rn(r.p[j], scale2);
            }
            return r;
        };
        float f = 1.f, rel = kE;
        if (want_z) {
            const float sum = ss.total();
            if constexpr (MX && HAS_Y) {
                st = warp_sum(st);
                rel = st > 0.f ? fmaf(sqrtf(st / sum), kE, kE) : kE;
                wild |= !(rel < 0x1p-12f);                          // also where sum = 0 < st: r cancelled altogether
            }
            const float m = fmaf(sum, p.inv_h, a.eps);
            wild |= !mean_ok(m) || (MX && !(wm < __int_as_float(0x7F800000)));   // a NaN weight passes every maximum
            f = __frsqrt_rn(m);
        }
        const float2 f2 = make_float2(f, f);
        auto z_chunk = [&](int ch, const V8& r) {
            const V8 w = unpack8(w_norm[ch]);
            V8 z;
#pragma unroll
            for (int j = 0; j < 4; ++j) z.p[j] = __fmul2_rn(__fmul2_rn(r.p[j], f2), w.p[j]);
            return z;
        };
        uint32_t row_max = 0, doubt = 0, zeros = 0;                 // bit i: the chunk of loop step i is not proven, is 0
        // r and z are stored at once, unless that would overwrite what a redo reads again
        const bool later = MX && p.in_place;
        if (!wild) {
            const float dt = t_max * f * wm * kE;
            uint32_t* code_row = reinterpret_cast<uint32_t*>(a.codes + (MX ? (size_t)row * (a.H >> 1) : 0));
            uint8_t* scale_row = a.scales + (MX ? mx_scale_offset(row, 0, p.tile_cols) : 0);   // + 512 per 16 chunks
            int i = 0;
#pragma unroll 1
            for (int c0 = 0; c0 < p.chunks16; c0 += 32, ++i) {      // whole groups of 16: the scale words' threads
                const int ch = c0 + lane;
                const bool ok = ch < chunks;
                V8 z;
                if (ok) {
                    const V8 r = r_chunk(ch);
                    if (a.resid_out && !later) store_resid(a, row, ch, r);
                    z = z_chunk(ch, r);
                    if (a.out && !later) row_max = max(row_max, store_out(a, row, ch, z));
                } else {
                    z = fill8(0.f);
                }
                if constexpr (MX) {
                    float zm = max_abs(z);
                    const float d = HAS_Y && ok ? fmaf(zm, rel, dt) : zm * rel;
                    float dm = d;
#pragma unroll
                    for (int o = 1; o < 4; o <<= 1) {
                        zm = fmaxf(zm, __shfl_xor_sync(0xFFFFFFFFu, zm, o));
                        dm = fmaxf(dm, __shfl_xor_sync(0xFFFFFFFFu, dm, o));
                    }
                    const uint32_t top = __float_as_uint(zm + dm), bot = __float_as_uint(fmaxf(zm - dm, 0.f));
                    // exponent field, at least 2; the byte is 2 less, and 1 / 2^e has the field 256 - it
                    const uint32_t field = max(top & 0x7F800000u, 0x01000000u);
                    const float inv = __uint_as_float(0x80000000u - field);
                    const float2 inv2 = make_float2(inv, inv);
                    // without y the bound is relative to each element
                    const float2 up = HAS_Y ? make_float2(d * inv, d * inv) : make_float2(rel, rel);
                    const float2 dn = make_float2(-up.x, -up.y);
                    float2 lo[4], hi[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 q = __fmul2_rn(z.p[j], inv2);
                        lo[j] = HAS_Y ? __fadd2_rn(q, dn) : __ffma2_rn(q, dn, q);
                        hi[j] = HAS_Y ? __fadd2_rn(q, up) : __ffma2_rn(q, up, q);
                    }
                    const uint32_t code =
                        cvt_e2m1x8(lo[0].x, lo[0].y, lo[1].x, lo[1].y, lo[2].x, lo[2].y, lo[3].x, lo[3].y);
                    const uint32_t other =
                        cvt_e2m1x8(hi[0].x, hi[0].y, hi[1].x, hi[1].y, hi[2].x, hi[2].y, hi[3].x, hi[3].y);
                    // also where the exponent is in doubt, or the values are near the ends of the range
                    const bool unsure = ((code ^ other) & kCodeBits<HAS_Y>) != 0u || ((top ^ bot) & 0x7F800000u) != 0u ||
                                        top - 0x21800000u >= 0x7F000000u - 0x21800000u;
                    doubt |= unsure ? 1u << i : 0u;
                    zeros |= top == 0u ? 1u << i : 0u;              // unsure, too
                    // zeros that agree: the end that kept their sign (x - 0 of each, or x + x rel)
                    if (ok) code_row[ch] = HAS_Y ? code : other;
                    uint32_t w = ok ? ((field >> 23) - 2u) << (8 * ((lane & 15) >> 2)) : 0u;
                    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
                    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
                    if ((lane & 15) == 0 && ch < p.chunks16) *reinterpret_cast<uint32_t*>(scale_row + 32 * ch) = w;
                }
            }
        }
        if constexpr (MX) {
            if (fmaxf(f, 1.f) * factors <= 0x1p18f) {
                doubt &= ~zeros;
            } else {
                for (; zeros; zeros &= zeros - 1) {
                    const int ch = 32 * (__ffs(zeros) - 1) + lane;
                    bool lost = ch < chunks && both_nonzero(HAS_Y ? r_chunk(ch) : load8<R>(sr, ch), unpack8(w_norm[ch]));
                    if constexpr (HAS_Y) lost = lost || (ch < chunks && lost_product<Y>(p, row, ch, g_row, y_row(row), w_post));
                    if (!lost) doubt &= ~(zeros & (0u - zeros));
                }
            }
        }
        doubt = __reduce_or_sync(0xFFFFFFFFu, doubt);               // from here on the same on every lane, as `wild` is
        if (wild || doubt != 0) {
            const uint8_t *y = sy, *v = sr;
            if (wild || !later) {                                   // r is not needed any more: the inputs once again
                if constexpr (HAS_Y) {
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) fetch(row);
                    mbar_wait(&full[wid], phase, &timeout, kErrTimeoutProducer);
                    phase ^= 1u;
                }
            } else {
                if constexpr (HAS_Y) y = y_row(row);
                v = a.resid ? v_row(row) : smem;
            }
            const uint32_t m = redo_row64<Y, R, MX>(p, row, doubt, wild, y, v, w_post, w_norm);
            row_max = wild ? m : row_max;
        }
        if (later && !wild) {
#pragma unroll 1
            for (int ch = lane; ch < chunks; ch += 32) {
                const V8 r = r_chunk(ch);
                if (a.resid_out) store_resid(a, row, ch, r);
                if (a.out) row_max = max(row_max, store_out(a, row, ch, z_chunk(ch, r)));
            }
        }
        zmax = max(zmax, row_max);
        fence_proxy_async();                                        // r's writes before the copies' ones
        __syncwarp();                                               // every lane is done with the buffer
        if (lane == 0 && next < a.T) fetch(next);
    }

    if constexpr (MX) zero_padding_rows(p);
    if (a.amax) {
        zmax = __reduce_max_sync(0xFFFFFFFFu, zmax);
        if (lane == 0) red_max[wid] = zmax;
        __syncthreads();
        if (wid == 0) {
            zmax = __reduce_max_sync(0xFFFFFFFFu, lane < warps ? red_max[lane] : 0u) << 16;
            if (lane == 0) atomicMax(reinterpret_cast<unsigned int*>(a.amax), zmax);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0 && timeout != 0) atomicCAS(p.err, 0, timeout);
}

int raise_smem(const void* kernel, std::atomic<bool> (&ready)[64]) {   // once per kernel and device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NVFP4B_ERR_CUDA;
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kNormMaxSmem);
        if (e != cudaSuccess) return record_cuda_error(e);
        ready[dev].store(true, std::memory_order_release);
    }
    return NVFP4B_OK;
}

// The row kernel's launch; `fits` false (nothing launched) where a row has more loop steps than a 32-bit mask, or where the
// row buffers that shared memory holds are too few.  With y and codes, which is the most to compute, six do (4096 wide,
// fp32 y and resid, 8192 rows: 122 us, 163 by CTAs; five, 8192 wide bf16: 243 and 248, but 1500 rows 74 and 58), if the
// scale is positive: it goes into the sum's terms there, which a scale below or at zero would give zeros of another sign.  Else
// all sixteen, or eight and four rounds of rows (4096 wide, bf16 y and resid to bf16, twelve warps: 8192 rows 55 us, 62 by
// CTAs; 4096 rows 35 and 34).
template <Src Y, Src R, bool MX>
int launch_block_norm_rows(NormParams& p, cudaStream_t s, bool& fits) {
    const auto kernel = block_norm_rows_kernel<Y, R, MX>;
    p.y_bytes = p.a.H * src_size(Y);
    p.stage_bytes = (p.a.H * (src_size(Y) + src_size(R)) + 127) / 128 * 128;
    p.weight_bytes = (p.a.H * (Y == kNone ? 2 : 4) + 127) / 128 * 128;
    int warps = (kNormMaxSmem - p.weight_bytes) / p.stage_bytes;
    if (warps > kRowWarps) warps = kRowWarps;
    fits = p.a.H <= 32 * 256 && (MX && Y != kNone ? warps >= 6 && p.a.scale > 0.f
                                                  : warps == kRowWarps || (warps >= 8 && p.a.T / warps >= 4 * sm_count()));
    if (!fits) return NVFP4B_OK;
    static std::atomic<bool> ready[64];
    const int st = raise_smem(reinterpret_cast<const void*>(kernel), ready);
    if (st) return st;
    const int grid = p.a.T < sm_count() ? p.a.T : sm_count();       // rows dealt over every SM first
    return launch_k(kernel, dim3((unsigned)grid), dim3(warps * 32), p.weight_bytes + warps * p.stage_bytes, s, p);
}

// Persistent grid: as many CTAs per SM as shared memory (and 2048 threads at up to 128 registers) hold.
template <Src Y, Src R, int NCH, bool MX>
int launch_block_norm(NormParams& p, cudaStream_t s) {
    const auto kernel = block_norm_kernel<Y, R, NCH, MX>;
    static std::atomic<bool> ready[64];
    const int st = raise_smem(reinterpret_cast<const void*>(kernel), ready);
    if (st) return st;
    const int threads = (p.a.H / 8 + NCH * 32 - 1) / (NCH * 32) * 32;
    const int row_bytes = p.a.H * src_size(Y) + (p.a.resid ? p.a.H * src_size(R) : 0);
    p.y_bytes = p.a.H * src_size(Y);                     // a multiple of 16
    p.stage_bytes = (row_bytes + 127) / 128 * 128;
    p.stages = 2 * p.stage_bytes <= kNormMaxSmem ? 2 : 1;
    const int smem = p.stages * p.stage_bytes;
    int per_sm = kNormMaxSmem / (smem + 1024);
    const int by_regs = 512 / threads;
    if (per_sm > by_regs) per_sm = by_regs;
    if (per_sm < 1) per_sm = 1;
    long long grid = (long long)sm_count() * per_sm;
    if (grid > p.a.T) grid = p.a.T;
    return launch_k(kernel, dim3((unsigned)grid), dim3(threads), smem, s, p);
}

// From kRowKernelRows rows per SM on a warp per row, where its buffers fit (900 x 2816 with y to MXFP4 16.3 us, 21.1 by
// CTAs; 700 rows 16.0 and 13.2, 741 rows, where the switch is, 16.0 and 13.3); not with an fp32 y and no codes, where there is
// little to compute and a row fills much shared memory (2900 x 2816 26.6 us by CTAs, 30.2 by warps).  Below a CTA per row: one
// chunk per thread, the shortest path through a row, as far as the rows make two rounds (64 x 2816 with y to MXFP4 6.2 us);
// then two, for more CTAs per SM (512 x 2816 fp32 to bf16 6.3 us, 7.2 with four; 739 x 4096 bf16 9.1 and 11.7), or with y and
// codes, where the threads compute most, four (600 x 2816 12.6 us, 13.8 with two).
constexpr int kRowKernelRows = 5;

template <Src Y, Src R, bool MX>
int dispatch_block_norm(NormParams& p, cudaStream_t s) {   // R = kBf16 without resid
    if constexpr (MX || Y != kF32) {
        if (p.a.T >= kRowKernelRows * sm_count()) {
            bool fits = false;
            const int st = launch_block_norm_rows<Y, R, MX>(p, s, fits);
            if (fits) return st;
        }
    }
    const int chunks = p.a.H / 8, resident = kNormMaxThreads / ((chunks + 31) / 32 * 32);    // CTAs per SM, one chunk each
    if (resident >= 1 && p.a.T <= 2 * sm_count() * resident) return launch_block_norm<Y, R, 1, MX>(p, s);
    if constexpr (!MX || Y == kNone) {
        if (chunks <= 2 * kNormMaxThreads) return launch_block_norm<Y, R, 2, MX>(p, s);
    }
    return launch_block_norm<Y, R, 4, MX>(p, s);
}

template <Src Y, Src R>
int dispatch_block_norm(NormParams& p, cudaStream_t s) {
    return p.a.codes ? dispatch_block_norm<Y, R, true>(p, s) : dispatch_block_norm<Y, R, false>(p, s);
}

bool bad_rows(const void* p, int f32, long long ld) { return !aligned16(p) || (ld * (f32 ? 4 : 2)) % 16; }

// Memory that a call reads or writes: n runs of `width` bytes, `pitch` bytes apart (p NULL: not there); one run where
// nothing lies between them.
struct Region {
    long long p, pitch, width, n;
    Region(const void* p_, long long width_, long long pitch_ = 0, long long n_ = 1)
        : p((long long)reinterpret_cast<uintptr_t>(p_)), pitch(pitch_), width(width_), n(n_) {
        if (n == 1 || pitch <= width) {
            width += (n - 1) * pitch;
            pitch = 0;
            n = 1;
        }
    }
    long long end() const { return p + (n - 1) * pitch + width; }
};

// Whether a run of `a` meets the one run `b`.
bool meets(const Region& a, const Region& b) {
    const long long d = b.p - a.p - a.width, i = d < 0 ? 0 : a.pitch ? d / a.pitch + 1 : 1;   // the first that ends behind b.p
    return i < a.n && a.p + i * a.pitch < b.p + b.width;
}

// Whether two regions share memory otherwise than run for run (`same` allowed) -- side by side in one pitch they do not; of
// different pitches that interleave it is assumed.
bool clash(const Region& a, const Region& b, bool same = false) {
    if (!a.p || !b.p || a.p >= b.end() || b.p >= a.end()) return false;
    if (same && a.p == b.p && a.width == b.width && a.pitch == b.pitch) return false;
    if (b.n == 1) return meets(a, b);
    if (a.n == 1) return meets(b, a);
    if (a.pitch != b.pitch) return true;
    const long long d = ((b.p - a.p) % a.pitch + a.pitch) % a.pitch;
    return d < a.width || d + b.width > a.pitch;
}

// Whether an output shares memory with another one, or with an input (resid_out and out may be resid or y themselves).
bool clashes(const nvfp4b_block_norm_args& a) {
    const auto rows = [&](const void* p, int f32, long long ld) {
        return Region(p, a.H * (f32 ? 4ll : 2ll), ld * (f32 ? 4 : 2), a.T);
    };
    const long long gate_size = a.gate_f32 ? 4 : 2;
    const Region out[] = {rows(a.resid_out, a.resid_out_f32, a.ld_resid_out), rows(a.out, 0, a.ld_out),
                          Region(a.codes, (long long)a.T * (a.H / 2)),
                          Region(a.scales, (long long)nvfp4b_mx_scale_buffer_bytes(a.T, a.H)), Region(a.amax, 4)};
    const Region in[] = {rows(a.resid, a.resid_f32, a.ld_resid), rows(a.y, a.y_f32, a.ld_y), Region(a.post_weight, a.H * 2ll),
                         Region(a.norm_weight, a.H * 2ll),
                         Region(a.gate, a.gate_col_stride ? a.H * gate_size : gate_size, a.gate_row_stride * gate_size, a.T)};
    for (int i = 0; i < 5; ++i) {
        for (int j = 0; j < 5; ++j)
            if (clash(out[i], in[j], i < 2 && j < 2)) return true;
        for (int j = 0; j < i; ++j)
            if (clash(out[i], out[j])) return true;
    }
    return false;
}

}  // namespace
}  // namespace nvfp4b

using namespace nvfp4b;

extern "C" int nvfp4b_block_norm(const nvfp4b_block_norm_args* args, void* stream) {
    if (!args) return NVFP4B_ERR_NULL;
    const nvfp4b_block_norm_args& a = *args;
    if (a.T <= 0 || a.H <= 0 || (a.H & 7) || a.H > NVFP4B_BLOCK_NORM_MAX_H || (a.codes && (a.H & 31)))
        return NVFP4B_ERR_SHAPE;
    if ((!a.resid && !a.y) || (!a.resid_out && !a.out && !a.codes) || !a.codes != !a.scales || (a.amax && !a.out))
        return NVFP4B_ERR_NULL;
    const int flags[] = {a.resid_f32, a.y_f32, a.gate_f32, a.resid_out_f32, a.post_norm};
    for (int f : flags)
        if (f != 0 && f != 1) return NVFP4B_ERR_ARG;
    if (a.gate_col_stride != 0 && a.gate_col_stride != 1) return NVFP4B_ERR_ARG;
    if (!(a.eps >= 0.0f) || ((a.post_weight || a.post_norm || a.gate) && !a.y)) return NVFP4B_ERR_ARG;
    if ((a.resid && a.ld_resid < a.H) || (a.y && a.ld_y < a.H) || (a.resid_out && a.ld_resid_out < a.H) ||
        (a.out && a.ld_out < a.H) || a.gate_row_stride < 0)
        return NVFP4B_ERR_SHAPE;
    if ((a.resid && bad_rows(a.resid, a.resid_f32, a.ld_resid)) || (a.y && bad_rows(a.y, a.y_f32, a.ld_y)) ||
        (a.resid_out && bad_rows(a.resid_out, a.resid_out_f32, a.ld_resid_out)) ||
        (a.out && bad_rows(a.out, 0, a.ld_out)) || !aligned16(a.post_weight) || !aligned16(a.norm_weight) ||
        !aligned16(a.codes) || !aligned16(a.scales) || (reinterpret_cast<uintptr_t>(a.gate) & (a.gate_f32 ? 3 : 1)) ||
        (reinterpret_cast<uintptr_t>(a.amax) & 3))
        return NVFP4B_ERR_ALIGN;
    if (clashes(a)) return NVFP4B_ERR_ARG;
    const cudaStream_t s = (cudaStream_t)stream;
    if (a.amax) {
        const cudaError_t e = cudaMemsetAsync(a.amax, 0, sizeof(float), s);
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    NormParams p;
    p.a = a;
    p.tile_cols = (a.H + 127) / 128;
    p.inv_h = 1.0f / (float)a.H;
    p.chunks16 = p.tile_cols * 16;
    p.weight_bytes = 0;
    p.in_place = (a.resid_out && (a.resid_out == a.resid || a.resid_out == a.y)) ||
                 (a.out && (a.out == a.resid || a.out == a.y));
    p.gate_vec = aligned16(a.gate) && (a.gate_row_stride * (a.gate_f32 ? 4 : 2)) % 16 == 0;
    p.err = device_error_ptr();
    if (!p.err) return NVFP4B_ERR_CUDA;
    const bool f32 = a.resid && a.resid_f32;
    if (a.y && a.y_f32)
        return f32 ? dispatch_block_norm<kF32, kF32>(p, s) : dispatch_block_norm<kF32, kBf16>(p, s);
    if (a.y) return f32 ? dispatch_block_norm<kBf16, kF32>(p, s) : dispatch_block_norm<kBf16, kBf16>(p, s);
    return f32 ? dispatch_block_norm<kNone, kF32>(p, s) : dispatch_block_norm<kNone, kBf16>(p, s);
}
