// mx_quant.cu -- MXFP4 quantisers (plain, and gated: gelu_tanh(gate) * up) and the dequantiser.
//
// All three are streams: the quantiser reads 2 or 4 bytes and writes 17/32 per element, the gated one reads 4, the
// dequantiser reads 17/32 and writes 2 or 4.  A thread owns 16 consecutive elements, two threads one block, eight
// threads the four blocks of one row of a scale tile; the four eighths of a warp take the rows m, m + 32, m + 64,
// m + 96 of one 128-row tile, whose scale words are neighbours in the tile layout, so a warp writes its 16 scale
// bytes as one run and reads four runs of 128 elements.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "mx.cuh"

namespace nvfp4b {
namespace {

constexpr int kMxThreads = 256;

struct MxPos {
    int m, k;          // row, first of the thread's 16 elements
    bool row_ok, ok;   // row < M; and k < K
};

// Work item -> this thread's elements.  Items run over (128-row tile, row in 0..31, column tile), columns fastest.
__device__ __forceinline__ MxPos mx_pos(long long item, int M, int K, int tile_cols) {
    const int lane = threadIdx.x & 31;
    const long long rowgrp = item / tile_cols;
    const int c = (int)(item - rowgrp * tile_cols);
    MxPos p;
    p.m = (int)(rowgrp >> 5) * 128 + (int)(rowgrp & 31) + (lane >> 3) * 32;
    p.k = c * 128 + (lane & 7) * 16;
    p.row_ok = p.m < M;
    p.ok = p.row_ok && p.k < K;
    return p;
}

// Gathers the four scale bytes of the eight-thread group (byte j from its threads 2j, 2j + 1) and writes the word.
__device__ __forceinline__ void mx_store_scales(uint8_t* scales, const MxPos& p, uint32_t byte, int tile_cols) {
    uint32_t w = byte << (8 * ((threadIdx.x & 7) >> 1));
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 2);
    w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
    if ((threadIdx.x & 7) == 0)
        *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(p.m, p.k >> 5, tile_cols)) = w;
}

template <typename T>
__device__ __forceinline__ void mx_load16(const T* p, float (&v)[16]);
template <>
__device__ __forceinline__ void mx_load16<uint16_t>(const uint16_t* p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint4 q = __ldg(reinterpret_cast<const uint4*>(p) + i);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[8 * i + 2 * j] = bf16lo(w[j]); v[8 * i + 2 * j + 1] = bf16hi(w[j]); }
    }
}
template <>
__device__ __forceinline__ void mx_load16<float>(const float* p, float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float4 q = __ldg(reinterpret_cast<const float4*>(p) + i);
        v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
}

__device__ __forceinline__ uint32_t mx_amax_bits16(const float (&v)[16]) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) b = max(b, __float_as_uint(v[i]) & 0x7FFFFFFFu);   // NaN orders above infinity
    return b;
}

template <typename T>
__global__ void __launch_bounds__(kMxThreads) mx_quantize_kernel(const T* __restrict__ x, long long ldx, int M, int K,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales, int tile_cols,
                                                                 long long items) {
    const long long step = (long long)gridDim.x * (kMxThreads / 32);
    for (long long it = (long long)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const MxPos p = mx_pos(it, M, K, tile_cols);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
        if (p.ok) mx_load16(x + (size_t)p.m * ldx + p.k, v);
        uint32_t a = mx_amax_bits16(v);
        a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
        const uint32_t byte = mx_byte(a);
        if (p.ok) {
            const float inv = mx_inv_scale(min(byte, 252u));
            uint2 c = make_uint2(mx_encode8(v, inv), mx_encode8(v + 8, inv));
            if (byte == 255u) c = make_uint2(0u, 0u);
            *reinterpret_cast<uint2*>(codes + (size_t)p.m * (K >> 1) + (p.k >> 1)) = c;
        }
        mx_store_scales(scales, p, byte, tile_cols);
    }
}

// gelu_tanh(g) * u = g u / (1 + exp(-2 t)), t = sqrt(2/pi) (g + 0.044715 g^3): no cancellation for negative g.
__device__ __forceinline__ double geglu64(double g, double u) {
    const double t2 = 1.5957691216057307117597842397375 * (g + 0.044715 * (g * g * g));
    return g / (1.0 + exp(-t2)) * u;
}

// float64 redo of one block by its two threads: stores the codes, returns the scale byte.
__device__ __noinline__ uint32_t geglu_block64(const uint16_t* gp, const uint16_t* up, uint8_t* codes,
                                               uint32_t pair_mask) {
    float g[16], u[16];
    mx_load16(gp, g);
    mx_load16(up, u);
    double a = 0.0;
    bool nan = false;
#pragma unroll 1
    for (int i = 0; i < 16; ++i) {
        const double h = fabs(geglu64((double)g[i], (double)u[i]));
        nan |= h != h;
        a = h > a ? h : a;
    }
    if (nan) a = __longlong_as_double(0x7FF8000000000000ll);
    const double b = __shfl_xor_sync(pair_mask, a, 1);
    a = (a != a || b != b) ? __longlong_as_double(0x7FF8000000000000ll) : (a > b ? a : b);
    const uint32_t byte = mx_byte64(a);
    unsigned long long c = 0;
#pragma unroll 1
    for (int i = 0; i < 16 && byte != 255u; ++i)
        c |= (unsigned long long)mx_code64(geglu64((double)g[i], (double)u[i]), byte) << (4 * i);
    *reinterpret_cast<unsigned long long*>(codes) = c;
    return byte;
}

// Gated quantiser: h = gelu_tanh(gate) * up of row [gate (I) | up (I)].  With w = 2 t / ln 2 the fp32 estimate
// g * rcp(1 + ex2(-w)) * u is off by at most |h| (max(-w, 1) 2^-22 + 2^-20): the five roundings of w leave the
// exponential |w| ln2 * 5 * 2^-24 off, which for w > 0 enters through ex2(-w) / (1 + ex2(-w)) only (below 1 / w);
// ex2.approx 2^-22, the sum, the reciprocal and the two products add 9 * 2^-24.  Where -w nears the end of the fp32
// range or h the subnormals, the estimate has no such bound; |h| <= |g u| 2^-100 then, and such an element has code
// 0 unless the whole block is that small, in which case the block counts as unproven.
__global__ void __launch_bounds__(kMxThreads) mx_geglu_kernel(const uint16_t* __restrict__ x, long long ldx, int M,
                                                              int I, uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, int tile_cols,
                                                              long long items) {
    const long long step = (long long)gridDim.x * (kMxThreads / 32);
    for (long long it = (long long)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const MxPos p = mx_pos(it, M, I, tile_cols);
        float h[16], d[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) h[i] = d[i] = 0.f;
        const uint16_t* gp = x + (size_t)(p.ok ? p.m : 0) * ldx + (p.ok ? p.k : 0);
        float tiny = 0.f;      // largest magnitude that the estimate may miss
        if (p.ok) {
            float g[16], u[16];
            mx_load16(gp, g);
            mx_load16(gp + I, u);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                // 2 sqrt(2/pi) / ln 2 = 2.3022082...
                const float w = 2.30220818f * g[i] * fmaf(0.044715f * g[i], g[i], 1.0f);
                float ex, rc;
                asm("ex2.approx.f32 %0, %1;" : "=f"(ex) : "f"(-w));
                asm("rcp.approx.f32 %0, %1;" : "=f"(rc) : "f"(1.0f + ex));
                h[i] = g[i] * rc * u[i];
                d[i] = fabsf(h[i]) * fmaf(fmaxf(-w, 1.0f), 0x1p-22f, 0x1p-20f);
                if (!(w > -100.f)) tiny = fmaxf(tiny, fabsf(g[i] * u[i]) * 0x1p-100f);
                else if (fabsf(h[i]) < 0x1p-100f && g[i] != 0.f && u[i] != 0.f) tiny = fmaxf(tiny, 0x1p-100f);
            }
        }
        uint32_t alo = 0, ahi = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const uint32_t lo = __float_as_uint(fabsf(h[i]) - d[i]) & 0x7FFFFFFFu;
            const uint32_t hi = __float_as_uint(fabsf(h[i]) + d[i]) & 0x7FFFFFFFu;
            alo = max(alo, lo);
            ahi = max(ahi, hi);
        }
        alo = max(alo, __shfl_xor_sync(0xFFFFFFFFu, alo, 1));
        ahi = max(ahi, __shfl_xor_sync(0xFFFFFFFFu, ahi, 1));
        uint32_t byte = mx_byte(ahi);
        const float inv = mx_inv_scale(min(byte, 252u));
        // the smallest magnitude with a code other than 0 is above A / 32
        bool redo = tiny > __uint_as_float(ahi) * 0x1p-6f || byte != mx_byte(alo) || (ahi >> 23) >= 254u;
        uint32_t c[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float lo[8], hi[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { lo[i] = h[8 * q + i] - d[8 * q + i]; hi[i] = h[8 * q + i] + d[8 * q + i]; }
            c[q] = mx_encode8(lo, inv);
            redo |= c[q] != mx_encode8(hi, inv);
        }
        redo |= __shfl_xor_sync(0xFFFFFFFFu, (int)redo, 1) != 0;      // both threads of a block, on every lane
        redo &= p.ok;
        uint8_t* cp = codes + (size_t)p.m * (I >> 1) + (p.k >> 1);
        if (p.ok && !redo) *reinterpret_cast<uint2*>(cp) = make_uint2(c[0], c[1]);
        if (redo) byte = geglu_block64(gp, gp + I, cp, 3u << (threadIdx.x & 30));
        __syncwarp();
        mx_store_scales(scales, p, byte, tile_cols);
    }
}

template <bool F32>
__global__ void __launch_bounds__(kMxThreads) mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, int M, int K,
                                                                   void* __restrict__ out, long long ldo,
                                                                   int tile_cols, long long items) {
    const long long step = (long long)gridDim.x * (kMxThreads / 32);
    for (long long it = (long long)blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const MxPos p = mx_pos(it, M, K, tile_cols);
        if (!p.ok) continue;
        const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + (size_t)p.m * (K >> 1) + (p.k >> 1)));
        const float s = mx_scale(__ldg(scales + mx_scale_offset(p.m, p.k >> 5, tile_cols)));
        float v[16];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = ((i < 4 ? c.x : c.y) >> (8 * (i & 3))) & 0xFFu;
            uint32_t h;
            asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"(b));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            v[2 * i] = f.x * s;
            v[2 * i + 1] = f.y * s;
        }
        if constexpr (F32) {
            float4* o = reinterpret_cast<float4*>(static_cast<float*>(out) + (size_t)p.m * ldo + p.k);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {   // every MXFP4 value is a bf16 value (or overflows to infinity under a byte above 252)
            uint4* o = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + (size_t)p.m * ldo + p.k);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
                    w[j] = *reinterpret_cast<const uint32_t*>(&t);
                }
                o[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

struct MxGrid { int tile_cols; long long items; unsigned blocks; };

// Items of a [M, K] problem: a warp each, grid-stride over at most 8 blocks per SM.
MxGrid mx_grid(int rows, int K) {
    MxGrid g;
    g.tile_cols = (K + 127) / 128;
    g.items = ((long long)rows + 127) / 128 * 32 * g.tile_cols;
    long long b = (g.items + kMxThreads / 32 - 1) / (kMxThreads / 32);
    const long long cap = (long long)sm_count() * 8;
    g.blocks = (unsigned)(b < cap ? b : cap);
    return g;
}

// Shape and alignment checks shared by the entry points; `ld` in elements of `esize` bytes.
int mx_check(const void* x, const void* codes, const void* scales, long long ld, int M, int K, int width, int esize) {
    if (M <= 0 || K <= 0 || (K & 31) || ld < width) return NVFP4B_ERR_SHAPE;
    if (!x || !codes || !scales) return NVFP4B_ERR_NULL;
    if (!aligned16(x) || !aligned16(codes) || !aligned16(scales) || (ld * esize) % 16) return NVFP4B_ERR_ALIGN;
    return NVFP4B_OK;
}

template <typename T>
int mx_launch_quantize(const T* x, long long ldx, int M, int K, uint8_t* codes, uint8_t* scales, void* stream) {
    const int st = mx_check(x, codes, scales, ldx, M, K, K, sizeof(T));
    if (st) return st;
    const MxGrid g = mx_grid(M, K);
    return launch_k(mx_quantize_kernel<T>, dim3(g.blocks), dim3(kMxThreads), 0, (cudaStream_t)stream, x, ldx, M, K,
                    codes, scales, g.tile_cols, g.items);
}

}  // namespace
}  // namespace nvfp4b

using namespace nvfp4b;

extern "C" size_t nvfp4b_mx_scale_buffer_bytes(int outer, int K) {
    if (outer <= 0 || K <= 0) return 0;
    return ((size_t)outer + 127) / 128 * (((size_t)K + 127) / 128) * 512;
}

extern "C" int nvfp4b_mx_swizzle_scales(const uint8_t* logical, uint8_t* swizzled, int outer, int K, void* stream) {
    if (outer <= 0 || K <= 0 || (K & 31)) return NVFP4B_ERR_SHAPE;
    return nvfp4b_swizzle_scales(logical, swizzled, outer, K / 2, stream);   // K/32 = (K/2)/16 bytes per row
}

extern "C" int nvfp4b_mx_quantize_bf16(const void* x, long long ldx, int M, int K, uint8_t* codes, uint8_t* scales,
                                       void* stream) {
    return mx_launch_quantize(static_cast<const uint16_t*>(x), ldx, M, K, codes, scales, stream);
}

extern "C" int nvfp4b_mx_quantize_f32(const float* x, long long ldx, int M, int K, uint8_t* codes, uint8_t* scales,
                                      void* stream) {
    return mx_launch_quantize(x, ldx, M, K, codes, scales, stream);
}

extern "C" int nvfp4b_mx_geglu_quantize(const void* gate_up, long long ld, int M, int I, uint8_t* codes,
                                        uint8_t* scales, void* stream) {
    if (I > (1 << 30)) return NVFP4B_ERR_SHAPE;
    const int st = mx_check(gate_up, codes, scales, ld, M, I, 2 * I, 2);
    if (st) return st;
    const MxGrid g = mx_grid(M, I);
    return launch_k(mx_geglu_kernel, dim3(g.blocks), dim3(kMxThreads), 0, (cudaStream_t)stream,
                    static_cast<const uint16_t*>(gate_up), ld, M, I, codes, scales, g.tile_cols, g.items);
}

extern "C" int nvfp4b_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int M, int K, void* out, int out_f32,
                                    long long ldo, void* stream) {
    if (out_f32 != 0 && out_f32 != 1) return NVFP4B_ERR_ARG;
    const int st = mx_check(out, codes, scales, ldo, M, K, K, out_f32 ? 4 : 2);
    if (st) return st;
    const MxGrid g = mx_grid(M, K);
    return launch_k(out_f32 ? mx_dequantize_kernel<true> : mx_dequantize_kernel<false>, dim3(g.blocks),
                    dim3(kMxThreads), 0, (cudaStream_t)stream, codes, scales, M, K, out, ldo, g.tile_cols, g.items);
}
