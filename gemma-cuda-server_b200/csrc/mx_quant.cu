// mx_quant.cu -- MXFP4 quantisers (plain, and gated: gelu_tanh(gate) * up) and the dequantiser.
//
// All three are streams: the quantiser reads 2 or 4 bytes and writes 17/32 per element, the gated one reads 4, the
// dequantiser reads 17/32 and writes 2 or 4.  In the quantisers a thread owns 16 consecutive elements, two threads one
// block, eight threads the four blocks of one row of a scale tile; the four eighths of a warp take the rows m, m + 32,
// m + 64, m + 96 of one 128-row tile, whose scale words are neighbours in the tile layout, so a warp writes its 16
// scale bytes as one run and reads four runs of 128 elements.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "mx.cuh"

namespace nvfp4b {
namespace {

constexpr int kMxThreads = 256;

struct MxPos {
    int m, k;          // row, first of the thread's 16 elements
    bool ok;           // both exist
};

// Work item -> this thread's elements.  Items run over (128-row tile, row in 0..31, column tile), columns fastest.
__device__ __forceinline__ MxPos mx_pos(uint32_t item, int M, int K, uint32_t tile_cols) {
    const int lane = threadIdx.x & 31;
    const uint32_t rowgrp = item / tile_cols, c = item - rowgrp * tile_cols;
    MxPos p;
    p.m = (int)(rowgrp >> 5) * 128 + (int)(rowgrp & 31) + (lane >> 3) * 32;
    p.k = (int)c * 128 + (lane & 7) * 16;
    p.ok = p.m < M && p.k < K;
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

// 32 bytes in one load where the address allows it (sm_100's 256-bit accesses), else two of 16.
struct Raw32 { uint32_t w[8]; };
template <bool WIDE>
__device__ __forceinline__ Raw32 load32(const void* p) {
    Raw32 r;
    if constexpr (WIDE) {
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]), "=r"(r.w[4]), "=r"(r.w[5]), "=r"(r.w[6]),
                       "=r"(r.w[7])
                     : "l"(p));
    } else {
        const uint4 a = __ldg(static_cast<const uint4*>(p)), b = __ldg(static_cast<const uint4*>(p) + 1);
        r = Raw32{{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
    }
    return r;
}
template <bool WIDE>
__device__ __forceinline__ void store32(void* p, const Raw32& r) {
    if constexpr (WIDE) {
        asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r.w[0]), "r"(r.w[1]), "r"(r.w[2]),
                     "r"(r.w[3]), "r"(r.w[4]), "r"(r.w[5]), "r"(r.w[6]), "r"(r.w[7]), "l"(p)
                     : "memory");
    } else {
        static_cast<uint4*>(p)[0] = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
        static_cast<uint4*>(p)[1] = make_uint4(r.w[4], r.w[5], r.w[6], r.w[7]);
    }
}

__device__ __forceinline__ float2 bf16x2(uint32_t w) { return make_float2(bf16lo(w), bf16hi(w)); }

// 16 elements as loaded (32 bytes of bf16 or 64 of fp32), and as eight pairs.
template <typename T, bool WIDE>
struct Raw16 {
    Raw32 r[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = load32<WIDE>(reinterpret_cast<const uint8_t*>(p) + 32 * i);
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = Raw32{{0, 0, 0, 0, 0, 0, 0, 0}};
    }
    __device__ __forceinline__ float2 pair(int j) const {
        if constexpr (sizeof(T) == 2) return bf16x2(r[0].w[j]);
        else return make_float2(__uint_as_float(r[j >> 2].w[2 * (j & 3)]), __uint_as_float(r[j >> 2].w[2 * (j & 3) + 1]));
    }
    // Largest magnitude as fp32 bits; NaN orders above infinity.
    __device__ __forceinline__ uint32_t amax() const {
        if constexpr (sizeof(T) == 2) {
            uint32_t b = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) b = __vmaxu2(b, r[0].w[j] & 0x7FFF7FFFu);
            return max(b << 16, b & 0xFFFF0000u);
        } else {
            uint32_t b = 0;
#pragma unroll
            for (int j = 0; j < 16; ++j) b = max(b, r[j >> 3].w[j & 7] & 0x7FFFFFFFu);
            return b;
        }
    }
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kMxThreads) mx_quantize_kernel(const T* __restrict__ x, long long ldx, int M, int K,
                                                                 uint8_t* __restrict__ codes,
                                                                 uint8_t* __restrict__ scales, uint32_t tile_cols,
                                                                 uint32_t items) {
    const uint32_t step = gridDim.x * (kMxThreads / 32);
    for (uint32_t it = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const MxPos p = mx_pos(it, M, K, tile_cols);
        Raw16<T, WIDE> r;
        r.zero();
        if (p.ok) r.load(x + (size_t)p.m * ldx + p.k);
        uint32_t a = r.amax();
        a = max(a, __shfl_xor_sync(0xFFFFFFFFu, a, 1));
        const uint32_t byte = mx_byte(a);
        if (p.ok) {
            const float inv = mx_inv_scale(min(byte, 252u));
            float2 q[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j] = __fmul2_rn(r.pair(j), make_float2(inv, inv));
            uint2 c = make_uint2(cvt_e2m1x8(q[0].x, q[0].y, q[1].x, q[1].y, q[2].x, q[2].y, q[3].x, q[3].y),
                                 cvt_e2m1x8(q[4].x, q[4].y, q[5].x, q[5].y, q[6].x, q[6].y, q[7].x, q[7].y));
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

// float64 redo of one block by a warp, an element per lane (by the block's two threads alone it took 7 us, which the
// last warps of a launch showed): stores the codes, returns the scale byte.
__device__ __noinline__ uint32_t geglu_block64(const uint16_t* gp, const uint16_t* up, uint8_t* codes) {
    const int lane = threadIdx.x & 31;
    const double h = geglu64((double)__uint_as_float((uint32_t)gp[lane] << 16),
                             (double)__uint_as_float((uint32_t)up[lane] << 16));
    double a = h != h ? __longlong_as_double(0x7FF0000000000000ll) : fabs(h);   // NaN as infinity: byte 0xFF
#pragma unroll
    for (int o = 16; o; o >>= 1) a = fmax(a, __shfl_xor_sync(0xFFFFFFFFu, a, o));
    const uint32_t byte = mx_byte64(a);
    uint32_t c = byte == 255u ? 0u : mx_code64(h, byte) << (4 * (lane & 7));
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) c |= __shfl_xor_sync(0xFFFFFFFFu, c, o);
    if ((lane & 7) == 0) reinterpret_cast<uint32_t*>(codes)[lane >> 3] = c;
    return byte;
}

// Whether estimates that have no relative bound matter: where -w nears the end of the fp32 range or h the subnormals,
// |h| <= |g u| 2^-100, and such an element has code 0 (the smallest magnitude with another one is above top / 32) unless
// the whole block is that small.  From g = -1.5e13 down w and its bound are infinities: 0 * inf would make both ends of a
// signed zero NaN, whose codes agree.
__device__ __noinline__ bool geglu_tiny(const uint16_t* gp, const uint16_t* up, float top) {
    const Raw32 rg = load32<false>(gp), ru = load32<false>(up);
    float tiny = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float g = (i & 1) ? bf16hi(rg.w[i >> 1]) : bf16lo(rg.w[i >> 1]);
        const float u = (i & 1) ? bf16hi(ru.w[i >> 1]) : bf16lo(ru.w[i >> 1]);
        if (g < -0x1p43f) return true;
        if (g != 0.f && u != 0.f) tiny = fmaxf(tiny, fmaxf(fabsf(g * u), 1.0f) * 0x1p-100f);
    }
    return tiny > top * 0x1p-6f;
}

// Gated quantiser: h = gelu_tanh(gate) * up of row [gate (I) | up (I)].  With w = 2 t / ln 2 the fp32 estimate
// g * rcp(1 + ex2(-w)) * u is off by at most |h| e, e = max(-w, 1) 2^-22 + 2^-20: the roundings of w leave it 3.5 * 2^-24
// off, so the exponential 2.5 |w| 2^-24, which for w > 0 enters through ex2(-w) / (1 + ex2(-w)) only (below 1 / w);
// ex2.approx 2^-22, the sum, the reciprocal and the products add 9 * 2^-24, h - d and h + d the rest.  The .ftz forms flush
// where w > 126 (the exponential adds nothing to 1) or w < -100 (no bound there, above).
template <bool WIDE>
__global__ void __launch_bounds__(kMxThreads) mx_geglu_kernel(const uint16_t* __restrict__ x, long long ldx, int M,
                                                              int I, uint8_t* __restrict__ codes,
                                                              uint8_t* __restrict__ scales, uint32_t tile_cols,
                                                              uint32_t items) {
    const uint32_t step = gridDim.x * (kMxThreads / 32);
    for (uint32_t it = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const MxPos p = mx_pos(it, M, I, tile_cols);
        const uint16_t* gp = x + (size_t)(p.ok ? p.m : 0) * ldx + (p.ok ? p.k : 0);
        Raw16<uint16_t, WIDE> rg, ru;
        rg.zero();
        ru.zero();
        if (p.ok) {
            rg.load(gp);
            ru.load(gp + I);
        }
        float2 h[8], e[8], sum = make_float2(0.f, 0.f);
        float w_min = 0.f, top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float2 g = rg.pair(j);
            // w / g = 2 sqrt(2/pi) / ln 2 * (1 + 0.044715 g^2)
            const float2 w = __fmul2_rn(g, __ffma2_rn(__fmul2_rn(g, g), make_float2(0.102943240f, 0.102943240f),
                                                      make_float2(2.30220820f, 2.30220820f)));
            float2 ex, rc;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ex.x) : "f"(-w.x));
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ex.y) : "f"(-w.y));
            ex = __fadd2_rn(ex, make_float2(1.f, 1.f));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rc.x) : "f"(ex.x));
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(rc.y) : "f"(ex.y));
            h[j] = __fmul2_rn(__fmul2_rn(g, rc), ru.pair(j));
            e[j] = __ffma2_rn(make_float2(fmaxf(-w.x, 1.f), fmaxf(-w.y, 1.f)), make_float2(0x1p-22f, 0x1p-22f),
                              make_float2(0x1p-20f, 0x1p-20f));
            w_min = fminf(w_min, fminf(w.x, w.y));
            top = fmaxf(top, fmaxf(fabsf(h[j].x), fabsf(h[j].y)));
            sum = __fadd2_rn(sum, h[j]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        // e is below 2^-15 down to w = -100
        const uint32_t hi = __float_as_uint(top * (1.f + 0x1p-15f)), lo = __float_as_uint(top * (1.f - 0x1p-15f));
        const uint32_t field = max(hi & 0x7F800000u, 0x01000000u);     // exponent field, at least 2: mx_byte + 2
        const float inv = __uint_as_float(0x80000000u - field);
        const float total = sum.x + sum.y;                             // NaN where an h is (no maximum shows it)
        bool redo = ((hi ^ lo) & 0x7F800000u) != 0u || hi >= 0x7F000000u || !(total == total);
        if (p.ok && (w_min <= -100.f || hi < 0x12800000u)) redo |= geglu_tiny(gp, gp + I, top);   // 2^-90
        uint32_t c[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float2 a[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 v = __fmul2_rn(h[4 * q + j], make_float2(inv, inv)), d = e[4 * q + j];
                a[j] = __ffma2_rn(v, make_float2(-d.x, -d.y), v);
                b[j] = __ffma2_rn(v, d, v);
            }
            c[q] = cvt_e2m1x8(a[0].x, a[0].y, a[1].x, a[1].y, a[2].x, a[2].y, a[3].x, a[3].y);
            const uint32_t hi_end = cvt_e2m1x8(b[0].x, b[0].y, b[1].x, b[1].y, b[2].x, b[2].y, b[3].x, b[3].y);
            redo |= ((c[q] ^ hi_end) & 0x77777777u) != 0u;             // a relative bound leaves no doubt about signs, and
            c[q] = hi_end;                                             // h + d keeps that of a zero
        }
        redo |= __shfl_xor_sync(0xFFFFFFFFu, (int)redo, 1) != 0;      // both threads of a block, on every lane
        redo &= p.ok;
        uint32_t byte = (field >> 23) - 2u;
        if (p.ok && !redo)
            *reinterpret_cast<uint2*>(codes + (size_t)p.m * (I >> 1) + (p.k >> 1)) = make_uint2(c[0], c[1]);
        for (uint32_t left = __ballot_sync(0xFFFFFFFFu, redo) & 0x55555555u; left; left &= left - 1) {
            const int src = __ffs(left) - 1;                           // the first thread of an unproven block
            const int m = __shfl_sync(0xFFFFFFFFu, p.m, src), k = __shfl_sync(0xFFFFFFFFu, p.k, src);
            const uint16_t* row = x + (size_t)m * ldx + k;
            const uint32_t b = geglu_block64(row, row + I, codes + (size_t)m * (I >> 1) + (k >> 1));
            if (((threadIdx.x & 31) ^ src) < 2) byte = b;
        }
        mx_store_scales(scales, p, byte, tile_cols);
    }
}

// A warp takes 512 consecutive elements of a row (fp32 out: 256), a lane the 16-byte (32-byte) piece of each quarter
// that makes its stores whole sectors in a row.
template <bool F32, bool WIDE>
__global__ void __launch_bounds__(kMxThreads) mx_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                                   const uint8_t* __restrict__ scales, int M, int K,
                                                                   void* __restrict__ out, long long ldo,
                                                                   uint32_t tile_cols, uint32_t spans, uint32_t items) {
    constexpr int kSteps = F32 ? 1 : 2;                       // 256 elements, 8 per lane, each
    const uint32_t step = gridDim.x * (kMxThreads / 32);
    const int lane = threadIdx.x & 31;
    for (uint32_t it = blockIdx.x * (kMxThreads / 32) + (threadIdx.x >> 5); it < items; it += step) {
        const uint32_t m = it / spans;
        const int k0 = (int)(it - m * spans) * (256 * kSteps) + 8 * lane;
        const uint8_t* row = codes + (size_t)m * (K >> 1);
        uint32_t c[kSteps], s[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int k = k0 + 256 * i;
            c[i] = s[i] = 0;
            if (k < K) {
                c[i] = __ldg(reinterpret_cast<const uint32_t*>(row + (k >> 1)));
                s[i] = __ldg(scales + mx_scale_offset((int)m, k >> 5, tile_cols));
            }
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int k = k0 + 256 * i;
            if (k >= K) continue;
            const float f = mx_scale(s[i]);
            float2 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t h;
                asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}"
                    : "=r"(h) : "r"((c[i] >> (8 * j)) & 0xFFu));
                v[j] = __fmul2_rn(__half22float2(*reinterpret_cast<const __half2*>(&h)), make_float2(f, f));
            }
            if constexpr (F32) {
                Raw32 r;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    r.w[2 * j] = __float_as_uint(v[j].x);
                    r.w[2 * j + 1] = __float_as_uint(v[j].y);
                }
                store32<WIDE>(static_cast<float*>(out) + (size_t)m * ldo + k, r);
            } else {   // every MXFP4 value is a bf16 value (or overflows to infinity under a byte above 252)
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const __nv_bfloat162 t = __floats2bfloat162_rn(v[j].x, v[j].y);
                    w[j] = *reinterpret_cast<const uint32_t*>(&t);
                }
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + (size_t)m * ldo + k) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

struct MxGrid { uint32_t tile_cols, items; unsigned blocks; };

// A warp per item, grid-stride over at most `per_sm` blocks per SM.  8192 x 2816: quantise 12.4 us at 16 and 13.5 at 8,
// dequantise 12.6 and 12.7; the gated quantiser, which computes more per item, 11.6 us at 8 and 12.2 at 16 (4096 x 2112).
unsigned mx_blocks(long long items, int per_sm) {
    const long long b = (items + kMxThreads / 32 - 1) / (kMxThreads / 32), cap = (long long)sm_count() * per_sm;
    return (unsigned)(b < cap ? b : cap);
}

// Items of a quantiser: 4 rows x 128 columns each.  False where there are more than 32-bit indices hold.
bool mx_grid(int rows, int K, int per_sm, MxGrid& g) {
    g.tile_cols = ((uint32_t)K + 127) / 128;
    const long long items = ((long long)rows + 127) / 128 * 32 * g.tile_cols;
    g.items = (uint32_t)items;
    g.blocks = mx_blocks(items, per_sm);
    return items < (1ll << 30);
}

bool aligned32(const void* p, long long pitch_bytes) {
    return (reinterpret_cast<uintptr_t>(p) & 31u) == 0 && pitch_bytes % 32 == 0;
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
    MxGrid g;
    if (!mx_grid(M, K, 16, g)) return NVFP4B_ERR_SHAPE;
    const auto kernel = aligned32(x, ldx * (long long)sizeof(T)) ? mx_quantize_kernel<T, true> : mx_quantize_kernel<T, false>;
    return launch_k(kernel, dim3(g.blocks), dim3(kMxThreads), 0, (cudaStream_t)stream, x, ldx, M, K, codes, scales,
                    g.tile_cols, g.items);
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
    if (I >= (1 << 30)) return NVFP4B_ERR_SHAPE;
    const int st = mx_check(gate_up, codes, scales, ld, M, I, 2 * I, 2);
    if (st) return st;
    MxGrid g;
    if (!mx_grid(M, I, 8, g)) return NVFP4B_ERR_SHAPE;
    const bool wide = aligned32(gate_up, ld * 2);      // the up half lies I, a multiple of 32, elements behind
    return launch_k(wide ? mx_geglu_kernel<true> : mx_geglu_kernel<false>, dim3(g.blocks), dim3(kMxThreads), 0,
                    (cudaStream_t)stream, static_cast<const uint16_t*>(gate_up), ld, M, I, codes, scales, g.tile_cols,
                    g.items);
}

extern "C" int nvfp4b_mx_dequantize(const uint8_t* codes, const uint8_t* scales, int M, int K, void* out, int out_f32,
                                    long long ldo, void* stream) {
    if (out_f32 != 0 && out_f32 != 1) return NVFP4B_ERR_ARG;
    const int st = mx_check(out, codes, scales, ldo, M, K, K, out_f32 ? 4 : 2);
    if (st) return st;
    const uint32_t span = out_f32 ? 256 : 512, spans = ((uint32_t)K + span - 1) / span;
    const long long items = (long long)M * spans;
    if (items >= (1ll << 30)) return NVFP4B_ERR_SHAPE;
    const auto kernel = !out_f32                     ? mx_dequantize_kernel<false, false>
                        : aligned32(out, ldo * 4LL) ? mx_dequantize_kernel<true, true>
                                                     : mx_dequantize_kernel<true, false>;
    return launch_k(kernel, dim3(mx_blocks(items, 16)), dim3(kMxThreads), 0, (cudaStream_t)stream, codes, scales, M, K, out,
                    ldo, ((uint32_t)K + 127) / 128, spans, (uint32_t)items);
}
