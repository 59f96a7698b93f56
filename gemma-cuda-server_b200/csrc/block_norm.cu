// block_norm.cu -- the norms around a transformer block, with its gate, residual and residual scale, in one pass:
//   n = rms(y; eps) * post_w,   r = scale * (resid + gate * n),   z = rms(r; eps) * norm_w
// r is written as the new residual; z as bf16 (with its max |.|, the dynamic scale of an NVFP4 quantiser) and/or as MXFP4
// codes and scales.  Each input is read once and each output written once: the row stays in registers.
//
// One CTA per row, 8 consecutive elements per thread and chunk; the two sums of squares are block reductions.  The codes
// stored are those of the float64 z: with u = 2^-24 the fp32 r is off by at most 17 u a, a = |scale| (|resid| +
// |gate n|) (12 u for rsqrt of a mean of squares -- 8 + 5 + 5 additions, half of them after the root -- and the
// products after it), and z by
//   d = |f w| (20 u a + |r| (16 u + 20 u k)),  k = sqrt(sum a^2 / sum r^2),  f = 1 / rms(r)
// (without y: r is one product, d = 20 u |z|).  Where the codes of z - d and z + d differ, or a sum of squares leaves
// the range in which the bounds hold, the CTA redoes its row in float64.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "mx.cuh"

namespace nvfp4b {
namespace {

constexpr int kNormMaxThreads = 512;

struct NormParams {
    nvfp4b_block_norm_args a;
    int tile_cols;
    float inv_h;
};

__device__ __forceinline__ void load8(const void* p, bool f32, long long i, float (&v)[8]) {
    if (f32) {
        const float4 q0 = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 q1 = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + 4);
        v[0] = q0.x; v[1] = q0.y; v[2] = q0.z; v[3] = q0.w;
        v[4] = q1.x; v[5] = q1.y; v[6] = q1.z; v[7] = q1.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { v[2 * j] = bf16lo(w[j]); v[2 * j + 1] = bf16hi(w[j]); }
    }
}

__device__ __forceinline__ float load1(const void* p, bool f32, long long i) {
    return f32 ? static_cast<const float*>(p)[i] : __uint_as_float((uint32_t)static_cast<const uint16_t*>(p)[i] << 16);
}

__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&t);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Gate of element (row, i): per token, per feature or per element by its strides; 1 without a gate.
__device__ __forceinline__ float gate_at(const nvfp4b_block_norm_args& a, int row, int i) {
    return a.gate ? load1(a.gate, a.gate_f32 != 0, row * a.gate_row_stride + (long long)i * a.gate_col_stride) : 1.0f;
}

// Block-wide sum, the same bits on every thread.  `red` (one value per warp) must not be in use.
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* red) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (lane == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? red[lane] : T(0);
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Whether a mean of squares (+ eps) is in the range where its fp32 value has its relative error bound.
__device__ __forceinline__ bool mean_ok(float m) { return m > 0x1p-80f && m < 0x1p100f; }

// r of element i in float64; f = 1 / rms(y).
__device__ __forceinline__ double r64(const nvfp4b_block_norm_args& a, int row, int i, double f) {
    double r = a.resid ? (double)load1(a.resid, a.resid_f32 != 0, row * a.ld_resid + i) : 0.0;
    if (a.y) {
        double n = (double)load1(a.y, a.y_f32 != 0, row * a.ld_y + i) * f;
        if (a.post_weight) n *= (double)load1(a.post_weight, false, i);
        r += (double)gate_at(a, row, i) * n;
    }
    return r * (double)a.scale;
}

template <int NCH, bool MX>
__global__ void __launch_bounds__(kNormMaxThreads) block_norm_kernel(const __grid_constant__ NormParams p) {
    __shared__ float red[3][kNormMaxThreads / 32];
    __shared__ double red64[2][kNormMaxThreads / 32];
    __shared__ uint32_t red_max[kNormMaxThreads / 32];
    const nvfp4b_block_norm_args& a = p.a;
    const int row = blockIdx.x, tid = threadIdx.x, threads = blockDim.x, chunks = a.H >> 3;
    const bool want_z = a.out || MX;
    bool redo = false;

    float r[NCH][8], bound[MX ? NCH : 1][8];      // bound: |scale| (|resid| + |gate n|)
    if (a.y) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
#pragma unroll
            for (int i = 0; i < 8; ++i) r[c][i] = 0.f;
            if (ch < chunks) load8(a.y, a.y_f32 != 0, row * a.ld_y + ch * 8, r[c]);
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(r[c][i], r[c][i], s);
            ss += s;
        }
        float f = 1.f;
        if (a.post_norm) {
            const float m = fmaf(block_sum(ss, red[0]), p.inv_h, a.eps);
            redo |= !mean_ok(m);
            f = __frsqrt_rn(m);
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
            if (ch >= chunks) {
                if constexpr (MX) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) bound[c][i] = 0.f;
                }
                continue;
            }
            float w[8], v[8], g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) { w[i] = 1.f; v[i] = 0.f; g[i] = 1.f; }
            if (a.post_weight) load8(a.post_weight, false, ch * 8, w);
            if (a.resid) load8(a.resid, a.resid_f32 != 0, row * a.ld_resid + ch * 8, v);
            if (a.gate) {
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = gate_at(a, row, ch * 8 + i);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float t = r[c][i] * f * w[i] * g[i];
                r[c][i] = a.scale * (v[i] + t);
                if constexpr (MX) bound[c][i] = fabsf(a.scale) * (fabsf(v[i]) + fabsf(t));
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
#pragma unroll
            for (int i = 0; i < 8; ++i) r[c][i] = 0.f;
            if (ch < chunks) load8(a.resid, a.resid_f32 != 0, row * a.ld_resid + ch * 8, r[c]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                r[c][i] *= a.scale;
                if constexpr (MX) bound[c][i] = fabsf(r[c][i]);
            }
        }
    }

    float z[NCH][8];
    uint32_t code[MX ? NCH : 1], byte[MX ? NCH : 1];
    if (want_z) {
        float ss = 0.f, sa = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            float s = 0.f, t = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                s = fmaf(r[c][i], r[c][i], s);
                if constexpr (MX) t = fmaf(bound[c][i], bound[c][i], t);
            }
            ss += s;
            sa += t;
        }
        ss = block_sum(ss, red[1]);
        const float m = fmaf(ss, p.inv_h, a.eps);
        redo |= !mean_ok(m);
        const float f = __frsqrt_rn(m);
        float rel = 0.f;                               // 16 u + 20 u k
        if constexpr (MX) {
            if (a.y) {
                sa = block_sum(sa, red[2]);
                rel = sa > 0.f ? fmaf(sqrtf(sa / ss), 0x1.4p-20f, 0x1p-20f) : 0.f;
                redo |= !(rel < 0x1p-10f);             // also where ss = 0 < sa: r cancelled altogether
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = 1.f;
            if (a.norm_weight && ch < chunks) load8(a.norm_weight, false, ch * 8, w);
#pragma unroll
            for (int i = 0; i < 8; ++i) z[c][i] = ch < chunks ? r[c][i] * f * w[i] : 0.f;
            if constexpr (MX) {
                float lo[8], hi[8];
                uint32_t alo = 0, ahi = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float d = ch >= chunks ? 0.f
                                    : a.y        ? fabsf(f * w[i]) * fmaf(fabsf(r[c][i]), rel, 0x1.4p-20f * bound[c][i])
                                                 : 0x1.4p-20f * fabsf(z[c][i]);
                    lo[i] = z[c][i] - d;
                    hi[i] = z[c][i] + d;
                    alo = max(alo, __float_as_uint(fmaxf(fabsf(z[c][i]) - d, 0.f)));
                    ahi = max(ahi, __float_as_uint(fabsf(z[c][i]) + d) & 0x7FFFFFFFu);
                }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    alo = max(alo, __shfl_xor_sync(0xFFFFFFFFu, alo, o));
                    ahi = max(ahi, __shfl_xor_sync(0xFFFFFFFFu, ahi, o));
                }
                byte[c] = mx_byte(ahi);
                const float inv = mx_inv_scale(min(byte[c], 252u));
                code[c] = mx_encode8(lo, inv);
                redo |= code[c] != mx_encode8(hi, inv) || byte[c] != mx_byte(alo) || (ahi >> 23) >= 254u ||
                        (ahi != 0u && ahi < 0x08800000u);     // below 2^-110 the products' bounds fail
            }
        }
    }

    if (__syncthreads_or(redo)) {                     // the whole row in float64, inputs read again
        double f = 1.0;
        if (a.y && a.post_norm) {
            double s = 0.0;
#pragma unroll 1
            for (int i = tid; i < a.H; i += threads) {
                const double v = (double)load1(a.y, a.y_f32 != 0, row * a.ld_y + i);
                s = fma(v, v, s);
            }
            f = 1.0 / sqrt(block_sum(s, red64[0]) / a.H + (double)a.eps);
        }
        double s = 0.0;
#pragma unroll 1
        for (int i = tid; i < a.H; i += threads) {
            const double v = r64(a, row, i, f);
            s = fma(v, v, s);
        }
        const double f2 = 1.0 / sqrt(block_sum(s, red64[1]) / a.H + (double)a.eps);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const int ch = tid + c * threads;
            double amax = 0.0;
            bool nan = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (ch >= chunks) continue;
                const double v = r64(a, row, ch * 8 + i, f);
                const double w = a.norm_weight ? (double)load1(a.norm_weight, false, ch * 8 + i) : 1.0;
                const double zz = v * f2 * w;
                r[c][i] = (float)v;
                z[c][i] = (float)zz;
                nan |= zz != zz;
                amax = fmax(amax, fabs(zz));
            }
            if constexpr (MX) {
                if (nan) amax = __longlong_as_double(0x7FF0000000000000ll);    // as an infinity: byte 0xFF
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) amax = fmax(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
                byte[c] = mx_byte64(amax);
                code[c] = 0u;
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                    if (ch >= chunks || byte[c] == 255u) continue;
                    const double v = r64(a, row, ch * 8 + i, f);
                    const double w = a.norm_weight ? (double)load1(a.norm_weight, false, ch * 8 + i) : 1.0;
                    code[c] |= mx_code64(v * f2 * w, byte[c]) << (4 * i);
                }
            }
        }
        __syncthreads();                              // every read of the row before the (possibly in-place) writes
    }

    uint32_t zmax = 0;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
        const int ch = tid + c * threads;
        const bool ok = ch < chunks;
        if (a.resid_out && ok) {
            if (a.resid_out_f32) {
                float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.resid_out) + row * a.ld_resid_out + ch * 8);
                o[0] = make_float4(r[c][0], r[c][1], r[c][2], r[c][3]);
                o[1] = make_float4(r[c][4], r[c][5], r[c][6], r[c][7]);
            } else {
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.resid_out) + row * a.ld_resid_out + ch * 8) =
                    pack8(r[c]);
            }
        }
        if (a.out && ok) {
            const uint4 q = pack8(z[c]);
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.ld_out + ch * 8) = q;
            const uint32_t w = __vmaxu2(__vmaxu2(q.x & 0x7FFF7FFFu, q.y & 0x7FFF7FFFu),
                                        __vmaxu2(q.z & 0x7FFF7FFFu, q.w & 0x7FFF7FFFu));
            zmax = max(zmax, max(w & 0xFFFFu, w >> 16));
        }
        if constexpr (MX) {
            if (ok) *reinterpret_cast<uint32_t*>(a.codes + (size_t)row * (a.H >> 1) + ch * 4) = code[c];
            uint32_t w = ok ? byte[c] << (8 * ((tid & 15) >> 2)) : 0u;
            w |= __shfl_xor_sync(0xFFFFFFFFu, w, 4);
            w |= __shfl_xor_sync(0xFFFFFFFFu, w, 8);
            if ((tid & 15) == 0 && (ch >> 4) < p.tile_cols)
                *reinterpret_cast<uint32_t*>(a.scales + mx_scale_offset(row, ch >> 2, p.tile_cols)) = w;
        }
    }
    if constexpr (MX) {                               // padding rows of the last scale tile row, dealt over the CTAs
        const int padded = (a.T + 127) / 128 * 128;
        for (int m = a.T + row; m < padded; m += gridDim.x)
            for (int t = tid; t < p.tile_cols; t += threads)
                *reinterpret_cast<uint32_t*>(a.scales + mx_scale_offset(m, 4 * t, p.tile_cols)) = 0u;
    }
    if (a.amax) {
        zmax = __reduce_max_sync(0xFFFFFFFFu, zmax);
        if ((tid & 31) == 0) red_max[tid >> 5] = zmax;
        __syncthreads();
        if (tid < 32) {
            zmax = __reduce_max_sync(0xFFFFFFFFu, tid < (threads >> 5) ? red_max[tid] : 0u) << 16;
            // same-address atomics serialise: a row that cannot raise the maximum seen so far skips its own
            if (tid == 0 && zmax > *reinterpret_cast<volatile uint32_t*>(a.amax))
                atomicMax(reinterpret_cast<unsigned int*>(a.amax), zmax);
        }
    }
}

template <int NCH>
int launch_block_norm(const NormParams& p, int threads, cudaStream_t s) {
    return launch_k(p.a.codes ? block_norm_kernel<NCH, true> : block_norm_kernel<NCH, false>, dim3(p.a.T),
                    dim3(threads), 0, s, p);
}

bool bad_rows(const void* p, int f32, long long ld) { return !aligned16(p) || (ld * (f32 ? 4 : 2)) % 16; }

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
    const cudaStream_t s = (cudaStream_t)stream;
    if (a.amax) {
        const cudaError_t e = cudaMemsetAsync(a.amax, 0, sizeof(float), s);
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    NormParams p;
    p.a = a;
    p.tile_cols = (a.H + 127) / 128;
    p.inv_h = 1.0f / (float)a.H;
    const int chunks = a.H / 8, nch = chunks <= kNormMaxThreads ? 1 : chunks <= 2 * kNormMaxThreads ? 2 : 4;
    const int threads = (chunks + nch * 32 - 1) / (nch * 32) * 32;
    if (nch == 1) return launch_block_norm<1>(p, threads, s);
    if (nch == 2) return launch_block_norm<2>(p, threads, s);
    return launch_block_norm<4>(p, threads, s);
}
