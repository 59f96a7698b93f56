// dense_epi.cuh -- epilogue policy of the dense GEMMs (NVFP4 and MXFP4): alpha times the accumulator as bf16 row-major,
// fp32 column-major or fp32 row-major.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "gemm_core.cuh"

namespace nvfp4b {

// STAGED (bf16 row-major only): each epilogue warp turns its 32-row x 32-column chunks around in a 2 KB
// shared-memory tile (16-byte segments XOR-swizzled by (row >> 1) & 3, conflict-free both ways) so every store
// instruction writes 8 rows x 64 contiguous bytes -- whole sectors -- instead of 32 rows x 16 bytes.
constexpr int kStoreTileBytes = 2048;   // per epilogue warp: one 32 x 32 bf16 tile

template <int OUT, bool STAGED = false>
struct DenseEpi {
    void* d;
    long long ldd;
    int M, N;
    float alpha, b_dequant;
    const float* d_a_amax;

    __device__ __forceinline__ void store_staged(int row0, int n0, int lane, const uint32_t (&r)[32], float a,
                                                 uint8_t* tile) const {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 h = __floats2bfloat162_rn(a * __uint_as_float(r[8 * v + 2 * i]),
                                                               a * __uint_as_float(r[8 * v + 2 * i + 1]));
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
            *reinterpret_cast<uint4*>(tile + lane * 64 + ((v ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int seg = lane & 3;
        const int col = n0 + 8 * seg;
        const bool vec = n0 + 32 <= N && (ldd & 7) == 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int rr = 8 * i + (lane >> 2);
            const uint4 val = *reinterpret_cast<const uint4*>(tile + rr * 64 + ((seg ^ ((rr >> 1) & 3)) << 4));
            const long long m = (long long)row0 + rr;
            if (m >= M) continue;
            __nv_bfloat16* D = static_cast<__nv_bfloat16*>(d) + m * ldd + col;
            if (vec) {
                *reinterpret_cast<uint4*>(D) = val;
            } else {
                const __nv_bfloat16* h = reinterpret_cast<const __nv_bfloat16*>(&val);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < N) D[e] = h[e];
            }
        }
        __syncwarp();
    }

    __device__ __forceinline__ void store(long long m, int n0, const uint32_t (&r)[32], float a) const {
        if constexpr (OUT == NVFP4B_OUT_BF16_ROWMAJOR) {
            __nv_bfloat16* D = static_cast<__nv_bfloat16*>(d) + m * ldd + n0;
            if (n0 + 32 <= N && (ldd & 7) == 0) {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const __nv_bfloat162 h = __floats2bfloat162_rn(a * __uint_as_float(r[8 * v + 2 * i]),
                                                                       a * __uint_as_float(r[8 * v + 2 * i + 1]));
                        w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    *reinterpret_cast<uint4*>(D + 8 * v) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (n0 + i < N) D[i] = __float2bfloat16_rn(a * __uint_as_float(r[i]));
            }
        } else if constexpr (OUT == NVFP4B_OUT_F32_COLMAJOR) {
            float* D = static_cast<float*>(d) + m;
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (n0 + i < N) D[(long long)(n0 + i) * ldd] = a * __uint_as_float(r[i]);
        } else {
            float* D = static_cast<float*>(d) + m * ldd + n0;
            if (n0 + 32 <= N && (ldd & 3) == 0) {
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    *reinterpret_cast<float4*>(D + 4 * v) =
                        make_float4(a * __uint_as_float(r[4 * v]), a * __uint_as_float(r[4 * v + 1]),
                                    a * __uint_as_float(r[4 * v + 2]), a * __uint_as_float(r[4 * v + 3]));
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (n0 + i < N) D[i] = a * __uint_as_float(r[i]);
            }
        }
    }

    __device__ __forceinline__ void finish() const {}
    __device__ __forceinline__ bool row_live(const TileInfo&, int) const { return true; }

    template <int CH>
    __device__ __forceinline__ void process(const TileInfo& ti, int row, int col_base, const uint32_t (&r)[CH][32],
                                            uint8_t* esm) const {
        const float a = d_a_amax ? __fdiv_rn(b_dequant, gscale_from_amax(__ldg(d_a_amax))) : alpha;
        if constexpr (STAGED && OUT == NVFP4B_OUT_BF16_ROWMAJOR) {
            const int lane = threadIdx.x & 31;
            uint8_t* tile = esm + ((threadIdx.x >> 5) - 4) * kStoreTileBytes;   // epilogue warps are 4..
            const int row0 = ti.a_row + row - lane;
            if (row0 >= M) return;                                            // warp-uniform
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int n0 = ti.n0 + col_base + 32 * c;                    // warp-uniform
                if (n0 < N) store_staged(row0, n0, lane, r[c], a, tile);
            }
            return;
        }
        const long long m = (long long)ti.a_row + row;
        if (m >= M) return;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int n0 = ti.n0 + col_base + 32 * c;
            if (n0 < N) store(m, n0, r[c], a);
        }
    }
};

}  // namespace nvfp4b
