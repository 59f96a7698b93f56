// mx_gemm.cu -- dense MXFP4 GEMM, D = alpha * A[M, K] @ B[N, K]^T, on the tcgen05 core (gemm_core.cuh, Kind::MXF4).
//
// One e8m0 scale per 32 elements: a 512-byte scale tile (128 rows x 4 blocks) serves two 64-element MMAs, so a K-tile
// needs half of the scale copies (tcgen05.cp) that NVFP4's scale per 16 does.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "gemm_core.cuh"
#include "sm100.cuh"

namespace nvfp4b {
namespace {

struct MxGemm {
    const uint8_t *a, *a_sf, *b, *b_sf;
    float alpha;
    int M, N, K;
    void* d;
    long long ldd;
};

// Epilogue of the CTA-pair tiles, which compute D^T = B A^T: a thread holds 32 columns of one row of the tile, so the lanes'
// elements lie together in row-major D and each is stored from its register, 64 or 128 bytes of a row per instruction, at
// any pitch.  The address goes up by additions: with a product for each element 4096 x 7000, K = 512 fp32 took 48% longer;
// through a swizzled tile in shared memory to 16 bytes per lane 14% (bf16 13%).
template <typename T>
struct MxEpi {
    T* d;
    long long ldd;                                                 // between the columns of the tile
    int M, N;                                                      // of D^T
    float alpha;

    __device__ __forceinline__ void finish() const {}

    template <int CH>
    __device__ __forceinline__ void process(const TileInfo& ti, int row, int col_base, const uint32_t (&r)[CH][32],
                                            uint8_t*) const {
        const int m = ti.a_row + row;
        if (m >= M) return;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int n0 = ti.n0 + col_base + 32 * c;              // warp-uniform
            T* at = d + n0 * ldd + m;
            if (n0 + 32 <= N) {
#pragma unroll
                for (int i = 0; i < 32; ++i, at += ldd) *at = T(alpha * __uint_as_float(r[c][i]));
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i, at += ldd)
                    if (n0 + i < N) *at = T(alpha * __uint_as_float(r[c][i]));
            }
        }
    }
};

using MxPair = PairCfg<6, 8, 0, Kind::MXF4>;

int mx_core_params(const MxGemm& g, CoreParams& cp) {
    cp.err = device_error_ptr();
    if (!cp.err) return NVFP4B_ERR_CUDA;
    cp.sfa = g.a_sf;
    cp.sfb = g.b_sf;
    cp.tile_cols = (g.K + 127) / 128;
    cp.mx_steps = (g.K + 63) / 64;
    cp.k_tiles = (g.K + 255) / 256;
    return NVFP4B_OK;
}

// ---------------------------------------------------------------------------------------------------------------
// Few rows: the weights as the M = 128 operand
// ---------------------------------------------------------------------------------------------------------------
// D^T = B A^T: 128 rows of B (the weights) against NT = 16, 32, 64 or 128 rows of A.  What a call of few rows does is
// stream the weights, so the tile is narrow in A's rows (the tensor pipe and the epilogue do no work for padding) and K
// is split over the S CTAs of a cluster while there are fewer tiles than SMs; the partial sums meet in distributed shared
// memory, each CTA adding up every S-th row in rank order (the same bits every time, no workspace).  One CTA per SM with
// about 200 KB of stages; persistent over tiles when S = 1, with two accumulators.
//   warp 0      producer: TMA loads of the weights (128 x 128 bytes) and of A (NT x 128 bytes), bulk loads of the scales
//   warp 1      TMEM owner and MMA issuer
//   warps 2..   epilogue, TMEM lane quadrant warp % 4: a thread holds one column n of D, 16 rows at a time.  Eight warps from
//               32 rows on, two to a quadrant: a warp's own instructions are what the epilogue takes (512 x 2816,
//               K = 2112 8.3 us with four, 7.9 with eight, no gain with sixteen)
//   last warp   scale copies (issued by the MMA thread they made a K-tile take 1330 cycles)
template <int NT_>
struct SkinnyCfg {
    static constexpr int NT = NT_, A_BYTES = NT * 128, W_BYTES = 128 * 128, SF_BYTES = 2 * 512;
    static constexpr int STAGE_BYTES = W_BYTES + A_BYTES + 2 * SF_BYTES;
    static constexpr int STAGES = 208 * 1024 / STAGE_BYTES;
    static constexpr int BAR_BYTES = 384;
    static constexpr int EPI_WARPS = NT >= 32 ? 8 : 4;
    static constexpr int TURN = 33, TURN_BYTES = EPI_WARPS * 16 * TURN * 4;   // per epilogue warp: 16 rows x 32 columns, padded
    static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + BAR_BYTES + TURN_BYTES + 1024;
    static constexpr int SF_COL0 = 2 * NT, SF_COLS = 16;          // per stage: 8 columns for the weights, 8 for A
    static constexpr int PART = 132;                              // row pitch of the partial sums, floats
    static constexpr int THREADS = 32 * (3 + EPI_WARPS);
    static_assert(SF_COL0 + STAGES * SF_COLS <= 512, "TMEM budget");
    static_assert((3 * STAGES + 4) * 8 + 16 <= BAR_BYTES, "barriers");
    static_assert(NT * PART * 4 <= STAGES * STAGE_BYTES, "partial sums");
    static_assert(SMEM_BYTES <= 232448, "shared memory budget");
};

// What issue_k_tile takes from its configuration.
template <int NT>
struct MmaOf {
    static constexpr Kind KIND = Kind::MXF4;
    static constexpr int BN = 128;                                // columns of one scale tile's copy: 4
};

struct SkinnyParams {
    const uint8_t *sfa, *sfw;
    void* d;
    long long ldd;
    float alpha;
    int M, N, n_tiles, m_tiles, tile_cols, k_steps, k_tiles;
    int wide;                // d and its pitch allow 16-byte stores
    int* err;
};

template <int OUT>
__device__ __forceinline__ void skinny_store(const SkinnyParams& p, int m, int n, float v) {
    v *= p.alpha;
    if constexpr (OUT == NVFP4B_OUT_BF16_ROWMAJOR) static_cast<__nv_bfloat16*>(p.d)[m * p.ldd + n] = __float2bfloat16_rn(v);
    else if constexpr (OUT == NVFP4B_OUT_F32_ROWMAJOR) static_cast<float*>(p.d)[m * p.ldd + n] = v;
    else static_cast<float*>(p.d)[n * p.ldd + m] = v;
}

// One warp stores rows m0.. (16 of them, `rows` exist) x columns n0.. (32) of D; lane = column in r.  Row-major a lane
// stores its own column, row by row: the lanes' elements lie together, at any pitch (turned around in shared memory to 16
// bytes per lane 512 x 2816, K = 2112 took 6% longer and 128 x 65536, K = 256 13%).  Column-major
// the rows are turned around in `t`.
template <int OUT>
__device__ __forceinline__ void skinny_store16(const SkinnyParams& p, int m0, int rows, int n0, const uint32_t (&r)[16],
                                               float* t) {
    const int lane = threadIdx.x & 31;
    if constexpr (OUT != NVFP4B_OUT_F32_COLMAJOR) {
        using T = std::conditional_t<OUT == NVFP4B_OUT_BF16_ROWMAJOR, __nv_bfloat16, float>;
        T* d = static_cast<T*>(p.d) + m0 * p.ldd + n0 + lane;
        const int mine = n0 + lane < p.N ? rows : 0;
#pragma unroll
        for (int i = 0; i < 16; ++i, d += p.ldd)
            if (i < mine) *d = T(p.alpha * __uint_as_float(r[i]));
    } else {
        constexpr int P = SkinnyCfg<16>::TURN;
#pragma unroll
        for (int i = 0; i < 16; ++i) t[i * P + lane] = p.alpha * __uint_as_float(r[i]);
        __syncwarp();
        if (p.wide && rows >= 16) {                               // a lane stores four rows of one column
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int n = i * 8 + (lane >> 2), m = 4 * (lane & 3);
                if (n0 + n < p.N)
                    *reinterpret_cast<float4*>(static_cast<float*>(p.d) + (n0 + n) * p.ldd + m0 + m) =
                        make_float4(t[m * P + n], t[(m + 1) * P + n], t[(m + 2) * P + n], t[(m + 3) * P + n]);
            }
        } else {                                                  // half a warp stores the 16 rows of one column
            const int m = lane & 15, n1 = m < rows ? min(32, p.N - n0) : 0;
            float* d = static_cast<float*>(p.d) + (n0 + (lane >> 4)) * p.ldd + m0 + m;
#pragma unroll
            for (int n = 0; n < 32; n += 2, d += 2 * p.ldd)
                if (n + (lane >> 4) < n1) *d = t[m * P + n + (lane >> 4)];
        }
    }
    __syncwarp();
}

// Sum, in rank order, of the four fp32 at one shared-memory address of the S <= 8 CTAs of the cluster; every load is issued
// before the first addition waits for one.
__device__ __forceinline__ float4 cluster_sum(uint32_t addr, int S) {
    float4 x[8];
#pragma unroll
    for (int q = 0; q < 8; ++q)
        x[q] = q < S ? sm100::ld_cluster_f32x4(sm100::mapa_shared(addr, (uint32_t)q)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int q = 1; q < 8; ++q) { x[0].x += x[q].x; x[0].y += x[q].y; x[0].z += x[q].z; x[0].w += x[q].w; }
    return x[0];
}

template <int NT, int OUT>
__global__ void __launch_bounds__(SkinnyCfg<NT>::THREADS, 1)
    mx_skinny_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_w,
                     const __grid_constant__ SkinnyParams p) {
    using namespace sm100;
    using C = SkinnyCfg<NT>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* sW = smem;
    uint8_t* sA = sW + C::STAGES * C::W_BYTES;
    uint8_t* sSF = sA + C::STAGES * C::A_BYTES;                   // per stage: weight scales, then A's
    uint64_t* full = reinterpret_cast<uint64_t*>(sSF + C::STAGES * 2 * C::SF_BYTES);
    uint64_t* empty = full + C::STAGES;
    uint64_t* tfull = empty + C::STAGES;
    uint64_t* tempty = tfull + 2;
    uint64_t* sf_full = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sf_full + C::STAGES);
    volatile int* sflag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    float* turn = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(full) + C::BAR_BYTES);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int S = (int)cluster_nctarank(), rank = (int)cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < C::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); mbar_init(&sf_full[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&tfull[b], 1); mbar_init(&tempty[b], 32 * C::EPI_WARPS); }
        *sflag = 0;
        fence_mbar_init();
        prefetch_tmap(&tma_a);
        prefetch_tmap(&tma_w);
    }
    if (warp == 1) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int tiles = p.n_tiles * p.m_tiles;
    const int t0 = (int)blockIdx.x / S, step = (int)gridDim.x / S;
    const int kt0 = p.k_tiles * rank / S, kt1 = p.k_tiles * (rank + 1) / S;   // none empty: S <= k_tiles

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int t = t0; t < tiles && ok; t += step) {
                const int nb = t / p.m_tiles, mb = t - nb * p.m_tiles;
                for (int kt = kt0; kt < kt1; ++kt) {
                    if (!mbar_wait(&empty[stage], phase ^ 1u, sflag, kErrTimeoutProducer)) { ok = false; break; }
                    const uint32_t sf = 512u * (uint32_t)min(2, p.tile_cols - 2 * kt);
                    uint8_t* f = sSF + stage * 2 * C::SF_BYTES;
                    mbar_arrive_expect_tx(&full[stage], C::W_BYTES + C::A_BYTES + 2 * sf);
                    tma_load_2d(sW + stage * C::W_BYTES, &tma_w, &full[stage], kt * 128, nb * 128);
                    bulk_load(f, p.sfw + ((long long)nb * p.tile_cols + 2 * kt) * 512, sf, &full[stage]);
                    tma_load_2d(sA + stage * C::A_BYTES, &tma_a, &full[stage], kt * 128, mb * NT);
                    bulk_load(f + C::SF_BYTES, p.sfa + ((long long)mb * p.tile_cols + 2 * kt) * 512, sf, &full[stage]);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, buf = 0;
            uint32_t phase = 0, aphase = 0;
            bool ok = true;
            constexpr uint32_t idesc = idesc_mxf4(128, NT);
            const uint64_t w_desc = desc_kmajor_sw128(smem_u32(sW)), a_desc = desc_kmajor_sw128(smem_u32(sA));
            for (int t = t0; t < tiles && ok; t += step) {
                if (!mbar_wait(&tempty[buf], aphase ^ 1u, sflag, kErrTimeoutMma)) break;
                tc_fence_after();
                const uint32_t d = tmem + (uint32_t)(buf * NT);
                for (int kt = kt0; kt < kt1; ++kt) {
                    if (!mbar_wait(&full[stage], phase, sflag, kErrTimeoutMma) ||
                        !mbar_wait(&sf_full[stage], phase, sflag, kErrTimeoutMma)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t fw = tmem + (uint32_t)(C::SF_COL0 + stage * C::SF_COLS);
                    issue_k_tile<MmaOf<NT>, false>(d, w_desc + stage * (C::W_BYTES >> 4), a_desc + stage * (C::A_BYTES >> 4),
                                                   idesc, fw, fw + 8, min(4, p.k_steps - 4 * kt), kt != kt0 ? 1u : 0u);
                    tc_commit(&empty[stage]);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
                if (!ok) break;
                tc_commit(&tfull[buf]);
                buf ^= 1;
                if (buf == 0) aphase ^= 1u;
            }
        }
    } else if (warp == 2 + C::EPI_WARPS) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            const uint64_t f_desc = desc_sf_32x16(smem_u32(sSF));
            for (int t = t0; t < tiles && ok; t += step) {
                for (int kt = kt0; kt < kt1; ++kt) {
                    if (!mbar_wait(&full[stage], phase, sflag, kErrTimeoutMma)) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t fd = f_desc + stage * (2 * C::SF_BYTES >> 4);
                    const uint32_t fw = tmem + (uint32_t)(C::SF_COL0 + stage * C::SF_COLS);
                    const int sf = min(2, p.tile_cols - 2 * kt);
                    for (int j = 0; j < sf; ++j) {
                        tmem_cp_32x128b_x4(fw + 4 * j, fd + j * (512 >> 4));
                        tmem_cp_32x128b_x4(fw + 8 + 4 * j, fd + ((C::SF_BYTES + j * 512) >> 4));
                    }
                    tc_commit(&sf_full[stage]);
                    if (++stage == C::STAGES) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else {
        const int quad = warp & 3, col = quad * 32 + lane;        // column of D within the tile
        float* my_turn = turn + (warp - 2) * 16 * C::TURN;
        int buf = 0;
        uint32_t aphase = 0;
        for (int t = t0; t < tiles; t += step) {
            const int nb = t / p.m_tiles, mb = t - nb * p.m_tiles;
            const int m0 = mb * NT, rows = min(NT, p.M - m0);
            if (!mbar_wait(&tfull[buf], aphase, sflag, kErrTimeoutEpilogue)) break;
            tc_fence_after();
            const uint32_t addr = tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * NT);
#pragma unroll 1
            for (int c0 = 16 * ((warp - 2) >> 2); c0 < rows; c0 += 4 * C::EPI_WARPS) {
                uint32_t r[16];
                tmem_ld_32x32b_x16(addr + c0, r);
                tmem_wait_ld();
                if (S == 1) {
                    skinny_store16<OUT>(p, m0 + c0, rows - c0, nb * 128 + quad * 32, r, my_turn);
                } else {                                          // the stages are free: every load and MMA is done
#pragma unroll
                    for (int i = 0; i < 16; ++i) reinterpret_cast<uint32_t*>(smem)[(c0 + i) * C::PART + col] = r[i];
                }
            }
            tc_fence_before();
            mbar_arrive(&tempty[buf]);
            buf ^= 1;
            if (buf == 0) aphase ^= 1u;
        }
    }
    __syncwarp();
    if (S > 1) {                                                  // one tile per cluster
        cluster_sync();
        const int nb = t0 / p.m_tiles, mb = t0 - nb * p.m_tiles;
        const int rows = min(NT, p.M - mb * NT), e = warp - 2;
        const uint32_t base = smem_u32(smem);
        if (e >= 0 && e < C::EPI_WARPS) {
            // Row-major D: a warp takes a row of the tile, four columns per lane.  Column-major: four columns of the tile,
            // a row per lane.  Either way the lanes' pieces lie together in D, and the padded pitch keeps the 16-byte
            // reads of a quarter-warp on distinct banks.
            constexpr bool COL = OUT == NVFP4B_OUT_F32_COLMAJOR;
            const int items = COL ? 32 * ((rows + 31) / 32) : rows;
            for (int i = rank * C::EPI_WARPS + e; i < items; i += C::EPI_WARPS * S) {
                const int c = COL ? (i >> 5) * 32 + lane : i, n = 4 * (COL ? i & 31 : lane);
                if (COL && c >= rows) continue;
                const float4 v = cluster_sum(base + 4u * (uint32_t)(c * C::PART + n), S);
                const int gm = mb * NT + c, gn = nb * 128 + n;
                const float x[4] = {v.x, v.y, v.z, v.w};
                if (!COL && p.wide && gn + 4 <= p.N) {
                    if constexpr (OUT == NVFP4B_OUT_BF16_ROWMAJOR) {
                        const __nv_bfloat162 h0 = __floats2bfloat162_rn(p.alpha * x[0], p.alpha * x[1]);
                        const __nv_bfloat162 h1 = __floats2bfloat162_rn(p.alpha * x[2], p.alpha * x[3]);
                        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.d) + gm * p.ldd + gn) =
                            make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
                    } else {
                        *reinterpret_cast<float4*>(static_cast<float*>(p.d) + gm * p.ldd + gn) =
                            make_float4(p.alpha * x[0], p.alpha * x[1], p.alpha * x[2], p.alpha * x[3]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (gn + k < p.N) skinny_store<OUT>(p, gm, gn + k, x[k]);
                }
            }
        }
        cluster_sync();                                           // no CTA leaves while a peer reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (threadIdx.x == 0 && *sflag != 0) atomicCAS(p.err, 0, *sflag);
}

// The CTAs that K is split over.  A split saves a CTA k_tiles (1 - 1/S) K-tiles of about 0.27 us and costs the meeting of
// the partial sums, which grows with the tile's rows and is twice as dear column-major (N = 2816: 16 rows, K = 2816, S = 6
// 5.2 against 7.3 us unsplit; 128 rows 8.0 and 8.4; K = 704, S = 3 5.0 and 4.6, 7.1 and 5.7), so it is taken from 3 +
// NT / 32 saved K-tiles on, and only as far as all clusters are resident at once (24 clusters of 6 are not: 14.4 us
// against 8.4 with 4).
template <int NT>
int skinny_split(int tiles, int k_tiles, bool col, const std::atomic<int> (&resident)[9]) {
    const int need = (3 + NT / 32) * (col ? 2 : 1);
    for (int S = k_tiles < 8 ? k_tiles : 8; S > 1; --S)
        if (tiles <= resident[S].load(std::memory_order_relaxed) && k_tiles * (S - 1) >= need * S) return S;
    return 1;
}

template <int NT, int OUT>
int mx_run_skinny(const MxGemm& g, cudaStream_t stream) {
    using C = SkinnyCfg<NT>;
    const auto kernel = mx_skinny_kernel<NT, OUT>;
    static std::atomic<bool> ready[64];                // per device: shared-memory limit raised, resident[] filled (host
    static std::atomic<int> resident[64][9];           // threads may race to, with the same values): clusters of S at once
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NVFP4B_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.blockDim = dim3(C::THREADS, 1, 1);
    cfg.dynamicSmemBytes = C::SMEM_BYTES;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!ready[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
        if (e != cudaSuccess) return record_cuda_error(e);
        for (int S = 2; S <= 8; ++S) {
            attr[0].val.clusterDim.x = (unsigned)S;
            cfg.gridDim = dim3((unsigned)(S * 148), 1, 1);
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();                    // this size is not taken
                n = 0;
            }
            resident[dev][S].store(n, std::memory_order_relaxed);
        }
        ready[dev].store(true, std::memory_order_release);
    }
    CUtensorMap ma, mw;
    int st = make_kmajor_map(&ma, g.a, g.M, g.K / 2, NT);
    if (st) return st;
    st = make_kmajor_map(&mw, g.b, g.N, g.K / 2, 128);
    if (st) return st;
    SkinnyParams p;
    p.sfa = g.a_sf;
    p.sfw = g.b_sf;
    p.d = g.d;
    p.ldd = g.ldd;
    p.alpha = g.alpha;
    p.M = g.M;
    p.N = g.N;
    p.n_tiles = (g.N + 127) / 128;
    p.m_tiles = (g.M + NT - 1) / NT;
    p.tile_cols = (g.K + 127) / 128;
    p.k_steps = (g.K + 63) / 64;
    p.k_tiles = (g.K + 255) / 256;
    p.wide = g.ldd % (OUT == NVFP4B_OUT_BF16_ROWMAJOR ? 8 : 4) == 0;     // d is 16-byte aligned
    p.err = device_error_ptr();
    if (!p.err) return NVFP4B_ERR_CUDA;
    const long long tiles = (long long)p.n_tiles * p.m_tiles;
    if (tiles > (1ll << 30)) return NVFP4B_ERR_SHAPE;
    const int sms = sm_count();
    const int S = tiles >= sms ? 1 : skinny_split<NT>((int)tiles, p.k_tiles, OUT == NVFP4B_OUT_F32_COLMAJOR, resident[dev]);
    attr[0].val.clusterDim.x = (unsigned)S;
    cfg.gridDim = dim3((unsigned)(S > 1 ? tiles * S : tiles < sms ? tiles : sms), 1, 1);
    cfg.stream = stream;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, ma, mw, p);
    return err == cudaSuccess ? NVFP4B_OK : record_cuda_error(err);
}

template <typename T>
int mx_run_pair(const MxGemm& g, cudaStream_t stream) {            // g.d as row-major [N, M]

    using C = MxPair;
    CUtensorMap ma, mb, msa, msb;
    int st = make_kmajor_map(&ma, g.a, g.M, g.K / 2, C::BM);
    if (st) return st;
    st = make_kmajor_map(&mb, g.b, g.N, g.K / 2, C::BN / 2);
    if (st) return st;
    st = make_scale_map(&msa, g.a_sf, (long long)nvfp4b_mx_scale_buffer_bytes(g.M, g.K), 2 * C::SF_TILES);
    if (st) return st;
    st = make_scale_map(&msb, g.b_sf, (long long)nvfp4b_mx_scale_buffer_bytes(g.N, g.K), 2 * C::SF_TILES);
    if (st) return st;
    CoreParams cp;
    st = mx_core_params(g, cp);
    if (st) return st;
    PairDenseSched s;
    s.m_tiles = (g.M + C::PAIR_M - 1) / C::PAIR_M;
    s.n_tiles = (g.N + C::BN - 1) / C::BN;
    s.group_m = 8;
    s.k_tiles = cp.k_tiles;
    const long long tiles = (long long)s.m_tiles * s.n_tiles;
    if (tiles > (1ll << 30)) return NVFP4B_ERR_SHAPE;
    return launch_pair<C>(ma, mb, msa, msb, cp, s, MxEpi<T>{static_cast<T*>(g.d), g.ldd, g.M, g.N, g.alpha}, (int)tiles,
                          stream);
}

// D^T = B A^T, stored where D is: column-major D is row-major D^T.
MxGemm swapped(const MxGemm& g) { return {g.b, g.b_sf, g.a, g.a_sf, g.alpha, g.N, g.M, g.K, g.d, g.ldd}; }

// Narrow tiles (128 x 128 above 64 rows) or CTA pairs (256 x 256)?  A round of narrow tiles takes about 0.42 us for each
// K-tile and 0.4 us, 1.3 at least (the stores of one tile under the products of the next); a round of pairs 0.42 us for
// each K-tile and 1.9 (one accumulator, so the stores are not hidden).  Narrow wins with few K-tiles, with one round, and
// where the pairs' last round is nearly empty (1024 x 4736, K = 704 7.8 against 10.2 us; 4096 x 7000, K = 512 22.3 and
// 26.2; K = 1408 38.0 and 34.8; 512 x 8448, K = 2816 14.2 and 11.5).
bool narrow_tiles(int M, int N, int K) {
    const long long sms = sm_count(), pairs = sms / 2, kt = (K + 255) / 256;
    const long long rn = ((M + 127) / 128 * ((N + 127ll) / 128) + sms - 1) / sms;
    const long long rp = ((M + 255) / 256 * ((N + 255ll) / 256) + pairs - 1) / pairs;
    return M <= 128 || rn * (kt > 2 ? 2 + 2 * kt : 6) <= rp * (9 + 2 * kt);
}

template <int OUT>
int mx_run(const MxGemm& g, cudaStream_t stream) {
    constexpr bool COL = OUT == NVFP4B_OUT_F32_COLMAJOR;
    if (g.M <= 16) return mx_run_skinny<16, OUT>(g, stream);
    if (g.M <= 32) return mx_run_skinny<32, OUT>(g, stream);
    if (g.M <= 64) return mx_run_skinny<64, OUT>(g, stream);
    if constexpr (COL) {                               // from 65 rows on either operand may be the wide one
        return mx_run<NVFP4B_OUT_F32_ROWMAJOR>(swapped(g), stream);
    } else {
        if (narrow_tiles(g.M, g.N, g.K)) return mx_run_skinny<128, OUT>(g, stream);
        return mx_run_pair<std::conditional_t<OUT == NVFP4B_OUT_BF16_ROWMAJOR, __nv_bfloat16, float>>(swapped(g), stream);
    }
}

}  // namespace
}  // namespace nvfp4b

using namespace nvfp4b;

extern "C" int nvfp4b_mx_gemm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales,
                              float alpha, int M, int N, int K, void* d, int out_kind, long long ldd, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || (K & 31)) return NVFP4B_ERR_SHAPE;
    if (M > 0x7fffff00 || N > 0x7fffff00 || K > 0x7fffff00) return NVFP4B_ERR_SHAPE;   // tile counts round up in 32 bits
    if (!a || !a_scales || !b || !b_scales || !d) return NVFP4B_ERR_NULL;
    if (out_kind < 0 || out_kind > 2) return NVFP4B_ERR_ARG;
    if (out_kind == NVFP4B_OUT_F32_COLMAJOR ? ldd < M : ldd < N) return NVFP4B_ERR_SHAPE;
    if (!aligned16(a) || !aligned16(b) || !aligned16(a_scales) || !aligned16(b_scales) || !aligned16(d))
        return NVFP4B_ERR_ALIGN;
    const MxGemm g = {a, a_scales, b, b_scales, alpha, M, N, K, d, ldd};
    const cudaStream_t s = (cudaStream_t)stream;
    switch (out_kind) {
        case NVFP4B_OUT_BF16_ROWMAJOR: return mx_run<NVFP4B_OUT_BF16_ROWMAJOR>(g, s);
        case NVFP4B_OUT_F32_COLMAJOR: return mx_run<NVFP4B_OUT_F32_COLMAJOR>(g, s);
        default: return mx_run<NVFP4B_OUT_F32_ROWMAJOR>(g, s);
    }
}
