// mx_gemm.cu -- dense MXFP4 GEMM, D = alpha * A[M, K] @ B[N, K]^T, on the tcgen05 core (gemm_core.cuh, Kind::MXF4).
//
// One e8m0 scale per 32 elements: a 512-byte scale tile (128 rows x 4 blocks) serves two 64-element MMAs, so a K-tile
// needs half of the scale copies (tcgen05.cp) that NVFP4's scale per 16 does.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "dense_epi.cuh"
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

using MxTile = KCfg<256, 4, 1, 8, Kind::MXF4>;
using MxPair = PairCfg<5, 8, 8 * kStoreTileBytes, Kind::MXF4>;   // + bf16 store staging tiles

template <class Epi>
Epi mx_epilogue(const MxGemm& g) {
    Epi e;
    e.d = g.d;
    e.ldd = g.ldd;
    e.M = g.M;
    e.N = g.N;
    e.alpha = e.b_dequant = g.alpha;
    e.d_a_amax = nullptr;
    return e;
}

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

template <int OUT>
int mx_run_tile(const MxGemm& g, cudaStream_t stream) {
    using C = MxTile;
    CUtensorMap ma, mb;
    int st = make_kmajor_map(&ma, g.a, g.M, g.K / 2, C::BM);
    if (st) return st;
    st = make_kmajor_map(&mb, g.b, g.N, g.K / 2, C::BN);
    if (st) return st;
    CoreParams cp;
    st = mx_core_params(g, cp);
    if (st) return st;
    DenseSched<C::BN> s;
    s.m_tiles = (g.M + C::BM - 1) / C::BM;
    s.n_tiles = (g.N + C::BN - 1) / C::BN;
    s.group_m = 16;
    s.N = g.N;
    s.b_row_tiles = (g.N + 127) / 128;
    s.k_tiles = cp.k_tiles;
    const int tiles = s.m_tiles * s.n_tiles;
    const int grid = tiles < sm_count() ? tiles : sm_count();
    return launch_core<C>(ma, mb, cp, s, mx_epilogue<DenseEpi<OUT>>(g), grid, stream);
}

template <int OUT>
int mx_run_pair(const MxGemm& g, cudaStream_t stream) {
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
    return launch_pair<C>(ma, mb, msa, msb, cp, s, mx_epilogue<DenseEpi<OUT, true>>(g), s.m_tiles * s.n_tiles, stream);
}

template <int OUT>
int mx_run(const MxGemm& g, cudaStream_t stream) {
    return g.M > 128 ? mx_run_pair<OUT>(g, stream) : mx_run_tile<OUT>(g, stream);
}

}  // namespace
}  // namespace nvfp4b

using namespace nvfp4b;

extern "C" int nvfp4b_mx_gemm(const uint8_t* a, const uint8_t* a_scales, const uint8_t* b, const uint8_t* b_scales,
                              float alpha, int M, int N, int K, void* d, int out_kind, long long ldd, void* stream) {
    if (M <= 0 || N <= 0 || K <= 0 || (K & 31)) return NVFP4B_ERR_SHAPE;
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
