// A layer with 4-bit microscaled weights on the host side: what its handle holds and what a forward is asked for.
#pragma once

#include "common.cuh"
#include "fp4_params.cuh"

namespace shrewq {

struct Fp4Weight {
    const uint8_t *codes = nullptr;   // the caller's, [N][Kp / 2]
    uint8_t *pieces = nullptr;        // owned: the scales in the order of the block-scaled matrix instructions
    Fp4Params *params = nullptr;      // owned, on the device
    bool nv = false;
    bool round_x = false;             // activations are quantized too
    float x_scale = 1.0f;             // NV: tensor scale of the activations
};

struct Fp4Forward {
    const Fp4Weight *w, *up;          // up null: a plain layer
    const float *bias, *bias_up;
    const float *alpha, *alpha_up;    // what the sums of a channel are multiplied by: the tensor scales (tcgen05 kernels)
    const void *w_tmap, *up_tmap;     // boxes of codes
    const void *x;
    int x_dtype;
    void *y;
    int y_dtype;
    size_t M, N, K, ldy;
    int epilogue;
    bool pdl;                         // weights are older than the previous kernel of the stream
};

// A launch whose grid is cut into clusters of S CTAs along x (S = 1: none), with or without programmatic stream serialization.
template <typename Kern, typename... Args>
inline cudaError_t launch_cluster(Kern kern, unsigned grid, unsigned block, size_t smem, cudaStream_t stream, bool pdl, int S, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (S > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)S;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kern, args...);
}

// How many CTAs (1, 2, 4 or 8) share the k range of a tile: as many as `room` holds of all tiles at once, each with at least
// min_rounds stages and none without one.
inline int split_over_cluster(size_t tiles, int rounds, int room, int min_rounds, int *rounds_per_cta) {
    int S = 1;
    while (S < 8 && tiles * (size_t)(2 * S) <= (size_t)room && rounds >= 2 * S * min_rounds) S *= 2;
    while (S > 1 && (S - 1) * ((rounds + S - 1) / S) >= rounds) S /= 2;
    *rounds_per_cta = (rounds + S - 1) / S;
    return S;
}

// pieces of 128 rows by 4 blocks along a row, out to whole 256 columns
inline size_t fp4_pieces(size_t K, bool nv) { return (K + 255) / 256 * (nv ? 4 : 2); }

int launch_quantize_fp4(shrewq_ctx *ctx, const void *x, int x_dtype, size_t rows, size_t cols, size_t ld, bool nv, float *g, int find_g,
                        void *codes, void *scales);
int launch_dequantize_fp4(shrewq_ctx *ctx, const void *codes, const void *scales, const float *g, size_t rows, size_t cols, bool nv, int out_dtype, void *out);
int launch_fp4_scale_pieces(shrewq_ctx *ctx, const uint8_t *scales, const float *g, size_t N, size_t blocks, size_t pieces, bool nv, uint8_t *out,
                            Fp4Params *params, float x_scale, float *alpha);
int encode_fp4_tmap(shrewq_ctx *ctx, const uint8_t *codes, size_t n, size_t k, int box_rows, int box_bytes, void *tmap_out);
int launch_gemm_w4_bf16(shrewq_ctx *ctx, const Fp4Forward &a);
int launch_gemm_fp4(shrewq_ctx *ctx, const Fp4Forward &a);
bool gemv_fp4_supported(const Fp4Forward &a);
int launch_gemm_w4_f16(shrewq_ctx *ctx, const Fp4Forward &a);
int launch_gemv_fp4(shrewq_ctx *ctx, const Fp4Forward &a);
int launch_residual_norm(shrewq_ctx *ctx, const shrewq_residual_norm_args *p);

}  // namespace shrewq
