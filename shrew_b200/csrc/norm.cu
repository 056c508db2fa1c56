// Launcher of the norms around a block (device code and its description: norm_kernels.cuh).
#include <cuda_fp16.h>

#include "linear_fp4.cuh"
#include "norm_kernels.cuh"

namespace shrewq {
namespace {

// A warp a row up to 1024 columns, else a CTA with two groups of 8 columns a thread (four above 16384).
template <typename TX, typename TB, typename TY>
cudaError_t launch_typed(shrewq_ctx *ctx, const NormArgs &a) {
    const bool pdl = ctx->tuning.pdl != 0;
    const size_t groups = ((size_t)a.D + 7) / 8;
    const unsigned most = 0x7FFFFFFFu;
    if (groups <= 128) {
        const size_t ctas = (a.M + 7) / 8;
        const dim3 grid((unsigned)(ctas < most ? ctas : most)), block(a.M >= 8 ? 256 : (unsigned)a.M * 32);
        if (groups <= 32) return launch_maybe_pdl(residual_norm_kernel<TX, TB, TY, 1, true>, grid, block, 0, ctx->stream, pdl, a);
        if (groups <= 64) return launch_maybe_pdl(residual_norm_kernel<TX, TB, TY, 2, true>, grid, block, 0, ctx->stream, pdl, a);
        return launch_maybe_pdl(residual_norm_kernel<TX, TB, TY, 4, true>, grid, block, 0, ctx->stream, pdl, a);
    }
    const int V = groups <= 2048 ? 2 : 4;
    const dim3 block((unsigned)(((groups + V - 1) / V + 31) / 32 * 32));
    // as many CTAs as are resident (64 registers a thread: 1024 threads an SM), row after row: 4096 rows of 4096 44.3 -> 43.8 us against a CTA a row
    const size_t resident = (size_t)ctx->sm_count * (1024 / block.x);
    const dim3 grid((unsigned)(a.M < resident ? a.M : resident));
    if (V == 2) return launch_maybe_pdl(residual_norm_kernel<TX, TB, TY, 2, false>, grid, block, 0, ctx->stream, pdl, a);
    return launch_maybe_pdl(residual_norm_kernel<TX, TB, TY, 4, false>, grid, block, 0, ctx->stream, pdl, a);
}

template <typename TX, typename TB>
cudaError_t launch_out(shrewq_ctx *ctx, const NormArgs &a, int y_dtype) {
    return y_dtype == SHREWQ_F32 ? launch_typed<TX, TB, float>(ctx, a) : launch_typed<TX, TB, __nv_bfloat16>(ctx, a);
}
template <typename TX>
cudaError_t launch_branch(shrewq_ctx *ctx, const NormArgs &a, int b_dtype, int y_dtype) {
    return b_dtype == SHREWQ_F32 ? launch_out<TX, float>(ctx, a, y_dtype) : launch_out<TX, __nv_bfloat16>(ctx, a, y_dtype);
}

}  // namespace

int launch_residual_norm(shrewq_ctx *ctx, const shrewq_residual_norm_args *p) {
    NormArgs a;
    a.x = p->x_dev; a.branch = p->branch_dev; a.gate = p->gate_dev;
    a.ldx = p->ldx; a.ldb = p->ldb; a.ldg = p->ldg;
    a.post_w = p->post_weight_dev; a.post_b = p->post_bias_dev; a.pre_w = p->pre_weight_dev; a.pre_b = p->pre_bias_dev;
    a.r = p->residual_dev; a.h = p->normed_dev;
    a.M = p->M; a.D = (int)p->D;
    a.post = p->branch_dev ? p->post_norm : SHREWQ_NORM_NONE;
    a.pre = p->pre_norm;
    a.gate_kind = p->branch_dev ? p->gate_kind : SHREWQ_GATE_NONE;
    a.post_eps = p->post_eps; a.pre_eps = p->pre_eps;
    a.residual_scale = p->residual_scale; a.branch_scale = p->branch_scale;
    // whole groups of 8: 32 bytes of f32, 16 of bf16
    const auto off = [&](const void *ptr, size_t ld, int dtype) {
        const size_t e = dtype == SHREWQ_F32 ? 4 : 2;
        return ptr && ((reinterpret_cast<uintptr_t>(ptr) | (ld * e)) % (8 * e));
    };
    const auto odd16 = [](const void *ptr) { return ptr && (reinterpret_cast<uintptr_t>(ptr) & 15); };
    a.vec = !(p->D % 8 || off(a.x, a.ldx, p->x_dtype) || off(a.branch, a.ldb, p->branch_dtype) ||
              (a.gate_kind == SHREWQ_GATE_FULL && off(a.gate, a.ldg, p->branch_dtype)) ||
              (a.gate_kind == SHREWQ_GATE_CHANNEL && off(a.gate, 0, p->branch_dtype)) || off(a.r, a.D, p->x_dtype) || off(a.h, a.D, p->normed_dtype) ||
              odd16(a.post_w) || odd16(a.post_b) || odd16(a.pre_w) || odd16(a.pre_b));
    const cudaError_t e = p->x_dtype == SHREWQ_F32 ? launch_branch<float>(ctx, a, p->branch_dtype, p->normed_dtype)
                                                   : launch_branch<__nv_bfloat16>(ctx, a, p->branch_dtype, p->normed_dtype);
    SHREWQ_CUDA_TRY(ctx, e);
    ctx->launches += 1;
    SHREWQ_CUDA_TRY(ctx, cudaGetLastError());
    return SHREWQ_OK;
}

}  // namespace shrewq
