// The entry points of the grouped and block-scaled products and of the quantiser: their checks, and their kernels' code object.
// Which kernel runs is groups.cpp's; the launcher (shim.cpp) knows neither.
#include <cstdio>
#include <cstring>

#include "groups.hpp"
#include "launcher.hpp"

extern "C" const unsigned char maize_embedded_groups[];

using maize::report;

namespace {

// The products' kernels, then the quantiser's.
const char* kernel_name(uint32_t index) {
    return index < maize::group_kernel_count() ? maize::group_kernel_name(index) : maize::quant_kernel_name(index - maize::group_kernel_count());
}
const maize::MoreKernels kernels = {maize_embedded_groups, "hipModuleLoadData(embedded code object of the grouped products)",
                                    maize::group_kernel_count() + maize::kQuantKernels, kernel_name};
[[maybe_unused]] const int added = maize::add_kernels(&kernels);

}  // namespace

extern "C" {

/* ---- products grouped by expert, and block-scaled 8-bit products -------------- */

int32_t maize_hip_gemm_grouped_validate(const maize_gemm_grouped_desc_t* d) {
    if (!d) return report(MAIZE_ERR_NULL, "gemm_grouped: descriptor is NULL");
    if (d->axis > MAIZE_GROUP_DEPTH) return report(MAIZE_ERR_ARG, "gemm_grouped: unknown axis %u", d->axis);
    const bool depth = d->axis == MAIZE_GROUP_DEPTH, bits8 = d->in_type == MAIZE_IN_E4M3, nt = d->layout == MAIZE_LAYOUT_NT;
    if ((d->layout != MAIZE_LAYOUT_NN && !nt) || (depth && nt))
        return report(MAIZE_ERR_LAYOUT, "gemm_grouped: layout %u (depth: MAIZE_LAYOUT_NN only)", d->layout);
    if (d->groups == 0 || d->groups >= (1u << 20)) return report(MAIZE_ERR_SHAPE, "gemm_grouped: %u groups (1 .. 2^20 - 1)", d->groups);
    const uint32_t rows = d->a.nrows;
    if (depth ? d->b.nrows != rows : d->c.nrows != rows)
        return report(MAIZE_ERR_SHAPE, "gemm_grouped: A has %u rows, %s has %u", rows, depth ? "B" : "C", depth ? d->b.nrows : d->c.nrows);
    const uint32_t kb = nt ? d->b.ncols : d->b.nrows, n = nt ? d->b.nrows : d->b.ncols;
    if (!depth && kb != d->a.ncols) return report(MAIZE_ERR_SHAPE, "gemm_grouped: inner dimensions differ (A has K=%u, B has K=%u)", d->a.ncols, kb);
    if (d->c.ncols != n || (depth && d->c.nrows != d->a.ncols))
        return report(MAIZE_ERR_SHAPE, "gemm_grouped: C is %ux%u, expected %ux%u", d->c.nrows, d->c.ncols, depth ? d->a.ncols : rows, n);
    if (d->a.ncols == 0 || n == 0) return report(MAIZE_ERR_SHAPE, "gemm_grouped: empty operand (%u columns of A, N=%u)", d->a.ncols, n);
    if (rows >= (1u << 31)) return report(MAIZE_ERR_SHAPE, "gemm_grouped: %u rows (offsets are int32)", rows);
    if (!d->offsets && d->groups != 1u) return report(MAIZE_ERR_NULL, "gemm_grouped: %u groups without offsets", d->groups);
    if (d->in_type != MAIZE_IN_BF16 && d->in_type != MAIZE_IN_F16 && !bits8)
        return report(MAIZE_ERR_ARG, "gemm_grouped: operand type %u (bf16, half, or E4M3 with block scales)", d->in_type);
    if (bits8 && depth) return report(MAIZE_ERR_ARG, "gemm_grouped: 8-bit operands are grouped by rows only");
    if (d->out_type != MAIZE_OUT_SAME && d->out_type != MAIZE_OUT_F32 && !(d->out_type == MAIZE_OUT_F16 && d->in_type != MAIZE_IN_BF16))
        return report(MAIZE_ERR_ARG, "gemm_grouped: output type %u for operand type %u", d->out_type, d->in_type);
    if (bits8 ? (!d->scale_a || !d->scale_b) : (d->scale_a || d->scale_b))
        return report(bits8 ? MAIZE_ERR_NULL : MAIZE_ERR_ARG, bits8 ? "gemm_grouped: E4M3 operands without scales" : "gemm_grouped: scales go with E4M3 operands");
    if (!d->b.ptr && !(depth && rows == 0)) return report(MAIZE_ERR_NULL, "gemm_grouped: NULL matrix pointer (B)");
    if ((!d->a.ptr && rows) || (!d->c.ptr && (rows || depth))) return report(MAIZE_ERR_NULL, "gemm_grouped: NULL matrix pointer");
    const uint32_t in_bytes = bits8 ? 1u : 2u, out_bytes = d->out_type == MAIZE_OUT_F32 ? 4u : 2u;
    if ((((uintptr_t)d->a.ptr | (uintptr_t)d->b.ptr) & (in_bytes - 1u)) || ((uintptr_t)d->c.ptr & (out_bytes - 1u)) ||
        (((uintptr_t)d->offsets | (uintptr_t)d->scale_a | (uintptr_t)d->scale_b) & 3u))
        return report(MAIZE_ERR_ALIGN, "gemm_grouped: pointers must be aligned to their element size");
    if ((d->lda && d->lda < d->a.ncols) || (d->ldb && d->ldb < d->b.ncols) || (d->ldc && d->ldc < d->c.ncols))
        return report(MAIZE_ERR_SHAPE, "gemm_grouped: a leading dimension is smaller than the row it strides (lda=%u ldb=%u ldc=%u)", d->lda, d->ldb, d->ldc);
    const uint32_t lda = d->lda ? d->lda : d->a.ncols, ldb = d->ldb ? d->ldb : d->b.ncols, ldc = d->ldc ? d->ldc : d->c.ncols, most = 1u << 21;
    if (lda >= most || ldb >= most || ldc >= most || (!depth && (d->b.nrows >= most)))
        return report(MAIZE_ERR_SHAPE, "gemm_grouped: a dimension reaches 2^21 (lda=%u ldb=%u ldc=%u, B %ux%u)", lda, ldb, ldc, d->b.nrows, d->b.ncols);
    if (d->groups > 1u) {
        const uint64_t one = depth ? (uint64_t)(d->c.nrows - 1u) * ldc + d->c.ncols : (uint64_t)(d->b.nrows - 1u) * ldb + d->b.ncols;
        if (d->stride < one && (depth || d->stride)) return report(MAIZE_ERR_SHAPE, "gemm_grouped: stride %llu is smaller than one matrix", (unsigned long long)d->stride);
    }
    if (bits8) {
        const uint32_t across = (d->b.ncols + 127u) / 128u;
        if ((d->ld_scale_a && d->ld_scale_a < rows) || (d->ld_scale_b && d->ld_scale_b < across))
            return report(MAIZE_ERR_SHAPE, "gemm_grouped: a leading dimension of the scales is smaller than their row (%u, %u)", d->ld_scale_a, d->ld_scale_b);
    }
    if (!(d->alpha == d->alpha) || !(d->beta == d->beta)) return report(MAIZE_ERR_ARG, "gemm_grouped: alpha or beta is NaN");
    return MAIZE_OK;
}

static int32_t group_planned(const maize_gemm_grouped_desc_t* d, uint32_t cus, maize::GroupPlan* plan, bool split = true) {
    if (maize::plan_group(*d, cus, plan, split)) return MAIZE_OK;
    return report(MAIZE_ERR_SHAPE, "gemm_grouped: more tiles than a launch has workgroups (%u rows, %u groups, N=%u)", d->a.nrows, d->groups, d->c.ncols);
}

int32_t maize_hip_gemm_grouped_plan(const maize_gemm_grouped_desc_t* d, uint32_t compute_units, maize_gemm_plan_t* out) {
    if (!out) return report(MAIZE_ERR_NULL, "gemm_grouped_plan: NULL argument");
    int32_t rc = maize_hip_gemm_grouped_validate(d);
    if (rc != MAIZE_OK) return rc;
    if (compute_units == 0) return report(MAIZE_ERR_ARG, "gemm_grouped_plan: compute_units must be positive");
    memset(out, 0, sizeof(*out));
    if (d->a.nrows == 0 && d->axis == MAIZE_GROUP_ROWS) return MAIZE_OK;       // nothing is launched
    maize::GroupPlan p;
    if ((rc = group_planned(d, compute_units, &p)) != MAIZE_OK) return rc;
    snprintf(out->kernel, sizeof(out->kernel), "%s", maize::group_kernel_name(p.kernel));
    out->grid[0] = p.grid;
    out->block[0] = p.block;
    out->grid[1] = out->grid[2] = out->block[1] = out->block[2] = 1;
    out->ksplit = p.ksplit;
    out->workspace_bytes = p.workspace_bytes;
    return MAIZE_OK;
}

int32_t maize_hip_gemm_grouped(maize_ctx_t* ctx, const maize_gemm_grouped_desc_t* d, void* stream) {
    if (!ctx) return report(MAIZE_ERR_NULL, "gemm_grouped: ctx is NULL");
    int32_t rc = maize_hip_gemm_grouped_validate(d);
    if (rc != MAIZE_OK) return rc;
    const bool depth = d->axis == MAIZE_GROUP_DEPTH;
    if (d->a.nrows == 0 && !depth) return MAIZE_OK;
    maize::GroupPlan p;
    if ((rc = group_planned(d, maize::compute_units(ctx), &p)) != MAIZE_OK) return rc;
    maize::GroupArgs args;
    memset(&args, 0, sizeof args);
    args.g.a = d->a.ptr; args.g.arows = d->a.nrows; args.g.acols = d->a.ncols;
    args.g.b = d->b.ptr; args.g.brows = d->b.nrows; args.g.bcols = d->b.ncols;
    args.g.c = d->c.ptr; args.g.crows = d->c.nrows; args.g.ccols = d->c.ncols;
    if (d->groups > 1u) (depth ? args.g.stride_c : args.g.stride_b) = d->stride;
    args.g.batch = 1;
    args.g.layout = d->layout;
    args.g.lda = d->lda; args.g.ldb = d->ldb; args.g.ldc = d->ldc;
    args.g.alpha = d->alpha; args.g.beta = d->beta;
    args.g.epi = (d->out_type == MAIZE_OUT_F32 ? 1u : 0u) | ((d->alpha != 1.0f || d->beta != 0.0f) ? 2u : 0u) |
                 (d->in_type == MAIZE_IN_F16 ? 4u : 0u) | (d->in_type == MAIZE_IN_E4M3 ? 8u : 0u) | (d->out_type == MAIZE_OUT_F16 ? 64u : 0u);
    args.offsets = d->offsets;
    args.groups = d->groups;
    args.rows = d->a.nrows;
    args.scale_a = d->scale_a;
    args.scale_b = d->scale_b;
    args.ld_scale_a = d->ld_scale_a ? d->ld_scale_a : d->a.nrows;
    args.ld_scale_b = d->ld_scale_b ? d->ld_scale_b : (d->b.ncols + 127u) / 128u;
    args.stride_scale_b = d->groups > 1u ? d->stride_scale_b : 0u;
    // No memory for the K ranges' parts: the same product without K ranges, which needs none.
    if (p.workspace_bytes && !maize::stream_workspace(ctx, stream, p.workspace_bytes, &args.g.workspace) &&
        (rc = group_planned(d, maize::compute_units(ctx), &p, false)) != MAIZE_OK)
        return rc;
    args.g.ksplit = p.ksplit;
    return maize::launch_more(ctx, p.kernel, p.grid, p.block, stream, &args, sizeof args);
}

int32_t maize_hip_quantize_blocks_validate(const maize_quantize_desc_t* d) {
    if (!d) return report(MAIZE_ERR_NULL, "quantize_blocks: descriptor is NULL");
    if (d->block_rows != 1u && d->block_rows != 128u) return report(MAIZE_ERR_ARG, "quantize_blocks: blocks of %u rows (1 or 128)", d->block_rows);
    if (d->in_type != MAIZE_IN_BF16 && d->in_type != MAIZE_IN_F16 && d->in_type != MAIZE_IN_F32)
        return report(MAIZE_ERR_ARG, "quantize_blocks: input type %u (bf16, half or fp32)", d->in_type);
    if (d->batch == 0) return report(MAIZE_ERR_SHAPE, "quantize_blocks: batch is 0");
    if (d->x.nrows != d->q.nrows || d->x.ncols != d->q.ncols)
        return report(MAIZE_ERR_SHAPE, "quantize_blocks: x is %ux%u, q is %ux%u", d->x.nrows, d->x.ncols, d->q.nrows, d->q.ncols);
    if (d->x.ncols == 0) return report(MAIZE_ERR_SHAPE, "quantize_blocks: no columns");
    if (d->x.nrows && (!d->x.ptr || !d->q.ptr || !d->scale)) return report(MAIZE_ERR_NULL, "quantize_blocks: NULL pointer");
    const uint32_t bytes = d->in_type == MAIZE_IN_F32 ? 4u : 2u;
    if (((uintptr_t)d->x.ptr & (bytes - 1u)) || ((uintptr_t)d->scale & 3u)) return report(MAIZE_ERR_ALIGN, "quantize_blocks: pointers must be aligned to their element size");
    const uint32_t across = (uint32_t)(((uint64_t)d->x.ncols + 127u) / 128u), down = (uint32_t)(((uint64_t)d->x.nrows + 127u) / 128u);
    const uint32_t scale_cols = d->block_rows == 1u ? d->x.nrows : across, scale_rows = d->block_rows == 1u ? across : down;
    if ((d->ldx && d->ldx < d->x.ncols) || (d->ldq && d->ldq < d->x.ncols) || (d->ld_scale && d->ld_scale < scale_cols))
        return report(MAIZE_ERR_SHAPE, "quantize_blocks: a leading dimension is smaller than the row it strides (ldx=%u ldq=%u ld_scale=%u)", d->ldx, d->ldq, d->ld_scale);
    if (d->batch > 1u && d->x.nrows) {
        const uint64_t ldq = d->ldq ? d->ldq : d->x.ncols, lds = d->ld_scale ? d->ld_scale : scale_cols;
        if (d->stride_q < (uint64_t)(d->x.nrows - 1u) * ldq + d->x.ncols || d->stride_scale < (uint64_t)(scale_rows - 1u) * lds + scale_cols)
            return report(MAIZE_ERR_SHAPE, "quantize_blocks: batch stride smaller than one matrix");
    }
    const uint64_t grid = (uint64_t)d->batch * across * (((uint64_t)d->x.nrows + (d->block_rows == 1u ? 15u : 127u)) / (d->block_rows == 1u ? 16u : 128u));
    if (grid >= (1u << 24)) return report(MAIZE_ERR_SHAPE, "quantize_blocks: more blocks than a launch has workgroups (%ux%u, batch %u)", d->x.nrows, d->x.ncols, d->batch);
    return MAIZE_OK;
}

int32_t maize_hip_quantize_blocks(maize_ctx_t* ctx, const maize_quantize_desc_t* d, void* stream) {
    if (!ctx) return report(MAIZE_ERR_NULL, "quantize_blocks: ctx is NULL");
    int32_t rc = maize_hip_quantize_blocks_validate(d);
    if (rc != MAIZE_OK || d->x.nrows == 0) return rc;
    const uint32_t across = (d->x.ncols + 127u) / 128u, by = d->block_rows == 1u ? 16u : 128u;
    maize::QuantArgs args;
    memset(&args, 0, sizeof args);
    args.x = d->x.ptr;
    args.q = d->q.ptr;
    args.scale = d->scale;
    args.rows = d->x.nrows;
    args.cols = d->x.ncols;
    args.ldx = d->ldx ? d->ldx : d->x.ncols;
    args.ldq = d->ldq ? d->ldq : d->x.ncols;
    args.ld_scale = d->ld_scale ? d->ld_scale : d->block_rows == 1u ? d->x.nrows : across;
    args.batch = d->batch;
    args.stride_x = d->stride_x;
    args.stride_q = d->stride_q;
    args.stride_scale = d->stride_scale;
    const uint32_t type = d->in_type == MAIZE_IN_BF16 ? 0u : d->in_type == MAIZE_IN_F16 ? 1u : 2u;
    const uint32_t kernel = maize::group_kernel_count() + 2u * type + (d->block_rows == 1u ? 0u : 1u);
    return maize::launch_more(ctx, kernel, d->batch * across * ((d->x.nrows + by - 1u) / by), 256, stream, &args, sizeof args);
}

}  // extern "C"
