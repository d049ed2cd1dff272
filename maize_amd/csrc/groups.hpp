// Which kernel of the groups' code object computes a grouped or block-scaled product, and its grid.  Host logic only; no HIP calls.
#pragma once
#include <stddef.h>
#include <stdint.h>

#include "maize_hip.h"

namespace maize {

uint32_t group_kernel_count();
const char* group_kernel_name(uint32_t index);

struct GroupPlan {
    uint32_t kernel;           // index; its name tells the operands' type, how they lie, and the tile
    uint32_t grid, block;
    uint32_t ksplit;           // K ranges per tile
    size_t workspace_bytes;
};
// false: the product needs more workgroups than a launch can have.  `split` false: no K ranges, and so no workspace.
bool plan_group(const maize_gemm_grouped_desc_t& d, uint32_t compute_units, GroupPlan* out, bool split = true);

// Kernel parameter blocks (kernels/gemm_group.hpp, kernels/quantize.hpp).
struct GroupArgs {
    maize_gemm_args_t g;
    const int32_t* offsets;
    uint32_t groups, rows;
    const float* scale_a;
    const float* scale_b;
    uint32_t ld_scale_a, ld_scale_b;
    uint64_t stride_scale_b;
};
static_assert(sizeof(GroupArgs) == 168, "kernel parameter block");
struct QuantArgs {
    const void* x;
    void* q;
    float* scale;
    uint32_t rows, cols, ldx, ldq, ld_scale, batch;
    uint64_t stride_x, stride_q, stride_scale;
};
static_assert(sizeof(QuantArgs) == 72, "kernel parameter block");
constexpr uint32_t kQuantKernels = 6;      // in_type (bf16, half, fp32) x (rows, blocks)
const char* quant_kernel_name(uint32_t index);

}  // namespace maize
