#include "groups.hpp"

#include "launcher.hpp"

#include <algorithm>
#include <cmath>

#include "dispatch.hpp"

namespace maize {
namespace {

// [type][layout][tile]; layouts: N x K, K x N, depth.  8-bit operands have no depth.
enum { kLarge, kMiddle, kFew, kTiles };
struct Shape { uint32_t bm, bn, threads; };
// 16-bit operands; 8-bit ones, N x K; K x N (rows of 64 8-bit columns would be half lines)
constexpr Shape kShape[3][kTiles] = {{{256, 256, 256}, {128, 128, 256}, {32, 64, 256}},
                                     {{256, 256, 512}, {128, 128, 256}, {32, 64, 256}},
                                     {{256, 256, 512}, {128, 128, 256}, {32, 128, 256}}};
const Shape* shapes(const maize_gemm_grouped_desc_t& d) { return kShape[d.in_type != MAIZE_IN_E4M3 ? 0 : d.layout == MAIZE_LAYOUT_NT ? 1 : 2]; }
#define MAIZE_ROW(tag, lay, few) "maize_group_" tag "_" lay "_256x256", "maize_group_" tag "_" lay "_128x128", "maize_group_" tag "_" lay "_32x" few
#define MAIZE_DEPTH(tag) "maize_group_" tag "_tn_256x256", "maize_group_" tag "_tn_128x128", nullptr
constexpr const char* kNames[] = {
    MAIZE_ROW("bf16", "nt", "64"), MAIZE_ROW("bf16", "nn", "64"), MAIZE_DEPTH("bf16"),
    MAIZE_ROW("f16", "nt", "64"),  MAIZE_ROW("f16", "nn", "64"),  MAIZE_DEPTH("f16"),
    MAIZE_ROW("e4m3", "nt", "64"), MAIZE_ROW("e4m3", "nn", "128"),
};
#undef MAIZE_ROW
#undef MAIZE_DEPTH
constexpr uint32_t kNameCount = sizeof(kNames) / sizeof(kNames[0]);
static_assert(kNameCount + kQuantKernels <= kMaxMoreKernels, "the launcher's table of functions");
constexpr const char* kQuant[kQuantKernels] = {"maize_quantize_bf16_rows", "maize_quantize_bf16_blocks", "maize_quantize_f16_rows",
                                               "maize_quantize_f16_blocks", "maize_quantize_f32_rows", "maize_quantize_f32_blocks"};

uint64_t cdiv(uint64_t a, uint64_t b) { return (a + b - 1u) / b; }

// The most tiles there can be, however the rows spread: every group that has rows may end in a tile that is not full.
uint64_t most_tiles(const maize_gemm_grouped_desc_t& d, const Shape& s) {
    if (d.axis == MAIZE_GROUP_DEPTH) return cdiv(d.c.nrows, s.bm) * cdiv(d.c.ncols, s.bn) * d.groups;
    const uint64_t rows = d.a.nrows, busy = d.offsets ? (d.groups < rows ? d.groups : rows) : 1u;
    return (rows + busy * (s.bm - 1u)) / s.bm * cdiv(d.c.ncols, s.bn);
}
// ... and the workgroups that may find one: of a depth product an eighth of each group's for every XCD.
uint64_t most_items(const maize_gemm_grouped_desc_t& d, const Shape& s, uint32_t ranges) {
    if (d.axis == MAIZE_GROUP_DEPTH) return cdiv(cdiv(d.c.nrows, s.bm) * cdiv(d.c.ncols, s.bn) * ranges, 8u) * 8u * d.groups;
    return most_tiles(d, s) * ranges;
}

// What a launch takes, in us, as fitted to 760 drawn products (one to 16384 rows, one to 64 groups, K and N from 256 to 16384, every type and
// layout; each on every tile and number of K ranges).  A workgroup: `fixed` and `step` for each K tile, `lone` times that while the
// launch leaves half of the places empty; `half`: a half tile's share of a whole one.  The tile that the model picks takes 2.2 % more
// than the best one on average, more than 10 % on 66 of the 760.  By even sizes: the host does not know how the rows spread.
struct Cost { double step[2], fixed, half, lone; };                // step: 16-bit, 8-bit operands (few rows, K x N: kStepFewKN)
constexpr Cost kCost[kTiles] = {{{1.17, 0.88}, 12.5, 0.60, 0.74}, {{0.77, 0.76}, 5.2, 0.76, 0.74}, {{0.32, 0.75}, 3.3, 1.0, 0.47}};
constexpr double kStepFewKN = 0.94;
constexpr double kRanges = 1.76, kRange = 0.55;                    // joining K ranges: at all, and for each
constexpr double kTail = 0.24, kBytesPerUs = 3.7e6, kLaunch = 2.4, kNorm = 3.65;

double estimate(const maize_gemm_grouped_desc_t& d, uint32_t tile, uint32_t ranges, uint32_t compute_units) {
    const bool bits8 = d.in_type == MAIZE_IN_E4M3, depth = d.axis == MAIZE_GROUP_DEPTH;
    const Shape& s = shapes(d)[tile];
    const Cost& c = kCost[tile];
    const double rows = d.a.nrows, busy = depth ? d.groups : std::max(1.0, std::min(rows, d.offsets ? (double)d.groups : 1.0)), each = rows / busy;
    const double k_tiles = depth ? std::max(1.0, each / 64.0) : (double)cdiv(d.a.ncols, bits8 ? 128u : 64u);
    double panels = depth ? (double)cdiv(d.c.nrows, s.bm) : 1.0;
    const double full = each / s.bm, places = tile == kLarge ? 1.0 : s.bn == 64u ? 3.0 : 2.0;      // workgroups on a compute unit
    if (!depth && tile == kFew) panels = each <= 20.0 ? 1.0 : std::max(1.0, full + 0.5);
    else if (!depth) panels = full <= 0.4 ? c.half : full < 1.0 ? c.half + (1.0 - c.half) * (full - 0.4) / 0.6 : full + 0.25;
    const double tiles = busy * panels * (double)cdiv(d.c.ncols, s.bn), rounds = tiles * ranges / (places * compute_units);
    const double one = c.fixed + (s.bm == 32u && s.bn == 128u ? kStepFewKN : c.step[bits8]) * k_tiles / ranges + (ranges > 1u ? kRanges + kRange * ranges : 0.0);
    const double compute = one * (rounds <= 0.5 ? c.lone : rounds <= 1.0 ? c.lone + (1.0 - c.lone) * (rounds - 0.5) * 2.0 : rounds + kTail * std::min(1.0, rounds - 1.0));
    const double in = bits8 ? 1.0 : 2.0, out = d.out_type == MAIZE_OUT_F32 ? 4.0 : 2.0, times = d.beta != 0.0f ? 2.0 : 1.0, n = d.c.ncols;
    const double bytes = (depth ? in * rows * (d.c.nrows + n) + out * times * d.groups * d.c.nrows * n : in * (rows * d.a.ncols + busy * d.a.ncols * n) + out * times * rows * n) +
                         (ranges > 1u ? tiles * ranges * s.bm * s.bn * 4.0 : 0.0);
    // (a few rows for each group: what the larger tiles add is theirs alone, and near ties go to the small ones: 16 rows of 8 groups on
    // 8-bit weights 91 us on 128 x 128, 78 on 32 x 64)
    return (!depth && tile != kFew && each <= 32.0 ? 1.05 : 1.0) * (kLaunch + std::pow(std::pow(compute, kNorm) + std::pow(bytes / kBytesPerUs, kNorm), 1.0 / kNorm));
}

}  // namespace

uint32_t group_kernel_count() { return kNameCount; }
const char* group_kernel_name(uint32_t index) { return index < kNameCount ? kNames[index] : nullptr; }
const char* quant_kernel_name(uint32_t index) { return index < kQuantKernels ? kQuant[index] : nullptr; }

bool plan_group(const maize_gemm_grouped_desc_t& d, uint32_t compute_units, GroupPlan* out, bool split) {
    const bool bits8 = d.in_type == MAIZE_IN_E4M3, depth = d.axis == MAIZE_GROUP_DEPTH;
    const Shape* shape = shapes(d);
    double best = 0.0;
    bool found = false;
    for (uint32_t tile = 0; tile < kTiles; ++tile) {
        if (tile == kFew && (depth || d.a.nrows > 4096u)) continue;
        const double k_tiles = depth ? (double)d.a.nrows / d.groups / 64.0 : (double)cdiv(d.a.ncols, bits8 ? 128u : 64u);
        const uint64_t tiles = most_tiles(d, shape[tile]);
        for (uint32_t ranges : {1u, 2u, 3u, 4u, 6u, 8u, 12u, 16u}) {
            // K ranges: of two K tiles or more; tiles that each have a ticket counter; parts for two rounds at most of 128 x 128 (two
            // workgroups on a compute unit), for 2.7 of 32 x 64 (three) and four of 32 x 128 (two)
            if (ranges > 1u && (!split || tile == kLarge || k_tiles < 2.0 * ranges || tiles > kTicketBytes / 4u || tiles * ranges > (tile == kFew ? 8u : 4u) * compute_units)) break;
            const uint64_t items = most_items(d, shape[tile], ranges);
            if (items >= (1u << 24) / (shape[tile].threads / 256u)) break;         // (a launch counts its work items in 32 bits)
            const double cost = estimate(d, tile, ranges, compute_units);
            if (found && cost >= best) continue;
            found = true;
            best = cost;
            out->kernel = (bits8 ? 18u : (d.in_type == MAIZE_IN_F16 ? 9u : 0u)) + (depth ? 6u : d.layout == MAIZE_LAYOUT_NT ? 0u : 3u) + tile;
            out->grid = (uint32_t)items;
            out->block = shape[tile].threads;
            out->ksplit = ranges;
            out->workspace_bytes = ranges > 1u ? kTicketBytes + (size_t)tiles * ranges * shape[tile].bm * shape[tile].bn * 4u : 0u;
        }
    }
    return found;
}

}  // namespace maize
