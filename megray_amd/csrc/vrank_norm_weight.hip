// Second launch of the norm's backward: the weight's gradient from the row groups' shares (vrank_fused.h).  Short, and bound by the latency of
// its loads: 2.9 us for 64 shares of 2048 columns (one load to a lane, 128 workgroups), 4.9 for 512 of 8192 (16 MiB, 32 loads to a lane, eight in flight).
#include "vrank_fused_impl.hpp"

namespace MegRay {
namespace vrank {

namespace {

using namespace fused;

// A workgroup takes `Cols` columns of one part; its lanes take the part's row groups in turn, a column each, and meet in LDS.
template <uint32_t Cols>
__global__ void __launch_bounds__(kNormWeightThreads) norm_weight(const NormWeightLaunch L) {
    constexpr uint32_t kTurns = kNormWeightThreads / Cols;
    __shared__ float share[kTurns][Cols];
    const uint32_t at = threadIdx.x % Cols, turn = threadIdx.x / Cols;
    const uint32_t col = blockIdx.x * Cols + at, part = blockIdx.y;
    float sum = 0.0f;
    if (col < L.cols) {
        const float* p = L.partial + uint64_t(part) * L.part_groups * L.cols + col;
#pragma unroll 8
        for (uint32_t g = turn; g < L.part_groups; g += kTurns) sum += p[uint64_t(g) * L.cols];
    }
    share[turn][at] = sum;
    __syncthreads();
    if (turn != 0 || col >= L.cols) return;
#pragma unroll
    for (uint32_t w = 1; w < kTurns; ++w) sum += share[w][at];
    if (L.nparts == 1)
        for (uint32_t r = 0; r < L.nranks; ++r) L.dweight[r][col] = sum;
    else
        L.dweight[part][col] = sum;
}

}  // namespace

const void* norm_weight_kernel(uint32_t cols) {
    return cols == 16 ? reinterpret_cast<const void*>(&norm_weight<16>) : reinterpret_cast<const void*>(&norm_weight<64>);
}

}  // namespace vrank
}  // namespace MegRay
