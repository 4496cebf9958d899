// Second launch of the norm's backward: the weight's gradient from the row groups' shares (vrank_fused.h).  Short, and bound by the
// latency of its loads: eight in flight to a lane, a line and a half of a share to a wavefront; 3.4 us for 64 shares of 2048 columns.
#include "vrank_fused_impl.hpp"

namespace MegRay {
namespace vrank {

namespace {

using namespace fused;

constexpr uint32_t kWaves = kNormWeightThreads / 64;

// A workgroup takes 64 columns of one part, a lane each; its wavefronts split the part's row groups and meet in LDS.
__global__ void __launch_bounds__(64 * kWaves) norm_weight(const NormWeightLaunch L) {
    __shared__ float share[kWaves][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t col = blockIdx.x * 64 + lane, part = blockIdx.y;
    float sum = 0.0f;
    if (col < L.cols) {
        const float* p = L.partial + uint64_t(part) * L.part_groups * L.cols + col;
#pragma unroll 8
        for (uint32_t g = wave; g < L.part_groups; g += kWaves) sum += p[uint64_t(g) * L.cols];
    }
    share[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || col >= L.cols) return;
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) sum += share[w][lane];
    if (L.nparts == 1)
        for (uint32_t r = 0; r < L.nranks; ++r) L.dweight[r][col] = sum;
    else
        L.dweight[part][col] = sum;
}

}  // namespace

const void* norm_weight_kernel() {
    return reinterpret_cast<const void*>(&norm_weight);
}

}  // namespace vrank
}  // namespace MegRay
