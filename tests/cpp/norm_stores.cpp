// Which rows of the norm behind a fold may leave by buffer stores, checked on the host: no GPU.
//
// vrank_fused.cpp is compiled as it is; this file supplies what it calls below that line.  A kernel "address" here says
// which kernel was asked for, and hipLaunchKernel() keeps it.  Buffer stores need a 4-byte boundary; a row's last piece is
// moved back to end with the row, so wherever the streaming kernels are chosen every piece of every stored buffer has to
// begin on one - and rows on cache lines for which that is so have to get them.
// Prints "ok" and the number of launches looked at, or the first violation.
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "megray/hip_context.h"
#include "vrank_fused.h"

using namespace MegRay;
using namespace MegRay::vrank;

namespace {

// [direction][streaming]: addresses that stand for kernels
char g_tags[2][2];
char g_weight_tag, g_adamw_tag;
const void* g_launched = nullptr;
dim3 g_grid;

NormKernels kernels(bool lines) {
    return {&g_tags[0][lines], &g_tags[1][lines]};
}

[[noreturn]] void violation(const char* format, ...) {
    va_list args;
    va_start(args, format);
    std::printf("VIOLATION: ");
    std::vprintf(format, args);
    std::printf("\n");
    std::exit(1);
}

}  // namespace

namespace MegRay {
namespace vrank {
NormKernels norm_kernels_f16(NormVariant, uint32_t, bool lines, bool) { return kernels(lines); }
NormKernels norm_kernels_f16_f32(NormVariant, uint32_t, bool lines, bool) { return kernels(lines); }
NormKernels norm_kernels_bf16(NormVariant, uint32_t, bool lines, bool) { return kernels(lines); }
NormKernels norm_kernels_bf16_f32(NormVariant, uint32_t, bool lines, bool) { return kernels(lines); }
NormKernels norm_kernels_f32(NormVariant, uint32_t, bool lines, bool) { return kernels(lines); }
const void* norm_weight_kernel(uint32_t) { return &g_weight_tag; }
const void* adamw_kernel_for(int, int, bool) { return &g_adamw_tag; }
const void* adamw_norm_kernel_for(int) { return &g_adamw_tag; }
const void* adamw_norm_join_kernel() { return &g_adamw_tag; }
}  // namespace vrank
}  // namespace MegRay

extern "C" {
hipError_t hipLaunchKernel(const void* kernel, dim3 grid, dim3, void**, size_t, hipStream_t) {
    if (kernel != &g_weight_tag) {
        g_launched = kernel;
        g_grid = grid;
    }
    return hipSuccess;
}
hipError_t hipGetDevice(int* device) { *device = 0; return hipSuccess; }
hipError_t hipGetLastError() { return hipSuccess; }
const char* hipGetErrorString(hipError_t) { return ""; }
hipError_t hipMalloc(void**, size_t) { return hipErrorOutOfMemory; }
hipError_t hipMemcpy(void*, const void*, size_t, hipMemcpyKind) { return hipErrorUnknown; }
hipError_t hipFree(void*) { return hipSuccess; }
}

namespace {

size_t size_of(int dtype) {
    return dtype == MEGRAY_FLOAT32 ? 4 : dtype == MRV_BFLOAT16 || dtype == MEGRAY_FLOAT16 ? 2 : 1;
}

// Whether every piece of a row of `cols` elements begins on a 4-byte boundary of a row that begins on one: pieces of
// eight, or of four where a 32-bit type takes part.
bool pieces_on_dwords(uint32_t cols, size_t elem, bool split) {
    const uint32_t width = split ? 4 : 8;
    for (uint32_t want = 0; want < cols; want += width) {
        const uint32_t at = want + width <= cols ? want : cols - width;
        if (at * elem % 4) return false;
    }
    return true;
}

constexpr uintptr_t kApart = uintptr_t(1) << 30;

}  // namespace

int main() {
    size_t seen = 0, streamed = 0;
    std::vector<void*> buffers[5];
    for (int b = 0; b < 5; ++b)
        for (uintptr_t r = 0; r < 3; ++r) buffers[b].push_back(reinterpret_cast<void*>((1 + uintptr_t(b) * 8 + r) * kApart));
    auto in = [&](int b) { return reinterpret_cast<const void* const*>(buffers[b].data()); };
    auto floats = [&](int b) { return reinterpret_cast<float* const*>(buffers[b].data()); };
    const void* const weight = reinterpret_cast<const void*>(60 * kApart);
    const int types[][2] = {{MRV_BFLOAT16, MRV_BFLOAT16}, {MEGRAY_FLOAT16, MEGRAY_FLOAT32}, {MEGRAY_FLOAT32, MEGRAY_FLOAT32}};
    for (const auto& type : types) {
        for (int collective : {int(MRV_ALL_REDUCE), int(MRV_REDUCE_SCATTER)}) {
            for (size_t rows : {1, 2, 5}) {
                for (uint32_t cols = 129; cols <= 16384; cols = cols < 1100 ? cols + 1 : cols + 509) {
                    // rows padded to a cache line of the narrowest type, or not padded (0)
                    for (size_t stride : {size_t(0), size_t(cols + 127) / 128 * 128}) {
                        for (int out : {type[0], int(MEGRAY_INT8)}) {
                            mrv_rms_norm_call c{};
                            c.sendbuffs = in(0);
                            c.residuals = in(1);
                            c.residual_outs = buffers[2].data();
                            c.outs = buffers[3].data();
                            c.scales = out == MEGRAY_INT8 ? floats(4) : nullptr;
                            c.weight = weight;
                            c.rows = rows, c.cols = cols;
                            c.send_stride = c.residual_stride = c.residual_out_stride = c.out_stride = stride;
                            c.nranks = 3;
                            c.dtype = c.weight_dtype = type[0], c.residual_dtype = type[1], c.out_dtype = out;
                            c.eps = 1e-5f;
                            NormPlan plan;
                            plan.plan_forward(collective, c);
                            plan.launch(nullptr);
                            const bool split = type[1] == MEGRAY_FLOAT32;
                            const bool dwords = pieces_on_dwords(cols, size_of(type[1]), split) && pieces_on_dwords(cols, size_of(out), split);
                            // several rows (of the fold, too) have to begin on lines each
                            const bool fold_rows = rows > 1 || collective == MRV_REDUCE_SCATTER;
                            const size_t step = stride ? stride : cols;
                            const bool lines = (!fold_rows || step * size_of(type[0]) % 128 == 0) &&
                                               (rows == 1 || (step * size_of(type[1]) % 128 == 0 && step * size_of(out) % 128 == 0));
                            const bool got = g_launched == &g_tags[0][1];
                            if (got && !dwords) violation("forward: %zu rows of %u, stride %zu, types %d %d -> %d stream off a dword", rows, cols, stride, type[0], type[1], out);
                            if (got != (lines && dwords)) violation("forward: %zu rows of %u, stride %zu, types %d %d -> %d: streamed %d", rows, cols, stride, type[0], type[1], out, got);
                            ++seen, streamed += got;
                        }
                        for (int what = 1; what < 4; ++what) {  // which gradients are stored
                            mrv_rms_norm_backward_call c{};
                            c.sendbuffs = in(0);
                            c.hiddens = in(1);
                            c.residual_out_grads = what & 1 ? buffers[2].data() : nullptr;
                            c.send_grads = what & 2 ? buffers[3].data() : nullptr;
                            c.weight = weight;
                            c.rows = rows, c.cols = cols;
                            c.send_stride = c.hidden_stride = c.residual_out_grad_stride = c.send_grad_stride = stride;
                            c.nranks = 3;
                            c.dtype = c.weight_dtype = type[0], c.residual_dtype = type[1];
                            c.eps = 1e-5f;
                            NormPlan plan;
                            plan.plan_backward(collective, c);
                            plan.launch(nullptr);
                            // pieces of four of the streaming kernels
                            const bool split = type[1] == MEGRAY_FLOAT32;
                            const bool dwords = (!(what & 1) || pieces_on_dwords(cols, size_of(type[1]), split)) &&
                                                (!(what & 2) || pieces_on_dwords(cols, size_of(type[0]), split));
                            const bool fold_rows = rows > 1 || collective == MRV_REDUCE_SCATTER;
                            const size_t step = stride ? stride : cols;
                            const bool lines = (!fold_rows || step * size_of(type[0]) % 128 == 0) &&
                                               (rows == 1 || (step * size_of(type[1]) % 128 == 0 && step * size_of(type[0]) % 128 == 0));
                            const bool got = g_launched == &g_tags[1][1];
                            if (got && !dwords) violation("backward: %zu rows of %u, stride %zu, types %d %d, stored %d stream off a dword", rows, cols, stride, type[0], type[1], what);
                            if (got != (lines && dwords)) violation("backward: %zu rows of %u, stride %zu, types %d %d, stored %d: streamed %d", rows, cols, stride, type[0], type[1], what, got);
                            ++seen, streamed += got;
                        }
                    }
                }
            }
        }
    }
    std::printf("ok %zu launches, %zu streamed\n", seen, streamed);
    return 0;
}
