// Folds with an epilogue: what a tensor- or data-parallel model does with the sum right behind its reduction, in the
// pass that makes the sum.  Launch descriptors, planning, and the entry points the C ABI calls.
//
//   rms_norm           h = residual + sum over ranks, y = h / rms(h) * weight, h and y to every rank (all_reduce) or each
//                      rank's rows to it (reduce_scatter); y in the sends' type or in 8 bits with a scale per row
//   rms_norm_backward  the fold of the partial gradients of y, the norm's backward behind it, the weight's gradient
//   Adamw              the norm of the folded gradients of many tensors, and the AdamW step that takes them
//
// Sums over ranks are taken in rank order 0 .. N-1 in 32 bits, whatever the sends' type: every result is rounded once,
// when it is stored, and is the same on every run.
#pragma once

#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <memory>
#include <utility>
#include <vector>

#include "megray_vrank.h"
#include "megray/common.h"
#include "vrank_types.h"

namespace MegRay {
namespace vrank {

// ---- the norm behind a fold ------------------------------------------------------------------

#ifdef __HIPCC__
#define MRV_DEVICE __device__ __forceinline__
#else
#define MRV_DEVICE inline
#endif

constexpr uint32_t kNormVec = 8;             // elements a lane holds of a row at a time: 16 bytes of a 16-bit type

// Which row a workgroup takes.  Workgroups go to the eight XCDs in turn; dealt out in runs of 2^shift, neighbouring rows are
// written by one XCD, through one L2, at about the same time.  Positions from `whole` on keep their own row.
struct Deal {
    uint32_t shift, whole;
    MRV_DEVICE uint32_t of(uint32_t n) const {
        if (n >= whole) return n;
        return (n >> (shift + 3) << (shift + 3)) + ((n & 7u) << shift) + ((n >> 3) & ((1u << shift) - 1u));
    }
};

// Whether a wavefront's stores go one at a time.
struct Pace {
    uint32_t on;
    MRV_DEVICE void wait() const {
#ifdef __HIP_DEVICE_COMPILE__
        if (on) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#endif
    }
};

struct NormLaunch {
    const void* send[kMaxRanks];  // the kernels read `send` and `hidden`, `out` and `scales` as one table each
    void* hidden[kMaxRanks];
    void* out[kMaxRanks];
    float* scales[kMaxRanks];
    const void* residual[kMaxRanks];  // all_reduce: entry 0; entry 0 null: no residual
    const void* weight;
    uint64_t send_stride, residual_stride, hidden_stride, out_stride;  // bytes from a row to the next
    uint32_t rows;       // of the fold: all of them
    uint32_t part_rows;  // rows of a destination: `rows` (all_reduce), rows / nranks (reduce_scatter)
    uint32_t cols;
    uint32_t nranks;
    uint32_t ndst;       // destinations of a row: nranks, or 1
    uint32_t weight32;   // the weight is FLOAT32 whatever the sends are
    uint32_t int8;       // 8-bit output: 1 INT8, 0 FLOAT8_E4M3
    uint32_t keep;       // stores leave their data in the last-level cache
    uint32_t has_hidden;
    float eps;
    uint32_t lanes;      // of a row, where a workgroup is one row: a multiple of 64
    uint32_t positions;  // rows in units of what a workgroup takes at a time
    uint32_t splits;     // workgroups that share a row's destinations, each folding the row for itself
    Deal deal;           // of the positions
    Pace pace;
};

struct NormBackLaunch {
    const void* send[kMaxRanks];         // partial gradients of y; read with `dhidden` as one table
    void* dhidden[kMaxRanks];            // entry 0 null: not wanted
    void* dsend[kMaxRanks];              // entry 0 null: not wanted; read with `hidden` as one table
    const void* hidden[kMaxRanks];       // all_reduce: entry 0
    const void* arriving[kMaxRanks];     // all_reduce: entry 0; null: none
    const void* weight;
    float* partial;                      // [groups][cols] sums of the weight's gradient; null: not wanted
    uint64_t send_stride, hidden_stride, arriving_stride, dhidden_stride, dsend_stride;  // bytes
    uint32_t rows;
    uint32_t part_rows;   // rows that share one weight gradient: all (all_reduce), a rank's (reduce_scatter)
    uint32_t part_groups; // row groups that walk them
    uint32_t groups;      // all row groups
    uint32_t cols;
    uint32_t nranks;
    uint32_t ndst;
    uint32_t weight32;
    uint32_t keep;
    float eps;
    uint32_t lanes;
    Deal deal;  // of a part's rows
};

struct NormWeightLaunch {  // the second launch of a backward: weight gradients from the row groups' sums
    const float* partial;
    float* dweight[kMaxRanks];
    uint32_t part_groups;
    uint32_t cols;
    uint32_t nparts;  // 1 (all_reduce: the same sum to every rank), nranks (reduce_scatter)
    uint32_t nranks;
};

// How a row is spread over lanes: rows of fewer than eight elements have a lane each (kNormNarrow), rows of up to 128 sixteen lanes (kNormShort), in
// the backward of up to 256 thirty-two (kNormShort32), of up to 512 a wavefront (kNormWave), rows of up to 8192 and 16384 a workgroup of as many wavefronts as they fill with one and two vectors per lane
// (kNormBlock, kNormBlock2), and longer ones are swept twice (kNormLong).
enum NormVariant { kNormNarrow, kNormShort, kNormShort32, kNormWave, kNormBlock, kNormBlock2, kNormLong };

struct NormKernels {  // addresses usable with hipLaunchKernel; null where the type has no such form
    const void* forward;
    const void* backward;
};

// in vrank_norm_<sends' type>[_<residual stream's type>].hip; `lines`: every row of every buffer begins on a cache line,
// and every stored row ends on a 4-byte boundary
NormKernels norm_kernels_f16(NormVariant v, uint32_t nranks, bool lines, bool q8);
NormKernels norm_kernels_f16_f32(NormVariant v, uint32_t nranks, bool lines, bool q8);
NormKernels norm_kernels_bf16(NormVariant v, uint32_t nranks, bool lines, bool q8);
NormKernels norm_kernels_bf16_f32(NormVariant v, uint32_t nranks, bool lines, bool q8);
NormKernels norm_kernels_f32(NormVariant v, uint32_t nranks, bool lines, bool q8);
constexpr uint32_t kNormWeightThreads = 1024;
const void* norm_weight_kernel(uint32_t cols);  // of a workgroup, 16 or 64; grid: workgroups along a row, parts

// ---- AdamW over many tensors -------------------------------------------------------------------

constexpr uint32_t kAdamVec = 8;               // elements of a lane
// Lanes of a workgroup: a large one reads and writes longer runs of a buffer at a time, a small one is sooner done with its chain
// of loads, scales and stores.  256 and 1024, BF16: the step with 32-bit states, 8 ranks, 98 M parameters 1088 and 1052 us, 1 rank, 157 M 766
// and 737 (but 1 rank, 13 M, 60.1 and 62.4); with 8-bit states, 4 ranks, 50 M, 274 and 309; the norm, 8 ranks, 98 M, 236 and 261.
constexpr uint32_t kAdamThreads = 1024;        // of the step with 32-bit states
constexpr uint32_t kAdamThreads8 = 256;        // of the step with 8-bit states
constexpr uint32_t kAdamNormThreads = 256;     // of the gradient norm
constexpr uint32_t kAdamBlock = 256;                       // elements that share a scale of an 8-bit state: half a wavefront's

struct AdamTensor {  // one per tensor, in device memory
    uint64_t len;
    float* master;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    float decay;
    uint32_t lines;  // every buffer of the tensor begins on a cache line
};

struct AdamTile {  // what a workgroup takes at a time: as many elements as its lanes hold
    uint32_t tensor;
    uint32_t tile;  // within the tensor
};

struct AdamLaunch {
    const AdamTensor* tensors;
    const AdamTile* tiles;
    const void* const* grads;  // [tensor][rank]
    void* const* params;       // [tensor][rank]
    uint32_t grad_ranks, param_ranks;
    uint32_t ntiles;
    Deal deal;  // of the tiles
    uint32_t keep;  // stores leave their data in the last-level cache
    Pace pace;
    float lr, beta1, beta2, eps;
    float rest1, rest2;  // 1 - beta1, 1 - beta2, from 64 bits: a beta near 1 has few bits of them left
    float rate;        // lr / (1 - beta1^step)
    float root_scale;  // 1 / sqrt(1 - beta2^step)
    float grad_scale;
    const float* clip;  // null: 1
};

struct AdamNormLaunch {
    const AdamTensor* tensors;
    const AdamTile* tiles;
    const void* const* grads;
    uint32_t grad_ranks;
    uint32_t ntiles;
    uint32_t groups;
    Deal deal;  // of the tiles
    float grad_scale;
    float max_norm;
    float* out;  // [0] the norm, [1] the coefficient, then `groups` 64-bit sums
};

const void* adamw_kernel_for(int grad_dtype, int param_dtype, bool state8);
const void* adamw_norm_kernel_for(int grad_dtype);
constexpr uint32_t kAdamJoinThreads = 1024;
const void* adamw_norm_join_kernel();

// ---- planning and launching ----------------------------------------------------------------------

// A HIP call failed while a handle was made.
struct HipFailure {};

// A fused collective with its arguments checked and its launches laid out: planned once, forward or backward.
class NormPlan {
public:
    NormPlan();
    NormPlan(const NormPlan&) = delete;
    NormPlan& operator=(const NormPlan&) = delete;
    // Contract violations throw MegRay::Exception.
    void plan_forward(int collective, const mrv_rms_norm_call& call);
    void plan_backward(int collective, const mrv_rms_norm_backward_call& call);
    Status launch(hipStream_t stream) const;
    size_t launch_count() const { return (m_first ? 1u : 0u) + (m_second ? 1u : 0u); }

private:
    const void* m_first = nullptr;
    const void* m_second = nullptr;
    const void* m_descriptor = nullptr;  // of the first launch: m_forward or m_backward
    uint32_t m_grid = 0, m_block = 0, m_weight_cols = 0;
    NormLaunch m_forward;
    NormBackLaunch m_backward;
    NormWeightLaunch m_weight;
};

// Bytes of workspace a backward with weight gradients needs.
size_t norm_backward_workspace(int collective, uint32_t nranks, size_t rows, size_t cols);

// Address ranges, added in the order of their beginnings.
class Taken {
public:
    void add(uintptr_t begin, uintptr_t end);
    bool overlaps(uintptr_t begin, uintptr_t end) const;

private:
    std::vector<std::pair<uintptr_t, uintptr_t>> m_runs;  // apart, ascending
};

class Adamw {
public:
    // Checks the tensors and uploads their tables (device allocation, synchronous).
    explicit Adamw(const mrv_adamw_tensors& t);
    ~Adamw();
    Adamw(const Adamw&) = delete;
    Adamw& operator=(const Adamw&) = delete;

    size_t norm_floats() const { return 2 + 2 * size_t(m_groups); }
    Status grad_norm(float grad_scale, float max_norm, float* out, hipStream_t stream) const;
    Status step(const mrv_adamw_step_args& args, hipStream_t stream) const;

private:
    void check_device() const;
    void* m_table = nullptr;  // device
    int m_device = 0;
    uint32_t m_groups = 0, m_threads = 0;
    bool m_can_step = false;
    Taken m_any, m_written;  // by the tensors
    AdamLaunch m_step{};
    AdamNormLaunch m_norm{};
    const void* m_step_kernel = nullptr;
    const void* m_norm_kernel = nullptr;
};

}  // namespace vrank
}  // namespace MegRay
