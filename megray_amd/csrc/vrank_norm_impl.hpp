// Kernels of the norm behind a fold and of its backward (vrank_fused.h).  Per-type translation units
// (vrank_norm_<type>.hip) instantiate them.
//
// A row is one reduction: `Lanes` lanes keep it in registers, `Vecs` vectors of eight elements each, so that everything
// is read once: N partial rows are summed as they arrive, the residual is added, the sum of squares (and, for 8-bit
// outputs, the largest |h * weight|, which times 1 / rms is the largest |y|) goes once across the lanes, and the row is
// stored to every destination from the registers.  The bound is HBM: two to four bytes of traffic per operation.
//
// A row whose length is no multiple of eight ends in a vector that is moved back to end with the row: the lane that owns
// it repeats up to seven elements of its neighbour, leaves them out of the sums, and stores the same values.  All loads of a
// row come before the reduction and all its stores behind it, so outputs that take an input's place are safe with that too.
#pragma once

#include "vrank_fused_impl.hpp"

namespace MegRay {
namespace vrank {
namespace detail {

using namespace fused;

constexpr uint32_t norm_block(uint32_t lanes) {
    return lanes < 256 ? 256 : lanes;  // rows of one wavefront go four to a workgroup
}

// Sums (and a maximum) over the lanes of a row.  `slot` alternates between rows that follow each other in a workgroup: a
// wavefront may be a row ahead of the others, never two.
template <uint32_t Lanes, int Sums, bool Max>
struct RowReduce {
    static constexpr uint32_t kWaves = Lanes / 64;
    struct Shared {
        float sum[2][Sums][kWaves];
        uint32_t max[2][Max ? kWaves : 1];
    };
    static __device__ __forceinline__ void run(Shared& s, uint32_t slot, float (&sum)[Sums], uint32_t& max) {
#pragma unroll
        for (int i = 0; i < Sums; ++i) sum[i] = across_wave(sum[i], Plus());
        if (Max) max = across_wave(max, Larger());
        if constexpr (kWaves > 1) {
            const uint32_t wave = threadIdx.x / 64;
            if (threadIdx.x % 64 == 0) {
#pragma unroll
                for (int i = 0; i < Sums; ++i) s.sum[slot][i][wave] = sum[i];
                if (Max) s.max[slot][wave] = max;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < Sums; ++i) {
                sum[i] = s.sum[slot][i][0];
#pragma unroll
                for (uint32_t w = 1; w < kWaves; ++w) sum[i] += s.sum[slot][i][w];
            }
            if (Max) {
                max = s.max[slot][0];
#pragma unroll
                for (uint32_t w = 1; w < kWaves; ++w) max = Larger()(max, s.max[slot][w]);
            }
        }
    }
};

// Which elements of a row this lane holds.
template <uint32_t Lanes, uint32_t Vecs>
struct RowPart {
    uint32_t col[Vecs];     // first element of vector k, never past cols - 8
    uint32_t repeat[Vecs];  // leading elements that belong to another lane (8 and more: all of them)
    __device__ __forceinline__ RowPart(uint32_t cols) {
        const uint32_t lane = threadIdx.x % Lanes;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            const uint32_t want = (k * Lanes + lane) * kNormVec;
            col[k] = want + kNormVec <= cols ? want : cols - kNormVec;
            repeat[k] = want - col[k];
        }
    }
    __device__ __forceinline__ bool stores(uint32_t k) const { return repeat[k] < kNormVec; }
};

// Adds rows `base + rank's offset` of `count` consecutive ranks to `acc`, all loads issued before the first sum.
// `left` ranks are there; those past them repeat the last one's loads and are not added.
template <typename T, uint32_t Vecs, uint32_t Ranks, bool Whole>
__device__ __forceinline__ void fold_ranks(const void* const* send, uint64_t row_offset, uint32_t left,
                                           const uint32_t (&col)[Vecs], float (&acc)[Vecs][8]) {
    Raw8<T> x[Ranks][Vecs];
#pragma unroll
    for (uint32_t r = 0; r < Ranks; ++r) {
        const char* p = static_cast<const char*>(send[Whole || r < left ? r : left - 1]) + row_offset;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[r][k] = load8<T, true>(p + col[k] * uint32_t(sizeof(T)));
    }
#pragma unroll
    for (uint32_t r = 0; r < Ranks; ++r) {
        if (Whole || r < left) {
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) {
                float f[8];
                widen<T>(x[r][k], f);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[k][i] += f[i];
            }
        }
    }
}

// Registers for about sixteen 16-byte loads in flight per lane.
template <typename T, uint32_t Vecs>
constexpr uint32_t ranks_at_once() {
    constexpr uint32_t loads = (sizeof(T) / 2) * Vecs;
    return loads >= 8 ? 1 : 8 / loads;
}

template <typename T, uint32_t Vecs>
__device__ __forceinline__ void fold_rows(const void* const* send, uint32_t nranks, uint64_t row_offset,
                                          const uint32_t (&col)[Vecs], float (&acc)[Vecs][8]) {
    constexpr uint32_t C = ranks_at_once<T, Vecs>();
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[k][i] = 0.0f;
    uint32_t r = 0;
    for (; r + C <= nranks; r += C) fold_ranks<T, Vecs, C, true>(send + r, row_offset, C, col, acc);
    if (r < nranks) fold_ranks<T, Vecs, C, false>(send + r, row_offset, nranks - r, col, acc);
}

template <typename T>
__device__ __forceinline__ void load_weight(const void* weight, uint32_t weight32, uint32_t col, float (&w)[8]) {
    if (weight32) widen<float>(load8<float, false>(static_cast<const char*>(weight) + uint64_t(col) * 4), w);
    else widen<T>(load8<T, false>(static_cast<const char*>(weight) + uint64_t(col) * sizeof(T)), w);
}

// R: the residual stream's type.  Q8: 8-bit output with a scale per row.
template <typename T, typename R, bool Q8, uint32_t Lanes, uint32_t Vecs>
__global__ void __launch_bounds__(norm_block(Lanes)) rms_norm_kernel(const NormLaunch L) {
    typedef RowReduce<Lanes, 1, Q8> Reduce;
    __shared__ typename Reduce::Shared shared;
    constexpr uint32_t kRows = norm_block(Lanes) / Lanes;
    const uint32_t row = blockIdx.x * kRows + (kRows > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / Lanes) : 0);
    if (kRows > 1 && row >= L.rows) return;  // a wavefront of its own: no barrier is missed
    const RowPart<Lanes, Vecs> part(L.cols);
    const uint32_t first = row / L.part_rows;  // destination (reduce_scatter); 0 (all_reduce)
    const uint32_t at = row - first * L.part_rows;

    float h[Vecs][8];
    fold_rows<T, Vecs>(L.send, L.nranks, uint64_t(row) * L.send_stride, part.col, h);
    if (L.residual[0]) {
        const char* p = static_cast<const char*>(L.residual[first]) + uint64_t(at) * L.residual_stride;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            float f[8];
            widen<R>(load8<R, true>(p + part.col[k] * uint32_t(sizeof(R))), f);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[k][i] += f[i];
        }
    }

    float w[Vecs][8];
    float sum[1] = {0.0f};
    uint32_t top = 0;
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) {
        load_weight<T>(L.weight, L.weight32, part.col[k], w[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sum[0] = __builtin_fmaf(h[k][i], uint32_t(i) >= part.repeat[k] ? h[k][i] : 0.0f, sum[0]);
            if (Q8) top = Larger()(top, magnitude(h[k][i] * w[k][i]));
        }
    }
    Reduce::run(shared, 0, sum, top);
    const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);

    float inverse = 0.0f;
    bool finite = true;
    if (Q8) {
        const float limit = L.int8 ? kInt8Max : kE4m3Max;
        float amax = r * __builtin_bit_cast(float, top);
        if (amax < kAmaxMin) amax = kAmaxMin;  // not true of a NaN
        finite = amax < __builtin_inff();
        inverse = limit / amax;
        if (threadIdx.x % Lanes == 0) {
            const float scale = finite ? amax / limit : __builtin_nanf("");
            for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[first + d] + at)) = scale;
        }
    }
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) {
        if (!part.stores(k)) continue;
        if (L.has_hidden) {
            const Raw8<R> x = narrow<R>(h[k]);
            const uint64_t off = uint64_t(at) * L.hidden_stride + part.col[k] * uint32_t(sizeof(R));
            for (uint32_t d = 0; d < L.ndst; ++d) store8<R>(static_cast<char*>(L.hidden[first + d]) + off, x, L.keep);
        }
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = h[k][i] * r * w[k][i];
        if constexpr (Q8) {
            const float limit = L.int8 ? kInt8Max : kE4m3Max;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = clamp_to(y[i] * inverse, limit);
            u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
            if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
            const uint64_t off = uint64_t(at) * L.out_stride + part.col[k];
            for (uint32_t d = 0; d < L.ndst; ++d) store_codes(static_cast<char*>(L.out[first + d]) + off, codes, L.keep);
        } else {
            const Raw8<T> x = narrow<T>(y);
            const uint64_t off = uint64_t(at) * L.out_stride + part.col[k] * uint32_t(sizeof(T));
            for (uint32_t d = 0; d < L.ndst; ++d) store8<T>(static_cast<char*>(L.out[first + d]) + off, x, L.keep);
        }
    }
}

// Rows of fewer than eight elements: a lane each.
template <typename T, typename R, bool Q8>
__global__ void __launch_bounds__(256) rms_norm_narrow_kernel(const NormLaunch L) {
    const uint32_t row = blockIdx.x * 256 + threadIdx.x;
    if (row >= L.rows) return;
    const uint32_t first = row / L.part_rows, at = row - first * L.part_rows;
    float h[kNormVec], w[kNormVec], sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) {
        h[c] = w[c] = 0.0f;
        if (c < L.cols) {
            for (uint32_t k = 0; k < L.nranks; ++k)
                h[c] += load_one<T>(static_cast<const char*>(L.send[k]) + uint64_t(row) * L.send_stride + c * sizeof(T));
            if (L.residual[0])
                h[c] += load_one<R>(static_cast<const char*>(L.residual[first]) + uint64_t(at) * L.residual_stride + c * sizeof(R));
            const char* p = static_cast<const char*>(L.weight);
            w[c] = L.weight32 ? load_one<float>(p + c * 4) : load_one<T>(p + c * sizeof(T));
            sum = __builtin_fmaf(h[c], h[c], sum);
            if (Q8) top = Larger()(top, magnitude(h[c] * w[c]));
        }
    }
    const float r = 1.0f / __builtin_sqrtf(sum / float(L.cols) + L.eps);
    float inverse = 0.0f;
    bool finite = true;
    const float limit = L.int8 ? kInt8Max : kE4m3Max;
    if (Q8) {
        float amax = r * __builtin_bit_cast(float, top);
        if (amax < kAmaxMin) amax = kAmaxMin;
        finite = amax < __builtin_inff();
        inverse = limit / amax;
        const float scale = finite ? amax / limit : __builtin_nanf("");
        for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[first + d] + at)) = scale;
    }
    float y[8];
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) y[c] = h[c] * r * w[c];
    if (Q8) {
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c) y[c] = clamp_to(y[c] * inverse, limit);
        u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
        if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c)
            if (c < L.cols)
                for (uint32_t d = 0; d < L.ndst; ++d)
                    *as_global<uint8_t>(static_cast<char*>(L.out[first + d]) + uint64_t(at) * L.out_stride + c) =
                            uint8_t(codes[c / 4] >> (8 * (c % 4)));
    }
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) {
        if (c >= L.cols) continue;
        for (uint32_t d = 0; d < L.ndst; ++d) {
            if (L.has_hidden)
                store_one<R>(static_cast<char*>(L.hidden[first + d]) + uint64_t(at) * L.hidden_stride + c * sizeof(R), h[c]);
            if (!Q8) store_one<T>(static_cast<char*>(L.out[first + d]) + uint64_t(at) * L.out_stride + c * sizeof(T), y[c]);
        }
    }
}

// Backward.  A row group (the lanes of one row) walks the rows of one part, `part_groups` apart, and carries its columns'
// share of the weight's gradient in registers; the shares meet in `partial`, and norm_weight_kernel adds them in order.
template <typename T, typename R, uint32_t Lanes, uint32_t Vecs>
__global__ void __launch_bounds__(norm_block(Lanes)) rms_norm_backward_kernel(const NormBackLaunch L) {
    typedef RowReduce<Lanes, 2, false> Reduce;
    __shared__ typename Reduce::Shared shared;
    constexpr uint32_t kGroups = norm_block(Lanes) / Lanes;
    const uint32_t group = blockIdx.x * kGroups + (kGroups > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / Lanes) : 0);
    if (kGroups > 1 && group >= L.groups) return;
    const RowPart<Lanes, Vecs> part(L.cols);
    const uint32_t first = group / L.part_groups;  // the destination whose rows these are (reduce_scatter); 0 (all_reduce)
    float w[Vecs][8], dw[Vecs][8];
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) {
        load_weight<T>(L.weight, L.weight32, part.col[k], w[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[k][i] = 0.0f;
    }
    const float mean = 1.0f / float(L.cols);
    uint32_t slot = 0;
    for (uint32_t at = group - first * L.part_groups; at < L.part_rows; at += L.part_groups, slot ^= 1) {
        const uint32_t row = first * L.part_rows + at;
        float g[Vecs][8], h[Vecs][8];
        fold_rows<T, Vecs>(L.send, L.nranks, uint64_t(row) * L.send_stride, part.col, g);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            const char* p = static_cast<const char*>(L.hidden[first]) + uint64_t(at) * L.hidden_stride;
            widen<R>(load8<R, true>(p + part.col[k] * uint32_t(sizeof(R))), h[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float mine = uint32_t(i) >= part.repeat[k] ? h[k][i] : 0.0f;
                sum[0] = __builtin_fmaf(h[k][i], mine, sum[0]);
                sum[1] = __builtin_fmaf(g[k][i] * w[k][i], mine, sum[1]);
            }
        }
        Raw8<R> arriving[Vecs];
        if (L.arriving[0]) {
            const char* p = static_cast<const char*>(L.arriving[first]) + uint64_t(at) * L.arriving_stride;
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) arriving[k] = load8<R, true>(p + part.col[k] * uint32_t(sizeof(R)));
        } else {
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) arriving[k] = Raw8<R>{};
        }
        uint32_t unused = 0;
        Reduce::run(shared, slot, sum, unused);
        const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        const float pull = r * r * r * (sum[1] * mean);
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            float dh[8];
            widen<R>(arriving[k], dh);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dh[i] += __builtin_fmaf(-pull, h[k][i], r * (g[k][i] * w[k][i]));
                dw[k][i] = __builtin_fmaf(g[k][i], h[k][i] * r, dw[k][i]);
            }
            if (!part.stores(k)) continue;
            if (L.dhidden[0]) {
                const Raw8<R> x = narrow<R>(dh);
                const uint64_t off = uint64_t(at) * L.dhidden_stride + part.col[k] * uint32_t(sizeof(R));
                for (uint32_t d = 0; d < L.ndst; ++d) store8<R>(static_cast<char*>(L.dhidden[first + d]) + off, x, L.keep);
            }
            if (L.dsend[0]) {
                const Raw8<T> x = narrow<T>(dh);
                const uint64_t off = uint64_t(at) * L.dsend_stride + part.col[k] * uint32_t(sizeof(T));
                for (uint32_t d = 0; d < L.ndst; ++d) store8<T>(static_cast<char*>(L.dsend[first + d]) + off, x, L.keep);
            }
        }
    }
    if (L.partial) {
        char* p = reinterpret_cast<char*>(L.partial + uint64_t(group) * L.cols);
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k)
            if (part.stores(k)) store8<float>(p + part.col[k] * 4, narrow<float>(dw[k]), true);
    }
}

// Rows of fewer than eight elements: a lane each, which is a row group of its own.
template <typename T, typename R>
__global__ void __launch_bounds__(256) rms_norm_backward_narrow_kernel(const NormBackLaunch L) {
    const uint32_t group = blockIdx.x * 256 + threadIdx.x;
    if (group >= L.groups) return;
    const uint32_t first = group / L.part_groups;
    float w[kNormVec], dw[kNormVec];
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) {
        const char* p = static_cast<const char*>(L.weight);
        w[c] = c >= L.cols ? 0.0f : L.weight32 ? load_one<float>(p + c * 4) : load_one<T>(p + c * sizeof(T));
        dw[c] = 0.0f;
    }
    for (uint32_t at = group - first * L.part_groups; at < L.part_rows; at += L.part_groups) {
        const uint64_t row = uint64_t(first) * L.part_rows + at;
        float g[kNormVec], h[kNormVec], a[kNormVec], square = 0.0f, inner = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c) {
            g[c] = h[c] = a[c] = 0.0f;
            if (c < L.cols) {
                for (uint32_t k = 0; k < L.nranks; ++k)
                    g[c] += load_one<T>(static_cast<const char*>(L.send[k]) + row * L.send_stride + c * sizeof(T));
                h[c] = load_one<R>(static_cast<const char*>(L.hidden[first]) + uint64_t(at) * L.hidden_stride + c * sizeof(R));
                if (L.arriving[0])
                    a[c] = load_one<R>(static_cast<const char*>(L.arriving[first]) + uint64_t(at) * L.arriving_stride + c * sizeof(R));
            }
            square = __builtin_fmaf(h[c], h[c], square);
            inner = __builtin_fmaf(g[c] * w[c], h[c], inner);
        }
        const float r = 1.0f / __builtin_sqrtf(square / float(L.cols) + L.eps);
        const float pull = r * r * r * (inner * (1.0f / float(L.cols)));
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c) {
            if (c >= L.cols) continue;
            const float dh = a[c] + __builtin_fmaf(-pull, h[c], r * (g[c] * w[c]));
            dw[c] = __builtin_fmaf(g[c], h[c] * r, dw[c]);
            for (uint32_t d = 0; d < L.ndst; ++d) {
                if (L.dhidden[0])
                    store_one<R>(static_cast<char*>(L.dhidden[first + d]) + uint64_t(at) * L.dhidden_stride + c * sizeof(R), dh);
                if (L.dsend[0])
                    store_one<T>(static_cast<char*>(L.dsend[first + d]) + uint64_t(at) * L.dsend_stride + c * sizeof(T), dh);
            }
        }
    }
    if (L.partial) {
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c)
            if (c < L.cols) L.partial[uint64_t(group) * L.cols + c] = dw[c];
    }
}

// Rows longer than the widest variant holds: the lanes sweep the row twice, the second time over data that the last-level
// cache mostly still has.  The vector at the row's end is taken element by element, so no element is read after another
// lane may have replaced it.
constexpr uint32_t kLongLanes = 1024;

template <typename T>
__device__ __forceinline__ void load_weight_part(const void* weight, uint32_t weight32, uint32_t col, uint32_t have, float (&w)[8]) {
    if (weight32) load_part<float>(static_cast<const char*>(weight) + uint64_t(col) * 4, have, w);
    else load_part<T>(static_cast<const char*>(weight) + uint64_t(col) * sizeof(T), have, w);
}
// The fold of `have` elements at byte `offset` of every rank's buffer.
template <typename T>
__device__ __forceinline__ void fold_part(const void* const* send, uint32_t nranks, uint64_t offset, uint32_t have, float (&acc)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < nranks; ++k) {
        float f[8];
        load_part<T>(static_cast<const char*>(send[k]) + offset, have, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += f[i];
    }
}

template <typename T, typename R, bool Q8>
__global__ void __launch_bounds__(kLongLanes) rms_norm_long_kernel(const NormLaunch L) {
    typedef RowReduce<kLongLanes, 1, Q8> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t row = blockIdx.x;
    const uint32_t first = row / L.part_rows, at = row - first * L.part_rows;
    const uint64_t send_row = uint64_t(row) * L.send_stride;
    const char* residual = L.residual[0] ? static_cast<const char*>(L.residual[first]) + uint64_t(at) * L.residual_stride : nullptr;
    float sum[1] = {0.0f};
    uint32_t top = 0;
    float r = 0.0f, inverse = 0.0f;
    bool finite = true;
    const float limit = L.int8 ? kInt8Max : kE4m3Max;
    for (uint32_t sweep = 0; sweep < 2; ++sweep) {
        for (uint64_t c = uint64_t(threadIdx.x) * kNormVec; c < L.cols; c += kLongLanes * kNormVec) {
            const uint32_t col = uint32_t(c);
            const uint32_t have = L.cols - col < kNormVec ? L.cols - col : kNormVec;
            float h[8], w[8];
            fold_part<T>(L.send, L.nranks, send_row + c * sizeof(T), have, h);
            if (residual) {
                float f[8];
                load_part<R>(residual + c * sizeof(R), have, f);
#pragma unroll
                for (int i = 0; i < 8; ++i) h[i] += f[i];
            }
            load_weight_part<T>(L.weight, L.weight32, col, have, w);
            if (sweep == 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum[0] = __builtin_fmaf(h[i], h[i], sum[0]);
                    if (Q8) top = Larger()(top, magnitude(h[i] * w[i]));
                }
                continue;
            }
            if (L.has_hidden)
                for (uint32_t d = 0; d < L.ndst; ++d)
                    store_part<R>(static_cast<char*>(L.hidden[first + d]) + uint64_t(at) * L.hidden_stride + c * sizeof(R), have, h, L.keep);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = h[i] * r * w[i];
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = clamp_to(y[i] * inverse, limit);
                u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
                if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
                for (uint32_t d = 0; d < L.ndst; ++d) {
                    char* p = static_cast<char*>(L.out[first + d]) + uint64_t(at) * L.out_stride + c;
                    if (have == kNormVec) {
                        store_codes(p, codes, L.keep);
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < kNormVec; ++i)
                            if (i < have) *as_global<uint8_t>(p + i) = uint8_t(codes[i / 4] >> (8 * (i % 4)));
                    }
                }
            } else {
                for (uint32_t d = 0; d < L.ndst; ++d)
                    store_part<T>(static_cast<char*>(L.out[first + d]) + uint64_t(at) * L.out_stride + c * sizeof(T), have, y, L.keep);
            }
        }
        if (sweep == 1) break;
        Reduce::run(shared, 0, sum, top);
        r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        if (Q8) {
            float amax = r * __builtin_bit_cast(float, top);
            if (amax < kAmaxMin) amax = kAmaxMin;
            finite = amax < __builtin_inff();
            inverse = limit / amax;
            if (threadIdx.x == 0) {
                const float scale = finite ? amax / limit : __builtin_nanf("");
                for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[first + d] + at)) = scale;
            }
        }
    }
}

template <typename T, typename R>
__global__ void __launch_bounds__(kLongLanes) rms_norm_backward_long_kernel(const NormBackLaunch L) {
    typedef RowReduce<kLongLanes, 2, false> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t group = blockIdx.x, first = group / L.part_groups;
    bool fresh = true;
    uint32_t slot = 0;
    for (uint32_t at = group - first * L.part_groups; at < L.part_rows; at += L.part_groups, slot ^= 1, fresh = false) {
        const uint64_t send_row = (uint64_t(first) * L.part_rows + at) * L.send_stride;
        const char* hidden = static_cast<const char*>(L.hidden[first]) + uint64_t(at) * L.hidden_stride;
        float sum[2] = {0.0f, 0.0f}, r = 0.0f, pull = 0.0f;
        for (uint32_t sweep = 0; sweep < 2; ++sweep) {
            for (uint64_t c = uint64_t(threadIdx.x) * kNormVec; c < L.cols; c += kLongLanes * kNormVec) {
                const uint32_t col = uint32_t(c);
                const uint32_t have = L.cols - col < kNormVec ? L.cols - col : kNormVec;
                float g[8], h[8], w[8];
                fold_part<T>(L.send, L.nranks, send_row + c * sizeof(T), have, g);
                load_part<R>(hidden + c * sizeof(R), have, h);
                load_weight_part<T>(L.weight, L.weight32, col, have, w);
                if (sweep == 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        sum[0] = __builtin_fmaf(h[i], h[i], sum[0]);
                        sum[1] = __builtin_fmaf(g[i] * w[i], h[i], sum[1]);
                    }
                    continue;
                }
                if (L.partial) {
                    char* share = reinterpret_cast<char*>(L.partial + uint64_t(group) * L.cols + c);
                    float dw[8] = {};
                    if (!fresh) load_part<float>(share, have, dw);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dw[i] = __builtin_fmaf(g[i], h[i] * r, dw[i]);
                    store_part<float>(share, have, dw, true);
                }
                float dh[8] = {};
                if (L.arriving[0])
                    load_part<R>(static_cast<const char*>(L.arriving[first]) + uint64_t(at) * L.arriving_stride + c * sizeof(R), have, dh);
#pragma unroll
                for (int i = 0; i < 8; ++i) dh[i] += __builtin_fmaf(-pull, h[i], r * (g[i] * w[i]));
                for (uint32_t d = 0; d < L.ndst; ++d) {
                    if (L.dhidden[0])
                        store_part<R>(static_cast<char*>(L.dhidden[first + d]) + uint64_t(at) * L.dhidden_stride + c * sizeof(R), have, dh, L.keep);
                    if (L.dsend[0])
                        store_part<T>(static_cast<char*>(L.dsend[first + d]) + uint64_t(at) * L.dsend_stride + c * sizeof(T), have, dh, L.keep);
                }
            }
            if (sweep == 1) break;
            uint32_t unused = 0;
            Reduce::run(shared, slot, sum, unused);
            r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
            pull = r * r * r * (sum[1] * (1.0f / float(L.cols)));
        }
    }
}

template <typename T, typename R, uint32_t Lanes, uint32_t Vecs>
NormKernels norm_kernels_of(bool q8) {
    return {q8 ? reinterpret_cast<const void*>(&rms_norm_kernel<T, R, true, Lanes, Vecs>)
               : reinterpret_cast<const void*>(&rms_norm_kernel<T, R, false, Lanes, Vecs>),
            reinterpret_cast<const void*>(&rms_norm_backward_kernel<T, R, Lanes, Vecs>)};
}

template <typename T, typename R>
NormKernels norm_kernels_for(NormVariant v, bool q8) {
    switch (v) {
        case kNormNarrow:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_narrow_kernel<T, R>)};
        case kNorm64x1: return norm_kernels_of<T, R, 64, 1>(q8);
        case kNorm64x2: return norm_kernels_of<T, R, 64, 2>(q8);
        case kNorm256x1: return norm_kernels_of<T, R, 256, 1>(q8);
        case kNorm256x2: return norm_kernels_of<T, R, 256, 2>(q8);
        case kNorm1024x1: return norm_kernels_of<T, R, 1024, 1>(q8);
        case kNorm1024x2: return norm_kernels_of<T, R, 1024, 2>(q8);
        case kNormLong:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_long_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_long_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_long_kernel<T, R>)};
    }
    return {nullptr, nullptr};
}

template <typename T>
NormKernels norm_kernels(NormVariant v, bool stream32, bool q8) {
    return stream32 ? norm_kernels_for<T, float>(v, q8) : norm_kernels_for<T, T>(v, q8);
}

}  // namespace detail
}  // namespace vrank
}  // namespace MegRay
