// Kernels of the norm behind a fold and of its backward (vrank_fused.h).  Per-type translation units
// (vrank_norm_<type>.hip) instantiate them.
//
// A row is one reduction: its lanes keep it in registers, `Vecs` vectors of eight elements each, so that everything
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

constexpr uint32_t kWaveRows = 4;  // rows of one wavefront go four to a workgroup

// Sums (and a maximum) over the lanes of a row, in a fixed order.  `slot` alternates between rows that follow each other in
// a workgroup: a wavefront may be a row ahead of the others, never two.
template <bool Wave, int Sums, bool Max>
struct RowReduce {
    struct Shared {
        float sum[2][Sums][Wave ? 1 : 16];
        uint32_t max[2][Max && !Wave ? 16 : 1];
    };
    static __device__ __forceinline__ void run(Shared& s, uint32_t waves, uint32_t slot, float (&sum)[Sums], uint32_t& max) {
#pragma unroll
        for (int i = 0; i < Sums; ++i) sum[i] = across_wave(sum[i], Plus());
        if (Max) max = across_wave(max, Larger());
        if constexpr (!Wave) {
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
                for (uint32_t w = 1; w < waves; ++w) sum[i] += s.sum[slot][i][w];
            }
            if (Max) {
                max = s.max[slot][0];
                for (uint32_t w = 1; w < waves; ++w) max = Larger()(max, s.max[slot][w]);
            }
        }
    }
};

// Which elements of a row a lane holds.
template <uint32_t Vecs>
struct RowPart {
    uint32_t col[Vecs];     // first element of vector k, never past cols - 8
    uint32_t repeat[Vecs];  // leading elements that belong to another lane (8 and more: all of them)
    __device__ __forceinline__ RowPart(uint32_t cols, uint32_t lanes, uint32_t lane) {
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            const uint32_t want = (k * lanes + lane) * kNormVec;
            col[k] = want + kNormVec <= cols ? want : cols - kNormVec;
            repeat[k] = want - col[k];
        }
    }
    __device__ __forceinline__ bool stores(uint32_t k) const { return repeat[k] < kNormVec; }
};

// Adds a row of `Ranks` consecutive ranks to `acc`, all loads issued before the first sum.  Not Whole: `left` of them are
// there, and the last one's loads are repeated, not added.
template <typename T, bool Lines, uint32_t Vecs, uint32_t Ranks, bool Whole>
__device__ __forceinline__ void fold_ranks(const void* const* send, uint64_t row_offset, uint32_t left,
                                           const uint32_t (&col)[Vecs], float (&acc)[Vecs][8]) {
    Raw8<T> x[Ranks][Vecs];
#pragma unroll
    for (uint32_t r = 0; r < Ranks; ++r) {
        const char* p = static_cast<const char*>(send[Whole || r < left ? r : left - 1]) + row_offset;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[r][k] = load8<T, Lines>(p + col[k] * uint32_t(sizeof(T)));
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

// The first `Ranks` ranks' part of a row, on its way.
template <typename T, bool Lines, uint32_t Vecs, uint32_t Ranks>
struct FirstRanks {
    Raw8<T> x[Ranks][Vecs];
    __device__ __forceinline__ void load(const void* const* send, uint32_t nranks, uint64_t row_offset, const uint32_t (&col)[Vecs]) {
#pragma unroll
        for (uint32_t r = 0; r < Ranks; ++r) {  // past the last rank: its buffer again, not added
            const char* p = static_cast<const char*>(send[r < nranks ? r : nranks - 1]) + row_offset;
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) x[r][k] = load8<T, Lines>(p + col[k] * uint32_t(sizeof(T)));
        }
    }
    // Adds them and the row's other ranks up.
    __device__ __forceinline__ void fold(const void* const* send, uint32_t nranks, uint64_t row_offset, const uint32_t (&col)[Vecs],
                                         float (&acc)[Vecs][8]) const {
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[k][i] = 0.0f;
#pragma unroll
        for (uint32_t r = 0; r < Ranks; ++r) {
            if (r < nranks) {
#pragma unroll
                for (uint32_t k = 0; k < Vecs; ++k) {
                    float f[8];
                    widen<T>(x[r][k], f);
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[k][i] += f[i];
                }
            }
        }
        uint32_t r = Ranks;
        for (; r + Ranks <= nranks; r += Ranks) fold_ranks<T, Lines, Vecs, Ranks, true>(send + r, row_offset, Ranks, col, acc);
        if (r < nranks) fold_ranks<T, Lines, Vecs, Ranks, false>(send + r, row_offset, nranks - r, col, acc);
    }
};

template <typename T, uint32_t Vecs>
__device__ __forceinline__ void load_weight(const void* weight, uint32_t weight32, const uint32_t (&col)[Vecs], float (&w)[Vecs][8]) {
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) {
        if (weight32) widen<float>(load8<float, false>(static_cast<const char*>(weight) + uint64_t(col[k]) * 4), w[k]);
        else widen<T>(load8<T, false>(static_cast<const char*>(weight) + uint64_t(col[k]) * sizeof(T)), w[k]);
    }
}

// A row of `ptr` (null: zeros), as it lies in memory.
template <typename R, bool Lines, uint32_t Vecs>
__device__ __forceinline__ void load_row(const void* ptr, uint64_t row_offset, const uint32_t (&col)[Vecs], Raw8<R> (&x)[Vecs]) {
    if (ptr) {
        const char* p = static_cast<const char*>(ptr) + row_offset;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[k] = load8<R, Lines>(p + col[k] * uint32_t(sizeof(R)));
    } else {
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[k] = Raw8<R>{};
    }
}

// Scale of a row whose largest |h * weight| is `top`, and 1 / scale; whether the row is finite (the scale is NaN if not).
__device__ __forceinline__ bool row_scale(float r, uint32_t top, uint32_t int8, float& scale, float& inverse) {
    float amax = r * __builtin_bit_cast(float, top);
    if (amax < kAmaxMin) amax = kAmaxMin;  // not true of a NaN
    scale = amax / (int8 ? kInt8Max : kE4m3Max);
    inverse = 1.0f / scale;
    if (amax < __builtin_inff()) return true;
    scale = __builtin_nanf("");
    return false;
}

// R: the residual stream's type.  Q8: 8-bit output with a scale per row.  Wave: a row is one wavefront's.  Lines: every row of every
// buffer begins on a cache line.
template <typename T, typename R, bool Q8, uint32_t Vecs, bool Wave, bool Lines, uint32_t Ranks>
__global__ void __launch_bounds__(Wave ? 64 * kWaveRows : 1024) rms_norm_kernel(const NormLaunch L) {
    typedef RowReduce<Wave, 1, Q8> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t lanes = Wave ? 64 : L.lanes, lane = Wave ? threadIdx.x % 64 : threadIdx.x;
    const uint32_t wave_row = Wave ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
    const RowPart<Vecs> part(L.cols, lanes, lane);
    float w[Vecs][8];
    load_weight<T, Vecs>(L.weight, L.weight32, part.col, w);

    // The next row's loads are issued before this one's stores: a workgroup that only stored would leave its share of the
    // reads idle.  Two vectors per lane leave no registers for that.
    constexpr bool kAhead = Vecs == 1;
    FirstRanks<T, Lines, Vecs, Ranks> ahead;
    Raw8<R> residual[Vecs];
    uint32_t row, first, at;
    auto find = [&](uint32_t position) -> bool {  // false: no such row (Wave: no barrier is missed)
        row = Wave ? L.deal.of(position) * kWaveRows + wave_row : L.deal.of(position);
        first = row / L.part_rows;  // destination (reduce_scatter); 0 (all_reduce)
        at = row - first * L.part_rows;
        return position < L.positions && row < L.rows;
    };
    auto fetch = [&] {
        load_row<R, Lines, Vecs>(L.residual[0] ? L.residual[first] : nullptr, uint64_t(at) * L.residual_stride, part.col, residual);
        ahead.load(L.send, L.nranks, uint64_t(row) * L.send_stride, part.col);
    };
    bool there = find(blockIdx.x);
    if (kAhead && there) fetch();
    uint32_t slot = 0;
    for (uint32_t position = blockIdx.x; there; slot ^= 1) {
        float h[Vecs][8];
        if (!kAhead) fetch();
        ahead.fold(L.send, L.nranks, uint64_t(row) * L.send_stride, part.col, h);
        float sum[1] = {0.0f};
        uint32_t top = 0;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            float f[8];
            widen<R>(residual[k], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[k][i] += f[i];
                sum[0] = __builtin_fmaf(h[k][i], uint32_t(i) >= part.repeat[k] ? h[k][i] : 0.0f, sum[0]);
                if (Q8) top = Larger()(top, magnitude(h[k][i] * w[k][i]));
            }
        }
        const uint32_t to = first, to_row = at;
        position += gridDim.x;
        there = find(position);
        if (kAhead && there) fetch();
        Reduce::run(shared, lanes / 64, slot, sum, top);
        const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);

        float scale = 0.0f, inverse = 0.0f;
        bool finite = true;
        if (Q8) {
            finite = row_scale(r, top, L.int8, scale, inverse);
            if (lane == 0)
                for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[to + d] + to_row)) = scale;
        }
        const uint64_t hidden_row = uint64_t(to_row) * L.hidden_stride, out_row = uint64_t(to_row) * L.out_stride;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            if (!part.stores(k)) continue;
            const Raw8<R> stored = narrow<R>(h[k]);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = h[k][i] * r * w[k][i];
            u32x2 codes = {0, 0};
            Raw8<T> result;
            if constexpr (Q8) {
                const float limit = L.int8 ? kInt8Max : kE4m3Max;
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = clamp_to(quotient(y[i], scale, inverse), limit);
                codes = L.int8 ? to_int8(y) : to_e4m3(y);
                if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
            } else {
                result = narrow<T>(y);
            }
            for (uint32_t d = 0; d < L.ndst; ++d) {
                if (L.has_hidden) {
                    store_row<R, Lines>(static_cast<char*>(L.hidden[to + d]) + hidden_row, part.col[k] * uint32_t(sizeof(R)), stored, L.keep);
                    L.pace.wait();
                }
                if constexpr (Q8)
                    store_row_codes<Lines>(static_cast<char*>(L.out[to + d]) + out_row, part.col[k], codes, L.keep);
                else
                    store_row<T, Lines>(static_cast<char*>(L.out[to + d]) + out_row, part.col[k] * uint32_t(sizeof(T)), result, L.keep);
                L.pace.wait();
            }
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
    float scale = 0.0f, inverse = 0.0f;
    bool finite = true;
    const float limit = L.int8 ? kInt8Max : kE4m3Max;
    if (Q8) {
        finite = row_scale(r, top, L.int8, scale, inverse);
        for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[first + d] + at)) = scale;
    }
    float y[8];
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) y[c] = h[c] * r * w[c];
    if (Q8) {
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c) y[c] = clamp_to(quotient(y[c], scale, inverse), limit);
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
template <typename T, typename R, uint32_t Vecs, bool Wave, bool Lines, uint32_t Ranks>
__global__ void __launch_bounds__(Wave ? 64 * kWaveRows : 1024) rms_norm_backward_kernel(const NormBackLaunch L) {
    typedef RowReduce<Wave, 2, false> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t lanes = Wave ? 64 : L.lanes, lane = Wave ? threadIdx.x % 64 : threadIdx.x;
    const uint32_t group = Wave ? blockIdx.x * kWaveRows + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : blockIdx.x;
    if (Wave && group >= L.groups) return;
    const RowPart<Vecs> part(L.cols, lanes, lane);
    const uint32_t first = group / L.part_groups;  // the destination whose rows these are (reduce_scatter); 0 (all_reduce)
    float w[Vecs][8], dw[Vecs][8];
    load_weight<T, Vecs>(L.weight, L.weight32, part.col, w);
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[k][i] = 0.0f;
    const float mean = 1.0f / float(L.cols);
    const void* const arriving_part = L.arriving[0] ? L.arriving[first] : nullptr;

    // As in the forward kernel the next row's loads are issued before this one's stores; two vectors per lane leave
    // no registers for that.
    constexpr bool kAhead = Vecs == 1;
    FirstRanks<T, Lines, Vecs, Ranks> ahead;
    constexpr bool kArrivingAhead = kAhead && sizeof(R) == 2;
    Raw8<R> hidden[Vecs], arriving[Vecs], arriving_ahead[Vecs];
    auto send_row = [&](uint32_t at) { return (uint64_t(first) * L.part_rows + at) * L.send_stride; };
    auto fetch = [&](uint32_t at) {
        load_row<R, Lines, Vecs>(L.hidden[first], uint64_t(at) * L.hidden_stride, part.col, hidden);
        if (kArrivingAhead) load_row<R, Lines, Vecs>(arriving_part, uint64_t(at) * L.arriving_stride, part.col, arriving_ahead);
        ahead.load(L.send, L.nranks, send_row(at), part.col);
    };
    uint32_t slot = 0, position = group - first * L.part_groups, next = L.deal.of(position);
    if (kAhead) fetch(next);
    for (; position < L.part_rows; slot ^= 1) {
        const uint32_t at = next;
        float g[Vecs][8], h[Vecs][8];
        if (!kAhead) fetch(at);
        ahead.fold(L.send, L.nranks, send_row(at), part.col, g);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            widen<R>(hidden[k], h[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float mine = uint32_t(i) >= part.repeat[k] ? h[k][i] : 0.0f;
                sum[0] = __builtin_fmaf(h[k][i], mine, sum[0]);
                sum[1] = __builtin_fmaf(g[k][i] * w[k][i], mine, sum[1]);
            }
        }
        if constexpr (kArrivingAhead) {
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) arriving[k] = arriving_ahead[k];
        } else {
            load_row<R, Lines, Vecs>(arriving_part, uint64_t(at) * L.arriving_stride, part.col, arriving);
        }
        position += L.part_groups;
        next = L.deal.of(position);
        if (kAhead && position < L.part_rows) fetch(next);
        uint32_t unused = 0;
        Reduce::run(shared, lanes / 64, slot, sum, unused);
        const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        const float pull = r * r * r * (sum[1] * mean);
        const uint64_t dhidden_row = uint64_t(at) * L.dhidden_stride, dsend_row = uint64_t(at) * L.dsend_stride;
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
            const Raw8<R> wide = narrow<R>(dh);
            const Raw8<T> slim = narrow<T>(dh);
            for (uint32_t d = 0; d < L.ndst; ++d) {
                if (L.dhidden[0]) {
                    store_row<R, Lines>(static_cast<char*>(L.dhidden[first + d]) + dhidden_row, part.col[k] * uint32_t(sizeof(R)), wide, L.keep);
                }
                if (L.dsend[0]) {
                    store_row<T, Lines>(static_cast<char*>(L.dsend[first + d]) + dsend_row, part.col[k] * uint32_t(sizeof(T)), slim, L.keep);
                }
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
    typedef RowReduce<false, 1, Q8> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t row = blockIdx.x;
    const uint32_t first = row / L.part_rows, at = row - first * L.part_rows;
    const uint64_t send_row = uint64_t(row) * L.send_stride;
    const char* residual = L.residual[0] ? static_cast<const char*>(L.residual[first]) + uint64_t(at) * L.residual_stride : nullptr;
    float sum[1] = {0.0f};
    uint32_t top = 0;
    float r = 0.0f, scale = 0.0f, inverse = 0.0f;
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
                for (int i = 0; i < 8; ++i) y[i] = clamp_to(quotient(y[i], scale, inverse), limit);
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
        Reduce::run(shared, kLongLanes / 64, 0, sum, top);
        r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        if (Q8) {
            finite = row_scale(r, top, L.int8, scale, inverse);
            if (threadIdx.x == 0)
                for (uint32_t d = 0; d < L.ndst; ++d) *as_global<float>(reinterpret_cast<char*>(L.scales[first + d] + at)) = scale;
        }
    }
}

template <typename T, typename R>
__global__ void __launch_bounds__(kLongLanes) rms_norm_backward_long_kernel(const NormBackLaunch L) {
    typedef RowReduce<false, 2, false> Reduce;
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
            Reduce::run(shared, kLongLanes / 64, slot, sum, unused);
            r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
            pull = r * r * r * (sum[1] * (1.0f / float(L.cols)));
        }
    }
}

// Ranks: how many ranks' loads are in flight together (past it, the others follow in groups of as many).  Loads of a buffer that
// is not there are repeats of the last one's and cost issue slots, and registers cost wavefronts: so no more than there are.
template <typename T, typename R, uint32_t Vecs, bool Wave, bool Lines, uint32_t Ranks, uint32_t BackRanks>
NormKernels norm_kernels_of(bool q8) {
    return {q8 ? reinterpret_cast<const void*>(&rms_norm_kernel<T, R, true, Vecs, Wave, Lines, Ranks>)
               : reinterpret_cast<const void*>(&rms_norm_kernel<T, R, false, Vecs, Wave, Lines, Ranks>),
            reinterpret_cast<const void*>(&rms_norm_backward_kernel<T, R, Vecs, Wave, Lines, BackRanks>)};
}

template <typename T, typename R, bool Wave, bool Lines>
NormKernels norm_kernels_ranks(uint32_t nranks, bool q8) {
    constexpr uint32_t kMost = sizeof(T) == 4 ? 4 : 8;  // eight 16-byte loads
    if (nranks <= 2) return norm_kernels_of<T, R, 1, Wave, Lines, 2, 2>(q8);
    if (nranks <= 4) return norm_kernels_of<T, R, 1, Wave, Lines, 4, 4>(q8);
    return norm_kernels_of<T, R, 1, Wave, Lines, kMost, kMost>(q8);
}

template <typename T, typename R, bool Lines>
NormKernels norm_kernels_lines(NormVariant v, uint32_t nranks, bool q8) {
    if (v == kNormWave) return norm_kernels_ranks<T, R, true, Lines>(nranks, q8);
    if (v == kNormBlock) return norm_kernels_ranks<T, R, false, Lines>(nranks, q8);
    return norm_kernels_of<T, R, 2, false, Lines, sizeof(T) == 4 ? 2 : 4, sizeof(T) == 4 ? 1 : 3>(q8);
}

template <typename T, typename R>
NormKernels norm_kernels_for(NormVariant v, uint32_t nranks, bool lines, bool q8) {
    switch (v) {
        case kNormNarrow:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_narrow_kernel<T, R>)};
        case kNormWave:
        case kNormBlock:
        case kNormBlock2: return lines ? norm_kernels_lines<T, R, true>(v, nranks, q8) : norm_kernels_lines<T, R, false>(v, nranks, q8);
        case kNormLong:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_long_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_long_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_long_kernel<T, R>)};
    }
    return {nullptr, nullptr};
}

}  // namespace detail
}  // namespace vrank
}  // namespace MegRay
