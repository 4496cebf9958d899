// Kernels of the norm behind a fold and of its backward (vrank_fused.h).  Per-type translation units
// (vrank_norm_<type>.hip) instantiate them.
//
// A row is one reduction: its lanes keep it in registers, `Vecs` vectors of eight elements each, so that everything
// is read once: N partial rows are summed as they arrive, the residual is added, the sum of squares (and, for 8-bit
// outputs, the largest |h * weight|, which times 1 / rms is the largest |y|) goes once across the lanes, and the row is
// stored to every destination from the registers.  The bound is HBM: two to four bytes of traffic per operation.
//
// A row whose length is no multiple of eight ends in a vector that is moved back to end with the row: the lane that owns
// it repeats up to seven elements of its neighbour, leaves them out of the sums, and stores the same values.  Where all loads of a
// row come before the reduction and all its stores behind it, outputs that take an input's place are safe with that too.  Two kernels load
// behind the reduction.  The backward with two vectors per lane reads the arriving gradient between its stores: it may not be replaced
// where rows end inside a vector (NormPlan::plan_backward takes the sweep there).  The kernels that sweep a row twice read it again
// as they store it: they move no vector back, and each element is read and stored by one lane alone.
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
                const float part = s.sum[slot][i][threadIdx.x % 16];  // anything, where there is no such wavefront
                sum[i] = across_row(threadIdx.x % 16 < waves ? part : 0.0f, Plus());
            }
            if (Max) {
                const uint32_t part = s.max[slot][threadIdx.x % 16];
                max = across_row(threadIdx.x % 16 < waves ? part : 0u, Larger());
            }
        }
    }
};

// Which elements of a row a lane holds: `Vecs` times one piece of eight, or two of four (Split: where a 32-bit type takes part, see Raw8).
// A piece that would pass the row's end is moved back to end with it.
template <uint32_t Vecs, bool Split>
struct RowPart {
    static constexpr uint32_t kPieces = Split ? 2 : 1, kWidth = kNormVec / kPieces;
    uint32_t col[Vecs][kPieces];     // first element, never past cols - kWidth
    uint32_t repeat[Vecs][kPieces];  // leading elements that belong to another lane (kWidth and more: all of them)
    __device__ __forceinline__ RowPart(uint32_t cols, uint32_t lanes, uint32_t lane) {
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
#pragma unroll
            for (uint32_t p = 0; p < kPieces; ++p) {
                const uint32_t first = Split ? (lane / 64 * 2 + p) * 64 + lane % 64 : lane;
                const uint32_t want = k * lanes * kNormVec + first * kWidth;
                col[k][p] = want + kWidth <= cols ? want : cols - kWidth;
                repeat[k][p] = want - col[k][p];
            }
        }
    }
    __device__ __forceinline__ bool mine(uint32_t k, uint32_t element) const {
        return element % kWidth >= repeat[k][element / kWidth];
    }
    // element vector k of the row at `row`
    template <typename T, bool Once>
    __device__ __forceinline__ Raw8<T> load(ConstBytes row, uint32_t k) const {
        if constexpr (Split) return load44<T, Once>(row + col[k][0] * uint32_t(sizeof(T)), row + col[k][kPieces - 1] * uint32_t(sizeof(T)));
        else return load8<T, Once>(row + col[k][0] * uint32_t(sizeof(T)));
    }
    // `w`: the vector's eight elements, `Size` bytes each.  Lines: a buffer store, whose offset has to be a multiple of four - that of a piece
    // that is moved back, too, which is why the row has to end on one.
    template <uint32_t Size, bool Lines>
    __device__ __forceinline__ void store(Bytes row, uint32_t k, const uint32_t* w, bool keep) const {
#pragma unroll
        for (uint32_t p = 0; p < kPieces; ++p)
            if (repeat[k][p] < kWidth) store_dwords<kWidth * Size, Lines, Size>(row, col[k][p] * Size, w + p * kWidth * Size / 4, keep);
    }
};

// Adds a row of `Ranks` consecutive ranks to `acc`, all loads issued before the first sum.  Not Whole: `left` of them are
// there, and the last one's loads are repeated, not added.
template <typename T, bool Lines, uint32_t Vecs, uint32_t Ranks, bool Whole, typename Part>
__device__ __forceinline__ void fold_ranks(const LaneTable& table, uint32_t from, uint64_t row_offset, uint32_t left, const Part& part,
                                           float (&acc)[Vecs][8]) {
    Raw8<T> x[Ranks][Vecs];
#pragma unroll
    for (uint32_t r = 0; r < Ranks; ++r) {
        const ConstBytes p = table.first(from + (Whole || r < left ? r : left - 1)) + row_offset;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[r][k] = part.template load<T, Lines>(p, k);
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
    template <typename Part>
    __device__ __forceinline__ void load(const LaneTable& table, uint32_t nranks, uint64_t row_offset, const Part& part) {
#pragma unroll
        for (uint32_t r = 0; r < Ranks; ++r) {  // past the last rank: its buffer again, not added
            const ConstBytes p = table.first(r < nranks ? r : nranks - 1) + row_offset;
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) x[r][k] = part.template load<T, Lines>(p, k);
        }
    }
    // Adds them and the row's other ranks up.
    template <typename Part>
    __device__ __forceinline__ void fold(const LaneTable& table, uint32_t nranks, uint64_t row_offset, const Part& part,
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
        for (; r + Ranks <= nranks; r += Ranks) fold_ranks<T, Lines, Vecs, Ranks, true>(table, r, row_offset, Ranks, part, acc);
        if (r < nranks) fold_ranks<T, Lines, Vecs, Ranks, false>(table, r, row_offset, nranks - r, part, acc);
    }
};

template <typename T, typename Part>
__device__ __forceinline__ void load_weight(const void* weight, uint32_t weight32, const Part& part, uint32_t k, float (&w)[8]) {
    if (weight32) widen<float>(part.template load<float, false>(bytes_of(weight), k), w);
    else widen<T>(part.template load<T, false>(bytes_of(weight), k), w);
}

// A row of `ptr` (null: zeros), as it lies in memory.
template <typename R, bool Lines, uint32_t Vecs, typename Part>
__device__ __forceinline__ void load_row(ConstBytes ptr, uint64_t row_offset, const Part& part, Raw8<R> (&x)[Vecs]) {
    if (ptr) {
        const ConstBytes p = ptr + row_offset;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[k] = part.template load<R, Lines>(p, k);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) x[k] = Raw8<R>{};
    }
}

// Scale of a row whose largest |h * weight| is `top`, and 1 / scale; whether the row is finite (the scale is NaN if not).
__device__ __forceinline__ bool row_scale(float r, uint32_t top, uint32_t int8, float& scale, float& inverse) {
    float amax = r * __builtin_bit_cast(float, top);
    if (amax < kAmaxMin) amax = kAmaxMin;  // not true of a NaN
    scale = amax * (int8 ? 1.0f / kInt8Max : 1.0f / kE4m3Max);
    inverse = 1.0f / scale;
    if (amax < __builtin_inff()) return true;
    scale = __builtin_nanf("");
    return false;
}

// R: the residual stream's type.  Q8: 8-bit output with a scale per row.  Wave: a row is one wavefront's.  Lines: every row of every
// buffer begins on a cache line, and every stored row ends on a 4-byte boundary.
template <typename T, typename R, bool Q8, uint32_t Vecs, bool Wave, bool Lines, uint32_t Ranks>
__global__ void __launch_bounds__(Wave ? 64 * kWaveRows : 1024, 4) rms_norm_kernel(const NormLaunch L) {
    typedef RowReduce<Wave, 1, Q8> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t lanes = Wave ? 64 : L.lanes, lane = Wave ? threadIdx.x % 64 : threadIdx.x;
    const uint32_t wave_row = Wave ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0;
    const LaneTable sends(offsetof(NormLaunch, send)), results(offsetof(NormLaunch, out));  // and hidden states; and scales
    const RowPart<Vecs, sizeof(T) == 4 || sizeof(R) == 4> part(L.cols, lanes, lane);
    float w[Vecs][8];
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) load_weight<T>(L.weight, L.weight32, part, k, w[k]);

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
        load_row<R, Lines, Vecs>(bytes_of(L.residual[0] ? L.residual[first] : nullptr), uint64_t(at) * L.residual_stride, part, residual);
        ahead.load(sends, L.nranks, uint64_t(row) * L.send_stride, part);
    };
    // destinations of this workgroup
    const uint32_t split = Wave || L.splits == 1 ? 0 : blockIdx.x % L.splits, start = Wave || L.splits == 1 ? blockIdx.x : blockIdx.x / L.splits;
    const uint32_t dst = L.ndst * split / L.splits, dst_end = L.ndst * (split + 1) / L.splits;
    bool there = find(start);
    if (kAhead && there) fetch();
    uint32_t slot = 0;
    for (uint32_t position = start; there; slot ^= 1) {
        float h[Vecs][8];
        if (!kAhead) fetch();
        ahead.fold(sends, L.nranks, uint64_t(row) * L.send_stride, part, h);
        float sum[1] = {0.0f};
        uint32_t top = 0;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            float f[8];
            widen<R>(residual[k], f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                h[k][i] += f[i];
                sum[0] = __builtin_fmaf(h[k][i], part.mine(k, uint32_t(i)) ? h[k][i] : 0.0f, sum[0]);
                if (Q8) top = Larger()(top, magnitude(h[k][i] * w[k][i]));
            }
        }
        const uint32_t to = first, to_row = at;
        position += gridDim.x;  // a launch with split rows has a workgroup for each
        there = find(position);
        if (kAhead && there) fetch();
        Reduce::run(shared, lanes / 64, slot, sum, top);
        const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);

        float scale = 0.0f, inverse = 0.0f;
        bool finite = true;
        if (Q8) {
            finite = row_scale(r, top, L.int8, scale, inverse);
            for (uint32_t d = dst; d < dst_end; ++d)
                if (lane == 0) *(MRV_GLOBAL float*)(results.second(to + d) + uint64_t(to_row) * 4) = scale;
        }
        const uint64_t hidden_row = uint64_t(to_row) * L.hidden_stride, out_row = uint64_t(to_row) * L.out_stride;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            const Raw8<R> stored = narrow<R>(h[k]);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = h[k][i] * r * w[k][i];
            Raw8<T> result;
            if constexpr (Q8) {
                const float limit = L.int8 ? kInt8Max : kE4m3Max;
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = clamp_to(quotient(y[i], scale, inverse), limit);
                u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
                if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
                result.w[0] = codes[0], result.w[1] = codes[1];
            } else {
                result = narrow<T>(y);
            }
            for (uint32_t d = dst; d < dst_end; ++d) {
                if (L.has_hidden) {
                    part.template store<sizeof(R), Lines>(sends.second(to + d) + hidden_row, k, stored.w, L.keep);
                    L.pace.wait();
                }
                part.template store<Q8 ? 1 : sizeof(T), Lines>(results.first(to + d) + out_row, k, result.w, L.keep);
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
                h[c] += load_one<T>(bytes_of(L.send[k]) + uint64_t(row) * L.send_stride + c * sizeof(T));
            if (L.residual[0])
                h[c] += load_one<R>(bytes_of(L.residual[first]) + uint64_t(at) * L.residual_stride + c * sizeof(R));
            const ConstBytes p = bytes_of(L.weight);
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
        for (uint32_t d = 0; d < L.ndst; ++d) L.scales[first + d][at] = scale;
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
                    *(MRV_GLOBAL uint8_t*)(bytes_of(L.out[first + d]) + uint64_t(at) * L.out_stride + c) =
                            uint8_t(codes[c / 4] >> (8 * (c % 4)));
    }
#pragma unroll
    for (uint32_t c = 0; c < kNormVec; ++c) {
        if (c >= L.cols) continue;
        for (uint32_t d = 0; d < L.ndst; ++d) {
            if (L.has_hidden)
                store_one<R>(bytes_of(L.hidden[first + d]) + uint64_t(at) * L.hidden_stride + c * sizeof(R), h[c]);
            if (!Q8) store_one<T>(bytes_of(L.out[first + d]) + uint64_t(at) * L.out_stride + c * sizeof(T), y[c]);
        }
    }
}

// Backward.  A row group (the lanes of one row) walks the rows of one part, `part_groups` apart, and carries its columns'
// share of the weight's gradient in registers; the shares meet in `partial`, and norm_weight_kernel adds them in order.
// dh is formed as r * (g * w - h * pull), pull = r * (r * mean(g * w * h)): pull is of dh's size and h * pull of g * w's, so neither leaves the
// range of 32 bits before dh does; r^3 would, from rows of 1e13 on and below 1e-13.
template <typename T, typename R, uint32_t Vecs, bool Wave, bool Lines, uint32_t Ranks>
__global__ void __launch_bounds__(Wave ? 64 * kWaveRows : 1024, 4) rms_norm_backward_kernel(const NormBackLaunch L) {
    typedef RowReduce<Wave, 2, false> Reduce;
    __shared__ typename Reduce::Shared shared;
    const uint32_t lanes = Wave ? 64 : L.lanes, lane = Wave ? threadIdx.x % 64 : threadIdx.x;
    const uint32_t group = Wave ? blockIdx.x * kWaveRows + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : blockIdx.x;
    if (Wave && group >= L.groups) return;
    const LaneTable sends(offsetof(NormBackLaunch, send)), others(offsetof(NormBackLaunch, dsend));  // and dhidden; and hidden
    // two of four of a 16-bit type only where that keeps whole lines whole: 3 ranks' 1365 x 5001 BF16 with a 32-bit stream 84 us
    // with pieces of eight, 100 with two of four (the same rows of one rank: 67 and 64)
    const RowPart<Vecs, sizeof(T) == 4 || (sizeof(R) == 4 && Lines)> part(L.cols, lanes, lane);
    const uint32_t first = group / L.part_groups;  // the destination whose rows these are (reduce_scatter); 0 (all_reduce)
    constexpr bool kAhead = Vecs == 1;
    float w[Vecs][8], dw[Vecs][8];
#pragma unroll
    for (uint32_t k = 0; k < Vecs; ++k) {
        if (kAhead) load_weight<T>(L.weight, L.weight32, part, k, w[k]);
#pragma unroll
        for (int i = 0; i < 8; ++i) dw[k][i] = 0.0f;
    }
    const float mean = 1.0f / float(L.cols);
    const ConstBytes arriving_part = bytes_of(L.arriving[0] ? L.arriving[first] : nullptr);

    // As in the forward kernel the next row's loads are issued before this one's stores; two vectors per lane leave
    // no registers for that, nor for the weight and the arriving gradient, which are read where they are used: the gradient may not be
    // replaced then where a lane repeats elements of another, which may be stored by that time (NormPlan::plan_backward).
    FirstRanks<T, Lines, Vecs, Ranks> ahead;
    constexpr bool kArrivingAhead = kAhead && sizeof(R) == 2 && Ranks < 8;
    Raw8<R> hidden[Vecs], arriving[Vecs], arriving_ahead[Vecs];
    auto send_row = [&](uint32_t at) { return (uint64_t(first) * L.part_rows + at) * L.send_stride; };
    auto fetch = [&](uint32_t at) {
        load_row<R, Lines, Vecs>(others.second(first), uint64_t(at) * L.hidden_stride, part, hidden);
        if (kArrivingAhead) load_row<R, Lines, Vecs>(arriving_part, uint64_t(at) * L.arriving_stride, part, arriving_ahead);
        ahead.load(sends, L.nranks, send_row(at), part);
    };
    uint32_t slot = 0, position = group - first * L.part_groups, next = L.deal.of(position);
    if (kAhead) fetch(next);
    for (; position < L.part_rows; slot ^= 1) {
        const uint32_t at = next;
        float g[Vecs][8], h[Vecs][8];
        if (!kAhead) fetch(at);
        ahead.fold(sends, L.nranks, send_row(at), part, g);
        float sum[2] = {0.0f, 0.0f};
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            widen<R>(hidden[k], h[k]);
            if (!kAhead) load_weight<T>(L.weight, L.weight32, part, k, w[k]);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float mine = part.mine(k, uint32_t(i)) ? h[k][i] : 0.0f;
                sum[0] = __builtin_fmaf(h[k][i], mine, sum[0]);
                sum[1] = __builtin_fmaf(g[k][i] * w[k][i], mine, sum[1]);
            }
        }
        if constexpr (kArrivingAhead) {
#pragma unroll
            for (uint32_t k = 0; k < Vecs; ++k) arriving[k] = arriving_ahead[k];
        } else if constexpr (kAhead) {
            load_row<R, Lines, Vecs>(arriving_part, uint64_t(at) * L.arriving_stride, part, arriving);
        }
        position += L.part_groups;
        next = L.deal.of(position);
        if (kAhead && position < L.part_rows) fetch(next);
        uint32_t unused = 0;
        Reduce::run(shared, lanes / 64, slot, sum, unused);
        const float r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        const float pull = r * (r * (sum[1] * mean));
        const uint64_t dhidden_row = uint64_t(at) * L.dhidden_stride, dsend_row = uint64_t(at) * L.dsend_stride;
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) {
            float dh[8];
            if (!kAhead) load_weight<T>(L.weight, L.weight32, part, k, w[k]);
            if constexpr (kAhead) widen<R>(arriving[k], dh);
            else widen<R>(arriving_part ? part.template load<R, Lines>(arriving_part + uint64_t(at) * L.arriving_stride, k) : Raw8<R>{}, dh);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                dh[i] = __builtin_fmaf(r, __builtin_fmaf(-pull, h[k][i], g[k][i] * w[k][i]), dh[i]);
                dw[k][i] = __builtin_fmaf(g[k][i], h[k][i] * r, dw[k][i]);
            }
            const Raw8<R> wide = narrow<R>(dh);
            const Raw8<T> slim = narrow<T>(dh);
            for (uint32_t d = 0; d < L.ndst; ++d) {
                if (L.dhidden[0]) {
                    part.template store<sizeof(R), Lines>(sends.second(first + d) + dhidden_row, k, wide.w, L.keep);
                }
                if (L.dsend[0]) {
                    part.template store<sizeof(T), Lines>(others.first(first + d) + dsend_row, k, slim.w, L.keep);
                }
            }
        }
    }
    if (L.partial) {
        const Bytes p = bytes_of(L.partial + uint64_t(group) * L.cols);
#pragma unroll
        for (uint32_t k = 0; k < Vecs; ++k) part.template store<4, false>(p, k, narrow<float>(dw[k]).w, true);
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
        const ConstBytes p = bytes_of(L.weight);
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
                    g[c] += load_one<T>(bytes_of(L.send[k]) + row * L.send_stride + c * sizeof(T));
                h[c] = load_one<R>(bytes_of(L.hidden[first]) + uint64_t(at) * L.hidden_stride + c * sizeof(R));
                if (L.arriving[0])
                    a[c] = load_one<R>(bytes_of(L.arriving[first]) + uint64_t(at) * L.arriving_stride + c * sizeof(R));
            }
            square = __builtin_fmaf(h[c], h[c], square);
            inner = __builtin_fmaf(g[c] * w[c], h[c], inner);
        }
        const float r = 1.0f / __builtin_sqrtf(square / float(L.cols) + L.eps);
        const float pull = r * (r * (inner * (1.0f / float(L.cols))));
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c) {
            if (c >= L.cols) continue;
            const float dh = __builtin_fmaf(r, __builtin_fmaf(-pull, h[c], g[c] * w[c]), a[c]);
            dw[c] = __builtin_fmaf(g[c], h[c] * r, dw[c]);
            for (uint32_t d = 0; d < L.ndst; ++d) {
                if (L.dhidden[0])
                    store_one<R>(bytes_of(L.dhidden[first + d]) + uint64_t(at) * L.dhidden_stride + c * sizeof(R), dh);
                if (L.dsend[0])
                    store_one<T>(bytes_of(L.dsend[first + d]) + uint64_t(at) * L.dsend_stride + c * sizeof(T), dh);
            }
        }
    }
    if (L.partial) {
#pragma unroll
        for (uint32_t c = 0; c < kNormVec; ++c)
            if (c < L.cols) L.partial[uint64_t(group) * L.cols + c] = dw[c];
    }
}

// The fold of a lane's eight elements, for lanes whose rows differ.
template <typename T, typename Part>
__device__ __forceinline__ void short_fold(const void* const* send, uint32_t nranks, uint64_t row_offset, const Part& part, float (&acc)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
#pragma unroll 8
    for (uint32_t k = 0; k < nranks; ++k) {
        float f[8];
        widen<T>(part.template load<T, false>(bytes_of(send[k]) + row_offset, 0), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += f[i];
    }
}

// Rows of up to 128 elements: sixteen lanes each, one row after the other in memory to a wavefront's four groups of lanes.  A wavefront for
// such a row would leave three quarters of its lanes idle.
constexpr uint32_t kShortLanes = 16;
constexpr uint32_t kShortRows = 256 / kShortLanes;  // of a workgroup

template <typename T, typename R, bool Q8>
__global__ void __launch_bounds__(256) rms_norm_short_kernel(const NormLaunch L) {
    const uint32_t lane = threadIdx.x % kShortLanes, row = L.deal.of(blockIdx.x) * kShortRows + threadIdx.x / kShortLanes;
    if (row >= L.rows) return;  // all of a row's lanes or none
    const uint32_t first = row / L.part_rows, at = row - first * L.part_rows;
    const RowPart<1, false> part(L.cols, kShortLanes, lane);
    float h[8], w[8], f[8];
    Raw8<R> residual[1];
    load_weight<T>(L.weight, L.weight32, part, 0, w);
    load_row<R, false, 1>(bytes_of(L.residual[0] ? L.residual[first] : nullptr), uint64_t(at) * L.residual_stride, part, residual);
    short_fold<T>(L.send, L.nranks, uint64_t(row) * L.send_stride, part, h);
    widen<R>(residual[0], f);
    float sum = 0.0f;
    uint32_t top = 0;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        h[i] += f[i];
        if (!part.mine(0, i)) continue;  // and lanes behind the row's end have none
        sum = __builtin_fmaf(h[i], h[i], sum);
        if (Q8) top = Larger()(top, magnitude(h[i] * w[i]));
    }
    sum = across_row(sum, Plus());
    if (Q8) top = across_row(top, Larger());
    const float r = 1.0f / __builtin_sqrtf(sum / float(L.cols) + L.eps);
    float scale = 0.0f, inverse = 0.0f;
    bool finite = true;
    if (Q8) {
        finite = row_scale(r, top, L.int8, scale, inverse);
        if (lane == 0)
            for (uint32_t d = 0; d < L.ndst; ++d) *(MRV_GLOBAL float*)(bytes_of(L.scales[first + d]) + uint64_t(at) * 4) = scale;
    }
    const Raw8<R> stored = narrow<R>(h);
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = h[i] * r * w[i];
    Raw8<T> result;
    if constexpr (Q8) {
        const float limit = L.int8 ? kInt8Max : kE4m3Max;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = clamp_to(quotient(y[i], scale, inverse), limit);
        u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
        if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
        result.w[0] = codes[0], result.w[1] = codes[1];
    } else {
        result = narrow<T>(y);
    }
    for (uint32_t d = 0; d < L.ndst; ++d) {
        if (L.has_hidden) part.template store<sizeof(R), false>(bytes_of(L.hidden[first + d]) + uint64_t(at) * L.hidden_stride, 0, stored.w, true);
        part.template store<Q8 ? 1 : sizeof(T), false>(bytes_of(L.out[first + d]) + uint64_t(at) * L.out_stride, 0, result.w, true);
    }
}

// Backward of rows of 8 * Lanes elements (16 or 32 lanes): a workgroup is a row group, whose rows at a time add their shares of the weight's
// gradient up in LDS at the end.
template <typename T, typename R, uint32_t Lanes>
__global__ void __launch_bounds__(256) rms_norm_backward_short_kernel(const NormBackLaunch L) {
    constexpr uint32_t kRows = 256 / Lanes;
    __shared__ float share[kRows][Lanes * kNormVec];
    const uint32_t lane = threadIdx.x % Lanes, slot = threadIdx.x / Lanes;
    const uint32_t first = blockIdx.x / L.part_groups;
    const RowPart<1, false> part(L.cols, Lanes, lane);
    float w[8], dw[8];
    load_weight<T>(L.weight, L.weight32, part, 0, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[i] = 0.0f;
    const ConstBytes hidden_part = bytes_of(L.hidden[first]), arriving_part = bytes_of(L.arriving[0] ? L.arriving[first] : nullptr);
    for (uint32_t at = (blockIdx.x - first * L.part_groups) * kRows + slot; at < L.part_rows; at += L.part_groups * kRows) {
        float g[8], h[8], dh[8];
        Raw8<R> hidden[1], arriving[1];
        load_row<R, false, 1>(hidden_part, uint64_t(at) * L.hidden_stride, part, hidden);
        load_row<R, false, 1>(arriving_part, uint64_t(at) * L.arriving_stride, part, arriving);
        short_fold<T>(L.send, L.nranks, (uint64_t(first) * L.part_rows + at) * L.send_stride, part, g);
        widen<R>(hidden[0], h);
        widen<R>(arriving[0], dh);
        float square = 0.0f, inner = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
            if (!part.mine(0, i)) continue;
            square = __builtin_fmaf(h[i], h[i], square);
            inner = __builtin_fmaf(g[i] * w[i], h[i], inner);
        }
        square = across_row(square, Plus());
        inner = across_row(inner, Plus());
        if (Lanes == 32) {
            square += __shfl_xor(square, 16, 64);
            inner += __shfl_xor(inner, 16, 64);
        }
        const float r = 1.0f / __builtin_sqrtf(square / float(L.cols) + L.eps);
        const float pull = r * (r * (inner * (1.0f / float(L.cols))));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            dh[i] = __builtin_fmaf(r, __builtin_fmaf(-pull, h[i], g[i] * w[i]), dh[i]);
            dw[i] = __builtin_fmaf(g[i], h[i] * r, dw[i]);
        }
        const Raw8<R> wide = narrow<R>(dh);
        const Raw8<T> slim = narrow<T>(dh);
        for (uint32_t d = 0; d < L.ndst; ++d) {
            if (L.dhidden[0]) part.template store<sizeof(R), false>(bytes_of(L.dhidden[first + d]) + uint64_t(at) * L.dhidden_stride, 0, wide.w, true);
            if (L.dsend[0]) part.template store<sizeof(T), false>(bytes_of(L.dsend[first + d]) + uint64_t(at) * L.dsend_stride, 0, slim.w, true);
        }
    }
    if (!L.partial) return;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (part.mine(0, i)) share[slot][part.col[0][0] + i] = dw[i];
    __syncthreads();
    if (threadIdx.x >= L.cols) return;
    float sum = share[0][threadIdx.x];
#pragma unroll
    for (uint32_t s = 1; s < kRows; ++s) sum += share[s][threadIdx.x];
    L.partial[uint64_t(blockIdx.x) * L.cols + threadIdx.x] = sum;
}

// Rows longer than the widest variant holds: the lanes sweep the row twice, the second time over data that the last-level
// cache mostly still has.  The vector at the row's end is taken element by element, so no element is read after another
// lane may have replaced it.
constexpr uint32_t kLongLanes = 1024;

template <typename T>
__device__ __forceinline__ void load_weight_part(const void* weight, uint32_t weight32, uint32_t col, uint32_t have, float (&w)[8]) {
    if (weight32) load_part<float>(bytes_of(weight) + uint64_t(col) * 4, have, w);
    else load_part<T>(bytes_of(weight) + uint64_t(col) * sizeof(T), have, w);
}
// The fold of `have` elements at byte `offset` of every rank's buffer.
template <typename T>
__device__ __forceinline__ void fold_part(const void* const* send, uint32_t nranks, uint64_t offset, uint32_t have, float (&acc)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.0f;
#pragma unroll 4
    for (uint32_t k = 0; k < nranks; ++k) {
        float f[8];
        load_part<T>(bytes_of(send[k]) + offset, have, f);
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
    const ConstBytes residual = L.residual[0] ? bytes_of(L.residual[first]) + uint64_t(at) * L.residual_stride : nullptr;
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
                    store_part<R>(bytes_of(L.hidden[first + d]) + uint64_t(at) * L.hidden_stride + c * sizeof(R), have, h);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = h[i] * r * w[i];
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = clamp_to(quotient(y[i], scale, inverse), limit);
                u32x2 codes = L.int8 ? to_int8(y) : to_e4m3(y);
                if (!finite) codes = L.int8 ? u32x2{0, 0} : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
                for (uint32_t d = 0; d < L.ndst; ++d) {
                    const Bytes p = bytes_of(L.out[first + d]) + uint64_t(at) * L.out_stride + c;
                    if (have == kNormVec) {
                        const uint32_t both[2] = {codes[0], codes[1]};
                        store_dwords<8, false, 1>(p, 0, both, true);
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < kNormVec; ++i)
                            if (i < have) *(MRV_GLOBAL uint8_t*)(p + i) = uint8_t(codes[i / 4] >> (8 * (i % 4)));
                    }
                }
            } else {
                for (uint32_t d = 0; d < L.ndst; ++d)
                    store_part<T>(bytes_of(L.out[first + d]) + uint64_t(at) * L.out_stride + c * sizeof(T), have, y);
            }
        }
        if (sweep == 1) break;
        Reduce::run(shared, kLongLanes / 64, 0, sum, top);
        r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
        if (Q8) {
            finite = row_scale(r, top, L.int8, scale, inverse);
            if (threadIdx.x == 0)
                for (uint32_t d = 0; d < L.ndst; ++d) L.scales[first + d][at] = scale;
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
        const ConstBytes hidden = bytes_of(L.hidden[first]) + uint64_t(at) * L.hidden_stride;
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
                    const Bytes share = bytes_of(L.partial + uint64_t(group) * L.cols + c);
                    float dw[8] = {};
                    if (!fresh) load_part<float>(share, have, dw);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dw[i] = __builtin_fmaf(g[i], h[i] * r, dw[i]);
                    store_part<float>(share, have, dw);
                }
                float dh[8] = {};
                if (L.arriving[0])
                    load_part<R>(bytes_of(L.arriving[first]) + uint64_t(at) * L.arriving_stride + c * sizeof(R), have, dh);
#pragma unroll
                for (int i = 0; i < 8; ++i) dh[i] = __builtin_fmaf(r, __builtin_fmaf(-pull, h[i], g[i] * w[i]), dh[i]);
                for (uint32_t d = 0; d < L.ndst; ++d) {
                    if (L.dhidden[0])
                        store_part<R>(bytes_of(L.dhidden[first + d]) + uint64_t(at) * L.dhidden_stride + c * sizeof(R), have, dh);
                    if (L.dsend[0])
                        store_part<T>(bytes_of(L.dsend[first + d]) + uint64_t(at) * L.dsend_stride + c * sizeof(T), have, dh);
                }
            }
            if (sweep == 1) break;
            uint32_t unused = 0;
            Reduce::run(shared, kLongLanes / 64, slot, sum, unused);
            r = 1.0f / __builtin_sqrtf(sum[0] / float(L.cols) + L.eps);
            pull = r * (r * (sum[1] * (1.0f / float(L.cols))));
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
    constexpr uint32_t kMost = sizeof(T) == 4 ? 4 : 8;  // 32 registers' worth
    constexpr uint32_t kBackMost = sizeof(T) == 4 ? 4 : sizeof(R) == 4 ? 6 : 8;  // what the backward's other values leave
    if (nranks <= 2) return norm_kernels_of<T, R, 1, Wave, Lines, 2, 2>(q8);
    if (nranks <= 4) return norm_kernels_of<T, R, 1, Wave, Lines, 4, 4>(q8);
    return norm_kernels_of<T, R, 1, Wave, Lines, kMost, kBackMost>(q8);
}

template <typename T, typename R, bool Lines>
NormKernels norm_kernels_lines(NormVariant v, uint32_t nranks, bool q8) {
    if (v == kNormWave) return norm_kernels_ranks<T, R, true, Lines>(nranks, q8);
    if (v == kNormBlock) return norm_kernels_ranks<T, R, false, Lines>(nranks, q8);
    return norm_kernels_of<T, R, 2, false, Lines, sizeof(T) == 4 ? 2 : 4, sizeof(R) == 4 ? 1 : 2>(q8);
}

template <typename T, typename R>
NormKernels norm_kernels_for(NormVariant v, uint32_t nranks, bool lines, bool q8) {
    switch (v) {
        case kNormNarrow:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_narrow_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_narrow_kernel<T, R>)};
        case kNormShort:
            return {q8 ? reinterpret_cast<const void*>(&rms_norm_short_kernel<T, R, true>)
                       : reinterpret_cast<const void*>(&rms_norm_short_kernel<T, R, false>),
                    reinterpret_cast<const void*>(&rms_norm_backward_short_kernel<T, R, 16>)};
        case kNormShort32: return {nullptr, reinterpret_cast<const void*>(&rms_norm_backward_short_kernel<T, R, 32>)};
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
