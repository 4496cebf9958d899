// Argument checks, planning and launching of the folds with an epilogue (vrank_fused.h).
#include "vrank_fused.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <iterator>
#include <new>

#include "megray/hip_context.h"
#include "vrank_kernels.h"

namespace MegRay {
namespace vrank {

namespace {

// ---- checks ----------------------------------------------------------------------------------

size_t float_size(int dtype, const char* what) {
    switch (dtype) {
        case MEGRAY_FLOAT16:
        case MRV_BFLOAT16: return 2;
        case MEGRAY_FLOAT32: return 4;
        default: MEGRAY_THROW(what);
    }
}

void check_pointer(const void* p, size_t align, const char* null_text) {
    if (!p) MEGRAY_THROW(null_text);
    if (reinterpret_cast<uintptr_t>(p) % align) MEGRAY_THROW("a buffer does not lie on a multiple of its element size");
}

// Rows of a buffer: `rows` of `bytes` bytes, `stride` bytes apart.
struct Rows {
    uintptr_t at;
    uint64_t rows, bytes, stride;
    uint32_t elem;
    uint64_t end() const { return rows ? at + (rows - 1) * stride + bytes : at; }
};

bool overlap(const Rows& a, const Rows& b) {
    if (!a.rows || !b.rows || a.at >= b.end() || b.at >= a.end()) return false;
    if (a.stride && a.stride == b.stride) {  // column ranges of one matrix lie between each other's rows
        const uint64_t d = (b.at >= a.at ? b.at - a.at : a.stride - (a.at - b.at) % a.stride) % a.stride;
        if (d >= a.bytes && d + b.bytes <= a.stride) return false;
    }
    return true;
}

bool same_place(const Rows& a, const Rows& b) {
    return a.at == b.at && a.elem == b.elem && (a.stride == b.stride || a.rows == 1);
}

// Every output against every input and output.  `replaces[o]` is the input that output o may be, or -1.  Whether one is.
bool check_rows(const std::vector<Rows>& outputs, const std::vector<int>& replaces, const std::vector<Rows>& inputs,
                const std::vector<Rows>& replaced) {
    bool in_place = false;
    for (size_t o = 0; o < outputs.size(); ++o) {
        for (size_t p = o + 1; p < outputs.size(); ++p)
            if (overlap(outputs[o], outputs[p])) MEGRAY_THROW("two outputs overlap");
        for (size_t i = 0; i < inputs.size(); ++i) {
            if (!overlap(outputs[o], inputs[i])) continue;
            if (replaces[o] != int(i) || !same_place(outputs[o], replaced[i])) MEGRAY_THROW("an output overlaps an input out of place");
            in_place = true;
        }
    }
    return in_place;
}

struct Shape {
    bool gathered;  // all_reduce
    uint32_t nranks, cols, part_rows, rows;
    size_t elem, stream_elem;
    bool stream32, weight32;
};

constexpr uint64_t kMaxStride = uint64_t(1) << 40;

uint64_t row_bytes(size_t stride, size_t cols, size_t elem) {
    if (!stride) stride = cols;
    if (stride < cols) MEGRAY_THROW("a row stride is less than the row's length");
    if (stride > kMaxStride) MEGRAY_THROW("a row stride is out of range");
    return uint64_t(stride) * elem;
}

void check_collective(int collective, uint32_t nranks) {
    if (collective != MRV_ALL_REDUCE && collective != MRV_REDUCE_SCATTER)
        MEGRAY_THROW("the norm stands behind an all_reduce or a reduce_scatter");
    if (nranks < 1 || nranks > kMaxRanks) MEGRAY_THROW("nranks must be in [1, 32]");
}

// Rows of the fold and row lengths that the launches count in 32 bits (grids in lanes, too).
void check_extent(uint64_t rows, uint64_t cols) {
    if (cols < 1) MEGRAY_THROW("a row needs at least one element");
    if (cols > (uint64_t(1) << 26)) MEGRAY_THROW("a row is too long");
    if (rows >= (uint64_t(1) << 22)) MEGRAY_THROW("too many rows");
}

Shape check_shape(int collective, uint32_t nranks, size_t rows, size_t cols, int dtype, int residual_dtype, int weight_dtype, float eps) {
    check_collective(collective, nranks);
    Shape s;
    s.gathered = collective == MRV_ALL_REDUCE;
    s.nranks = nranks;
    s.elem = float_size(dtype, "unknown dtype");
    s.stream_elem = float_size(residual_dtype, "unknown residual dtype");
    (void)float_size(weight_dtype, "unknown weight dtype");
    if (residual_dtype != dtype && residual_dtype != MEGRAY_FLOAT32) MEGRAY_THROW("the residual's dtype is the sends' or FLOAT32");
    if (weight_dtype != dtype && weight_dtype != MEGRAY_FLOAT32) MEGRAY_THROW("the weight's dtype is the sends' or FLOAT32");
    s.stream32 = residual_dtype == MEGRAY_FLOAT32;
    s.weight32 = weight_dtype == MEGRAY_FLOAT32;
    if (!(eps >= 0.0f) || !std::isfinite(eps)) MEGRAY_THROW("eps must be finite and not negative");
    if (rows >= (uint64_t(1) << 22)) MEGRAY_THROW("too many rows");
    check_extent(s.gathered ? rows : uint64_t(rows) * nranks, cols);
    s.cols = uint32_t(cols);
    s.part_rows = uint32_t(rows);
    s.rows = s.gathered ? s.part_rows : s.part_rows * nranks;
    return s;
}

// ---- how a norm is laid out --------------------------------------------------------------------

// A wavefront to a row up to 512 elements against a workgroup of one wavefront: 20000 x 384 BF16 of 8 ranks 77 and 79 us, 16384 x 509 of 8 ranks
// 96 and 117, 40000 x 504 of 1 rank 31.5 and 32.6 (backward 51.4 and 51.8); at 512 itself they are level (24.4 and 24.6, 16384 rows of
// 8 ranks 78 and 80, backward 75 and 66).  One vector per lane up to 8192 against two: 4096 x 8192 of 8 ranks 286 and 321 us, of 2 ranks 88 and
// 104, backward 76 and 85.  Two up to 16384 against the row swept twice: 4096 x 16384 of 8 ranks 611 and 782, backward 467 and 744.
// Sixteen lanes to a row up to 128 elements against a wavefront: 65536 x 64 BF16 of 1 rank 9.2 and 23.6 us, backward 16.6 and 43.4; 65536 x 128 of 8 ranks 93 and
// 150, backward 78 and 77; 30000 x 127 of 2 ranks 11.5 and 18.7, backward 15.9 and 31.8 (FP32, 7000 x 99 of 4 ranks 10.1 and 8.7, backward 12.6 and 19.1).
// Thirty-two lanes to a row up to 256 and the workgroup's shares added in LDS against a wavefront and a share of each: backward of 65536 x 256 BF16 of 1 rank 33.9 and
// 50.4 us, 16384 x 256 of 8 ranks 37.7 and 40.3, 20000 x 130 of 4 ranks 18.2 and 26.7 (forward of 8 ranks 44.9 and 36.2, of 1 rank 22.7 and 28.5;
// a wavefront's lanes with the shares in LDS, up to 512: 16384 x 512 of 8 ranks 77.7 and 72.7, 16384 x 509 76.1 and 84.1).  The rule knows widths alone; where
// two figures of a width differ by rank count or type (256 forward, 99 of FP32) it takes what serves the wider range of the backward and the rank counts.
NormVariant norm_variant(uint32_t cols, bool backward) {
    if (cols < kNormVec) return kNormNarrow;
    if (cols <= 16 * kNormVec) return kNormShort;
    if (cols <= 32 * kNormVec && backward) return kNormShort32;
    if (cols <= 64 * kNormVec) return kNormWave;
    if (cols <= 1024 * kNormVec) return kNormBlock;
    if (cols <= 2 * 1024 * kNormVec) return kNormBlock2;
    return kNormLong;
}

// Lanes of a workgroup, and the rows (forward) or row groups (backward) it takes.
struct Layout {
    uint32_t lanes, each;
};

Layout norm_layout(NormVariant v, uint32_t cols, bool backward) {
    const uint32_t per_lane = v == kNormBlock2 ? 2 * kNormVec : kNormVec;
    switch (v) {
        case kNormNarrow: return {256, 256};
        case kNormShort: return {256, backward ? 1u : 16u};
        case kNormShort32: return {256, 1};
        case kNormWave: return {256, 4};
        case kNormLong: return {1024, 1};
        default: return {(cols + 64 * per_lane - 1) / (64 * per_lane) * 64, 1};
    }
}

constexpr uint32_t kComputeUnits = 256;

// Workgroups that the device holds at a time, by the registers of the kernels for so many ranks (norm_kernels_ranks in
// vrank_norm_impl.hpp): a walk over rows with more of them than that would run its second half after its first.  The least over the types with one vector per
// lane: a CU holds 24 - 32 wavefronts of the forward for up to two ranks, 20 - 28 for up to four (16 - 24 with a 32-bit stream), 16 above; of the backward 20,
// 16 - 20 and 16.  Two vectors per lane leave 16 (BF16's backward 20): rows of 8193 to at most 12288 elements of up to four ranks get twice the workgroups
// that are held.  (Twice as many and half as many: 8192 x 8192 BF16 of 8 ranks, forward, 575 -> 579, 575 us, backward 423 -> 423, 424; 2048 x 4096 of 4
// ranks 35.9 -> 36.2, 36.0, backward 35.2 -> 39.6, 33.3.)
uint32_t resident(uint32_t lanes, uint32_t nranks, bool stream32, bool backward) {
    const uint32_t waves = backward ? (nranks <= 2 ? 20 : 16) : nranks <= 2 ? 24 : nranks <= 4 && !stream32 ? 20 : 16;
    return kComputeUnits * std::max(1u, waves * 64 / lanes);
}

// Row groups of a backward, per part: enough to fill the device and no more than twice that, sixteen rows to each if there are (a group
// writes its share of the weight's gradient once), as many to each as to the others.  (Eight rows to each and 32: 8192 x 8192 BF16 of 8 ranks 423 ->
// 422, 429 us, of 2 ranks 145 -> 145, 142; up to once and four times what the device holds: 427, 423, and 141, 145.  Half as many groups of up to 256 lanes:
// 65536 x 1024 of 1 rank 113 -> 101, 8192 x 512 of 8 ranks 44.1 -> 39.2, 8192 x 1024 59.8 -> 55.5, 2000 x 2048 35.6 -> 33.1, 3000 x 300 of 2 ranks
// 15.4 -> 12.5, but 16384 x 2048 of 1 rank 53.4 -> 56.3 and 20000 x 1500 of 4 ranks 128.3 -> 128.4; a quarter: 141, 39.7, 62.4, 35.5, 12.6, 74.5.)
uint32_t backward_groups(NormVariant v, uint32_t cols, uint32_t part_rows, uint32_t nranks, uint32_t nparts) {
    if (!part_rows) return 0;
    const Layout layout = norm_layout(v, cols, true);
    uint32_t target = v == kNormNarrow ? 16384 : v == kNormLong ? kComputeUnits : resident(layout.lanes, nranks, false, true) * layout.each;
    target = std::max(1u, target / nparts);
    const uint32_t rows_at_a_time = v == kNormShort ? 16 : 8;
    if (v == kNormShort || v == kNormShort32) target = std::min(target, (part_rows + 2 * rows_at_a_time - 1) / (2 * rows_at_a_time));
    else if (v != kNormNarrow) target = std::min(std::max(target, part_rows / 16), 2 * target);
    const uint32_t each = (part_rows + target - 1) / target;
    return (part_rows + each - 1) / each;
}

// Written in all, from which a launch is a long one: its stores go one at a time.  Off and on, rows of 8192 BF16 with the hidden state:
// 16384 of 2 ranks 367 -> 344 us, 8192 of 4 ranks 315 -> 306, 8192 of 8 ranks 581 -> 575; below, 1024 of 8 ranks, nothing (76 and 76).
// AdamW with 32-bit states: 1 rank, 2.2 GB written, 737 -> 709 us, 352 MB 119.6 -> 118.0; 8 ranks, 2.7 GB 1052 -> 1037, 704 MB 281 -> 279,
// 352 MB 149 -> 151; below, 1 rank, 176 MB, 62.4 -> 62.7, 8 ranks, 88 MB, 34.9 -> 35.8.
constexpr uint64_t kLongBytes = uint64_t(256) << 20;

// Whether each row has a workgroup of its own, or the workgroups that the device holds walk the rows, each loading its next row before it
// stores this one.  Rows so wide that a CU holds one workgroup need the walk (8192 x 8192 BF16 of 1 rank: walk 101, own 120 us; with
// 8-bit outputs 118 and 132, of 3 ranks 201 and 232) - but not where a long launch has four destinations and more and a store is what
// the wavefronts wait for (of 4 ranks 16384 x 8192: 649 and 593; of 8 ranks 8192 x 8192 624 and 576; 8192 x 6144 of 4 ranks 237 and 228; but 8192 x
// 5120 of 5 ranks 265 and 291).  Of narrower rows a CU holds several, which overlap by themselves, and a launch of many has no
// need of a walk (32768 x 2048 of 2 ranks 172 and 154, 65536 x 1024 of 1 rank 98 and 89, reduce_scatter of 8 ranks 2048 x 4096 258 and 234), one
// of few has (1024 x 4096 of 2 ranks 10.9 and 12.4, 2048 x 4096 of 1 rank 13.7 and 14.8); nor have rows of one wavefront (65536 x 128 26 and 33).
bool one_row_each(NormVariant v, uint32_t lanes, uint32_t nranks, uint32_t turns, bool stores_bound) {
    if (lanes >= 768) return stores_bound;
    return v == kNormBlock && lanes >= 128 && lanes <= (nranks == 1 ? 256u : 512u) && turns >= 8;
}

// Few rows: a CU would fold a row and store it to every destination while others idle.  Workgroups share the destinations
// instead, up to 256 lanes for each CU, and each folds the row for itself, from the caches (8 ranks,
// all of it by one workgroup and shared by eight, four, two: 1 x 8192 BF16 7.8 -> 6.3, 6.2, 6.8 us; 32 x 8192 8.3 -> 11.0, 7.4, 7.2; 64 x 4096
// 5.5 -> 9.9, 6.8, 5.3; 32 x 2048 5.6 -> 4.9, 5.0, 5.2).  Not where a destination is an input: it would be read after it is written.
constexpr uint32_t kSharedLanes = 65536;

uint32_t shares(uint32_t ndst, uint64_t lanes) {
    uint32_t n = 1;
    while (2 * n <= ndst && 2 * n * lanes <= kSharedLanes) n *= 2;
    return n;
}

// Of a buffer that an XCD writes in one run.  None, 64 KiB, 256 KiB, 1 MiB: 8192 x 8192 BF16 of 8 ranks, forward 601, 603, 577, 568 us, backward
// 465, 439, 425, 420; 8192 x 4096 of 2 ranks 84.7, 83.7, 84.3, 84.6 and 75.1, 73.3, 73.2, 73.1; AdamW, 8 ranks, 98 M parameters, none and
// 256 KiB: 1112 and 1043.
constexpr uint32_t kDealBytes = 256 << 10;

Deal deal_blocks(uint32_t blocks, uint64_t block_bytes) {
    Deal d{0, 0};
    while (d.shift < 6 && (block_bytes << (d.shift + 1)) <= kDealBytes) ++d.shift;
    d.whole = blocks >> (d.shift + 3) << (d.shift + 3);
    return d;
}

// Whether rows may stream past the caches: then no line is written in two parts.  Streamed and through the caches: 8192 x 8192 BF16 of 8
// ranks 577 and 617 us, backward 425 and 463, of 2 ranks 73 and 81; 1024 x 8192 of 8 ranks 76 and 90.  What streams leaves by buffer stores, which
// need a 4-byte boundary: a stored row's last piece ends with the row, so the row has to end on one.  BF16 rows of 4160 elements' distance, 4099 of them
// used (through the caches) and 4100 (streamed): 8192 of 8 ranks 355 and 436, backward 257 and 232, of 1 rank 56 and 52, backward 100 and 93.
bool on_lines(const std::vector<Rows>& buffers, const std::vector<Rows>& stored) {
    for (const Rows& b : buffers)
        if (b.at % 128 || (b.rows > 1 && b.stride % 128)) return false;
    for (const Rows& b : stored)
        if (b.bytes % 4) return false;
    return true;
}

NormKernels kernels_for(int dtype, NormVariant v, uint32_t nranks, bool stream32, bool lines, bool q8) {
    switch (dtype) {
        case MEGRAY_FLOAT16: return (stream32 ? norm_kernels_f16_f32 : norm_kernels_f16)(v, nranks, lines, q8);
        case MRV_BFLOAT16: return (stream32 ? norm_kernels_bf16_f32 : norm_kernels_bf16)(v, nranks, lines, q8);
        default: return norm_kernels_f32(v, nranks, lines, q8);
    }
}

// Columns of a workgroup of the weight gradient's launch: few make many workgroups, many read whole lines of the shares.  64 and 16, both launches
// together: 5099 x 88 of 8 ranks 22.1 and 17.7 us, 40000 x 256 of 1 rank 41.6 and 37.4, 65536 x 1024 117.6 and 114.6, 8192 x 4096 57.5 and 58.6,
// 8192 x 8192 120 and 124, 4096 x 16384 of 4 ranks 249 and 259.
uint32_t weight_cols(uint32_t cols) {
    return cols < 4096 ? 16 : 64;
}

Status launch_kernel(const void* kernel, dim3 grid, uint32_t block, const void* descriptor, hipStream_t stream) {
    if (!grid.x) return MEGRAY_OK;
    void* args[] = {const_cast<void*>(descriptor)};
    HIP_CHECK(hipLaunchKernel(kernel, grid, dim3(block), args, 0, stream));
    return MEGRAY_OK;
}

}  // namespace

NormPlan::NormPlan() {
    std::memset(&m_forward, 0, sizeof(m_forward));
    std::memset(&m_backward, 0, sizeof(m_backward));
    std::memset(&m_weight, 0, sizeof(m_weight));
}

void NormPlan::plan_forward(int collective, const mrv_rms_norm_call& c) {
    const Shape s = check_shape(collective, c.nranks, c.rows, c.cols, c.dtype, c.residual_dtype, c.weight_dtype, c.eps);
    const bool q8 = c.out_dtype == MEGRAY_INT8 || c.out_dtype == MRV_FLOAT8_E4M3;
    if (!q8 && c.out_dtype != c.dtype) MEGRAY_THROW("the output's dtype is the sends', INT8 or FLOAT8_E4M3");
    const size_t out_elem = q8 ? 1 : s.elem;
    if (!c.sendbuffs) MEGRAY_THROW("sendbuffs is null");
    if (!c.outs) MEGRAY_THROW("outs is null");
    if (q8 && !c.scales) MEGRAY_THROW("an 8-bit output needs scales");
    NormLaunch& L = m_forward;
    L.send_stride = row_bytes(c.send_stride, s.cols, s.elem);
    L.residual_stride = row_bytes(c.residual_stride, s.cols, s.stream_elem);
    L.hidden_stride = row_bytes(c.residual_out_stride, s.cols, s.stream_elem);
    L.out_stride = row_bytes(c.out_stride, s.cols, out_elem);
    if (!s.rows) return;  // nothing to launch
    std::vector<Rows> inputs, replaced, outputs, rows;
    std::vector<int> replaces;
    auto input = [&](const void* p, uint64_t count, uint64_t stride, size_t elem, uint64_t own_row) {
        inputs.push_back({reinterpret_cast<uintptr_t>(p), count, s.cols * elem, stride, uint32_t(elem)});
        rows.push_back(inputs.back());
        replaced.push_back(inputs.back());
        replaced.back().at += own_row * stride;
    };
    auto output = [&](void* p, uint64_t stride, size_t elem, int replacing) {
        outputs.push_back({reinterpret_cast<uintptr_t>(p), s.part_rows, s.cols * elem, stride, uint32_t(elem)});
        rows.push_back(outputs.back());
        replaces.push_back(replacing);
    };
    for (uint32_t r = 0; r < s.nranks; ++r) {
        check_pointer(c.sendbuffs[r], s.elem, "a send buffer is null");
        L.send[r] = c.sendbuffs[r];
        input(c.sendbuffs[r], s.rows, L.send_stride, s.elem, s.gathered ? 0 : uint64_t(r) * s.part_rows);
    }
    const uint32_t residuals = c.residuals ? (s.gathered ? 1 : s.nranks) : 0;
    for (uint32_t r = 0; r < residuals; ++r) {
        check_pointer(c.residuals[r], s.stream_elem, "a residual is null");
        L.residual[r] = c.residuals[r];
        input(c.residuals[r], s.part_rows, L.residual_stride, s.stream_elem, 0);
    }
    check_pointer(c.weight, s.weight32 ? 4 : s.elem, "weight is null");
    L.weight = c.weight;
    inputs.push_back({reinterpret_cast<uintptr_t>(c.weight), 1, uint64_t(s.cols) * (s.weight32 ? 4 : s.elem), 0, 0});
    replaced.push_back(inputs.back());
    uint64_t written = 0;
    for (uint32_t r = 0; r < s.nranks; ++r) {
        check_pointer(c.outs[r], out_elem, "an output is null");
        L.out[r] = c.outs[r];
        output(c.outs[r], L.out_stride, out_elem, q8 ? -1 : int(r));
        if (c.residual_outs) {
            check_pointer(c.residual_outs[r], s.stream_elem, "a residual output is null");
            L.hidden[r] = c.residual_outs[r];
            output(c.residual_outs[r], L.hidden_stride, s.stream_elem, residuals ? int(s.nranks + (s.gathered ? 0 : r)) : -1);
        }
        if (q8) {
            check_pointer(c.scales[r], 4, "a scale buffer is null");
            L.scales[r] = c.scales[r];
            outputs.push_back({reinterpret_cast<uintptr_t>(c.scales[r]), 1, uint64_t(s.part_rows) * 4, 0, 4});
            replaces.push_back(-1);
        }
        written += uint64_t(s.part_rows) * s.cols * (out_elem + (c.residual_outs ? s.stream_elem : 0));
    }
    const bool in_place = check_rows(outputs, replaces, inputs, replaced);
    L.rows = s.rows;
    L.part_rows = s.part_rows;
    L.cols = s.cols;
    L.nranks = s.nranks;
    L.ndst = s.gathered ? s.nranks : 1;
    L.weight32 = s.weight32;
    L.int8 = c.out_dtype == MEGRAY_INT8;
    L.keep = written <= kKeepMaxBytes;
    L.has_hidden = c.residual_outs != nullptr;
    L.eps = c.eps;
    const NormVariant v = norm_variant(s.cols, false);
    const Layout layout = norm_layout(v, s.cols, false);
    m_first = kernels_for(c.dtype, v, s.nranks, s.stream32, on_lines(rows, outputs), q8).forward;
    L.positions = (s.rows + layout.each - 1) / layout.each;
    m_block = L.lanes = layout.lanes;
    const bool long_launch = written >= kLongBytes;
    const uint32_t at_a_time = resident(layout.lanes, s.nranks, s.stream32, false);
    const bool one_each = v == kNormNarrow || v == kNormShort || v == kNormLong || one_row_each(v, layout.lanes, s.nranks, L.positions / at_a_time, long_launch && L.ndst >= 4 && !q8);
    m_grid = one_each ? L.positions : std::min(L.positions, at_a_time);
    L.splits = v == kNormBlock && !in_place ? shares(L.ndst, uint64_t(L.positions) * layout.lanes) : 1;
    m_grid *= L.splits;
    L.deal = deal_blocks(L.positions, layout.each * L.send_stride);
    L.pace.on = long_launch && L.ndst > 1;
    m_descriptor = &m_forward;
}

size_t norm_backward_workspace(int collective, uint32_t nranks, size_t rows, size_t cols) {
    check_collective(collective, nranks);
    const uint32_t nparts = collective == MRV_ALL_REDUCE ? 1 : nranks;
    if (rows >= (uint64_t(1) << 22)) MEGRAY_THROW("too many rows");
    check_extent(uint64_t(rows) * nparts, cols);
    return size_t(backward_groups(norm_variant(uint32_t(cols), true), uint32_t(cols), uint32_t(rows), nranks, nparts)) * nparts * cols * sizeof(float);
}

void NormPlan::plan_backward(int collective, const mrv_rms_norm_backward_call& c) {
    const Shape s = check_shape(collective, c.nranks, c.rows, c.cols, c.dtype, c.residual_dtype, c.weight_dtype, c.eps);
    if (!c.sendbuffs) MEGRAY_THROW("sendbuffs is null");
    if (!c.hiddens) MEGRAY_THROW("hiddens is null");
    if (!c.residual_out_grads && !c.send_grads && !c.weight_grads) MEGRAY_THROW("no gradient is asked for");
    NormBackLaunch& L = m_backward;
    L.send_stride = row_bytes(c.send_stride, s.cols, s.elem);
    L.hidden_stride = row_bytes(c.hidden_stride, s.cols, s.stream_elem);
    L.arriving_stride = row_bytes(c.residual_grad_stride, s.cols, s.stream_elem);
    L.dhidden_stride = row_bytes(c.residual_out_grad_stride, s.cols, s.stream_elem);
    L.dsend_stride = row_bytes(c.send_grad_stride, s.cols, s.elem);
    std::vector<Rows> inputs, replaced, outputs, rows;
    std::vector<int> replaces;
    const uint32_t copies = s.gathered ? 1 : s.nranks;
    auto input = [&](const void* p, uint64_t count, uint64_t stride, size_t elem, uint64_t own_row) {
        inputs.push_back({reinterpret_cast<uintptr_t>(p), count, s.cols * elem, stride, uint32_t(elem)});
        rows.push_back(inputs.back());
        replaced.push_back(inputs.back());
        replaced.back().at += own_row * stride;
    };
    if (s.rows) {
        for (uint32_t r = 0; r < s.nranks; ++r) {
            check_pointer(c.sendbuffs[r], s.elem, "a send buffer is null");
            L.send[r] = c.sendbuffs[r];
            input(c.sendbuffs[r], s.rows, L.send_stride, s.elem, s.gathered ? 0 : uint64_t(r) * s.part_rows);
        }
        for (uint32_t r = 0; r < copies; ++r) {
            check_pointer(c.hiddens[r], s.stream_elem, "a hidden state is null");
            L.hidden[r] = c.hiddens[r];
            input(c.hiddens[r], s.part_rows, L.hidden_stride, s.stream_elem, 0);
        }
        for (uint32_t r = 0; c.residual_grads && r < copies; ++r) {
            check_pointer(c.residual_grads[r], s.stream_elem, "a residual gradient is null");
            L.arriving[r] = c.residual_grads[r];
            input(c.residual_grads[r], s.part_rows, L.arriving_stride, s.stream_elem, 0);
        }
        check_pointer(c.weight, s.weight32 ? 4 : s.elem, "weight is null");
        L.weight = c.weight;
        inputs.push_back({reinterpret_cast<uintptr_t>(c.weight), 1, uint64_t(s.cols) * (s.weight32 ? 4 : s.elem), 0, 0});
        replaced.push_back(inputs.back());
    }
    const NormVariant v = norm_variant(s.cols, true);
    const uint32_t nparts = s.gathered ? 1 : s.nranks;
    const uint32_t part_groups = backward_groups(v, s.cols, s.part_rows, s.nranks, nparts);
    uint64_t written = 0;
    bool replaced_arriving = false;
    for (uint32_t r = 0; r < s.nranks; ++r) {
        const int own = int(s.gathered ? 0 : r);
        if (c.residual_out_grads && s.rows) {
            check_pointer(c.residual_out_grads[r], s.stream_elem, "a residual gradient output is null");
            L.dhidden[r] = c.residual_out_grads[r];
            outputs.push_back({reinterpret_cast<uintptr_t>(L.dhidden[r]), s.part_rows, s.cols * s.stream_elem, L.dhidden_stride, uint32_t(s.stream_elem)});
            rows.push_back(outputs.back());
            // in the hidden state's place, or in the arriving gradient's
            const bool arriving = c.residual_grads && L.dhidden[r] == L.arriving[own];
            replaced_arriving |= arriving;
            replaces.push_back(int(s.nranks) + (arriving ? int(copies) : 0) + own);
            written += uint64_t(s.part_rows) * s.cols * s.stream_elem;
        }
        if (c.send_grads && s.rows) {
            check_pointer(c.send_grads[r], s.elem, "a send gradient is null");
            L.dsend[r] = c.send_grads[r];
            outputs.push_back({reinterpret_cast<uintptr_t>(L.dsend[r]), s.part_rows, s.cols * s.elem, L.dsend_stride, uint32_t(s.elem)});
            rows.push_back(outputs.back());
            replaces.push_back(int(r));
            written += uint64_t(s.part_rows) * s.cols * s.elem;
        }
        if (c.weight_grads) {
            check_pointer(c.weight_grads[r], 4, "a weight gradient is null");
            m_weight.dweight[r] = c.weight_grads[r];
            outputs.push_back({reinterpret_cast<uintptr_t>(c.weight_grads[r]), 1, uint64_t(s.cols) * 4, 0, 4});
            replaces.push_back(-1);
        }
    }
    if (c.weight_grads) {
        const size_t need = size_t(part_groups) * nparts * s.cols * sizeof(float);
        if (need) {
            check_pointer(c.workspace, 4, "weight gradients need a workspace");
            if (c.workspace_bytes < need) MEGRAY_THROW("the workspace is too small (see mrv_rms_norm_backward_workspace)");
            outputs.push_back({reinterpret_cast<uintptr_t>(c.workspace), 1, need, 0, 4});
            replaces.push_back(-1);
        }
        L.partial = static_cast<float*>(c.workspace);
        m_weight.partial = L.partial;
        m_weight.part_groups = part_groups;
        m_weight.cols = s.cols;
        m_weight.nparts = nparts;
        m_weight.nranks = s.nranks;
        m_weight_cols = weight_cols(s.cols);
        m_second = norm_weight_kernel(m_weight_cols);
    }
    check_rows(outputs, replaces, inputs, replaced);
    if (!s.rows) return;  // the weight gradients are zero then
    L.rows = s.rows;
    L.part_rows = s.part_rows;
    L.part_groups = part_groups;
    L.groups = part_groups * nparts;
    L.cols = s.cols;
    L.nranks = s.nranks;
    L.ndst = s.gathered ? s.nranks : 1;
    L.weight32 = s.weight32;
    L.keep = written <= kKeepMaxBytes;
    L.eps = c.eps;
    // Two vectors per lane read the arriving gradient between their stores.  Where it is replaced and rows end inside a vector, the sweep
    // takes the row groups instead: it reads and stores every element in one lane.
    const NormVariant taken = v == kNormBlock2 && replaced_arriving && s.cols % kNormVec ? kNormLong : v;
    const Layout layout = norm_layout(taken, s.cols, true);
    m_first = kernels_for(c.dtype, taken, s.nranks, s.stream32, on_lines(rows, outputs), false).backward;
    m_grid = (L.groups + layout.each - 1) / layout.each;
    m_block = L.lanes = layout.lanes;
    L.deal = deal_blocks(v == kNormWave || v == kNormShort || v == kNormShort32 ? 0 : s.part_rows, L.send_stride);
    m_descriptor = &m_backward;
}

Status NormPlan::launch(hipStream_t stream) const {
    if (m_first) {
        const Status st = launch_kernel(m_first, dim3(m_grid), m_block, m_descriptor, stream);
        if (st != MEGRAY_OK) return st;
    }
    if (m_second)
        return launch_kernel(m_second, dim3((m_weight.cols + m_weight_cols - 1) / m_weight_cols, m_weight.nparts), kNormWeightThreads, &m_weight, stream);
    return MEGRAY_OK;
}

// ---- AdamW ---------------------------------------------------------------------------------------

namespace {

struct Interval {
    uintptr_t begin, end;
    bool written;
};

// No output may overlap anything else.  Returns what is taken by all tensors and by those that are written.
void check_intervals(std::vector<Interval>& all, Taken& any, Taken& written) {
    std::sort(all.begin(), all.end(), [](const Interval& a, const Interval& b) { return a.begin < b.begin; });
    for (const Interval& x : all) {
        if ((x.written ? any : written).overlaps(x.begin, x.end)) MEGRAY_THROW("a tensor that is written overlaps another");
        any.add(x.begin, x.end);
        if (x.written) written.add(x.begin, x.end);
    }
}

}  // namespace

void Taken::add(uintptr_t begin, uintptr_t end) {
    if (!m_runs.empty() && begin <= m_runs.back().second) m_runs.back().second = std::max(m_runs.back().second, end);
    else m_runs.push_back({begin, end});
}

bool Taken::overlaps(uintptr_t begin, uintptr_t end) const {
    auto next = std::lower_bound(m_runs.begin(), m_runs.end(), end, [](const std::pair<uintptr_t, uintptr_t>& run, uintptr_t at) { return run.first < at; });
    return next != m_runs.begin() && std::prev(next)->second > begin;  // the last run that begins before `end`
}

namespace {

// Workgroups of the gradient norm.  Few bytes in flight to each, or a tile or few, want many of them; where a lane loads 16 bytes of an element at
// once or more and all of its ranks together, the fewer keep closer together.  512 and 2048: BF16, 98 M of 1 rank 87 and 38 us, 79 M of 3 ranks 100 and 76, of 4
// ranks 110 and 99, 39 M of 16 ranks 203 and 196, 14 M of 8 ranks 49.6 and 41.2; 98 M of 8 ranks 235 and 244, 25 M 62.4 and 65.4 (but 29 M
// 80.7 and 78.2); FP32, 24 M of 4 ranks 58.9 and 60.6, 39 M of 8 ranks 185 and 189.
uint32_t norm_groups(uint64_t tiles, uint32_t ranks, size_t elem) {
    return tiles >= 8192 && ranks <= 8 && ranks * elem >= 16 ? 512 : uint32_t(std::min<uint64_t>(tiles, 2048));
}

}  // namespace

Adamw::Adamw(const mrv_adamw_tensors& t) {
    if (t.grad_ranks < 1 || t.grad_ranks > kMaxRanks) MEGRAY_THROW("grad_ranks must be in [1, 32]");
    const size_t grad_elem = float_size(t.grad_dtype, "unknown gradient dtype");
    if (t.ntensors && (!t.lens || !t.grads)) MEGRAY_THROW("lens or grads is null");
    m_can_step = t.params != nullptr;
    size_t param_elem = 0;
    bool state8 = false;
    if (m_can_step) {
        if (t.param_ranks < 1 || t.param_ranks > kMaxRanks) MEGRAY_THROW("param_ranks must be in [1, 32]");
        param_elem = float_size(t.param_dtype, "unknown parameter dtype");
        if (t.state_dtype != MEGRAY_FLOAT32 && t.state_dtype != MRV_FLOAT8_E4M3) MEGRAY_THROW("states are FLOAT32 or FLOAT8_E4M3");
        state8 = t.state_dtype == MRV_FLOAT8_E4M3;
        if (!t.masters && t.param_dtype != MEGRAY_FLOAT32) MEGRAY_THROW("masters is null and the parameters are not FLOAT32");
        if (!t.exp_avgs || !t.exp_avg_sqs) MEGRAY_THROW("exp_avgs or exp_avg_sqs is null");
        if (state8 && (!t.exp_avg_scales || !t.exp_avg_sq_scales)) MEGRAY_THROW("8-bit states need scales");
    }
    const uint32_t param_ranks = m_can_step ? t.param_ranks : 0;

    // The norm's tiles and the step's, which may be larger ones.
    const uint32_t threads = state8 ? kAdamThreads8 : kAdamThreads;
    const uint64_t norm_tile = kAdamNormThreads * kAdamVec, step_tile = uint64_t(threads) * kAdamVec;
    uint64_t norm_tiles = 0, step_tiles = 0;
    for (size_t n = 0; n < t.ntensors; ++n) {
        if (t.lens[n] > (uint64_t(1) << 40)) MEGRAY_THROW("a tensor is too long");
        norm_tiles += (t.lens[n] + norm_tile - 1) / norm_tile;
        step_tiles += m_can_step ? (t.lens[n] + step_tile - 1) / step_tile : 0;
        // a grid counts its lanes in 32 bits, and a tensor may be a tile of a few elements
        if (norm_tiles >= (uint64_t(1) << 24) || step_tiles * threads >= uint64_t(1) << 32) MEGRAY_THROW("too many elements for one handle");
    }
    if (t.ntensors >= (uint64_t(1) << 24)) MEGRAY_THROW("too many tensors for one handle");

    // one table: tensors, the norm's tiles, the step's tiles, gradient pointers, parameter pointers
    const size_t tensors_bytes = t.ntensors * sizeof(AdamTensor);
    const size_t norm_bytes = size_t(norm_tiles) * sizeof(AdamTile), tiles_bytes = norm_bytes + size_t(step_tiles) * sizeof(AdamTile);
    const size_t grads_bytes = t.ntensors * t.grad_ranks * sizeof(void*), params_bytes = t.ntensors * param_ranks * sizeof(void*);
    std::vector<char> host(tensors_bytes + tiles_bytes + grads_bytes + params_bytes);
    auto* tensors = reinterpret_cast<AdamTensor*>(host.data());
    auto* norm_at = reinterpret_cast<AdamTile*>(host.data() + tensors_bytes);
    auto* step_at = norm_at + norm_tiles;
    auto* grads = reinterpret_cast<const void**>(host.data() + tensors_bytes + tiles_bytes);
    auto* params = reinterpret_cast<void**>(host.data() + tensors_bytes + tiles_bytes + grads_bytes);
    std::vector<Interval> used;
    uintptr_t bits = 0;  // of the current tensor's buffers' addresses
    auto take = [&](const void* p, uint64_t bytes, size_t align, bool written, const char* null_text) {
        check_pointer(p, align, null_text);
        const uintptr_t a = reinterpret_cast<uintptr_t>(p);
        used.push_back({a, a + bytes, written});
        bits |= a;
    };
    for (size_t n = 0; n < t.ntensors; ++n) {
        const uint64_t len = t.lens[n];
        AdamTensor& x = tensors[n];
        std::memset(&x, 0, sizeof(x));
        x.len = len;
        if (!len) continue;
        bits = 0;
        for (uint64_t k = 0; k * norm_tile < len; ++k) *norm_at++ = {uint32_t(n), uint32_t(k)};
        for (uint64_t k = 0; m_can_step && k * step_tile < len; ++k) *step_at++ = {uint32_t(n), uint32_t(k)};
        for (uint32_t r = 0; r < t.grad_ranks; ++r) {
            const void* p = t.grads[size_t(r) * t.ntensors + n];
            take(p, len * grad_elem, grad_elem, false, "a gradient is null");
            grads[n * t.grad_ranks + r] = p;
        }
        if (!m_can_step) continue;
        for (uint32_t r = 0; r < param_ranks; ++r) {
            void* p = t.params[size_t(r) * t.ntensors + n];
            take(p, len * param_elem, param_elem, true, "a parameter is null");
            params[n * param_ranks + r] = p;
        }
        x.master = t.masters ? t.masters[n] : static_cast<float*>(params[n * param_ranks]);
        const bool shared = t.param_dtype == MEGRAY_FLOAT32 && x.master == params[n * param_ranks];
        if (!shared) take(x.master, len * 4, 4, true, "a master is null");
        const uint64_t blocks = (len + kAdamBlock - 1) / kAdamBlock;
        x.m = t.exp_avgs[n];
        x.v = t.exp_avg_sqs[n];
        x.decay = t.weight_decays ? t.weight_decays[n] : 0.0f;
        if (!std::isfinite(x.decay)) MEGRAY_THROW("a weight decay is not finite");
        take(x.m, len * (state8 ? 1 : 4), state8 ? 1 : 4, true, "a running mean is null");
        take(x.v, len * (state8 ? 1 : 4), state8 ? 1 : 4, true, "a running mean of squares is null");
        x.lines = bits % 128 == 0;  // the scales, a float per block, do not matter for it
        if (state8) {
            x.m_scale = t.exp_avg_scales[n];
            x.v_scale = t.exp_avg_sq_scales[n];
            take(x.m_scale, blocks * 4, 4, true, "a scale buffer is null");
            take(x.v_scale, blocks * 4, 4, true, "a scale buffer is null");
        }
    }
    check_intervals(used, m_any, m_written);

    uint64_t written = 0;
    for (const Interval& x : used) written += x.written ? x.end - x.begin : 0;
    m_step.keep = written <= kKeepMaxBytes;
    m_step.pace.on = !state8 && written >= kLongBytes;
    m_groups = norm_groups(norm_tiles, t.grad_ranks, grad_elem);
    if (hipGetDevice(&m_device) != hipSuccess) {
        (void)hipGetLastError();
        throw HipFailure();
    }
    if (!host.empty()) {
        if (hipMalloc(&m_table, host.size()) != hipSuccess) {
            (void)hipGetLastError();
            m_table = nullptr;
            throw HipFailure();
        }
        if (hipMemcpy(m_table, host.data(), host.size(), hipMemcpyHostToDevice) != hipSuccess) {
            (void)hipGetLastError();
            (void)hipFree(m_table);
            m_table = nullptr;
            throw HipFailure();
        }
    }
    const char* table = static_cast<const char*>(m_table);
    m_norm.tensors = m_step.tensors = reinterpret_cast<const AdamTensor*>(table);
    m_norm.tiles = reinterpret_cast<const AdamTile*>(table + tensors_bytes);
    m_step.tiles = reinterpret_cast<const AdamTile*>(table + tensors_bytes + norm_bytes);
    m_norm.grads = m_step.grads = reinterpret_cast<const void* const*>(table + tensors_bytes + tiles_bytes);
    m_step.params = reinterpret_cast<void* const*>(const_cast<char*>(table) + tensors_bytes + tiles_bytes + grads_bytes);
    m_norm.grad_ranks = m_step.grad_ranks = t.grad_ranks;
    m_step.param_ranks = param_ranks;
    m_norm.ntiles = uint32_t(norm_tiles);
    m_step.ntiles = uint32_t(step_tiles);
    m_threads = threads;
    m_norm.groups = m_groups;
    m_norm.deal = deal_blocks(m_norm.ntiles, norm_tile * grad_elem);
    m_step.deal = deal_blocks(m_step.ntiles, step_tile * grad_elem);
    m_norm_kernel = adamw_norm_kernel_for(t.grad_dtype);
    if (m_can_step) m_step_kernel = adamw_kernel_for(t.grad_dtype, t.param_dtype, state8);
}

Adamw::~Adamw() {
    if (m_table) (void)hipFree(m_table);
}

void Adamw::check_device() const {
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess) {
        (void)hipGetLastError();
        throw HipFailure();
    }
    if (device != m_device) MEGRAY_THROW("the handle's tables are on another device than the current one");
}

Status Adamw::grad_norm(float grad_scale, float max_norm, float* out, hipStream_t stream) const {
    if (!out) MEGRAY_THROW("out is null");
    if (reinterpret_cast<uintptr_t>(out) % 8) MEGRAY_THROW("out does not lie on a multiple of 8 bytes");
    if (!std::isfinite(grad_scale)) MEGRAY_THROW("grad_scale is not finite");
    if (!(max_norm >= 0.0f)) MEGRAY_THROW("max_norm must not be negative");
    if (m_any.overlaps(reinterpret_cast<uintptr_t>(out), reinterpret_cast<uintptr_t>(out + norm_floats()))) MEGRAY_THROW("out overlaps a tensor");
    check_device();
    AdamNormLaunch L = m_norm;
    L.grad_scale = grad_scale;
    L.max_norm = max_norm;
    L.out = out;
    const Status st = launch_kernel(m_norm_kernel, dim3(m_groups), kAdamNormThreads, &L, stream);
    if (st != MEGRAY_OK) return st;
    return launch_kernel(adamw_norm_join_kernel(), dim3(1), kAdamJoinThreads, &L, stream);
}

Status Adamw::step(const mrv_adamw_step_args& a, hipStream_t stream) const {
    if (!m_can_step) MEGRAY_THROW("the handle was made without parameters: it has no step");
    if (!std::isfinite(float(a.lr)) || !std::isfinite(float(a.grad_scale))) MEGRAY_THROW("lr or grad_scale is not finite");
    if (!(a.beta1 >= 0 && a.beta1 < 1 && a.beta2 >= 0 && a.beta2 < 1)) MEGRAY_THROW("beta1 and beta2 must be in [0, 1)");
    if (!(a.eps >= 0) || !std::isfinite(float(a.eps))) MEGRAY_THROW("eps must be finite and not negative");
    if (a.step < 1) MEGRAY_THROW("step counts from 1");
    if (reinterpret_cast<uintptr_t>(a.clip) % 4) MEGRAY_THROW("clip does not lie on a multiple of 4 bytes");
    if (a.clip && m_written.overlaps(reinterpret_cast<uintptr_t>(a.clip), reinterpret_cast<uintptr_t>(a.clip + 1)))
        MEGRAY_THROW("clip lies in a tensor that the step writes");
    check_device();
    AdamLaunch L = m_step;
    L.lr = float(a.lr);
    L.beta1 = float(a.beta1);
    L.beta2 = float(a.beta2);
    L.rest1 = float(1 - a.beta1);
    L.rest2 = float(1 - a.beta2);
    L.eps = float(a.eps);
    L.rate = float(a.lr / (1 - std::pow(a.beta1, double(a.step))));
    L.root_scale = float(1 / std::sqrt(1 - std::pow(a.beta2, double(a.step))));
    L.grad_scale = float(a.grad_scale);
    L.clip = a.clip;
    return launch_kernel(m_step_kernel, dim3(L.ntiles), m_threads, &L, stream);
}

}  // namespace vrank
}  // namespace MegRay
