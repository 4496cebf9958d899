// Device helpers of the folds with an epilogue: eight elements of a row or tensor at a time.
//
// Rows and tensors start anywhere: the 128-bit global accesses of gfx950 take any element boundary, so one code path
// serves every alignment (an access off the 16-byte grid costs its wavefront one more cache line, nothing else).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>
#include <type_traits>

#include "vrank_fused.h"

namespace MegRay {
namespace vrank {
namespace fused {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int Align>
struct Unaligned;
#define MRV_UNALIGNED(n)                             \
    template <>                                      \
    struct Unaligned<n> {                            \
        typedef u32x4 v4 __attribute__((aligned(n))); \
        typedef u32x2 v2 __attribute__((aligned(n))); \
    };
MRV_UNALIGNED(1)
MRV_UNALIGNED(2)
MRV_UNALIGNED(4)
#undef MRV_UNALIGNED

// Pointers out of a descriptor or a table are global memory; saying so keeps flat instructions out of the kernels.
#define MRV_GLOBAL __attribute__((address_space(1)))
typedef MRV_GLOBAL char* Bytes;
typedef const MRV_GLOBAL char* ConstBytes;
__device__ __forceinline__ ConstBytes bytes_of(const void* p) {
    return (ConstBytes)(uintptr_t)p;
}
__device__ __forceinline__ Bytes bytes_of(void* p) {
    return (Bytes)(uintptr_t)p;
}
__device__ __forceinline__ Bytes bytes_of(float* p) {
    return (Bytes)(uintptr_t)p;
}

// Two pointer tables of a launch descriptor that lie behind each other, entry l in lane l: one access reads them, and they take two vector
// registers where 64 entries would not fit the scalar ones.
struct LaneTable {
    uint32_t lo, hi;
    __device__ __forceinline__ explicit LaneTable(size_t offset) {  // in the kernel's only argument
        static_assert(2 * kMaxRanks == 64, "an entry per lane");
        typedef const __attribute__((address_space(4))) char* Constant;
        const Constant p = Constant(__builtin_amdgcn_kernarg_segment_ptr()) + offset + threadIdx.x % 64 * sizeof(void*);
        lo = reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(p)[0];
        hi = reinterpret_cast<const __attribute__((address_space(4))) uint32_t*>(p)[1];
    }
    __device__ __forceinline__ Bytes at(uint32_t entry) const {  // the same entry for the whole wavefront
        const uint32_t a = __builtin_amdgcn_readlane(lo, entry), b = __builtin_amdgcn_readlane(hi, entry);
        return (Bytes)(uint64_t(b) << 32 | a);
    }
    __device__ __forceinline__ Bytes first(uint32_t entry) const { return at(entry); }
    __device__ __forceinline__ Bytes second(uint32_t entry) const { return at(kMaxRanks + entry); }
};

// Eight elements of T as they lie in memory: one piece of eight, or two pieces of four.  A wavefront's accesses have to cover whole cache
// lines one instruction at a time: eight 32-bit elements per lane are two 16-byte accesses 32 bytes apart, half of every line twice, which
// past the caches (a store that streams) costs more than twice the time.  So wherever a 32-bit type takes part, the
// lanes hold two pieces of four elements, the wavefront's second 256 elements behind its first: 16 bytes of a 32-bit type, 8 of a 16-bit one.
template <typename T>
struct Raw8 {
    uint32_t w[2 * sizeof(T)];
};

template <uint32_t Count, bool Once, int Align>
__device__ __forceinline__ void load_dwords(ConstBytes p, uint32_t* w) {
    if constexpr (Count == 8) {
        typedef typename Unaligned<Align>::v2 V;
        const u32x2 x = Once ? __builtin_nontemporal_load((const MRV_GLOBAL V*)p) : *(const MRV_GLOBAL V*)p;
        w[0] = x[0], w[1] = x[1];
    } else {
        typedef typename Unaligned<Align>::v4 V;
#pragma unroll
        for (uint32_t i = 0; i < Count / 16; ++i) {
            const u32x4 x = Once ? __builtin_nontemporal_load((const MRV_GLOBAL V*)p + i) : ((const MRV_GLOBAL V*)p)[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
        }
    }
}

// Eight consecutive elements.  `Once`: the data is read by no one else soon, so it need not stay in the caches.
template <typename T, bool Once>
__device__ __forceinline__ Raw8<T> load8(ConstBytes p) {
    Raw8<T> x;
    load_dwords<8 * sizeof(T), Once, sizeof(T)>(p, x.w);
    return x;
}
// Two pieces of four.
template <typename T, bool Once>
__device__ __forceinline__ Raw8<T> load44(ConstBytes p, ConstBytes q) {
    Raw8<T> x;
    load_dwords<4 * sizeof(T), Once, sizeof(T)>(p, x.w);
    load_dwords<4 * sizeof(T), Once, sizeof(T)>(q, x.w + sizeof(T));
    return x;
}

template <typename T>
__device__ __forceinline__ void widen(const Raw8<T>& x, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __builtin_bit_cast(float, x.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (__is_same(T, __bf16)) {
                f[2 * i] = __builtin_bit_cast(float, x.w[i] << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, x.w[i] & 0xffff0000u);
            } else {
                f[2 * i] = float(__builtin_bit_cast(_Float16, uint16_t(x.w[i])));
                f[2 * i + 1] = float(__builtin_bit_cast(_Float16, uint16_t(x.w[i] >> 16)));
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ Raw8<T> narrow(const float (&f)[8]) {
    Raw8<T> x;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.w[i] = __builtin_bit_cast(uint32_t, f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typedef T Pair __attribute__((ext_vector_type(2)));
            typedef float Wide __attribute__((ext_vector_type(2)));
            x.w[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((Wide{f[2 * i], f[2 * i + 1]}), Pair));
        }
    }
    return x;
}

// Stores.  Rows on cache lines go past the caches like the collectives' own results (or stay in the last-level cache:
// `keep`); others leave lines that two wavefronts, or two rows, write a part of, and those are put together in the L2.
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
constexpr int kStream = 18;  // sc1 | nt
constexpr int kStay = 16;    // sc1
template <uint32_t Count, bool Lines, int Align>
__device__ __forceinline__ void store_dwords(Bytes base, uint32_t offset, const uint32_t* w, bool keep) {
    if constexpr (Lines) {  // `base` is the same for the whole wavefront, base + offset a multiple of four: what a buffer store needs
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, -1, 0x00020000);
        if constexpr (Count == 4) {
            if (keep) __builtin_amdgcn_raw_buffer_store_b32(int32_t(w[0]), rsrc, int(offset), 0, kStay);
            else __builtin_amdgcn_raw_buffer_store_b32(int32_t(w[0]), rsrc, int(offset), 0, kStream);
        } else if constexpr (Count == 8) {
            const i32x2 x = {int32_t(w[0]), int32_t(w[1])};
            if (keep) __builtin_amdgcn_raw_buffer_store_b64(x, rsrc, int(offset), 0, kStay);
            else __builtin_amdgcn_raw_buffer_store_b64(x, rsrc, int(offset), 0, kStream);
        } else {
            static_assert(Count == 16, "a piece of at most 16 bytes");
            const i32x4 x = {int32_t(w[0]), int32_t(w[1]), int32_t(w[2]), int32_t(w[3])};
            if (keep) __builtin_amdgcn_raw_buffer_store_b128(x, rsrc, int(offset), 0, kStay);
            else __builtin_amdgcn_raw_buffer_store_b128(x, rsrc, int(offset), 0, kStream);
        }
    } else if constexpr (Count == 4) {
        typedef uint32_t V __attribute__((aligned(1)));
        *(MRV_GLOBAL V*)(base + offset) = w[0];
    } else if constexpr (Count == 8) {
        typedef typename Unaligned<Align>::v2 V;
        *(MRV_GLOBAL V*)(base + offset) = u32x2{w[0], w[1]};
    } else {
        typedef typename Unaligned<Align>::v4 V;
#pragma unroll
        for (uint32_t i = 0; i < Count / 16; ++i)
            ((MRV_GLOBAL V*)(base + offset))[i] = u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
    }
}
// Eight consecutive elements, through the caches.
template <typename T>
__device__ __forceinline__ void store8(Bytes p, const Raw8<T>& x) {
    store_dwords<8 * sizeof(T), false, sizeof(T)>(p, 0, x.w, true);
}

template <typename T>
__device__ __forceinline__ float load_one(ConstBytes p) {
    return float(*(const MRV_GLOBAL T*)p);
}
template <typename T>
__device__ __forceinline__ void store_one(Bytes p, float x) {
    *(MRV_GLOBAL T*)p = T(x);
}

// The first `have` elements of eight, the others 0 / left alone.
template <typename T>
__device__ __forceinline__ void load_part(ConstBytes p, uint32_t have, float (&f)[8]) {
    if (have == 8u) {
        widen<T>(load8<T, false>(p), f);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) f[i] = i < have ? load_one<T>(p + i * sizeof(T)) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_part(Bytes p, uint32_t have, const float (&f)[8]) {
    if (have == 8u) {
        store8<T>(p, narrow<T>(f));
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i)
            if (i < have) store_one<T>(p + i * sizeof(T), f[i]);
    }
}

// ---- 8 bits ------------------------------------------------------------------------------------

constexpr float kE4m3Max = 448.0f;
constexpr float kInt8Max = 127.0f;
constexpr float kAmaxMin = 0x1p-100f;  // what a scale is made from at least: Q / amax stays finite, a row of zeros needs no case

__device__ __forceinline__ float clamp_to(float x, float limit) {
    return __builtin_fmaxf(__builtin_fminf(x, limit), -limit);
}

// x / y, `inverse` = 1 / y: one correction of the product makes the quotient the rounded one (Markstein 1990), so that a code
// is the one its definition says also where a product's last bit would move it across a border.
__device__ __forceinline__ float quotient(float x, float y, float inverse) {
    const float q = x * inverse;
    return __builtin_fmaf(__builtin_fmaf(-q, y, x), inverse, q);
}

__device__ __forceinline__ uint32_t to_e4m3(float a, float b, float c, float d) {  // at most 448 in magnitude
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return uint32_t(w);
}
__device__ __forceinline__ u32x2 to_e4m3(const float (&f)[8]) {
    return {to_e4m3(f[0], f[1], f[2], f[3]), to_e4m3(f[4], f[5], f[6], f[7])};
}

__device__ __forceinline__ void from_e4m3(u32x2 x, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(x[i]), false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(x[i]), true);
        f[4 * i] = lo[0];
        f[4 * i + 1] = lo[1];
        f[4 * i + 2] = hi[0];
        f[4 * i + 3] = hi[1];
    }
}

__device__ __forceinline__ u32x2 to_int8(const float (&f)[8]) {  // |f| <= 127
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) w |= (uint32_t(int(__builtin_rintf(f[4 * i + j]))) & 0xffu) << (8 * j);
        r[i] = w;
    }
    return r;
}

// |x| as an integer that orders like it, NaN above everything: a maximum over these does not lose a NaN.
__device__ __forceinline__ uint32_t magnitude(float x) {
    return __builtin_bit_cast(uint32_t, x) & 0x7fffffffu;
}

// ---- over the lanes of a wavefront ---------------------------------------------------------------

// Sixteen lanes' values combined, the same bits in each of them: by rotations, after the step of n lanes the values repeat
// every n, so that a lane combines the same pairs as its neighbours.
template <typename V, typename Op>
__device__ __forceinline__ V across_row(V x, Op op) {
    auto turned = [](V v, auto n) {
        const int i = __builtin_bit_cast(int, v);
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(i, i, 0x120 + decltype(n)::value, 0xf, 0xf, false));  // row_ror:n
    };
    x = op(x, turned(x, std::integral_constant<int, 8>()));
    x = op(x, turned(x, std::integral_constant<int, 4>()));
    x = op(x, turned(x, std::integral_constant<int, 2>()));
    return op(x, turned(x, std::integral_constant<int, 1>()));
}
// All 64 lanes' values: the four rows through scalar registers.
template <typename V, typename Op>
__device__ __forceinline__ V across_wave(V x, Op op) {
    if constexpr (sizeof(V) == 4) {
        x = across_row(x, op);
        auto row = [&](int lane) { return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane)); };
        return op(op(row(0), row(16)), op(row(32), row(48)));
    } else {
#pragma unroll
        for (int d = 32; d; d >>= 1) x = op(x, __shfl_xor(x, d, 64));
        return x;
    }
}
struct Plus {
    template <typename V>
    __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Larger {
    __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a > b ? a : b; }
};

}  // namespace fused
}  // namespace vrank
}  // namespace MegRay
