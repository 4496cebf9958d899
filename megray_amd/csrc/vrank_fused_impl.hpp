// Device helpers of the folds with an epilogue: eight elements of a row or tensor at a time.
//
// Rows and tensors start anywhere: the 128-bit global accesses of gfx950 take any element boundary, so one code path
// serves every alignment (an access off the 16-byte grid costs its wavefront one more cache line, nothing else).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "vrank_fused.h"

namespace MegRay {
namespace vrank {
namespace fused {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <int Align>
struct Unaligned;
template <>
struct Unaligned<1> {
    typedef u32x4 v4 __attribute__((aligned(1)));
    typedef u32x2 v2 __attribute__((aligned(1)));
};
template <>
struct Unaligned<2> {
    typedef u32x4 v4 __attribute__((aligned(2)));
};
template <>
struct Unaligned<4> {
    typedef u32x4 v4 __attribute__((aligned(4)));
};

// Pointers out of a descriptor or a table are global memory; saying so keeps flat instructions out of the kernels.
#define MRV_GLOBAL __attribute__((address_space(1)))
template <typename V>
__device__ __forceinline__ const MRV_GLOBAL V* as_global(const char* p) {
    return (const MRV_GLOBAL V*)(uintptr_t)p;
}
template <typename V>
__device__ __forceinline__ MRV_GLOBAL V* as_global(char* p) {
    return (MRV_GLOBAL V*)(uintptr_t)p;
}

// Eight elements of T as they lie in memory.
template <typename T>
struct Raw8 {
    u32x4 q[sizeof(T) / 2];
};

// `once`: the data is read by no one else soon, so it need not stay in the caches.
template <typename T, bool Once>
__device__ __forceinline__ Raw8<T> load8(const char* p) {
    typedef typename Unaligned<sizeof(T)>::v4 V;
    Raw8<T> x;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 2; ++i) {
        if constexpr (Once) x.q[i] = __builtin_nontemporal_load(as_global<V>(p) + i);
        else x.q[i] = as_global<V>(p)[i];
    }
    return x;
}

template <typename T>
__device__ __forceinline__ void widen(const Raw8<T>& x, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __builtin_bit_cast(float, uint32_t(x.q[i / 4][i % 4]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = x.q[0][i];
            if constexpr (__is_same(T, __bf16)) {
                f[2 * i] = __builtin_bit_cast(float, w << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, w & 0xffff0000u);
            } else {
                f[2 * i] = float(__builtin_bit_cast(_Float16, uint16_t(w)));
                f[2 * i + 1] = float(__builtin_bit_cast(_Float16, uint16_t(w >> 16)));
            }
        }
    }
}

template <typename T>
__device__ __forceinline__ Raw8<T> narrow(const float (&f)[8]) {
    Raw8<T> x;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x.q[i / 4][i % 4] = __builtin_bit_cast(uint32_t, f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            typedef T Pair __attribute__((ext_vector_type(2)));
            typedef float Wide __attribute__((ext_vector_type(2)));
            x.q[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((Wide{f[2 * i], f[2 * i + 1]}), Pair));
        }
    }
    return x;
}

template <typename T>
__device__ __forceinline__ void store8(char* p, const Raw8<T>& x, bool keep) {
    typedef typename Unaligned<sizeof(T)>::v4 V;
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 2; ++i) {
        if (keep) as_global<V>(p)[i] = x.q[i];
        else __builtin_nontemporal_store(x.q[i], as_global<V>(p) + i);
    }
}

// Row stores.  Rows on cache lines go past the caches like the collectives' own results (or stay in the last-level cache:
// `keep`); others leave lines that two wavefronts, or two rows, write a part of, and those are put together in the L2.
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
constexpr int kStream = 18;  // sc1 | nt
constexpr int kStay = 16;    // sc1
template <typename T, bool Lines>
__device__ __forceinline__ void store_row(char* row, uint32_t offset, const Raw8<T>& x, bool keep) {
    if constexpr (Lines) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(row, 0, -1, 0x00020000);
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i) {
            if (keep) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, x.q[i]), rsrc, int(offset + 16 * i), 0, kStay);
            else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(i32x4, x.q[i]), rsrc, int(offset + 16 * i), 0, kStream);
        }
    } else {
        store8<T>(row + offset, x, true);
    }
}

__device__ __forceinline__ void store_codes(char* p, u32x2 x, bool keep) {
    typedef Unaligned<1>::v2 V;
    if (keep) *as_global<V>(p) = x;
    else __builtin_nontemporal_store(x, as_global<V>(p));
}

template <bool Lines>
__device__ __forceinline__ void store_row_codes(char* row, uint32_t offset, u32x2 x, bool keep) {
    if constexpr (Lines) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(row, 0, -1, 0x00020000);
        if (keep) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i32x2, x), rsrc, int(offset), 0, kStay);
        else __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(i32x2, x), rsrc, int(offset), 0, kStream);
    } else {
        store_codes(row + offset, x, true);
    }
}

template <typename T>
__device__ __forceinline__ float load_one(const char* p) {
    return float(*as_global<T>(p));
}
template <typename T>
__device__ __forceinline__ void store_one(char* p, float x) {
    *as_global<T>(p) = T(x);
}

// The first `have` elements of eight, the others 0 / left alone.
template <typename T>
__device__ __forceinline__ void load_part(const char* p, uint32_t have, float (&f)[8]) {
    if (have == 8u) {
        widen<T>(load8<T, true>(p), f);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) f[i] = i < have ? load_one<T>(p + i * sizeof(T)) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ void store_part(char* p, uint32_t have, const float (&f)[8], bool keep) {
    if (have == 8u) {
        store8<T>(p, narrow<T>(f), keep);
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

__device__ __forceinline__ u32x2 to_e4m3(const float (&f)[8]) {  // |f| <= 448
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], w, true);
        r[i] = uint32_t(w);
    }
    return r;
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

template <typename V, typename Op>
__device__ __forceinline__ V across_half(V x, Op op) {  // over 32 lanes, the same in each of them
#pragma unroll
    for (int d = 16; d; d >>= 1) x = op(x, __shfl_xor(x, d, 64));
    return x;
}
template <typename V, typename Op>
__device__ __forceinline__ V across_wave(V x, Op op) {
    x = across_half(x, op);
    return op(x, __shfl_xor(x, 32, 64));
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
