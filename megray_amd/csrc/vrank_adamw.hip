// The AdamW step over many tensors, and the norm of their gradients (vrank_fused.h).
//
// Both are one pass over the ranks' gradients, which are summed on the way: N reads of a gradient, and for the step one read
// and one write of master, m and v and N writes of the parameter - 4 to 7 bytes per operation, HBM bound.  A workgroup
// takes kAdamTile elements of one tensor (a table says which), a lane eight of them: 16 bytes per access of a
// 16-bit type.  32 lanes hold the 256 elements that share the scale of an 8-bit state, so the block's maximum is a
// reduction over half a wavefront and the new codes leave from the same registers.
#include "vrank_fused_impl.hpp"

namespace MegRay {
namespace vrank {

namespace {

using namespace fused;

// The sum over ranks of `have` elements from element `i` on; `ptrs` are the tensor's buffers.
template <typename G>
__device__ __forceinline__ void fold_grads(const void* const* ptrs, uint32_t nranks, uint64_t i, uint32_t have, float (&g)[8]) {
    constexpr uint32_t C = sizeof(G) == 4 ? 4 : 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = 0.0f;
    if (have == 8) {
        for (uint32_t r0 = 0; r0 < nranks; r0 += C) {
            const uint32_t left = nranks - r0;
            Raw8<G> x[C];
#pragma unroll
            for (uint32_t r = 0; r < C; ++r)  // past the last rank: its buffer again, not added
                x[r] = load8<G, true>(static_cast<const char*>(ptrs[r0 + (r < left ? r : left - 1)]) + i * sizeof(G));
#pragma unroll
            for (uint32_t r = 0; r < C; ++r) {
                if (r < left) {
                    float f[8];
                    widen<G>(x[r], f);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] += f[j];
                }
            }
        }
    } else if (have) {
        for (uint32_t r = 0; r < nranks; ++r) {
            float f[8];
            load_part<G>(static_cast<const char*>(ptrs[r]) + i * sizeof(G), have, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += f[j];
        }
    }
}

__device__ __forceinline__ u32x2 load_codes(const char* p, uint32_t have) {
    if (have == 8) return __builtin_nontemporal_load(as_global<Unaligned<1>::v2>(p));
    u32x2 x = {0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (i < have) x[i / 4] |= uint32_t(*as_global<uint8_t>(p + i)) << (8 * (i % 4));
    return x;
}

__device__ __forceinline__ void store_codes_part(char* p, uint32_t have, u32x2 x) {
    if (have == 8) {
        store_codes(p, x, false);
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (i < have) *as_global<uint8_t>(p + i) = uint8_t(x[i / 4] >> (8 * (i % 4)));
}

// Codes and scale of a block; all 32 lanes of it call this.  KeepAlive: a value above zero gets at least the smallest code, so that a
// root of v that is small beside its block's largest does not vanish from the denominator.
template <bool KeepAlive>
__device__ __forceinline__ u32x2 to_block(const float (&x)[8], float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = Larger()(top, magnitude(x[i]));
    top = across_half(top, Larger());
    float amax = __builtin_bit_cast(float, top);
    if (amax < kAmaxMin) amax = kAmaxMin;  // not true of a NaN
    const bool finite = amax < __builtin_inff();
    scale = amax / kE4m3Max;
    const float inverse = 1.0f / scale;
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        q[i] = clamp_to(quotient(x[i], scale, inverse), kE4m3Max);
        if (KeepAlive && x[i] > 0.0f) q[i] = __builtin_fmaxf(q[i], 0x1p-9f);
    }
    if (!finite) scale = __builtin_nanf("");
    return finite ? to_e4m3(q) : u32x2{0x7f7f7f7fu, 0x7f7f7f7fu};
}

template <typename G, typename P, bool State8>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const AdamLaunch L) {
    float factor = L.grad_scale;
    if (L.clip) {
        const float clip = *L.clip;
        if (!(__builtin_fabsf(clip) < __builtin_inff())) return;
        factor *= clip;
    }
    const AdamTile where = L.tiles[blockIdx.x];
    const AdamTensor t = L.tensors[where.tensor];
    const uint64_t i = uint64_t(where.tile) * kAdamTile + threadIdx.x * kAdamVec;
    const uint32_t have = i >= t.len ? 0u : t.len - i < kAdamVec ? uint32_t(t.len - i) : kAdamVec;
    const uint64_t block = i / kAdamBlock;

    float g[8], m[8], v[8], p[8];
    float m_scale = 0.0f, v_scale = 0.0f;
    u32x2 m_codes = {0, 0}, v_codes = {0, 0};
    if constexpr (State8) {
        if (have) {
            m_codes = load_codes(static_cast<const char*>(t.m) + i, have);
            v_codes = load_codes(static_cast<const char*>(t.v) + i, have);
            m_scale = *as_global<float>(reinterpret_cast<const char*>(t.m_scale + block));
            v_scale = *as_global<float>(reinterpret_cast<const char*>(t.v_scale + block));
        }
    } else {
        load_part<float>(static_cast<const char*>(t.m) + i * 4, have, m);
        load_part<float>(static_cast<const char*>(t.v) + i * 4, have, v);
    }
    load_part<float>(reinterpret_cast<const char*>(t.master + i), have, p);
    fold_grads<G>(L.grads + uint64_t(where.tensor) * L.grad_ranks, L.grad_ranks, i, have, g);
    if constexpr (State8) {
        from_e4m3(m_codes, m);
        from_e4m3(v_codes, v);
    }
    const float shrink = L.lr * t.decay;
    float root[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = g[j] * factor;
        if constexpr (State8) {
            m[j] *= m_scale;
            v[j] *= v_scale;
            v[j] *= v[j];
        }
        m[j] = L.beta1 * m[j] + L.rest1 * x;
        v[j] = L.beta2 * v[j] + L.rest2 * x * x;
        root[j] = __builtin_sqrtf(v[j]);
        const float update = L.rate * m[j] / __builtin_fmaf(root[j], L.root_scale, L.eps);
        p[j] = __builtin_fmaf(-shrink, p[j], p[j]) - update;
    }
    store_part<float>(reinterpret_cast<char*>(t.master + i), have, p, false);
    for (uint32_t r = 0; r < L.param_ranks; ++r) {
        char* q = static_cast<char*>(L.params[uint64_t(where.tensor) * L.param_ranks + r]);
        store_part<P>(q + i * sizeof(P), have, p, false);
    }
    if constexpr (State8) {
        if (have < 8) {  // elements behind the tensor's end do not count for the block's maximum
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (j >= have) m[j] = root[j] = 0.0f;
        }
        m_codes = to_block<false>(m, m_scale);
        v_codes = to_block<true>(root, v_scale);
        if (have) {
            store_codes_part(static_cast<char*>(t.m) + i, have, m_codes);
            store_codes_part(static_cast<char*>(t.v) + i, have, v_codes);
            if (threadIdx.x % (kAdamBlock / kAdamVec) == 0) {
                *as_global<float>(reinterpret_cast<char*>(t.m_scale + block)) = m_scale;
                *as_global<float>(reinterpret_cast<char*>(t.v_scale + block)) = v_scale;
            }
        }
    } else {
        store_part<float>(static_cast<char*>(t.m) + i * 4, have, m, false);
        store_part<float>(static_cast<char*>(t.v) + i * 4, have, v, false);
    }
}

// Sum over a workgroup in a fixed order; the result is valid in lane 0.
template <uint32_t Threads>
__device__ __forceinline__ double workgroup_sum(double x) {
    __shared__ double part[Threads / 64];
    x = across_wave(x, Plus());
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = x;
    __syncthreads();
    x = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < Threads / 64; ++w) x += part[w];
    return x;
}

// Squares are summed in 64 bits: no gradient that is finite in 32 bits overflows, and the number of terms does not matter.
template <typename G>
__global__ void __launch_bounds__(kAdamThreads) adamw_norm_kernel(const AdamNormLaunch L) {
    double sum = 0.0;
    for (uint32_t n = blockIdx.x; n < L.ntiles; n += L.groups) {
        const AdamTile where = L.tiles[n];
        const uint64_t len = L.tensors[where.tensor].len;
        const uint64_t i = uint64_t(where.tile) * kAdamTile + threadIdx.x * kAdamVec;
        const uint32_t have = i >= len ? 0u : len - i < kAdamVec ? uint32_t(len - i) : kAdamVec;
        float g[8];
        fold_grads<G>(L.grads + uint64_t(where.tensor) * L.grad_ranks, L.grad_ranks, i, have, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = double(g[j] * L.grad_scale);
            sum = __builtin_fma(x, x, sum);
        }
    }
    sum = workgroup_sum<kAdamThreads>(sum);
    if (threadIdx.x == 0) reinterpret_cast<double*>(L.out + 2)[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kAdamJoinThreads) adamw_norm_join(const AdamNormLaunch L) {
    double sum = 0.0;
    for (uint32_t n = threadIdx.x; n < L.groups; n += kAdamJoinThreads) sum += reinterpret_cast<const double*>(L.out + 2)[n];
    sum = workgroup_sum<kAdamJoinThreads>(sum);
    if (threadIdx.x == 0) {
        const float norm = float(__builtin_sqrt(sum));
        const float ratio = L.max_norm / (norm + 1e-6f);
        L.out[0] = norm;
        L.out[1] = norm < __builtin_inff() ? (ratio < 1.0f ? ratio : 1.0f) : __builtin_nanf("");
    }
}

template <typename G, typename P>
const void* step_kernel(bool state8) {
    return state8 ? reinterpret_cast<const void*>(&adamw_kernel<G, P, true>) : reinterpret_cast<const void*>(&adamw_kernel<G, P, false>);
}
template <typename G>
const void* step_kernel_for(int param_dtype, bool state8) {
    switch (param_dtype) {
        case MEGRAY_FLOAT16: return step_kernel<G, _Float16>(state8);
        case MRV_BFLOAT16: return step_kernel<G, __bf16>(state8);
        case MEGRAY_FLOAT32: return step_kernel<G, float>(state8);
        default: return nullptr;
    }
}

}  // namespace

const void* adamw_kernel_for(int grad_dtype, int param_dtype, bool state8) {
    switch (grad_dtype) {
        case MEGRAY_FLOAT16: return step_kernel_for<_Float16>(param_dtype, state8);
        case MRV_BFLOAT16: return step_kernel_for<__bf16>(param_dtype, state8);
        case MEGRAY_FLOAT32: return step_kernel_for<float>(param_dtype, state8);
        default: return nullptr;
    }
}

const void* adamw_norm_kernel_for(int grad_dtype) {
    switch (grad_dtype) {
        case MEGRAY_FLOAT16: return reinterpret_cast<const void*>(&adamw_norm_kernel<_Float16>);
        case MRV_BFLOAT16: return reinterpret_cast<const void*>(&adamw_norm_kernel<__bf16>);
        case MEGRAY_FLOAT32: return reinterpret_cast<const void*>(&adamw_norm_kernel<float>);
        default: return nullptr;
    }
}

const void* adamw_norm_join_kernel() {
    return reinterpret_cast<const void*>(&adamw_norm_join);
}

}  // namespace vrank
}  // namespace MegRay
