// The AdamW step over many tensors, and the norm of their gradients (vrank_fused.h).
//
// Both are one pass over the ranks' gradients, which are summed on the way: N reads of a gradient, and for the step one read
// and one write of master, m and v and N writes of the parameter - 4 to 7 bytes per operation, HBM bound.  A workgroup
// takes a tile of one tensor (a table says which); a wavefront takes 512 elements, a lane two pieces of four, 256 apart (see
// Raw8).  So a piece of a wavefront is just the 256 elements that share the scale of an 8-bit state: their maximum is
// one reduction across it, and the new codes leave from the same registers.
//
// Measured, BF16 gradients and parameters: 8 ranks, 98 M parameters, 32-bit states 1037 us (5.5 GB, 5.31 TB/s); 1 rank, 157 M 709 us (6.21
// TB/s); 4 ranks, 50 M in tensors that begin off the cache lines, 8-bit states 274 us (5.2 TB/s); the norm of 8 ranks' 98 M 236 us (6.7 TB/s).  A
// step that walks its tiles and loads the next one before it stores this one is slower (1215 us: it leaves fewer wavefronts), and so are
// half the loads in flight (1108 us), tiles of a workgroup 32 apart (1196) and stores whose ranks begin elsewhere in each tile (1045).
#include "vrank_fused_impl.hpp"

namespace MegRay {
namespace vrank {

namespace {

using namespace fused;

// The elements of a tensor that a lane works on.
struct Elements {
    uint64_t at[2];    // first element of each piece of four
    uint32_t have[2];  // how many of the four are there
    __device__ __forceinline__ Elements(uint64_t tile_at, uint64_t len) {  // the workgroup's first element
        const uint64_t first = tile_at + threadIdx.x / 64 * 512u + threadIdx.x % 64 * 4u;
#pragma unroll
        for (uint32_t p = 0; p < 2; ++p) {
            at[p] = first + p * kAdamBlock;
            have[p] = at[p] >= len ? 0u : len - at[p] < 4 ? uint32_t(len - at[p]) : 4u;
        }
    }
    __device__ __forceinline__ bool whole() const { return have[1] == 4; }
    template <typename T, bool Once>
    __device__ __forceinline__ Raw8<T> load(ConstBytes base) const {  // whole() lanes only
        return load44<T, Once>(base + at[0] * sizeof(T), base + at[1] * sizeof(T));
    }
    template <typename T>
    __device__ __forceinline__ void load_some(ConstBytes base, float (&f)[8]) const {
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) f[i] = i % 4 < have[i / 4] ? load_one<T>(base + (at[i / 4] + i % 4) * sizeof(T)) : 0.0f;
    }
    // `Size` bytes per element; `tile_at`: the workgroup's first element
    template <uint32_t Size, bool Lines>
    __device__ __forceinline__ void store(Bytes base, uint64_t tile_at, const uint32_t* w, bool keep) const {
        if (whole()) {
            const Bytes tile = base + tile_at * Size;  // the same for the whole wavefront
#pragma unroll
            for (uint32_t p = 0; p < 2; ++p) store_dwords<4 * Size, Lines, Size>(tile, uint32_t(at[p] - tile_at) * Size, w + p * Size, keep);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (i % 4 >= have[i / 4]) continue;
                const Bytes q = base + (at[i / 4] + i % 4) * Size;
                if constexpr (Size == 4) *(MRV_GLOBAL uint32_t*)q = w[i];
                else if constexpr (Size == 2) *(MRV_GLOBAL uint16_t*)q = uint16_t(w[i / 2] >> (16 * (i % 2)));
                else *(MRV_GLOBAL uint8_t*)q = uint8_t(w[i / 4] >> (8 * (i % 4)));
            }
        }
    }
};

// The sum over ranks of a lane's elements; `ptrs` are the tensor's buffers.
template <typename G, bool Once>
__device__ __forceinline__ void fold_grads(const void* const* ptrs, uint32_t nranks, const Elements& e, float (&g)[8]) {
    constexpr uint32_t C = sizeof(G) == 4 ? 4 : 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] = 0.0f;
    if (e.whole()) {
        for (uint32_t r0 = 0; r0 < nranks; r0 += C) {
            const uint32_t left = nranks - r0;
            Raw8<G> x[C];
#pragma unroll
            for (uint32_t r = 0; r < C; ++r)
                if (r < left) x[r] = e.load<G, Once>(bytes_of(ptrs[r0 + r]));
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
    } else if (e.have[0]) {
        for (uint32_t r = 0; r < nranks; ++r) {
            float f[8];
            e.load_some<G>(bytes_of(ptrs[r]), f);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] += f[j];
        }
    }
}

// Codes and scale of a block, four elements of it in each lane.  KeepAlive: a value above zero gets at least the smallest code, so
// that a root of v that is small beside its block's largest does not vanish from the denominator.
template <bool KeepAlive>
__device__ __forceinline__ uint32_t to_block(const float* x, float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = Larger()(top, magnitude(x[i]));
    float amax = __builtin_bit_cast(float, across_wave(top, Larger()));
    if (amax < kAmaxMin) amax = kAmaxMin;  // not true of a NaN
    const bool finite = amax < __builtin_inff();
    scale = amax * (1.0f / kE4m3Max);
    const float inverse = 1.0f / scale;
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        q[i] = clamp_to(quotient(x[i], scale, inverse), kE4m3Max);
        if (KeepAlive && x[i] > 0.0f) q[i] = __builtin_fmaxf(q[i], 0x1p-9f);
    }
    if (!finite) scale = __builtin_nanf("");
    return finite ? to_e4m3(q[0], q[1], q[2], q[3]) : 0x7f7f7f7fu;
}

template <bool State8>
constexpr uint32_t kThreads = State8 ? kAdamThreads8 : kAdamThreads;

// Lines: the tensor's buffers all begin on a cache line.
template <typename G, typename P, bool State8, bool Lines>
__device__ __forceinline__ void adamw_tile(const AdamLaunch& L, const AdamTensor& t, uint32_t tensor, uint32_t tile, float factor) {
    const uint64_t tile_at = uint64_t(tile) * (kThreads<State8> * kAdamVec);
    const Elements e(tile_at, t.len);
    const uint64_t block = tile_at / kAdamBlock + __builtin_amdgcn_readfirstlane(threadIdx.x / 64) * 2;

    float g[8], m[8], v[8], p[8];
    uint32_t m_codes[2] = {0, 0}, v_codes[2] = {0, 0};
    float m_scale[2] = {0.0f, 0.0f}, v_scale[2] = {0.0f, 0.0f};
    if (e.whole()) {
        Raw8<float> pr = e.load<float, Lines>(bytes_of(t.master)), mr, vr;
        if constexpr (State8) {
            typedef uint32_t V __attribute__((aligned(1)));
#pragma unroll
            for (uint32_t q = 0; q < 2; ++q) {
                m_codes[q] = *(const MRV_GLOBAL V*)(bytes_of(t.m) + e.at[q]);
                v_codes[q] = *(const MRV_GLOBAL V*)(bytes_of(t.v) + e.at[q]);
            }
        } else {
            mr = e.load<float, Lines>(bytes_of(t.m));
            vr = e.load<float, Lines>(bytes_of(t.v));
        }
        widen<float>(pr, p);
        if constexpr (!State8) {
            widen<float>(mr, m);
            widen<float>(vr, v);
        }
    } else {
        e.load_some<float>(bytes_of(t.master), p);
        if constexpr (State8) {
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) {
                if (i % 4 >= e.have[i / 4]) continue;
                m_codes[i / 4] |= uint32_t(*(const MRV_GLOBAL uint8_t*)(bytes_of(t.m) + e.at[i / 4] + i % 4)) << (8 * (i % 4));
                v_codes[i / 4] |= uint32_t(*(const MRV_GLOBAL uint8_t*)(bytes_of(t.v) + e.at[i / 4] + i % 4)) << (8 * (i % 4));
            }
        } else {
            e.load_some<float>(bytes_of(t.m), m);
            e.load_some<float>(bytes_of(t.v), v);
        }
    }
    if constexpr (State8) {
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) {
            if ((block + q) * kAdamBlock < t.len) {
                m_scale[q] = load_one<float>(bytes_of(t.m_scale + block + q));
                v_scale[q] = load_one<float>(bytes_of(t.v_scale + block + q));
            }
        }
    }
    fold_grads<G, Lines>(L.grads + uint64_t(tensor) * L.grad_ranks, L.grad_ranks, e, g);
    if constexpr (State8) {
        from_e4m3(u32x2{m_codes[0], m_codes[1]}, m);
        from_e4m3(u32x2{v_codes[0], v_codes[1]}, v);
    }
    const float shrink = L.lr * t.decay;
    float root[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = g[j] * factor;
        if constexpr (State8) {
            m[j] *= m_scale[j / 4];
            v[j] *= v_scale[j / 4];
            v[j] *= v[j];
        }
        m[j] = L.beta1 * m[j] + L.rest1 * x;
        v[j] = L.beta2 * v[j] + L.rest2 * x * x;
        root[j] = __builtin_sqrtf(v[j]);
        const float update = L.rate * m[j] / __builtin_fmaf(root[j], L.root_scale, L.eps);
        p[j] = __builtin_fmaf(-shrink, p[j], p[j]) - update;
    }
    e.store<4, Lines>(bytes_of(t.master), tile_at, narrow<float>(p).w, L.keep);
    L.pace.wait();
    const Raw8<P> param = narrow<P>(p);
    for (uint32_t r = 0; r < L.param_ranks; ++r) {
        e.store<sizeof(P), Lines>(bytes_of(L.params[uint64_t(tensor) * L.param_ranks + r]), tile_at, param.w, L.keep);
        L.pace.wait();
    }
    if constexpr (State8) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)  // elements behind the tensor's end do not count for the block's maximum
            if (j % 4 >= e.have[j / 4]) m[j] = root[j] = 0.0f;
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) {
            m_codes[q] = to_block<false>(m + 4 * q, m_scale[q]);
            v_codes[q] = to_block<true>(root + 4 * q, v_scale[q]);
            if (threadIdx.x % 64 == 0 && (block + q) * kAdamBlock < t.len) {
                store_one<float>(bytes_of(t.m_scale + block + q), m_scale[q]);
                store_one<float>(bytes_of(t.v_scale + block + q), v_scale[q]);
            }
        }
        e.store<1, Lines>(bytes_of(t.m), tile_at, m_codes, L.keep);
        e.store<1, Lines>(bytes_of(t.v), tile_at, v_codes, L.keep);
    } else {
        e.store<4, Lines>(bytes_of(t.m), tile_at, narrow<float>(m).w, L.keep);
        L.pace.wait();
        e.store<4, Lines>(bytes_of(t.v), tile_at, narrow<float>(v).w, L.keep);
    }
}

template <typename G, typename P, bool State8>
__global__ void __launch_bounds__(kThreads<State8>) adamw_kernel(const AdamLaunch L) {
    float factor = L.grad_scale;
    if (L.clip) {
        const float clip = *L.clip;
        if (!(__builtin_fabsf(clip) < __builtin_inff())) return;
        factor *= clip;
    }
    const AdamTile where = L.tiles[L.deal.of(blockIdx.x)];
    const AdamTensor t = L.tensors[where.tensor];
    if (t.lines) adamw_tile<G, P, State8, true>(L, t, where.tensor, where.tile, factor);
    else adamw_tile<G, P, State8, false>(L, t, where.tensor, where.tile, factor);
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

// Squares are summed in 64 bits: no gradient that is finite in 32 bits overflows, and the number of terms does not matter.  The gradients are loaded as
// data that need not stay in the caches; the step that follows reads them again, of a large model (1.5 GB above) from memory either way.
template <typename G>
__global__ void __launch_bounds__(kAdamNormThreads) adamw_norm_kernel(const AdamNormLaunch L) {
    double sum = 0.0;
    for (uint32_t n = blockIdx.x; n < L.ntiles; n += L.groups) {
        const AdamTile where = L.tiles[L.deal.of(n)];
        const Elements e(uint64_t(where.tile) * (kAdamNormThreads * kAdamVec), L.tensors[where.tensor].len);
        float g[8];
        fold_grads<G, true>(L.grads + uint64_t(where.tensor) * L.grad_ranks, L.grad_ranks, e, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = double(g[j] * L.grad_scale);
            sum = __builtin_fma(x, x, sum);
        }
    }
    sum = workgroup_sum<kAdamNormThreads>(sum);
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
