// Device helpers of the head's kernels: 16-bit and f32 elements in runs of eight, at any alignment.
#pragma once

#include <hip/hip_runtime.h>

#include "head.h"

namespace lg {
namespace head_detail {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Vectors in memory at any byte address: gfx950 loads and stores them whole, aligned or not.
typedef u32x2 u32x2_any __attribute__((aligned(1)));
typedef u32x4 u32x4_any __attribute__((aligned(1)));

template <uint32_t DT>
constexpr uint32_t elem_size = DT == LG_DTYPE_F32 ? 4 : 2;

// One element as f32, from its bits.
template <uint32_t DT>
__device__ inline float widen(uint32_t bits) {
    if constexpr (DT == LG_DTYPE_F32) {
        return __uint_as_float(bits);
    } else if constexpr (DT == LG_DTYPE_BF16) {
        return __uint_as_float(bits << 16);
    } else {
        return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
    }
}

// One element at p; the address is a multiple of the element's size.
template <uint32_t DT>
__device__ inline float load_one(const char* p) {
    if constexpr (DT == LG_DTYPE_F32) {
        return *reinterpret_cast<const float*>(p);
    } else {
        return widen<DT>(*reinterpret_cast<const uint16_t*>(p));
    }
}

template <uint32_t DT>
__device__ inline void store_one(char* p, float v) {
    if constexpr (DT == LG_DTYPE_F32) {
        *reinterpret_cast<float*>(p) = v;
    } else if constexpr (DT == LG_DTYPE_BF16) {
        *reinterpret_cast<__bf16*>(p) = static_cast<__bf16>(v);  // to nearest, ties to even
    } else {
        *reinterpret_cast<_Float16*>(p) = static_cast<_Float16>(v);
    }
}

// Eight consecutive elements as they lie in memory.
template <uint32_t DT>
struct Run {
    u32x4 w[elem_size<DT> / 2];

    __device__ inline void load(const char* p) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(elem_size<DT> / 2); ++i) w[i] = *reinterpret_cast<const u32x4_any*>(p + 16 * i);
    }
    // Elements are widened from here on again, and not held as f32 since an earlier use.
    __device__ inline void keep() {
#pragma unroll
        for (int i = 0; i < static_cast<int>(elem_size<DT> / 2); ++i) __asm__ volatile("" : "+v"(w[i]));
    }
    // Eight times -inf.
    __device__ inline void clear() {
        const uint32_t none = DT == LG_DTYPE_F32 ? 0xff800000u : DT == LG_DTYPE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
        for (int i = 0; i < static_cast<int>(elem_size<DT> / 2); ++i) w[i] = u32x4{none, none, none, none};
    }
    __device__ inline float operator[](int e) const {
        if constexpr (DT == LG_DTYPE_F32) {
            return __uint_as_float(w[e / 4][e % 4]);
        } else if constexpr (DT == LG_DTYPE_BF16) {
            const uint32_t v = w[0][e / 2];
            return __uint_as_float(e % 2 ? v & 0xffff0000u : v << 16);
        } else {
            const uint32_t v = w[0][e / 2];
            return widen<DT>(e % 2 ? v >> 16 : v & 0xffffu);
        }
    }
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Two f32 values rounded to the 16-bit type, to nearest, ties to even, in one word.
template <uint32_t DT>
__device__ inline uint32_t pack2(float a, float b) {
    if constexpr (DT == LG_DTYPE_BF16) {
        const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    } else {
        const f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    }
}

template <uint32_t DT>
__device__ inline void store_run(char* p, const float (&v)[8]) {
    if constexpr (DT == LG_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __float_as_uint(v[4 * i + e]);
            *reinterpret_cast<u32x4_any*>(p + 16 * i) = o;
        }
    } else {
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(v[2 * e], v[2 * e + 1]);
        *reinterpret_cast<u32x4_any*>(p) = o;
    }
}

// A lane's value moved within the wave by a data-parallel step; `otherwise` where the step has no source.
template <int STEP, int ROWS>
__device__ inline float moved(float v, float otherwise) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(otherwise), __float_as_int(v), STEP, ROWS, 0xf, false));
}
template <int STEP, int ROWS>
__device__ inline double moved(double v, double otherwise) {
    const uint64_t a = __builtin_bit_cast(uint64_t, v), b = __builtin_bit_cast(uint64_t, otherwise);
    const int lo = __builtin_amdgcn_update_dpp(static_cast<int>(b), static_cast<int>(a), STEP, ROWS, 0xf, false);
    const int hi = __builtin_amdgcn_update_dpp(static_cast<int>(b >> 32), static_cast<int>(a >> 32), STEP, ROWS, 0xf, false);
    return __builtin_bit_cast(double, static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo));
}
// Shifts by 1, 2, 4 and 8 within rows of sixteen lanes, then the last lane of a row to the next and of the lower half to
// the upper: lane 63 ends with all. Every lane returns it.
__device__ inline float wave_max(float v) {
    v = fmaxf(v, moved<0x111, 0xf>(v, v));
    v = fmaxf(v, moved<0x112, 0xf>(v, v));
    v = fmaxf(v, moved<0x114, 0xf>(v, v));
    v = fmaxf(v, moved<0x118, 0xf>(v, v));
    v = fmaxf(v, moved<0x142, 0xa>(v, v));
    v = fmaxf(v, moved<0x143, 0xc>(v, v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ inline double wave_sum(double v) {
    v += moved<0x111, 0xf>(v, 0.0);
    v += moved<0x112, 0xf>(v, 0.0);
    v += moved<0x114, 0xf>(v, 0.0);
    v += moved<0x118, 0xf>(v, 0.0);
    v += moved<0x142, 0xa>(v, 0.0);
    v += moved<0x143, 0xc>(v, 0.0);
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b), 63));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(b >> 32), 63));
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ inline uint32_t wave_sum(uint32_t u) {
    int v = static_cast<int>(u);
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, 63));
}

inline void launched(Context* ctx, const char* name) {
    check_hip(hipGetLastError(), name);
    note_launch(ctx, name);
}

}  // namespace head_detail
}  // namespace lg
