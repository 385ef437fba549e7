// attention_device.hpp -- what the kernels around a quantised key-value cache share: 16-bit and 8-bit types, reductions over
// groups of lanes.
#pragma once

#include <hip/hip_runtime.h>

#include "attention_common.hpp"

namespace fkattn {

using half2_t = _Float16 __attribute__((ext_vector_type(2)));
using half8_t = _Float16 __attribute__((ext_vector_type(8)));
using float2_t = float __attribute__((ext_vector_type(2)));
using float4_t = float __attribute__((ext_vector_type(4)));
using uint2_t = uint32_t __attribute__((ext_vector_type(2)));
using uint4_t = uint32_t __attribute__((ext_vector_type(4)));

constexpr float kTopInt8 = 127.0f, kTopE4M3 = 448.0f;

// Launches a kernel of one argument; the runtime's code, of this launch and not of what was before it.
template <typename A> int launch(void (*kernel)(A), dim3 grid, dim3 block, void* stream, A args, size_t lds = 0) {
    void* ptrs[] = {&args};
    return int(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, ptrs, lds, static_cast<hipStream_t>(stream)));
}

// ---- 16-bit types ----------------------------------------------------------------------------------------------------

// Two elements of a dword as float32, and back (rounded to the nearest, ties to even).
template <int TYPE> __device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
    if constexpr (TYPE == FKLHIP_BF16) {
        a = __builtin_bit_cast(float, w << 16);
        b = __builtin_bit_cast(float, w & 0xffff0000u);
    } else {
        const half2_t h = __builtin_bit_cast(half2_t, w);
        a = float(h.x);
        b = float(h.y);
    }
}
template <int TYPE> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (TYPE == FKLHIP_BF16) {
        using bf2 = __bf16 __attribute__((ext_vector_type(2)));
        const bf2 r = {__bf16(a), __bf16(b)};
        return __builtin_bit_cast(uint32_t, r);
    } else {
        const half2_t r = {_Float16(a), _Float16(b)};
        return __builtin_bit_cast(uint32_t, r);
    }
}

// ---- 8-bit codes -----------------------------------------------------------------------------------------------------

// Four codes of a dword as float32.
template <int CODES> __device__ __forceinline__ void decode4(uint32_t w, float* x) {
    if constexpr (CODES == FKLHIP_CODES_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = float(int32_t(w << (24 - 8 * i)) >> 24);
    } else {
        x[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
    }
}
// Four values that are at most the top code in size (up to rounding) as codes.
template <int CODES> __device__ __forceinline__ uint32_t encode4(const float* x) {
    if constexpr (CODES == FKLHIP_CODES_INT8) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = int(__builtin_rintf(__builtin_amdgcn_fmed3f(x[i], -kTopInt8, kTopInt8)));
            w |= uint32_t(c & 0xff) << (8 * i);
        }
        return w;
    } else {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_amdgcn_fmed3f(x[i], -kTopE4M3, kTopE4M3);
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true));
    }
}

// ---- reductions over a power of two of neighbouring lanes (8, 16 or 32), every lane getting the result ---------------

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t v) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, true));
}
template <int LANES, typename F> __device__ __forceinline__ uint32_t reduce_lanes(uint32_t v, F f) {
    static_assert(LANES == 8 || LANES == 16 || LANES == 32);
    v = f(v, dpp<0xb1>(v));                          // quad_perm [1, 0, 3, 2]
    v = f(v, dpp<0x4e>(v));                          // quad_perm [2, 3, 0, 1]
    v = f(v, dpp<0x141>(v));                         // row_half_mirror: the other quad of eight
    if constexpr (LANES >= 16) v = f(v, dpp<0x140>(v));   // row_mirror: the other half of sixteen
    if constexpr (LANES >= 32) v = f(v, uint32_t(__builtin_amdgcn_ds_swizzle(int(v), 0x401f)));   // xor 16
    return v;
}
template <int LANES> __device__ __forceinline__ float sum_lanes(float v) {
    return __builtin_bit_cast(float, reduce_lanes<LANES>(__builtin_bit_cast(uint32_t, v), [](uint32_t a, uint32_t b) {
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b)); }));
}
template <int LANES> __device__ __forceinline__ uint32_t max_lanes(uint32_t v) {
    return reduce_lanes<LANES>(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// x / n by a multiplication: magic = ceil(2^32 / n), exact for x * n < 2^32 (n = 1: magic 0).
__device__ __forceinline__ uint32_t divide(uint32_t x, uint32_t magic) { return magic ? __umulhi(x, magic) : x; }

} // namespace fkattn
