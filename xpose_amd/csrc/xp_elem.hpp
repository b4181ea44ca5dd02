// Elements of rows and caches as 32-bit floats, eight at a time.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "xp_device.hpp"
#include "xp_rows.hpp"

namespace xp {

typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float f16_lo(uint32_t w) { return f16_bits_to_f32(w & 0xFFFFu); }
__device__ __forceinline__ float f16_hi(uint32_t w) { return f16_bits_to_f32(w >> 16); }
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return uint32_t(f32_to_f16_bits(a)) | (uint32_t(f32_to_f16_bits(b)) << 16);
}
// Two floats to bf16, to nearest even; a NaN stays one.
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v{a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}

template <int ELEM>
__device__ __forceinline__ float load1(const void* base, uint64_t i) {
    if constexpr (ELEM == XP_ELEM_F32) return static_cast<const float*>(base)[i];
    else if constexpr (ELEM == XP_ELEM_F16) return f16_bits_to_f32(static_cast<const uint16_t*>(base)[i]);
    else if constexpr (ELEM == XP_ELEM_BF16) return bf16lo(static_cast<const uint16_t*>(base)[i]);
    else if constexpr (ELEM == XP_ELEM_I8) return float(static_cast<const int8_t*>(base)[i]);
    else return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(base)[i], 0);
}
template <int ELEM>
__device__ __forceinline__ void store1(void* base, uint64_t i, float x) {
    if constexpr (ELEM == XP_ELEM_F32) static_cast<float*>(base)[i] = x;
    else if constexpr (ELEM == XP_ELEM_F16) static_cast<uint16_t*>(base)[i] = f32_to_f16_bits(x);
    else static_cast<uint16_t*>(base)[i] = uint16_t(pack_bf16(x, x));
}

// Eight elements as they lie in memory: 32 bytes of f32, 16 of 16 bits, 8 of 8 bits,
// aligned to that or to 16.
template <int ELEM>
struct Raw8 {
    u32x4 a, b;
    __device__ __forceinline__ void load(const void* base, uint64_t i) {
        const u32x4* p = reinterpret_cast<const u32x4*>(static_cast<const float*>(base) + i);
        a = p[0];
        b = p[1];
    }
    __device__ __forceinline__ void zero() { a = b = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(a[j]), x[4 + j] = __uint_as_float(b[j]);
    }
};
template <bool F16>
struct Raw8x16 {
    u32x4 a;
    __device__ __forceinline__ void load(const void* base, uint64_t i) {
        a = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + i);
    }
    __device__ __forceinline__ void zero() { a = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = F16 ? f16_lo(a[j]) : bf16lo(a[j]);
            x[2 * j + 1] = F16 ? f16_hi(a[j]) : bf16hi(a[j]);
        }
    }
};
template <bool I8>
struct Raw8x8 {
    u32x2 a;
    __device__ __forceinline__ void load(const void* base, uint64_t i) {
        a = *reinterpret_cast<const u32x2*>(static_cast<const uint8_t*>(base) + i);
    }
    __device__ __forceinline__ void zero() { a = u32x2{0u, 0u}; }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            if constexpr (I8) {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * w + j] = float(int8_t(a[w] >> (8 * j)));
            } else {
                const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(int(a[w]), false);
                const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8(int(a[w]), true);
                x[4 * w] = lo[0], x[4 * w + 1] = lo[1], x[4 * w + 2] = hi[0], x[4 * w + 3] = hi[1];
            }
        }
    }
};
template <> struct Raw8<XP_ELEM_F16> : Raw8x16<true> {};
template <> struct Raw8<XP_ELEM_BF16> : Raw8x16<false> {};
template <> struct Raw8<XP_ELEM_I8> : Raw8x8<true> {};
template <> struct Raw8<XP_ELEM_E4M3> : Raw8x8<false> {};

template <int ELEM>
__device__ __forceinline__ void load8(const void* base, uint64_t i, float (&x)[8]) {
    Raw8<ELEM> r;
    r.load(base, i);
    r.floats(x);
}
template <int ELEM>
__device__ __forceinline__ void store8(void* base, uint64_t i, const float (&x)[8]) {
    if constexpr (ELEM == XP_ELEM_F32) {
        u32x4* p = reinterpret_cast<u32x4*>(static_cast<float*>(base) + i);
        u32x4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] = __float_as_uint(x[j]), b[j] = __float_as_uint(x[4 + j]);
        p[0] = a;
        p[1] = b;
    } else {
        static_assert(ELEM == XP_ELEM_F16 || ELEM == XP_ELEM_BF16, "8-bit rows need their scale");
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            a[j] = ELEM == XP_ELEM_F16 ? pack_f16(x[2 * j], x[2 * j + 1]) : pack_bf16(x[2 * j], x[2 * j + 1]);
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + i) = a;
    }
}

}  // namespace xp
