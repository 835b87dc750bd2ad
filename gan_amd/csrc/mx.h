// Element types (fp32, bf16, fp16) and the microscaled formats of the norm / product / loss kernels.
//
// A microscaled block is 32 values along the contraction axis that share one power-of-two scale, held as the byte e + 127:
// e4m3 elements one byte each (largest 448), e2m1 elements four bits each (largest 6; the first of two in the low half).
// e is the smallest integer in [-126, 127] with max |x| <= largest * 2^e, so no element saturates and the gradient of the
// quantiser can be passed straight through without a mask.  A block that holds an infinity or a NaN has scale byte 255 and
// stands for NaN in all its values.  An all-zero block has scale byte 1.
#pragma once
#include <atomic>
#include <type_traits>

#include "common.h"

namespace gan {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8), aligned(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Vec8;
template <> struct Vec8<float> { typedef f32x8 type; };
template <> struct Vec8<bf16_t> { typedef bf16x8 type; };
template <> struct Vec8<f16_t> { typedef f16x8 type; };

inline size_t dtype_bytes(int dtype) { return dtype == GAN_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == GAN_F32 || dtype == GAN_BF16 || dtype == GAN_F16; }
inline bool mx_fmt_ok(int fmt) { return fmt == GAN_MX_E4M3 || fmt == GAN_MX_E2M1; }
inline bool aligned16(const void* p) { return (reinterpret_cast<size_t>(p) & 15) == 0; }
// Rows of microscaled values are filled up with zeros to whole groups of 128 (4 blocks), the step of the products.
__host__ __device__ __forceinline__ int mx_groups(int c) { return (c + 127) / 128; }

// Eight consecutive values from index i0 of a row of c; 0 beyond its end.  `vec`: the row is 16-byte aligned, so whole
// chunks load at once.
template <typename T>
__device__ __forceinline__ void load8(const T* __restrict__ row, int i0, int c, bool vec, float (&v)[8]) {
    if (vec && i0 + 8 <= c) {
        const typename Vec8<T>::type t = *reinterpret_cast<const typename Vec8<T>::type*>(row + i0);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)t[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = i0 + j < c ? (float)row[i0 + j] : 0.f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* __restrict__ row, int i0, int c, bool vec, const float (&v)[8]) {
    if (vec && i0 + 8 <= c) {
        typename Vec8<T>::type t;
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = (T)v[j];
        *reinterpret_cast<typename Vec8<T>::type*>(row + i0) = t;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i0 + j < c) row[i0 + j] = (T)v[j];
    }
}

// Reductions over the 64 lanes of a wave, the result in all of them: four steps inside the rows of 16 lanes as operand swizzles
// (neighbour, pair, mirrored half row, mirrored row), then the four rows by scalar reads.  No trip through LDS.
template <int CTRL>
__device__ __forceinline__ float row_swizzle(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ double row_swizzle(double v) {
    const long u = __builtin_bit_cast(long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_mov_dpp((int)u, CTRL, 0xf, 0xf, true);
    const unsigned hi = (unsigned)__builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xf, 0xf, true);
    return __builtin_bit_cast(double, (unsigned long)hi << 32 | lo);
}
__device__ __forceinline__ float from_lane(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ double from_lane(double v, int lane) {
    const long u = __builtin_bit_cast(long, v);
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)u, lane), hi = (unsigned)__builtin_amdgcn_readlane((int)(u >> 32), lane);
    return __builtin_bit_cast(double, (unsigned long)hi << 32 | lo);
}
template <typename S>
__device__ __forceinline__ S wave_all_sum(S v) {
    v += row_swizzle<0xb1>(v);
    v += row_swizzle<0x4e>(v);
    v += row_swizzle<0x141>(v);
    v += row_swizzle<0x140>(v);
    return (from_lane(v, 0) + from_lane(v, 16)) + (from_lane(v, 32) + from_lane(v, 48));
}
__device__ __forceinline__ float wave_all_max(float v) {
    v = fmaxf(v, row_swizzle<0xb1>(v));
    v = fmaxf(v, row_swizzle<0x4e>(v));
    v = fmaxf(v, row_swizzle<0x141>(v));
    v = fmaxf(v, row_swizzle<0x140>(v));
    return fmaxf(fmaxf(from_lane(v, 0), from_lane(v, 16)), fmaxf(from_lane(v, 32), from_lane(v, 48)));
}

// |x| as an ordered integer: NaN > infinity > every number, so the maximum over a block tells all three apart.
__device__ __forceinline__ unsigned mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Scale byte of a block whose largest magnitude has the bits `a`.
template <int FMT>
__device__ __forceinline__ unsigned mx_scale_byte(unsigned a) {
    if (a >= 0x7f800000u) return 255u;
    // largest element value: 1.75 * 2^8 (e4m3), 1.5 * 2^2 (e2m1)
    const int e = (int)(a >> 23) - 127 - (FMT == GAN_MX_E4M3 ? 8 : 2) +
                  ((a & 0x7fffffu) > (FMT == GAN_MX_E4M3 ? 0x600000u : 0x400000u) ? 1 : 0);
    return (unsigned)((e < -126 ? -126 : e) + 127);
}

// 2^-e of a scale byte in 1..254 (NaN for 255): what the block's values are multiplied by, exactly, before rounding.
__device__ __forceinline__ float mx_inverse_scale(unsigned byte) {
    return byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - byte) << 23);
}
// 2^e of a scale byte (NaN for 255, the subnormal 2^-127 for 0)
__device__ __forceinline__ float mx_scale(unsigned byte) {
    return __uint_as_float(byte == 255u ? 0x7fc00000u : byte == 0u ? 0x400000u : byte << 23);
}

// Four / eight scaled values to one dword of codes, round to nearest even.
__device__ __forceinline__ unsigned pack_e4m3(float a, float b, float c, float d) {
    int u = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, u, true);
}
__device__ __forceinline__ unsigned pack_e2m1(const float* v) {
    unsigned u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], 1.f, 0);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[2], v[3], 1.f, 1);
    u = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[4], v[5], 1.f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(u, v[6], v[7], 1.f, 3);
}

// Eight codes to eight bf16 values, scale included.  Exact: an element has at most 4 significant bits, the scale is a power of
// two (products below bf16's smallest normal value may round).  `u`: one dword of e2m1 codes, or two of e4m3 codes.
__device__ __forceinline__ bf16x8 e2m1_to_bf16(unsigned u, float scale) {
    bf16x8 r;
    bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 0);
    r[0] = t[0]; r[1] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 1);
    r[2] = t[0]; r[3] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 2);
    r[4] = t[0]; r[5] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(u, scale, 3);
    r[6] = t[0]; r[7] = t[1];
    return r;
}
__device__ __forceinline__ bf16x8 e4m3_to_bf16(unsigned lo, unsigned hi, float scale) {
    bf16x8 r;
    bf16x2 t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
    r[0] = t[0]; r[1] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    r[2] = t[0]; r[3] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
    r[4] = t[0]; r[5] = t[1];
    t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    r[6] = t[0]; r[7] = t[1];
    return r;
}

// Four lanes in a row (lane & 3) hold the 32 values of a block, eight each.  Returns the block's scale byte and leaves the
// lane's codes in `code` (two dwords e4m3, one e2m1).
template <int FMT>
__device__ __forceinline__ unsigned mx_quantize_lane8(const float (&v)[8], unsigned (&code)[2]) {
    unsigned a = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) a = max(a, mag_bits(v[j]));
    a = max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true));
    a = max(a, (unsigned)__builtin_amdgcn_mov_dpp((int)a, 0x4e, 0xf, 0xf, true));
    const unsigned byte = mx_scale_byte<FMT>(a);
    const float inv = mx_inverse_scale(byte);
    float s[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = v[j] * inv;
    if (FMT == GAN_MX_E4M3) {
        code[0] = pack_e4m3(s[0], s[1], s[2], s[3]);
        code[1] = pack_e4m3(s[4], s[5], s[6], s[7]);
    } else {
        code[0] = pack_e2m1(s);
        code[1] = 0;
    }
    return byte;
}

// A kernel's launches may use up to `bytes` of dynamic LDS.  Asked for once a device; `devices` remembers where.
inline hipError_t allow_lds(const void* kernel, int bytes, std::atomic<unsigned long>& devices) {
    int device = 0;
    hipError_t rc = hipGetDevice(&device);
    if (rc != hipSuccess || (device < 64 && devices.load(std::memory_order_relaxed) >> device & 1)) return rc;
    rc = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (rc == hipSuccess && device < 64) devices.fetch_or(1ul << device, std::memory_order_relaxed);
    return rc;
}

// Calls f with a null pointer of the element type `dtype` names.
template <typename F>
inline int with_dtype(int dtype, F f) {
    switch (dtype) {
        case GAN_F32: return f(static_cast<float*>(nullptr));
        case GAN_BF16: return f(static_cast<bf16_t*>(nullptr));
        default: return f(static_cast<f16_t*>(nullptr));
    }
}

}  // namespace gan
