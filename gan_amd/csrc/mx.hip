// Microscaled quantisation: rows of activations, weight matrices in the product's layout, and back.  All memory-bound, one
// launch each, every tensor read and written once.  From memory (twelve matrices in turn), us and TB/s for 2048 x 8192 and 8192 x 8192:
// packing fp32 15 = 5.0 and 56 = 5.5, back to fp32 14 = 5.4 and 54 = 5.6, bf16 to e4m3 rows 12 = 4.2 and 34 = 6.0, back 10 = 5.1 and
// 33 = 6.1.  Inside a traced training step, behind other kernels' writes, packing 2048 x 8192 takes 26.  Below 10 us a call is the host's.
#include "mx.h"

namespace gan {

// [rows][c] of T -> codes [rows][128 groups] (one byte or half a byte a value), scale bytes [rows][4 groups].  A lane takes
// eight values, four lanes a block.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const T* __restrict__ x, long ldx, unsigned char* __restrict__ codes,
                                                          unsigned char* __restrict__ scales, long rows, int c, bool vec) {
    const int chunks = mx_groups(c) * 16;
    const long total = rows * chunks, step = (long)gridDim.x * 256;
    // (total and step are multiples of 4: the four lanes of a block stay together)
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long row = i / chunks;
        const int chunk = (int)(i - row * chunks), i0 = chunk * 8;
        float v[8];
        load8(x + row * ldx, i0, i0 < c ? c : 0, vec, v);
        unsigned code[2];
        const unsigned byte = mx_quantize_lane8<FMT>(v, code);
        if (FMT == GAN_MX_E4M3) *reinterpret_cast<uint2*>(codes + i * 8) = make_uint2(code[0], code[1]);
        else *reinterpret_cast<unsigned*>(codes + i * 4) = code[0];
        if ((chunk & 3) == 0) scales[i / 4] = (unsigned char)byte;
    }
}

__device__ __forceinline__ float e2m1_value(unsigned code) {
    const unsigned m = code & 7;    // 0 0.5 1 1.5 2 3 4 6
    const float v = m < 2 ? 0.5f * m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1) << 22);
    return code & 8 ? -v : v;
}

template <typename T, int FMT>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(const unsigned char* __restrict__ codes,
                                                            const unsigned char* __restrict__ scales, T* __restrict__ y,
                                                            long rows, int c, bool vec) {
    const int chunks = (c + 7) / 8, pitch = mx_groups(c) * 16;
    const long total = rows * chunks, step = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += step) {
        const long row = i / chunks;
        const int chunk = (int)(i - row * chunks);
        const long at = row * pitch + chunk;
        const float s = mx_scale(scales[at / 4]);
        float v[8];
        if (FMT == GAN_MX_E4M3) {
            const uint2 u = *reinterpret_cast<const uint2*>(codes + at * 8);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int w = (int)(j ? u.y : u.x);
                v[4 * j + 0] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * s;
                v[4 * j + 1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * s;
                v[4 * j + 2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * s;
                v[4 * j + 3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * s;
            }
        } else {
            const unsigned u = *reinterpret_cast<const unsigned*>(codes + at * 4);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = e2m1_value(u >> (4 * j)) * s;
        }
        store8(y + row * c, chunk * 8, c, vec, v);
    }
}

// A matrix [in][out] quantised in blocks of 32 along `in`, in the order the matrix pipe takes it: codes [in / 32][out][16 bytes]
// -- one lane's fragment is one block, 16 bytes, and neighbouring outputs lie side by side -- and scales [in / 128][out][4
// bytes], a lane's four blocks of a 128-deep step in one dword.  `in` is filled up with zeros to whole groups of 128.
// A workgroup takes 64 outputs x 4 blocks, a lane one block: reads of a row and the 16-byte stores are contiguous over lanes.
template <typename T>
__global__ __launch_bounds__(256) void mx_pack_kernel(const T* __restrict__ m, long ld, unsigned char* __restrict__ codes,
                                                      unsigned char* __restrict__ scales, int in_dim, int out_dim) {
    __shared__ __align__(4) unsigned char bytes[64][4];
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), kb = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (n < out_dim) {
        float v[32];
        unsigned a = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const int k = kb * 32 + j;
            v[j] = k < in_dim ? (float)m[k * ld + n] : 0.f;
            a = max(a, mag_bits(v[j]));
        }
        const unsigned byte = mx_scale_byte<GAN_MX_E2M1>(a);
        const float inv = mx_inverse_scale(byte);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= inv;
        uint4 u;
        u.x = pack_e2m1(v);
        u.y = pack_e2m1(v + 8);
        u.z = pack_e2m1(v + 16);
        u.w = pack_e2m1(v + 24);
        reinterpret_cast<uint4*>(codes)[(long)kb * out_dim + n] = u;
        bytes[threadIdx.x & 63][threadIdx.x >> 6] = (unsigned char)byte;
    }
    __syncthreads();
    if (threadIdx.x < 64 && n < out_dim)
        reinterpret_cast<unsigned*>(scales)[(long)blockIdx.y * out_dim + n] = *reinterpret_cast<const unsigned*>(bytes[threadIdx.x]);
}

template <typename T>
__global__ __launch_bounds__(256) void mx_unpack_kernel(const unsigned char* __restrict__ codes,
                                                        const unsigned char* __restrict__ scales, T* __restrict__ m, int in_dim,
                                                        int out_dim) {
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), kb = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (n >= out_dim) return;
    const uint4 u = reinterpret_cast<const uint4*>(codes)[(long)kb * out_dim + n];
    const float s = mx_scale(scales[((long)blockIdx.y * out_dim + n) * 4 + (kb & 3)]);
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        const int k = kb * 32 + j;
        if (k < in_dim) m[(long)k * out_dim + n] = (T)(e2m1_value(w[j >> 3] >> (4 * (j & 7))) * s);
    }
}

}  // namespace gan

using namespace gan;

extern "C" {

int gan_mx_quantize(int dtype, int fmt, long rows, int c, const void* x, long ldx, void* codes, void* scales,
                    gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype) && mx_fmt_ok(fmt), "gan_mx_quantize: unknown element type %d or format %d", dtype, fmt);
    GAN_CHECK_ARG(rows >= 0 && rows < (1L << 31) && c >= 1 && c <= (1 << 28) && ldx >= c, "gan_mx_quantize: %ld rows of %d values, stride %ld",
                  rows, c, ldx);
    if (rows == 0) return 0;
    GAN_CHECK_ARG(x && codes && scales, "gan_mx_quantize: null pointer");
    GAN_CHECK_ARG((reinterpret_cast<size_t>(codes) & 7) == 0, "gan_mx_quantize: codes are not 8-byte aligned");
    const long total = rows * mx_groups(c) * 16;
    const dim3 grid((unsigned)(total / 256 + 1 < 8192 ? total / 256 + 1 : 8192));
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        const bool vec = aligned16(x) && ldx * sizeof(T) % 16 == 0;
        unsigned char* co = static_cast<unsigned char*>(codes);
        unsigned char* sc = static_cast<unsigned char*>(scales);
        if (fmt == GAN_MX_E4M3)
            hipLaunchKernelGGL((mx_quantize_kernel<T, GAN_MX_E4M3>), grid, dim3(256), 0, as_stream(stream),
                               static_cast<const T*>(x), ldx, co, sc, rows, c, vec);
        else
            hipLaunchKernelGGL((mx_quantize_kernel<T, GAN_MX_E2M1>), grid, dim3(256), 0, as_stream(stream),
                               static_cast<const T*>(x), ldx, co, sc, rows, c, vec);
        return check_launch("gan_mx_quantize");
    });
}

int gan_mx_dequantize(int dtype, int fmt, long rows, int c, const void* codes, const void* scales, void* y,
                      gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype) && mx_fmt_ok(fmt), "gan_mx_dequantize: unknown element type %d or format %d", dtype, fmt);
    GAN_CHECK_ARG(rows >= 0 && rows < (1L << 31) && c >= 1 && c <= (1 << 28), "gan_mx_dequantize: %ld rows of %d values", rows, c);
    if (rows == 0) return 0;
    GAN_CHECK_ARG(y && codes && scales, "gan_mx_dequantize: null pointer");
    GAN_CHECK_ARG((reinterpret_cast<size_t>(codes) & 7) == 0, "gan_mx_dequantize: codes are not 8-byte aligned");
    const long total = rows * ((c + 7) / 8);
    const dim3 grid((unsigned)(total / 256 + 1 < 8192 ? total / 256 + 1 : 8192));
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        const bool vec = aligned16(y) && c * sizeof(T) % 16 == 0;
        const unsigned char* co = static_cast<const unsigned char*>(codes);
        const unsigned char* sc = static_cast<const unsigned char*>(scales);
        if (fmt == GAN_MX_E4M3)
            hipLaunchKernelGGL((mx_dequantize_kernel<T, GAN_MX_E4M3>), grid, dim3(256), 0, as_stream(stream), co, sc,
                               static_cast<T*>(y), rows, c, vec);
        else
            hipLaunchKernelGGL((mx_dequantize_kernel<T, GAN_MX_E2M1>), grid, dim3(256), 0, as_stream(stream), co, sc,
                               static_cast<T*>(y), rows, c, vec);
        return check_launch("gan_mx_dequantize");
    });
}

int gan_mx_pack(int dtype, int in_dim, int out_dim, const void* matrix, long ld, void* codes, void* scales,
                gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype), "gan_mx_pack: unknown element type %d", dtype);
    GAN_CHECK_ARG(in_dim >= 1 && in_dim <= GAN_MX_MAX_IN && out_dim >= 1 && out_dim <= GAN_MX_MAX_IN && ld >= out_dim,
                  "gan_mx_pack: matrix of %d x %d, row stride %ld (up to %d of each are served)", in_dim, out_dim, ld, GAN_MX_MAX_IN);
    GAN_CHECK_ARG(matrix && codes && scales, "gan_mx_pack: null pointer");
    GAN_CHECK_ARG(aligned16(codes) && (reinterpret_cast<size_t>(scales) & 3) == 0,
                  "gan_mx_pack: codes have to be 16-byte and scales 4-byte aligned");
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        hipLaunchKernelGGL(mx_pack_kernel<T>, dim3((out_dim + 63) / 64, mx_groups(in_dim)), dim3(256), 0, as_stream(stream),
                           static_cast<const T*>(matrix), ld, static_cast<unsigned char*>(codes),
                           static_cast<unsigned char*>(scales), in_dim, out_dim);
        return check_launch("gan_mx_pack");
    });
}

int gan_mx_unpack(int dtype, int in_dim, int out_dim, const void* codes, const void* scales, void* matrix,
                  gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype), "gan_mx_unpack: unknown element type %d", dtype);
    GAN_CHECK_ARG(in_dim >= 1 && in_dim <= GAN_MX_MAX_IN && out_dim >= 1 && out_dim <= GAN_MX_MAX_IN, "gan_mx_unpack: matrix of %d x %d", in_dim, out_dim);
    GAN_CHECK_ARG(matrix && codes && scales, "gan_mx_unpack: null pointer");
    GAN_CHECK_ARG(aligned16(codes) && (reinterpret_cast<size_t>(scales) & 3) == 0,
                  "gan_mx_unpack: codes have to be 16-byte and scales 4-byte aligned");
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        hipLaunchKernelGGL(mx_unpack_kernel<T>, dim3((out_dim + 63) / 64, mx_groups(in_dim)), dim3(256), 0, as_stream(stream),
                           static_cast<const unsigned char*>(codes), static_cast<const unsigned char*>(scales),
                           static_cast<T*>(matrix), in_dim, out_dim);
        return check_launch("gan_mx_unpack");
    });
}

}  // extern "C"
