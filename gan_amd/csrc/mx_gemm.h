// Pieces shared by the two tiled products (mx_matmul.hip: scaled 8- / 4-bit pipe; mx_grad.hip: bf16 pipe).
#pragma once
#include "mx.h"

namespace gan {

typedef __attribute__((address_space(1))) const void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// 16 bytes a lane from global memory straight into LDS: lane l's bytes land at dst + 16 l (dst the same in all lanes).
__device__ __forceinline__ void copy_to_lds16(const void* src, void* dst) {
    __builtin_amdgcn_global_load_lds((global_ptr)src, (lds_ptr)dst, 16, 0, 0);
}

// All of this wave's copies into LDS have landed, and all waves have got here.
__device__ __forceinline__ void copies_done_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

// Launch position -> tile.  Workgroups go to the 8 XCDs round robin, each with an L2 of its own: position p works on tile
// (p % 8) * (tiles / 8) + p / 8, so that one XCD holds a contiguous run of tiles, and a run walks bands of 8 row tiles, so that
// tiles in flight together share their operand rows and columns in that L2.
__device__ __forceinline__ void tile_of(int p, int ti, int tj, int& i, int& j) {
    const int total = ti * tj, per = total / 8, extra = total % 8, x = p % 8, q = p / 8;
    const int t = x * per + min(x, extra) + q;
    const int band = t / (8 * tj), in = t - band * 8 * tj, high = min(8, ti - band * 8);
    i = band * 8 + in % high;
    j = in / high;
}

// Four consecutive results of a row, from column j on.
template <typename T>
__device__ __forceinline__ void store4(T* __restrict__ row, int j, int n, bool vec, f32x4 v, const float* __restrict__ bias,
                                       int accumulate) {
    if (vec) {      // (n and the row are multiples of 4 values then: all four are inside or none)
        if (j >= n) return;
        if (bias) v += *reinterpret_cast<const f32x4*>(bias + j);
        if constexpr (std::is_same<T, float>::value) {
            if (accumulate) v += *reinterpret_cast<const f32x4*>(row + j);
            *reinterpret_cast<f32x4*>(row + j) = v;
        } else {
            typedef T vec4 __attribute__((ext_vector_type(4)));
            vec4 t;
#pragma unroll
            for (int k = 0; k < 4; ++k) t[k] = (T)v[k];
            *reinterpret_cast<vec4*>(row + j) = t;
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (j + k < n) {
            float s = v[k] + (bias ? bias[j + k] : 0.f);
            if constexpr (std::is_same<T, float>::value)
                if (accumulate) s += row[j + k];
            row[j + k] = (T)s;
        }
}

// out[i][j] (+)= bias[j] + sum over slabs, in slab order: the end of a product whose contraction was split over workgroups.
template <typename T>
__global__ __launch_bounds__(256) void mx_join_kernel(const float* __restrict__ slabs, int splits, T* __restrict__ out, long rows,
                                                      int n, const float* __restrict__ bias, int accumulate, bool vec) {
    const int quads = (n + 3) / 4;
    const long total = rows * quads, slab = rows * (long)quads * 4;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / quads;
        const int j = (int)(i - row * quads) * 4;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f32x4*>(slabs + s * slab + i * 4);
        store4(out + row * n, j, n, vec, v, bias, accumulate);
    }
}

template <typename T>
inline void join_slabs(const float* slabs, int splits, T* out, long rows, int n, const float* bias, int accumulate, bool vec,
                       hipStream_t st) {
    const long blocks = (rows * ((n + 3) / 4) + 255) / 256;
    hipLaunchKernelGGL((mx_join_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, slabs, splits, out,
                       rows, n, bias, accumulate, vec);
}
inline size_t slab_bytes(int splits, long rows, int n) { return splits > 1 ? (size_t)splits * rows * ((n + 3) / 4) * 16 : 0; }

// In how many parts a contraction of `steps` steps is cut when `tiles` workgroups alone would not fill the 256 CUs: no part
// shorter than `least` steps, about two workgroups a CU in all.
inline int contraction_splits(long tiles, int steps, int least) {
    long s = tiles >= 256 ? 1 : 512 / tiles;
    if (s > steps / least) s = steps / least;
    return s < 1 ? 1 : (int)s;
}

// The bf16-pipe product of mx_grad.hip: C[i][j] (+)= bias[j] + sum over parts and c of P[i][c] Q[j][c].
struct Bf16Product {
    const bf16_t* p;
    const bf16_t* q;
    long ldp, ldq, pstep, qstep;    // row strides; step from one part to the next
    int parts, depth;               // depth of one part: a multiple of 64, rows filled up with zeros to it
    int rows, cols;                 // of C, dense
    const float* bias;
    int accumulate;
};
size_t bf16_product_workspace(int rows, int cols, int parts, int depth);
template <typename T>
int bf16_product(const Bf16Product& p, T* out, void* ws, hipStream_t st, const char* what);

// [rows][groups * 128] bf16 and [out][groups * 128] bf16 of microscaled operands (forward with fp32 results).
void mx_rows_to_bf16(int fmt, const void* codes, const void* scales, bf16_t* out, long rows, int in_dim, hipStream_t st);
void mx_weights_to_bf16(const void* codes, const void* scales, bf16_t* out, int in_dim, int out_dim, hipStream_t st);

}  // namespace gan
