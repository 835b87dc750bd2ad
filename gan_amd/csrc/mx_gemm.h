// Pieces shared by the two tiled products (mx_matmul.hip: scaled 8- / 4-bit pipe; mx_grad.hip: bf16 pipe).
#pragma once
#include "mx.h"

namespace gan {

typedef __attribute__((address_space(3))) void* lds_ptr;

// 16 (4) bytes a lane from global memory straight into LDS: lane l's bytes, from base + offset, land at dst + 16 l (4 l); base and
// dst are the same in all lanes.  As buffer loads: base in scalar registers, so that a copy is one instruction.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t copy_source(const unsigned char* base) {
    // (offsets are taken within the tensors by their callers: no range of its own)
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(base), 0, 0xffffffffu, 0x00027000);
}
__device__ __forceinline__ void copy_to_lds16(__amdgpu_buffer_rsrc_t src, unsigned offset, void* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr)dst, 16, (int)offset, 0, 0, 0);
}
__device__ __forceinline__ void copy_to_lds4(__amdgpu_buffer_rsrc_t src, unsigned offset, void* dst) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (lds_ptr)dst, 4, (int)offset, 0, 0, 0);
}

// The order of instructions among MFMAS matrix instructions: READS LDS reads early, so that they have returned when the next
// matrix instructions want them, then COPIES copies (which the compiler keeps behind the reads, both being accesses to LDS).  The
// masks are those of the builtin: 8 matrix, 0x100 LDS read, 0x20 global read.
template <int MFMAS, int READS, int COPIES, int I = 0>
__device__ __forceinline__ void interleave() {
    if constexpr (I < MFMAS) {
        constexpr int early = COPIES > 0 ? (MFMAS + 1) / 2 : (MFMAS * 3 + 3) / 4, late = MFMAS - early > 0 ? MFMAS - early : 1;
        constexpr int r = I < early ? (I + 1) * READS / early - I * READS / early : 0;
        constexpr int k = I - (MFMAS - late), c = k >= 0 ? (k + 1) * COPIES / late - k * COPIES / late : 0;
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
        if constexpr (c > 0) __builtin_amdgcn_sched_group_barrier(0x20, c, 0);
        interleave<MFMAS, READS, COPIES, I + 1>();
    }
}

// This wave's copies into LDS have landed but for the last N it issued, its reads of LDS have returned, and all waves have got
// here.  (Not __syncthreads, which would wait for all copies.)
template <int N>
__device__ __forceinline__ void landed_barrier() {
    static_assert(N >= 0 && N < 63, "vmcnt has six bits");
    __builtin_amdgcn_sched_barrier(0);      // (the matrix instructions of either side stay on it)
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// Launch position -> tile and part of the contraction.  Workgroups go to the 8 XCDs round robin, each with an L2 of its own: position
// p works on item (p % 8) * (items / 8) + p / 8, so that one XCD holds a contiguous run, of whole parts first, and within a part the
// run walks bands of 8 row tiles: workgroups in flight together share their operand rows and columns in that L2.
__device__ __forceinline__ void tile_of(int p, int ti, int tj, int splits, int& i, int& j, int& split) {
    const int total = ti * tj * splits, per = total / 8, extra = total % 8, x = p % 8, q = p / 8;
    int t = x * per + min(x, extra) + q;
    split = t / (ti * tj);
    t -= split * ti * tj;
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

// A wave's 32 rows x (32 F) columns, as F accumulators of the 32x32 instruction (lane: one row, four times four consecutive
// columns of each), to memory: by way of `stage`, 32 (32 F + 4) floats of LDS of its own, so that whole runs of a row are stored.
// Straight from the accumulators every store would touch 32 rows for 16 bytes each (a 4096 x 4096 bf16 result: 18 us more).
template <typename T, int F, typename Pick>
__device__ __forceinline__ void store_rows(Pick acc, float* stage, int row0, int col0, int rows, int cols, T* __restrict__ out,
                                           long pitch, const float* __restrict__ bias, int accumulate, bool vec) {
    constexpr int PITCH = 32 * F + 4, N = sizeof(T) == 2 ? 8 : 4, LANES = 32 * F / N;     // lanes a row
    const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const f32x16& a = acc(f);
            *reinterpret_cast<f32x4*>(stage + l32 * PITCH + 32 * f + 8 * q + 4 * half) = f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int c = lane % LANES * N, col = col0 + c;
    f32x4 b[N / 4];
#pragma unroll
    for (int k = 0; k < N / 4; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) b[k][j] = bias && col + 4 * k + j < cols ? bias[col + 4 * k + j] : 0.f;
#pragma unroll
    for (int i = 0; i < 32 * LANES / 64; ++i) {
        const int r = i * (64 / LANES) + lane / LANES, row = row0 + r;
        f32x4 v[N / 4];
#pragma unroll
        for (int k = 0; k < N / 4; ++k) v[k] = *reinterpret_cast<const f32x4*>(stage + r * PITCH + c + 4 * k) + b[k];
        if (row >= rows) continue;
        T* to = out + row * pitch + col;
        if (vec && col + N <= cols) {
            typedef T vecn __attribute__((ext_vector_type(N), aligned(16)));
            vecn t;
            if constexpr (N == 4) {
                if (accumulate) v[0] += *reinterpret_cast<const f32x4*>(to);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) t[j] = (T)v[j / 4][j % 4];
            *reinterpret_cast<vecn*>(to) = t;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (col + j < cols) to[j] = (T)(N == 4 && accumulate ? v[j / 4][j % 4] + (float)to[j] : v[j / 4][j % 4]);
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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

// In how many parts a contraction of `steps` steps is cut when `tiles` workgroups alone leave CUs idle: up to `workgroups` in all, no
// part shorter than `least` steps.
inline int contraction_splits(long tiles, int workgroups, int steps, int least) {
    long s = workgroups / tiles;
    if (s > steps / least) s = steps / least;
    return s < 1 ? 1 : (int)s;
}

// The bf16-pipe product of mx_grad.hip: C[i][j] (+)= bias[j] + sum over parts and c of P[i][c] Q[j][c], with PT of P[c][i],
// with QT of Q[c][j].
struct Bf16Product {
    const bf16_t* p;
    const bf16_t* q;
    long ldp, ldq, pstep, qstep;    // row strides; step from one part to the next
    int parts, depth;               // depth of one part: a multiple of 64, operands filled up with zeros to it
    int rows, cols;                 // of C, dense
    const float* bias;
    int accumulate;
};
size_t bf16_product_workspace(int rows, int cols, int parts, int depth);
template <bool PT, bool QT, typename T>
int bf16_product(const Bf16Product& p, T* out, void* ws, hipStream_t st, const char* what);

// [rows][groups * 128] and [out][groups * 128] bf16 of microscaled operands.
void mx_product_images(int fmt, const void* a_codes, const void* a_scales, bf16_t* a, int rows, const void* w_codes, const void* w_scales,
                       bf16_t* w, int in_dim, int out_dim, hipStream_t st);

}  // namespace gan
