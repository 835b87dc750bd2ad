// The bf16-pipe product and the gradients of the microscaled product.
//
//   dA[r][k] = sum_n dY[r][n] W[k][n]      dW[k][n] = sum_r A[r][k] dY[r][n]      dbias[n] = sum_r dY[r][n]
//
// with A and W the quantised values (the gradient of the quantisers is passed straight through).  Quantised values are exact in
// bf16; dY is split exactly into one (bf16), two (fp16: 11 = 8 + 3 bits) or three (fp32: 24 = 8 + 8 + 8) bf16 parts, whose
// products are summed in fp32.  So a gradient carries the error of an fp32 sum of exact products whatever the type.
//
// All three products contract over rows that are contiguous in memory: memory-bound passes turn the operands into bf16 images
// with the contraction axis innermost and filled up with zeros to a multiple of 64, then one compute-bound kernel runs.
#include "mx_gemm.h"

namespace gan {

// C[i][j] over a tile of BI x BJ, WI x WJ waves, 32x32x16 instructions with Q as their first operand (a lane ends with four
// consecutive j of one i).  A stage in LDS is 64 deep: 128 bytes of every row -- whole cache lines; 64 bytes a row and stage cost
// twice the requests to the L2 --, their 16-byte chunks swapped by row so that a fragment read hits all banks.  STAGES stages form
// a ring that direct copies keep filled.  The fragments of the next 16 are read while the matrix pipe works on these; the one
// barrier of a stage stands before its last quarter, when all of it has been read: it asks for the next stage and frees this one.
// Large tiles have two waves a SIMD with 128 x 64 outputs each: LDS then gives 96 bytes a clock of its 128; one wave of
// 128 x 128 needs less of it, but nothing covers its waits (4096^3: 126 us against 115, the weights' image included).
// 4096 x 4096 x 8192: 1.25 PF/s, a library product of that size 1.45.
template <typename T, int BI, int BJ, int WI, int WJ, int STAGES>
__global__ __launch_bounds__(64 * WI * WJ) void bf16_product_kernel(Bf16Product p, T* out, float* slabs, int splits, bool vec) {
    constexpr int WAVES = WI * WJ, THREADS = 64 * WAVES, FI = BI / WI / 32, FJ = BJ / WJ / 32, STAGE = (BI + BJ) * 128;
    constexpr int COPIES = STAGE / 16 / THREADS;        // of a wave for a stage
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wj = wave % WJ, wi = wave / WJ;
    const int l32 = lane & 31, half = lane >> 5;
    int ti, tj;
    tile_of(blockIdx.x, (p.rows + BI - 1) / BI, (p.cols + BJ - 1) / BJ, ti, tj);
    const int i0 = ti * BI, j0 = tj * BJ;
    const int per = p.depth / 64;
    const long steps = (long)per * p.parts;
    const int s0 = (int)(steps * blockIdx.y / splits), s1 = (int)(steps * (blockIdx.y + 1) / splits);

    // where this lane's copies begin, and the two operands' places in the part at hand (rows beyond the last: the last again)
    constexpr int PC = BI * 8 / THREADS, QC = BJ * 8 / THREADS;
    unsigned p_off[PC], q_off[QC];
#pragma unroll
    for (int i = 0; i < PC; ++i) {
        const int row = ((i * WAVES + wave) * 64 + lane) >> 3, chunk = (lane & 7) ^ (row & 7);
        p_off[i] = (unsigned)min(row, p.rows - 1 - i0) * (unsigned)(p.ldp * 2) + chunk * 16;
    }
#pragma unroll
    for (int i = 0; i < QC; ++i) {
        const int row = ((i * WAVES + wave) * 64 + lane) >> 3, chunk = (lane & 7) ^ (row & 7);
        q_off[i] = (unsigned)min(row, p.cols - 1 - j0) * (unsigned)(p.ldq * 2) + chunk * 16;
    }
    int filled = s0, in_part = s0 % per;
    const unsigned char* pp = reinterpret_cast<const unsigned char*>(p.p + (long)i0 * p.ldp + (s0 / per) * p.pstep + in_part * 64L);
    const unsigned char* qp = reinterpret_cast<const unsigned char*>(p.q + (long)j0 * p.ldq + (s0 / per) * p.qstep + in_part * 64L);
    const long p_jump = (p.pstep - (per - 1) * 64L) * 2, q_jump = (p.qstep - (per - 1) * 64L) * 2;
    // copies of the stage after the last one copied, into LDS from `to` on; past the end the last one again, which nobody reads
    auto fill = [&](int to) {
        unsigned char* base = lds + to;
#pragma unroll
        for (int i = 0; i < PC; ++i) copy_to_lds16(copy_source(pp), p_off[i], base + (i * WAVES + wave) * 1024);
#pragma unroll
        for (int i = 0; i < QC; ++i) copy_to_lds16(copy_source(qp), q_off[i], base + BI * 128 + (i * WAVES + wave) * 1024);
        const bool more = ++filled < s1, jump = in_part == per - 1;
        in_part = jump ? 0 : in_part + 1;
        pp += more ? (jump ? p_jump : 128L) : 0L;
        qp += more ? (jump ? q_jump : 128L) : 0L;
    };
    struct Fragments {
        bf16x8 p[FI], q[FJ];
    };
    auto read = [&](int at, int k, Fragments& f) {
        const unsigned char* base = lds + at;
#pragma unroll
        for (int j = 0; j < FJ; ++j) {
            const int row = BI + (wj * FJ + j) * 32 + l32;
            f.q[j] = *reinterpret_cast<const bf16x8*>(base + row * 128 + (((2 * k + half) ^ (row & 7)) * 16));
        }
#pragma unroll
        for (int i = 0; i < FI; ++i) {
            const int row = (wi * FI + i) * 32 + l32;
            f.p[i] = *reinterpret_cast<const bf16x8*>(base + row * 128 + (((2 * k + half) ^ (row & 7)) * 16));
        }
    };
    f32x16 acc[FJ][FI];
#pragma unroll
    for (int j = 0; j < FJ; ++j)
#pragma unroll
        for (int i = 0; i < FI; ++i)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[j][i][k] = 0.f;
    auto multiply = [&](const Fragments& f) {
#pragma unroll
        for (int j = 0; j < FJ; ++j)
#pragma unroll
            for (int i = 0; i < FI; ++i) acc[j][i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f.q[j], f.p[i], acc[j][i], 0, 0, 0);
    };
#pragma unroll
    for (int s = 0; s < STAGES; ++s) fill(s * STAGE);
    landed_barrier<(STAGES - 1) * COPIES>();
    Fragments f[2];
    read(0, 0, f[0]);
    int at = 0;
    for (int s = s0; s < s1; ++s) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            read(at, k + 1, f[(k + 1) % 2]);
            multiply(f[k % 2]);
            interleave<FI * FJ, FI + FJ, 0>();
        }
        landed_barrier<(STAGES - 2) * COPIES>();        // the next stage is there; STAGES - 2 more are on their way
        const int freed = at;
        at = at + STAGE == STAGES * STAGE ? 0 : at + STAGE;
        read(at, 0, f[0]);
        fill(freed);
        multiply(f[1]);
        interleave<FI * FJ, FI + FJ, COPIES>();
    }
    landed_barrier<0>();        // (no copy is in flight when the workgroup gives its LDS back)
    float* stage = reinterpret_cast<float*>(lds) + wave * 32 * (32 * FJ + 4);
    static_assert(WAVES * 32 * (32 * FJ + 4) * 4 <= STAGES * STAGE, "the results pass through the stages' LDS");
    const int n4 = (p.cols + 3) / 4 * 4, col0 = j0 + wj * FJ * 32;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        const int row0 = i0 + (wi * FI + i) * 32;
        auto pick = [&](int j) -> const f32x16& { return acc[j][i]; };
        if (slabs) store_rows<float, FJ>(pick, stage, row0, col0, p.rows, n4, slabs + (long)blockIdx.y * p.rows * n4, n4, nullptr, 0, true);
        else store_rows<T, FJ>(pick, stage, row0, col0, p.rows, p.cols, out, p.cols, p.bias, p.accumulate, vec);
    }
}

enum { BF16_128, BF16_256_128, BF16_256 };      // tiles
struct Bf16Plan {
    int tile, splits;
};
static Bf16Plan bf16_plan(int rows, int cols, int parts, int depth) {
    // 256 x 256 tiles where they fill the chip, alone (4096^3: 115 us against 132) or in parts of 32 stages or more
    // (1024 x 1024 <- 32768: 98 us in 16 parts against 110 with small tiles in 6; 1024 x 4096 <- 4096, parts of 16: 58 against 53)
    const long large = (long)((rows + 255) / 256) * ((cols + 255) / 256), all = (long)parts * (depth / 64);
    const int steps = (int)(all < (1 << 30) ? all : 1 << 30);
    if (large >= 192) return {BF16_256, 1};
    // (4096 x 2048 <- 8192: 125 us, 133 in two parts of 256 x 256 tiles)
    if ((long)((rows + 255) / 256) * ((cols + 127) / 128) >= 192) return {BF16_256_128, 1};
    if (steps / (256 / large) >= 32) return {BF16_256, (int)(256 / large)};
    return {BF16_128, contraction_splits((long)((rows + 127) / 128) * ((cols + 127) / 128), 384, steps, 8)};
}

size_t bf16_product_workspace(int rows, int cols, int parts, int depth) {
    return slab_bytes(bf16_plan(rows, cols, parts, depth).splits, rows, cols);
}

template <typename T, int BI, int BJ, int WI, int WJ>
static int launch_bf16(const Bf16Product& p, T* out, float* slabs, int splits, bool vec, hipStream_t st, const char* what) {
    // 128 x 128: two workgroups a CU
    constexpr int STAGES = BI + BJ == 384 ? 3 : 2, LDS = STAGES * (BI + BJ) * 128;
    auto kernel = bf16_product_kernel<T, BI, BJ, WI, WJ, STAGES>;
    static std::atomic<unsigned long> devices{0};
    const hipError_t set = allow_lds(reinterpret_cast<const void*>(kernel), LDS, devices);
    if (set != hipSuccess) return fail("%s: %d bytes of LDS refused: %s", what, LDS, hipGetErrorString(set));
    const long tiles = (long)((p.rows + BI - 1) / BI) * ((p.cols + BJ - 1) / BJ);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, splits), dim3(64 * WI * WJ), LDS, st, p, out, slabs, splits, vec);
    return 0;
}

template <typename T>
int bf16_product(const Bf16Product& p, T* out, void* ws, hipStream_t st, const char* what) {
    const Bf16Plan plan = bf16_plan(p.rows, p.cols, p.parts, p.depth);
    const bool vec = p.cols * sizeof(T) % 16 == 0 && aligned16(out), vec4 = vec && aligned16(p.bias);
    float* slabs = plan.splits > 1 ? static_cast<float*>(ws) : nullptr;
    const int rc = plan.tile == BF16_256       ? launch_bf16<T, 256, 256, 2, 4>(p, out, slabs, plan.splits, vec, st, what)
                   : plan.tile == BF16_256_128 ? launch_bf16<T, 256, 128, 4, 2>(p, out, slabs, plan.splits, vec, st, what)
                                               : launch_bf16<T, 128, 128, 2, 2>(p, out, slabs, plan.splits, vec, st, what);
    if (rc) return rc;
    if (slabs) join_slabs(slabs, plan.splits, out, (long)p.rows, p.cols, p.bias, p.accumulate, vec4, st);
    return check_launch(what);
}
template int bf16_product<float>(const Bf16Product&, float*, void*, hipStream_t, const char*);

// ------------------------------------------------------------------------------------------------ operand images
// Part `part` of the exact split of v into bf16 values, largest first.  By truncation: it cannot overflow, and what is left is
// exact.  An infinity or a NaN is in part 0 alone.
__device__ __forceinline__ bf16_t split_part(float v, int part) {
    for (int i = 0; i < part; ++i) {
        const unsigned u = __float_as_uint(v);
        v = (u & 0x7f800000u) == 0x7f800000u ? 0.f : v - __uint_as_float(u & 0xffff0000u);
    }
    const unsigned u = __float_as_uint(v);
    const unsigned nan = (u & 0x7fffffffu) > 0x7f800000u ? 0x400000u : 0u;
    return __builtin_bit_cast(bf16_t, (unsigned short)((u | nan) >> 16));
}

template <typename T> struct Parts;
template <> struct Parts<bf16_t> { static constexpr int n = 1; };
template <> struct Parts<f16_t> { static constexpr int n = 2; };
template <> struct Parts<float> { static constexpr int n = 3; };

__host__ __device__ __forceinline__ long to64(long n) { return (n + 63) / 64 * 64; }

// dY [rows][n] -> parts [rows][n filled up to 64] bf16.
template <typename T>
__global__ __launch_bounds__(256) void split_rows_kernel(const T* __restrict__ y, bf16_t* __restrict__ out, long rows, int n,
                                                         bool vec) {
    const long np = to64(n), chunks = np / 8, total = rows * chunks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long row = i / chunks;
        const int i0 = (int)(i - row * chunks) * 8;
        float v[8];
        load8(y + row * n, i0, i0 < n ? n : 0, vec, v);
#pragma unroll
        for (int part = 0; part < Parts<T>::n; ++part) {
            bf16x8 b;
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = split_part(v[j], part);
            *reinterpret_cast<bf16x8*>(out + (part * rows + row) * np + i0) = b;
        }
    }
}

// dY [rows][n] -> parts [n][rows filled up to 64] bf16, and the sums of 64 rows of each column (dbias).  64 x 64 tiles through
// LDS.
template <typename T>
__global__ __launch_bounds__(256) void split_transpose_kernel(const T* __restrict__ y, bf16_t* __restrict__ out,
                                                              float* __restrict__ colsum, int rows, int n, bool vec) {
    __shared__ float tile[64][65];
    const long rp = to64(rows);
    const int n0 = blockIdx.x * 64, r0 = blockIdx.y * 64, t = threadIdx.x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h * 32 + t / 8, i0 = n0 + (t % 8) * 8;
        float v[8];
        load8(y + (long)min(r0 + row, rows - 1) * n, i0, r0 + row < rows && i0 < n ? n : 0, vec, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[row][(t % 8) * 8 + j] = v[j];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int col = h * 32 + t / 8, r8 = (t % 8) * 8;
        float v[8], s = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = tile[r8 + j][col];
            s += v[j];
        }
        if (n0 + col < n) {
#pragma unroll
            for (int part = 0; part < Parts<T>::n; ++part) {
                bf16x8 b;
#pragma unroll
                for (int j = 0; j < 8; ++j) b[j] = split_part(v[j], part);
                *reinterpret_cast<bf16x8*>(out + ((long)part * n + n0 + col) * rp + r0 + r8) = b;
            }
        }
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        s += __shfl_xor(s, 4, 64);
        if (colsum && (t & 7) == 0 && n0 + col < n) colsum[(long)blockIdx.y * n + n0 + col] = s;
    }
}

// A [rows][in] microscaled -> [in][rows filled up to 64] bf16, 64 rows x 64 values a workgroup.
template <int FMT>
__global__ __launch_bounds__(256) void mx_rows_transpose_kernel(const unsigned char* __restrict__ codes,
                                                                const unsigned char* __restrict__ scales, bf16_t* __restrict__ out,
                                                                int rows, int in_dim) {
    __shared__ bf16_t tile[64][66];
    const long rp = to64(rows), pitch = mx_groups(in_dim) * 16L;
    const int k0 = blockIdx.x * 64, r0 = blockIdx.y * 64, t = threadIdx.x;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = h * 32 + t / 8;
        bf16x8 b;
        if (r0 + row < rows) {
            const long at = (long)(r0 + row) * pitch + k0 / 8 + t % 8;
            const float s = mx_scale(scales[at / 4]);
            if constexpr (FMT == GAN_MX_E4M3) {
                const uint2 u = *reinterpret_cast<const uint2*>(codes + at * 8);
                b = e4m3_to_bf16(u.x, u.y, s);
            } else {
                b = e2m1_to_bf16(*reinterpret_cast<const unsigned*>(codes + at * 4), s);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = (bf16_t)0.f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[row][(t % 8) * 8 + j] = b[j];
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int col = h * 32 + t / 8, r8 = (t % 8) * 8;
        if (k0 + col >= in_dim) continue;
        bf16x8 b;
#pragma unroll
        for (int j = 0; j < 8; ++j) b[j] = tile[r8 + j][col];
        *reinterpret_cast<bf16x8*>(out + (long)(k0 + col) * rp + r0 + r8) = b;
    }
}

template <int FMT>
__global__ __launch_bounds__(256) void mx_rows_bf16_kernel(const unsigned char* __restrict__ codes,
                                                           const unsigned char* __restrict__ scales, bf16_t* __restrict__ out,
                                                           long total) {
    for (long at = (long)blockIdx.x * 256 + threadIdx.x; at < total; at += (long)gridDim.x * 256) {
        const float s = mx_scale(scales[at / 4]);
        bf16x8 b;
        if constexpr (FMT == GAN_MX_E4M3) {
            const uint2 u = *reinterpret_cast<const uint2*>(codes + at * 8);
            b = e4m3_to_bf16(u.x, u.y, s);
        } else {
            b = e2m1_to_bf16(*reinterpret_cast<const unsigned*>(codes + at * 4), s);
        }
        *reinterpret_cast<bf16x8*>(out + at * 8) = b;
    }
}

// Packed W -> [out][groups * 128] bf16: a lane writes one block, 64 bytes.
__global__ __launch_bounds__(256) void mx_weights_bf16_kernel(const unsigned char* __restrict__ codes,
                                                              const unsigned char* __restrict__ scales, bf16_t* __restrict__ out,
                                                              int groups, int out_dim) {
    // 4 blocks of 64 outputs; neighbouring lanes take the four blocks of one output, so that 256 bytes of a row are written
    const int q = threadIdx.x & 3, n = blockIdx.x * 64 + threadIdx.x / 4, g = blockIdx.y;
    if (n >= out_dim) return;
    const uint4 u = reinterpret_cast<const uint4*>(codes)[((long)g * 4 + q) * out_dim + n];
    const float s = mx_scale(scales[((long)g * out_dim + n) * 4 + q]);
    bf16x8* o = reinterpret_cast<bf16x8*>(out + ((long)n * groups + g) * 128 + q * 32);
    o[0] = e2m1_to_bf16(u.x, s);
    o[1] = e2m1_to_bf16(u.y, s);
    o[2] = e2m1_to_bf16(u.z, s);
    o[3] = e2m1_to_bf16(u.w, s);
}

// Packed W -> [in][out filled up to 64] bf16: a lane takes one block of one output; the lanes of a wave are neighbouring
// outputs, so each of the 32 stores is contiguous.
__global__ __launch_bounds__(256) void mx_weights_transpose_kernel(const unsigned char* __restrict__ codes,
                                                                   const unsigned char* __restrict__ scales,
                                                                   bf16_t* __restrict__ out, int in_dim, int out_dim) {
    const long np = to64(out_dim);
    const int n = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6, k0 = blockIdx.y * 128 + q * 32;
    uint4 u = make_uint4(0, 0, 0, 0);
    float s = 1.f;
    if (n < out_dim) {
        u = reinterpret_cast<const uint4*>(codes)[((long)blockIdx.y * 4 + q) * out_dim + n];
        s = mx_scale(scales[((long)blockIdx.y * out_dim + n) * 4 + q]);
    }
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bf16x8 b = e2m1_to_bf16(w[i], s);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k0 + i * 8 + j < in_dim) out[(long)(k0 + i * 8 + j) * np + n] = b[j];
    }
}

// dbias[n] (+)= sum over blocks of 64 rows.
__global__ __launch_bounds__(256) void mx_dbias_kernel(const float* __restrict__ colsum, float* __restrict__ out, int blocks, int n,
                                                       int accumulate) {
    __shared__ float red[8][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float s = 0.f;
    if (col < n)
        for (int i = part; i < blocks; i += 8) s += colsum[(long)i * n + col];
    red[part][threadIdx.x & 31] = s;
    __syncthreads();
    if (part == 0 && col < n) {
        s = 0.f;
        for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
        out[col] = (accumulate ? out[col] : 0.f) + s;
    }
}

static dim3 flat_grid(long items) {
    const long blocks = (items + 255) / 256;
    return dim3((unsigned)(blocks < 8192 ? (blocks < 1 ? 1 : blocks) : 8192));
}

void mx_rows_to_bf16(int fmt, const void* codes, const void* scales, bf16_t* out, long rows, int in_dim, hipStream_t st) {
    const long total = rows * mx_groups(in_dim) * 16;
    const unsigned char* c = static_cast<const unsigned char*>(codes);
    const unsigned char* s = static_cast<const unsigned char*>(scales);
    if (fmt == GAN_MX_E4M3) hipLaunchKernelGGL(mx_rows_bf16_kernel<GAN_MX_E4M3>, flat_grid(total), dim3(256), 0, st, c, s, out, total);
    else hipLaunchKernelGGL(mx_rows_bf16_kernel<GAN_MX_E2M1>, flat_grid(total), dim3(256), 0, st, c, s, out, total);
}

void mx_weights_to_bf16(const void* codes, const void* scales, bf16_t* out, int in_dim, int out_dim, hipStream_t st) {
    hipLaunchKernelGGL(mx_weights_bf16_kernel, dim3((out_dim + 63) / 64, mx_groups(in_dim)), dim3(256), 0, st,
                       static_cast<const unsigned char*>(codes), static_cast<const unsigned char*>(scales), out, mx_groups(in_dim),
                       out_dim);
}

static int parts_of(int dtype) { return dtype == GAN_BF16 ? 1 : dtype == GAN_F16 ? 2 : 3; }

// dY itself is the operand of dA when it is bf16 in whole 64s.
static bool dy_as_is(int dtype, int out_dim) { return dtype == GAN_BF16 && out_dim % 64 == 0; }

}  // namespace gan

using namespace gan;

extern "C" {

size_t gan_mx_matmul_dgrad_workspace_bytes(int dtype, int rows, int in_dim, int out_dim) {
    if (rows < 1 || rows > GAN_MX_MAX_ROWS || in_dim < 1 || in_dim > GAN_MX_MAX_IN || out_dim < 1 || out_dim > GAN_MX_MAX_IN || !dtype_ok(dtype)) return 0;
    const size_t np = to64(out_dim), parts = parts_of(dtype);
    return in_dim * np * 2 + (dy_as_is(dtype, out_dim) ? 0 : parts * rows * np * 2) +
           bf16_product_workspace(rows, in_dim, (int)parts, (int)np);
}

int gan_mx_matmul_dgrad(int dtype, int rows, int in_dim, int out_dim, const void* dy, const void* w_codes, const void* w_scales,
                        void* dx, void* ws, size_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype), "gan_mx_matmul_dgrad: unknown element type %d", dtype);
    GAN_CHECK_ARG(rows >= 0 && rows <= GAN_MX_MAX_ROWS && in_dim >= 1 && in_dim <= GAN_MX_MAX_IN && out_dim >= 1 && out_dim <= GAN_MX_MAX_IN,
                  "gan_mx_matmul_dgrad: %d rows, %d inputs, %d outputs (up to %d rows and %d of the others are served)", rows, in_dim, out_dim, GAN_MX_MAX_ROWS, GAN_MX_MAX_IN);
    if (rows == 0) return 0;
    GAN_CHECK_ARG(dy && w_codes && w_scales && dx, "gan_mx_matmul_dgrad: null pointer");
    GAN_CHECK_ARG(aligned16(dy) && aligned16(w_codes) && (reinterpret_cast<size_t>(w_scales) & 3) == 0,
                  "gan_mx_matmul_dgrad: dy and codes have to be 16-byte and scales 4-byte aligned");
    const size_t need = gan_mx_matmul_dgrad_workspace_bytes(dtype, rows, in_dim, out_dim);
    GAN_CHECK_ARG(ws && aligned16(ws) && ws_bytes >= need,
                  "gan_mx_matmul_dgrad: workspace of %zu bytes needed (16-byte aligned), %zu given", need, ws_bytes);
    const hipStream_t st = as_stream(stream);
    const long np = to64(out_dim);
    const int parts = parts_of(dtype);
    bf16_t* w = static_cast<bf16_t*>(ws);
    bf16_t* y = w + in_dim * np;
    hipLaunchKernelGGL(mx_weights_transpose_kernel, dim3((unsigned)(np / 64), mx_groups(in_dim)), dim3(256), 0, st,
                       static_cast<const unsigned char*>(w_codes), static_cast<const unsigned char*>(w_scales), w, in_dim, out_dim);
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        const bf16_t* dyp = static_cast<const bf16_t*>(dy);
        bf16_t* end = y;
        if (!dy_as_is(dtype, out_dim)) {
            hipLaunchKernelGGL((split_rows_kernel<T>), flat_grid(rows * np / 8), dim3(256), 0, st, static_cast<const T*>(dy), y,
                               (long)rows, out_dim, out_dim * sizeof(T) % 16 == 0);
            dyp = y;
            end = y + (long)parts * rows * np;
        }
        const Bf16Product p{dyp, w, np, np, rows * np, 0, parts, (int)np, rows, in_dim, nullptr, 0};
        return bf16_product(p, static_cast<T*>(dx), end, st, "gan_mx_matmul_dgrad");
    });
}

size_t gan_mx_matmul_wgrad_workspace_bytes(int dtype, int rows, int in_dim, int out_dim) {
    if (rows < 1 || rows > GAN_MX_MAX_ROWS || in_dim < 1 || in_dim > GAN_MX_MAX_IN || out_dim < 1 || out_dim > GAN_MX_MAX_IN || !dtype_ok(dtype)) return 0;
    const size_t rp = to64(rows), parts = parts_of(dtype);
    return (in_dim + parts * out_dim) * rp * 2 + (rp / 64 * out_dim * 4 + 15) / 16 * 16 +
           bf16_product_workspace(in_dim, out_dim, (int)parts, (int)rp);
}

int gan_mx_matmul_wgrad(int dtype, int fmt, int rows, int in_dim, int out_dim, const void* a_codes, const void* a_scales,
                        const void* dy, float* dmatrix, float* dbias, int accumulate, void* ws, size_t ws_bytes,
                        gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype) && mx_fmt_ok(fmt), "gan_mx_matmul_wgrad: unknown element type %d or format %d", dtype, fmt);
    GAN_CHECK_ARG(rows >= 1 && rows <= GAN_MX_MAX_ROWS && in_dim >= 1 && in_dim <= GAN_MX_MAX_IN && out_dim >= 1 && out_dim <= GAN_MX_MAX_IN,
                  "gan_mx_matmul_wgrad: %d rows, %d inputs, %d outputs (up to %d rows and %d of the others are served)", rows, in_dim, out_dim, GAN_MX_MAX_ROWS, GAN_MX_MAX_IN);
    GAN_CHECK_ARG(dy && a_codes && a_scales && dmatrix, "gan_mx_matmul_wgrad: null pointer");
    GAN_CHECK_ARG(aligned16(dy) && aligned16(a_codes), "gan_mx_matmul_wgrad: dy and codes have to be 16-byte aligned");
    const size_t need = gan_mx_matmul_wgrad_workspace_bytes(dtype, rows, in_dim, out_dim);
    GAN_CHECK_ARG(ws && aligned16(ws) && ws_bytes >= need,
                  "gan_mx_matmul_wgrad: workspace of %zu bytes needed (16-byte aligned), %zu given", need, ws_bytes);
    const hipStream_t st = as_stream(stream);
    const long rp = to64(rows);
    const int parts = parts_of(dtype), blocks = (int)(rp / 64);
    bf16_t* a = static_cast<bf16_t*>(ws);
    bf16_t* y = a + in_dim * rp;
    float* colsum = reinterpret_cast<float*>(y + (long)parts * out_dim * rp);
    void* end = reinterpret_cast<char*>(colsum) + ((size_t)blocks * out_dim * 4 + 15) / 16 * 16;
    const dim3 ga((in_dim + 63) / 64, blocks), gy((out_dim + 63) / 64, blocks);
    const unsigned char* c = static_cast<const unsigned char*>(a_codes);
    const unsigned char* s = static_cast<const unsigned char*>(a_scales);
    if (fmt == GAN_MX_E4M3) hipLaunchKernelGGL(mx_rows_transpose_kernel<GAN_MX_E4M3>, ga, dim3(256), 0, st, c, s, a, rows, in_dim);
    else hipLaunchKernelGGL(mx_rows_transpose_kernel<GAN_MX_E2M1>, ga, dim3(256), 0, st, c, s, a, rows, in_dim);
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        hipLaunchKernelGGL((split_transpose_kernel<T>), gy, dim3(256), 0, st, static_cast<const T*>(dy), y,
                           dbias ? colsum : nullptr, rows, out_dim, out_dim * sizeof(T) % 16 == 0);
        if (dbias)
            hipLaunchKernelGGL(mx_dbias_kernel, dim3((out_dim + 31) / 32), dim3(256), 0, st, colsum, dbias, blocks, out_dim, accumulate);
        const Bf16Product p{a, y, rp, rp, 0, out_dim * rp, parts, (int)rp, in_dim, out_dim, nullptr, accumulate};
        return bf16_product(p, dmatrix, end, st, "gan_mx_matmul_wgrad");
    });
}

}  // extern "C"
