// The bf16-pipe product and the gradients of the microscaled product.
//
//   dA[r][k] = sum_n dY[r][n] W[k][n]      dW[k][n] = sum_r A[r][k] dY[r][n]      dbias[n] = sum_r dY[r][n]
//
// with A and W the quantised values (the gradient of the quantisers is passed straight through).  Quantised values are exact in
// bf16; dY is split exactly into one (bf16), two (fp16: 11 = 8 + 3 bits) or three (fp32: 24 = 8 + 8 + 8) bf16 parts, whose
// products are summed in fp32.  So a gradient carries the error of an fp32 sum of exact products whatever the type (of an fp32 dY
// below 2^-110 what lies under bf16's smallest step of 2^-133 is lost).
//
// Memory-bound passes turn the operands into bf16 images whose contraction axis is filled up with zeros to a multiple of 64 -- one
// image of dY for both products, none where dY is bf16 in whole 64s --, then one compute-bound kernel runs each product.  It takes
// operands that contract over contiguous values (dY for dA) and over rows (W for dA, A and dY for dW) as they are.
#include "mx_gemm.h"

namespace gan {

// The LDS's transposing read.  (The restrict is for the compiler's waits: of an access that it knows nothing about it assumes that it
// reads what a copy in flight writes, and waits for all of them.)
typedef __attribute__((address_space(3))) i16x4* lds_i16x4;
__device__ __forceinline__ i16x4 read_transposed(lds_i16x4 __restrict__ from) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16(from); }

// C[i][j] over a tile of BI x BJ, WI x WJ waves, 32x32x16 instructions with Q as their first operand (a lane ends with four
// consecutive j of one i).  A stage in LDS is 64 deep: 128 bytes of every row -- whole cache lines; 64 bytes a row and stage cost
// twice the requests to the L2 --, their 16-byte chunks swapped by row so that a fragment read hits all banks.  STAGES stages form
// a ring that direct copies keep filled.  The fragments of the next 16 are read while the matrix pipe works on these; the one
// barrier of a stage stands before its last quarter, when all of it has been read: it asks for the next stage and frees this one.
// Large tiles have two waves a SIMD with 128 x 64 outputs each: LDS then gives 96 bytes a clock of its 128; one wave of
// 128 x 128 needs less of it, but nothing covers its waits (4096^3: 126 us against 115, the weights' image included).
// 4096 x 4096 x 8192: 1.25 PF/s, a library product of that size 1.45.  The gradients of 1024 x 1024 x 32768 fp32 (three parts): dx 186
// us, dmatrix 207 us, 28 of them for its 134 MB.
// PT, QT: an operand lies the other way round, [contraction][rows (columns) of C].  Its part of a stage then is 64 rows of BI (BJ)
// values, their 64-byte pieces swapped by row; a fragment, eight consecutive of the contraction for each of 32 values, is read by the
// LDS's transposing read: 16 lanes fetch 4 x 16 values, lane i keeps column i.
template <typename T, int BI, int BJ, int WI, int WJ, int STAGES, bool PT, bool QT>
__global__ __launch_bounds__(64 * WI * WJ) void bf16_product_kernel(Bf16Product p, T* out, float* slabs, int splits, bool vec) {
    constexpr int WAVES = WI * WJ, THREADS = 64 * WAVES, FI = BI / WI / 32, FJ = BJ / WJ / 32, STAGE = (BI + BJ) * 128;
    constexpr int COPIES = STAGE / 16 / THREADS;        // of a wave for a stage
    extern __shared__ __align__(16) unsigned char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wj = wave % WJ, wi = wave / WJ;
    const int l32 = lane & 31, half = lane >> 5;
    int ti, tj, split;
    tile_of(blockIdx.x, (p.rows + BI - 1) / BI, (p.cols + BJ - 1) / BJ, splits, ti, tj, split);
    const int i0 = ti * BI, j0 = tj * BJ;
    // the parts of one 64 follow each other: the operand they share then comes from the L2
    const long steps = (long)(p.depth / 64) * p.parts;
    const int s0 = (int)(steps * split / splits), s1 = (int)(steps * (split + 1) / splits);

    // where this lane's copies begin, and the two operands' places in the part at hand (rows beyond the last: the last again)
    constexpr int PC = BI * 8 / THREADS, QC = BJ * 8 / THREADS;
    unsigned p_off[PC], q_off[QC];
    auto offset = [&](auto trans, int at, auto width, int first, int last, long ld) -> unsigned {
        constexpr int kChunks = decltype(width)::value / 8;
        if constexpr (decltype(trans)::value) {      // (chunks beyond the row: its last again)
            const int k = at / kChunks, chunk = at % kChunks ^ (k & 3) << 2;
            return (unsigned)k * (unsigned)(ld * 2) + (unsigned)min(first + chunk * 8, (int)ld - 8) * 2u;
        } else {
            const int row = at >> 3, chunk = (at & 7) ^ (row & 7);
            return (unsigned)min(row, last - first) * (unsigned)(ld * 2) + chunk * 16;
        }
    };
#pragma unroll
    for (int i = 0; i < PC; ++i)
        p_off[i] = offset(std::bool_constant<PT>(), (i * WAVES + wave) * 64 + lane, std::integral_constant<int, BI>(), i0, p.rows - 1, p.ldp);
#pragma unroll
    for (int i = 0; i < QC; ++i)
        q_off[i] = offset(std::bool_constant<QT>(), (i * WAVES + wave) * 64 + lane, std::integral_constant<int, BJ>(), j0, p.cols - 1, p.ldq);
    int filled = s0, part = s0 % p.parts;
    const long p_step = PT ? 64 * p.ldp : 64, q_step = QT ? 64 * p.ldq : 64;
    const unsigned char* pp =
        reinterpret_cast<const unsigned char*>(p.p + (PT ? 0 : i0 * p.ldp) + s0 / p.parts * p_step + part * p.pstep);
    const unsigned char* qp =
        reinterpret_cast<const unsigned char*>(p.q + (QT ? 0 : j0 * p.ldq) + s0 / p.parts * q_step + part * p.qstep);
    const long p_jump = (p_step - (p.parts - 1) * p.pstep) * 2, q_jump = (q_step - (p.parts - 1) * p.qstep) * 2;
    // copies of the stage after the last one copied, into LDS from `to` on; past the end the last one again, which nobody reads
    auto fill = [&](int to) {
        unsigned char* base = lds + to;
#pragma unroll
        for (int i = 0; i < PC; ++i) copy_to_lds16(copy_source(pp), p_off[i], base + (i * WAVES + wave) * 1024);
#pragma unroll
        for (int i = 0; i < QC; ++i) copy_to_lds16(copy_source(qp), q_off[i], base + BI * 128 + (i * WAVES + wave) * 1024);
        const bool more = ++filled < s1, jump = part == p.parts - 1;
        part = jump ? 0 : part + 1;
        pp += more ? (jump ? p_jump : 2 * p.pstep) : 0L;
        qp += more ? (jump ? q_jump : 2 * p.qstep) : 0L;
    };
    struct Fragments {
        bf16x8 p[FI], q[FJ];
    };
    auto fragment = [&](auto trans, const unsigned char* base, auto width, int f, int k) -> bf16x8 {     // the f-th 32 of an operand
        if constexpr (decltype(trans)::value) {
            constexpr int kPitch = decltype(width)::value * 2;
            const int row = k * 16 + half * 8 + (lane >> 2 & 3);        // (row + 4 has the same swap)
            const unsigned char* at = base + row * kPitch + ((f ^ (row & 3)) * 64) + (lane >> 4 & 1) * 32 + (lane & 3) * 8;
            const i16x4 a = read_transposed((lds_i16x4)at), b = read_transposed((lds_i16x4)(at + 4 * kPitch));
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            const int row = f * 32 + l32;
            return *reinterpret_cast<const bf16x8*>(base + row * 128 + (((2 * k + half) ^ (row & 7)) * 16));
        }
    };
    auto read = [&](int at, int k, Fragments& f) {
        const unsigned char* base = lds + at;
#pragma unroll
        for (int j = 0; j < FJ; ++j) f.q[j] = fragment(std::bool_constant<QT>(), base + BI * 128, std::integral_constant<int, BJ>(), wj * FJ + j, k);
#pragma unroll
        for (int i = 0; i < FI; ++i) f.p[i] = fragment(std::bool_constant<PT>(), base, std::integral_constant<int, BI>(), wi * FI + i, k);
    };
    constexpr int READS = FI * (PT ? 2 : 1) + FJ * (QT ? 2 : 1);
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
            interleave<FI * FJ, READS, 0>();
        }
        landed_barrier<(STAGES - 2) * COPIES>();        // the next stage is there; STAGES - 2 more are on their way
        const int freed = at;
        at = at + STAGE == STAGES * STAGE ? 0 : at + STAGE;
        read(at, 0, f[0]);
        fill(freed);
        multiply(f[1]);
        interleave<FI * FJ, READS, COPIES>();
    }
    landed_barrier<0>();        // (no copy is in flight when the workgroup gives its LDS back)
    float* stage = reinterpret_cast<float*>(lds) + wave * 32 * (32 * FJ + 4);
    static_assert(WAVES * 32 * (32 * FJ + 4) * 4 <= STAGES * STAGE, "the results pass through the stages' LDS");
    const int n4 = (p.cols + 3) / 4 * 4, col0 = j0 + wj * FJ * 32;
#pragma unroll
    for (int i = 0; i < FI; ++i) {
        const int row0 = i0 + (wi * FI + i) * 32;
        auto pick = [&](int j) -> const f32x16& { return acc[j][i]; };
        if (slabs) store_rows<float, FJ>(pick, stage, row0, col0, p.rows, n4, slabs + (long)split * p.rows * n4, n4, nullptr, 0, true);
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

template <bool PT, bool QT, typename T, int BI, int BJ, int WI, int WJ>
static int launch_bf16(const Bf16Product& p, T* out, float* slabs, int splits, bool vec, hipStream_t st, const char* what) {
    // 128 x 128: two workgroups a CU
    constexpr int STAGES = BI + BJ == 384 ? 3 : 2, LDS = STAGES * (BI + BJ) * 128;
    auto kernel = bf16_product_kernel<T, BI, BJ, WI, WJ, STAGES, PT, QT>;
    static std::atomic<unsigned long> devices{0};
    const hipError_t set = allow_lds(reinterpret_cast<const void*>(kernel), LDS, devices);
    if (set != hipSuccess) return fail("%s: %d bytes of LDS refused: %s", what, LDS, hipGetErrorString(set));
    const long tiles = (long)((p.rows + BI - 1) / BI) * ((p.cols + BJ - 1) / BJ);
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles * splits), dim3(64 * WI * WJ), LDS, st, p, out, slabs, splits, vec);
    return 0;
}

template <bool PT, bool QT, typename T>
int bf16_product(const Bf16Product& p, T* out, void* ws, hipStream_t st, const char* what) {
    const Bf16Plan plan = bf16_plan(p.rows, p.cols, p.parts, p.depth);
    const bool vec = p.cols * sizeof(T) % 16 == 0 && aligned16(out), vec4 = vec && aligned16(p.bias);
    float* slabs = plan.splits > 1 ? static_cast<float*>(ws) : nullptr;
    const int rc = plan.tile == BF16_256       ? launch_bf16<PT, QT, T, 256, 256, 2, 4>(p, out, slabs, plan.splits, vec, st, what)
                   : plan.tile == BF16_256_128 ? launch_bf16<PT, QT, T, 256, 128, 4, 2>(p, out, slabs, plan.splits, vec, st, what)
                                               : launch_bf16<PT, QT, T, 128, 128, 2, 2>(p, out, slabs, plan.splits, vec, st, what);
    if (rc) return rc;
    if (slabs) join_slabs(slabs, plan.splits, out, (long)p.rows, p.cols, p.bias, p.accumulate, vec4, st);
    return check_launch(what);
}
template int bf16_product<false, false, float>(const Bf16Product&, float*, void*, hipStream_t, const char*);

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

// dY [rows][n] -> parts [rows filled up to 64][n filled up to 64] bf16, and the sums of 64 rows of each column (for dbias); either may
// be null.  Memory-bound; a workgroup takes 64 rows x 256 columns, a thread 8 rows x 8 columns (1024 x 32768 fp32, 335 MB: 61 us =
// 5.5 TB/s).
template <typename T>
__device__ __forceinline__ void split_block(const T* __restrict__ y, bf16_t* __restrict__ out, float* __restrict__ colsum, int rows,
                                            int n, bool vec, int accumulate, int bx, int by, float (*red)[256]) {
    const int rp = (int)to64(rows), np = (int)to64(n);
    const int t = threadIdx.x % 32, group = threadIdx.x / 32, i0 = bx * 256 + t * 8, r0 = by * 64 + group;
    float s[8] = {}, v[8][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int row = r0 + 8 * k;
        load8(y + (long)min(row, rows - 1) * n, i0, row < rows && i0 < n ? n : 0, vec, v[k]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += v[k][j];
        if (!out || i0 >= np) continue;
#pragma unroll
        for (int part = 0; part < Parts<T>::n; ++part) {
            bf16x8 b;
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = split_part(v[k][j], part);
            *reinterpret_cast<bf16x8*>(out + ((long)part * rp + r0 + 8 * k) * np + i0) = b;
        }
    }
    if (!colsum) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) red[group][t * 8 + j] = s[j];
    __syncthreads();
    const int col = bx * 256 + threadIdx.x;
    float total = 0.f;
#pragma unroll
    for (int g = 0; g < 8; ++g) total += red[g][threadIdx.x];
    if (col < n) colsum[(long)by * n + col] = (accumulate ? colsum[(long)by * n + col] : 0.f) + total;
}

// A microscaled [rows][groups * 128] -> bf16, by eights: `live` of them, then zeros up to `total`.
template <int FMT>
__device__ __forceinline__ void rows_block(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                           bf16_t* __restrict__ out, long live, long total, int block, int blocks) {
    for (long at = (long)block * 256 + threadIdx.x; at < total; at += (long)blocks * 256) {
        const float s = at < live ? mx_scale(scales[at / 4]) : 0.f;
        bf16x8 b;
        if (at >= live) {
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = (bf16_t)0.f;
        } else if constexpr (FMT == GAN_MX_E4M3) {
            const uint2 u = *reinterpret_cast<const uint2*>(codes + at * 8);
            b = e4m3_to_bf16(u.x, u.y, s);
        } else {
            b = e2m1_to_bf16(*reinterpret_cast<const unsigned*>(codes + at * 4), s);
        }
        *reinterpret_cast<bf16x8*>(out + at * 8) = b;
    }
}

// Packed W -> [filled][groups * 128] bf16, outputs and then zeros: a lane turns 8 codes of one output into 16 bytes, 16 lanes write
// 256 bytes of a row.  64 outputs of one group a workgroup.
__device__ __forceinline__ void weights_block(const unsigned char* __restrict__ codes, const unsigned char* __restrict__ scales,
                                              bf16_t* __restrict__ out, int groups, int out_dim, int filled, int bx, int g) {
    const int c = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = bx * 64 + i * 16 + threadIdx.x / 16;
        if (n >= filled) continue;
        const long at = min(n, out_dim - 1);
        const unsigned u = reinterpret_cast<const unsigned*>(codes)[(((long)g * 4 + c / 4) * out_dim + at) * 4 + c % 4];
        const float s = mx_scale(scales[((long)g * out_dim + at) * 4 + c / 4]);
        *reinterpret_cast<bf16x8*>(out + ((long)n * groups + g) * 128 + c * 8) = e2m1_to_bf16(n < out_dim ? u : 0u, n < out_dim ? s : 1.f);
    }
}

// All images that a call needs, in one launch: first the workgroups of dY, then A's, then W's.
struct Images {
    const void* dy;
    bf16_t* y;
    float* colsum;
    int rows, n;
    bool vec;
    int accumulate;                 // into colsum: up to 64 rows, of which it is dbias itself
    const unsigned char *a_codes, *a_scales;
    bf16_t* a;
    long live, total;
    const unsigned char *w_codes, *w_scales;
    bf16_t* w;
    int groups, out_dim, filled;
    int y_blocks, a_blocks, w_blocks;
};
template <typename T, int FMT>
__global__ __launch_bounds__(256) void images_kernel(Images p) {
    __shared__ float red[8][256];
    int b = blockIdx.x;
    if (b < p.y_blocks) {
        const int across = (int)((to64(p.n) + 255) / 256);
        split_block(static_cast<const T*>(p.dy), p.y, p.colsum, p.rows, p.n, p.vec, p.accumulate, b % across, b / across, red);
        return;
    }
    b -= p.y_blocks;
    if (b < p.a_blocks) {
        rows_block<FMT>(p.a_codes, p.a_scales, p.a, p.live, p.total, b, p.a_blocks);
        return;
    }
    b -= p.a_blocks;
    weights_block(p.w_codes, p.w_scales, p.w, p.groups, p.out_dim, p.filled, b / p.groups, b % p.groups);
}
// Adds A [rows][groups * 128], filled up to `filled` rows, or W, filled up to `filled` outputs, to the images of a call.
static void add_a(Images& m, const void* codes, const void* scales, bf16_t* a, long rows, long filled, int in_dim) {
    m.a_codes = static_cast<const unsigned char*>(codes);
    m.a_scales = static_cast<const unsigned char*>(scales);
    m.a = a;
    m.live = rows * mx_groups(in_dim) * 16;
    m.total = filled * mx_groups(in_dim) * 16;
    const long blocks = (m.total + 255) / 256;
    m.a_blocks = (int)(blocks < 8192 ? blocks : 8192);
}
static void add_w(Images& m, const void* codes, const void* scales, bf16_t* w, int in_dim, int out_dim, int filled) {
    m.w_codes = static_cast<const unsigned char*>(codes);
    m.w_scales = static_cast<const unsigned char*>(scales);
    m.w = w;
    m.groups = mx_groups(in_dim);
    m.out_dim = out_dim;
    m.filled = filled;
    m.w_blocks = (filled + 63) / 64 * m.groups;
}
template <typename T>
static void make_images(const Images& m, int fmt, hipStream_t st) {
    const dim3 grid((unsigned)m.y_blocks + (unsigned)m.a_blocks + (unsigned)m.w_blocks);
    if (grid.x == 0) return;
    if (fmt == GAN_MX_E4M3) hipLaunchKernelGGL((images_kernel<T, GAN_MX_E4M3>), grid, dim3(256), 0, st, m);
    else hipLaunchKernelGGL((images_kernel<T, GAN_MX_E2M1>), grid, dim3(256), 0, st, m);
}
void mx_product_images(int fmt, const void* a_codes, const void* a_scales, bf16_t* a, int rows, const void* w_codes, const void* w_scales,
                       bf16_t* w, int in_dim, int out_dim, hipStream_t st) {
    Images m{};
    add_a(m, a_codes, a_scales, a, rows, rows, in_dim);
    add_w(m, w_codes, w_scales, w, in_dim, out_dim, out_dim);
    make_images<float>(m, fmt, st);
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

static int parts_of(int dtype) { return dtype == GAN_BF16 ? 1 : dtype == GAN_F16 ? 2 : 3; }

// The gradients of one product, dx and dmatrix both or either, with their images' places in the workspace.
struct Gradients {
    int dtype, fmt, rows, in_dim, out_dim;
    const void *a_codes, *a_scales, *w_codes, *w_scales, *dy;
    void* dx;
    float *dmatrix, *dbias;
    int accumulate;
};
struct GradientImages {
    bool as_is;                     // dY itself is the operand: bf16, nothing to fill up
    long ldy, rp, kp;               // row strides of dY's image and of A's and W's; rows of the first two
    size_t y, w, a, colsum, slabs, bytes;       // offsets
};

static GradientImages gradient_images(int dtype, int rows, int in_dim, int out_dim, bool dx, bool dmatrix) {
    GradientImages g;
    // (dx contracts over outputs, dmatrix over rows: steps of 64)
    g.as_is = dtype == GAN_BF16 && (!dx || out_dim % 64 == 0) && (!dmatrix || (rows % 64 == 0 && out_dim % 8 == 0));
    g.ldy = g.as_is ? out_dim : to64(out_dim);
    g.rp = to64(rows);
    g.kp = mx_groups(in_dim) * 128L;
    const int parts = parts_of(dtype);
    const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    size_t slabs = 0;
    if (dx) slabs = bf16_product_workspace(rows, in_dim, parts, (int)to64(out_dim));
    if (dmatrix) {
        const size_t more = bf16_product_workspace(in_dim, out_dim, parts, (int)g.rp);
        slabs = more > slabs ? more : slabs;
    }
    g.y = 0;
    g.w = g.y + (g.as_is ? 0 : up((size_t)parts * g.rp * g.ldy * 2));
    g.a = g.w + (dx ? up((size_t)to64(out_dim) * g.kp * 2) : 0);
    g.colsum = g.a + (dmatrix ? up((size_t)g.rp * g.kp * 2) : 0);
    g.slabs = g.colsum + (dmatrix ? up((size_t)g.rp / 64 * out_dim * 4) : 0);
    g.bytes = g.slabs + slabs;
    return g;
}

static bool gradient_sizes_ok(int rows, int in_dim, int out_dim) {
    return rows <= GAN_MX_MAX_ROWS && in_dim >= 1 && in_dim <= GAN_MX_MAX_IN && out_dim >= 1 && out_dim <= GAN_MX_MAX_IN;
}
static size_t gradient_bytes(int dtype, int rows, int in_dim, int out_dim, bool dx, bool dmatrix) {
    if (rows < 1 || !gradient_sizes_ok(rows, in_dim, out_dim) || !dtype_ok(dtype)) return 0;
    return gradient_images(dtype, rows, in_dim, out_dim, dx, dmatrix).bytes;
}

static int gradients(const Gradients& g, void* ws, size_t ws_bytes, hipStream_t st, const char* what) {
    const bool dm = g.dmatrix != nullptr, dx = g.dx != nullptr;
    GAN_CHECK_ARG(dtype_ok(g.dtype) && mx_fmt_ok(g.fmt), "%s: unknown element type %d or format %d", what, g.dtype, g.fmt);
    GAN_CHECK_ARG(g.rows >= (dm ? 1 : 0) && gradient_sizes_ok(g.rows, g.in_dim, g.out_dim),
                  "%s: %d rows, %d inputs, %d outputs (up to %d rows and %d of the others are served)", what, g.rows, g.in_dim,
                  g.out_dim, GAN_MX_MAX_ROWS, GAN_MX_MAX_IN);
    if (g.rows == 0) return 0;
    GAN_CHECK_ARG(g.dy && (dx || dm) && (!dx || (g.w_codes && g.w_scales)) && (!dm || (g.a_codes && g.a_scales)), "%s: null pointer", what);
    GAN_CHECK_ARG(aligned16(g.dy) && aligned16(g.w_codes) && aligned16(g.a_codes) &&
                  ((reinterpret_cast<size_t>(g.w_scales) | reinterpret_cast<size_t>(g.a_scales)) & 3) == 0,
                  "%s: dy and codes have to be 16-byte and scales 4-byte aligned", what);
    const GradientImages im = gradient_images(g.dtype, g.rows, g.in_dim, g.out_dim, dx, dm);
    GAN_CHECK_ARG(im.bytes == 0 || (ws && aligned16(ws) && ws_bytes >= im.bytes),
                  "%s: workspace of %zu bytes needed (16-byte aligned), %zu given", what, im.bytes, ws_bytes);
    char* base = static_cast<char*>(ws);
    float* colsum = dm && g.dbias ? reinterpret_cast<float*>(base + im.colsum) : nullptr;
    bf16_t* w = reinterpret_cast<bf16_t*>(base + im.w);
    bf16_t* a = reinterpret_cast<bf16_t*>(base + im.a);
    bf16_t* image = im.as_is ? nullptr : reinterpret_cast<bf16_t*>(base + im.y);
    const bf16_t* y = im.as_is ? static_cast<const bf16_t*>(g.dy) : image;
    const int parts = parts_of(g.dtype), blocks = (int)(im.rp / 64);
    const long np = to64(g.out_dim);
    return with_dtype(g.dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        Images m{};
        if (image || colsum) {
            m.dy = g.dy;
            m.y = image;
            m.colsum = colsum && blocks == 1 ? g.dbias : colsum;
            m.accumulate = blocks == 1 && g.accumulate;
            m.rows = g.rows;
            m.n = g.out_dim;
            m.vec = g.out_dim * sizeof(T) % 16 == 0;
            m.y_blocks = (int)((np + 255) / 256) * blocks;
        }
        if (dm) add_a(m, g.a_codes, g.a_scales, a, g.rows, im.rp, g.in_dim);
        if (dx) add_w(m, g.w_codes, g.w_scales, w, g.in_dim, g.out_dim, (int)np);
        make_images<T>(m, g.fmt, st);
        if (dm) {
            if (g.dbias && blocks > 1)
                hipLaunchKernelGGL(mx_dbias_kernel, dim3((g.out_dim + 31) / 32), dim3(256), 0, st, colsum, g.dbias, blocks, g.out_dim,
                                   g.accumulate);
            const Bf16Product p{a, y, im.kp, im.ldy, 0, im.rp * im.ldy, parts, (int)im.rp, g.in_dim, g.out_dim, nullptr, g.accumulate};
            if (const int rc = bf16_product<true, true>(p, g.dmatrix, base + im.slabs, st, what)) return rc;
        }
        if (!dx) return 0;
        const Bf16Product p{y, w, im.ldy, im.kp, im.rp * im.ldy, 0, parts, (int)np, g.rows, g.in_dim, nullptr, 0};
        return bf16_product<false, true>(p, static_cast<T*>(g.dx), base + im.slabs, st, what);
    });
}

}  // namespace gan

using namespace gan;

extern "C" {

size_t gan_mx_matmul_dgrad_workspace_bytes(int dtype, int rows, int in_dim, int out_dim) {
    return gradient_bytes(dtype, rows, in_dim, out_dim, true, false);
}

int gan_mx_matmul_dgrad(int dtype, int rows, int in_dim, int out_dim, const void* dy, const void* w_codes, const void* w_scales,
                        void* dx, void* ws, size_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(rows == 0 || dx, "gan_mx_matmul_dgrad: null pointer");
    const Gradients g{dtype, GAN_MX_E4M3, rows, in_dim, out_dim, nullptr, nullptr, w_codes, w_scales, dy, dx, nullptr, nullptr, 0};
    return gradients(g, ws, ws_bytes, as_stream(stream), "gan_mx_matmul_dgrad");
}

size_t gan_mx_matmul_wgrad_workspace_bytes(int dtype, int rows, int in_dim, int out_dim) {
    return gradient_bytes(dtype, rows, in_dim, out_dim, false, true);
}

int gan_mx_matmul_wgrad(int dtype, int fmt, int rows, int in_dim, int out_dim, const void* a_codes, const void* a_scales,
                        const void* dy, float* dmatrix, float* dbias, int accumulate, void* ws, size_t ws_bytes,
                        gan_stream_t stream) {
    GAN_CHECK_ARG(dmatrix, "gan_mx_matmul_wgrad: null pointer");
    const Gradients g{dtype, fmt, rows, in_dim, out_dim, a_codes, a_scales, nullptr, nullptr, dy, nullptr, dmatrix, dbias, accumulate};
    return gradients(g, ws, ws_bytes, as_stream(stream), "gan_mx_matmul_wgrad");
}

size_t gan_mx_matmul_bwd_workspace_bytes(int dtype, int rows, int in_dim, int out_dim) {
    return gradient_bytes(dtype, rows, in_dim, out_dim, true, true);
}

int gan_mx_matmul_bwd(int dtype, int fmt, int rows, int in_dim, int out_dim, const void* a_codes, const void* a_scales,
                      const void* w_codes, const void* w_scales, const void* dy, void* dx, float* dmatrix, float* dbias,
                      int accumulate, void* ws, size_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(dx && dmatrix, "gan_mx_matmul_bwd: null pointer");
    const Gradients g{dtype, fmt, rows, in_dim, out_dim, a_codes, a_scales, w_codes, w_scales, dy, dx, dmatrix, dbias, accumulate};
    return gradients(g, ws, ws_bytes, as_stream(stream), "gan_mx_matmul_bwd");
}

}  // extern "C"
