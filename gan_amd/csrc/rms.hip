// Root-mean-square norm with the residual's addition, forward and backward.
//
//   h = T(x + r)   s = 1 / sqrt(mean(h^2) + eps)   y = h s gamma
//   g = dy gamma   n = h s   dx = dr = s (g - n mean(g n)) + dh   dgamma = sum over rows of dy n
//
// h is rounded to the tensors' type before it is normalised: it is the residual stream that is stored and that the backward
// pass reads again, so forward and backward see one h.  The sum of squares is fp64, so that no finite row overflows it; the
// backward's sums are fp32.  In front of the 8-bit output y is fp64 too: the row is one division away from a grid with steps of
// 1/8, and with y rounded once from 64 bits a value next to a border falls on its own side (fp64 runs at the fp32 rate here, and
// the kernel waits for memory: no cost was measurable).
//
// Memory-bound.  A team of 8 to 1024 threads keeps a whole row in registers, eight values a chunk, so every tensor is read and
// written once.  bf16 with a residual: 8192 x 4096 to 8 bits 45 us = 5.2 TB/s; 16384 x 2048 forward 46 us = 5.8 TB/s, backward 51 + 4
// us = 4.9 TB/s (a large copy reaches 4.8 TB/s on this card, an addition in place 5.9); one row of 4096 3.2 us, which is the launch and
// two trips to memory.
#include "mx.h"

namespace gan {

// Sum over the TPR threads of a team, in all of them: lanes of a wave, or whole waves by way of `red`.
template <int TPR, typename S>
__device__ __forceinline__ S team_sum(S v, S* red) {
    if constexpr (TPR < 64) {
        v += row_swizzle<0xb1>(v);
        v += row_swizzle<0x4e>(v);
        v += row_swizzle<0x141>(v);
        if constexpr (TPR >= 16) v += row_swizzle<0x140>(v);
        if constexpr (TPR == 32) v += __shfl_xor(v, 16, 64);
    } else {
        v = wave_all_sum(v);
        if constexpr (TPR > 64) {
            __syncthreads();
            if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
            __syncthreads();
            v = 0;
#pragma unroll
            for (int i = 0; i < TPR / 64; ++i) v += red[i];
        }
    }
    return v;
}

struct RmsFwd {
    const void* x;
    const void* res;
    const float* gamma;
    void* h;
    void* y;
    unsigned char* codes;
    unsigned char* scales;
    float* rstd;
    long rows, ldx, ldr;
    int c;
    float eps;
    bool vec_x, vec_r, vec_o, vec_g;
};

template <typename T, int TPR, int NV, bool MX>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_fwd_kernel(RmsFwd p) {
    constexpr int TEAMS = TPR < 256 ? 256 / TPR : 1;
    __shared__ double red[TPR / 64 + 1];
    const int t = threadIdx.x % TPR, team = threadIdx.x / TPR;
    const int c = p.c, chunks = MX ? mx_groups(c) * 16 : (c + 7) / 8;
    const long row = ((long)blockIdx.y * gridDim.x + blockIdx.x) * TEAMS + team;
    const bool live = row < p.rows;
    const T* xr = static_cast<const T*>(p.x) + (live ? row : 0) * p.ldx;
    const T* rr = p.res ? static_cast<const T*>(p.res) + (live ? row : 0) * p.ldr : nullptr;
    float v[NV][8], g[NV][8];
    double s = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int i0 = (i * TPR + t) * 8;
        load8(xr, i0, i0 < c ? c : 0, p.vec_x, v[i]);
        if (rr) load8(rr, i0, i0 < c ? c : 0, p.vec_r, g[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int i0 = (i * TPR + t) * 8;
        if (rr) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = (float)(T)(v[i][j] + g[i][j]);
            if (live && i0 < c) store8(static_cast<T*>(p.h) + row * c, i0, c, p.vec_o, v[i]);
        }
        load8(p.gamma, i0, i0 < c ? c : 0, p.vec_g, g[i]);      // (on its way while the row is summed)
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fma((double)v[i][j], (double)v[i][j], s);
    }
    const double inv = 1.0 / sqrt(team_sum<TPR>(s, red) / c + (double)p.eps);
    const float rstd = (float)inv;
    // (1 / a subnormal root is beyond fp32: such rows are lifted by a power of two, all others multiplied by 1)
    const bool lifted = inv > 0x1p100;
    const float up = lifted ? 0x1p100f : 1.f, norm = lifted ? (float)(inv * 0x1p-100) : rstd;
    if (!live) return;
    if (p.rstd && t == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int chunk = i * TPR + t, i0 = chunk * 8;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            y[j] = MX ? (float)((double)v[i][j] * inv * (double)g[i][j]) : v[i][j] * up * norm * g[i][j];
        if (MX) {
            unsigned code[2];
            const unsigned byte = mx_quantize_lane8<GAN_MX_E4M3>(y, code);   // (all lanes: the block's four exchange maxima)
            if (chunk < chunks) {
                *reinterpret_cast<uint2*>(p.codes + row * (chunks * 8L) + i0) = make_uint2(code[0], code[1]);
                if ((chunk & 3) == 0) p.scales[row * (chunks / 4L) + chunk / 4] = (unsigned char)byte;
            }
        } else if (i0 < c) {
            store8(static_cast<T*>(p.y) + row * c, i0, c, p.vec_o, y);
        }
    }
}

struct RmsBwd {
    const void* h;
    const float* gamma;
    const float* rstd;
    const void* dy;
    const void* dh;
    void* dx;
    float* partial;     // [workgroups][c], or null
    long rows, ldh;
    int c;
    bool vec_h, vec_o, vec_g;
};

constexpr int kRmsTwice = 4;        // chunks a thread from which a row is read twice

// Every team walks the rows from its own number on in steps of the number of teams and adds dy n up in registers (the columns of a
// thread are the same in every row).  The teams of a workgroup join their sums in LDS, rms_dgamma_kernel those of the workgroups,
// both in a fixed order.
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_bwd_kernel(RmsBwd p) {
    constexpr int TEAMS = TPR < 256 ? 256 / TPR : 1;
    __shared__ float red[TPR / 64 + 1];
    const int t = threadIdx.x % TPR, c = p.c;
    const long team = (long)blockIdx.x * TEAMS + threadIdx.x / TPR, teams = (long)gridDim.x * TEAMS;
    // 1024 threads have 128 registers each: with one chunk gamma stays in them and dh comes with the row, with two gamma and dh are
    // read when they are wanted, with four the sums are in LDS and the row is read again for its gradient (32M bf16 values in rows of
    // 32768: 208 us held and spilled, 86 so)
    constexpr bool kHold = TPR < 1024 || NV == 1, kTwice = NV == kRmsTwice;
    extern __shared__ __align__(16) float sums[];      // [NV * 8][TPR], kTwice only
    float acc[kTwice ? 1 : NV][8], w[kTwice ? 1 : NV][8];
    if constexpr (kTwice) {
        for (int i = 0; i < NV * 8; ++i) sums[i * TPR + t] = 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int i0 = (i * TPR + t) * 8;
            if constexpr (kHold) load8(p.gamma, i0, i0 < c ? c : 0, p.vec_g, w[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = 0.f;
        }
    }
    for (long row = team; row < p.rows; row += teams) {
        const T* hr = static_cast<const T*>(p.h) + row * p.ldh;
        const T* yr = static_cast<const T*>(p.dy) + row * c;
        const T* dhr = p.dh && p.dx ? static_cast<const T*>(p.dh) + row * c : nullptr;
        const float rstd = p.rstd[row];
        if constexpr (kTwice) {
            float s = 0.f;
#pragma unroll 2
            for (int i = 0; i < NV; ++i) {
                const int i0 = (i * TPR + t) * 8, cc = i0 < c ? c : 0;
                float n[8], g[8];
                load8(hr, i0, cc, p.vec_h, n);
                load8(yr, i0, cc, p.vec_o, g);
                load8(p.gamma, i0, cc, p.vec_g, w[0]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    n[j] *= rstd;
                    sums[(i * 8 + j) * TPR + t] = fmaf(g[j], n[j], sums[(i * 8 + j) * TPR + t]);
                    s = fmaf(g[j] * w[0][j], n[j], s);
                }
            }
            if (!p.dx) continue;
            const float m = team_sum<TPR>(s, red) / c;
#pragma unroll 2
            for (int i = 0; i < NV; ++i) {
                const int i0 = (i * TPR + t) * 8;
                if (i0 >= c) continue;
                float n[8], g[8], d[8], o[8];
                load8(hr, i0, c, p.vec_h, n);
                load8(yr, i0, c, p.vec_o, g);
                load8(p.gamma, i0, c, p.vec_g, w[0]);
                if (dhr) load8(dhr, i0, c, p.vec_o, d);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[j] = rstd * (g[j] * w[0][j] - n[j] * rstd * m);
                    if (dhr) o[j] += d[j];
                }
                store8(static_cast<T*>(p.dx) + row * c, i0, c, p.vec_o, o);
            }
            continue;
        } else {
            float n[NV][8], g[NV][8], d[NV][8], s = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int i0 = (i * TPR + t) * 8, cc = i0 < c ? c : 0;
                load8(hr, i0, cc, p.vec_h, n[i]);
                load8(yr, i0, cc, p.vec_o, g[i]);
                if (kHold && dhr) load8(dhr, i0, cc, p.vec_o, d[i]);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!kHold) load8(p.gamma, (i * TPR + t) * 8, (i * TPR + t) * 8 < c ? c : 0, p.vec_g, w[0]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    n[i][j] *= rstd;
                    acc[i][j] = fmaf(g[i][j], n[i][j], acc[i][j]);
                    g[i][j] *= w[kHold ? i : 0][j];
                    s = fmaf(g[i][j], n[i][j], s);
                }
            }
            if (!p.dx) continue;
            const float m = team_sum<TPR>(s, red) / c;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int i0 = (i * TPR + t) * 8;
                if (i0 >= c) continue;
                float o[8];
                if (!kHold && dhr) load8(dhr, i0, c, p.vec_o, d[i]);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[j] = rstd * (g[i][j] - n[i][j] * m);
                    if (dhr) o[j] += d[i][j];
                }
                store8(static_cast<T*>(p.dx) + row * c, i0, c, p.vec_o, o);
            }
        }
    }
    if (!p.partial) return;
    float* out = p.partial + (long)blockIdx.x * c;
    if constexpr (TEAMS == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int i0 = (i * TPR + t) * 8;
            if constexpr (kTwice) {
#pragma unroll
                for (int j = 0; j < 8; ++j) acc[0][j] = sums[(i * 8 + j) * TPR + t];
            }
            if (i0 < c) store8(out, i0, c, (c & 3) == 0, acc[kTwice ? 0 : i]);
        }
    } else {
        constexpr int W = TPR * NV * 8;
        __shared__ __align__(16) float join[TEAMS * W];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            *reinterpret_cast<f32x8*>(join + threadIdx.x / TPR * W + (i * TPR + t) * 8) =
                f32x8{acc[i][0], acc[i][1], acc[i][2], acc[i][3], acc[i][4], acc[i][5], acc[i][6], acc[i][7]};
        __syncthreads();
        for (int col = threadIdx.x; col < c; col += 256) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < TEAMS; ++i) s += join[i * W + col];
            out[col] = s;
        }
    }
}

// dgamma[col] (+)= sum over workgroups of partial[workgroup][col]: 32 columns a block, 32 rows side by side, joined in LDS.
__global__ __launch_bounds__(1024) void rms_dgamma_kernel(const float* __restrict__ partial, float* __restrict__ out, int rows,
                                                          int c, int accumulate) {
    __shared__ float red[32][33];
    const int col = blockIdx.x * 32 + (threadIdx.x & 31), part = threadIdx.x >> 5;
    float s = 0.f;
    if (col < c) {
#pragma unroll 8
        for (int i = part; i < rows; i += 32) s += partial[(long)i * c + col];
    }
    red[part][threadIdx.x & 31] = s;
    __syncthreads();
    if (part == 0 && col < c) {
        s = 0.f;
        for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
        out[col] = (accumulate ? out[col] : 0.f) + s;
    }
}

// Calls f(threads a row, chunks a thread) with a shape that holds `chunks` chunks of eight.  One chunk a thread keeps rows in few
// registers and many of them in flight: backward of 32M bf16 values (floor 45 us) with rows of 2048 52 us (two chunks 79), of 4096 54
// (72 to 80), of 8192 54 (75 to 88); a wave for a row of 1024 is better than four, 56 against 81.  In the forward pass two chunks
// in front of the 8-bit output cost less than the wider team's exchange: rows of 4096 42 us against 45, without it 46 against 43.
template <bool MX, typename F>
static void with_shape(int chunks, F f) {
#define GAN_SHAPE(tpr, nv) return f(std::integral_constant<int, tpr>(), std::integral_constant<int, nv>())
    if constexpr (!MX) {        // (8-bit rows are filled up to 16 chunks)
        if (chunks <= 8) GAN_SHAPE(8, 1);
    }
    if (chunks <= 16) GAN_SHAPE(16, 1);
    if (chunks <= 32) GAN_SHAPE(32, 1);
    if (chunks <= 64) GAN_SHAPE(64, 1);
    if (chunks <= 128) GAN_SHAPE(64, 2);
    if (chunks <= 256) GAN_SHAPE(256, 1);
    if constexpr (MX) {
        if (chunks <= 512) GAN_SHAPE(256, 2);
        if (chunks <= 1024) GAN_SHAPE(512, 2);
    } else {
        if (chunks <= 512) GAN_SHAPE(512, 1);
        if (chunks <= 1024) GAN_SHAPE(1024, 1);
    }
    if (chunks <= 2048) GAN_SHAPE(1024, 2);
    GAN_SHAPE(1024, 4);
#undef GAN_SHAPE
}

// Workgroups of the backward grid: enough to fill the chip, and few, since each leaves a row of partial sums.
static int rms_bwd_groups(long rows, int c) {
    const int chunks = (c + 7) / 8, teams = chunks <= 8 ? 32 : chunks <= 16 ? 16 : chunks <= 32 ? 8 : chunks <= 128 ? 4 : 1;    // (a workgroup's)
    const long groups = c <= 2048 ? 1024 : c <= 4096 ? 512 : 256, most = (rows + 4 * teams - 1) / (4 * teams);
    return (int)(groups < most ? groups : most);
}

constexpr int kRmsMaxWidth = 32768;

}  // namespace gan

using namespace gan;

extern "C" {

int gan_rms_norm_fwd(int dtype, long rows, int c, const void* x, long ldx, const void* residual, long ldr, const float* gamma,
                     float eps, void* h, void* y, void* mx_codes, void* mx_scales, float* rstd, gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype), "gan_rms_norm_fwd: unknown element type %d", dtype);
    GAN_CHECK_ARG(rows >= 0 && rows < (1L << 31) && c >= 1 && c <= kRmsMaxWidth,
                  "gan_rms_norm_fwd: %ld rows of %d values (1..%d values are served)", rows, c, kRmsMaxWidth);
    const bool mx = mx_codes != nullptr;
    GAN_CHECK_ARG(gamma && (rows == 0 || (x && (mx ? mx_scales && !y : y != nullptr) && (residual != nullptr) == (h != nullptr))),
                  "gan_rms_norm_fwd: null pointer (x, gamma, one of y or mx_codes with mx_scales; h exactly with a residual)");
    GAN_CHECK_ARG(ldx >= c && (!residual || ldr >= c), "gan_rms_norm_fwd: row stride smaller than the row");
    GAN_CHECK_ARG(eps >= 0.f, "gan_rms_norm_fwd: epsilon %g", (double)eps);
    GAN_CHECK_ARG(!mx || ((reinterpret_cast<size_t>(mx_codes) & 7) == 0), "gan_rms_norm_fwd: mx_codes is not 8-byte aligned");
    if (rows == 0) return 0;
    return with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        RmsFwd p{x, residual, gamma, h, y, static_cast<unsigned char*>(mx_codes), static_cast<unsigned char*>(mx_scales), rstd,
                 rows, ldx, ldr, c, eps,
                 aligned16(x) && ldx * sizeof(T) % 16 == 0, aligned16(residual) && ldr * sizeof(T) % 16 == 0,
                 c * sizeof(T) % 16 == 0 && aligned16(h) && aligned16(y), aligned16(gamma)};
        auto go = [&](auto tpr, auto nv, auto to_mx) {
            constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, TEAMS = TPR < 256 ? 256 / TPR : 1;
            // (fewer than 2^32 threads along x)
            const long blocks = (rows + TEAMS - 1) / TEAMS, along = blocks < (1L << 21) ? blocks : 1L << 21;
            const dim3 grid((unsigned)along, (unsigned)((blocks + along - 1) / along)), block(TPR < 256 ? 256 : TPR);
            hipLaunchKernelGGL((rms_fwd_kernel<T, TPR, NV, decltype(to_mx)::value>), grid, block, 0, as_stream(stream), p);
        };
        if (mx) with_shape<true>(mx_groups(c) * 16, [&](auto tpr, auto nv) { go(tpr, nv, std::true_type()); });
        else with_shape<false>((c + 7) / 8, [&](auto tpr, auto nv) { go(tpr, nv, std::false_type()); });
        return check_launch("gan_rms_norm_fwd");
    });
}

size_t gan_rms_norm_workspace_bytes(long rows, int c) {
    if (rows <= 0 || c < 1) return 0;
    return (size_t)rms_bwd_groups(rows, c) * c * sizeof(float);
}

int gan_rms_norm_bwd(int dtype, long rows, int c, const void* h, long ldh, const float* gamma, const float* rstd, const void* dy,
                     const void* dh, void* dx, float* dgamma, int accumulate, void* ws, size_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype), "gan_rms_norm_bwd: unknown element type %d", dtype);
    GAN_CHECK_ARG(rows >= 0 && rows < (1L << 31) && c >= 1 && c <= kRmsMaxWidth,
                  "gan_rms_norm_bwd: %ld rows of %d values (1..%d values are served)", rows, c, kRmsMaxWidth);
    GAN_CHECK_ARG(gamma && (rows == 0 || (h && rstd && dy)) && (dx || dgamma), "gan_rms_norm_bwd: null pointer");
    GAN_CHECK_ARG(ldh >= c, "gan_rms_norm_bwd: row stride smaller than the row");
    const size_t need = dgamma ? gan_rms_norm_workspace_bytes(rows, c) : 0;
    GAN_CHECK_ARG(ws_bytes >= need && (need == 0 || (ws && aligned16(ws))),
                  "gan_rms_norm_bwd: workspace of %zu bytes needed (16-byte aligned), %zu given", need, ws_bytes);
    const int groups = rows ? rms_bwd_groups(rows, c) : 0;
    float* partial = dgamma ? static_cast<float*>(ws) : nullptr;
    if (rows) {
        const int rc = with_dtype(dtype, [&](auto* tag) {
            typedef typename std::remove_pointer<decltype(tag)>::type T;
            RmsBwd p{h, gamma, rstd, dy, dh, dx, partial, rows, ldh, c,
                     aligned16(h) && ldh * sizeof(T) % 16 == 0,
                     c * sizeof(T) % 16 == 0 && aligned16(dy) && aligned16(dh) && aligned16(dx), aligned16(gamma)};
            hipError_t set = hipSuccess;
            with_shape<false>((c + 7) / 8, [&](auto tpr, auto nv) {
                constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, LDS = NV == kRmsTwice ? NV * 8 * TPR * 4 : 0;
                if constexpr (LDS > 0) {
                    static std::atomic<unsigned long> devices{0};
                    set = allow_lds(reinterpret_cast<const void*>(rms_bwd_kernel<T, TPR, NV>), LDS, devices);
                    if (set != hipSuccess) return;
                }
                hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, NV>), dim3(groups), dim3(TPR < 256 ? 256 : TPR), LDS,
                                   as_stream(stream), p);
            });
            if (set != hipSuccess) return fail("gan_rms_norm_bwd: LDS refused: %s", hipGetErrorString(set));
            return check_launch("gan_rms_norm_bwd");
        });
        if (rc) return rc;
    }
    if (dgamma) {
        hipLaunchKernelGGL(rms_dgamma_kernel, dim3((c + 31) / 32), dim3(1024), 0, as_stream(stream), partial, dgamma, groups, c,
                           accumulate);
        return check_launch("gan_rms_norm_bwd");
    }
    return 0;
}

}  // extern "C"
