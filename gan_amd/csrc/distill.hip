// Distillation from a teacher's top logits: mean over rows of a Kullback-Leibler divergence, fused with its gradient.
//
//   z = s / tau, t' = t / tau; list entries whose class is outside [0, classes) or whose logit is -inf are left out.  Maxima and
//   differences are taken before the division, which could carry a mask of the type's lowest value to -inf
//   p_i = softmax of t' over the list, or exp(t'_i - lse) where the teacher's log-sum-exp is given
//   l = sum_i p_i (log p_i - log q_i)  [+ p_r (log p_r - log q_r)],   q = softmax z
//   p_r = max(0, 1 - sum p), q_r = sum of q over the classes not listed (with lse only; where q_r is 0, with every class listed or
//   all others at -inf, l has no such term and p_r is 0)
//   dl/dz_j = P q_j - p_j (listed), P q_j - p_r q_j / q_r (others), P = sum p + p_r
//
// Memory-bound: the logits are read once, held in registers, and their gradient is written once (2048 x 131072 bf16, the half of a
// row beyond the registers read twice: 244 us = 4.4 TB/s of logits and gradient; 1024 x 32768 fp32 51 us = 5.3 TB/s).  One workgroup
// a row, its threads hold the row in 16-byte chunks of the tensor's type; maximum and sum of exponentials come from two passes over
// the registers, joined over the workgroup in one exchange; a third pass writes the gradient.
// q_r is never 1 - sum q_i, which cancels: a bit per class marks the list, and sums over the marked and the unmarked classes
// are taken apart.  The same bits tell whether a class is listed twice (its probabilities add up).
// Statistics are fp32 in an order fixed by the thread number, so results are deterministic.
#include "mx.h"

namespace gan {

struct Distill {
    const void* logits;
    void* grad;             // dense [rows][classes], or null
    const void* teacher;
    const void* index;
    const float* lse;
    const float* weight;
    const float* total;     // sum of the weights; null: the kernel adds them up itself
    float* row_loss;
    long ld, rows;
    int classes, top, teacher_dtype, index64;
    float inv_tau, grad_scale;
};

__device__ __forceinline__ float teacher_at(const Distill& p, long i) {
    if (p.teacher_dtype == GAN_F32) return static_cast<const float*>(p.teacher)[i];
    if (p.teacher_dtype == GAN_BF16) return (float)static_cast<const bf16_t*>(p.teacher)[i];
    return (float)static_cast<const f16_t*>(p.teacher)[i];
}

// e^((x - m) / tau) as 2^((x - m) c2), c2 = log2(e) / tau, with -inf as the maximum of nothing: of -inf and -inf it is 0 here.
// Maxima stay in the logits' own units: a mask of the type's lowest value times log2(e) would be an infinity.
__device__ __forceinline__ float power(float x, float m, float c2) {
    return __builtin_amdgcn_exp2f((x - (m == -INFINITY ? 0.f : m)) * c2);
}

// Maximum and sum of powers, joined: (m, s) <- (max(m, m2), s e^((m - max) / tau) + s2 e^((m2 - max) / tau)).
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2, float c2) {
    const float mm = fmaxf(m, m2);
    s = s * power(m, mm, c2) + s2 * power(m2, mm, c2);
    m = mm;
}

// 16 bytes of a row.
template <typename T> struct Chunk {
    static constexpr int n = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack(const i32x4& r, float (&v)[4], float) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __int_as_float(r[j]);
}
__device__ __forceinline__ void unpack(const i32x4& r, float (&v)[8], bf16_t) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[2 * j] = __int_as_float(r[j] << 16);
        v[2 * j + 1] = __int_as_float(r[j] & 0xffff0000);
    }
}
__device__ __forceinline__ void unpack(const i32x4& r, float (&v)[8], f16_t) {
    const f16x8 h = __builtin_bit_cast(f16x8, r);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)h[j];
}
// -inf in the places `marked` names
template <typename T>
__device__ __forceinline__ void strike(i32x4& r, unsigned marked) {
    constexpr int n = Chunk<T>::n;
    if constexpr (n == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = marked >> j & 1 ? 0xff800000 : r[j];
    } else {
        constexpr unsigned low = std::is_same<T, bf16_t>::value ? 0xff80u : 0xfc00u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned m = (marked >> (2 * j) & 1) * 0xffffu | (marked >> (2 * j + 1) & 1) * 0xffff0000u;
            r[j] = (int)(((unsigned)r[j] & ~m) | (low * 0x10001u & m));
        }
    }
}

template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_all_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
    for (int i = 0; i < NT / 64; ++i) v += red[i];
    return v;
}

// NV chunks a thread in registers; what a row has beyond them is read twice.
template <typename T, int NT, int NV, bool REST>
__global__ __launch_bounds__(NT) void distill_kernel(Distill p) {
    constexpr int N = Chunk<T>::n;
    constexpr bool kKeep = sizeof(T) == 4;      // a power takes the place of its value, and is not computed twice
    extern __shared__ __align__(16) unsigned char lds[];
    __shared__ float red[2 * NT / 64];
    // of the list: any, sum p, p_r, maximum, sum of powers, repeated classes
    __shared__ float told[6];
    __shared__ float wsum[NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, classes = p.classes;
    const long row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.ld;
    T* gr = static_cast<T*>(p.grad) + (p.grad ? row * classes : 0);
    // the row: up to N - 1 values before its first 16-byte border, whole chunks, up to N - 1 values behind them; of the loose
    // values a thread has at most one
    const int head = min(classes, (int)((16 - (reinterpret_cast<size_t>(x) & 15)) & 15) / (int)sizeof(T));
    const int chunks = (classes - head) / N, tail = head + chunks * N;
    const bool gvec = ((reinterpret_cast<size_t>(gr) ^ reinterpret_cast<size_t>(x)) & 15) == 0;
    const int loose = tid < head ? tid : tid >= 8 && tail + tid - 8 < classes && tid < 16 ? tail + tid - 8 : -1;
    unsigned* bits = reinterpret_cast<unsigned*>(lds);      // bit e - head + 8: class e is listed
    const int words = (classes + 8 + 127) / 128 * 4;
    int* l_id = reinterpret_cast<int*>(bits + words);
    float* l_p = reinterpret_cast<float*>(l_id + p.top);
    float* l_lp = l_p + p.top;
    float* l_z = l_lp + p.top;
    auto marks = [&](int chunk) -> unsigned {
        const int at = chunk * N + 8;
        return bits[at >> 5] >> (at & 31) & ((1u << N) - 1);
    };
    auto store = [&](int chunk, const float (&g)[N]) {
        T* to = gr + head + chunk * N;
        if (gvec) {
            typedef T vec __attribute__((ext_vector_type(N)));
            vec r;
#pragma unroll
            for (int j = 0; j < N; ++j) r[j] = (T)g[j];
            *reinterpret_cast<vec*>(to) = r;
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) to[j] = (T)g[j];
        }
    };

    const float w = p.weight ? p.weight[row] : 1.f;
    const float c2 = p.inv_tau * 1.44269504f;
    if (w != 0.f && tid < 64) {     // the list, by the first wave, before its share of the row
        for (int i = lane; i < words / 4; i += 64) reinterpret_cast<uint4*>(bits)[i] = make_uint4(0, 0, 0, 0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        int any = 0, twice = 0;
        float m = -INFINITY;
        for (int i = lane; i < p.top; i += 64) {
            const long at = row * p.top + i;
            const long id64 = p.index64 ? static_cast<const long*>(p.index)[at] : static_cast<const int*>(p.index)[at];
            const float t = teacher_at(p, at);
            const bool in = id64 >= 0 && id64 < classes && t != -INFINITY;
            const int id = in ? (int)id64 : -1;
            l_id[i] = id;
            l_lp[i] = t;
            l_z[i] = in ? (float)x[id] : 0.f;
            if (in) {
                any = 1;
                m = fmaxf(m, t);
                const int place = id - head + 8;
                const unsigned bit = 1u << (place & 31);
                twice |= (atomicOr(&bits[place >> 5], bit) & bit) != 0;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        any = __any(any);
        twice = __any(twice);
        float norm = 0.f;
        if (REST) {
            norm = p.lse[row];
            m = 0.f;
        } else {
            m = wave_all_max(m);
            float s = 0.f;
            for (int i = lane; i < p.top; i += 64)
                if (l_id[i] >= 0) s += expf((l_lp[i] - m) * p.inv_tau);
            norm = logf(wave_all_sum(s));
        }
        float mass = 0.f;
        for (int i = lane; i < p.top; i += 64) {
            const float lp = (l_lp[i] - m) * p.inv_tau - norm, pr = l_id[i] >= 0 ? expf(lp) : 0.f;
            l_lp[i] = lp;
            l_p[i] = pr;
            mass += pr;
        }
        float ml = -INFINITY, sl = 0.f;
        if (REST) {     // statistics of the listed classes, each once
            mass = wave_all_sum(mass);
            for (int i = lane; i < p.top; i += 64)
                if (l_id[i] >= 0) ml = fmaxf(ml, l_z[i]);
            ml = wave_all_max(ml);
            for (int i = lane; i < p.top; i += 64) {
                bool first = l_id[i] >= 0;
                if (twice)
                    for (int j = 0; j < i && first; ++j) first = l_id[j] != l_id[i];
                if (first) sl += power(l_z[i], ml, c2);
            }
            sl = wave_all_sum(sl);
        }
        if (lane == 0) {
            const float rest = REST ? fmaxf(0.f, 1.f - mass) : 0.f;
            told[0] = any ? 1.f : 0.f;
            told[1] = REST ? mass : 1.f;
            told[2] = rest;
            told[3] = ml;
            told[4] = sl;
            told[5] = twice ? 1.f : 0.f;
        }
    }
    i32x4 raw[NV];
    float lone = -INFINITY;         // the thread's loose value
    if (w != 0.f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int chunk = i * NT + tid;
            if (chunk < chunks) {
                raw[i] = *reinterpret_cast<const i32x4*>(x + head + chunk * N);
            } else {
                raw[i] = i32x4{0, 0, 0, 0};
                strike<T>(raw[i], (1u << N) - 1);
            }
        }
        if (loose >= 0) lone = (float)x[loose];
    }
    if (p.weight && !p.total) {
        float s = 0.f;
#pragma unroll 4
        for (int i = tid; i < (int)p.rows; i += NT) s += p.weight[i];
        s = wave_all_sum(s);
        if (lane == 0) wsum[tid >> 6] = s;
    }
    __syncthreads();
    if (w == 0.f || told[0] == 0.f) {       // nothing to learn in this row
        if (p.grad) {
            const float zero[N] = {};
            for (int c = tid; c < chunks; c += NT) store(c, zero);
            if (loose >= 0) gr[loose] = (T)0.f;
        }
        if (tid == 0) p.row_loss[row] = 0.f;
        return;
    }
    float total = (float)p.rows;
    if (p.weight) {
        if (p.total) {
            total = p.total[0];
        } else {
            total = 0.f;
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) total += wsum[i];
        }
    }
    const bool lone_listed = loose >= 0 && (bits[(loose - head + 8) >> 5] >> ((loose - head + 8) & 31) & 1);
    if (REST && lone_listed) lone = -INFINITY;

    // maximum and sum of powers of the unlisted classes (REST) or of all
    const int wave0 = __builtin_amdgcn_readfirstlane(tid & ~63);     // (chunks past the end of the row are skipped by whole waves)
    float m = lone, s = 0.f, own;
    {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * NT + wave0 >= chunks) continue;
            if (REST && i * NT + tid < chunks) {
                const unsigned marked = marks(i * NT + tid);
                if (marked) strike<T>(raw[i], marked);
            }
            float v[N];
            unpack(raw[i], v, T());
#pragma unroll
            for (int j = 0; j < N; ++j) m = fmaxf(m, v[j]);
        }
        const float off = m == -INFINITY ? 0.f : m;
        own = m;        // (of a thread with masked classes alone -inf, whose power is 0)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * NT + wave0 >= chunks) continue;
            asm volatile("" : "+v"(raw[i]));        // unpack again here: keeping every pass's values costs more registers than there are
            float v[N];
            unpack(raw[i], v, T());
#pragma unroll
            for (int j = 0; j < N; ++j) {
                v[j] = __builtin_amdgcn_exp2f((v[j] - off) * c2);
                s += v[j];
                if constexpr (kKeep) raw[i][j] = __float_as_int(v[j]);
            }
        }
        s += __builtin_amdgcn_exp2f((lone - off) * c2);
        for (int c = NV * NT + tid; c < chunks; c += NT) {
            i32x4 r = *reinterpret_cast<const i32x4*>(x + head + c * N);
            if (REST) {
                const unsigned marked = marks(c);
                if (marked) strike<T>(r, marked);
            }
            float v[N], mc = -INFINITY, sc = 0.f;
            unpack(r, v, T());
#pragma unroll
            for (int j = 0; j < N; ++j) mc = fmaxf(mc, v[j]);
#pragma unroll
            for (int j = 0; j < N; ++j) sc += power(v[j], mc, c2);
            join_stats(m, s, mc, sc, c2);
        }
    }
    {
        const float mw = wave_all_max(m);
        s = wave_all_sum(s * power(m, mw, c2));
        m = mw;
        if (lane == 0) {
            red[2 * (tid >> 6)] = m;
            red[2 * (tid >> 6) + 1] = s;
        }
        __syncthreads();
        const float mi = lane < NT / 64 ? red[2 * (lane & (NT / 64 - 1))] : -INFINITY;
        const float si = lane < NT / 64 ? red[2 * (lane & (NT / 64 - 1)) + 1] : 0.f;
        m = wave_all_max(mi);
        s = wave_all_sum(si * power(mi, m, c2));
    }
    float mall = m, sall = s;
    if (REST) join_stats(mall, sall, told[3], told[4], c2);
    const float log_sall = logf(sall);
    // (classes outside the list, if any has mass: m is their maximum)
    const float rest = told[2];
    const bool there = REST && rest > 0.f && m > -INFINITY;
    const float P = told[1] + (there ? rest : 0.f);
    const float gs = total != 0.f ? p.grad_scale * (w / total) : 0.f;
    if (p.grad) {
        // e^((x - m) / tau) times one factor for every class that is not listed
        const float f = gs * (REST ? P * power(m, mall, c2) / sall - (there ? rest / s : 0.f) : P / s);
        const float off = m == -INFINITY ? 0.f : m;
        const float f_own = f * power(own, m, c2);      // (of a kept power, which goes by the thread's own maximum)
        auto gradient = [&](int chunk, const i32x4& r) {
            float v[N];
            unpack(r, v, T());
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = __builtin_amdgcn_exp2f((v[j] - off) * c2) * f;
            store(chunk, v);
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * NT + wave0 >= chunks) continue;
            asm volatile("" : "+v"(raw[i]));
            const int chunk = i * NT + tid;
            if (chunk >= chunks) continue;
            if constexpr (kKeep) {
                float v[N];
                unpack(raw[i], v, T());
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] *= f_own;
                store(chunk, v);
            } else {
                gradient(chunk, raw[i]);
            }
        }
        for (int c = NV * NT + tid; c < chunks; c += NT) gradient(c, *reinterpret_cast<const i32x4*>(x + head + c * N));
        if (loose >= 0) gr[loose] = (T)(__builtin_amdgcn_exp2f((lone - off) * c2) * f);
        __syncthreads();        // (these stores come before those of the listed classes, which are written once more)
    }
    if (tid < 64) {
        const bool twice = told[5] != 0.f;
        float l = 0.f;
        for (int i = lane; i < p.top; i += 64) {
            const int id = l_id[i];
            if (id < 0) continue;
            if (l_p[i] > 0.f || l_p[i] != l_p[i]) l += l_p[i] * (l_lp[i] - ((l_z[i] - mall) * p.inv_tau - log_sall));
            if (!p.grad) continue;
            float pi = l_p[i];
            bool first = true;
            if (twice) {
                pi = 0.f;
                for (int j = 0; j < p.top; ++j)
                    if (l_id[j] == id) {
                        if (j < i) first = false;
                        pi += l_p[j];
                    }
            }
            if (first) gr[id] = (T)(gs * (P * power(l_z[i], mall, c2) / sall - pi));
        }
        l = wave_all_sum(l);
        if (there) l += rest * (logf(rest) - ((m - mall) * p.inv_tau + logf(s) - log_sall));
        if (lane == 0) p.row_loss[row] = w * l;
    }
}

// Sum of x: one workgroup, fixed order, eight loads of a thread in flight.
__device__ float sum_by_block(const float* __restrict__ x, long n, float* red) {
    float s = 0.f;
    for (long i = threadIdx.x; i < n; i += 8 * 1024) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i + k * 1024 < n ? x[i + k * 1024] : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) s += v[k];
    }
    return block_sum<1024>(s, red);
}
__global__ __launch_bounds__(1024) void distill_weights_kernel(const float* __restrict__ weight, long rows, float* out) {
    __shared__ float red[16];
    const float s = sum_by_block(weight, rows, red);
    if (threadIdx.x == 0) out[0] = s;
}
__global__ __launch_bounds__(1024) void distill_mean_kernel(const float* __restrict__ row_loss, const float* __restrict__ weight,
                                                            const float* __restrict__ weights, long rows, float scale,
                                                            int accumulate, float* __restrict__ out) {
    __shared__ float red[16];
    const float s = sum_by_block(row_loss, rows, red);
    const float total = weights ? weights[0] : weight ? sum_by_block(weight, rows, red) : (float)rows;
    if (threadIdx.x == 0) out[0] = (accumulate ? out[0] : 0.f) + (total != 0.f ? scale * (s / total) : 0.f);
}

constexpr int kMaxClasses = 1 << 20, kMaxTop = 1024;

template <typename T, int NT, int NV>
static int launch_distill(const Distill& p, hipStream_t st) {
    const size_t lds = ((size_t)p.classes + 8 + 127) / 128 * 16 + (size_t)p.top * 16;
    auto go = [&](auto kernel) {
        // the list's bits of the largest vocabulary and the longest list
        constexpr int most = kMaxClasses / 8 + 64 + kMaxTop * 16;
        static std::atomic<unsigned long> devices{0};
        const hipError_t set = lds > 65536 ? allow_lds(reinterpret_cast<const void*>(kernel), most, devices) : hipSuccess;
        if (set != hipSuccess) return fail("gan_distill_topk_mean: %zu bytes of LDS refused: %s", lds, hipGetErrorString(set));
        hipLaunchKernelGGL(kernel, dim3((unsigned)p.rows), dim3(NT), lds, st, p);
        return 0;
    };
    return p.lse ? go(distill_kernel<T, NT, NV, true>) : go(distill_kernel<T, NT, NV, false>);
}

}  // namespace gan

using namespace gan;

extern "C" {

size_t gan_distill_topk_workspace_bytes(long rows) { return rows > 0 ? ((size_t)rows + 4) * sizeof(float) : 0; }

int gan_distill_topk_mean(int dtype, long rows, int classes, const void* logits, long ld, int teacher_dtype, const void* teacher,
                          const void* index, int index_bytes, int top, const float* teacher_lse, const float* row_weight,
                          float temperature, float weight, int accumulate, float* loss_out, void* dlogits, void* ws,
                          size_t ws_bytes, gan_stream_t stream) {
    GAN_CHECK_ARG(dtype_ok(dtype) && dtype_ok(teacher_dtype), "gan_distill_topk_mean: unknown element type %d or %d", dtype, teacher_dtype);
    GAN_CHECK_ARG(rows >= 1 && rows <= GAN_MX_MAX_ROWS, "gan_distill_topk_mean: %ld rows (1..%d are served)", rows, GAN_MX_MAX_ROWS);
    GAN_CHECK_ARG(classes >= 1 && classes <= kMaxClasses, "gan_distill_topk_mean: %d classes (1..%d are served)", classes, kMaxClasses);
    GAN_CHECK_ARG(top >= 1 && top <= kMaxTop, "gan_distill_topk_mean: lists of %d (1..%d are served)", top, kMaxTop);
    GAN_CHECK_ARG(index_bytes == 4 || index_bytes == 8, "gan_distill_topk_mean: indices of %d bytes", index_bytes);
    GAN_CHECK_ARG(temperature >= 0x1p-40f && temperature <= 0x1p40f, "gan_distill_topk_mean: temperature %g (2^-40..2^40 are served)",
                  (double)temperature);
    GAN_CHECK_ARG(logits && teacher && index && loss_out, "gan_distill_topk_mean: null pointer");
    GAN_CHECK_ARG(ld >= classes, "gan_distill_topk_mean: row stride %ld smaller than the row", ld);
    GAN_CHECK_ARG(ws && ws_bytes >= gan_distill_topk_workspace_bytes(rows), "gan_distill_topk_mean: workspace of %zu bytes needed, %zu given",
                  gan_distill_topk_workspace_bytes(rows), ws_bytes);
    const hipStream_t st = as_stream(stream);
    float* row_loss = static_cast<float*>(ws);
    float* total = nullptr;
    if (row_weight && rows > 4096) {    // (up to there every workgroup adds the weights up itself: 16 KB from the L2)
        total = row_loss + rows;
        hipLaunchKernelGGL(distill_weights_kernel, dim3(1), dim3(1024), 0, st, row_weight, rows, total);
    }
    const Distill p{logits, dlogits, teacher, index, teacher_lse, row_weight, total, row_loss, ld, rows, classes, top,
                    teacher_dtype, index_bytes == 8, 1.f / temperature, weight * temperature};
    const int rc = with_dtype(dtype, [&](auto* tag) {
        typedef typename std::remove_pointer<decltype(tag)>::type T;
        const int chunks = classes / Chunk<T>::n;
        // What is in flight on a CU counts, not only that nothing is read twice: of 131072 bf16 classes (16384 chunks) 2048 rows
        // take 249 us with half of a row in registers and 262 with all of it, of 32000 (4000 chunks) 4096 rows 124 us with 512
        // threads, 143 with 1024, 134 with 256 x 16 chunks.  Few rows want every thread: 256 rows of 131072 41 us against 46.
        // Many short rows go to a wave each: 65536 x 100 fp32 227 us with 256 threads, 110 so, 16384 x 1000 60 against 42, 8192 x 4000
        // bf16 61 against 50 (of 8000 77 against 95); 64 rows of 100 10.0 against 11.4 us.
        if (rows >= 2048 && chunks <= 512) {
            if (chunks <= 64) return launch_distill<T, 64, 1>(p, st);
            return chunks <= 256 ? launch_distill<T, 64, 4>(p, st) : launch_distill<T, 64, 8>(p, st);
        }
        if (chunks <= 256) return launch_distill<T, 256, 1>(p, st);
        if (chunks <= 512) return launch_distill<T, 256, 2>(p, st);
        if (chunks <= 1024) return launch_distill<T, 256, 4>(p, st);
        if (chunks <= 2048) return launch_distill<T, 256, 8>(p, st);
        if (chunks <= 4096) return launch_distill<T, 512, 8>(p, st);
        if (chunks <= 8192 || (chunks <= 16384 && rows > 512)) return launch_distill<T, 1024, 8>(p, st);
        return launch_distill<T, 1024, 16>(p, st);
    });
    if (rc) return rc;
    hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(1024), 0, st, row_loss, row_weight, total, rows, weight * temperature * temperature,
                       accumulate, loss_out);
    return check_launch("gan_distill_topk_mean");
}

}  // extern "C"
