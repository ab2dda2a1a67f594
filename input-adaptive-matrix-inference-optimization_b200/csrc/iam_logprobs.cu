// iam_logprobs.cu -- log probabilities of given tokens, their rank, the entropy and the best alternatives
// of rows of logits (the reference ends its step in an argmax, test_generation.cpp:276).
//
// With m = max x, L = sum exp(x - m):  logprob = x_t - m - ln L,  entropy = ln L - sum (x - m) exp(x - m) / L.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "iam_types.cuh"

namespace iam {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = kThreads / 2;  // maxima that bound the k-th largest value from below
constexpr int kMaxTop = 64;
constexpr int kCand = kThreads;        // candidates ranked directly
constexpr int kMaxCluster = 16;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LogprobParams {
    const void* logits;
    long long stride;
    int vocab, top_k;
    const int32_t* targets;
    float *logprob, *lse, *entropy;
    int32_t* rank;
    float* top_logprob;
    int32_t* top_index;
};

// Orderable key of (value, index): the larger value wins, then the smaller index; NaN above all.
IAM_DEV unsigned long long order_key(float v, int index) {
    const unsigned u = __float_as_uint(v + 0.0f);  // -0 as 0
    const unsigned ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((unsigned long long)ord << 32) | (unsigned long long)(0xffffffffu - (unsigned)index);
}
IAM_DEV float key_value(unsigned long long k) {
    const unsigned ord = (unsigned)(k >> 32);
    return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7fffffffu) : ~ord);
}
IAM_DEV int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }

IAM_DEV float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Makes the compiler widen the 16-bit values anew in each pass over them: kept as fp32 they spill.
template <class T, int VEC, int NV>
IAM_DEV void keep_packed(Vec<T, VEC> (&raw)[NV]) {
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            uint4& w = *reinterpret_cast<uint4*>(&raw[k]);
            asm volatile("" : "+r"(w.x), "+r"(w.y), "+r"(w.z), "+r"(w.w));
        }
}

// What one CTA knows of its part of the row.
struct Part {
    float m, l, s;  // maximum, sum of exp2(y), sum of y exp2(y), y = (x - m) log2(e)
    int ahead;      // tokens ahead of the target
    int n_top;
    unsigned long long top[kMaxTop];  // largest keys first
};

// One cluster per row, its CTAs side by side in the row.  A CTA reads its part once, NV 16-byte accesses a
// thread, all issued before the first is used, and keeps it in registers: the maximum, the sums and the
// search for the alternatives then cost no further traffic.  Bound by the bytes of the logits.
// The alternatives: of the maxima of 128 pairs of threads the k-th largest is a lower bound of the k-th
// largest value, and hardly more than k values reach it; these are collected and ranked.
template <class T, int NV>
__global__ void __launch_bounds__(kThreads, 2) logprobs_kernel(LogprobParams p) {
    constexpr int VEC = 16 / (int)sizeof(T);
    using V = Vec<T, VEC>;
    __shared__ Part part;
    __shared__ float s_m[kWarps], s_l[kWarps], s_s[kWarps];
    __shared__ int s_ahead[kWarps];
    __shared__ __align__(16) float s_group[kGroups];
    __shared__ float s_floor;
    __shared__ int s_count;
    __shared__ unsigned long long s_cand[kCand];
    __shared__ unsigned long long s_best[kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / C;
    const T* x = static_cast<const T*>(p.logits) + row * p.stride;
    // aligned accesses: the row begins `lead` elements into the first one
    const int lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    const T* x0 = x - lead;
    const int all = (p.vocab + lead + VEC - 1) / VEC, per = (all + C - 1) / C;
    const int v0 = rank * per, v1 = min(all, v0 + per);
    V raw[NV];
    auto at = [&](int k) { return v0 + tid + k * kThreads; };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int v = at(k), first = v * VEC - lead;
        if (v < v1 && first >= 0 && first + VEC <= p.vocab) {
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(x0 + (size_t)v * VEC));
            raw[k] = *reinterpret_cast<const V*>(&w);
        } else {  // the row's ends, element by element, and nothing behind them
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                raw[k].v[e] = v < v1 && first + e >= 0 && first + e < p.vocab ? x[first + e] : from_f32<T>(-INFINITY);
        }
    }
    const int target = p.targets ? p.targets[row] : -1;
    const bool named = target >= 0 && target < p.vocab;
    const float xt = named ? to_f32(x[target]) : INFINITY;

    float m = -INFINITY;
    int ahead = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float top = to_f32(raw[k].v[0]);
#pragma unroll
        for (int e = 1; e < VEC; ++e) top = fmaxf(top, to_f32(raw[k].v[e]));
        m = fmaxf(m, top);
        if (top >= xt) {
            const int first = at(k) * VEC - lead;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float f = to_f32(raw[k].v[e]);
                ahead += f > xt || (f == xt && (unsigned)(first + e) < (unsigned)target);
            }
        }
    }
    keep_packed(raw);
    // (the difference is taken first: one rounding relative to it, however far the logits are from 0, and no
    // overflow at the type's lowest value)
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, s = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float y = (to_f32(raw[k].v[e]) - ref) * kLog2e;
            const float t = exp2_fast(y);
            l += t;
            s = fmaf(fmaxf(y, -200.0f), t, s);  // (the term of -inf is 0, not -inf times 0)
        }
    // ---- the CTA's sums, in warp order
    {
        float wm = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
        const float d = m == -INFINITY ? 0.0f : (m - wm) * kLog2e;
        const float f = exp2_fast(d);
        // terms y exp2(y) at another maximum: (y + d) exp2(y + d)
        s = (s + fmaxf(d, -200.0f) * l) * f;
        l *= f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
            s += __shfl_xor_sync(0xffffffffu, s, o);
            ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
        }
        if (lane == 0) {
            s_m[warp] = wm;
            s_l[warp] = l;
            s_s[warp] = s;
            s_ahead[warp] = ahead;
        }
        const float pair = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
        if (!(tid & 1)) s_group[tid >> 1] = pair;
        if (tid == 0) s_count = 0;
    }
    __syncthreads();
    if (tid == 0) {
        float M = s_m[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) M = fmaxf(M, s_m[w]);
        float L = 0.0f, S = 0.0f;
        int A = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float d = s_m[w] == -INFINITY ? 0.0f : (s_m[w] - M) * kLog2e;
            const float f = exp2_fast(d);
            S += (s_s[w] + fmaxf(d, -200.0f) * s_l[w]) * f;
            L = fmaf(s_l[w], f, L);
            A += s_ahead[w];
        }
        part.m = M;
        part.l = L;
        part.s = S;
        part.ahead = A;
    }
    if (p.top_k > 0) {
        const int here = max(0, min(p.vocab, v1 * VEC - lead) - max(0, v0 * VEC - lead));
        const int want = min(p.top_k, here);
        if (want > 0) {
            if (tid < kGroups) {
                const float mine = s_group[tid];
                int above = 0;
#pragma unroll 8
                for (int j = 0; j < kGroups; j += 4) {
                    const float4 o = *reinterpret_cast<const float4*>(s_group + j);
                    above += (o.x > mine || (o.x == mine && j < tid)) + (o.y > mine || (o.y == mine && j + 1 < tid)) +
                             (o.z > mine || (o.z == mine && j + 2 < tid)) + (o.w > mine || (o.w == mine && j + 3 < tid));
                }
                if (above == want - 1) s_floor = mine;
            }
            __syncthreads();
            const float bound = s_floor;
            keep_packed(raw);
            if (m >= bound) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int first = at(k) * VEC - lead;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float f = to_f32(raw[k].v[e]);
                        if (f >= bound && at(k) < v1 && (unsigned)(first + e) < (unsigned)p.vocab) {
                            const int c = atomicAdd(&s_count, 1);
                            if (c < kCand) s_cand[c] = order_key(f, first + e);
                        }
                    }
                }
            }
            __syncthreads();
            const int n = s_count;
            if (n >= want && n <= kCand) {
                if (tid < n) {
                    const unsigned long long mine = s_cand[tid];
                    int above = 0;
                    for (int j = 0; j < n; ++j) above += s_cand[j] > mine;
                    if (above < want) part.top[above] = mine;
                }
            } else {  // many equal values (or NaN): one pass over the registers for each alternative
                unsigned long long last = ~0ull;
                for (int j = 0; j < want; ++j) {
                    keep_packed(raw);
                    unsigned long long best = 0ull;
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const int first = at(k) * VEC - lead;
#pragma unroll
                        for (int e = 0; e < VEC; ++e)
                            if (at(k) < v1 && (unsigned)(first + e) < (unsigned)p.vocab) {
                                const unsigned long long key = order_key(to_f32(raw[k].v[e]), first + e);
                                if (key < last && key > best) best = key;
                            }
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) {
                        const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
                        best = other > best ? other : best;
                    }
                    if (lane == 0) s_best[warp] = best;
                    __syncthreads();
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) best = s_best[w] > best ? s_best[w] : best;
                    if (tid == 0) part.top[j] = best;
                    last = best;
                    __syncthreads();
                }
            }
        }
        if (tid == 0) part.n_top = want;
    }
    // ---- the row's result from the cluster's parts, in order
    if (C > 1) cluster.sync();
    else __syncthreads();
    if (rank == 0) {
        float M = -INFINITY;
        for (int c = 0; c < C; ++c) M = fmaxf(M, cluster.map_shared_rank(&part, c)->m);
        float L = 0.0f, S = 0.0f;
        int A = 0;
        for (int c = 0; c < C; ++c) {
            const Part* o = cluster.map_shared_rank(&part, c);
            const float d = o->m == -INFINITY ? 0.0f : (o->m - M) * kLog2e;
            const float f = exp2_fast(d);
            S += (o->s + fmaxf(d, -200.0f) * o->l) * f;
            L = fmaf(o->l, f, L);
            A += o->ahead;
        }
        const bool any = M != -INFINITY || L != L;  // some token has a probability (or is NaN)
        const float log_l = any ? logf(L) : NAN;
        if (tid == 0) {
            if (p.logprob) p.logprob[row] = target < 0 ? 0.0f : named ? (xt - M) - log_l : NAN;
            if (p.lse) p.lse[row] = any ? M + log_l : -INFINITY;
            if (p.entropy) p.entropy[row] = any ? log_l - S / L * kLn2 : NAN;
            if (p.rank) p.rank[row] = named ? A : -1;
        }
        if (p.top_k > 0) {
            float* tl = p.top_logprob + row * p.top_k;
            int32_t* ti = p.top_index + row * p.top_k;
            for (int i = tid; i < C * p.top_k; i += kThreads) {
                const int c = i / p.top_k, j = i - c * p.top_k;
                const Part* o = cluster.map_shared_rank(&part, c);
                if (j >= o->n_top) continue;
                const unsigned long long mine = o->top[j];
                int above = j;  // its own part is in order
                for (int b = 0; b < C && above < p.top_k; ++b) {
                    if (b == c) continue;
                    const Part* q = cluster.map_shared_rank(&part, b);
                    for (int k = 0; k < q->n_top && q->top[k] > mine; ++k) ++above;
                }
                if (above < p.top_k) {
                    tl[above] = (key_value(mine) - M) - log_l;
                    ti[above] = key_index(mine);
                }
            }
        }
    }
    if (C > 1) cluster.sync();  // no CTA leaves while its part is read
}

template <class T, int NV>
int launch(const LogprobParams& p, int n_rows, int cluster, cudaStream_t s) {
    auto kern = logprobs_kernel<T, NV>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); }));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_rows * cluster);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    IAM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p));
    return IAM_OK;
}

}  // namespace
}  // namespace iam

using namespace iam;

extern "C" int iam_logprobs(const void* logits_dev, int dtype, int n_rows, int vocab, long long row_stride, const int32_t* targets_dev,
                            float* logprob_dev, float* lse_dev, float* entropy_dev, int32_t* rank_dev, int top_k, float* top_logprob_dev,
                            int32_t* top_index_dev, void* stream) {
    if (!dtype_ok(dtype)) return fail(IAM_ERR_ARG, "logprobs: dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    if (n_rows < 0 || vocab <= 0) return fail(IAM_ERR_ARG, "logprobs: bad sizes");
    if (n_rows > 1 && row_stride < vocab) return fail(IAM_ERR_ARG, "logprobs: rows overlap");
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab) return fail(IAM_ERR_ARG, "logprobs: top_k must be in [0, min(64, vocab)]");
    if (top_k > 0 && n_rows > 0 && (!top_logprob_dev || !top_index_dev)) return fail(IAM_ERR_ARG, "logprobs: null top outputs");
    if (n_rows == 0) return IAM_OK;
    const size_t elem = dtype_size(dtype);
    if (!logits_dev || reinterpret_cast<uintptr_t>(logits_dev) % elem) return fail(IAM_ERR_ARG, "logprobs: null or misaligned logits");
    if (!targets_dev && (logprob_dev || rank_dev)) return fail(IAM_ERR_ARG, "logprobs: logprob and rank need targets");
    const long long vecs = ((long long)vocab * (long long)elem + 15) / 16 + 1;  // accesses of a row, at any alignment
    if (vecs > 16LL * kThreads * kMaxCluster) return fail(IAM_ERR_UNSUPPORTED, "logprobs: a row must be below 1 MiB");
    int dev = 0;
    static std::atomic<int> sm_count{0};
    int sms = sm_count.load(std::memory_order_relaxed);
    if (!sms) {
        IAM_CUDA_TRY(cudaGetDevice(&dev));
        IAM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        sm_count.store(sms, std::memory_order_relaxed);
    }
    // as few CTAs as hold the row in registers; for few rows up to 8 each, while that fills idle SMs and
    // leaves every thread an access
    int c = 1;
    while ((vecs + c - 1) / c > 16 * kThreads) c *= 2;
    while (c < 8 && (long long)n_rows * c * 2 <= 2 * sms && vecs / (2 * c) >= kThreads) c *= 2;
    if ((long long)n_rows * c > INT32_MAX) return fail(IAM_ERR_ARG, "logprobs: too many rows");
    const long long per = (vecs + c - 1) / c;
    LogprobParams p{logits_dev, row_stride, vocab, top_k, targets_dev, logprob_dev, lse_dev, entropy_dev, rank_dev, top_logprob_dev, top_index_dev};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        if (per <= 4 * kThreads) return launch<T, 4>(p, n_rows, c, s);
        if (per <= 8 * kThreads) return launch<T, 8>(p, n_rows, c, s);
        return launch<T, 16>(p, n_rows, c, s);
    });
}
