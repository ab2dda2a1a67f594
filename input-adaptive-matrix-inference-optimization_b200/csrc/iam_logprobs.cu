// iam_logprobs.cu -- log probabilities of given tokens, their rank, the entropy and the best alternatives
// of rows of logits (the reference ends its step in an argmax, test_generation.cpp:276).
//
// With m = max x, L = sum exp(x - m):  logprob = x_t - m - ln L,  entropy = ln L - sum (x - m) exp(x - m) / L.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "iam_tc.cuh"
#include "iam_types.cuh"

namespace iam {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kPerSm = 2;       // CTAs an SM
constexpr int kSlots = 64;      // candidates of a row that a warp keeps at most; above half of it they are cut to the best
constexpr int kList = kWarps * kSlots;
constexpr int kMaxTop = 64;
constexpr int kMaxCluster = 8;
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

// What one CTA knows of its part of a row.
struct Part {
    float m, l, s;  // maximum, sum of exp2(y), sum of y exp2(y), y = (x - m) log2(e)
    int ahead;      // tokens ahead of the target
    int n_top;
    unsigned long long top[kMaxTop];  // largest keys first
};

// (m, l, s) of two disjoint sets of values, as one: terms y exp2(y) at another maximum are (y + d) exp2(y + d).
IAM_DEV void join(float& m, float& l, float& s, float m2, float l2, float s2) {
    const float M = fmaxf(m, m2);
    const float d1 = m == -INFINITY ? 0.0f : (m - M) * kLog2e, d2 = m2 == -INFINITY ? 0.0f : (m2 - M) * kLog2e;
    const float f1 = exp2_fast(d1), f2 = exp2_fast(d2);
    s = (s + fmaxf(d1, -200.0f) * l) * f1 + (s2 + fmaxf(d2, -200.0f) * l2) * f2;
    l = l * f1 + l2 * f2;
    m = M;
}

// The value before x in its type's order, as fp32: f >= x is f > before(x).
IAM_DEV float before(float x) {
    const int b = __float_as_int(x);
    return __int_as_float(x > 0.0f ? b - 1 : x < 0.0f ? b + 1 : (int)0x80000001);
}

// A cluster takes rows in turn, its CTAs side by side in each row, and a CTA its part in chunks of NV 16-byte
// accesses a thread.  A chunk comes into shared memory by one bulk copy, from there into registers, and the next
// chunk (of this row or the next) is on its way while this one is worked on, so the copies hardly pause: the
// kernel is bound by the bytes of the logits.  (Copies by the threads themselves do pause: an SM accepts about
// 64 KB of outstanding loads, and the warps that issue more wait.)  Large chunks, because each costs a chain of
// short steps with a barrier apiece: 16 KB ones in four CTAs an SM took twice as long.
// The alternatives: of the maxima of 64 groups of threads (128 when more than 32 are wanted) the k-th largest is a
// lower bound of the chunk's, and so of the row's, k-th largest value, and hardly more than k values reach it; these
// are collected and ranked.
// 2048 rows of 32000 (262 MB in fp32): 50 us without alternatives (5.2 TB/s; bf16 48), 95 with 20 (127): the threads'
// comparisons among groups, the collection and the ranking are a chain of barriers that two CTAs an SM hide only in part.  With
// -inf in a tenth of every third row's tokens 79 and 117 (55 and 133): a target among them is counted element by element, and its
// row holds up its CTA.  One row: 7.7 us.
template <class T, int NV>
__global__ void __launch_bounds__(kThreads, kPerSm) logprobs_kernel(LogprobParams p, int n_rows) {
    constexpr int VEC = 16 / (int)sizeof(T), CHUNK = NV * kThreads;
    using V = Vec<T, VEC>;
    extern __shared__ __align__(16) char s_chunk[];  // [CHUNK] accesses
    __shared__ Part s_part[2][kMaxCluster];          // the cluster's first CTA holds every CTA's part, rows in turn
    __shared__ __align__(8) uint64_t s_full;
    __shared__ unsigned s_lost;  // 1: a wait gave up, and this row and all later ones are NaN
    __shared__ float s_m[kWarps], s_l[kWarps], s_s[kWarps];
    __shared__ int s_ahead[kWarps];
    __shared__ __align__(16) float s_group[kThreads / 2];
    __shared__ float s_floor;
    __shared__ __align__(16) int s_count[kWarps];
    __shared__ unsigned long long s_cand[kWarps][kSlots], s_list[kList];
    __shared__ unsigned long long s_best[kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = cluster.num_blocks(), rank = cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int step = gridDim.x / C;
    const bool wide = p.top_k > 32;

    // This CTA's part of a row, in aligned accesses: the row begins `lead` elements into its first one.
    struct Where {
        const T* x;
        int lead, v0, v1;  // accesses of this part
        int f0, f1;        // those wholly inside the row
    };
    auto where = [&](int row) {
        Where w;
        w.x = static_cast<const T*>(p.logits) + row * p.stride;
        w.lead = (int)((reinterpret_cast<uintptr_t>(w.x) & 15) / sizeof(T));
        const int all = (p.vocab + w.lead + VEC - 1) / VEC, per = C == 1 ? all : (all + C - 1) / C;
        w.v0 = min(all, rank * per);
        w.v1 = min(all, w.v0 + per);
        w.f0 = max(w.v0, w.lead ? 1 : 0);
        w.f1 = min(w.v1, (p.vocab + w.lead) / VEC);
        return w;
    };
    auto fetch = [&](const Where& w, int c0) {  // one thread: the whole accesses among c0 .. c0 + CHUNK
        const int a = max(w.f0, c0), b = min(w.f1, c0 + CHUNK);
        const uint32_t bytes = b > a ? (uint32_t)(b - a) * 16u : 0u;
        mbar_expect_tx(&s_full, bytes);
        if (bytes) bulk_load(s_chunk + (size_t)(a - c0) * 16, w.x - w.lead + (size_t)a * VEC, bytes, &s_full);
    };
    if (C > 1) cluster.barrier_arrive();
    if (tid == 0) {
        s_lost = 0u;
        mbar_init(&s_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    int row = blockIdx.x / C;
    if (tid == 0 && row < n_rows) fetch(where(row), where(row).v0);
    // The first CTA's shared memory takes the others' parts only once that CTA runs; the first chunk is on its way meanwhile.
    if (C > 1) {
        __syncwarp();
        cluster.barrier_wait();
    }
    uint32_t phase = 0;
    for (int turn = 0; row < n_rows; row += step, turn ^= 1) {  // (every CTA of a cluster makes the same turns)
        const Where w = where(row);
        const int target = p.targets ? p.targets[row] : -1;
        const bool named = target >= 0 && target < p.vocab;
        const float xt = named ? to_f32(w.x[target]) : INFINITY, xt_or_more = before(xt);
        Part* home = C > 1 ? cluster.map_shared_rank(&s_part[turn][rank], 0) : &s_part[turn][0];
        float m = -INFINITY, l = 0.0f, s = 0.0f;
        float bound = -INFINITY;  // a lower bound of the k-th largest value of the chunks so far
        int ahead = 0, n_mine = 0;  // (n_mine: candidates of this warp)
        if (named && warp == 0) {  // of the target's own access: the tokens before it that equal it
            const int v = (target + w.lead) / VEC, i = target - 1 - lane;
            if (v >= w.v0 && v < w.v1 && i >= 0 && i >= v * VEC - w.lead) ahead += to_f32(w.x[i]) == xt;
        }
        for (int c0 = w.v0;; c0 += CHUNK) {
            V raw[NV];
            mbar_wait_unless(&s_full, phase, &s_lost, 1u);
            phase ^= 1u;
            const V* got = reinterpret_cast<const V*>(s_chunk) + tid;
            if (c0 >= w.f0 && c0 + CHUNK <= w.f1) {
#pragma unroll
                for (int k = 0; k < NV; ++k) raw[k] = got[k * kThreads];
            } else {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
#pragma unroll
                    for (int e = 0; e < VEC; ++e) raw[k].v[e] = from_f32<T>(-INFINITY);
                    const int v = c0 + tid + k * kThreads;
                    if (v >= w.f0 && v < w.f1) raw[k] = got[k * kThreads];
                }
                if (w.f0 > w.v0 || w.f1 < w.v1)  // the row's ends, element by element
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const int v = c0 + tid + k * kThreads;
                        if (v < w.v1 && (v < w.f0 || v >= w.f1)) {
                            const int first = v * VEC - w.lead;
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                if (first + e >= 0 && first + e < p.vocab) raw[k].v[e] = w.x[first + e];
                        }
                    }
            }
            __syncthreads();  // the chunk is in registers
            const bool more = c0 + CHUNK < w.v1;
            if (tid == 0) {
                if (more) fetch(w, c0 + CHUNK);
                else if (row + step < n_rows) fetch(where(row + step), where(row + step).v0);
            }
            auto first_of = [&](int k) { return (c0 + tid + k * kThreads) * VEC - w.lead; };
            auto inside = [&](int k, int i) { return c0 + tid + k * kThreads < w.v1 && (unsigned)i < (unsigned)p.vocab; };
            auto top_of = [&](int k) {
                float top = to_f32(raw[k].v[0]);
#pragma unroll
                for (int e = 1; e < VEC; ++e) top = fmaxf(top, to_f32(raw[k].v[e]));
                return top;
            };

            float cm = -INFINITY;
#pragma unroll
            for (int k = 0; k < NV; ++k) cm = fmaxf(cm, top_of(k));
            if (p.top_k > 0) {
                float gm = fmaxf(cm, __shfl_xor_sync(0xffffffffu, cm, 1));
                if (!wide) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, 2));
                if (wide ? !(tid & 1) : !(tid & 3)) s_group[wide ? tid >> 1 : tid >> 2] = gm;
                __syncthreads();
                // two or four threads a group, each with its share of the comparisons
                const int lanes = wide ? 2 : 4, share = wide ? 64 : 16;
                const int j = tid / lanes, q = (tid & (lanes - 1)) * share;
                const float mine = s_group[j];
                int above = 0;
                for (int i0 = q; i0 < q + share; i0 += 16)
#pragma unroll
                    for (int i = i0; i < i0 + 16; i += 4) {
                        const float4 o = *reinterpret_cast<const float4*>(s_group + i);
                        above += (o.x > mine || (o.x == mine && i < j)) + (o.y > mine || (o.y == mine && i + 1 < j)) +
                                 (o.z > mine || (o.z == mine && i + 2 < j)) + (o.w > mine || (o.w == mine && i + 3 < j));
                    }
                above += __shfl_xor_sync(0xffffffffu, above, 1);
                if (!wide) above += __shfl_xor_sync(0xffffffffu, above, 2);
                if (above == p.top_k - 1 && (tid & (lanes - 1)) == 0) s_floor = mine;  // (read behind the sums' barrier)
            }
            if (named) {
                // tokens ahead of the target: from its own logit on in the accesses before its own, above it in
                // the others
                const int before_k = (target + w.lead) / VEC - c0 - tid;  // access k lies before it: k * kThreads < before_k
                if (xt > -INFINITY) {
#pragma unroll
                    for (int k = 0; k < NV; ++k) {
                        const float limit = k * kThreads < before_k ? xt_or_more : xt;
#pragma unroll
                        for (int e = 0; e < VEC; ++e) ahead += to_f32(raw[k].v[e]) > limit;
                    }
                } else {
#pragma unroll 1
                    for (int k = 0; k < NV; ++k)
                        for (int e = 0; e < VEC; ++e) {
                            const int v = c0 + tid + k * kThreads, i = v * VEC - w.lead + e;
                            if (v >= w.v1 || (unsigned)i >= (unsigned)p.vocab) continue;
                            const float f = to_f32(w.x[i]);
                            ahead += f > xt || (f == xt && k * kThreads < before_k);
                        }
                }
            }
            keep_packed(raw);
            {   // the sums at the thread's new maximum
                const float M = fmaxf(m, cm), d = m == -INFINITY ? 0.0f : (m - M) * kLog2e, f = exp2_fast(d);
                s = (s + fmaxf(d, -200.0f) * l) * f;
                l *= f;
                m = M;
            }
            // (the difference is taken first: one rounding relative to it, however far the logits are from 0, and no
            // overflow at the type's lowest value)
            const float ref = m == -INFINITY ? 0.0f : m;
            float l2 = 0.0f, s2 = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float y = (to_f32(raw[k].v[e]) - ref) * kLog2e;
                    const float t = exp2_fast(y);
                    float& la = e & 1 ? l2 : l;
                    float& sa = e & 1 ? s2 : s;
                    la += t;
                    sa = fmaf(fmaxf(y, -200.0f), t, sa);  // (the term of -inf is 0, not -inf times 0)
                }
            l += l2;
            s += s2;
            if (p.top_k > 0) {
                __syncthreads();
                bound = fmaxf(bound, s_floor);
                const int n_before = n_mine;
                if (bound > -INFINITY && __any_sync(0xffffffffu, cm >= bound)) {
                    keep_packed(raw);
                    unsigned which = 0;  // accesses with a value that reaches the bound: this lane's, then the warp's
#pragma unroll
                    for (int k = 0; k < NV; ++k) which |= top_of(k) >= bound ? 1u << k : 0u;
                    which = __reduce_or_sync(0xffffffffu, which);
#pragma unroll
                    for (int k = 0; k < NV; ++k)
                        if (which >> k & 1u) {
                            const int first = first_of(k);
                            unsigned hits[VEC];
#pragma unroll
                            for (int e = 0; e < VEC; ++e) hits[e] = __ballot_sync(0xffffffffu, to_f32(raw[k].v[e]) >= bound);
#pragma unroll
                            for (int e = 0; e < VEC; ++e) {
                                const int c = n_mine + __popc(hits[e] & ((1u << lane) - 1u));
                                if ((hits[e] >> lane & 1u) && c < kSlots) s_cand[warp][c] = order_key(to_f32(raw[k].v[e]), first + e);
                                n_mine += __popc(hits[e]);
                            }
                        }
                }
                if (lane == 0) s_count[warp] = n_mine;
                const int state = (__syncthreads_or(n_mine > kSlots) ? 1 : 0) | (bound == -INFINITY ? 1 : 0);
                if (state) {  // many equal values, or few tokens left: a pass over the registers for each of the chunk's best
                    const int here = max(0, min(p.vocab, min(w.v1, c0 + CHUNK) * VEC - w.lead) - max(0, c0 * VEC - w.lead));
                    const int want = min(p.top_k, here);
                    n_mine = n_before;
                    unsigned long long last = ~0ull;
                    for (int j = 0; j < want; ++j) {
                        keep_packed(raw);
                        unsigned long long best = 0ull;
#pragma unroll
                        for (int k = 0; k < NV; ++k) {
                            const int first = first_of(k);
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                if (inside(k, first + e)) {
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
                        for (int v = 0; v < kWarps; ++v) best = s_best[v] > best ? s_best[v] : best;
                        if ((j & (kWarps - 1)) == warp) {
                            if (lane == 0) s_cand[warp][n_mine] = best;
                            ++n_mine;
                        }
                        last = best;
                        __syncthreads();
                    }
                    if (lane == 0) s_count[warp] = n_mine;
                    __syncthreads();
                }
                int total = 0, mine0 = 0, most = 0;
#pragma unroll
                for (int v = 0; v < kWarps; ++v) {
                    const int c = s_count[v];
                    mine0 += v < warp ? c : 0;
                    total += c;
                    most = max(most, c);
                }
                if (!more || most > kSlots / 2) {  // the best of them: in order, into the part, or back among the candidates
                    for (int c = lane; c < n_mine; c += 32) s_list[mine0 + c] = s_cand[warp][c];
                    __syncthreads();
                    if (more) n_mine = (min(total, p.top_k) + kWarps - 1 - warp) / kWarps;
                    for (int c0 = 0; c0 < total; c0 += kThreads / 4) {  // four threads a candidate
                        const int c = c0 + (tid >> 2);
                        const unsigned long long mine = c < total ? s_list[c] : 0ull;
                        int above = 0;
#pragma unroll 4
                        for (int j = tid & 3; j < total; j += 4) above += s_list[j] > mine;
                        above += __shfl_xor_sync(0xffffffffu, above, 1);
                        above += __shfl_xor_sync(0xffffffffu, above, 2);
                        if (c < total && above < p.top_k && !(tid & 3)) {
                            if (more) s_cand[above & (kWarps - 1)][above / kWarps] = mine;
                            else home->top[above] = mine;
                        }
                    }
                }
                if (more) __syncthreads();  // what this chunk shares is read before the next one writes it
            }
            if (!more) break;
        }
        // ---- the CTA's sums: lanes at the warp's maximum, then the warps
        {
            float wm = m;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) wm = fmaxf(wm, __shfl_xor_sync(0xffffffffu, wm, o));
            const float d = m == -INFINITY ? 0.0f : (m - wm) * kLog2e;
            const float f = exp2_fast(d);
            s = (s + fmaxf(d, -200.0f) * l) * f;
            l *= f;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                l += __shfl_xor_sync(0xffffffffu, l, o);
                s += __shfl_xor_sync(0xffffffffu, s, o);
            }
            ahead = __reduce_add_sync(0xffffffffu, ahead);
            if (lane == 0) {
                s_m[warp] = wm;
                s_l[warp] = *(volatile unsigned*)&s_lost ? NAN : l;
                s_s[warp] = s;
                s_ahead[warp] = ahead;
            }
        }
        __syncthreads();
        float M = s_m[lane & (kWarps - 1)], L = s_l[lane & (kWarps - 1)], S = s_s[lane & (kWarps - 1)];
        int A = s_ahead[lane & (kWarps - 1)];
#pragma unroll
        for (int o = 1; o < kWarps; o <<= 1) {
            join(M, L, S, __shfl_xor_sync(0xffffffffu, M, o), __shfl_xor_sync(0xffffffffu, L, o), __shfl_xor_sync(0xffffffffu, S, o));
            A += __shfl_xor_sync(0xffffffffu, A, o);
        }
        const Part* parts = s_part[turn];
        if (C > 1) {
            if (tid == 0) {
                home->m = M;
                home->l = L;
                home->s = S;
                home->ahead = A;
                home->n_top = min(p.top_k, max(0, min(p.vocab, w.v1 * VEC - w.lead) - max(0, w.v0 * VEC - w.lead)));
            }
            // One barrier a row is enough: the parts of the row after next overwrite these, and the first CTA has
            // read them before it arrives at the next row's barrier.
            cluster.sync();
            if (rank != 0) continue;
            M = parts[0].m;
            L = parts[0].l;
            S = parts[0].s;
            A = parts[0].ahead;
            for (int c = 1; c < C; ++c) {
                join(M, L, S, parts[c].m, parts[c].l, parts[c].s);
                A += parts[c].ahead;
            }
        }
        const bool any = M != -INFINITY || L != L;  // some token has a probability (or is NaN)
        const float log_l = any ? logf(L) : NAN;
        if (tid == kThreads - 1) {
            if (p.logprob) p.logprob[row] = target < 0 ? 0.0f : named ? (xt - M) - log_l : NAN;
            if (p.lse) p.lse[row] = any ? M + log_l : -INFINITY;
            if (p.entropy) p.entropy[row] = any ? log_l - S / L * kLn2 : NAN;
            if (p.rank) p.rank[row] = named ? A : -1;
        }
        if (C == 1) {
            if (tid < p.top_k) {
                const unsigned long long key = parts[0].top[tid];
                p.top_logprob[(size_t)row * p.top_k + tid] = (key_value(key) - M) - log_l;
                p.top_index[(size_t)row * p.top_k + tid] = key_index(key);
            }
        } else {
            for (int i = tid; i < C * p.top_k; i += kThreads) {
                const int c = i / p.top_k, j = i - c * p.top_k;
                if (j >= parts[c].n_top) continue;
                const unsigned long long mine = parts[c].top[j];
                int above = j;  // its own part is in order
                for (int b = 0; b < C; ++b) {
                    const int n = b == c ? 0 : parts[b].n_top;
#pragma unroll 8
                    for (int k = 0; k < n; ++k) above += parts[b].top[k] > mine;
                }
                if (above < p.top_k) {
                    p.top_logprob[(size_t)row * p.top_k + above] = (key_value(mine) - M) - log_l;
                    p.top_index[(size_t)row * p.top_k + above] = key_index(mine);
                }
            }
        }
    }
}

template <class T, int NV>
int launch(const LogprobParams& p, int n_rows, int cluster, int sms, cudaStream_t s) {
    constexpr size_t smem = (size_t)NV * kThreads * 16;
    auto kern = logprobs_kernel<T, NV>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min(n_rows, std::max(1, kPerSm * sms / cluster)) * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    IAM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, p, n_rows));
    return IAM_OK;
}

}  // namespace
}  // namespace iam

using namespace iam;

extern "C" int iam_logprobs(const void* logits_dev, int dtype, int n_rows, int vocab, long long row_stride, const int32_t* targets_dev,
                            float* logprob_dev, float* lse_dev, float* entropy_dev, int32_t* rank_dev, int top_k, float* top_logprob_dev,
                            int32_t* top_index_dev, void* stream) {
    if (!dtype_ok(dtype)) return fail(IAM_ERR_ARG, "logprobs: dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    if (n_rows > 1 << 30) return fail(IAM_ERR_ARG, "logprobs: more than 2^30 rows");
    if (n_rows < 0 || vocab <= 0) return fail(IAM_ERR_ARG, "logprobs: bad sizes");
    if (n_rows > 1 && row_stride < vocab) return fail(IAM_ERR_ARG, "logprobs: rows overlap");
    if (top_k < 0 || top_k > kMaxTop || top_k > vocab) return fail(IAM_ERR_ARG, "logprobs: top_k must be in [0, min(64, vocab)]");
    if (top_k > 0 && n_rows > 0 && (!top_logprob_dev || !top_index_dev)) return fail(IAM_ERR_ARG, "logprobs: null top outputs");
    if (n_rows == 0) return IAM_OK;
    const size_t elem = dtype_size(dtype);
    if (!logits_dev || reinterpret_cast<uintptr_t>(logits_dev) % elem) return fail(IAM_ERR_ARG, "logprobs: null or misaligned logits");
    if (!targets_dev && (logprob_dev || rank_dev)) return fail(IAM_ERR_ARG, "logprobs: logprob and rank need targets");
    if ((long long)vocab * (long long)elem > INT32_MAX) return fail(IAM_ERR_UNSUPPORTED, "logprobs: a row must be below 2 GiB");
    const long long vecs = ((long long)vocab * (long long)elem + 15) / 16 + 1;  // accesses of a row, at any alignment
    int dev = 0;
    static std::atomic<int> sm_count{0};
    int sms = sm_count.load(std::memory_order_relaxed);
    if (!sms) {
        IAM_CUDA_TRY(cudaGetDevice(&dev));
        IAM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        sm_count.store(sms, std::memory_order_relaxed);
    }
    // one CTA a row; for few rows up to 8, while that fills idle SMs and leaves every thread an access
    int c = 1;
    while (c < kMaxCluster && (long long)n_rows * c * 2 <= 2 * sms && vecs / (2 * c) >= kThreads) c *= 2;
    const long long per = (vecs + c - 1) / c;
    LogprobParams p{logits_dev, row_stride, vocab, top_k, targets_dev, logprob_dev, lse_dev, entropy_dev, rank_dev, top_logprob_dev, top_index_dev};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // chunks of 64 KB (16-bit types: 32 KB, as many values; 64 KB of them do not fit the registers), or as
        // much as a shorter part of a row fills
        if (per <= 4 * kThreads) return launch<T, 4>(p, n_rows, c, sms, s);
        if (per <= 8 * kThreads || sizeof(T) == 2) return launch<T, 8>(p, n_rows, c, sms, s);
        return launch<T, sizeof(T) == 2 ? 8 : 16>(p, n_rows, c, sms, s);
    });
}
