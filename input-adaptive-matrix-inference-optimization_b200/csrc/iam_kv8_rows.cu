// iam_kv8_rows.cu -- attention of many query rows per sequence (prompts, drafted tokens) over the 8-bit
// paged cache.
#include <algorithm>
#include <atomic>

#include "iam_kv8_plan.cuh"

namespace iam {
namespace {

constexpr int kRows = 64;       // query rows of a tile: 16 for each warp
constexpr int kThreads = 128;
constexpr int kTile = 64;       // tokens of a work unit
constexpr int kPerSm = 3;       // CTAs per SM at most (scratch)
constexpr int kMinUnits = 8;    // units of a CTA at least, while there are enough: a context in few parts is joined faster
// Row tile (16 rows a warp) times tokens: scores with the queries as A and the tokens as B of m16n8k16, the
// probabilities (fp16, one or two terms) from the accumulators' own registers as A and the values as B.
// Codes arrive by cp.async one tile ahead and become fp16 in shared memory once per tile for all warps.  Bound by the
// MMAs' and the softmax's issue.  This kernel serves what the other two do not: 64 rows of one 8192-token
// sequence take it 76 us (the decode kernel 35), of 32 x 2000 tokens 172 (234); fp32 and head_dim 256 prompts always (2048 rows on
// 8192 earlier tokens: 32 heads of 128 over 8 in fp32 2716 us, 8 heads of 256 over 1 in bf16 1524, in fp32 1895).
template <class T, int FMT, int HD, int TERMS>
__global__ void __launch_bounds__(kThreads) kv8_rows_kernel(Kv8Attn p) {
    constexpr int KS = HD / 16, NT = kTile / 8, CB = HD / 16;  // CB: 16-byte pieces of a code row
    constexpr int PITCH = HD + 4;
    extern __shared__ __align__(16) char smem[];
    char* s_q = smem;                                    // [TERMS][kRows][HD] fp16
    char* s_k = s_q + TERMS * kRows * HD * 2;            // [kTile][HD] fp16
    char* s_v = s_k + kTile * HD * 2;                    // [kTile][HD] fp16
    char* s_raw = s_v + kTile * HD * 2;                  // [2 stages][K, V][kTile][HD] codes
    __shared__ float s_ks[2][4], s_vs[2][4];             // scales of the stage's groups
    __shared__ int s_ok[2][4];
    __shared__ float s_rf[kRows];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
    const int plog = 31 - __clz(p.c.page_size), kvh = p.c.n_kv_heads;
    const uint32_t q_s = (uint32_t)__cvta_generic_to_shared(s_q), k_s = (uint32_t)__cvta_generic_to_shared(s_k),
                   v_s = (uint32_t)__cvta_generic_to_shared(s_v);
    auto off = [](int row, int piece) { return row * (HD * 2) + ((piece ^ (row & 7)) << 4); };

    const Plan plan{p.s.plan};
    const int items = plan.items();
    const int per_head = plan.unit()[items];
    const long long total = (long long)per_head * kvh;
    if (total == 0) return;
    const int run = min(kMinUnits, per_head / max(1, items));  // (short contexts: a row tile a CTA)
    const long long ctas = min((long long)gridDim.x, (total + run - 1) / max(1, run));
    if (blockIdx.x >= ctas) return;
    const long long u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
    int item = find_item(plan, items, (int)(u0 % per_head));
    int head = (int)(u0 / per_head);

    long long u = u0;
    while (u < u1) {
        const long long item0 = (long long)head * per_head + plan.unit()[item], item1 = (long long)head * per_head + plan.unit()[item + 1];
        const int seq = plan.seq()[item], rtile = plan.rtile()[item];
        const SeqRows r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr);
        const RowItem it = item_of<kRows, kTile>(p, r, rtile);
        const int tile = (int)(u - item0);
        const long long seg_end = min(u1, item1);
        const int n_tiles = (int)(seg_end - u);
        const int t_first = it.lo + tile * kTile;
        const int32_t* table = p.c.block_table + (size_t)seq * p.c.max_pages;

        auto issue = [&](int i) {  // tile i of the segment into stage i & 1
            const int t0 = t_first + i * kTile, st = i & 1;
            char* rk = s_raw + (size_t)(2 * st) * kTile * HD;
            char* rv = rk + kTile * HD;
#pragma unroll
            for (int f0 = 0; f0 < kTile * CB; f0 += kThreads) {
                const int f = f0 + tid, row = f / CB, c = f - row * CB, t = t0 + row;
                int id = -1;
                if (t < r.cap && t >= (it.first & ~(kKv8Group - 1))) {
                    id = __ldg(table + (t >> plog));
                    if (id < 0 || id >= p.c.n_pages) {
                        atomicOr(p.s.err, kKv8ErrRange);
                        id = -1;
                    }
                }
                if (c == 0 && (row & (kKv8Group - 1)) == 0) {
                    s_ok[st][row / kKv8Group] = id >= 0;
                    s_ks[st][row / kKv8Group] = id >= 0 ? p.c.k_scale[(size_t)id * kvh + head] : 0.0f;
                    s_vs[st][row / kKv8Group] = id >= 0 ? p.c.v_scale[(size_t)id * kvh + head] : 0.0f;
                }
                char* dk = rk + row * HD + c * 16;
                char* dv = rv + row * HD + c * 16;
                if (id >= 0) {
                    const size_t at = ((((size_t)id * kvh + head) << plog) + (t & (p.c.page_size - 1))) * HD + c * 16;
                    cp_async16(dk, static_cast<const uint8_t*>(p.c.k) + at);
                    cp_async16(dv, static_cast<const uint8_t*>(p.c.v) + at);
                } else {  // behind the last token or before the window: nothing is read
                    *reinterpret_cast<uint4*>(dk) = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(dv) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        issue(0);

        // ---- queries, a row at a time, shifted into fp16's range and rounded (or split in two)
        for (int row = warp; row < kRows; row += kThreads / 32) {
            const int rr = rtile * kRows + row;
            const bool have = row < it.n_rows;
            const T* src = have ? static_cast<const T*>(p.q.data) + (size_t)(r.row0 + rr / p.gq) * p.q.token_stride +
                                      (head * p.gq + rr % p.gq) * p.q.head_stride
                                : nullptr;
            float f[HD / 32], amax = 0.0f;
#pragma unroll
            for (int e = 0; e < HD / 32; e += 2)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    f[e + k] = have ? to_f32(src[e * 32 + lane * 2 + k]) : 0.0f;
                    amax = fmaxf(amax, fabsf(f[e + k]));
                }
            const int sh = query_shift(warp_max(amax));
            const float up = pow2f(sh);
#pragma unroll
            for (int e = 0; e < HD / 32; e += 2) {
                const int d = e * 32 + lane * 2;
                char* to = s_q + off(row, d >> 3) + (d & 7) * 2;
                *reinterpret_cast<uint32_t*>(to) = pack_h2(f[e] * up, f[e + 1] * up);
                if (TERMS == 2)
                    *reinterpret_cast<uint32_t*>(to + kRows * HD * 2) = pack_h2(split_lo(f[e] * up), split_lo(f[e + 1] * up));
            }
            if (lane == 0) s_rf[row] = pow2f(-sh) * p.scale_log2;
        }
        __syncthreads();
        const int row_a = warp * 16 + g;
        float rf[2] = {s_rf[row_a], s_rf[row_a + 8]};
        int pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            pos[h] = row_a + 8 * h < it.n_rows ? r.start + (rtile * kRows + row_a + 8 * h) / p.gq : -1;

        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[HD / 8][4];
#pragma unroll
        for (int n = 0; n < HD / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

        for (int i = 0; i < n_tiles; ++i) {
            const int t0 = t_first + i * kTile, st = i & 1;
            cp_async_wait_all();
            __syncthreads();  // the stage has arrived; the fp16 tiles of the previous tile are consumed
            {
                const char* rk = s_raw + (size_t)(2 * st) * kTile * HD;
#pragma unroll
                for (int f0 = 0; f0 < kTile * CB; f0 += kThreads) {
                    const int f = f0 + tid, row = f / CB, c = f - row * CB;
                    const bool zero = t0 + row >= r.cap || t0 + row < it.first;
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        uint4 w = *reinterpret_cast<const uint4*>(rk + kv * kTile * HD + row * HD + c * 16);
                        if (zero) w = make_uint4(0u, 0u, 0u, 0u);
                        uint4 a, b;
                        codes_to_half<FMT>(w.x, a.x, a.y);
                        codes_to_half<FMT>(w.y, a.z, a.w);
                        codes_to_half<FMT>(w.z, b.x, b.y);
                        codes_to_half<FMT>(w.w, b.z, b.w);
                        char* to = kv ? s_v : s_k;
                        *reinterpret_cast<uint4*>(to + off(row, 2 * c)) = a;
                        *reinterpret_cast<uint4*>(to + off(row, 2 * c + 1)) = b;
                    }
                }
            }
            float ks4[4], vs4[4];
            bool ok4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                ks4[k] = s_ks[st][k];
                vs4[k] = s_vs[st][k];
                ok4[k] = s_ok[st][k];
            }
            __syncthreads();
            if (i + 1 < n_tiles) issue(i + 1);
            __syncwarp();  // (pages may part the warp, and the matrix instructions take it together)

            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint32_t a[TERMS][4];
#pragma unroll
                for (int x = 0; x < TERMS; ++x)
                    ldsm_x4(a[x], q_s + x * kRows * HD * 2 + off(warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * ks + (lane >> 4)));
#pragma unroll
                for (int n2 = 0; n2 < NT / 2; ++n2) {
                    uint32_t b[4];
                    ldsm_x4(b, k_s + off(n2 * 16 + (lane & 7) + (lane >> 4) * 8, 2 * ks + ((lane >> 3) & 1)));
#pragma unroll
                    for (int x = 0; x < TERMS; ++x) {
                        mma_16816(sc[2 * n2], a[x], b[0], b[1]);
                        mma_16816(sc[2 * n2 + 1], a[x], b[2], b[3]);
                    }
                }
            }
            const bool all_ok = ok4[0] && ok4[1] && ok4[2] && ok4[3];
            const bool whole = all_ok && t0 + kTile - 1 <= it.pos_lo && t0 + kTile <= r.cap && (p.window == 0 || t0 > it.pos_hi - p.window);
            float rescale[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = m[h];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float f = fminf(ks4[n >> 1] * rf[h], 3.402823466e38f);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = sc[n][2 * h + e] * f;
                        const int t = t0 + n * 8 + 2 * tig + e;
                        if (!whole && (!ok4[n >> 1] || t > pos[h] || t >= r.cap || (p.window > 0 && t <= pos[h] - p.window))) v = -INFINITY;
                        sc[n][2 * h + e] = v;
                        mx = fmaxf(mx, v);
                    }
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float ref = mx == -INFINITY ? 0.0f : mx;
                rescale[h] = ex2(m[h] - ref);
                m[h] = mx;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = ex2(sc[n][2 * h + e] - ref);
                        sc[n][2 * h + e] = v;
                        sum += v;
                    }
                l[h] = fmaf(l[h], rescale[h], sum);  // this lane's tokens only
            }
            // The groups' value scales: the largest goes on the products in fp32, the ratios to it (powers of
            // two, at most 1) on the probabilities, which are lifted by 2^12 so that a ratio of 2^-12 costs
            // none of fp16's 11 bits.
            const float vmax = fmaxf(fmaxf(vs4[0], vs4[1]), fmaxf(vs4[2], vs4[3]));
            uint32_t pa[TERMS][4][4];
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) {
                const float lift = vmax > 0.0f ? __fdividef(vs4[kt], vmax) * 4096.0f : 0.0f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float x = sc[2 * kt + (q >> 1)][(q & 1) * 2] * lift, y = sc[2 * kt + (q >> 1)][(q & 1) * 2 + 1] * lift;
                    pa[0][kt][q] = pack_h2(x, y);
                    if (TERMS == 2) pa[TERMS - 1][kt][q] = pack_h2(split_lo(x), split_lo(y));
                }
            }
            const float vf = vmax * (1.0f / 4096.0f);
            __syncwarp();
#pragma unroll
            for (int n2 = 0; n2 < HD / 16; ++n2) {
                float acc[2][4];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[x][e] = 0.0f;
#pragma unroll
                for (int kt = 0; kt < 4; ++kt) {
                    uint32_t b[4];
                    ldsm_x4_t(b, v_s + off(16 * kt + (lane & 7) + ((lane >> 3) & 1) * 8, 2 * n2 + (lane >> 4)));
#pragma unroll
                    for (int x = 0; x < TERMS; ++x) {
                        mma_16816(acc[0], pa[x][kt], b[0], b[1]);
                        mma_16816(acc[1], pa[x][kt], b[2], b[3]);
                    }
                }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[2 * n2 + x][e] = fmaf(acc[x][e], vf, o[2 * n2 + x][e] * rescale[e >> 1]);
            }
        }

        // ---- results, or this CTA's part of them
        const bool complete = tile == 0 && seg_end == item1;
        const int cta0 = (int)(((item0 + 1) * ctas - 1) / total), cta1 = (int)((item1 * ctas - 1) / total);
        float* part = p.s.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == cta0 ? 1 : 0)) * kRows * PITCH;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
            const int row = row_a + 8 * h;
            if (row >= it.n_rows) continue;
            const int rr = rtile * kRows + row;
            const size_t to = (size_t)(r.row0 + rr / p.gq);
            const int qh = head * p.gq + rr % p.gq;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = n * 8 + 2 * tig + e;
                    if (complete) store_result<T>(p, to, qh, d, o[n][2 * h + e], l[h]);
                    else __stcg(part + row * PITCH + d, o[n][2 * h + e]);
                }
            if (tig == 0) {
                if (complete) {
                    store_lse(p, to, qh, m[h], l[h]);
                } else {
                    __stcg(part + row * PITCH + HD, m[h]);
                    __stcg(part + row * PITCH + HD + 1, l[h]);
                }
            }
        }
        if (!complete) {  // the last CTA to arrive joins the parts in CTA order
            __syncthreads();
            if (tid == 0) s_last = arrive(p.s.ctr + cta0) == cta1 - cta0;
            __syncthreads();
            if (s_last) {
                const int parts = cta1 - cta0 + 1;
                auto part_of = [&](int k) { return p.s.part + (size_t)(2 * (cta0 + k) + (k == 0 ? 1 : 0)) * kRows * PITCH; };
                // a thread's 16 bytes of a row from every part, eight parts in flight
                for (int e = tid; e < it.n_rows * (HD / 4); e += kThreads) {
                    const int row = e / (HD / 4), d = (e - row * (HD / 4)) * 4;
                    float top = -INFINITY, sum = 0.0f;
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    constexpr int B = 8;
                    for (int k0 = 0; k0 < parts; k0 += B) {
                        float2 ml[B];
                        float4 v[B];
#pragma unroll
                        for (int k = 0; k < B; ++k) {
                            ml[k] = make_float2(-INFINITY, 0.0f);
                            v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (k0 + k < parts) {
                                const float* from = part_of(k0 + k) + row * PITCH;
                                ml[k] = __ldcg(reinterpret_cast<const float2*>(from + HD));
                                v[k] = __ldcg(reinterpret_cast<const float4*>(from + d));
                            }
                        }
                        const float before = top;
#pragma unroll
                        for (int k = 0; k < B; ++k) top = fmaxf(top, ml[k].x);
                        const float ref = top == -INFINITY ? 0.0f : top, f0 = ex2(before - ref);
                        sum *= f0;
                        acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
                        for (int k = 0; k < B; ++k) {
                            const float f = ex2(ml[k].x - ref);
                            sum = fmaf(f, ml[k].y, sum);
                            acc = make_float4(fmaf(f, v[k].x, acc.x), fmaf(f, v[k].y, acc.y), fmaf(f, v[k].z, acc.z), fmaf(f, v[k].w, acc.w));
                        }
                    }
                    const int rr = rtile * kRows + row, qh = head * p.gq + rr % p.gq;
                    const size_t to = (size_t)(r.row0 + rr / p.gq);
                    store_result<T>(p, to, qh, d, acc.x, sum);
                    store_result<T>(p, to, qh, d + 1, acc.y, sum);
                    store_result<T>(p, to, qh, d + 2, acc.z, sum);
                    store_result<T>(p, to, qh, d + 3, acc.w, sum);
                    if (d == 0) store_lse(p, to, qh, top, sum);
                }
                if (tid == 0) p.s.ctr[cta0] = 0;  // ready for the next call
            }
        }
        __syncthreads();  // shared memory is reused by the next segment
        u = seg_end;
        if (u == item1 && ++item == items) {
            item = 0;
            ++head;
        }
    }
}

template <class T, int FMT, int HD>
int launch(const Kv8Attn& a, cudaStream_t s) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
    constexpr size_t smem = (size_t)TERMS * kRows * HD * 2 + 2 * (size_t)kTile * HD * 2 + 4 * (size_t)kTile * HD;
    auto kern = kv8_rows_kernel<T, FMT, HD, TERMS>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
    static std::atomic<int> resident{0};
    int n = resident.load(std::memory_order_relaxed);
    if (n == 0) {
        IAM_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, smem));
        resident.store(n, std::memory_order_relaxed);
    }
    plan_kernel<kRows, kTile><<<1, kPlanThreads, 0, s>>>(a);
    IAM_CUDA_TRY(cudaGetLastError());
    kern<<<std::min(kPerSm, n) * a.sms, kThreads, smem, s>>>(a);
    IAM_CUDA_TRY(cudaGetLastError());
    return IAM_OK;
}

template <class T, int FMT>
int launch_dim(const Kv8Attn& a, cudaStream_t s) {
    switch (a.c.head_dim) {
        case 64: return launch<T, FMT, 64>(a, s);
        case 128: return launch<T, FMT, 128>(a, s);
        default: return launch<T, FMT, 256>(a, s);
    }
}

}  // namespace

size_t kv8_plan_words() { return 2 + 3 * (size_t)kKv8MaxItems; }
size_t kv8_rows_part_floats(int head_dim, int sms) { return (size_t)2 * kPerSm * sms * kRows * (head_dim + 4); }

int kv8_rows_launch(const Kv8Attn& a, int dtype, cudaStream_t s) {
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return a.c.format == IAM_KV8_INT8 ? launch_dim<T, IAM_KV8_INT8>(a, s) : launch_dim<T, IAM_KV8_E4M3>(a, s);
    });
}

}  // namespace iam
