// iam_kv8_decode.cu -- attention of few query rows per sequence (decoding) over the 8-bit paged cache.
//
// out = sum_t softmax_t(scale q.k_t) v_t in one pass with a running maximum and sum.  The rows of a
// (sequence, KV head), up to 8, are the N of the tensor cores' m16n8k16 and the tokens (for the scores)
// or the dims (for the values) its M, so a code enters one MMA and no row of the tile is padding for
// want of queries.  The codes go from global memory into the registers of the fragments they belong to:
// which physical dim plays a fragment's k (scores) or row (values) is free as long as the queries and
// the output agree, and the choice below makes every access 16 bytes of adjacent codes of one token.
#include <algorithm>
#include <atomic>

#include "iam_kv8.cuh"

namespace iam {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTile = kWarps * kKv8Group;  // tokens of a work unit: one group for each warp
constexpr int kMinUnits = 2;               // work units of a CTA at least, while there are enough

// The call's work: units of kTile tokens, in the order (sequence, KV head, row tile, token), cut into
// equal runs, one per CTA, whatever the sequences' lengths.
struct Item {
    int rt, nt;      // row tiles of the sequence, units of one
    int lo;          // first token read (a multiple of kKv8Group)
    long long units; // of the whole sequence
};

template <int RT>
IAM_DEV Item item_of(const Kv8Attn& p, const SeqRows& r) {
    Item it;
    it.rt = (r.n * p.gq + RT - 1) / RT;
    it.lo = p.window > 0 ? max(0, r.start - p.window + 1) & ~(kKv8Group - 1) : 0;
    it.nt = max(1, (r.cap - it.lo + kTile - 1) / kTile);  // a sequence without tokens still gets its rows written
    it.units = (long long)it.rt * it.nt * p.c.n_kv_heads;
    return it;
}

// C += A B with A a 16 x 16 tile; the transpose of an 8 x 8 tile of 16-bit values across the warp.
IAM_DEV uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// T: query and output type; TERMS 2 (fp32): columns 0..3 of the tile hold the rows' high fp16 terms and
// 4..7 the low ones (and so for the probabilities), which carries 22 bits of both through fp16 products.
template <class T, int FMT, int HD, int TERMS>
__global__ void __launch_bounds__(kThreads) kv8_decode_kernel(Kv8Attn p) {
    constexpr int RT = 8 / TERMS;
    constexpr int KS = HD / 16, KL = HD / 64, VW = HD / 32, MT = HD / 16;
    constexpr int PITCH = HD + 4;
    __shared__ __align__(16) float s_o[kWarps][8][PITCH];
    __shared__ float s_m[kWarps][8], s_l[kWarps][8];
    __shared__ float s_top[8], s_sum[8];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
    const int plog = 31 - __clz(p.c.page_size), kvh = p.c.n_kv_heads;

    // ---- this CTA's run of units (every warp finds it by itself)
    long long total = 0;
    for (int i = lane; i < p.c.n_seqs; i += 32)
        total += item_of<RT>(p, seq_rows(p.c, p.cu, p.lens, p.n_rows, i, blockIdx.x == 0 ? p.s.err : nullptr)).units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (total == 0) return;
    const long long ctas = min((long long)gridDim.x, (total + kMinUnits - 1) / kMinUnits);
    if (blockIdx.x >= ctas) return;
    const long long u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
    long long base = 0;  // units before sequence `seq`
    int seq = 0;
    for (int i0 = 0;; i0 += 32) {
        long long mine = 0;
        if (i0 + lane < p.c.n_seqs) mine = item_of<RT>(p, seq_rows(p.c, p.cu, p.lens, p.n_rows, i0 + lane, nullptr)).units;
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base + sum > u0);
        if (past) {
            const int at = __ffs(past) - 1;
            base += __shfl_sync(0xffffffffu, sum - mine, at);
            seq = i0 + at;
            break;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }

    long long u = u0;
    while (u < u1) {
        SeqRows r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr);
        Item it = item_of<RT>(p, r);
        while (u >= base + it.units) {  // (sequences without rows have no units)
            base += it.units;
            ++seq;
            r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr);
            it = item_of<RT>(p, r);
        }
        const long long rel = u - base;
        const int tile = (int)(rel % it.nt), rth = (int)(rel / it.nt);
        const int head = rth / it.rt, rtile = rth - head * it.rt;
        const long long item0 = u - tile, item1 = item0 + it.nt;
        const long long seg_end = min(u1, item1);
        const int t0 = it.lo + tile * kTile, t1 = min(r.cap, t0 + (int)(seg_end - u) * kTile);
        const int n_rows = min(RT, r.n * p.gq - rtile * RT);  // rows of this tile
        const int pos_lo = r.start + rtile * RT / p.gq, pos_hi = r.start + (rtile * RT + n_rows - 1) / p.gq;

        // ---- this warp's groups of 16 tokens: t0 + 16 (warp + kWarps i), i < cnt
        const int first = t0 + warp * kKv8Group;
        const int cnt = first < t1 ? (t1 - first + kTile - 1) / kTile : 0;
        const int32_t* table = p.c.block_table + (size_t)seq * p.c.max_pages;
        // lane l keeps page and scales of group (i & ~31) + l
        int ids = -1;
        float kss = 0.0f, vss = 0.0f;
        auto look_up = [&](int i) {
            const int t = first + (i + lane) * kTile;
            ids = -1;
            if (t < t1) {
                ids = table[t >> plog];
                if (ids < 0 || ids >= p.c.n_pages) {
                    *p.s.err = 1u;
                    ids = -1;
                }
            }
            kss = ids >= 0 ? p.c.k_scale[(size_t)ids * kvh + head] : 0.0f;
            vss = ids >= 0 ? p.c.v_scale[(size_t)ids * kvh + head] : 0.0f;
        };
        uint4 kq[2][KL];
        uint32_t vq[4][VW];
        auto row_at = [&](const void* codes, int id, int t) {
            return static_cast<const uint8_t*>(codes) + ((((size_t)id * kvh + head) << plog) + (t & (p.c.page_size - 1))) * HD;
        };
        auto load_k = [&](int id, int t) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int c = 0; c < KL; ++c) kq[half][c] = make_uint4(0u, 0u, 0u, 0u);
            if (id < 0) return;
            const uint8_t* src = row_at(p.c.k, id, t) + g * HD + tig * 16;
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int c = 0; c < KL; ++c) kq[half][c] = __ldcs(reinterpret_cast<const uint4*>(src + half * 8 * HD + c * 64));
        };
        auto load_v = [&](int id, int t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int tok = 2 * tig + (j & 1) + (j >> 1) * 8;
#pragma unroll
                for (int c = 0; c < VW; ++c) vq[j][c] = 0u;
                if (id < 0 || t + tok >= r.cap) continue;  // what is behind the last token is not read
                const uint8_t* src = row_at(p.c.v, id, t) + tok * HD;
                if constexpr (VW == 2) {
                    const uint2 w = __ldcs(reinterpret_cast<const uint2*>(src + g * 8));
                    vq[j][0] = w.x;
                    vq[j][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src + c * 128 + g * 16));
                        vq[j][4 * c] = w.x;
                        vq[j][4 * c + 1] = w.y;
                        vq[j][4 * c + 2] = w.z;
                        vq[j][4 * c + 3] = w.w;
                    }
                }
            }
        };
        int id = -1;
        if (cnt > 0) {
            look_up(0);
            id = __shfl_sync(0xffffffffu, ids, 0);
            load_k(id, first);
            load_v(id, first);
        }

        // ---- queries: column g's fragment; dims 64 c + 16 tig + 4 w + {0, 1} and {2, 3} are k-step
        // 4 c + w's columns 2 tig + {0, 1} and + 8
        uint32_t bq[KS][2];
        float rf[2];    // of columns 2 tig, 2 tig + 1: query shift undone, score scale, log2(e)
        int pos[2];
        {
            const int col = TERMS == 2 ? g & 3 : g;
            const int rr = rtile * RT + col;
            const bool have = col < n_rows;
            const T* src = have ? static_cast<const T*>(p.q.data) + (size_t)(r.row0 + rr / p.gq) * p.q.token_stride +
                                      (head * p.gq + rr % p.gq) * p.q.head_stride
                                : nullptr;
            float f[KS][4];
            float amax = 0.0f;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[ks][e] = have ? to_f32(src[(ks >> 2) * 64 + tig * 16 + (ks & 3) * 4 + e]) : 0.0f;
                    amax = fmaxf(amax, fabsf(f[ks][e]));
                }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int sh = query_shift(amax);
            const float up = pow2f(sh);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    f[ks][e] *= up;
                    if (TERMS == 2 && g >= 4) f[ks][e] = split_lo(f[ks][e]);
                }
                bq[ks][0] = pack_h2(f[ks][0], f[ks][1]);
                bq[ks][1] = pack_h2(f[ks][2], f[ks][3]);
            }
            const float mine = pow2f(-sh) * p.scale_log2;
            const int c0 = TERMS == 2 ? 2 * (tig & 1) : 2 * tig;
            rf[0] = __shfl_sync(0xffffffffu, mine, 4 * c0);
            rf[1] = __shfl_sync(0xffffffffu, mine, 4 * c0 + 4);
#pragma unroll
            for (int h = 0; h < 2; ++h) pos[h] = c0 + h < n_rows ? r.start + (rtile * RT + c0 + h) / p.gq : -1;
        }

        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[MT][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][e] = 0.0f;

        for (int i = 0; i < cnt; ++i) {
            const int t = first + i * kTile;
            const float ks_now = __shfl_sync(0xffffffffu, kss, i & 31), vs_now = __shfl_sync(0xffffffffu, vss, i & 31);
            const bool bad = id < 0;
            // scores of tokens g and g + 8 (rows), columns 2 tig and 2 tig + 1
            float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t w0 = reinterpret_cast<const uint32_t*>(&kq[0][ks >> 2])[ks & 3];
                const uint32_t w1 = reinterpret_cast<const uint32_t*>(&kq[1][ks >> 2])[ks & 3];
                uint32_t a[4];
                codes_to_half<FMT>(w0, a[0], a[2]);
                codes_to_half<FMT>(w1, a[1], a[3]);
                mma_16816(sc, a, bq[ks][0], bq[ks][1]);
            }
            int id_next = -1;
            if (i + 1 < cnt) {
                if (((i + 1) & 31) == 0) look_up(i + 1);
                id_next = __shfl_sync(0xffffffffu, ids, (i + 1) & 31);
                load_k(id_next, t + kTile);
            }
            if (TERMS == 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[e] += __shfl_xor_sync(0xffffffffu, sc[e], 2);
            const bool whole = !bad && t + kKv8Group - 1 <= pos_lo && t + kKv8Group <= r.cap &&
                               (p.window == 0 || t > pos_hi - p.window);
            float rescale[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float f = fminf(ks_now * rf[h], 3.402823466e38f);
                float s0 = sc[h] * f, s1 = sc[2 + h] * f;
                if (!whole) {
                    const int ta = t + g, tb = ta + 8;
                    if (bad || ta > pos[h] || ta >= r.cap || (p.window > 0 && ta <= pos[h] - p.window)) s0 = -INFINITY;
                    if (bad || tb > pos[h] || tb >= r.cap || (p.window > 0 && tb <= pos[h] - p.window)) s1 = -INFINITY;
                }
                float mx = fmaxf(s0, s1);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                mx = fmaxf(mx, m[h]);
                const float ref = mx == -INFINITY ? 0.0f : mx;  // nothing seen yet: every term is 0
                rescale[h] = ex2(m[h] - ref);
                m[h] = mx;
                sc[h] = ex2(s0 - ref);
                sc[2 + h] = ex2(s1 - ref);
                l[h] = fmaf(l[h], rescale[h], sc[h] + sc[2 + h]);  // this lane's tokens only
            }
            if (TERMS == 2 && tig >= 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[e] = split_lo(sc[e]);
            const uint32_t b0 = transpose8(pack_h2(sc[0], sc[1])), b1 = transpose8(pack_h2(sc[2], sc[3]));
            // values: word c of tokens 2 tig, 2 tig + 1 (a, b) and + 8 (cc, d) makes m-tiles 2 c and 2 c + 1,
            // whose rows g and g + 8 are dims 4 c' + {0, 1} and {2, 3} of this lane's piece
#pragma unroll
            for (int c = 0; c < VW; ++c) {
                const uint32_t ab01 = __byte_perm(vq[0][c], vq[1][c], 0x5140), ab23 = __byte_perm(vq[0][c], vq[1][c], 0x7362);
                const uint32_t cd01 = __byte_perm(vq[2][c], vq[3][c], 0x5140), cd23 = __byte_perm(vq[2][c], vq[3][c], 0x7362);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t a[4];
                    codes_to_half<FMT>(e ? ab23 : ab01, a[0], a[1]);
                    codes_to_half<FMT>(e ? cd23 : cd01, a[2], a[3]);
                    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    mma_16816(acc, a, b0, b1);
                    // the page's scale in fp32: no probability is rounded at another scale than its own
                    float(&om)[4] = o[2 * c + e];
                    om[0] = fmaf(acc[0], vs_now, om[0] * rescale[0]);
                    om[1] = fmaf(acc[1], vs_now, om[1] * rescale[1]);
                    om[2] = fmaf(acc[2], vs_now, om[2] * rescale[0]);
                    om[3] = fmaf(acc[3], vs_now, om[3] * rescale[1]);
                }
            }
            if (i + 1 < cnt) load_v(id_next, t + kTile);
            id = id_next;
        }

        // ---- join the warps in warp order
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
            if (g == 0) {
                s_m[warp][2 * tig + h] = m[h];
                s_l[warp][2 * tig + h] = l[h];
            }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = mt >> 1;
                const int dim = (VW == 2 ? 8 * g + 4 * c : (c >> 2) * 128 + 16 * g + 4 * (c & 3)) + 2 * (mt & 1) + (e >> 1);
                s_o[warp][2 * tig + (e & 1)][dim] = o[mt][e];
            }
        __syncthreads();
        const bool complete = tile == 0 && seg_end == item1;
        // CTAs that share this row tile: the owner of its first unit to the owner of its last
        const int cta0 = (int)(((item0 + 1) * ctas - 1) / total), cta1 = (int)((item1 * ctas - 1) / total);
        float* part = p.s.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == cta0 ? 1 : 0)) * 8 * PITCH;
        for (int e = tid; e < n_rows * HD; e += kThreads) {
            const int col = e / HD, d = e - col * HD;
            float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w][col]);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = ex2(s_m[w][col] - ref);
                sum = fmaf(f, s_l[w][col], sum);
                float v = s_o[w][col][d];
                if (TERMS == 2) v += s_o[w][col + 4][d];
                acc = fmaf(f, v, acc);
            }
            if (complete) {
                const int rr = rtile * RT + col;
                const size_t row = (size_t)(r.row0 + rr / p.gq);
                const int qh = head * p.gq + rr % p.gq;
                store_result<T>(p, row, qh, d, acc, sum);
                if (d == 0) store_lse(p, row, qh, top, sum);
            } else {
                __stcg(part + col * PITCH + d, acc);
                if (d == 0) {
                    __stcg(part + col * PITCH + HD, top);
                    __stcg(part + col * PITCH + HD + 1, sum);
                }
            }
        }
        if (!complete) {  // the last CTA to arrive joins the parts in CTA order
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(p.s.ctr + cta0, 1) == cta1 - cta0;
            __syncthreads();
            if (s_last) {
                __threadfence();
                const int parts = cta1 - cta0 + 1;
                auto part_of = [&](int k) { return p.s.part + (size_t)(2 * (cta0 + k) + (k == 0 ? 1 : 0)) * 8 * PITCH; };
                for (int col = warp; col < n_rows; col += kWarps) {
                    float top = -INFINITY;
                    for (int k = lane; k < parts; k += 32) top = fmaxf(top, __ldcg(part_of(k) + col * PITCH + HD));
                    top = warp_max(top);
                    const float ref = top == -INFINITY ? 0.0f : top;
                    float sum = 0.0f;
                    for (int k = lane; k < parts; k += 32)
                        sum = fmaf(ex2(__ldcg(part_of(k) + col * PITCH + HD) - ref), __ldcg(part_of(k) + col * PITCH + HD + 1), sum);
#pragma unroll
                    for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
                    if (lane == 0) {
                        s_top[col] = top;
                        s_sum[col] = sum;
                    }
                }
                __syncthreads();
                for (int e = tid; e < n_rows * (HD / 4); e += kThreads) {
                    const int col = e / (HD / 4), d = (e - col * (HD / 4)) * 4;
                    const float ref = s_top[col] == -INFINITY ? 0.0f : s_top[col];
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int k = 0; k < parts; ++k) {
                        const float* from = part_of(k) + col * PITCH;
                        const float f = ex2(__ldcg(from + HD) - ref);
                        const float4 v = __ldcg(reinterpret_cast<const float4*>(from + d));
                        acc.x = fmaf(f, v.x, acc.x);
                        acc.y = fmaf(f, v.y, acc.y);
                        acc.z = fmaf(f, v.z, acc.z);
                        acc.w = fmaf(f, v.w, acc.w);
                    }
                    const int rr = rtile * RT + col;
                    const size_t row = (size_t)(r.row0 + rr / p.gq);
                    const int qh = head * p.gq + rr % p.gq;
                    store_result<T>(p, row, qh, d, acc.x, s_sum[col]);
                    store_result<T>(p, row, qh, d + 1, acc.y, s_sum[col]);
                    store_result<T>(p, row, qh, d + 2, acc.z, s_sum[col]);
                    store_result<T>(p, row, qh, d + 3, acc.w, s_sum[col]);
                    if (d == 0) store_lse(p, row, qh, s_top[col], s_sum[col]);
                }
                if (tid == 0) p.s.ctr[cta0] = 0;  // ready for the next call
            }
        }
        __syncthreads();  // shared memory is reused by the next segment
        u = seg_end;
    }
}

template <class T, int FMT, int HD>
int launch(const Kv8Attn& a, cudaStream_t s) {
    auto kern = kv8_decode_kernel<T, FMT, HD, sizeof(T) == 4 ? 2 : 1>;
    static std::atomic<int> resident{0};
    int n = resident.load(std::memory_order_relaxed);
    if (n == 0) {
        IAM_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, 0));
        resident.store(n, std::memory_order_relaxed);
    }
    kern<<<std::min(a.s.max_ctas, n * a.sms), kThreads, 0, s>>>(a);
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

int kv8_decode_launch(const Kv8Attn& a, int dtype, cudaStream_t s) {
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return a.c.format == IAM_KV8_INT8 ? launch_dim<T, IAM_KV8_INT8>(a, s) : launch_dim<T, IAM_KV8_E4M3>(a, s);
    });
}

}  // namespace iam
