// iam_kv8_decode.cu -- attention of few query rows per sequence (decoding) over the 8-bit paged cache.
//
// out = sum_t softmax_t(scale q.k_t) v_t in one pass with a running maximum and sum.  The rows of a
// (sequence, KV head), up to 8, are the N of the tensor cores' m16n8k16 and the tokens (for the scores)
// or the dims (for the values) its M, so a code enters one MMA and no row of the tile is padding for
// want of queries.  Which physical dim plays a fragment's k (scores) or row (values) is free as long as the
// queries and the output agree: the choice below makes every access 16 bytes of adjacent codes of one token.
#include <climits>
#include <algorithm>
#include <atomic>

#include "iam_kv8.cuh"
#include "iam_tc.cuh"

namespace iam {
namespace {

constexpr int kMinUnits = 8;  // work units of a CTA at least, while there are enough

// Warps of a CTA (one CTA an SM) and groups of 16 tokens in each warp's ring: 192 KB of codes on their way.
template <int HD>
struct Shape {
    static constexpr int kWarps = HD == 256 ? 8 : 16;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kHalves = HD == 256 ? 2 : 1;          // 128-byte columns of a row
    static constexpr int kBox = kKv8Group * HD / kHalves;      // bytes of one copy
    static constexpr int kStage = 2 * kHalves * kBox;          // a group's keys and values
    static constexpr int kStages = 192 * 1024 / (kWarps * kStage);
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kPitch = HD + 4;
    static_assert(kWarps * 8 * kPitch * 4 <= kRing, "the warps' results are joined where the codes were");
};

// The call's work: groups of 16 tokens in the order (sequence, KV head, row tile, token), cut into equal runs, one
// per CTA, whatever the sequences' lengths.
struct Item {
    int rt, nt;    // row tiles of the sequence, groups of one
    int lo;        // first token read (a multiple of kKv8Group)
    int units;     // of the whole sequence (the sum over the sequences is checked against 2^31)
};

template <int RT>
IAM_DEV Item item_of(const Kv8Attn& p, const SeqRows& r) {
    Item it;
    it.rt = (r.n * p.gq + RT - 1) / RT;
    it.lo = p.window > 0 ? max(0, r.start - p.window + 1) & ~(kKv8Group - 1) : 0;
    it.nt = max(1, (r.cap - it.lo + kKv8Group - 1) / kKv8Group);  // a sequence without tokens still gets its rows written
    const long long units = (long long)it.rt * it.nt * p.c.n_kv_heads;
    it.units = (int)min(units, (long long)INT_MAX);
    return it;
}

// Run of CTA c when `total` units are cut into `ctas` runs, and the CTA that has unit u.
struct Cut {
    int q, rem;  // units of a run, and how many runs have one more
    IAM_DEV int first(int c) const { return q * c + min(c, rem); }
    IAM_DEV int owner(int u) const {
        const int big = rem * (q + 1);
        return u < big ? u / (q + 1) : rem + (u - big) / q;
    }
};

// C += A B with A a 16 x 16 tile; the transpose of an 8 x 8 tile of 16-bit values across the warp.
IAM_DEV uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// T: query and output type; TERMS 2 (fp32): columns 0..3 of the tile hold the rows' high fp16 terms and
// 4..7 the low ones (and so for the probabilities), which carries 22 bits of both through fp16 products.
// Each warp streams its own groups of tokens through its own ring in shared memory: lane 0 has TMA fetch a group's
// keys and values (16 rows each, swizzled so that the reads below meet no bank twice) as soon as the warp has
// taken the group before out of that place; no warp waits for another.  The fragments' rows are tokens in the
// order 0 4 2 6 5 1 7 3 for the same reason: eight lanes then read eight different 16-byte columns both as
// keys (two tokens, four columns) and as values (four tokens, two columns).
template <class T, int FMT, int HD, int TERMS>
__global__ void __launch_bounds__(Shape<HD>::kThreads, 1)
    kv8_decode_kernel(const Kv8Attn p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = Shape<HD>;
    constexpr int RT = 8 / TERMS, W = S::kWarps;
    constexpr int KS = HD / 16, KL = HD / 64, VW = HD / 32, MT = HD / 16;
    constexpr int PITCH = S::kPitch;
    extern __shared__ unsigned char s_raw[];
    __shared__ __align__(8) uint64_t s_full[W][S::kStages];
    __shared__ float s_m[W][8], s_l[W][8];
    __shared__ float s_top[8], s_sum[8];
    __shared__ int s_last;
    unsigned char* ring = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    auto s_o = reinterpret_cast<float (*)[8][PITCH]>(ring);  // the warps' results, when the codes are used up
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
    const int plog = 31 - __clz(p.c.page_size), kvh = p.c.n_kv_heads;
    unsigned char* mine_ring = ring + (size_t)warp * S::kStages * S::kStage;
    if (lane == 0) {
        for (int i = 0; i < S::kStages; ++i) mbar_init(&s_full[warp][i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();

    // ---- this CTA's run of units (every warp finds it by itself)
    long long all = 0;
    for (int i = lane; i < p.c.n_seqs; i += 32)
        all += item_of<RT>(p, seq_rows(p.c, p.cu, p.lens, p.n_rows, i, blockIdx.x == 0 && warp == 0 ? p.s.err : nullptr)).units;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (all == 0) return;
    if (all > INT_MAX / 2) {  // (more than 16 G tokens)
        if (blockIdx.x == 0 && tid == 0) atomicOr(p.s.err, kKv8ErrRange);
        return;
    }
    const int total = (int)all, ctas = min((int)gridDim.x, (total + kMinUnits - 1) / kMinUnits);
    if ((int)blockIdx.x >= ctas) return;
    const Cut cut{total / ctas, total % ctas};
    const int u0 = cut.first(blockIdx.x), u1 = cut.first(blockIdx.x + 1);
    int base = 0;  // units before sequence `seq`
    int seq = 0;
    for (int i0 = 0; p.c.n_seqs > 1; i0 += 32) {
        int mine = 0;
        if (i0 + lane < p.c.n_seqs) mine = item_of<RT>(p, seq_rows(p.c, p.cu, p.lens, p.n_rows, i0 + lane, nullptr)).units;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
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

    uint32_t phases = 0;  // of the ring's barriers, a bit each
    int u = u0;
    while (u < u1) {
        SeqRows r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr);
        Item it = item_of<RT>(p, r);
        while (u >= base + it.units) {  // (sequences without rows have no units)
            base += it.units;
            ++seq;
            r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr);
            it = item_of<RT>(p, r);
        }
        const int rel = u - base;
        const int rth = rel / it.nt, tile = rel - rth * it.nt;
        const int head = rth / it.rt, rtile = rth - head * it.rt;
        const int item0 = u - tile, item1 = item0 + it.nt;
        const int seg_end = min(u1, item1);
        const int t0 = it.lo + tile * kKv8Group, t1 = min(r.cap, t0 + (seg_end - u) * kKv8Group);
        const int n_rows = min(RT, r.n * p.gq - rtile * RT);  // rows of this tile
        const int pos_lo = r.start + rtile * RT / p.gq, pos_hi = r.start + (rtile * RT + n_rows - 1) / p.gq;

        // ---- this warp's groups of 16 tokens: t0 + 16 (warp + W i), i < cnt
        constexpr int STRIDE = W * kKv8Group;
        const int first = t0 + warp * kKv8Group;
        const int cnt = first < t1 ? (t1 - first + STRIDE - 1) / STRIDE : 0;
        const int32_t* table = p.c.block_table + (size_t)seq * p.c.max_pages;
        // lane l keeps the page of group (i & ~31) + l, looked up when the copies get there, and its scales
        int ids = -1, ids_before = -1;
        float kss = 0.0f, vss = 0.0f, kss_before = 0.0f, vss_before = 0.0f;
        auto look_up = [&](int i) {
            const int t = first + (i + lane) * STRIDE;
            ids_before = ids;
            kss_before = kss;
            vss_before = vss;
            ids = -1;
            if (t < t1) {
                ids = table[t >> plog];
                if (ids < 0 || ids >= p.c.n_pages) {
                    atomicOr(p.s.err, kKv8ErrRange);
                    ids = -1;
                }
            }
            kss = ids >= 0 ? p.c.k_scale[(size_t)ids * kvh + head] : 0.0f;
            vss = ids >= 0 ? p.c.v_scale[(size_t)ids * kvh + head] : 0.0f;
        };
        auto issue = [&](int i) {  // group i into stage i % kStages
            if ((i & 31) == 0) look_up(i);
            const int id = __shfl_sync(0xffffffffu, ids, i & 31);
            if (lane == 0 && id >= 0) {
                const int t = first + i * STRIDE, st = i % S::kStages;
                const int row = (int)((((long long)id * kvh + head) << plog) + (t & (p.c.page_size - 1)));
                unsigned char* to = mine_ring + st * S::kStage;
                mbar_expect_tx(&s_full[warp][st], S::kStage);
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h) {
                    tma_load_2d(to + h * S::kBox, &map_k, 128 * h, row, &s_full[warp][st]);
                    tma_load_2d(to + (S::kHalves + h) * S::kBox, &map_v, 128 * h, row, &s_full[warp][st]);
                }
            }
        };
        for (int i = 0; i < min(cnt, S::kStages); ++i) issue(i);

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

        // fragment row j is token order[j] of its eight
        auto token = [](int j) { return HD == 64 ? j : (0x37156240 >> (4 * j)) & 7; };
        // the 16-byte column c of a row in the swizzled box
        auto column = [](int row, int c) {
            return HD == 64 ? row * 64 + ((c ^ ((row >> 1) & 3)) << 4) : row * 128 + ((c ^ (row & 7)) << 4);
        };
        const int tok_g = token(g);
        for (int i = 0; i < cnt; ++i) {
            const int t = first + i * STRIDE, st = i % S::kStages;
            // (the copies may already be a batch of 32 look-ups further)
            const bool older = (i & ~31) != (min(i + S::kStages - 1, cnt - 1) & ~31);
            const int id = __shfl_sync(0xffffffffu, older ? ids_before : ids, i & 31);
            const float ks_now = __shfl_sync(0xffffffffu, older ? kss_before : kss, i & 31);
            const float vs_now = __shfl_sync(0xffffffffu, older ? vss_before : vss, i & 31);
            const bool bad = id < 0;
            const unsigned char* box_k = mine_ring + st * S::kStage;
            const unsigned char* box_v = box_k + S::kHalves * S::kBox;
            if (!bad) {
                if (!mbar_wait(&s_full[warp][st], (phases >> st) & 1u, nullptr)) atomicOr(p.s.err, kKv8ErrWait);
                phases ^= 1u << st;
            }
            // scores of fragment rows g and g + 8, columns 2 tig and 2 tig + 1
            float sc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sd[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < KL; ++c) {
                const unsigned char* half = box_k + (HD == 256 ? (c >> 1) * S::kBox : 0);
                const int piece = HD == 256 ? (c & 1) * 4 + tig : c * 4 + tig;
                const uint4 q0 = *reinterpret_cast<const uint4*>(half + column(tok_g, piece));
                const uint4 q1 = *reinterpret_cast<const uint4*>(half + column(tok_g + 8, piece));
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    uint32_t a[4];
                    codes_to_half<FMT>(reinterpret_cast<const uint32_t*>(&q0)[w], a[0], a[2]);
                    codes_to_half<FMT>(reinterpret_cast<const uint32_t*>(&q1)[w], a[1], a[3]);
                    mma_16816(w & 1 ? sd : sc, a, bq[4 * c + w][0], bq[4 * c + w][1]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[e] += sd[e];
            uint32_t vq[4][VW];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int tok = token(2 * tig + (j & 1)) + (j >> 1) * 8;
                if constexpr (VW == 2) {
                    const uint2 w = *reinterpret_cast<const uint2*>(box_v + column(tok, g >> 1) + (g & 1) * 8);
                    vq[j][0] = w.x;
                    vq[j][1] = w.y;
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const uint4 w = *reinterpret_cast<const uint4*>(box_v + c * S::kBox + column(tok, g));
                        vq[j][4 * c] = w.x;
                        vq[j][4 * c + 1] = w.y;
                        vq[j][4 * c + 2] = w.z;
                        vq[j][4 * c + 3] = w.w;
                    }
                }
            }
            __syncwarp();
            if (i + S::kStages < cnt) issue(i + S::kStages);
            if (t + kKv8Group > r.cap || bad) {  // what stands behind the last token has no part in the sums
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (bad || t + token(2 * tig + (j & 1)) + (j >> 1) * 8 >= r.cap)
#pragma unroll
                        for (int c = 0; c < VW; ++c) vq[j][c] = 0u;
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
                    const int ta = t + tok_g, tb = ta + 8;
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
            // values: word c of fragment columns 2 tig, 2 tig + 1 (a, b) and + 8 (cc, d) makes m-tiles 2 c and 2 c + 1,
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
        }

        // ---- join the warps in warp order
        __syncthreads();  // every warp's codes are used up
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
        const int cta0 = cut.owner(item0), cta1 = cut.owner(item1 - 1);
        float* part = p.s.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == cta0 ? 1 : 0)) * 8 * PITCH;
        for (int e = tid; e < n_rows * HD; e += S::kThreads) {
            const int col = e / HD, d = e - col * HD;
            float top = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, s_m[w][col]);
            const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
            for (int w = 0; w < W; ++w) {
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
                for (int col = warp; col < n_rows; col += W) {
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
                for (int e = tid; e < n_rows * (HD / 4); e += S::kThreads) {
                    const int col = e / (HD / 4), d = (e - col * (HD / 4)) * 4;
                    const float ref = s_top[col] == -INFINITY ? 0.0f : s_top[col];
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
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
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring is the copies' again
        __syncthreads();
        u = seg_end;
    }
}

// The cache's codes as rows of head_dim bytes, copied 16 rows (of at most 128 bytes) at a time.
template <int HD>
int make_map(CUtensorMap* map, const void* codes, const iam_kv8_cache& c) {
    auto fn = tensor_map_encoder();
    if (fn == nullptr) return fail(IAM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {HD, (cuuint64_t)c.n_pages * c.n_kv_heads * c.page_size};
    const cuuint64_t strides[1] = {HD};
    const cuuint32_t box[2] = {HD > 128 ? 128 : HD, kKv8Group};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, HD == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(IAM_ERR_CUDA, "kv8: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return IAM_OK;
}

template <class T, int FMT, int HD>
int launch(const Kv8Attn& a, cudaStream_t s) {
    constexpr size_t smem = Shape<HD>::kRing + 1024;
    auto kern = kv8_decode_kernel<T, FMT, HD, sizeof(T) == 4 ? 2 : 1>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
    CUtensorMap mk, mv;
    int rc = make_map<HD>(&mk, a.c.k, a.c);
    if (rc == IAM_OK) rc = make_map<HD>(&mv, a.c.v, a.c);
    if (rc) return rc;
    kern<<<a.sms, Shape<HD>::kThreads, smem, s>>>(a, mk, mv);
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

int kv8_max_ctas(int sms) { return 4 * sms; }
size_t kv8_decode_part_floats(int head_dim, int sms) { return (size_t)2 * sms * 8 * (head_dim + 4); }

int kv8_decode_launch(const Kv8Attn& a, int dtype, cudaStream_t s) {
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return a.c.format == IAM_KV8_INT8 ? launch_dim<T, IAM_KV8_INT8>(a, s) : launch_dim<T, IAM_KV8_E4M3>(a, s);
    });
}

}  // namespace iam
