// iam_kv8_decode.cu -- attention of few query rows per sequence (decoding) over the 8-bit paged cache.
//
// out = sum_t softmax_t(scale q.k_t) v_t in one pass with a running maximum and sum.  The rows of a
// (sequence, KV head), up to 8, are the N of the tensor cores' m16n8k16 and the tokens (for the scores)
// or the dims (for the values) its M, so a code enters one MMA and no row of the tile is padding for
// want of queries.  Which physical dim plays a fragment's k (scores) or row (values) is free as long as the
// queries and the output agree: the choice below makes every access 16 bytes of adjacent codes of one token.
//
// Long contexts (one sequence of 131071 tokens, 8 KV heads of 128, 268 MB of e4m3: 56.8 us, 4.7 TB/s; int8, whose conversion
// takes more instructions: 63; 48 ragged requests, 429 MB: 91 us, 4.7 TB/s) are bound by the fixed latencies of a warp's chain from
// codes to products: the registers allow three warps a scheduler, which issue every second cycle while no unit is more than half
// busy.  Short ones by the start (finding the run, the first page numbers, scales and copies one after another: 4 us) and
// the join (8192 tokens in fp32: 13.5 us for 17 MB).
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "iam_kv8.cuh"
#include "iam_tc.cuh"

namespace iam {
namespace {

// Groups of tokens of a CTA at least, where a context is shared (1 x 1024 tokens: 10.5 us; with 4 10.8, with 16 11.6; long
// contexts do not tell them apart).
constexpr int kMinGroups = 8;
// What opening and joining a piece of a context costs, in groups (48 ragged requests 92 us, 200 of up to 600 tokens 59, 13 x 7 drafted
// rows 34; with 8 groups 101, 70, 63; with 48 98, 64, 31; with 96 109, 67, 36).
constexpr int kItemCost = 24;
// Probabilities (at most 1) are lifted by this before they are rounded to fp16, whose smallest step is 2^-24: a weight of 2^-28
// still has all of its 11 bits, and what is lost of smaller ones is 2^-39 of the largest value a token.
constexpr float kLift = 16384.0f;

// Warps of a CTA (one CTA an SM; as many as have the registers they need) and groups of 16 tokens in each warp's
// ring: 128 to 144 KB of codes on their way.
template <int HD>
struct Shape {
    static constexpr int kWarps = HD == 256 ? 8 : HD == 128 ? 12 : 16;
    static constexpr int kThreads = 32 * kWarps;
    static constexpr int kHalves = HD == 256 ? 2 : 1;          // 128-byte columns of a row
    static constexpr int kBox = kKv8Group * HD / kHalves;      // bytes of one copy
    static constexpr int kStage = 2 * kHalves * kBox;          // a group's keys and values
    static constexpr int kStages = HD == 256 ? 2 : HD == 128 ? 3 : 4;
    static constexpr int kRing = kWarps * kStages * kStage;
    static constexpr int kPitch = HD + 4;
    static constexpr int kHeads = HD == 64 ? 8 : 4;             // heads of an item at most
    static constexpr int kSmem = kRing + kWarps * 8 * kPitch * 4 + 1024;
};

// A (sequence, group of `hg` KV heads, row tile) is an item: nt groups of 16 tokens from token lo on, of each of its
// heads; a CTA's warps are dealt to the heads.  (One head an item while items are fewer than SMs; more
// where there are many, for a piece's opening and join are paid once for all of its heads.)  Items are laid end to
// end, each preceded by kItemCost groups of nothing, and the line is cut into equal runs, one per CTA, whatever
// the sequences' lengths.  With at most half as many items as SMs each gets CTAs of its own in proportion, so
// that none opens a second piece.
struct Items {
    int n;   // items of the sequence
    int rt;  // row tiles of a group of heads
    int nt, lo;
};

template <int RT>
IAM_DEV Items items_of(const Kv8Attn& p, int hg, const SeqRows& r) {
    Items it;
    it.rt = (r.n * p.gq + RT - 1) / RT;
    it.n = (int)min((long long)it.rt * (p.c.n_kv_heads / hg), (long long)INT_MAX);
    it.lo = p.window > 0 ? max(0, r.start - p.window + 1) & ~(kKv8Group - 1) : 0;
    it.nt = max(1, (r.cap - it.lo + kKv8Group - 1) / kKv8Group);  // a sequence without tokens still gets its rows written
    return it;
}

// The line of `total` units cut into `ctas` runs: the first unit of CTA c's, and the CTA that has unit u.
struct Cut {
    int q, rem;  // units of a run, and how many runs have one more
    IAM_DEV int first(int c) const { return q * c + min(c, rem); }
    IAM_DEV int owner(int u) const {
        const int big = rem * (q + 1);
        return u < big ? u / (q + 1) : rem + (u - big) / q;
    }
};

IAM_DEV long long warp_sum(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// C += A B with A a 16 x 16 tile; the transpose of an 8 x 8 tile of 16-bit values across the warp.
IAM_DEV uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// T: query and output type; TERMS 2 (fp32): columns 0..3 of the tile hold the rows' high fp16 terms and
// 4..7 the low ones (and so for the probabilities), which carries 22 bits of both through fp16 products (of a probability, down
// to 2^-17 of its warp's maximum, where the low term meets fp16's smallest step).
// TERMS 1 (16-bit types): one fp16 term, so a probability is off by 2^-12 of itself, where the result's own rounding is 2^-11
// (fp16) or 2^-8 (bf16) and the errors of a row's tokens average.  Off by (2-norm, against 64 bits) 2.23e-4 instead of 2.07e-4 with a
// second term for 131071 tokens in fp16, 1.657e-3 instead of 1.655e-3 for 48 ragged requests in bf16; that term's
// products take 66 us instead of 58 and 109 instead of 94.  A caller who wants 22 bits passes fp32 queries.
// Each warp streams its own groups of tokens through its own ring in shared memory: TMA fetches a group's keys and
// values (16 rows each, swizzled so that the reads below meet no bank twice) as soon as the warp has taken an
// earlier group out of that place, into the next piece of context already; the warps wait for one another only
// to join a piece's results.  (One feeding warp for all of them was slower: its lanes share the wait for each
// look-up.)  The fragments' rows are tokens in the order 0 4 2 6 5 1 7 3 for the same reason: eight lanes then
// read eight different 16-byte columns both as keys (two tokens, four columns) and as values (four tokens, two
// columns).
template <class T, int FMT, int HD, int TERMS>
__global__ void __launch_bounds__(Shape<HD>::kThreads, 1)
    kv8_decode_kernel(const Kv8Attn p, int hg, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = Shape<HD>;
    constexpr int RT = 8 / TERMS, W = S::kWarps;
    constexpr int KS = HD / 16, KL = HD / 64, VW = HD / 32, MT = HD / 16;
    constexpr int PITCH = S::kPitch, QE = HD / 32;
    extern __shared__ unsigned char s_raw[];
    __shared__ __align__(8) uint64_t s_full[W][S::kStages];
    __shared__ float4 s_group[W][S::kStages];  // key scale, value scale, page (as bits) of the group in a place
    __shared__ __align__(16) __half s_q[S::kHeads][8][HD + 8];  // [head of the item][column]
    __shared__ float s_rf[S::kHeads][8];
    __shared__ float s_m[W][8], s_l[W][8];
    __shared__ float s_weight[W][8], s_top[S::kHeads][8], s_sum[S::kHeads][8];
    __shared__ int s_last;
    unsigned char* ring = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    auto s_o = reinterpret_cast<float (*)[8][PITCH]>(ring + S::kRing);  // the warps' results
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, tig = lane & 3;
    const int plog = 31 - __clz(p.c.page_size), kvh = p.c.n_kv_heads;
    const int per_head = W / hg;  // warps that share a head
    if (lane == 0) {
        for (int i = 0; i < S::kStages; ++i) mbar_init(&s_full[warp][i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    }
    __syncwarp();

    // ---- this CTA's run (every warp finds it by itself)
    long long n_items = 0, n_groups = 0;
    for (int i = lane; i < p.c.n_seqs; i += 32) {
        const Items it = items_of<RT>(p, hg, seq_rows(p.c, p.cu, p.lens, p.n_rows, i, blockIdx.x == 0 && warp == 0 ? p.s.err : nullptr));
        n_items += it.n;
        n_groups += (long long)it.n * it.nt;
    }
    n_items = warp_sum(n_items);
    n_groups = warp_sum(n_groups);
    if (n_items == 0) return;
    const long long line = n_groups + n_items * kItemCost;
    if (line > INT_MAX / 2) {  // (more than 16 G tokens)
        if (blockIdx.x == 0 && tid == 0) atomicOr(p.s.err, kKv8ErrRange);
        return;
    }
    const int grid = gridDim.x;
    const bool few = n_items * 2 <= grid;
    // few: the CTAs that share an item, so that their sum over the items is at most the grid
    auto sharers = [&](const Items& it) {
        return min(1 + (int)((long long)it.nt * (grid - n_items) / n_groups), (it.nt + kMinGroups - 1) / kMinGroups);
    };
    const int total = (int)line, ctas = (int)min((long long)grid, max(n_items, (n_groups + kMinGroups - 1) / kMinGroups));
    if (!few && (int)blockIdx.x >= ctas) return;
    const Cut cut{total / ctas, total % ctas};
    const int u0 = few ? (int)blockIdx.x : cut.first(blockIdx.x), u1 = few ? u0 + 1 : cut.first(blockIdx.x + 1);
    int base0 = 0, seq0 = 0;  // what stands before sequence seq0: CTAs (few) or units
    for (int i0 = 0; p.c.n_seqs > 1; i0 += 32) {
        int mine = 0;
        if (i0 + lane < p.c.n_seqs) {
            const Items it = items_of<RT>(p, hg, seq_rows(p.c, p.cu, p.lens, p.n_rows, i0 + lane, nullptr));
            mine = it.n * (few ? sharers(it) : it.nt + kItemCost);
        }
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += up;
        }
        const unsigned past = __ballot_sync(0xffffffffu, base0 + sum > u0);
        if (past) {
            const int at = __ffs(past) - 1;
            base0 += __shfl_sync(0xffffffffu, sum - mine, at);
            seq0 = i0 + at;
            break;
        }
        base0 += __shfl_sync(0xffffffffu, sum, 31);
        if (i0 + 32 >= p.c.n_seqs) return;  // (few: more CTAs than shares)
    }

    // A piece of an item: groups [ta, tb) of it, shared by CTAs cta0 .. cta1.  One state walks the pieces for the
    // copies, another one behind it for the sums.
    struct Piece {
        int u, base, seq;  // place on the line, units (or CTAs) before the sequence
        SeqRows r;
        int head, rtile, ta, tb, lo, cta0, cta1;  // head: the first of its group
    };
    auto open = [&](Piece& c) {  // the piece at c.u < u1; advances c.u behind it
        for (;;) {
            c.r = seq_rows(p.c, p.cu, p.lens, p.n_rows, c.seq, nullptr);
            const Items it = items_of<RT>(p, hg, c.r);
            const int share = few ? sharers(it) : it.nt + kItemCost, end = c.base + it.n * share;
            if (c.u >= end) {  // (sequences without rows have no items)
                c.base = end;
                if (++c.seq >= p.c.n_seqs) {
                    c.u = u1;
                    c.ta = c.tb = 0;
                    return false;
                }
                continue;
            }
            const int rel = c.u - c.base, item = rel / share, idx = rel - item * share;
            c.lo = it.lo;
            c.head = item / it.rt;
            c.rtile = item - c.head * it.rt;
            c.head *= hg;
            const int item0 = c.u - idx;
            if (few) {
                c.ta = (int)((long long)it.nt * idx / share);
                c.tb = (int)((long long)it.nt * (idx + 1) / share);
                c.cta0 = item0;
                c.cta1 = item0 + share - 1;
                ++c.u;
                return true;
            }
            const int stop = min(u1, item0 + share);
            c.ta = max(0, idx - kItemCost);
            c.tb = max(0, stop - item0 - kItemCost);
            c.cta0 = cut.owner(item0 + kItemCost);
            c.cta1 = cut.owner(item0 + share - 1);
            c.u = stop;
            if (c.tb > c.ta) return true;
            if (c.u >= u1) return false;  // nothing of the item but its cost
        }
    };
    Piece now;
    now.u = u0;
    now.base = base0;
    now.seq = seq0;

    const int hh = warp % hg;  // this warp's head of the item
    unsigned char* mine_ring = ring + (size_t)warp * S::kStages * S::kStage;
    // The queries of a piece, a row (of hg * RT) a warp and turn: lane l has dims QE l ..; asked for before anything
    // waits.
    constexpr int TURNS = (S::kHeads * RT + W - 1) / W;
    float qf[QE];
    auto ask = [&](const Piece& c, int row, float (&f)[QE]) {
        const int rr = c.rtile * RT + row % RT;
        if (row < hg * RT && rr < c.r.n * p.gq) {
            const T* src = static_cast<const T*>(p.q.data) + (size_t)(c.r.row0 + rr / p.gq) * p.q.token_stride +
                           ((c.head + row / RT) * p.gq + rr % p.gq) * p.q.head_stride + lane * QE;
#pragma unroll
            for (int e = 0; e < QE; ++e) f[e] = to_f32(src[e]);
        }
    };
    // The stream of the warp's groups, kStages ahead of their use and into the next pieces.
    bool left = now.u < u1 && open(now);
    Piece ahead = now;
    int t_ahead = now.ta + warp / hg, n_issued = 0, batch = 32;
    bool more = left;
    int ids = -1;  // lane l: page and scales of group t_ahead + per_head l, as of the last look-up
    float kss = 0.0f, vss = 0.0f;
    auto issue = [&] {
        while (more && t_ahead >= ahead.tb) {
            more = ahead.u < u1 && open(ahead);
            if (more) t_ahead = ahead.ta + warp / hg;
            batch = 32;
        }
        if (!more) return;
        if (batch == 32) {
            const int t = t_ahead + per_head * lane;
            ids = -1;
            if (t < ahead.tb && ahead.lo + t * kKv8Group < ahead.r.cap) {
                ids = __ldg(p.c.block_table + (size_t)ahead.seq * p.c.max_pages + ((ahead.lo + t * kKv8Group) >> plog));
                if (ids < 0 || ids >= p.c.n_pages) {
                    atomicOr(p.s.err, kKv8ErrRange);
                    ids = -1;
                }
            }
            kss = ids >= 0 ? __ldg(p.c.k_scale + (size_t)ids * kvh + ahead.head + hh) : 0.0f;
            vss = ids >= 0 ? __ldg(p.c.v_scale + (size_t)ids * kvh + ahead.head + hh) : 0.0f;
            batch = 0;
        }
        if (lane == batch) {  // the lane that looked it up
            const int st = n_issued % S::kStages;
            mbar_expect_tx(&s_full[warp][st], ids >= 0 ? S::kStage : 0);
            if (ids >= 0) {
                const int tok = ahead.lo + t_ahead * kKv8Group;
                const int row = (int)((((long long)ids * kvh + ahead.head + hh) << plog) + (tok & (p.c.page_size - 1)));
                unsigned char* to = mine_ring + st * S::kStage;
#pragma unroll
                for (int h = 0; h < S::kHalves; ++h) {
                    tma_load_2d(to + h * S::kBox, &map_k, 128 * h, row, &s_full[warp][st]);
                    tma_load_2d(to + (S::kHalves + h) * S::kBox, &map_v, 128 * h, row, &s_full[warp][st]);
                }
            }
            s_group[warp][st] = make_float4(kss, vss, __int_as_float(ids), 0.0f);  // (the copies do not wait for the scales)
        }
        ++n_issued;
        ++batch;
        t_ahead += per_head;
    };
    if (left) ask(now, warp, qf);
    for (int i = 0; i < S::kStages; ++i) issue();

    int n_used = 0;
    while (left) {
        const SeqRows& r = now.r;
        const int head = now.head, rtile = now.rtile;
        const int n_rows = min(RT, r.n * p.gq - rtile * RT);  // rows of this tile
        const int pos_lo = r.start + rtile * RT / p.gq, pos_hi = r.start + (rtile * RT + n_rows - 1) / p.gq;

        // ---- queries: a warp takes a row, shifts it into fp16's range and rounds it or splits it in two
#pragma unroll
        for (int turn = 0; turn < TURNS; ++turn) {
            const int row = warp + turn * W, col = row % RT;
            if (row >= hg * RT) break;
            if (turn > 0) ask(now, row, qf);
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < QE; ++e) {
                qf[e] = col < n_rows ? qf[e] : 0.0f;
                amax = fmaxf(amax, fabsf(qf[e]));
            }
            const int sh = query_shift(warp_max(amax));
            const float up = pow2f(sh);
            uint32_t* hi = reinterpret_cast<uint32_t*>(&s_q[row / RT][col][lane * QE]);
            uint32_t* lo = reinterpret_cast<uint32_t*>(&s_q[row / RT][(col + 4) & 7][lane * QE]);
#pragma unroll
            for (int e = 0; e < QE; e += 2) {
                hi[e / 2] = pack_h2(qf[e] * up, qf[e + 1] * up);
                if (TERMS == 2) lo[e / 2] = pack_h2(split_lo(qf[e] * up), split_lo(qf[e + 1] * up));
            }
            if (lane == 0) s_rf[row / RT][col] = pow2f(-sh) * p.scale_log2;
        }
        __syncthreads();
        // column g's fragment: dims 64 c + 16 tig + 4 w + {0, 1} and {2, 3} are k-step 4 c + w's columns
        // 2 tig + {0, 1} and + 8
        uint32_t bq[KS][2];
#pragma unroll
        for (int c = 0; c < KL; ++c)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const uint4 q = *reinterpret_cast<const uint4*>(&s_q[hh][g][c * 64 + tig * 16 + w * 8]);
                bq[4 * c + 2 * w][0] = q.x;
                bq[4 * c + 2 * w][1] = q.y;
                bq[4 * c + 2 * w + 1][0] = q.z;
                bq[4 * c + 2 * w + 1][1] = q.w;
            }
        float rf[2];  // of columns 2 tig, 2 tig + 1: query shift undone, score scale, log2(e)
        int pos[2];
        const int c0 = TERMS == 2 ? 2 * (tig & 1) : 2 * tig;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            rf[h] = s_rf[hh][c0 + h];
            pos[h] = c0 + h < n_rows ? r.start + (rtile * RT + c0 + h) / p.gq : -1;
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
        float unit = 0.0f;  // the value scale that o is in units of
        for (int tile = now.ta + warp / hg; tile < now.tb; tile += per_head) {
            const int t = now.lo + tile * kKv8Group, st = n_used % S::kStages;
            const unsigned char* box_k = mine_ring + st * S::kStage;
            const unsigned char* box_v = box_k + S::kHalves * S::kBox;
            mbar_wait_unless(&s_full[warp][st], (n_used / S::kStages) & 1, p.s.err, kKv8ErrWait);
            __syncwarp();  // (lanes may leave the wait one by one; the matrix instructions take the warp together)
            const float4 group = s_group[warp][st];
            const float ks_now = group.x, vs_now = group.y;
            const bool bad = __float_as_int(group.z) < 0;
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
            ++n_used;
            __syncwarp();
            issue();  // (what parts the warp here and in the masks meets again at the maxima's shuffles)
            // what stands behind the last token or before the window has no part in the sums
            if (t + kKv8Group > r.cap || bad || (p.window > 0 && t <= pos_lo - p.window)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int at = t + token(2 * tig + (j & 1)) + (j >> 1) * 8;
                    if (bad || at >= r.cap || (p.window > 0 && at <= pos_lo - p.window))
#pragma unroll
                        for (int c = 0; c < VW; ++c) vq[j][c] = 0u;
                }
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
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[e] *= kLift;  // (the sums l are of the weights as they are)
            if (TERMS == 2 && tig >= 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[e] = split_lo(sc[e]);
            const uint32_t b0 = transpose8(pack_h2(sc[0], sc[1])), b1 = transpose8(pack_h2(sc[2], sc[3]));
            // o is kept in units of the largest value scale so far, and at the running maxima: both seldom change, and
            // then the products go straight into it.  A page of a smaller scale is added in fp32, so no
            // probability is rounded at another scale than its own.
            const bool larger = vs_now > unit;
            if (__any_sync(0xffffffffu, larger || rescale[0] != 1.0f || rescale[1] != 1.0f)) {
                const float f = larger ? __fdividef(unit, vs_now) : 1.0f;
                const float f0 = f * rescale[0], f1 = f * rescale[1];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    o[mt][0] *= f0;
                    o[mt][1] *= f1;
                    o[mt][2] *= f0;
                    o[mt][3] *= f1;
                }
                unit = larger ? vs_now : unit;
            }
            const bool same = vs_now == unit;
            const float ratio = unit > 0.0f ? __fdividef(vs_now, unit) : 0.0f;
            // values: word c of fragment columns 2 tig, 2 tig + 1 (a, b) and + 8 (cc, d) makes m-tiles 2 c and 2 c + 1,
            // whose rows g and g + 8 are dims 4 c' + {0, 1} and {2, 3} of this lane's piece
            auto products = [&](auto direct) {
#pragma unroll
                for (int c = 0; c < VW; ++c) {
                    const uint32_t ab01 = __byte_perm(vq[0][c], vq[1][c], 0x5140), ab23 = __byte_perm(vq[0][c], vq[1][c], 0x7362);
                    const uint32_t cd01 = __byte_perm(vq[2][c], vq[3][c], 0x5140), cd23 = __byte_perm(vq[2][c], vq[3][c], 0x7362);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        uint32_t a[4];
                        codes_to_half<FMT>(e ? ab23 : ab01, a[0], a[1]);
                        codes_to_half<FMT>(e ? cd23 : cd01, a[2], a[3]);
                        float(&om)[4] = o[2 * c + e];
                        if constexpr (decltype(direct)::value) {
                            mma_16816(om, a, b0, b1);
                        } else {
                            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                            mma_16816(acc, a, b0, b1);
#pragma unroll
                            for (int x = 0; x < 4; ++x) om[x] = fmaf(acc[x], ratio, om[x]);
                        }
                    }
                }
            };
            if (same) products(std::true_type{});
            else products(std::false_type{});
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
                s_o[warp][2 * tig + (e & 1)][dim] = o[mt][e] * (1.0f / kLift) * unit;
            }
        __syncthreads();
        // the next piece's queries are on their way while this one's results are joined
        Piece next = now;
        const bool more_left = next.u < u1 && open(next);
        if (more_left) ask(next, warp, qf);
        const bool complete = now.cta0 == now.cta1;
        constexpr int PART = 64 * PITCH;  // [head of the item][row]
        float* part = p.s.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == now.cta0 ? 1 : 0)) * PART;
        const int n_out = hg * n_rows;
        for (int k = warp; k < n_out; k += W) {  // a row's weights: lane i has the i-th warp's of its head
            const int h = k / n_rows, col = k - h * n_rows;
            const float wm = lane < per_head ? s_m[h + hg * lane][col] : -INFINITY, wl = lane < per_head ? s_l[h + hg * lane][col] : 0.0f;
            const float top = warp_max(wm), f = ex2(wm - (top == -INFINITY ? 0.0f : top));
            float sum = f * wl;
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
            if (lane < per_head) s_weight[h + hg * lane][col] = f;
            if (lane == 0) {
                s_top[h][col] = top;
                s_sum[h][col] = sum;
            }
        }
        __syncthreads();
        auto write = [&](int h, int col, int d, const float4& v, float top, float sum) {
            const int rr = rtile * RT + col, qh = (head + h) * p.gq + rr % p.gq;
            const size_t row = (size_t)(r.row0 + rr / p.gq);
            store_result<T>(p, row, qh, d, v.x, sum);
            store_result<T>(p, row, qh, d + 1, v.y, sum);
            store_result<T>(p, row, qh, d + 2, v.z, sum);
            store_result<T>(p, row, qh, d + 3, v.w, sum);
            if (d == 0) store_lse(p, row, qh, top, sum);
        };
        for (int e = tid; e < n_out * (HD / 4); e += S::kThreads) {
            const int k = e / (HD / 4), d = (e - k * (HD / 4)) * 4, h = k / n_rows, col = k - h * n_rows;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (int i = 0; i < per_head; ++i) {
                const int w = h + hg * i;
                const float f = s_weight[w][col];
                float4 v = *reinterpret_cast<const float4*>(&s_o[w][col][d]);
                if (TERMS == 2) {
                    const float4 lo = *reinterpret_cast<const float4*>(&s_o[w][col + 4][d]);
                    v = make_float4(v.x + lo.x, v.y + lo.y, v.z + lo.z, v.w + lo.w);
                }
                acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
            }
            if (complete) {
                write(h, col, d, acc, s_top[h][col], s_sum[h][col]);
            } else {
                float* to = part + (h * 8 + col) * PITCH;
                __stcg(reinterpret_cast<float4*>(to + d), acc);
                if (d == 0) __stcg(reinterpret_cast<float2*>(to + HD), make_float2(s_top[h][col], s_sum[h][col]));
            }
        }
        if (!complete) {  // the last CTA to arrive joins the parts in CTA order
            __syncthreads();
            if (tid == 0) s_last = arrive(p.s.ctr + now.cta0) == now.cta1 - now.cta0;
            __syncthreads();
            if (s_last) {
                const int parts = now.cta1 - now.cta0 + 1;
                auto part_of = [&](int k) { return p.s.part + (size_t)(2 * (now.cta0 + k) + (k == 0 ? 1 : 0)) * PART; };
                // With few rows, groups of threads take every split-th part, so that one trip to L2 (about a
                // microsecond for what another SM wrote) brings most of them; their sums meet in shared memory.
                constexpr int B = 8;  // parts in flight
                const int work = n_out * (HD / 4), split = max(1, min(per_head, S::kThreads / work));
                const int lanes = split > 1 ? work : S::kThreads, group = split > 1 ? tid / work : 0;
                auto s_j = reinterpret_cast<float (*)[PITCH]>(s_o);  // [group][row], tops and sums behind the values
                for (int e = tid - group * lanes; group < split && e < work; e += lanes) {
                    const int k = e / (HD / 4), d = (e - k * (HD / 4)) * 4, h = k / n_rows, col = k - h * n_rows;
                    float top = -INFINITY, sum = 0.0f;
                    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int k0 = group; k0 < parts; k0 += B * split) {
                        float pm[B], pl[B];
                        float4 pv[B];
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const int at = k0 + i * split;
                            pm[i] = -INFINITY;
                            pl[i] = 0.0f;
                            pv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (at < parts) {
                                const float* from = part_of(at) + (h * 8 + col) * PITCH;
                                const float2 ml = __ldcg(reinterpret_cast<const float2*>(from + HD));
                                pv[i] = __ldcg(reinterpret_cast<const float4*>(from + d));
                                pm[i] = ml.x;
                                pl[i] = ml.y;
                            }
                        }
                        const float before = top;
#pragma unroll
                        for (int i = 0; i < B; ++i) top = fmaxf(top, pm[i]);
                        const float ref = top == -INFINITY ? 0.0f : top;
                        const float f0 = ex2(before - ref);
                        sum *= f0;
                        acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
#pragma unroll
                        for (int i = 0; i < B; ++i) {
                            const float f = ex2(pm[i] - ref);
                            sum = fmaf(f, pl[i], sum);
                            acc = make_float4(fmaf(f, pv[i].x, acc.x), fmaf(f, pv[i].y, acc.y), fmaf(f, pv[i].z, acc.z), fmaf(f, pv[i].w, acc.w));
                        }
                    }
                    if (split == 1) {
                        write(h, col, d, acc, top, sum);
                    } else {
                        *reinterpret_cast<float4*>(&s_j[group * n_out + k][d]) = acc;
                        if (d == 0) *reinterpret_cast<float2*>(&s_j[group * n_out + k][HD]) = make_float2(top, sum);
                    }
                }
                if (split > 1) {
                    __syncthreads();
                    for (int e = tid; e < work; e += S::kThreads) {
                        const int k = e / (HD / 4), d = (e - k * (HD / 4)) * 4, h = k / n_rows, col = k - h * n_rows;
                        float top = -INFINITY, sum = 0.0f;
                        float4 out = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        for (int i = 0; i < split; ++i) top = fmaxf(top, s_j[i * n_out + k][HD]);
                        const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
                        for (int i = 0; i < split; ++i) {
                            const float2 ml = *reinterpret_cast<const float2*>(&s_j[i * n_out + k][HD]);
                            const float4 v = *reinterpret_cast<const float4*>(&s_j[i * n_out + k][d]);
                            const float f = ex2(ml.x - ref);
                            sum = fmaf(f, ml.y, sum);
                            out = make_float4(fmaf(f, v.x, out.x), fmaf(f, v.y, out.y), fmaf(f, v.z, out.z), fmaf(f, v.w, out.w));
                        }
                        write(h, col, d, out, top, sum);
                    }
                }
                if (tid == 0) p.s.ctr[now.cta0] = 0;  // ready for the next call
            }
        }
        // (the next piece's queries pass a barrier before anything of this one's is overwritten)
        now = next;
        left = more_left;
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
    constexpr size_t smem = Shape<HD>::kSmem;
    auto kern = kv8_decode_kernel<T, FMT, HD, sizeof(T) == 4 ? 2 : 1>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
    CUtensorMap mk, mv;
    int rc = make_map<HD>(&mk, a.c.k, a.c);
    if (rc == IAM_OK) rc = make_map<HD>(&mv, a.c.v, a.c);
    if (rc) return rc;
    // KV heads of an item: more than one only where (sequence, head) pairs outnumber the SMs
    int hg = 1;
    while (hg < Shape<HD>::kHeads && a.c.n_kv_heads % (2 * hg) == 0 && (long long)a.c.n_seqs * (a.c.n_kv_heads / hg) > a.sms) hg *= 2;
    kern<<<a.sms, Shape<HD>::kThreads, smem, s>>>(a, hg, mk, mv);
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
size_t kv8_decode_part_floats(int head_dim, int sms) { return (size_t)2 * sms * 64 * (head_dim + 4); }

int kv8_decode_launch(const Kv8Attn& a, int dtype, cudaStream_t s) {
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        return a.c.format == IAM_KV8_INT8 ? launch_dim<T, IAM_KV8_INT8>(a, s) : launch_dim<T, IAM_KV8_E4M3>(a, s);
    });
}

}  // namespace iam
