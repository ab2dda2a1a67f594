// iam_kv8_prompt.cu -- attention of prompts over the 8-bit paged cache on the tcgen05 tensor cores (fp16 and bf16
// queries, head_dim 64 and 128).
//
// A CTA holds two tiles of 128 query rows and walks the tokens 64 at a time.  Scores S = Q K^T and values O += P V are
// tcgen05.mma (fp16 products, fp32 sums; in tensor memory, for each row tile, S, two tiles of probabilities as left
// operands, and O: 512 columns).  No product is written over what another one in flight may read: the tensor cores
// keep the order of products of one shape only.  S of the next tokens is computed as soon as the softmax has this
// one's in registers.  The codes become fp16 in shared memory once for both row tiles.  By warp:
//   0..3, 4..7   softmax of row tile 0, 1: a thread owns a row, so maxima and sums need no exchange
//   8..11        codes to fp16: keys as they lie, values turned so that a dim's tokens are adjacent (both operands
//                are then K-major with the 128-byte swizzle)
//   12           the MMAs, issued by one thread: while one row tile's probabilities are made, the other's products run
//   13           the copies (TMA, 16 rows a box, so any page size)
// 128 x 128 rows and tokens cost the tensor cores 512 cycles for S and as many for P V (head_dim 128), and their 16384
// powers cost the special-function units 1024: the two are level, and neither can wait for the other.  2048 rows on 8192
// earlier tokens (32 heads of 128 over 8): 497 us, 623 TFLOP/s (queries and results moved 2 bytes at a time: 606); 2 x 141 rows
// on 222 tokens 85, nearly all of it start and join.  Bound by the softmax's chain from one tile's scores to its
// probabilities, some 3200 cycles for 256 x 64; the mma.sync kernel for rows took 2001.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "iam_kv8_plan.cuh"
#include "iam_tc.cuh"

namespace iam {
namespace {

constexpr int kQ = 128;            // rows of a tile: the MMA's M
constexpr int kRows = 2 * kQ;
constexpr int kTile = 64;          // tokens of a unit
constexpr int kGroups = kTile / kKv8Group;
constexpr int kMinUnits = 8;       // units of a CTA at least, while there are enough: a context in few parts is joined faster
constexpr int kThreads = 16 * 32;  // (warps 14 and 15 only complete the last four)
constexpr int kInfo = 8;           // tiles whose scales are kept: the softmax may be four behind the copies
constexpr int kLiftLog = 7;        // probabilities (at most 2^kLag) are lifted by 2^kLiftLog before they are rounded to fp16
constexpr float kLag = 8.0f;       // a row's reference is raised when its maximum outgrows it by more than this (log2)

template <int HD>
struct Smem {
    static constexpr int kQBytes = kQ * HD * 2;
    static constexpr int kCodes = kTile * HD;           // K or V codes of a tile
    static constexpr int kHalf = kTile * HD * 2;        // the same in fp16
    static constexpr int q = 0;                         // [2] row tiles
    static constexpr int k16 = 2 * kQBytes;
    static constexpr int v16 = k16 + 2 * kHalf;         // two of each
    static constexpr int raw = v16 + 2 * kHalf;         // [2] stages of K, V codes
    static constexpr int total = raw + 4 * kCodes;
    static constexpr size_t bytes = total + 1024;
    static_assert(bytes + 2048 <= 227 * 1024, "shared memory per CTA");
};

// D[tmem] (+)= A[tmem] * B[smem]^T
IAM_DEV void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
        : "memory");
}
// 32 consecutive columns of this thread's lane.
IAM_DEV void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// Ends the wait for tmem_ld32; the registers pass through it so that no use is scheduled before.
IAM_DEV void tmem_ld_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])::"memory");
}
IAM_DEV void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(
            r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// True in one lane of a converged warp, always the same one.  (What the elected lane hands to tcgen05 has to be the same
// in the whole warp, and known to be: a value that the compiler must first move there costs each instruction some
// 100 cycles.)
IAM_DEV bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0u;
}
IAM_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
IAM_DEV uint32_t cvt_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// A CTA's share of an item, as every role sees it.
struct Share {
    int item, head;
    SeqRows r;
    RowItem it;
    int seq, rtile, tile, n_tiles, t_first;
    long long item0, item1;
};

template <class T, int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1)
    kv8_prompt_kernel(const Kv8Attn p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using M = Smem<HD>;
    constexpr int PITCH = HD + 4;
    extern __shared__ unsigned char s_raw[];
    // [2] of the first six by tile, of the others by row tile.  No barrier may complete two phases before its waiter has
    // looked, nor lag one behind: a row tile's next probabilities can be ready before this one's are waited for, and its sums are
    // waited for seldom, when the products of the tile before may not be in yet (the other row tile's come first), hence two
    // barriers each, taken in turn.
    __shared__ __align__(8) uint64_t b_raw_full[2], b_raw_free[2], b_k_ready[2], b_k_free[2], b_v_ready[2], b_v_free[2], b_q_ready[2],
        b_s_ready[2], b_s_free[2], b_p_ready[2][2], b_o_done[2][2];
    __shared__ float4 s_info[kInfo][kGroups];  // key scale, value scale, 1 if the page is one of the cache's, log2 of the value scale
    __shared__ uint32_t s_tmem;
    __shared__ int s_last;
    unsigned char* smem = s_raw + ((1024u - (smem_u32(s_raw) & 1023u)) & 1023u);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int plog = 31 - __clz(p.c.page_size), kvh = p.c.n_kv_heads;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&b_raw_full[i], kGroups);
            mbar_init(&b_raw_free[i], 4);
            mbar_init(&b_q_ready[i], 4);
            mbar_init(&b_s_ready[i], 1);
            mbar_init(&b_s_free[i], 4);
            mbar_init(&b_p_ready[i][0], 4);
            mbar_init(&b_p_ready[i][1], 4);
            mbar_init(&b_o_done[i][0], 1);
            mbar_init(&b_o_done[i][1], 1);
            mbar_init(&b_k_ready[i], 4);
            mbar_init(&b_k_free[i], 1);
            mbar_init(&b_v_ready[i], 4);
            mbar_init(&b_v_free[i], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        tmem_alloc(&s_tmem, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // of row tile i: S, the probabilities of the c-th tile that it sees, and O
    auto tm_s = [&](int i) { return tmem + (uint32_t)(i * kTile); };
    auto tm_p = [&](int i, int c) { return tmem + (uint32_t)(2 * kTile + (2 * i + (c & 1)) * (kTile / 2)); };
    auto tm_o = [&](int i) { return tmem + (uint32_t)(4 * kTile + i * HD); };

    const Plan plan{p.s.plan};
    const int items = plan.items();
    const int per_head = plan.unit()[items];
    const long long total = (long long)per_head * kvh;
    const int run = min(kMinUnits, per_head / max(1, items));  // (short contexts: a row tile a CTA)
    const long long ctas = min((long long)gridDim.x, (total + run - 1) / max(1, run));
    const bool idle = (long long)blockIdx.x >= ctas;
    const long long u0 = idle ? 0 : total * blockIdx.x / ctas, u1 = idle ? 0 : total * (blockIdx.x + 1) / ctas;

    Share w;
    w.item = idle ? 0 : find_item(plan, items, (int)(u0 % per_head));
    w.head = idle ? 0 : (int)(u0 / per_head);
    long long u = u0;
    auto open = [&] {  // the share at u
        w.item0 = (long long)w.head * per_head + plan.unit()[w.item];
        w.item1 = (long long)w.head * per_head + plan.unit()[w.item + 1];
        w.seq = plan.seq()[w.item];
        w.rtile = plan.rtile()[w.item];
        w.r = seq_rows(p.c, p.cu, p.lens, p.n_rows, w.seq, nullptr);
        w.it = item_of<kRows, kTile>(p, w.r, w.rtile);
        w.tile = (int)(u - w.item0);
        w.n_tiles = (int)(min(u1, w.item1) - u);
        w.t_first = w.it.lo + w.tile * kTile;
    };
    auto close = [&] {
        u += w.n_tiles;
        if (u == w.item1 && ++w.item == items) {
            w.item = 0;
            ++w.head;
        }
    };
    bool dead = false;  // a wait gave up: the rest is passed through without waiting
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (!dead && !mbar_wait(b, parity & 1u, nullptr)) {
            atomicOr(p.s.err, kKv8ErrWait);
            dead = true;
        }
        __syncwarp();  // (lanes may leave the wait one by one, and what follows it takes the whole warp together)
    };
    auto give = [&](uint64_t* b) {  // one arrival for this warp
        __syncwarp();
        if (lane == 0) mbar_arrive(b);
    };

    // The registers of a block of 16 warps, 128 a thread, go where they are needed: 152 for the softmax, 104 for the
    // conversion and the rest (512 for the four warps that share a scheduler, as at the launch).
    if (warp >= 12) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    else if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");
    if (warp >= 14) {
    } else if (warp == 13) {  // ---- copies: lane g has group g of every tile
        for (int n = 0; u < u1; close()) {
            open();
            const int32_t* table = p.c.block_table + (size_t)w.seq * p.c.max_pages;
            const int from = w.it.first & ~(kKv8Group - 1);  // (pages wholly before the window may be anyone's)
            auto page_of = [&](int j) {
                const int t = w.t_first + j * kTile + lane * kKv8Group;
                return lane < kGroups && j < w.n_tiles && t < w.r.cap && t >= from ? __ldg(table + (t >> plog)) : -1;
            };
            int id = page_of(0);
            for (int j = 0; j < w.n_tiles; ++j, ++n) {
                const int st = n & 1, t = w.t_first + j * kTile + lane * kKv8Group;
                const int id_next = page_of(j + 1);
                wait(&b_raw_free[st], (n >> 1) + 1);
                if (lane < kGroups) {
                    if (t < w.r.cap && t >= from && (id < 0 || id >= p.c.n_pages)) {
                        atomicOr(p.s.err, kKv8ErrRange);
                        id = -1;
                    }
                    const size_t slot = (size_t)id * kvh + w.head;
                    if (id >= 0) {
                        const float vs = __ldg(p.c.v_scale + slot);
                        s_info[n % kInfo][lane] = make_float4(__ldg(p.c.k_scale + slot), vs, 1.0f, __log2f(vs));
                    }
                    else s_info[n % kInfo][lane] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    mbar_expect_tx(&b_raw_full[st], id >= 0 ? 2 * kKv8Group * HD : 0);
                    if (id >= 0) {
                        const int row = (int)((((long long)id * kvh + w.head) << plog) + (t & (p.c.page_size - 1)));
                        unsigned char* to = smem + M::raw + 2 * st * M::kCodes + lane * kKv8Group * HD;
                        tma_load_2d(to, &map_k, 0, row, &b_raw_full[st]);
                        tma_load_2d(to + M::kCodes, &map_v, 0, row, &b_raw_full[st]);
                    }
                }
                id = id_next;
            }
        }
    } else if (warp == 12) {  // ---- products
        constexpr uint32_t kDescS = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kQ >> 4) << 24);
        constexpr uint32_t kDescO = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kQ >> 4) << 24);
        // (descriptors count in 16 bytes; building each anew took the issuing thread longer than the products)
        const uint64_t desc_q = sw128_desc(smem + M::q), desc_k = sw128_desc(smem + M::k16), desc_v = sw128_desc(smem + M::v16);
        int n = 0, piece = 0;  // n: the tile (of all) whose values are next
        int f0 = 0, f1 = 0, n1 = 0, piece1 = 0;  // tiles that left S; values and pieces of the second row tile
        for (; u < u1; close(), ++piece) {
            open();
            const bool two = w.it.n_rows > kQ;
            auto scores = [&](int i, int j) {  // row tile i times the keys of tile j (of all)
                const int half = __shfl_sync(0xffffffffu, j & 1, 0);
                const uint64_t q = desc_q + (uint64_t)(i * (M::kQBytes >> 4)), keys = desc_k + (uint64_t)(half * (M::kHalf >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < HD / 16; ++k)
                        tc_mma(tm_s(i), q + (uint64_t)(((k >> 2) * (kQ * 128) >> 4) + 2 * (k & 3)),
                               keys + (uint64_t)(((k >> 2) * (kTile * 128) >> 4) + 2 * (k & 3)), kDescS, k > 0);
                    tc_commit(&b_s_ready[i]);
                }
            };
            auto values = [&](int i, int c, int j, bool first) {  // its c-th probabilities times the values of tile j
                const int half = __shfl_sync(0xffffffffu, j & 1, 0), place = __shfl_sync(0xffffffffu, c & 1, 0);
                const uint64_t vals = desc_v + (uint64_t)(half * (M::kHalf >> 4));
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kTile / 16; ++k)
                        tc_mma_ts(tm_o(i), tm_p(i, place) + 8 * k, vals + (uint64_t)(2 * k), kDescO, !first || k > 0);
                    tc_commit(&b_o_done[i][place]);
                }
            };
            auto commit = [&](uint64_t* b) {
                if (elect_one()) tc_commit(b);
            };
            wait(&b_q_ready[0], piece);
            if (two) wait(&b_q_ready[1], piece1++);
            wait(&b_k_ready[n & 1], n >> 1);
            tc_fence_after();
            scores(0, n);
            if (two) scores(1, n);
            commit(&b_k_free[n & 1]);
            for (int j = 0; j < w.n_tiles; ++j, ++n) {
                if (j + 1 < w.n_tiles) {  // the next tile's scores, as soon as the softmax has this one's in registers
                    wait(&b_k_ready[(n + 1) & 1], (n + 1) >> 1);
                    wait(&b_s_free[0], f0++);
                    tc_fence_after();
                    scores(0, n + 1);
                    if (two) {
                        wait(&b_s_free[1], f1++);
                        tc_fence_after();
                        scores(1, n + 1);
                    }
                    commit(&b_k_free[(n + 1) & 1]);
                } else {
                    wait(&b_s_free[0], f0++);
                    if (two) wait(&b_s_free[1], f1++);
                }
                wait(&b_v_ready[n & 1], n >> 1);
                wait(&b_p_ready[0][n & 1], n >> 1);
                tc_fence_after();
                values(0, n, n, j == 0);
                if (two) {
                    wait(&b_p_ready[1][n1 & 1], n1 >> 1);
                    tc_fence_after();
                    values(1, n1++, n, j == 0);
                }
                commit(&b_v_free[n & 1]);
            }
            __syncwarp();
        }
    } else if (warp >= 8) {  // ---- codes to fp16
        const int c_tid = tid - 256;
        for (int n = 0; u < u1; close()) {
            open();
            for (int j = 0; j < w.n_tiles; ++j, ++n) {
                const int st = n & 1, t0 = w.t_first + j * kTile;
                const unsigned char* raw_k = smem + M::raw + 2 * st * M::kCodes;
                const unsigned char* raw_v = raw_k + M::kCodes;
                wait(&b_raw_full[st], n >> 1);
                wait(&b_k_free[st], (n >> 1) + 1);
                // keys: 16 codes of a token to 32 bytes of its row; four lanes take half of a token's 128, so that the
                // stores meet no bank twice
                constexpr int PIECES = HD / 16;  // of a token
#pragma unroll
                for (int i = 0; i < kTile * PIECES / 128; ++i) {
                    const int f = i * 128 + c_tid;
                    const int row = PIECES == 8 ? ((f >> 4) << 1 | (f >> 2 & 1)) : f >> 2;
                    const int c = PIECES == 8 ? ((f >> 3 & 1) << 2 | (f & 3)) : f & 3;
                    const uint4 q = *reinterpret_cast<const uint4*>(raw_k + row * HD + c * 16);
                    uint4 a, b;
                    codes_to_half<FMT>(q.x, a.x, a.y);
                    codes_to_half<FMT>(q.y, a.z, a.w);
                    codes_to_half<FMT>(q.z, b.x, b.y);
                    codes_to_half<FMT>(q.w, b.z, b.w);
                    unsigned char* to = smem + M::k16 + st * M::kHalf + (c >> 2) * (kTile * 128) + row * 128;
                    const int piece = (c & 3) * 2;
                    *reinterpret_cast<uint4*>(to + ((piece ^ (row & 7)) << 4)) = a;
                    *reinterpret_cast<uint4*>(to + (((piece + 1) ^ (row & 7)) << 4)) = b;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                give(&b_k_ready[st]);
                wait(&b_v_free[st], (n >> 1) + 1);
                // values: 4 dims of 8 tokens to 4 rows of 16 bytes; lanes take the tokens in turn, so that neither
                // reads nor stores meet a bank twice
                constexpr int WORDS = HD / 4;
                const bool ends = t0 + kTile > w.r.cap || t0 < w.it.first;
                unsigned ok = 0;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) ok |= s_info[n % kInfo][k].z != 0.0f ? 1u << k : 0u;
#pragma unroll
                for (int i = 0; i < WORDS * (kTile / 8) / 128; ++i) {
                    const int f = i * 128 + c_tid;
                    const int word = f % WORDS, t8 = (f / WORDS + (word >> 1)) % (kTile / 8);
                    uint32_t v[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint32_t*>(raw_v + (t8 * 8 + k) * HD + word * 4);
                    if (ends || ok != (1u << kGroups) - 1u)  // what stands behind the last token or before the window has no part in the sums
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const int at = t0 + t8 * 8 + k;
                            if (at >= w.r.cap || at < w.it.first || !(ok >> (t8 >> 1) & 1u)) v[k] = 0u;
                        }
                    uint32_t h[4][4];  // [dim][pair of tokens]
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        codes_to_half<FMT>(__byte_perm(v[2 * k], v[2 * k + 1], 0x5140), h[0][k], h[1][k]);
                        codes_to_half<FMT>(__byte_perm(v[2 * k], v[2 * k + 1], 0x7362), h[2][k], h[3][k]);
                    }
                    unsigned char* to = smem + M::v16 + st * M::kHalf;
#pragma unroll
                    for (int d = 0; d < 4; ++d) {
                        const int row = word * 4 + d;
                        *reinterpret_cast<uint4*>(to + row * 128 + ((t8 ^ (row & 7)) << 4)) = make_uint4(h[d][0], h[d][1], h[d][2], h[d][3]);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                give(&b_v_ready[st]);
                give(&b_raw_free[st]);
            }
        }
    } else {  // ---- softmax
        const int i = warp >> 2;                       // row tile
        const int row = tid & (kQ - 1);                // of the row tile: this thread's lane of tensor memory
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t to = tm_o(i) + lanes;
        int n = 0, ni = 0;  // tiles; tiles that had this row tile
        for (; u < u1; close()) {
            open();
            const int mine = i * kQ + row;
            const bool have = mine < w.it.n_rows;
            const int rr = w.rtile * kRows + mine;
            const size_t q_row = (size_t)(w.r.row0 + rr / p.gq);
            const int q_head = w.head * p.gq + rr % p.gq;
            const bool tile_there = w.it.n_rows > i * kQ;  // of the whole row tile
            float rf = 0.0f;
            if (tile_there) {  // this thread's query, shifted into fp16's range
                const T* src = have ? static_cast<const T*>(p.q.data) + q_row * p.q.token_stride + q_head * p.q.head_stride : nullptr;
                // (16 bytes at a time where the row allows it: as many trips less for the start of a piece)
                const bool wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
                auto eight = [&](int c) { return wide ? load_vec<true, T, 8>(src + c * 8) : load_vec<false, T, 8>(src + c * 8); };
                float amax = 0.0f;
                if (have)
#pragma unroll 8
                    for (int c = 0; c < HD / 8; ++c) {
                        const Vec<T, 8> x = eight(c);
#pragma unroll
                        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(to_f32(x.v[e])));
                    }
                const int sh = query_shift(amax);
                const float up = pow2f(sh);
                rf = pow2f(-sh) * p.scale_log2;
#pragma unroll 2
                for (int c = 0; c < HD / 8; ++c) {
                    float f[8];
                    Vec<T, 8> x;
                    if (have) x = eight(c);
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] = have ? to_f32(x.v[e]) * up : 0.0f;
                    *reinterpret_cast<uint4*>(smem + M::q + i * M::kQBytes + (c >> 3) * (kQ * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4)) =
                        make_uint4(cvt_h2(f[0], f[1]), cvt_h2(f[2], f[3]), cvt_h2(f[4], f[5]), cvt_h2(f[6], f[7]));
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                give(&b_q_ready[i]);
            }
            const int pos = have ? w.r.start + rr / p.gq : -1;
            // positions of the row tile's first and last row
            const int pos_lo = w.r.start + (w.rtile * kRows + i * kQ) / p.gq;
            const int pos_hi = w.r.start + (w.rtile * kRows + min(w.it.n_rows, (i + 1) * kQ) - 1) / p.gq;
            float m = -INFINITY, l = 0.0f, unit = 0.0f;
            if (!tile_there) n += w.n_tiles;
            for (int j = 0; tile_there && j < w.n_tiles; ++j, ++n, ++ni) {
                wait(&b_s_ready[i], ni);
                // (S of this tile was issued after the products of the tile before last: their probabilities' place is free)
                const uint32_t ts = tm_s(i) + lanes, tp = tm_p(i, ni) + lanes;
                tc_fence_after();
                uint32_t s[2][32];  // the row's scores
                tmem_ld32(ts, s[0]);
                tmem_ld32(ts + 32, s[1]);
                const int t0 = w.t_first + j * kTile;
                const float4* info = s_info[n % kInfo];
                bool all_ok = true;
                float vmax = 0.0f, vmin = INFINITY;
#pragma unroll
                for (int k = 0; k < kGroups; ++k) {
                    all_ok = all_ok && info[k].z != 0.0f;
                    vmax = fmaxf(vmax, info[k].y);
                    vmin = fminf(vmin, info[k].y);
                }
                const bool whole = all_ok && t0 + kTile - 1 <= pos_lo && t0 + kTile <= w.r.cap && (p.window == 0 || t0 > pos_hi - p.window);
                auto seen = [&](int t, int k) {
                    return info[k].z != 0.0f && t <= pos && t < w.r.cap && (p.window == 0 || t > pos - p.window);
                };
                const bool grown = vmax > unit;
                const float new_unit = grown ? vmax : unit;
                // The usual tile: every row sees all of it, and the value scales are close enough to go into the
                // exponent (below); both loops are kept free of the other case's work.
                const bool plain = whole && vmin >= new_unit * 0x1p-20f && new_unit > 0.0f;
                const float unit_log = __log2f(new_unit) - kLiftLog;
                tmem_ld_wait(s[0]);
                tmem_ld_wait(s[1]);
                tc_fence_before();
                give(&b_s_free[i]);
                auto tile = [&](auto is_plain) {
                    constexpr bool PLAIN = decltype(is_plain)::value;
                    float mx = -INFINITY;
#pragma unroll
                    for (int k = 0; k < kGroups; ++k) {
                        uint32_t* x = s[k >> 1] + 16 * (k & 1);
                        const float f = fminf(info[k].x * rf, 3.402823466e38f);
                        float gm = -INFINITY;
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            if (!PLAIN) {
                                if (!seen(t0 + 16 * k + e, k)) x[e] = 0xff800000u;
                                if (!seen(t0 + 16 * k + e + 1, k)) x[e + 1] = 0xff800000u;
                            }
                            gm = fmaxf(gm, fmaxf(__uint_as_float(x[e]), __uint_as_float(x[e + 1])));
                        }
                        mx = fmaxf(mx, gm == -INFINITY ? gm : gm * f);
                    }
                    if constexpr (!PLAIN) __syncwarp();  // (the masks may part the warp; nothing behind them does)
                    // The reference follows the maximum with a lag: powers of up to 2^kLag are as exact, and O is
                    // rarely rewritten.  O is in units of the largest value scale so far.
                    const bool raise = mx > m + kLag || (m == -INFINITY && mx > -INFINITY);
                    if (__any_sync(0xffffffffu, raise) || grown) {
                        const float fm = raise ? (m == -INFINITY ? 0.0f : ex2(m - mx)) : 1.0f;
                        const float fo = fm * (grown ? __fdividef(unit, vmax) : 1.0f);
                        l *= fm;
                        m = raise ? mx : m;
                        if (j > 0) {
                            wait(&b_o_done[i][(ni - 1) & 1], (ni - 1) >> 1);  // the products of the tile before are in
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < HD / 16; ++c) {
                                uint32_t x[16];
                                tmem_ld16(to + 16 * c, x);
#pragma unroll
                                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * fo);
                                tmem_st16(to + 16 * c, x);
                            }
                        }
                    }
                    const float ref = m == -INFINITY ? 0.0f : m;
                    // powers, rounded to fp16 with the group's value scale (relative to the unit) and the lift in them; a
                    // plain tile has both in the exponent and takes them out of the sum again
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t h[16];
#pragma unroll
                        for (int k = 2 * c; k < 2 * c + 2; ++k) {
                            const uint32_t* x = s[c] + 16 * (k & 1);
                            const float4 g = info[k];
                            const float f = fminf(g.x * rf, 3.402823466e38f);
                            const float lift = g.w - unit_log, bias = PLAIN ? lift - ref : -ref;
                            const float ratio = PLAIN || new_unit == 0.0f ? 0.0f : __fdividef(g.y, new_unit) * (float)(1 << kLiftLog);
                            float sum[2] = {0.0f, 0.0f};
#pragma unroll
                            for (int e = 0; e < 16; e += 2) {
                                const float xa = __uint_as_float(x[e]), xb = __uint_as_float(x[e + 1]);
                                float a = ex2(fmaf(xa, f, bias)), b = ex2(fmaf(xb, f, bias));
                                if (!PLAIN) {  // (-inf times a scale of 0 is no -inf)
                                    a = xa == -INFINITY ? 0.0f : a;
                                    b = xb == -INFINITY ? 0.0f : b;
                                }
                                sum[0] += a;
                                sum[1] += b;
                                if (!PLAIN) {
                                    a *= ratio;
                                    b *= ratio;
                                }
                                h[8 * (k & 1) + e / 2] = cvt_h2(a, b);
                            }
                            l = fmaf(sum[0] + sum[1], PLAIN ? ex2(-lift) : 1.0f, l);
                        }
                        tmem_st16(tp + 16 * c, h);
                    }
                };
                if (plain) tile(std::true_type{});
                else tile(std::false_type{});
                unit = new_unit;
                tmem_st_wait();
                tc_fence_before();
                give(&b_p_ready[i][ni & 1]);
            }
            // ---- results, or this CTA's part of them
            const bool complete = w.tile == 0 && w.n_tiles == w.item1 - w.item0;
            const int cta0 = (int)(((w.item0 + 1) * ctas - 1) / total), cta1 = (int)((w.item1 * ctas - 1) / total);
            constexpr int PART = kRows * PITCH;
            float* part = p.s.part + (size_t)(2 * blockIdx.x + ((int)blockIdx.x == cta0 ? 1 : 0)) * PART;
            if (tile_there) {
                wait(&b_o_done[i][(ni - 1) & 1], (ni - 1) >> 1);
                tc_fence_after();
                const float scale = unit * (1.0f / (1 << kLiftLog));
                // (decided once for all rows, so that the warp stays together)
                const bool wide = ((reinterpret_cast<uintptr_t>(p.out.data) | (uintptr_t)(p.out.token_stride * (long long)sizeof(T)) |
                                    (uintptr_t)(p.out.head_stride * (long long)sizeof(T))) & 15) == 0;
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) {
                    uint32_t x[32];
                    __syncwarp();  // a row tile's last rows may be none: the load takes all lanes together
                    tmem_ld32(to + 32 * c, x);
                    tmem_ld_wait(x);
                    if (have) {
                        if (complete && wide) {
                            T* const out = static_cast<T*>(p.out.data) + q_row * p.out.token_stride + q_head * p.out.head_stride + 32 * c;
#pragma unroll
                            for (int e = 0; e < 32; e += 8) {
                                Vec<T, 8> v;
#pragma unroll
                                for (int k = 0; k < 8; ++k) v.v[k] = result<T>(__uint_as_float(x[e + k]) * scale, l);
                                store_vec<true>(out + e, v);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 v = make_float4(__uint_as_float(x[e]) * scale, __uint_as_float(x[e + 1]) * scale,
                                                             __uint_as_float(x[e + 2]) * scale, __uint_as_float(x[e + 3]) * scale);
                                if (complete) {
                                    store_result<T>(p, q_row, q_head, 32 * c + e, v.x, l);
                                    store_result<T>(p, q_row, q_head, 32 * c + e + 1, v.y, l);
                                    store_result<T>(p, q_row, q_head, 32 * c + e + 2, v.z, l);
                                    store_result<T>(p, q_row, q_head, 32 * c + e + 3, v.w, l);
                                } else {
                                    __stcg(reinterpret_cast<float4*>(part + mine * PITCH + 32 * c + e), v);
                                }
                            }
                        }
                    }
                }
                if (have) {
                    if (complete) store_lse(p, q_row, q_head, m, l);
                    else __stcg(reinterpret_cast<float2*>(part + mine * PITCH + HD), make_float2(m, l));
                }
                tc_fence_before();
            }
            if (!complete) {  // the last CTA to arrive joins the parts in CTA order
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (tid == 0) s_last = arrive(p.s.ctr + cta0) == cta1 - cta0;
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (s_last) {
                    const int parts = cta1 - cta0 + 1;
                    auto part_of = [&](int k) { return p.s.part + (size_t)(2 * (cta0 + k) + (k == 0 ? 1 : 0)) * PART; };
                    for (int r0 = warp; r0 < w.it.n_rows; r0 += 8) {
                        float top = -INFINITY, sum = 0.0f, acc[HD / 32];
#pragma unroll
                        for (int e = 0; e < HD / 32; ++e) acc[e] = 0.0f;
#pragma unroll 4
                        for (int k = 0; k < parts; ++k) {
                            const float* from = part_of(k) + r0 * PITCH;
                            const float2 ml = __ldcg(reinterpret_cast<const float2*>(from + HD));
                            const float now = fmaxf(top, ml.x), ref = now == -INFINITY ? 0.0f : now;
                            const float f0 = ex2(top - ref), f1 = ex2(ml.x - ref);
                            sum = sum * f0 + ml.y * f1;
#pragma unroll
                            for (int e = 0; e < HD / 32; ++e) acc[e] = acc[e] * f0 + __ldcg(from + e * 32 + lane) * f1;
                            top = now;
                        }
                        const int ri = w.rtile * kRows + r0, qh = w.head * p.gq + ri % p.gq;
                        const size_t qr = (size_t)(w.r.row0 + ri / p.gq);
#pragma unroll
                        for (int e = 0; e < HD / 32; ++e) store_result<T>(p, qr, qh, e * 32 + lane, acc[e], sum);
                        if (lane == 0) store_lse(p, qr, qh, top, sum);
                    }
                    if (tid == 0) p.s.ctr[cta0] = 0;  // ready for the next call
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");  // s_last is read by all
            }
        }
    }
    __syncthreads();
    if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int HD>
int make_map(CUtensorMap* map, const void* codes, const iam_kv8_cache& c) {
    auto fn = tensor_map_encoder();
    if (fn == nullptr) return fail(IAM_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {HD, (cuuint64_t)c.n_pages * c.n_kv_heads * c.page_size};
    const cuuint64_t strides[1] = {HD};
    const cuuint32_t box[2] = {HD, kKv8Group};
    const cuuint32_t estr[2] = {1u, 1u};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(IAM_ERR_CUDA, "kv8: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return IAM_OK;
}

template <class T, int FMT, int HD>
int launch(const Kv8Attn& a, cudaStream_t s) {
    constexpr size_t smem = Smem<HD>::bytes;
    auto kern = kv8_prompt_kernel<T, FMT, HD>;
    static std::atomic<unsigned long long> done{0};
    IAM_CUDA_TRY(once_per_device(done, [&] { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); }));
    CUtensorMap mk, mv;
    int rc = make_map<HD>(&mk, a.c.k, a.c);
    if (rc == IAM_OK) rc = make_map<HD>(&mv, a.c.v, a.c);
    if (rc) return rc;
    plan_kernel<kRows, kTile><<<1, kPlanThreads, 0, s>>>(a);
    IAM_CUDA_TRY(cudaGetLastError());
    kern<<<a.sms, kThreads, smem, s>>>(a, mk, mv);
    IAM_CUDA_TRY(cudaGetLastError());
    return IAM_OK;
}

template <class T, int FMT>
int launch_dim(const Kv8Attn& a, cudaStream_t s) {
    return a.c.head_dim == 64 ? launch<T, FMT, 64>(a, s) : launch<T, FMT, 128>(a, s);
}

}  // namespace

size_t kv8_prompt_part_floats(int head_dim, int sms) { return head_dim > 128 ? 0 : (size_t)2 * sms * kRows * (head_dim + 4); }

int kv8_prompt_launch(const Kv8Attn& a, int dtype, cudaStream_t s) {
    if (dtype == IAM_BF16) return a.c.format == IAM_KV8_INT8 ? launch_dim<__nv_bfloat16, IAM_KV8_INT8>(a, s) : launch_dim<__nv_bfloat16, IAM_KV8_E4M3>(a, s);
    return a.c.format == IAM_KV8_INT8 ? launch_dim<__half, IAM_KV8_INT8>(a, s) : launch_dim<__half, IAM_KV8_E4M3>(a, s);
}

}  // namespace iam
