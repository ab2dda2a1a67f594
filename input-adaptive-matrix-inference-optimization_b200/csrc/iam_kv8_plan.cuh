// iam_kv8_plan.cuh -- how the attention of many query rows is shared out: every (sequence, tile of ROWS rows of a KV
// head's group) has as many units as it sees tiles of TILE tokens; the units of all KV heads and row tiles lie on a line
// that is cut into equal runs, one per CTA.
#pragma once

#include <climits>

#include "iam_kv8.cuh"

namespace iam {
namespace {

constexpr int kPlanThreads = 1024;

// Words of the schedule: the number of row tiles; then, of each, its sequence, its number within the
// sequence, and the units of tokens before it (one more entry: all units).
struct Plan {
    int* words;
    IAM_DEV int& items() const { return words[0]; }
    IAM_DEV int* seq() const { return words + 1; }
    IAM_DEV int* rtile() const { return words + 1 + kKv8MaxItems; }
    IAM_DEV int* unit() const { return words + 1 + 2 * kKv8MaxItems; }
};

struct RowItem {
    int lo, nt, pos_lo, pos_hi, n_rows;  // first token of the first unit (a multiple of TILE), units, first and last position
    int first;                           // first token that a row sees: pages wholly before it are not looked up
};

template <int ROWS, int TILE>
IAM_DEV RowItem item_of(const Kv8Attn& p, const SeqRows& r, int rtile) {
    RowItem it;
    it.n_rows = min(ROWS, r.n * p.gq - rtile * ROWS);
    it.pos_lo = r.start + rtile * ROWS / p.gq;
    it.pos_hi = r.start + (rtile * ROWS + it.n_rows - 1) / p.gq;
    it.first = p.window > 0 ? max(0, it.pos_lo - p.window + 1) : 0;
    it.lo = it.first & ~(TILE - 1);
    const int hi = min(it.pos_hi + 1, r.cap);
    it.nt = max(1, (hi - it.lo + TILE - 1) / TILE);
    return it;
}

IAM_DEV int block_scan(int v, int* s_warp, int& total) {  // exclusive
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
    }
    __syncthreads();  // (s_warp of an earlier call is consumed)
    if (lane == 31) s_warp[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int w = s_warp[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += up;
        }
        s_warp[lane] = w;
    }
    __syncthreads();
    total = s_warp[kPlanThreads / 32 - 1];
    return sum - v + (warp ? s_warp[warp - 1] : 0);
}

// The row tiles of the call in order, and how many units of tokens stand before each.
template <int ROWS, int TILE>
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(Kv8Attn p) {
    __shared__ int s_warp[32];
    const Plan plan{p.s.plan};
    const int tid = threadIdx.x;
    int items = 0, total;
    for (int i0 = 0; i0 < p.c.n_seqs; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int n = 0;
        if (i < p.c.n_seqs) n = (seq_rows(p.c, p.cu, p.lens, p.n_rows, i, p.s.err).n * p.gq + ROWS - 1) / ROWS;
        const int at = items + block_scan(n, s_warp, total);
        for (int k = 0; k < n && at + k < kKv8MaxItems; ++k) {
            plan.seq()[at + k] = i;
            plan.rtile()[at + k] = k;
        }
        items = min(items + total, kKv8MaxItems);  // (more only when the row offsets do not ascend)
    }
    __syncthreads();
    long long units = 0;
    for (int i0 = 0; i0 < items; i0 += kPlanThreads) {
        const int i = i0 + tid;
        int n = 0;
        if (i < items) {
            const int seq = plan.seq()[i];
            n = item_of<ROWS, TILE>(p, seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, nullptr), plan.rtile()[i]).nt;
        }
        const long long at = units + block_scan(n, s_warp, total);  // (1024 tiles of at most 2^20 units)
        if (i < items) plan.unit()[i] = (int)min(at, (long long)INT_MAX);
        units += total;
    }
    if (tid == 0) {
        const bool fits = units < INT_MAX;
        if (!fits) atomicOr(p.s.err, kKv8ErrRange);
        plan.unit()[fits ? items : 0] = fits ? (int)units : 0;
        plan.items() = fits ? items : 0;
    }
}

// The last row tile whose first unit is at most `want`: 32 probes a round, by a whole warp.
IAM_DEV int find_item(const Plan& plan, int items, int want) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = items;  // unit[lo] <= want < unit[hi]
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int at = min(lo + lane * step, hi);
        const unsigned le = __ballot_sync(0xffffffffu, at < hi && plan.unit()[at] <= want);
        const int last = 31 - __clz(le);  // lane 0 always holds
        hi = min(hi, lo + (last + 1) * step);
        lo = lo + last * step;
    }
    return lo;
}

}  // namespace
}  // namespace iam
