// iam_kv8.cu -- the 8-bit paged KV cache: its handle, the append and the entry points of the attention.
// (The reference's cache is fp32, one buffer per layer, model.hpp:97-98, attention.hpp:281-309.)
#include <algorithm>
#include <cmath>
#include <new>
#include <type_traits>

#include "iam_kv8.cuh"

namespace iam {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kFewRows = 16;     // rows a sequence, on average, up to which a warp does what a block does else
constexpr int kAppendKeep = 4;  // 16-byte accesses of the new values that a thread keeps between the two passes

template <int FMT>
constexpr float code_top() { return FMT == IAM_KV8_INT8 ? 127.0f : 448.0f; }

// Exponent of the smallest power of two >= 2^-126 that brings amax (finite, not negative) within the
// largest code: 127 = 1.984375 * 2^6, 448 = 1.75 * 2^8, so it follows from amax's exponent and one
// comparison of its mantissa.
template <int FMT>
IAM_DEV int scale_exponent(float amax) {
    const int bits = __float_as_int(amax);
    const int e = (bits >> 23) - 127, m = bits & 0x7fffff;
    constexpr int kTopE = FMT == IAM_KV8_INT8 ? 6 : 8, kTopM = FMT == IAM_KV8_INT8 ? 0x7e0000 : 0x600000;
    const int s = e - kTopE + (m > kTopM ? 1 : 0);
    return (bits >> 23) == 0 ? -126 : max(-126, s);
}

// A value times the reciprocal of the scale to its code: to nearest, ties to even; infinities become the
// largest code and NaN 0.
template <int FMT>
IAM_DEV uint32_t encode(float x) {
    x = x != x ? 0.0f : fminf(fmaxf(x, -code_top<FMT>()), code_top<FMT>());
    if constexpr (FMT == IAM_KV8_INT8) {
        return (uint32_t)__float2int_rn(x) & 0xffu;
    } else {
        uint16_t r;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(x));
        return r & 0xffu;
    }
}
// Four of them, the first in the lowest byte.
template <int FMT>
IAM_DEV uint32_t encode4(float a, float b, float c, float d) {
    if constexpr (FMT == IAM_KV8_INT8) {
        return encode<FMT>(a) | encode<FMT>(b) << 8 | encode<FMT>(c) << 16 | encode<FMT>(d) << 24;
    } else {  // (the conversion itself saturates)
        a = a == a ? a : 0.0f;
        b = b == b ? b : 0.0f;
        c = c == c ? c : 0.0f;
        d = d == d ? d : 0.0f;
        uint32_t r;
        asm("{\n.reg .b16 l, h;\ncvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\nmov.b32 %0, {l, h};\n}"
            : "=r"(r)
            : "f"(a), "f"(b), "f"(c), "f"(d));
        return r;
    }
}
template <int FMT>
IAM_DEV float decode_code(uint32_t b) {
    if constexpr (FMT == IAM_KV8_INT8) return (float)(int8_t)b;
    uint32_t h;
    asm("{\n.reg .b16 a;\ncvt.u16.u32 a, %1;\ncvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(h) : "r"(b));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

struct AppendParams {
    iam_kv8_cache c;
    iam_rows x[2];
    const int32_t* cu;
    const int32_t* lens;
    int n_rows;
    unsigned* err;
};

// The pages that the call touches are numbered without knowing the lengths on the host: a sequence of
// n rows touches at most n / page + 2 pages (1 when n is 1), and cu[i] / page + 2 i is below the sum
// of that over the sequences before it, so slot w belongs to the last sequence whose base is <= w.
IAM_DEV int slot_base(int cu, int i, int page_log2) { return (cu >> page_log2) + 2 * i; }

// NT threads (a block, or one warp of it) per (touched page, KV head, K or V), the only ones that write that page and
// head: pass 1 finds the largest new value, they agree on the scale, pass 2 rounds (and, when the scale grew,
// shifts the codes that the page held).  Bound by bytes for prompts (the values are read once and kept
// in registers up to kAppendKeep accesses a thread; of a 64-token page of fp32, half is read twice), by the chain of dependent
// loads for single tokens.  15000 tokens of 8 heads of 128, bf16 to e4m3 (91 MB): 27.7 us, 3.3 TB/s, with 68 % of the issue slots
// busy (with the KV heads of a page apart and single conversions 57); fp32 (152 MB): 46 us; 64 sequences of one token: 3.1 us.
template <class T, int FMT, bool WIDE, int NT>
__global__ void __launch_bounds__(kAppendThreads, 4) kv8_append_kernel(AppendParams p) {
    constexpr int VEC = WIDE ? 16 / (int)sizeof(T) : 4;
    using V = Vec<T, VEC>;
    __shared__ float s_max[NT / 32];
    const int tid = threadIdx.x % NT, lane = tid & 31, warp = tid >> 5;
    // the KV heads of a page side by side, so that blocks at work together read whole token rows
    constexpr int ABREAST = kAppendThreads / NT;
    const int lots = 2 * p.c.n_kv_heads, per_slot = (lots + ABREAST - 1) / ABREAST, slot_no = blockIdx.x / per_slot;
    const int lot = (blockIdx.x - slot_no * per_slot) * ABREAST + threadIdx.x / NT, head = lot >> 1, which = lot & 1;
    const int page = p.c.page_size, plog = 31 - __clz(page), hd = p.c.head_dim;
    int seq = slot_no, nth = 0;
    if (p.cu) {  // the last sequence whose base is at most this slot: a probe a thread and round
        int lo = 0, hi = p.c.n_seqs;
        while (hi - lo > 1) {
            const int step = (hi - lo + kAppendThreads - 1) / kAppendThreads, at = lo + threadIdx.x * step;
            const int below = __syncthreads_count(at < hi && slot_base(p.cu[at], at, plog) <= slot_no);
            if (below == 0) return;  // (offsets that do not start at 0)
            hi = min(hi, lo + below * step);
            lo += (below - 1) * step;
        }
        seq = lo;
        nth = slot_no - slot_base(p.cu[seq], seq, plog);
        if (nth < 0) return;  // (offsets that do not ascend)
    }
    if (lot >= lots) return;  // (no barrier of the block behind this with several lots)
    const SeqRows r = seq_rows(p.c, p.cu, p.lens, p.n_rows, seq, p.err);
    const int first = max(r.start, 0);  // tokens before position 0 are skipped
    const long long page_at = (long long)(first / page + nth) * page;  // the page's first token
    if (r.n == 0 || page_at >= r.cap) return;  // (tokens behind the table are flagged by seq_rows)
    const int index = first / page + nth;
    const int lo = max(first, (int)page_at), hi = min(r.len, (int)page_at + page);
    if (lo >= hi) return;
    // the new values are asked for first; the page they go to is looked up meanwhile
    const iam_rows rows = which ? p.x[1] : p.x[0];
    const T* x = static_cast<const T*>(rows.data) + (size_t)(r.row0 + lo - r.start) * rows.token_stride + head * rows.head_stride;
    const int row_log = 31 - __clz(hd / VEC), n_vec = (hi - lo) << row_log;  // (head_dim is a power of two)
    V keep[kAppendKeep];
    auto load = [&](int f) {
        const int row = f >> row_log, c = f - (row << row_log);
        return load_vec<WIDE, T, VEC>(x + (size_t)row * rows.token_stride + c * VEC);
    };
#pragma unroll
    for (int k = 0; k < kAppendKeep; ++k) {
        const int f = tid + k * NT;
        if (f < n_vec) keep[k] = load(f);
    }
    const int id = p.c.block_table[(size_t)seq * p.c.max_pages + index];
    if (id < 0 || id >= p.c.n_pages) {
        if (tid == 0) atomicOr(p.err, kKv8ErrRange);
        return;
    }
    const size_t slot = (size_t)id * p.c.n_kv_heads + head;
    uint8_t* codes = static_cast<uint8_t*>(which ? p.c.v : p.c.k) + slot * page * hd;
    float* scale_at = (which ? p.c.v_scale : p.c.k_scale) + slot;
    const int held = lo - (int)page_at;  // earlier tokens in the page
    const float old = held > 0 ? *scale_at : 0.0f;

    // the largest finite magnitude: of all first (fmaxf passes NaN over), and without the infinities if there are any
    float amax = 0.0f;
    auto each = [&](auto&& f) {
#pragma unroll
        for (int k = 0; k < kAppendKeep; ++k)
            if (tid + k * NT < n_vec) f(keep[k]);
        for (int g = tid + kAppendKeep * NT; g < n_vec; g += NT) f(load(g));
    };
    each([&](const V& v) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) amax = fmaxf(amax, fabsf(to_f32(v.v[e])));
    });
    if (amax > 3.402823466e38f) {
        amax = 0.0f;
        each([&](const V& v) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float a = fabsf(to_f32(v.v[e]));
                amax = a <= 3.402823466e38f ? fmaxf(amax, a) : amax;
            }
        });
    }
    amax = warp_max(amax);
    if constexpr (NT > 32) {
        if (lane == 0) s_max[warp] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NT / 32; ++w) amax = fmaxf(amax, s_max[w]);
    } else {
        __syncwarp();  // every lane has read the old scale before one overwrites it
    }
    const float fresh = pow2f(scale_exponent<FMT>(amax));
    const float scale = old > fresh ? old : fresh;
    const float inv = __fdiv_rn(1.0f, scale);

    auto store = [&](int f, const V& v) {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int e = 0; e < VEC; e += 4)
            w[e / 4] = encode4<FMT>(to_f32(v.v[e]) * inv, to_f32(v.v[e + 1]) * inv, to_f32(v.v[e + 2]) * inv, to_f32(v.v[e + 3]) * inv);
        uint32_t* to = reinterpret_cast<uint32_t*>(codes + (size_t)held * hd + (size_t)f * VEC);
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
        else *to = w[0];
    };
#pragma unroll
    for (int k = 0; k < kAppendKeep; ++k) {
        const int f = tid + k * NT;
        if (f < n_vec) store(f, keep[k]);
    }
    for (int f = tid + kAppendKeep * NT; f < n_vec; f += NT) store(f, load(f));
    if (held > 0 && old < scale) {
        const float shift = __fdiv_rn(old, scale);
        uint4* c16 = reinterpret_cast<uint4*>(codes);
#pragma unroll 4
        for (int f = tid; f < held * hd / 16; f += NT) {
            const uint4 w = c16[f];
            auto moved = [&](uint32_t x) {
                uint32_t o = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) o |= encode<FMT>(decode_code<FMT>((x >> (8 * e)) & 0xffu) * shift) << (8 * e);
                return o;
            };
            c16[f] = make_uint4(moved(w.x), moved(w.y), moved(w.z), moved(w.w));
        }
    }
    if (tid == 0) *scale_at = scale;
}

int check_cache(const iam_kv8_cache* c) {
    if (!c) return fail(IAM_ERR_ARG, "kv8: null cache");
    if (c->format != IAM_KV8_INT8 && c->format != IAM_KV8_E4M3) return fail(IAM_ERR_ARG, "kv8: unknown format");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(IAM_ERR_ARG, "kv8: page_size must be 16, 32, 64 or 128");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(IAM_ERR_UNSUPPORTED, "kv8: head_dim must be 64, 128 or 256");
    if (c->n_kv_heads <= 0 || c->n_pages <= 0 || c->max_pages <= 0 || c->n_seqs < 0) return fail(IAM_ERR_ARG, "kv8: bad cache sizes");
    if (c->n_kv_heads > 65535) return fail(IAM_ERR_ARG, "kv8: more than 65535 KV heads");
    if ((long long)c->max_pages * c->page_size > kKv8MaxTokens) return fail(IAM_ERR_UNSUPPORTED, "kv8: a table of more than 2^26 tokens");
    if ((long long)c->n_pages * c->n_kv_heads * c->page_size > INT32_MAX) return fail(IAM_ERR_UNSUPPORTED, "kv8: 2^31 rows of codes or more");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || (c->n_seqs > 0 && !c->block_table)) return fail(IAM_ERR_ARG, "kv8: null cache array");
    if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16)
        return fail(IAM_ERR_ARG, "kv8: codes must be 16-byte aligned");
    return IAM_OK;
}

int check_rows(const iam_rows* r, size_t elem, const char* what) {
    if (!r || !r->data) return fail(IAM_ERR_ARG, std::string("kv8: null ") + what);
    if (reinterpret_cast<uintptr_t>(r->data) % elem) return fail(IAM_ERR_ARG, std::string("kv8: misaligned ") + what);
    return IAM_OK;
}

}  // namespace
}  // namespace iam

using namespace iam;

struct iam_kv8_s {
    int device = 0, sms = 0, n_heads = 0, n_kv_heads = 0, head_dim = 0;
    Kv8Scratch s{};
};

extern "C" int iam_kv8_create(iam_kv8_t* out, int n_heads, int n_kv_heads, int head_dim, int device) {
    if (!out) return fail(IAM_ERR_ARG, "kv8: null handle");
    if (n_heads <= 0 || n_kv_heads <= 0 || n_heads % n_kv_heads) return fail(IAM_ERR_ARG, "kv8: n_heads must be a multiple of n_kv_heads");
    if (head_dim != 64 && head_dim != 128 && head_dim != 256) return fail(IAM_ERR_UNSUPPORTED, "kv8: head_dim must be 64, 128 or 256");
    int sms = 0;
    int rc = iam_device_info(device, &sms, nullptr, nullptr);
    if (rc) return rc;
    DeviceGuard g(device);
    IAM_CUDA_TRY(g.err);
    iam_kv8_s* h = new (std::nothrow) iam_kv8_s;
    if (!h) return fail(IAM_ERR_NOMEM, "kv8: out of host memory");
    h->device = device;
    h->sms = sms;
    h->n_heads = n_heads;
    h->n_kv_heads = n_kv_heads;
    h->head_dim = head_dim;
    h->s.max_ctas = kv8_max_ctas(sms);
    h->s.part_floats = std::max(std::max(kv8_decode_part_floats(head_dim, sms), kv8_rows_part_floats(head_dim, sms)), kv8_prompt_part_floats(head_dim, sms));
    cudaError_t e = cudaMalloc(&h->s.part, h->s.part_floats * sizeof(float));
    if (e == cudaSuccess) e = cudaMalloc(&h->s.ctr, h->s.max_ctas * sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(h->s.ctr, 0, h->s.max_ctas * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&h->s.plan, kv8_plan_words() * sizeof(int));
    if (e == cudaSuccess) e = cudaMalloc(&h->s.err, sizeof(unsigned));
    if (e == cudaSuccess) e = cudaMemset(h->s.err, 0, sizeof(unsigned));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) {
        iam_kv8_destroy(h);
        return cuda_fail(e, "kv8: scratch");
    }
    *out = h;
    return IAM_OK;
}

extern "C" int iam_kv8_destroy(iam_kv8_t h) {
    if (!h) return IAM_OK;
    DeviceGuard g(h->device);
    cudaFree(h->s.part);
    cudaFree(h->s.ctr);
    cudaFree(h->s.plan);
    cudaFree(h->s.err);
    delete h;
    return IAM_OK;
}

extern "C" int iam_kv8_status(iam_kv8_t h) {
    if (!h) return fail(IAM_ERR_ARG, "kv8: null handle");
    DeviceGuard g(h->device);
    IAM_CUDA_TRY(g.err);
    IAM_CUDA_TRY(cudaDeviceSynchronize());
    unsigned e = 0;
    IAM_CUDA_TRY(cudaMemcpy(&e, h->s.err, sizeof(e), cudaMemcpyDeviceToHost));
    if (!e) return IAM_OK;
    IAM_CUDA_TRY(cudaMemset(h->s.err, 0, sizeof(e)));
    if (e & kKv8ErrWait) return fail(IAM_ERR_TIMEOUT, "kv8: a wait of the attention gave up");
    return fail(IAM_ERR_ARG, "kv8: a page number, a length or a row offset was out of range");
}

extern "C" int iam_kv8_append(iam_kv8_t h, const iam_kv8_cache* cache, int dtype, int n_rows, const iam_rows* k, const iam_rows* v,
                              const int32_t* cu_dev, const int32_t* seq_lens_dev, void* stream) {
    if (!h) return fail(IAM_ERR_ARG, "kv8: null handle");
    int rc = check_cache(cache);
    if (rc) return rc;
    if (!dtype_ok(dtype)) return fail(IAM_ERR_ARG, "kv8: dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    if (cache->head_dim != h->head_dim || cache->n_kv_heads != h->n_kv_heads) return fail(IAM_ERR_ARG, "kv8: the cache has other heads than the handle");
    if (n_rows < 0) return fail(IAM_ERR_ARG, "kv8: negative rows");
    if (!cu_dev && n_rows != cache->n_seqs) return fail(IAM_ERR_ARG, "kv8: without cu there is one row per sequence");
    if (n_rows == 0 || cache->n_seqs == 0) return IAM_OK;
    const size_t elem = dtype_size(dtype);
    if ((rc = check_rows(k, elem, "keys")) || (rc = check_rows(v, elem, "values"))) return rc;
    if (!seq_lens_dev) return fail(IAM_ERR_ARG, "kv8: null sequence lengths");
    // slots as numbered on the device (slot_base); one page per sequence when each has one row
    const long long slots = cu_dev ? (long long)n_rows / cache->page_size + 2LL * cache->n_seqs : cache->n_seqs;
    if (slots * 2 * cache->n_kv_heads > INT32_MAX) return fail(IAM_ERR_ARG, "kv8: too many sequences");
    AppendParams p{*cache, {*k, *v}, cu_dev, seq_lens_dev, n_rows, h->s.err};
    const bool wide = rows_aligned(*k, elem, 16) && rows_aligned(*v, elem, 16);
    // A block for each page and head, or a warp where there are more of them than blocks run at once and few rows in each
    // (64 sequences of 1 row: 3.0 us against 7.6, of 16: 5 against 10, of 64: 19 against 16; 512 of 1: 10 against 56; but
    // 2 of 32, 80 blocks: 5.2 against 3.3).
    const bool few = n_rows <= kFewRows * (long long)cache->n_seqs && slots * 2 * cache->n_kv_heads > 4LL * h->sms;
    const int abreast = few ? kAppendThreads / 32 : 1;
    const dim3 grid((unsigned)(slots * ((2 * cache->n_kv_heads + abreast - 1) / abreast)));
    DeviceGuard g(h->device);
    IAM_CUDA_TRY(g.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    rc = with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // 16-byte reads where every row allows them, else one element at a time
        auto with_format = [&](auto fmt) {
            constexpr int FMT = decltype(fmt)::value;
            if (few) {
                if (wide) kv8_append_kernel<T, FMT, true, 32><<<grid, kAppendThreads, 0, s>>>(p);
                else kv8_append_kernel<T, FMT, false, 32><<<grid, kAppendThreads, 0, s>>>(p);
            } else {
                if (wide) kv8_append_kernel<T, FMT, true, kAppendThreads><<<grid, kAppendThreads, 0, s>>>(p);
                else kv8_append_kernel<T, FMT, false, kAppendThreads><<<grid, kAppendThreads, 0, s>>>(p);
            }
        };
        if (cache->format == IAM_KV8_INT8) with_format(std::integral_constant<int, IAM_KV8_INT8>{});
        else with_format(std::integral_constant<int, IAM_KV8_E4M3>{});
        IAM_CUDA_TRY(cudaGetLastError());
        return (int)IAM_OK;
    });
    return rc;
}

extern "C" int iam_kv8_attention(iam_kv8_t h, const iam_kv8_cache* cache, int dtype, int n_rows, int max_q, const iam_rows* q,
                                 const int32_t* cu_dev, const int32_t* seq_lens_dev, float scale, int window, const iam_rows* out,
                                 float* lse_dev, void* stream) {
    if (!h) return fail(IAM_ERR_ARG, "kv8: null handle");
    int rc = check_cache(cache);
    if (rc) return rc;
    if (!dtype_ok(dtype)) return fail(IAM_ERR_ARG, "kv8: dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    if (cache->head_dim != h->head_dim || cache->n_kv_heads != h->n_kv_heads) return fail(IAM_ERR_ARG, "kv8: the cache has other heads than the handle");
    if (n_rows < 0 || max_q < 0) return fail(IAM_ERR_ARG, "kv8: negative rows");
    if (!cu_dev && n_rows != cache->n_seqs) return fail(IAM_ERR_ARG, "kv8: without cu there is one row per sequence");
    if (!(scale >= 0.0f) || !std::isfinite(scale)) return fail(IAM_ERR_ARG, "kv8: scale must be finite and not negative (0: 1/sqrt(head_dim))");
    if (window < 0) return fail(IAM_ERR_ARG, "kv8: negative window");
    if (n_rows == 0 || cache->n_seqs == 0) return IAM_OK;
    const size_t elem = dtype_size(dtype);
    if ((rc = check_rows(q, elem, "queries")) || (rc = check_rows(out, elem, "output"))) return rc;
    if (!seq_lens_dev) return fail(IAM_ERR_ARG, "kv8: null sequence lengths");
    if (q->data == out->data && ((n_rows > 1 && q->token_stride != out->token_stride) || (h->n_heads > 1 && q->head_stride != out->head_stride)))
        return fail(IAM_ERR_ARG, "kv8: results over the queries need the same strides for both");
    Kv8Attn a{};
    a.c = *cache;
    a.cu = cu_dev;
    a.lens = seq_lens_dev;
    a.n_rows = n_rows;
    a.n_heads = h->n_heads;
    a.gq = h->n_heads / h->n_kv_heads;
    a.window = std::min(window, 1 << 30);  // (beyond every table; position - window stays an int)
    a.scale_log2 = (float)((scale > 0.0f ? (double)scale : 1.0 / std::sqrt((double)h->head_dim)) * 1.4426950408889634074);
    a.q = *q;
    a.out = *out;
    a.lse = lse_dev;
    a.s = h->s;
    a.sms = h->sms;
    const long long rows = (long long)(cu_dev ? (max_q > 0 ? std::min(max_q, n_rows) : n_rows) : 1) * a.gq;
    DeviceGuard g(h->device);
    IAM_CUDA_TRY(g.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((long long)n_rows * a.gq / 64 + cache->n_seqs > kKv8MaxItems)
        return fail(IAM_ERR_ARG, "kv8: more query rows than one call takes (65536 tiles of 64)");
    // The decode kernel reads the context once for 8 rows of a KV head (fp32: 4), the rows kernel once for 64, the prompt
    // kernel once for 256.  In us, decode | rows | prompt kernel, e4m3, head_dim 128, 8 KV heads where not said: re-reading
    // from L2 costs less than the others' schedule and join up to 4 passes (32 rows: 1 sequence of 8192 tokens 22 | 60 | 39, 32
    // of 2000 126 | 151 | 142; fp32, 16 rows: 23 | 63 and 116 | 179), and up to 8 where the sequences' KV heads do not fill
    // the SMs by themselves (64 rows: 1 x 8192 35 | 76 | 48, but 32 x 2000 234 | 172 | 148; fp32, 32 rows: 36 | 70, but
    // 218 | 188).  The prompt kernel takes over where there are many rows (512 of 13 x 5000 tokens, 2 KV heads:
    // 426 | 267 | 130) or heads to fill the SMs (128 of 32 x 2000: 447 | 295 | 166).  Head_dim 64 and 256 lie alike (64 rows of
    // 1 x 8192: 28 | 50 | 41 and 53 | 118).  The bounds are older than the prompt kernel's present start: between them, where the rows
    // kernel is still chosen for 16-bit queries, one of the others is faster by now (128 rows of 1 x 8192 58 | 79 | 68, of
    // 4 x 2000 71 | 78 | 47).
    const long long passes = (rows + (dtype == IAM_F32 ? 3 : 7)) / (dtype == IAM_F32 ? 4 : 8), items = (long long)cache->n_seqs * h->n_kv_heads;
    if (passes <= 4 || (passes <= 8 && items <= h->sms)) return kv8_decode_launch(a, dtype, s);
    if (dtype != IAM_F32 && h->head_dim <= 128 && rows > 64 && (rows > 256 || items >= h->sms)) return kv8_prompt_launch(a, dtype, s);
    return kv8_rows_launch(a, dtype, s);
}
