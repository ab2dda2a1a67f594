// iam_rope.cu -- rotary positions (rope_mx, aux.cl:227-248, generalised): half or interleaved pairs, the
// first rot_dim dims of a head, frequencies scaled for contexts longer than the model was trained on.
//
// Pair i of a token at position p turns by the angle p * w[i]:
//   (a, b) -> f * (a cos - b sin, b cos + a sin),
// with w[i] = theta^(-2i/rot) changed by the scaling (rope_frequencies) and f its factor (1 but for YaRN).
#include <algorithm>
#include <cmath>
#include <new>

#include "iam_rope.h"
#include "iam_types.cuh"

namespace iam {

constexpr int kRopeThreads = 256;
constexpr int kRopeMaxPairs = 512;
constexpr double kTwoPi = 6.283185307179586476925286766559;

int rope_check(const iam_rope_config* c) {
    if (!c) return fail(IAM_ERR_ARG, "rope: null config");
    if (c->head_dim < 2 || c->head_dim > 2 * kRopeMaxPairs) return fail(IAM_ERR_ARG, "rope: head_dim must be in [2, 1024]");
    if (c->rot_dim < 2 || c->rot_dim > c->head_dim || c->rot_dim % 2)
        return fail(IAM_ERR_ARG, "rope: rot_dim must be even and in [2, head_dim]");
    if (!(c->theta > 1.0) || !std::isfinite(c->theta)) return fail(IAM_ERR_ARG, "rope: theta must be finite and above 1");
    if (c->scaling < IAM_ROPE_NONE || c->scaling > IAM_ROPE_BANDED) return fail(IAM_ERR_ARG, "rope: unknown scaling");
    if (c->scaling != IAM_ROPE_NONE && (!(c->factor >= 1.0) || !std::isfinite(c->factor)))
        return fail(IAM_ERR_ARG, "rope: a scaling's factor must be finite and at least 1");
    if (c->scaling == IAM_ROPE_YARN || c->scaling == IAM_ROPE_BANDED) {
        if (c->original_ctx <= 0) return fail(IAM_ERR_ARG, "rope: this scaling needs original_ctx");
        if (!(c->low_turns >= 0.0) || !(c->high_turns >= 0.0) || !std::isfinite(c->low_turns) || !std::isfinite(c->high_turns))
            return fail(IAM_ERR_ARG, "rope: low_turns and high_turns must be finite and not negative");
        const double lo = c->low_turns > 0 ? c->low_turns : 1.0;
        const double hi = c->high_turns > 0 ? c->high_turns : c->scaling == IAM_ROPE_YARN ? 32.0 : 4.0;
        if (!(lo < hi)) return fail(IAM_ERR_ARG, "rope: low_turns must be below high_turns");
    }
    if (!(c->attn_factor >= 0.0) || !std::isfinite(c->attn_factor))
        return fail(IAM_ERR_ARG, "rope: attn_factor must be finite and not negative (0: the scaling's own)");
    return IAM_OK;
}

void rope_frequencies(const iam_rope_config& c, double* w, double* factor) {
    const int d = c.rot_dim;
    const double lo = c.low_turns > 0 ? c.low_turns : 1.0;
    const double hi = c.high_turns > 0 ? c.high_turns : c.scaling == IAM_ROPE_YARN ? 32.0 : 4.0;
    double theta = c.theta, f = 1.0, first = 0.0, last = 0.0;
    if (c.scaling == IAM_ROPE_NTK && d > 2) theta *= std::pow(c.factor, (double)d / (d - 2));
    if (c.scaling == IAM_ROPE_YARN) {
        // the pair that turns `n` times within the training length: theta^(-2i/d) * original = 2 pi n
        auto pair_of = [&](double n) { return d * std::log(c.original_ctx / (n * kTwoPi)) / (2.0 * std::log(c.theta)); };
        first = std::fmax(std::floor(pair_of(hi)), 0.0);
        last = std::fmin(std::ceil(pair_of(lo)), d - 1.0);
        if (c.factor > 1.0) f = 0.1 * std::log(c.factor) + 1.0;
    }
    for (int i = 0; i < d / 2; ++i) {
        const double base = std::pow(theta, -2.0 * i / d);
        double keep = 1.0;  // share of the unscaled frequency
        if (c.scaling == IAM_ROPE_LINEAR) keep = 0.0;
        if (c.scaling == IAM_ROPE_BANDED) keep = std::fmin(1.0, std::fmax(0.0, (c.original_ctx * base / kTwoPi - lo) / (hi - lo)));
        if (c.scaling == IAM_ROPE_YARN) keep = 1.0 - std::fmin(1.0, std::fmax(0.0, (i - first) / std::fmax(last - first, 0.001)));
        w[i] = keep == 1.0 ? base : base * keep + base / c.factor * (1.0 - keep);
    }
    *factor = c.attn_factor > 0.0 ? c.attn_factor : f;
}

namespace {

struct RopeParams {
    iam_rows in[2], out[2];  // q and k (k.data null: q alone)
    int heads[2];
    int n_tokens, head_dim, rot;
    const int32_t* positions;
    const double* turns;  // [rot / 2] turns (2 pi) per position
    float factor;
};

// `group` tokens per blockIdx.x; a thread keeps one place of a head (an access, or a pair of them in the half layout) and
// walks the (token, head) rows, which are spread over the block and blockIdx.y.  Bound by the bytes; the angles cost one
// reduction in 64 bits and one sincospif per pair and token, shared by all its heads through shared memory.  2048
// tokens of 32 + 8 heads of 128 (bf16, 42 MB): 11.1 us, 3.8 TB/s; 8191 tokens of 16 + 16 heads, 64 of 128 dims
// interleaved (fp16, 134 MB): 35.2 us, 3.8 TB/s (in place 36.6: the dims that do not turn are moved all the same); one token: 2.1 us,
// the launch.  (Rows asked for before the angles are
// made, one to four a thread, took 12.4 to 20 us for the first.)  The angle in turns is exact to 2^-53 of its size, so a position of 2^31 still has its phase to 2^-24.
template <class T, bool INTER, bool WIDE>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(RopeParams p, int group) {
    constexpr int VEC = WIDE ? 16 / (int)sizeof(T) : INTER ? 2 : 1;  // elements of a rotating access
    constexpr int PASS = WIDE ? VEC : 1;                             // and of one behind them
    __shared__ __align__(16) float2 cs[kRopeMaxPairs];               // [token of the group][pair]
    const int token0 = blockIdx.x * group, tokens = min(group, p.n_tokens - token0), pairs = p.rot / 2;
    for (int i = threadIdx.x; i < tokens * pairs; i += kRopeThreads) {
        const int k = i / pairs;
        const double t = (double)p.positions[token0 + k] * p.turns[i - k * pairs];
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        cs[i] = make_float2(c * p.factor, s * p.factor);
    }
    __syncthreads();
    const int turned = INTER ? p.rot / VEC : pairs / VEC;  // places of a head that rotate
    const int per_head = turned + (p.head_dim - p.rot) / PASS;
    const int heads = p.heads[0] + p.heads[1], n_rows = tokens * heads;
    // whole heads to the block's threads; a head with more places than threads in turns
    const int abreast = max(1, kRopeThreads / per_head);
    const int my_row = per_head <= kRopeThreads ? threadIdx.x / per_head : 0;
    if (my_row >= abreast) return;
    using V = Vec<T, VEC>;
    for (int j = threadIdx.x - my_row * per_head; j < per_head; j += kRopeThreads) {
#pragma unroll 2
        for (int row = blockIdx.y * abreast + my_row; row < n_rows; row += gridDim.y * abreast) {
            const int k = row / heads;
            int head = row - k * heads;
            const int which = head >= p.heads[0];
            head -= which ? p.heads[0] : 0;
            const iam_rows& ri = p.in[which];
            const iam_rows& ro = p.out[which];
            const T* x = static_cast<const T*>(ri.data) + (token0 + k) * ri.token_stride + head * ri.head_stride;
            T* y = static_cast<T*>(ro.data) + (token0 + k) * ro.token_stride + head * ro.head_stride;
            const float2* turn = cs + k * pairs;
            if (j >= turned) {  // dims behind the rotated ones
                const int d = p.rot + (j - turned) * PASS;
                store_vec<WIDE>(y + d, load_vec<WIDE, T, PASS>(x + d));
            } else if constexpr (INTER) {
                const V a = load_vec<WIDE, T, VEC>(x + j * VEC);
                V o;
#pragma unroll
                for (int e = 0; e < VEC; e += 2) {
                    const float2 t = turn[(j * VEC + e) / 2];
                    const float u = to_f32(a.v[e]), w = to_f32(a.v[e + 1]);
                    o.v[e] = from_f32<T>(u * t.x - w * t.y);
                    o.v[e + 1] = from_f32<T>(w * t.x + u * t.y);
                }
                store_vec<WIDE>(y + j * VEC, o);
            } else {
                const V a = load_vec<WIDE, T, VEC>(x + j * VEC), b = load_vec<WIDE, T, VEC>(x + pairs + j * VEC);
                V oa, ob;
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float2 t = turn[j * VEC + e];
                    const float u = to_f32(a.v[e]), w = to_f32(b.v[e]);
                    oa.v[e] = from_f32<T>(u * t.x - w * t.y);
                    ob.v[e] = from_f32<T>(w * t.x + u * t.y);
                }
                store_vec<WIDE>(y + j * VEC, oa);
                store_vec<WIDE>(y + pairs + j * VEC, ob);
            }
        }
    }
}

template <class T, bool INTER, bool WIDE>
int launch_rope(const RopeParams& p, int sms, cudaStream_t s) {
    constexpr int VEC = WIDE ? 16 / (int)sizeof(T) : INTER ? 2 : 1;
    const int per_head = (INTER ? p.rot : p.rot / 2) / VEC + (p.head_dim - p.rot) / (WIDE ? VEC : 1);
    const int abreast = std::max(1, kRopeThreads / per_head), heads = p.heads[0] + p.heads[1];
    // Many tokens: four a block, so that its threads have several rows each; few: a token's heads over as many blocks
    // as leave a row to a thread
    const bool many = p.n_tokens >= 8 * sms && 4 * (p.rot / 2) <= kRopeMaxPairs;
    const int group = many ? 4 : 1;
    long long split = 1;
    if (p.n_tokens < 2 * sms) split = std::min<long long>((heads + abreast - 1) / abreast, (2 * sms + p.n_tokens - 1) / p.n_tokens);
    rope_kernel<T, INTER, WIDE><<<dim3((p.n_tokens + group - 1) / group, (unsigned)std::max<long long>(1, split)), kRopeThreads, 0, s>>>(p, group);
    IAM_CUDA_TRY(cudaGetLastError());
    return IAM_OK;
}

}  // namespace
}  // namespace iam

using namespace iam;

struct iam_rope_s {
    iam_rope_config cfg{};
    int device = 0, sms = 0;
    float factor = 1.0f;
    double* turns = nullptr;
};

extern "C" int iam_rope_frequencies(const iam_rope_config* cfg, double* radians_out, double* factor_out) {
    int rc = rope_check(cfg);
    if (rc) return rc;
    if (!radians_out) return fail(IAM_ERR_ARG, "rope: null output");
    double f;
    rope_frequencies(*cfg, radians_out, &f);
    if (factor_out) *factor_out = f;
    return IAM_OK;
}

extern "C" int iam_rope_create(iam_rope_t* out, const iam_rope_config* cfg, int device) {
    if (!out) return fail(IAM_ERR_ARG, "rope: null handle");
    int rc = rope_check(cfg);
    if (rc) return rc;
    int sms = 0;
    if ((rc = iam_device_info(device, &sms, nullptr, nullptr))) return rc;
    DeviceGuard g(device);
    IAM_CUDA_TRY(g.err);
    double w[kRopeMaxPairs], factor;
    rope_frequencies(*cfg, w, &factor);
    for (int i = 0; i < cfg->rot_dim / 2; ++i) w[i] /= kTwoPi;
    iam_rope_s* h = new (std::nothrow) iam_rope_s;
    if (!h) return fail(IAM_ERR_NOMEM, "rope: out of host memory");
    h->cfg = *cfg;
    h->device = device;
    h->sms = sms;
    h->factor = (float)factor;
    const size_t bytes = sizeof(double) * (cfg->rot_dim / 2);
    cudaError_t e = cudaMalloc(&h->turns, bytes);
    if (e == cudaSuccess) e = cudaMemcpy(h->turns, w, bytes, cudaMemcpyHostToDevice);
    if (e != cudaSuccess) {
        cudaFree(h->turns);
        delete h;
        return cuda_fail(e, "rope: frequencies");
    }
    *out = h;
    return IAM_OK;
}

extern "C" int iam_rope_destroy(iam_rope_t h) {
    if (!h) return IAM_OK;
    DeviceGuard g(h->device);
    cudaFree(h->turns);
    delete h;
    return IAM_OK;
}

extern "C" int iam_rope_apply(iam_rope_t h, int dtype, int n_tokens, const int32_t* positions_dev, int n_heads, const iam_rows* q_in,
                              const iam_rows* q_out, int n_kv_heads, const iam_rows* k_in, const iam_rows* k_out, void* stream) {
    if (!h) return fail(IAM_ERR_ARG, "rope: null handle");
    if (!dtype_ok(dtype)) return fail(IAM_ERR_ARG, "rope: dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    if (n_tokens > 1 << 30) return fail(IAM_ERR_ARG, "rope: more than 2^30 tokens");
    if (n_tokens < 0 || n_heads < 0 || n_kv_heads < 0) return fail(IAM_ERR_ARG, "rope: negative count");
    if ((long long)n_heads + n_kv_heads > 65536) return fail(IAM_ERR_ARG, "rope: more than 65536 heads");
    if (n_tokens == 0 || n_heads + n_kv_heads == 0) return IAM_OK;
    if (!positions_dev) return fail(IAM_ERR_ARG, "rope: null positions");
    RopeParams p{};
    const iam_rows* in[2] = {q_in, k_in};
    const iam_rows* out[2] = {q_out, k_out};
    const int heads[2] = {n_heads, n_kv_heads};
    const size_t elem = dtype_size(dtype);
    const int vec = (int)(16 / elem);
    const int rot = h->cfg.rot_dim, unit = h->cfg.interleaved ? rot : rot / 2;
    bool wide = unit % vec == 0 && rot % vec == 0 && h->cfg.head_dim % vec == 0;
    for (int i = 0; i < 2; ++i) {
        if (heads[i] == 0) continue;
        if (!in[i] || !out[i] || !in[i]->data || !out[i]->data) return fail(IAM_ERR_ARG, "rope: null rows");
        if (reinterpret_cast<uintptr_t>(in[i]->data) % elem || reinterpret_cast<uintptr_t>(out[i]->data) % elem)
            return fail(IAM_ERR_ARG, "rope: rows not aligned to their type");
        if (in[i]->data == out[i]->data && ((n_tokens > 1 && in[i]->token_stride != out[i]->token_stride) ||
                                            (heads[i] > 1 && in[i]->head_stride != out[i]->head_stride)))
            return fail(IAM_ERR_ARG, "rope: in place needs the same strides for input and output");
        p.in[i] = *in[i];
        p.out[i] = *out[i];
        p.heads[i] = heads[i];
        wide = wide && rows_aligned(*in[i], elem, 16) && rows_aligned(*out[i], elem, 16);
    }
    p.n_tokens = n_tokens;
    p.head_dim = h->cfg.head_dim;
    p.rot = rot;
    p.positions = positions_dev;
    p.turns = h->turns;
    p.factor = h->factor;
    DeviceGuard g(h->device);
    IAM_CUDA_TRY(g.err);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return with_dtype(dtype, [&](auto t) {
        using T = decltype(t);
        // 16-byte accesses where every row allows them, else one element at a time (rows at odd
        // offsets or strides, or a rotated part that is no whole number of vectors)
        if (h->cfg.interleaved) return wide ? launch_rope<T, true, true>(p, h->sms, s) : launch_rope<T, true, false>(p, h->sms, s);
        return wide ? launch_rope<T, false, true>(p, h->sms, s) : launch_rope<T, false, false>(p, h->sms, s);
    });
}
