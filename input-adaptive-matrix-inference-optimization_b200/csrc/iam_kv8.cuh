// iam_kv8.cuh -- device side of the 8-bit paged KV cache: codes to fp16, where a sequence's rows and
// tokens are, and the join of a context that several CTAs share.
#pragma once

#include "iam_kv8.h"
#include "iam_mma.cuh"
#include "iam_types.cuh"

namespace iam {

// Every code is exact in fp16 (int8: 8 bits; e4m3: 4 bits in 2^-9 .. 448), so the tensor cores see the
// cache's own values and only the scales are applied in fp32.  Bytes 0, 1 -> lo, bytes 2, 3 -> hi.
template <int FMT>
IAM_DEV void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == IAM_KV8_E4M3) {
        asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        // 0x64xx is 1024 + xx in fp16: with the code's sign bit flipped, 1024 + 128 + code
        const uint32_t x = w ^ 0x80808080u;
        const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
        const uint32_t a = __byte_perm(x, 0x64646464u, 0x4140), b = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 l = __hsub2(*reinterpret_cast<const __half2*>(&a), off), h = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&l);
        hi = *reinterpret_cast<const uint32_t*>(&h);
    }
}

IAM_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Rows and tokens of one sequence: rows [row0, row0 + n) at positions start .. len - 1.  `cap` is the
// number of tokens whose page the table names.
struct SeqRows {
    int row0, n, len, start, cap;
};

IAM_DEV SeqRows seq_rows(const iam_kv8_cache& c, const int32_t* cu, const int32_t* lens, int n_rows, int i, unsigned* err) {
    SeqRows r;
    r.row0 = cu ? cu[i] : i;
    const int end = cu ? cu[i + 1] : i + 1;
    r.len = lens[i];
    const bool ok = r.row0 >= 0 && end >= r.row0 && end <= n_rows && r.len >= 0;
    r.n = ok ? end - r.row0 : 0;
    r.len = ok ? r.len : 0;
    const long long room = (long long)c.max_pages * c.page_size;
    r.cap = r.len <= room ? r.len : (int)room;
    if ((!ok || r.len > room) && err) atomicOr(err, kKv8ErrRange);
    r.start = r.len - r.n;
    return r;
}

// 2^e for -126 <= e <= 127
IAM_DEV float pow2f(int e) { return __int_as_float((e + 127) << 23); }

// The power of two that brings a row's largest magnitude into [2^13, 2^14) before it is rounded to fp16
// (one term) or split in two (hi + lo): fp16's range then never limits a query, whatever its type's.
IAM_DEV int query_shift(float amax) {
    const int e = (__float_as_int(amax) >> 23) & 0xff;  // amax is not negative
    return e == 0 || e == 0xff ? 0 : max(-120, min(120, 13 - (e - 127)));
}

IAM_DEV float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Counts one arrival, with what the CTA's threads wrote before their last barrier, and returns the number before it;
// what earlier arrivals brought is visible to the CTA behind its next barrier.
IAM_DEV int arrive(int* ctr) {
    int before;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(before) : "l"(__cvta_generic_to_global(ctr)) : "memory");
    return before;
}

constexpr float kLn2 = 0.69314718055994530942f;

// A row's result from its running maximum (log2 domain), sum and value sums.
template <class T>
IAM_DEV T result(float o, float l) {
    return from_f32<T>(l > 0.0f || l != l ? __fdiv_rn(o, l) : 0.0f);
}
template <class T>
IAM_DEV void store_result(const Kv8Attn& p, size_t row, int head, int d, float o, float l) {
    T* out = static_cast<T*>(p.out.data) + row * p.out.token_stride + head * p.out.head_stride;
    out[d] = result<T>(o, l);
}
IAM_DEV void store_lse(const Kv8Attn& p, size_t row, int head, float m, float l) {
    if (p.lse) p.lse[row * p.n_heads + head] = l > 0.0f || l != l ? (m + log2f(l)) * kLn2 : -INFINITY;
}

}  // namespace iam
