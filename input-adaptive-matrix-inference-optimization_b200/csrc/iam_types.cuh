// iam_types.cuh -- element types of the stand-alone operators (rotary positions, 8-bit KV cache,
// log probabilities): fp32, fp16 or bf16 in memory, fp32 in registers.
#pragma once

#include <cuda_bf16.h>

#include "iam_common.cuh"

namespace iam {

IAM_DEV float to_f32(float v) { return v; }
IAM_DEV float to_f32(__half v) { return __half2float(v); }
IAM_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
IAM_DEV T from_f32(float v);
template <>
IAM_DEV float from_f32<float>(float v) { return v; }
template <>
IAM_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
IAM_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements moved as one access of N * sizeof(T) bytes (at most 16).
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

template <bool WIDE, class T, int N>
IAM_DEV Vec<T, N> load_vec(const T* p) {
    if constexpr (WIDE) {
        return *reinterpret_cast<const Vec<T, N>*>(p);
    } else {
        Vec<T, N> o;
#pragma unroll
        for (int e = 0; e < N; ++e) o.v[e] = p[e];
        return o;
    }
}
template <bool WIDE, class T, int N>
IAM_DEV void store_vec(T* p, const Vec<T, N>& o) {
    if constexpr (WIDE) {
        *reinterpret_cast<Vec<T, N>*>(p) = o;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = o.v[e];
    }
}

inline size_t dtype_size(int dtype) { return dtype == IAM_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == IAM_F32 || dtype == IAM_F16 || dtype == IAM_BF16; }

// Calls f(T{}) with the element type that `dtype` names.
template <class F>
int with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case IAM_F32: return f(float{});
        case IAM_F16: return f(__half{});
        case IAM_BF16: return f(__nv_bfloat16{});
        default: return fail(IAM_ERR_ARG, "dtype must be IAM_F32, IAM_F16 or IAM_BF16");
    }
}

// Makes `device` current for the life of the object and puts the caller's device back.
struct DeviceGuard {
    int before = -1;
    cudaError_t err = cudaSuccess;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

// Rows of heads: whether every access of `bytes` bytes at a multiple of it from a head's start is aligned.
inline bool rows_aligned(const iam_rows& r, size_t elem, size_t bytes) {
    return (reinterpret_cast<uintptr_t>(r.data) % bytes) == 0 && (r.token_stride * (long long)elem) % (long long)bytes == 0 &&
           (r.head_stride * (long long)elem) % (long long)bytes == 0;
}

}  // namespace iam
