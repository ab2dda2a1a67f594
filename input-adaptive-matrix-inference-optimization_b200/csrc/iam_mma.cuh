// iam_mma.cuh -- warp-level matrix instructions and shared-memory fragment loads.
#pragma once

#include "iam_common.cuh"

namespace iam {

// 16-byte global -> shared copy that does not wait (cp.async; completed by cp_async_wait_all).
IAM_DEV void cp_async16(void* dst_smem, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst_smem)),
                 "l"(__cvta_generic_to_global(src))
                 : "memory");
}
IAM_DEV void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// mma.sync m16n8k16, f16 x f16 -> f32 (fragments as the PTX ISA lays them out: A rows
// g = lane / 4 and g + 8, columns 2 * (lane % 4) + {0, 1} and + 8; B rows 2 * (lane % 4) + {0, 1}
// and + 8, column g; C rows g and g + 8, columns 2 * (lane % 4) + {0, 1}).
IAM_DEV void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
IAM_DEV void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
IAM_DEV void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
IAM_DEV uint32_t pack_h2(float a, float b) {  // a in the low half, both rounded to fp16
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | ((uint32_t)__half_as_ushort(__float2half_rn(b)) << 16);
}
// x = hi + lo with hi = fp16(x): the low part of a two-term fp16 split (exact in fp32)
IAM_DEV float split_lo(float x) { return __fsub_rn(x, __half2float(__float2half_rn(x))); }

}  // namespace iam
