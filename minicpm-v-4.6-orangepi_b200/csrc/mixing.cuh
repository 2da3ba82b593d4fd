// Shared pieces of the token-mixing operators (mrope.cu, paged_attention.cu,
// gated_delta.cu): warp-level fp16 MMA and its operand loads, asynchronous
// 16-byte copies with zero fill, the checks of strided rows and of a paged
// cache.  sm_100a.
#pragma once

#include "common.cuh"

namespace mcv {

// Device-side error bit of the token-mixing operators: an index read from
// device memory (page, sequence row, state slot, sequence bound) was out of
// range.  It is never followed.
enum : unsigned { kDevErrIndex = 2u };
// A gated delta prompt ended in a state that is not finite.
enum : unsigned { kDevErrRange = 4u };

// Host checks; both set the error message and return a status.
int check_rows(const char* who, const char* what, const mcv_rows* r, int64_t heads, int64_t dim);
int check_kv_cache(const char* who, const mcv_kv_cache* c);

// q = n / d for 0 <= n < 2^31 by one multiplication: q = (n * mul) >> shift
// with shift = 31 + ceil(log2 d), mul = ceil(2^shift / d) (Granlund and
// Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
    uint32_t mul, shift, d;
    explicit FastDiv(uint32_t div) : d(div) {
        uint32_t l = 0;
        while ((uint64_t{1} << l) < div) ++l;
        shift = 31 + l;
        mul = static_cast<uint32_t>(((uint64_t{1} << shift) + div - 1) / div);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
    }
};

// 16-byte asynchronous copy; copies nothing and writes zeros when !take (src
// is then not read).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Four 8x8 fp16 matrices; lanes 8i..8i+7 give the row addresses of matrix i.
// Lane (g = lane / 4, t = lane % 4) receives elements (g, 2t), (g, 2t + 1) of
// each, of its transpose in the _t form.
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Transposes an 8x8 fp16 matrix held as lane (g, t) = elements (g, 2t), (g, 2t + 1).
__device__ __forceinline__ uint32_t movm_t(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
// c (16x8 fp32) += a (16x16 fp16, rows) x b (16x8 fp16, columns).
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x, y as two fp16 pairs hi + lo: x - (hi + lo) is at most 2^-22 |x| (and 2^-25
// where lo is subnormal), so that a product of hi and lo with fp16 operands
// keeps fp32's accuracy.  The remainder is exact, in one mixed-precision FMA.
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = h2_as_u32(__floats2half2_rn(x, y));
    fma2_f16_f32(x, y, hi, 0xbc00bc00u);      // - 1 hi
    lo = h2_as_u32(__floats2half2_rn(x, y));
}

}  // namespace mcv
