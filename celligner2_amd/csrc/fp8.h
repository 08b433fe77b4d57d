// Shared by the 8-bit quantiser (fp8.hip) and the 8-bit products (gemm_fp8.hip, rows_fp8.hip).
#pragma once
#include "vec8.h"

namespace c2 {
namespace fp8 {

typedef __attribute__((ext_vector_type(8))) int i32x8;

__device__ __forceinline__ float finite_abs(float x) {  // (a comparison with NaN is false)
    const float a = fabsf(x);
    return a < INFINITY ? a : 0.f;
}

// exponent s of a block whose largest finite magnitude is amax
template <int FMT>
__device__ __forceinline__ int block_exponent(float amax) {
    const unsigned u = __builtin_bit_cast(unsigned, amax);
    if (u == 0) return 0;
    const int s = (int)(u >> 23) - 127 - (FMT == C2_E4M3 ? 8 : 15) + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(s, -126);  // (an amax below the normal range ends here too)
}
__device__ __forceinline__ float exp2i(int e) { return __builtin_bit_cast(float, (unsigned)(e + 127) << 23); }  // -126 .. 127

// four values, already multiplied by 2^-s, as four 8-bit numbers
template <int FMT>
__device__ __forceinline__ unsigned pack8(float a, float b, float c, float d) {
    int r = 0;
    if (FMT == C2_E4M3) {
        r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    } else {
        r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, r, false);
        r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
    }
    return (unsigned)r;
}

// Products with fp32 results run on the bf16 instruction, which adds its products in fp32: every 8-bit number times its scale is
// exact in bf16.  Eight numbers of FMT (four in lo, four in hi) times the scale `x`, see wide_scale.
template <int FMT>
__device__ __forceinline__ bf16x8 widen8(unsigned lo, unsigned hi, float x) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
    bf16x2 a, b, c, d;
    if (FMT == C2_E4M3) {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, x, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, x, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, x, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, x, true);
    } else {
        a = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, x, false);
        b = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(lo, x, true);
        c = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, x, false);
        d = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(hi, x, true);
    }
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The scale byte as the conversion takes it (a float's exponent), one below: a block near fp32's largest number may hold an element
// that is rounded up to 2^128, which neither fp32 nor bf16 has.  kWideBack times the sum makes up for both operands' halves.  An
// element under 2^-132 is rounded to a multiple of that (bf16's own smallest step).
constexpr float kWideBack = 4.f;
__device__ __forceinline__ float wide_scale(unsigned byte) { return __builtin_bit_cast(float, (byte << 23) - 0x800000u); }

__device__ __forceinline__ int64_t scale_at(int64_t kb, int64_t r64, int64_t row) {
    return ((kb * r64 + (row >> 6)) * 16 + (row & 15)) * 4 + ((row >> 4) & 3);
}

// rows_fp8.hip: products with few rows of A.  x_dtype: C2_F32 / C2_BF16 / C2_F16 (quantised inside, e4m3), or kQuantised (A, sA
// in format a_fmt).
constexpr int kQuantised = -1;
struct RowPlan {
    enum { kNone, kOneLaunch, kParts } form;  // kNone: not such a product
    int splits, kb_per_split;
    int64_t lds;  // row pitch of the parts, [splits][M][lds] floats in ws where splits > 1
};
RowPlan row_plan(int64_t M, int64_t N, int64_t K);
inline bool in_rows(int64_t M, int64_t N, int64_t K) { return row_plan(M, N, K).form != RowPlan::kNone; }
void launch_few_rows(const void* A, int x_dtype, int64_t lda, const uint8_t* sA, int a_fmt, const uint8_t* B, int64_t ldb,
                     const uint8_t* sB, int64_t M, int64_t N, int64_t K, void* Y, int y_dtype, int64_t ldy, const float* bias,
                     const float* alpha_dev, float* ws, hipStream_t st);
// gemm_fp8.hip: Y = alpha * sum of the parts + bias
void join_slabs(const float* ws, int64_t slab, int64_t lds, int splits, int64_t M, int64_t N, void* Y, int y_dtype, int64_t ldy,
                const float* bias, const float* alpha_dev, hipStream_t st);

}  // namespace fp8
}  // namespace c2
