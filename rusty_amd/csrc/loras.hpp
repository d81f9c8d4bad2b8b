// An adapter's t = factor X . A^T on the way to its product with fp16 B, shared by the kernels that add
// adapters to many rows (loras.hip, gemm.hip).
//
// A row of t is scaled by a power of two that puts its largest finite value in [2^14, 2^15), and each value x is
// two fp16 terms, hi = fp16(x) and lo = fp16(2^11 (x - hi)), whose products with B are summed apart and joined as
// hi + 2^-11 lo: off by at most 2^-22 of x where x is a normal number of fp16, from 2^-14 on.  A row with a value other than 0
// below that, more than 2^28 under its largest, is `low`: columns that only such values reach would lose bits that a sum
// in f32 has, so 16 rows with one that is low take f32 instructions, t as it is (8 for 2).
#pragma once

#include <hip/hip_runtime.h>

namespace rq {

typedef _Float16 lora_half8 __attribute__((ext_vector_type(8)));
typedef float lora_float4 __attribute__((ext_vector_type(4)));

constexpr float kLoraLo = 1.0f / 2048.0f;  // of a second term

// The exponent of a row's scale, for its largest finite |t| (at most 2^126, so that the inverse is a normal number).
__device__ __forceinline__ int lora_exponent(float most) {
    return most > 0.0f ? min(15 - __builtin_amdgcn_frexp_expf(most), 126) : 0;
}
__device__ __forceinline__ bool lora_low(float x) { return x != 0.0f && fabsf(x) < 6.103515625e-5f; }
// The terms of a scaled value (infinite and NaN: in hi alone).
__device__ __forceinline__ void lora_split(float x, _Float16 &hi, _Float16 &lo) {
    hi = (_Float16)x;
    lo = __builtin_isfinite((float)hi) ? (_Float16)((x - (float)hi) * 2048.0f) : (_Float16)0.0f;
}
// The two products joined.  An infinite B makes the second one infinite of either sign, or NaN as 0 times infinity; the
// first has what the sum is then, so the second is kept finite.
__device__ __forceinline__ float lora_join(float hi, float lo) {
    return __builtin_fmaf(__builtin_amdgcn_fmed3f(lo, -3e38f, 3e38f), kLoraLo, hi);
}
// acc + B^T . t^T in f32 instructions: b and t of 32 ranks as operands of v_mfma_f32_16x16x32_f16 (a lane: column or row
// lane % 16, ranks 8 (lane / 16) ..); instruction e takes rank e of each quarter wave.
__device__ __forceinline__ lora_float4 lora_add_f32(lora_half8 b, const lora_float4 (&t)[2], lora_float4 acc) {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32((float)b[e], t[e / 4][e % 4], acc, 0, 0, 0);
    return acc;
}

}  // namespace rq
