// gelu.h — the erf GELU of the encoder's FFN (GEMM epilogues and the int8 row kernels).
#pragma once
#include <hip/hip_runtime.h>

namespace hcr {

// GELU(x) = x/2 (1 + erf(x / sqrt 2)) (HF BERT "gelu", exact-erf form).  erf by Abramowitz &
// Stegun 7.1.26 (|error| <= 1.5e-7, far below the fp16/bf16 output rounding) on v_rcp / v_exp:
// ~12 instructions instead of the ~50 of the library erff -- the FFN1 epilogue evaluates 128 of
// them per lane per tile.  The reference-precision mode uses it too: its error (<= ~3e-7
// absolute with the rcp / exp2 approximations, a few fp32 ulps of erf near 1) leaves the
// encoder's max |diff| vs fp32 BertModel at the 1e-6 level (tests/test_encoder_gpu.py, 1e-4
// bar); HCRAG_GELU_LIBERF=1 selects the library erff there.
__device__ __forceinline__ float erf_as(float x) {
  const float ax = fabsf(x);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, ax, 1.f));
  float p = fmaf(t, 1.061405429f, -1.453152027f);
  p = fmaf(t, p, 1.421413741f);
  p = fmaf(t, p, -0.284496736f);
  p = fmaf(t, p, 0.254829592f);
  const float e = __builtin_amdgcn_exp2f(-ax * ax * 1.4426950408889634f);
  const float r = fmaf(-p * t, e, 1.f);
  return copysignf(r, x);
}
__device__ __forceinline__ float gelu_erf(float x) { return 0.5f * x * (1.f + erf_as(x * 0.70710678118654752f)); }

}  // namespace hcr
