// int8_kernels.h — kernels of the 8-bit integer operators (C ABI in include/hcrag.h, host side in
// int8_ops.hip; the encoder's HCR_I8 mode calls them):
//   rows_to_int8_kernel   [residual add + LayerNorm / RMS norm | activation] -> int8 rows + scales
//   int8_to_rows_kernel   the values that int8 rows and scales stand for
//   int8_linear_direct    y = x . w^T of int8 rows, few tokens
#pragma once
#include "device_common.h"
#include "hcrag.h"
#include "int8_args.h"

namespace hcr {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef unsigned int uintx4 __attribute__((ext_vector_type(4)));

// -------------------------------------------------------------------------------------
// Rows -> int8.  Per row: v = f(x) (below), a = max |v|, scale = a / 127,
// q = round_half_even(v * (127 / a)).
//   I8_QUANT  v = x                        I8_GELU  v = gelu(x) (exact-erf form)
//   I8_LAYER  h = x + r, v = (h - mean) rsqrt(var + eps) g + b
//   I8_RMS    h = x + r, v = h rsqrt(mean(h^2) + eps) g + b       (b may be absent)
// A row is read once: its elements stay in registers (NCH chunks of 8 per thread) through the
// centred second moment (as layernorm4_kernel) and the maximum.  Everything between the loads
// and the stores is fp32: v is computed from the unrounded h, and the int8 rounding is the only
// one q carries; sum (h) and y (v) are rounded once to their own types.
// The maximum is taken over the bit patterns of |v|: an infinity or a NaN is larger than every
// finite value, and such a row gets scale NaN and q = 0, so that a product with it is NaN.  A row
// below 2^-100 counts as zeros (scale 0, q 0): 127 / a would leave fp32's range.
// Bound by memory (MI355X, calls back to back on one input; a copy of 8 GiB moves 4.6 TB/s): RMS norm with
// residual of 65521 x 4096 bf16 1.88 GB in 317 us (5.9 TB/s), LayerNorm of 32749 x 768 (f16 + f32 -> f32)
// 51 us (5.4 TB/s), quantisation of 65521 x 4096 f16 116 us (7.0 TB/s), with GELU 155-163 us by the board,
// where arithmetic and memory meet.
// -------------------------------------------------------------------------------------

// gelu(x) = x Phi(x) = x / (1 + 2^-z), z = log2(Phi / (1 - Phi)) = x g(x^2): g as a polynomial fitted so
// that Phi is within 3.6e-8 everywhere (its last coefficient is positive: z keeps x's sign past the
// fit, where Phi is 0 or 1).  Fewer instructions than erf_as's form, whose error in Phi it also halves:
// this kernel is bound by arithmetic (65521 x 4096: 207 us with erf_as, 160 so).  In fp32, exp2 and the
// reciprocal each off by one ulp at most, |dv| <= 0.81 (1.6e-7 |x| + 2.4e-7 |v|).  That is an absolute
// bound: in the negative tail nothing of v may be left (i8_gelu_tail).
__device__ __forceinline__ float i8_gelu(float x) {
  const float t = x * x;
  float g = 5.067230635091846e-09f;
  g = fmaf(g, t, -3.816310822912783e-07f);
  g = fmaf(g, t, 1.1439830814197194e-05f);
  g = fmaf(g, t, -1.5957992582116276e-04f);
  g = fmaf(g, t, -9.4049253675621e-05f);
  g = fmaf(g, t, 1.0483512282371521e-01f);
  g = fmaf(g, t, 2.3022093772888184e+00f);
  return x * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-(g * x)));
}

// gelu(x) relative to itself, for the rows whose scale is a value of the negative tail: no element of such
// a row is larger than I8_GELU_SMALL, so it is either below -3 (x Phi(x) = -phi(x) W(1 / x^2), W as a
// polynomial fitted within 5e-7 for x < -2.5, phi the normal density with its factor in W's coefficients)
// or within 0.008 of 0, where the logistic form is relative already.
// |dv| <= (1e-6 + (1.25 x^2 + 24) 2^-24) |v|.  65521 x 4096 f16: rows in the tail 249 us, others 163
// (without this branch 161), rows of zeros 144.
constexpr uint32_t I8_GELU_SMALL = 0x3B800000u;        // 2^-8, as bits
__device__ __forceinline__ float i8_gelu_tail(float x) {
  const float t = x * x, s = __builtin_amdgcn_rcpf(t);
  float p = 105.96810913085938f;
  p = fmaf(p, s, -73.01840209960938f);
  p = fmaf(p, s, 23.39447784423828f);
  p = fmaf(p, s, -5.247370719909668f);
  p = fmaf(p, s, 1.1810914278030396f);
  p = fmaf(p, s, -0.39880889654159546f);
  p = fmaf(p, s, 0.39894208312034607f);
  const float tail = -(__builtin_amdgcn_exp2f(t * -0.72134752044448f) * p);   // (log2(e) / 2)
  return x < -2.5f ? tail : i8_gelu(x);
}

// v inv, rounded, plus 1.5 * 2^23, rounded: the low byte is v inv to the nearest whole number, ties to
// even.  (Not as one fma: q is defined by the rounded product.)
__device__ __forceinline__ uint32_t i8_step(float v, float inv) {
#pragma clang fp contract(off)
  const float p = v * inv;
  return __float_as_uint(p + 12582912.f);
}

// 16 bytes at any alignment: one instruction, the hardware takes unaligned vectors (rows of odd
// widths, 65521 x 1531 bf16: 139 us element by element).
typedef uint32_t uintx4_any __attribute__((ext_vector_type(4), aligned(2)));
// NT: not to be kept in the caches (non-temporal).
template <bool NT = false>
__device__ __forceinline__ uintx4 i8_load16(const char* p) {
  const uintx4_any* v = reinterpret_cast<const uintx4_any*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(v);
  else return *v;
}
template <bool NT = false>
__device__ __forceinline__ void i8_store16(char* p, uintx4 u) {
  uintx4_any* v = reinterpret_cast<uintx4_any*>(p);
  if constexpr (NT) __builtin_nontemporal_store((uintx4_any)u, v);
  else *v = u;
}

struct I8Raw { uintx4 a, b; };     // 8 elements as loaded: 16-bit types in a, f32 in a and b

// elements [i, i + 8) of a row of cols: whole chunks as vectors, the row's last, partial one element
// by element (the row's last element again past its end: the caller drops those)
template <bool F32, bool NT = false>
__device__ __forceinline__ void i8_load(I8Raw& o, const char* row, int i, int cols) {
  if (i + 8 <= cols) {
    const char* p = row + (int64_t)i * (F32 ? 4 : 2);
    o.a = i8_load16<NT>(p);
    if constexpr (F32) o.b = i8_load16(p + 16);
  } else if (i < cols) {
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = min(i + e, cols - 1);
      w[e] = F32 ? reinterpret_cast<const uint32_t*>(row)[j] : reinterpret_cast<const uint16_t*>(row)[j];
    }
    if constexpr (F32) {
      o.a = uintx4{w[0], w[1], w[2], w[3]};
      o.b = uintx4{w[4], w[5], w[6], w[7]};
    } else {
      o.a = uintx4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
    }
  }
}
__device__ __forceinline__ void i8_convert(float (&v)[8], const I8Raw& o, int type) {
  if (type == HCR_F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = __uint_as_float(o.a[e]); v[4 + e] = __uint_as_float(o.b[e]); }
  } else if (type == HCR_BF16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = __uint_as_float(o.a[e] << 16);
      v[2 * e + 1] = __uint_as_float(o.a[e] & 0xFFFF0000u);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = (float)__builtin_bit_cast(_Float16, (uint16_t)o.a[e]);
      v[2 * e + 1] = (float)__builtin_bit_cast(_Float16, (uint16_t)(o.a[e] >> 16));
    }
  }
}
// Both rounded at once (v_cvt_pk): element by element, the f16 conversion after an fma becomes one
// v_fma_mixlo, which leaves f16 subnormals as zeros.
template <typename T>
__device__ __forceinline__ uint32_t i8_pack2(float x, float y) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  typedef T T2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{x, y}), T2));
}
// elements [i, i + 8) of a row of cols, those that exist
template <bool NT>
__device__ __forceinline__ void i8_store(char* row, int type, int i, int cols, const float (&v)[8]) {
  if (type == HCR_F32) {
    char* p = row + (int64_t)i * 4;
    if (i + 8 <= cols) {
      i8_store16(p, uintx4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
      i8_store16(p + 16, uintx4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e) if (i + e < cols) reinterpret_cast<float*>(p)[e] = v[e];
    }
    return;
  }
  uintx4 h;
  if (type == HCR_BF16) h = uintx4{i8_pack2<__bf16>(v[0], v[1]), i8_pack2<__bf16>(v[2], v[3]), i8_pack2<__bf16>(v[4], v[5]), i8_pack2<__bf16>(v[6], v[7])};
  else h = uintx4{i8_pack2<_Float16>(v[0], v[1]), i8_pack2<_Float16>(v[2], v[3]), i8_pack2<_Float16>(v[4], v[5]), i8_pack2<_Float16>(v[6], v[7])};
  char* p = row + (int64_t)i * 2;
  if (i + 8 <= cols) {
    i8_store16<NT>(p, h);
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (i + e < cols) reinterpret_cast<uint16_t*>(p)[e] = (uint16_t)(h[e >> 1] >> (16 * (e & 1)));
  }
}

// Reductions over the WAVES waves that share a row (WAVES == 1: each wave has its own row), the same
// result in every lane.  Within 16 lanes by DPP, over the rest by lane swaps: no LDS round trips.
template <int CTRL>
__device__ __forceinline__ uint32_t i8_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
template <typename F>
__device__ __forceinline__ uint32_t i8_wave_reduce(uint32_t v, F f) {
  v = f(v, i8_dpp<0xB1>(v));       // quad_perm [1 0 3 2]
  v = f(v, i8_dpp<0x4E>(v));       // quad_perm [2 3 0 1]
  v = f(v, i8_dpp<0x141>(v));      // mirrored in 8 lanes
  v = f(v, i8_dpp<0x140>(v));      // mirrored in 16 lanes
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = f(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return f(b[0], b[1]);
}
template <int WAVES, typename F>
__device__ __forceinline__ uint32_t i8_row_reduce(uint32_t v, uint32_t* red, int wave, int lane, F f) {
  v = i8_wave_reduce(v, f);
  if constexpr (WAVES > 1) {
    __syncthreads();               // (the previous reduction's reads of red are done)
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v = f(v, red[w]);
  }
  return v;
}
template <int WAVES>
__device__ __forceinline__ float i8_row_sum(float s, uint32_t* red, int wave, int lane) {
  return __uint_as_float(i8_row_reduce<WAVES>(__float_as_uint(s), red, wave, lane, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// One row per WAVES waves; WAVES == 1 puts 4 rows in a workgroup.  Covers cols <= 512 WAVES NCH.
// NT: x, the residual and what is stored pass by the caches (but f32 rows, of which a lane takes two
// vectors, each half of its lines, and the int8 rows of a mere quantisation: 65521 x 4096 f16 118 us, with
// them 125 on the same board).
template <int MODE, int WAVES, int NCH, bool NT>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, WAVES == 1 && MODE == I8_GELU ? 8 : 1)
rows_to_int8_kernel(I8RowArgs a) {
  __shared__ uint32_t red[WAVES > 1 ? WAVES : 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned at = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  if (WAVES == 1 && at >= a.rows) return;
  const int64_t row = a.row0 + at;
  const int tid = WAVES == 1 ? lane : threadIdx.x;
  constexpr int NTH = 64 * WAVES;
  constexpr bool NORM = MODE == I8_LAYER || MODE == I8_RMS;
  const bool x32 = a.xt == HCR_F32, r32 = a.rt == HCR_F32;
  const char* xr = reinterpret_cast<const char*>(a.x) + row * a.ldx * (x32 ? 4 : 2);
  const char* rr = reinterpret_cast<const char*>(a.r) + row * a.ldr * (r32 ? 4 : 2);
  I8Raw xs[NCH], rs[NORM ? NCH : 1];
  // (one branch on the element size around all of a row's loads: they are in flight together)
  if (x32) {
#pragma unroll
    for (int c = 0; c < NCH; ++c) i8_load<true>(xs[c], xr, (tid + NTH * c) * 8, a.cols);
  } else {
#pragma unroll
    for (int c = 0; c < NCH; ++c) i8_load<false, NT>(xs[c], xr, (tid + NTH * c) * 8, a.cols);
  }
  if constexpr (NORM) {
    if (a.r) {
      if (r32) {
#pragma unroll
        for (int c = 0; c < NCH; ++c) i8_load<true>(rs[c], rr, (tid + NTH * c) * 8, a.cols);
      } else {
#pragma unroll
        for (int c = 0; c < NCH; ++c) i8_load<false, NT>(rs[c], rr, (tid + NTH * c) * 8, a.cols);
      }
    }
  }
  float v[NCH][8];                 // (elements past the row's end are 0)
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    i8_convert(v[c], xs[c], a.xt);
    if constexpr (NORM) {
      if (a.r) {
        float r[8];
        i8_convert(r, rs[c], a.rt);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] += r[e];
      }
    }
    if constexpr (MODE == I8_GELU) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = i8_gelu(v[c][e]);
    }
    const int n = a.cols - (tid + NTH * c) * 8;
    if (n < 8) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = e < n ? v[c][e] : 0.f;
    }
  }
  if constexpr (NORM) {
    float mean = 0.f;
    if constexpr (MODE == I8_LAYER) {
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        s += ((v[c][0] + v[c][1]) + (v[c][2] + v[c][3])) + ((v[c][4] + v[c][5]) + (v[c][6] + v[c][7]));
      mean = i8_row_sum<WAVES>(s, red, wave, lane) / (float)a.cols;
    }
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int n = a.cols - (tid + NTH * c) * 8;
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = v[c][e] - mean;
      if (n < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = e < n ? d[e] : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(d[e], d[e], s);
    }
    const float var = i8_row_sum<WAVES>(s, red, wave, lane) / (float)a.cols;
    // (squares past fp32's range: the row is not representable, and all of it becomes NaN)
    const float rstd = var < INFINITY ? rsqrtf(var + a.eps) : __uint_as_float(0x7FC00000u);
    if (a.sum) {
      char* sr = reinterpret_cast<char*>(a.sum) + row * a.ldsum * (r32 ? 4 : 2);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int i = (tid + NTH * c) * 8;
        if (i < a.cols) i8_store<NT>(sr, a.rt, i, a.cols, v[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      const int i = (tid + NTH * c) * 8, n = a.cols - i;
      if (n <= 0) continue;
      I8Raw raw;
      float g[8], b[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      i8_load<true>(raw, reinterpret_cast<const char*>(a.g), i, a.cols);
      i8_convert(g, raw, HCR_F32);
      if (a.b) {
        i8_load<true>(raw, reinterpret_cast<const char*>(a.b), i, a.cols);
        i8_convert(b, raw, HCR_F32);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[c][e] = fmaf((v[c][e] - mean) * rstd, g[e], b[e]);
      if (n < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[c][e] = e < n ? v[c][e] : 0.f;
      }
    }
    if (a.y) {
      char* yr = reinterpret_cast<char*>(a.y) + row * a.ldy * (a.yt == HCR_F32 ? 4 : 2);
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        const int i = (tid + NTH * c) * 8;
        if (i < a.cols) i8_store<NT>(yr, a.yt, i, a.cols, v[c]);
      }
    }
  }
  // the largest pattern as signed (of the positive elements) and as unsigned (of the negative ones,
  // if there are any): one three-way maximum per two elements each
  uint32_t mn;
  auto largest = [&]() __attribute__((always_inline)) {
    int mp = 0;
    mn = 0u;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t u0 = __float_as_uint(v[c][e]), u1 = __float_as_uint(v[c][e + 1]);
        mp = max(max(mp, (int)u0), (int)u1);
        mn = max(max(mn, u0), u1);
      }
    const uint32_t m = max((uint32_t)mp, (mn >> 31) ? mn & 0x7FFFFFFFu : 0u);
    return i8_row_reduce<WAVES>(m, red, wave, lane, [](uint32_t p, uint32_t q) { return max(p, q); });
  };
  uint32_t m = largest();
  if constexpr (MODE == I8_GELU) {
    if ((uint32_t)__builtin_amdgcn_readfirstlane((int)m) < I8_GELU_SMALL) {
      // (v keeps x's sign, also where nothing is left of it: rows of zeros, as padding is, end here)
      const int negative = (int)(mn >> 31);
      if (WAVES == 1 ? __any(negative) : __syncthreads_or(negative)) {
        // The row again, relative to its values.  Read again, a chunk at a time: held for this, its
        // elements would cost every row registers.  (The address is one that the compiler cannot take for
        // the first reads'.)
        const char* xa = xr;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
          const int i = (tid + NTH * c) * 8, n = a.cols - i;
          asm volatile("" : "+v"(xa)::"memory");
          I8Raw raw;
          if (x32) i8_load<true>(raw, xa, i, a.cols);
          else i8_load<false>(raw, xa, i, a.cols);
          i8_convert(v[c], raw, a.xt);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[c][e] = e < n ? i8_gelu_tail(v[c][e]) : 0.f;
        }
        m = largest();
      }
    }
  }
  const float amax = __uint_as_float(m);
  const bool bad = m >= 0x7F800000u;
  const bool zero = bad || amax < 0x1p-100f;
  const float inv = zero ? 0.f : 127.f / amax;
  if (tid == 0) a.scale[row] = bad ? __uint_as_float(0x7FC00000u) : zero ? 0.f : amax / 127.f;
  int8_t* qr = a.q + row * a.ldq;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const int i = (tid + NTH * c) * 8, n = a.cols - i;
    if (n <= 0) continue;
    // |v inv| <= 127 (1 + 2^-23), which rounds to 127; two's complement in the low byte (bad and
    // zero rows: 0 whatever v is)
    uint32_t u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = i8_step(v[c][e], inv);
    uint32_t w[2];
#pragma unroll
    for (int d = 0; d < 2; ++d) {
      const uint32_t lo = __builtin_amdgcn_perm(u[4 * d + 1], u[4 * d], 0x0C0C0400u);
      const uint32_t hi = __builtin_amdgcn_perm(u[4 * d + 3], u[4 * d + 2], 0x0C0C0400u);
      w[d] = zero ? 0u : lo | hi << 16;
    }
    if (n >= 8) {                  // (q rows start on 16 bytes)
      typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));
      uintx2* p = reinterpret_cast<uintx2*>(qr + i);
      if constexpr (NT && NORM) __builtin_nontemporal_store(uintx2{w[0], w[1]}, p);
      else *p = uintx2{w[0], w[1]};
    } else
#pragma unroll
      for (int e = 0; e < 7; ++e) if (e < n) qr[i + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
  }
}

// out = q * scale, rounded once to the output's type.  One thread per 8 elements; the last 8 of a row
// that is no multiple of 8 overlap the ones before (the same values are stored twice).
template <bool NT>
__global__ void __launch_bounds__(256)
int8_to_rows_kernel(const int8_t* __restrict__ q, int64_t ldq, const float* __restrict__ scale, unsigned rows,
                    int cols, void* __restrict__ out, int ot, int64_t ldo) {
  const unsigned per = (unsigned)(cols + 7) >> 3;
  const unsigned id = blockIdx.x * 256 + threadIdx.x, row = id / per;            // (the host: below 2^32)
  if (row >= rows) return;
  const int i = min((int)(id - row * per) * 8, max(cols - 8, 0));
  const int8_t* qr = q + row * ldq + i;
  char* orow = reinterpret_cast<char*>(out) + row * ldo * (ot == HCR_F32 ? 4 : 2);
  const float s = scale[row];
  float v[8];
  if (cols >= 8) {
    typedef uint32_t uintx2_any __attribute__((ext_vector_type(2), aligned(1)));
    const uintx2_any w = *reinterpret_cast<const uintx2_any*>(qr);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)(int8_t)(w[e >> 2] >> (8 * (e & 3))) * s;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)qr[min(e, cols - 1)] * s;
  }
  i8_store<NT>(orow, ot, i, cols, v);
}

// -------------------------------------------------------------------------------------
// y[t][f] = (sum_k x[t][k] w[f][k]) * sx[t] * sw[f] + bias[f].  The sum is exact in int32
// (|x w| <= 2^14, K <= 131071), so any split of k gives the same bits; the conversion to fp32
// rounds it once (sums above 2^24), and y is rounded once more to its type.
// K need not fill a stage: w's bytes at k >= K are replaced by zeros in registers, so what the
// padding of either operand holds does not matter.
// -------------------------------------------------------------------------------------
__device__ __forceinline__ intx4 i8_mfma(intx4 a, intx4 b, intx4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// bytes of a 16-byte chunk that starts n bytes before the row's end, the others zero (n >= 16: all)
__device__ __forceinline__ intx4 i8_keep(intx4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int left = n - 4 * d;
    v[d] = left >= 4 ? v[d] : left <= 0 ? 0 : v[d] & (int)((1u << (8 * left)) - 1u);
  }
  return v;
}

// 4 consecutive features of token t
__device__ __forceinline__ void i8_store_out4(const I8LinearArgs& a, int64_t t, int f, const float (&v)[4]) {
  if (a.ot == HCR_F32) {
    float* p = reinterpret_cast<float*>(a.out) + t * a.ldo + f;
    if (a.vec && f + 4 <= a.N) *reinterpret_cast<float4*>(p) = float4{v[0], v[1], v[2], v[3]};
    else
#pragma unroll
      for (int r = 0; r < 4; ++r) if (f + r < a.N) p[r] = v[r];
    return;
  }
  const uint2 h = a.ot == HCR_BF16 ? uint2{i8_pack2<__bf16>(v[0], v[1]), i8_pack2<__bf16>(v[2], v[3])}
                                   : uint2{i8_pack2<_Float16>(v[0], v[1]), i8_pack2<_Float16>(v[2], v[3])};
  uint16_t* p = reinterpret_cast<uint16_t*>(a.out) + t * a.ldo + f;
  if (a.vec && f + 4 <= a.N) *reinterpret_cast<uint2*>(p) = h;
  else
#pragma unroll
    for (int r = 0; r < 4; ++r) if (f + r < a.N) p[r] = (uint16_t)((r < 2 ? h.x : h.y) >> (16 * (r & 1)));
}

// Operands straight from memory to the matrix cores: 16 FB features x 16 TB tokens per workgroup,
// whose KW waves take every KW-th 128-byte piece of the rows (a lane's 32 bytes are contiguous,
// a row's 128 bytes one line; the contraction order is the same for both operands) and add their
// int32 sums through LDS.
template <int FB, int TB, int KW>
__global__ void __launch_bounds__(64 * KW)
int8_linear_direct(I8LinearArgs a) {
  __shared__ __attribute__((aligned(16))) intx4 red[KW][FB * TB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int li = lane & 15, lg = lane >> 4;
  const unsigned nfb = (unsigned)((a.N + 16 * FB - 1) / (16 * FB));
  const int f0 = (int)(blockIdx.x % nfb) * (16 * FB), t0 = (int)(blockIdx.x / nfb) * (16 * TB);
  const int8_t* wr[FB];
  const int8_t* xr[TB];
#pragma unroll
  for (int c = 0; c < FB; ++c) wr[c] = a.w + (int64_t)min(f0 + 16 * c + li, a.N - 1) * a.ldw;
#pragma unroll
  for (int b = 0; b < TB; ++b) xr[b] = a.x + (int64_t)min(t0 + 16 * b + li, a.T - 1) * a.ldx;
  intx4 acc[FB][TB];
#pragma unroll
  for (int c = 0; c < FB; ++c)
#pragma unroll
    for (int b = 0; b < TB; ++b) acc[c][b] = intx4{0, 0, 0, 0};
  const int whole = a.K / 128 * 128;
  for (int k = wave * 128; k < whole; k += KW * 128) {
    intx4 w[FB][2], x[TB][2];
#pragma unroll
    for (int c = 0; c < FB; ++c)
#pragma unroll
      for (int j = 0; j < 2; ++j) w[c][j] = reinterpret_cast<const intx4*>(wr[c] + k + lg * 32)[j];
#pragma unroll
    for (int b = 0; b < TB; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j) x[b][j] = reinterpret_cast<const intx4*>(xr[b] + k + lg * 32)[j];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < FB; ++c)
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[c][b] = i8_mfma(w[c][j], x[b][j], acc[c][b]);
  }
  if (whole < a.K && (whole / 128) % KW == wave) {      // the rows' last, partial piece
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = whole + lg * 32 + j * 16, n = a.K - k;
      const int kk = n > 0 ? k : 0;                     // (a chunk past the row: any, times 0)
      intx4 x[TB];
#pragma unroll
      for (int b = 0; b < TB; ++b) x[b] = *reinterpret_cast<const intx4*>(xr[b] + kk);
#pragma unroll
      for (int c = 0; c < FB; ++c) {
        const intx4 w = i8_keep(*reinterpret_cast<const intx4*>(wr[c] + kk), n);
#pragma unroll
        for (int b = 0; b < TB; ++b) acc[c][b] = i8_mfma(w, x[b], acc[c][b]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < FB; ++c)
#pragma unroll
    for (int b = 0; b < TB; ++b) red[wave][c * TB + b][lane] = acc[c][b];
  __syncthreads();
  for (int i = wave; i < FB * TB; i += KW) {
    intx4 s = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < KW; ++w) s += red[w][i][lane];
    // lane: features f .. f + 3 of token t
    const int t = t0 + 16 * (i % TB) + li, f = f0 + 16 * (i / TB) + 4 * lg;
    if (t >= a.T || f >= a.N) continue;
    const float sx = a.sx[t];
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int fr = min(f + r, a.N - 1);
      v[r] = fmaf((float)s[r] * sx, a.sw[fr], a.bias ? a.bias[fr] : 0.f);
    }
    i8_store_out4(a, t, f, v);
  }
}

}  // namespace hcr
