// int8_args.h — what the kernels of the 8-bit integer operators are given (int8_kernels.h,
// int8_gemm.h); the C ABI's checks and the encoder fill these in.
#pragma once
#include <cstdint>

namespace hcr {

// what a row kernel computes before it quantises
enum : int { I8_QUANT = 0, I8_GELU = 1, I8_LAYER = 2, I8_RMS = 3 };

struct I8RowArgs {
  const void* x; int64_t ldx;
  const void* r; int64_t ldr;      // residual (NULL: none)
  void* sum; int64_t ldsum;        // h in r's type (NULL: not stored); may be r itself
  void* y; int64_t ldy;            // v in yt (NULL: not stored); may be x or r itself
  const float* g; const float* b;  // (b NULL: 0)
  int8_t* q; int64_t ldq;
  float* scale;
  int64_t rows, row0;              // rows [row0, row0 + rows) (the host cuts very long calls)
  int cols;
  float eps;
  int xt, rt, yt;                  // hcr_dtype of x, r (and sum), y
};

struct I8LinearArgs {
  const int8_t* x; int64_t ldx; const float* sx;
  const int8_t* w; int64_t ldw; const float* sw;
  const float* bias;               // (NULL: 0)
  void* out; int64_t ldo; int ot;  // hcr_dtype of out
  int T, N, K;
  int vec;                         // out's rows start on 4 elements
};

}  // namespace hcr
