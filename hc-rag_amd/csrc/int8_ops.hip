// int8_ops.hip — host side of the 8-bit integer operators' C ABI (include/hcrag.h): argument
// checks and the choice of a kernel.  Nothing here allocates, synchronises or keeps state, so
// every call can be captured into a graph and run from several threads and streams at once.
#include <hip/hip_runtime.h>

#include <initializer_list>

#include "int8_kernels.h"
#include "int8_gemm.h"
#include "int8_ops.h"
#include "host_common.h"

using namespace hcr;

namespace hcr {

// What a call reads or writes beyond the 256 MiB of the memory-side cache is evicted before its next
// use, so it goes past the caches (quantisation of 65521 x 4096 f16 137 us, so 116; dequantisation
// 138, 116; RMS norm 328, 317; with GELU 160, 156).  Below that the next kernel pays more than this
// one gains: 65521 x 768 f16, dequantisation and an addition 70 us, 77 so; quantisation and a product 70, 76.
constexpr int64_t kNtBytes = (int64_t)256 << 20;

constexpr int64_t kLaunchThreads = (int64_t)1 << 31;   // per launch; a grid of 2^32 threads is refused

template <int MODE, int WAVES, int NCH, bool NT>
static void launch_rows_nt(const I8RowArgs& a, hipStream_t st) {
  constexpr int64_t most = kLaunchThreads / (64 * WAVES);        // rows per launch
  for (int64_t r = 0; r < a.rows; r += most) {
    I8RowArgs c = a;
    c.row0 = r;
    c.rows = std::min(most, a.rows - r);
    const unsigned grid = WAVES == 1 ? (unsigned)((c.rows + 3) / 4) : (unsigned)c.rows;
    hipLaunchKernelGGL((rows_to_int8_kernel<MODE, WAVES, NCH, NT>), dim3(grid), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0,
                       st, c);
  }
}
template <int MODE, int WAVES, int NCH>
static void launch_rows(const I8RowArgs& a, hipStream_t st) {
  const int64_t n = a.rows * a.cols;
  const int64_t in = n * (i8_size(a.xt) + (a.r ? i8_size(a.rt) : 0));
  const int64_t out = n * (1 + (a.sum ? i8_size(a.rt) : 0) + (a.y ? i8_size(a.yt) : 0));
  if (std::max(in, out) >= kNtBytes) launch_rows_nt<MODE, WAVES, NCH, true>(a, st);
  else launch_rows_nt<MODE, WAVES, NCH, false>(a, st);
}
// The narrowest layout that holds a row.  Up to 2048 columns a wave per row (a workgroup per row
// pays its barriers three times: 60000 x 384 LayerNorm 45 us, 89 with 4 waves a row; 65536 x 2048
// RMS 172, 184), above that 2 chunks per thread (30000 x 8192 RMS 313 us, 349 with 4 waves x 4 chunks,
// 416 with 16 x 1; 20000 x 16384: 449, 493 with 16 x 4).  Idle lanes cost where arithmetic counts (GELU of
// 65521 x 5000: 6 waves 240 us, 8 waves 281; 65521 x 2560: 3 waves 119, 4 waves 145).
template <int MODE>
static void launch_rows_mode(const I8RowArgs& a, hipStream_t st) {
  if (a.cols <= 512) launch_rows<MODE, 1, 1>(a, st);
  else if (a.cols <= 1024) launch_rows<MODE, 1, 2>(a, st);
  else if (a.cols <= 2048) launch_rows<MODE, 1, 4>(a, st);
  else if (a.cols <= 3 * 1024) launch_rows<MODE, 3, 2>(a, st);
  else if (a.cols <= 4096) launch_rows<MODE, 4, 2>(a, st);
  else if (a.cols <= 6 * 1024) launch_rows<MODE, 6, 2>(a, st);
  else if (a.cols <= 8192) launch_rows<MODE, 8, 2>(a, st);
  else if (a.cols <= 16384) launch_rows<MODE, 16, 2>(a, st);
  else launch_rows<MODE, 16, 4>(a, st);
}

int int8_rows_launch(int mode, const I8RowArgs& a, hipStream_t st) {
  if (mode == I8_QUANT) launch_rows_mode<I8_QUANT>(a, st);
  else if (mode == I8_GELU) launch_rows_mode<I8_GELU>(a, st);
  else if (mode == I8_LAYER) launch_rows_mode<I8_LAYER>(a, st);
  else launch_rows_mode<I8_RMS>(a, st);
  HIPC(hipGetLastError());
  return HCR_OK;
}

template <int FB, int TB, int KW>
static int launch_direct(const I8LinearArgs& a, hipStream_t st) {
  const int64_t blocks = (int64_t)((a.N + 16 * FB - 1) / (16 * FB)) * ((a.T + 16 * TB - 1) / (16 * TB));
  hipLaunchKernelGGL((int8_linear_direct<FB, TB, KW>), dim3((unsigned)blocks), dim3(64 * KW), 0, st, a);
  HIPC(hipGetLastError());
  return HCR_OK;
}
static int64_t tiles_of(const I8LinearArgs& a, int features, int tokens) {
  return (int64_t)((a.N + features - 1) / features) * ((a.T + tokens - 1) / tokens);
}
template <int OT, bool ODD, int MT, int WM, int WN, int NST, int OCC, bool NT = false>
static void launch_tile(const I8LinearArgs& a, hipStream_t st) {
  constexpr int FT = 16 * MT * WM, TT = 64 * WN;
  hipLaunchKernelGGL((int8_linear_tiles<OT, ODD, MT, WM, WN, NST, OCC, NT>), dim3((unsigned)tiles_of(a, FT, TT)),
                     dim3(64 * WM * WN), 0, st, a, (a.N + FT - 1) / FT);
}
// Results of kNtBytes and more (T = 65536, K = 1024, N = 4096, f16, 512 MiB: 319 us, so 297; T = 24576, 192 MiB:
// 112, 115), unless rows are no whole number of 16 bytes (T = 30001, K = 777, N = 2051, f32: 127, 268).
static bool nt_out(const I8LinearArgs& a) { return (int64_t)a.T * a.N * i8_size(a.ot) >= kNtBytes; }

// The widest tile that leaves every CU one, down to 64 x 128 (features x tokens; us on MI355X):
//   64 x 128   4 waves of 32 x 64: a round takes 2.75 + 0.235 per 64 of depth (T = 2000, N = 1024, K = 4096:
//              18.5, 128 x 128 22.8, 128 x 256 31.1; T = 4000: 30.3, 24.0, 31.7; T = 1000, N = 768, K = 768:
//              5.7, 6.7, 9.5)
//   128 x 128  8 waves of 32 x 64
//   128 x 256  8 waves of 64 x 64, two workgroups per CU (T = 6000, N = 1024, K = 4096: 33.1, 128 x 128 36.6;
//              T = 21853, N = 768, K = 768: 27.4, 4 waves of 128 x 64 29.4, alternating wave groups as in
//              the streaming kernel 26.4, but 5 % behind at K = 384)
template <int OT, bool ODD>
static void launch_tiles(const I8LinearArgs& a, hipStream_t st) {
  if (tiles_of(a, 64, 128) <= 256) launch_tile<OT, ODD, 2, 2, 2, 4, 3>(a, st);
  else if (tiles_of(a, 128, 128) <= 256) launch_tile<OT, ODD, 2, 4, 2, 4, 4>(a, st);
  else if (!ODD && nt_out(a)) launch_tile<OT, ODD, 4, 2, 4, 3, 4, !ODD>(a, st);
  else launch_tile<OT, ODD, 4, 2, 4, 3, 4>(a, st);
}
template <int OT, bool ODD>
static void launch_stream(const I8LinearArgs& a, hipStream_t st) {
  const int nft = (a.N + 255) / 256;
  const unsigned tiles = (unsigned)nft * ((a.T + 255) / 256);
  const dim3 grid(std::min((tiles + 7) & ~7u, 256u));
  if (!ODD && nt_out(a)) hipLaunchKernelGGL((int8_linear_stream<OT, ODD, !ODD>), grid, dim3(512), 0, st, a, nft, tiles);
  else hipLaunchKernelGGL((int8_linear_stream<OT, ODD, false>), grid, dim3(512), 0, st, a, nft, tiles);
}
template <int OT>
static void launch_linear(const I8LinearArgs& a, bool stream, hipStream_t st) {
  const bool odd = a.N % (16 / i8_size(OT)) != 0;
  if (stream) odd ? launch_stream<OT, true>(a, st) : launch_stream<OT, false>(a, st);
  else odd ? launch_tiles<OT, true>(a, st) : launch_tiles<OT, false>(a, st);
}

// Features and tokens per workgroup of the direct kernel, in 16s: the wider the less it reads for an
// output, as long as the device is filled (us on MI355X; G the number of workgroups):
//   2 x 4  from 256 of them at depths where reading dominates (T = 512, N = 1024, K = 4096: 14.4, with
//          2 x 2 17.3; K = 384, N = 1152: 5.4, 4.9)
//   2 x 2  from 144 (T = 256, N = 768, K = 768: 4.0, with 1 x 2 4.5; T = 128, G = 96: 3.9, 3.5)
//   1 x 2  from 192 (T = 128, N = 1024, K = 4096: 8.0, with 1 x 1 9.6; T = 64, G = 128: 7.8, 5.9)
static int launch_direct_for(const I8LinearArgs& a, hipStream_t st) {
  auto groups = [&](int fb, int tb) { return (int64_t)((a.N + 16 * fb - 1) / (16 * fb)) * ((a.T + 16 * tb - 1) / (16 * tb)); };
  if (a.T > 16) {
    if (a.K >= 1024 && groups(2, 4) >= 256) return launch_direct<2, 4, 4>(a, st);
    if (groups(2, 2) >= 144) return launch_direct<2, 2, 4>(a, st);
    if (groups(1, 2) >= 192) return launch_direct<1, 2, 4>(a, st);
  }
  return launch_direct<1, 1, 4>(a, st);
}

// Which kernel (us on MI355X, f16 results):
//   direct  up to 2^19 outputs of at most 16 MiB of x: its time grows with the work from 2.6 us on (about
//           280 TOP/s), that of a round of small tiles is 2.75 + 0.235 per 64 of depth whatever there is
//           to do (T = 512, N = 768, K = 768: 5.3, tiles 5.6; T = 768: 6.6, 5.6; T = 512, N = 1024, K = 4096:
//           14.0, 16.9; T = 768: 24.4, 17.6); many narrow rows are read from memory once per 32 features
//           (T = 10000, N = 130, K = 4096: 55, tiles 31)
//   stream  where its 256 x 256 tiles fill its rounds (one per CU) to 3/4 at a depth of 1024, to 9/10
//           from 768 on: a round takes 5.6 + 0.88 per 64 of depth, 512 tiles 2 + 1.15 (T = 65536,
//           N = 4096, K = 1024: 324, tiles 420; T = 8192, N = 2048, K = 2048: 36, tiles 41; T = 65536,
//           N = 2304, K = 768: 163, tiles 202; 1.34 rounds, T = 21853, N = 1024, K = 1024: 36, tiles 33)
//   tiles   otherwise
// A last round of at most 1/4 of its tiles is cut off: the tokens that the full rounds do not cover are
// a product of their own (T = 21853, N = 2304, K = 768, 3.02 rounds: 56 us, so 51; T = 16400, N = 1024,
// K = 4096: 92, 66).
int int8_linear_launch(const I8LinearArgs& a, hipStream_t st) {
  // rows of w, x and out that 31-bit byte offsets reach, in whole tiles
  const int64_t fmost = INT32_MAX / a.ldw / 256 * 256;
  const int64_t tmost = INT32_MAX / std::max<int64_t>(a.ldx, a.ldo * i8_size(a.ot)) / 256 * 256;
  const bool near = fmost > 0 && tmost > 0;
  const int64_t fstep = std::min<int64_t>(near ? fmost : a.N, 1 << 22);
  // (far: the direct kernel's offsets have 64 bits; its workgroups take 32 features at most and a thread 4
  // outputs, so 2^30 tokens x features, in whole 32s of features, are 2^28 threads, and 512 tokens 2^29)
  const int64_t fwide = (std::min<int64_t>(a.N, fstep) + 31) / 32 * 32;
  const int64_t tstep = near ? tmost : std::max<int64_t>((1 << 30) / fwide / 64 * 64, 512);
  for (int64_t f = 0; f < a.N; f += fstep) {
    I8LinearArgs c = a;
    c.N = (int)std::min(fstep, a.N - f);
    c.w = a.w + f * a.ldw;
    c.sw = a.sw + f;
    if (a.bias) c.bias = a.bias + f;
    for (int64_t t = 0; t < a.T; t += c.T) {
      c.T = (int)std::min(tstep, a.T - t);
      c.x = a.x + t * a.ldx;
      c.sx = a.sx + t;
      c.out = static_cast<char*>(a.out) + (t * a.ldo + f) * i8_size(a.ot);
      if (!near || ((int64_t)c.T * c.N <= 1 << 19 && (int64_t)c.T * c.K <= 16 << 20)) {
        CHECK(launch_direct_for(c, st));
        continue;
      }
      const int64_t nf = (c.N + 255) / 256, nt = (c.T + 255) / 256, over = nf * nt % 256;
      const int64_t full = nf * nt / 256 * 256 / nf * 256;         // tokens that the full rounds cover
      if (full > 0 && over > 0 && over <= 64 && full < c.T) c.T = (int)full;
      const int64_t big = nf * ((c.T + 255) / 256), slots = (big + 255) / 256 * 256;
      const bool stream = c.K >= 1024 ? big * 4 >= slots * 3 : c.K >= 768 && big * 10 >= slots * 9;
      if (c.ot == HCR_F32) launch_linear<HCR_F32>(c, stream, st);
      else if (c.ot == HCR_BF16) launch_linear<HCR_BF16>(c, stream, st);
      else launch_linear<HCR_F16>(c, stream, st);
      HIPC(hipGetLastError());
    }
  }
  return HCR_OK;
}

}  // namespace hcr

static size_t float_size(int dt) { return dt == HCR_F32 ? 4 : 2; }
static bool is_float(int dt) { return dt == HCR_F16 || dt == HCR_BF16 || dt == HCR_F32; }
static bool on(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// a [rows][cols] operand of a floating type: its type, stride and alignment
static int check_floats(const char* what, const void* p, int dt, int64_t ld, int64_t cols) {
  if (!is_float(dt)) return hcr_set_errorf(HCR_EINVAL, "%s: dtype must be HCR_F16, HCR_BF16 or HCR_F32, got %d", what, dt);
  if (ld < cols) return hcr_set_errorf(HCR_EINVAL, "%s: row stride %lld is below %lld columns", what, (long long)ld, (long long)cols);
  if (!on(p, float_size(dt))) return hcr_set_errorf(HCR_EINVAL, "%s: not aligned to its elements", what);
  return HCR_OK;
}
static int check_int8(const char* what, const void* p, int64_t ld, int64_t cols) {
  if (ld < cols) return hcr_set_errorf(HCR_EINVAL, "%s: row stride %lld is below %lld columns", what, (long long)ld, (long long)cols);
  if (!on(p, 16) || (ld & 15))
    return hcr_set_errorf(HCR_EINVAL, "%s: int8 rows must start on 16 bytes (aligned pointer, row stride a multiple of 16)", what);
  return HCR_OK;
}
static int check_rows(int64_t rows, int64_t cols, int64_t max_cols) {
  if (rows < 0 || rows > kI8MaxRows) return hcr_set_errorf(HCR_EINVAL, "rows must be in [0, 2^30], got %lld", (long long)rows);
  if (cols < 1 || cols > max_cols) return hcr_set_errorf(HCR_EINVAL, "cols must be in [1, %lld], got %lld", (long long)max_cols, (long long)cols);
  return HCR_OK;
}
// rows in one buffer as another operand's: the same element for element, or refused
static int check_same(const char* what, const void* p, int dt, int64_t ld, const char* other, const void* o, int odt, int64_t old) {
  if (p && p == o && (dt != odt || ld != old))
    return hcr_set_errorf(HCR_EINVAL, "%s in the buffer of %s: needs its dtype and row stride", what, other);
  return HCR_OK;
}
struct Operand { const char* what; const void* p; };
static int check_apart(const Operand& out, std::initializer_list<Operand> others) {
  for (const Operand& o : others)
    if (out.p && out.p == o.p) return hcr_set_errorf(HCR_EINVAL, "%s and %s must not overlap", out.what, o.what);
  return HCR_OK;
}

extern "C" int hcr_quant_rows_device(const void* d_x, int x_dtype, int64_t ldx, int64_t rows, int64_t cols, int act,
                                     int8_t* d_q, int64_t ldq, float* d_scale, void* stream) {
  CHECK(check_rows(rows, cols, kI8MaxRowCols));
  if (act != HCR_ACT_NONE && act != HCR_ACT_GELU) return hcr_set_errorf(HCR_EINVAL, "unknown activation %d", act);
  if (rows == 0) return HCR_OK;
  if (!d_x || !d_q || !d_scale) return hcr_set_error(HCR_EINVAL, "NULL buffer");
  CHECK(check_floats("x", d_x, x_dtype, ldx, cols));
  CHECK(check_int8("q", d_q, ldq, cols));
  if (!on(d_scale, 4)) return hcr_set_error(HCR_EINVAL, "scale: not aligned to its elements");
  CHECK(check_apart({"q", d_q}, {{"x", d_x}}));
  CHECK(check_apart({"scale", d_scale}, {{"x", d_x}, {"q", d_q}}));
  I8RowArgs a{};
  a.x = d_x; a.ldx = ldx; a.xt = x_dtype;
  a.q = d_q; a.ldq = ldq; a.scale = d_scale; a.rows = rows; a.cols = (int)cols;
  return int8_rows_launch(act == HCR_ACT_GELU ? I8_GELU : I8_QUANT, a, (hipStream_t)stream);
}

extern "C" int hcr_norm_quant_rows_device(const hcr_norm_quant_args* args, void* stream) {
  if (!args) return hcr_set_error(HCR_EINVAL, "args is NULL");
  const hcr_norm_quant_args& n = *args;
  CHECK(check_rows(n.rows, n.cols, kI8MaxRowCols));
  if (n.norm != HCR_NORM_LAYER && n.norm != HCR_NORM_RMS) return hcr_set_errorf(HCR_EINVAL, "unknown norm %d", n.norm);
  if (!(n.eps >= 0.f)) return hcr_set_error(HCR_EINVAL, "eps must be >= 0");
  if (n.sum && !n.residual) return hcr_set_error(HCR_EINVAL, "a sum output needs a residual");
  if (n.rows == 0) return HCR_OK;
  if (!n.x || !n.weight || !n.q || !n.scale) return hcr_set_error(HCR_EINVAL, "NULL buffer");
  CHECK(check_floats("x", n.x, n.x_dtype, n.ldx, n.cols));
  if (n.residual) CHECK(check_floats("residual", n.residual, n.residual_dtype, n.ldr, n.cols));
  if (n.sum) CHECK(check_floats("sum", n.sum, n.residual_dtype, n.ldsum, n.cols));
  if (n.norm_out) CHECK(check_floats("norm output", n.norm_out, n.norm_dtype, n.ldnorm, n.cols));
  CHECK(check_int8("q", n.q, n.ldq, n.cols));
  if (!on(n.scale, 4) || !on(n.weight, 4) || !on(n.bias, 4))
    return hcr_set_error(HCR_EINVAL, "scale, weight or bias: not aligned to its elements");
  CHECK(check_same("the sum", n.sum, n.residual_dtype, n.ldsum, "the residual", n.residual, n.residual_dtype, n.ldr));
  CHECK(check_same("the norm output", n.norm_out, n.norm_dtype, n.ldnorm, "x", n.x, n.x_dtype, n.ldx));
  CHECK(check_same("the norm output", n.norm_out, n.norm_dtype, n.ldnorm, "the residual", n.residual, n.residual_dtype, n.ldr));
  const Operand x{"x", n.x}, residual{"the residual", n.residual}, weight{"weight", n.weight}, bias{"bias", n.bias},
      sum{"the sum", n.sum}, norm_out{"the norm output", n.norm_out}, q{"q", n.q};
  CHECK(check_apart(sum, {x, weight, bias, norm_out}));
  CHECK(check_apart(norm_out, {weight, bias}));
  CHECK(check_apart(q, {x, residual, weight, bias, sum, norm_out}));
  CHECK(check_apart({"scale", n.scale}, {x, residual, weight, bias, sum, norm_out, q}));
  I8RowArgs a{};
  a.x = n.x; a.ldx = n.ldx; a.xt = n.x_dtype;
  a.r = n.residual; a.ldr = n.ldr; a.rt = n.residual ? n.residual_dtype : HCR_F32;
  a.sum = n.sum; a.ldsum = n.ldsum;
  a.y = n.norm_out; a.ldy = n.ldnorm; a.yt = n.norm_dtype;
  a.g = n.weight; a.b = n.bias; a.eps = n.eps;
  a.q = n.q; a.ldq = n.ldq; a.scale = n.scale; a.rows = n.rows; a.cols = (int)n.cols;
  return int8_rows_launch(n.norm == HCR_NORM_LAYER ? I8_LAYER : I8_RMS, a, (hipStream_t)stream);
}

extern "C" int hcr_dequant_rows_device(const int8_t* d_q, int64_t ldq, const float* d_scale, int64_t rows, int64_t cols,
                                       void* d_out, int out_dtype, int64_t ldo, void* stream) {
  CHECK(check_rows(rows, cols, kI8MaxDepth));
  if (rows == 0) return HCR_OK;
  if (!d_q || !d_scale || !d_out) return hcr_set_error(HCR_EINVAL, "NULL buffer");
  CHECK(check_int8("q", d_q, ldq, cols));
  CHECK(check_floats("out", d_out, out_dtype, ldo, cols));
  if (!on(d_scale, 4)) return hcr_set_error(HCR_EINVAL, "scale: not aligned to its elements");
  CHECK(check_apart({"out", d_out}, {{"q", d_q}, {"scale", d_scale}}));
  if (rows * cols > kI8MaxElements) return hcr_set_error(HCR_EINVAL, "more than 2^40 elements");
  const int64_t per = (cols + 7) / 8, most = kLaunchThreads / per;   // threads per row, rows per launch
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = std::min(most, rows - r);
    auto kernel = rows * cols * (int64_t)float_size(out_dtype) >= kNtBytes ? int8_to_rows_kernel<true> : int8_to_rows_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)((n * per + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                       d_q + r * ldq, ldq, d_scale + r, (unsigned)n, (int)cols,
                       static_cast<char*>(d_out) + r * ldo * (int64_t)float_size(out_dtype), out_dtype, ldo);
    HIPC(hipGetLastError());
  }
  return HCR_OK;
}

extern "C" int hcr_int8_linear_device(const int8_t* d_x, int64_t ldx, const float* d_x_scale, int64_t rows,
                                      const int8_t* d_w, int64_t ldw, const float* d_w_scale, int64_t features,
                                      int64_t depth, const float* d_bias, void* d_out, int out_dtype, int64_t ldo,
                                      void* stream) {
  CHECK(check_rows(rows, depth, kI8MaxDepth));
  if (features < 0 || features > kI8MaxRows)
    return hcr_set_errorf(HCR_EINVAL, "features must be in [0, 2^30], got %lld", (long long)features);
  if (rows == 0 || features == 0) return HCR_OK;
  if (!d_x || !d_x_scale || !d_w || !d_w_scale || !d_out) return hcr_set_error(HCR_EINVAL, "NULL buffer");
  CHECK(check_int8("x", d_x, ldx, depth));
  CHECK(check_int8("w", d_w, ldw, depth));
  CHECK(check_floats("out", d_out, out_dtype, ldo, features));
  if (!on(d_x_scale, 4) || !on(d_w_scale, 4) || !on(d_bias, 4))
    return hcr_set_error(HCR_EINVAL, "scales or bias: not aligned to their elements");
  CHECK(check_apart({"out", d_out}, {{"x", d_x}, {"w", d_w}, {"x's scale", d_x_scale}, {"w's scale", d_w_scale}, {"bias", d_bias}}));
  if (rows * features > kI8MaxElements) return hcr_set_error(HCR_EINVAL, "more than 2^40 outputs");
  I8LinearArgs a{};
  a.x = d_x; a.ldx = ldx; a.sx = d_x_scale;
  a.w = d_w; a.ldw = ldw; a.sw = d_w_scale;
  a.bias = d_bias; a.out = d_out; a.ldo = ldo; a.ot = out_dtype;
  a.T = (int)rows; a.N = (int)features; a.K = (int)depth;
  a.vec = ldo % 4 == 0 && on(d_out, 4 * float_size(out_dtype));
  return int8_linear_launch(a, (hipStream_t)stream);
}
