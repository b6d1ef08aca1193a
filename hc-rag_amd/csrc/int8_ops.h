// int8_ops.h — launchers of the 8-bit integer operators (int8_ops.hip), shared with the encoder.
// Arguments are checked by the C ABI entry points; these only choose a kernel and launch it.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace hcr {
struct I8RowArgs;
struct I8LinearArgs;
constexpr int kI8MaxRowCols = 32768;       // 16 waves x 4 chunks x 512 elements
constexpr int kI8MaxRows = 1 << 30;        // rows and features (32-bit row indices)
constexpr int64_t kI8MaxElements = (int64_t)1 << 40;   // of a product's or a dequantisation's result
constexpr int kI8MaxDepth = 131071;        // 2^14 K < 2^31: the int32 sums stay exact
int int8_rows_launch(int mode, const I8RowArgs& a, hipStream_t st);
int int8_linear_launch(const I8LinearArgs& a, hipStream_t st);
}  // namespace hcr
