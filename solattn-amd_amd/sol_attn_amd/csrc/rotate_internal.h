// Parameter block and launcher of the heads' rotation and norms (rotate.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace sol {

// One of Q and K: its rows and where they go, by element strides, and its norm.
struct RotateOperand {
  const uint16_t* rows;
  uint16_t* out;
  int64_t sb, st, sh;     // of rows: {batch, token, head}
  int64_t ob, ot, oh;     // of out
  const void* weight;     // [D] fp32 or BF16, null: no norm
  int heads;              // 0: none
};

struct RotateParams {
  RotateOperand x[2];
  const int32_t* positions;  // [batch, tokens, axes], the axes contiguous
  int64_t pb, pt;            // its element strides
  const double* frequencies; // [D / 2]
  const int32_t* axis;       // [D / 2]
  int axes, tokens;          // tokens of a batch entry
  int64_t rows;              // batch * tokens
  int weights_bf16;
  float eps;
};

hipError_t launch_rotate(const RotateParams& p, int D, bool pairs, hipStream_t stream);

}  // namespace sol
