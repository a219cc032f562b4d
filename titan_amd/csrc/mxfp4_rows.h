// The product of one mxfp4 matrix with a few rows (mxfp4_rows.hip).
#pragma once

#include "common.h"

namespace qmoe_mx {

constexpr int64_t kFewRows = 64;

struct RowsArgs {
  const uint16_t* x;      // bf16 rows, ldx elements apart
  const uint32_t* xq;     // or codes [n_x, K/8]
  const uint8_t* xs;      // and scales [n_x, K/32]
  const int32_t* x_rows;  // null: row m reads x[m]
  int64_t M, n_x, ldx;
  const uint32_t* w;
  const uint8_t* s;
  int64_t N, K;
  void* out;
  int out_f32;
};

// At most kFewRows rows; arguments checked by the caller.
int rows_product(const RowsArgs& a, bool qq, hipStream_t st);

}  // namespace qmoe_mx
