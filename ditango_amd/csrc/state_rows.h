// Rows of an attention state between the two layouts of its lse.
#pragma once

#include "dt_common.h"

namespace dt {

struct RowIndex {         // row ((b * Sq) + s) * H + h of B * Sq * H < 2^31 -> its place in the [B,H,Sq] layout
  int32_t Sq, H;
  uint32_t rows;          // B * Sq * H
  Quotient by_h, by_s;
};
__device__ __forceinline__ uint32_t bhs_of(const RowIndex& at, uint32_t row) {
  const uint32_t bs = quotient(row, at.by_h), h = row - bs * (uint32_t)at.H;
  const uint32_t b = quotient(bs, at.by_s), q = bs - b * (uint32_t)at.Sq;
  return (b * (uint32_t)at.H + h) * (uint32_t)at.Sq + q;
}
__device__ __forceinline__ uint32_t bsh_of(const RowIndex& at, uint32_t row) {   // the other way round
  const uint32_t bh = quotient(row, at.by_s), q = row - bh * (uint32_t)at.Sq;
  const uint32_t b = quotient(bh, at.by_h), h = bh - b * (uint32_t)at.H;
  return (b * (uint32_t)at.Sq + q) * (uint32_t)at.H + h;
}
static RowIndex row_index(int B, int Sq, int H) {
  RowIndex at{};
  at.Sq = Sq;
  at.H = H;
  at.rows = (uint32_t)((int64_t)B * Sq * H);
  at.by_h = quotient_by(H);
  at.by_s = quotient_by(Sq);
  return at;
}
}  // namespace dt
