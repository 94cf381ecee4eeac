// Act8Copy: the 8-bit copy of an activation that a function keeps between its
// forward and its backward (the format is described at nblahip_act8_pack).
// Also the rows-by-columns view of the transformer-block functions.
#pragma once

#include <nbla/hip/common.hpp>
#include <nbla/nd_array.hpp>
#include <nbla/variable.hpp>

#include <algorithm>

namespace nbla {

// "" : none, "int8", "e4m3".
inline int act8_format(const string &checkpoint) {
  if (checkpoint.empty()) return NBLAHIP_ACT8_NONE;
  if (checkpoint == "int8") return NBLAHIP_ACT8_INT8;
  NBLA_CHECK(checkpoint == "e4m3", error_code::value,
             "checkpoint must be \"\", \"int8\" or \"e4m3\" (given \"%s\").", checkpoint.c_str());
  return NBLAHIP_ACT8_E4M3;
}

class Act8Copy {
  Variable codes_, scales_;

public:
  void reshape(Size_t rows, Size_t cols) {
    codes_.reshape(Shape_t{rows * cols}, true);
    scales_.reshape(Shape_t{rows * static_cast<Size_t>(nblahip_act8_scales_per_row(cols))}, true);
  }
  uint8_t *codes(const Context &ctx) {
    return codes_.data()->cast(dtypes::UBYTE, ctx, true)->pointer<uint8_t>();
  }
  uint8_t *scales(const Context &ctx) {
    return scales_.data()->cast(dtypes::UBYTE, ctx, true)->pointer<uint8_t>();
  }
  const uint8_t *kept_codes(const Context &ctx) {
    return codes_.data()->get(dtypes::UBYTE, ctx)->const_pointer<uint8_t>();
  }
  const uint8_t *kept_scales(const Context &ctx) {
    return scales_.data()->get(dtypes::UBYTE, ctx)->const_pointer<uint8_t>();
  }
};

// Rows (the batch axes, which must be the leading ones) and columns of x.
inline void rows_and_columns(const string &name, const Shape_t &shape, vector<int> &batch_axis,
                             Size_t &rows, Size_t &cols) {
  const int ndim = static_cast<int>(shape.size());
  NBLA_CHECK(!batch_axis.empty(), error_code::value, "batch_axis must not be empty.");
  for (int &b : batch_axis) {
    if (b < 0) b += ndim;
    NBLA_CHECK(b >= 0 && b < ndim, error_code::value, "batch_axis out of range.");
  }
  std::sort(batch_axis.begin(), batch_axis.end());
  rows = 1;
  for (size_t i = 0; i < batch_axis.size(); ++i) {
    NBLA_CHECK(batch_axis[i] == static_cast<int>(i), error_code::not_implemented,
               "%s: the batch axes must be the leading axes, each once.", name.c_str());
    rows *= shape[i];
  }
  cols = 1;
  for (size_t i = batch_axis.size(); i < shape.size(); ++i) cols *= shape[i];
  NBLA_CHECK(cols < (Size_t(1) << 27), error_code::value,
             "%s: fewer than 2^27 elements per row required.", name.c_str());
}

} // namespace nbla
