// How an expert's rows are divided into parts of a weight gradient; for host and device.
#pragma once

#include <cstdint>

#include "host_device.h"

namespace lgbm_b200 {
namespace experts {

// Rows of each of `parts` parts of n rows: whole blocks, as few as cover them. The last parts are
// shorter or empty.
LGBM_HOST_DEVICE int32_t part_rows(int32_t n, int32_t parts, int32_t block) {
  const int32_t blocks = n / block + (n % block != 0);
  return (blocks + parts - 1) / parts * block;
}

}  // namespace experts
}  // namespace lgbm_b200
