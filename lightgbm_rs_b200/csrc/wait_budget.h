// How long a bounded wait lasts; for host and device.
#pragma once

#include <cstdint>

#include "host_device.h"

namespace lgbm_b200 {
namespace experts {

// A wait looks at the clock every few polls and ends when its time is used up. The clock runs on
// while the process is switched off the device, which is no sign of a stuck wait, so the time
// between two looks counts as `kStep` at most: a hundred looks that found nothing are needed.
struct WaitBudget {
  static constexpr uint64_t kTotal = 2000000000;  // ns
  static constexpr uint64_t kStep = kTotal / 100;
  uint64_t last;  // the clock at the last look
  uint64_t left;

  LGBM_HOST_DEVICE explicit WaitBudget(uint64_t now) : last(now), left(kTotal) {}
  // False when the time is used up.
  LGBM_HOST_DEVICE bool spend(uint64_t now) {
    const uint64_t passed = now - last < kStep ? now - last : kStep;
    last = now;
    left = passed < left ? left - passed : 0;
    return left > 0;
  }
};

}  // namespace experts
}  // namespace lgbm_b200
