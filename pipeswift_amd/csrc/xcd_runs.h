// How equal runs of work fall on the eight XCDs: plain arithmetic, for kernels
// (cached_queries.h), their launches and the host alike.
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define PSK_HOST_DEVICE __host__ __device__
#else
#define PSK_HOST_DEVICE
#endif

namespace psk_detail {

// Workgroups that share a step's runs, of `slots` at most where that leaves whole
// rounds of the XCDs: run_of_xcd() reaches every run of such a launch, and of no other.
PSK_HOST_DEVICE constexpr int64_t xcd_rounds(int64_t slots) { return slots < 8 ? 8 : slots / 8 * 8; }

// The idx-th of `runs` runs on an XCD, consecutive ones on each; `runs` where it has
// no more.
PSK_HOST_DEVICE constexpr int64_t run_of_xcd(int64_t runs, int64_t xcd, int64_t idx) {
  const int64_t per = (runs + 7) >> 3;
  return idx < per ? xcd * per + idx : runs;
}

}  // namespace psk_detail
