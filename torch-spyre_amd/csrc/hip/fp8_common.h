// OCP e4m3 codes with one fp32 scale per group of 128 columns: what the 8-bit
// row kernels and products share.
#pragma once

#include "sph_common.h"

namespace sph {
namespace fp8 {

constexpr int kGroup = 128;        // columns of one scale
constexpr float kTop = 448.f;      // e4m3's largest finite value
// A group's largest magnitude counts as at least 2^-100, so that 448 / amax
// stays finite for groups of zeros and of tiny values.  As bits: magnitudes are
// compared as unsigned integers, which lets a NaN (its bits are above those of
// infinity) win, where fmaxf would drop it.
constexpr uint32_t kLeastBits = 0x0d800000u;

inline int64_t groups(int64_t cols) { return ceil_div(cols, kGroup); }

// A grid dimension holds fewer than 2^32 threads.
inline int check_grid(const char* what, int64_t workgroups, int64_t threads) {
  SPH_REQUIRE(workgroups <= UINT32_MAX / threads, SPH_ERR_TOO_LARGE,
              std::string(what) + ": more workgroups than a launch holds");
  return SPH_OK;
}

}  // namespace fp8
}  // namespace sph
