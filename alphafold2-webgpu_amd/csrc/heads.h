// What the operators over [batch][tokens][heads][channels] share: strides in
// bytes and the checks of their descriptors (rotary.hip, window.hip).
#pragma once

#include "internal.h"

namespace afhip {

constexpr int kMaxHeadDim = 128;

// afhip_strides in bytes, packed ones filled in.
struct HeadStrides {
  int64_t batch, token, head;
};

inline HeadStrides head_strides(const afhip_strides& s, int64_t tokens, int64_t heads, int64_t channels, int dtype) {
  const int64_t es = (int64_t)dtype_size(dtype);
  if (s.token == 0) return {tokens * heads * channels * es, heads * channels * es, channels * es};
  return {s.batch * es, s.token * es, s.head * es};
}

// Strides that 16-byte accesses of whole rows can take, and 64 rows of which
// stay within a buffer's 2 GiB; what is written has no two elements in one
// place along an axis.
inline int check_strides(const char* name, const HeadStrides& s, int64_t batch, int64_t tokens, int64_t heads,
                         int64_t channels, int dtype, bool written) {
  const int64_t row = channels * (int64_t)dtype_size(dtype);
  AFHIP_REQUIRE(s.batch >= 0 && s.token >= 0 && s.head >= 0, "%s has a negative stride", name);
  AFHIP_REQUIRE(((s.batch | s.token | s.head) & 15) == 0, "%s has a stride that is not a multiple of 16 bytes", name);
  AFHIP_REQUIRE(s.token <= ((int64_t)1 << 24), "%s has a token stride of more than 16 MiB", name);
  AFHIP_REQUIRE(s.batch <= ((int64_t)1 << 46) && s.head <= ((int64_t)1 << 46), "%s has a stride that is too large",
                name);
  if (tokens > 1) AFHIP_REQUIRE(s.token >= row, "%s has tokens that overlap", name);
  if (written) {
    // From the narrowest axis on, each stride clears all that the ones before reach.
    int64_t stride[] = {s.batch, s.token, s.head}, count[] = {batch, tokens, heads}, reach = row;
    for (int left = 3; left > 0; left--) {
      int n = 0;
      for (int i = 1; i < left; i++)
        if (stride[i] < stride[n]) n = i;
      if (count[n] > 1) {
        AFHIP_REQUIRE(stride[n] >= reach, "%s is written, and has entries that overlap", name);
        reach += (count[n] - 1) * stride[n];
      }
      stride[n] = stride[left - 1];
      count[n] = count[left - 1];
    }
  }
  return AFHIP_OK;
}

inline int check_address(const char* name, const void* p) {
  AFHIP_REQUIRE(p != nullptr, "%s is NULL", name);
  AFHIP_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "%s is not aligned to 16 bytes", name);
  return AFHIP_OK;
}

// A launch has fewer than 2^32 threads.
inline int check_grid(int64_t groups, int threads) {
  AFHIP_REQUIRE(groups * threads < ((int64_t)1 << 32), "%lld workgroups of %d threads are too many for one launch",
                (long long)groups, threads);
  return AFHIP_OK;
}

}  // namespace afhip
