// fa2_host.h - host helpers that the library's translation units share.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>
#include <random>

#include "fa2_device.h"

namespace fa2 {

constexpr int kMaxDevices = 64;
inline std::once_flag g_cu_once[kMaxDevices];
inline int g_cu_count[kMaxDevices];

inline int cu_count_current_device() {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 256;
  std::call_once(g_cu_once[dev], [dev] {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
      n = 256;
    g_cu_count[dev] = n;
  });
  return g_cu_count[dev];
}

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline int elt_bytes(int dtype) { return dtype == FA2_DTYPE_F32 ? 4 : 2; }

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline bool stride_ok(int64_t s, int eb) { return ((s * eb) & 15) == 0; }

// Tag of one call's merge words (KArgs::merge_tag): a process-wide counter
// from a random start, skipping the values a cleared or all-ones word holds.
inline uint64_t next_merge_tag() {
  constexpr uint64_t kMask = (uint64_t(1) << kMergeTagBits) - 1;
  static std::atomic<uint64_t> next{[] {
    std::random_device rd;
    return (static_cast<uint64_t>(rd()) << 32) ^ rd();
  }()};
  for (;;) {
    const uint64_t t = next.fetch_add(1, std::memory_order_relaxed) & kMask;
    if (t != 0 && t != kMask) return t;
  }
}

}  // namespace fa2
