// One error word per device, written by kernels whose bounded waits give up
// (0 = ok, otherwise a code naming the wait site) or that meet an index in device memory
// outside its buffer, whose access they skip (codes from kIndexSite on).  Allocated on first use.
#pragma once
#include "common.h"

namespace rt {
constexpr int kIndexSite = 1000;
constexpr int kSiteCacheWrite = 1001, kSiteCacheRead = 1002, kSiteCachedAttention = 1003, kSiteToken = 1004;
int* device_error_word();
// Synchronises the device, reads and clears the word.
rt_status check_device_error(const char* what);
}  // namespace rt
