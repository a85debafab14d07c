// cache_args.h -- checks of sm120n_qk_cache_args shared by the Q/K norm + RoPE +
// KV store kernels.
#pragma once

#include <cstdint>

#include "sm120norm_b200.h"

namespace sm120n {

enum CacheKind : int { kNoCache = 0, kSameType = 1, kFp8 = 2 };

// Validates the arguments and says which kind of cache they store to.
int check_cache_args(const sm120n_qk_cache_args* a, int* cache_kind);

inline bool aligned_to(const void* p, uintptr_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace sm120n
