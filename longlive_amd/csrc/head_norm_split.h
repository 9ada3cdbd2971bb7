// How the tokens of ll_head_norm_rope are divided over launches: host arithmetic.
#pragma once
#include <stdint.h>

namespace ll {

constexpr int kHeadNormThreads = 256;
// Waves of a launch: HIP takes fewer than 2^32 threads, 2^26 waves, in a dimension of the grid.
constexpr int64_t kHeadNormMostWaves = 1ll << 25;

// Tokens of a launch at most, of which each takes `per_token` waves.
inline int64_t head_norm_tokens(uint32_t per_token) { return kHeadNormMostWaves / per_token; }
// Workgroups of a launch of so many tokens.
inline uint32_t head_norm_groups(int64_t tokens, uint32_t per_token) {
  constexpr int64_t kWaves = kHeadNormThreads / 64;
  return (uint32_t)((tokens * per_token + kWaves - 1) / kWaves);
}

}  // namespace ll
