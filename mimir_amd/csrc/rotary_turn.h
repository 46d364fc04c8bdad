// The angle of a rotary pair, from a position and a frequency in units of 2^-64 of a turn
// (prefixlm_rotary.hip says why); shared by the kernels that turn.
#pragma once

#include "prefixlm_common.h"

namespace mimir {

// cos and sin of 2 pi p / 2^64.
__device__ __forceinline__ void sincos_turn(uint64_t p, float& c, float& s) {
  const uint64_t quarter = p + (1ull << 61);                     // nearest quarter turn: its top two bits
  const int64_t r = (int64_t)(p - (quarter & (3ull << 62)));     // in [-2^61, 2^61)
  const float x = (float)(int)(r >> 30) * (float)(6.283185307179586 / 17179869184.0);  // 2 pi / 2^34
  const float y = x * x;
  const float sn = x * (1.f + y * (-1.f / 6 + y * (1.f / 120 + y * (-1.f / 5040 + y * (1.f / 362880)))));
  const float cs = 1.f + y * (-0.5f + y * (1.f / 24 + y * (-1.f / 720 + y * (1.f / 40320 + y * (-1.f / 3628800)))));
  const int n = (int)(quarter >> 62);
  const float a = n & 1 ? sn : cs, b = n & 1 ? cs : sn;
  c = n == 1 || n == 2 ? -a : a;
  s = n >= 2 ? -b : b;
}

}  // namespace mimir
