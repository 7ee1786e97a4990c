// The 8-bit KV cache: layout and conversions shared by the kernels that write, move and attend it.
//
// A row (slot, kv head) of K or V is hd e4m3 codes and one exponent byte b: value = code * 2^(b - 127), with
// the least power of two that keeps the row's largest magnitude at or below 448 (b >= 27). A power of two
// costs a float code at most one of its 16 binades and makes every step exact: x * 2^-e before the one
// rounding to four significant bits, and code * 2^e, which is a bf16 value, after it (infinity where the row's
// largest rounds to 2^128, from 1.9375 * 2^127 on).
//
// One (layer, sequence, kv head) holds max_len slots (a multiple of 64) of K and of V, hd bytes a slot, in
// 64-slot blocks stored as the attention's MFMA operands, 16 bytes a lane and 1 KiB a load:
//  K: tile (kt, p) lane (g * 16 + i) = K[slot 64b + 16 kt + i][64 p + 16 g .. + 16]: the A operands of
//     S^T = K Q^T for key tile kt and k-steps 2p (first 8 dims) and 2p + 1 (last 8).
//  V: tile dt lane (g * 16 + i), byte 8c + t = V[slot 64b + 32c + 16 (t / 4) + 4g + t % 4][16 dt + i]: the A
//     operands of O^T = V^T P^T for dim tile dt and key halves c. The scores leave the MFMA as keys 16 kt +
//     4g + e of lane group g, which is this order: they are the P^T operand without a move between lanes.
//  Exponents: byte 16 g + 4 kt + e of a block = slot 64b + 16 kt + 4g + e: a lane's sixteen keys are one load.
#pragma once
#include "common.h"

namespace ssd {

__device__ __forceinline__ size_t q8_k_off(int s, int d, int hd) {
  return ((size_t)((s >> 4) * (hd >> 6) + (d >> 6)) << 10) + ((((d >> 4) & 3) * 16 + (s & 15)) << 4) + (d & 15);
}
__device__ __forceinline__ size_t q8_v_off(int s, int d, int hd) {
  return ((size_t)((s >> 6) * (hd >> 4) + (d >> 4)) << 10) + ((((s >> 2) & 3) * 16 + (d & 15)) << 4) +
         (((s >> 5) & 1) << 3) + (((s >> 4) & 1) << 2) + (s & 3);
}
__device__ __forceinline__ int q8_x_off(int s) {
  return (s & ~63) + (((s >> 2) & 3) << 4) + (((s >> 4) & 3) << 2) + (s & 3);
}

// A launch holds at most 2^32 - 1 threads.
__host__ inline bool grid_too_large(int64_t workgroups, int threads) { return workgroups * threads > (int64_t)UINT32_MAX; }

constexpr int Q8_MIN_EXP = 27;  // exponent byte of 2^-100: codes, scales and their products stay normal numbers

// Exponent byte for a row whose largest finite magnitude is amax: 448 = 0.875 * 2^9, so with amax = f * 2^n,
// f in [1, 2), it is n - 8 where f <= 1.75 and n - 7 above.
__device__ __forceinline__ int q8_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int b = (int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return b < Q8_MIN_EXP ? Q8_MIN_EXP : b;
}
__device__ __forceinline__ float q8_scale(uint32_t b) { return __uint_as_float(b << 23); }
__device__ __forceinline__ float q8_inv_scale(int b) { return __uint_as_float((uint32_t)(254 - b) << 23); }

}  // namespace ssd
