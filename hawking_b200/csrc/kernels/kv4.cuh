// Inside of a unit of the 4-bit paged KV cache: 16 tokens of one kv head, 18 * HD bytes.
//
// A value is c + s * (code - 8): a 4-bit code, and per token and 64 head dims one float16 pair
// (s, c): 4.5 bits a value. The codes lie in the order in which the attention kernels' matrix
// fragments take them, so that a warp reads its operands as whole 16-byte pieces without bank
// conflicts and a few bit operations on each 32-bit word give pairs of operands:
//
//   keys     words [HD / 128][token 16][t 4][i]: nibble p + 4 e = head dim 128 plane + 32 i + 8 t + 2 p + e
//   values   words [HD / 64][g 8][t 4][i 2][h 2]: nibble p + 4 e = token 8 h + 2 t + e, dim 64 plane + 32 i + 4 g + p
//   pairs    keys [token 16][HD / 64] (s, c), then values likewise
//
// (g = lane / 4 and t = lane % 4 of the mma.m16n8k16 fragments; (w & 0x000f000f) and its shifts by
// 4, 8 and 12 are the nibble pairs (p, p + 4).)
#pragma once
#include "common.cuh"
#include "kv4.h"
#include "sm100.cuh"

namespace hk {
namespace kv4 {

template <int HD>
struct Unit {
  static constexpr int kGroups = HD / 64;                // (s, c) pairs of one token's K (or V)
  static constexpr int kRow = (HD < 128 ? HD : 128) / 2;  // bytes of one token's key codes in a plane
  static constexpr int kCodes = 8 * HD;                  // bytes of the key (or value) codes
  static constexpr int kPairsK = 16 * HD;                // byte offset of the key pairs
  static constexpr int kPairsV = 17 * HD;                // byte offset of the value pairs
  static constexpr int kBytes = 18 * HD;

  // byte of the key word holding dims [d, d + 8) (d % 8 == 0) of token `tok`
  __host__ __device__ static constexpr int key_word(int tok, int d) {
    return (d >> 7) * 16 * kRow + tok * kRow + ((d >> 3) & 3) * (kRow / 4) + ((d & 127) >> 5) * 4;
  }
  // byte of the value half word holding dims [d, d + 4) (d % 4 == 0) of token `tok`
  __host__ __device__ static constexpr int value_half(int tok, int d) {
    return kCodes + (d >> 6) * 512 + ((d >> 2) & 7) * 64 + ((tok & 7) >> 1) * 16 + ((d >> 5) & 1) * 8 + (tok >> 3) * 4 +
           (tok & 1) * 2;
  }
  // byte of the (s, c) pair of group `grp` of token `tok`
  __host__ __device__ static constexpr int pair(bool value, int tok, int grp) {
    return (value ? kPairsV : kPairsK) + tok * (4 * kGroups) + grp * 4;
  }
};

// Codes less 8, exact, as float16 pairs of the even (0x000f000f) and odd (0x00f000f0) nibbles of w: 1024 + m
// and 1024 + 16 m are the bit patterns themselves.
__device__ __forceinline__ uint32_t centre_even(uint32_t w) {
  const uint32_t x = (w & 0x000f000fu) | 0x64006400u, k = 0xe408e408u;  // -1032
  const __half2 r = __hadd2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t centre_odd(uint32_t w) {
  const uint32_t x = (w & 0x00f000f0u) | 0x64006400u, s = 0x2c002c00u, k = 0xd480d480u;  // 1 / 16, -72
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&s),
                            *reinterpret_cast<const __half2*>(&k));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Largest magnitude a group holds: larger finite values are clamped to it, so that the centre and
// the ends c - 8 s, c + 7 s of every group stay finite in float16.
constexpr float kMaxValue = 65024.f;

// ---- sinks of the attention kernels ----
// A head's extra logit as log2 of its weight: NaN stays, and +infinity becomes a number that no score reaches, so that it
// takes all the weight and no difference of infinities arises, whether a row is merged from parts or not.
__device__ __forceinline__ float min_keeping_nan(float x, float y) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float sink_log2(float sink) { return min_keeping_nan(sink * 1.4426950408889634f, 1e30f); }
// log2 of its weight relative to a row's reference, of which the power stays finite
__device__ __forceinline__ float sink_over(float sink, float ref) { return min_keeping_nan(sink_log2(sink) - ref, 126.f); }

// ---- waits of the attention kernels ----
// A wait that ran out: over a bad argument's code, which is the lesser failure.
__device__ __forceinline__ void timed_out(int* status) { atomicExch(status, HK_ERR_MBAR_TIMEOUT); }

// A warp's bounded wait, with one answer for all lanes: those that give up leave the code in which a warp votes, or
// issues instructions as one, together. It gives up after `polls` polls, or early once a wait anywhere has. (A bad
// argument's code in the status word, of this launch or an earlier one, ends no wait: its rows read as zeros and the
// other rows go on.)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status, uint32_t polls) {
  bool done = false;
  for (uint32_t left = polls; left && !(done = sm100::mbar_try_wait(bar, parity)); --left)
    if ((left & 1023) == 1 && *reinterpret_cast<volatile int*>(status) == HK_ERR_MBAR_TIMEOUT) break;
  done = __all_sync(0xffffffffu, done);
  if (!done) timed_out(status);
  return done;
}

// The wait for a CTA's own copies or products before it gives up its memory: whatever the status word says, and
// however short the other waits are.
__device__ __forceinline__ bool drain(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kKv4WaitPolls; ++i)
    if (sm100::mbar_try_wait(bar, parity)) return true;
  return false;
}

}  // namespace kv4
}  // namespace hk
