// Device-side building blocks and launchers of the 4-bit paged cache (kv4.h).
#pragma once

#include "../../include/kv4.h"
#include "kv8_common.h"

namespace rf {

constexpr uint32_t kNibbles = 0x000f000fu;     // bits 0..3 of both halves
constexpr uint32_t kNibbles4 = 0x00f000f0u;    // bits 4..7
constexpr uint32_t kStepBits = 0xfff0fff0u;    // a word's step, both halves
// fp16 numbers that end in a nibble: 1024 + n with n in bits 0..3, 64 + n with n in
// bits 4..7.
constexpr uint32_t kBase = 0x64006400u, kBase4 = 0x54005400u;

// (a & m) | c in one instruction, the mask in a scalar register.
__device__ __forceinline__ uint32_t mask_or(uint32_t a, uint32_t m, uint32_t c) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "s"(m), "v"(c));
  return r;
}

__device__ __forceinline__ half2v as_half2(uint32_t v) { return __builtin_bit_cast(half2v, v); }
__device__ __forceinline__ half8 join8(half2v a, half2v b, half2v c, half2v d) {
  return __builtin_shufflevector(__builtin_shufflevector(a, b, 0, 1, 2, 3), __builtin_shufflevector(c, d, 0, 1, 2, 3),
                                 0, 1, 2, 3, 4, 5, 6, 7);
}

// Tile and byte of a token's numbers inside a 32-token group of one head.
// Keys: the four bytes of dimensions [d, d + 8).
template <int D>
__device__ __forceinline__ int k4_at(int token, int d) {
  const int l = d % 64 / 16 * 16 + token / 8 * 4 + token % 4;
  return d / 64 * kTileBytes + l * 16 + token / 4 % 2 * 8 + d % 16 / 8 * 4;
}
// Values: the two bytes of dimensions [d, d + 4).
template <int D>
__device__ __forceinline__ int v4_at(int token, int d) {
  const int l = token / 8 * 16 + d % 64 / 4;
  return d / 64 * kTileBytes + l * 16 + token % 8 / 2 * 4 + token % 2 * 2;
}

// Validated arguments, as the C ABI passes them on (kv4_capi.hip).
hipError_t launch_kv4_append(const rf_kv4_cache& c, const rf_kv8_heads& k, const rf_kv8_heads& v,
                             int dtype, const int32_t* slots, int64_t tokens, hipStream_t stream);
hipError_t launch_kv4_read(const rf_kv4_cache& c, const int32_t* slots, int64_t n, int dtype,
                           void* k_out, void* v_out, hipStream_t stream);
PagedPlan plan_kv4_attention(const rf_kv4_attention_args& a, int cus);
hipError_t launch_kv4_attention(const rf_kv4_attention_args& a, const PagedPlan& p, hipStream_t stream);

}  // namespace rf
