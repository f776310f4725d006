// Device-side building blocks and launchers of the int8 paged cache (kv8.h).
#pragma once

#include "../../include/kv8.h"
#include "w8a16_common.h"
#include "w8a16_internal.h"

namespace rf {

typedef float floatx8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Eight consecutive values of a 16-bit type <-> fp32.
template <typename T>
struct Eight;
template <>
struct Eight<_Float16> {
  static __device__ __forceinline__ floatx8 load(const void* p) {
    return __builtin_convertvector(__builtin_bit_cast(half8, load_u4(p)), floatx8);
  }
  static __device__ __forceinline__ void store(void* p, floatx8 v) {
    *reinterpret_cast<half8*>(p) = __builtin_convertvector(v, half8);
  }
};
template <>
struct Eight<__bf16> {
  static __device__ __forceinline__ floatx8 load(const void* p) {
    return __builtin_convertvector(__builtin_bit_cast(bf16x8, load_u4(p)), floatx8);
  }
  static __device__ __forceinline__ void store(void* p, floatx8 v) {
    *reinterpret_cast<bf16x8*>(p) = __builtin_convertvector(v, bf16x8);
  }
};
template <>
struct Eight<float> {
  static __device__ __forceinline__ void store(void* p, floatx8 v) {
    *reinterpret_cast<floatx8*>(p) = v;
  }
};

// A launch holds fewer than 2^32 threads along x: with more it runs those modulo
// 2^32, without an error.  What needs more workgroups runs in several launches.
constexpr int64_t kMaxThreads = ((int64_t)1 << 32) - 1;

// Validated arguments, as the C ABI passes them on (kv8_capi.hip).
// (m: the same call's axes, or null: one axis)
hipError_t launch_qk_norm_rope(const rf_kv8_rope_args& a, const rf_kv8_mrope_args* m, hipStream_t stream);
hipError_t launch_kv8_plan(const rf_kv8_plan_args& a, hipStream_t stream);
hipError_t launch_kv8_append(const rf_kv8_cache& c, const rf_kv8_heads& k, const rf_kv8_heads& v,
                             int dtype, const int32_t* slots, int64_t tokens, hipStream_t stream);
hipError_t launch_kv8_read(const rf_kv8_cache& c, const int32_t* slots, int64_t n, int dtype,
                           void* k_out, void* v_out, hipStream_t stream);

// How a call of the attention is launched: rows (query, head of the group) of
// one tile, workgroups over the tokens of one tile, partial results.
struct PagedPlan {
  int kernel;     // 0: tokens split over the wavefronts (few rows), 1: rows split over them
  int gangs = 1;  // groups of four wavefronts that take a tile's tokens in turn
  int rows;       // rows of a tile
  int64_t tiles;  // upper bound of tiles per key/value head
  int splits;     // of a tile: all of them, or at most where `shares` is set
  int least;      // 32-token groups of a split, at least
  bool merge;     // a second kernel adds the splits
  int shares = 0; // of all tiles of a key/value head together, for batches of unequal lengths
  int aim = 0;    // that many of them, unless there are more tiles
  int64_t grid;   // workgroups
  int64_t partials;  // rows of partial results
  size_t workspace;  // their bytes
};
PagedPlan plan_kv8_attention(const rf_kv8_attention_args& a, int cus);
hipError_t launch_kv8_attention(const rf_kv8_attention_args& a, const PagedPlan& p,
                                hipStream_t stream);

}  // namespace rf
