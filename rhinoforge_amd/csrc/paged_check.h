// Checks of arguments that the paged caches' C entries share (kv8_capi.hip,
// kv4_capi.hip).
#pragma once

#include "kv8_common.h"

namespace rf {
namespace {

constexpr int64_t kMaxSize = (int64_t)1 << 30;  // tokens, requests, slots of one call

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

int check_device(DeviceInfo* dev) {
  const int st = device_info(dev);
  if (st != RF_W8A16_OK) return st;
  return dev->gfx950 ? RF_W8A16_OK : RF_W8A16_EDEVICE;
}

bool half_dtype(int dtype) { return dtype == RF_W8A16_DTYPE_F16 || dtype == RF_W8A16_DTYPE_BF16; }

int check_heads(const rf_kv8_heads& h) {
  if (!h.data || h.heads < 1 || h.heads > 4096) return RF_W8A16_EINVAL;
  if (!aligned(h.data, 16) || h.token_stride % 8 || h.head_stride % 8) return RF_W8A16_EALIGN;
  return RF_W8A16_OK;
}

// The cache's sizes (rf_kv8_cache or the like).
template <typename Cache>
bool sizes_fit(const Cache& c) {
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return false;
  if (c.block_size != 32 && c.block_size != 64 && c.block_size != 128) return false;
  if (c.kv_heads < 1 || c.kv_heads > 4096 || c.num_blocks < 1) return false;
  return c.num_blocks <= 0x7fffffff / c.block_size;  // slots are int32
}

// All of an attention call but its cache (checked before: `st`).
template <typename Args>
int check_paged_attention(const Args* a, int st) {
  if (st == RF_W8A16_OK) st = check_heads(a->q);
  if (st != RF_W8A16_OK) return st;
  if (!half_dtype(a->dtype) || !a->kv_lens || !a->block_table || !a->out) return RF_W8A16_EINVAL;
  if (a->q.heads % a->cache.kv_heads) return RF_W8A16_EINVAL;
  if (a->tokens < 0 || a->tokens > kMaxSize || a->requests < 1 || a->requests > kMaxSize)
    return RF_W8A16_EINVAL;
  if (a->tokens * a->q.heads > 0x7fffffff) return RF_W8A16_EINVAL;
  if (!a->cu_q && a->tokens % a->requests) return RF_W8A16_EINVAL;
  if (a->width < 1 || a->table_stride < a->width || a->width > kMaxSize / a->cache.block_size)
    return RF_W8A16_EINVAL;
  if (!(a->scale > 0.0f) || !(a->scale < __builtin_inff())) return RF_W8A16_EINVAL;
  if (a->window < 0 || (a->window > 0 && !a->causal)) return RF_W8A16_EINVAL;
  if (a->max_q_len < 0 || a->max_kv_len < 0) return RF_W8A16_EINVAL;
  if (!aligned(a->out, 16) || !aligned(a->lse, 4) || !aligned(a->cu_q, 4) ||
      !aligned(a->kv_lens, 4) || !aligned(a->block_table, 4))
    return RF_W8A16_EALIGN;
  return RF_W8A16_OK;
}

int status_of(hipError_t e) { return e == hipSuccess ? RF_W8A16_OK : RF_W8A16_EHIP; }

}  // namespace
}  // namespace rf
