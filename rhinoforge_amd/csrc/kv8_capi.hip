// C-ABI layer of the int8 paged cache (kv8.h): every refusal happens here,
// before any launch.
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

int check_cache(const rf_kv8_cache& c) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return RF_W8A16_EINVAL;
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return RF_W8A16_EINVAL;
  if (c.block_size != 32 && c.block_size != 64 && c.block_size != 128) return RF_W8A16_EINVAL;
  if (c.kv_heads < 1 || c.kv_heads > 4096 || c.num_blocks < 1) return RF_W8A16_EINVAL;
  // slots are int32
  if (c.num_blocks > 0x7fffffff / c.block_size) return RF_W8A16_EINVAL;
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 4) || !aligned(c.v_scale, 4))
    return RF_W8A16_EALIGN;
  return RF_W8A16_OK;
}

int check_attention(const rf_kv8_attention_args* a) {
  if (!a) return RF_W8A16_EINVAL;
  int st = check_cache(a->cache);
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

struct Ints {
  const int32_t* p;
  int64_t n;
};

int status_of(hipError_t e) { return e == hipSuccess ? RF_W8A16_OK : RF_W8A16_EHIP; }

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_kv8_qk_norm_rope(const rf_kv8_rope_args* a, void* stream) {
  if (!a) return RF_W8A16_EINVAL;
  int st = check_heads(a->q);
  if (st == RF_W8A16_OK) st = check_heads(a->k);
  if (st != RF_W8A16_OK) return st;
  if (!a->q_out || !a->k_out || !half_dtype(a->dtype) || a->tokens < 0 || a->tokens > kMaxSize)
    return RF_W8A16_EINVAL;
  if (a->head_dim < 8 || a->head_dim > 512 || a->head_dim % 8) return RF_W8A16_EINVAL;
  if (a->rot < 0 || a->rot > a->head_dim || a->rot % 16) return RF_W8A16_EINVAL;
  if (a->rot > 0) {
    if (!a->cos || !a->sin || a->table_rows < 1) return RF_W8A16_EINVAL;
    if (!a->positions && a->table_rows < a->tokens) return RF_W8A16_EINVAL;
    if (!aligned(a->cos, 16) || !aligned(a->sin, 16)) return RF_W8A16_EALIGN;
  }
  if (!aligned(a->q_out, 16) || !aligned(a->k_out, 16) || !aligned(a->q_weight, 16) ||
      !aligned(a->k_weight, 16) || !aligned(a->positions, a->positions64 ? 8 : 4))
    return RF_W8A16_EALIGN;
  if (a->tokens == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_qk_norm_rope(*a, static_cast<hipStream_t>(stream)));
}

int rf_kv8_plan(const rf_kv8_plan_args* a, void* stream) {
  if (!a || a->requests < 1 || a->requests > RF_KV8_MAX_REQUESTS || a->tokens < 0 ||
      a->tokens > kMaxSize || a->width < 1 || a->width > kMaxSize || a->table_stride < a->width ||
      a->num_free < 0)
    return RF_W8A16_EINVAL;
  if (a->block_size != 32 && a->block_size != 64 && a->block_size != 128) return RF_W8A16_EINVAL;
  if (!a->block_table || !a->cached || !a->fresh || !a->free_start || !a->cu || !a->kv_lens ||
      !a->free_next || (a->num_free > 0 && !a->free_blocks) ||
      (a->tokens > 0 && (!a->slots || !a->positions)))
    return RF_W8A16_EINVAL;
  for (const void* p : {(const void*)a->block_table, (const void*)a->cached, (const void*)a->fresh,
                        (const void*)a->free_blocks, (const void*)a->free_start,
                        (const void*)a->slots, (const void*)a->positions, (const void*)a->cu,
                        (const void*)a->kv_lens, (const void*)a->free_next})
    if (!aligned(p, 4)) return RF_W8A16_EALIGN;
  const Ints in[] = {{a->cached, a->requests}, {a->fresh, a->requests}, {a->free_blocks, a->num_free}, {a->free_start, 1}};
  const Ints out[] = {{a->slots, a->tokens}, {a->positions, a->tokens}, {a->cu, a->requests + 1},
                      {a->kv_lens, a->requests}, {a->free_next, 1}};
  for (const Ints& o : out)
    for (const Ints& i : in)
      if (o.n > 0 && i.n > 0 && o.p < i.p + i.n && i.p < o.p + o.n) return RF_W8A16_EINVAL;
  DeviceInfo dev;
  const int st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_kv8_plan(*a, static_cast<hipStream_t>(stream)));
}

int rf_kv8_append(const rf_kv8_cache* cache, const rf_kv8_heads* k, const rf_kv8_heads* v,
                  int32_t dtype, const int32_t* slots, int64_t tokens, void* stream) {
  if (!cache || !k || !v) return RF_W8A16_EINVAL;
  int st = check_cache(*cache);
  if (st == RF_W8A16_OK) st = check_heads(*k);
  if (st == RF_W8A16_OK) st = check_heads(*v);
  if (st != RF_W8A16_OK) return st;
  if (!half_dtype(dtype) || k->heads != cache->kv_heads || v->heads != cache->kv_heads ||
      tokens < 0 || tokens > kMaxSize || (tokens > 0 && !slots))
    return RF_W8A16_EINVAL;
  if (!aligned(slots, 4)) return RF_W8A16_EALIGN;
  if (tokens == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_kv8_append(*cache, *k, *v, dtype, slots, tokens,
                                     static_cast<hipStream_t>(stream)));
}

int rf_kv8_read(const rf_kv8_cache* cache, const int32_t* slots, int64_t n, int32_t dtype,
                void* k_out, void* v_out, void* stream) {
  if (!cache) return RF_W8A16_EINVAL;
  int st = check_cache(*cache);
  if (st != RF_W8A16_OK) return st;
  if ((!half_dtype(dtype) && dtype != RF_W8A16_DTYPE_F32) || n < 0 || n > kMaxSize ||
      (n > 0 && (!slots || !k_out || !v_out)))
    return RF_W8A16_EINVAL;
  const size_t out = dtype == RF_W8A16_DTYPE_F32 ? 32 : 16;
  if (!aligned(slots, 4) || !aligned(k_out, out) || !aligned(v_out, out)) return RF_W8A16_EALIGN;
  if (n == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_kv8_read(*cache, slots, n, dtype, k_out, v_out,
                                   static_cast<hipStream_t>(stream)));
}

size_t rf_kv8_attention_workspace(const rf_kv8_attention_args* a) {
  DeviceInfo dev;
  if (check_attention(a) != RF_W8A16_OK || a->tokens == 0 || device_info(&dev) != RF_W8A16_OK) return 0;
  return plan_kv8_attention(*a, dev.cus).workspace;
}

int rf_kv8_attention(const rf_kv8_attention_args* a, void* stream) {
  int st = check_attention(a);
  if (st != RF_W8A16_OK) return st;
  if (a->tokens == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  const Kv8AttnPlan p = plan_kv8_attention(*a, dev.cus);
  if (p.workspace > 0) {
    const rf_w8a16_scratch* w = a->scratch;
    if (!w || !w->counters || !w->partials || w->partial_bytes < p.workspace) return RF_W8A16_EWORKSPACE;
    if (!aligned(w->counters, 4) || !aligned(w->partials, 16)) return RF_W8A16_EALIGN;
  }
  if (p.grid > 0x7fffffff) return RF_W8A16_EINVAL;
  return status_of(launch_kv8_attention(*a, p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
