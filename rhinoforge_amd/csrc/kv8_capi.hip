// C-ABI layer of the int8 paged cache (kv8.h): every refusal happens here,
// before any launch.
#include "paged_check.h"

namespace rf {
namespace {

int check_cache(const rf_kv8_cache& c) {
  if (!c.k || !c.v || !c.k_scale || !c.v_scale) return RF_W8A16_EINVAL;
  if (!sizes_fit(c)) return RF_W8A16_EINVAL;
  if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 4) || !aligned(c.v_scale, 4))
    return RF_W8A16_EALIGN;
  return RF_W8A16_OK;
}

int check_attention(const rf_kv8_attention_args* a) {
  return a ? check_paged_attention(a, check_cache(a->cache)) : RF_W8A16_EINVAL;
}

int check_rope(const rf_kv8_rope_args* a) {
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
  return RF_W8A16_OK;
}

struct Ints {
  const int32_t* p;
  int64_t n;
};

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_kv8_qk_norm_rope(const rf_kv8_rope_args* a, void* stream) {
  int st = check_rope(a);
  if (st != RF_W8A16_OK || a->tokens == 0) return st;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_qk_norm_rope(*a, nullptr, static_cast<hipStream_t>(stream)));
}

int rf_kv8_qk_norm_mrope(const rf_kv8_mrope_args* a, void* stream) {
  if (!a) return RF_W8A16_EINVAL;
  int st = check_rope(&a->rope);
  if (st != RF_W8A16_OK) return st;
  if (a->rope.rot < 1 || !a->rope.positions || a->axes < 1 || a->axes > RF_KV8_MAX_AXES) return RF_W8A16_EINVAL;
  if (a->axis_stride < a->rope.tokens) return RF_W8A16_EINVAL;
  int64_t pairs = 0;
  for (int i = 0; i < a->axes; ++i) {
    if (a->sections[i] < 0 || a->sections[i] > a->rope.rot / 2) return RF_W8A16_EINVAL;
    pairs += a->sections[i];
    // (mixed: the last pair of axis i is axes * (section - 1) + i)
    if (a->mixed && i > 0 && a->sections[i] > 0 && a->axes * (a->sections[i] - 1) + i >= a->rope.rot / 2)
      return RF_W8A16_EINVAL;
  }
  if (pairs != a->rope.rot / 2) return RF_W8A16_EINVAL;
  if (a->rope.tokens == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  return status_of(launch_qk_norm_rope(a->rope, a, static_cast<hipStream_t>(stream)));
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
  const PagedPlan p = plan_kv8_attention(*a, dev.cus);
  if (p.workspace > 0) {
    const rf_w8a16_scratch* w = a->scratch;
    if (!w || !w->counters || !w->partials || w->partial_bytes < p.workspace) return RF_W8A16_EWORKSPACE;
    if (!aligned(w->counters, 4) || !aligned(w->partials, 16)) return RF_W8A16_EALIGN;
  }
  if (p.grid > 0x7fffffff) return RF_W8A16_EINVAL;
  return status_of(launch_kv8_attention(*a, p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
