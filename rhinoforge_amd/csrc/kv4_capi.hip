// C-ABI layer of the 4-bit paged cache (kv4.h): every refusal happens here,
// before any launch.
#include "kv4_common.h"
#include "paged_check.h"

namespace rf {
namespace {

int check_cache(const rf_kv4_cache& c) {
  if (!c.k || !c.v || !c.rows || !sizes_fit(c)) return RF_W8A16_EINVAL;
  return aligned(c.k, 16) && aligned(c.v, 16) && aligned(c.rows, 16) ? RF_W8A16_OK : RF_W8A16_EALIGN;
}

int check_attention(const rf_kv4_attention_args* a) {
  return a ? check_paged_attention(a, check_cache(a->cache)) : RF_W8A16_EINVAL;
}

}  // namespace
}  // namespace rf

using namespace rf;

extern "C" {

int rf_kv4_append(const rf_kv4_cache* cache, const rf_kv8_heads* k, const rf_kv8_heads* v,
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
  return status_of(launch_kv4_append(*cache, *k, *v, dtype, slots, tokens,
                                     static_cast<hipStream_t>(stream)));
}

int rf_kv4_read(const rf_kv4_cache* cache, const int32_t* slots, int64_t n, int32_t dtype,
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
  return status_of(launch_kv4_read(*cache, slots, n, dtype, k_out, v_out,
                                   static_cast<hipStream_t>(stream)));
}

size_t rf_kv4_attention_workspace(const rf_kv4_attention_args* a) {
  DeviceInfo dev;
  if (check_attention(a) != RF_W8A16_OK || a->tokens == 0 || device_info(&dev) != RF_W8A16_OK) return 0;
  return plan_kv4_attention(*a, dev.cus).workspace;
}

int rf_kv4_attention(const rf_kv4_attention_args* a, void* stream) {
  int st = check_attention(a);
  if (st != RF_W8A16_OK) return st;
  if (a->tokens == 0) return RF_W8A16_OK;
  DeviceInfo dev;
  st = check_device(&dev);
  if (st != RF_W8A16_OK) return st;
  const PagedPlan p = plan_kv4_attention(*a, dev.cus);
  if (p.workspace > 0) {
    const rf_w8a16_scratch* w = a->scratch;
    if (!w || !w->counters || !w->partials || w->partial_bytes < p.workspace) return RF_W8A16_EWORKSPACE;
    if (!aligned(w->counters, 4) || !aligned(w->partials, 16)) return RF_W8A16_EALIGN;
  }
  if (p.grid > 0x7fffffff) return RF_W8A16_EINVAL;
  return status_of(launch_kv4_attention(*a, p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"
