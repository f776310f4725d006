// Torch-library ops over the rf_kv4 C ABI (namespace `kv4`; PyTorch-ROCm):
//   append(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) rows, Tensor k, Tensor v,
//          Tensor slots) -> ()
//   read(Tensor k_cache, Tensor v_cache, Tensor rows, Tensor slots, ScalarType dtype)
//        -> (Tensor, Tensor)
//   attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor rows, Tensor block_table,
//             Tensor kv_lens, Tensor? cu_q, int max_q_len, int max_kv_len, bool causal, int window,
//             float scale, bool return_lse) -> (Tensor, Tensor)
// Checks in the manner of kv8_torch.cpp; there is no CPU computation.
#include "paged_torch.h"

namespace {

using namespace rf_torch;

// k_cache, v_cache: uint8 [blocks, kv_heads, block_size / 32, head_dim / 64, 1024];
// rows: int16 [blocks, kv_heads, block_size / 32, 2, 32].
void check_cache(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows, const char* op) {
  TORCH_CHECK(kc.scalar_type() == at::kByte && vc.scalar_type() == at::kByte, op,
              ": k_cache and v_cache must be uint8 tiles");
  TORCH_CHECK(kc.dim() == 5 && kc.sym_size(4) == 1024 && kc.is_contiguous() && vc.is_contiguous() &&
                  kc.sym_sizes() == vc.sym_sizes(),
              op, ": k_cache and v_cache must be contiguous tiles [blocks, kv_heads, block_size / 32, "
              "head_dim / 64, 1024] of one shape, got ", kc.sym_sizes(), " and ", vc.sym_sizes());
  TORCH_CHECK(kc.sym_size(0) >= 1 && kc.sym_size(1) >= 1, op, ": the cache is empty");
  const c10::SymInt g = kc.sym_size(2), d = kc.sym_size(3);
  TORCH_CHECK(g == 1 || g == 2 || g == 4, op, ": block_size must be 32, 64 or 128, got ", g * 32);
  TORCH_CHECK(d == 1 || d == 2 || d == 4, op, ": head_dim must be 64, 128 or 256, got ", d * 64);
  TORCH_CHECK(rows.scalar_type() == at::kShort && rows.dim() == 5 && rows.is_contiguous() &&
                  rows.sym_size(0) == kc.sym_size(0) && rows.sym_size(1) == kc.sym_size(1) &&
                  rows.sym_size(2) == g && rows.sym_size(3) == 2 && rows.sym_size(4) == 32,
              op, ": rows must be contiguous int16 [", kc.sym_size(0), ", ", kc.sym_size(1), ", ", g,
              ", 2, 32], got ", rows.scalar_type(), " ", rows.sym_sizes());
}

rf_kv4_cache cache_of(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows, const char* op) {
  check_same_device(kc, kc, op, "k_cache");
  check_same_device(vc, kc, op, "v_cache");
  check_same_device(rows, kc, op, "rows");
  return {kc.data_ptr(), vc.data_ptr(), reinterpret_cast<uint16_t*>(rows.data_ptr<int16_t>()), kc.size(0),
          (int32_t)kc.size(1), (int32_t)kc.size(3) * 64, (int32_t)kc.size(2) * 32};
}

void check_append(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
                  const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& slots) {
  const char* op = "kv4::append";
  check_cache(kc, vc, rows, op);
  check_half(k, op, "k");
  check_ints(slots, 1, op, "slots");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": v must be ", k.scalar_type(), " as k");
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->dim() == 3 && t->sym_size(0) == slots.sym_size(0) &&
                    t->sym_size(1) == kc.sym_size(1) && t->sym_size(2) == kc.sym_size(3) * 64,
                op, ": k and v must be [", slots.sym_size(0), " tokens, ", kc.sym_size(1),
                " kv_heads, ", kc.sym_size(3) * 64, " head_dim], got ", t->sym_sizes());
}

void append_hip(at::Tensor& kc, at::Tensor& vc, at::Tensor& rows, const at::Tensor& k,
                const at::Tensor& v, const at::Tensor& slots) {
  RECORD_FUNCTION("kv4::append", {});
  const char* op = "kv4::append";
  check_append(kc, vc, rows, k, v, slots);
  const rf_kv4_cache c = cache_of(kc, vc, rows, op);
  check_same_device(k, kc, op, "k");
  check_same_device(v, kc, op, "v");
  check_same_device(slots, kc, op, "slots");
  if (slots.numel() == 0) return;
  c10::DeviceGuard dev_guard(kc.device());
  at::Tensor keep[2];
  const rf_kv8_heads kh = heads_of(k, &keep[0]), vh = heads_of(v, &keep[1]);
  check_status(rf_kv4_append(&c, &kh, &vh, dtype_code(k.scalar_type()), slots.data_ptr<int32_t>(),
                             slots.numel(), stream_of(kc)),
               op);
}

void append_meta(at::Tensor& kc, at::Tensor& vc, at::Tensor& rows, const at::Tensor& k,
                 const at::Tensor& v, const at::Tensor& slots) {
  check_append(kc, vc, rows, k, v, slots);
}

void append_cpu(at::Tensor& kc, at::Tensor& vc, at::Tensor& rows, const at::Tensor& k,
                const at::Tensor& v, const at::Tensor& slots) {
  check_append(kc, vc, rows, k, v, slots);
  no_cpu("kv4::append");
}

void check_read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows, const at::Tensor& slots, at::ScalarType dtype) {
  const char* op = "kv4::read";
  check_cache(kc, vc, rows, op);
  check_ints(slots, 1, op, "slots");
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16 || dtype == at::kFloat, op,
              ": dtype must be float16, bfloat16 or float32, got ", dtype);
}

Two read_meta(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
              const at::Tensor& slots, at::ScalarType dtype) {
  check_read(kc, vc, rows, slots, dtype);
  const std::vector<c10::SymInt> shape = {slots.sym_size(0), kc.sym_size(1), kc.sym_size(3) * 64};
  const auto o = kc.options().dtype(dtype);
  return {at::empty_symint(shape, o), at::empty_symint(shape, o)};
}

Two read_hip(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
             const at::Tensor& slots, at::ScalarType dtype) {
  RECORD_FUNCTION("kv4::read", {});
  const char* op = "kv4::read";
  check_read(kc, vc, rows, slots, dtype);
  const rf_kv4_cache c = cache_of(kc, vc, rows, op);
  check_same_device(slots, kc, op, "slots");
  const std::vector<int64_t> shape = {slots.size(0), kc.size(1), kc.size(3) * 64};
  Two out{new_tensor(shape, dtype, kc), new_tensor(shape, dtype, kc)};
  if (slots.numel() == 0) return out;
  c10::DeviceGuard dev_guard(kc.device());
  check_status(rf_kv4_read(&c, slots.data_ptr<int32_t>(), slots.numel(), dtype_code(dtype),
                           std::get<0>(out).data_ptr(), std::get<1>(out).data_ptr(), stream_of(kc)),
               op);
  return out;
}

Two read_cpu(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
             const at::Tensor& slots, at::ScalarType dtype) {
  check_read(kc, vc, rows, slots, dtype);
  no_cpu("kv4::read");
}

// ---- attention -------------------------------------------------------------------
void check_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
                     const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                     int64_t max_kv, bool causal, int64_t window, double scale) {
  const char* op = "kv4::attention";
  check_half(q, op, "q");
  check_cache(kc, vc, rows, op);
  rf_torch::check_attention(op, q, kc.sym_size(1), kc.sym_size(3) * 64, table, lens, cu, max_q, max_kv, causal,
                            window, scale);
}

Two attention_hip(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                  int64_t max_kv, bool causal, int64_t window, double scale, bool return_lse) {
  RECORD_FUNCTION("kv4::attention", {});
  const char* op = "kv4::attention";
  check_attention(q, kc, vc, rows, table, lens, cu, max_q, max_kv, causal, window, scale);
  check_same_device(q, q, op, "q");
  rf_kv4_attention_args a{};
  a.cache = cache_of(kc, vc, rows, op);
  check_same_device(kc, q, op, "k_cache");
  return run_attention(op, a, rf_kv4_attention, rf_kv4_attention_workspace, q, table, lens, cu, max_q, max_kv,
                       causal, window, scale, return_lse);
}

Two attention_meta(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
                   const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                   int64_t max_kv, bool causal, int64_t window, double scale, bool return_lse) {
  check_attention(q, kc, vc, rows, table, lens, cu, max_q, max_kv, causal, window, scale);
  return attention_outputs(q, return_lse);
}

Two attention_cpu(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& rows,
                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                  int64_t max_kv, bool causal, int64_t window, double scale, bool) {
  check_attention(q, kc, vc, rows, table, lens, cu, max_q, max_kv, causal, window, scale);
  no_cpu("kv4::attention");
}

}  // namespace

TORCH_LIBRARY(kv4, m) {
  m.def("append(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) rows, Tensor k, Tensor v, "
        "Tensor slots) -> ()");
  m.def("read(Tensor k_cache, Tensor v_cache, Tensor rows, Tensor slots, ScalarType dtype) "
        "-> (Tensor, Tensor)");
  m.def("attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor rows, Tensor block_table, "
        "Tensor kv_lens, Tensor? cu_q, int max_q_len, int max_kv_len, bool causal, int window, "
        "float scale, bool return_lse) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(kv4, CUDA, m) {
  m.impl("append", TORCH_FN(append_hip));
  m.impl("read", TORCH_FN(read_hip));
  m.impl("attention", TORCH_FN(attention_hip));
}
TORCH_LIBRARY_IMPL(kv4, Meta, m) {
  m.impl("append", TORCH_FN(append_meta));
  m.impl("read", TORCH_FN(read_meta));
  m.impl("attention", TORCH_FN(attention_meta));
}
TORCH_LIBRARY_IMPL(kv4, CPU, m) {
  m.impl("append", TORCH_FN(append_cpu));
  m.impl("read", TORCH_FN(read_cpu));
  m.impl("attention", TORCH_FN(attention_cpu));
}
// Not differentiable, as the other cache's ops: autograd falls through.
TORCH_LIBRARY_IMPL(kv4, Autograd, m) {
  for (const char* op : {"append", "read", "attention"}) m.impl(op, torch::CppFunction::makeFallthrough());
}
