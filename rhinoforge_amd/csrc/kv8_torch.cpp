// Torch-library ops over the rf_kv8 C ABI (namespace `kv8`; PyTorch-ROCm):
//   qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, Tensor? sin,
//                Tensor? positions, float eps, bool interleaved) -> (Tensor, Tensor)
//   plan(Tensor(a!) block_table, Tensor cached_lens, Tensor new_lens, Tensor free_blocks,
//        Tensor free_start, int num_tokens, int block_size)
//        -> (Tensor, Tensor, Tensor, Tensor, Tensor)
//   append(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale,
//          Tensor k, Tensor v, Tensor slots) -> ()
//   read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor slots,
//        ScalarType dtype) -> (Tensor, Tensor)
//   attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale,
//             Tensor block_table, Tensor kv_lens, Tensor? cu_q, int max_q_len, int max_kv_len,
//             bool causal, int window, float scale, bool return_lse) -> (Tensor, Tensor)
// and of namespace `rope`, the same norms and rotation by positions of several axes:
//   qk_norm_mrope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, Tensor sin,
//                 Tensor positions, int[] sections, bool mixed, float eps, bool interleaved)
//                 -> (Tensor, Tensor)
// They are what the reference's decoders run between the W8A16 projections
// (src/fused/rpu_qwen3_model.h: head norms, RoPE, KV insert, SDPA).  Checks in
// the manner of w8a16_torch.cpp: dtype and shape first (shared with the Meta
// kernels), then devices; invalid input raises, there is no CPU computation.
#include "paged_torch.h"

namespace {

using namespace rf_torch;

// ---- norms and rotation ----------------------------------------------------------
// All of a call but its positions.
void check_rope_operands(const char* op, const at::Tensor& q, const at::Tensor& k, const OptTensor& qw,
                         const OptTensor& kw, const OptTensor& cos, const OptTensor& sin) {
  check_half(q, op, "q");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), op, ": k must be ", q.scalar_type(), " as q, got ",
              k.scalar_type());
  TORCH_CHECK(q.dim() == 3 && k.dim() == 3 && q.sym_size(0) == k.sym_size(0) &&
                  q.sym_size(2) == k.sym_size(2),
              op, ": q and k must be [tokens, heads, head_dim] with the same tokens and head_dim, got ",
              q.sym_sizes(), " and ", k.sym_sizes());
  const c10::SymInt D = q.sym_size(2);
  TORCH_CHECK(q.sym_size(1) >= 1 && k.sym_size(1) >= 1, op, ": q and k need at least one head");
  TORCH_CHECK(D >= 8 && D <= 512 && D % 8 == 0, op, ": head_dim ", D,
              " must be a multiple of 8 up to 512");
  for (const OptTensor* w : {&qw, &kw}) {
    if (!given(*w)) continue;
    TORCH_CHECK((*w)->scalar_type() == q.scalar_type() && (*w)->dim() == 1 &&
                    (*w)->sym_size(0) == D && (*w)->is_contiguous(),
                op, ": a norm weight must be a contiguous ", q.scalar_type(), " [", D, "], got ",
                (*w)->scalar_type(), " ", (*w)->sym_sizes());
  }
  TORCH_CHECK(given(cos) == given(sin), op, ": cos and sin go together");
  if (given(cos)) {
    for (const OptTensor* c : {&cos, &sin})
      TORCH_CHECK((*c)->scalar_type() == at::kFloat && (*c)->dim() == 2 && (*c)->is_contiguous(), op,
                  ": cos and sin must be contiguous float32 [rows, rot / 2]");
    TORCH_CHECK(cos->sym_sizes() == sin->sym_sizes(), op, ": cos and sin differ in shape");
    const c10::SymInt rot = cos->sym_size(1) * 2;
    TORCH_CHECK(rot >= 16 && rot % 16 == 0 && rot <= D, op, ": rotated dimensions ", rot,
                " must be a multiple of 16 up to head_dim ", D);
    TORCH_CHECK(cos->sym_size(0) >= 1, op, ": cos and sin have no rows");
  }
}

void check_rope(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
                const OptTensor& cos, const OptTensor& sin, const OptTensor& pos) {
  const char* op = "kv8::qk_norm_rope";
  check_rope_operands(op, q, k, qw, kw, cos, sin);
  if (!given(cos)) return;
  if (given(pos)) {
    TORCH_CHECK((pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong) &&
                    pos->dim() == 1 && pos->sym_size(0) == q.sym_size(0) && pos->is_contiguous(),
                op, ": positions must be a contiguous int32 or int64 [tokens]");
  } else {
    TORCH_CHECK(cos->sym_size(0) >= q.sym_size(0), op,
                ": without positions cos and sin need a row for each token");
  }
}

// The operands as the C ABI takes them, checked for their devices, and the outputs.
struct RopeCall {
  at::Tensor q, k;
  at::Tensor keep[6];
};

void fill_rope(RopeCall& c, rf_kv8_rope_args& a, const char* op, const at::Tensor& q, const at::Tensor& k,
               const OptTensor& qw, const OptTensor& kw, const OptTensor& cos, const OptTensor& sin,
               const OptTensor& pos, double eps, bool interleaved) {
  a.q = heads_of(q, &c.keep[0]);
  a.k = heads_of(k, &c.keep[1]);
  c.q = new_tensor(q.sizes(), q.scalar_type(), q);
  c.k = new_tensor(k.sizes(), k.scalar_type(), k);
  a.q_out = c.q.data_ptr();
  a.k_out = c.k.data_ptr();
  if (given(qw)) a.q_weight = (c.keep[2] = aligned_copy(*qw)).data_ptr();
  if (given(kw)) a.k_weight = (c.keep[3] = aligned_copy(*kw)).data_ptr();
  if (given(cos)) {
    a.cos = (c.keep[4] = aligned_copy(*cos)).data_ptr<float>();
    a.sin = (c.keep[5] = aligned_copy(*sin)).data_ptr<float>();
    a.rot = (int32_t)cos->size(1) * 2;
    a.table_rows = cos->size(0);
    if (given(pos)) {
      a.positions = pos->data_ptr();
      a.positions64 = pos->scalar_type() == at::kLong;
    }
  }
  a.tokens = q.size(0);
  a.head_dim = (int32_t)q.size(2);
  a.dtype = dtype_code(q.scalar_type());
  a.interleaved = interleaved;
  a.eps = (float)eps;
}

Two rope_hip(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
             const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, double eps,
             bool interleaved) {
  RECORD_FUNCTION("kv8::qk_norm_rope", {});
  const char* op = "kv8::qk_norm_rope";
  check_rope(q, k, qw, kw, cos, sin, pos);
  check_same_device(k, q, op, "k");
  for (const OptTensor* t : {&qw, &kw, &cos, &sin, &pos})
    if (given(*t)) check_same_device(**t, q, op, "an argument");
  c10::DeviceGuard dev_guard(q.device());
  RopeCall c;
  rf_kv8_rope_args a{};
  fill_rope(c, a, op, q, k, qw, kw, cos, sin, pos, eps, interleaved);
  if (a.tokens > 0) check_status(rf_kv8_qk_norm_rope(&a, stream_of(q)), op);
  return {c.q, c.k};
}

Two rope_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
              const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, double, bool) {
  check_rope(q, k, qw, kw, cos, sin, pos);
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}

Two rope_cpu(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
             const OptTensor& cos, const OptTensor& sin, const OptTensor& pos, double, bool) {
  check_rope(q, k, qw, kw, cos, sin, pos);
  no_cpu("kv8::qk_norm_rope");
}

// Several axes: positions [axes, tokens]; sections: pairs of each.
void check_mrope(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
                 const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& pos,
                 at::IntArrayRef sections, bool mixed) {
  const char* op = "rope::qk_norm_mrope";
  check_rope_operands(op, q, k, qw, kw, cos, sin);
  const int64_t axes = (int64_t)sections.size();
  TORCH_CHECK(axes >= 1 && axes <= RF_KV8_MAX_AXES, op, ": between 1 and ", RF_KV8_MAX_AXES,
              " sections, got ", axes);
  TORCH_CHECK((pos.scalar_type() == at::kInt || pos.scalar_type() == at::kLong) && pos.dim() == 2 &&
                  pos.sym_size(0) == axes && pos.sym_size(1) == q.sym_size(0),
              op, ": positions must be int32 or int64 [", axes, " axes, ", q.sym_size(0), " tokens], got ",
              pos.scalar_type(), " ", pos.sym_sizes());
  const c10::SymInt pairs = cos.sym_size(1);
  c10::SymInt sum = 0;
  for (const int64_t n : sections) TORCH_CHECK(n >= 0, op, ": sections must not be negative, got ", sections);
  for (int64_t i = 0; i < axes; ++i) {
    TORCH_CHECK(pairs >= sections[i], op, ": sections ", sections, " must add up to the ", pairs,
                " pairs of cos and sin");
    sum += sections[i];
  }
  TORCH_CHECK(sum == pairs, op, ": sections ", sections, " must add up to the ", pairs, " pairs of cos and sin");
  for (int64_t i = 1; i < axes; ++i)
    TORCH_CHECK(!mixed || sections[i] == 0 || pairs > axes * (sections[i] - 1) + i, op, ": sections ", sections,
                " cannot be mixed, axis ", i, " has more pairs than places");
}

Two mrope_hip(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
              const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& pos,
              at::IntArrayRef sections, bool mixed, double eps, bool interleaved) {
  RECORD_FUNCTION("rope::qk_norm_mrope", {});
  const char* op = "rope::qk_norm_mrope";
  check_mrope(q, k, qw, kw, cos, sin, pos, sections, mixed);
  check_same_device(k, q, op, "k");
  for (const OptTensor* t : {&qw, &kw})
    if (given(*t)) check_same_device(**t, q, op, "a norm weight");
  for (const at::Tensor* t : {&cos, &sin, &pos}) check_same_device(*t, q, op, "an argument");
  c10::DeviceGuard dev_guard(q.device());
  const bool rows = (pos.size(1) <= 1 || pos.stride(1) == 1) && (pos.size(0) <= 1 || pos.stride(0) >= pos.size(1));
  const at::Tensor p = rows ? pos : pos.contiguous();
  RopeCall c;
  rf_kv8_mrope_args a{};
  fill_rope(c, a.rope, op, q, k, qw, kw, cos, sin, p, eps, interleaved);
  a.axes = (int32_t)sections.size();
  a.axis_stride = a.axes == 1 ? a.rope.tokens : p.stride(0);
  a.mixed = mixed;
  for (int i = 0; i < a.axes; ++i) a.sections[i] = (int32_t)sections[i];
  if (a.rope.tokens > 0) check_status(rf_kv8_qk_norm_mrope(&a, stream_of(q)), op);
  return {c.q, c.k};
}

Two mrope_meta(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
               const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& pos,
               at::IntArrayRef sections, bool mixed, double, bool) {
  check_mrope(q, k, qw, kw, cos, sin, pos, sections, mixed);
  return {at::empty_symint(q.sym_sizes(), q.options()), at::empty_symint(k.sym_sizes(), k.options())};
}

Two mrope_cpu(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
              const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& pos,
              at::IntArrayRef sections, bool mixed, double, bool) {
  check_mrope(q, k, qw, kw, cos, sin, pos, sections, mixed);
  no_cpu("rope::qk_norm_mrope");
}

// ---- block tables and slots ------------------------------------------------------
void check_plan(const at::Tensor& table, const at::Tensor& cached, const at::Tensor& fresh,
                const at::Tensor& free_blocks, const at::Tensor& start, int64_t tokens, int64_t bs) {
  const char* op = "kv8::plan";
  check_ints(table, 2, op, "block_table");
  check_ints(cached, 1, op, "cached_lens");
  check_ints(fresh, 1, op, "new_lens");
  check_ints(free_blocks, 1, op, "free_blocks");
  check_ints(start, 1, op, "free_start");
  const c10::SymInt B = cached.sym_size(0);
  TORCH_CHECK(B >= 1 && B <= RF_KV8_MAX_REQUESTS, op, ": between 1 and ", RF_KV8_MAX_REQUESTS,
              " requests, got ", B);
  TORCH_CHECK(fresh.sym_size(0) == B && table.sym_size(0) == B, op,
              ": block_table, cached_lens and new_lens differ in requests");
  TORCH_CHECK(table.sym_size(1) >= 1 && table.sym_stride(1) == 1 &&
                  (B <= 1 || table.sym_stride(0) >= table.sym_size(1)),
              op, ": block_table must have rows of unit stride, one after the other");
  TORCH_CHECK(start.sym_size(0) == 1, op, ": free_start must have one element");
  TORCH_CHECK(tokens >= 0 && tokens <= ((int64_t)1 << 30), op, ": num_tokens ", tokens,
              " is negative or too large");
  TORCH_CHECK(bs == 32 || bs == 64 || bs == 128, op, ": block_size must be 32, 64 or 128, got ", bs);
}

using Five = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

Five plan_outputs(const at::Tensor& cached, int64_t tokens) {
  const auto o = cached.options();
  const c10::SymInt B = cached.sym_size(0);
  return {at::empty({tokens}, o), at::empty({tokens}, o), at::empty_symint({B + 1}, o),
          at::empty_symint({B}, o), at::empty({1}, o)};
}

Five plan_hip(at::Tensor& table, const at::Tensor& cached, const at::Tensor& fresh,
              const at::Tensor& free_blocks, const at::Tensor& start, int64_t tokens, int64_t bs) {
  RECORD_FUNCTION("kv8::plan", {});
  const char* op = "kv8::plan";
  check_plan(table, cached, fresh, free_blocks, start, tokens, bs);
  check_same_device(cached, table, op, "cached_lens");
  check_same_device(fresh, table, op, "new_lens");
  check_same_device(free_blocks, table, op, "free_blocks");
  check_same_device(start, table, op, "free_start");
  c10::DeviceGuard dev_guard(table.device());
  const int64_t B = cached.size(0);
  const auto ints = [&](int64_t n) { return new_tensor({n}, at::kInt, table); };
  Five out{ints(tokens), ints(tokens), ints(B + 1), ints(B), ints(1)};
  rf_kv8_plan_args a{};
  a.block_table = table.data_ptr<int32_t>();
  a.cached = cached.data_ptr<int32_t>();
  a.fresh = fresh.data_ptr<int32_t>();
  a.free_blocks = free_blocks.numel() ? free_blocks.data_ptr<int32_t>() : nullptr;
  a.free_start = start.data_ptr<int32_t>();
  a.slots = std::get<0>(out).data_ptr<int32_t>();
  a.positions = std::get<1>(out).data_ptr<int32_t>();
  a.cu = std::get<2>(out).data_ptr<int32_t>();
  a.kv_lens = std::get<3>(out).data_ptr<int32_t>();
  a.free_next = std::get<4>(out).data_ptr<int32_t>();
  a.requests = cached.size(0);
  a.width = table.size(1);
  a.table_stride = a.requests <= 1 ? a.width : table.stride(0);
  a.num_free = free_blocks.numel();
  a.tokens = tokens;
  a.block_size = (int32_t)bs;
  check_status(rf_kv8_plan(&a, stream_of(table)), op);
  return out;
}

Five plan_meta(at::Tensor& table, const at::Tensor& cached, const at::Tensor& fresh,
               const at::Tensor& free_blocks, const at::Tensor& start, int64_t tokens, int64_t bs) {
  check_plan(table, cached, fresh, free_blocks, start, tokens, bs);
  return plan_outputs(cached, tokens);
}

Five plan_cpu(at::Tensor& table, const at::Tensor& cached, const at::Tensor& fresh,
              const at::Tensor& free_blocks, const at::Tensor& start, int64_t tokens, int64_t bs) {
  check_plan(table, cached, fresh, free_blocks, start, tokens, bs);
  no_cpu("kv8::plan");
}

// ---- the cache -------------------------------------------------------------------
// k_cache, v_cache: uint8 [blocks, kv_heads, block_size / 32, head_dim / 32, 1024].
void check_cache(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                 const at::Tensor& vs, const char* op) {
  TORCH_CHECK(kc.scalar_type() == at::kByte && vc.scalar_type() == at::kByte, op,
              ": k_cache and v_cache must be uint8 tiles");
  TORCH_CHECK(kc.dim() == 5 && kc.sym_size(4) == 1024 && kc.is_contiguous() && vc.is_contiguous() &&
                  kc.sym_sizes() == vc.sym_sizes(),
              op, ": k_cache and v_cache must be contiguous tiles [blocks, kv_heads, block_size / 32, "
              "head_dim / 32, 1024] of one shape, got ", kc.sym_sizes(), " and ", vc.sym_sizes());
  TORCH_CHECK(kc.sym_size(0) >= 1 && kc.sym_size(1) >= 1, op, ": the cache is empty");
  const c10::SymInt g = kc.sym_size(2), d = kc.sym_size(3);
  TORCH_CHECK(g == 1 || g == 2 || g == 4, op, ": block_size must be 32, 64 or 128, got ", g * 32);
  TORCH_CHECK(d == 2 || d == 4 || d == 8, op, ": head_dim must be 64, 128 or 256, got ", d * 32);
  for (const at::Tensor* s : {&ks, &vs})
    TORCH_CHECK(s->scalar_type() == at::kFloat && s->dim() == 2 && s->is_contiguous() &&
                    s->sym_size(0) == kc.sym_size(0) && s->sym_size(1) == kc.sym_size(1),
                op, ": k_scale and v_scale must be contiguous float32 [", kc.sym_size(0), ", ",
                kc.sym_size(1), "], got ", s->scalar_type(), " ", s->sym_sizes());
}

rf_kv8_cache cache_of(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                      const at::Tensor& vs, const char* op) {
  check_same_device(kc, kc, op, "k_cache");
  check_same_device(vc, kc, op, "v_cache");
  check_same_device(ks, kc, op, "k_scale");
  check_same_device(vs, kc, op, "v_scale");
  return {kc.data_ptr(), vc.data_ptr(), ks.data_ptr<float>(), vs.data_ptr<float>(), kc.size(0),
          (int32_t)kc.size(1), (int32_t)kc.size(3) * 32, (int32_t)kc.size(2) * 32};
}

void check_append(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                  const at::Tensor& vs, const at::Tensor& k, const at::Tensor& v,
                  const at::Tensor& slots) {
  const char* op = "kv8::append";
  check_cache(kc, vc, ks, vs, op);
  check_half(k, op, "k");
  check_ints(slots, 1, op, "slots");
  TORCH_CHECK(v.scalar_type() == k.scalar_type(), op, ": v must be ", k.scalar_type(), " as k");
  for (const at::Tensor* t : {&k, &v})
    TORCH_CHECK(t->dim() == 3 && t->sym_size(0) == slots.sym_size(0) &&
                    t->sym_size(1) == kc.sym_size(1) && t->sym_size(2) == kc.sym_size(3) * 32,
                op, ": k and v must be [", slots.sym_size(0), " tokens, ", kc.sym_size(1),
                " kv_heads, ", kc.sym_size(3) * 32, " head_dim], got ", t->sym_sizes());
}

void append_hip(at::Tensor& kc, at::Tensor& vc, at::Tensor& ks, at::Tensor& vs, const at::Tensor& k,
                const at::Tensor& v, const at::Tensor& slots) {
  RECORD_FUNCTION("kv8::append", {});
  const char* op = "kv8::append";
  check_append(kc, vc, ks, vs, k, v, slots);
  const rf_kv8_cache c = cache_of(kc, vc, ks, vs, op);
  check_same_device(k, kc, op, "k");
  check_same_device(v, kc, op, "v");
  check_same_device(slots, kc, op, "slots");
  if (slots.numel() == 0) return;
  c10::DeviceGuard dev_guard(kc.device());
  at::Tensor keep[2];
  const rf_kv8_heads kh = heads_of(k, &keep[0]), vh = heads_of(v, &keep[1]);
  check_status(rf_kv8_append(&c, &kh, &vh, dtype_code(k.scalar_type()), slots.data_ptr<int32_t>(),
                             slots.numel(), stream_of(kc)),
               op);
}

void append_meta(at::Tensor& kc, at::Tensor& vc, at::Tensor& ks, at::Tensor& vs, const at::Tensor& k,
                 const at::Tensor& v, const at::Tensor& slots) {
  check_append(kc, vc, ks, vs, k, v, slots);
}

void append_cpu(at::Tensor& kc, at::Tensor& vc, at::Tensor& ks, at::Tensor& vs, const at::Tensor& k,
                const at::Tensor& v, const at::Tensor& slots) {
  check_append(kc, vc, ks, vs, k, v, slots);
  no_cpu("kv8::append");
}

void check_read(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks,
                const at::Tensor& vs, const at::Tensor& slots, at::ScalarType dtype) {
  const char* op = "kv8::read";
  check_cache(kc, vc, ks, vs, op);
  check_ints(slots, 1, op, "slots");
  TORCH_CHECK(dtype == at::kHalf || dtype == at::kBFloat16 || dtype == at::kFloat, op,
              ": dtype must be float16, bfloat16 or float32, got ", dtype);
}

Two read_meta(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
              const at::Tensor& slots, at::ScalarType dtype) {
  check_read(kc, vc, ks, vs, slots, dtype);
  const std::vector<c10::SymInt> shape = {slots.sym_size(0), kc.sym_size(1), kc.sym_size(3) * 32};
  const auto o = kc.options().dtype(dtype);
  return {at::empty_symint(shape, o), at::empty_symint(shape, o)};
}

Two read_hip(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
             const at::Tensor& slots, at::ScalarType dtype) {
  RECORD_FUNCTION("kv8::read", {});
  const char* op = "kv8::read";
  check_read(kc, vc, ks, vs, slots, dtype);
  const rf_kv8_cache c = cache_of(kc, vc, ks, vs, op);
  check_same_device(slots, kc, op, "slots");
  const std::vector<int64_t> shape = {slots.size(0), kc.size(1), kc.size(3) * 32};
  Two out{new_tensor(shape, dtype, kc), new_tensor(shape, dtype, kc)};
  if (slots.numel() == 0) return out;
  c10::DeviceGuard dev_guard(kc.device());
  check_status(rf_kv8_read(&c, slots.data_ptr<int32_t>(), slots.numel(), dtype_code(dtype),
                           std::get<0>(out).data_ptr(), std::get<1>(out).data_ptr(), stream_of(kc)),
               op);
  return out;
}

Two read_cpu(const at::Tensor& kc, const at::Tensor& vc, const at::Tensor& ks, const at::Tensor& vs,
             const at::Tensor& slots, at::ScalarType dtype) {
  check_read(kc, vc, ks, vs, slots, dtype);
  no_cpu("kv8::read");
}

// ---- attention -------------------------------------------------------------------
void check_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                     const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                     const at::Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t max_kv,
                     bool causal, int64_t window, double scale) {
  const char* op = "kv8::attention";
  check_half(q, op, "q");
  check_cache(kc, vc, ks, vs, op);
  rf_torch::check_attention(op, q, kc.sym_size(1), kc.sym_size(3) * 32, table, lens, cu, max_q, max_kv, causal,
                            window, scale);
}

Two attention_hip(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                  const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                  const at::Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t max_kv,
                  bool causal, int64_t window, double scale, bool return_lse) {
  RECORD_FUNCTION("kv8::attention", {});
  const char* op = "kv8::attention";
  check_attention(q, kc, vc, ks, vs, table, lens, cu, max_q, max_kv, causal, window, scale);
  check_same_device(q, q, op, "q");
  rf_kv8_attention_args a{};
  a.cache = cache_of(kc, vc, ks, vs, op);
  check_same_device(kc, q, op, "k_cache");
  return run_attention(op, a, rf_kv8_attention, rf_kv8_attention_workspace, q, table, lens, cu, max_q, max_kv,
                       causal, window, scale, return_lse);
}

Two attention_meta(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                   const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                   const at::Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t max_kv,
                   bool causal, int64_t window, double scale, bool return_lse) {
  check_attention(q, kc, vc, ks, vs, table, lens, cu, max_q, max_kv, causal, window, scale);
  return attention_outputs(q, return_lse);
}

Two attention_cpu(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                  const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                  const at::Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t max_kv,
                  bool causal, int64_t window, double scale, bool) {
  check_attention(q, kc, vc, ks, vs, table, lens, cu, max_q, max_kv, causal, window, scale);
  no_cpu("kv8::attention");
}

}  // namespace

TORCH_LIBRARY(kv8, m) {
  m.def("qk_norm_rope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor? cos, "
        "Tensor? sin, Tensor? positions, float eps, bool interleaved) -> (Tensor, Tensor)");
  m.def("plan(Tensor(a!) block_table, Tensor cached_lens, Tensor new_lens, Tensor free_blocks, "
        "Tensor free_start, int num_tokens, int block_size) "
        "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("append(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, "
        "Tensor k, Tensor v, Tensor slots) -> ()");
  m.def("read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor slots, "
        "ScalarType dtype) -> (Tensor, Tensor)");
  m.def("attention(Tensor q, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor kv_lens, Tensor? cu_q, int max_q_len, int max_kv_len, "
        "bool causal, int window, float scale, bool return_lse) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(kv8, CUDA, m) {
  m.impl("qk_norm_rope", TORCH_FN(rope_hip));
  m.impl("plan", TORCH_FN(plan_hip));
  m.impl("append", TORCH_FN(append_hip));
  m.impl("read", TORCH_FN(read_hip));
  m.impl("attention", TORCH_FN(attention_hip));
}
TORCH_LIBRARY_IMPL(kv8, Meta, m) {
  m.impl("qk_norm_rope", TORCH_FN(rope_meta));
  m.impl("plan", TORCH_FN(plan_meta));
  m.impl("append", TORCH_FN(append_meta));
  m.impl("read", TORCH_FN(read_meta));
  m.impl("attention", TORCH_FN(attention_meta));
}
TORCH_LIBRARY_IMPL(kv8, CPU, m) {
  m.impl("qk_norm_rope", TORCH_FN(rope_cpu));
  m.impl("plan", TORCH_FN(plan_cpu));
  m.impl("append", TORCH_FN(append_cpu));
  m.impl("read", TORCH_FN(read_cpu));
  m.impl("attention", TORCH_FN(attention_cpu));
}
// Not differentiable, as the W8A16 ops: autograd falls through.
TORCH_LIBRARY_IMPL(kv8, Autograd, m) {
  for (const char* op : {"qk_norm_rope", "plan", "append", "read", "attention"})
    m.impl(op, torch::CppFunction::makeFallthrough());
}

// Norms and rotation do not depend on the cache: the forms for several axes have a
// namespace of their own.
TORCH_LIBRARY(rope, m) {
  m.def("qk_norm_mrope(Tensor q, Tensor k, Tensor? q_weight, Tensor? k_weight, Tensor cos, "
        "Tensor sin, Tensor positions, int[] sections, bool mixed, float eps, bool interleaved) "
        "-> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(rope, CUDA, m) { m.impl("qk_norm_mrope", TORCH_FN(mrope_hip)); }
TORCH_LIBRARY_IMPL(rope, Meta, m) { m.impl("qk_norm_mrope", TORCH_FN(mrope_meta)); }
TORCH_LIBRARY_IMPL(rope, CPU, m) { m.impl("qk_norm_mrope", TORCH_FN(mrope_cpu)); }
TORCH_LIBRARY_IMPL(rope, Autograd, m) { m.impl("qk_norm_mrope", torch::CppFunction::makeFallthrough()); }
