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
// They are what the reference's decoders run between the W8A16 projections
// (src/fused/rpu_qwen3_model.h: head norms, RoPE, KV insert, SDPA).  Checks in
// the manner of w8a16_torch.cpp: dtype and shape first (shared with the Meta
// kernels), then devices; invalid input raises, there is no CPU computation.
#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <vector>

#include "../../include/kv8.h"
#include "torch_scratch.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void check_status(int st, const char* op) {
  TORCH_CHECK(st == RF_W8A16_OK, op, ": ", rf_w8a16_status_str(st), " (status ", st, ")");
}

int32_t dtype_code(at::ScalarType t) {
  return t == at::kHalf ? RF_W8A16_DTYPE_F16 : t == at::kBFloat16 ? RF_W8A16_DTYPE_BF16 : RF_W8A16_DTYPE_F32;
}

void check_half(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, op, ": ", name,
              " must be float16 or bfloat16, got ", t.scalar_type());
}

void check_ints(const at::Tensor& t, int64_t dim, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must have ", dim, " dimension(s), got shape ",
              t.sym_sizes());
  TORCH_CHECK(dim != 1 || t.is_contiguous(), op, ": ", name, " must be contiguous");
}

void check_same_device(const at::Tensor& t, const at::Tensor& first, const char* op,
                       const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name,
              " must be on a HIP device (there is no CPU implementation)");
  TORCH_CHECK(t.device() == first.device(), op, ": ", name, " must be on ", first.device(), ", got ",
              t.device());
}

[[noreturn]] void no_cpu(const char* op) {
  TORCH_CHECK(false, op, ": tensors are on the CPU; the kernels run on a HIP device (gfx950) only "
              "and there is no CPU implementation");
}

void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A new contiguous tensor, straight from the caching allocator (at::empty's way
// there through the dispatcher is a third of what a single-token call costs).
at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A [tokens, heads, D] operand as the C ABI takes it; one of another layout is
// copied (kept alive in *keep).
rf_kv8_heads heads_of(const at::Tensor& t, at::Tensor* keep) {
  const auto fits = [](const at::Tensor& x) {
    return x.stride(2) == 1 && (x.size(0) <= 1 || x.stride(0) % 8 == 0) &&
           (x.size(1) <= 1 || x.stride(1) % 8 == 0) && aligned16(x);
  };
  *keep = fits(t) ? t : t.is_contiguous() ? t.clone() : t.contiguous();
  const at::Tensor& x = *keep;
  return {x.data_ptr(), x.size(0) <= 1 ? x.size(1) * x.size(2) : x.stride(0),
          x.size(1) <= 1 ? x.size(2) : x.stride(1), (int32_t)x.size(1)};
}

at::Tensor aligned_copy(const at::Tensor& t) { return aligned16(t) ? t : t.clone(); }

// ---- norms and rotation ----------------------------------------------------------
void check_rope(const at::Tensor& q, const at::Tensor& k, const OptTensor& qw, const OptTensor& kw,
                const OptTensor& cos, const OptTensor& sin, const OptTensor& pos) {
  const char* op = "kv8::qk_norm_rope";
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
    if (given(pos)) {
      TORCH_CHECK((pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong) &&
                      pos->dim() == 1 && pos->sym_size(0) == q.sym_size(0) && pos->is_contiguous(),
                  op, ": positions must be a contiguous int32 or int64 [tokens]");
    } else {
      TORCH_CHECK(cos->sym_size(0) >= q.sym_size(0), op,
                  ": without positions cos and sin need a row for each token");
    }
  }
}

using Two = std::tuple<at::Tensor, at::Tensor>;

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
  at::Tensor keep[6];
  rf_kv8_rope_args a{};
  a.q = heads_of(q, &keep[0]);
  a.k = heads_of(k, &keep[1]);
  at::Tensor qo = new_tensor(q.sizes(), q.scalar_type(), q), ko = new_tensor(k.sizes(), k.scalar_type(), k);
  a.q_out = qo.data_ptr();
  a.k_out = ko.data_ptr();
  if (given(qw)) a.q_weight = (keep[2] = aligned_copy(*qw)).data_ptr();
  if (given(kw)) a.k_weight = (keep[3] = aligned_copy(*kw)).data_ptr();
  if (given(cos)) {
    a.cos = (keep[4] = aligned_copy(*cos)).data_ptr<float>();
    a.sin = (keep[5] = aligned_copy(*sin)).data_ptr<float>();
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
  if (a.tokens > 0) check_status(rf_kv8_qk_norm_rope(&a, stream_of(q)), op);
  return {qo, ko};
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
  const std::vector<int64_t> shape = {slots.size(0), kc.size(1), kc.size(3) * 32};
  Two out{new_tensor(shape, dtype, kc), new_tensor(shape, dtype, kc)};
  const rf_kv8_cache c = cache_of(kc, vc, ks, vs, op);
  check_same_device(slots, kc, op, "slots");
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
  check_ints(table, 2, op, "block_table");
  check_ints(lens, 1, op, "kv_lens");
  TORCH_CHECK(q.dim() == 3 && q.sym_size(2) == kc.sym_size(3) * 32, op,
              ": q must be [tokens, heads, ", kc.sym_size(3) * 32, "], got ", q.sym_sizes());
  TORCH_CHECK(q.sym_size(1) >= 1 && q.sym_size(1) % kc.sym_size(1) == 0, op, ": q's heads ",
              q.sym_size(1), " must be a multiple of the cache's ", kc.sym_size(1));
  const c10::SymInt B = lens.sym_size(0);
  TORCH_CHECK(B >= 1 && table.sym_size(0) == B, op, ": block_table and kv_lens differ in requests");
  TORCH_CHECK(table.sym_size(1) >= 1 && table.sym_stride(1) == 1 &&
                  (B <= 1 || table.sym_stride(0) >= table.sym_size(1)),
              op, ": block_table must have rows of unit stride, one after the other");
  if (given(cu)) {
    check_ints(*cu, 1, op, "cu_q");
    TORCH_CHECK(cu->sym_size(0) == B + 1, op, ": cu_q must have ", B + 1, " elements, got ",
                cu->sym_size(0));
  } else {
    TORCH_CHECK(q.sym_size(0) % B == 0, op, ": without cu_q the tokens (", q.sym_size(0),
                ") must be a multiple of the requests (", B, ")");
  }
  TORCH_CHECK(scale > 0 && (float)scale < std::numeric_limits<float>::infinity() && (float)scale > 0,
              op, ": scale must be positive and finite, got ", scale);
  TORCH_CHECK(window >= 0 && (window == 0 || causal), op,
              ": window must be 0 (none), or positive with causal");
  TORCH_CHECK(max_q >= 0 && max_kv >= 0, op, ": max_q_len and max_kv_len must not be negative");
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
  check_same_device(table, q, op, "block_table");
  check_same_device(lens, q, op, "kv_lens");
  if (given(cu)) check_same_device(*cu, q, op, "cu_q");
  c10::DeviceGuard dev_guard(q.device());
  at::Tensor out = new_tensor(q.sizes(), q.scalar_type(), q);
  at::Tensor lse = return_lse ? new_tensor({q.size(0), q.size(1)}, at::kFloat, q) : new_tensor({0}, at::kFloat, q);
  if (q.size(0) == 0) return {out, lse};
  at::Tensor keep;
  a.q = heads_of(q, &keep);
  if (given(cu)) a.cu_q = cu->data_ptr<int32_t>();
  a.kv_lens = lens.data_ptr<int32_t>();
  a.block_table = table.data_ptr<int32_t>();
  a.out = out.data_ptr();
  a.lse = return_lse ? lse.data_ptr<float>() : nullptr;
  a.tokens = q.size(0);
  a.requests = lens.size(0);
  a.width = table.size(1);
  a.table_stride = a.requests <= 1 ? a.width : table.stride(0);
  a.max_q_len = max_q;
  a.max_kv_len = max_kv;
  a.dtype = dtype_code(q.scalar_type());
  a.causal = causal;
  a.window = window;
  a.scale = (float)scale;
  void* stream = stream_of(q);
  const int st = rf_torch::with_scratch(
      q.device(), stream, op,
      [&](const rf_w8a16_scratch* scratch) {
        a.scratch = scratch;
        return rf_kv8_attention(&a, stream);
      },
      [&] { return rf_kv8_attention_workspace(&a) + RF_W8A16_WS_COUNTER_BYTES; });
  check_status(st, op);
  return {out, lse};
}

Two attention_meta(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& vc,
                   const at::Tensor& ks, const at::Tensor& vs, const at::Tensor& table,
                   const at::Tensor& lens, const OptTensor& cu, int64_t max_q, int64_t max_kv,
                   bool causal, int64_t window, double scale, bool return_lse) {
  check_attention(q, kc, vc, ks, vs, table, lens, cu, max_q, max_kv, causal, window, scale);
  const auto o = q.options().dtype(at::kFloat);
  return {at::empty_symint(q.sym_sizes(), q.options()),
          return_lse ? at::empty_symint({q.sym_size(0), q.sym_size(1)}, o) : at::empty({0}, o)};
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
