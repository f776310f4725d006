// What the torch ops of the paged caches share (kv8_torch.cpp, kv4_torch.cpp): checks,
// operands as the C ABI takes them, attention calls.
#pragma once

#include <ATen/ATen.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <vector>

#include "../../include/kv4.h"
#include "torch_scratch.h"

namespace rf_torch {


using OptTensor = c10::optional<at::Tensor>;

inline bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

inline void check_status(int st, const char* op) {
  TORCH_CHECK(st == RF_W8A16_OK, op, ": ", rf_w8a16_status_str(st), " (status ", st, ")");
}

inline int32_t dtype_code(at::ScalarType t) {
  return t == at::kHalf ? RF_W8A16_DTYPE_F16 : t == at::kBFloat16 ? RF_W8A16_DTYPE_BF16 : RF_W8A16_DTYPE_F32;
}

inline void check_half(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16, op, ": ", name,
              " must be float16 or bfloat16, got ", t.scalar_type());
}

inline void check_ints(const at::Tensor& t, int64_t dim, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.dim() == dim, op, ": ", name, " must have ", dim, " dimension(s), got shape ",
              t.sym_sizes());
  TORCH_CHECK(dim != 1 || t.is_contiguous(), op, ": ", name, " must be contiguous");
}

inline void check_same_device(const at::Tensor& t, const at::Tensor& first, const char* op,
                       const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name,
              " must be on a HIP device (there is no CPU implementation)");
  TORCH_CHECK(t.device() == first.device(), op, ": ", name, " must be on ", first.device(), ", got ",
              t.device());
}

[[noreturn]] inline void no_cpu(const char* op) {
  TORCH_CHECK(false, op, ": tensors are on the CPU; the kernels run on a HIP device (gfx950) only "
              "and there is no CPU implementation");
}

inline void* stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// A new contiguous tensor, straight from the caching allocator (at::empty's way
// there through the dispatcher is a third of what a single-token call costs).
inline at::Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}

inline bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A [tokens, heads, D] operand as the C ABI takes it; one of another layout is
// copied (kept alive in *keep).
inline rf_kv8_heads heads_of(const at::Tensor& t, at::Tensor* keep) {
  const auto fits = [](const at::Tensor& x) {
    return x.stride(2) == 1 && (x.size(0) <= 1 || x.stride(0) % 8 == 0) &&
           (x.size(1) <= 1 || x.stride(1) % 8 == 0) && aligned16(x);
  };
  *keep = fits(t) ? t : t.is_contiguous() ? t.clone() : t.contiguous();
  const at::Tensor& x = *keep;
  return {x.data_ptr(), x.size(0) <= 1 ? x.size(1) * x.size(2) : x.stride(0),
          x.size(1) <= 1 ? x.size(2) : x.stride(1), (int32_t)x.size(1)};
}

inline at::Tensor aligned_copy(const at::Tensor& t) { return aligned16(t) ? t : t.clone(); }

// All of an attention call but its cache; `heads` and `D` are the cache's.
inline void check_attention(const char* op, const at::Tensor& q, const c10::SymInt& heads, const c10::SymInt& D,
                            const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                            int64_t max_kv, bool causal, int64_t window, double scale) {
  check_ints(table, 2, op, "block_table");
  check_ints(lens, 1, op, "kv_lens");
  TORCH_CHECK(q.dim() == 3 && q.sym_size(2) == D, op,
              ": q must be [tokens, heads, ", D, "], got ", q.sym_sizes());
  TORCH_CHECK(q.sym_size(1) >= 1 && q.sym_size(1) % heads == 0, op, ": q's heads ",
              q.sym_size(1), " must be a multiple of the cache's ", heads);
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

using Two = std::tuple<at::Tensor, at::Tensor>;

// The call itself: `a` holds the cache, `call` and `workspace` are the C ABI's.
template <typename Args, typename Call, typename Workspace>
Two run_attention(const char* op, Args& a, Call attention, Workspace workspace, const at::Tensor& q,
                  const at::Tensor& table, const at::Tensor& lens, const OptTensor& cu, int64_t max_q,
                  int64_t max_kv, bool causal, int64_t window, double scale, bool return_lse) {
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
        return attention(&a, stream);
      },
      [&] { return workspace(&a) + RF_W8A16_WS_COUNTER_BYTES; });
  check_status(st, op);
  return {out, lse};
}

inline Two attention_outputs(const at::Tensor& q, bool return_lse) {
  const auto o = q.options().dtype(at::kFloat);
  return {at::empty_symint(q.sym_sizes(), q.options()),
          return_lse ? at::empty_symint({q.sym_size(0), q.sym_size(1)}, o) : at::empty({0}, o)};
}

}  // namespace rf_torch
