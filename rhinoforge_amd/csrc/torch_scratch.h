// Scratch of the split launches behind the torch ops (w8a16_torch.cpp,
// kv8_torch.cpp): one set per device and stream, shared by all of them.
#pragma once

#include <ATen/ATen.h>
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "../../include/w8a16.h"

namespace rf_torch {

// Scratch per (device, stream), in two parts (the C ABI's rf_w8a16_scratch).
// Calls on one stream are ordered and leave the counters zero, so one set per
// stream is safe to reuse.
//   counters  allocated and cleared once, on the stream itself; for a stream
//             first seen under graph capture the library's own, which nothing
//             has to clear.  Never replaced: a fill recorded into a graph would
//             clear them on that graph's replays only, and every other call on
//             the stream might find anything.
//   partials  at least kMinPartials bytes, never cleared.  A buffer that has to
//             grow, under capture too, is retired, never freed: a HIP graph
//             captured earlier on that stream may still reference it.  The next
//             one is at least twice as large, so that needs which vary from call
//             to call (the attention's) hold less than four times the largest.
constexpr int64_t kMinPartials = 16 << 20;

inline bool capturing(void* stream) {
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(static_cast<hipStream_t>(stream), &st) == hipSuccess &&
         st != hipStreamCaptureStatusNone;
}

struct ScratchCache {
  std::mutex mu;
  std::map<std::pair<int, void*>, rf_w8a16_scratch> sets;
  std::vector<at::Tensor> kept;  // every buffer handed out, until the process ends

  void* keep(at::Tensor t) {
    kept.push_back(t);
    return t.data_ptr();
  }

  // The stream's scratch with at least `bytes` of partials (current device: dev).
  rf_w8a16_scratch get(const at::Device& dev, void* stream, size_t bytes, const char* op) {
    std::lock_guard<std::mutex> g(mu);
    rf_w8a16_scratch& s = sets[std::make_pair((int)dev.index(), stream)];
    const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
    if (!s.counters) {
      if (capturing(stream)) {
        const int st = rf_w8a16_stream_counters(stream, &s.counters);
        TORCH_CHECK(st == RF_W8A16_OK, op, ": no split-K counters for a stream first used under "
                    "graph capture (status ", st, "); make one call on it before the capture "
                    "begins");
      } else {
        s.counters = keep(at::zeros({RF_W8A16_WS_COUNTER_BYTES}, opts));
      }
    }
    if (!s.partials || s.partial_bytes < bytes) {
      const auto megabytes = [](int64_t n) { return (n + (1 << 20) - 1) >> 20 << 20; };
      const int64_t need = std::max<int64_t>((int64_t)bytes, kMinPartials);
      int64_t sz = megabytes(std::max<int64_t>(need, s.partials ? 2 * (int64_t)s.partial_bytes : 0));
      try {
        s.partials = keep(at::empty({sz}, opts));
      } catch (const c10::OutOfMemoryError&) {  // what the call needs may fit still
        if (sz == megabytes(need)) throw;
        sz = megabytes(need);
        s.partials = keep(at::empty({sz}, opts));
      }
      s.partial_bytes = (size_t)sz;
    }
    return s;
  }
};

inline ScratchCache& scratch_cache() {
  static ScratchCache* c = new ScratchCache();  // lives until process exit
  return *c;
}

// Runs call(scratch) with the stream's cached scratch.  The C ABI refuses one
// that is too small with RF_W8A16_EWORKSPACE before it launches anything; only
// then is the size the shape needs queried (a second launch plan: need()
// returns the one-buffer size, counters included), the partials grown and the
// call repeated.
template <typename Call, typename Need>
int with_scratch(const at::Device& dev, void* stream, const char* op, Call call, Need need) {
  ScratchCache& cache = scratch_cache();
  rf_w8a16_scratch s = cache.get(dev, stream, 0, op);
  int st = call(&s);
  if (st == RF_W8A16_EWORKSPACE) {
    const size_t bytes = need();
    TORCH_CHECK(bytes > RF_W8A16_WS_COUNTER_BYTES, op, ": ", rf_w8a16_status_str(RF_W8A16_EINVAL));
    s = cache.get(dev, stream, bytes - RF_W8A16_WS_COUNTER_BYTES, op);
    st = call(&s);
  }
  return st;
}

}  // namespace rf_torch
