// What surrounds the attention over the 4-bit paged cache (kv4.h): the quantizing
// append and the read-back.  Both are bound by the 16-bit side's bytes on long
// batches and by the launch on single tokens.
#include "kv4_common.h"

namespace rf {
namespace {

constexpr int kThreads = 256;

// LP = D / 8 lanes hold one row (token, head, side), eight dimensions each; the
// lanes after them hold the other side's row.  A workgroup takes the tokens of one
// head, 256 / (2 LP) at a time, kTurns times: 32 tokens that follow each other are
// what fills the cache lines they are written to.
template <typename Op>
__device__ __forceinline__ float over_lanes(float v, int lp, Op op) {
  const auto step = [&](auto ctrl) {
    v = op(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl(), 0xf,
                                                                    0xf, true)));
  };
  step([] { return 0xB1; });             // lanes 1, 0, 3, 2 of a quad
  step([] { return 0x4E; });             // 2, 3, 0, 1
  step([] { return 0x141; });            // mirrored in eight
  if (lp >= 16) step([] { return 0x140; });  // mirrored in sixteen
  if (lp >= 32) v = op(v, __shfl_xor(v, 16));
  return v;
}

// rint(x / s), where r is 1 / s to an ulp: the quotient's one correction, t + r (x -
// t s) (Markstein 1990), makes it exact where it is a tie, and x / s with x of 11
// bits and s of 7 is at least 2^-19 of itself away from every other one.
__device__ __forceinline__ float rounded_quotient(float x, float s, float r) {
  const float t = x * r;
  return __builtin_rintf(__builtin_fmaf(__builtin_fmaf(-t, s, x), r, t));
}

struct AppendArgs {
  const uint8_t* x[2];   // k, v
  int64_t ts[2], hs[2];  // bytes
  uint8_t* store[2];
  uint16_t* rows;
  const int32_t* slots;
  int64_t tokens, num_blocks;
  int heads, shift;      // log2(block size)
};

template <typename T, int D, int kTurns>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(AppendArgs a) {
  constexpr int LP = D / 8, kTokens = kThreads / (2 * LP);
  const int tid = threadIdx.x, sub = tid % LP, side = tid / LP % 2, d = sub * 8;
  const unsigned part = blockIdx.x / (unsigned)a.heads;
  const int h = (int)(blockIdx.x - part * a.heads);
  const int64_t t0 = (int64_t)part * (kTokens * kTurns) + tid / (2 * LP);
  const uint8_t* src = (side ? a.x[1] : a.x[0]) + h * (side ? a.hs[1] : a.hs[0]) + d * 2;
  const int64_t ts = side ? a.ts[1] : a.ts[0];
  uint4 raw[kTurns];
  int32_t slot[kTurns];
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const int64_t t = t0 + i * kTokens;
    raw[i] = make_uint4(0, 0, 0, 0);
    slot[i] = -1;
    if (t < a.tokens) {
      raw[i] = load_u4(src + t * ts);
      slot[i] = a.slots[t];
    }
  }
#pragma unroll
  for (int i = 0; i < kTurns; ++i) {
    const floatx8 x = Eight<T>::load(&raw[i]);
    float low = 0.0f, high = 0.0f, nan = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      low = fminf(low, x[j]);
      high = fmaxf(high, x[j]);
      nan = __builtin_fmaf(x[j], 0.0f, nan);  // (NaN where x is not finite)
    }
    low = over_lanes(low, LP, [](float u, float v) { return fminf(u, v); });
    high = over_lanes(high, LP, [](float u, float v) { return fmaxf(u, v); });
    // either side of the token's row
    const uint64_t odd = __ballot(nan != nan);
    const int lane = tid % kWave, from = lane / (2 * LP) * (2 * LP);
    const bool bad = (odd >> from & (~0ull >> (kWave - 2 * LP))) != 0;
    const float span = high - low;
    // the least step of seven bits (of 2^-20 where fp16 has no more) with 15 of it
    // at least the span: span / 15 cut to those bits, and one up where that was less
    const float least = fminf(fmaxf(span * (1.0f / 15.0f), 0x1p-20f), 4352.0f);
    const uint32_t power = __builtin_bit_cast(uint32_t, least) & 0x7f800000u;
    const float ulp = fmaxf(__builtin_bit_cast(float, power) * 0x1p-6f, 0x1p-20f);
    const float inv = __builtin_bit_cast(float, 0x7f000000u - __builtin_bit_cast(uint32_t, ulp));
    float s = __builtin_truncf(least * inv) * ulp;
    if (15.0f * s < span) s = fminf(s + ulp, 4352.0f);
    const float r = __builtin_amdgcn_rcpf(s);
    const float z = fminf(rounded_quotient(-low, s, r), 15.0f);
    uint32_t n[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      n[j] = (uint32_t)__builtin_amdgcn_fmed3f(rounded_quotient(x[j], s, r) + z, 0.0f, 15.0f);
    uint32_t word = __builtin_bit_cast(uint16_t, (_Float16)s) | (uint32_t)z;
    uint32_t even = n[0] | n[2] << 4 | n[4] << 8 | n[6] << 12, odds = n[1] | n[3] << 4 | n[5] << 8 | n[7] << 12;
    uint32_t lo = n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12, hi = n[4] | n[5] << 4 | n[6] << 8 | n[7] << 12;
    if (bad) {
      word = side ? RF_KV4_EMPTY : RF_KV4_NAN;
      even = odds = lo = hi = 0;
    }
    const int64_t block = slot[i] >> a.shift;
    if (slot[i] < 0 || block >= a.num_blocks) continue;
    const int o = slot[i] & ((1 << a.shift) - 1);
    const int64_t group = (block * a.heads + h) * (1 << (a.shift - 5)) + o / 32;
    if (side) {
      uint8_t* p = a.store[1] + group * (16 * D) + v4_at<D>(o % 32, d);
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)lo;
      *reinterpret_cast<uint16_t*>(p + 16) = (uint16_t)hi;
    } else {
      *reinterpret_cast<uint32_t*>(a.store[0] + group * (16 * D) + k4_at<D>(o % 32, d)) = even | odds << 16;
    }
    if (sub == 0) a.rows[group * 64 + side * 32 + o % 32] = (uint16_t)word;
  }
}

// ---------------------------------------------------------------------------
// Read-back.  A workgroup takes kEntries entries of the list and one head.  Entries
// whose slots follow each other inside eight tokens are a unit: a thread loads 16
// bytes of one, which are sixteen dimensions of two of its keys, or four dimensions
// of all eight values, and writes those that the list asks for.  A list of runs,
// wherever they begin, moves few bytes twice that way (9001 tokens, 8 heads of 128:
// 10.6 us, 4.4 TB/s; token by token 19.8).  Where the entries are mostly single
// tokens, a thread takes eight dimensions of one.
// ---------------------------------------------------------------------------
struct ReadArgs {
  const uint8_t* store[2];
  const uint16_t* rows;
  const int32_t* slots;
  int64_t n, num_blocks;
  int heads, shift;
  uint8_t* out[2];
};

// The value of one number, NaN where the token's word of the keys says so.
struct Row {
  float s, z;
  __device__ __forceinline__ Row(uint32_t word, uint32_t key) : z((float)(word & 15)) {
    s = key == RF_KV4_NAN ? __builtin_nanf("") : (float)__builtin_bit_cast(_Float16, (uint16_t)(word & 0xfff0u));
  }
  __device__ __forceinline__ float at(uint32_t n) const { return ((float)(n & 15) - z) * s; }
};

template <typename T>
__device__ __forceinline__ void store4(void* p, floatx4 v) {
  typedef T tx4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<tx4*>(p) = __builtin_convertvector(v, tx4);
}

template <typename T, int D, int kEntries>
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(ReadArgs a) {
  constexpr int kItems = D / 4;  // of a unit and side
  __shared__ int firsts[kEntries + 1], places[kEntries], all[kEntries];
  const int tid = threadIdx.x, lane = tid % kWave;
  const unsigned part = blockIdx.x / (unsigned)a.heads;
  const int h = (int)(blockIdx.x - part * a.heads);
  const int64_t t0 = (int64_t)part * kEntries;
  const int count = (int)(a.n - t0 < kEntries ? a.n - t0 : kEntries);
  int32_t slot = lane < count ? a.slots[t0 + lane] : -1;
  if ((slot >> a.shift) >= a.num_blocks) slot = -1;
  const int32_t before = __shfl_up(slot, 1);
  const bool first = lane < count && (lane == 0 || slot < 0 || slot != before + 1 || slot % 8 == 0);
  const uint32_t mask = (uint32_t)__ballot(first);
  const int units = __popc(mask);
  if (tid < kWave) {
    if (lane < count) all[lane] = slot;
    if (first) {
      const int u = __popc(mask & ((1u << lane) - 1));
      firsts[u] = lane;
      places[u] = slot;
    }
    if (lane == 0) firsts[units] = count;
  }
  __syncthreads();
  if (2 * units > count) {
    for (int it = tid; it < count * kItems; it += kThreads) {
      const int e = it / kItems, d = it % (D / 8) * 8, side = it / (D / 8) % 2;
      const int32_t place = all[e];
      const int64_t block = place >> a.shift;
      const int o = place & ((1 << a.shift) - 1);
      const int64_t group = (block * a.heads + h) * (1 << (a.shift - 5)) + o / 32;
      uint32_t x = 0, y = 0, word = 0, key = 0;
      if (place >= 0) {
        const uint8_t* p = (side ? a.store[1] : a.store[0]) + group * (16 * D) +
                           (side ? v4_at<D>(o % 32, d) : k4_at<D>(o % 32, d));
        x = *reinterpret_cast<const uint16_t*>(p);
        y = *reinterpret_cast<const uint16_t*>(p + (side ? 16 : 2));
        word = a.rows[group * 64 + side * 32 + o % 32];
        key = a.rows[group * 64 + o % 32];
      }
      const Row r(word, key);
      // keys: even dimensions, odd ones; values: the first four, the next
      floatx8 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float f = r.at(x >> (4 * j)), g = r.at(y >> (4 * j));
        if (side) v[j] = f, v[4 + j] = g;
        else v[2 * j] = f, v[2 * j + 1] = g;
      }
      Eight<T>::store((side ? a.out[1] : a.out[0]) + (((t0 + e) * a.heads + h) * D + d) * (int64_t)sizeof(T), v);
    }
    return;
  }
  for (int it = tid; it < 2 * units * kItems; it += kThreads) {
    const bool side = it >= units * kItems;
    const int u = (side ? it - units * kItems : it) / kItems, item = it % kItems;
    const int e0 = firsts[u], e1 = firsts[u + 1], place = places[u];
    const int64_t block = place >> a.shift;
    const int o = place & ((1 << a.shift) - 1), token = o % 32 & ~7, skip = o % 8;
    const int64_t group = (block * a.heads + h) * (1 << (a.shift - 5)) + o / 32;
    const uint16_t* words = a.rows + group * 64 + token;
    const int64_t row = (t0 + e0) * a.heads + h;  // of the unit's first entry
    if (side) {
      uint4 n = make_uint4(0, 0, 0, 0), vw = n, kw = n;
      if (place >= 0) {
        n = load_u4(a.store[1] + group * (16 * D) + v4_at<D>(token, item * 4));
        vw = load_u4(words + 32);
        kw = load_u4(words);
      }
      const uint32_t ns[4] = {n.x, n.y, n.z, n.w}, vs[4] = {vw.x, vw.y, vw.z, vw.w}, ks[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = place < 0 ? i : i - skip;
        if (at < 0 || e0 + at >= e1) continue;
        const uint32_t x = ns[i / 2] >> (16 * (i % 2));
        const Row r(vs[i / 2] >> (16 * (i % 2)) & 0xffffu, ks[i / 2] >> (16 * (i % 2)) & 0xffffu);
        store4<T>(a.out[1] + ((row + (int64_t)at * a.heads) * D + item * 4) * (int64_t)sizeof(T),
                  floatx4{r.at(x), r.at(x >> 4), r.at(x >> 8), r.at(x >> 12)});
      }
    } else {
      const int b = item % 4, d = item / 4 * 16;
      uint4 n = make_uint4(0, 0, 0, 0);
      uint32_t w[2] = {0, 0};
      if (place >= 0) {
        n = load_u4(a.store[0] + group * (16 * D) + k4_at<D>(token + b, d));
        w[0] = words[b];
        w[1] = words[b + 4];
      }
      const uint32_t ns[4] = {n.x, n.y, n.z, n.w};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int at = place < 0 ? 4 * i + b : 4 * i + b - skip;
        if (at < 0 || e0 + at >= e1) continue;
        const Row r(w[i], w[i]);
        uint8_t* to = a.out[0] + ((row + (int64_t)at * a.heads) * D + d) * (int64_t)sizeof(T);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          floatx8 y;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = r.at(ns[2 * i + j] >> (4 * (e / 2 + 4 * (e % 2))));
          Eight<T>::store(to + j * 8 * sizeof(T), y);
        }
      }
    }
  }
}

inline int log2i(int v) { return __builtin_ctz((unsigned)v); }

// Workgroups of one turn while they leave CUs idle, of 32 tokens after.
template <int D>
bool few(int64_t tokens, int heads) {
  return tokens * heads <= 256 * (kThreads / (D / 4)) * 4;
}

template <typename T, int D, int kTurns>
hipError_t append_turns(AppendArgs a, hipStream_t stream) {
  constexpr int64_t kTokens = kThreads / (D / 4) * kTurns;
  const int64_t most = kMaxThreads / kThreads / a.heads * kTokens;  // tokens of a launch
  for (int64_t left = a.tokens; left > 0; left -= most) {
    a.tokens = left < most ? left : most;
    kv4_append_kernel<T, D, kTurns><<<(unsigned)(ceil_div(a.tokens, kTokens) * a.heads), kThreads, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.slots += a.tokens;
    for (int i = 0; i < 2; ++i) a.x[i] += a.tokens * a.ts[i];
  }
  return hipSuccess;
}

template <typename T, int D>
hipError_t append_sized(const AppendArgs& a, hipStream_t stream) {
  return few<D>(a.tokens, a.heads) ? append_turns<T, D, 1>(a, stream) : append_turns<T, D, D / 32>(a, stream);
}

template <typename T>
hipError_t append_typed(const AppendArgs& a, int D, hipStream_t stream) {
  return D == 64 ? append_sized<T, 64>(a, stream)
         : D == 128 ? append_sized<T, 128>(a, stream)
                    : append_sized<T, 256>(a, stream);
}

template <typename T, int D, int kEntries>
hipError_t read_sized(ReadArgs a, hipStream_t stream) {
  const int64_t most = kMaxThreads / kThreads / a.heads * kEntries;  // entries of a launch
  for (int64_t left = a.n; left > 0; left -= most) {
    a.n = left < most ? left : most;
    kv4_read_kernel<T, D, kEntries><<<(unsigned)(ceil_div(a.n, kEntries) * a.heads), kThreads, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.slots += a.n;
    for (int i = 0; i < 2; ++i) a.out[i] += a.n * a.heads * D * (int64_t)sizeof(T);
  }
  return hipSuccess;
}

template <typename T>
hipError_t read_typed(const ReadArgs& a, int D, hipStream_t stream) {
  // (few entries: in pieces of 8, which leave fewer CUs idle)
  const bool few = a.n * a.heads <= 8192;
  return D == 64    ? few ? read_sized<T, 64, 8>(a, stream) : read_sized<T, 64, 32>(a, stream)
         : D == 128 ? few ? read_sized<T, 128, 8>(a, stream) : read_sized<T, 128, 32>(a, stream)
                    : few ? read_sized<T, 256, 8>(a, stream) : read_sized<T, 256, 32>(a, stream);
}

}  // namespace

hipError_t launch_kv4_append(const rf_kv4_cache& c, const rf_kv8_heads& k, const rf_kv8_heads& v,
                             int dtype, const int32_t* slots, int64_t tokens, hipStream_t stream) {
  AppendArgs a{};
  a.x[0] = (const uint8_t*)k.data;
  a.x[1] = (const uint8_t*)v.data;
  a.ts[0] = k.token_stride * 2;
  a.ts[1] = v.token_stride * 2;
  a.hs[0] = k.head_stride * 2;
  a.hs[1] = v.head_stride * 2;
  a.store[0] = (uint8_t*)c.k;
  a.store[1] = (uint8_t*)c.v;
  a.rows = c.rows;
  a.slots = slots;
  a.tokens = tokens;
  a.num_blocks = c.num_blocks;
  a.heads = c.kv_heads;
  a.shift = log2i(c.block_size);
  return dtype == RF_W8A16_DTYPE_F16 ? append_typed<_Float16>(a, c.head_dim, stream)
                                     : append_typed<__bf16>(a, c.head_dim, stream);
}

hipError_t launch_kv4_read(const rf_kv4_cache& c, const int32_t* slots, int64_t n, int dtype,
                           void* k_out, void* v_out, hipStream_t stream) {
  const ReadArgs a{{(const uint8_t*)c.k, (const uint8_t*)c.v}, c.rows, slots, n, c.num_blocks,
                   c.kv_heads, log2i(c.block_size), {(uint8_t*)k_out, (uint8_t*)v_out}};
  return dtype == RF_W8A16_DTYPE_F16    ? read_typed<_Float16>(a, c.head_dim, stream)
         : dtype == RF_W8A16_DTYPE_BF16 ? read_typed<__bf16>(a, c.head_dim, stream)
                                        : read_typed<float>(a, c.head_dim, stream);
}

}  // namespace rf
