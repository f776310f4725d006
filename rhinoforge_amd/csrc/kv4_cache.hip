// What surrounds the attention over the 4-bit paged cache (kv4.h): the quantizing
// append and the read-back.  Both are bound by the 16-bit side's bytes on long
// batches and by the launch on single tokens.
#include "kv4_common.h"

namespace rf {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Append.  LP = D / 16 lanes hold one row (token, head, side), sixteen dimensions
// each; the LP lanes after them hold the other side's row.  A workgroup takes 256 /
// (2 LP) tokens of one head.  A prompt runs in one or two rounds of workgroups, which
// load, compute and store one after the other, so what counts beside the bytes are
// the vector instructions: 6874 tokens of 8 heads of 128 take 10.6 us (35.6 MB, 3.4
// TB/s), with eight dimensions a lane and the numbers put together by shifts and ORs
// 13.8.  Workgroups that take several tokens a lane gain nothing (2000 tokens: 5.0
// us, in half as many workgroups 5.0; 1000: 3.1 and 3.8).
// ---------------------------------------------------------------------------
template <typename Op>
__device__ __forceinline__ float over_lanes(float v, int lp, Op op) {
  const auto step = [&](auto ctrl) {
    v = op(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl(), 0xf, 0xf,
                                                                    true)));
  };
  step([] { return 0xB1; });                 // lanes 1, 0, 3, 2 of a quad
  step([] { return 0x4E; });                 // 2, 3, 0, 1
  if (lp >= 8) step([] { return 0x141; });   // mirrored in eight
  if (lp >= 16) step([] { return 0x140; });  // mirrored in sixteen
  return v;
}

// x / s, where r is 1 / s to an ulp: the quotient's one correction, t + r (x - t s)
// (Markstein 1990), makes it exact where it is a tie, and x / s with x of 11 bits and
// s of 7 is at least 2^-19 of itself away from every other one.
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float t = x * r;
  return __builtin_fmaf(__builtin_fmaf(-t, s, x), r, t);
}

// The bits of 1.5 2^23: the sum with a small number holds its nearest integer (ties
// to even) in its low bits, and sums of those with shifts of 4, 8, .. put numbers
// next to each other.
constexpr float kMagic = 12582912.0f;
constexpr int kMagicBits = 0x4b400000;

struct AppendArgs {
  const uint8_t* x[2];   // k, v
  int64_t ts[2], hs[2];  // bytes
  uint8_t* store[2];
  uint16_t* rows;
  const int32_t* slots;
  int64_t tokens, num_blocks;
  int heads, shift;      // log2(block size)
};

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(AppendArgs a) {
  constexpr int LP = D / 16, kTokens = kThreads / (2 * LP);
  const int tid = threadIdx.x, sub = tid % LP, side = tid / LP % 2, d = sub * 16;
  const unsigned part = blockIdx.x / (unsigned)a.heads;
  const int h = (int)(blockIdx.x - part * a.heads);
  const int64_t t = (int64_t)part * kTokens + tid / (2 * LP);
  const uint8_t* src = (side ? a.x[1] : a.x[0]) + h * (side ? a.hs[1] : a.hs[0]) + d * 2;
  uint4 raw[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  int32_t slot = -1;
  if (t < a.tokens) {
    src += t * (side ? a.ts[1] : a.ts[0]);
    raw[0] = load_u4(src);
    raw[1] = load_u4(src + 16);
    slot = a.slots[t];
  }
  float x[16];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const floatx8 f = Eight<T>::load(&raw[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[8 * j + e] = f[e];
  }
  float low = 0.0f, high = 0.0f;  // (NaN where an x is)
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    low = __builtin_elementwise_minimum(low, x[j]);
    high = __builtin_elementwise_maximum(high, x[j]);
  }
  // an infinity or NaN on either side of the token's row
  const uint64_t odd = __ballot(!(high < __builtin_inff()) || !(low > -__builtin_inff()));
  const int lane = tid % kWave, from = lane / (2 * LP) * (2 * LP);
  const bool bad = (odd >> from & (~0ull >> (kWave - 2 * LP))) != 0;
  low = over_lanes(low, LP, [](float u, float v) { return fminf(u, v); });
  high = over_lanes(high, LP, [](float u, float v) { return fmaxf(u, v); });
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
  const int z = (int)fminf(__builtin_rintf(quotient(-low, s, r)), 15.0f);
  // numbers plus (magic - z), within magic - z .. magic - z + 15
  const int base = kMagicBits - z;
  const float least_n = __builtin_bit_cast(float, base), most_n = __builtin_bit_cast(float, base + 15);
  uint32_t word[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    uint32_t sum = 0;
#pragma unroll
    for (int e = 7; e >= 0; --e) {
      const float n = __builtin_amdgcn_fmed3f(quotient(x[8 * j + e], s, r) + kMagic, least_n, most_n);
      sum = (sum << 4) + __builtin_bit_cast(uint32_t, n);
    }
    word[j] = sum - (uint32_t)base * 0x11111111u;
  }
  uint32_t row = __builtin_bit_cast(uint16_t, (_Float16)s) | (uint32_t)z;
  if (bad) {
    row = side ? RF_KV4_EMPTY : RF_KV4_NAN;
    word[0] = word[1] = 0;
  }
  const int64_t block = slot >> a.shift;
  if (slot < 0 || block >= a.num_blocks) return;
  const int o = slot & ((1 << a.shift) - 1);
  const int64_t group = (block * a.heads + h) * (1 << (a.shift - 5)) + o / 32;
  if (side) {
    uint8_t* p = a.store[1] + group * (16 * D) + v4_at<D>(o % 32, d);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint16_t*>(p + 16 * j) = (uint16_t)(word[j / 2] >> (16 * (j % 2)));
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // even dimensions to the low half, odd ones to the high half
      uint32_t w = word[j];
      uint32_t m = (w ^ (w >> 4)) & 0x00f000f0u;
      w ^= m ^ (m << 4);
      m = (w ^ (w >> 8)) & 0x0000ff00u;
      word[j] = w ^ m ^ (m << 8);
    }
    *reinterpret_cast<uint2*>(a.store[0] + group * (16 * D) + k4_at<D>(o % 32, d)) = make_uint2(word[0], word[1]);
  }
  if (sub == 0) a.rows[group * 64 + side * 32 + o % 32] = (uint16_t)row;
}

// ---------------------------------------------------------------------------
// Read-back.  A workgroup takes kEntries entries of the list and one head.  Entries
// whose slots follow each other inside eight tokens are a unit: a thread loads 16
// bytes of one, which are sixteen dimensions of two of its keys, or four dimensions
// of all eight values, and writes those that the list asks for.  A list of runs,
// wherever they begin, moves few bytes twice that way (9001 tokens, 8 heads of 128:
// 10.9 us, 4.3 TB/s; token by token 19.8).  Where the entries are mostly single
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

template <typename T, int D>
hipError_t append_sized(AppendArgs a, hipStream_t stream) {
  constexpr int64_t kTokens = kThreads / (D / 8);
  const int64_t most = kMaxThreads / kThreads / a.heads * kTokens;  // tokens of a launch
  for (int64_t left = a.tokens; left > 0; left -= most) {
    a.tokens = left < most ? left : most;
    kv4_append_kernel<T, D><<<(unsigned)(ceil_div(a.tokens, kTokens) * a.heads), kThreads, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    a.slots += a.tokens;
    for (int i = 0; i < 2; ++i) a.x[i] += a.tokens * a.ts[i];
  }
  return hipSuccess;
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
  // Few entries go in pieces of 8, which single tokens need to have enough loads under
  // way; runs fill one round of workgroups either way (8 heads of 128, pieces of 32 and of
  // 8: 128 single tokens 4.8 and 3.1 us, 1024 6.7 and 5.5, 4096 13.1 and 13.2; tokens in
  // runs of 64, 128 of them 3.3 and 4.1, 1024 3.8 and 4.6, 4096 6.9 and 9.7).
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
