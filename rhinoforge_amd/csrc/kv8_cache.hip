// What surrounds the attention over the int8 paged cache (kv8.h): norms and
// rotation of the heads, block tables and slots, the quantizing append and the
// read-back.  All bound by memory on long batches and by the launch on single
// tokens.
#include "kv8_common.h"

namespace rf {
namespace {

// ---------------------------------------------------------------------------
// Norms and rotation.  LP lanes hold one head, eight dimensions each (16-byte
// loads and stores); a wavefront takes 64 / LP heads of one token at a time,
// with that token's cos and sin and both weights in registers for all of them.
// ---------------------------------------------------------------------------
struct RopeArgs {
  const uint8_t *q, *k;
  uint8_t *q_out, *k_out;
  int64_t q_ts, q_hs, k_ts, k_hs;  // bytes
  const uint8_t *qw, *kw;
  const float *cos, *sin;
  const void* pos;
  int64_t tokens, table_rows;
  int pos64, hq, hk, D, rot, interleaved;
  int per_wave;  // heads of a wavefront
  float eps;
};

template <typename T, int LP>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int kHeads = kWave / LP;
  const int lane = threadIdx.x % kWave, sub = lane % LP;
  const int64_t t = blockIdx.x;
  const int heads = a.hq + a.hk;
  const int first = (blockIdx.y * (blockDim.x / kWave) + threadIdx.x / kWave) * a.per_wave;
  if (first >= heads) return;
  const int end = min(first + a.per_wave, heads);
  const int d0 = sub * 8;
  const bool mine = d0 < a.D;

  // cos and sin of this lane's eight dimensions; signs so that y' = y c + partner s.
  floatx8 c = 1.0f, s = 0.0f;
  int src = lane;
  const int half = a.rot / 2;
  if (a.rot > 0) {
    const int64_t row = a.pos == nullptr ? t
                        : a.pos64        ? reinterpret_cast<const int64_t*>(a.pos)[t]
                                         : reinterpret_cast<const int32_t*>(a.pos)[t];
    const bool ok = row >= 0 && row < a.table_rows;
    const float* cr = a.cos + (ok ? row : 0) * half;
    const float* sr = a.sin + (ok ? row : 0) * half;
    const float bad = ok ? 0.0f : __builtin_nanf("");
    c = 1.0f + bad;
    if (d0 >= a.rot) {
    } else if (a.interleaved) {
      const floatx4 cv = *reinterpret_cast<const floatx4*>(cr + d0 / 2);
      const floatx4 sv = *reinterpret_cast<const floatx4*>(sr + d0 / 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[2 * i] = c[2 * i + 1] = cv[i] + bad;
        s[2 * i] = -sv[i];
        s[2 * i + 1] = sv[i];
      }
    } else {
      const bool low = d0 < half;
      const int at = low ? d0 : d0 - half;
      src = low ? lane + half / 8 : lane - half / 8;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const floatx4 cv = *reinterpret_cast<const floatx4*>(cr + at + i);
        const floatx4 sv = *reinterpret_cast<const floatx4*>(sr + at + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          c[i + j] = cv[j] + bad;
          s[i + j] = low ? -sv[j] : sv[j];
        }
      }
    }
  }
  floatx8 qw = 1.0f, kw = 1.0f;
  if (mine && a.qw) qw = Eight<T>::load(a.qw + d0 * 2);
  if (mine && a.kw) kw = Eight<T>::load(a.kw + d0 * 2);

  for (int h0 = first; h0 < end; h0 += kHeads) {
    const int h = h0 + lane / LP;
    const bool on = mine && h < end;
    const bool isq = h < a.hq;
    const uint8_t* in = isq ? a.q + t * a.q_ts + h * a.q_hs : a.k + t * a.k_ts + (h - a.hq) * a.k_hs;
    floatx8 x = 0.0f;
    if (on) x = Eight<T>::load(in + d0 * 2);
    if (isq ? a.qw != nullptr : a.kw != nullptr) {
      float ss = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i];
#pragma unroll
      for (int m = 1; m < LP; m <<= 1) ss += __shfl_xor(ss, m);
      const float r = 1.0f / sqrtf(ss / (float)a.D + a.eps);
      x = x * r * (isq ? qw : kw);
    }
    floatx8 y;
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i] * c[i] + x[i ^ 1] * s[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = x[i] * c[i] + __shfl(x[i], src) * s[i];
    }
    if (on) {
      uint8_t* out = isq ? a.q_out + (t * a.hq + h) * (int64_t)a.D * 2
                         : a.k_out + (t * a.hk + (h - a.hq)) * (int64_t)a.D * 2;
      Eight<T>::store(out + d0 * 2, y);
    }
  }
}

// ---------------------------------------------------------------------------
// Block tables and slots.  Every workgroup adds up the batch's lengths for
// itself (a scan of at most 8192 requests in LDS, cheaper than a second
// launch), then writes its share of the tokens and of the table rows.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;

__global__ __launch_bounds__(kPlanThreads) void kv8_plan_kernel(rf_kv8_plan_args a, int shift) {
  extern __shared__ int32_t lds[];
  const int B = (int)a.requests, tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int32_t* cu = lds;             // [B + 1] new tokens before request i
  int32_t* blocks = lds + B + 1; // [B + 1] new blocks before request i
  __shared__ int64_t wave_sum[2][kPlanThreads / kWave];
  const int64_t bs = a.block_size;
  const auto need_of = [&](int i, int64_t* tokens) -> int64_t {
    const int64_t c = max(a.cached[i], 0), n = max(a.fresh[i], 0);
    *tokens = n;
    return ((c + n + bs - 1) >> shift) - ((c + bs - 1) >> shift);
  };
  const int per = (B + kPlanThreads - 1) / kPlanThreads;
  const int lo = min(tid * per, B), hi = min(lo + per, B);
  int64_t st = 0, sb = 0;
  for (int i = lo; i < hi; ++i) {
    int64_t n;
    sb += need_of(i, &n);
    st += n;
  }
  int64_t pt = st, pb = sb;  // inclusive over the wavefront
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const int64_t u = __shfl_up(pt, m), v = __shfl_up(pb, m);
    if (lane >= m) {
      pt += u;
      pb += v;
    }
  }
  if (lane == kWave - 1) {
    wave_sum[0][wave] = pt;
    wave_sum[1][wave] = pb;
  }
  __syncthreads();
  pt -= st;
  pb -= sb;
  for (int w = 0; w < wave; ++w) {
    pt += wave_sum[0][w];
    pb += wave_sum[1][w];
  }
  constexpr int64_t kTop = 0x7fffffff;
  for (int i = lo; i < hi; ++i) {
    cu[i] = (int32_t)min(pt, kTop);
    blocks[i] = (int32_t)min(pb, kTop);
    int64_t n;
    pb += need_of(i, &n);
    pt += n;
  }
  if (tid == kPlanThreads - 1) {
    cu[B] = (int32_t)min(pt, kTop);
    blocks[B] = (int32_t)min(pb, kTop);
  }
  __syncthreads();

  const int64_t start = max(*a.free_start, 0);
  const auto free_at = [&](int64_t i) -> int32_t { return i < a.num_free ? a.free_blocks[i] : -1; };
  const int64_t stride = (int64_t)gridDim.x * kPlanThreads;
  const int64_t me = (int64_t)blockIdx.x * kPlanThreads + tid;
  for (int64_t i = me; i <= B; i += stride) {
    a.cu[i] = cu[i];
    if (i < B) {
      const int64_t len = (int64_t)max(a.cached[i], 0) + max(a.fresh[i], 0);
      a.kv_lens[i] = (int32_t)min(len, kTop);
    } else {
      *a.free_next = (int32_t)min(start + blocks[B], kTop);
    }
  }
  // New table entries: new block n of the batch belongs to the last request
  // that begins at or before it.
  for (int64_t n = me; n < blocks[B]; n += stride) {
    int l = 0, r = B;  // blocks[l] <= n < blocks[r]
    while (r - l > 1) {
      const int m = (l + r) / 2;
      if (blocks[m] <= n) l = m; else r = m;
    }
    const int64_t j = (((int64_t)max(a.cached[l], 0) + bs - 1) >> shift) + (n - blocks[l]);
    if (j < a.width) a.block_table[l * a.table_stride + j] = free_at(start + n);
  }
  for (int64_t t = me; t < a.tokens; t += stride) {
    int32_t slot = -1, position = 0;
    if (t < cu[B]) {
      int l = 0, r = B;
      while (r - l > 1) {
        const int m = (l + r) / 2;
        if (cu[m] <= t) l = m; else r = m;
      }
      const int64_t cached = max(a.cached[l], 0), pos = cached + (t - cu[l]);
      const int64_t j = pos >> shift, have = (cached + bs - 1) >> shift;
      // (entries from `have` on are being written by this launch)
      const int64_t block = j >= a.width ? -1
                            : j < have   ? a.block_table[l * a.table_stride + j]
                                         : free_at(start + blocks[l] + (j - have));
      position = (int32_t)min(pos, kTop);
      if (block >= 0) slot = (int32_t)min(block * bs + (pos & (bs - 1)), kTop);
    }
    a.slots[t] = slot;
    a.positions[t] = position;
  }
}

// ---------------------------------------------------------------------------
// Append.  A run is a maximal sequence of consecutive slots inside one block
// among consecutive tokens; one workgroup quantizes one head of it, k or v:
// the largest magnitude, the new scale, the held values again if the scale
// rose, the new ones.  v is gathered by tiles of dimensions, through LDS.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const uint8_t* x[2];     // k, v
  int64_t ts[2], hs[2];    // bytes
  uint8_t* store[2];
  float* scale[2];
  const int32_t* slots;
  int64_t tokens, num_blocks;
  int heads, shift;        // log2(block size)
  int chunk;               // consecutive tokens whose runs one workgroup begins
};

constexpr float kLeastAmax = 0x1p-100f;

// rint(x / step) as a stored byte.  x / step by a correctly rounded reciprocal
// and one correction, t + r (x - t step) (Markstein 1990).
__device__ __forceinline__ uint32_t quant_byte(float x, float step, float r) {
  const float t = x * r;
  const float q = rintf(__builtin_fmaf(__builtin_fmaf(-t, step, x), r, t));
  return (uint32_t)((int)fminf(fmaxf(q, -127.0f), 127.0f) + 128);
}
__device__ __forceinline__ uint32_t requant_byte(uint32_t u, float ratio) {
  return (uint32_t)((int)rintf((float)((int)u - 128) * ratio) + 128) & 0xffu;
}
__device__ __forceinline__ uint32_t byte_of(uint4 v, int i) {
  const uint32_t w = i < 4 ? v.x : i < 8 ? v.y : i < 12 ? v.z : v.w;
  return (w >> (8 * (i & 3))) & 0xffu;
}

template <typename T, int D, int NT>
__global__ __launch_bounds__(NT) void kv8_append_kernel(AppendArgs a) {
  extern __shared__ uint8_t staged[];  // v: [tokens of the run][D] bytes
  __shared__ uint32_t wave_amax[NT / kWave];
  const int tid = threadIdx.x, lane = tid % kWave;
  const int h = blockIdx.y, side = blockIdx.z;
  const int bs = 1 << a.shift;
  const uint8_t* x0 = a.x[side] + h * a.hs[side];
  const int64_t ts = a.ts[side];
  const int64_t t_end = min((int64_t)(blockIdx.x + 1) * a.chunk, a.tokens);
  for (int64_t t = (int64_t)blockIdx.x * a.chunk; t < t_end; ++t) {
    // ---- the run that begins at t, if one does (the same in every wavefront)
    const int32_t slot = a.slots[t];
    const int64_t block = slot >> a.shift;
    const int o0 = slot & (bs - 1);
    if (slot < 0 || block >= a.num_blocks) continue;
    if (o0 != 0 && t > 0 && a.slots[t - 1] == slot - 1) continue;
    int n = 0;
    for (bool more = true; more && n < bs - o0;) {
      const int i = n + lane;
      const bool same = i < bs - o0 && t + i < a.tokens && a.slots[t + i] == slot + i;
      const uint64_t b = __ballot(same);
      const int len = b == ~0ull ? kWave : __builtin_ctzll(~b);
      n += len;
      more = len == kWave;
    }
    // ---- the largest magnitude, as the bits of |x| (a NaN is above infinity)
    uint32_t top = 0;
    for (int it = tid; it < n * (D / 8); it += NT) {
      const int i = it / (D / 8), d = it % (D / 8) * 8;
      const uint4 v = load_u4(x0 + (t + i) * ts + d * 2);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        top = max(top, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    if (lane == 0) wave_amax[tid / kWave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / kWave; ++w) top = max(top, wave_amax[w]);
    const float amax = (float)__builtin_bit_cast(T, (uint16_t)top);
    float* scale = a.scale[side] + block * a.heads + h;
    const float before = o0 > 0 ? *scale : 0.0f;
    const float fresh = amax < kLeastAmax ? 0.0f : amax * (1.0f / 127.0f);
    // max of the two; either one not finite makes the block not finite
    const float step = before >= fresh || before != before ? before : fresh;
    const bool rise = o0 > 0 && !(step == before) && before == before;
    const float ratio = rise ? before / step : 1.0f;
    const bool some = step > 0.0f && step < __builtin_inff();  // else all zeros
    const float r = some ? 1.0f / step : 0.0f;
    __syncthreads();  // every thread has read the scale and wave_amax
    if (tid == 0) *scale = step;
    uint8_t* dst = a.store[side] + (block * a.heads + h) * ((int64_t)D << a.shift);
    if (side == 0) {
      // 16 dimensions of one token are 16 consecutive bytes.
      const int begin = rise ? 0 : o0 * (D / 16);
      for (int it = begin + tid; it < (o0 + n) * (D / 16); it += NT) {
        const int o = it / (D / 16), dc = it % (D / 16);  // token, 16 dimensions
        uint8_t* p = dst + (o >> 5) * (32 * D) + ((o >> 4 & 1) * (D / 64) + (dc >> 2)) * kTileBytes +
                     ((dc & 3) * 16 + (o & 15)) * 16;
        uint32_t w[4];
        if (o < o0) {
          const uint4 v = load_u4(p);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) w[j] |= requant_byte(byte_of(v, 4 * j + b), ratio) << (8 * b);
          }
        } else {
          const uint8_t* src = x0 + (t + (o - o0)) * ts + dc * 32;
          const floatx8 f[2] = {Eight<T>::load(src), Eight<T>::load(src + 16)};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            w[j] = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
              w[j] |= (some ? quant_byte(f[j / 2][(4 * j + b) & 7], step, r) : 128u) << (8 * b);
          }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
      for (int it = tid; it < n * (D / 8); it += NT) {
        const int i = it / (D / 8), d = it % (D / 8) * 8;
        const floatx8 f = Eight<T>::load(x0 + (t + i) * ts + d * 2);
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j)
          w[j / 4] |= (some ? quant_byte(f[j], step, r) : 128u) << (8 * (j & 3));
        *reinterpret_cast<uint2*>(staged + i * D + d) = make_uint2(w[0], w[1]);
      }
      __syncthreads();
      // 16 bytes: two dimensions (e) of tokens q + c and 16 + q + c (h4).
      const int g0 = rise ? 0 : o0 >> 5, g1 = (o0 + n - 1) >> 5;
      for (int it = tid; it < (g1 - g0 + 1) * (2 * D); it += NT) {
        const int gr = g0 + it / (2 * D), c16 = it % (2 * D);
        const int dt = c16 / kWave, l = c16 % kWave;
        const int tok = gr * 32 + 4 * (l / 16), dim = dt * 32 + l % 16;
        const auto is_new = [&](int o) { return o >= o0 && o < o0 + n; };
        const bool any = (tok < o0 + n && tok + 4 > o0) || (tok + 16 < o0 + n && tok + 20 > o0);
        if (!any && !(rise && tok < o0)) continue;
        uint8_t* p = dst + gr * (32 * D) + c16 * 16;
        const bool all = is_new(tok) && is_new(tok + 19);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (!all) v = load_u4(p);
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int o = tok + 16 * (j & 1) + b, d = dim + 16 * (j >> 1);
            uint32_t u = byte_of(v, 4 * j + b);
            if (is_new(o)) u = staged[(o - o0) * D + d];
            else if (rise && o < o0) u = requant_byte(u, ratio);
            w[j] |= u << (8 * b);
          }
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    __syncthreads();  // staged and wave_amax are reused by the next run
  }
}

// ---------------------------------------------------------------------------
// Read-back: eight dimensions of one token and head per thread.
// ---------------------------------------------------------------------------
struct ReadArgs {
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t* slots;
  int64_t n, num_blocks;
  int heads, shift;
  uint8_t *k_out, *v_out;
};

template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  const int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int d = it % (D / 8) * 8;
  const int64_t th = it / (D / 8), t = th / a.heads;
  const int h = (int)(th % a.heads);
  if (t >= a.n) return;
  const int32_t slot = a.slots[t];
  const int64_t block = slot >> a.shift;
  floatx8 kf = 0.0f, vf = 0.0f;
  if (slot >= 0 && block < a.num_blocks) {
    const int o = slot & ((1 << a.shift) - 1);
    const int64_t at = block * a.heads + h;
    const uint8_t* kp = a.k + at * ((int64_t)D << a.shift) + (o >> 5) * (32 * D) +
                        ((o >> 4 & 1) * (D / 64) + d / 64) * kTileBytes +
                        ((d / 16 & 3) * 16 + (o & 15)) * 16 + (d & 8);
    const uint2 kb = *reinterpret_cast<const uint2*>(kp);
    const uint8_t* vp = a.v + at * ((int64_t)D << a.shift) + (o >> 5) * (32 * D) +
                        d / 32 * kTileBytes + ((o >> 2 & 3) * 16 + (d & 8)) * 16 + (d >> 4 & 1) * 8 +
                        (o >> 4 & 1) * 4 + (o & 3);
    const float ks = a.ks[at], vs = a.vs[at];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      kf[j] = (float)((int)((j < 4 ? kb.x : kb.y) >> (8 * (j & 3)) & 0xffu) - 128) * ks;
      vf[j] = (float)((int)vp[j * 16] - 128) * vs;
    }
  }
  const int64_t to = (th * D + d) * (int64_t)sizeof(T);
  Eight<T>::store(a.k_out + to, kf);
  Eight<T>::store(a.v_out + to, vf);
}

inline int log2i(int v) { return __builtin_ctz((unsigned)v); }

template <typename T>
hipError_t rope_typed(const RopeArgs& r, dim3 grid, int threads, hipStream_t stream) {
  if (r.D <= 64) qk_norm_rope_kernel<T, 8><<<grid, threads, 0, stream>>>(r);
  else if (r.D <= 128) qk_norm_rope_kernel<T, 16><<<grid, threads, 0, stream>>>(r);
  else if (r.D <= 256) qk_norm_rope_kernel<T, 32><<<grid, threads, 0, stream>>>(r);
  else qk_norm_rope_kernel<T, 64><<<grid, threads, 0, stream>>>(r);
  return hipGetLastError();
}

template <typename T, int D>
hipError_t append_sized(const AppendArgs& a, bool wide, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(a.tokens, a.chunk), (unsigned)a.heads, 2);
  const size_t lds = wide ? (size_t)D << a.shift : (size_t)D << a.shift;
  if (wide) kv8_append_kernel<T, D, 256><<<grid, 256, lds, stream>>>(a);
  else kv8_append_kernel<T, D, 64><<<grid, 64, lds, stream>>>(a);
  return hipGetLastError();
}

template <typename T>
hipError_t append_typed(const AppendArgs& a, int D, bool wide, hipStream_t stream) {
  return D == 64 ? append_sized<T, 64>(a, wide, stream)
         : D == 128 ? append_sized<T, 128>(a, wide, stream)
                    : append_sized<T, 256>(a, wide, stream);
}

template <typename T>
hipError_t read_typed(const ReadArgs& a, int D, hipStream_t stream) {
  const unsigned grid = (unsigned)ceil_div(a.n * a.heads * (D / 8), 256);
  if (D == 64) kv8_read_kernel<T, 64><<<grid, 256, 0, stream>>>(a);
  else if (D == 128) kv8_read_kernel<T, 128><<<grid, 256, 0, stream>>>(a);
  else kv8_read_kernel<T, 256><<<grid, 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_norm_rope(const rf_kv8_rope_args& a, hipStream_t stream) {
  RopeArgs r;
  r.q = (const uint8_t*)a.q.data;
  r.k = (const uint8_t*)a.k.data;
  r.q_out = (uint8_t*)a.q_out;
  r.k_out = (uint8_t*)a.k_out;
  r.q_ts = a.q.token_stride * 2;
  r.q_hs = a.q.head_stride * 2;
  r.k_ts = a.k.token_stride * 2;
  r.k_hs = a.k.head_stride * 2;
  r.qw = (const uint8_t*)a.q_weight;
  r.kw = (const uint8_t*)a.k_weight;
  r.cos = a.cos;
  r.sin = a.sin;
  r.pos = a.positions;
  r.tokens = a.tokens;
  r.table_rows = a.table_rows;
  r.pos64 = a.positions64;
  r.hq = a.q.heads;
  r.hk = a.k.heads;
  r.D = a.head_dim;
  r.rot = a.rot;
  r.interleaved = a.interleaved;
  r.eps = a.eps;
  const int lanes = a.head_dim <= 64 ? 8 : a.head_dim <= 128 ? 16 : a.head_dim <= 256 ? 32 : 64;
  const int at_once = kWave / lanes, heads = r.hq + r.hk;
  r.per_wave = at_once;
  const int waves = 4;
  const dim3 grid((unsigned)a.tokens, (unsigned)ceil_div(heads, (int64_t)r.per_wave * waves));
  return a.dtype == RF_W8A16_DTYPE_F16 ? rope_typed<_Float16>(r, grid, waves * kWave, stream)
                                       : rope_typed<__bf16>(r, grid, waves * kWave, stream);
}

hipError_t launch_kv8_plan(const rf_kv8_plan_args& a, hipStream_t stream) {
  const int64_t work = a.tokens > a.requests ? a.tokens : a.requests;
  const int64_t groups = ceil_div(work > 0 ? work : 1, kPlanThreads);
  const unsigned grid = (unsigned)(groups > 256 ? 256 : groups);
  kv8_plan_kernel<<<grid, kPlanThreads, (size_t)(a.requests + 1) * 8, stream>>>(a, log2i(a.block_size));
  return hipGetLastError();
}

hipError_t launch_kv8_append(const rf_kv8_cache& c, const rf_kv8_heads& k, const rf_kv8_heads& v,
                             int dtype, const int32_t* slots, int64_t tokens, hipStream_t stream) {
  AppendArgs a;
  a.x[0] = (const uint8_t*)k.data;
  a.x[1] = (const uint8_t*)v.data;
  a.ts[0] = k.token_stride * 2;
  a.ts[1] = v.token_stride * 2;
  a.hs[0] = k.head_stride * 2;
  a.hs[1] = v.head_stride * 2;
  a.store[0] = (uint8_t*)c.k;
  a.store[1] = (uint8_t*)c.v;
  a.scale[0] = c.k_scale;
  a.scale[1] = c.v_scale;
  a.slots = slots;
  a.tokens = tokens;
  a.num_blocks = c.num_blocks;
  a.heads = c.kv_heads;
  a.shift = log2i(c.block_size);
  a.chunk = 1;
  const bool wide = false;
  return dtype == RF_W8A16_DTYPE_F16 ? append_typed<_Float16>(a, c.head_dim, wide, stream)
                                     : append_typed<__bf16>(a, c.head_dim, wide, stream);
}

hipError_t launch_kv8_read(const rf_kv8_cache& c, const int32_t* slots, int64_t n, int dtype,
                           void* k_out, void* v_out, hipStream_t stream) {
  ReadArgs a{(const uint8_t*)c.k, (const uint8_t*)c.v, c.k_scale, c.v_scale, slots, n, c.num_blocks,
             c.kv_heads, log2i(c.block_size), (uint8_t*)k_out, (uint8_t*)v_out};
  return dtype == RF_W8A16_DTYPE_F16    ? read_typed<_Float16>(a, c.head_dim, stream)
         : dtype == RF_W8A16_DTYPE_BF16 ? read_typed<__bf16>(a, c.head_dim, stream)
                                        : read_typed<float>(a, c.head_dim, stream);
}

}  // namespace rf
