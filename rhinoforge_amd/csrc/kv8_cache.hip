// What surrounds the attention over the int8 paged cache (kv8.h): norms and
// rotation of the heads, block tables and slots, the quantizing append and the
// read-back.  All bound by memory on long batches and by the launch on single
// tokens.
#include "kv8_common.h"

namespace rf {
namespace {

// ---------------------------------------------------------------------------
// Norms and rotation.  LP lanes hold one head; a lane's eight dimensions are
// two runs of four, a0.. and b0.., which with halves as pairs are each other's
// partners, so the rotation needs no other lane and one set of four cosines.
// A wavefront walks query heads or key heads of one token, kHeads at a time,
// with that token's cos and sin and the weight in registers and the next heads'
// loads in flight; heads advance a scalar base, so they cost no address math
// (4001 tokens of 64 + 8 heads: 46 us with per-lane addresses and IEEE square
// root and division, 27.8 so).
// ---------------------------------------------------------------------------
struct RopeArgs {
  const uint8_t *q, *k;
  uint8_t *q_out, *k_out;
  int64_t q_ts, q_hs, k_ts, k_hs;  // bytes
  const uint8_t *qw, *kw;
  const float *cos, *sin;
  const void* pos;
  int64_t table_rows;
  int tokens, pos64, hq, hk, D, rot;
  int turns;           // of kHeads heads each, per wavefront
  int q_parts, parts;  // wavefronts of one token: for q, for both
  float eps;
};

// Sum over the LP lanes of a head, in all of them.
template <int LP>
__device__ __forceinline__ float sum_lanes(float v) {
  const auto add = [&](auto ctrl) {
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl(),
                                                               0xf, 0xf, true));
  };
  add([] { return 0xB1; } );   // lanes 1, 0, 3, 2 of a quad
  add([] { return 0x4E; });    // 2, 3, 0, 1
  add([] { return 0x141; });   // mirrored in eight
  if (LP >= 16) add([] { return 0x140; });  // mirrored in sixteen
  if (LP >= 32) v += __shfl_xor(v, 16);
  if (LP >= 64) v += __shfl_xor(v, 32);
  return v;
}

// kPart: some dimensions are not rotated.  A form of its own: where all are, the
// selects that it takes would cost a wavefront per SIMD (27.8 -> 29.3 us), and here
// fewer loads ahead pay for them (half of 128 rotated, 4001 tokens, 64 + 8 heads:
// 31.5 us with four, 30.0 with two; interleaved 31.7, 30.8 with three).
template <typename T, int LP, bool kInterleaved, bool kPart>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeArgs a) {
  constexpr int kHeads = kWave / LP, kAhead = !kPart ? 4 : kInterleaved ? 3 : 2;
  typedef T tx4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x % kWave, sub = lane % LP;
  const unsigned w = blockIdx.x * (256 / kWave) + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t = (int)(w / (unsigned)a.parts), part = (int)(w - (unsigned)t * a.parts);
  if (t >= a.tokens) return;
  const bool isq = part < a.q_parts;
  const int heads = isq ? a.hq : a.hk, first = (isq ? part : part - a.q_parts) * a.turns * kHeads;
  const int left = heads - first;  // heads from here on
  const bool mine = sub * 8 < a.D, turned = sub < a.rot / 8;
  const int a0 = turned ? 4 * sub : a.rot + 4 * (sub - a.rot / 8);
  const int b0 = a0 + (turned ? a.rot / 2 : (a.D - a.rot) / 2);
  const int64_t hs = isq ? a.q_hs : a.k_hs;
  const uint8_t* src = (isq ? a.q + t * a.q_ts : a.k + t * a.k_ts) + first * hs;
  uint8_t* dst = (isq ? a.q_out : a.k_out) + ((int64_t)t * heads + first) * a.D * 2;
  const int64_t in_a = lane / LP * hs + a0 * 2, in_b = lane / LP * hs + b0 * 2;
  const int out_a = (lane / LP * a.D + a0) * 2, out_b = (lane / LP * a.D + b0) * 2;
  const int turns = min(a.turns, (left + kHeads - 1) / kHeads);

  // The first heads go out before the position's and the table's round trips.
  tx4 xa[kAhead], xb[kAhead];
  const auto load = [&](int u, int turn) {
    if (mine && turn * kHeads + lane / LP < left) {
      const uint8_t* p = src + turn * (kHeads * hs);
      xa[u] = *reinterpret_cast<const tx4*>(p + in_a);
      xb[u] = *reinterpret_cast<const tx4*>(p + in_b);
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    xa[u] = xb[u] = (T)0.0f;
    if (u < turns) load(u, u);
  }

  floatx4 ca = 1.0f, sa = 0.0f, cb = 1.0f, sb = 0.0f;  // (halves as pairs: ca and sa only)
  if (a.rot > 0) {
    const int64_t row = a.pos == nullptr ? t
                        : a.pos64        ? reinterpret_cast<const int64_t*>(a.pos)[t]
                                         : reinterpret_cast<const int32_t*>(a.pos)[t];
    const bool ok = row >= 0 && row < a.table_rows;
    const float* cr = a.cos + (ok ? row : 0) * (a.rot / 2);
    const float* sr = a.sin + (ok ? row : 0) * (a.rot / 2);
    if (turned) {
      if (kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          ca[i] = cr[a0 / 2 + i / 2], cb[i] = cr[b0 / 2 + i / 2];
          sa[i] = sr[a0 / 2 + i / 2], sb[i] = sr[b0 / 2 + i / 2];
        }
      } else {
        ca = *reinterpret_cast<const floatx4*>(cr + a0);
        sa = *reinterpret_cast<const floatx4*>(sr + a0);
      }
    }
    if (!ok) ca = cb = __builtin_nanf("");
  }
  if (!kInterleaved) cb = ca;
  const uint8_t* weight = isq ? a.qw : a.kw;
  floatx4 wa = 1.0f, wb = 1.0f;
  if (mine && weight) {
    wa = __builtin_convertvector(*reinterpret_cast<const tx4*>(weight + a0 * 2), floatx4);
    wb = __builtin_convertvector(*reinterpret_cast<const tx4*>(weight + b0 * 2), floatx4);
  }
  const float over = 1.0f / (float)a.D;

  for (int turn0 = 0; turn0 < turns; turn0 += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int turn = turn0 + u;
      if (turn >= turns) break;
      floatx4 x = __builtin_convertvector(xa[u], floatx4), y = __builtin_convertvector(xb[u], floatx4);
      if (turn + kAhead < turns) load(u, turn + kAhead);
      if (weight) {
        const floatx4 sq = x * x + y * y;
        const float ss = sum_lanes<LP>((sq[0] + sq[1]) + (sq[2] + sq[3]));
        const float r = __builtin_amdgcn_rsqf(ss * over + a.eps);  // (within 2^-23)
        x = x * r * wa;
        y = y * r * wb;
      }
      floatx4 xo, yo;
      if (kInterleaved) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          xo[i] = x[i] * ca[i] - x[i + 1] * sa[i];
          xo[i + 1] = x[i + 1] * ca[i] + x[i] * sa[i];
          yo[i] = y[i] * cb[i] - y[i + 1] * sb[i];
          yo[i + 1] = y[i + 1] * cb[i] + y[i] * sb[i];
        }
      } else {
        xo = x * ca - y * sa;
        yo = y * cb + x * sa;
      }
      if (kPart && !turned) {  // (0 times an infinity or NaN of another dimension is not 0)
        xo = x * ca;
        yo = y * cb;
      }
      if (mine && turn * kHeads + lane / LP < left) {
        uint8_t* out = dst + (int64_t)turn * kHeads * a.D * 2;
        *reinterpret_cast<tx4*>(out + out_a) = __builtin_convertvector(xo, tx4);
        *reinterpret_cast<tx4*>(out + out_b) = __builtin_convertvector(yo, tx4);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Block tables and slots.  Every workgroup adds up the batch's lengths for
// itself (a scan of at most 8192 requests in LDS, cheaper than a second
// launch), then writes its share of the tokens and of the table rows.
// Bound by its round trips and barriers: 64 requests of one token 3.9 us (2.5
// in a replayed graph), 200 prompts of up to 700 tokens 5.4.
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
// among consecutive tokens; for one head of it, k or v: the largest magnitude,
// the new scale, the held values again if the scale rose, the new ones.
// ---------------------------------------------------------------------------
struct AppendArgs {
  const uint8_t* x[2];     // k, v
  int64_t ts[2], hs[2];    // bytes
  uint8_t* store[2];
  float* scale[2];
  const int32_t* slots;
  int64_t tokens, num_blocks;
  int heads, shift;        // log2(block size)
  int chunk;               // long runs: consecutive tokens whose runs a workgroup begins
  int64_t first;           // token that the launch begins at
};

constexpr float kLeastAmax = 0x1p-100f;

// b is i slots after a (slots reach up to 2^31)
__device__ __forceinline__ bool follows(int32_t a, int i, int32_t b) {
  return (uint32_t)b - (uint32_t)a == (uint32_t)i;
}

// x / step, correctly rounded, plus 1.5 * 2^23 + 128: the sum rounds the
// quotient to the nearest integer (ties to even), and its low byte is the
// stored byte.  The quotient comes from a correctly rounded reciprocal and one
// correction, t + r (x - t step) (Markstein 1990); |x / step| < 127.0001.
__device__ __forceinline__ uint32_t quant_bits(float x, float step, float r) {
  const float t = x * r;
  return __builtin_bit_cast(uint32_t, __builtin_fmaf(__builtin_fmaf(-t, step, x), r, t) + 12583040.0f);
}
// The low bytes of four words, in order.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
  return lo | hi;
}
__device__ __forceinline__ uint32_t requant_byte(uint32_t u, float ratio) {
  return (uint32_t)((int)rintf((float)((int)u - 128) * ratio) + 128) & 0xffu;
}
__device__ __forceinline__ uint32_t byte_of(uint4 v, int i) {
  const uint32_t w = i < 4 ? v.x : i < 8 ? v.y : i < 12 ? v.z : v.w;
  return (w >> (8 * (i & 3))) & 0xffu;
}

// What a block's scale becomes.
struct Step {
  float step, ratio;  // held values change by `ratio` where `rise`
  float r;            // 1 / step, 0 where everything is stored as 0
  bool rise, some;
  __device__ __forceinline__ Step(float step, float r) : step(step), ratio(1.0f), r(r), rise(false), some(r != 0.0f) {}
  __device__ __forceinline__ Step(float amax, bool held, float scale) {
    const float before = held ? scale : 0.0f;
    const float fresh = amax < kLeastAmax ? 0.0f : amax * (1.0f / 127.0f);
    // the larger; either one not finite makes the block not finite
    step = before >= fresh || before != before ? before : fresh;
    rise = held && !(step == before) && before == before;
    ratio = rise ? before / step : 1.0f;
    some = step > 0.0f && step < __builtin_inff();
    r = some ? 1.0f / step : 0.0f;
  }
  __device__ __forceinline__ uint2 bytes(floatx8 f) const {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = quant_bits(f[j], step, r);
    return some ? make_uint2(low_bytes(w[0], w[1], w[2], w[3]), low_bytes(w[4], w[5], w[6], w[7]))
                : make_uint2(0x80808080u, 0x80808080u);
  }
};

// Bits of the largest |x| of eight values (a NaN is above infinity).
__device__ __forceinline__ uint32_t top_bits(uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, max(w[j] & 0x7fffu, (w[j] >> 16) & 0x7fffu));
  return top;
}

// Byte offsets within a head's block.
template <int D>
__device__ __forceinline__ int k_at(int o, int d) {  // 16 bytes for d % 16 == 0
  return (o >> 5) * (32 * D) + ((o >> 4 & 1) * (D / 64) + (d >> 6)) * kTileBytes +
         ((d >> 4 & 3) * 16 + (o & 15)) * 16 + (d & 15);
}
template <int D>
__device__ __forceinline__ int v_at(int o, int d) {
  return (o >> 5) * (32 * D) + (d >> 5) * kTileBytes + ((o >> 2 & 3) * 16 + (d & 15)) * 16 +
         (d >> 4 & 1) * 8 + (o >> 4 & 1) * 4 + (o & 3);
}

// Held bytes of tokens [0, o0) rounded to a larger step, by a workgroup of 256;
// v chunks hold tokens past o0 too, whose bytes stay.  Four chunks a thread are
// loaded together: what this costs is its round trips.
template <int D>
__device__ __forceinline__ void requantize(uint8_t* dst, int side, int o0, float ratio, int tid) {
  const int end = ((o0 + 31) >> 5) * 2 * D;
  for (int it0 = tid; it0 < end; it0 += 4 * 256) {
    uint4 v[4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (it0 + n * 256 < end) v[n] = load_u4(dst + (it0 + n * 256) * 16);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int it = it0 + n * 256;
      // 16 bytes of one token (k), or of tokens tok + c and tok + 16 + c (v)
      const int gr = it / (2 * D), l = it % kWave;
      const int tok = gr * 32 + (side ? 4 * (l / 16) : (it % (2 * D) / kWave / (D / 64)) * 16 + l % 16);
      if (it >= end || tok >= o0) continue;
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t u = byte_of(v[n], 4 * j + b);
          const bool held = !side || tok + 16 * (j & 1) + b < o0;
          w[j] |= (held ? requant_byte(u, ratio) : u) << (8 * b);
        }
      }
      *reinterpret_cast<uint4*>(dst + it * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// A workgroup begins the runs of `chunk` consecutive tokens, for one head of k
// or v.  Runs of up to kShort tokens (single tokens, drafted ones) are done all
// at once, a thread for every eight values: the time is the chain of round
// trips slots, values and scales, stores, whatever their number.  Longer ones
// come one after the other: the values are read once, stay in registers until
// the scale is known and go out through LDS in 16-byte chunks.  Bound by those
// round trips for few tokens (48 single ones: 5.3 us, 256: 5.6), by the bytes for
// many (6874 tokens in prompts, 8 heads of 128: 14.8 us, 2.9 TB/s).  A wavefront
// for each run, which single tokens alone would like (3.7 us for 48, 4.7 for 256),
// needs 127 us for a prompt of 1024 tokens, where this takes 6.0.  256 runs of 8
// tokens take 13.0 us, of 9, one after the other, 21.0.
constexpr int kShort = 8;

template <typename T, int D, int BS>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs a) {
  constexpr int kRow = D / 8, kItems = BS * kRow / 256, kPitch = D + 16;
  constexpr int kAtOnce = 64 * kRow / 256;
  __shared__ int32_t near_slots[256];
  __shared__ uint32_t wave_top[4], token_top[64];
  __shared__ float steps[64], inverse[64], ratios[64];
  __shared__ uint64_t rising;
  extern __shared__ __align__(16) uint8_t staged[];  // [tokens of the run][kPitch]
  const int tid = threadIdx.x, lane = tid % kWave;
  const unsigned both = 2u * (unsigned)a.heads, part = blockIdx.x / both, which = blockIdx.x - part * both;
  const int side = which >= (unsigned)a.heads, h = (int)which - (side ? a.heads : 0);
  constexpr int bs = BS;
  const int64_t t0 = a.first + (int64_t)part * a.chunk;
  {  // token t0 - 1 + tid (chunk + 128 < 256)
    const int64_t at = t0 - 1 + tid;
    near_slots[tid] = at >= 0 && at < a.tokens ? a.slots[at] : -1;
  }
  __syncthreads();
  const int64_t ts = a.ts[side];
  uint8_t* const store = a.store[side];
  // tokens of the chunk that begin a run, those of runs of few tokens, and those
  uint64_t begins, brief, valid;
  int length;  // of the run that this lane's token begins, within the chunk
  {
    const int32_t slot = near_slots[min(lane + 1, 255)], prev = near_slots[min(lane, 255)];
    const int64_t block = slot >> a.shift;
    const bool ok = lane <= a.chunk && slot >= 0 && block < a.num_blocks;
    const bool first = (slot & (bs - 1)) == 0 || t0 + lane == 0 || !follows(prev, 1, slot);
    valid = __ballot(ok && lane < a.chunk);
    begins = __ballot(ok && lane < a.chunk && first);
    // does the last run go on after the chunk?  (chunk == 64: its slot is past the lanes)
    const int32_t last = near_slots[a.chunk], past = near_slots[a.chunk + 1];
    const bool over = (past & (bs - 1)) != 0 && follows(last, 1, past) && past >= 0;
    const uint64_t on = lane == 63 ? 0 : (valid & ~begins) >> (lane + 1);
    length = 1 + (int)__builtin_ctzll(~on);
    brief = __ballot((begins >> lane & 1) && length <= kShort && !(over && lane + length == a.chunk));
  }
  if (brief != 0) {
    // which run token i belongs to: 64 where it is none of these
    const auto run_of = [&](int i) {
      const uint64_t upto = begins & (~0ull >> (63 - i));
      if (!(valid >> i & 1) || upto == 0) return 64;
      const int c = 63 - (int)__builtin_clzll(upto);
      return brief >> c & 1 ? c : 64;
    };
    const uint8_t* x0 = a.x[side] + h * a.hs[side] + t0 * ts;
    uint4 raw[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int it = k * 256 + tid, i = it / kRow;
      raw[k] = make_uint4(0, 0, 0, 0);
      if (i < a.chunk && run_of(i) < 64) raw[k] = load_u4(x0 + i * ts + it % kRow * 16);
    }
    const bool mine = tid < kWave && (brief >> tid & 1);
    const int32_t slot = near_slots[min(tid + 1, 255)];
    const int64_t at = (int64_t)(slot >> a.shift) * a.heads + h;
    const int o0 = slot & (bs - 1);
    float held = 0.0f;
    if (mine && o0 > 0) held = a.scale[side][at];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int it = k * 256 + tid, i = it / kRow;
      uint32_t top = top_bits(raw[k]);
#pragma unroll
      for (int m = 1; m < kRow; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
      if (i < a.chunk && it % kRow == 0) token_top[i] = top;
    }
    __syncthreads();
    if (tid < kWave) {
      bool rise = false;
      if (mine) {
        uint32_t top = 0;
        for (int i = 0; i < length; ++i) top = max(top, token_top[tid + i]);
        const Step s((float)__builtin_bit_cast(T, (uint16_t)top), o0 > 0, held);
        a.scale[side][at] = s.step;
        steps[tid] = s.step;
        inverse[tid] = s.r;
        ratios[tid] = s.ratio;
        rise = s.rise;
      }
      const uint64_t all = __ballot(rise);
      if (tid == 0) rising = all;
    }
    __syncthreads();
    if (rising != 0) {
      for (uint64_t r = rising; r != 0; r &= r - 1) {
        const int c = (int)__builtin_ctzll(r);
        const int32_t slot = near_slots[c + 1];
        requantize<D>(store + ((int64_t)(slot >> a.shift) * a.heads + h) * ((int64_t)D << a.shift), side,
                      slot & (bs - 1), ratios[c], tid);
      }
      __syncthreads();  // the held bytes are written before the new ones among them
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int it = k * 256 + tid, i = it / kRow, d = it % kRow * 8;
      const int c = i < a.chunk ? run_of(i) : 64;
      if (c == 64) continue;
      const int32_t slot = near_slots[i + 1];
      uint8_t* dst = store + ((int64_t)(slot >> a.shift) * a.heads + h) * ((int64_t)D << a.shift);
      const uint2 q = Step(steps[c], inverse[c]).bytes(Eight<T>::load(&raw[k]));
      if (side == 0) {
        *reinterpret_cast<uint2*>(dst + k_at<D>(slot & (bs - 1), d)) = q;
      } else {
        uint8_t* p = dst + v_at<D>(slot & (bs - 1), d);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j * 16] = (uint8_t)((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
      }
    }
    begins &= ~brief;
  }
  for (; begins != 0; begins &= begins - 1) {
    const int c = (int)__builtin_ctzll(begins);
    const int32_t slot = __builtin_amdgcn_readfirstlane(near_slots[c + 1]);
    const int64_t block = slot >> a.shift;
    const int o0 = slot & (bs - 1);
    int n = 0;
    for (bool more = true; more && n < bs - o0;) {  // (slots past the batch are -1 there)
      const int i = n + lane;
      const uint64_t b = __ballot(i < bs - o0 && follows(slot, i, near_slots[min(c + 1 + i, 255)]));
      const int len = ~b == 0 ? kWave : (int)__builtin_ctzll(~b);
      n += len;
      more = len == kWave;
    }
    const uint8_t* x0 = a.x[side] + h * a.hs[side] + (t0 + c) * ts;
    float* scale = a.scale[side] + block * a.heads + h;
    const float held_scale = o0 > 0 ? *scale : 0.0f;
    uint4 raw[kItems];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int it = k * 256 + tid;
      if (it < n * kRow) raw[k] = load_u4(x0 + (it / kRow) * ts + it % kRow * 16);
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      if (k * 256 + tid < n * kRow) top = max(top, top_bits(raw[k]));
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, m));
    if (lane == 0) wave_top[tid / kWave] = top;
    __syncthreads();  // (and the scale has been read)
    top = max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3]));
    const Step s((float)__builtin_bit_cast(T, (uint16_t)top), o0 > 0, held_scale);
    if (tid == 0) *scale = s.step;
    uint8_t* dst = a.store[side] + (block * a.heads + h) * ((int64_t)D << a.shift);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int it = k * 256 + tid;
      if (it < n * kRow)
        *reinterpret_cast<uint2*>(staged + it / kRow * kPitch + it % kRow * 8) =
            s.bytes(Eight<T>::load(&raw[k]));
    }
    if (s.rise) requantize<D>(dst, side, o0, s.ratio, tid);
    __syncthreads();  // staged; the held bytes are written
    if (side == 0) {
      // chunks in memory order: 16 dimensions of one token each
      const int g0 = o0 >> 4, g1 = (o0 + n - 1) >> 4;  // 16-token tiles
      for (int it = tid; it < (g1 - g0 + 1) * D; it += 256) {
        const int o = (g0 + it / D) * 16 + it % 16, dd = it % D / 16 * 16;
        if (o < o0 || o >= o0 + n) continue;
        *reinterpret_cast<uint4*>(dst + k_at<D>(o, dd)) =
            *reinterpret_cast<const uint4*>(staged + (o - o0) * kPitch + dd);
      }
    } else {
      // Four dimensions of eight tokens a thread: bytes [token][dimension] of
      // LDS become 8 bytes [token] of each dimension's chunk.
      const int g0 = o0 >> 5, g1 = (o0 + n - 1) >> 5;
      for (int it = tid; it < (g1 - g0 + 1) * D; it += 256) {
        const int gr = g0 + it / D, dq = it % 4, e = it / 4 % 2, g = it / 8 % 4, dt = it % D / 32;
        const int tok = gr * 32 + 4 * g, dim = dt * 32 + 16 * e + 4 * dq;
        const auto fresh = [&](int o) { return o >= o0 && o < o0 + n; };
        const bool any = (tok < o0 + n && tok + 4 > o0) || (tok + 16 < o0 + n && tok + 20 > o0);
        if (!any) continue;
        uint8_t* p = dst + gr * (32 * D) + dt * kTileBytes + (g * 16 + 4 * dq) * 16 + 8 * e;
        uint32_t out[4][2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t w[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int o = min(max(tok + 16 * half + b - o0, 0), n - 1);
            w[b] = *reinterpret_cast<const uint32_t*>(staged + o * kPitch + dim);
          }
          const uint32_t l01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // dims 0, 1 of tokens 0, 1
          const uint32_t h01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);  // dims 2, 3
          const uint32_t l23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
          const uint32_t h23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
          out[0][half] = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
          out[1][half] = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
          out[2][half] = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
          out[3][half] = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
        }
        if (fresh(tok) && fresh(tok + 19)) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint2*>(p + j * 16) = make_uint2(out[j][0], out[j][1]);
        } else {  // the run begins or ends among these tokens
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int b = 0; b < 8; ++b)
              if (fresh(tok + 16 * (b / 4) + b % 4)) p[j * 16 + b] = (uint8_t)(out[j][b / 4] >> (8 * (b % 4)));
        }
      }
    }
    __syncthreads();  // staged and wave_top are reused by the next run
  }
}

// ---------------------------------------------------------------------------
// Read-back: a workgroup takes 32 consecutive entries of `slots`, one head.
// Where they are one 32-token group of a block its bytes are read in memory
// order and turned in LDS into rows of tokens; any other 32 are gathered, eight
// dimensions of one token per thread.  Bound by the values it writes: 6874
// tokens, 8 heads of 128: 12.6 us, 3.4 TB/s (gathering all of them: 19).
// ---------------------------------------------------------------------------
struct ReadArgs {
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t* slots;
  int64_t n, num_blocks;
  int heads, shift;
  uint8_t *k_out, *v_out;
};

// Eight stored bytes.
__device__ __forceinline__ floatx8 values_of(uint2 u, float scale) {
  floatx8 f;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    f[j] = ((float)((j < 4 ? u.x : u.y) >> (8 * (j & 3)) & 0xffu) - 128.0f) * scale;
  return f;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_read_kernel(ReadArgs a) {
  constexpr int kRow = D / 8, kPitch = D + 16;
  __shared__ __align__(16) uint8_t rows[2][32 * kPitch];  // k, v: bytes [token][dimension]
  const int tid = threadIdx.x, lane = tid % kWave;
  const unsigned part = blockIdx.x / (unsigned)a.heads;
  const int h = (int)(blockIdx.x - part * a.heads);
  const int64_t t0 = (int64_t)part * 32;
  const int32_t mine = lane < 32 && t0 + lane < a.n ? a.slots[t0 + lane] : -1;
  const int32_t first = __builtin_amdgcn_readfirstlane(mine);
  const bool whole = first >= 0 && (first & 31) == 0 && (first >> a.shift) < a.num_blocks &&
                     __ballot(lane >= 32 || (mine >= 0 && follows(first, lane, mine))) == ~0ull;
  uint8_t* const outs[2] = {a.k_out, a.v_out};
  if (whole) {
    const int64_t at = (int64_t)(first >> a.shift) * a.heads + h;
    const int64_t base = at * ((int64_t)D << a.shift) + (first & ((1 << a.shift) - 1)) * D;
    const float ks = a.ks[at], vs = a.vs[at];
    for (int it = tid; it < 2 * D; it += 256) {  // 16 dimensions of one token
      const int tile = it / kWave, l = it % kWave;
      *reinterpret_cast<uint4*>(rows[0] + (tile / (D / 64) * 16 + l % 16) * kPitch + tile % (D / 64) * 64 + l / 16 * 16) =
          load_u4(a.k + base + it * 16);
    }
    for (int it = tid; it < D; it += 256) {  // four dimensions of eight tokens
      const int dq = it % 4, e = it / 4 % 2, g = it / 8 % 4, dt = it / 32;
      const uint8_t* p = a.v + base + dt * kTileBytes + (g * 16 + 4 * dq) * 16 + 8 * e;
      uint2 in[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) in[j] = *reinterpret_cast<const uint2*>(p + j * 16);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = half ? in[j].y : in[j].x;
        const uint32_t l01 = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u);  // tokens 0, 1 of dims 0, 1
        const uint32_t h01 = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);  // tokens 2, 3
        const uint32_t l23 = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u);
        const uint32_t h23 = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
        uint8_t* q = rows[1] + (4 * g + 16 * half) * kPitch + dt * 32 + 16 * e + 4 * dq;
        *reinterpret_cast<uint32_t*>(q) = __builtin_amdgcn_perm(l23, l01, 0x05040100u);
        *reinterpret_cast<uint32_t*>(q + kPitch) = __builtin_amdgcn_perm(l23, l01, 0x07060302u);
        *reinterpret_cast<uint32_t*>(q + 2 * kPitch) = __builtin_amdgcn_perm(h23, h01, 0x05040100u);
        *reinterpret_cast<uint32_t*>(q + 3 * kPitch) = __builtin_amdgcn_perm(h23, h01, 0x07060302u);
      }
    }
    __syncthreads();
#pragma unroll
    for (int it = tid; it < 32 * kRow; it += 256) {
      const int i = it / kRow, d = it % kRow * 8;
      const int64_t to = (((t0 + i) * a.heads + h) * D + d) * (int64_t)sizeof(T);
#pragma unroll
      for (int side = 0; side < 2; ++side)
        Eight<T>::store(outs[side] + to, values_of(*reinterpret_cast<const uint2*>(rows[side] + i * kPitch + d),
                                                   side ? vs : ks));
    }
    return;
  }
  for (int it = tid; it < 32 * kRow; it += 256) {
    const int i = it / kRow, d = it % kRow * 8;
    if (t0 + i >= a.n) return;
    const int32_t slot = a.slots[t0 + i];
    const int64_t block = slot >> a.shift;
    floatx8 kf = 0.0f, vf = 0.0f;
    if (slot >= 0 && block < a.num_blocks) {
      const int o = slot & ((1 << a.shift) - 1);
      const int64_t at = block * a.heads + h, base = at * ((int64_t)D << a.shift);
      const uint8_t* vp = a.v + base + v_at<D>(o, d);
      uint32_t w[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = vp[j * 16];
      kf = values_of(*reinterpret_cast<const uint2*>(a.k + base + k_at<D>(o, d)), a.ks[at]);
      vf = values_of(make_uint2(low_bytes(w[0], w[1], w[2], w[3]), low_bytes(w[4], w[5], w[6], w[7])), a.vs[at]);
    }
    const int64_t to = (((t0 + i) * a.heads + h) * D + d) * (int64_t)sizeof(T);
    Eight<T>::store(a.k_out + to, kf);
    Eight<T>::store(a.v_out + to, vf);
  }
}

inline int log2i(int v) { return __builtin_ctz((unsigned)v); }

template <typename T, int LP>
hipError_t rope_sized(const RopeArgs& r, bool interleaved, unsigned grid, hipStream_t stream) {
  const bool part = r.rot < r.D;
  if (interleaved && part) qk_norm_rope_kernel<T, LP, true, true><<<grid, 256, 0, stream>>>(r);
  else if (interleaved) qk_norm_rope_kernel<T, LP, true, false><<<grid, 256, 0, stream>>>(r);
  else if (part) qk_norm_rope_kernel<T, LP, false, true><<<grid, 256, 0, stream>>>(r);
  else qk_norm_rope_kernel<T, LP, false, false><<<grid, 256, 0, stream>>>(r);
  return hipGetLastError();
}

template <typename T>
hipError_t rope_typed(const RopeArgs& r, bool interleaved, unsigned grid, hipStream_t stream) {
  return r.D <= 64    ? rope_sized<T, 8>(r, interleaved, grid, stream)
         : r.D <= 128 ? rope_sized<T, 16>(r, interleaved, grid, stream)
         : r.D <= 256 ? rope_sized<T, 32>(r, interleaved, grid, stream)
                      : rope_sized<T, 64>(r, interleaved, grid, stream);
}

template <typename T, int D>
hipError_t append_sized(AppendArgs a, hipStream_t stream) {
  const size_t lds = (size_t)(D + 16) << a.shift;
  const int64_t parts = ceil_div(a.tokens, a.chunk), most = kMaxThreads / 256 / (2 * a.heads);
  for (int64_t i = 0; i < parts; i += most) {
    a.first = i * a.chunk;
    const unsigned grid = (unsigned)((parts - i < most ? parts - i : most) * 2 * a.heads);
    if (a.shift == 5) kv8_append_kernel<T, D, 32><<<grid, 256, lds, stream>>>(a);
    else if (a.shift == 6) kv8_append_kernel<T, D, 64><<<grid, 256, lds, stream>>>(a);
    else kv8_append_kernel<T, D, 128><<<grid, 256, lds, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t append_typed(const AppendArgs& a, int D, hipStream_t stream) {
  return D == 64 ? append_sized<T, 64>(a, stream)
         : D == 128 ? append_sized<T, 128>(a, stream)
                    : append_sized<T, 256>(a, stream);
}

template <typename T>
hipError_t read_typed(ReadArgs a, int D, hipStream_t stream) {
  const int64_t most = kMaxThreads / 256 / a.heads * 32;  // entries of a launch
  for (int64_t left = a.n; left > 0; left -= most) {
    a.n = left < most ? left : most;
    const unsigned grid = (unsigned)(ceil_div(a.n, 32) * a.heads);
    if (D == 64) kv8_read_kernel<T, 64><<<grid, 256, 0, stream>>>(a);
    else if (D == 128) kv8_read_kernel<T, 128><<<grid, 256, 0, stream>>>(a);
    else kv8_read_kernel<T, 256><<<grid, 256, 0, stream>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t bytes = a.n * a.heads * D * (int64_t)sizeof(T);
    a.slots += a.n;
    a.k_out += bytes;
    a.v_out += bytes;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_qk_norm_rope(const rf_kv8_rope_args& a, hipStream_t stream) {
  RopeArgs r;
  r.q_ts = a.q.token_stride * 2;
  r.q_hs = a.q.head_stride * 2;
  r.k_ts = a.k.token_stride * 2;
  r.k_hs = a.k.head_stride * 2;
  r.qw = (const uint8_t*)a.q_weight;
  r.kw = (const uint8_t*)a.k_weight;
  r.cos = a.cos;
  r.sin = a.sin;
  r.pos = a.positions;
  r.table_rows = a.table_rows;
  r.pos64 = a.positions64;
  r.hq = a.q.heads;
  r.hk = a.k.heads;
  r.D = a.head_dim;
  r.rot = a.rot;
  r.eps = a.eps;
  const int lanes = r.D <= 64 ? 8 : r.D <= 128 ? 16 : r.D <= 256 ? 32 : 64;
  // Few tokens: a wavefront per kHeads heads.  Many: as many heads per wavefront
  // as leave about 16 wavefronts for each CU.
  const int64_t at_once = kWave / lanes, q_turns = ceil_div(r.hq, at_once), k_turns = ceil_div(r.hk, at_once);
  int64_t each = a.tokens * (q_turns + k_turns) / 4096;
  each = each < 1 ? 1 : each > q_turns ? q_turns : each;
  r.turns = (int)each;
  r.q_parts = (int)ceil_div(q_turns, each);
  r.parts = r.q_parts + (int)ceil_div(k_turns, each);
  // (a wavefront counts the wavefronts before it in 32 bits, fewer than threads)
  const int64_t most = kMaxThreads / 256 * (256 / kWave) / r.parts;  // tokens of a launch
  for (int64_t t = 0; t < a.tokens; t += most) {
    r.tokens = (int)(a.tokens - t < most ? a.tokens - t : most);
    r.q = (const uint8_t*)a.q.data + t * r.q_ts;
    r.k = (const uint8_t*)a.k.data + t * r.k_ts;
    r.q_out = (uint8_t*)a.q_out + t * r.hq * r.D * 2;
    r.k_out = (uint8_t*)a.k_out + t * r.hk * r.D * 2;
    if (a.positions) {
      r.pos = (const uint8_t*)a.positions + t * (a.positions64 ? 8 : 4);
    } else if (r.rot > 0) {  // token t has row t
      r.cos = a.cos + t * (r.rot / 2);
      r.sin = a.sin + t * (r.rot / 2);
      r.table_rows = a.table_rows - t;
    }
    const unsigned grid = (unsigned)ceil_div((int64_t)r.tokens * r.parts, 256 / kWave);
    const hipError_t e = a.dtype == RF_W8A16_DTYPE_F16 ? rope_typed<_Float16>(r, a.interleaved, grid, stream)
                                                       : rope_typed<__bf16>(r, a.interleaved, grid, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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
  AppendArgs a{};
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
  // Small chunks while they leave CUs idle, large ones after (8 heads of 128, 256
  // single tokens: 5.3 us in chunks of 16, 8.1 of 64; prompts of 8192: 22.0, 13.2).
  a.chunk = tokens * c.kv_heads <= 8192 ? 16 : 64;
  return dtype == RF_W8A16_DTYPE_F16 ? append_typed<_Float16>(a, c.head_dim, stream)
                                     : append_typed<__bf16>(a, c.head_dim, stream);
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
