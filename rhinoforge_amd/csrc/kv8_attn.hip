// Attention over the int8 paged cache (kv8.h), gfx950.
//
// For query row q (one query, one head) over its seen tokens j:
//   x_j = (q . k_j) ks scale log2(e),  p_j = 2^(x_j - m),  o = vs sum p_j v_j / sum p_j
// with integer k_j, v_j and the scales ks, vs of the token's block.  One pass
// over the tokens with a running m: p only has to stay in fp16's range, so m
// follows the largest x when that is 8 or more above it, not at every step;
// results do not depend on how m is chosen beyond rounding.
//
// Both products run on the matrix cores with the cache as the A operand and the
// queries as columns: S^T = K Q^T leaves each lane with scores of one query row
// (its column), and after exp2 those are the B operand of O^T = V^T P^T as they
// stand (the v tiles hold tokens in that order).  int8 -> fp16 is exact.
//   * Queries: fp16 as they are.  bf16 times a power of two per row, which
//     brings the row's largest magnitude to [2^14, 2^15): exact in fp16 down to
//     2^-38 of it; the power goes into that row's score factor.
//   * p is rounded to fp16 (11 bits, round to nearest): 2^-12 relative, as much
//     as the output's own rounding in fp16.  2^7 p is what is rounded, so that
//     small weights stay normal.
//   * vs goes into p as vs / max(vs so far): 2^log2 of it joins the exponent.
//     The sum over p divides it out again.  m, the sums and o stay in fp32.
#include "kv8_common.h"

namespace rf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRaise = 8.0f;  // m follows x from here on: 2^(7 + 8) < 65504
constexpr float kShift = 7.0f;

struct AttnArgs {
  const uint8_t* q;
  int64_t q_ts, q_hs;  // bytes
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int32_t *cu, *lens, *table;
  uint8_t* out;
  float* lse;
  float* part;         // [tokens * heads][splits][D] fp32, unnormalized
  floatx4* stat;       // [tokens * heads][splits] (m, l): see Stat
  int64_t tokens, table_stride, num_blocks;
  int requests, width, hq, hk, group, shift;
  int per_request;     // cu == nullptr: queries of a request
  int splits, tiles;
  int causal;
  int64_t window;      // 0: none
  float scale_log2e;
};

// Where a workgroup works: request, its queries, this tile's first row.
struct Tile {
  int64_t first_token;  // of the request
  int64_t queries;
  int64_t row0;         // first row (query * group + head of the group) of the tile
  int64_t kv_len;
  const int32_t* table;
  bool pad;             // the tokens past the batch: nothing is seen
};

__device__ __forceinline__ int64_t cu_at(const AttnArgs& a, int b) {
  if (b <= 0) return 0;
  if (b > a.requests) return a.tokens;
  const int64_t c = a.cu[b];
  return c < 0 ? 0 : c > a.tokens ? a.tokens : c;
}

// Tile x of the launch: request b's tiles begin at floor(cu[b] group / R) + b,
// which leaves room for all of them.  Every lane looks at one boundary at a
// time: two rounds for up to 4096 requests.
template <int R>
__device__ bool find_tile(const AttnArgs& a, int64_t x, Tile* t) {
  int b;
  if (a.cu == nullptr) {
    const int64_t rows = (int64_t)a.per_request * a.group, per = (rows + R - 1) / R;
    b = (int)(x / per);
    if (b >= a.requests) return false;
    t->first_token = (int64_t)b * a.per_request;
    t->queries = a.per_request;
    t->row0 = (x - (int64_t)b * per) * R;
  } else {
    const int lane = threadIdx.x % kWave;
    const int last = a.requests;  // the tokens past the batch
    int lo = 0, n = last + 1;     // the answer is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + kWave - 1) / kWave;
      const int at = lo + lane * step;
      const bool below = at < lo + n && cu_at(a, at) * a.group / R + at <= x;
      const int hits = __popcll(__ballot(below));
      const int base = lo + (hits > 0 ? hits - 1 : 0) * step;
      n = min(step, lo + n - base);
      lo = base;
    }
    b = __builtin_amdgcn_readfirstlane(lo);
    t->first_token = cu_at(a, b);
    const int64_t next = cu_at(a, b + 1);
    t->queries = next > t->first_token ? next - t->first_token : 0;
    t->row0 = (x - (t->first_token * a.group / R + b)) * R;
  }
  if (t->row0 < 0 || t->row0 >= t->queries * a.group) return false;
  t->pad = b >= a.requests;
  const int64_t most = (int64_t)a.width << a.shift;
  const int64_t len = t->pad ? 0 : a.lens[b];
  t->kv_len = len < 0 ? 0 : len > most ? most : len;
  t->table = a.table + (t->pad ? 0 : (int64_t)b * a.table_stride);
  return true;
}

// Tokens [lo, hi) that row `row` of a request sees.
__device__ __forceinline__ void seen(const AttnArgs& a, const Tile& t, int64_t row, int64_t* lo,
                                     int64_t* hi) {
  *lo = 0;
  *hi = t.kv_len;
  if (a.causal) {
    const int64_t pos = t.kv_len - t.queries + row / a.group;
    *hi = pos < 0 ? 0 : pos + 1 < t.kv_len ? pos + 1 : t.kv_len;
    if (a.window > 0 && pos - a.window + 1 > 0) *lo = pos - a.window + 1;
  }
}

// One 32-token group of a head: where its bytes are and its scales.  A block id
// outside the cache: block 0 with scales of NaN.
struct Group {
  int64_t at;  // block * hk + h
  int sub;     // group within the block
  bool ok;
};
__device__ __forceinline__ Group group_of(const AttnArgs& a, const Tile& t, int h, int g) {
  Group r;
  const int per = a.shift - 5;
  const int64_t id = t.table[g >> per];
  r.ok = id >= 0 && id < a.num_blocks;
  r.at = (r.ok ? id : 0) * a.hk + h;
  r.sub = g & ((1 << per) - 1);
  return r;
}

// Eight query values as fp16 times 2^-e.
template <typename T>
__device__ __forceinline__ float load_amax(uint4 v, float m) {
  const floatx8 f = Eight<T>::load(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(f[i]));
  return m;
}

// exponent e with |x| 2^-e in [2^14, 2^15) for the largest |x| (0: for 0, inf, NaN)
__device__ __forceinline__ int row_exponent(float amax) {
  const int be = (int)(__builtin_bit_cast(uint32_t, amax) >> 23 & 0xff);
  return be == 0 || be == 255 ? 0 : be - 127 - 14;
}
__device__ __forceinline__ float pow2(int e) {  // |e| <= 126
  return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23);
}

// Running softmax of one query row, as the lanes of its column hold it: m and
// svm agree over them, l is each lane's own share of the sum.
struct Running {
  float m;  // log2 units; -inf: nothing seen
  float l;
};

__device__ __forceinline__ float safe(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ bool larger(float vs, float top) {
  return vs > top && vs < __builtin_inff();
}

// log2(vs / top) for the exponent.  A block of zeros counts as if its scale
// were the largest; one 2^60 below it as 2^-60 (what it adds is far below one
// rounding of the result).  A scale that is not finite gives NaN.
__device__ __forceinline__ float ratio_log2(float vs, float top) {
  if (!(vs < __builtin_inff())) return __builtin_nanf("");
  if (vs == 0.0f || vs == top) return 0.0f;
  const float r = vs / top;
  return r < 0x1p-60f ? -60.0f : __builtin_amdgcn_logf(r);
}

// ---------------------------------------------------------------------------
// Few rows (single tokens, a few drafted ones): RT tiles of 16 rows, held by
// all four wavefronts; the wavefronts take 32-token groups in turn and read the
// cache straight into MFMA operands (no LDS), two groups ahead of the products.
// Bound by the cache's bytes.  At the end the wavefronts' sums meet in LDS.
// ---------------------------------------------------------------------------
constexpr int kWaves = 4;

template <int D>
struct Bytes {
  uint4 k[D / 32], v[D / 32];
  float ks, vs;
};

template <int D>
__device__ __forceinline__ void fetch(const AttnArgs& a, const Group& g, int lane, Bytes<D>& b) {
  const int64_t base = (g.at << a.shift) * D + g.sub * (32 * D);
  const uint8_t* kp = a.k + base;
  const uint8_t* vp = a.v + base;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) b.k[i] = load_u4_stream(kp + i * kTileBytes + lane * 16);
#pragma unroll
  for (int i = 0; i < D / 32; ++i) b.v[i] = load_u4_stream(vp + i * kTileBytes + lane * 16);
  const float nan = __builtin_nanf("");
  b.ks = g.ok ? a.ks[g.at] : nan;
  b.vs = g.ok ? a.vs[g.at] : nan;
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kWaves* kWave) void kv8_decode_kernel(AttnArgs a) {
  constexpr int R = 16 * RT;
  __shared__ __align__(16) float red[kWaves][16][D + 4];
  __shared__ float red_m[kWaves][R], red_l[kWaves][R];
  __shared__ float red_v[kWaves];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 16, lg = lane / 16;
  int64_t id = blockIdx.x;
  const int h = (int)(id % a.hk);
  id /= a.hk;
  const int split = (int)(id % a.splits);
  Tile t;
  if (!find_tile<R>(a, id / a.splits, &t)) return;
  const int64_t rows = t.queries * a.group;

  // ---- queries, as B operands: column = row, 16 dimensions 64 kb + 16 lg + ..
  half8 q[RT][D / 32];
  float factor[RT];
  int64_t lo[RT], hi[RT];
  int64_t lo_min = INT64_MAX, lo_max = 0, hi_min = INT64_MAX, hi_max = 0;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    int64_t row = t.row0 + 16 * r + col;
    if (row >= rows) row = rows - 1;
    const int64_t qi = row / a.group;
    const uint8_t* p = a.q + (t.first_token + qi) * a.q_ts +
                       (h * a.group + (row - qi * a.group)) * a.q_hs + lg * 32;
    uint4 raw[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) raw[i] = load_u4(p + (i / 2) * 128 + (i % 2) * 16);
    factor[r] = a.scale_log2e;
    if constexpr (sizeof(T) == 2 && !__is_same(T, _Float16)) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) m = load_amax<T>(raw[i], m);
      m = fmaxf(m, __shfl_xor(m, 16));
      m = fmaxf(m, __shfl_xor(m, 32));
      const int e = row_exponent(m), e1 = e / 2, e2 = e - e1;
      const float f1 = pow2(-e1), f2 = pow2(-e2);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        q[r][i] = __builtin_convertvector(Eight<T>::load(&raw[i]) * f1 * f2, half8);
      factor[r] = a.scale_log2e * pow2(e1) * pow2(e2);
    } else {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) q[r][i] = as_half8(raw[i]);
    }
    seen(a, t, row, &lo[r], &hi[r]);
  }
  // the tile's first and last rows bound what any row sees
  {
    const int64_t last = min(t.row0 + R, rows) - 1;
    seen(a, t, t.row0, &lo_min, &hi_min);
    seen(a, t, last, &lo_max, &hi_max);
  }
  const int g_lo = (int)(lo_min >> 5), g_hi = (int)((hi_max + 31) >> 5);
  int begin = g_lo, end = g_hi;
  if (a.splits > 1) {
    const int n = g_hi - g_lo;
    const int per = max((n + a.splits - 1) / a.splits, kWaves);
    begin = min(g_lo + split * per, g_hi);
    end = min(begin + per, g_hi);
  }

  floatx4 acc[RT][D / 16];
  Running run[RT];
  float top = 0.0f;  // largest vs so far
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    run[r] = {-__builtin_inff(), 0.0f};
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[r][i] = floatx4{0, 0, 0, 0};
  }

  const auto step = [&](const Bytes<D>& b, int g) {
    floatx4 s[RT][2];
#pragma unroll
    for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][tt] = floatx4{0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < D / 64; ++kb) {
        const uint4 d = b.k[tt * (D / 64) + kb];
        const half8 k0 = dequant8(d.x, d.y), k1 = dequant8(d.z, d.w);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          s[r][tt] = mfma16x16x32(k0, q[r][2 * kb], s[r][tt]);
          s[r][tt] = mfma16x16x32(k1, q[r][2 * kb + 1], s[r][tt]);
        }
      }
    }
    const int64_t t0 = (int64_t)g << 5;
    const bool edge = t0 < lo_max || t0 + 32 > hi_min;
    bool raise = larger(b.vs, top);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float c = b.ks * factor[r];
      float mx = -__builtin_inff();
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = s[r][tt][i] * c;
          if (edge) {
            const int64_t tok = t0 + 16 * tt + 4 * lg + i;
            if (tok < lo[r] || tok >= hi[r]) x = -__builtin_inff();
          }
          s[r][tt][i] = x;
          mx = fmaxf(mx, x);
        }
      raise |= mx > run[r].m + (run[r].m == -__builtin_inff() ? 0.0f : kRaise);
    }
    if (__ballot(raise)) {
      const float to = larger(b.vs, top) ? b.vs : top;
      const float fv = to > 0.0f ? top / to : 1.0f;
      top = to;
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float mx = run[r].m;
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[r][tt][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float f = exp2_fast(run[r].m - safe(mx));
        run[r].m = mx;
        run[r].l *= f;
        const float fa = f * fv;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[r][i] *= fa;
      }
    }
    const float lr = ratio_log2(b.vs, top), back = exp2_fast(-lr);
    half8 p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float off = kShift + lr - safe(run[r].m);
      float sum = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = exp2_fast(s[r][tt][i] + off);
          if (edge && s[r][tt][i] == -__builtin_inff()) e = 0.0f;
          sum += e;
          p[r][tt * 4 + i] = (_Float16)e;
        }
      run[r].l += sum == 0.0f ? 0.0f : sum * back;  // (0 of a group whose scale is not finite)
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const half8 v0 = dequant8(b.v[i].x, b.v[i].y), v1 = dequant8(b.v[i].z, b.v[i].w);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        acc[r][2 * i] = mfma16x16x32(v0, p[r], acc[r][2 * i]);
        acc[r][2 * i + 1] = mfma16x16x32(v1, p[r], acc[r][2 * i + 1]);
      }
    }
  };

  if (begin + wave < end) {
    // group g's bytes are loaded while group g - kWaves is worked on, and its
    // block id one turn before that.
    const auto id_of = [&](int g) { return group_of(a, t, h, min(g, end - 1)); };
    int g = begin + wave;
    Bytes<D> b0, b1;
    fetch<D>(a, id_of(g), lane, b0);
    Group next = id_of(g + kWaves);
    while (true) {
      fetch<D>(a, next, lane, b1);
      next = id_of(g + 2 * kWaves);
      step(b0, g);
      g += kWaves;
      if (g >= end) break;
      fetch<D>(a, next, lane, b0);
      next = id_of(g + 2 * kWaves);
      step(b1, g);
      g += kWaves;
      if (g >= end) break;
    }
  }

  // ---- the four wavefronts' results
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    float l = run[r].l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    run[r].l = l;
    if (lg == 0) {
      red_m[wave][16 * r + col] = run[r].m;
      red_l[wave][16 * r + col] = l;
    }
  }
  if (lane == 0) red_v[wave] = top;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    __syncthreads();
    const int rr = 16 * r + col;
    float m = red_m[0][rr];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red_m[w][rr]);
    // nothing seen by this wavefront: its sums are 0 and their factor too
    const float f = exp2_fast(run[r].m - safe(m)) * top;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      *reinterpret_cast<floatx4*>(&red[wave][col][16 * i + 4 * lg]) = acc[r][i] * f;
    __syncthreads();
    for (int it = tid; it < 16 * (D / 8); it += kWaves * kWave) {
      const int c = it / (D / 8), d = it % (D / 8) * 8, rc = 16 * r + c;
      const int64_t row = t.row0 + rc;
      if (row >= rows) continue;
      float mm = red_m[0][rc];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, red_m[w][rc]);
      float l = 0.0f;
      floatx8 o = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        l += red_l[w][rc] * exp2_fast(red_m[w][rc] - safe(mm));
        const floatx4 x = *reinterpret_cast<const floatx4*>(&red[w][c][d]);
        const floatx4 y = *reinterpret_cast<const floatx4*>(&red[w][c][d + 4]);
        o += __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
      }
      const int64_t qi = row / a.group;
      const int64_t to = (t.first_token + qi) * a.hq + h * a.group + (row - qi * a.group);
      if (a.splits > 1) {
        float* part = a.part + (to * a.splits + split) * D + d;
        *reinterpret_cast<floatx8*>(part) = o;
        if (d == 0) a.stat[to * a.splits + split] = floatx4{mm, l, 0, 0};
      } else {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        if (l == 0.0f) o = 0.0f;
        Eight<T>::store(a.out + (to * D + d) * 2, o * inv);
        if (d == 0 && a.lse)
          a.lse[to] = l == 0.0f ? -__builtin_inff() : (mm - kShift + __builtin_amdgcn_logf(l)) * kLn2;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Many rows (prompts): four wavefronts of 32 * RT rows each.  A step's K and V
// bytes are loaded once per workgroup, turned into fp16 on their way into LDS,
// in operand order (a wavefront reads 1 KB in lane order per MFMA), and the
// next step's are loaded meanwhile.
// ---------------------------------------------------------------------------
__device__ __forceinline__ floatx16 mfma32x32x16(half8 a, half8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kWaves* kWave)
__attribute__((amdgpu_waves_per_eu(RT == 1 ? 2 : 1))) void kv8_prefill_kernel(AttnArgs a) {
  constexpr int R = 32 * RT * kWaves;
  constexpr int NG = D <= 128 ? 2 : 1;          // 32-token groups of a step
  constexpr int kBuf = NG * 32 * D * 2 * 2;     // bytes of a step's K and V in fp16
  constexpr int kChunks = NG * D / 128;         // 16-byte chunks of K (and of V) per thread
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 32, lh = lane / 32;
  int64_t id = blockIdx.x;
  const int h = (int)(id % a.hk);
  id /= a.hk;
  const int split = (int)(id % a.splits);
  Tile t;
  // the last tiles of a request see the most tokens: they begin first
  if (!find_tile<R>(a, a.tiles - 1 - id / a.splits, &t)) return;
  const int64_t rows = t.queries * a.group;

  // Size 256: the sums take 128 registers, so the queries stay in LDS, where
  // each lane reads its own.
  constexpr bool kQLds = D > 128;
  half8 q[RT][kQLds ? 1 : D / 16];
  half8* q_lds = reinterpret_cast<half8*>(lds + 2 * kBuf) + wave * (RT * D / 16) * kWave + lane;
  const auto put_q = [&](int r, int i, half8 v) {
    if constexpr (kQLds) q_lds[(r * (D / 16) + i) * kWave] = v;
    else q[r][i] = v;
  };
  const auto get_q = [&](int r, int i) {
    if constexpr (kQLds) return q_lds[(r * (D / 16) + i) * kWave];
    else return q[r][i];
  };
  float factor[RT];
  int64_t lo[RT], hi[RT];
  int64_t my_lo_min, my_lo_max, my_hi_min, my_hi_max, lo_min, hi_max, unused;
  const int64_t wrow = t.row0 + wave * 32 * RT;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    int64_t row = wrow + 32 * r + col;
    if (row >= rows) row = rows - 1;
    const int64_t qi = row / a.group;
    const uint8_t* p = a.q + (t.first_token + qi) * a.q_ts +
                       (h * a.group + (row - qi * a.group)) * a.q_hs + lh * 16;
    uint4 raw[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) raw[i] = load_u4(p + i * 32);
    factor[r] = a.scale_log2e;
    if constexpr (!__is_same(T, _Float16)) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) m = load_amax<T>(raw[i], m);
      m = fmaxf(m, __shfl_xor(m, 32));
      const int e = row_exponent(m), e1 = e / 2, e2 = e - e1;
      const float f1 = pow2(-e1), f2 = pow2(-e2);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        put_q(r, i, __builtin_convertvector(Eight<T>::load(&raw[i]) * f1 * f2, half8));
      factor[r] = a.scale_log2e * pow2(e1) * pow2(e2);
    } else {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) put_q(r, i, as_half8(raw[i]));
    }
    seen(a, t, row, &lo[r], &hi[r]);
  }
  seen(a, t, t.row0, &lo_min, &unused);
  seen(a, t, min(t.row0 + R, rows) - 1, &unused, &hi_max);
  const bool idle = wrow >= rows;
  seen(a, t, idle ? rows - 1 : wrow, &my_lo_min, &my_hi_min);
  seen(a, t, min(wrow + 32 * RT, rows) - 1, &my_lo_max, &my_hi_max);
  const int g_lo = (int)(lo_min >> 5), g_hi = (int)((hi_max + 31) >> 5);
  int begin = g_lo, end = g_hi;
  if (a.splits > 1) {
    const int n = g_hi - g_lo;
    const int per = max((n + a.splits - 1) / a.splits, NG);
    begin = min(g_lo + split * per, g_hi);
    end = min(begin + per, g_hi);
  }

  floatx16 acc[RT][D / 32];
  Running run[RT];
  float top = 0.0f;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    run[r] = {-__builtin_inff(), 0.0f};
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[r][i] = 0.0f;
  }

  // Chunk c of this wavefront is 1 KB tile c * kWaves + wave of the step.
  uint4 kr[kChunks], vr[kChunks];
  const auto load = [&](int g) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int tile = c * kWaves + wave;
      const Group gr = group_of(a, t, h, min(g + tile / (D / 32), end - 1));
      const int64_t at = (gr.at << a.shift) * D + gr.sub * (32 * D) + tile % (D / 32) * kTileBytes + lane * 16;
      kr[c] = load_u4(a.k + at);
      vr[c] = load_u4(a.v + at);
    }
  };
  const int g16 = lane / 16, l16 = lane % 16;
  const auto stage = [&](uint8_t* buf) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int tile = c * kWaves + wave, gr = tile / (D / 32), i = tile % (D / 32);
      {  // token row order: see the file's head (16 tt + 4 x + c -> 16 (x / 2) + 8 tt + 4 (x % 2) + c)
        const int tt = i / (D / 64), kb = i % (D / 64), x = l16 / 4;
        const int row = 16 * (x / 2) + 8 * tt + 4 * (x % 2) + l16 % 4;
        uint8_t* p = buf + ((gr * (D / 16) + kb * 4 + g16) * kWave + row) * 16;
        *reinterpret_cast<half8*>(p) = dequant8(kr[c].x, kr[c].y);
        *reinterpret_cast<half8*>(p + 32 * 16) = dequant8(kr[c].z, kr[c].w);
      }
      {
        uint8_t* p = buf + kBuf / 2 +
                     (((gr * (D / 32) + i) * 2 + g16 / 2) * kWave + (g16 % 2) * 32 + l16) * 16;
        *reinterpret_cast<half8*>(p) = dequant8(vr[c].x, vr[c].y);
        *reinterpret_cast<half8*>(p + 16 * 16) = dequant8(vr[c].z, vr[c].w);
      }
    }
  };
  const auto step = [&](const uint8_t* buf, int g) {
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      const int64_t t0 = (int64_t)(g + n) << 5;
      if (g + n >= end || idle || t0 >= my_hi_max || t0 + 32 <= my_lo_min) continue;
      const Group gr = group_of(a, t, h, g + n);
      const float nan = __builtin_nanf("");
      const float ks = gr.ok ? a.ks[gr.at] : nan, vs = gr.ok ? a.vs[gr.at] : nan;
      floatx16 s[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        const half8 k = *reinterpret_cast<const half8*>(buf + ((n * (D / 16) + i) * kWave + lane) * 16);
#pragma unroll
        for (int r = 0; r < RT; ++r) s[r] = mfma32x32x16(k, get_q(r, i), s[r]);
      }
      const bool edge = t0 < my_lo_max || t0 + 32 > my_hi_min;
      bool raise = larger(vs, top);
      float c[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        c[r] = ks == 0.0f ? 1.0f : ks * factor[r];  // (a block of zeros: every score is 0)
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (edge) {
            const int64_t tok = t0 + 16 * (i / 4 % 2) + 4 * (2 * (i / 8) + lh) + i % 4;
            if (tok < lo[r] || tok >= hi[r]) s[r][i] = -__builtin_inff();
          }
          mx = fmaxf(mx, s[r][i]);
        }
        raise |= mx * c[r] > run[r].m + (run[r].m == -__builtin_inff() ? 0.0f : kRaise);
      }
      if (__ballot(raise)) {
        const float to = larger(vs, top) ? vs : top;
        const float fv = to > 0.0f ? top / to : 1.0f;
        top = to;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          float mx = -__builtin_inff();
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[r][i]);
          mx = fmaxf(run[r].m, mx * c[r]);
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float f = exp2_fast(run[r].m - safe(mx));
          run[r].m = mx;
          run[r].l *= f;
          const float fa = f * fv;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) acc[r][i] *= fa;
        }
      }
      const float lr = ratio_log2(vs, top), back = exp2_fast(-lr);
      half8 p[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float off = kShift + lr - safe(run[r].m);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float e = exp2_fast(__builtin_fmaf(s[r][i], c[r], off));
          if (edge && s[r][i] == -__builtin_inff()) e = 0.0f;
          sum += e;
          p[r][i / 8][i % 8] = (_Float16)e;
        }
        run[r].l += sum == 0.0f ? 0.0f : sum * back;  // (0 of a group whose scale is not finite)
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const half8 v = *reinterpret_cast<const half8*>(
              buf + kBuf / 2 + (((n * (D / 32) + i) * 2 + u) * kWave + lane) * 16);
#pragma unroll
          for (int r = 0; r < RT; ++r) acc[r][i] = mfma32x32x16(v, p[r][u], acc[r][i]);
        }
    }
  };

  if (begin < end) {
    load(begin);
    stage(lds);
    __syncthreads();
    int at = 0;
    for (int g = begin; g < end; g += NG) {
      const bool more = g + NG < end;
      if (more) load(g + NG);
      step(lds + at * kBuf, g);
      if (more) stage(lds + (1 - at) * kBuf);
      __syncthreads();
      at = 1 - at;
    }
  }

#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int64_t row = wrow + 32 * r + col;
    float l = run[r].l;
    l += __shfl_xor(l, 32);
    if (row >= rows) continue;
    const int64_t qi = row / a.group;
    const int64_t to = (t.first_token + qi) * a.hq + h * a.group + (row - qi * a.group);
    const float f = a.splits > 1 ? top : l == 0.0f ? 0.0f : top / l;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        floatx4 o;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] = acc[r][i][4 * j + c] * f;
        const int d = 32 * i + 8 * j + 4 * lh;
        if (a.splits > 1) {
          *reinterpret_cast<floatx4*>(a.part + (to * a.splits + split) * D + d) = o;
        } else {
          typedef T tx4 __attribute__((ext_vector_type(4)));
          *reinterpret_cast<tx4*>(a.out + (to * D + d) * 2) = __builtin_convertvector(o, tx4);
        }
      }
    if (lh == 0) {
      if (a.splits > 1) a.stat[to * a.splits + split] = floatx4{run[r].m, l, 0, 0};
      else if (a.lse)
        a.lse[to] = l == 0.0f ? -__builtin_inff() : (run[r].m - kShift + __builtin_amdgcn_logf(l)) * kLn2;
    }
  }
}

// ---------------------------------------------------------------------------
// The splits of one row, in their order: eight dimensions a thread.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256) void kv8_merge_kernel(AttnArgs a) {
  const int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = it / (D / 8);
  const int d = it % (D / 8) * 8;
  if (row >= a.tokens * a.hq) return;
  const floatx4* stat = a.stat + row * a.splits;
  float m = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, stat[s][0]);
  float l = 0.0f;
  floatx8 o = 0.0f;
  for (int s = 0; s < a.splits; ++s) {
    const float f = exp2_fast(stat[s][0] - safe(m));
    l += stat[s][1] * f;
    const floatx8 x = *reinterpret_cast<const floatx8*>(a.part + (row * a.splits + s) * D + d);
    o += x * f;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = 0.0f;
  Eight<T>::store(a.out + (row * D + d) * 2, o * inv);
  if (d == 0 && a.lse)
    a.lse[row] = l == 0.0f ? -__builtin_inff() : (m - kShift + __builtin_amdgcn_logf(l)) * kLn2;
}

template <typename T, int D>
hipError_t launch_sized(const AttnArgs& a, const Kv8AttnPlan& p, hipStream_t stream) {
  const unsigned grid = (unsigned)(p.tiles * a.hk * a.splits);
  if (p.kernel == 0) {
    if (p.rows == 16) kv8_decode_kernel<T, D, 1><<<grid, kWaves * kWave, 0, stream>>>(a);
    else if constexpr (D <= 128) kv8_decode_kernel<T, D, 2><<<grid, kWaves * kWave, 0, stream>>>(a);
  } else {
    const size_t lds = 2 * (D <= 128 ? 2 : 1) * 32 * D * 2 * 2 + (D > 128 ? kWaves * 32 * D * 2 : 0);
    kv8_prefill_kernel<T, D, 1><<<grid, kWaves * kWave, lds, stream>>>(a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  kv8_merge_kernel<T, D><<<(unsigned)ceil_div(a.tokens * a.hq * (D / 8), 256), 256, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

Kv8AttnPlan plan_kv8_attention(const rf_kv8_attention_args& a, int cus) {
  Kv8AttnPlan p;
  const int64_t group = a.q.heads / a.cache.kv_heads;
  int64_t most_q = a.cu_q ? a.max_q_len : ceil_div(a.tokens, a.requests);
  if (most_q < 1 || most_q > a.tokens) most_q = a.tokens;
  const int64_t most_rows = most_q * group;
  p.kernel = most_rows > 64 ? 1 : 0;
  // (two tiles of 16 rows of size 256 would not fit the registers)
  p.rows = p.kernel ? 128 : most_rows <= 16 || a.cache.head_dim > 128 ? 16 : 32;
  p.tiles = a.cu_q ? a.tokens * group / p.rows + a.requests + 1
                   : a.requests * ceil_div(most_rows, p.rows);
  int64_t most_kv = a.width * a.cache.block_size;
  if (a.max_kv_len > 0 && a.max_kv_len < most_kv) most_kv = a.max_kv_len;
  if (a.window > 0 && a.window + most_q < most_kv) most_kv = a.window + most_q;
  // Useful tiles, of which each is cut along its tokens until the launch has
  // about `want` workgroups, in pieces of at least `least` groups.
  const int64_t tiles = p.kernel ? ceil_div(a.tokens * group, p.rows) : a.requests * ceil_div(most_rows, p.rows);
  const int64_t busy = tiles * a.cache.kv_heads;
  const int64_t want = p.kernel ? 2 * cus : 4 * cus, least = p.kernel ? 16 : 4;
  const int64_t groups = ceil_div(most_kv, RF_KV8_GROUP);
  int64_t s = want / (busy > 0 ? busy : 1);
  if (s > groups / least) s = groups / least;
  p.splits = (int)(s < 1 ? 1 : s > 128 ? 128 : s);
  const int64_t D = a.cache.head_dim;
  p.workspace = p.splits == 1 ? 0 : (size_t)(a.tokens * a.q.heads * p.splits) * (D + 4) * 4;
  return p;
}

hipError_t launch_kv8_attention(const rf_kv8_attention_args& in, const Kv8AttnPlan& p,
                                hipStream_t stream) {
  AttnArgs a;
  a.q = (const uint8_t*)in.q.data;
  a.q_ts = in.q.token_stride * 2;
  a.q_hs = in.q.head_stride * 2;
  a.k = (const uint8_t*)in.cache.k;
  a.v = (const uint8_t*)in.cache.v;
  a.ks = in.cache.k_scale;
  a.vs = in.cache.v_scale;
  a.cu = in.cu_q;
  a.lens = in.kv_lens;
  a.table = in.block_table;
  a.out = (uint8_t*)in.out;
  a.lse = in.lse;
  const int D = in.cache.head_dim;
  const int64_t rows = in.tokens * in.q.heads * p.splits;
  a.stat = (floatx4*)in.workspace;
  a.part = (float*)in.workspace + rows * 4;
  a.tokens = in.tokens;
  a.table_stride = in.table_stride;
  a.num_blocks = in.cache.num_blocks;
  a.requests = (int)in.requests;
  a.width = (int)in.width;
  a.hq = in.q.heads;
  a.hk = in.cache.kv_heads;
  a.group = a.hq / a.hk;
  a.shift = __builtin_ctz((unsigned)in.cache.block_size);
  a.per_request = in.cu_q ? 0 : (int)(in.tokens / in.requests);
  a.splits = p.splits;
  a.tiles = (int)p.tiles;
  a.causal = in.causal;
  a.window = in.window;
  a.scale_log2e = in.scale * kLog2e;
  const bool f16 = in.dtype == RF_W8A16_DTYPE_F16;
  if (D == 64)
    return f16 ? launch_sized<_Float16, 64>(a, p, stream) : launch_sized<__bf16, 64>(a, p, stream);
  if (D == 128)
    return f16 ? launch_sized<_Float16, 128>(a, p, stream) : launch_sized<__bf16, 128>(a, p, stream);
  return f16 ? launch_sized<_Float16, 256>(a, p, stream) : launch_sized<__bf16, 256>(a, p, stream);
}

}  // namespace rf
