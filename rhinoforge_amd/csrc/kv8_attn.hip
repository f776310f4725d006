// Attention over the int8 paged cache (kv8.h), gfx950.
//
// For query row q (one query, one head) over its seen tokens j:
//   x_j = (q . k_j) ks scale log2(e),  p_j = 2^(x_j - m),  o = vs sum p_j v_j / sum p_j
// with integer k_j, v_j and the scales ks, vs of the token's block.  One pass
// over the tokens with two running references for each row: m follows its
// largest x, m + d its largest x + log2 vs.  The sum l is kept relative to m, the
// weights w_j = 2^(x_j + log2 vs_j - m - d) and o relative to m + d.  Both only
// have to stay in range, so they move when something is 8 or more above them, not
// at every step.
//
// Both products run on the matrix cores with the cache as the A operand and the
// queries as columns: S^T = K Q^T leaves each lane with scores of one query row
// (its column), and after exp2 those are the B operand of O^T = V^T P^T as they
// stand (the v tiles hold tokens in that order).  int8 -> fp16 is exact.
//   * Queries: fp16 as they are.  bf16 times a power of two per row, which
//     brings the row's largest magnitude to [2^14, 2^15): exact in fp16 down to
//     2^-31 of it, within 2^-39 of it below; the power goes into that row's score
//     factor.
//   * w is rounded to fp16 (11 bits, round to nearest): 2^-11 relative, as much
//     as the output's own rounding in fp16.  2^7 w is what is rounded: the row's
//     largest lies in [2^7, 2^15), and a weight below fp16's normal range loses at
//     most 2^-25, 2^-32 of the largest p vs that the row sees.  What other rows
//     see, and blocks without weight, do not count.
//   * A sum over w of one block, times 2^-(log2 vs - d), is its part of l.
//     m, d, the sums and o stay in fp32.
#include "paged_attn.h"

namespace rf {
namespace {

struct AttnArgs : PagedArgs {
  const float *ks, *vs;
};

// A scale's bits (kept as an integer: compares and branches on it are scalar).
// Scales are not negative, so their order is that of the bits.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t scale_bits(const float* p, const Group& g) {
  const uint32_t v = read_scalar(reinterpret_cast<const uint32_t*>(p), g.at);
  return g.ok ? v : kInfBits;
}
__device__ __forceinline__ float as_float(uint32_t bits) { return __builtin_bit_cast(float, bits); }

// Running softmax of one query row, as the lanes of its column hold it: m and
// d agree over them, l is each lane's own share of the sum.
struct Running {
  float m = -__builtin_inff();  // log2 units; -inf: nothing seen
  float l = 0.0f;
  float d = 0.0f;               // the sums of p vs v are in units of 2^(m + d)
};

// s c - m, both steps rounded: 0 where m is that product.
__device__ __forceinline__ float product_minus(float s, float c, float m) {
#pragma clang fp contract(off)
  return s * c - m;
}

// log2 of a value scale; of 0, so low that 2^ it is 0 and differences stay finite.
__device__ __forceinline__ float scale_log2(uint32_t vs) {
  float log = log2_fast(as_float(vs));
  if (vs < 0x00800000u) {  // (the instruction takes denormals as 0)
    keep_branch();
    log = fmaxf(log2_fast(as_float(vs) * 0x1p64f) - 64.0f, -300.0f);
  }
  return log;
}
// log2 vs relative to the row's d, for the exponent, not below -60: 2^7 w is then
// below 2^(15 - 60), which rounds to 0 in fp16.
__device__ __forceinline__ float ratio_log2(float log_vs, const Running& r) {
  return fmaxf(log_vs - r.d, -60.0f);
}

// A row's references once m is its largest score, and new scores with log2 vs lie at
// most `above` over that; by how much l and the sums of p vs v change.  (d comes from
// differences of scores: a score's sum with log2 vs would not hold it from 2^24 on.)
struct Change {
  float l, o;
};
__device__ __forceinline__ Change raise_to(Running& r, float m, float above) {
  const float fall = r.m - safe(m), d = m == -__builtin_inff() ? 0.0f : fmaxf(r.d + fall, above);
  const Change c = {exp2_fast(fall), exp2_fast(fall + (r.d - d))};
  r.m = m;
  r.d = d;
  return c;
}
// 2^(d / 2), to be applied twice: 2^d itself may leave fp32's normal range.
__device__ __forceinline__ float half_unit(const Running& r) { return exp2_fast(0.5f * r.d); }

// A group with a scale that is not finite (or negative): its scores become NaN
// (those of tokens that a row does not see are overwritten after that) and the
// scales harmless.
__device__ __forceinline__ bool not_finite(uint32_t ks, uint32_t vs) {
  return (ks > vs ? ks : vs) >= kInfBits;
}
constexpr uint32_t kOneBits = 0x3f800000u;

// ---------------------------------------------------------------------------
// Few rows (single tokens, a few drafted ones): RT tiles of 16 rows, held by
// all four wavefronts; the wavefronts take 32-token groups in turn and read the
// cache straight into MFMA operands (no LDS), one turn ahead of the products.  At
// the end the wavefronts' sums meet in LDS.  Bound by the cache's bytes: 130999
// tokens, 32 + 8 heads of 128, in 47.1 us, 5.7 TB/s (a plain read of as many bytes
// reaches 6.7); short contexts by their round trips: 777 tokens 8.4 us, of which
// 4.4 remain for 64 tokens.  Eight wavefronts a workgroup gave the same times:
// one CU takes in about 64 GB/s however many of them ask.
// ---------------------------------------------------------------------------
template <int D>
struct Bytes {
  uint4 k[D / 32], v[D / 32];
  uint32_t ks, vs;
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
  // (the scales' wait would otherwise come before the bytes go out)
  if constexpr (D <= 128) __builtin_amdgcn_sched_barrier(0);
  b.ks = scale_bits(a.ks, g);
  b.vs = scale_bits(a.vs, g);
}

template <typename T, int D, int RT>
__global__ __launch_bounds__(kWaves* kWave)
__attribute__((amdgpu_waves_per_eu(2))) void kv8_decode_kernel(AttnArgs a) {
  constexpr int R = 16 * RT;
  __shared__ __align__(16) float red[kWaves][16][D + 4];
  __shared__ float red_m[kWaves][R], red_l[kWaves][R];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int col = lane % 16, lg = lane / 16;
  const unsigned id = a.first + blockIdx.x, pair = id / (unsigned)a.hk;
  const int h = (int)(id - pair * a.hk);
  int split, splits;
  Tile t;
  if (a.shares) {
    if (!find_share<R>(a, (int)pair, &t, &split, &splits)) return;
  } else {
    const int x = (int)(pair / (unsigned)a.splits);
    if (!find_tile<R>(a, x, &t)) return;
    splits = a.splits;
    split = (int)(pair - (unsigned)x * splits);
  }
  const int rows = min(t.queries * a.group - t.row0, R);  // of this tile
  // its first and last rows bound what any row sees
  int lo_min, lo_max, hi_min, hi_max;
  seen(a, t, t.row0, &lo_min, &hi_min);
  seen(a, t, t.row0 + rows - 1, &lo_max, &hi_max);
  lo_max = uniform(lo_max), hi_min = uniform(hi_min);
  const Share share = share_of(a, lo_min >> 5, (hi_max + 31) >> 5, split, splits);
  if (split >= share.splits) {
    if (a.merge) no_share(a, t, h, rows, split);
    return;
  }
  const int begin = uniform(share.begin), end = uniform(share.end);
  const bool partial = share.splits > 1 || a.merge;

  // ---- queries, as B operands: column = row, 16 dimensions 64 kb + 16 lg + ..
  half8 q[RT][D / 32];
  float factor[RT];
  int lo[RT], hi[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = t.row0 + min(16 * r + col, rows - 1);
    const int qi = (int)((unsigned)row / (unsigned)a.group);
    const uint8_t* p = a.q + (int64_t)(t.first_token + qi) * a.q_ts +
                       (int64_t)(h * a.group + (row - qi * a.group)) * a.q_hs + lg * 32;
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
    factor[r] = in_range(factor[r]);
    seen(a, t, row, &lo[r], &hi[r]);
  }
  floatx4 acc[RT][D / 16];
  Running run[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[r][i] = floatx4{0, 0, 0, 0};

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
    uint32_t ks = b.ks, vs = b.vs;
    if (not_finite(ks, vs)) {
      keep_branch();
      ks = kOneBits;
      vs = 0;
#pragma unroll
      for (int r = 0; r < RT; ++r) s[r][0] = s[r][1] = __builtin_nanf("");
    }
    const int t0 = opaque(g << 5);
    const bool edge = t0 < lo_max || t0 + 32 > hi_min;
    const float log_vs = scale_log2(vs);
    bool raise = false;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float c = in_range(as_float(ks) * factor[r]);
      const int first = lo[r] - t0 - 4 * lg, past = hi[r] - t0 - 4 * lg;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) s[r][tt] *= c;
      if (edge) {
        keep_branch();
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int tok = 16 * tt + i;  // past t0 + 4 lg
            s[r][tt][i] = (tok < first) | (tok >= past) ? -__builtin_inff() : s[r][tt][i];
          }
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[r][tt][i]);
      raise |= minus(mx, run[r].m) + fmaxf(log_vs - run[r].d, 0.0f) > kRaise;  // (NaN: nothing seen yet)
    }
    if (__ballot(raise)) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int tt = 0; tt < 2; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[r][tt][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m = fmaxf(run[r].m, mx);
        const Change f = raise_to(run[r], m, minus(mx, safe(m)) + log_vs);
        run[r].l *= f.l;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[r][i] *= f.o;
      }
    }
    float lr[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) lr[r] = 0.0f;
    if (opaque(t0) >= 0) {  // (always: see the prefill kernel)
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        lr[r] = ratio_log2(log_vs, run[r]);
        asm volatile("" : "+v"(lr[r]));
      }
    }
    half8 p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float off = kShift + lr[r], m = safe(run[r].m);
      float sum = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = exp2_fast(minus(s[r][tt][i], m) + off);
          sum += e;
          p[r][tt * 4 + i] = (_Float16)e;
        }
      run[r].l += sum * exp2_fast(-lr[r]);
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
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    __syncthreads();
    const int rr = 16 * r + col;
    float m = red_m[0][rr];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red_m[w][rr]);
    // nothing seen by this wavefront: its sums are 0 and their factor too
    const float half = half_unit(run[r]), f = exp2_fast(run[r].m - safe(m)) * half;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      *reinterpret_cast<floatx4*>(&red[wave][col][16 * i + 4 * lg]) = acc[r][i] * half * f;
    __syncthreads();
    for (int it = tid; it < 16 * (D / 4); it += kThreads) {
      const int c = it / (D / 4), d = it % (D / 4) * 4, rc = 16 * r + c;
      if (rc >= rows) continue;
      float mm = red_m[0][rc];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) mm = fmaxf(mm, red_m[w][rc]);
      float l = 0.0f;
      floatx4 o = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        l += red_l[w][rc] * exp2_fast(red_m[w][rc] - safe(mm));
        o += *reinterpret_cast<const floatx4*>(&red[w][c][d]);
      }
      const int64_t to = out_row(a, t, h, rc);
      if (partial) {
        const Partials parts(a);
        const int i = a.merge ? (int)to * a.splits + split : (int)id * R + rc;
        parts.store(i * D + d, o);
        if (d == 0) parts.store_stat(i, mm, l);
      } else {
        finish<T>(a, to, D, d, o, mm, l);
      }
    }
  }
  if (partial && !a.merge)
    join<T, D, R, kThreads>(a, t, h, rows, share.splits, ((int)id - split * a.hk) * R, a.hk * R,
               a.counters + (id - (unsigned)(split * a.hk)), &red[0][0][0]);
}

// ---------------------------------------------------------------------------
// Many rows (prompts): four wavefronts of 32 rows each.  A step's K and V bytes
// are loaded once per workgroup, turned into fp16 on their way into LDS, in
// operand order (a wavefront reads 1 KB in lane order per MFMA), and those of
// the next two steps are loaded meanwhile.  G = 2: two gangs of four wavefronts
// take the steps of the same rows in turn, and their sums join at the end: what
// the longest tile takes is halved, which is what a prompt takes that does not
// fill the chip several times (2500 tokens, 16 + 8 heads: 69 us with one gang, 49
// with two; 1000 tokens, 32 + 8: 32 and 26; but 7999, 64 + 8: 1127 and 1224).
// 7999 tokens, 64 + 8 heads of 128:
// 1089 to 1174 us on different cards, 963 to 893 TFLOP/s, where a library product
// of 16384^3 reaches 1300.
// Vector units 63% and matrix units 45% busy at 1.9 of 2.4 GHz: the clock gives
// way to the power they draw.  Variants with other orders of the same
// instructions (products and weights interleaved one by one, operands read
// ahead, loads one step ahead instead of two) differ by up to 6% in cycles and
// by 1% in time.
// ---------------------------------------------------------------------------
template <typename T, int D, int G>
__global__ __launch_bounds__(G* kWaves* kWave)
__attribute__((amdgpu_waves_per_eu(2))) void kv8_prefill_kernel(AttnArgs a) {
  constexpr int R = 32 * kWaves;
  constexpr int NG = D <= 128 ? 2 : 1;          // 32-token groups of a step
  constexpr int kBuf = NG * 32 * D * 2 * 2;     // bytes of a step's K and V in fp16
  constexpr int kChunks = NG * D / 128;         // 16-byte chunks of K (and of V) per thread
  constexpr bool kQLds = D > 128;               // see below
  // (sized at the launch: with the size known here the register allocator
  // trades registers for it, and spills)
  extern __shared__ __align__(16) uint8_t lds[];
  const int tid = threadIdx.x, lane = tid % kWave, any_wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wave = any_wave % kWaves, gang = any_wave / kWaves;
  uint8_t* const bufs = lds + gang * 2 * kBuf;
  const int col = lane % 32, lh = lane / 32;
  const unsigned id = a.first + blockIdx.x, pair = id / (unsigned)a.hk;
  const int h = (int)(id - pair * a.hk), turn = (int)(pair / (unsigned)a.splits);
  const int split = (int)(pair - (unsigned)turn * a.splits);
  // the last tiles of a request see the most tokens: they begin first
  const int x = a.tiles - 1 - turn;
  Tile t;
  if (!find_tile<R>(a, x, &t)) return;
  const int rows = min(t.queries * a.group - t.row0, R);  // of this tile
  int lo_min, hi_max, unused;
  seen(a, t, t.row0, &lo_min, &unused);
  seen(a, t, t.row0 + rows - 1, &unused, &hi_max);
  const Share share = share_of(a, lo_min >> 5, (hi_max + 31) >> 5, split, a.splits);
  if (split >= share.splits) {
    no_share(a, t, h, rows, split);
    return;
  }
  const int begin = uniform(share.begin), end = uniform(share.end);
  const bool partial = a.splits > 1;  // merge_splits_kernel adds them

  // Size 256: the sums take 128 registers, so the queries stay in LDS, where
  // each lane reads its own.
  half8 q[kQLds ? 1 : D / 16];
  half8* q_lds = reinterpret_cast<half8*>(lds + G * 2 * kBuf) + wave * (D / 16) * kWave + lane;
  const auto put_q = [&](int i, half8 v) {
    if constexpr (kQLds) q_lds[i * kWave] = v;
    else q[i] = v;
  };
  const auto get_q = [&](int i) {
    if constexpr (kQLds) return q_lds[i * kWave];
    else return q[i];
  };
  float factor = a.scale_log2e;
  int lo, hi;
  const int wrow = wave * 32;  // this wavefront's first row of the tile
  {
    const int row = t.row0 + min(wrow + col, rows - 1);
    const int qi = (int)((unsigned)row / (unsigned)a.group);
    const uint8_t* p = a.q + (int64_t)(t.first_token + qi) * a.q_ts +
                       (int64_t)(h * a.group + (row - qi * a.group)) * a.q_hs + lh * 16;
    uint4 raw[D / 16];
#pragma unroll
    for (int i = 0; i < D / 16; ++i) raw[i] = load_u4(p + i * 32);
    if constexpr (!__is_same(T, _Float16)) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) m = load_amax<T>(raw[i], m);
      m = fmaxf(m, __shfl_xor(m, 32));
      const int e = row_exponent(m), e1 = e / 2, e2 = e - e1;
      const float f1 = pow2(-e1), f2 = pow2(-e2);
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        put_q(i, __builtin_convertvector(Eight<T>::load(&raw[i]) * f1 * f2, half8));
      factor = a.scale_log2e * pow2(e1) * pow2(e2);
    } else {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) put_q(i, as_half8(raw[i]));
    }
    factor = in_range(factor);
    seen(a, t, row, &lo, &hi);
    hi = min(hi, end * 32);
  }
  const bool idle = wrow >= rows;
  int my_lo_min, my_lo_max, my_hi_min, my_hi_max;
  seen(a, t, t.row0 + min(wrow, rows - 1), &my_lo_min, &my_hi_min);
  seen(a, t, t.row0 + min(wrow + 32, rows) - 1, &my_lo_max, &my_hi_max);
  my_lo_min = uniform(my_lo_min), my_lo_max = uniform(my_lo_max);
  my_hi_min = min(uniform(my_hi_min), end * 32), my_hi_max = min(uniform(my_hi_max), end * 32);

  floatx16 acc[D / 32];
  Running run;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;

  // Chunk c of this wavefront is 1 KB tile c * kWaves + wave of the step.  A
  // step's bytes and scales are loaded two steps ahead (a short share is bound
  // by their round trip), its block ids three.
  struct Ahead {
    uint4 k[kChunks], v[kChunks];
    uint32_t ks[NG], vs[NG];
  };
  Group ids[NG];
  const auto look = [&](int g) {
#pragma unroll
    for (int n = 0; n < NG; ++n) ids[n] = group_of(a, t, h, min(g + n, end - 1));
  };
  const auto load = [&](Ahead& x) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int tile = c * kWaves + wave;
      const Group& gr = NG == 1 || (D == 64 ? wave < 2 : c == 0) ? ids[0] : ids[NG - 1];
      const int64_t at = (gr.at << a.shift) * D + gr.sub * (32 * D) + tile % (D / 32) * kTileBytes + lane * 16;
      x.k[c] = load_u4(a.k + at);
      x.v[c] = load_u4(a.v + at);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      x.ks[n] = scale_bits(a.ks, ids[n]);
      x.vs[n] = scale_bits(a.vs, ids[n]);
    }
  };
  const int g16 = lane / 16, l16 = lane % 16;
  const auto stage = [&](uint8_t* buf, const Ahead& x) {
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
      const int tile = c * kWaves + wave, gr = tile / (D / 32), i = tile % (D / 32);
      {  // token row order: see the file's head (16 tt + 4 x + c -> 16 (x / 2) + 8 tt + 4 (x % 2) + c)
        const int tt = i / (D / 64), kb = i % (D / 64), quad = l16 / 4;
        const int row = 16 * (quad / 2) + 8 * tt + 4 * (quad % 2) + l16 % 4;
        uint8_t* p = buf + ((gr * (D / 16) + kb * 4 + g16) * kWave + row) * 16;
        *reinterpret_cast<half8*>(p) = dequant8(x.k[c].x, x.k[c].y);
        *reinterpret_cast<half8*>(p + 32 * 16) = dequant8(x.k[c].z, x.k[c].w);
      }
      {
        uint8_t* p = buf + kBuf / 2 +
                     (((gr * (D / 32) + i) * 2 + g16 / 2) * kWave + (g16 % 2) * 32 + l16) * 16;
        *reinterpret_cast<half8*>(p) = dequant8(x.v[c].x, x.v[c].y);
        *reinterpret_cast<half8*>(p + 16 * 16) = dequant8(x.v[c].z, x.v[c].w);
      }
    }
  };
  // One step of a wavefront: all of its scores, one look at their maximum, then
  // the weights.  The products of a group with V are issued among the weights of
  // the next group, the last ones among the conversion of the next step's bytes:
  // those take the vector units, these the matrix units.  A wavefront's priority
  // rises through the step, so that of two that share a SIMD the one ahead stays
  // ahead and they are in different phases (five prompts with a window 151.9 ->
  // 143.6 us, 2500 tokens 50.4 -> 48.6; on another card 155.0 -> 148.6).
  const auto step = [&](const uint8_t* buf, int g, const uint32_t (&kss)[NG], const uint32_t (&vss)[NG],
                        uint8_t* out, const Ahead& next) {
    const int t0 = opaque(g << 5);
    if (idle || t0 >= my_hi_max || t0 + 32 * NG <= my_lo_min) {
      stage(out, next);
      return;
    }
    floatx16 s[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) s[n] = 0.0f;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const half8 k = *reinterpret_cast<const half8*>(buf + ((n * (D / 16) + i) * kWave + lane) * 16);
        s[n] = mfma32x32x16(k, get_q(i), s[n]);
      }
    __builtin_amdgcn_s_setprio(2);
    uint32_t ks[NG];
    float log_vs[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      ks[n] = kss[n];
      uint32_t vs = vss[n];
      if (not_finite(ks[n], vs)) {
        keep_branch();
        ks[n] = kOneBits;
        vs = 0;
        s[n] = __builtin_nanf("");
      }
      log_vs[n] = scale_log2(vs);
    }
    if (t0 < my_lo_max || t0 + 32 * NG > my_hi_min) {
      keep_branch();
      const int first = lo - t0 - 4 * lh, past = hi - t0 - 4 * lh;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int tok = 32 * n + 16 * (i / 4 % 2) + 8 * (i / 8) + i % 4;  // past t0 + 4 lh
          s[n][i] = (tok < first) | (tok >= past) ? -__builtin_inff() : s[n][i];
        }
    }
    // the largest scores, and how far they, or with log2 vs what is above d, are over m
    float c[NG], most[NG], over = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      // (not 0, also where ks is 0 or the product underflows: masked scores are
      // -inf here already, and -inf * 0 is NaN)
      c[n] = in_range(as_float(ks[n]) * factor);
      most[n] = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; ++i) most[n] = fmaxf(most[n], s[n][i]);
      most[n] *= c[n];
      over = fmaxf(over, minus(most[n], run.m) + fmaxf(log_vs[n] - run.d, 0.0f));
    }
    if (__ballot(over > kRaise)) {
      float mx = fmaxf(most[0], most[NG - 1]);
      mx = fmaxf(run.m, fmaxf(mx, __shfl_xor(mx, 32)));
      float above = fmaxf(minus(most[0], safe(mx)) + log_vs[0], minus(most[NG - 1], safe(mx)) + log_vs[NG - 1]);
      above = fmaxf(above, __shfl_xor(above, 32));
      const Change f = raise_to(run, mx, above);
      run.l *= f.l;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] *= f.o;
    }
    // (a branch the compiler cannot fold: in one block with the merge above it
    // would keep the sums twice, 256 registers instead of 211, and spill)
    float lr[NG];
#pragma unroll
    for (int n = 0; n < NG; ++n) lr[n] = 0.0f;
    if (opaque(t0) >= 0) {  // (always: a block of its own)
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        lr[n] = ratio_log2(log_vs[n], run);
        asm volatile("" : "+v"(lr[n]));
      }
    }
    // Scores of ordinary size take one instruction for their product with c and the
    // difference from m.  Of large ones m, rounded, would be off by more than the
    // weights have room for: the products are rounded as m was.
    float base = safe(run.m);
    if (__ballot(fabsf(base) > kFar)) {
      keep_branch();
#pragma unroll
      for (int n = 0; n < NG; ++n) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = product_minus(s[n][i], c[n], base);
        c[n] = 1.0f;
      }
      base = 0.0f;
    }
    half8 p[2];
    const auto weights = [&](int n) {
      const float off = kShift + lr[n] - base;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_fast(__builtin_fmaf(s[n][i], c[n], off));
        sum += e;
        p[i / 8][i % 8] = (_Float16)e;
      }
      run.l += sum * exp2_fast(-lr[n]);
    };
    const auto add = [&](int n, const half8 (&p)[2]) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const half8 v = *reinterpret_cast<const half8*>(
              buf + kBuf / 2 + (((n * (D / 32) + i) * 2 + u) * kWave + lane) * 16);
          acc[i] = mfma32x32x16(v, p[u], acc[i]);
        }
    };
    __builtin_amdgcn_s_setprio(3);
    weights(0);
    if constexpr (NG == 2) {
      const half8 p0[2] = {p[0], p[1]};
      add(0, p0);
      weights(1);
    }
    add(NG - 1, p);
    __builtin_amdgcn_s_setprio(0);
    stage(out, next);
  };

  if (begin < end) {
    // (past the end the last group is loaded again, and masked)
    constexpr int kStride = G * NG;
    const int turns = (end - begin + kStride - 1) / kStride;
    int g = begin + gang * NG;
    Ahead x0, x1;
    look(g);
    load(x0);
    look(g + kStride);
    load(x1);
    look(g + 2 * kStride);
    stage(bufs, x0);
    __syncthreads();
    const auto turn = [&](Ahead& now, Ahead& next, const uint8_t* in, uint8_t* out, int g) {
      uint32_t ks[NG], vs[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        ks[n] = now.ks[n];
        vs[n] = now.vs[n];
      }
      load(now);
      look(g + 3 * kStride);
      step(in, g, ks, vs, out, next);
      __syncthreads();
    };
    for (int i = 0; i < turns; i += 2, g += 2 * kStride) {
      turn(x0, x1, bufs, bufs + kBuf, g);
      if (i + 1 < turns) turn(x1, x0, bufs + kBuf, bufs, g + kStride);
    }
  }

  if constexpr (G == 2) {  // the second gang's sums join the first's, lane by lane
    float* sums = reinterpret_cast<float*>(lds) + wave * (D / 2) * kWave + lane;
    float* stats = reinterpret_cast<float*>(lds) + kWaves * (D / 2) * kWave + wave * 2 * kWave + lane;
    const float half = half_unit(run);
    if (gang == 1) {
#pragma unroll
      for (int i = 0; i < D / 2; ++i) sums[i * kWave] = acc[i / 16][i % 16] * half * half;
      stats[0] = run.m;
      stats[kWave] = run.l;
    }
    __syncthreads();
    if (gang == 0) {
      const float om = stats[0], m = fmaxf(run.m, om);
      const float f = exp2_fast(run.m - safe(m)), of = exp2_fast(om - safe(m));
      const float fa = f * half;
#pragma unroll
      for (int i = 0; i < D / 2; ++i) acc[i / 16][i % 16] = acc[i / 16][i % 16] * half * fa + sums[i * kWave] * of;
      run.m = m;
      run.l = run.l * f + stats[kWave] * of;
      run.d = 0.0f;
    }
    __syncthreads();  // the rows go out through the same memory
    if (gang == 1) return;
  }

  // Rows go out through LDS (each wavefront its own part, free after the last
  // barrier), 64 dimensions at a time: straight from the registers every lane
  // would store four values of another row.
  constexpr int kPitch = 64 + 4;
  float* mine = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
  float l = run.l;
  l += __shfl_xor(l, 32);
  const int left = rows - wrow;  // rows of this wavefront's tile
  const float half = half_unit(run), f = partial ? half : l == 0.0f ? 0.0f : half / l;
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      floatx4 o;
#pragma unroll
      for (int c = 0; c < 4; ++c) o[c] = acc[i + j / 4][4 * (j % 4) + c] * half * f;
      *reinterpret_cast<floatx4*>(mine + col * kPitch + 8 * j + 4 * lh) = o;
    }
    const int d = lane % 8 * 8;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int rr = 8 * n + lane / 8;
      if (rr >= left) continue;
      const float* src = mine + rr * kPitch + d;
      const floatx4 x = *reinterpret_cast<const floatx4*>(src);
      const floatx4 y = *reinterpret_cast<const floatx4*>(src + 4);
      const int64_t to = out_row(a, t, h, wrow + rr);
      if (partial) {
        float* part = a.part + (to * a.splits + split) * D + 32 * i + d;
        *reinterpret_cast<floatx4*>(part) = x;
        *reinterpret_cast<floatx4*>(part + 4) = y;
      } else {
        Eight<T>::store(a.out + (to * D + 32 * i + d) * 2,
                        __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
      }
    }
  }
  if (lh == 0 && col < left) {
    const int64_t to = out_row(a, t, h, wrow + col);
    if (partial) Partials(a).store_stat((int)to * a.splits + split, run.m, l);
    else if (a.lse)
      a.lse[to] = l == 0.0f ? -__builtin_inff() : (run.m - kShift + log2_fast(l)) * kLn2;
  }
}

template <typename T, int D>
hipError_t launch_sized(AttnArgs a, const PagedPlan& p, hipStream_t stream) {
  constexpr size_t kLds = D == 64 ? kWaves * 32 * 68 * 4
                                  : 2 * (D <= 128 ? 2 : 1) * 32 * D * 2 * 2 + (D > 128 ? 128 * D * 2 : 0);
  constexpr size_t kLds2 = 4 * 2 * 32 * D * 2 * 2;
  // (no workgroup waits for another, so those of one tile may be in two launches)
  const int64_t most = kMaxThreads / (p.gangs * kThreads);
  for (int64_t i = 0; i < p.grid; i += most) {
    a.first = (unsigned)i;
    const unsigned grid = (unsigned)(p.grid - i < most ? p.grid - i : most);
    if (p.kernel == 1 && p.gangs == 1) kv8_prefill_kernel<T, D, 1><<<grid, kThreads, kLds, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 16 && p.gangs == 1) kv8_decode_kernel<T, D, 1><<<grid, kThreads, 0, stream>>>(a);
    else if constexpr (D <= 128) {
      if (p.kernel == 1 && p.gangs == 2) kv8_prefill_kernel<T, D, 2><<<grid, 2 * kThreads, kLds2, stream>>>(a);
      else if (p.kernel == 0 && p.rows == 32 && p.gangs == 1) kv8_decode_kernel<T, D, 2><<<grid, kThreads, 0, stream>>>(a);
      else return hipErrorInvalidValue;
    } else {
      return hipErrorInvalidValue;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.merge) return hipSuccess;
  merge_splits_kernel<T, D>
      <<<(unsigned)ceil_div((int64_t)a.tokens * a.hq * (D / 4), kThreads), kThreads, 0, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

// The launch: which kernel, and in how many splits each tile's tokens (batches
// of unequal lengths cut them into equal shares, below).  The kernels' times
// follow from the number of workgroups and the turns each makes (decode: four
// 32-token groups, one per wavefront; prefill: one step of each gang), with the
// constants below fitted to 18 shapes at 1, 2, 4, 8 and 16 splits on either
// kernel and to 19 prompts on one and two gangs.  Small batches of a few hundred
// rows run on the decode kernel (4 x 50 queries, 32 + 8 heads, 1018 tokens: 14.3
// us unsplit, the prefill kernel 19.1 at its best), prompts that fill the chip on
// the prefill kernel (7999 tokens, 64 + 8 heads: 1.13 ms, the decode kernel 1.57).
//
// Batches of several requests, in workgroups of shares (16 requests of 4 to 20
// thousand tokens, 32 + 8 heads, 1, 1.25, 2 and 3 workgroups a CU: 64.8, 74.8, 63.5,
// 65.4 us; 48 of up to 9000, 64 + 8 heads: 2, 2.5, 3 and 4: 95.9, 87.8, 83.5, 88.9),
// whose least length is that of the join they cost (32 requests of up to 500 tokens:
// 8.0 us, in shares of 8 groups 11.5; 4 x 50 queries after 968 tokens, 32 rows: 14.0
// and 20.9).
namespace {

struct Kv8Costs {
  static double base(bool prefill, int rows, int D) {
    return prefill ? (D == 64 ? 1.1 : D == 128 ? 1.5 : 1.35)
                   : D == 256 ? 1.1 : (rows == 16 ? 0.55 : 0.85) * (D == 64 ? 0.75 : 1.0);
  }
  static double more(bool prefill, int rows, int D) {
    return prefill ? (D == 256 ? 0.6 : 0.4) : D == 256 ? 1.2 : (rows == 16 ? 0.25 : 0.58) * (D == 64 ? 0.6 : 1.0);
  }
  // (prompts of size 256: LDS holds one on each CU, the fitted constants go with two)
  static double slots(bool prefill, int gangs, int rows, int D) {
    return gangs == 2 ? 1.0 : prefill || D == 256 || rows > 16 ? 2.0 : 3.0;
  }
  static double token_bytes(int D) { return 2.0 * D; }
  // (two tiles of 16 rows of size 256 would not fit the registers)
  static int few(int64_t rows, int D) { return rows <= 16 || D > 128 ? 16 : 32; }
  static Estimate decode(int64_t requests, int rows, double tiles, double groups, double longest, double tokens_heads,
                         bool ragged, double shared, int most_rows, int D, int hk, int cus) {
    return estimate<Kv8Costs>(false, 1, rows, tiles, groups, longest, tokens_heads, ragged, shared, most_rows, D, hk, cus);
  }
  static bool cut(double, double, int, int) { return true; }
  static constexpr bool aim = false;
  // (the multiple of the CUs that leaves tiles half a share each to cut)
  static int64_t shares(double tiles, double groups, int D, int cus) {
    return ceil_div(3 * (int64_t)tiles, 2 * cus) * cus;
  }
  static int share_least(int rows, int D, double longest) { return rows == 32 ? 32 : D == 256 ? 8 : 16; }
};

}  // namespace

PagedPlan plan_kv8_attention(const rf_kv8_attention_args& a, int cus) {
  return plan_paged_attention<Kv8Costs>(shape_of(a), cus);
}

hipError_t launch_kv8_attention(const rf_kv8_attention_args& in, const PagedPlan& p,
                                hipStream_t stream) {
  AttnArgs a;
  fill_paged(a, in, p);
  a.ks = in.cache.k_scale;
  a.vs = in.cache.v_scale;
  const int D = in.cache.head_dim;
  const bool f16 = in.dtype == RF_W8A16_DTYPE_F16;
  if (D == 64)
    return f16 ? launch_sized<_Float16, 64>(a, p, stream) : launch_sized<__bf16, 64>(a, p, stream);
  if (D == 128)
    return f16 ? launch_sized<_Float16, 128>(a, p, stream) : launch_sized<__bf16, 128>(a, p, stream);
  return f16 ? launch_sized<_Float16, 256>(a, p, stream) : launch_sized<__bf16, 256>(a, p, stream);
}

}  // namespace rf
