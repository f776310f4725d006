// Attention over the 4-bit paged cache (kv4.h), gfx950.
//
// For query row q (one query, one head) over its seen tokens j, which hold whole
// numbers k_j, v_j, steps a_j, b_j and zero points y_j, z_j:
//   x_j = (q . k_j - y_j sum(q)) a_j scale log2(e),  p_j = 2^(x_j - m)
//   o   = sum p_j b_j (v_j - z_j) / sum p_j
// in one pass over the tokens with a running reference m.
//
// Both products run on the matrix cores with the cache as the A operand and the
// queries as columns, as over the int8 cache (kv8_attn.hip): scores leave the first
// product as the second one takes its operand.
//
// Few rows: a token's numbers meet one tile of rows or two, so as little as
// possible is done to them.  Keys: k - 8, exact in fp16 (without the 8 the products
// would have one sign, and the matrix cores' sums lose two bits more: an lse off by
// 6e-7 instead of 1e-7); what the zero point differs from 8, and the step, go into
// the scores, of which there is one for 64 or more numbers.  Values: v - z, exact
// in fp16; the step goes into the weight.
// Many rows: every number is turned into the fp16 value that it stands for (exact),
// once for 128 rows, and what is left is attention over fp16.
//
//   * Queries: fp16 as they are.  bf16 times a power of two per row, which
//     brings the row's largest magnitude to [2^14, 2^15): exact in fp16 down to
//     2^-31 of it, within 2^-39 of it below; the power goes into that row's score
//     factor.
//   * Weights p b (or p) are rounded to fp16 (11 bits, to nearest): 2^-11
//     relative, as much as the output's own rounding in fp16.  2^7 times the weight
//     is what is rounded, the row's largest so far lies in [2^7, 2^15), and what is
//     below fp16's normal range loses at most 2^-25: 2^-32 of the largest weight.
//   * m, the sums and o stay in fp32.  m is a score before its factor, and scores are
//     taken as differences from it: scores of any size keep their weights.
#include "kv4_common.h"
#include "paged_attn.h"

namespace rf {
namespace {

struct AttnArgs : PagedArgs {
  const uint16_t* rows;
};

// Nothing seen yet.  (Finite: differences from scores of -inf are not NaN.  Scores
// before their factor are sums of at most 256 products of two fp16 numbers, below 2^41.)
constexpr float kNothing = -1e30f;
constexpr float kLeastStep = -24.0f;  // log2 of less than any value step
// A row's reference as partial results hold it, in log2 units, -inf where nothing was
// seen (l = 0), and by how much the rounding moved it, as a factor of the sums.  (At
// most 2: past 2^24 scores are no more exact than that.  Scores past fp32's range are
// as its largest number.)
__device__ __forceinline__ float reference(float m, float factor, float l, float* to) {
  const float at = __builtin_amdgcn_fmed3f(m * factor, -0x1.fffffep127f, 0x1.fffffep127f);
  *to = l == 0.0f ? -__builtin_inff() : at;
  return exp2_fast(__builtin_amdgcn_fmed3f(__builtin_fmaf(m, factor, -at), -1.0f, 1.0f));
}

// (n - z) of a token pair's numbers: base - (base + z), exact in fp16.
__device__ __forceinline__ half2v less(uint32_t v, uint32_t z) { return as_half2(v) - as_half2(z); }

// ---------------------------------------------------------------------------
// Few rows (single tokens, a few drafted ones): RT tiles of 16 rows, held by
// all four or eight wavefronts; the wavefronts take 32-token groups in turn and read
// the cache straight into MFMA operands (no LDS), one turn ahead of the products.
// At the end the wavefronts' sums meet in LDS.
//
// Long contexts are bound by the cache's bytes, and by what comes before and after
// them: 130999 tokens, 32 + 8 heads of 128 (138 MB), take 29.7 us, a plain read of as
// much 23.4; 48 requests of up to 9000, 64 + 8 heads (237 MB), 51.1 and 36.6.  Short
// ones by round trips: 777 tokens take 8.5 us, of which it is 1.3 until the request
// is found, 1.2 for ids and queries, 1 a turn, 1 in LDS and, split, 4 to store, count and
// join.
//
// A product has 16 columns, and a single token of a model with four query heads to
// a key head fills four of them.  W = 2, 4: tiles of 16 / W rows, each of which has
// W columns; of the eight scores that a lane has of its row it takes N = 8 / W on,
// and the weights meet in the first of the columns.
// ---------------------------------------------------------------------------
// Loads of one group: its place in scalar registers, 32 bits of each lane.  (As
// plain pointers the addresses were summed in vector registers that loads under way
// may be writing, and waited for them.)
struct Base {
  static constexpr int kStream = 2;  // nt: read once
  __amdgpu_buffer_rsrc_t p;
  __device__ __forceinline__ Base(const void* q, int bytes)
      : p(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(q), 0, bytes, 0x00027000)) {}
  __device__ __forceinline__ uint4 stream16(int at, int more) const {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(p, at, more, kStream));
  }
  template <int kBytes>
  __device__ __forceinline__ auto load(int at, int more) const {
    if constexpr (kBytes == 4) return __builtin_amdgcn_raw_buffer_load_b32(p, at, more, 0);
    else if constexpr (kBytes == 8) return __builtin_amdgcn_raw_buffer_load_b64(p, at, more, 0);
    else return __builtin_amdgcn_raw_buffer_load_b128(p, at, more, 0);
  }
};

template <int N>
struct Words {  // of N tokens, two of 16 bits each
  typedef uint32_t vec __attribute__((ext_vector_type(N / 2)));
  vec w;
  __device__ __forceinline__ void load(const Base& b, int at, int more) {
    w = __builtin_bit_cast(vec, b.load<2 * N>(at, more));
  }
  __device__ __forceinline__ uint32_t at(int i) const { return w[i]; }
};

template <int D, int N>
struct Bytes {
  uint4 k[D / 64], v[D / 64];
  Words<N> kw, vs;  // of the tokens whose scores the lane takes on
  Words<8> vw;      // of its eight tokens
};

template <int D, int N>
__device__ __forceinline__ void fetch(const AttnArgs& a, const Group& g, int lane, Bytes<D, N>& b) {
  const int64_t group = (g.at << (a.shift - 5)) + g.sub;
  const Base k(a.k + group * (16 * D), 16 * D), v(a.v + group * (16 * D), 16 * D), rows(a.rows + group * 64, 128);
  const int first = lane / 16 * 16, mine = first + lane % 16 / (2 * N) * (2 * N);
  b.kw.load(rows, mine, 0);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) b.k[i] = k.stream16(lane * 16, i * kTileBytes);
  b.vs.load(rows, mine, 64);
  b.vw.load(rows, first, 64);
#pragma unroll
  for (int i = 0; i < D / 64; ++i) b.v[i] = v.stream16(lane * 16, i * kTileBytes);
}

// What lane n + N of a row of 16 lanes holds (0 past the row).
template <int N>
__device__ __forceinline__ uint32_t from_above(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x100 + N, 0xf, 0xf, true);
}

// op over the lanes that differ by multiples of C (4, 8 or 16), in all of them: turns of
// a row of 16, then exchanges between rows.  (Through LDS, as __shfl_xor goes, each step
// is a round trip, up to eight before the first weights: 2000 tokens, 12 heads of 64, 9.1
// us, so 8.9.)
template <int C, typename Op>
__device__ __forceinline__ float over_columns(float v, Op op) {
  const auto turned = [&](auto ctrl) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl(), 0xf, 0xf, true));
  };
  if constexpr (C <= 4) v = op(v, turned([] { return 0x124; }));  // row_ror:4
  if constexpr (C <= 8) v = op(v, turned([] { return 0x128; }));  // row_ror:8
  const auto pair = [&](auto both) {
    const uint32_t x = both[0], y = both[1];
    return op(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
  };
  uint32_t u = __builtin_bit_cast(uint32_t, v);
  v = pair(__builtin_amdgcn_permlane16_swap(u, u, false, false));
  u = __builtin_bit_cast(uint32_t, v);
  return pair(__builtin_amdgcn_permlane32_swap(u, u, false, false));
}
__device__ __forceinline__ float add(float u, float v) { return u + v; }
__device__ __forceinline__ float larger(float u, float v) { return fmaxf(u, v); }

// Eight numbers less 8, in the order of their dimensions.
__device__ __forceinline__ half8 centred8(uint32_t d) {
  constexpr uint32_t k8 = 0x64086408u, k84 = 0x54805480u;  // 1024 + 8, 64 + 8
  const uint32_t d8 = d >> 8;
  return join8(less(mask_or(d, kNibbles, kBase), k8), less(mask_or(d, kNibbles4, kBase4), k84),
               less(mask_or(d8, kNibbles, kBase), k8), less(mask_or(d8, kNibbles4, kBase4), k84));
}

// The wavefronts' sums meet in LDS, and go out or wait for those of other splits.
// (Lane numbers are made anew here: kept through the loop, what follows from them
// would take registers there.)
template <typename T, int D, int RT, int W, int NW>
__device__ __forceinline__ void finish_tile(const AttnArgs& a, const Tile& t, int h, int rows, int split, int splits,
                                            bool partial, unsigned id, const float (&m)[RT], const float (&d)[RT],
                                            const float (&factor)[RT], float (&l)[RT],
                                            const floatx4 (&acc)[RT][D / 16], float (&red)[NW][16 / W][D + 4],
                                            float (&red_m)[NW][16 / W * RT], float (&red_l)[NW][16 / W * RT]) {
  constexpr int C = 16 / W, R = C * RT, A = D / 64;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lg = lane / 16, col = lane % C, part = lane % 16 / C;
  float top_w[RT], unit[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
#pragma unroll
    for (int n = C; n < kWave; n *= 2) l[r] += __shfl_xor(l[r], n);
    unit[r] = reference(m[r], factor[r], l[r], &top_w[r]) * exp2_fast(d[r]);
    l[r] *= unit[r];
    if (lane < C) {
      red_m[wave][C * r + col] = top_w[r];
      red_l[wave][C * r + col] = l[r];
    }
  }
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    __syncthreads();
    const int rr = C * r + col;
    float top = red_m[0][rr];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, red_m[w][rr]);
    const float f = exp2_fast(top_w[r] - safe(top)) * unit[r];
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < A; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          floatx4 o;
#pragma unroll
          for (int n = 0; n < 4; ++n) o[n] = acc[r][4 * i + n][j] * f;
          *reinterpret_cast<floatx4*>(&red[wave][col][64 * i + 16 * lg + 4 * j]) = o;
        }
    }
    __syncthreads();
    for (int it = tid; it < C * (D / 4); it += NW * kWave) {
      const int c = it / (D / 4), d = it % (D / 4) * 4, rc = C * r + c;
      if (rc >= rows) continue;
      float mm = red_m[0][rc];
#pragma unroll
      for (int w = 1; w < NW; ++w) mm = fmaxf(mm, red_m[w][rc]);
      float ll = 0.0f;
      floatx4 o = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        ll += red_l[w][rc] * exp2_fast(red_m[w][rc] - safe(mm));
        o += *reinterpret_cast<const floatx4*>(&red[w][c][d]);
      }
      const int64_t to = out_row(a, t, h, rc);
      if (partial) {
        const Partials parts(a);
        const int i = a.merge ? (int)to * a.splits + split : (int)id * R + rc;
        parts.store(i * D + d, o);
        if (d == 0) parts.store_stat(i, mm, ll);
      } else {
        finish<T>(a, to, D, d, o, mm, ll);
      }
    }
  }
  if (partial && !a.merge)
    join<T, D, R, NW * kWave>(a, t, h, rows, splits, ((int)id - split * a.hk) * R, a.hk * R,
               a.counters + (id - (unsigned)(split * a.hk)), &red[0][0][0]);
}

template <typename T, int D, int RT, int W, int NW>
__global__ __launch_bounds__(NW* kWave)
__attribute__((amdgpu_waves_per_eu(D <= 128 && RT == 1 ? 3 : 2))) void kv4_decode_kernel(AttnArgs a) {
  static_assert(RT == 1 || W == 1);
  constexpr int C = 16 / W, N = 8 / W, R = C * RT, A = D / 64, kAhead = 1;
  // (join() wants room for the splits' numbers)
  constexpr int kRed = NW * C * (D + 4), kJoin = R * 64 * 2 + NW * kWave * 4;
  __shared__ __align__(16) float lds[kRed > kJoin ? kRed : kJoin];
  float(&red)[NW][C][D + 4] = *reinterpret_cast<float(*)[NW][C][D + 4]>(&lds);
  __shared__ float red_m[NW][R], red_l[NW][R];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lg = lane / 16, col = lane % C, part = lane % 16 / C;
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

  // ---- queries, as B operands: column = row, dimensions 64 i + 16 lg + 8 j + ..
  uint4 raw[RT][2 * A];
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int row = t.row0 + min(C * r + col, rows - 1);
    const int qi = (int)((unsigned)row / (unsigned)a.group);
    const uint8_t* p = a.q + (int64_t)(t.first_token + qi) * a.q_ts +
                       (int64_t)(h * a.group + (row - qi * a.group)) * a.q_hs + lg * 32;
#pragma unroll
    for (int i = 0; i < 2 * A; ++i) raw[r][i] = load_u4(p + (i / 2) * 128 + (i % 2) * 16);
  }

  // The bytes of kAhead turns are under way while one is worked on, and the block
  // ids of the turn after them.  The first go out before the queries are looked at.
  const auto id_of = [&](int g) { return group_of(a, t, h, min(g, end - 1)); };
  constexpr int kBufs = kAhead + 1;
  int g = begin + wave, to = g + kAhead * NW;
  Bytes<D, N> b[kBufs];
  bool ok[kBufs];
  Group next;
  if (g < end) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const Group x = id_of(g + i * NW);
      ok[i] = x.ok;
      fetch(a, x, lane, b[i]);
      __builtin_amdgcn_sched_barrier(0);  // (in this order: what is waited for is counted back)
    }
    next = id_of(to);
  }

  half8 q[RT][2 * A];
  float factor[RT], qsum[RT];  // qsum: -sum(q)
  int pos[RT];                 // of the row's query
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    factor[r] = a.scale_log2e;
    if constexpr (!__is_same(T, _Float16)) {
      float m = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * A; ++i) m = load_amax<T>(raw[r][i], m);
      m = over_columns<16>(m, larger);
      const int e = row_exponent(m), e1 = e / 2, e2 = e - e1;
      const float f1 = pow2(-e1), f2 = pow2(-e2);
#pragma unroll
      for (int i = 0; i < 2 * A; ++i)
        q[r][i] = __builtin_convertvector(Eight<T>::load(&raw[r][i]) * f1 * f2, half8);
      factor[r] = a.scale_log2e * pow2(e1) * pow2(e2);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * A; ++i) q[r][i] = as_half8(raw[r][i]);
    }
    factor[r] = in_range(factor[r]);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * A; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += (float)q[r][i][j];
    qsum[r] = -over_columns<16>(sum, add);
    pos[r] = t.kv_len - t.queries + (int)((unsigned)(t.row0 + min(C * r + col, rows - 1)) / (unsigned)a.group);
  }
  floatx4 acc[RT][4 * A];
  // Weights are relative to 2^(m factor + d): m is the row's largest score, before its
  // factor, when it was last raised, d what the largest of the scores with log2 of their
  // value steps had above that (-24 to 13).  Scores count by their difference from m,
  // which is right for any size of them; m factor, rounded, would be off by more than a
  // weight's range from 2^28 on.
  float m[RT], d[RT], l[RT];  // l: each lane's own share of the sum
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    m[r] = kNothing;
    d[r] = kLeastStep;
    l[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * A; ++i) acc[r][i] = floatx4{0, 0, 0, 0};
  }

  const auto step = [&](const Bytes<D, N>& b, int g, bool ok) {
    floatx4 all[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) all[r][0] = all[r][1] = floatx4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < A; ++i) {
      const uint32_t d[4] = {b.k[i].x, b.k[i].y, b.k[i].z, b.k[i].w};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const half8 k = centred8(d[w]);
#pragma unroll
        for (int r = 0; r < RT; ++r) all[r][w / 2] = mfma16x16x32(k, q[r][2 * i + w % 2], all[r][w / 2]);
      }
    }
    half2v ks[(N + 1) / 2], kz[(N + 1) / 2], vs[(N + 1) / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      ks[i] = as_half2(b.kw.at(i) & kStepBits);
      kz[i] = less(mask_or(b.kw.at(i), kNibbles, kBase), 0x64086408u);  // less 8
      vs[i] = as_half2(b.vs.at(i) & kStepBits);
    }
    const int t0 = opaque(g << 5);
    const bool edge = t0 < lo_max || t0 + 32 > hi_min;
    float s[RT][N];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x = all[r][i / 4][i % 4];
#pragma unroll
        for (int n = 1; n < W; ++n) x = part == n ? all[r][(n * N + i) / 4][(n * N + i) % 4] : x;
        x = __builtin_fmaf((float)kz[i / 2][i % 2], qsum[r], x);
        s[r][i] = __builtin_fmaf((float)ks[i / 2][i % 2], x, 0.0f);
      }
      if (!ok) {
        keep_branch();
#pragma unroll
        for (int i = 0; i < N; ++i) s[r][i] = __builtin_nanf("");
      }
      if (edge) {
        keep_branch();
        const int at = t0 + 8 * lg + N * part;
        const int first = a.window > 0 ? pos[r] - a.window + 1 - at : -at, past = (a.causal ? pos[r] + 1 : t.kv_len) - at;
#pragma unroll
        for (int i = 0; i < N; ++i) s[r][i] = ((i < first) | (i >= past)) ? -__builtin_inff() : s[r][i];
      }
    }
    typedef _Float16 halfN __attribute__((ext_vector_type(N)));
    halfN mine[RT];
    float sum[RT];
    bool raise = false;
    const auto weights = [&](int r) {  // the largest of them
      const float off = kShift - d[r];
      float most = 0.0f;
      sum[r] = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float e = exp2_fast(__builtin_fmaf(minus(s[r][i], m[r]), factor[r], off));
        const float w = __builtin_fmaf((float)vs[i / 2][i % 2], e, 0.0f);
        sum[r] += e;
        most = fmaxf(most, w);
        mine[r][i] = (_Float16)w;
      }
      return most;
    };
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float most = weights(r);
      raise |= most > 32768.0f || sum[r] == __builtin_inff();
    }
    if (__ballot(raise)) {
      keep_branch();
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        float top = m[r];
#pragma unroll
        for (int i = 0; i < N; ++i) top = fmaxf(top, s[r][i]);
        top = over_columns<C>(top, larger);
        const float fall = (m[r] - top) * factor[r];
        float above = d[r] + fall;
#pragma unroll
        for (int i = 0; i < N; ++i)
          above = fmaxf(above, __builtin_fmaf(minus(s[r][i], top), factor[r],
                                              log2_fast(fmaxf((float)vs[i / 2][i % 2], 0x1p-24f))));
        above = over_columns<C>(above, larger);
        const float f = exp2_fast(fall + (d[r] - above));
        m[r] = top;
        d[r] = above;
        l[r] *= f;
#pragma unroll
        for (int i = 0; i < 4 * A; ++i) acc[r][i] *= f;
        weights(r);
      }
    }
    half8 p[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      l[r] += sum[r];
      if constexpr (W == 1) {
        p[r] = mine[r];
      } else if constexpr (W == 2) {
        const uint2 u = __builtin_bit_cast(uint2, mine[r]);
        p[r] = as_half8(make_uint4(u.x, u.y, from_above<C>(u.x), from_above<C>(u.y)));
      } else {
        const uint32_t u = __builtin_bit_cast(uint32_t, mine[r]);
        p[r] = as_half8(make_uint4(u, from_above<C>(u), from_above<2 * C>(u), from_above<3 * C>(u)));
      }
    }
    const uint32_t vw[4] = {b.vw.at(0), b.vw.at(1), b.vw.at(2), b.vw.at(3)};
    uint32_t z[4], z4[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[i] = mask_or(vw[i], kNibbles, kBase);
      z4[i] = mask_or(vw[i] << 4, kNibbles4, kBase4);
    }
#pragma unroll
    for (int i = 0; i < A; ++i) {
      const uint32_t d[4] = {b.v[i].x, b.v[i].y, b.v[i].z, b.v[i].w};
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        half2v v[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t x = n < 2 ? d[w] : d[w] >> 8;
          v[w] = n % 2 ? less(mask_or(x, kNibbles4, kBase4), z4[w]) : less(mask_or(x, kNibbles, kBase), z[w]);
        }
        const half8 v8 = join8(v[0], v[1], v[2], v[3]);
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[r][4 * i + n] = mfma16x16x32(v8, p[r], acc[r][4 * i + n]);
      }
    }
  };

  if (g < end) {
    const auto turn = [&](int now) {
      const int last = (now + kAhead) % kBufs;
      ok[last] = next.ok;
      fetch(a, next, lane, b[last]);
      to += NW;
      next = id_of(to);
      // (they go out before anything of this turn waits for its own)
      __builtin_amdgcn_sched_barrier(0);
      step(b[now], g, ok[now]);
      g += NW;
      return g < end;
    };
    while (turn(0) && turn(1)) {}
  }

  // ---- the wavefronts' results
  finish_tile<T, D, RT, W, NW>(a, t, h, rows, split, share.splits, partial, id, m, d, factor, l, acc, red, red_m,
                               red_l);
}

// ---------------------------------------------------------------------------
// Many rows (prompts): four wavefronts of 32 rows each.  A step's numbers are
// loaded once per workgroup, turned into the fp16 values that they stand for on
// their way into LDS, in operand order (a wavefront reads 1 KB in lane order per
// MFMA), and those of the next two steps are loaded meanwhile.  G = 2: two gangs
// of four wavefronts take the steps of the same rows in turn, and their sums join
// at the end: what the longest tile takes is halved, which is what a prompt takes
// that does not fill the chip several times (1000 tokens, 32 + 8 heads of 128: 33.3 us,
// two gangs 26.8; 7999 tokens, 64 + 8 heads: 1145, and 916 TFLOP/s with one).  Bound by
// the vector instructions beside the products, at the power's clock: matrix units 44%
// busy, vector units 67% (over int8 45% and 63%).
// ---------------------------------------------------------------------------
template <typename T, int D, int G>
__global__ __launch_bounds__(G* kWaves* kWave)
__attribute__((amdgpu_waves_per_eu(2))) void kv4_prefill_kernel(AttnArgs a) {
  constexpr int R = 32 * kWaves, A = D / 64;
  constexpr int NG = D <= 128 ? 2 : 1;          // 32-token groups of a step
  constexpr int kBuf = NG * 32 * D * 2 * 2;     // bytes of a step's K and V in fp16
  // A step has NG * A tiles of keys and as many of values: one of each per
  // wavefront, or, of size 64, one of either.
  constexpr bool kBoth = NG * A == kWaves;
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
  float m = kNothing, l = 0.0f;  // weights are relative to 2^(m factor)
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.0f;

  // A step's bytes and words are loaded two steps ahead (a short share is bound
  // by their round trip), its block ids three.
  const int g16 = lane / 16, l16 = lane % 16;
  const int tile = kBoth ? wave : wave % (kWaves / 2), my_group = tile / A, my_tile = tile % A;
  const bool my_k = kBoth || wave < kWaves / 2, my_v = kBoth || wave >= kWaves / 2;
  struct Ahead {
    uint4 k, v, vw;
    uint32_t kw;  // words of the lane's two tokens
    bool ok[NG];
  };
  Group ids[NG];
  const auto look = [&](int g) {
#pragma unroll
    for (int n = 0; n < NG; ++n) ids[n] = group_of(a, t, h, min(g + n, end - 1));
  };
  const auto load = [&](Ahead& x) {
    const Group& gr = NG == 1 || my_group == 0 ? ids[0] : ids[NG - 1];
    const int64_t group = (gr.at << (a.shift - 5)) + gr.sub;
    const int64_t at = group * (16 * D) + my_tile * kTileBytes + lane * 16;
    const uint16_t* rp = a.rows + group * 64;
    if (my_k) {
      const int token = l16 / 4 * 8 + l16 % 4;
      x.k = load_u4(a.k + at);
      x.kw = rp[token] | (uint32_t)rp[token + 4] << 16;
    }
    if (my_v) {
      x.v = load_u4(a.v + at);
      x.vw = load_u4(rp + 32 + g16 * 8);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) x.ok[n] = ids[n].ok;
  };
  // Element e of a value operand is token 16 u + 8 lh + e, so the first product's
  // rows are in the order 16 u + 8 x + 4 lh + c for token 16 u + 8 lh + 4 x + c.  A
  // 32-dimension tile of values holds dimension 4 c + b in row 8 b + c.
  const auto stage = [&](uint8_t* buf, const Ahead& x) {
    if (my_k) {
      const uint32_t d[4] = {x.k.x, x.k.y, x.k.z, x.k.w};
#pragma unroll
      for (int tt = 0; tt < 2; ++tt) {
        const uint32_t w = __builtin_amdgcn_perm(x.kw, x.kw, tt ? 0x03020302u : 0x01000100u);
        const half2v s = as_half2(w & kStepBits);
        const uint32_t z = mask_or(w, kNibbles, kBase), z4 = mask_or(w << 4, kNibbles4, kBase4);
        const int row = 16 * (l16 / 8) + 8 * tt + 4 * (l16 / 4 % 2) + l16 % 4;
        uint8_t* p = buf + ((my_group * (D / 16) + my_tile * 4 + g16) * kWave + row) * 16;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t u = d[2 * tt + j], u8 = u >> 8;
          *reinterpret_cast<half8*>(p + j * 32 * 16) =
              join8(less(mask_or(u, kNibbles, kBase), z) * s, less(mask_or(u, kNibbles4, kBase4), z4) * s,
                    less(mask_or(u8, kNibbles, kBase), z) * s, less(mask_or(u8, kNibbles4, kBase4), z4) * s);
        }
      }
    }
    if (my_v) {
      const uint32_t d[4] = {x.v.x, x.v.y, x.v.z, x.v.w}, w[4] = {x.vw.x, x.vw.y, x.vw.z, x.vw.w};
      uint8_t* p = buf + kBuf / 2 + (((my_group * (D / 32) + my_tile * 2 + l16 / 8) * 2 + g16 / 2) * kWave +
                                     (g16 % 2) * 32 + l16 % 8) * 16;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        half2v v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t u = n < 2 ? d[i] : d[i] >> 8;
          const half2v s = as_half2(w[i] & kStepBits);
          v[i] = n % 2 ? less(mask_or(u, kNibbles4, kBase4), mask_or(w[i] << 4, kNibbles4, kBase4)) * s
                       : less(mask_or(u, kNibbles, kBase), mask_or(w[i], kNibbles, kBase)) * s;
        }
        *reinterpret_cast<half8*>(p + n * 8 * 16) = join8(v[0], v[1], v[2], v[3]);
      }
    }
  };
  // One step of a wavefront: all of its scores, one look at their maximum, then
  // the weights.  The products of a group with V are issued among the weights of
  // the next group, the last ones among the conversion of the next step's bytes:
  // those take the vector units, these the matrix units.  A wavefront's priority
  // rises through the step, so that of two that share a SIMD the one ahead stays
  // ahead and they are in different phases.
  const auto step = [&](const uint8_t* buf, int g, const bool (&ok)[NG], uint8_t* out, const Ahead& next) {
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
#pragma unroll
    for (int n = 0; n < NG; ++n)
      if (!ok[n]) {
        keep_branch();
        s[n] = __builtin_nanf("");
      }
    if (t0 < my_lo_max || t0 + 32 * NG > my_hi_min) {
      keep_branch();
      const int first = lo - t0 - 8 * lh, past = hi - t0 - 8 * lh;
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int tok = 32 * n + 16 * (i / 8) + i % 8;  // past t0 + 8 lh
          s[n][i] = ((tok < first) | (tok >= past)) ? -__builtin_inff() : s[n][i];
        }
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
    if (__ballot(minus(mx, m) * factor > kRaise)) {
      const float top = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32))), f = exp2_fast((m - top) * factor);
      m = top;
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] *= f;
    }
    // (a value the compiler cannot fold into the branch above: merged with it, it
    // would keep the sums twice, and spill)
    float off = 0.0f;
    if (opaque(t0) >= 0) {  // (always: a block of its own)
      off = __builtin_fmaf(-m, factor, kShift);
      asm volatile("" : "+v"(off));
    }
    // Scores of ordinary size take one instruction for their difference from m.  Of
    // large ones both terms are rounded, from 2^22 on to more than the fp16 weights have
    // room for: first the difference, then the factor.
    if (__ballot(fabsf(off) > kFar)) {
      keep_branch();
#pragma unroll
      for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = minus(s[n][i], m);
      off = kShift;
    }
    half8 p[2];
    const auto weights = [&](int n) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = exp2_fast(__builtin_fmaf(s[n][i], factor, off));
        sum += e;
        p[i / 8][i % 8] = (_Float16)e;
      }
      l += sum;
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
      bool ok[NG];
#pragma unroll
      for (int n = 0; n < NG; ++n) ok[n] = now.ok[n];
      load(now);
      look(g + 3 * kStride);
      step(in, g, ok, out, next);
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
    if (gang == 1) {
#pragma unroll
      for (int i = 0; i < D / 2; ++i) sums[i * kWave] = acc[i / 16][i % 16];
      stats[0] = m;
      stats[kWave] = l;
    }
    __syncthreads();
    if (gang == 0) {
      const float om = stats[0], top = fmaxf(m, om);
      const float f = exp2_fast((m - top) * factor), of = exp2_fast((om - top) * factor);
#pragma unroll
      for (int i = 0; i < D / 2; ++i) acc[i / 16][i % 16] = acc[i / 16][i % 16] * f + sums[i * kWave] * of;
      m = top;
      l = l * f + stats[kWave] * of;
    }
    __syncthreads();  // the rows go out through the same memory
    if (gang == 1) return;
  }

  // Rows go out through LDS (each wavefront its own part, free after the last
  // barrier), 64 dimensions at a time: straight from the registers every lane
  // would store four values of another row.
  constexpr int kPitch = 64 + 4;
  float* mine = reinterpret_cast<float*>(lds) + wave * 32 * kPitch;
  l += __shfl_xor(l, 32);
  const int left = rows - wrow;  // rows of this wavefront's tile
  float top_w;
  const float unit = reference(m, factor, l, &top_w), f = partial ? unit : l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int i = 0; i < D / 32; i += 2) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {  // dimensions 32 (j / 4) + 16 lh + 4 (j % 4) + ..
      floatx4 o;
#pragma unroll
      for (int b = 0; b < 4; ++b) o[b] = acc[i + j / 4][4 * b + j % 4] * f;
      *reinterpret_cast<floatx4*>(mine + col * kPitch + 32 * (j / 4) + 16 * lh + 4 * (j % 4)) = o;
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
    if (partial) Partials(a).store_stat((int)to * a.splits + split, top_w, l * unit);
    else if (a.lse)
      a.lse[to] = l == 0.0f ? -__builtin_inff() : __builtin_fmaf(m, factor, log2_fast(l) - kShift) * kLn2;
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
    if (p.kernel == 1 && p.gangs == 1) kv4_prefill_kernel<T, D, 1><<<grid, kThreads, kLds, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 4 && p.gangs == 2) kv4_decode_kernel<T, D, 1, 4, 8><<<grid, 512, 0, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 8 && p.gangs == 2) kv4_decode_kernel<T, D, 1, 2, 8><<<grid, 512, 0, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 4 && p.gangs == 1) kv4_decode_kernel<T, D, 1, 4, 4><<<grid, kThreads, 0, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 8 && p.gangs == 1) kv4_decode_kernel<T, D, 1, 2, 4><<<grid, kThreads, 0, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 16 && p.gangs == 1) kv4_decode_kernel<T, D, 1, 1, 4><<<grid, kThreads, 0, stream>>>(a);
    else if constexpr (D <= 128) {
      if (p.kernel == 1 && p.gangs == 2) kv4_prefill_kernel<T, D, 2><<<grid, 2 * kThreads, kLds2, stream>>>(a);
      else if (p.kernel == 0 && p.rows == 32 && p.gangs == 1) kv4_decode_kernel<T, D, 2, 1, 4><<<grid, kThreads, 0, stream>>>(a);
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

struct Kv4Costs {
  // (of the kernel for many rows alone: the one for few has an estimate of its own)
  static double base(bool, int, int D) { return D == 64 ? 1.1 : D == 128 ? 1.5 : 1.35; }
  static double more(bool, int, int D) { return D == 256 ? 0.6 : 0.4; }
  static double slots(bool, int gangs, int, int) { return gangs == 2 ? 1.0 : 2.0; }
  static double token_bytes(int D) { return D + 4.0; }
  static int few(int64_t rows, int D) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 || D > 128 ? 16 : 32; }
  // Tiles are not cut where they are short, or so many that the CUs have others to go on
  // with (200 requests of up to 1000 tokens, 64 + 8 heads: 32 us, cut 41; 128 of up to
  // 8000 105.8 and 107.6; 48 of those 62.1 and 46.5; 12 heads of 64, 128 of up to 2000: 29.1
  // and 34.5; 64 of up to 4000 31.9 and 30.2; 8 + 1 heads of 256, 400 of up to 2000: 33.5
  // and 47.5; 128 of those 23.0 and 18.2).
  static bool cut(double tiles, double longest, int D, int cus) {
    return longest > 33 && tiles < cus * (D == 64 ? 4.0 : D == 128 ? 2.0 : 1.5);
  }
  // The decode kernel, with four or eight wavefronts a workgroup, fitted to 1 x 100 to
  // 131000 tokens of four head layouts at 1 to 64 splits on either: us of a turn, of what
  // surrounds the turns, and of the join, which one workgroup does for a tile (32 rows
  // of 128, 8 and 32 splits of 4000 tokens: 20.8 and 27 us, with the second kernel 13.9 and
  // 14; 4 rows, 8 splits of 777: 8.6 and 8.2, but 9.4 and 11.8 for a caller that launches
  // them itself: a call of one launch takes the host 8.7 us, one of two 11.7).
  // Eight wavefronts halve the splits of long contexts (131000 tokens, 32 + 8 heads: 64
  // splits of four 31.3 us, 32 of eight 29.5; 60000 tokens, 8 + 1 heads of 256: 27.5 and
  // 22.7) and do without any in middling ones (777 tokens, 12 heads of 64: 7.5 and 6.8).
  static Estimate decode(int64_t requests, int rows, double tiles, double groups, double longest, double tokens_heads,
                         bool ragged, double shared, int most_rows, int D, int hk, int cus) {
    const int held = rows < most_rows ? rows : most_rows, cap = most_splits(rows);
    constexpr double kOneLaunch = 8.5, kTwoLaunches = 11.5;
    const bool whole = requests > 1 && !cut(tiles * hk, longest, D, cus);
    Estimate best{1e30, 1, false};
    double least = 1e30;
    for (int gangs = 1; gangs <= (rows <= 8 && requests == 1 ? 2 : 1); ++gangs) {
      const double compute = rows <= 8 ? 1.0 : rows == 16 ? 1.15 : 1.65;
      const double turn = compute * (D == 64 ? (gangs == 1 ? 0.43 : 0.63) : D == 128 ? (gangs == 1 ? 0.61 : 0.94)
                                                                                     : (gangs == 1 ? 1.02 : 1.66));
      const int slots = rows == 32 ? 2 : gangs == 1 ? (D == 64 ? 4 : D == 128 ? 3 : 2) : (D == 64 ? 2 : 1);
      for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
        if (s > cap || (s > 1 && (s > groups || whole))) break;
        const double turns = ceil(ceil(groups / s) / (kWaves * gangs)), w = tiles * hk * s;
        const auto round = [&](double n) {  // n workgroups at a time
          // (the CUs share the memory evenly, so those with a workgroup more are the last: 131000
          // tokens, 12 heads of 64, 24 splits of eight wavefronts 34 us, 64 of four 28)
          const double as_if = rows <= 8 && n > cus ? ceil(n / cus) * cus : n;
          const double bytes = as_if * kWaves * gangs * 32.0 * token_bytes(D) * shared / (gangs == 1 ? 6.5e6 : 7.0e6);
          const double beside = turn * (1.0 + 0.3 * (n > cus ? n / cus - 1.0 : 0.0));
          return turns * (beside > bytes ? beside : bytes);
        };
        const double room = (double)cus * slots, full = floor(w / room), rest = w - full * room;
        double us = 4.2 + 0.5 * gangs + full * round(room) + (rest >= 1 ? round(rest) : 0.0) + 1.5 * (ceil(w / room) - 1.0);
        // (workgroups that start together hold each other up: 8000 tokens, 32 + 8 heads, 16 and
        // 32 splits 11.1 and 12.2 us, 12 heads of 64 10.9 and 12.9)
        if (rows <= 8) us += 2.2 * (w < 2 * cus ? w / cus : 2.0);
        // (prompts: the kernel for many rows has its say; 13, 19 and 49 shapes of heads of 256,
        // 64 and 128 within 0.76 to 1.17 of it)
        const double tile = D == 64 ? 1.2 + 0.73 * turns : D == 128 ? 2.3 + 0.9 * turns : 2.9 + 1.05 * turns;
        const double many = (D == 64 ? 6.1 : D == 128 ? 7.9 : 7.1) + w / cus * tile;
        if (most_rows > 16 && w > cus && us < many) us = many;
        bool merge = false;
        if (s > 1) {
          const double x = held * D / 512.0;
          const double join = rows <= 8 ? (gangs == 1 && D <= 128 ? 2.0 : 3.1) + 0.2 * x + (0.03 + 0.028 * x) * s * (gangs == 2 ? 0.42 : 1.0)
                                        : 2.2 + 0.08 * s + x * (0.7 + 0.037 * s);
          const double second = 2.9 + 0.09 * s + tokens_heads * s * D * 8.0 / 3e6;
          // (a caller that does not replay graphs pays for the second launch)
          merge = (second < join && us + join > kTwoLaunches) || tiles * hk > kMaxSplitCounters;
          us += merge ? second : join;
        }
        const double host = merge ? kTwoLaunches : kOneLaunch, call = us > host ? us : host;
        if (call + 0.1 * us < least) least = call + 0.1 * us, best = {call, s, merge, gangs};
      }
    }
    return best;
  }
  // (48 requests of up to 9000 tokens, 64 + 8 heads: 776 workgroups, four on eight of the
  // CUs and three on the others, take 60 us, 768 of them 52)
  static constexpr bool aim = true;
  // Workgroups of a batch, a multiple of the CUs: those that a CU runs at a time where
  // they get enough to do (16 requests of up to 15000 tokens, 32 + 8 heads, 1, 2, 3 and
  // 4 a CU: 38.2, 31.6, 32.3, 36.3 us; of 15000 each 52.2, 51.9, 49.5, 54.7; of 4000 each
  // 20.5, 19.9, 20.3, 24.4; 12 heads of 64, of 15000: 64.0, 47.5, 40.7, 41.8; 8 + 1 heads of
  // 256: 22.0, 27.0, 37.4, 40.1), and room for the tiles to be cut.
  static int64_t shares(double tiles, double groups, int D, int cus) {  // of all heads
    const double most = D == 256 ? 1 : D == 64 || tiles * groups > 3 * 45.0 * cus ? 3 : 2;
    const double room = ceil(1.5 * tiles / cus);
    return (int64_t)(room > most ? room : most) * cus;
  }
  // (4 requests of up to 2000 tokens, 32 + 8 heads, 8, 12, 16 and 24 groups: 10.0, 10.4, 10.9,
  // 12.0 us; 16 of those 12.4, 12.2, 13.0, 12.3; 8 + 1 heads of 256, 16 of up to 2000: 13.2,
  // 14.2, 15.1, 16.9)
  static int share_least(int rows, int D, double) { return rows == 32 ? 16 : D == 256 ? 8 : 12; }
};

}  // namespace

PagedPlan plan_kv4_attention(const rf_kv4_attention_args& a, int cus) {
  return plan_paged_attention<Kv4Costs>(shape_of(a), cus);
}

hipError_t launch_kv4_attention(const rf_kv4_attention_args& in, const PagedPlan& p, hipStream_t stream) {
  AttnArgs a;
  fill_paged(a, in, p);
  a.rows = in.cache.rows;
  const int D = in.cache.head_dim;
  const bool f16 = in.dtype == RF_W8A16_DTYPE_F16;
  if (D == 64)
    return f16 ? launch_sized<_Float16, 64>(a, p, stream) : launch_sized<__bf16, 64>(a, p, stream);
  if (D == 128)
    return f16 ? launch_sized<_Float16, 128>(a, p, stream) : launch_sized<__bf16, 128>(a, p, stream);
  return f16 ? launch_sized<_Float16, 256>(a, p, stream) : launch_sized<__bf16, 256>(a, p, stream);
}

}  // namespace rf
