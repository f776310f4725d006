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
#include <math.h>

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
  uint32_t* counters;  // one per tile and key head, at most, zero between launches
  float* part;         // unnormalized, [tokens * heads][splits][D], or [workgroups][R][D]
  uint64_t* stat;      // m, l, likewise
  int64_t table_stride;
  int num_blocks;
  int tokens, requests, width, hq, hk, group, shift;
  int per_request;     // cu == nullptr: queries of a request
  int splits, least, tiles;
  unsigned first;      // workgroup that the launch begins at
  int shares;          // find_share: of all tiles together (0: not used)
  bool merge;          // partial results are added by kv8_merge_kernel, else by join()
  int causal, window;  // window 0: none
  float scale_log2e;
};

// Where a workgroup works.  Rows (query * group + head of the group), tokens
// and positions fit 32 bits (checked on the host).
struct Tile {
  int first_token, queries;  // of the request
  int row0;                  // first row of the tile
  int kv_len;
  const int32_t* table;
};

// A value that is the same in all lanes, in a scalar register: the compiler
// does not see it through the loads and searches below, and would carry every
// bound, id and branch of the loops per lane (the builtin it folds away where
// it knows the value uniform but has it in a vector register).  The wait states
// are the ones the compiler keeps around its own instruction but cannot know
// of here: the vector register may be written by the instruction before it,
// and the scalar one be a load's address in the one after.
__device__ __forceinline__ int uniform(int v) {
  int r;
  asm("s_nop 1\n\tv_readfirstlane_b32 %0, %1\n\ts_nop 4" : "=s"(r) : "v"(v));
  return r;
}
// The same for a value that is in one: not to be merged with per-lane counters.
__device__ __forceinline__ int opaque(int v) {
  asm("" : "+s"(v));
  return v;
}
// Ids, lengths and scales are read only, at uniform addresses: scalar loads,
// which do not queue behind the cache's bytes.
template <typename T>
__device__ __forceinline__ T read_scalar(const T* p, int64_t i) {
  return reinterpret_cast<const __attribute__((address_space(4))) T*>(reinterpret_cast<uintptr_t>(p))[i];
}

__device__ __forceinline__ int cu_at(const AttnArgs& a, int b) {
  if (b <= 0) return 0;
  if (b > a.requests) return a.tokens;
  return min(max(a.cu[b], 0), a.tokens);
}

// Tile x of the launch: request b's tiles begin at floor(cu[b] group / R) + b,
// which leaves room for all of them.  Each lane looks at one boundary (and up
// to 62 requests at their lengths too: one memory round trip); more requests
// take a round per factor of 64.
template <int R>
__device__ __forceinline__ bool find_tile(const AttnArgs& a, int x, Tile* t) {
  int b, len;
  if (a.cu == nullptr) {
    const int per = (a.per_request * a.group + R - 1) / R;
    b = (int)((unsigned)x / (unsigned)per);
    if (b >= a.requests) return false;
    t->first_token = b * a.per_request;
    t->queries = a.per_request;
    t->row0 = (x - b * per) * R;
    len = a.lens[b];
  } else {
    const int lane = threadIdx.x % kWave;
    const auto begin = [&](int c, int i) { return (int)((int64_t)c * a.group / R) + i; };
    int first, next;
    if (a.requests < kWave - 1) {
      const int c = cu_at(a, lane);
      const int n = lane < a.requests ? a.lens[lane] : 0;
      const int hits = __popcll(__ballot(lane <= a.requests && begin(c, lane) <= x));
      b = hits - 1;
      first = __builtin_amdgcn_readlane(c, b);
      next = __builtin_amdgcn_readlane(c, b + 1);
      len = __builtin_amdgcn_readlane(n, b);
    } else {
      int lo = 0, n = a.requests + 1;  // the answer is in [lo, lo + n)
      while (n > 1) {
        const int step = (n + kWave - 1) / kWave, at = lo + lane * step;
        const bool below = at < lo + n && begin(cu_at(a, at), at) <= x;
        const int hits = __popcll(__ballot(below));
        const int base = lo + (hits > 0 ? hits - 1 : 0) * step;
        n = min(step, lo + n - base);
        lo = base;
      }
      b = __builtin_amdgcn_readfirstlane(lo);
      first = cu_at(a, b);
      next = cu_at(a, b + 1);
      len = b < a.requests ? a.lens[b] : 0;
    }
    t->first_token = first;
    t->queries = max(next - first, 0);
    t->row0 = (x - begin(first, b)) * R;
  }
  if (t->row0 < 0 || t->row0 >= t->queries * a.group) return false;
  // (b == requests: the tokens past the batch, which see nothing)
  b = uniform(b);
  t->first_token = uniform(t->first_token);
  t->queries = uniform(t->queries);
  t->row0 = uniform(t->row0);
  t->kv_len = uniform(min(max(len, 0), a.width << a.shift));
  t->table = a.table + (b < a.requests ? b * a.table_stride : 0);
  return true;
}

// Sums and maxima over the lanes up to each one.
template <typename Op>
__device__ __forceinline__ int scan(int v, Op op) {  // op(v, 0) == v
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr:1
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));  // row_shr:2
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));  // row_shr:4
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));  // row_shr:8
  v = op(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));  // row_bcast:15
  return op(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));  // row_bcast:31
}

// Tokens [lo, hi) that row `row` of a request sees.
__device__ __forceinline__ void seen(const AttnArgs& a, const Tile& t, int row, int* lo, int* hi) {
  *lo = 0;
  *hi = t.kv_len;
  if (a.causal) {
    const int pos = t.kv_len - t.queries + (int)((unsigned)row / (unsigned)a.group);
    *hi = max(pos + 1, 0);
    if (a.window > 0) *lo = max(pos - a.window + 1, 0);
  }
}

// Split `split` of tile `tile` as workgroup x of a batch of unequal lengths
// finds it.  Every tile is cut into shares of at most L groups, with the
// smallest L that leaves no more than `shares` of them: a batch takes as long as
// its mean, not as its longest request, and its workgroups fill the CUs evenly.
// Each lane holds ceil(requests / 64) requests, so up to 64 of them cost one
// memory round trip; for more, L is a bound that needs no search.
template <int R>
__device__ __forceinline__ bool find_share(const AttnArgs& a, int x, Tile* t, int* split, int* splits) {
  struct Entry {
    int first, queries, tiles, len, n;  // n: groups that its last tile sees
  };
  const int lane = threadIdx.x % kWave, entries = a.requests + (a.cu ? 1 : 0);
  const int per = (int)((unsigned)(entries + kWave - 1) / kWave);
  const auto entry = [&](int b) {  // (b == requests: the tokens past the batch, which see nothing)
    Entry e;
    e.len = b < a.requests ? min(max(a.lens[b], 0), a.width << a.shift) : 0;
    e.first = a.cu ? cu_at(a, b) : b * a.per_request;
    e.queries = b >= entries ? 0 : a.cu ? max(cu_at(a, b + 1) - e.first, 0) : a.per_request;
    e.tiles = (int)(((unsigned)(e.queries * a.group) + R - 1) / R);
    int lo = 0;
    if (a.causal && a.window > 0) {
      const int query = (int)((unsigned)(max(e.tiles - 1, 0) * R) / (unsigned)a.group);
      lo = max(e.len - e.queries + query - a.window + 1, 0);
    }
    e.n = max(((e.len + 31) >> 5) - (lo >> 5), 0);
    return e;
  };
  const auto add = [](int u, int v) { return u + v; };
  const auto most = [](int u, int v) { return max(u, v); };
  Entry e;
  int work = 0, longest = 0, tiles = 0;
  for (int j = 0; j < per; ++j) {
    e = entry(lane * per + j);
    work += e.tiles * e.n;
    longest = max(longest, e.n);
    tiles += e.tiles;
  }
  const auto all = [&](int v) { return __builtin_amdgcn_readlane(scan(v, add), kWave - 1); };
  const unsigned total = (unsigned)all(work);
  const int over = a.shares - all(tiles);  // sum ceil(n / L) < sum n / L + tiles
  longest = __builtin_amdgcn_readlane(scan(longest, most), kWave - 1);
  const auto ratio = [](unsigned u, unsigned v) { return (u + v - 1) / v; };
  const unsigned least = max((unsigned)a.least, ratio((unsigned)longest, (unsigned)a.splits));
  unsigned length = max(over > 0 ? min(ratio(total, (unsigned)over), (unsigned)longest) : (unsigned)longest, least);
  // ceil(n / length) or, by rounding, one less (never more: there is room for
  // `shares`); all workgroups come to the same
  const auto cut = [](int n, unsigned length) {
    const float inv = (1.0f - 0x1p-20f) * __builtin_amdgcn_rcpf((float)length);
    return max((int)__builtin_ceilf((float)n * inv), 1);
  };
  if (per == 1) {
    unsigned few = max(ratio(total, (unsigned)a.shares), least) - 1;  // too short, or not allowed
    for (int i = 0; i < 7 && few + 1 < length; ++i) {
      const unsigned mid = (few + length) / 2;
      const bool fits = all(__mul24(e.tiles, cut(e.n, mid))) <= a.shares;
      if (fits) length = mid;
      else few = mid;
    }
  }
  int count = 0;
  if (per == 1) count = e.tiles * cut(e.n, length);
  else
    for (int j = 0; j < per; ++j) {
      const Entry o = entry(lane * per + j);
      count += o.tiles * cut(o.n, length);
    }
  const int upto = scan(count, add);
  const int holder = __popcll(__ballot(upto <= x));
  if (holder >= kWave) return false;
  int rest = x - (__builtin_amdgcn_readlane(upto, holder) - __builtin_amdgcn_readlane(count, holder));
  int b = holder * per;
  if (per == 1) {
    e.first = __builtin_amdgcn_readlane(e.first, b);
    e.queries = __builtin_amdgcn_readlane(e.queries, b);
    e.len = __builtin_amdgcn_readlane(e.len, b);
    e.n = __builtin_amdgcn_readlane(e.n, b);
  } else {
    for (int j = 0; j < per; ++j, ++b) {
      e = entry(b);
      const int its = e.tiles * cut(e.n, length);
      if (rest < its || j == per - 1) break;
      rest -= its;
    }
  }
  const int c = cut(e.n, length), tile = (int)((unsigned)rest / (unsigned)c);
  *split = uniform(rest - tile * c);
  *splits = uniform(c);
  b = uniform(b);
  t->first_token = uniform(e.first);
  t->queries = uniform(e.queries);
  t->row0 = uniform(tile * R);
  t->kv_len = uniform(e.len);
  t->table = a.table + (b < a.requests ? b * a.table_stride : 0);
  // (offsets that are not in order may ask for more tiles than there is room
  // for: then a tile runs with all of its shares or not at all)
  return t->row0 < t->queries * a.group && x - *split + *splits <= a.shares;
}

// The 32-token groups [begin, end) of one split of a tile, and how many splits
// the tile has: the launch's, or fewer of at least `least` groups.
struct Share {
  int begin, end, splits;
};
__device__ __forceinline__ Share share_of(const AttnArgs& a, int g_lo, int g_hi, int split, int splits) {
  const int n = max(g_hi - g_lo, 0);
  const int per = max((n + splits - 1) / splits, a.least);
  Share r;
  r.begin = g_lo + min(split * per, n);
  r.end = min(r.begin + per, g_lo + n);
  r.splits = max((n + per - 1) / per, 1);
  return r;
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
  const int id = read_scalar(t.table, g >> per);
  const bool ok = (unsigned)id < (unsigned)a.num_blocks;
  r.at = (int64_t)(ok ? id : 0) * a.hk + h;
  r.sub = g & ((1 << per) - 1);
  r.ok = ok;
  return r;
}
// A scale's bits (kept as an integer: compares and branches on it are scalar).
// Scales are not negative, so their order is that of the bits.
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t scale_bits(const float* p, const Group& g) {
  const uint32_t v = read_scalar(reinterpret_cast<const uint32_t*>(p), g.at);
  return g.ok ? v : kInfBits;
}
__device__ __forceinline__ float as_float(uint32_t bits) { return __builtin_bit_cast(float, bits); }

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

// Inside a branch on a uniform condition: keeps the compiler from turning it
// into a select per value that every group would pay for.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

// Running softmax of one query row, as the lanes of its column hold it: m and
// d agree over them, l is each lane's own share of the sum.
struct Running {
  float m = -__builtin_inff();  // log2 units; -inf: nothing seen
  float l = 0.0f;
  float d = 0.0f;               // the sums of p vs v are in units of 2^(m + d)
};

__device__ __forceinline__ float safe(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

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

// A row's references after scores of at most x, and of at most xv with log2 vs;
// by how much l and the sums of p vs v change.
struct Change {
  float l, o;
};
__device__ __forceinline__ Change raise_to(Running& r, float x, float xv) {
  const float m = fmaxf(r.m, x), top = fmaxf(r.m + r.d, xv);
  const float d = m == -__builtin_inff() ? 0.0f : top - m, fall = r.m - safe(m);
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
// Splits of one tile.  Each workgroup stores its rows' sums and (m, l), waits
// for its stores and counts itself; the last one adds all of them in split
// order, so the order of arrival does not show.  Stores and loads go past the
// XCD's own L2 (device scope).  One workgroup adds at what its own loads in
// flight allow: where a tile has many rows a second kernel does it (4 requests
// of 50 queries, 8 heads of 256, 8 splits: 87 us with join(), 36 with it).
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kDeviceScope = 16;  // sc1 of a buffer access

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// Partial results, addressed by byte offsets below 2^31 (checked on the host).
struct Partials {
  __amdgpu_buffer_rsrc_t part, stat;
  __device__ __forceinline__ Partials(const AttnArgs& a)
      : part(__builtin_amdgcn_make_buffer_rsrc(a.part, 0, 0x7fffffff, 0x00027000)),
        stat(__builtin_amdgcn_make_buffer_rsrc(a.stat, 0, 0x7fffffff, 0x00027000)) {}
  __device__ __forceinline__ void store(int i, floatx4 v) const {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), part, i * 4, 0, kDeviceScope);
  }
  __device__ __forceinline__ floatx4 load(int i) const {
    return __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(part, i * 4, 0, kDeviceScope));
  }
  __device__ __forceinline__ void store_stat(int i, float m, float l) const {
    const floatx2 v = {m, l};
    __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, v), stat, i * 8, 0, kDeviceScope);
  }
  __device__ __forceinline__ floatx2 load_stat(int i) const {  // m, l
    return __builtin_bit_cast(floatx2, __builtin_amdgcn_raw_buffer_load_b64(stat, i * 8, 0, kDeviceScope));
  }
};

// Output row of tile row rc: token * heads + head.
__device__ __forceinline__ int64_t out_row(const AttnArgs& a, const Tile& t, int h, int rc) {
  const int row = t.row0 + rc, qi = (int)((unsigned)row / (unsigned)a.group);
  return (int64_t)(t.first_token + qi) * a.hq + h * a.group + (row - qi * a.group);
}

template <typename T>
__device__ __forceinline__ void finish(const AttnArgs& a, int64_t to, int D, int d, floatx4 o, float m,
                                       float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = 0.0f;
  typedef T tx4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<tx4*>(a.out + (to * D + d) * 2) = __builtin_convertvector(o * inv, tx4);
  if (d == 0 && a.lse)
    a.lse[to] = l == 0.0f ? -__builtin_inff() : (m - kShift + log2_fast(l)) * kLn2;
}

// A split with nothing to do, for kv8_merge_kernel.
__device__ __forceinline__ void no_share(const AttnArgs& a, const Tile& t, int h, int rows, int split) {
  const Partials parts(a);
  for (int rc = threadIdx.x; rc < rows; rc += kThreads)
    parts.store_stat((int)out_row(a, t, h, rc) * a.splits + split, -__builtin_inff(), 0.0f);
}

// All threads call it after their stores of partial results.  buf: LDS of
// rows * splits * 8 + 4096 bytes, free for use.  Row rc of split s is at
// first + s * stride + rc of the partial results.
template <typename T, int D>
__device__ __forceinline__ void join(const AttnArgs& a, const Tile& t, int h, int rows, int splits,
                                     int first, int stride, uint32_t* counter, float* buf) {
  const int tid = threadIdx.x;
  __shared__ int is_last;
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wavefront's stores are done
  __syncthreads();
  if (tid == 0) {
    const uint32_t before =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = before == (uint32_t)(splits - 1);
    if (is_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;
  const Partials parts(a);
  // One thread per row and four dimensions; where that leaves threads over,
  // `ways` of them share the splits and meet in LDS.  What counts is that many
  // loads are in flight: a round trip takes longer than the bytes.
  constexpr int kFlight = 8;
  const int units = rows * (D / 4);
  int ways = 1;
  while (units * ways * 2 <= kThreads && ways * 2 <= splits) ways *= 2;
  float* stat = buf;  // [rows][splits][m, l]
  floatx4* sums = reinterpret_cast<floatx4*>(buf + (rows * splits * 2 + 3) / 4 * 4);
  for (int i = tid; i < rows * splits; i += kThreads) {
    const int rc = (int)((unsigned)i / (unsigned)splits);
    *reinterpret_cast<floatx2*>(stat + 2 * i) =
        parts.load_stat(first + (i - rc * splits) * stride + rc);
  }
  for (int u0 = 0; u0 < units; u0 += kThreads) {
    const int way = ways == 1 ? 0 : (int)((unsigned)tid / (unsigned)units);
    const int u = u0 + (ways == 1 ? tid : tid - way * units);
    const bool on = u < units && way < ways;
    const int rc = on ? u / (D / 4) : 0, d = u % (D / 4) * 4;
    const int64_t to = out_row(a, t, h, rc);
    const int at = (first + rc) * D + d, next = stride * D;
    floatx4 x[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) x[k] = parts.load(at + min(way + k * ways, splits - 1) * next);
    if (u0 == 0) __syncthreads();  // stat
    const float* st = stat + rc * splits * 2;
    float m = -__builtin_inff(), l = 0.0f;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, st[2 * s]);
    for (int s = 0; s < splits; ++s) l += st[2 * s + 1] * exp2_fast(st[2 * s] - safe(m));
    floatx4 o = 0.0f;
    for (int s0 = way; s0 < splits; s0 += kFlight * ways) {
      floatx4 y[kFlight];
#pragma unroll
      for (int k = 0; k < kFlight; ++k) y[k] = x[k];
      if (s0 + kFlight * ways < splits) {
#pragma unroll
        for (int k = 0; k < kFlight; ++k)
          x[k] = parts.load(at + min(s0 + (kFlight + k) * ways, splits - 1) * next);
      }
#pragma unroll
      for (int k = 0; k < kFlight; ++k) {
        const int s = s0 + k * ways;
        if (s < splits) o += y[k] * exp2_fast(st[2 * s] - safe(m));
      }
    }
    if (ways > 1) {  // (units < kThreads: one turn of the outer loop)
      sums[tid] = o;
      __syncthreads();
      if (on && way == 0)
        for (int w = 1; w < ways; ++w) o += sums[tid + w * units];
    }
    if (on && way == 0) finish<T>(a, to, D, d, o, m, l);
  }
}

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
constexpr int kWaves = 4;

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
      const float c = as_float(ks) * factor[r];
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
      raise |= mx + fmaxf(log_vs - run[r].d, 0.0f) > run[r].m + (run[r].m == -__builtin_inff() ? 0.0f : kRaise);
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
        const Change f = raise_to(run[r], mx, mx + log_vs);
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
      const float off = kShift + lr[r] - safe(run[r].m);
      float sum = 0.0f;
#pragma unroll
      for (int tt = 0; tt < 2; ++tt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = exp2_fast(s[r][tt][i] + off);
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
    join<T, D>(a, t, h, rows, share.splits, ((int)id - split * a.hk) * R, a.hk * R,
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
__device__ __forceinline__ floatx16 mfma32x32x16(half8 a, half8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

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
  const bool partial = a.splits > 1;  // kv8_merge_kernel adds them

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
    // the largest score, with log2 vs, and as much of that as is above d
    float c[NG], mx = -__builtin_inff(), mv = mx, over = mx;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      // (not 0, also where ks is 0 or the product underflows: masked scores are
      // -inf here already, and -inf * 0 is NaN; any score times 2^-126 is 0 to exp2)
      c[n] = fmaxf(as_float(ks[n]) * factor, 0x1p-126f);
      float most = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, s[n][i]);
      most *= c[n];
      mx = fmaxf(mx, most);
      mv = fmaxf(mv, most + log_vs[n]);
      over = fmaxf(over, most + fmaxf(log_vs[n] - run.d, 0.0f));
    }
    if (__ballot(over > run.m + (run.m == -__builtin_inff() ? 0.0f : kRaise))) {
      const Change f = raise_to(run, fmaxf(mx, __shfl_xor(mx, 32)), fmaxf(mv, __shfl_xor(mv, 32)));
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
    half8 p[2];
    const auto weights = [&](int n) {
      const float off = kShift + lr[n] - safe(run.m);
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

// ---------------------------------------------------------------------------
// The splits of every row, in their order: four dimensions a thread.  Its cost,
// about 5 us and 8 bytes per value and split at 3 TB/s with the stores that feed
// it, is what bounds the number of splits of prompts.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void kv8_merge_kernel(AttnArgs a) {
  const int64_t it = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = it / (D / 4);
  const int d = it % (D / 4) * 4;
  if (row >= (int64_t)a.tokens * a.hq) return;
  const floatx2* stat = reinterpret_cast<const floatx2*>(a.stat) + row * a.splits;
  const float* part = a.part + row * a.splits * D + d;
  float m = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, stat[s][0]);
  float l = 0.0f;
  floatx4 o = 0.0f;
#pragma unroll 8
  for (int s = 0; s < a.splits; ++s) {
    const float ls = stat[s][1], f = exp2_fast(stat[s][0] - safe(m));
    floatx4 x = *reinterpret_cast<const floatx4*>(part + (int64_t)s * D);
    if (ls == 0.0f) x = 0.0f;  // (not written)
    l += ls * f;
    o += x * f;
  }
  finish<T>(a, row, D, d, o, m, l);
}

template <typename T, int D>
hipError_t launch_sized(AttnArgs a, const Kv8AttnPlan& p, hipStream_t stream) {
  constexpr size_t kLds = D == 64 ? kWaves * 32 * 68 * 4
                                  : 2 * (D <= 128 ? 2 : 1) * 32 * D * 2 * 2 + (D > 128 ? 128 * D * 2 : 0);
  constexpr size_t kLds2 = 4 * 2 * 32 * D * 2 * 2;
  // (no workgroup waits for another, so those of one tile may be in two launches)
  const int64_t most = kMaxThreads / (p.gangs * kThreads);
  for (int64_t i = 0; i < p.grid; i += most) {
    a.first = (unsigned)i;
    const unsigned grid = (unsigned)(p.grid - i < most ? p.grid - i : most);
    if (p.kernel == 1 && p.gangs == 1) kv8_prefill_kernel<T, D, 1><<<grid, kThreads, kLds, stream>>>(a);
    else if (p.kernel == 0 && p.rows == 16) kv8_decode_kernel<T, D, 1><<<grid, kThreads, 0, stream>>>(a);
    else if constexpr (D <= 128) {
      if (p.kernel == 1) kv8_prefill_kernel<T, D, 2><<<grid, 2 * kThreads, kLds2, stream>>>(a);
      else kv8_decode_kernel<T, D, 2><<<grid, kThreads, 0, stream>>>(a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (!a.merge) return hipSuccess;
  kv8_merge_kernel<T, D>
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
namespace {

// Splits of a tile that join()'s LDS holds.
int most_splits(int rows) { return rows == 32 ? 48 : 64; }
// Requests up to which every workgroup adds up their lengths: eight round trips.
constexpr int64_t kShareRequests = 512;

struct Estimate {
  double us;
  int splits;
  bool merge;
};

Estimate estimate(bool prefill, int gangs, int rows, double tiles, double groups, double longest, double tokens_heads, bool ragged,
                  double shared, int most_rows, int D, int hk, int cus) {
  // us of a turn; slots: workgroups that run at a time (prompts of size 256: LDS
  // holds one on each CU, the fitted constants go with two)
  const double base = prefill ? (D == 64 ? 1.1 : D == 128 ? 1.5 : 1.35)
                              : D == 256 ? 1.1 : (rows == 16 ? 0.55 : 0.85) * (D == 64 ? 0.75 : 1.0);
  const double more = prefill ? (D == 256 ? 0.6 : 0.4) : D == 256 ? 1.2 : (rows == 16 ? 0.25 : 0.58) * (D == 64 ? 0.6 : 1.0);
  const int per_turn = prefill ? (D == 256 ? 1 : 2 * gangs) : kWaves;
  const double slots = cus * (gangs == 2 ? 1.0 : prefill || D == 256 || rows > 16 ? 2.0 : 3.0);
  const int held = rows < most_rows ? rows : most_rows;
  const int cap = most_splits(rows);
  Estimate best{1e30, 1, false};
  for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (s > cap || (s > 1 && s > groups)) break;
    const double turns = ceil(ceil(groups / s) / per_turn), w = tiles * hk * s;
    const auto round = [&](double n) {  // n workgroups at a time
      // the cache's bytes of a turn, at 6.5 TB/s, where they come from memory
      const double bytes = n * per_turn * 64.0 * D * shared / 6.5e6;
      const double turn = base + more * (gangs * n / cus);
      return 2.5 + turns * (turn > bytes ? turn : bytes);
    };
    const double full = floor(w / slots), rest = w - full * slots;
    double us = full * round(slots) + (rest >= 1 ? round(rest) : 0.0);
    // the last tile of a prompt sees the most, beside shorter ones
    const double alone = 2.5 + ceil(ceil(longest / s) / per_turn) * (base + more * (gangs == 2 ? 1.75 : prefill ? 0.3 : 0.2));
    us = 3.0 + (prefill ? 2 * gangs - 1 : 0) + (us > alone ? us : alone);
    if (ragged) us += 0.1 * round(w < slots ? w : slots);  // the longest request runs on
    bool merge = false;
    if (s > 1) {
      const double units = held * (D / 4), ways = units < kThreads ? kThreads / units : 1.0;
      const double join = 2.0 + 1.2 * ceil(units / kThreads) * ceil(s / (8.0 * ways));
      const double second = 4.5 + tokens_heads * s * D * 8.0 / 3e6;
      merge = prefill || second < join || tiles * hk > kMaxSplitCounters;
      us += merge ? second : join;
    }
    if (us < best.us) best = {us, s, merge};
  }
  return best;
}

}  // namespace

Kv8AttnPlan plan_kv8_attention(const rf_kv8_attention_args& a, int cus) {
  Kv8AttnPlan p;
  const int64_t group = a.q.heads / a.cache.kv_heads, hk = a.cache.kv_heads;
  const int D = a.cache.head_dim;
  int64_t most_q = a.cu_q ? a.max_q_len : a.tokens / a.requests;
  if (most_q < 1 || most_q > a.tokens) most_q = a.tokens;
  const int64_t most_rows = most_q * group;
  int64_t most_kv = a.width * a.cache.block_size;
  if (a.max_kv_len > 0 && a.max_kv_len < most_kv) most_kv = a.max_kv_len;
  if (a.window > 0 && a.window < most_kv - most_q) most_kv = a.window + most_q;  // (a window may be any int64)
  const bool ragged = a.cu_q && a.requests > 1;
  // tiles that have work, and the upper bound that the grid covers
  const auto useful = [&](int rows) {
    const int64_t each = a.requests * ceil_div(most_rows, rows), all = a.tokens * group / rows + a.requests;
    return each < all ? each : all;
  };
  const auto bound = [&](int rows) {
    return a.cu_q ? a.tokens * group / rows + a.requests + 1 : a.requests * ceil_div(most_rows, rows);
  };
  const auto groups = [&](int rows) {  // seen by a tile, on average
    const double first = a.causal ? (most_q > rows / group ? most_q - rows / (double)group : 0.0) / 2 : 0.0;
    const double n = most_kv - first;
    return (n < 1 ? 1 : n) / RF_KV8_GROUP + 0.5;
  };
  const double tokens_heads = (double)a.tokens * a.q.heads, longest = most_kv / (double)RF_KV8_GROUP + 0.5;
  // (two tiles of 16 rows of size 256 would not fit the registers)
  const int few = most_rows <= 16 || D > 128 ? 16 : 32;
  const int most = (int)(most_rows < 1024 ? most_rows : 1024);
  Estimate e = estimate(false, 1, few, (double)useful(few), groups(few), longest, tokens_heads, ragged,
                        1.0 / ceil_div(most_rows, few), most, D, (int)hk, cus);
  p.kernel = 0;
  p.rows = few;
  if (most_rows > 16) {
    for (int gangs = 1; gangs <= (D == 256 ? 1 : 2); ++gangs) {
      const Estimate e1 = estimate(true, gangs, 128, (double)useful(128), groups(128), longest, tokens_heads, ragged,
                                   1.0 / ceil_div(most_rows, 128), most, D, (int)hk, cus);
      if (e1.us >= e.us) continue;
      e = e1;
      p.kernel = 1;
      p.gangs = gangs;
      p.rows = 128;
    }
  }
  p.tiles = bound(p.rows);
  p.least = p.kernel ? (D == 256 ? 1 : 2) : kWaves;
  p.splits = e.splits;
  p.merge = e.merge;
  p.grid = p.tiles * hk * p.splits;
  // Partial results are addressed by 31 bits; joined tiles take a counter each.
  const auto fits = [&](int64_t rows, int64_t grid) {
    p.partials = rows;
    p.workspace = (size_t)rows * (D + 2) * 4;
    return p.workspace <= 0x7fffffff && grid <= (p.merge ? 0x7fffffff : kMaxSplitCounters);
  };
  // (the sums of tiles times groups fit, whatever the offsets say)
  if (p.kernel == 0 && !p.merge && a.requests > 1 && a.requests < kShareRequests &&
      (double)p.tiles * (double)a.requests * (double)(a.width * a.cache.block_size / RF_KV8_GROUP + 1) < 2147483647.0) {
    // Workgroups: the multiple of the CUs that leaves tiles half a share each to
    // cut (16 requests of 4 to 20 thousand tokens, 32 + 8 heads, 1, 1.25, 2 and 3
    // workgroups a CU: 64.8, 74.8, 63.5, 65.4 us; 48 of up to 9000, 64 + 8 heads:
    // 2, 2.5, 3 and 4: 95.9, 87.8, 83.5, 88.9).  Shares are long enough for the
    // join they cost (32 requests of up to 500 tokens: 8.0 us, in shares of 8
    // groups 11.5; 4 x 50 queries after 968 tokens, 32 rows: 14.0 and 20.9).
    int64_t shares = ceil_div(3 * useful(p.rows) * hk, 2 * cus) * cus / hk;
    if (shares < p.tiles) shares = p.tiles;
    // (16 workgroups a CU even out by themselves, and their partial results stay
    // below 70 MB)
    if (shares * hk <= 16 * cus && fits(shares * hk * p.rows, shares * hk)) {
      p.shares = (int)shares;
      p.splits = most_splits(p.rows);
      p.least = p.rows == 32 ? 32 : D == 256 ? 8 : 16;
      p.grid = shares * hk;
      return p;
    }
  }
  if (p.splits == 1 || !fits(p.merge ? a.tokens * a.q.heads * p.splits : p.grid * p.rows, p.grid)) {
    p.splits = 1;
    p.merge = false;
    p.grid = p.tiles * hk;
    p.partials = 0;
    p.workspace = 0;
  }
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
  a.counters = nullptr;
  a.stat = nullptr;
  a.part = nullptr;
  if (p.workspace > 0) {
    a.counters = (uint32_t*)in.scratch->counters;
    a.part = (float*)in.scratch->partials;
    a.stat = (uint64_t*)(a.part + p.partials * D);
  }
  a.table_stride = in.table_stride;
  a.num_blocks = (int)in.cache.num_blocks;
  a.tokens = (int)in.tokens;
  a.requests = (int)in.requests;
  a.width = (int)in.width;
  a.hq = in.q.heads;
  a.hk = in.cache.kv_heads;
  a.group = a.hq / a.hk;
  a.shift = __builtin_ctz((unsigned)in.cache.block_size);
  a.per_request = in.cu_q ? 0 : (int)(in.tokens / in.requests);
  a.splits = p.splits;
  a.least = p.least;
  a.merge = p.merge;
  a.shares = p.shares;
  a.tiles = (int)p.tiles;
  a.causal = in.causal;
  a.window = in.window > (1 << 30) ? 1 << 30 : (int)in.window;
  a.scale_log2e = in.scale * kLog2e;
  const bool f16 = in.dtype == RF_W8A16_DTYPE_F16;
  if (D == 64)
    return f16 ? launch_sized<_Float16, 64>(a, p, stream) : launch_sized<__bf16, 64>(a, p, stream);
  if (D == 128)
    return f16 ? launch_sized<_Float16, 128>(a, p, stream) : launch_sized<__bf16, 128>(a, p, stream);
  return f16 ? launch_sized<_Float16, 256>(a, p, stream) : launch_sized<__bf16, 256>(a, p, stream);
}

}  // namespace rf
