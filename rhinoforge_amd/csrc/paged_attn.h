// What attention over a paged cache shares whatever the cache holds (kv8_attn.hip,
// kv4_attn.hip): where a workgroup finds its rows and tokens, how the splits of a
// tile are added, and how a call's launch is chosen.
#pragma once

#include <math.h>

#include "kv8_common.h"

namespace rf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kRaise = 8.0f;  // m follows x from here on: 2^(7 + 8) < 65504
constexpr float kShift = 7.0f;
// Scores (log2 units) from which on their differences are taken first: rounding one of
// this size costs 2^-12.
constexpr float kFar = 4096.0f;

struct PagedArgs {
  const uint8_t* q;
  int64_t q_ts, q_hs;  // bytes
  const uint8_t *k, *v;
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
  int shares;          // find_share: of all tiles together, at most (0: not used)
  int aim;             // that many of them, unless there are more tiles
  bool merge;          // partial results are added by merge_splits_kernel, else by join()
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

// First token of request b's queries and its keys, for any b >= 0 (b >= requests: the
// tokens past the batch, which see nothing).  No branches, and loads apart from what
// looks at them: the compiler waits for a load at the end of a branch.
__device__ __forceinline__ int read_cu(const PagedArgs& a, int b) { return a.cu[min(b, a.requests)]; }
__device__ __forceinline__ int read_len(const PagedArgs& a, int b) { return a.lens[min(b, a.requests - 1)]; }
__device__ __forceinline__ int checked_cu(const PagedArgs& a, int b, int c) {
  const int lo = b > a.requests ? a.tokens : 0, hi = b <= 0 ? 0 : a.tokens;
  return min(max(c, lo), hi);
}
__device__ __forceinline__ int checked_len(const PagedArgs& a, int b, int len) {
  return min(max(len, 0), b < a.requests ? a.width << a.shift : 0);
}
__device__ __forceinline__ int cu_at(const PagedArgs& a, int b) { return checked_cu(a, b, read_cu(a, b)); }
__device__ __forceinline__ int len_at(const PagedArgs& a, int b) { return checked_len(a, b, read_len(a, b)); }

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

// Requests up to which every workgroup counts all tiles: eight of them a lane.
constexpr int kCountRequests = 512;

// Tile x of the launch.  The wavefront counts the tiles of up to 512 requests, whose
// offsets and lengths it reads at once, so that the tiles follow each other and what the
// grid has more, for any offsets, ends after them.  (With tiles at places that the
// offsets alone give, floor(cu[b] group / R) + b, half the workgroups of a batch of
// single tokens were empty ones among the others: 128 x 300 tokens, 64 + 8 heads of a
// 4-bit cache 25 us, now 14.5.)  More requests are found like that, 64 boundaries at a
// time.
template <int R>
__device__ __forceinline__ bool find_tile(const PagedArgs& a, int x, Tile* t) {
  int b, len;
  if (a.cu == nullptr) {
    const int per = (a.per_request * a.group + R - 1) / R;
    b = (int)((unsigned)x / (unsigned)per);
    if (b >= a.requests) return false;
    t->first_token = b * a.per_request;
    t->queries = a.per_request;
    t->row0 = (x - b * per) * R;
    len = len_at(a, b);
  } else if (a.requests < kCountRequests) {
    const int lane = threadIdx.x % kWave;
    constexpr int kChunks = kCountRequests / kWave;
    int first[kChunks], next[kChunks], lens[kChunks];
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (i == 0 || i * kWave <= a.requests) {
        const int at = i * kWave + lane;
        first[i] = read_cu(a, at);
        next[i] = read_cu(a, at + 1);
        lens[i] = read_len(a, at);
      }
    int before = 0;
    bool found = false;
#pragma unroll
    for (int i = 0; i < kChunks; ++i)
      if (!found && (i == 0 || i * kWave <= a.requests)) {
        const int at = i * kWave + lane, from = checked_cu(a, at, first[i]);
        const int queries = max(checked_cu(a, at + 1, next[i]) - from, 0);
        const int tiles = (int)(((unsigned)(queries * a.group) + R - 1) / R);
        const int upto = scan(tiles, [](int u, int v) { return u + v; }) + before;
        const int holder = __popcll(__ballot(upto <= x));
        found = holder < kWave;
        if (found) {
          b = i * kWave + holder;
          t->first_token = __builtin_amdgcn_readlane(from, holder);
          t->queries = __builtin_amdgcn_readlane(queries, holder);
          t->row0 = (x - __builtin_amdgcn_readlane(upto - tiles, holder)) * R;
          len = checked_len(a, b, __builtin_amdgcn_readlane(lens[i], holder));
        } else {
          before = __builtin_amdgcn_readlane(upto, kWave - 1);
        }
      }
    if (!found) return false;
  } else {
    const int lane = threadIdx.x % kWave;
    const auto begin = [&](int c, int i) { return (int)((int64_t)c * a.group / R) + i; };
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
    const int first = cu_at(a, b);
    t->first_token = first;
    t->queries = max(cu_at(a, b + 1) - first, 0);
    t->row0 = (x - begin(first, b)) * R;
    len = len_at(a, b);
  }
  if (t->row0 < 0 || t->row0 >= t->queries * a.group) return false;
  b = uniform(b);
  t->first_token = uniform(t->first_token);
  t->queries = uniform(t->queries);
  t->row0 = uniform(t->row0);
  t->kv_len = uniform(len);
  t->table = a.table + (b < a.requests ? b * a.table_stride : 0);
  return true;
}

// Tokens [lo, hi) that row `row` of a request sees.
__device__ __forceinline__ void seen(const PagedArgs& a, const Tile& t, int row, int* lo, int* hi) {
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
// smallest L that leaves no more than `aim` of them: a batch takes as long as
// its mean, not as its longest request, and its workgroups fill the CUs evenly.
// Each lane holds ceil(requests / 64) requests, so up to 64 of them cost one
// memory round trip; for more, L is a bound that needs no search.
template <int R>
__device__ __forceinline__ bool find_share(const PagedArgs& a, int x, Tile* t, int* split, int* splits) {
  struct Entry {
    int first, queries, tiles, len, n;  // n: groups that its last tile sees
  };
  const int lane = threadIdx.x % kWave, entries = a.requests + (a.cu ? 1 : 0);
  const int per = (int)((unsigned)(entries + kWave - 1) / kWave);
  const auto entry = [&](int b) {
    Entry e;
    e.len = len_at(a, b);
    e.first = b * a.per_request;
    e.queries = a.per_request;
    if (a.cu) {
      e.first = cu_at(a, b);
      e.queries = max(cu_at(a, b + 1) - e.first, 0);
    }
    if (b >= entries) e.queries = 0;
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
  const int over = a.aim - all(tiles);  // sum ceil(n / L) < sum n / L + tiles
  longest = __builtin_amdgcn_readlane(scan(longest, most), kWave - 1);
  const auto ratio = [](unsigned u, unsigned v) { return (u + v - 1) / v; };
  const unsigned least = max((unsigned)a.least, ratio((unsigned)longest, (unsigned)a.splits));
  unsigned length = max(over > 0 ? min(ratio(total, (unsigned)over), (unsigned)longest) : (unsigned)longest, least);
  // ceil(n / length) or, by rounding, one less (never more: there is room for
  // `aim`); all workgroups come to the same
  const auto cut = [](int n, unsigned length) {
    const float inv = (1.0f - 0x1p-20f) * __builtin_amdgcn_rcpf((float)length);
    return max((int)__builtin_ceilf((float)n * inv), 1);
  };
  if (per == 1) {
    unsigned few = max(ratio(total, (unsigned)a.aim), least) - 1;  // too short, or not allowed
    for (int i = 0; i < 7 && few + 1 < length; ++i) {
      const unsigned mid = (few + length) / 2;
      const bool fits = all(__mul24(e.tiles, cut(e.n, mid))) <= a.aim;
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
__device__ __forceinline__ Share share_of(const PagedArgs& a, int g_lo, int g_hi, int split, int splits) {
  const int n = max(g_hi - g_lo, 0);
  const int per = max((n + splits - 1) / splits, a.least);
  Share r;
  r.begin = g_lo + min(split * per, n);
  r.end = min(r.begin + per, g_lo + n);
  r.splits = max((n + per - 1) / per, 1);
  return r;
}

// One 32-token group of a head: where its bytes are.  A block id outside the cache:
// block 0, and not ok (the kernels make its scores NaN).
struct Group {
  int64_t at;  // block * hk + h
  int sub;     // group within the block
  bool ok;
};
__device__ __forceinline__ Group group_of(const PagedArgs& a, const Tile& t, int h, int g) {
  Group r;
  const int per = a.shift - 5;
  const int id = read_scalar(t.table, g >> per);
  const bool ok = (unsigned)id < (unsigned)a.num_blocks;
  r.at = (int64_t)(ok ? id : 0) * a.hk + h;
  r.sub = g & ((1 << per) - 1);
  r.ok = ok;
  return r;
}
// The largest magnitude of eight query values and m.
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

__device__ __forceinline__ float safe(float m) { return m == -__builtin_inff() ? 0.0f : m; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float log2_fast(float x) { return __builtin_amdgcn_logf(x); }

// Score factors stay finite and above 0: a masked score is -inf whatever it is
// multiplied by, a score of 0 is 0, and scores beyond these ranges are 0 or infinite to
// exp2.
__device__ __forceinline__ float in_range(float factor) { return fminf(fmaxf(factor, 0x1p-126f), 0x1p127f); }

// A difference of scores, both rounded.  (Taken together with the product that one of
// them is, in one rounding, it would not be 0 for the largest score.)
__device__ __forceinline__ float minus(float s, float m) {
#pragma clang fp contract(off)
  return s - m;
}

// ---------------------------------------------------------------------------
// Splits of one tile.  Each workgroup stores its rows' sums and (m, l), waits
// for its stores and counts itself; the last one adds all of them in split
// order, so the order of arrival does not show.  Stores and loads go past the
// XCD's own L2 (device scope).  One workgroup adds at what its own loads in
// flight allow: where a tile has many rows a second kernel does it (4 requests
// of 50 queries, 8 heads of 256, 8 splits: 87 us with join(), 36 with it).
// ---------------------------------------------------------------------------
constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kDeviceScope = 16;  // sc1 of a buffer access

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float floatx2 __attribute__((ext_vector_type(2)));

// Partial results, addressed by byte offsets below 2^31 (checked on the host).
struct Partials {
  __amdgpu_buffer_rsrc_t part, stat;
  __device__ __forceinline__ Partials(const PagedArgs& a)
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
__device__ __forceinline__ int64_t out_row(const PagedArgs& a, const Tile& t, int h, int rc) {
  const int row = t.row0 + rc, qi = (int)((unsigned)row / (unsigned)a.group);
  return (int64_t)(t.first_token + qi) * a.hq + h * a.group + (row - qi * a.group);
}

template <typename T>
__device__ __forceinline__ void finish(const PagedArgs& a, int64_t to, int D, int d, floatx4 o, float m,
                                       float l) {
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (l == 0.0f) o = 0.0f;
  typedef T tx4 __attribute__((ext_vector_type(4)));
  *reinterpret_cast<tx4*>(a.out + (to * D + d) * 2) = __builtin_convertvector(o * inv, tx4);
  if (d == 0 && a.lse)
    a.lse[to] = l == 0.0f ? -__builtin_inff() : (m - kShift + log2_fast(l)) * kLn2;
}

// A split with nothing to do, for merge_splits_kernel.
__device__ __forceinline__ void no_share(const PagedArgs& a, const Tile& t, int h, int rows, int split) {
  const Partials parts(a);
  for (int rc = threadIdx.x; rc < rows; rc += blockDim.x)
    parts.store_stat((int)out_row(a, t, h, rc) * a.splits + split, -__builtin_inff(), 0.0f);
}

// All threads call it after their stores of partial results.  buf: LDS of
// rows * splits * 8 + 16 kT bytes, free for use; kT threads, up to kRows rows.  Row rc of split s is at
// first + s * stride + rc of the partial results.
template <typename T, int D, int kRows, int kT>
__device__ __forceinline__ void join(const PagedArgs& a, const Tile& t, int h, int rows, int splits,
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
  while (units * ways * 2 <= kT && ways * 2 <= splits) ways *= 2;
  float* stat = buf;  // [rows][splits][2^(m - the row's), l]
  floatx4* sums = reinterpret_cast<floatx4*>(buf + (rows * splits * 2 + 3) / 4 * 4);
  __shared__ float tops[kRows];
  constexpr int kEach = (kRows + kT / kWave - 1) / (kT / kWave);
  // A wavefront takes some of the rows, a lane one of its splits (at most 64).
  const int lane = tid % kWave, wave = tid / kWave;
  floatx2 own[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i)  // (no branches, which would wait for each load)
    own[i] = parts.load_stat(first + min(lane, splits - 1) * stride + min(wave + i * (kT / kWave), rows - 1));
  const auto factors = [&] {
    float top[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) top[i] = own[i][0];  // (lanes from `splits` on: the last one's)
    for (int n = 1; n < splits; n *= 2)
#pragma unroll
      for (int i = 0; i < kEach; ++i) top[i] = fmaxf(top[i], __shfl_xor(top[i], n));
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int rc = wave + i * (kT / kWave);
      if (rc >= rows) break;
      if (lane == 0) tops[rc] = top[i];
      if (lane < splits)
        *reinterpret_cast<floatx2*>(stat + 2 * (rc * splits + lane)) =
            floatx2{exp2_fast(own[i][0] - safe(top[i])), own[i][1]};
    }
  };
  for (int u0 = 0; u0 < units; u0 += kT) {
    const int way = ways == 1 ? 0 : (int)((unsigned)tid / (unsigned)units);
    const int u = u0 + (ways == 1 ? tid : tid - way * units);
    const bool on = u < units && way < ways;
    const int rc = on ? u / (D / 4) : 0, d = u % (D / 4) * 4;
    const int64_t to = out_row(a, t, h, rc);
    const int at = (first + rc) * D + d, next = stride * D;
    floatx4 x[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) x[k] = parts.load(at + min(way + k * ways, splits - 1) * next);
    if (u0 == 0) {
      factors();
      __syncthreads();
    }
    const floatx2* st = reinterpret_cast<const floatx2*>(stat) + rc * splits;
    const float m = tops[rc];
    float l = 0.0f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) l += st[s][1] * st[s][0];
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
        if (s < splits) o += y[k] * st[s][0];
      }
    }
    if (ways > 1) {  // (units < kT: one turn of the outer loop)
      sums[tid] = o;
      __syncthreads();
      if (on && way == 0)
        for (int w = 1; w < ways; ++w) o += sums[tid + w * units];
    }
    if (on && way == 0) finish<T>(a, to, D, d, o, m, l);
  }
}


__device__ __forceinline__ floatx16 mfma32x32x16(half8 a, half8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// ---------------------------------------------------------------------------
// The splits of every row, in their order: four dimensions a thread.  Its cost,
// about 5 us and 8 bytes per value and split at 3 TB/s with the stores that feed
// it, is what bounds the number of splits of prompts.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(kThreads) void merge_splits_kernel(PagedArgs a) {
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

// Splits of a tile that join()'s LDS holds.
int most_splits(int rows) { return rows == 32 ? 48 : 64; }
// Requests up to which every workgroup adds up their lengths: eight round trips.
constexpr int64_t kShareRequests = 512;

struct Estimate {
  double us;
  int splits;
  bool merge;
  int gangs = 1;
};

// Times of the kernels, fitted (Costs, one for each cache): base and more, us of a
// workgroup's turn alone and for each workgroup beside it on its CU; slots, the
// workgroups that a CU runs at a time; token_bytes, a token's keys and values; few, rows of a
// tile of the decode kernel; decode, its estimate; cut, whether the tiles of a batch of
// several requests are cut into shares; shares, how many, and aim, whether no more of
// them where the grid has room for more tiles; share_least, 32-token groups of one, at
// least.
template <typename Costs>
Estimate estimate(bool prefill, int gangs, int rows, double tiles, double groups, double longest, double tokens_heads, bool ragged,
                  double shared, int most_rows, int D, int hk, int cus) {
  const double base = Costs::base(prefill, rows, D), more = Costs::more(prefill, rows, D);
  const int per_turn = prefill ? (D == 256 ? 1 : 2 * gangs) : kWaves;
  const double slots = cus * Costs::slots(prefill, gangs, rows, D);
  const int held = rows < most_rows ? rows : most_rows;
  const int cap = most_splits(rows);
  Estimate best{1e30, 1, false};
  for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
    if (s > cap || (s > 1 && s > groups)) break;
    const double turns = ceil(ceil(groups / s) / per_turn), w = tiles * hk * s;
    const auto round = [&](double n) {  // n workgroups at a time
      // the cache's bytes of a turn, at 6.5 TB/s, where they come from memory
      const double bytes = n * per_turn * 32.0 * Costs::token_bytes(D) * shared / 6.5e6;
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


// What of a call its launch depends on.
struct PagedShape {
  int64_t tokens, requests, width;
  int heads, kv_heads, head_dim, block_size;
  bool ragged;  // offsets of the requests' queries are given
  int64_t max_q_len, max_kv_len;
  int causal;
  int64_t window;
};

template <typename Costs>
PagedPlan plan_paged_attention(const PagedShape& a, int cus) {
  PagedPlan p;
  const int64_t group = a.heads / a.kv_heads, hk = a.kv_heads;
  const int D = a.head_dim;
  int64_t most_q = a.ragged ? a.max_q_len : a.tokens / a.requests;
  if (most_q < 1 || most_q > a.tokens) most_q = a.tokens;
  const int64_t most_rows = most_q * group;
  int64_t most_kv = a.width * a.block_size;
  if (a.max_kv_len > 0 && a.max_kv_len < most_kv) most_kv = a.max_kv_len;
  if (a.window > 0 && a.window < most_kv - most_q) most_kv = a.window + most_q;  // (a window may be any int64)
  const bool ragged = a.ragged && a.requests > 1;
  // tiles that have work, and the upper bound that the grid covers
  const auto useful = [&](int rows) {
    const int64_t each = a.requests * ceil_div(most_rows, rows), all = a.tokens * group / rows + a.requests;
    return each < all ? each : all;
  };
  const auto bound = [&](int rows) {
    return a.ragged ? a.tokens * group / rows + a.requests + 1 : a.requests * ceil_div(most_rows, rows);
  };
  const auto groups = [&](int rows) {  // seen by a tile, on average
    const double first = a.causal ? (most_q > rows / group ? most_q - rows / (double)group : 0.0) / 2 : 0.0;
    const double n = most_kv - first;
    return (n < 1 ? 1 : n) / RF_KV8_GROUP + 0.5;
  };
  const double tokens_heads = (double)a.tokens * a.heads, longest = most_kv / (double)RF_KV8_GROUP + 0.5;
  const int few = Costs::few(most_rows, D);
  const int most = (int)(most_rows < 1024 ? most_rows : 1024);
  Estimate e = Costs::decode(a.requests, few, (double)useful(few), groups(few), longest, tokens_heads, ragged,
                             1.0 / ceil_div(most_rows, few), most, D, (int)hk, cus);
  p.kernel = 0;
  p.gangs = e.gangs;
  p.rows = few;
  if (most_rows > 16) {
    for (int gangs = 1; gangs <= (D == 256 ? 1 : 2); ++gangs) {
      const Estimate e1 = estimate<Costs>(true, gangs, 128, (double)useful(128), groups(128), longest, tokens_heads, ragged,
                                   1.0 / ceil_div(most_rows, 128), most, D, (int)hk, cus);
      if (e1.us >= e.us) continue;
      e = e1;
      p.kernel = 1;
      p.gangs = gangs;
      p.rows = 128;
    }
  }
  p.tiles = bound(p.rows);
  p.least = p.kernel ? (D == 256 ? 1 : 2) : kWaves * p.gangs;
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
  if (p.kernel == 0 && p.gangs == 1 && !p.merge && a.requests > 1 && a.requests < kShareRequests &&
      Costs::cut((double)(useful(p.rows) * hk), longest, D, cus) &&
      (double)p.tiles * (double)a.requests * (double)(a.width * a.block_size / RF_KV8_GROUP + 1) < 2147483647.0) {
    // Shares that are long enough for the join they cost (what was measured stands
    // at each Costs).
    int64_t shares = Costs::shares((double)(useful(p.rows) * hk), groups(p.rows), D, cus) / hk;
    p.aim = (int)shares;
    if (shares < p.tiles) shares = p.tiles;
    if (!Costs::aim || p.aim < 1) p.aim = (int)shares;
    // (16 workgroups a CU even out by themselves, and their partial results stay
    // below 70 MB)
    if (shares * hk <= 16 * cus && fits(shares * hk * p.rows, shares * hk)) {
      p.shares = (int)shares;
      p.splits = most_splits(p.rows);
      p.least = Costs::share_least(p.rows, D, longest);
      p.grid = shares * hk;
      return p;
    }
  }
  if (p.splits == 1 || !fits(p.merge ? a.tokens * a.heads * p.splits : p.grid * p.rows, p.grid)) {
    p.splits = 1;
    p.merge = false;
    p.grid = p.tiles * hk;
    p.partials = 0;
    p.workspace = 0;
  }
  return p;
}

// The kernels' arguments from a call's (rf_kv8_attention_args or the like).
template <typename In>
void fill_paged(PagedArgs& a, const In& in, const PagedPlan& p) {
  a.q = (const uint8_t*)in.q.data;
  a.q_ts = in.q.token_stride * 2;
  a.q_hs = in.q.head_stride * 2;
  a.k = (const uint8_t*)in.cache.k;
  a.v = (const uint8_t*)in.cache.v;
  a.cu = in.cu_q;
  a.lens = in.kv_lens;
  a.table = in.block_table;
  a.out = (uint8_t*)in.out;
  a.lse = in.lse;
  a.counters = nullptr;
  a.stat = nullptr;
  a.part = nullptr;
  if (p.workspace > 0) {
    a.counters = (uint32_t*)in.scratch->counters;
    a.part = (float*)in.scratch->partials;
    a.stat = (uint64_t*)(a.part + p.partials * in.cache.head_dim);
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
  a.aim = p.aim;
  a.tiles = (int)p.tiles;
  a.causal = in.causal;
  a.window = in.window > (1 << 30) ? 1 << 30 : (int)in.window;
  a.scale_log2e = in.scale * kLog2e;
}

template <typename In>
PagedShape shape_of(const In& a) {
  return {a.tokens, a.requests, a.width, a.q.heads, a.cache.kv_heads, a.cache.head_dim, a.cache.block_size,
          a.cu_q != nullptr, a.max_q_len, a.max_kv_len, a.causal, a.window};
}

}  // namespace
}  // namespace rf
