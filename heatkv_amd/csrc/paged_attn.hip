// Attention over a paged K/V cache: every query of a request sees the rows of
// its request's blocks (with a causal limit, a sliding window and first rows
// that stay visible), and of a prefix that all requests share.
//
// The queries of one request and K/V head are a matrix of n * group rows (token
// by token, the heads of a group side by side) against one stream of keys.  Two
// kernels run tiles of those rows:
//  * wide_tile, 128 rows: prompts and scales, bound by the matrix cores (and, as
//    the segmented kernel, by the chains of its softmax).  A prompt of 8192 tokens,
//    32 heads on 8: 560 us, 980 TFLOP/s; library products of random bf16 reach
//    1130 to 1350 on the same card.
//  * narrow_tile, 16 rows: single tokens, bound by the bytes of the cache.  64
//    requests of 800 to 16000 rows, 2.33 GB: 404 us, 5.8 TB/s; a copy of 2 GiB
//    moves 4.95.
//
// Plan.  Nothing about the requests is known on the host, so up to 64 requests every
// wave finds its work from lengths and query_starts itself (1 to 2 us, beside other
// workgroups' work in all but the smallest launches); for more, paged_plan_kernel
// writes each unit's work first, about 5 us (planned by every workgroup: 128 requests of
// 500 rows 65.4 us against 59.4, 1024 of 62 rows 283 against 106; two requests to a lane
// would save 3 us up to 128 requests and cost the calls of a few 0.2).  The plan is tiles
// of rows per request, 64-key chunks per tile, and, so that few rows over long keys
// still fill the card, parts of a tile's chunks.  part_chunks gives the chunks of a
// part from the total of the launch, so that the host knows how many units and
// records there can be at most.  A tile that is not cut writes its output.  Parts of
// narrow tiles are joined by the last of them (join_parts): a pair of tokens over
// 6425 rows, 16 heads, 27.3 us against 30.7 with a launch for it.  Parts of wide
// tiles, whose records are 66 KB, and the prefix's and own results of one row are
// joined by paged_combine_kernel (joining wide parts in place: 8 requests of 17
// tokens behind 1000 rows 50 us against 22).  Either way in part order, so results do
// not depend on the order of arrival.
#include "attn_common.h"
#include "paged.h"

namespace hkv {
namespace {

using namespace attn;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* lds_s16x4_ptr;
typedef __attribute__((address_space(3))) void* lds_void_ptr;

constexpr int kWideRows = 128;
constexpr int kNarrowRows = 16;
constexpr int kPlanned = 64;  // requests that each wave plans by itself
constexpr float kNoMax = -1e30f;

// ---------------------------------------------------------------- plan

// One launch: the requests' own rows, or (shared) the prefix for the rows of
// all requests together.
struct PagedPass {
  int32_t shared;       // one pseudo request: all live tokens, the prefix's keys
  int32_t with_prefix;  // each tile's keys begin with the prefix
  int32_t rows;         // rows of a tile
  int32_t tile_tokens;  // tokens that a tile spans at most
  int32_t least;        // chunks of a part at least
  int32_t wanted;       // units per K/V head that fill the card once
  int32_t most;         // ... and that parts may make at most
  int32_t cap;          // chunks of a part from which more than `wanted` are made
  int32_t step;         // parts are multiples of this many chunks (a power of two)
  int32_t uncut;        // tiles of up to this many chunks are not cut
  int32_t always;       // every tile leaves records (a shared prefix's are joined to them)
  int32_t combined;     // a combine launch follows: write meta
  int32_t join;         // the last part of a cut tile joins its records (counters)
  int32_t limit;        // records there is room for
  int32_t units;        // units there are workgroups for (per K/V head)
  const int4* list;     // the units' work, for more than kPlanned requests
  float* records;       // per record and K/V head: rows * D values, rows maxima, rows sums
  int2* meta;           // per live row: first record, parts | row in tile << 16
};

__device__ __forceinline__ int32_t uniform(int32_t v) { return __builtin_amdgcn_readfirstlane(v); }

__host__ __device__ __forceinline__ int64_t up_div(int64_t a, int32_t b) {
  // 32-bit where that does (64-bit divisions cost about 150 instructions)
  const int64_t n = a + b - 1;
  return n >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(n) / static_cast<uint32_t>(b)) : n / b;
}

// Chunks of a part in a launch of `total` chunks (per K/V head): enough units to fill
// the card once, more where parts would be longer than `cap`.
__host__ __device__ __forceinline__ int64_t part_chunks(const PagedPass& p, int64_t total) {
  int64_t c = up_div(total, p.wanted);
  if (c > p.cap) {
    c = up_div(total, p.most);
    c = c > p.cap ? c : p.cap;
  }
  c = c > p.least ? c : p.least;
  return (c + p.step - 1) & ~static_cast<int64_t>(p.step - 1);
}

struct Geometry {
  int32_t n;      // queries
  int32_t first;  // token of query 0
  int32_t len;    // rows
};

__device__ __forceinline__ int32_t clamp32(int32_t v, int32_t lo, int32_t hi) {
  return v < lo ? lo : (v > hi ? hi : v);
}

__device__ __forceinline__ int32_t live_tokens(const PagedAttnArgs& a) {
  return a.requests > 0 ? clamp32(a.query_starts[a.requests], 0, a.num_tokens) : 0;
}

// Tokens before the first request (none, as a rule).
__device__ __forceinline__ int32_t first_token(const PagedAttnArgs& a) {
  return clamp32(a.query_starts[0], 0, a.num_tokens);
}

__device__ __forceinline__ Geometry load_request(const PagedAttnArgs& a, const PagedPass& p, int32_t r) {
  Geometry g;
  if (p.shared) {
    g.first = 0;
    g.n = live_tokens(a);
    g.len = a.prefix_len;
    return g;
  }
  g.first = clamp32(a.query_starts[r], 0, a.num_tokens);
  g.n = clamp32(a.query_starts[r + 1], g.first, a.num_tokens) - g.first;
  g.len = clamp32(a.lengths[r], 0, a.table_width << a.block_shift);
  return g;
}

// The keys that queries [i0, i1] of a request see: rows [0, sinks) and
// [lo, hi), as chunks [0, na) and [b0, b0 + nb) behind the prefix's np.
struct Keys {
  int32_t lo, hi, sinks;
  int32_t np, na, b0, nb;
  __device__ __forceinline__ int32_t chunks() const { return np + na + nb; }
};

__device__ __forceinline__ Keys keys_of(const PagedAttnArgs& a, const PagedPass& p, const Geometry& g, int32_t i0,
                                        int32_t i1) {
  Keys k{0, 0, 0, 0, 0, 0, 0};
  if (p.shared) {
    k.hi = g.len;
  } else {
    const int32_t p0 = g.len - g.n + i0, p1 = g.len - g.n + i1;
    k.hi = p1 < 0 ? 0 : (a.causal ? p1 + 1 : g.len);
    if (a.window > 0 && p0 >= a.window) {
      k.lo = p0 - a.window + 1;
      k.sinks = a.sinks < k.hi ? a.sinks : k.hi;
      if (k.lo <= k.sinks) k.lo = k.sinks = 0;
    }
    if (p.with_prefix) k.np = (a.prefix_len + kBN - 1) / kBN;
  }
  if (k.hi > 0) {
    k.na = (k.sinks + kBN - 1) / kBN;
    k.b0 = k.lo / kBN > k.na ? k.lo / kBN : k.na;
    k.nb = (k.hi + kBN - 1) / kBN - k.b0;
    if (k.nb < 0) k.nb = 0;
  }
  return k;
}

struct Load {
  int32_t tiles, chunks;  // of a request: tiles of rows, chunks of a longest tile
};

__device__ __forceinline__ Load load_of(const PagedAttnArgs& a, const PagedPass& p, const Geometry& g) {
  const int32_t group = a.group;
  Load l{0, 0};
  if (g.n == 0) return l;
  l.tiles = (g.n * group + p.rows - 1) >> (p.rows == kWideRows ? 7 : 4);
  // causal: the last tile's, else the first's
  const int32_t span = g.n < p.tile_tokens ? g.n : p.tile_tokens;
  const int32_t i0 = a.causal && !p.shared ? g.n - span : 0;
  l.chunks = keys_of(a, p, g, i0, i0 + span - 1).chunks();
  return l;
}

struct Work {
  int32_t request;  // -1: none
  int32_t tile;
  int32_t part;
  int32_t parts;    // of the request's tiles
  int32_t record;   // of the tile's part 0
  Geometry g;       // of the request
  int32_t head, end;  // the requests' tokens
};

__device__ __forceinline__ int32_t parts_of(const PagedPass& p, const Load& l, int64_t c) {
  if (l.chunks <= c || l.chunks <= p.uncut) return 1;
  // wide tiles: to the nearest, so that a little over one round is not two
  if (p.rows == kWideRows) return (l.chunks + static_cast<int32_t>(c) / 2) / static_cast<int32_t>(c);
  return static_cast<int32_t>(up_div(l.chunks, static_cast<int32_t>(c)));
}

// Units, and records, of a request.
__device__ __forceinline__ int2 units_of(const PagedPass& p, const Load& l, int64_t c) {
  const int32_t parts = parts_of(p, l, c);
  const int32_t units = l.tiles * parts;
  return int2{units, parts > 1 || p.always ? units : 0};
}

// Sum, and prefix sums, of the first n lanes (the others hold zeros).
__device__ __forceinline__ int64_t wave_sum64(int64_t v, int n = 64) {
  for (int off = 1; off < n; off <<= 1) v += __shfl_xor(v, off, 64);
  return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int32_t>(v)))) |
                              static_cast<uint64_t>(uniform(static_cast<int32_t>(v >> 32))) << 32);
}

// Counts of units and records that more than can be launched do not overflow.
__device__ __forceinline__ int2 add_units(const int2& a, const int2& b) {
  constexpr int32_t kMost = 0x3fffffff;
  const int32_t x = a.x + b.x, y = a.y + b.y;
  return int2{x < kMost ? x : kMost, y < kMost ? y : kMost};
}

__device__ __forceinline__ int2 wave_prefix(int2 v, int n = 64) {
  const int lane = threadIdx.x & 63;
  for (int off = 1; off < n; off <<= 1) {
    const int2 o{__shfl_up(v.x, off, 64), __shfl_up(v.y, off, 64)};
    if (lane >= off) v = add_units(v, o);
  }
  return v;
}

// Work of unit `unit` (per K/V head): up to kPlanned requests every wave plans by
// itself, a request per lane.
__device__ __forceinline__ Work find_work(const PagedAttnArgs& a, const PagedPass& p, int32_t unit) {
  const int32_t R = p.shared ? 1 : a.requests;
  const int lane = threadIdx.x & 63;
  Work w{-1, 0, 0, 1, 0, {0, 0, 0}, 0, 0};
  if (R <= kPlanned) {
    Load l{0, 0};
    Geometry g{0, 0, 0};
    if (lane < R) {
      g = load_request(a, p, lane);
      l = load_of(a, p, g);
    }
    if (R > 0) {
      w.head = __builtin_amdgcn_readlane(g.first, 0);
      w.end = __builtin_amdgcn_readlane(g.first + g.n, R - 1);
      if (w.end < w.head) w.end = w.head;
    }
    const int64_t total = wave_sum64(static_cast<int64_t>(l.tiles) * l.chunks, R);
    const int64_t c = part_chunks(p, total);
    const int2 mine = units_of(p, l, c);
    const int2 end = wave_prefix(mine, R);
    const uint64_t hit = __ballot(lane < R && unit >= end.x - mine.x && unit < end.x);
    if (hit == 0) return w;
    const int src = __builtin_ctzll(hit);
    const int32_t parts = __builtin_amdgcn_readlane(parts_of(p, l, c), src);
    const int32_t in = uniform(unit - __builtin_amdgcn_readlane(end.x - mine.x, src));
    w.request = src;
    w.parts = parts;
    w.part = in % parts;
    w.tile = __builtin_amdgcn_readlane(l.tiles, src) - 1 - in / parts;  // causal tiles: longest first
    w.record = __builtin_amdgcn_readlane(end.y - mine.y, src) + w.tile * parts;
    w.g = Geometry{__builtin_amdgcn_readlane(g.n, src), __builtin_amdgcn_readlane(g.first, src),
                   __builtin_amdgcn_readlane(g.len, src)};
    return w;
  }
  // what paged_plan_kernel wrote
  const int4 x = p.list[2 * static_cast<int64_t>(unit)], y = p.list[2 * static_cast<int64_t>(unit) + 1];
  const int4 range = p.list[2 * static_cast<int64_t>(p.units)];
  w.head = uniform(range.x);
  w.end = uniform(range.y);
  w.request = uniform(x.x);
  w.tile = uniform(x.y);
  w.part = uniform(x.z);
  w.parts = uniform(x.w);
  w.record = uniform(y.x);
  w.g = Geometry{uniform(y.y), uniform(y.z), uniform(y.w)};
  return w;
}

// The work of every unit of a launch of more than kPlanned requests, 32 bytes each, and
// behind them the range of live tokens.  Each workgroup plans all requests, up to four
// to a thread, and finds its own units' requests by bisection.  256 threads up to 1024
// requests: 128 requests of 500 rows 56.6 us, with 1024 threads 57.7.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_plan_kernel(const PagedAttnArgs a, const PagedPass p,
                                                              int4* __restrict__ list) {
  constexpr int kWaves = kThreads / 64, kRun = kMaxRequests / 1024, kMost = kThreads * kRun;
  __shared__ int64_t wave_total[kWaves];
  __shared__ int2 wave_units[kWaves];
  __shared__ int32_t start[kMost], record[kMost], tiles[kMost], cut[kMost];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = tid >> 6;
  const int32_t R = a.requests;
  const int32_t run = (R + kThreads - 1) / kThreads;
  const int32_t r0 = tid * run;
  Load l[kRun];
  int64_t sum = 0;
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    l[i] = Load{0, 0};
    if (i < run && r0 + i < R) l[i] = load_of(a, p, load_request(a, p, r0 + i));
    sum += static_cast<int64_t>(l[i].tiles) * l[i].chunks;
  }
  sum = wave_sum64(sum);
  if (lane == 0) wave_total[wave] = sum;
  __syncthreads();
  int64_t total = 0;
  for (int i = 0; i < kWaves; ++i) total += wave_total[i];
  const int64_t c = part_chunks(p, total);
  int2 mine{0, 0};
#pragma unroll
  for (int i = 0; i < kRun; ++i) mine = add_units(mine, units_of(p, l[i], c));
  int2 end = wave_prefix(mine);
  if (lane == 63) wave_units[wave] = end;
  int2 at{__shfl_up(end.x, 1, 64), __shfl_up(end.y, 1, 64)};
  if (lane == 0) at = int2{0, 0};
  __syncthreads();
  int2 all{0, 0};
  for (int i = 0; i < kWaves; ++i) {
    if (i == wave) at = add_units(all, at);
    all = add_units(all, wave_units[i]);
  }
#pragma unroll
  for (int i = 0; i < kRun; ++i) {
    if (i >= run || r0 + i >= R) break;
    start[r0 + i] = at.x;
    record[r0 + i] = at.y;
    tiles[r0 + i] = l[i].tiles;
    cut[r0 + i] = parts_of(p, l[i], c);
    at = add_units(at, units_of(p, l[i], c));
  }
  __syncthreads();
  for (int32_t u = blockIdx.x * kThreads + tid; u < p.units; u += gridDim.x * kThreads) {
    int4 x{-1, 0, 0, 1}, y{0, 0, 0, 0};
    if (u < all.x) {
      int32_t r = 0;  // the last request that starts at or before u
      for (int32_t step = kMost / 2; step > 0; step >>= 1)
        if (r + step < R && start[r + step] <= u) r += step;
      const Geometry g = load_request(a, p, r);
      const int32_t in = u - start[r], parts = cut[r];
      const int32_t tile = tiles[r] - 1 - in / parts;  // causal tiles: longest first
      x = int4{r, tile, in % parts, parts};
      y = int4{record[r] + tile * parts, g.n, g.first, g.len};
    }
    list[2 * static_cast<int64_t>(u)] = x;
    list[2 * static_cast<int64_t>(u) + 1] = y;
  }
  if (blockIdx.x == 0 && tid == 0) {
    const int32_t head = first_token(a), last = live_tokens(a);
    list[2 * static_cast<int64_t>(p.units)] = int4{head, last < head ? head : last, 0, 0};
  }
}

// ---------------------------------------------------------------- a tile of rows

struct Tile {
  Geometry g;
  Keys keys;
  const int32_t* blocks;  // of the request's own keys (shared: the prefix's)
  int32_t row0, rows;     // rows of the request's matrix
  int32_t t0, t1;         // chunks of this part
  int32_t parts;          // of this tile
  int32_t one;            // all rows stand at one position
};

// Whether there is work; part and tile of `w` as its tile cuts them.
__device__ __forceinline__ bool make_tile(const PagedAttnArgs& a, const PagedPass& p, const Work& w, int32_t unit,
                                          Tile& t) {
  const int32_t group = a.group;
  t.g = w.g;
  t.row0 = w.tile * p.rows;
  t.rows = t.g.n * group - t.row0;
  t.rows = t.rows < p.rows ? t.rows : p.rows;
  if (w.tile < 0 || t.rows <= 0) return false;
  const int32_t i0 = t.row0 / group, i1 = (t.row0 + t.rows - 1) / group;
  t.one = i0 == i1;
  t.keys = keys_of(a, p, t.g, i0, i1);
  t.blocks = p.shared ? a.prefix_blocks : a.block_tables + w.request * a.table_stride;
  const int32_t n = t.keys.chunks();
  // a tile with fewer chunks than its request's longest is cut in fewer parts
  const int32_t most = n > p.uncut ? (n + p.least - 1) / p.least : 1;
  t.parts = w.parts < most ? w.parts : (most > 1 ? most : 1);
  // Where query_starts do not ascend, tiles may be more than the launch has room for:
  // one without a record or a unit for each part is not cut.
  if (w.record + w.parts > p.limit || unit - w.part + w.parts > p.units) {
    if (p.always) return false;
    t.parts = 1;
  }
  if (w.part >= t.parts) return false;
  const int32_t each = n / t.parts, more = n - each * t.parts;  // the first `more` parts have one chunk more
  t.t0 = each * w.part + (w.part < more ? w.part : more);
  t.t1 = t.t0 + each + (w.part < more ? 1 : 0);
  return true;
}

// First row of the part's t-th chunk, and whether it is the prefix's.
__device__ __forceinline__ int32_t chunk_row(const Keys& k, int32_t t, bool& prefix) {
  prefix = t < k.np;
  if (prefix) return t * kBN;
  t -= k.np;
  return (t < k.na ? t : t - k.na + k.b0) * kBN;
}

// The row to load for row j of a chunk: rows that no query of the tile sees
// (past the end, or between the sinks and the window) stand for one that is
// seen, so that their weight of 0 meets no stray NaN and no stale table entry.
__device__ __forceinline__ int32_t row_to_load(const PagedAttnArgs& a, const Keys& k, int32_t j, bool prefix) {
  if (prefix) return j < a.prefix_len ? j : a.prefix_len - 1;
  if (j >= k.hi) return k.hi - 1;
  if (j < k.lo && j >= k.sinks) return (j & ~(kBN - 1)) < k.sinks ? k.sinks - 1 : k.lo;
  return j;
}

// Byte offset in the cache of a request's row whose table entry is `id` (an
// entry outside the cache stands for block 0).  32-bit strides in bytes.
__device__ __forceinline__ int64_t row_offset(const PagedAttnArgs& a, const PagedCacheStrides& s, int32_t id,
                                              int32_t row) {
  const uint32_t b = static_cast<uint32_t>(id) < static_cast<uint32_t>(a.num_blocks) ? id : 0;
  const uint32_t r = row & ((1 << a.block_shift) - 1);
  return static_cast<int64_t>(static_cast<uint64_t>(b) * static_cast<uint32_t>(s.block * 2) +
                              r * static_cast<uint32_t>(s.row * 2));
}

// What a query (row of the matrix) sees of its request's own rows.
struct Sight {
  int32_t lo, hi;
};

__device__ __forceinline__ Sight sight_of(const PagedAttnArgs& a, const PagedPass& p, const Geometry& g, int32_t i) {
  Sight s{0, g.len};
  if (!p.shared) {
    const int32_t pos = g.len - g.n + i;
    if (pos < 0) s.hi = 0;
    else if (a.causal) s.hi = pos + 1;
    if (a.window > 0 && pos >= a.window) s.lo = pos - a.window + 1;
  }
  return s;
}

// Whether each query of the tile sees each row of the 64 (or `n`) from j.
__device__ __forceinline__ bool all_seen(const PagedAttnArgs& a, const Sight& first, const Sight& last, int32_t j,
                                         bool prefix, int32_t n = kBN) {
  if (prefix) return j + n <= a.prefix_len;
  return j + n <= first.hi && (j >= last.lo || j + n <= a.sinks);
}

// 16 bytes per lane from `src` straight to LDS at lds + 16 lane (uniform lds).
// Inline assembly, so that the compiler, which cannot see the LDS write, does not
// make LDS reads wait for every load: the kernels wait themselves.  M0 is
// written here and nothing else in these kernels uses it.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dword %1, off" : : "s"(lds), "v"(src) : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_ptr)(p)));
}

__device__ __forceinline__ u32x2_t ds_read_tr(const uint8_t* p) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(p)));
}

// Takes the values that are not finite out of an operand: 1 in `up` for +inf and
// NaN, in `down` for -inf and NaN.
template <int DT>
__device__ __forceinline__ void split_finite(u32x4_t& v, u32x4_t& up, u32x4_t& down) {
  constexpr uint32_t kExp = DT == kF16 ? 0x7c00u : 0x7f80u;
  constexpr uint32_t kOne = DT == kF16 ? 0x3c00u : 0x3f80u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t x[2] = {v[i] & 0xffffu, v[i] >> 16};
    uint32_t keep[2], hi[2], lo[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const bool odd = (x[k] & kExp) == kExp;
      const bool nan = odd && (x[k] & 0x7fffu) != kExp;
      keep[k] = odd ? 0u : x[k];
      hi[k] = odd && (nan || x[k] < 0x8000u) ? kOne : 0u;
      lo[k] = odd && (nan || x[k] >= 0x8000u) ? kOne : 0u;
    }
    v[i] = keep[0] | keep[1] << 16;
    up[i] = hi[0] | hi[1] << 16;
    down[i] = lo[0] | lo[1] << 16;
  }
}

// Zeros (lse -inf) for the tokens outside [head, live), the requests', shared by
// all workgroups.
template <int kThreads>
__device__ __forceinline__ void fill_tail(const PagedAttnArgs& a, int32_t head, int32_t live, int32_t block,
                                          int32_t blocks) {
  const int64_t row = static_cast<int64_t>(a.heads) * (a.head_dim / 8);  // 16-byte pieces of a token
  const int64_t gap = live - head;
  uint4* const out = reinterpret_cast<uint4*>(a.out);
  const int64_t at = static_cast<int64_t>(block) * kThreads + threadIdx.x % kThreads;
  const int64_t step = static_cast<int64_t>(blocks) * kThreads;
  for (int64_t i = at; i < (a.num_tokens - gap) * row; i += step)
    out[i < head * row ? i : i + gap * row] = uint4{0, 0, 0, 0};
  if (a.lse == nullptr) return;
  const int64_t rest = a.num_tokens - gap;
  for (int64_t i = at; i < rest * a.heads; i += step) {
    const int64_t t = i % rest;
    a.lse[(i / rest) * a.num_tokens + (t < head ? t : t + gap)] = -__builtin_inff();
  }
}

// Record of (part of a tile, K/V head).
template <int D>
__device__ __forceinline__ float* record_of(const PagedAttnArgs& a, const PagedPass& p, int32_t record, int32_t kvh) {
  return p.records + (static_cast<int64_t>(record) * a.kv_heads + kvh) * (p.rows * (D + 2));
}

template <int kThreads>
__device__ __forceinline__ void write_meta(const PagedAttnArgs& a, const PagedPass& p, const Tile& t, const Work& w,
                                           int32_t kvh) {
  if (!p.combined || w.part != 0 || kvh != 0) return;
  const int32_t group = a.group;
  for (int32_t i = threadIdx.x % kThreads; i < t.rows; i += kThreads)
    p.meta[static_cast<int64_t>(t.g.first) * group + t.row0 + i] = int2{w.record, t.parts | i << 16};
}

// ---------------------------------------------------------------- wide tiles
//
// Four waves of 32 rows; per 64-key chunk S^T = K Q^T and O^T += V^T P^T on the
// 32x32x16 MFMAs, softmax in the exp2 domain with a lazily moved maximum, as
// the segmented kernel (seg_attn_direct.hip, whose operand order in LDS this
// one shares): chunks go straight to LDS, two stages, K one chunk ahead of V, so
// iteration t runs S(t + 1) on the matrix cores beside the exponentials of S(t).
// Waves 0 and 1 load the K rows, 2 and 3 the V rows, each lane the rows of its
// own (its address is made once per lane and chunk, V lanes take theirs from LDS:
// 560 against 598 us a prompt of 8192 with an address for each of a V lane's four
// rows); the table entries of the next chunk are read one iteration ahead.
template <int D>
struct WideLds {
  static constexpr int kTensor = kBN * D * 2;  // bytes of a chunk's K or V
  static constexpr int kStage = 2 * kTensor;
  static constexpr int kPitch = D * 2 + 16;    // of a row of the output
  uint8_t ring[2 * kStage < 4 * 32 * kPitch ? 4 * 32 * kPitch : 2 * kStage];
  const uint8_t* v_rows[2][32];
};

// Workgroup `block` of `blocks`.
template <int DT, int D>
__device__ __forceinline__ void wide_tile(const PagedAttnArgs& a, const PagedPass& p, const Scalars& sc,
                                          int32_t block, int32_t blocks, WideLds<D>& lds_wide) {
  constexpr int kThreads = 256;
  constexpr int KS = D / 16;               // k-steps of S
  constexpr int DB = D / 32;               // 32-wide blocks of O
  constexpr int NP = D / 64;               // V DMAs per 8 rows
  constexpr int kTensor = WideLds<D>::kTensor;
  constexpr int kStage = WideLds<D>::kStage;
  constexpr int kPitch = WideLds<D>::kPitch;
  uint8_t* const ring = lds_wide.ring;
  auto& v_rows = lds_wide.v_rows;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 5;
  const int32_t group = a.group;
  const int32_t unit = block / a.kv_heads;
  const int32_t kvh = block - unit * a.kv_heads;
  const Work w = find_work(a, p, unit);
  if (a.fill_tail && !p.shared && w.end - w.head < a.num_tokens)
    fill_tail<kThreads>(a, w.head, w.end, block, blocks);
  Tile t;
  if (w.request < 0 || !make_tile(a, p, w, unit, t)) return;
  write_meta<kThreads>(a, p, t, w, kvh);

  // this lane's row (rows past the tile's last repeat it and are not stored)
  const int32_t row = wave * 32 + (lane & 31);
  const int32_t mat = t.row0 + (row < t.rows ? row : t.rows - 1);
  const int32_t tok = mat / group;
  const Sight mine = sight_of(a, p, t.g, tok);
  const Sight first = sight_of(a, p, t.g, t.row0 / group);
  const Sight last = sight_of(a, p, t.g, (t.row0 + t.rows - 1) / group);
  u32x4_t qf[KS];
  {
    const uint16_t* const q = static_cast<const uint16_t*>(a.q) + (t.g.first + tok) * a.q_token +
                              (kvh * group + (mat - tok * group)) * a.q_head + g * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4_t*>(q + ks * 16);
  }

  f32x16_t oacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) oacc[i] = f32x16_t{};
  float m_run = kNoMax, l_run = 0.f;

  if (t.t0 < t.t1) {
    // Rows of this wave in a chunk: [32 half, + 32), a row's address per lane.  K
    // lanes load their own row, V lanes rows 8 i + 4 (lp / 16) + (lp % 8) / 2, i < 4.
    const bool k_wave = wave < 2;
    const int half = wave & 1;
    const int lp = lane & 31;
    const int v_row = 4 * (lp >> 4) + ((lp & 7) >> 1);
    const int col = k_wave ? 16 * g : 2 * (32 * g + 16 * ((lp >> 3) & 1) + 8 * (lp & 1));
    const PagedCacheStrides cs = k_wave ? a.ks : a.vs;
    const uint8_t* const cache = static_cast<const uint8_t*>(k_wave ? a.k_cache : a.v_cache) + kvh * cs.head * 2;
    const uint32_t lds = lds_address(ring) + (k_wave ? half * (KS * 1024) : kTensor + half * (4 * NP * 1024));
    int32_t my_row = 0, my_id = 0;
    // the table entry of this lane's row of the chunk at stream position c
    auto look_up = [&](int32_t c) {
      bool prefix;
      const int32_t j0 = chunk_row(t.keys, c, prefix) + 32 * half;
      my_row = row_to_load(a, t.keys, j0 + lp, prefix);
      my_id = (prefix ? a.prefix_blocks : t.blocks)[my_row >> a.block_shift];
    };
    // the chunk that was looked up, into stage c % 2
    auto issue = [&](int32_t c) {
      const uint32_t dst = lds + (c & 1) * kStage;
      const uint8_t* const mine = cache + row_offset(a, cs, my_id, my_row);
      if (k_wave) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) dma16(mine + col + 32 * ks, dst + 1024 * ks);
      } else {
        v_rows[half][lp] = mine;
        __builtin_amdgcn_wave_barrier();  // a wave's LDS operations run in order
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint8_t* const src = v_rows[half][8 * i + v_row] + col;
#pragma unroll
          for (int n = 0; n < NP; ++n) dma16(src + 128 * n, dst + 1024 * (i * NP + n));
        }
      }
    };

    auto qk = [&](f32x16_t (&sx)[2], int32_t c) {
      const uint8_t* const kst = ring + (c & 1) * kStage + lane * 16;
      sx[0] = f32x16_t{};
      sx[1] = f32x16_t{};
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          sx[kb] = mfma32<DT>(*reinterpret_cast<const u32x4_t*>(kst + (kb * KS + ks) * 1024), qf[ks], sx[kb]);
    };
    auto v_operand = [&](const uint8_t* vst, int u, int db) {
      const uint8_t* const at = vst + (u * 2 * NP + (db >> 1)) * 1024 + (db & 1) * 512;
      const u32x2_t lo = ds_read_tr(at), hi = ds_read_tr(at + NP * 1024);
      return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
    };
    auto pv = [&](const u32x4_t (&pf)[4], int32_t c) {
      const uint8_t* const vst = ring + (c & 1) * kStage + kTensor + lane * 8;
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] = mfma32<DT>(v_operand(vst, u, db), pf[u], oacc[db]);
    };
    // Rows of chunk c that this lane's query does not see: score -inf.
    auto hide = [&](f32x16_t (&sx)[2], int32_t j0, bool prefix) {
      const int32_t hi = (prefix ? a.prefix_len : mine.hi) - j0 - 4 * g;
      const int32_t lo = (prefix ? 0 : mine.lo) - j0 - 4 * g;
      const int32_t sinks = a.sinks - j0 - 4 * g;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int32_t j = kb * 32 + 8 * (i >> 2) + (i & 3);
          sx[kb][i] = (j >= hi) | ((j < lo) & (j >= sinks)) ? -__builtin_inff() : sx[kb][i];
        }
    };
    auto pack = [&](const f32x16_t (&sx)[2], u32x4_t (&pf)[4]) {
#pragma unroll
      for (int u = 0; u < 4; ++u) pf[u] = p_operand<DT>(sx, u);
    };
    auto move = [&](float mx) {
      if (__any(mx - m_run > sc.thresh)) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * sc.c);
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
        m_run = m_new;
      }
    };
    auto hidden = [&](int32_t c, int32_t& j0, bool& prefix) {
      j0 = chunk_row(t.keys, c, prefix);
      return !all_seen(a, first, last, j0, prefix);
    };

    // Prologue: chunk t0 whole, K(t0 + 1) in flight; V waves look up t0 + 1, K waves t0 + 2.
    look_up(t.t0);
    issue(t.t0);
    if (t.t0 + 1 < t.t1) look_up(t.t0 + 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] ^= sc.q_sign;
    wait_vmcnt<0>();
    __syncthreads();
    if (k_wave && t.t0 + 1 < t.t1) {
      issue(t.t0 + 1);
      if (t.t0 + 2 < t.t1) look_up(t.t0 + 2);
    }
    f32x16_t sa[2], sb[2];
    int32_t j0;
    bool prefix;
    qk(sa, t.t0);
    if (hidden(t.t0, j0, prefix)) hide(sa, j0, prefix);
    move(tile_max(sa));

    auto weigh = [&](f32x16_t (&s)[2], int32_t c) {
      u32x4_t pf[4];
      exp_tile(s, m_run, sc.c, l_run);
      pack(s, pf);
      pv(pf, c);
    };
    auto step = [&](f32x16_t (&cur)[2], f32x16_t (&next)[2], int32_t c) {
      wait_vmcnt<0>();
      __syncthreads();
      const int32_t ahead = c + (k_wave ? 2 : 1);
      if (ahead < t.t1) {
        issue(ahead);
        if (ahead + 1 < t.t1) look_up(ahead + 1);
      }
      qk(next, c + 1);
      weigh(cur, c);
      asm volatile("" : "+v"(l_run));
      float mx = tile_max(next);
      asm volatile("" : "+v"(mx));
      if (hidden(c + 1, j0, prefix)) {
        hide(next, j0, prefix);
        mx = tile_max(next);
      }
      move(mx);
    };
    int32_t c = t.t0;
    for (; c + 2 < t.t1; c += 2) {
      step(sa, sb, c);
      step(sb, sa, c + 1);
    }
    const bool two = c + 1 < t.t1;
    if (two) step(sa, sb, c++);
    wait_vmcnt<0>();
    __syncthreads();
    if (two) weigh(sb, c);
    else weigh(sa, c);

    // A V value that is not finite in a chunk that some queries see only in part
    // has reached the others through a weight of 0.  Where the result shows
    // one, the tile runs again, chunk by chunk and with the same arithmetic,
    // without such values, and each is added to the queries that see it.
    if (!t.one) {
      float z = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) z = __builtin_fmaf(oacc[db][i], 0.f, z);
      if (__builtin_expect(__syncthreads_or(z != 0.f), 0)) {
#pragma unroll
        for (int i = 0; i < DB; ++i) oacc[i] = f32x16_t{};
        m_run = kNoMax;
        l_run = 0.f;
#pragma unroll 1
        for (c = t.t0; c < t.t1; ++c) {
          __syncthreads();
          look_up(c);
          issue(c);
          wait_vmcnt<0>();
          __syncthreads();
          __builtin_amdgcn_sched_barrier(0);
          qk(sa, c);
          if (hidden(c, j0, prefix)) hide(sa, j0, prefix);
          move(tile_max(sa));
          u32x4_t pf[4];
          exp_tile(sa, m_run, sc.c, l_run);
          pack(sa, pf);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sa[kb][i] = 1.f;
          hide(sa, j0, prefix);
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sa[kb][i] = fmaxf(sa[kb][i], 0.f);
          u32x4_t seen[4];
          pack(sa, seen);
          __builtin_amdgcn_sched_barrier(0);
          const uint8_t* const vst = ring + (c & 1) * kStage + kTensor + lane * 8;
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            f32x16_t above{}, below{};  // how many +inf or NaN, -inf or NaN each query sees
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              u32x4_t v = v_operand(vst, u, db), up, down;
              split_finite<DT>(v, up, down);
              oacc[db] = mfma32<DT>(v, pf[u], oacc[db]);
              above = mfma32<DT>(up, seen[u], above);
              below = mfma32<DT>(down, seen[u], below);
              __builtin_amdgcn_sched_barrier(0);  // as few registers as it takes
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if (above[i] > 0.f) oacc[db][i] += __builtin_inff();
              if (below[i] > 0.f) oacc[db][i] -= __builtin_inff();
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  }

  const float l = pair_sum(l_run);
  if (t.parts > 1 || p.always) {
    float* const rec = record_of<D>(a, p, w.record + w.part, kvh);
    if (row < t.rows) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int jb = 0; jb < 4; ++jb)
          *reinterpret_cast<f32x4_t*>(rec + row * D + db * 32 + 8 * jb + 4 * g) =
              f32x4_t{oacc[db][4 * jb], oacc[db][4 * jb + 1], oacc[db][4 * jb + 2], oacc[db][4 * jb + 3]};
      if (g == 0) {
        rec[p.rows * D + row] = m_run;
        rec[p.rows * (D + 1) + row] = l;
      }
    }
    return;
  }
  // Output through LDS, whole rows per store.  A row that sees nothing has l = 0.
  const float inv = l == 0.f ? 0.f : 1.f / l;
  __syncthreads();  // every wave is past its last chunk: the ring is free
  uint8_t* const stage = ring + wave * 32 * kPitch;
  uint8_t* const own = stage + (lane & 31) * kPitch;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int jb = 0; jb < 4; ++jb) {
      u32x2_t o;
      o[0] = pack2<DT>(oacc[db][4 * jb + 0] * inv, oacc[db][4 * jb + 1] * inv);
      o[1] = pack2<DT>(oacc[db][4 * jb + 2] * inv, oacc[db][4 * jb + 3] * inv);
      *reinterpret_cast<u32x2_t*>(own + (db * 32 + 8 * jb + 4 * g) * 2) = o;
    }
  __builtin_amdgcn_wave_barrier();  // a wave's LDS operations run in order
  constexpr int kLanes = D / 8;     // lanes per row
  constexpr int kAtOnce = 64 / kLanes;
#pragma unroll
  for (int k = 0; k < 32 / kAtOnce; ++k) {
    const int r = k * kAtOnce + lane / kLanes;
    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(stage + r * kPitch + (lane % kLanes) * 16);
    if (wave * 32 + r < t.rows) {
      const int32_t mr = t.row0 + wave * 32 + r;
      const int32_t i = mr / group;
      const int64_t at = (static_cast<int64_t>(t.g.first + i) * a.heads + kvh * group + (mr - i * group)) * D;
      *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(a.out) + at + (lane % kLanes) * 8) = v;
    }
  }
  if (a.lse != nullptr && g == 0 && row < t.rows)
    a.lse[static_cast<int64_t>(kvh * group + (mat - tok * group)) * a.num_tokens + t.g.first + tok] =
        l == 0.f ? -__builtin_inff() : (m_run * sc.c + __log2f(l)) * 0.6931471805599453f;
}

template <int DT, int D>
__global__ __launch_bounds__(256, 2) void paged_wide_kernel(const PagedAttnArgs a, const PagedPass p,
                                                            const Scalars sc) {
  __shared__ __attribute__((aligned(1024))) WideLds<D> lds;
  wide_tile<DT, D>(a, p, sc, static_cast<int32_t>(blockIdx.x), static_cast<int32_t>(gridDim.x), lds);
}

// ---------------------------------------------------------------- narrow tiles
//
// 16 rows on the 16x16x32 MFMAs; bound by the bytes of the cache.  The 32-key
// halves of the part's chunks are dealt to NW waves, each with its own stages in
// LDS and its own softmax, joined at the end: no barrier in the loop.  Per stage a wave sends 32
// rows of K and of V straight to LDS, whole rows side by side (16-byte pieces of
// a row exchanged by its number, so that reads of one piece from 16 rows meet
// 16 different banks).  Row addresses come from table entries that arrive in LDS
// the same way, NS stages ahead of the rows, so no load is waited for but by
// count: a group is the rows of stage k and the entries of stage k + NS, and NS - 1
// younger groups stay in flight.  128 KB of the cache are in flight per CU either
// way: two workgroups of two waves with two stages, or one of eight waves with one.
template <int DT>
__device__ __forceinline__ f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                   c, 0, 0, 0);
}

// Maximum / sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48 of a query.
__device__ __forceinline__ float quad_max(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return pair_max(fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])),
                        __builtin_bit_cast(float, static_cast<uint32_t>(r[1]))));
}
__device__ __forceinline__ float quad_sum(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v);
  const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
  return pair_sum(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])) +
                  __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

// 8 bytes of a record, coherent across the XCDs (attn_common.h has the reasons).
__device__ __forceinline__ f32x2_t ld_agent2(const float* p) {
  return __builtin_bit_cast(f32x2_t, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT));
}

// Counts in a part of a cut tile, whose record every wave has written its share of;
// true, in all waves, for the last one to do so.  Nothing waits: a part that is not
// the last is done.
__device__ __forceinline__ bool last_part(const PagedAttnArgs& a, const Tile& t, const Work& w, int32_t kvh,
                                          int32_t& turn) {
  int32_t* const counter = a.counters + 2 * (static_cast<int64_t>(w.record) * a.kv_heads + kvh);
  wait_vmcnt<0>();  // the record is written before it is counted
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last =
        __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == t.parts - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    turn = last;
  }
  __syncthreads();
  return turn != 0;
}

// The last part of a cut tile joins the records of all in part order, a wave per row.
template <int DT, int D, int NW>
__device__ __forceinline__ void join_parts(const PagedAttnArgs& a, const PagedPass& p, const Scalars& sc,
                                           const Tile& t, const Work& w, int32_t kvh) {
  const int lane = threadIdx.x & 63;
  const int wave = uniform(threadIdx.x >> 6);
  constexpr int kLanes = D / 2;         // of a part's row
  constexpr int kAtOnce = 64 / kLanes;  // parts per load
  const int32_t group = a.group;
  const int64_t stride = static_cast<int64_t>(a.kv_heads) * (p.rows * (D + 2));
  const float* const rec0 = record_of<D>(a, p, w.record, kvh);
  for (int32_t row = wave; row < t.rows; row += NW) {
    float top = kNoMax, sum = 0.f;
    f32x2_t acc{};
    for (int32_t q0 = 0; q0 < t.parts; q0 += 64) {
      const int32_t count = t.parts - q0 < 64 ? t.parts - q0 : 64;
      float pm = kNoMax, pl = 0.f;
      if (lane < count) {
        const float* const ml = rec0 + (q0 + lane) * stride + p.rows * D + row;
        pm = ld_agent(ml);
        pl = ld_agent(ml + p.rows);
      }
      float mn = pm;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
      mn = fmaxf(top, mn);
      const float x = __builtin_amdgcn_exp2f((top - mn) * sc.c), y = __builtin_amdgcn_exp2f((pm - mn) * sc.c);
      float add = pl * y;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) add += __shfl_xor(add, off, 64);
      sum = sum * x + add;
      top = mn;
      acc *= x;
      const float* const o = rec0 + q0 * stride + row * D + (lane % kLanes) * 2;
#pragma unroll 1
      for (int32_t base = 0; base < count; base += 8 * kAtOnce) {
        f32x2_t v[8];
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int32_t mine = base + i * kAtOnce + lane / kLanes;
          const int32_t at = mine < count ? mine : 0;
          v[i] = ld_agent2(o + at * stride);
          z[i] = __shfl(y, at, 64);
          if (mine >= count) v[i] = f32x2_t{};
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc += v[i] * z[i];
      }
    }
    if constexpr (kAtOnce > 1) {
      acc[0] += __shfl_xor(acc[0], 32, 64);
      acc[1] += __shfl_xor(acc[1], 32, 64);
    }
    const int32_t mat = t.row0 + row;
    const int32_t tok = mat / group;
    const int32_t head = kvh * group + (mat - tok * group);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t at = static_cast<int64_t>(t.g.first + tok) * a.heads + head;
    if (lane < kLanes)
      *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at * D + lane * 2) =
          pack2<DT>(acc[0] * inv, acc[1] * inv);
    if (a.lse != nullptr && lane == 0)
      a.lse[static_cast<int64_t>(head) * a.num_tokens + t.g.first + tok] =
          sum == 0.f ? -__builtin_inff() : (top * sc.c + __log2f(sum)) * 0.6931471805599453f;
  }
}

// A wave's LDS: NS stages of 32 rows of K and V, their table entries, row addresses.
template <int D, int NS>
struct NarrowLds {
  uint8_t ring[NS * 2 * 32 * D * 2];
  int32_t ids[NS][64];
  const uint8_t* rows[2][32];
};

// Workgroup `block` of `blocks`, or (PAIR) one of the two in a workgroup of twice the
// waves: they meet at the one barrier and nowhere else.
template <int DT, int D, int NW, int NS, bool PAIR = false>
__device__ __forceinline__ void narrow_tile(const PagedAttnArgs& a, const PagedPass& p, const Scalars& sc,
                                            int32_t block, int32_t blocks, NarrowLds<D, NS> (&lds_waves)[NW],
                                            int32_t& turn) {
  constexpr int kThreads = NW * 64;
  constexpr int kKeys = 32;                // of a stage
  constexpr int kRow = D * 2;              // bytes
  constexpr int kTensor = kKeys * kRow;
  constexpr int kStage = 2 * kTensor;
  constexpr int NI = kTensor / 1024;       // DMAs of K, and of V, per stage
  constexpr int kGroup = 2 * NI + 1;       // ... and one of table entries
  constexpr int KS = D / 32;               // k-steps of S
  constexpr int DB = D / 16;               // 16-wide blocks of O
  constexpr int kPieces = D / 8;           // 16-byte pieces of a row
  const int tid = threadIdx.x % kThreads;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int q = lane & 15;
  const int g = lane >> 4;
  const int32_t group = a.group;
  const int32_t unit = block / a.kv_heads;
  const int32_t kvh = block - unit * a.kv_heads;
  if (PAIR && block >= blocks) {
    __syncthreads();
    return;
  }
  const Work w = find_work(a, p, unit);
  if (a.fill_tail && !p.shared && w.end - w.head < a.num_tokens)
    fill_tail<kThreads>(a, w.head, w.end, block, blocks);
  Tile t;
  if (w.request < 0 || !make_tile(a, p, w, unit, t)) {
    if constexpr (PAIR) __syncthreads();
    return;
  }
  write_meta<kThreads>(a, p, t, w, kvh);

  const int32_t mat = t.row0 + (q < t.rows ? q : t.rows - 1);
  const int32_t tok = mat / group;
  const int32_t head = kvh * group + (mat - tok * group);
  const Sight mine = sight_of(a, p, t.g, tok);
  const Sight first = sight_of(a, p, t.g, t.row0 / group);
  const Sight last = sight_of(a, p, t.g, (t.row0 + t.rows - 1) / group);

  NarrowLds<D, NS>& my = lds_waves[wave];
  const uint32_t ring_lds = lds_address(my.ring);
  // the part's 32-key halves of chunks are dealt to the waves in turn
  const int32_t n = (2 * (t.t1 - t.t0) - wave + NW - 1) / NW;
  const auto stage_row = [&](int32_t k, bool& prefix) {
    const int32_t s = (k < n ? k : n - 1) * NW + wave;
    return chunk_row(t.keys, t.t0 + (s >> 1), prefix) + kKeys * (s & 1);
  };
  // Lanes l and l + 32 stand for row l % 32 of a stage, one for K, one for V.
  auto look_up = [&](int32_t k) {
    bool prefix;
    const int32_t j = stage_row(k, prefix) + (lane & 31);
    dma4((prefix ? a.prefix_blocks : t.blocks) + (row_to_load(a, t.keys, j, prefix) >> a.block_shift),
         lds_address(my.ids[k % NS]));
  };
  const bool for_k = lane < 32;
  PagedCacheStrides cs;
  cs.block = for_k ? a.ks.block : a.vs.block;
  cs.row = for_k ? a.ks.row : a.vs.row;
  const uint8_t* const cache = static_cast<const uint8_t*>(for_k ? a.k_cache : a.v_cache) +
                               kvh * (for_k ? a.ks.head : a.vs.head) * 2;
  auto issue = [&](int32_t k) {
    bool prefix;
    const int32_t r = row_to_load(a, t.keys, stage_row(k, prefix) + (lane & 31), prefix);
    my.rows[lane >> 5][lane & 31] = cache + row_offset(a, cs, my.ids[k % NS][lane], r);
    const uint32_t dst = ring_lds + (k % NS) * kStage;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      constexpr int kLanes = kPieces;  // lanes of a row
      const int row = i * (64 / kLanes) + lane / kLanes;
      const int piece = (lane % kLanes) ^ (D == 128 ? row & 15 : (row >> 1) & 7);
      dma16(my.rows[0][row] + piece * 16, dst + i * 1024);
      dma16(my.rows[1][row] + piece * 16, dst + kTensor + i * 1024);
    }
  };

  f32x4_t oacc[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) oacc[i] = f32x4_t{};
  float m_run = kNoMax, l_run = 0.f;
  u32x4_t qf[KS];

  const int k_swap = D == 128 ? q : q >> 1;
  const int v_row = 4 * g + (q >> 2);
  const int v_swap = D == 128 ? v_row : v_row >> 1;
  auto scores = [&](f32x4_t (&s)[2], const uint8_t* st) {
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      s[kb] = f32x4_t{};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        s[kb] = mfma16<DT>(
            *reinterpret_cast<const u32x4_t*>(st + (16 * kb + q) * kRow + (((4 * ks + g) ^ k_swap) * 16)), qf[ks], s[kb]);
    }
  };
  auto hide = [&](f32x4_t (&s)[2], int32_t j0, bool prefix) {
    const int32_t hi = (prefix ? a.prefix_len : mine.hi) - j0 - 4 * g;
    const int32_t lo = (prefix ? 0 : mine.lo) - j0 - 4 * g;
    const int32_t sinks = a.sinks - j0 - 4 * g;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int32_t j = 16 * kb + i;
        s[kb][i] = (j >= hi) | ((j < lo) & (j >= sinks)) ? -__builtin_inff() : s[kb][i];
      }
  };
  auto weigh = [&](f32x4_t (&s)[2]) {
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = quad_max(mx);
    if (__any(mx - m_run > sc.thresh)) {
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f((m_run - m_new) * sc.c);
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] *= alpha;
      m_run = m_new;
    }
    const float mc = m_run * sc.c;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][i], sc.c, -mc));
    l_run += ((s[0][0] + s[0][1]) + (s[0][2] + s[0][3])) + ((s[1][0] + s[1][1]) + (s[1][2] + s[1][3]));
  };
  // P^T's k slots 8 g .. + 7 are keys 4 g .. + 3 and 16 + 4 g .. + 3, as S^T leaves the MFMA
  auto pack = [&](const f32x4_t (&s)[2]) {
    return u32x4_t{pack2<DT>(s[0][0], s[0][1]), pack2<DT>(s[0][2], s[0][3]), pack2<DT>(s[1][0], s[1][1]),
                   pack2<DT>(s[1][2], s[1][3])};
  };
  auto v_operand = [&](const uint8_t* st, int db) {
    const uint8_t* const at =
        st + kTensor + v_row * kRow + (((2 * db + ((q & 3) >> 1)) ^ v_swap) * 16) + (q & 1) * 8;
    const u32x2_t lo = ds_read_tr(at), hi = ds_read_tr(at + 16 * kRow);
    return u32x4_t{lo[0], lo[1], hi[0], hi[1]};
  };

  if (n > 0) {
#pragma unroll
    for (int k = 0; k < NS; ++k)
      if (k < n) look_up(k);
    {
      const uint16_t* const src = static_cast<const uint16_t*>(a.q) + (t.g.first + tok) * a.q_token + head * a.q_head +
                                  g * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const u32x4_t*>(src + ks * 32);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) qf[ks] ^= sc.q_sign;
    }
    wait_vmcnt<0>();
#pragma unroll
    for (int k = 0; k < NS; ++k)
      if (k < n) {
        issue(k);
        look_up(k + NS);
      }
    for (int32_t k = 0; k < n; ++k) {
      // stage k and its successors' entries have landed; up to NS - 1 groups stay in flight
      const int32_t rest = n - 1 - k;
      if (rest >= NS - 1) wait_vmcnt<(NS - 1) * kGroup>();
      else if (NS > 3 && rest == 2) wait_vmcnt<(NS > 3 ? 2 : 0) * kGroup>();
      else if (NS > 2 && rest == 1) wait_vmcnt<(NS > 2 ? 1 : 0) * kGroup>();
      else wait_vmcnt<0>();
      asm volatile("" ::: "memory");
      const uint8_t* const st = my.ring + (k % NS) * kStage;
      bool prefix;
      const int32_t j0 = stage_row(k, prefix);
      f32x4_t s[2];
      scores(s, st);
      if (!all_seen(a, first, last, j0, prefix, kKeys)) hide(s, j0, prefix);
      weigh(s);
      const u32x4_t pf = pack(s);
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[db] = mfma16<DT>(v_operand(st, db), pf, oacc[db]);
      if (k + NS < n) {
        // the stage's reads are done before it is written again
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        issue(k + NS);
        look_up(k + 2 * NS);
      }
    }
    // Again without values that are not finite, as in the wide kernel; a wave is on its own here.
    if (!t.one) {
      float z = 0.f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) z = __builtin_fmaf(oacc[db][i], 0.f, z);
      if (__builtin_expect(__any(z != 0.f), 0)) {
#pragma unroll
        for (int i = 0; i < DB; ++i) oacc[i] = f32x4_t{};
        m_run = kNoMax;
        l_run = 0.f;
#pragma unroll 1
        for (int32_t k = 0; k < n; ++k) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          look_up(k);
          wait_vmcnt<0>();
          issue(k);
          wait_vmcnt<0>();
          asm volatile("" ::: "memory");
          const uint8_t* const st = my.ring + (k % NS) * kStage;
          bool prefix;
          const int32_t j0 = stage_row(k, prefix);
          f32x4_t s[2];
          scores(s, st);
          if (!all_seen(a, first, last, j0, prefix, kKeys)) hide(s, j0, prefix);
          weigh(s);
          const u32x4_t pf = pack(s);
          s[0] = s[1] = f32x4_t{1.f, 1.f, 1.f, 1.f};
          hide(s, j0, prefix);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = fmaxf(s[i >> 2][i & 3], 0.f);
          const u32x4_t seen = pack(s);
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            u32x4_t v = v_operand(st, db), up, down;
            split_finite<DT>(v, up, down);
            oacc[db] = mfma16<DT>(v, pf, oacc[db]);
            const f32x4_t above = mfma16<DT>(up, seen, f32x4_t{}), below = mfma16<DT>(down, seen, f32x4_t{});
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (above[i] > 0.f) oacc[db][i] += __builtin_inff();
              if (below[i] > 0.f) oacc[db][i] -= __builtin_inff();
            }
          }
        }
      }
    }
  }
  float l = quad_sum(l_run);

  // the waves' results are joined in their order, each wave taking its share of the dimensions
  constexpr int kMine = (DB + NW - 1) / NW;
  float* const left = reinterpret_cast<float*>(my.ring);
#pragma unroll
  for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4_t*>(left + (db * 64 + lane) * 4) = oacc[db];
  left[DB * 256 + lane] = m_run;
  left[DB * 256 + 64 + lane] = l;
  __syncthreads();
  float ms[NW];
  f32x4_t o[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) o[i] = f32x4_t{};
  m_run = kNoMax;
  l = 0.f;
#pragma unroll
  for (int v = 0; v < NW; ++v) {
    ms[v] = reinterpret_cast<const float*>(lds_waves[v].ring)[DB * 256 + lane];
    m_run = fmaxf(m_run, ms[v]);
  }
  const int db0 = wave * kMine;
#pragma unroll
  for (int v = 0; v < NW; ++v) {
    const float* const other = reinterpret_cast<const float*>(lds_waves[v].ring);
    const float y = __builtin_amdgcn_exp2f((ms[v] - m_run) * sc.c);
    l += other[DB * 256 + 64 + lane] * y;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
      if (db0 + i < DB) o[i] += *reinterpret_cast<const f32x4_t*>(other + ((db0 + i) * 64 + lane) * 4) * y;
  }
  if (t.parts > 1 || p.always) {
    float* const rec = record_of<D>(a, p, w.record + w.part, kvh);
    const bool join = !PAIR && t.parts > 1 && p.join;
    if (q < t.rows) {
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        if (db0 + i >= DB) break;
        float* const to = rec + q * D + (db0 + i) * 16 + 4 * g;
        if (join) {
#pragma unroll
          for (int k = 0; k < 4; ++k) st_agent(to + k, o[i][k]);
        } else {
          *reinterpret_cast<f32x4_t*>(to) = o[i];
        }
      }
      if (wave == 0 && g == 0) {
        st_agent(rec + p.rows * D + q, m_run);
        st_agent(rec + p.rows * (D + 1) + q, l);
      }
    }
    if (join && last_part(a, t, w, kvh, turn)) join_parts<DT, D, NW>(a, p, sc, t, w, kvh);
    return;
  }
  if (q >= t.rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = (static_cast<int64_t>(t.g.first + tok) * a.heads + head) * D + 4 * g;
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    if (db0 + i < DB) store4<DT>(a.out, at + (db0 + i) * 16, o[i] * inv);
  if (a.lse != nullptr && wave == 0 && g == 0)
    a.lse[static_cast<int64_t>(head) * a.num_tokens + t.g.first + tok] =
        l == 0.f ? -__builtin_inff() : (m_run * sc.c + __log2f(l)) * 0.6931471805599453f;
}

template <int DT, int D, int NW, int NS>
__global__ __launch_bounds__(NW * 64, NW * NS * D <= 256 ? 2 : 1) void paged_narrow_kernel(const PagedAttnArgs a,
                                                                                 const PagedPass p,
                                                                                 const Scalars sc) {
  __shared__ __attribute__((aligned(1024))) NarrowLds<D, NS> lds[NW];
  __shared__ int32_t turn;
  narrow_tile<DT, D, NW, NS>(a, p, sc, static_cast<int32_t>(blockIdx.x), static_cast<int32_t>(gridDim.x), lds, turn);
}

// ---------------------------------------------------------------- prefix and own rows
//
// The prefix's tiles (wide: bound by the matrix cores) and the requests' own (narrow:
// bound by bytes) in one launch, so that each CU runs one of either.  Workgroups go
// to the 8 XCDs in turn and to an XCD's 32 CUs in turn, twice: the kinds alternate
// from CU to CU, and the other way round for a CU's second workgroup.  128 tokens
// behind 16384 rows, 32 heads on 8: 88.9 us with the combine, 104.2 in two launches (51
// and 43, and 11); 16 tokens behind 2000 rows, 16 heads: 18.8 / 25.2.  With more own
// tiles than CUs a workgroup runs two of them, on two waves each (the 128 tokens 69 us of
// this kernel against 79, part of that by the plan launch).
template <int DT, int D, bool WIDE, bool PAIR>
__global__ __launch_bounds__(256, 2) void paged_prefix_kernel(const PagedAttnArgs a, const PagedPass pre,
                                                              const PagedPass own, const Scalars sc,
                                                              const int32_t pre_blocks, const int32_t own_blocks) {
  constexpr int NW = 4, NS = D == 128 ? 1 : 2;
  union Lds {
    WideLds<D> wide;
    NarrowLds<D, NS> narrow[NW];
  };
  __shared__ __attribute__((aligned(1024))) uint8_t lds[sizeof(Lds)];
  __shared__ int32_t turn;
  // the id-th workgroup of its kind: of 16 neighbours 8 are the prefix's, while both kinds last
  const int32_t both = (pre_blocks < own_blocks ? pre_blocks : own_blocks) / 256 * 256;
  const int32_t b = static_cast<int32_t>(blockIdx.x);
  bool prefix;
  int32_t id;
  if (b < 2 * both) {
    const int32_t j = b >> 3;  // place in its XCD
    prefix = ((j + (j >> 5)) & 1) == 0;
    id = (j >> 1) * 8 + (b & 7);
  } else {
    id = b - 2 * both + both;
    prefix = id < pre_blocks;
    if (!prefix) id -= pre_blocks - both;
  }
  if (prefix) {
    if constexpr (WIDE) wide_tile<DT, D>(a, pre, sc, id, pre_blocks, *reinterpret_cast<WideLds<D>*>(lds));
    else
      narrow_tile<DT, D, NW, NS>(a, pre, sc, id, pre_blocks, *reinterpret_cast<NarrowLds<D, NS>(*)[NW]>(lds), turn);
  } else if constexpr (PAIR) {
    const int half = uniform(threadIdx.x >> 7);
    narrow_tile<DT, D, 2, NS, true>(a, own, sc, 2 * id + half, own.units * a.kv_heads,
                                    reinterpret_cast<NarrowLds<D, NS>(*)[2]>(lds)[half], turn);
  } else {
    narrow_tile<DT, D, NW, NS>(a, own, sc, id, own_blocks, *reinterpret_cast<NarrowLds<D, NS>(*)[NW]>(lds), turn);
  }
}

// ---------------------------------------------------------------- combine

// Joins the records of one row and K/V head: a wave per row.  Up to 64 parts at
// once: a lane per part for the maxima and sums, then D / 4 lanes per part for its
// values, so that all of a batch's loads are in flight together.  `chunk` rows of
// meta per wave, of which only cut ones are joined.
template <int DT, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(const PagedAttnArgs a, const PagedPass own,
                                                            const PagedPass pre, const Scalars sc,
                                                            const int32_t chunk) {
  constexpr int kLanes = D / 4;         // of a part's row
  constexpr int kAtOnce = 64 / kLanes;  // parts per load
  const int lane = threadIdx.x & 63;
  const int32_t group = a.group;
  const int64_t head = static_cast<int64_t>(first_token(a)) * group;
  const int64_t rows = static_cast<int64_t>(live_tokens(a)) * group;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 4 + uniform(threadIdx.x >> 6);
  const int32_t kvh = static_cast<int32_t>(id % a.kv_heads);
  const int64_t r0 = id / a.kv_heads * chunk;
  if (r0 >= rows) return;
  const int n = static_cast<int>(rows - r0 < chunk ? rows - r0 : chunk);
  int2 mo{0, 0}, mp{0, 0};
  if (lane < n) {
    mo = own.meta[r0 + lane];
    if (pre.combined) mp = pre.meta[r0 + lane];
  }
  const auto sound = [](const PagedPass& p, const int2& m) {
    const int32_t parts = m.y & 0xffff;
    return m.x >= 0 && m.x < p.limit && parts <= p.limit - m.x && (m.y >> 16) >= 0 && (m.y >> 16) < p.rows;
  };
  uint64_t todo = __ballot(lane < n && r0 + lane >= head && (own.always || (mo.y & 0xffff) > 1) && sound(own, mo) &&
                           (!pre.combined || sound(pre, mp)));
  while (todo != 0) {
    const int i = __builtin_ctzll(todo);
    todo &= todo - 1;
    float m = kNoMax, l = 0.f;
    f32x4_t acc{};
    auto join = [&](const PagedPass& p, int32_t record, int32_t info) {
      const int32_t parts = info & 0xffff, row = info >> 16;
      const int64_t stride = static_cast<int64_t>(a.kv_heads) * (p.rows * (D + 2));
      const float* const rec0 = record_of<D>(a, p, record, kvh);
      for (int32_t q0 = 0; q0 < parts; q0 += 64) {
        const int32_t count = parts - q0 < 64 ? parts - q0 : 64;
        float pm = kNoMax, pl = 0.f;
        if (lane < count) {
          const float* const ml = rec0 + (q0 + lane) * stride + p.rows * D + row;
          pm = ml[0];
          pl = ml[p.rows];
        }
        float mn = pm;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) mn = fmaxf(mn, __shfl_xor(mn, off, 64));
        mn = fmaxf(m, mn);
        const float x = __builtin_amdgcn_exp2f((m - mn) * sc.c), y = __builtin_amdgcn_exp2f((pm - mn) * sc.c);
        float sum = pl * y;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        l = l * x + sum;
        m = mn;
        acc *= x;
        const float* const o = rec0 + q0 * stride + row * D + (lane % kLanes) * 4;
#pragma unroll 8
        for (int32_t q = 0; q < count; q += kAtOnce) {
          const int32_t mine = q + lane / kLanes;
          const float z = __shfl(y, mine < count ? mine : 0, 64);
          if (mine < count) acc += *reinterpret_cast<const f32x4_t*>(o + mine * stride) * z;
        }
      }
    };
    if (pre.combined) join(pre, __builtin_amdgcn_readlane(mp.x, i), __builtin_amdgcn_readlane(mp.y, i));
    join(own, __builtin_amdgcn_readlane(mo.x, i), __builtin_amdgcn_readlane(mo.y, i));
#pragma unroll
    for (int off = kLanes; off < 64; off <<= 1)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[k] += __shfl_xor(acc[k], off, 64);
    const int64_t mat = r0 + i;
    const int64_t tok = mat / group;
    const int64_t h = kvh * group + (mat - tok * group);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (lane < kLanes) store4<DT>(a.out, (tok * a.heads + h) * D + lane * 4, acc * inv);
    if (a.lse != nullptr && lane == 0)
      a.lse[h * a.num_tokens + tok] =
          l == 0.f ? -__builtin_inff() : (m * sc.c + __log2f(l)) * 0.6931471805599453f;
  }
}

// ---------------------------------------------------------------- launch

// What runs a launch's tiles.
enum Form : int32_t {
  kWide,        // paged_wide_kernel, two workgroups per CU
  kNarrowMany,  // paged_narrow_kernel: two waves of two stages, two workgroups per CU
  kNarrowMost,  // ... two waves of one stage, four workgroups per CU
  kNarrowOne,   // ... eight waves of one stage, one workgroup per CU
};

struct Layout {
  int32_t shared;    // a pass of its own for the prefix ...
  int32_t pairs;     // ... two of a request's own tiles to a workgroup
  int32_t together;  // ... in one launch with narrow tiles of the requests' own rows
  Form own_form, pre_form;
  PagedPass own, pre;
  int64_t own_units, pre_units;  // per K/V head
  int64_t bytes;
};

int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// Units per K/V head of a launch of up to `tiles` tiles of up to `chunks` chunks each.
int64_t units_bound(const PagedPass& p, int64_t tiles, int64_t chunks) {
  // total / c for any total up to this one: c >= least, and c >= total / wanted or
  // else c >= cap and c >= total / most
  if (chunks <= p.least || chunks <= p.uncut) return tiles;
  const int64_t total = tiles * chunks;
  int64_t cuts = total / p.cap < p.most ? total / p.cap : p.most;
  if (cuts < p.wanted) cuts = p.wanted;
  if (cuts > total / p.least) cuts = total / p.least;
  return tiles + cuts;
}

// How a launch of up to `tiles` tiles (per K/V head) of up to `chunks` chunks runs.
// 256 stands for the CUs.  us on the device:
// * wide, few tiles: parts of 4 chunks and more, one unit per CU first (32 tiles of
//   65 chunks: 32.1, two per CU 37.8) and two from 12 chunks a part (128 tiles of 135: 98
//   against 110); up to 16 chunks whole (40 tiles of 15: 21 against 31).  Many tiles: up
//   to 32 chunks whole (470 tiles of up to 14: 36 against 54; but 64 tiles of 33, 38
//   cut, 65 whole).
// * narrow, up to one tile and 32 chunks per CU: eight waves on one tile, whole up to 16
//   chunks (8 heads, 300 rows 7.8, cut 10.3; 16 requests of 500 behind a prefix 10.3 / 13.9;
//   1000 rows 11.4 / 10.7), else in parts of 4 and its multiples, a stage for each wave (8
//   requests of up to 2000 rows: 14.0, in parts of 5 chunks 20.3, two waves on a tile 17.7).
// * long tiles: eight waves, in parts of up to 48 chunks (64 requests of up to 16000 rows
//   418, two waves 436; one of 64000 58 / 68); many short ones: two waves, two workgroups
//   per CU (256 requests of up to 1200 rows 143, eight waves 160 to 169), whole up to 16
//   chunks (32 requests of 1000 rows 30.7 / 34.7), and with more than 512 tiles of up to 16
//   chunks four workgroups of one stage each, so that one's start is hidden by three
//   others (128 requests of 500 rows 58.0, two 60.5; 1024 of 62 rows 70 / 106; but 64 of
//   500, 512 tiles, 30.8 / 30.2, and the 256 of up to 1200 140 / 138).
Form shape(PagedPass& p, bool narrow, int64_t tiles, int64_t chunks, int32_t kv_heads) {
  p.cap = 0x7fffffff;
  p.step = 1;
  p.uncut = 0;
  if (!narrow) {
    const bool few = tiles * kv_heads < 256;
    p.least = few || p.always ? 4 : 8;
    p.uncut = p.always ? 0 : (few ? 16 : 32);
    p.wanted = (256 + kv_heads - 1) / kv_heads;
    p.most = 2 * p.wanted;
    p.cap = 12;
    return kWide;
  }
  const int64_t per_cu = tiles * kv_heads * chunks / 256;
  p.least = 4;
  if (per_cu <= 32 && tiles * kv_heads <= 256) {
    p.step = 4;  // one stage for each wave
    p.uncut = 16;
    p.wanted = p.most = (256 + kv_heads - 1) / kv_heads;
    return kNarrowOne;
  }
  const bool one = chunks >= 32 && per_cu >= 32;
  p.wanted = ((one ? 256 : 512) + kv_heads - 1) / kv_heads;
  p.most = 4 * p.wanted;
  p.cap = 48;
  p.step = one ? 4 : 1;
  p.uncut = one ? 0 : 16;
  if (one) return kNarrowOne;
  return tiles * kv_heads > 512 && chunks <= 16 ? kNarrowMost : kNarrowMany;
}

Layout layout_of(int32_t tokens, int32_t requests, int32_t heads, int32_t kv_heads, int32_t dim, int64_t table_rows,
                 int32_t prefix_len, int64_t window, int64_t sinks, bool causal, void* workspace, bool counters) {
  Layout l{};
  const int64_t group = heads / kv_heads;
  const int64_t rows = tokens * group;
  const int64_t busy = requests < tokens ? requests : tokens;  // requests with queries
  const int64_t prefix_chunks = (static_cast<int64_t>(prefix_len) + kBN - 1) / kBN;
  const int64_t table_chunks = (table_rows + kBN - 1) / kBN;
  // A prefix has a pass of its own where its rows are read by few rows per
  // request; else, and where it is short, it heads each tile's keys.  us, a pass of
  // its own / heading the keys, by requests x chunks x K/V heads: 1760 14.4 / 9.7, 3608
  // 14.6 / 16.1, 4096 20.9 / 18.9, 8192 18.8 / 32.
  l.shared = prefix_len > 0 && rows < 64 * busy && busy * prefix_chunks * kv_heads > 2048;
  // 16-row tiles up to 16 rows per request; up to 48 (up to three readings of its
  // keys) where those are few or the prefix's tiles run beside them.  us, 16-row /
  // 128-row tiles: 32 requests over 2000 rows, 20 rows each 66.8 / 63.3, 36 rows 87 / 62; 36
  // rows each behind 4000 rows 33.6 / 43; 18 rows each over 200 rows 8.6 / 12.9.
  const bool light = busy * (table_chunks + prefix_chunks) * kv_heads <= 2048;
  bool narrow = rows <= (l.shared || light ? 3 : 1) * kNarrowRows * busy;
  const auto set_rows = [&](PagedPass& p, bool narrow) {
    p.rows = narrow ? kNarrowRows : kWideRows;
    p.tile_tokens = static_cast<int32_t>((p.rows + 2 * group - 2) / group);
  };
  set_rows(l.own, narrow);
  int64_t longest = table_chunks;  // of a tile
  if (window > 0) {
    const int64_t span = causal && l.own.tile_tokens < tokens ? l.own.tile_tokens : tokens;
    const int64_t seen = (window + span) / kBN + 2 + (sinks + kBN - 1) / kBN;
    if (seen < longest) longest = seen;
  }
  l.own.with_prefix = prefix_len > 0 && !l.shared;
  if (l.own.with_prefix) longest += prefix_chunks;
  l.own.always = l.shared;
  int64_t tiles = rows / l.own.rows + busy;
  const int64_t singly = tokens * ((group + l.own.rows - 1) / l.own.rows);  // a request each
  if (singly < tiles) tiles = singly;
  if (tiles == 0) tiles = 1;  // without requests, the tail is filled
  l.own_form = shape(l.own, narrow, tiles, longest, kv_heads);
  l.own_units = units_bound(l.own, tiles, longest);
  l.own.units = static_cast<int32_t>(l.own_units < 0x7fffffff ? l.own_units : 0x7fffffff);
  const bool may_cut = longest > l.own.least && longest > l.own.uncut;
  // a record's counter is 8 bytes of the counters
  l.own.join = counters && may_cut && l.own_form != kWide && !l.shared &&
               (2 * (l.own_units - tiles) + 1) * kv_heads * 8 <= kPagedCounterBytes;
  l.own.combined = l.shared || (may_cut && !l.own.join);
  int64_t at = 0;
  // records: of tiles that are cut, at most twice the cuts; of all where all are joined
  auto place = [&](PagedPass& p, int64_t units, int64_t tiles) {
    char* const base = static_cast<char*>(workspace);
    const int64_t limit = p.always ? units : 2 * (units - tiles) + 1;
    p.limit = static_cast<int32_t>(limit < 0x7fffffff ? limit : 0x7fffffff);
    p.records = reinterpret_cast<float*>(base + at);
    at += round256(limit * kv_heads * p.rows * (dim + 2) * 4);
    p.meta = reinterpret_cast<int2*>(base + at);
    at += round256(rows * 8);
  };
  if (may_cut || l.shared) place(l.own, l.own_units, tiles);
  if (requests > kPlanned) {
    l.own.list = reinterpret_cast<const int4*>(static_cast<char*>(workspace) + at);
    at += round256((2 * l.own_units + 1) * 16);
  }
  if (l.shared) {
    l.pre = l.own;
    l.pre.shared = 1;
    narrow = rows <= kNarrowRows;
    set_rows(l.pre, narrow);
    const int64_t tiles = (rows + l.pre.rows - 1) / l.pre.rows;
    l.pre_form = shape(l.pre, narrow, tiles, prefix_chunks, kv_heads);
    l.together = l.own_form != kWide;
    if (l.together && l.pre_form == kWide) {
      // one per CU beside the requests' own tiles (two: 100 against 88.9 us above)
      l.pre.wanted = l.pre.most = (256 + kv_heads - 1) / kv_heads;
      l.pre.cap = 0x7fffffff;
      // us, one tile / two to a workgroup: 256 tiles 31.0 / 31.1, 384 26.9 / 23.3, 2048 103 / 95
      l.pairs = l.own_units * kv_heads > 256;
    }
    l.pre_units = units_bound(l.pre, tiles, prefix_chunks);
    l.pre.units = static_cast<int32_t>(l.pre_units < 0x7fffffff ? l.pre_units : 0x7fffffff);
    place(l.pre, l.pre_units, tiles);
  }
  l.bytes = at;
  return l;
}

template <int DT, int D>
hipError_t launch(const PagedAttnArgs& a, const Scalars& sc, hipStream_t stream) {
  const Layout l = layout_of(a.num_tokens, a.requests, a.heads, a.kv_heads, D,
                             static_cast<int64_t>(a.table_width) << a.block_shift, a.prefix_len, a.window, a.sinks,
                             a.causal != 0, a.workspace, a.counters != nullptr);
  const auto grid = [&](int64_t units) { return dim3(static_cast<uint32_t>(units * a.kv_heads)); };
  if ((l.own_units > l.pre_units ? l.own_units : l.pre_units) * a.kv_heads > 0x7fffffffLL / 256)
    return hipErrorInvalidConfiguration;
  if (a.requests > kPlanned) {
    const bool few = a.requests <= 1024;
    const int64_t groups = few ? (l.own_units + 255) / 256 : (l.own_units + 4095) / 4096;
    const dim3 plan(static_cast<uint32_t>(groups < 256 ? groups : 256));
    int4* const list = const_cast<int4*>(l.own.list);
    if (few) paged_plan_kernel<256><<<plan, 256, 0, stream>>>(a, l.own, list);
    else paged_plan_kernel<1024><<<plan, 1024, 0, stream>>>(a, l.own, list);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const auto run = [&](const PagedPass& p, Form form, int64_t units) {
    constexpr int kMore = D == 128 ? 1 : 2;  // rows of 64 are half as long
    switch (form) {
      case kWide: paged_wide_kernel<DT, D><<<grid(units), 256, 0, stream>>>(a, p, sc); break;
      case kNarrowMany: paged_narrow_kernel<DT, D, 2, 2 * kMore><<<grid(units), 128, 0, stream>>>(a, p, sc); break;
      case kNarrowMost: paged_narrow_kernel<DT, D, 2, kMore><<<grid(units), 128, 0, stream>>>(a, p, sc); break;
      case kNarrowOne: paged_narrow_kernel<DT, D, 8, kMore><<<grid(units), 512, 0, stream>>>(a, p, sc); break;
    }
  };
  if (l.together) {
    const int64_t pre = l.pre_units * a.kv_heads;
    const int64_t own = l.pairs ? (l.own_units * a.kv_heads + 1) / 2 : l.own_units * a.kv_heads;
    if (pre + own > 0x7fffffffLL / 256) return hipErrorInvalidConfiguration;
    const dim3 all(static_cast<uint32_t>(pre + own));
    const int32_t p = static_cast<int32_t>(pre), o = static_cast<int32_t>(own);
    if (l.pre_form == kWide && l.pairs)
      paged_prefix_kernel<DT, D, true, true><<<all, 256, 0, stream>>>(a, l.pre, l.own, sc, p, o);
    else if (l.pre_form == kWide)
      paged_prefix_kernel<DT, D, true, false><<<all, 256, 0, stream>>>(a, l.pre, l.own, sc, p, o);
    else
      paged_prefix_kernel<DT, D, false, false><<<all, 256, 0, stream>>>(a, l.pre, l.own, sc, p, o);
  } else {
    if (l.shared) run(l.pre, l.pre_form, l.pre_units);
    run(l.own, l.own_form, l.own_units);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !l.own.combined) return e;
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.group;
  // about 8192 waves; where every row is joined, one each
  const int64_t per = l.own.always ? 1 : rows * a.kv_heads / 8192;
  const int32_t chunk = static_cast<int32_t>(per < 1 ? 1 : (per > 64 ? 64 : per));
  const int64_t waves = (rows + chunk - 1) / chunk * a.kv_heads;
  if ((waves + 3) / 4 > 0x7fffffffLL / 256) return hipErrorInvalidConfiguration;
  paged_combine_kernel<DT, D><<<dim3(static_cast<uint32_t>((waves + 3) / 4)), 256, 0, stream>>>(a, l.own, l.pre, sc,
                                                                                             chunk);
  return hipGetLastError();
}

}  // namespace

int64_t paged_attention_workspace(int32_t tokens, int32_t requests, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                  int64_t table_rows, int32_t prefix_len, int32_t window, int32_t sinks, bool causal) {
  return layout_of(tokens, requests, heads, kv_heads, head_dim, table_rows, prefix_len, window, sinks, causal, nullptr,
                   false).bytes;
}

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.num_tokens <= 0) return hipSuccess;
  const float c = fabsf(a.softmax_scale) * kLog2e;
  Scalars sc;
  sc.c = c > kMinC ? c : kMinC;
  sc.thresh = kRescaleLog2 / sc.c;
  sc.q_sign = a.softmax_scale < 0.f ? 0x80008000u : 0u;
  if (a.dtype == kBF16)
    return a.head_dim == 128 ? launch<kBF16, 128>(a, sc, stream) : launch<kBF16, 64>(a, sc, stream);
  return a.head_dim == 128 ? launch<kF16, 128>(a, sc, stream) : launch<kF16, 64>(a, sc, stream);
}

}  // namespace hkv
