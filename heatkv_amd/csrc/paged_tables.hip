// Bookkeeping and append of the paged K/V cache.
//
// Tables of one step.  A request that holds `len` rows and brings `n` tokens
// needs ceil((len + n) / block) blocks and has ceil(len / block); the missing
// ones are popped from the head of a ring of free blocks, in request order.
// Blocks that no later token sees (all of an ended request's; with a window W,
// those from behind the sinks' blocks up to row len + n - W + 1) are pushed
// behind the ring's tail.  A step pops only blocks that were free before it,
// so what it pushes may still be read until the next step.  Three prefix sums
// over the requests (tokens, popped, pushed) give every token, popped and
// pushed block its place; then each is written by a thread of its own, which
// finds its request by a search of the prefix sum.
#include "hkv_internal.h"
#include "paged.h"
#include "stream_mem.h"

namespace hkv {
namespace {

// A sum of the prefix sums; saturating, so that sums past 32 bits refuse the step.
struct Sum3 {
  uint32_t tokens, popped, pushed;
};

__device__ __forceinline__ Sum3 add(const Sum3& a, const Sum3& b) {
  return Sum3{__builtin_elementwise_add_sat(a.tokens, b.tokens), __builtin_elementwise_add_sat(a.popped, b.popped),
              __builtin_elementwise_add_sat(a.pushed, b.pushed)};
}

// What one request does in a step.
struct Request {
  int64_t have, need;  // blocks
  int64_t front;       // ended: blocks [0, front) are pushed, too
  int64_t from, to;    // logical blocks [from, to) are pushed
};

// First block that the tokens from position `rows` on still see behind the sinks.
__device__ __forceinline__ int64_t first_live(int64_t rows, int64_t kept, const PagedTablesArgs& a) {
  const int64_t low = rows - a.window + 1;
  const int64_t b = low > 0 ? low >> a.block_shift : 0;
  return b > kept ? b : kept;
}

// A request that holds `held` rows and brings n tokens, or (n < 0) has ended.
__device__ __forceinline__ Request request_of(const PagedTablesArgs& a, int64_t held, int64_t n) {
  Request q;
  const int64_t block = 1LL << a.block_shift;
  const bool ended = n < 0;
  if (ended) n = 0;
  q.have = (held + block - 1) >> a.block_shift;
  q.need = (held + n + block - 1) >> a.block_shift;
  const int64_t kept = a.window > 0 ? (a.sinks + block - 1) >> a.block_shift : 0;
  q.front = 0;
  q.from = 0;
  q.to = 0;
  if (ended) {
    const int64_t low = a.window > 0 ? first_live(held, kept, a) : 0;
    q.front = kept < q.have ? kept : q.have;
    q.from = low < q.have ? low : q.have;
    q.to = q.have;
  } else if (a.window > 0) {
    q.from = first_live(held, kept, a);
    q.to = first_live(held + n, kept, a);
  }
  return q;
}

// The r with prefix[r] <= i < prefix[r + 1]; prefix[0] = 0 <= i < prefix[n].
__device__ __forceinline__ int32_t find(const uint32_t* prefix, int32_t n, uint32_t i) {
  int32_t lo = 0, hi = n;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (prefix[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ Sum3 wave_scan(Sum3 v) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const Sum3 o{__shfl_up(v.tokens, off, 64), __shfl_up(v.popped, off, 64), __shfl_up(v.pushed, off, 64)};
    if (static_cast<int>(threadIdx.x & 63) >= off) v = add(v, o);
  }
  return v;
}

// Every workgroup computes the prefix sums of all requests for itself (a few
// thousand integers) and takes its share of the blocks and tokens, so that one
// launch does it all: no workgroup reads what another writes.  Popped are table
// entries behind those held, pushed ring entries behind those free; only where
// free and pushed together exceed the ring (a prompt longer than its window on an
// almost empty cache) would a push meet an entry yet to be popped, and there the first
// workgroup takes everything, in order.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void paged_tables_kernel(const PagedTablesArgs a) {
  constexpr int kWaves = kThreads / 64;
  constexpr int32_t kEnded = static_cast<int32_t>(0x80000000u);
  __shared__ uint32_t starts[kMaxRequests + 1], popped[kMaxRequests + 1], pushed[kMaxRequests + 1];
  __shared__ int32_t rows[kMaxRequests];  // held, kEnded set where the request has ended
  __shared__ Sum3 wave_total[kWaves];
  __shared__ int32_t too_long;
  const int tid = threadIdx.x;
  const int wave = tid >> 6;
  const int32_t R = a.requests, N = a.ring_size;
  const int32_t given0 = a.free_range[0], given1 = a.free_range[1];
  if (tid == 0) too_long = 0;
  Sum3 carry{0, 0, 0};
  for (int32_t r0 = 0; r0 < R || r0 == 0; r0 += kThreads) {
    const int32_t r = r0 + tid;
    Sum3 mine{0, 0, 0};
    bool over = false;
    if (r < R) {
      const int32_t n = a.new_counts[r];
      int32_t held = a.lengths[r];
      held = held > 0 ? held : 0;
      const Request q = request_of(a, held, n);
      const int64_t push = q.front + q.to - q.from;
      mine = Sum3{n > 0 ? static_cast<uint32_t>(n) : 0u, static_cast<uint32_t>(q.need - q.have),
                  static_cast<uint32_t>(push)};
      over = q.need > a.table_width || held + (n > 0 ? static_cast<int64_t>(n) : 0) > 0x7fffffffLL;
      rows[r] = n < 0 ? held | kEnded : held;
    }
    const Sum3 incl = wave_scan(mine);
    if ((tid & 63) == 63) wave_total[wave] = incl;
    __syncthreads();  // also the first: too_long is clear
    if (over) too_long = 1;
    Sum3 before = add(carry, incl);
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before = add(before, wave_total[w]);
      carry = add(carry, wave_total[w]);
    }
    if (r < R) {
      starts[r + 1] = before.tokens;
      popped[r + 1] = before.popped;
      pushed[r + 1] = before.pushed;
    }
    if (r == 0) starts[0] = popped[0] = pushed[0] = 0;
    __syncthreads();
  }
  int32_t free = given1 < 0 ? 0 : (given1 > N ? N : given1);
  int32_t first = N > 0 ? given0 % N : 0;
  if (first < 0) first += N;
  const int64_t left = static_cast<int64_t>(free) - carry.popped + carry.pushed;
  const int32_t status = (carry.popped > static_cast<uint32_t>(free) ? 1 : 0) | (too_long != 0 ? 2 : 0) |
                         (carry.tokens > static_cast<uint32_t>(a.num_tokens) ? 4 : 0);
  // blocks given back that the ring has no room for: not the blocks of this cache
  const int32_t state = status == 0 && left > N ? 8 : status;
  const bool fine = state == 0;
  const auto ring_at = [&](int64_t i) {
    int64_t at = first + i;  // i < 2 N
    if (at >= N) at -= N;
    if (at >= N) at -= N;
    return at;
  };
  const bool alone = static_cast<int64_t>(free) + carry.pushed > N;
  const int64_t step = alone ? kThreads : static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t at = alone ? tid : static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  if (blockIdx.x == 0) {
    for (int32_t r = tid; r <= R; r += kThreads) a.query_starts[r] = fine ? static_cast<int32_t>(starts[r]) : 0;
    if (a.lengths_out != a.lengths) {
      for (int32_t r = tid; r < R; r += kThreads) {
        const int32_t n = static_cast<int32_t>(starts[r + 1] - starts[r]);
        a.lengths_out[r] = !fine ? a.lengths[r] : (rows[r] & kEnded) != 0 ? 0 : rows[r] + n;
      }
    }
    if (tid == 0) {
      a.status[0] = state;
      a.status[1] = fine ? static_cast<int32_t>(carry.popped) : 0;
      a.status[2] = fine ? static_cast<int32_t>(carry.pushed) : 0;
      if (a.range_out != a.free_range) {
        a.range_out[0] = fine && N > 0 ? static_cast<int32_t>(ring_at(carry.popped)) : given0;
        a.range_out[1] = fine ? static_cast<int32_t>(left) : given1;
      }
    }
  }
  if (alone && blockIdx.x != 0) return;
  const auto request = [&](int32_t r) {
    const int32_t x = rows[r];
    return (x & kEnded) != 0 ? request_of(a, x & ~kEnded, -1) : request_of(a, x, starts[r + 1] - starts[r]);
  };
  // Slot of a token: its request's block of the row, and the row in it.
  const auto slot = [&](int64_t t) {
    int64_t to = -1;
    if (fine && t < carry.tokens) {
      const int32_t r = find(starts, R, static_cast<uint32_t>(t));
      const int64_t row = (rows[r] & ~kEnded) + (t - starts[r]);
      const int64_t j = row >> a.block_shift;
      const int64_t have = ((rows[r] & ~kEnded) + (1LL << a.block_shift) - 1) >> a.block_shift;
      const int64_t b = j < have ? a.block_tables[r * a.table_stride + j]
                                 : a.free_blocks[ring_at(popped[r] + (j - have))];
      to = (b << a.block_shift) + (row & ((1LL << a.block_shift) - 1));
    }
    a.slot_map[t] = to;
  };
  const auto pop = [&](int64_t i) {
    const int32_t r = find(popped, R, static_cast<uint32_t>(i));
    a.block_tables[r * a.table_stride + request(r).have + (i - popped[r])] = a.free_blocks[ring_at(i)];
  };
  const auto push = [&](int64_t i) {
    const int32_t r = find(pushed, R, static_cast<uint32_t>(i));
    const Request q = request(r);
    const int64_t k = i - pushed[r];
    const int64_t j = k < q.front ? k : q.from + (k - q.front);
    // a block that this step pops is read where it is popped from, or (alone) to
    const int32_t b = j < q.have || alone ? a.block_tables[r * a.table_stride + j]
                                          : a.free_blocks[ring_at(popped[r] + (j - q.have))];
    a.free_blocks[ring_at(static_cast<int64_t>(free) + i)] = b;
  };
  const int64_t tokens = a.num_tokens, pops = fine ? carry.popped : 0, pushes = fine ? carry.pushed : 0;
  if (!alone) {
    // side by side, so that no thread waits for one kind before it begins the next
    for (int64_t i = at; i < tokens + pops + pushes; i += step) {
      if (i < tokens) slot(i);
      else if (i < tokens + pops) pop(i - tokens);
      else push(i - tokens - pops);
    }
    return;
  }
  for (int64_t i = at; i < tokens; i += step) slot(i);
  for (int64_t i = at; i < pops; i += step) pop(i);
  __syncthreads();
  for (int64_t i = at; i < pushes; i += step) push(i);
}

// The state in place, once no workgroup of the step reads the old one any more.
__global__ __launch_bounds__(256) void paged_state_kernel(const PagedTablesArgs a) {
  if (a.status[0] != 0) return;
  for (int32_t r = threadIdx.x; r < a.requests; r += 256) {
    const int32_t held = a.lengths[r] > 0 ? a.lengths[r] : 0;
    a.lengths_out[r] = a.new_counts[r] < 0 ? 0 : held + (a.query_starts[r + 1] - a.query_starts[r]);
  }
  if (threadIdx.x == 0 && a.ring_size > 0) {
    const int64_t N = a.ring_size;
    const int32_t given0 = a.free_range[0], given1 = a.free_range[1];
    int64_t first = given0 % N;
    if (first < 0) first += N;
    a.range_out[0] = static_cast<int32_t>((first + a.status[1]) % N);
    a.range_out[1] = (given1 < 0 ? 0 : given1) - a.status[1] + a.status[2];
  }
}

// K/V rows of the step's tokens to their slots: one thread per 16 bytes (2
// where the strides or pointers ask for it) of K and of V, both in flight.
template <typename U, bool STREAM>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a, const int32_t units_shift) {
  constexpr int kPer = sizeof(U) / 2;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const uint32_t row = static_cast<uint32_t>(i >> units_shift);  // (token, head)
  const int64_t c = (i & ((1 << units_shift) - 1)) * kPer;
  const uint32_t t = row / static_cast<uint32_t>(a.kv_heads);
  if (t >= static_cast<uint32_t>(a.num_tokens)) return;
  const int64_t h = row - t * static_cast<uint32_t>(a.kv_heads);
  const int64_t slot = a.slot_map[t];
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t b = slot >> a.block_shift, r = slot & ((1 << a.block_shift) - 1);
  const U* const sk = reinterpret_cast<const U*>(static_cast<const uint16_t*>(a.k) + t * a.k_token + h * a.k_head + c);
  const U* const sv = reinterpret_cast<const U*>(static_cast<const uint16_t*>(a.v) + t * a.v_token + h * a.v_head + c);
  U* const dk = reinterpret_cast<U*>(static_cast<uint16_t*>(a.k_cache) + b * a.ks.block + h * a.ks.head +
                                     r * a.ks.row + c);
  U* const dv = reinterpret_cast<U*>(static_cast<uint16_t*>(a.v_cache) + b * a.vs.block + h * a.vs.head +
                                     r * a.vs.row + c);
  if constexpr (STREAM) {
    const U xk = stream_load(sk), xv = stream_load(sv);
    stream_store(dk, xk);
    stream_store(dv, xv);
  } else {
    const U xk = *sk, xv = *sv;
    *dk = xk;
    *dv = xv;
  }
}

typedef uint32_t U16B __attribute__((ext_vector_type(4)));

}  // namespace

hipError_t launch_paged_tables(const PagedTablesArgs& a, hipStream_t stream) {
  // a workgroup per 1024 tokens, and per 32 requests whose blocks may move
  int64_t blocks = (a.num_tokens + 1023LL) / 1024 + a.requests / 32;
  blocks = blocks < 1 ? 1 : (blocks > 128 ? 128 : blocks);
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (a.requests <= 256 && blocks == 1) paged_tables_kernel<256><<<grid, 256, 0, stream>>>(a);
  else paged_tables_kernel<1024><<<grid, 1024, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || (a.lengths_out != a.lengths && a.range_out != a.free_range)) return e;
  paged_state_kernel<<<1, 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.num_tokens <= 0) return hipSuccess;
  const int64_t strides = a.k_token | a.k_head | a.v_token | a.v_head | a.ks.block | a.ks.head | a.ks.row |
                          a.vs.block | a.vs.head | a.vs.row;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
  const bool wide = strides % 8 == 0 && ptrs % 16 == 0;
  const int32_t shift = (a.head_dim == 128 ? 7 : 6) - (wide ? 3 : 0);
  const int64_t rows = static_cast<int64_t>(a.num_tokens) * a.kv_heads;
  const int64_t blocks = ((rows << shift) + 255) / 256;
  if (rows > 0x7fffffffLL || blocks > 0xffffffffLL / 256) return hipErrorInvalidConfiguration;
  const dim3 grid(static_cast<uint32_t>(blocks));
  // Past the caches, rows are moved without a place in them: 134 MB written 52.5 -> 48.3 us
  // (5.5 TB/s), but 34 MB 12.2 -> 14.2.
  const bool once = rows * a.head_dim * 4 >= (1LL << 26);
  if (!wide) paged_append_kernel<uint16_t, false><<<grid, 256, 0, stream>>>(a, shift);
  else if (once) paged_append_kernel<U16B, true><<<grid, 256, 0, stream>>>(a, shift);
  else paged_append_kernel<U16B, false><<<grid, 256, 0, stream>>>(a, shift);
  return hipGetLastError();
}

}  // namespace hkv
