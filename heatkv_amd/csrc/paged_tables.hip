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

constexpr int kTableThreads = 1024;
constexpr int kTableWaves = kTableThreads / 64;

struct Sum3 {
  int64_t tokens, popped, pushed;
};

__device__ __forceinline__ Sum3 add(const Sum3& a, const Sum3& b) {
  return Sum3{a.tokens + b.tokens, a.popped + b.popped, a.pushed + b.pushed};
}

// What one request does in a step.
struct Request {
  int64_t held;  // rows before the step
  int64_t n;     // new tokens
  int64_t have, need;
  int64_t front;       // ended: blocks [0, front) are pushed, too
  int64_t from, to;    // logical blocks [from, to) are pushed
  bool ended;
};

// First block that the tokens from position `rows` on still see behind the sinks.
__device__ __forceinline__ int64_t first_live(int64_t rows, int64_t kept, const PagedTablesArgs& a) {
  const int64_t low = rows - a.window + 1;
  const int64_t b = low > 0 ? low >> a.block_shift : 0;
  return b > kept ? b : kept;
}

__device__ __forceinline__ Request load_request(const PagedTablesArgs& a, int32_t r) {
  Request q;
  const int32_t count = a.new_counts[r];
  const int32_t len = a.lengths[r];
  const int64_t block = 1LL << a.block_shift;
  q.ended = count < 0;
  q.n = count > 0 ? count : 0;
  q.held = len > 0 ? len : 0;
  q.have = (q.held + block - 1) >> a.block_shift;
  q.need = (q.held + q.n + block - 1) >> a.block_shift;
  const int64_t kept = a.window > 0 ? (a.sinks + block - 1) >> a.block_shift : 0;
  q.front = 0;
  q.from = 0;
  q.to = 0;
  if (q.ended) {
    const int64_t low = a.window > 0 ? first_live(q.held, kept, a) : 0;
    q.front = kept < q.have ? kept : q.have;
    q.from = low < q.have ? low : q.have;
    q.to = q.have;
  } else if (a.window > 0) {
    q.from = first_live(q.held, kept, a);
    q.to = first_live(q.held + q.n, kept, a);
  }
  return q;
}

// The r with prefix[r] <= i < prefix[r + 1]; prefix[0] = 0 <= i < prefix[n].
__device__ __forceinline__ int32_t find(const int32_t* prefix, int32_t n, int32_t i) {
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

__global__ __launch_bounds__(kTableThreads) void paged_tables_kernel(PagedTablesArgs a) {
  __shared__ int32_t starts[kMaxRequests + 1], popped[kMaxRequests + 1], pushed[kMaxRequests + 1];
  __shared__ Sum3 wave_total[kTableWaves];
  __shared__ int32_t too_long;
  const int tid = threadIdx.x;
  const int wave = tid >> 6;
  const int32_t R = a.requests, N = a.ring_size;
  int32_t first = a.free_range[0], free = a.free_range[1];
  free = free < 0 ? 0 : (free > N ? N : free);
  first = N > 0 ? first % N : 0;
  if (first < 0) first += N;
  if (tid == 0) too_long = 0;
  __syncthreads();
  Sum3 carry{0, 0, 0};
  for (int32_t r0 = 0; r0 < R; r0 += kTableThreads) {
    const int32_t r = r0 + tid;
    Sum3 mine{0, 0, 0};
    if (r < R) {
      const Request q = load_request(a, r);
      mine = Sum3{q.n, q.need - q.have, q.front + q.to - q.from};
      if (q.need > a.table_width || q.have > a.table_width || q.held + q.n > 0x7fffffffLL) too_long = 1;
    }
    const Sum3 incl = wave_scan(mine);
    if ((tid & 63) == 63) wave_total[wave] = incl;
    __syncthreads();
    Sum3 before = carry;
    for (int w = 0; w < kTableWaves; ++w) {
      if (w == wave) before = add(before, incl);
      carry = add(carry, wave_total[w]);
      if (w < wave) before = add(before, wave_total[w]);
    }
    if (r < R) {
      // sums past 32 bits refuse the step below
      starts[r + 1] = static_cast<int32_t>(before.tokens);
      popped[r + 1] = static_cast<int32_t>(before.popped);
      pushed[r + 1] = static_cast<int32_t>(before.pushed);
    }
    __syncthreads();
  }
  if (tid == 0) starts[0] = popped[0] = pushed[0] = 0;
  __syncthreads();
  const int32_t status =
      (carry.popped > free ? 1 : 0) | (too_long != 0 ? 2 : 0) | (carry.tokens > a.num_tokens ? 4 : 0);
  const bool fine = status == 0;
  // lengths_out may be lengths, so each is read before it is written and not again
  const auto ring_at = [&](int64_t i) { return static_cast<int32_t>((first + i) % N); };
  if (fine) {
    for (int32_t i = tid; i < static_cast<int32_t>(carry.popped); i += kTableThreads) {
      const int32_t r = find(popped, R, i);
      const Request q = load_request(a, r);
      a.block_tables[r * a.table_stride + q.have + (i - popped[r])] = a.free_blocks[ring_at(i)];
    }
    for (int32_t i = tid; i < static_cast<int32_t>(carry.pushed); i += kTableThreads) {
      const int32_t r = find(pushed, R, i);
      const Request q = load_request(a, r);
      const int32_t k = i - pushed[r];
      const int64_t j = k < q.front ? k : q.from + (k - q.front);
      // a block that this step pops is read where it is popped from
      const int32_t b = j < q.have ? a.block_tables[r * a.table_stride + j]
                                   : a.free_blocks[ring_at(popped[r] + (j - q.have))];
      a.free_blocks[ring_at(static_cast<int64_t>(free) + i)] = b;
    }
  }
  __syncthreads();
  for (int32_t r = tid; r < R; r += kTableThreads) {
    const Request q = load_request(a, r);
    const int32_t after = q.ended ? 0 : static_cast<int32_t>(q.held + q.n);
    const int32_t was = a.lengths[r];
    a.query_starts[r] = fine ? starts[r] : 0;
    a.lengths_out[r] = fine ? after : was;
  }
  if (tid == 0) {
    a.query_starts[R] = fine ? starts[R] : 0;
    a.status[0] = status;
    const int32_t f0 = a.free_range[0], f1 = a.free_range[1];
    a.range_out[0] = fine ? (N > 0 ? ring_at(carry.popped) : 0) : f0;
    a.range_out[1] = fine ? static_cast<int32_t>(free - carry.popped + carry.pushed) : f1;
  }
}

// Slot of each token: its request's block of the row, and the row in it.
__global__ __launch_bounds__(256) void paged_slots_kernel(PagedTablesArgs a) {
  __shared__ int32_t starts[kMaxRequests + 1];
  const int32_t R = a.requests;
  for (int32_t r = threadIdx.x; r <= R; r += 256) starts[r] = a.query_starts[r];
  __syncthreads();
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < a.num_tokens;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    int64_t slot = -1;
    if (t < starts[R]) {
      const int32_t r = find(starts, R, static_cast<int32_t>(t));
      const int32_t row = a.lengths_out[r] - starts[r + 1] + static_cast<int32_t>(t);
      const int64_t b = a.block_tables[r * a.table_stride + (row >> a.block_shift)];
      slot = (b << a.block_shift) + (row & ((1 << a.block_shift) - 1));
    }
    a.slot_map[t] = slot;
  }
}

// K/V rows of the step's tokens to their slots: one thread per 16 bytes (2
// where the strides or pointers ask for it) of K and of V, both in flight.
template <typename U>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedAppendArgs a, int32_t units, int64_t total) {
  constexpr int kPer = sizeof(U) / 2;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / units;
    const int32_t c = static_cast<int32_t>(i - row * units) * kPer;
    const int64_t t = row / a.kv_heads;
    const int64_t h = row - t * a.kv_heads;
    const int64_t slot = a.slot_map[t];
    if (slot < 0 || slot >= a.num_slots) continue;
    const int64_t b = slot >> a.block_shift, r = slot & ((1 << a.block_shift) - 1);
    const uint16_t* sk = static_cast<const uint16_t*>(a.k) + t * a.k_token + h * a.k_head + c;
    const uint16_t* sv = static_cast<const uint16_t*>(a.v) + t * a.v_token + h * a.v_head + c;
    uint16_t* dk = static_cast<uint16_t*>(a.k_cache) + b * a.ks.block + h * a.ks.head + r * a.ks.row + c;
    uint16_t* dv = static_cast<uint16_t*>(a.v_cache) + b * a.vs.block + h * a.vs.head + r * a.vs.row + c;
    const U xk = *reinterpret_cast<const U*>(sk);
    const U xv = *reinterpret_cast<const U*>(sv);
    *reinterpret_cast<U*>(dk) = xk;
    *reinterpret_cast<U*>(dv) = xv;
  }
}

typedef uint32_t U16B __attribute__((ext_vector_type(4)));

}  // namespace

hipError_t launch_paged_tables(const PagedTablesArgs& a, hipStream_t stream) {
  paged_tables_kernel<<<1, kTableThreads, 0, stream>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.num_tokens == 0) return e;
  const int64_t blocks = (a.num_tokens + 255LL) / 256;
  paged_slots_kernel<<<dim3(static_cast<uint32_t>(blocks < 1024 ? blocks : 1024)), 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.num_tokens <= 0) return hipSuccess;
  const int64_t strides = a.k_token | a.k_head | a.v_token | a.v_head | a.ks.block | a.ks.head | a.ks.row |
                          a.vs.block | a.vs.head | a.vs.row | a.head_dim;
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                         reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache);
  const bool wide = strides % 8 == 0 && ptrs % 16 == 0;
  const int32_t units = wide ? a.head_dim / 8 : a.head_dim;
  const int64_t total = static_cast<int64_t>(a.num_tokens) * a.kv_heads * units;
  const int64_t blocks = (total + 255) / 256;
  const dim3 grid(static_cast<uint32_t>(blocks < (1 << 20) ? blocks : (1 << 20)));
  if (wide) paged_append_kernel<U16B><<<grid, 256, 0, stream>>>(a, units, total);
  else paged_append_kernel<uint16_t><<<grid, 256, 0, stream>>>(a, units, total);
  return hipGetLastError();
}

}  // namespace hkv
