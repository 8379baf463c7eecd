// Attention over a paged K/V cache: every query of a request sees the rows of
// its request's blocks (with a causal limit, a sliding window and first rows
// that stay visible), and of a prefix that all requests share.
//
// One wave per (token, query head): 64 keys at a time, a key per lane for the
// scores, two dimensions per lane for the values.
#include "attn_common.h"
#include "paged.h"

namespace hkv {
namespace {

using namespace attn;

template <int DT>
__device__ __forceinline__ float widen(uint16_t v) {
  if constexpr (DT == kF16) return f16_to_f32(v);
  else return __builtin_bit_cast(float, static_cast<uint32_t>(v) << 16);
}

template <int DT>
__device__ __forceinline__ uint16_t narrow(float v) {
  return static_cast<uint16_t>(pack2<DT>(v, v) & 0xffffu);
}

template <int DT, int D>
__global__ __launch_bounds__(64) void paged_attn_kernel(PagedAttnArgs a) {
  constexpr int kPer = D / 64;
  __shared__ float qs[D];
  const int lane = threadIdx.x;
  const int32_t t = static_cast<int32_t>(blockIdx.x);
  const int32_t h = static_cast<int32_t>(blockIdx.y);
  const int32_t kvh = h / (a.heads / a.kv_heads);
  const int32_t R = a.requests;
  uint16_t* const out = static_cast<uint16_t*>(a.out) + (static_cast<int64_t>(t) * a.heads + h) * D;
  // the request of the token: the last one that starts at or before it
  const int32_t end = R > 0 ? a.query_starts[R] : 0;
  if (t >= end) {
    if (a.fill_tail) {
      for (int i = 0; i < kPer; ++i) out[lane * kPer + i] = 0;
      if (a.lse != nullptr && lane == 0) a.lse[static_cast<int64_t>(h) * a.num_tokens + t] = -__builtin_inff();
    }
    return;
  }
  int32_t lo = 0, hi = R;
  while (hi - lo > 1) {
    const int32_t mid = (lo + hi) >> 1;
    if (a.query_starts[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int64_t cap = static_cast<int64_t>(a.table_width) << a.block_shift;
  int64_t len = a.lengths[lo];
  len = len < 0 ? 0 : (len > cap ? cap : len);
  const int64_t pos = len - (a.query_starts[lo + 1] - t);
  const uint16_t* const q = static_cast<const uint16_t*>(a.q) + t * a.q_token + h * a.q_head;
  for (int i = lane; i < D; i += 64) qs[i] = widen<DT>(q[i]) * a.softmax_scale;
  __syncthreads();
  float m = -__builtin_inff(), l = 0.f, acc[kPer] = {};
  // keys [k0, k1) of `blocks`
  const auto walk = [&](const int32_t* blocks, int64_t k0, int64_t k1) {
    for (int64_t base = k0; base < k1; base += 64) {
      const int64_t j = base + lane < k1 ? base + lane : k1 - 1;
      const uint32_t raw = static_cast<uint32_t>(blocks[j >> a.block_shift]);
      const int64_t b = raw < static_cast<uint32_t>(a.num_blocks) ? raw : 0;
      const int64_t r = j & ((1 << a.block_shift) - 1);
      const uint16_t* k = static_cast<const uint16_t*>(a.k_cache) + b * a.ks.block + kvh * a.ks.head + r * a.ks.row;
      const uint16_t* v = static_cast<const uint16_t*>(a.v_cache) + b * a.vs.block + kvh * a.vs.head + r * a.vs.row;
      float s = 0.f;
      for (int i = 0; i < D; ++i) s = __builtin_fmaf(qs[i], widen<DT>(k[i]), s);
      const bool in = base + lane < k1;
      float mx = in ? s : -__builtin_inff();
      for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      const float mn = fmaxf(m, mx);
      const float p = in ? expf(s - mn) : 0.f;
      const float al = m == mn ? 1.f : expf(m - mn);
      float sum = p;
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
      l = l * al + sum;
      m = mn;
      for (int i = 0; i < kPer; ++i) acc[i] *= al;
      const int64_t vp = reinterpret_cast<int64_t>(v);
      const int n = static_cast<int>(k1 - base < 64 ? k1 - base : 64);
      for (int jj = 0; jj < n; ++jj) {
        const uint16_t* row = reinterpret_cast<const uint16_t*>(__shfl(vp, jj, 64));
        const float pj = __shfl(p, jj, 64);
        for (int i = 0; i < kPer; ++i) acc[i] = __builtin_fmaf(pj, widen<DT>(row[lane * kPer + i]), acc[i]);
      }
    }
  };
  if (a.prefix_len > 0) walk(a.prefix_blocks, 0, a.prefix_len);
  if (pos >= 0) {
    const int32_t* const blocks = a.block_tables + lo * a.table_stride;
    const int64_t last = a.causal && pos + 1 < len ? pos + 1 : len;
    const int64_t low = a.window > 0 && pos + 1 > a.window ? pos + 1 - a.window : 0;
    walk(blocks, 0, low < a.sinks ? low : a.sinks);
    walk(blocks, low, last);
  }
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  for (int i = 0; i < kPer; ++i) out[lane * kPer + i] = narrow<DT>(acc[i] * inv);
  if (a.lse != nullptr && lane == 0) a.lse[static_cast<int64_t>(h) * a.num_tokens + t] = m + logf(l);
}

}  // namespace

hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream) {
  if (a.num_tokens <= 0) return hipSuccess;
  const dim3 grid(static_cast<uint32_t>(a.num_tokens), static_cast<uint32_t>(a.heads));
  if (a.dtype == kBF16) {
    if (a.head_dim == 128) paged_attn_kernel<kBF16, 128><<<grid, 64, 0, stream>>>(a);
    else paged_attn_kernel<kBF16, 64><<<grid, 64, 0, stream>>>(a);
  } else {
    if (a.head_dim == 128) paged_attn_kernel<kF16, 128><<<grid, 64, 0, stream>>>(a);
    else paged_attn_kernel<kF16, 64><<<grid, 64, 0, stream>>>(a);
  }
  return hipGetLastError();
}

}  // namespace hkv
