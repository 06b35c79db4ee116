// Attention of single new tokens over a paged cache: the token of sequence b stands at position len - 1 (len = seq_lens[b], itself in
// the cache already) and sees the positions p < len with p >= len - W or p < n_sink.
#pragma once

#include "sink_rows.cuh"

namespace swa {
namespace sink {

struct DecodeArgs {
  View4 q, o;               // [B, Hq, 1, d]
  View4 k, v;               // caches [pages, Hkv, slots, d]
  const int32_t *page_table, *seq_lens;
  int B, Hq, Hkv, G, dqk, dv, W, ns, max_pages, n_pages, page_size;
  float c2;
};

// The page and slot of position p as an element offset into a cache, or false: a page number outside the cache holds nothing.
__device__ __forceinline__ bool cache_row(const DecodeArgs& a, int b, int p, int64_t* page, int* slot) {
  const int lp = p / a.page_size;
  const int pg = a.page_table[(int64_t)b * a.max_pages + lp];
  *page = pg;
  *slot = p - lp * a.page_size;
  return pg >= 0 && pg < a.n_pages;
}

__device__ __forceinline__ int decode_len(const DecodeArgs& a, int b) {
  const int64_t most = (int64_t)a.max_pages * a.page_size;
  const int n = a.seq_lens[b];
  return n < 0 ? 0 : (int64_t)n > most ? (int)most : n;
}

// One warp per query row: every type, stride and head dim up to 256.
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) decode_rows_kernel(const __grid_constant__ DecodeArgs a) {
  __shared__ float smem[kRowWarps][kMaxDim];
  pdl_enter();
  pdl_wait();
  const int lane = threadIdx.x & 31, h = blockIdx.x * kRowWarps + (threadIdx.x >> 5), b = blockIdx.y;
  if (h >= a.Hq) return;
  float* s = smem[threadIdx.x >> 5];
  const int hk = h / a.G, len = decode_len(a, b);
  stage_row(s, row_ptr<T>(a.q, b, h, 0), a.q.s3, a.dqk, lane);
  __syncwarp();
  const bool vec = vec_rows<T>(a.k, a.dqk);
  float acc[kDimsPerLane] = {};
  float m = -INFINITY, l = 0.f;
  bool any = false;
  const int lo = (int)max((int64_t)0, (int64_t)len - a.W), sinks = min(a.ns, lo);
  for (int j0 = 0; j0 < len; j0 += 32) {
    if (j0 >= sinks && j0 + 32 <= lo) {
      j0 += (lo - j0) / 32 * 32 - 32;
      continue;
    }
    const int j = j0 + lane;
    int64_t page = 0;
    int slot = 0;
    bool on = j < len && (j < sinks || j >= lo);
    if (on) on = cache_row(a, b, j, &page, &slot);
    uint32_t see = __ballot_sync(0xffffffffu, on);
    if (!see) continue;
    any = true;
    const float x = on ? dot_row(s, (const T*)a.k.ptr + page * a.k.s0 + hk * a.k.s1 + slot * a.k.s2, a.k.s3, a.dqk, vec) * a.c2 : -INFINITY;
    const float mn = fmaxf(m, lanes_max(x));
    const float f = m == mn ? 1.f : exp2f(m - mn);
    const float p = on && x != -INFINITY ? exp2f(x - mn) : 0.f;
    l = l * f + lanes_sum(p);
    m = mn;
#pragma unroll
    for (int t = 0; t < kDimsPerLane; ++t) acc[t] *= f;
    const int64_t vo = page * a.v.s0 + hk * a.v.s1 + slot * a.v.s2;
    while (see) {
      const int y = __ffs(see) - 1;
      see &= see - 1;
      const float w = __shfl_sync(0xffffffffu, p, y);
      const T* r = (const T*)a.v.ptr + __shfl_sync(0xffffffffu, vo, y);
#pragma unroll
      for (int t = 0; t < kDimsPerLane; ++t)
        if (lane + 32 * t < a.dv) acc[t] = fmaf(w, to_f(r[(lane + 32 * t) * a.v.s3]), acc[t]);
    }
  }
  store_row<T>(a.o, b, h, 0, acc, any ? 1.f / l : 0.f, a.dv, lane);
}

}  // namespace sink
}  // namespace swa
