// Attention of single new tokens over a paged cache: the token of sequence b stands at position len - 1 (len = seq_lens[b], itself in
// the cache already) and sees the positions p < len with p >= len - W or p < n_sink.
#pragma once

#include <type_traits>

#include "sink_rows.cuh"

namespace swa {
namespace sink {

struct DecodeArgs {
  View4 q, o;               // [B, Hq, 1, d]
  View4 k, v;               // caches [pages, Hkv, slots, d]
  const int32_t *page_table, *seq_lens;
  int B, Hq, Hkv, G, dqk, dv, W, ns, max_pages, n_pages, page_size;
  int split, page_shift;    // decode_split_kernel: CTAs of a cluster; log2 of the page size, or -1
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

// ---- the split kernel ---------------------------------------------------------------------------------------------------
// A cluster of C CTAs of four warps works on one sequence, one key head and up to 16 of the query heads that share it; the tokens it
// sees (sinks, then window, in tiles of KT) are dealt out evenly to its 4 C warps, so that a few long sequences fill the GPU as
// well as many do.  Each warp runs the one-pass softmax over its tiles -- cp.async into a ring of its own, no barrier with
// the other warps -- and the partial results (maximum, sum, O) are joined once at the end, in the order of the warps, through
// the shared memories of the cluster: one launch, no workspace, the same bits every time.
// Bound by HBM: each visible key and value is read once for all heads of its group.  With 16-bit types both products are warp MMAs with
// the heads as columns, S^T = K Q^T (16 keys x 8 heads) and O^T += V^T P^T, P rounded to the type of V as in the forward kernel: with the heads
// as 16 rows a tile took 627 instructions and 64 accumulators a thread, most of them for heads that are not there.  fp32 runs on the CUDA
// cores, lanes by keys for the scores and by columns for O.
// The weights are taken at the running maximum, so that no tile waits for a reduction over its lanes (64 sequences, 4100 tokens, 32 heads of
// 128 on 8, bf16: 186 us, 5.8 TB/s of 6.5 measured for a copy; one sequence of 2052 tokens 9.7 us, most of it the chain length -> page ->
// data -> join).  fp32: 16 sequences of 2004 tokens 81 us, 3.2 TB/s, bound by the multiply-adds' shared memory reads.
// Rows of a tile that are not seen (behind the end, before the window, no page) are zero-filled instead of loaded.
constexpr int kDecWarps = 4, kDecHeads = 16, kMaxSplit = 16;
// The maximum of rows that have seen something is at least this: -inf is left to those that have seen nothing, whose output is zero,
// while a row of nothing but scores of -inf ends as 0 / 0.
constexpr float kLowest = -3.0e38f;

template <typename T, int DK, int DV>
struct DecodeShape {
  static constexpr int KT = sizeof(T) == 4 ? 8 : 16;
  static constexpr int kRowK = DK * sizeof(T), kRowV = DV * sizeof(T), kStage = KT * (kRowK + kRowV);
  static constexpr int kStages = DK + DV == 256 ? 3 : DK + DV == 192 ? 4 : 6;
  static constexpr int kRing = kDecWarps * kStages * kStage;
  static constexpr int kQ = sizeof(T) == 4 ? kDecHeads * DK * 4 + kDecWarps * KT * kDecHeads * 4 : 0;    // fp32: queries, weights of a tile
  static constexpr int kSmem = kRing + kQ;
  static_assert(kDecWarps * kDecHeads * DV * 4 + kDecHeads * DV * 4 <= kRing, "partial results lie over the ring");
};

__device__ __forceinline__ uint32_t smem_of(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of 16-bit elements held by a warp.
__device__ __forceinline__ uint32_t movm_t(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float x, float y) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_peer(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}

// grid = C * B * Hkv * head groups, clusters of C = a.split.  HPL: 16-bit types, eights of heads; fp32, heads per lane of the
// scores (4 HPL heads at most).
template <typename T, int DK, int DV, int HPL>
__global__ void __launch_bounds__(32 * kDecWarps) decode_split_kernel(const __grid_constant__ DecodeArgs a) {
  using S = DecodeShape<T, DK, DV>;
  constexpr int KT = S::KT, E = 16 / sizeof(T);
  constexpr bool kMma = sizeof(T) == 2;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ml[2][kDecWarps][kDecHeads], cml[2][kDecHeads], cw[2][kDecHeads][kMaxSplit + 1];
  pdl_enter();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t C = a.split, rank = C > 1 ? cluster_rank() : 0u;
  const int groups = (a.G + kDecHeads - 1) / kDecHeads, unit = blockIdx.x / C;
  const int grp = unit % groups, hk = unit / groups % a.Hkv, b = unit / groups / a.Hkv;
  const int h0 = hk * a.G + grp * kDecHeads, nh = min(kDecHeads, a.G - grp * kDecHeads);
  const int len = decode_len(a, b);
  const int lo = (int)max((int64_t)0, (int64_t)len - a.W), sinks = min(a.ns, lo), first = lo / KT * KT;
  const int n_sink = (sinks + KT - 1) / KT, tiles = n_sink + (len - first + KT - 1) / KT;
  const int me = rank * kDecWarps + warp, parts = C * kDecWarps;
  const int t0 = (int)((int64_t)tiles * me / parts), t1 = (int)((int64_t)tiles * (me + 1) / parts);

  uint8_t* ring = smem + warp * S::kStages * S::kStage;
  // LR lanes share a row of a tile: its page and slot (page -1 if nothing of it is seen), and units u, u + LR, .. of it, so that
  // an instruction asks for whole 32-byte sectors and a row's address is computed once.
  constexpr int LR = 32 / KT, CK = DK / E, CV = DV / E;          // units of a row
  const int lr = lane / LR, lu = lane % LR;
  struct Where { int page, slot; };
  const int32_t* table = a.page_table + (int64_t)b * a.max_pages;
  auto locate = [&](int t) {
    Where w{-1, 0};
    const int p = t < n_sink ? t * KT + lr : first + (t - n_sink) * KT + lr;
    if (t < t1 && (t < n_sink ? p < sinks : p >= lo && p < len)) {
      const int lp = a.page_shift >= 0 ? p >> a.page_shift : p / a.page_size;
      w.page = table[lp];
      w.slot = p - lp * a.page_size;
    }
    return w;
  };
  // (strides of pages and slots fit 32 bits here)
  const int32_t ks0 = (int32_t)a.k.s0, ks2 = (int32_t)a.k.s2, vs0 = (int32_t)a.v.s0, vs2 = (int32_t)a.v.s2;
  const T* const k_base = (const T*)a.k.ptr + hk * a.k.s1 + lu * E;
  const T* const v_base = (const T*)a.v.ptr + hk * a.v.s1 + lu * E;
  const uint32_t x0 = (uint32_t)((lu ^ (lr & 7)) << 4);          // unit lu of the row, swizzled: unit c lies at c ^ (row & 7)
  auto load = [&](int stage, const Where& w) {
    const uint32_t k_s = smem_of(ring + stage * S::kStage) + lr * S::kRowK, v_s = smem_of(ring + stage * S::kStage) + KT * S::kRowK + lr * S::kRowV;
    const bool on = (uint32_t)w.page < (uint32_t)a.n_pages;
    const T* kp = k_base + (on ? (int64_t)w.page * ks0 + (int64_t)w.slot * ks2 : 0);
    const T* vp = v_base + (on ? (int64_t)w.page * vs0 + (int64_t)w.slot * vs2 : 0);
    // units of this lane that exist; a source of 0 bytes is not read
    const int nk = on ? a.dqk - lu * E : 0, nv = on ? a.dv - lu * E : 0;
#pragma unroll
    for (int x = 0; x < CK / LR; ++x) cp_async16(k_s + (x0 ^ (x * LR << 4)), kp + x * LR * E, x * LR * E < nk ? 16 : 0);
#pragma unroll
    for (int x = 0; x < CV / LR; ++x) cp_async16(v_s + (x0 ^ (x * LR << 4)), vp + x * LR * E, x * LR * E < nv ? 16 : 0);
  };

  // the ring holds tiles t .. t + kStages - 2; `sees` the visible keys of each, a bit per lane
  uint32_t sees[S::kStages];
  Where w0 = locate(t0), w1 = locate(t0 + 1);
#pragma unroll
  for (int s = 0; s < S::kStages - 1; ++s) {
    sees[s] = __ballot_sync(0xffffffffu, (uint32_t)w0.page < (uint32_t)a.n_pages);
    load(s, w0);
    cp_commit();
    w0 = w1;
    w1 = locate(t0 + s + 2);
  }

  // queries: MMA fragments in registers (head lane / 4 of each eight), or fp32 in shared memory
  constexpr int NT = kMma ? HPL : 1;                             // eights of heads
  uint32_t qf[kMma ? DK / 16 : 1][2 * NT];
  float* qs = reinterpret_cast<float*>(smem + S::kRing);
  if constexpr (kMma) {
#pragma unroll
    for (int k = 0; k < DK / 16; ++k)
#pragma unroll
      for (int x = 0; x < 2 * NT; ++x) {
        const int r = (lane >> 2) + 8 * (x >> 1), c = 16 * k + 2 * (lane & 3) + 8 * (x & 1);
        uint32_t v = 0;
        if (r < nh && c < a.dqk) v = *reinterpret_cast<const uint32_t*>(row_ptr<T>(a.q, b, h0 + r, 0) + c);
        qf[k][x] = v;
      }
  } else {
    for (int x = threadIdx.x; x < kDecHeads * DK; x += 32 * kDecWarps) {
      const int r = x / DK, c = x % DK;
      qs[x] = r < nh && c < a.dqk ? to_f(row_ptr<T>(a.q, b, h0 + r, 0)[c]) : 0.f;
    }
    __syncthreads();
  }
  // Running maximum and sum.  MMA: of heads 8 n + 2 (lane % 4) and + 1, O^T of those heads and dims 16 x + lane / 4 and + 8;
  // fp32: of heads HPL (lane / 8) .., O of all heads and four columns.
  constexpr int NH = kMma ? 2 * NT : HPL;
  float o[kMma ? DV / 16 * 4 * NT : 4 * 4 * HPL];
  float m[NH], l[NH];
#pragma unroll
  for (auto& x : o) x = 0.f;
#pragma unroll
  for (int x = 0; x < NH; ++x) {
    m[x] = -INFINITY;
    l[x] = 0.f;
  }
  int stage = 0;
#pragma unroll 1
  for (int t = t0; t < t1; ++t) {
    cp_wait<S::kStages - 2>();
    __syncwarp();
    const uint32_t see = sees[0];
    const uint32_t k_s = smem_of(ring + stage * S::kStage), v_s = k_s + KT * S::kRowK;
    // the tile after those in flight, into the stage that was read last
    auto refill = [&]() {
#pragma unroll
      for (int s = 0; s + 2 < S::kStages; ++s) sees[s] = sees[s + 1];
      sees[S::kStages - 2] = __ballot_sync(0xffffffffu, (uint32_t)w0.page < (uint32_t)a.n_pages);
      load(stage == 0 ? S::kStages - 1 : stage - 1, w0);
      cp_commit();
      w0 = w1;
      w1 = locate(t + S::kStages + 1);
      if (++stage == S::kStages) stage = 0;
    };
    if constexpr (kMma) {
      float s[NT][4], s2[NT][4];                                 // (two chains of accumulations)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
      // lanes 0-15: the keys, 16-31: the same keys' next 8 dims
      const int kr = lane & 15;
      const uint32_t ka = k_s + kr * S::kRowK, kx = (uint32_t)(((lane >> 4) ^ (kr & 7)) << 4);
      uint32_t kf[DK / 16][4];
#pragma unroll
      for (int k = 0; k < DK / 16; ++k) ldsm4(kf[k], ka + (kx ^ (k << 5)));
#pragma unroll
      for (int k = 0; k < DK / 16; k += 2) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma16816<T>(s[n], kf[k], qf[k][2 * n], qf[k][2 * n + 1]);
          mma16816<T>(s2[n], kf[k + 1], qf[k + 1][2 * n], qf[k + 1][2 * n + 1]);
        }
      }
      // lanes 0-7: keys 0-7, 8-15: the same keys' next 8 columns, 16-31: keys 8-15
      const int vr = (lane & 7) + (lane >> 4) * 8;
      const uint32_t va = v_s + vr * S::kRowV, vx = (uint32_t)(((lane >> 3 & 1) ^ (vr & 7)) << 4);
      uint32_t vf[DV / 16][4];
#pragma unroll
      for (int x = 0; x < DV / 16; ++x) ldsm4t(vf[x], va + (vx ^ (x << 5)));
      refill();
      // keys lane / 4 and + 8: bits 2 * key
      const bool on0 = see >> (2 * (lane >> 2)) & 1u, on1 = see >> (2 * (lane >> 2) + 16) & 1u;
      // The weights are taken at the running maximum, without waiting for the tile's own; only when a score is beyond it by 2^8
      // (the first tile, then rarely) the maximum is reduced over the tile and the sums are scaled.
      float w[NT][4];
      bool grow = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[n][e] = (e < 2 ? on0 : on1) ? (s[n][e] + s2[n][e]) * a.c2 : -INFINITY;
          const float mh = m[2 * n + (e & 1)];
          grow |= w[n][e] - mh > 8.f || (see && mh == -INFINITY);
        }
      if (__any_sync(0xffffffffu, grow)) {
        float f[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          float v = fmaxf(w[h >> 1][h & 1], w[h >> 1][(h & 1) + 2]);
#pragma unroll
          for (int z = 4; z < 32; z <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, z));
          const float mn = fmaxf(fmaxf(m[h], v), kLowest);
          f[h] = m[h] == mn ? 1.f : ex2(m[h] - mn);
          m[h] = mn;
          l[h] *= f[h];
        }
#pragma unroll
        for (int x = 0; x < DV / 16 * 4 * NT; ++x) o[x] *= f[x / 4 % NT * 2 + (x & 1)];
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[n][e] = w[n][e] == -INFINITY ? 0.f : ex2(w[n][e] - m[2 * n + (e & 1)]);
          l[2 * n + (e & 1)] += w[n][e];
        }
        pf[n][0] = movm_t(pack_pair<T>(w[n][0], w[n][1]));
        pf[n][1] = movm_t(pack_pair<T>(w[n][2], w[n][3]));
      }
#pragma unroll
      for (int x = 0; x < DV / 16; ++x)
#pragma unroll
        for (int n = 0; n < NT; ++n) mma16816<T>(o + 4 * (x * NT + n), vf[x], pf[n][0], pf[n][1]);
    } else {
      // scores: lane = key (lane & 7) x heads HPL * (lane / 8) ..; weights through shared memory; O: lane = 4 columns
      float* ws = reinterpret_cast<float*>(smem + S::kRing + kDecHeads * DK * 4) + warp * KT * kDecHeads;
      refill();
      const int key = lane & 7, hl = (lane >> 3) * HPL;
      const uint8_t* kp = smem + (k_s - smem_of(smem)) + key * S::kRowK;
      const uint8_t* vp = smem + (v_s - smem_of(smem));
      float s[HPL] = {};
#pragma unroll 8
      for (int c = 0; c < DK / 4; ++c) {
        const float4 kv = *reinterpret_cast<const float4*>(kp + ((c ^ key) << 4));
#pragma unroll
        for (int x = 0; x < HPL; ++x) {
          const float4 qv = *reinterpret_cast<const float4*>(qs + (hl + x) * DK + 4 * c);
          s[x] = fmaf(kv.x, qv.x, fmaf(kv.y, qv.y, fmaf(kv.z, qv.z, fmaf(kv.w, qv.w, s[x]))));
        }
      }
      bool moved = false;
#pragma unroll
      for (int x = 0; x < HPL; ++x) {
        // (m, l of lane's own heads at index x; the other lanes' heads are read through shared memory at the end)
        const float v0 = see >> (4 * key) & 1u ? s[x] * a.c2 : -INFINITY;
        float v = v0;
#pragma unroll
        for (int y = 4; y; y >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, y));
        const float mn = see ? fmaxf(fmaxf(m[x], v), kLowest) : m[x], f = m[x] == mn ? 1.f : exp2f(m[x] - mn);
        const float w = v0 == -INFINITY ? 0.f : exp2f(v0 - mn);
        float sum = w;
#pragma unroll
        for (int y = 4; y; y >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, y);
        l[x] = l[x] * f + sum;
        m[x] = mn;
        s[x] = f;
        moved |= f != 1.f;
        ws[key * kDecHeads + hl + x] = w;
      }
      __syncwarp();
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int h = 0; h < 4 * HPL; ++h) {
          const float f = __shfl_sync(0xffffffffu, s[h % HPL], h / HPL * 8);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[4 * h + e] *= f;
        }
      }
      if (4 * lane < DV) {
#pragma unroll
        for (int k = 0; k < KT; ++k) {
          const float4 vv = *reinterpret_cast<const float4*>(vp + k * S::kRowV + ((lane ^ k) << 4));
#pragma unroll
          for (int h = 0; h < 4 * HPL; ++h) {
            const float w = ws[k * kDecHeads + h];
            o[4 * h] = fmaf(w, vv.x, o[4 * h]);
            o[4 * h + 1] = fmaf(w, vv.y, o[4 * h + 1]);
            o[4 * h + 2] = fmaf(w, vv.z, o[4 * h + 2]);
            o[4 * h + 3] = fmaf(w, vv.w, o[4 * h + 3]);
          }
        }
      }
      __syncwarp();
    }
  }
  cp_wait<0>();
  __syncthreads();

  // ---- join: warps of the CTA, then CTAs of the cluster
  float* po = reinterpret_cast<float*>(smem);                    // [warp][head][DV]
  float* co = po + kDecWarps * kDecHeads * DV;                   // [head][DV]
  if constexpr (kMma) {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
      for (int z = 4; z < 32; z <<= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], z);
      const int r = 8 * (h >> 1) + 2 * (lane & 3) + (h & 1);
      if (lane < 4) {
        ml[0][warp][r] = m[h];
        ml[1][warp][r] = l[h];
      }
      if (r < nh) {
#pragma unroll
        for (int x = 0; x < DV / 16; ++x)
#pragma unroll
          for (int z = 0; z < 2; ++z)
            po[(warp * kDecHeads + r) * DV + 16 * x + 8 * z + (lane >> 2)] = o[4 * (x * NT + (h >> 1)) + 2 * z + (h & 1)];
      }
    }
  } else {
    if ((lane & 7) == 0) {
#pragma unroll
      for (int x = 0; x < HPL; ++x) {
        ml[0][warp][(lane >> 3) * HPL + x] = m[x];
        ml[1][warp][(lane >> 3) * HPL + x] = l[x];
      }
    }
    if (4 * lane < DV) {
#pragma unroll
      for (int h = 0; h < 4 * HPL; ++h)
        if (h < nh) *reinterpret_cast<float4*>(po + (warp * kDecHeads + h) * DV + 4 * lane) = make_float4(o[4 * h], o[4 * h + 1], o[4 * h + 2], o[4 * h + 3]);
    }
  }
  __syncthreads();
  T* const out = (T*)a.o.ptr + b * a.o.s0;
  for (int x = threadIdx.x; x < nh * (DV / 4); x += 32 * kDecWarps) {
    const int r = x / (DV / 4), c = x % (DV / 4) * 4;
    float mx = -INFINITY, sum = 0.f, acc[4] = {};
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) mx = fmaxf(mx, ml[0][w][r]);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float f = ml[0][w][r] == -INFINITY ? 0.f : exp2f(ml[0][w][r] - mx);
      const float4 v = *reinterpret_cast<const float4*>(po + (w * kDecHeads + r) * DV + c);
      sum = fmaf(f, ml[1][w][r], sum);
      acc[0] = fmaf(f, v.x, acc[0]); acc[1] = fmaf(f, v.y, acc[1]); acc[2] = fmaf(f, v.z, acc[2]); acc[3] = fmaf(f, v.w, acc[3]);
    }
    if (C == 1) {
      const float inv = mx == -INFINITY ? 0.f : 1.f / sum;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.dv) out[(int64_t)(h0 + r) * a.o.s1 + (c + e) * a.o.s3] = from_f<T>(acc[e] * inv);
    } else {
      *reinterpret_cast<float4*>(co + r * DV + c) = make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (c == 0) {
        cml[0][r] = mx;
        cml[1][r] = sum;
      }
    }
  }
  if (C == 1) return;
  cluster_sync();
  // weight of each CTA's part of a head, then the sums; a thread's loads from its peers are in flight together
  for (int x = threadIdx.x; x < nh * (int)C; x += 32 * kDecWarps) {
    const int r = x / C, k = x % C;
    cw[0][r][k] = ld_peer(smem_of(&cml[0][r]), k);
    cw[1][r][k] = ld_peer(smem_of(&cml[1][r]), k);
  }
  __syncthreads();
  if (threadIdx.x < nh) {
    const int r = threadIdx.x;
    float mx = -INFINITY, sum = 0.f;
    for (int k = 0; k < (int)C; ++k) mx = fmaxf(mx, cw[0][r][k]);
    for (int k = 0; k < (int)C; ++k) {
      const float f = cw[0][r][k] == -INFINITY ? 0.f : exp2f(cw[0][r][k] - mx);
      sum = fmaf(f, cw[1][r][k], sum);
      cw[0][r][k] = f;
    }
    cw[0][r][kMaxSplit] = mx == -INFINITY ? 0.f : 1.f / sum;
  }
  __syncthreads();
  for (int x = rank * 32 * kDecWarps + threadIdx.x; x < nh * DV; x += C * 32 * kDecWarps) {
    const int r = x / DV, c = x % DV;
    float v[kMaxSplit], acc = 0.f;
#pragma unroll
    for (int k = 0; k < kMaxSplit; ++k)
      if (k < (int)C) v[k] = ld_peer(smem_of(co + r * DV + c), k);
#pragma unroll
    for (int k = 0; k < kMaxSplit; ++k)
      if (k < (int)C) acc = fmaf(cw[0][r][k], v[k], acc);
    if (c < a.dv) out[(int64_t)(h0 + r) * a.o.s1 + c * a.o.s3] = from_f<T>(acc * cw[0][r][kMaxSplit]);
  }
  cluster_sync();                                                // nobody leaves while its shared memory is read
}

}  // namespace sink
}  // namespace swa
