// tcgen05 forward kernel of the attention with a sliding window and sink tokens (definition: sink_rows.cuh).
//
// One pass over the keys with the running maximum and sum of the softmax: per row i, over blocks of 128 keys,
//   S = Q K^T;  m' = max(m, max S);  P = exp2(c (S - m'));  l = l exp2(c (m - m')) + sum P;  O = O exp2(c (m - m')) + P V
// and o = O / l, lse = c m + log2 l.
//
// A CTA (one per SM, 384 threads, persistent) works on a pair of tiles of 128 queries that meet the same blocks: two heads of one
// key head where heads come in pairs, else two neighbouring tiles of one head; keys and values are loaded once for both
// (at d = 128 a tile of its own would want 64 bytes a cycle of L2, more than it gives).  The blocks are those of
// the window, from the diagonal down, then the blocks of sinks the window does not reach, of which only the sinks' columns, in
// steps of 16, are multiplied.
//   warp 0       TMA producer: queries, rings of key and value blocks
//   warp 1       issues every MMA: S_t of the next block behind O_t += P_t V of this one, tile by tile, so that the tensor pipe works on
//                one tile while the other's softmax runs
//   warps 4-7, 8-11   softmax and epilogue of tile 0 and 1, one thread per row; P (16-bit) goes over the scores in tensor memory
// Tensor memory: S_0, S_1 (128 columns each), O_0, O_1.  The maximum a row is scaled by is raised only when it has grown by 2^8, so the
// accumulator is touched rarely; S_t of a block is complete only after P_t V of the block before (one issuing thread, in order),
// which is what makes the accumulator safe to touch.
//
// A hidden pair has P = 0, which is nothing to a sum until the value is an infinity or a NaN: a row that ends as one is done again
// by row_forward, which touches only what the row sees, after the CTA's last tile.
//
// All waits are bounded (umma.cuh); a warp whose wait gave up leaves its loops, the others run into their own limit.
#pragma once

#include "sink_rows.cuh"
#include "swa_tc_common.cuh"
#include "umma.cuh"

namespace swa {
namespace sink {

constexpr int kFwdThreadsS = 384, kTile = 128;
constexpr uint32_t kChunk = 16384;              // 128 rows of 64 elements
constexpr float kGrow = 8.f;                    // a row's maximum may lag by 2^8

struct FwdParams {
  Args a;
  int n_items, n_y, n_x, pair_heads, stages;    // items: n_y query positions (descending) x B x n_x
  int32_t* status;
};

struct FwdShared {
  uint64_t q_full, q_empty, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], p_full[2], o_full[2], o_empty[2];
  uint32_t tmem_base;
  int abort_flag, bad;
};

// The blocks of one pair of tiles.
struct FwdItem {
  int b, hk, len, h[2], q0[2];
  int hi[2], lo[2];                             // a tile's blocks in its window; hi = -1: no rows
  int bhi, blo, sbn, sb, nwin, nb;              // union; blocks that hold sinks, those of them below the union; counts
  __device__ __forceinline__ int block(int n) const { return n < nwin ? bhi - n : sb - 1 - (n - nwin); }
  __device__ __forceinline__ bool takes(int t, int blk) const { return blk <= hi[t] && (blk >= lo[t] || blk < sbn); }
  __device__ __forceinline__ int last(int t) const { return sb > 0 || blo < sbn ? nb - 1 : bhi - lo[t]; }
};

__device__ __forceinline__ FwdItem fwd_item(const FwdParams& p, int item) {
  const Args& a = p.a;
  FwdItem w;
  const int per = a.B * p.n_x, y = p.n_y - 1 - item / per, r = item % per;
  w.b = r / p.n_x;
  const int x = r % p.n_x;
  w.len = seq_len(a, w.b);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w.h[t] = p.pair_heads ? 2 * x + t : x;
    w.q0[t] = (p.pair_heads ? y : 2 * y + t) * kTile;
    w.hi[t] = w.q0[t] < w.len ? w.q0[t] / kTile : -1;          // the diagonal block: the tile's rows see no later one
    w.lo[t] = max(0, w.q0[t] - a.W + 1) / kTile;
  }
  w.hk = w.h[0] / a.G;
  w.sbn = (a.ns + kTile - 1) / kTile;
  w.bhi = max(w.hi[0], w.hi[1]);
  w.blo = w.lo[0];
  w.sb = min(w.sbn, w.blo);
  w.nwin = w.bhi < 0 ? 0 : w.bhi - w.blo + 1;
  w.nb = w.bhi < 0 ? 0 : w.nwin + w.sb;
  return w;
}

// Columns of a block that a tile multiplies: all of a window's block, of a block of sinks only the sinks, in steps of 16.
__device__ __forceinline__ int fwd_cols(const Args& a, int blk, int lo) {
  return blk >= lo ? kTile : min(kTile, (a.ns - blk * kTile + 15) & ~15);
}

// Bits of columns 32 w .. 32 w + 31 below n.
__device__ __forceinline__ uint32_t below(int n, int w) {
  n -= 32 * w;
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

template <bool BF16>
__device__ __forceinline__ void exp_pack32(const float* s, uint64_t c22, uint64_t nmc2, uint64_t* ls, uint32_t* w) {
  using namespace ptx;
#pragma unroll
  for (int h = 0; h < 16; ++h) {
    const float2 x = f2_unpack(f2_fma(f2_pack(s[2 * h], s[2 * h + 1]), c22, nmc2));
    const float p0 = exp2f(x.x), p1 = exp2f(x.y);
    ls[h & 1] = f2_add(ls[h & 1], f2_pack(p0, p1));
    w[h] = tc::pack2<BF16>(p0, p1);
  }
}

template <bool BF16, int QC, int VC>
__global__ void __launch_bounds__(kFwdThreadsS, 1)
sink_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ FwdParams p) {
  using namespace ptx;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const Args& a = p.a;
  uint8_t* q_smem = smem;                                        // tile, chunk
  uint8_t* k_smem = q_smem + 2 * QC * kChunk;                    // stage, chunk
  uint8_t* v_smem = k_smem + p.stages * QC * kChunk;
  FwdShared* sh = reinterpret_cast<FwdShared*>(v_smem + p.stages * VC * kChunk);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kO = 256, kOCols = VC * 64;                 // tensor memory: O_t at kO + t * kOCols

  if (threadIdx.x < offsetof(FwdShared, tmem_base) / 8) {
    uint64_t* bar = reinterpret_cast<uint64_t*>(sh) + threadIdx.x;
    const bool warps4 = (bar >= sh->p_full && bar < sh->p_full + 2) || (bar >= sh->o_empty && bar < sh->o_empty + 2);
    mbar_init(bar, warps4 ? 4 : 1);
  }
  if (threadIdx.x == 0) sh->abort_flag = sh->bad = 0;
  fence_barrier_init();
  if (warp == 1) {
    tmem_alloc(&sh->tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_enter();
  pdl_wait();
  const uint32_t tmem = sh->tmem_base;
  bool ok = true;                                                // warp-uniform: false once a wait has given up
  auto wait = [&](uint64_t* bar, uint32_t parity) { ok &= __all_sync(0xffffffffu, mbar_wait_polls<0>(smem_u32(bar), parity)) != 0; };

  if (warp < 4) {
    setmaxnreg_dec<72>();
    if (warp == 0) {
      // ---------------------------------------------------------------- producer
      const uint32_t el = elect_one();
      int st = 0, par = 1, q_par = 1;
      for (int item = blockIdx.x; ok && item < p.n_items; item += gridDim.x) {
        const FwdItem w = fwd_item(p, item);
        if (!w.nb) continue;
        wait(&sh->q_empty, q_par);
        q_par ^= 1;
        if (!ok) break;
        mbar_expect_tx_el(el, smem_u32(&sh->q_full), 2 * QC * kChunk);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int c = 0; c < QC; ++c)
            tma_load_4d_el(el, smem_u32(q_smem) + (t * QC + c) * kChunk, &tm_q, smem_u32(&sh->q_full), 64 * c, w.q0[t], w.h[t], w.b);
        for (int n = 0; n < w.nb; ++n) {
          const int row = w.block(n) * kTile;
          wait(&sh->k_empty[st], par);
          if (!ok) break;
          mbar_expect_tx_el(el, smem_u32(&sh->k_full[st]), QC * kChunk);
#pragma unroll
          for (int c = 0; c < QC; ++c)
            tma_load_4d_el(el, smem_u32(k_smem) + (st * QC + c) * kChunk, &tm_k, smem_u32(&sh->k_full[st]), 64 * c, row, w.hk, w.b);
          wait(&sh->v_empty[st], par);
          if (!ok) break;
          mbar_expect_tx_el(el, smem_u32(&sh->v_full[st]), VC * kChunk);
#pragma unroll
          for (int c = 0; c < VC; ++c)
            tma_load_4d_el(el, smem_u32(v_smem) + (st * VC + c) * kChunk, &tm_v, smem_u32(&sh->v_full[st]), 64 * c, row, w.hk, w.b);
          if (++st == p.stages) { st = 0; par ^= 1; }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t el = elect_one();
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint32_t hi_sw = smem_desc_hi(1024, true);
      const uint64_t q_d = smem_desc_from(smem_u32(q_smem), 16, hi_sw), k_d = smem_desc_from(smem_u32(k_smem), 16, hi_sw),
                     v_d = smem_desc_from(smem_u32(v_smem), kChunk, hi_sw);
      const uint32_t id_pv = instr_desc(fmt, 128, kOCols, 0, 1);
      int ks = 0, kpar = 0, vs = 0, vpar = 0, q_par = 0;
      uint32_t p_par = 0, o_par = 3;                             // a bit per tile
      auto scores = [&](const FwdItem& w, int t, int blk) {      // S_t = Q_t K^T from key stage ks
        const uint32_t id = instr_desc(fmt, 128, fwd_cols(a, blk, w.lo[t]), 0, 0);
        const uint64_t qd = q_d + (uint64_t)(t * QC * (kChunk >> 4)), kd = k_d + (uint64_t)(ks * QC * (kChunk >> 4));
#pragma unroll
        for (int k = 0; k < 4 * QC; ++k)
          umma_ss_el(el, tmem + t * 128, qd + (k >> 2) * (kChunk >> 4) + 2 * (k & 3), kd + (k >> 2) * (kChunk >> 4) + 2 * (k & 3), id, k ? 1u : 0u);
        umma_commit_el(el, &sh->s_full[t]);
      };
      auto next_k = [&]() {
        umma_commit_el(el, &sh->k_empty[ks]);
        if (++ks == p.stages) { ks = 0; kpar ^= 1; }
      };
      for (int item = blockIdx.x; ok && item < p.n_items; item += gridDim.x) {
        const FwdItem w = fwd_item(p, item);
        if (!w.nb) continue;
        wait(&sh->q_full, q_par);
        q_par ^= 1;
        wait(&sh->k_full[ks], kpar);
        if (!ok) break;
        tc_fence_after();
        for (int t = 0; t < 2; ++t)
          if (w.takes(t, w.bhi)) scores(w, t, w.bhi);
        next_k();
        if (w.nb == 1) umma_commit_el(el, &sh->q_empty);
        for (int n = 0; n < w.nb; ++n) {
          const int blk = w.block(n);
          const bool more = n + 1 < w.nb;
          const int nxt = more ? w.block(n + 1) : -1;
          if (more) wait(&sh->k_full[ks], kpar);
          wait(&sh->v_full[vs], vpar);
          for (int t = 0; t < 2; ++t) {
            if (w.takes(t, blk)) {
              if (n == w.bhi - w.hi[t]) {                        // the tile's first block: its accumulator has been read
                wait(&sh->o_empty[t], o_par >> t & 1u);
                o_par ^= 1u << t;
              }
              wait(&sh->p_full[t], p_par >> t & 1u);
              p_par ^= 1u << t;
              if (!ok) break;
              tc_fence_after();
              const uint32_t first = n == w.bhi - w.hi[t] ? 0u : 1u;
              const uint64_t vd = v_d + (uint64_t)(vs * VC * (kChunk >> 4));
              const int steps = fwd_cols(a, blk, w.lo[t]) >> 4;
              if (steps == 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k) umma_ts_el(el, tmem + kO + t * kOCols, tmem + t * 128 + 8 * k, vd + 128 * k, id_pv, k ? 1u : first);
              } else {
                for (int k = 0; k < steps; ++k) umma_ts_el(el, tmem + kO + t * kOCols, tmem + t * 128 + 8 * k, vd + 128 * k, id_pv, k ? 1u : first);
              }
              if (n == w.last(t)) umma_commit_el(el, &sh->o_full[t]);
            }
            if (more && w.takes(t, nxt)) {
              tc_fence_after();
              scores(w, t, nxt);
            }
          }
          if (!ok) break;
          if (more) {
            next_k();
            if (n + 2 == w.nb) umma_commit_el(el, &sh->q_empty);
          }
          umma_commit_el(el, &sh->v_empty[vs]);
          if (++vs == p.stages) { vs = 0; vpar ^= 1; }
        }
      }
    }
  } else {
    setmaxnreg_inc<208>();
    // ------------------------------------------------------------------ softmax and epilogue, one thread per row
    const int t = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tm = lanes + t * 128, o_tm = lanes + kO + t * kOCols;
    const float c2 = a.c2;
    const uint64_t c22 = f2_pack(c2, c2);
    uint32_t s_par = 0, o_par = 0;
    for (int item = blockIdx.x; ok && item < p.n_items; item += gridDim.x) {
      const FwdItem w = fwd_item(p, item);
      const int i = w.q0[t] + r, h = w.h[t];
      float m = -INFINITY, l = 0.f;
      const int n0 = w.bhi - w.hi[t], n1 = w.hi[t] < 0 ? -1 : w.last(t);
      for (int n = n0; n <= n1; ++n) {
        const int blk = w.block(n);
        if (!w.takes(t, blk)) continue;
        const int kb = blk * kTile, cols = fwd_cols(a, blk, w.lo[t]);
        const bool first = n == n0;
        // what the row sees of the block: columns up to cr, from cl on or below cs
        const int cr = min(i, w.len - 1) - kb, cl = i - a.W + 1 - kb, cs = a.ns - kb;
        const bool edge = blk >= w.lo[t] ? kb + kTile - 1 > w.q0[t] || (kb <= w.q0[t] + kTile - 1 - a.W && cs < kTile) || kb + kTile > w.len
                                         : cs < cols;
        wait(&sh->s_full[t], s_par);
        s_par ^= 1;
        if (!ok) break;
        tc_fence_after();
        auto grow = [&](float mx) {                              // the maximum the row is scaled by
          if (first) {
            m = mx;
            return;
          }
          const bool need = (mx - m) * c2 > kGrow || (m == -INFINITY && mx > m);
          if (__any_sync(0xffffffffu, need)) {
            const float f = need ? exp2f((m - mx) * c2) : 1.f;
#pragma unroll 1
            for (int c = 0; c < (int)kOCols; c += 16) {
              uint32_t x[16];
              tmem_ld16(o_tm + c, x);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
              tmem_st16(o_tm + c, x);
            }
            if (need) { m = mx; l *= f; }
          }
        };
        uint64_t ls[2] = {0ull, 0ull};
        if (cols == kTile) {
          float s[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(s_tm + 32 * c, reinterpret_cast<uint32_t*>(s) + 32 * c);
          tmem_wait_ld();
          if (edge) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint32_t see = below(cr + 1, c) & (~below(cl, c) | below(cs, c));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(see >> e & 1u)) s[32 * c + e] = -INFINITY;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 128; e += 2) mx[(e >> 1) & 3] = fmaxf(mx[(e >> 1) & 3], fmaxf(s[e], s[e + 1]));
          grow(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const float mc = m == -INFINITY ? 0.f : m * c2;
          const uint64_t nmc2 = f2_pack(-mc, -mc);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pw[16];
            exp_pack32<BF16>(s + 32 * c, c22, nmc2, ls, pw);
            tmem_st16(s_tm + 16 * c, pw);
          }
        } else {
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < cols; c += 16) {
            uint32_t s[16];
            tmem_ld16(s_tm + c, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c + e < cs) mx = fmaxf(mx, __uint_as_float(s[e]));
          }
          grow(mx);
          const float mc = m == -INFINITY ? 0.f : m * c2;
#pragma unroll 1
          for (int c = 0; c < cols; c += 16) {
            uint32_t s[16], pw[8];
            tmem_ld16(s_tm + c, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float p0 = c + 2 * e < cs ? exp2f(fmaf(__uint_as_float(s[2 * e]), c2, -mc)) : 0.f;
              const float p1 = c + 2 * e + 1 < cs ? exp2f(fmaf(__uint_as_float(s[2 * e + 1]), c2, -mc)) : 0.f;
              ls[e & 1] = f2_add(ls[e & 1], f2_pack(p0, p1));
              pw[e] = tc::pack2<BF16>(p0, p1);
            }
            tmem_st8(s_tm + (c >> 1), pw);
          }
        }
        const float2 l0 = f2_unpack(ls[0]), l1 = f2_unpack(ls[1]);
        l += (l0.x + l0.y) + (l1.x + l1.y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[t]);
      }
      if (!ok) break;
      const bool live = i < w.len, in = i < a.N;
      T* orow = (T*)a.o.ptr + w.b * a.o.s0 + h * a.o.s1 + (int64_t)i * a.o.s2;
      if (w.hi[t] < 0) {
        if (in)
          for (int c = 0; c < a.dv_dim; c += 8) *reinterpret_cast<uint4*>(orow + c) = make_uint4(0, 0, 0, 0);
      } else {
        wait(&sh->o_full[t], o_par);
        o_par ^= 1;
        if (!ok) break;
        tc_fence_after();
        const float inv = live ? 1.f / l : 0.f;
        const uint64_t inv2 = f2_pack(inv, inv);
        uint64_t z = 0ull;                                       // becomes a NaN with any infinity or NaN
#pragma unroll
        for (int c = 0; c < (int)kOCols; c += 32) {
          uint32_t x[32];
          tmem_ld32(o_tm + c, x);
          tmem_wait_ld();
          if (c + 32 == (int)kOCols) {                           // the last column has been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->o_empty[t]);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t wd[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint64_t y = f2_mul(f2_pack(__uint_as_float(x[8 * u + 2 * e]), __uint_as_float(x[8 * u + 2 * e + 1])), inv2);
              z = f2_fma(y, 0ull, z);
              const float2 f = f2_unpack(y);
              wd[e] = live ? tc::pack2<BF16>(f.x, f.y) : 0u;
            }
            if (in && c + 8 * u < a.dv_dim) *reinterpret_cast<uint4*>(orow + c + 8 * u) = make_uint4(wd[0], wd[1], wd[2], wd[3]);
          }
        }
        const float2 zz = f2_unpack(z);
        if (live && !(zz.x == 0.f && zz.y == 0.f)) sh->bad = 1;
      }
      if (in) a.lse[((int64_t)w.b * a.Hq + h) * a.N + i] = live ? fmaf(m, c2, log2f(l)) : -INFINITY;
    }
  }

  // -------------------------------------------------------------------- teardown
  if (!ok) sh->abort_flag = 1;
  tc_fence_before();
  __syncthreads();
  if (*(volatile int*)&sh->abort_flag) {
    // let whatever is still in flight (TMA, MMA) land before shared memory and tensor memory are released
#pragma unroll 1
    for (int n = 0; n < 64; ++n) __nanosleep(1000);
    if (threadIdx.x == 0) tc::report_abort(p.status, 7, 0);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (*(volatile int*)&sh->bad && !*(volatile int*)&sh->abort_flag) {
    // rows that ended as an infinity or a NaN once more, over the pairs that see each other only
    float* s = reinterpret_cast<float*>(smem) + warp * 2 * kMaxDim;
    for (int item = blockIdx.x; item < p.n_items; item += gridDim.x) {
      const FwdItem w = fwd_item(p, item);
#pragma unroll 1
      for (int x = warp; x < 2 * kTile; x += kFwdThreadsS / 32) {
        const int t = x >> 7, i = w.q0[t] + (x & 127);
        if (i >= w.len) continue;
        bool bad = false;
        const T* o = row_ptr<T>(a.o, w.b, w.h[t], i);
        for (int d = lane; d < a.dv_dim; d += 32) bad |= !(fabsf(to_f(o[d])) <= 3.0e38f);
        if (__any_sync(0xffffffffu, bad)) row_forward<T>(a, w.b, w.h[t], i, s);
      }
    }
  }
}

}  // namespace sink
}  // namespace swa
