// tcgen05 forward kernel of the attention with a sliding window and sink tokens (definition: sink_rows.cuh).
//
// One pass over the keys with the running maximum and sum of the softmax: per row i, over blocks of keys,
//   S = Q K^T;  m' = max(m, max S);  P = exp2(c (S - m'));  l = l exp2(c (m - m')) + sum P;  O = O exp2(c (m - m')) + P V
// and o = O / l, lse = c m + log2 l.
//
// A CTA (one per SM, persistent) works on a pair of tiles of 128 queries that meet the same blocks: two heads of one
// key head where heads come in pairs, else two neighbouring tiles of one head; keys and values are loaded once for both
// (at d = 128 a tile of its own would want 64 bytes a cycle of L2, more than it gives).  The blocks are those of
// the window, from the diagonal down, then the blocks of sinks the window does not reach, of which only the sinks' columns, in
// steps of 16, are multiplied.
//   warp 0       TMA producer: queries, rings of key and value blocks      warp 2   hands out the items
//   warp 1       issues S_t = Q K^T      warp 3   issues O_t += P V   (one warp for both was the bottleneck: 3500 cycles for a
//                pair of tiles and 80 keys, whose products take 1456)
//   warps 4-7, 8-11   softmax of tile 0 and 1, one thread per row      warps 12-15   epilogue
// Tensor memory: S_t (128 columns), O_t, and P_t (16-bit).  With d_v up to 64 P has columns of its own: the scores of the next block are made as
// soon as a group has taken these into registers.  Above, P lies over the scores, and the next ones are made when P V is done with
// it; the two tiles then take turns, one group's exponentials running beside the other tile's products, and P V starts on the first
// half of P.  (Blocks of 80 keys leave room for P there too, but cost more between blocks: 8192 tokens, window 4096, 16 heads of 128
// 255 us.)
// The maximum a row is scaled by is raised only when it has grown by 2^8, so the accumulator is touched rarely.
// P is rounded to the type of V: an MMA's operands have one, and a second product for what that leaves would be half of the kernel's products
// again.  O's error against 64 bits is 1.3 times that of its own rounding (l is the sum of the weights before theirs).
//
// Measured (bf16, head dims 128, 16 heads on 4): 8192 tokens, window 4096 219 us, 940 TFLOP/s of visible pairs; 16384 tokens, window
// 1024, 64 sinks 165 us, 850.  Tensor pipe 48 % busy, exponential unit 48 %: a group's chain is what is left (scores to registers 280 cycles,
// maximum 400, exponentials 1700 beside the other group's, the wait for P V and Q K^T 1400).  Tried and not kept: a part of the exponentials
// as polynomials on the fp32 pipes (one pair in eight 235 us, in two 287: issue slots, not the exponential unit, run short); reading the
// scores twice from tensor memory instead of holding 128 in registers (304 us); the running maximum of the block before with a second
// look (298 us, spills).
//
// A hidden pair has P = 0, which is nothing to a sum until the value is an infinity or a NaN: a row that ends as one is done again
// by row_forward, which touches only what the row sees, after the CTA's last tile.  Padding behind a sequence's end costs no row
// that: it is zeros before it is multiplied (zero_rows).
//
// All waits are bounded (umma.cuh); a warp whose wait gave up leaves its loops, the others run into their own limit.
#pragma once

#include "sink_tc_common.cuh"

namespace swa {
namespace sink {

constexpr float kGrow = 8.f;                    // a row's maximum may lag by 2^8

struct FwdParams {
  Args a;
  int n_items, n_y, n_x, pair_heads, stages;    // items: n_y query positions (descending) x B x n_x
  int32_t* status;
};

// The blocks of one pair of tiles.
struct FwdItem {
  int nb;                                       // blocks; -1: no more items
  int b, hk, len, h[2], q0[2];
  int hi[2], lo[2];                             // a tile's blocks in its window; hi = -1: no rows
  int bhi, blo, sbn, sb, nwin;                  // union; blocks that hold sinks, those of them below the union; blocks of the window
  __device__ __forceinline__ int block(int n) const { return n < nwin ? bhi - n : sb - 1 - (n - nwin); }
  __device__ __forceinline__ bool takes(int t, int blk) const { return blk <= hi[t] && (blk >= lo[t] || blk < sbn); }
  __device__ __forceinline__ int last(int t) const { return sb > 0 || blo < sbn ? nb - 1 : bhi - lo[t]; }
};

struct FwdShared {
  uint64_t q_full, q_empty, k_full[4], k_empty[4], v_full[4], v_empty[4], s_full[2], s_free[2], p_half[2], p_full[2], pv_done[2], o_full[2], o_empty[2],
      l_full[2], l_empty[2], item_full[kItems], item_empty[kItems], padded;
  FwdItem item[kItems];
  float inv[2][kTile];                          // 1 / l of a tile's rows
  uint32_t tmem_base;
  int abort_flag, bad;
};

template <int N>
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
    w.hi[t] = w.q0[t] < w.len ? min(w.q0[t] + kTile - 1, w.len - 1) / N : -1;
    w.lo[t] = max(0, w.q0[t] - a.W + 1) / N;
  }
  w.hk = w.h[0] / a.G;
  w.sbn = (a.ns + N - 1) / N;
  w.bhi = max(w.hi[0], w.hi[1]);
  w.blo = w.lo[0];
  w.sb = min(w.sbn, w.blo);
  w.nwin = w.bhi < 0 ? 0 : w.bhi - w.blo + 1;
  w.nb = w.bhi < 0 ? 0 : w.nwin + w.sb;
  return w;
}

// Columns of a block that a tile multiplies: all of a window's block, of a block of sinks only the sinks, in steps of 16.
template <int N>
__device__ __forceinline__ int fwd_cols(const Args& a, int blk, int lo) {
  return blk >= lo ? N : min(N, (a.ns - blk * N + 15) & ~15);
}

template <int QC, int VC>
struct FwdShape {
  static constexpr int N = 128;
  static constexpr bool kOver = VC > 1;                          // P over S
  static constexpr uint32_t kP = kOver ? 0 : 2 * N, kPStep = kOver ? N : N / 2, kO = 512 - 2 * VC * 64;     // S_t at t N, P_t at kP + t kPStep, O_t
  static constexpr uint32_t kKStage = QC * N * 128, kVStage = VC * N * 128;
  static_assert((kOver ? 2 * N : 3 * N) <= kO, "tensor memory");
};

template <bool BF16, int QC, int VC>
__global__ void __launch_bounds__(kThreads, 1)
sink_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ FwdParams p) {
  using namespace ptx;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using S = FwdShape<QC, VC>;
  constexpr int N = S::N;
  constexpr uint32_t kOCols = VC * 64, kB = N * 128;             // kB: bytes of a chunk of a block
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const Args& a = p.a;
  uint8_t* q_smem = smem;                                        // tile, chunk
  uint8_t* k_smem = q_smem + 2 * QC * kChunk;                    // stage, chunk
  uint8_t* v_smem = k_smem + p.stages * S::kKStage;
  uint8_t* stg_smem = v_smem + p.stages * S::kVStage;
  FwdShared* sh = reinterpret_cast<FwdShared*>(stg_smem + 4 * kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x < offsetof(FwdShared, item) / 8) {
    uint64_t* bar = reinterpret_cast<uint64_t*>(sh) + threadIdx.x;
    auto in = [&](uint64_t* x, int n) { return bar >= x && bar < x + n; };
    const bool warps4 = in(sh->s_free, 2) || in(sh->p_half, 2) || in(sh->p_full, 2) || in(sh->o_empty, 2) || in(sh->l_full, 2) || in(sh->l_empty, 2);
    mbar_init(bar, warps4 ? 4 : in(sh->item_empty, kItems) ? 15 : 1);
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
  // The next item from the ring; a consumer is done with it once it has copied what it needs.
  int ii = 0, ipar = 0;
  auto take = [&](FwdItem& w) {
    wait(&sh->item_full[ii], ipar);
    if (!ok) return false;
    w = sh->item[ii];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->item_empty[ii]);
    if (++ii == kItems) { ii = 0; ipar ^= 1; }
    return w.nb >= 0;
  };

  if (warp < 4) {
    setmaxnreg_dec<kRegsIssue>();
    if (warp == 0) {
      // ---------------------------------------------------------------- producer
      const uint32_t el = elect_one();
      int st = 0, par = 1, q_par = 1, pad_par = 0;
      FwdItem w;
      while (take(w)) {
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
          const int row = w.block(n) * N;
          wait(&sh->k_empty[st], par);
          if (!ok) break;
          mbar_expect_tx_el(el, smem_u32(&sh->k_full[st]), S::kKStage);
#pragma unroll
          for (int c = 0; c < QC; ++c)
            tma_load_4d_el(el, smem_u32(k_smem) + st * S::kKStage + c * kB, &tm_k, smem_u32(&sh->k_full[st]), 64 * c, row, w.hk, w.b);
          wait(&sh->v_empty[st], par);
          if (!ok) break;
          const bool pad = holds_padding<N>(row, w.len, a.N);    // (scores of hidden keys are never used, their values are multiplied)
          const uint32_t vs = smem_u32(v_smem) + st * S::kVStage, vbar = smem_u32(pad ? &sh->padded : &sh->v_full[st]);
          mbar_expect_tx_el(el, vbar, S::kVStage);
#pragma unroll
          for (int c = 0; c < VC; ++c) tma_load_4d_el(el, vs + c * kB, &tm_v, vbar, 64 * c, row, w.hk, w.b);
          if (pad) {
            wait(&sh->padded, pad_par);
            if (!ok) break;
            pad_par ^= 1;
            zero_rows<N, VC>(vs, w.len - row, lane);
            if (lane == 0) mbar_arrive(&sh->v_full[st]);
          }
          if (++st == p.stages) { st = 0; par ^= 1; }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- scores
      const uint32_t el = elect_one();
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint32_t hi_sw = smem_desc_hi(1024, true);
      const uint64_t q_d = smem_desc_from(smem_u32(q_smem), 16, hi_sw), k_d = smem_desc_from(smem_u32(k_smem), 16, hi_sw);
      const uint32_t id_full = instr_desc(fmt, 128, N, 0, 0);
      const int kq = steps16(a.dqk);
      int ks = 0, kpar = 0, q_par = 0;
      uint32_t sf_par = 3;                                       // a bit per tile
      FwdItem w;
      while (take(w)) {
        if (!w.nb) continue;
        wait(&sh->q_full, q_par);
        q_par ^= 1;
        for (int n = 0; ok && n < w.nb; ++n) {
          const int blk = w.block(n);
          wait(&sh->k_full[ks], kpar);
          const uint64_t kd = k_d + (uint64_t)(ks * (S::kKStage >> 4));
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!w.takes(t, blk)) continue;
            // the group has taken the scores before, or the product has read the P that lies over them
            wait(S::kOver ? &sh->pv_done[t] : &sh->s_free[t], sf_par >> t & 1u);
            sf_par ^= 1u << t;
            if (!ok) break;
            tc_fence_after();
            const uint32_t id = blk >= w.lo[t] ? id_full : instr_desc(fmt, 128, fwd_cols<N>(a, blk, w.lo[t]), 0, 0);
            const uint64_t qd = q_d + (uint64_t)(t * QC * (kChunk >> 4));
            scores_mma<QC>(el, tmem + t * N, qd, kd, kChunk >> 4, kB >> 4, id, kq);
            umma_commit_el(el, &sh->s_full[t]);
          }
          if (!ok) break;
          umma_commit_el(el, &sh->k_empty[ks]);
          if (++ks == p.stages) { ks = 0; kpar ^= 1; }
        }
        if (!ok) break;
        umma_commit_el(el, &sh->q_empty);
      }
    } else if (warp == 3) {
      // ---------------------------------------------------------------- O_t += P_t V
      const uint32_t el = elect_one();
      const uint32_t id_pv = instr_desc(BF16 ? 1u : 0u, 128, 16 * steps16(a.dv_dim), 0, 1);
      const uint64_t v_d = smem_desc_from(smem_u32(v_smem), kB, smem_desc_hi(1024, true));
      int vs = 0, vpar = 0;
      uint32_t p_par = 0, o_par = 3;                             // a bit per tile
      FwdItem w;
      while (take(w)) {
        const int n1[2] = {w.last(0), w.last(1)};
        for (int n = 0; ok && n < w.nb; ++n) {
          const int blk = w.block(n);
          wait(&sh->v_full[vs], vpar);
          const uint64_t vd = v_d + (uint64_t)(vs * (S::kVStage >> 4));
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!w.takes(t, blk)) continue;
            const uint32_t first = n == w.bhi - w.hi[t] ? 0u : 1u;
            if (!first) {                                        // the tile's first block: its accumulator has been read
              wait(&sh->o_empty[t], o_par >> t & 1u);
              o_par ^= 1u << t;
            }
            const uint32_t o_tm = tmem + S::kO + t * kOCols, p_tm = tmem + S::kP + t * S::kPStep;
            constexpr int kHalf = S::kOver ? N / 32 : 0;         // steps that begin on the first half of P
            if constexpr (S::kOver) {
              wait(&sh->p_half[t], p_par >> t & 1u);
              if (!ok) break;
              if (blk >= w.lo[t]) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < kHalf; ++k) umma_ts_el(el, o_tm, p_tm + 8 * k, vd + 128 * k, id_pv, k ? 1u : first);
              }
            }
            wait(&sh->p_full[t], p_par >> t & 1u);
            p_par ^= 1u << t;
            if (!ok) break;
            tc_fence_after();
            if (blk >= w.lo[t]) {
#pragma unroll
              for (int k = kHalf; k < N / 16; ++k) umma_ts_el(el, o_tm, p_tm + 8 * k, vd + 128 * k, id_pv, k ? 1u : first);
            } else {
              const int steps = fwd_cols<N>(a, blk, w.lo[t]) >> 4;
              for (int k = 0; k < steps; ++k) umma_ts_el(el, o_tm, p_tm + 8 * k, vd + 128 * k, id_pv, k ? 1u : first);
            }
            umma_commit_el(el, &sh->pv_done[t]);
            if (n == n1[t]) umma_commit_el(el, &sh->o_full[t]);
          }
          if (!ok) break;
          umma_commit_el(el, &sh->v_empty[vs]);
          if (++vs == p.stages) { vs = 0; vpar ^= 1; }
        }
        if (!ok) break;
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- items
      int s = 0, par = 1;
      for (int item = blockIdx.x; ok; item += gridDim.x) {
        const bool end = item >= p.n_items;
        FwdItem w;
        if (!end) w = fwd_item<N>(p, item);
        wait(&sh->item_empty[s], par);
        if (!ok) break;
        if (lane == 0) {
          if (!end) sh->item[s] = w;
          else sh->item[s].nb = -1;
          mbar_arrive(&sh->item_full[s]);
        }
        if (end) break;
        if (++s == kItems) { s = 0; par ^= 1; }
      }
    }
  } else if (warp < 12) {
    setmaxnreg_inc<kRegsCompute>();
    // ------------------------------------------------------------------ softmax, one thread per row
    const int t = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t s_tm = lanes + t * N, p_tm = lanes + S::kP + t * S::kPStep, o_tm = lanes + S::kO + t * kOCols;
    const float c2 = a.c2;
    const uint64_t c22 = f2_pack(c2, c2);
    uint32_t s_par = 0, l_par = 1, pv_par = 0;
    bool pv_open = false;                                        // a product of this tile that has not been waited for
    auto wait_pv = [&]() {                                       // (P over S: these scores came after it)
      if (S::kOver || !pv_open) return;
      wait(&sh->pv_done[t], pv_par);
      pv_par ^= 1;
      pv_open = false;
    };
    FwdItem w;
    while (take(w)) {
      const int q0 = w.q0[t], t_hi = w.hi[t], t_lo = w.lo[t], i = q0 + r;
      if (t_hi < 0) {
        if (i < a.N) a.lse[((int64_t)w.b * a.Hq + w.h[t]) * a.N + i] = -INFINITY;
        continue;
      }
      float m = -INFINITY, l = 0.f;
      const int n0 = w.bhi - t_hi, n1 = w.last(t);
      // keys the row sees: lo .. hi, and the sinks
      const int hi = min(i, w.len - 1), lo = i - a.W + 1;
      const int sbn = w.sbn, nwin = w.nwin, sb = w.sb;
      int blk = t_hi;
      for (int n = n0; n <= n1; ++n, --blk) {
        if (n == nwin) blk = sb - 1;                             // below the window: the blocks of sinks
        if (blk < t_lo && blk >= sbn) continue;
        const int kb = blk * N, cols = fwd_cols<N>(a, blk, t_lo);
        const int first = lo - kb, last = hi - kb, sinks = a.ns - kb;        // as columns of the block
        const bool full = __all_sync(0xffffffffu, last >= cols - 1 && (first <= 0 || sinks >= cols));
        wait(&sh->s_full[t], s_par);
        s_par ^= 1;
        if (!ok) break;
        tc_fence_after();
        auto taken = [&]() {                                     // the scores are in registers
          tmem_wait_ld();
          if constexpr (S::kOver) return;
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->s_free[t]);
        };
        auto grow = [&](float mx) {                              // the maximum the row is scaled by
          // (a row that has met nothing has an accumulator of zeros)
          const bool need = m != -INFINITY && (mx - m) * c2 > kGrow;
          if (__any_sync(0xffffffffu, need)) {
            wait_pv();
            if (!ok) return;
            tc_fence_after();
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
            if (need) l *= f;
          }
          if (need || m == -INFINITY) m = mx;
        };
        uint64_t ls[2] = {0ull, 0ull};
        auto half = [&]() {                                      // the first half of P is there
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->p_half[t]);
        };
        // C chunks of 16 columns
        auto block = [&](auto count) {
          constexpr int C = decltype(count)::value;
          float s[16 * C];
#pragma unroll
          for (int c = 0; c < C; ++c) tmem_ld16(s_tm + 16 * c, reinterpret_cast<uint32_t*>(s) + 16 * c);
          taken();
          if (!full) {
#pragma unroll
            for (int c = 0; c < (C + 1) / 2; ++c) {
              const uint32_t see = below(last + 1, c) & (~below(first, c) | below(sinks, c));
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (32 * c + e < 16 * C && !(see >> e & 1u)) s[32 * c + e] = -INFINITY;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < 16 * C; e += 2) mx[(e >> 1) & 3] = fmaxf(mx[(e >> 1) & 3], fmaxf(s[e], s[e + 1]));
          grow(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
          const float mc = m == -INFINITY ? 0.f : m * c2;
          const uint64_t nmc2 = f2_pack(-mc, -mc);
          wait_pv();                                             // the product that read P last
#pragma unroll
          for (int c = 0; c < C; ++c) {
            uint32_t pw[8];
#pragma unroll
            for (int h = 0; h < 8; ++h) {
              const float2 x = f2_unpack(f2_fma(f2_pack(s[16 * c + 2 * h], s[16 * c + 2 * h + 1]), c22, nmc2));
              const float p0 = exp2f(x.x), p1 = exp2f(x.y);
              ls[h & 1] = f2_add(ls[h & 1], f2_pack(p0, p1));
              pw[h] = tc::pack2<BF16>(p0, p1);
            }
            tmem_st8(p_tm + 8 * c, pw);
            if (S::kOver && C == N / 16 && c == C / 2 - 1) half();
          }
        };
        if (cols == N) block(std::integral_constant<int, N / 16>());
        else if (cols == 16) block(std::integral_constant<int, 1>());
        else if (cols == 64) block(std::integral_constant<int, 4>());
        else {
          // a block of sinks of another width: chunk by chunk, twice (16384 tokens, window 1024, heads of 128, us with 16, 64 and 128 sinks 163,
          // 164, 165; with 32 and 48 163, 164, with 80, 96 and 112 171, 177, 179)
          float mx = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < cols; c += 16) {
            uint32_t s[16];
            tmem_ld16(s_tm + c, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (c + e < sinks && c + e <= last) mx = fmaxf(mx, __uint_as_float(s[e]));
          }
          grow(mx);
          const float mc = m == -INFINITY ? 0.f : m * c2;
          wait_pv();
#pragma unroll 1
          for (int c = 0; c < cols; c += 16) {
            uint32_t s[16], pw[8];
            tmem_ld16(s_tm + c, s);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int k = c + 2 * e;
              const float p0 = k < sinks && k <= last ? exp2f(fmaf(__uint_as_float(s[2 * e]), c2, -mc)) : 0.f;
              const float p1 = k + 1 < sinks && k + 1 <= last ? exp2f(fmaf(__uint_as_float(s[2 * e + 1]), c2, -mc)) : 0.f;
              ls[e & 1] = f2_add(ls[e & 1], f2_pack(p0, p1));
              pw[e] = tc::pack2<BF16>(p0, p1);
            }
            tmem_st8(p_tm + (c >> 1), pw);
          }
          taken();
        }
        if (S::kOver && cols != N) half();
        if (!ok) break;
        const float2 l0 = f2_unpack(ls[0]), l1 = f2_unpack(ls[1]);
        l += (l0.x + l0.y) + (l1.x + l1.y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[t]);
        pv_open = true;
      }
      if (!ok) break;
      const bool live = i < w.len;
      if (i < a.N) a.lse[((int64_t)w.b * a.Hq + w.h[t]) * a.N + i] = live ? fmaf(m, c2, log2f(l)) : -INFINITY;
      wait(&sh->l_empty[t], l_par);
      l_par ^= 1;
      if (!ok) break;
      sh->inv[t][r] = 1.f / l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->l_full[t]);
    }
  } else {
    setmaxnreg_dec<kRegsEpilogue>();
    // ------------------------------------------------------------------ epilogue, one thread per row of each tile
    const int e = warp & 3, r = e * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(e * 32) << 16);
    uint8_t* stg = stg_smem + e * kStage;
    uint32_t par = 0;                                            // a bit per tile
    FwdItem w;
    while (take(w)) {
      for (int t = 0; t < 2; ++t) {
        const int row0 = w.q0[t] + e * 32;
        if (w.hi[t] < 0) {
          if (row0 < a.N) store_zeros<BF16>(stg, lane, &tm_o, a.dv_dim, row0, w.h[t], w.b);
          continue;
        }
        wait(&sh->l_full[t], par >> t & 1u);
        wait(&sh->o_full[t], par >> t & 1u);
        par ^= 1u << t;
        if (!ok) break;
        tc_fence_after();
        const bool live = w.q0[t] + r < w.len;
        const float inv = sh->inv[t][r];
        uint64_t z = 0ull;
#pragma unroll 1
        for (int c = 0; c < (int)kOCols; c += 32) {
          uint32_t x[32];
          tmem_ld32(lanes + S::kO + t * kOCols + c, x);
          tmem_wait_ld();
          if (c + 32 == (int)kOCols) {                           // the accumulator and the sums have been read
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&sh->o_empty[t]);
              mbar_arrive(&sh->l_empty[t]);
            }
          }
          if (row0 < a.N && c < a.dv_dim) store_columns<BF16>(x, inv, live, z, stg, lane, &tm_o, c, a.dv_dim, row0, w.h[t], w.b);
        }
        if (live && has_nan(z)) sh->bad = 1;
      }
      if (!ok) break;
    }
    if (lane == 0) tma_store_wait_all();
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
      const FwdItem w = fwd_item<N>(p, item);
#pragma unroll 1
      for (int x = warp; x < 2 * kTile; x += kThreads / 32) {
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
