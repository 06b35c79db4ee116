// tcgen05 backward kernels of the attention with a sliding window and sink tokens: one template, KIND 1 dQ and KIND 2 dK / dV.
//
//   P = exp2(c S - lse),  dP = dO V^T,  dS = P (dP - delta):   dQ = scale dS K;   dV = P^T dO,  dK = scale dS^T Q
//
// A CTA (one per SM, persistent) holds a resident tile X of 128 rows -- queries and their dO, or keys and their values --
// and streams blocks Y of N rows of the other side:  S = X_qk Y_qk^T and dP = X_v Y_v^T (for keys: their transposes), and
// dQ += dS Y_qk, or dV += P Y_v and dK += dS Y_qk, with P and dS as A operands in tensor memory over the scores they came from.
// dQ and dK/dV in kernels of their own, seven products where five would do: the fifth of a joint kernel, dQ summed by
// atomics over the key tiles, would make results depend on the order of CTAs.  Heads that share a key head follow each other
// in the stream of its dK/dV tile, so that their sum is in a fixed order too.
//
//   warp 0      TMA producer      warp 1   issues S and dP      warp 3   issues the products of P and dS
//   warp 2      hands out the items, and -lse and -delta: KIND 1 of an item's rows with it, KIND 2 of the streamed rows block by block
//   warps 4-11  two groups, one thread per resident row each, on half of a block's columns: P while dP is being made, then dS
//   warps 12-15 epilogue
// Tensor memory: two score buffers, one dP buffer, the accumulators.  dK/dV: N = 128, 96 (d_qk and d_v on different sides of 64) or 80 (both
// above) is what then fits; dQ: 128, and 96 with wide heads, whose blocks of 128 leave room for two stages only, so that every load was
// waited for.  The scores of the next block are made while a block's P and dS are, its dP as soon as
// this block's has been read, and this block's products run behind it.
//
// Measured (bf16, 16384 tokens, window 1024, 64 sinks, 16 heads of 128 on 4): dQ 217 to 236 us, tensor pipe 56 % busy; dK/dV 266 to 293 us, 67 %; with what the
// kernels execute, 7 products and whole blocks, that is 1.05 to 1.15 PFLOP/s.  Left: per block about 200 cycles of waits, 860 for 48 columns of P,
// 380 for dS, 350 of loop.  Tried and not kept: the groups on alternate whole blocks with a dP buffer each, which wants N = 96 and 64 (dQ 222 us,
// dK/dV 291; with heads of 64 dQ 91 -> 109 and dK/dV 119 -> 132).
//
// Blocks of dK/dV that hold sinks are seen by every later query: their stream is cut into pieces about as long as another block's, the
// partial sums go to scratch in fp32 and join_kernel (sink_rows.cuh) adds them in order.
//
// P and dS are rounded to the type of the tensors they are multiplied with, as in the forward kernel; delta is made from the rounded O.  Error
// against 64 bits, as multiples of the results' own rounding: dV 1.4, dQ and dK 1.46 to 1.53 (1.05 to 1.1 with P and dS in fp32: what delta adds).
//
// Infinities and NaN: as in the forward kernel, rows of the result that end as one are done again by row_dq / row_dkdv, rows of a piece's
// sums by row_piece; padding behind a sequence's end is zeros before it is multiplied.
#pragma once

#include "sink_tc_common.cuh"

namespace swa {
namespace sink {

struct BwdParams {
  Args a;
  int n_items, stages, xbufs;
  int n_t;                                      // tiles of 128 resident rows
  int n_sb, pieces, piece_len, near, n_sink_items;    // KIND 2: blocks that hold sinks, their pieces (cut_pieces)
  float* part;                                  // [B, Hkv, n_sb, pieces, 128, d_qk + d_v]
  int32_t* status;
};

template <int KIND, int XC, int VC>
struct BwdShape {
  static constexpr int N = XC + VC == 2 ? 128 : KIND == 1 ? (XC + VC == 3 ? 128 : 96) : XC + VC == 3 ? 96 : 80;
  static constexpr int kS = 0, kDP = 2 * N, kAcc = 3 * N;        // tensor memory
  static constexpr int kAccV = kAcc, kAccQK = KIND == 1 ? kAcc : kAcc + VC * 64;
  static constexpr int CH = (N / 2 + 15) / 16;                   // 16-column chunks of a group, the first's
  static_assert(kAccQK + XC * 64 <= 512, "tensor memory");
};

// What an item streams: KIND 1 key blocks, KIND 2 query blocks of the heads that share the key head.
struct BwdItem {
  int nb;                                       // blocks; -1: no more items
  int b, h, x0, len;                            // h: head of the resident rows; x0: their first
  int hi, lo, sb;                               // KIND 1: window's blocks, blocks of sinks below them
  int per_head, first, piece;                   // KIND 2: blocks of a head, the first of this piece; piece < 0: results go straight out
};

struct BwdShared {
  // ds_ready: a barrier per score buffer.  Both issuers wait for it, and the second may be behind by a block, waiting for the epilogue; the
  // next phase of a buffer's barrier needs scores that are made only after the products of the one before (s_done).
  uint64_t x_full[2], x_empty[2], y_full[4], y_empty[4], s_full[2], s_done[2], ds_ready[2], dp_full, acc_full, acc_empty, vec_full[4], vec_empty[4],
      item_full[kItems], item_empty[kItems], padded;
  // KIND 2: -lse and -delta of the streamed rows, a ring by blocks; KIND 1: of the resident rows, a ring by items
  alignas(16) float vec[4][2][kTile];
  BwdItem item[kItems];
  uint32_t tmem_base;
  int abort_flag, bad;
};
static_assert(kItems == 4, "vec is a ring of items too");

// Where a piece leaves its sums: [column / 4][row][4], so that a warp's rows lie side by side.
__device__ __forceinline__ float* piece_sums(const BwdParams& p, const BwdItem& w) {
  return p.part + ((((int64_t)w.b * p.a.Hkv + w.h) * p.n_sb + w.x0 / kTile) * p.pieces + w.piece) * (int64_t)kTile * (p.a.dqk + p.a.dv_dim);
}

template <int KIND, int N>
__device__ __forceinline__ BwdItem bwd_item(const BwdParams& p, int item) {
  const Args& a = p.a;
  BwdItem w;
  if constexpr (KIND == 1) {
    const int per = a.B * a.Hq, r = item % per;
    w.b = r / a.Hq;
    w.h = r % a.Hq;
    w.x0 = (p.n_t - 1 - item / per) * kTile;
    w.len = seq_len(a, w.b);
    w.hi = min(w.x0 + kTile - 1, max(w.len, 1) - 1) / N;
    w.lo = max(0, w.x0 - a.W + 1) / N;
    w.sb = min((a.ns + N - 1) / N, w.lo);
    w.nb = w.x0 < w.len ? w.hi - w.lo + 1 + w.sb : 0;
    w.piece = -1;
    w.first = w.per_head = 0;
  } else {
    const int per = a.B * a.Hkv;
    w.hi = w.lo = w.sb = 0;
    int blk, piece = 0;
    int r;
    if (item < p.n_sink_items) {
      r = item % per;
      piece = item / per % p.pieces;
      blk = item / per / p.pieces;
    } else {
      r = (item - p.n_sink_items) % per;
      blk = p.n_sb + (item - p.n_sink_items) / per;
    }
    w.b = r / a.Hkv;
    w.h = r % a.Hkv;
    w.x0 = blk * kTile;
    w.len = seq_len(a, w.b);
    const int end = blk < p.n_sb ? w.len : (int)min((int64_t)w.len, (int64_t)w.x0 + kTile - 1 + a.W);
    w.per_head = w.x0 < w.len ? (end - w.x0 + N - 1) / N : 0;
    const int all = w.per_head * a.G;
    w.first = piece * p.piece_len;
    w.nb = blk < p.n_sb ? max(0, min(p.piece_len, all - w.first)) : all;
    if (blk >= p.n_sb) w.first = 0;
    w.piece = blk < p.n_sb && all > p.piece_len ? piece : -1;
  }
  return w;
}

// The blocks of an item one after the other: first row, and head, of each.  (Incremental: with the divisions that find block n from scratch
// the top of the compute groups' loop took 600 cycles.)
template <int KIND, int N>
struct BwdWalk {
  int y0, h, n, i;                              // i: blocks left of the window (KIND 1), of the head (KIND 2)
  __device__ __forceinline__ BwdWalk(const BwdItem& w, int G) : n(0) {
    if constexpr (KIND == 1) {
      y0 = w.hi * N;
      h = w.h / G;
      i = w.hi - w.lo + 1;
    } else {
      const int heads = w.first ? w.first / w.per_head : 0, at = w.first - heads * w.per_head;
      y0 = w.x0 + at * N;
      h = w.h * G + heads;
      i = w.per_head - at;
    }
  }
  __device__ __forceinline__ bool window() const { return KIND == 2 || i > 0; }
  __device__ __forceinline__ int cols(int ns) const { return window() ? N : min(N, (ns - y0 + 15) & ~15); }
  __device__ __forceinline__ void next(const BwdItem& w) {
    ++n;
    --i;
    if constexpr (KIND == 1) {
      y0 -= N;
      if (i == 0) y0 = (w.sb - 1) * N;          // below the window: the blocks of sinks
    } else {
      y0 += N;
      if (i == 0) {
        y0 = w.x0;
        ++h;
        i = w.per_head;
      }
    }
  }
};

// Rows of this CTA's items that ended as an infinity or a NaN once more, over the pairs that see each other only; a warp a row.
template <typename T, int KIND, int N>
__device__ __noinline__ void bwd_repair(const BwdParams& p, float* s) {
  const Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int item = blockIdx.x; item < p.n_items; item += gridDim.x) {
    const BwdItem w = bwd_item<KIND, N>(p, item);
    if (!w.nb) continue;
    const bool near = KIND == 2 && w.piece >= 0 && piece_near(w.first, w.nb, w.per_head, p.near);
#pragma unroll 1
    for (int i = w.x0 + warp; i < min(w.len, w.x0 + kTile); i += kThreads / 32) {
      if (KIND == 2 && w.piece >= 0) {
        float* part = piece_sums(p, w) + (i - w.x0) * 4;
        if ((i < a.ns || near) && bad_piece(a, part, 4 * kTile, lane))
          row_piece<T>(a, w.b, w.h, i, w.x0, w.first, w.nb, w.per_head, N, part, 4 * kTile, s);
        continue;
      }
      bool bad = false;
      const T* x = row_ptr<T>(KIND == 1 ? a.dq : a.dk, w.b, w.h, i);
      for (int d = lane; d < a.dqk; d += 32) bad |= !(fabsf(to_f(x[d])) <= 3.0e38f);
      if constexpr (KIND == 2) {
        const T* y = row_ptr<T>(a.dv, w.b, w.h, i);
        for (int d = lane; d < a.dv_dim; d += 32) bad |= !(fabsf(to_f(y[d])) <= 3.0e38f);
      }
      if (!__any_sync(0xffffffffu, bad)) continue;
      if constexpr (KIND == 1) row_dq<T>(a, w.b, w.h, i, s);
      else row_dkdv<T>(a, w.b, w.h, i, s);
    }
  }
}

template <bool BF16, int KIND, int XC, int VC>
__global__ void __launch_bounds__(kThreads, 1)
sink_bwd_kernel(const __grid_constant__ CUtensorMap tm_xqk, const __grid_constant__ CUtensorMap tm_xv, const __grid_constant__ CUtensorMap tm_yqk,
                const __grid_constant__ CUtensorMap tm_yv, const __grid_constant__ CUtensorMap tm_oqk, const __grid_constant__ CUtensorMap tm_ov,
                const __grid_constant__ BwdParams p) {
  using namespace ptx;
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  using S = BwdShape<KIND, XC, VC>;
  constexpr int N = S::N, CH = S::CH;
  constexpr uint32_t kY = N * 128, kYStage = (XC + VC) * kY, kX = (XC + VC) * kChunk;      // bytes: chunk of a block, block, resident tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const Args& a = p.a;
  uint8_t* x_smem = smem;                                        // buffer: qk chunks, v chunks
  uint8_t* y_smem = x_smem + p.xbufs * kX;
  uint8_t* stg_smem = y_smem + p.stages * kYStage;
  BwdShared* sh = reinterpret_cast<BwdShared*>(stg_smem + 4 * kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x < offsetof(BwdShared, vec) / 8) {
    uint64_t* bar = reinterpret_cast<uint64_t*>(sh) + threadIdx.x;
    // consumers of items: producer, two issuers, 8 warps of the groups, 4 of the epilogue
    mbar_init(bar, (bar >= sh->ds_ready && bar < sh->ds_ready + 2) || (bar >= sh->vec_empty && bar < sh->vec_empty + 4) ? 8 : bar == &sh->acc_empty ? 4
                   : bar >= sh->item_empty && bar < sh->item_empty + kItems ? 15 : 1);
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
  bool ok = true;
  auto wait = [&](uint64_t* bar, uint32_t parity) { ok &= __all_sync(0xffffffffu, mbar_wait_polls<0>(smem_u32(bar), parity)) != 0; };
  using Walk = BwdWalk<KIND, N>;
  // The next item from the ring, its slot in `ii`; done() once nothing of it is read there any more.
  int ii = kItems - 1, ipar = 1;
  auto done = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->item_empty[ii]);
  };
  auto take = [&](BwdItem& w, bool keep = false) {
    if (++ii == kItems) ii = 0;
    if (ii == 0) ipar ^= 1;
    wait(&sh->item_full[ii], ipar);
    if (!ok) return false;
    w = sh->item[ii];
    if (!keep || w.nb <= 0) done();
    return w.nb >= 0;
  };

  if (warp < 4) {
    setmaxnreg_dec<kRegsIssue>();
    if (warp == 0) {
      // ---------------------------------------------------------------- producer
      const uint32_t el = elect_one();
      int st = 0, par = 1, xb = 0, x_par = 1, pad_par = 0;
      BwdItem w;
      while (take(w)) {
        if (!w.nb) continue;
        wait(&sh->x_empty[xb], x_par);
        if (!ok) break;
        const uint32_t xs = smem_u32(x_smem) + xb * kX, xbar = smem_u32(&sh->x_full[xb]);
        mbar_expect_tx_el(el, xbar, kX);
#pragma unroll
        for (int c = 0; c < XC; ++c) tma_load_4d_el(el, xs + c * kChunk, &tm_xqk, xbar, 64 * c, w.x0, w.h, w.b);
#pragma unroll
        for (int c = 0; c < VC; ++c) tma_load_4d_el(el, xs + (XC + c) * kChunk, &tm_xv, xbar, 64 * c, w.x0, w.h, w.b);
        if (++xb == p.xbufs) { xb = 0; x_par ^= 1; }
        Walk y(w, a.G);
        for (; y.n < w.nb; y.next(w)) {
          const int row = y.y0, h = y.h;
          wait(&sh->y_empty[st], par);
          if (!ok) break;
          const bool pad = holds_padding<N>(row, w.len, a.N);
          const uint32_t ys = smem_u32(y_smem) + st * kYStage, ybar = smem_u32(pad ? &sh->padded : &sh->y_full[st]);
          mbar_expect_tx_el(el, ybar, kYStage);
#pragma unroll
          for (int c = 0; c < XC; ++c) tma_load_4d_el(el, ys + c * kY, &tm_yqk, ybar, 64 * c, row, h, w.b);
#pragma unroll
          for (int c = 0; c < VC; ++c) tma_load_4d_el(el, ys + (XC + c) * kY, &tm_yv, ybar, 64 * c, row, h, w.b);
          if (pad) {
            wait(&sh->padded, pad_par);
            if (!ok) break;
            pad_par ^= 1;
            zero_rows<N, XC + VC>(ys, w.len - row, lane);
            if (lane == 0) mbar_arrive(&sh->y_full[st]);
          }
          if (++st == p.stages) { st = 0; par ^= 1; }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------- S and dP
      const uint32_t el = elect_one();
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint32_t hi_sw = smem_desc_hi(1024, true);
      const uint64_t x_d = smem_desc_from(smem_u32(x_smem), 16, hi_sw), y_d = smem_desc_from(smem_u32(y_smem), 16, hi_sw);
      const int kq = steps16(a.dqk), kv = steps16(a.dv_dim);
      int st = 0, y_par = 0, xb = 0, x_par = 0, buf = 0;
      uint32_t ds_par = 0, sd_par = 3;                           // sd_par: a bit per score buffer
      bool open = false;                                         // a block whose dP has not been read yet
      BwdItem w;
      while (take(w)) {
        if (!w.nb) continue;
        wait(&sh->x_full[xb], x_par);
        const uint64_t xq = x_d + (uint64_t)(xb * (kX >> 4)), xv = xq + (XC * kChunk >> 4);
        for (Walk y(w, a.G); ok && y.n < w.nb; y.next(w)) {
          const uint32_t id = instr_desc(fmt, 128, y.cols(a.ns), 0, 0);
          const uint64_t yq = y_d + (uint64_t)(st * (kYStage >> 4)), yv = yq + (XC * kY >> 4);
          wait(&sh->y_full[st], y_par);
          wait(&sh->s_done[buf], sd_par >> buf & 1u);            // the products have read the P and dS over the scores before the last
          sd_par ^= 1u << buf;
          if (!ok) break;
          tc_fence_after();
          scores_mma<XC>(el, tmem + buf * N, xq, yq, kChunk >> 4, kY >> 4, id, kq);
          umma_commit_el(el, &sh->s_full[buf]);
          if (open) {                                            // the groups have read the dP before
            wait(&sh->ds_ready[buf ^ 1], ds_par >> (buf ^ 1) & 1u);
            ds_par ^= 1u << (buf ^ 1);
            if (!ok) break;
            tc_fence_after();
          }
          open = true;
          scores_mma<VC>(el, tmem + S::kDP, xv, yv, kChunk >> 4, kY >> 4, id, kv);
          umma_commit_el(el, &sh->dp_full);
          buf ^= 1;
          if (++st == p.stages) { st = 0; y_par ^= 1; }
        }
        if (!ok) break;
        umma_commit_el(el, &sh->x_empty[xb]);
        if (++xb == p.xbufs) { xb = 0; x_par ^= 1; }
      }
    } else if (warp == 3) {
      // ---------------------------------------------------------------- dQ += dS K, or dV += P dO and dK += dS Q
      const uint32_t el = elect_one();
      const uint32_t fmt = BF16 ? 1u : 0u;
      const uint64_t y_d = smem_desc_from(smem_u32(y_smem), kY, smem_desc_hi(1024, true));
      const uint32_t id_qk = instr_desc(fmt, 128, 16 * steps16(a.dqk), 0, 1), id_v = instr_desc(fmt, 128, 16 * steps16(a.dv_dim), 0, 1);
      int st = 0, buf = 0;
      uint32_t ds_par = 0, acc_par = 1;
      BwdItem w;
      while (take(w)) {
        if (!w.nb) continue;
        wait(&sh->acc_empty, acc_par);                           // the accumulators of the item before have been read
        acc_par ^= 1;
        for (Walk y(w, a.G); ok && y.n < w.nb; y.next(w)) {
          const uint32_t s_tm = tmem + buf * N, acc = y.n ? 1u : 0u;
          const uint64_t yq = y_d + (uint64_t)(st * (kYStage >> 4)), yv = yq + (XC * kY >> 4);
          wait(&sh->ds_ready[buf], ds_par >> buf & 1u);
          ds_par ^= 1u << buf;
          if (!ok) break;
          tc_fence_after();
          // a chunk of 16 columns holds 16 P (KIND 2) and 16 dS, packed into 8 columns each
          if constexpr (KIND == 2) {
#pragma unroll
            for (int k = 0; k < N / 16; ++k) umma_ts_el(el, tmem + S::kAccV, s_tm + 16 * k, yv + 128 * k, id_v, k ? 1u : acc);
#pragma unroll
            for (int k = 0; k < N / 16; ++k) umma_ts_el(el, tmem + S::kAccQK, s_tm + 16 * k + 8, yq + 128 * k, id_qk, k ? 1u : acc);
          } else if (y.window()) {
#pragma unroll
            for (int k = 0; k < N / 16; ++k) umma_ts_el(el, tmem + S::kAccQK, s_tm + 16 * k, yq + 128 * k, id_qk, k ? 1u : acc);
          } else {
            const int steps = y.cols(a.ns) >> 4;
            for (int k = 0; k < steps; ++k) umma_ts_el(el, tmem + S::kAccQK, s_tm + 16 * k, yq + 128 * k, id_qk, k ? 1u : acc);
          }
          umma_commit_el(el, &sh->s_done[buf]);
          umma_commit_el(el, &sh->y_empty[st]);
          buf ^= 1;
          if (++st == p.stages) st = 0;
        }
        if (!ok) break;
        umma_commit_el(el, &sh->acc_full);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- items and softmax statistics
      int s = 0, par = 1, item = blockIdx.x, v = 0, v_par = 1;
      // the next item into the ring, with the end mark after the last; false once it is in, or a wait gave up
      auto hand_out = [&](BwdItem& w) {
        w.nb = -1;
        if (item < p.n_items) w = bwd_item<KIND, N>(p, item);
        float l[4], d[4];
        if (KIND == 1 && w.nb > 0) {
          const int64_t at = ((int64_t)w.b * a.Hq + w.h) * a.N + w.x0;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int r = lane + 32 * x;
            l[x] = w.x0 + r < w.len ? a.lse[at + r] : INFINITY;
            d[x] = w.x0 + r < w.len ? a.delta[at + r] : 0.f;
          }
        }
        wait(&sh->item_empty[s], par);
        if (!ok) return false;
        if (KIND == 1 && w.nb > 0) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            sh->vec[s][0][lane + 32 * x] = -l[x];
            sh->vec[s][1][lane + 32 * x] = -d[x];
          }
        }
        if (lane == 0) sh->item[s] = w;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->item_full[s]);
        if (++s == kItems) { s = 0; par ^= 1; }
        item += gridDim.x;
        return w.nb >= 0;
      };
      BwdItem w, next;
      bool more = hand_out(w);
      // KIND 2: one item ahead of the one whose blocks' statistics are written
      while (KIND == 1 && more) more = hand_out(w);
      while (KIND == 2 && more) {
        more = hand_out(next);
        if (!ok) break;
        if (w.nb)
          for (Walk y(w, a.G); y.n < w.nb; y.next(w)) {
            const int row = y.y0;
            const int64_t at = ((int64_t)w.b * a.Hq + y.h) * a.N + row;
            float l[4], d[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int r = lane + 32 * x;
              const bool in = r < N && row + r < w.len;
              l[x] = in ? a.lse[at + r] : INFINITY;               // a row behind the end: P = exp2(-inf)
              d[x] = in ? a.delta[at + r] : 0.f;
            }
            wait(&sh->vec_empty[v], v_par);
            if (!ok) break;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              sh->vec[v][0][lane + 32 * x] = -l[x];
              sh->vec[v][1][lane + 32 * x] = -d[x];
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->vec_full[v]);
            if (++v == 4) { v = 0; v_par ^= 1; }
          }
        if (!ok) break;
        w = next;
      }
    }
  } else if (warp < 12) {
    setmaxnreg_inc<kRegsCompute>();
    // ------------------------------------------------------------------ P and dS, one thread per resident row and group
    const int g = (warp - 4) >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int c0 = g * CH * 16;                                  // this group's columns: c0 .. c0 + 16 nch
    const uint64_t c22 = f2_pack(a.c2, a.c2);
    int buf = 0, v = 0, v_par = 0;
    uint32_t s_par = 0, dp_par = 0;
    BwdItem w;
    while (take(w, KIND == 1)) {
      if (!w.nb) continue;
      const int x = w.x0 + r;
      float nlse = -INFINITY, ndelta = 0.f;                      // KIND 1: of the thread's query
      // rows of the other side that the thread's row sees: lo .. hi, and (KIND 1) the sinks up to hi
      int lo, hi;
      if constexpr (KIND == 1) {
        hi = x < w.len ? x : -1;
        lo = x - a.W + 1;
        nlse = sh->vec[ii][0][r];
        ndelta = sh->vec[ii][1][r];
        done();
      } else {
        lo = x;
        hi = x < a.ns ? w.len - 1 : (int)min((int64_t)w.len - 1, (int64_t)x + a.W - 1);
      }
      for (Walk y(w, a.G); y.n < w.nb; y.next(w)) {
        const int base = y.y0 + c0, width = 16 * max(0, min(CH, (y.cols(a.ns) - c0) >> 4));
        // the same as columns of this group, and whether the warp's rows see all of them, or none
        const int first = lo - base, last = hi - base, sinks = KIND == 1 ? a.ns - base : 0;
        const bool full = __all_sync(0xffffffffu, last >= width - 1 && (first <= 0 || sinks >= width));
        const bool none = width == 0 || __all_sync(0xffffffffu, last < 0 || (first >= width && sinks <= 0));
        const uint32_t s_tm = lanes + buf * N + c0, d_tm = lanes + S::kDP + c0;
        [[maybe_unused]] const float* vec = sh->vec[v][0] + c0;
        if constexpr (KIND == 2) wait(&sh->vec_full[v], v_par);
        wait(&sh->s_full[buf], s_par >> buf & 1u);
        s_par ^= 1u << buf;
        if (!ok) break;
        tc_fence_after();
        if (none) {                                              // all of the warp's pairs are hidden
          wait(&sh->dp_full, dp_par);
          if (!ok) break;
          uint32_t zero[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) zero[e] = 0u;
          for (int i = 0; i < width; i += 16) {
            if constexpr (KIND == 2) tmem_st16(s_tm + i, zero);
            else tmem_st8(s_tm + i, zero);
          }
        } else {
          // C chunks of 16 columns: P while dP is being made, then dS.  (A hidden pair has P = 0 and dS = 0 * what it holds.)
          auto block = [&](auto count) {
            constexpr int C = decltype(count)::value;
            float s[16 * C];
#pragma unroll
            for (int i = 0; i < C; ++i) tmem_ld16(s_tm + 16 * i, reinterpret_cast<uint32_t*>(s) + 16 * i);
            tmem_wait_ld();
            if (!full) {
              uint32_t see[(C + 1) / 2];
#pragma unroll
              for (int i = 0; i < (C + 1) / 2; ++i) {
                see[i] = below(last + 1, i) & ~below(first, i);
                if constexpr (KIND == 1) see[i] |= below(last + 1, i) & below(sinks, i);
              }
#pragma unroll
              for (int e = 0; e < 16 * C; ++e)
                if (!(see[e >> 5] >> (e & 31) & 1u)) s[e] = -INFINITY;
            }
            [[maybe_unused]] uint32_t pw[8];
#pragma unroll
            for (int e = 0; e < 8 * C; e += 2) {
              uint64_t nl[2];
              if constexpr (KIND == 2) {
                const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(vec + 2 * e);
                nl[0] = t.x; nl[1] = t.y;
              } else {
                nl[0] = nl[1] = f2_pack(nlse, nlse);
              }
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const float2 t = f2_unpack(f2_fma(f2_pack(s[2 * e + 2 * z], s[2 * e + 2 * z + 1]), c22, nl[z]));
                s[2 * e + 2 * z] = exp2f(t.x);
                s[2 * e + 2 * z + 1] = exp2f(t.y);
                if constexpr (KIND == 2) pw[(e + z) & 7] = tc::pack2<BF16>(s[2 * e + 2 * z], s[2 * e + 2 * z + 1]);
              }
              if constexpr (KIND == 2)
                if ((e & 7) == 6) tmem_st8(s_tm + 2 * (e - 6), pw);
            }
            // (P before the wait, not sunk below it)
            if constexpr (KIND == 1) {
#pragma unroll
              for (int e = 0; e < 16 * C; ++e) asm volatile("" : "+f"(s[e]));
            }
            wait(&sh->dp_full, dp_par);
            if (!ok) return;
            tc_fence_after();
            float d[16 * C];
#pragma unroll
            for (int i = 0; i < C; ++i) tmem_ld16(d_tm + 16 * i, reinterpret_cast<uint32_t*>(d) + 16 * i);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 8 * C; e += 2) {
              uint64_t nd[2];
              if constexpr (KIND == 2) {
                const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(vec + 128 + 2 * e);
                nd[0] = t.x; nd[1] = t.y;
              } else {
                nd[0] = nd[1] = f2_pack(ndelta, ndelta);
              }
#pragma unroll
              for (int z = 0; z < 2; ++z) {
                const int c = 2 * e + 2 * z;
                const float2 t = f2_unpack(f2_mul(f2_pack(s[c], s[c + 1]), f2_add(f2_pack(d[c], d[c + 1]), nd[z])));
                pw[(e + z) & 7] = tc::pack2<BF16>(t.x, t.y);
              }
              if ((e & 7) == 6) tmem_st8(s_tm + 2 * (e - 6) + (KIND == 2 ? 8 : 0), pw);
            }
          };
          if (width == 16 * CH) block(std::integral_constant<int, CH>());
          else if (width == 16 * (CH - 1)) block(std::integral_constant<int, CH - 1>());
          else if (width == 32) block(std::integral_constant<int, 2>());      // (KIND 1: few sinks)
          else block(std::integral_constant<int, 1>());
          if (!ok) break;
        }
        dp_par ^= 1;
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sh->ds_ready[buf]);
          if constexpr (KIND == 2) mbar_arrive(&sh->vec_empty[v]);
        }
        buf ^= 1;
        if (++v == 4) { v = 0; v_par ^= 1; }
      }
      if (!ok) break;
    }
  } else {
    setmaxnreg_dec<kRegsEpilogue>();
    // ------------------------------------------------------------------ epilogue, one thread per resident row
    const int e = warp & 3, r = e * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(e * 32) << 16);
    uint8_t* stg = stg_smem + e * kStage;
    uint32_t par = 0;
    BwdItem w;
    while (take(w)) {
      const int row0 = w.x0 + e * 32;
      if (!w.nb) {
        if (row0 < a.N && w.piece < 0 && w.first == 0) {
          store_zeros<BF16>(stg, lane, &tm_oqk, a.dqk, row0, w.h, w.b);
          if constexpr (KIND == 2) store_zeros<BF16>(stg, lane, &tm_ov, a.dv_dim, row0, w.h, w.b);
        }
        continue;
      }
      wait(&sh->acc_full, par);
      par ^= 1;
      if (!ok) break;
      tc_fence_after();
      const bool live = w.x0 + r < w.len;
      const bool counts = KIND == 2 && w.piece >= 0 && (w.x0 + r < a.ns || piece_near(w.first, w.nb, w.per_head, p.near));
      uint64_t z = 0ull;
      // accumulators, 32 columns at a time: dV, then dQ or dK
      constexpr int kV = KIND == 2 ? 2 * VC : 0, kAll = kV + 2 * XC;
#pragma unroll 1
      for (int c = 0; c < kAll; ++c) {
        const bool is_v = c < kV;
        const int col = 32 * (is_v ? c : c - kV);
        uint32_t q[32];
        tmem_ld32(lanes + (is_v ? S::kAccV : S::kAccQK) + col, q);
        tmem_wait_ld();
        if (c + 1 == kAll) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->acc_empty);
        }
        if (col >= (is_v ? a.dv_dim : a.dqk)) continue;
        if (KIND == 2 && w.piece >= 0) {
          float* part = piece_sums(p, w) + (int64_t)((is_v ? a.dqk : 0) + col) * kTile + r * 4;
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (counts && col + 4 * u < (is_v ? a.dv_dim : a.dqk)) {
              *reinterpret_cast<uint4*>(part + u * 4 * kTile) = make_uint4(q[4 * u], q[4 * u + 1], q[4 * u + 2], q[4 * u + 3]);
#pragma unroll
              for (int x = 0; x < 4; x += 2) z = f2_fma(f2_pack(__uint_as_float(q[4 * u + x]), __uint_as_float(q[4 * u + x + 1])), 0ull, z);
            }
        } else if (row0 < a.N) {
          store_columns<BF16>(q, is_v ? 1.f : a.scale, live, z, stg, lane, is_v ? &tm_ov : &tm_oqk, col, is_v ? a.dv_dim : a.dqk, row0, w.h, w.b);
        }
      }
      if (live && has_nan(z)) sh->bad = 1;
    }
    if (lane == 0) tma_store_wait_all();
  }

  // -------------------------------------------------------------------- teardown (as in the forward kernel)
  if (!ok) sh->abort_flag = 1;
  tc_fence_before();
  __syncthreads();
  if (*(volatile int*)&sh->abort_flag) {
#pragma unroll 1
    for (int n = 0; n < 64; ++n) __nanosleep(1000);
    if (threadIdx.x == 0) tc::report_abort(p.status, 7 + KIND, 0);
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (*(volatile int*)&sh->bad && !*(volatile int*)&sh->abort_flag) bwd_repair<T, KIND, N>(p, reinterpret_cast<float*>(smem) + warp * 2 * kMaxDim);
}

}  // namespace sink
}  // namespace swa
