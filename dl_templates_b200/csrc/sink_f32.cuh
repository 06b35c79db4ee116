// fp32 kernels of the attention with a sliding window and sink tokens, on the CUDA cores: KIND 0 forward, 1 dQ, 2 dK / dV (the products
// are those of sink_tc_fwd.cuh and sink_tc_bwd.cuh).
//
// A block of 128 threads holds 32 resident rows and streams blocks of 64 rows of the other side through shared memory.  Thread
// (ty, tx) owns the scores of rows ty + 8 i and columns tx + 16 j, i, j < 4, and columns 4 tx + 64 c of the accumulators of the
// same rows: a row belongs to one half warp, so that maxima and sums are shuffles and the weights go from the scores'
// threads to the second product's through shared memory without a barrier.  Rows in shared memory are 4 floats longer than the
// head: 16 rows read at the same column then lie in different banks.
// Bound by the fp32 pipes: 8 16-byte loads feed 64 multiply-adds, issued as 32 packed ones.
//
// Measured: 4000 tokens, window 1000, 16 heads of 128, batch 2: forward 1.88 ms (31 TFLOP/s of 74 nominal), backward 6.2 ms; 777 tokens, window 256, 8
// heads of 64 33 and 103 us.  With 64 resident rows and 256 threads 1.93 and 6.5 ms, 40 and 115 us: fewer and longer blocks (the fp32 pipes 50 to
// 54 % busy; 753 tokens, d_v = 128, 128 heads the other way round, 413 us against 446).  Tried and not kept beside that: 512 threads for 64 rows
// (46 us), scalar multiply-adds in the second product (2.02 ms).  Tensor cores (three tf32 products for one) would accumulate with
// truncation, over a whole window to 1e-5 and more: not what a caller of fp32 asks for.
//
// Neither started early under their predecessor nor letting their successor start: blocks of a small grid that start while the one before
// is still running are packed two and three to an SM onto the SMs that it left idle, and stay there (104 blocks each: 230 us a
// training step instead of 170).
//
// dK/dV of blocks with sinks, which every later query sees, are cut into pieces and joined in order, as in sink_tc_bwd.cuh; rows that
// end as an infinity or a NaN, of a piece too, are done again by the row functions.
#pragma once

#include "sink_rows.cuh"
#include "umma.cuh"

namespace swa {
namespace sink {

constexpr int kF32X = 32, kF32Rows = 64, kF32Threads = 4 * kF32X, kF32PPitch = kF32Rows + 4;      // resident, streamed rows
constexpr int kF32Y = kF32Threads / 16;           // rows ty + kF32Y i of a thread

struct F32Params {
  Args a;
  int n_t, n_sb, pieces, piece_len, near, n_sink_items;   // KIND 2: blocks that hold sinks, their pieces (cut_pieces)
  float* part;                                      // [B, Hkv, n_sb, pieces, kF32X, d_qk + d_v]
};

template <int KIND, int DQ, int DV>
struct F32Shape {
  static constexpr int PQ = DQ + 4, PV = DV + 4;
  static constexpr int kX = kF32X * (PQ + (KIND ? PV : 0)), kY = kF32Rows * (PQ + PV);
  static constexpr int kSmem = 4 * (kX + kY + kF32X * kF32PPitch);
};

// ROWS rows of a [B, H, N, d] tensor from row `n0` on into rows of `pitch` floats; zeros behind the sequence's last row and the last element (a weight
// of zero would make a NaN of what padding may hold).
template <int ROWS>
__device__ __forceinline__ void f32_load(float* s, int pitch, int dmax, const View4& t, int b, int h, int n0, int len, int d) {
  const float* p = (const float*)t.ptr + b * t.s0 + h * t.s1;
  const int units = dmax / 4;
  for (int x = threadIdx.x; x < ROWS * units; x += kF32Threads) {
    const int r = x / units, c = x % units * 4;
    const bool on = n0 + r < len && c < d;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(ptx::smem_u32(s + r * pitch + c)),
                 "l"(on ? p + (int64_t)(n0 + r) * t.s2 + c : (const float*)t.ptr), "r"(on ? 16 : 0) : "memory");
  }
}

// acc[i][j] = x row (ty + kF32Y i) . y row (tx + 16 j)
template <int D>
__device__ __forceinline__ void f32_scores(float (*acc)[4], const float* x, const float* y, int ty, int tx) {
  using namespace ptx;
  uint64_t s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = 0ull;
#pragma unroll 4
  for (int c = 0; c < D; c += 4) {
    ulonglong2 p[4], q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = *reinterpret_cast<const ulonglong2*>(x + (ty + kF32Y * i) * (D + 4) + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const ulonglong2*>(y + (tx + 16 * j) * (D + 4) + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = f2_fma(p[i].y, q[j].y, f2_fma(p[i].x, q[j].x, s[i][j]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = f2_unpack(s[i][j]);
      acc[i][j] = f.x + f.y;
    }
}

// acc[i][2 c + e] (pairs of columns 4 tx + 64 c + 2 e) += w row (ty + kF32Y i) . y columns
template <int D>
__device__ __forceinline__ void f32_product(uint64_t (*acc)[D / 32], const float* w, const float* y, int ty, int tx) {
  using namespace ptx;
#pragma unroll 2
  for (int k = 0; k < kF32Rows; k += 4) {
    float p[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(p[i]) = *reinterpret_cast<const float4*>(w + (ty + kF32Y * i) * kF32PPitch + k);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(y + (k + e) * (D + 4) + 4 * tx + 64 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint64_t pp = f2_pack(p[i][e], p[i][e]);
          acc[i][2 * c] = f2_fma(pp, v.x, acc[i][2 * c]);
          acc[i][2 * c + 1] = f2_fma(pp, v.y, acc[i][2 * c + 1]);
        }
      }
  }
}

template <int KIND, int DQ, int DV>
__global__ void __launch_bounds__(kF32Threads, (KIND == 2 && DQ + DV > 128 ? 1 : 2) * 256 / kF32Threads) f32_kernel(const __grid_constant__ F32Params p) {
  using namespace ptx;
  using S = F32Shape<KIND, DQ, DV>;
  extern __shared__ __align__(16) float f32_smem[];
  __shared__ int bad_row[kF32X];
  float *xq = f32_smem, *xv = xq + kF32X * S::PQ, *yq = f32_smem + S::kX, *yv = yq + kF32Rows * S::PQ, *ws = yv + kF32Rows * S::PV;
  const Args& a = p.a;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;

  // ---- the item: resident rows x0 .. x0 + kF32X - 1 of head h, the blocks it streams
  int b, h, x0, piece = -1, nb, first = 0, per_head = 0, hi = 0, lo = 0, sb = 0;
  if constexpr (KIND != 2) {
    const int per = a.B * a.Hq, r = blockIdx.x % per;
    b = r / a.Hq;
    h = r % a.Hq;
    x0 = (p.n_t - 1 - (int)(blockIdx.x / per)) * kF32X;
  } else {
    const int per = a.B * a.Hkv;
    int r, blk, pc = 0;
    if ((int)blockIdx.x < p.n_sink_items) {
      r = blockIdx.x % per;
      pc = blockIdx.x / per % p.pieces;
      blk = blockIdx.x / per / p.pieces;
    } else {
      r = (blockIdx.x - p.n_sink_items) % per;
      blk = p.n_sb + (blockIdx.x - p.n_sink_items) / per;
    }
    b = r / a.Hkv;
    h = r % a.Hkv;
    x0 = blk * kF32X;
    piece = pc;
  }
  const int len = seq_len(a, b);
  if constexpr (KIND != 2) {
    hi = min(x0 + kF32X - 1, max(len, 1) - 1) / kF32Rows;
    lo = max(0, x0 - a.W + 1) / kF32Rows;
    sb = min((a.ns + kF32Rows - 1) / kF32Rows, lo);
    nb = x0 < len ? hi - lo + 1 + sb : 0;
  } else {
    const bool sink_block = x0 / kF32X < p.n_sb;
    const int end = sink_block ? len : (int)min((int64_t)len, (int64_t)x0 + kF32X - 1 + a.W);
    per_head = x0 < len ? (end - x0 + kF32Rows - 1) / kF32Rows : 0;
    const int all = per_head * a.G;
    if (sink_block) {
      first = piece * p.piece_len;
      nb = max(0, min(p.piece_len, all - first));
      if (all <= p.piece_len) piece = piece ? -2 : -1;           // not cut: the first piece is all of it
    } else {
      nb = all;
      piece = -1;
    }
    if (nb == 0 && (piece != -1)) return;
  }

  const View4 &tq = KIND == 2 ? a.k : a.q, &tv = KIND == 2 ? a.v : a.d_o;          // resident
  const View4 &sq = KIND == 2 ? a.q : a.k, &sv = KIND == 2 ? a.d_o : a.v;          // streamed
  if (nb) {
    f32_load<kF32X>(xq, S::PQ, DQ, tq, b, h, x0, len, a.dqk);
    if constexpr (KIND != 0) f32_load<kF32X>(xv, S::PV, DV, tv, b, h, x0, len, a.dv_dim);
  }
  // statistics of the resident rows (KIND 0 running, 1 given)
  float m[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = x0 + ty + kF32Y * i;
    m[i] = KIND == 0 ? -INFINITY : 0.f;
    l[i] = 0.f;
    if (KIND == 1 && x < len) {
      m[i] = a.lse[((int64_t)b * a.Hq + h) * a.N + x];
      l[i] = a.delta[((int64_t)b * a.Hq + h) * a.N + x];
    }
  }
  uint64_t acc[4][DV / 32], acq[4][DQ / 32];                     // O, dV; dQ, dK
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int c = 0; c < DV / 32; ++c) acc[i][c] = 0ull;
#pragma unroll
    for (int c = 0; c < DQ / 32; ++c) acq[i][c] = 0ull;
  }

#pragma unroll 1
  for (int n = 0; n < nb; ++n) {
    int y0, hy;
    if constexpr (KIND != 2) {
      y0 = (n <= hi - lo ? hi - n : sb - 1 - (n - (hi - lo + 1))) * kF32Rows;
      hy = h / a.G;
    } else {
      y0 = x0 + (first + n) % per_head * kF32Rows;
      hy = h * a.G + (first + n) / per_head;
    }
    __syncthreads();                                             // the block before has been read
    f32_load<kF32Rows>(yq, S::PQ, DQ, sq, b, hy, y0, len, a.dqk);
    f32_load<kF32Rows>(yv, S::PV, DV, sv, b, hy, y0, len, a.dv_dim);
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float s[4][4];
    f32_scores<DQ>(s, xq, yq, ty, tx);
    uint32_t see = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int x = x0 + ty + kF32Y * i, y = y0 + tx + 16 * j, qi = KIND == 2 ? y : x, kj = KIND == 2 ? x : y;
        if (kj <= qi && qi < len && (kj > qi - a.W || kj < a.ns)) see |= 1u << (4 * i + j);
      }
    if constexpr (KIND == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = see >> (4 * i + j) & 1u ? s[i][j] * a.c2 : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[i], mx), f = m[i] == mn ? 1.f : exp2f(m[i] - mn);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float w = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - mn);
          sum += w;
          ws[(ty + kF32Y * i) * kF32PPitch + tx + 16 * j] = w;
        }
#pragma unroll
        for (int o = 8; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * f + sum;
        m[i] = mn;
        const uint64_t ff = f2_pack(f, f);
#pragma unroll
        for (int c = 0; c < DV / 32; ++c) acc[i][c] = f2_mul(acc[i][c], ff);
      }
      __syncwarp();
      f32_product<DV>(acc, ws, yv, ty, tx);
    } else {
      float dp[4][4];
      f32_scores<DV>(dp, xv, yv, ty, tx);
      float ly[4], dy[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int y = y0 + tx + 16 * j;
        ly[j] = dy[j] = 0.f;
        if (KIND == 2 && y < len) {
          ly[j] = a.lse[((int64_t)b * a.Hq + hy) * a.N + y];
          dy[j] = a.delta[((int64_t)b * a.Hq + hy) * a.N + y];
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool on = see >> (4 * i + j) & 1u;
          const float w = on ? exp2f(fmaf(s[i][j], a.c2, -(KIND == 1 ? m[i] : ly[j]))) : 0.f;
          dp[i][j] = on ? w * (dp[i][j] - (KIND == 1 ? l[i] : dy[j])) : 0.f;
          ws[(ty + kF32Y * i) * kF32PPitch + tx + 16 * j] = KIND == 1 ? dp[i][j] : w;
        }
      __syncwarp();
      if constexpr (KIND == 2) {
        f32_product<DV>(acc, ws, yv, ty, tx);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) ws[(ty + kF32Y * i) * kF32PPitch + tx + 16 * j] = dp[i][j];
        __syncwarp();
      }
      f32_product<DQ>(acq, ws, yq, ty, tx);
    }
    __syncwarp();
  }

  // ---- store
  __syncthreads();
  if (threadIdx.x < kF32X) bad_row[threadIdx.x] = 0;
  __syncthreads();
  const bool near = KIND == 2 && piece >= 0 && piece_near(first, nb, per_head, p.near);         // (rows other than sinks count)
  auto put = [&](auto& v, const View4& t, int dmax, int d, float* part, int i, float f) {
    const int r = ty + kF32Y * i, x = x0 + r;
    float z = 0.f;
    for (int c = 0; c < dmax / 64; ++c) {
      const int col = 4 * tx + 64 * c;
      const float2 u = f2_unpack(v[i][2 * c]), w = f2_unpack(v[i][2 * c + 1]);
      float4 o = make_float4(u.x * f, u.y * f, w.x * f, w.y * f);
      z += 0.f * o.x + 0.f * o.y + 0.f * o.z + 0.f * o.w;
      if (x >= len) o = make_float4(0.f, 0.f, 0.f, 0.f);
      if (col >= d) continue;
      if (part) *reinterpret_cast<float4*>(part + (int64_t)r * (a.dqk + a.dv_dim) + col) = o;
      else if (x < a.N) *reinterpret_cast<float4*>((float*)t.ptr + b * t.s0 + h * t.s1 + (int64_t)x * t.s2 + col) = o;
    }
    if (x < len && (!part || x < a.ns || near) && !(z == 0.f)) bad_row[r] = 1;
  };
  float* part = KIND == 2 && piece >= 0 ? p.part + (((((int64_t)b * a.Hkv + h) * p.n_sb + x0 / kF32X) * p.pieces + piece) * kF32X) * (a.dqk + a.dv_dim) : nullptr;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int x = x0 + ty + kF32Y * i;
    if constexpr (KIND == 0) {
      put(acc, a.o, DV, a.dv_dim, nullptr, i, x < len ? 1.f / l[i] : 0.f);
      if (tx == 0 && x < a.N) a.lse[((int64_t)b * a.Hq + h) * a.N + x] = x < len ? m[i] + log2f(l[i]) : -INFINITY;
    } else if constexpr (KIND == 1) {
      put(acq, a.dq, DQ, a.dqk, nullptr, i, a.scale);
    } else {
      put(acq, a.dk, DQ, a.dqk, part, i, part ? 1.f : a.scale);
      put(acc, a.dv, DV, a.dv_dim, part ? part + a.dqk : nullptr, i, 1.f);
    }
  }
  __syncthreads();
  float* s = f32_smem + (threadIdx.x >> 5) * 2 * kMaxDim;        // (the tiles are done with)
#pragma unroll 1
  for (int r = threadIdx.x >> 5; r < kF32X; r += kF32Threads / 32) {
    if (!bad_row[r]) continue;
    if constexpr (KIND == 0) row_forward<float>(a, b, h, x0 + r, s);
    if constexpr (KIND == 1) row_dq<float>(a, b, h, x0 + r, s);
    if constexpr (KIND == 2) {
      if (part) row_piece<float>(a, b, h, x0 + r, x0, first, nb, per_head, kF32Rows, part + r * (a.dqk + a.dv_dim), 4, s);
      else row_dkdv<float>(a, b, h, x0 + r, s);
    }
  }
}

}  // namespace sink
}  // namespace swa
