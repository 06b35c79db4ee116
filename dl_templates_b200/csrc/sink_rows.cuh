// Attention with a sliding window and sink tokens, one warp per row: token i of a sequence of `len` tokens sees token j if
//   j <= i,  i < len  and  (j > i - W  or  j < n_sink).
// These functions are the definition the tiled kernels are held to: only pairs that see each other are touched, so that an
// infinity or a NaN stays with the rows that see it.  They serve every type, stride and head dim up to 256, and the tiled kernels
// fall back on them for the rows (and only those) in which an infinity or a NaN has turned up: a hidden pair weighs 0 there, and
// 0 * inf is a NaN.
#pragma once

#include "../../include/swa_sequence.h"
#include "common.cuh"

namespace swa {
namespace sink {

// SMs of a B200.  The rules that cut work take this number and do not ask the device: the cut decides in which order sums are made, so that a
// part of a GPU gives the same bits.
constexpr int kSms = 148;
constexpr int kMaxDim = 256, kDimsPerLane = kMaxDim / 32;

struct Args {
  View4 q, k, v, o, d_o, dq, dk, dv;
  float* lse;            // [B, Hq, N], base 2
  float* delta;          // [B, Hq, N]: sum of o * do
  const int32_t* lens;   // [B] or nullptr: all N
  int B, Hq, Hkv, G, N, dqk, dv_dim, W, ns;
  float scale, c2;       // c2 = scale * log2(e)
};

__device__ __forceinline__ int seq_len(const Args& a, int b) {
  if (!a.lens) return a.N;
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.N ? a.N : n;
}

template <typename T>
__device__ __forceinline__ const T* row_ptr(const View4& v, int b, int h, int n) {
  return (const T*)v.ptr + b * v.s0 + h * v.s1 + (int64_t)n * v.s2;
}

template <typename T>
__device__ __forceinline__ void stage_row(float* s, const T* p, int64_t st, int d, int lane) {
  for (int t = lane; t < d; t += 32) s[t] = to_f(p[t * st]);
}

// s . row, the row read by one lane; by 16 bytes where the tensor allows.
template <typename T>
__device__ __forceinline__ float dot_row(const float* s, const T* p, int64_t st, int d, bool vec) {
  float acc = 0.f;
  if (vec) {
    constexpr int E = 16 / sizeof(T);
    for (int t = 0; t < d; t += E) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + t);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int x = 0; x < E; ++x) acc = fmaf(s[t + x], to_f(e[x]), acc);
    }
  } else {
    for (int t = 0; t < d; ++t) acc = fmaf(s[t], to_f(p[t * st]), acc);
  }
  return acc;
}

template <typename T>
__device__ __forceinline__ bool vec_rows(const View4& v, int d) {
  constexpr int E = 16 / sizeof(T);
  return v.s3 == 1 && d % E == 0 && reinterpret_cast<uintptr_t>(v.ptr) % 16 == 0 && v.s0 % E == 0 && v.s1 % E == 0 && v.s2 % E == 0;
}

__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// acc += sum over the chunk's keys of w[key] * row[key]: each lane owns dims lane, lane + 32, ...; `see` has a bit per key.
template <typename T>
__device__ __forceinline__ void add_rows(float* acc, float w, uint32_t see, const T* base, int64_t s2, int64_t s3, int d, int lane) {
  while (see) {
    const int j = __ffs(see) - 1;
    see &= see - 1;
    const float x = __shfl_sync(0xffffffffu, w, j);
    const T* p = base + j * s2;
#pragma unroll
    for (int t = 0; t < kDimsPerLane; ++t)
      if (lane + 32 * t < d) acc[t] = fmaf(x, to_f(p[(lane + 32 * t) * s3]), acc[t]);
  }
}

template <typename T>
__device__ __forceinline__ void store_row(const View4& v, int b, int h, int n, const float* acc, float f, int d, int lane) {
  T* p = (T*)v.ptr + b * v.s0 + h * v.s1 + (int64_t)n * v.s2;
#pragma unroll
  for (int t = 0; t < kDimsPerLane; ++t)
    if (lane + 32 * t < d) p[(lane + 32 * t) * v.s3] = from_f<T>(acc[t] * f);
}

// Calls body(first key, bits of its 32 keys that row i sees) for every chunk with such a key.
template <typename F>
__device__ __forceinline__ void for_key_chunks(const Args& a, int i, int lane, F&& body) {
  const int lo = max(0, i - a.W + 1), sinks = min(a.ns, lo);
  for (int j0 = 0; j0 < sinks; j0 += 32) body(j0, __ballot_sync(0xffffffffu, j0 + lane < sinks));
  for (int j0 = lo; j0 <= i; j0 += 32) body(j0, __ballot_sync(0xffffffffu, j0 + lane <= i));
}

// Forward: o_i and lse_i.  `s` is a warp's shared memory, 2 * kMaxDim floats.
template <typename T>
__device__ __noinline__ void row_forward(const Args& a, int b, int h, int i, float* s) {
  const int lane = threadIdx.x & 31, hk = h / a.G;
  float acc[kDimsPerLane] = {};
  float m = -INFINITY, l = 0.f;
  bool any = false;
  if (i < seq_len(a, b)) {
    any = true;
    __syncwarp();
    stage_row(s, row_ptr<T>(a.q, b, h, i), a.q.s3, a.dqk, lane);
    __syncwarp();
    const bool vec = vec_rows<T>(a.k, a.dqk);
    for_key_chunks(a, i, lane, [&](int j0, uint32_t see) {
      const float x = see >> lane & 1u ? dot_row(s, row_ptr<T>(a.k, b, hk, j0 + lane), a.k.s3, a.dqk, vec) * a.c2 : -INFINITY;
      // (a NaN is left to the sums: fmaxf passes over it)
      const float mn = fmaxf(m, lanes_max(x));
      const float f = m == mn ? 1.f : exp2f(m - mn);
      const float p = see >> lane & 1u && x != -INFINITY ? exp2f(x - mn) : 0.f;       // (a row of nothing but -inf: 0 / 0 at the end)
#pragma unroll
      for (int t = 0; t < kDimsPerLane; ++t) acc[t] *= f;
      l = l * f + lanes_sum(p);
      m = mn;
      add_rows(acc, p, see, row_ptr<T>(a.v, b, hk, j0), a.v.s2, a.v.s3, a.dv_dim, lane);
    });
  }
  store_row<T>(a.o, b, h, i, acc, any ? 1.f / l : 0.f, a.dv_dim, lane);
  if (lane == 0) a.lse[((int64_t)b * a.Hq + h) * a.N + i] = any ? m + log2f(l) : -INFINITY;
}

// dq_i = scale * sum_j p_ij (do_i . v_j - delta_i) k_j
template <typename T>
__device__ __noinline__ void row_dq(const Args& a, int b, int h, int i, float* s) {
  const int lane = threadIdx.x & 31, hk = h / a.G;
  float acc[kDimsPerLane] = {};
  if (i < seq_len(a, b)) {
    __syncwarp();
    stage_row(s, row_ptr<T>(a.q, b, h, i), a.q.s3, a.dqk, lane);
    stage_row(s + kMaxDim, row_ptr<T>(a.d_o, b, h, i), a.d_o.s3, a.dv_dim, lane);
    __syncwarp();
    const bool kvec = vec_rows<T>(a.k, a.dqk), vvec = vec_rows<T>(a.v, a.dv_dim);
    const int64_t at = ((int64_t)b * a.Hq + h) * a.N + i;
    const float lse = a.lse[at], delta = a.delta[at];
    for_key_chunks(a, i, lane, [&](int j0, uint32_t see) {
      float ds = 0.f;
      if (see >> lane & 1u) {
        const float p = exp2f(dot_row(s, row_ptr<T>(a.k, b, hk, j0 + lane), a.k.s3, a.dqk, kvec) * a.c2 - lse);
        ds = p * (dot_row(s + kMaxDim, row_ptr<T>(a.v, b, hk, j0 + lane), a.v.s3, a.dv_dim, vvec) - delta);
      }
      add_rows(acc, ds, see, row_ptr<T>(a.k, b, hk, j0), a.k.s2, a.k.s3, a.dqk, lane);
    });
  }
  store_row<T>(a.dq, b, h, i, acc, a.scale, a.dqk, lane);
}

// Adds what queries lo .. end - 1 of head h give to dk and dv of the key staged in `s`, p_ij (do_i . v_j - delta_i) q_i and p_ij do_i.
template <typename T>
__device__ __forceinline__ void add_queries(const Args& a, int b, int h, int lo, int end, const float* s, bool qvec, bool ovec, float* dk, float* dv, int lane) {
  const int64_t at = ((int64_t)b * a.Hq + h) * a.N;
  for (int i0 = lo; i0 < end; i0 += 32) {
    const uint32_t see = __ballot_sync(0xffffffffu, i0 + lane < end);
    float p = 0.f, ds = 0.f;
    if (see >> lane & 1u) {
      p = exp2f(dot_row(s, row_ptr<T>(a.q, b, h, i0 + lane), a.q.s3, a.dqk, qvec) * a.c2 - a.lse[at + i0 + lane]);
      ds = p * (dot_row(s + kMaxDim, row_ptr<T>(a.d_o, b, h, i0 + lane), a.d_o.s3, a.dv_dim, ovec) - a.delta[at + i0 + lane]);
    }
    add_rows(dv, p, see, row_ptr<T>(a.d_o, b, h, i0), a.d_o.s2, a.d_o.s3, a.dv_dim, lane);
    add_rows(dk, ds, see, row_ptr<T>(a.q, b, h, i0), a.q.s2, a.q.s3, a.dqk, lane);
  }
}
// Behind the last query that sees key j.
__device__ __forceinline__ int queries_end(const Args& a, int j, int len) { return j < a.ns ? len : (int)min((int64_t)len, (int64_t)j + a.W); }

// dk_j = scale * sum_i p_ij (do_i . v_j - delta_i) q_i,  dv_j = sum_i p_ij do_i, over the heads that share key head hk, in order.
template <typename T>
__device__ __noinline__ void row_dkdv(const Args& a, int b, int hk, int j, float* s) {
  const int lane = threadIdx.x & 31, len = seq_len(a, b);
  float dk[kDimsPerLane] = {}, dv[kDimsPerLane] = {};
  if (j < len) {
    __syncwarp();
    stage_row(s, row_ptr<T>(a.k, b, hk, j), a.k.s3, a.dqk, lane);
    stage_row(s + kMaxDim, row_ptr<T>(a.v, b, hk, j), a.v.s3, a.dv_dim, lane);
    __syncwarp();
    const bool qvec = vec_rows<T>(a.q, a.dqk), ovec = vec_rows<T>(a.d_o, a.dv_dim);
    const int end = queries_end(a, j, len);
    for (int g = 0; g < a.G; ++g) add_queries<T>(a, b, hk * a.G + g, j, end, s, qvec, ovec, dk, dv, lane);
  }
  store_row<T>(a.dk, b, hk, j, dk, a.scale, a.dqk, lane);
  store_row<T>(a.dv, b, hk, j, dv, 1.f, a.dv_dim, lane);
}

// A piece of a block with sinks, as the tiled kernels cut its stream (cut_pieces): `nb` blocks of `stream` queries, the first of them block `first`
// of the per_head blocks that every head of the group has from query x0 on.  bad_piece: whether a sum that the kernel left for row j is an
// infinity or a NaN; row_piece: the row's sums over the piece once more, over the pairs that see each other only.  `part`: the row's place,
// column c of dK and then dV at c / 4 * s_col4 + c % 4.
__device__ __forceinline__ bool bad_piece(const Args& a, const float* part, int s_col4, int lane) {
  bool bad = false;
  for (int c = lane; c < a.dqk + a.dv_dim; c += 32) bad |= !(fabsf(part[(c >> 2) * s_col4 + (c & 3)]) <= 3.0e38f);
  return __any_sync(0xffffffffu, bad);
}
template <typename T>
__device__ __noinline__ void row_piece(const Args& a, int b, int hk, int j, int x0, int first, int nb, int per_head, int stream, float* part, int s_col4,
                                       float* s) {
  const int lane = threadIdx.x & 31, len = seq_len(a, b);
  float dk[kDimsPerLane] = {}, dv[kDimsPerLane] = {};
  __syncwarp();
  stage_row(s, row_ptr<T>(a.k, b, hk, j), a.k.s3, a.dqk, lane);
  stage_row(s + kMaxDim, row_ptr<T>(a.v, b, hk, j), a.v.s3, a.dv_dim, lane);
  __syncwarp();
  const bool qvec = vec_rows<T>(a.q, a.dqk), ovec = vec_rows<T>(a.d_o, a.dv_dim);
  const int end = queries_end(a, j, len);
  for (int n = first; n < first + nb;) {
    const int g = n / per_head, at = n - g * per_head, blocks = min(per_head - at, first + nb - n);
    add_queries<T>(a, b, hk * a.G + g, max(j, x0 + at * stream), min(end, x0 + (at + blocks) * stream), s, qvec, ovec, dk, dv, lane);
    n += blocks;
  }
#pragma unroll
  for (int t = 0; t < kDimsPerLane; ++t) {
    const int c = lane + 32 * t, e = a.dqk + c;
    if (c < a.dqk) part[(c >> 2) * s_col4 + (c & 3)] = dk[t];
    if (c < a.dv_dim) part[(e >> 2) * s_col4 + (e & 3)] = dv[t];
  }
}

// KIND 0 forward, 1 dQ, 2 dK/dV.  grid = (rows / 8, heads, B); 8 warps.
constexpr int kRowWarps = 8;
template <typename T, int KIND>
__global__ void __launch_bounds__(32 * kRowWarps) rows_kernel(const __grid_constant__ Args a) {
  __shared__ float s[kRowWarps][2 * kMaxDim];
  pdl_enter();
  pdl_wait();
  const int warp = threadIdx.x >> 5;
  for (int64_t n = (int64_t)blockIdx.x * kRowWarps + warp; n < a.N; n += (int64_t)gridDim.x * kRowWarps) {
    if constexpr (KIND == 0) row_forward<T>(a, blockIdx.z, blockIdx.y, (int)n, s[warp]);
    if constexpr (KIND == 1) row_dq<T>(a, blockIdx.z, blockIdx.y, (int)n, s[warp]);
    if constexpr (KIND == 2) row_dkdv<T>(a, blockIdx.z, blockIdx.y, (int)n, s[warp]);
  }
}

// ---- delta = sum of o * do -----------------------------------------------------------------------------------------------
// Rows of whole 16-byte units: `group` lanes (the power of two that holds a row's units) take kDeltaRows rows, whose loads are in flight
// together (72000 rows of 80 16-bit elements: 8.7 us; a row at a time 11.9).  Rows behind a sequence's end are left out.
constexpr int kDeltaRows = 4;
template <typename T>
__global__ void __launch_bounds__(256) delta_rows_kernel(const __grid_constant__ Args a, int units, int group) {
  pdl_enter();
  pdl_wait();
  constexpr int E = 16 / sizeof(T);
  const int part = threadIdx.x & (group - 1), b = blockIdx.z, h = blockIdx.y, len = seq_len(a, b);
  const int per_block = 256 / group, n0 = blockIdx.x * per_block * kDeltaRows + threadIdx.x / group;
  uint4 x[kDeltaRows], y[kDeltaRows];
#pragma unroll
  for (int r = 0; r < kDeltaRows; ++r) {
    const int n = n0 + r * per_block;
    x[r] = y[r] = make_uint4(0, 0, 0, 0);
    if (n < len && part < units) {
      x[r] = *reinterpret_cast<const uint4*>(row_ptr<T>(a.o, b, h, n) + part * E);
      y[r] = *reinterpret_cast<const uint4*>(row_ptr<T>(a.d_o, b, h, n) + part * E);
    }
  }
#pragma unroll
  for (int r = 0; r < kDeltaRows; ++r) {
    const T *p = reinterpret_cast<const T*>(&x[r]), *q = reinterpret_cast<const T*>(&y[r]);
    float acc = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) acc += to_f(p[e]) * to_f(q[e]);
    for (int off = group >> 1; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    const int n = n0 + r * per_block;
    if (part == 0 && n < len) a.delta[((int64_t)b * a.Hq + h) * a.N + n] = acc;
  }
}

// Any type, stride and head dim: a warp a row.  grid = (rows / 8, Hq, B).
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) delta_any_kernel(const __grid_constant__ Args a) {
  pdl_enter();
  pdl_wait();
  const int lane = threadIdx.x & 31, n = blockIdx.x * kRowWarps + (threadIdx.x >> 5), h = blockIdx.y, b = blockIdx.z;
  if (n >= seq_len(a, b)) return;
  const T *x = row_ptr<T>(a.o, b, h, n), *y = row_ptr<T>(a.d_o, b, h, n);
  float acc = 0.f;
  for (int d = lane; d < a.dv_dim; d += 32) acc = fmaf(to_f(x[d * a.o.s3]), to_f(y[d * a.d_o.s3]), acc);
  acc = lanes_sum(acc);
  if (lane == 0) a.delta[((int64_t)b * a.Hq + h) * a.N + n] = acc;
}

// ---- dK and dV of blocks with sinks --------------------------------------------------------------------------------------
// Every later query sees them: the tiled kernels cut the G * ceil((len - x0) / stream) blocks they stream for such a block of `rows` resident
// rows into pieces of piece_len, each of which leaves its sums in part [B, Hkv, n_sb, pieces, rows * (d_qk + d_v)], row j and column c of
// them at j * s_row + c / 4 * s_col4 + c % 4.  Added here in the order of the pieces, one warp per row; a block that is a single piece
// has gone straight out.  Sums that are an infinity or a NaN have been done again by the kernel that left them (row_piece), so that nothing
// is left to repeat here: a row's warps, which have 32 columns each, depend on nothing but the pieces.
// Pieces of blocks with sinks: as long as an ordinary block's stream (G * near blocks, near = those that rows other than sinks can see), but
// no more of them than keep every SM busy four times over, or than keep a piece from outlasting the kernels' waits.  So they are less than
// twice 592 of `rows` rows together (155 MB of 128 rows of d_qk + d_v = 256) until G * N passes 2^24.
struct Pieces { int near, len, most; };
inline Pieces cut_pieces(const Args& a, int n_sb, int rows, int stream) {
  Pieces c;
  c.near = (rows - 1 + a.W + stream - 1) / stream;
  const int64_t all = (int64_t)a.G * ((a.N + stream - 1) / stream), blocks = (int64_t)a.B * a.Hkv * n_sb;
  const int64_t busy = (4 * kSms + blocks - 1) / (blocks > 0 ? blocks : 1), patient = ((int64_t)a.G * a.N >> 24) + 1;
  const int64_t cap = busy > patient ? busy : patient, shortest = (all + cap - 1) / cap, ordinary = (int64_t)a.G * c.near;
  const int64_t len = ordinary > shortest ? ordinary : shortest;
  c.len = (int)(len < INT32_MAX ? len : INT32_MAX);
  c.most = n_sb ? (int)((all + c.len - 1) / c.len) : 0;
  return c;
}

// Whether `nb` blocks of the stream from `first` on hold one that rows other than sinks can see: the first `near` of a head's `per_head`.  The
// other pieces leave sums for the sinks' rows only.
__device__ __forceinline__ bool piece_near(int first, int nb, int per_head, int near) {
  const int at = first % per_head;
  return at < near || at + nb > per_head;
}

struct JoinParams {
  Args a;
  int n_sb, pieces, piece_len, near, rows, stream, s_row, s_col4;
  const float* part;
};

// grid = (rows / 8, Hkv * 8, B): a warp has one row and 32 of its columns (with a warp for all of a row's columns 16384 tokens' 14 pieces took 17 us).
template <typename T>
__global__ void __launch_bounds__(32 * kRowWarps) join_kernel(const __grid_constant__ JoinParams p) {
  pdl_enter();
  pdl_wait();
  const Args& a = p.a;
  const int lane = threadIdx.x & 31, j = blockIdx.x * kRowWarps + (threadIdx.x >> 5), hk = blockIdx.y >> 3, c = 32 * (blockIdx.y & 7) + lane, b = blockIdx.z;
  const int len = seq_len(a, b), blk = j / p.rows, x0 = blk * p.rows, d = a.dqk + a.dv_dim;
  if (j >= a.N || blk >= p.n_sb || x0 >= len || c - lane >= d) return;            // (a block behind the end: zeros, written by its first piece)
  const int all = (len - x0 + p.stream - 1) / p.stream * a.G;
  if (all <= p.piece_len) return;
  const int pieces = j < len ? (all + p.piece_len - 1) / p.piece_len : 0, per_head = all / a.G;
  const bool sink = j < a.ns;
  const int64_t step = (int64_t)p.rows * d;
  const float* part = p.part + (((int64_t)b * a.Hkv + hk) * p.n_sb + blk) * p.pieces * step + (j - x0) * p.s_row + (c >> 2) * p.s_col4 + (c & 3);
  float acc = 0.f;
  for (int p0 = 0; p0 < pieces; p0 += 32) {
    const int mine = p0 + lane;
    uint32_t has = __ballot_sync(0xffffffffu, mine < pieces && (sink || piece_near(mine * p.piece_len, min(p.piece_len, all - mine * p.piece_len), per_head, p.near)));
    if (c >= d) has = 0;
    const float* from = part + p0 * step;
#pragma unroll 1
    for (int x = 0; has >> x; x += 8, from += 8 * step) {
      float v[8];                                                // eight pieces in flight
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = has >> x >> e & 1u ? from[e * step] : 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc += v[e];
      if (x == 24) break;
    }
  }
  if (c < a.dqk) ((T*)a.dk.ptr)[b * a.dk.s0 + hk * a.dk.s1 + (int64_t)j * a.dk.s2 + c * a.dk.s3] = from_f<T>(acc * a.scale);
  else if (c < d) ((T*)a.dv.ptr)[b * a.dv.s0 + hk * a.dv.s1 + (int64_t)j * a.dv.s2 + (c - a.dqk) * a.dv.s3] = from_f<T>(acc);
}

}  // namespace sink
}  // namespace swa
