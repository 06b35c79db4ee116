// Rotary positions with several axes, stand-alone and on the way into a paged cache.
//
// Axis a turns R_a pairs by the angle of the token's position on it: with off_a = 2 (R_0 + .. + R_{a-1}), pair i is the elements
// off_a + i and off_a + R_a + i of a row,
//   y0 = x0 cos - x1 sin,   y1 = x0 sin + x1 cos      (inverse, for gradients: sin -> -sin),
// cos and sin from the axis' fp32 table (angles of far positions want 64 bits, which the table was made in).  A negative position
// turns nothing, one behind the table's end takes the table's last row; elements behind the last axis are copied.
//
// Bound by HBM: every byte is moved once, and q and k (and v on its way into the cache) share one launch.  Measured (bf16, 32 and 8 heads of
// 128, 32768 rows): 102 us, 6.6 TB/s; 16-bit rows whose axes start off 16-byte boundaries move in smaller units: 10 pairs an axis, by 4
// bytes, 3.3 TB/s.  Four heads a thread: 32 us for 168 MB; one 41, two 35, eight 35.  The data's loads ahead of the position's gained the
// append 1 us of 40 and cost the rotation 3 of 32.
#pragma once

#include "../../include/swa_sequence.h"
#include "common.cuh"

namespace swa {
namespace axes {

constexpr int kMaxAxes = 4;

// Heads of one tensor: `paged` ones go to the pages of a cache [pages, heads, slots, d] instead of a tensor [B, heads, N, d].
struct Group {
  View4 src, dst;
  int H, d, rotate, paged, chunks;       // chunks of heads
};

struct Args {
  Group g[3];
  int n_axes, R[kMaxAxes], max_pos[kMaxAxes], pairs;
  const float* cs[kMaxAxes];
  const int32_t* pos;                    // element [b, a, n] at b * pos_b + a * pos_a + n
  int64_t pos_b, pos_a;
  int N, slots;                          // tokens; slots of a row, the widest group's
  float sign;
  const int32_t *page_table, *seq_lens, *new_lens;
  int max_pages, n_pages, page_size;
};

template <int BYTES> struct Unit;
template <> struct Unit<16> { using type = uint4; };
template <> struct Unit<8> { using type = uint2; };
template <> struct Unit<4> { using type = uint32_t; };
template <> struct Unit<2> { using type = uint16_t; };

// Row of token n (of N new ones) in a cache, or -1: page * ps0 + place * ps2.  A page number outside the cache is no page.
__device__ __forceinline__ bool paged_row(const Args& a, const View4& c, int b, int n, int64_t* at) {
  int fresh = a.N;
  if (a.new_lens) fresh = min(max(a.new_lens[b], 0), a.N);
  if (n >= fresh) return false;
  const int64_t p = (int64_t)a.seq_lens[b] - fresh + n;
  if (p < 0 || p >= (int64_t)a.max_pages * a.page_size) return false;
  const int lp = (int)(p / a.page_size);
  const int page = a.page_table[(int64_t)b * a.max_pages + lp];
  if (page < 0 || page >= a.n_pages) return false;
  *at = page * c.s0 + (p - (int64_t)lp * a.page_size) * c.s2;
  return true;
}

// One thread: one slot of a token's row in HEADS heads of a group -- VE pairs of an axis, or two units of VE elements that are
// copied.  The position, the table values and the index arithmetic serve all its heads, and its loads are in flight together.
// VE elements are what rows, axes and tensors are aligned to, 16 bytes at most.  The chunks of heads, tokens and slots of a sequence are one
// index (a step of one token has 16 slots a head: with a block for each chunk of heads it took 5.5 us, most threads without
// work), grid = (all of them / 256, 1, B).
template <typename T, int VE, int HEADS>
__global__ void __launch_bounds__(256) rotate_kernel(const __grid_constant__ Args a) {
  using U = typename Unit<VE * sizeof(T)>::type;
  pdl_enter();
  pdl_wait();
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x, row = gid / (uint32_t)a.slots, sl = gid - row * a.slots;
  const uint32_t chunk = row / (uint32_t)a.N, tok = row - chunk * a.N;
  int y = (int)chunk, gi = 0;
  while (gi < 3 && y >= a.g[gi].chunks) y -= a.g[gi++].chunks;
  if (gi == 3) return;                                           // (no such group: its chunks are 0)
  const Group& g = a.g[gi];
  const int b = blockIdx.z;
  const uint32_t rot_slots = g.rotate ? (uint32_t)a.pairs / VE : 0u;
  const uint32_t spr = rot_slots + (((uint32_t)g.d / VE - 2 * rot_slots + 1) >> 1);
  if (sl >= spr) return;
  int64_t to = b * g.dst.s0 + (int64_t)tok * g.dst.s2;
  if (g.paged && !paged_row(a, g.dst, b, (int)tok, &to)) return;
  const T* src = (const T*)g.src.ptr + b * g.src.s0 + (int64_t)tok * g.src.s2;
  T* dst = (T*)g.dst.ptr + to;
  int e0, e1;
  bool two = true, turn = false;
  float cs[2 * VE];
  if (sl < rot_slots) {
    int ax = 0, off = 0;
    uint32_t i = sl * VE;
    while (i >= (uint32_t)a.R[ax]) {
      i -= a.R[ax];
      off += 2 * a.R[ax++];
    }
    e0 = off + (int)i;
    e1 = e0 + a.R[ax];
    int p = a.pos[b * a.pos_b + ax * a.pos_a + tok];
    if (p >= 0) {
      turn = true;
      p = min(p, a.max_pos[ax] - 1);
      const float* tab = a.cs[ax] + ((int64_t)p * a.R[ax] + i) * 2;
      if constexpr (VE == 1) {
        cs[0] = tab[0];
        cs[1] = tab[1];
      } else {
#pragma unroll
        for (int j = 0; j < 2 * VE; j += 4) *reinterpret_cast<float4*>(cs + j) = *reinterpret_cast<const float4*>(tab + j);
      }
    }
  } else {
    e0 = 2 * (g.rotate ? a.pairs : 0) + (int)(sl - rot_slots) * 2 * VE;
    e1 = e0 + VE;
    two = e1 < g.d;
  }
  const int h0 = y * HEADS;
  U u[HEADS], w[HEADS];
#pragma unroll
  for (int x = 0; x < HEADS; ++x)
    if (h0 + x < g.H) {
      const T* r = src + (h0 + x) * g.src.s1;
      u[x] = *reinterpret_cast<const U*>(r + e0 * g.src.s3);
      if (two) w[x] = *reinterpret_cast<const U*>(r + e1 * g.src.s3);
    }
#pragma unroll
  for (int x = 0; x < HEADS; ++x)
    if (h0 + x < g.H) {
      if (turn) {
        T* p0 = reinterpret_cast<T*>(&u[x]);
        T* p1 = reinterpret_cast<T*>(&w[x]);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float c = cs[2 * j], s = cs[2 * j + 1] * a.sign, x0 = to_f(p0[j]), x1 = to_f(p1[j]);
          p0[j] = from_f<T>(x0 * c - x1 * s);
          p1[j] = from_f<T>(x0 * s + x1 * c);
        }
      }
      T* r = dst + (h0 + x) * g.dst.s1;
      *reinterpret_cast<U*>(r + e0 * g.dst.s3) = u[x];
      if (two) *reinterpret_cast<U*>(r + e1 * g.dst.s3) = w[x];
    }
}

}  // namespace axes
}  // namespace swa
