// What the tcgen05 kernels of the attention with a sliding window and sink tokens share: work items handed out by one warp, the epilogue's
// stores, column masks.
//
// A CTA has 512 threads: warps 0-3 load, issue and hand out items, warps 4-11 are the two compute groups, warps 12-15 the epilogue.  An item
// is worked out once, by one warp, and read from a ring by all others: with every role doing its own divisions and loads the
// compute groups spent 1400 to 1900 cycles between items.  The epilogue in warps of its own takes an accumulator out of
// tensor memory while the compute groups are in the next item (in the compute groups it cost 1300 to 4000 cycles an item, most of
// it for stores of 16 bytes from 32 rows at a time), and stores it through shared memory by TMA.
#pragma once

#include "sink_rows.cuh"
#include "swa_tc_common.cuh"
#include "umma.cuh"

namespace swa {
namespace sink {

constexpr int kThreads = 512, kTile = 128;
constexpr uint32_t kChunk = 16384;              // 128 rows of 64 elements
constexpr int kItems = 4;                       // ring of items
// registers: loaders and issuers, compute groups, epilogue: (56 + 2 * 184 + 88) * 128 = 64 Ki
constexpr uint32_t kRegsIssue = 56, kRegsCompute = 184, kRegsEpilogue = 88;
constexpr uint32_t kStage = 2048;               // staging of an epilogue warp: 32 rows of 32 elements, 64-byte swizzle

// Bits of columns 32 w .. 32 w + 31 below n.
__device__ __forceinline__ uint32_t below(int n, int w) {
  n -= 32 * w;
  return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u;
}

// Whether a block of N streamed rows from `row` on holds rows behind the end of a sequence of `len` tokens that the tensor has (TMA fills with
// zeros what it has not).
template <int N>
__device__ __forceinline__ bool holds_padding(int row, int len, int n_rows) { return row < len && len < row + N && len < n_rows; }

// Zeros in rows `keep` .. N - 1 of such a block, CHUNKS chunks of N rows of 128 bytes (the swizzle stays within a row): padding may be anything, and a
// weight of zero makes a NaN of an infinity or a NaN, so that every row that meets the block would have to be done again (a training step of 4
// sequences of 500 to 1500 tokens padded with NaN: 23 ms instead of 0.13).  By the warp that loaded the block, once it is there and
// before it says so: the products read it behind the fence.  One block a sequence and head; no other waits.
template <int N, int CHUNKS>
__device__ __forceinline__ void zero_rows(uint32_t block, int keep, int lane) {
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c)
#pragma unroll 1
    for (int x = keep * 128 + lane * 16; x < N * 128; x += 512) ptx::sts128(block + c * N * 128 + x, 0u, 0u, 0u, 0u);
  ptx::fence_proxy_async_smem();
  __syncwarp();
}

// 32 columns of an accumulator, from column `col` of d on: this thread's row, times f, as 16-bit values through the warp's staging buffer to
// rows row0 .. row0 + 31 of the output; `z` becomes a NaN with any infinity or NaN.  The warp's lanes together; `keep`: the row
// counts, else zeros.  (Columns from d on have never been written.)
template <bool BF16>
__device__ __forceinline__ void store_columns(const uint32_t* x, float f, bool keep, uint64_t& z, uint8_t* stg, int lane, const CUtensorMap* map,
                                              int col, int d, int row0, int h, int b) {
  using namespace ptx;
  const uint64_t f2 = f2_pack(f, f);
  const uint32_t row = smem_u32(stg) + lane * 64, sw = (uint32_t)(lane >> 1 & 3) << 4;
  tma_store_wait_read();                                         // (of the lane that issued the store before)
  __syncwarp();
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    uint32_t w[4];
    if (col + 8 * u >= d) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint64_t y = f2_mul(f2_pack(__uint_as_float(x[8 * u + 2 * e]), __uint_as_float(x[8 * u + 2 * e + 1])), f2);
      z = f2_fma(y, 0ull, z);
      const float2 t = f2_unpack(y);
      w[e] = keep ? tc::pack2<BF16>(t.x, t.y) : 0u;
    }
    sts128(row + ((uint32_t)(u << 4) ^ sw), w[0], w[1], w[2], w[3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(smem_u32(stg)), "r"(col), "r"(row0), "r"(h), "r"(b) : "memory");
    tma_store_commit();
  }
}

// Zeros in rows row0 .. of columns 0 .. d - 1 (tiles behind a sequence's end).
template <bool BF16>
__device__ __forceinline__ void store_zeros(uint8_t* stg, int lane, const CUtensorMap* map, int d, int row0, int h, int b) {
  uint32_t x[32];
#pragma unroll
  for (int e = 0; e < 32; ++e) x[e] = 0u;
  uint64_t z = 0ull;
  for (int c = 0; c < d; c += 32) store_columns<BF16>(x, 0.f, false, z, stg, lane, map, c, d, row0, h, b);
}

// Steps of 16 elements of a contraction over a head dim, and the columns of an accumulator of that many: heads that fill no chunk of 64
// pay for what they have (d = 80 as 128: 63 % more of every product).
__device__ __forceinline__ int steps16(int d) { return (d + 15) >> 4; }

// D = A B^T over `steps` steps of 16 elements of chunks of 64, `a16` and `b16` bytes / 16 apart; a whole number of chunks without a test
// per step (with one, the products of d = 128 waited for their issue: 8 % of the forward kernel).
template <int CHUNKS>
__device__ __forceinline__ void scores_mma(uint32_t el, uint32_t d_tm, uint64_t ad, uint64_t bd, uint32_t a16, uint32_t b16, uint32_t id, int steps) {
  if (steps == 4 * CHUNKS) {
#pragma unroll
    for (int k = 0; k < 4 * CHUNKS; ++k) ptx::umma_ss_el(el, d_tm, ad + (k >> 2) * a16 + 2 * (k & 3), bd + (k >> 2) * b16 + 2 * (k & 3), id, k ? 1u : 0u);
  } else {
#pragma unroll 1
    for (int k = 0; k < steps; ++k) ptx::umma_ss_el(el, d_tm, ad + (k >> 2) * a16 + 2 * (k & 3), bd + (k >> 2) * b16 + 2 * (k & 3), id, k ? 1u : 0u);
  }
}

__device__ __forceinline__ bool has_nan(uint64_t z) {
  const float2 t = ptx::f2_unpack(z);
  return !(t.x == 0.f && t.y == 0.f);
}

}  // namespace sink
}  // namespace swa
