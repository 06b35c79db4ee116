// Host side of the tcgen05 kernels for attention with a sliding window and sink tokens: which calls they take, tensor maps, launches.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstdio>
#include <cstring>
#include <type_traits>

#include "sink_tc.cuh"
#include "sink_tc_bwd.cuh"
#include "sink_tc_fwd.cuh"
#include "swa_tc.cuh"

namespace swa {
namespace sink {

namespace {

thread_local char g_err[256] = "";
constexpr int kSmem = 227 * 1024;

int fail(const char* what, const char* why) {
  snprintf(g_err, sizeof(g_err), "%s: %s", what, why);
  return -1;
}

// (element, token, head, batch) of a [B, H, N, d] tensor; boxes of `cols` elements x `rows` tokens, swizzled in rows of 128 bytes (cols 64,
// loads) or 64 (cols 32, stores), zero fill.
bool make_map(CUtensorMap* m, const View4& t, int dtype, int B, int H, int N, int d, int rows, int cols = 64) {
  auto fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(tc::tensor_map_encoder());
  if (!fn) {
    fail("tensor map", "cuTensorMapEncodeTiled entry point not available");
    return false;
  }
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)N, (cuuint64_t)H, (cuuint64_t)B};
  cuuint64_t strides[3] = {(cuuint64_t)t.s2 * 2, (cuuint64_t)t.s1 * 2, (cuuint64_t)t.s0 * 2};
  for (int i = 0; i < 3; ++i)                     // a dimension of extent 1 may carry any stride; give it a legal one
    if (dims[i + 1] == 1) strides[i] = 16;
  cuuint32_t box[4] = {(cuuint32_t)cols, (cuuint32_t)rows, 1u, 1u}, estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, dtype == SWA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.ptr, dims, strides, box,
                        estr, CU_TENSOR_MAP_INTERLEAVE_NONE, cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    snprintf(g_err, sizeof(g_err), "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return false;
  }
  return true;
}

}  // namespace

const char* tc_unsupported(const sink_geom_t* g, const swa_tensor_t* const* ts, int n) {
  if (g->dtype == SWA_F32) return "fp32";
  if (g->d_qk % 8 || g->d_v % 8 || g->d_qk > 128 || g->d_v > 128) return "head dims must be multiples of 8 up to 128";
  if (!(g->sm_scale > 0.f)) return "sm_scale must be positive";
  if ((int64_t)((g->N + kTile - 1) / kTile) * g->B * g->Hq > (1 << 30)) return "too many tiles";
  // The kernels' waits last about a second: a dK/dV tile's stream of G window rows has to end well before (a block of 64 to 128 takes a
  // microsecond).
  if ((int64_t)(g->Hq / g->Hkv) * (g->window < g->N ? g->window : g->N) > (1 << 25)) return "query heads per key head times window is above 2^25";
  for (int i = 0; ts && i < n; ++i) {                            // q, k, v, o[, do, dq, dk, dv]
    const int64_t* s = ts[i]->stride;
    const bool of_k = i == 1 || i == 2 || i >= 6;
    const int64_t extent[3] = {g->B, of_k ? g->Hkv : g->Hq, g->N};
    if (s[3] != 1 || (uintptr_t)ts[i]->ptr % 16) return "rows must be contiguous and start on 16-byte boundaries";
    for (int d = 0; d < 3; ++d)
      if (extent[d] > 1 && (s[d] <= 0 || s[d] % 8 || s[d] >= (int64_t)1 << 38)) return "strides must be positive multiples of 8";
  }
  return nullptr;
}

const char* tc_error() { return g_err; }

namespace {

template <int QC, int VC>
int launch_fwd(const Args& a, int dtype, int32_t* status, cudaStream_t st) {
  using S = FwdShape<QC, VC>;
  FwdParams p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.status = status;
  p.pair_heads = a.G % 2 == 0;
  const int tiles = (a.N + kTile - 1) / kTile;
  p.n_y = p.pair_heads ? tiles : (tiles + 1) / 2;
  p.n_x = p.pair_heads ? a.Hq / 2 : a.Hq;
  p.n_items = p.n_y * a.B * p.n_x;
  const int fixed = 2 * QC * (int)kChunk + 1024 + 4 * (int)kStage + (int)sizeof(FwdShared), stage = S::kKStage + S::kVStage;
  p.stages = std::min(4, (kSmem - fixed) / stage);
  const int smem = fixed + p.stages * stage;
  CUtensorMap tq, tk, tv, to;
  if (!make_map(&tq, a.q, dtype, a.B, a.Hq, a.N, a.dqk, kTile) || !make_map(&tk, a.k, dtype, a.B, a.Hkv, a.N, a.dqk, S::N) ||
      !make_map(&tv, a.v, dtype, a.B, a.Hkv, a.N, a.dv_dim, S::N) || !make_map(&to, a.o, dtype, a.B, a.Hq, a.N, a.dv_dim, 32, 32))
    return -1;
  const auto kern = dtype == SWA_BF16 ? sink_fwd_kernel<true, QC, VC> : sink_fwd_kernel<false, QC, VC>;
  cudaError_t e = allow_smem((const void*)kern);
  if (e == cudaSuccess) e = launch_pdl(kern, dim3(std::min(p.n_items, tc::sm_count())), kThreads, smem, st, tq, tk, tv, to, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail("launch", cudaGetErrorString(e));
  }
  return 0;
}

}  // namespace

int tc_fwd(const Args& a, int dtype, int32_t* status, cudaStream_t st) {
  if (a.dqk <= 64) return a.dv_dim <= 64 ? launch_fwd<1, 1>(a, dtype, status, st) : launch_fwd<1, 2>(a, dtype, status, st);
  return a.dv_dim <= 64 ? launch_fwd<2, 1>(a, dtype, status, st) : launch_fwd<2, 2>(a, dtype, status, st);
}

namespace {

template <int KIND, int XC, int VC>
int launch_bwd(const Args& a, int dtype, void* scratch, int32_t* status, cudaStream_t st, BwdParams* out) {
  using S = BwdShape<KIND, XC, VC>;
  constexpr int N = S::N, kYStage = (XC + VC) * N * 128, kX = (XC + VC) * (int)kChunk;
  BwdParams p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.status = status;
  p.n_t = (a.N + kTile - 1) / kTile;
  const int room = kSmem - 1024 - 4 * (int)kStage - (int)sizeof(BwdShared);
  p.xbufs = room - 2 * kX >= 3 * kYStage ? 2 : 1;
  p.stages = std::min(4, (room - p.xbufs * kX) / kYStage);
  const int smem = kSmem - room + p.xbufs * kX + p.stages * kYStage;
  if constexpr (KIND == 1) {
    p.n_items = p.n_t * a.B * a.Hq;
  } else {
    p.n_sb = std::min(p.n_t, (a.ns + kTile - 1) / kTile);
    const Pieces c = cut_pieces(a, p.n_sb, kTile, N);
    p.near = c.near;
    p.piece_len = c.len;
    p.pieces = c.most;
    p.n_sink_items = p.n_sb * p.pieces * a.B * a.Hkv;
    p.n_items = p.n_sink_items + (p.n_t - p.n_sb) * a.B * a.Hkv;
    p.part = (float*)scratch;
  }
  *out = p;
  if (!scratch) return 0;                          // asked for its plan only
  CUtensorMap txq, txv, tyq, tyv, toq, tov;
  bool ok = KIND == 1
      ? make_map(&txq, a.q, dtype, a.B, a.Hq, a.N, a.dqk, kTile) && make_map(&txv, a.d_o, dtype, a.B, a.Hq, a.N, a.dv_dim, kTile) &&
            make_map(&tyq, a.k, dtype, a.B, a.Hkv, a.N, a.dqk, N) && make_map(&tyv, a.v, dtype, a.B, a.Hkv, a.N, a.dv_dim, N)
      : make_map(&txq, a.k, dtype, a.B, a.Hkv, a.N, a.dqk, kTile) && make_map(&txv, a.v, dtype, a.B, a.Hkv, a.N, a.dv_dim, kTile) &&
            make_map(&tyq, a.q, dtype, a.B, a.Hq, a.N, a.dqk, N) && make_map(&tyv, a.d_o, dtype, a.B, a.Hq, a.N, a.dv_dim, N);
  ok = ok && make_map(&toq, KIND == 1 ? a.dq : a.dk, dtype, a.B, KIND == 1 ? a.Hq : a.Hkv, a.N, a.dqk, 32, 32);
  tov = toq;
  if (KIND == 2) ok = ok && make_map(&tov, a.dv, dtype, a.B, a.Hkv, a.N, a.dv_dim, 32, 32);
  if (!ok) return -1;
  const auto kern = dtype == SWA_BF16 ? sink_bwd_kernel<true, KIND, XC, VC> : sink_bwd_kernel<false, KIND, XC, VC>;
  cudaError_t e = allow_smem((const void*)kern);
  if (e == cudaSuccess) e = launch_pdl(kern, dim3(std::min(p.n_items, tc::sm_count())), kThreads, smem, st, txq, txv, tyq, tyv, toq, tov, p);
  if (e == cudaSuccess && KIND == 2 && p.pieces > 1) {
    const dim3 grid(std::min(p.n_sb * kTile, a.N + kRowWarps - 1) / kRowWarps, a.Hkv * 8, a.B);
    const JoinParams jp{a, p.n_sb, p.pieces, p.piece_len, p.near, kTile, N, 4, 4 * kTile, p.part};
    e = dtype == SWA_BF16 ? launch_pdl(join_kernel<__nv_bfloat16>, grid, 32 * kRowWarps, 0, st, jp)
                          : launch_pdl(join_kernel<__half>, grid, 32 * kRowWarps, 0, st, jp);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail("launch", cudaGetErrorString(e));
  }
  return 0;
}

template <int KIND>
int launch_bwd(const Args& a, int dtype, void* scratch, int32_t* status, cudaStream_t st, BwdParams* out) {
  const int x = a.dqk > 64, v = a.dv_dim > 64;
  return x ? v ? launch_bwd<KIND, 2, 2>(a, dtype, scratch, status, st, out) : launch_bwd<KIND, 2, 1>(a, dtype, scratch, status, st, out)
           : v ? launch_bwd<KIND, 1, 2>(a, dtype, scratch, status, st, out) : launch_bwd<KIND, 1, 1>(a, dtype, scratch, status, st, out);
}

}  // namespace

int64_t tc_bwd_scratch(const Args& a) {
  BwdParams p;
  launch_bwd<2>(a, SWA_BF16, nullptr, nullptr, nullptr, &p);
  return p.pieces > 1 ? (int64_t)a.B * a.Hkv * p.n_sb * p.pieces * kTile * (a.dqk + a.dv_dim) * 4 : 0;
}

int tc_bwd(const Args& a, int dtype, void* scratch, int32_t* status, cudaStream_t st, int* launches) {
  BwdParams p;
  if (launch_bwd<1>(a, dtype, scratch, status, st, &p)) return -1;
  if (launch_bwd<2>(a, dtype, scratch, status, st, &p)) return -1;
  *launches = p.pieces > 1 ? 3 : 2;
  return 0;
}

}  // namespace sink
}  // namespace swa
