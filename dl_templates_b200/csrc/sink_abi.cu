// C ABI (include/swa2d.h) of the operators for token sequences: argument validation, kernel-family selection, launches.
#include <algorithm>
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "common.cuh"
#include "rope_axes.cuh"
#include "sink_decode.cuh"
#include "sink_f32.cuh"
#include "sink_rows.cuh"
#include "sink_tc.cuh"

namespace swa {
int abi_fail(int code, const char* msg);
int abi_launched(const char* what);
}  // namespace swa

namespace {

using swa::abi_launched;

enum : int { E_NULL = -1, E_DTYPE = -2, E_SHAPE = -3, E_ROPE = -4, E_IMPL = -5, E_LAUNCH = -6, E_STRIDE = -7 };

int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return swa::abi_fail(code, msg);
}

int check_tensor(const swa_tensor_t* t, const char* name) {
  if (!t || !t->ptr) return fail(E_NULL, "%s is NULL", name);
  return 0;
}
int check_dtype(int32_t dtype) {
  if (dtype < SWA_F32 || dtype > SWA_BF16) return fail(E_DTYPE, "unknown dtype %d", dtype);
  return 0;
}

int check_axes(const rope_axes_t* r, int32_t C) {
  if (!r) return fail(E_NULL, "rope axes are NULL");
  if (r->n_axes < 1 || r->n_axes > ROPE_MAX_AXES) return fail(E_ROPE, "n_axes must be in [1, %d]", ROPE_MAX_AXES);
  int64_t pairs = 0;
  for (int a = 0; a < r->n_axes; ++a) {
    if (r->n_pairs[a] <= 0 || r->max_pos[a] <= 0) return fail(E_ROPE, "axis %d: pairs and table rows must be positive", a);
    if (!r->cs[a]) return fail(E_ROPE, "axis %d: table is NULL", a);
    pairs += r->n_pairs[a];
  }
  if (2 * pairs > C) return fail(E_ROPE, "2 * pairs of all axes (%lld) exceeds the head dim %d", (long long)(2 * pairs), C);
  return 0;
}

int check_heads(int32_t B, int32_t Hq, int32_t Hkv) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0) return fail(E_SHAPE, "batch and heads must be positive");
  if (Hq % Hkv) return fail(E_SHAPE, "query heads (%d) must be a multiple of key heads (%d)", Hq, Hkv);
  if (B > 65535 || Hq > 65535 || Hkv > 8191) return fail(E_SHAPE, "batch and query heads must be at most 65535, key heads at most 8191");
  return 0;
}

int check_geom(const sink_geom_t* g) {
  if (!g) return fail(E_NULL, "geometry is NULL");
  if (int e = check_dtype(g->dtype)) return e;
  if (int e = check_heads(g->B, g->Hq, g->Hkv)) return e;
  if (g->N <= 0 || g->N > (1 << 30)) return fail(E_SHAPE, "tokens must be in [1, 2^30]");
  if (g->d_qk <= 0 || g->d_v <= 0 || g->d_qk > swa::sink::kMaxDim || g->d_v > swa::sink::kMaxDim)
    return fail(E_SHAPE, "head dims must be in [1, %d]", swa::sink::kMaxDim);
  if (g->window < 1) return fail(E_SHAPE, "window must be at least 1 (a token sees itself)");
  if (g->n_sink < 0 || g->n_sink > SINK_MAX_SINKS) return fail(E_SHAPE, "n_sink must be in [0, %d]", SINK_MAX_SINKS);
  if (g->impl < SWA_IMPL_AUTO || g->impl > SWA_IMPL_TC) return fail(E_IMPL, "unknown impl %d", g->impl);
  return 0;
}

swa::sink::Args make_args(const sink_geom_t* g) {
  swa::sink::Args a;
  memset(&a, 0, sizeof(a));
  a.lens = g->lens;
  a.B = g->B; a.Hq = g->Hq; a.Hkv = g->Hkv; a.G = g->Hq / g->Hkv; a.N = g->N;
  a.dqk = g->d_qk; a.dv_dim = g->d_v;
  a.W = std::min(g->window, g->N);
  a.ns = std::min(g->n_sink, g->N);
  a.scale = g->sm_scale;
  a.c2 = g->sm_scale * swa::kLog2e;
  return a;
}

int resolve(const sink_geom_t* g, const swa_tensor_t* const* ts, int n) {
  const char* why = swa::sink::tc_unsupported(g, ts, n);
  if (g->impl == SWA_IMPL_SIMT) return SWA_IMPL_SIMT;
  if (!why) return SWA_IMPL_TC;
  if (g->impl == SWA_IMPL_TC) return fail(E_IMPL, "tensor-core path unavailable: %s", why);
  return SWA_IMPL_SIMT;
}

#define SINK_DISPATCH(dtype, ...)                                 \
  do {                                                            \
    switch (dtype) {                                              \
      case SWA_F32: { using T = float; __VA_ARGS__; break; }      \
      case SWA_F16: { using T = __half; __VA_ARGS__; break; }     \
      default: { using T = __nv_bfloat16; __VA_ARGS__; break; }   \
    }                                                             \
  } while (0)

int launched(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(E_LAUNCH, "%s launch failed: %s", what, cudaGetErrorString(e));
  }
  return abi_launched(what);
}

template <int KIND>
int launch_rows(const swa::sink::Args& a, int dtype, cudaStream_t st) {
  const dim3 grid((unsigned)((a.N + swa::sink::kRowWarps - 1) / swa::sink::kRowWarps), KIND == 2 ? a.Hkv : a.Hq, a.B);
  cudaError_t e = cudaSuccess;
  SINK_DISPATCH(dtype, e = swa::launch_pdl(swa::sink::rows_kernel<T, KIND>, grid, 32 * swa::sink::kRowWarps, 0, st, a));
  return launched(e, KIND == 0 ? "sink rows forward" : KIND == 1 ? "sink rows dQ" : "sink rows dK/dV");
}

// ---- fp32 tiles --------------------------------------------------------------------------------------------------------
bool f32_shape(const sink_geom_t* g) { return g->dtype == SWA_F32 && g->d_qk % 4 == 0 && g->d_v % 4 == 0 && g->d_qk <= 128 && g->d_v <= 128; }

bool f32_tiles(const sink_geom_t* g, const swa_tensor_t* const* ts, int n) {
  if (!f32_shape(g)) return false;
  for (int i = 0; i < n; ++i)
    if (ts[i]->stride[3] != 1 || (uintptr_t)ts[i]->ptr % 16 || ts[i]->stride[0] % 4 || ts[i]->stride[1] % 4 || ts[i]->stride[2] % 4) return false;
  return true;
}

// Plan of a kernel: tiles, pieces of the blocks with sinks (KIND 2).
template <int KIND>
swa::sink::F32Params f32_plan(const swa::sink::Args& a, float* part) {
  constexpr int R = swa::sink::kF32X;
  swa::sink::F32Params p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.n_t = (a.N + R - 1) / R;
  p.part = part;
  if (KIND == 2) {
    p.n_sb = std::min(p.n_t, (a.ns + R - 1) / R);
    const swa::sink::Pieces c = swa::sink::cut_pieces(a, p.n_sb, R, swa::sink::kF32Rows);
    p.near = c.near;
    p.piece_len = c.len;
    p.pieces = c.most;
    p.n_sink_items = p.n_sb * p.pieces * a.B * a.Hkv;
  }
  return p;
}
int64_t f32_scratch(const swa::sink::Args& a) {
  const swa::sink::F32Params p = f32_plan<2>(a, nullptr);
  return p.pieces > 1 ? (int64_t)a.B * a.Hkv * p.n_sb * p.pieces * swa::sink::kF32X * (a.dqk + a.dv_dim) * 4 : 0;
}

template <int KIND, int DQ, int DV>
cudaError_t launch_f32_as(const swa::sink::F32Params& p, int64_t items, cudaStream_t st) {
  const auto kern = swa::sink::f32_kernel<KIND, DQ, DV>;
  constexpr int smem = swa::sink::F32Shape<KIND, DQ, DV>::kSmem;
  cudaError_t e = swa::set_once((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = swa::set_once((const void*)kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  kern<<<dim3((unsigned)items), swa::sink::kF32Threads, smem, st>>>(p);
  return cudaGetLastError();
}

template <int KIND>
int launch_f32(const swa::sink::Args& a, float* part, cudaStream_t st) {
  const swa::sink::F32Params p = f32_plan<KIND>(a, part);
  const int64_t items = KIND == 2 ? p.n_sink_items + (int64_t)(p.n_t - p.n_sb) * a.B * a.Hkv : (int64_t)p.n_t * a.B * a.Hq;
  if (items > INT32_MAX) return fail(E_SHAPE, "too many tiles");
  cudaError_t e = a.dqk <= 64 ? a.dv_dim <= 64 ? launch_f32_as<KIND, 64, 64>(p, items, st) : launch_f32_as<KIND, 64, 128>(p, items, st)
                              : a.dv_dim <= 64 ? launch_f32_as<KIND, 128, 64>(p, items, st) : launch_f32_as<KIND, 128, 128>(p, items, st);
  if (int c = launched(e, "sink fp32 tiles")) return c;
  if (KIND != 2 || p.pieces <= 1) return 0;
  constexpr int R = swa::sink::kF32X, WARPS = swa::sink::kRowWarps;
  const swa::sink::JoinParams jp{a, p.n_sb, p.pieces, p.piece_len, p.near, R, swa::sink::kF32Rows, a.dqk + a.dv_dim, 4, part};
  e = swa::launch_pdl(swa::sink::join_kernel<float>, dim3(std::min(p.n_sb * R, a.N + WARPS - 1) / WARPS, a.Hkv * 8, a.B), 32 * WARPS, 0, st, jp);
  return launched(e, "sink join");
}

// ---- rotation --------------------------------------------------------------------------------------------------------
bool aligned(const swa_tensor_t& t, int ve, int esz) {
  if (ve == 1) return true;
  return t.stride[3] == 1 && (uintptr_t)t.ptr % (ve * esz) == 0 && t.stride[0] % ve == 0 && t.stride[1] % ve == 0 && t.stride[2] % ve == 0;
}

// Launches the groups of `a` (g[i].H > 0) with the widest unit that all of them, the axes and the tables allow.
int launch_rotate(swa::axes::Args& a, int n_groups, const swa_tensor_t* const* tensors, int n_tensors, int dtype, int B, cudaStream_t st) {
  const int esz = dtype == SWA_F32 ? 4 : 2;
  bool rotates = false;
  for (int i = 0; i < n_groups; ++i) rotates |= a.g[i].rotate != 0;
  auto fits = [&](int ve) {
    for (int i = 0; i < n_groups; ++i)
      if (a.g[i].d % ve) return false;
    for (int i = 0; i < n_tensors; ++i)
      if (!aligned(*tensors[i], ve, esz)) return false;
    for (int x = 0; rotates && x < a.n_axes; ++x)
      if (a.R[x] % ve || (ve > 1 && (uintptr_t)a.cs[x] % 16)) return false;
    return true;
  };
  int ve = 16 / esz;
  while (!fits(ve)) ve >>= 1;
  int64_t spr = 0;
  int heads = 0;
  for (int i = 0; i < n_groups; ++i) {
    const int64_t rot = a.g[i].rotate ? a.pairs / ve : 0;
    spr = std::max(spr, rot + (a.g[i].d / ve - 2 * rot + 1) / 2);
    heads += a.g[i].H;
  }
  // Four heads a thread where that leaves two blocks for every place on the SMs (8 of 148): their loads are in flight together and the
  // table is read once (168 MB of bf16 rows: 32 us, one head a thread 41); fewer rows want the blocks (173 tokens: 2.1 us).
  const bool four = a.N * spr / 256 * B * ((heads + 3) / 4) >= 2 * 8 * swa::sink::kSms;
  int64_t chunks = 0;
  for (int i = 0; i < n_groups; ++i) chunks += a.g[i].chunks = four ? (a.g[i].H + 3) / 4 : a.g[i].H;
  if (a.N * spr > INT32_MAX || a.N * spr * chunks > INT32_MAX) return fail(E_SHAPE, "too many tokens in one call");
  a.slots = (int)spr;
  const dim3 grid((unsigned)((a.N * spr * chunks + 255) / 256), 1, B);
  cudaError_t e = cudaSuccess;
#define ROT(T, VE) e = four ? swa::launch_stream(swa::axes::rotate_kernel<T, VE, 4>, grid, 256, st, a) : swa::launch_stream(swa::axes::rotate_kernel<T, VE, 1>, grid, 256, st, a)
#define ROT16(T) do { if (ve == 8) ROT(T, 8); else if (ve == 4) ROT(T, 4); else if (ve == 2) ROT(T, 2); else ROT(T, 1); } while (0)
  if (dtype == SWA_F32) {
    if (ve == 4) ROT(float, 4); else if (ve == 2) ROT(float, 2); else ROT(float, 1);
  } else if (dtype == SWA_F16) {
    ROT16(__half);
  } else {
    ROT16(__nv_bfloat16);
  }
#undef ROT16
#undef ROT
  return launched(e, "rotate");
}

void set_axes(swa::axes::Args* a, const rope_axes_t* r) {
  a->n_axes = r->n_axes;
  a->pairs = 0;
  for (int x = 0; x < r->n_axes; ++x) {
    a->R[x] = r->n_pairs[x];
    a->max_pos[x] = r->max_pos[x];
    a->cs[x] = r->cs[x];
    a->pairs += r->n_pairs[x];
  }
  a->pos = r->pos;
  a->pos_b = r->pos_stride[0];
  a->pos_a = r->pos_stride[1];
}

int check_cache(const sink_cache_t* c) {
  if (!c) return fail(E_NULL, "cache is NULL");
  if (int e = check_tensor(&c->k, "k cache")) return e;
  if (int e = check_tensor(&c->v, "v cache")) return e;
  if (!c->page_table || !c->seq_lens) return fail(E_NULL, "page_table or seq_lens is NULL");
  if (c->n_pages <= 0 || c->page_size <= 0 || c->max_pages <= 0) return fail(E_SHAPE, "pages, page size and table width must be positive");
  if ((int64_t)c->max_pages * c->page_size > (1 << 30)) return fail(E_SHAPE, "a sequence may hold at most 2^30 tokens");
  return 0;
}

// ---- decode ------------------------------------------------------------------------------------------------------------
// nullptr when the split kernel takes the call, else the reason it does not.
const char* split_unsupported(int dtype, const swa::sink::DecodeArgs& a) {
  const int e = dtype == SWA_F32 ? 4 : 8, esz = 16 / e;
  if (a.dqk % e || a.dv % e || a.dqk > 128 || a.dv > 128) return "head dims must be multiples of 16 bytes, up to 128 elements";
  for (const swa::View4* c : {&a.k, &a.v})
    if (c->s3 != 1 || (uintptr_t)c->ptr % 16 || c->s0 % e || c->s1 % e || c->s2 % e) return "rows of the cache must be contiguous and start on 16-byte boundaries";
  if (a.q.s3 != 1 || (uintptr_t)a.q.ptr % (2 * esz) || a.q.s0 % 2 || a.q.s1 % 2) return "rows of q must be contiguous and start on even elements";
  for (const swa::View4* c : {&a.k, &a.v})
    if (c->s0 > INT32_MAX || c->s2 > INT32_MAX) return "pages of the cache are too far apart";
  if ((int64_t)a.B * a.Hkv * ((a.G + 15) / 16) > (1 << 26)) return "too many sequences and heads";
  return nullptr;
}

template <typename T, int DK, int DV, int HPL>
cudaError_t launch_split_as(const swa::sink::DecodeArgs& a, unsigned units, cudaStream_t st) {
  const auto kern = swa::sink::decode_split_kernel<T, DK, DV, HPL>;
  constexpr int smem = swa::sink::DecodeShape<T, DK, DV>::kSmem;
  cudaError_t e = swa::set_once((const void*)kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e == cudaSuccess) e = swa::set_once((const void*)kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) e = swa::set_once((const void*)kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * a.split);
  cfg.blockDim = dim3(32 * swa::sink::kDecWarps);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = a.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

template <typename T, int HPL>
cudaError_t launch_split_dims(const swa::sink::DecodeArgs& a, unsigned units, cudaStream_t st) {
  if (a.dqk <= 64) return a.dv <= 64 ? launch_split_as<T, 64, 64, HPL>(a, units, st) : launch_split_as<T, 64, 128, HPL>(a, units, st);
  return a.dv <= 64 ? launch_split_as<T, 128, 64, HPL>(a, units, st) : launch_split_as<T, 128, 128, HPL>(a, units, st);
}

cudaError_t launch_split(int dtype, swa::sink::DecodeArgs& a, cudaStream_t st) {
  const unsigned units = (unsigned)a.B * a.Hkv * ((a.G + swa::sink::kDecHeads - 1) / swa::sink::kDecHeads);
  // CTAs of a cluster: as many as there is room for at once, while every warp keeps two tiles of 16 tokens.  Clusters of up to 4 find two
  // places on every SM; larger ones have to fit into a GPC: those of 8 gain while there is an SM for each CTA, those of 16 while each has a
  // GPC, of which there are eight, of its own.  Measured (bf16, d = 128, us of a launch with 16 / 8 / 4 CTAs, cold L2):
  //   pairs of sequence and key head     2052 tokens           6004 tokens
  //                               4      14.3 / 14.3 / 17.6    16.4 / 20.5 / 28.0
  //                               8      16.4 / 15.4 / 18.4    20.6 / 20.5 / 28.7      (launches in a row, 2052 tokens: 10.2 / 10.5)
  //                               9      16.4 / 16.4 / 18.4    22.5 / 20.6 / 28.7
  //                              12      17.6 / 16.4 / 18.4    23.8 / 22.5 / 28.7
  //                              16      26.5 / 18.4 / 18.4    36.9 / 30.7 / 30.2
  //                              24         - / 20.1 / 18.4       - / 34.8 / 33.0
  //                              40         - / 30.7 / 26.6       - / 55.3 / 53.3
  // and with 4 / 2 / 1: 64 pairs, 6004 tokens 41 / 62 / 104; 512 pairs, 4100 tokens 213 / 202 / 187.
  const int64_t seen = std::min((int64_t)a.W + a.ns, (int64_t)a.max_pages * a.page_size);
  using swa::sink::kSms;
  auto room = [](int c) { return c <= 4 ? 2 * kSms + 24 : c == 8 ? kSms : 8 * 16; };
  a.split = 1;
  while (a.split < 16 && (int64_t)units * a.split * 2 <= room(2 * a.split) && seen > (int64_t)a.split * swa::sink::kDecWarps * 32) a.split *= 2;
  a.page_shift = -1;
  if ((a.page_size & (a.page_size - 1)) == 0)
    for (a.page_shift = 0; 1 << a.page_shift < a.page_size;) ++a.page_shift;
  const int nh = std::min(a.G, swa::sink::kDecHeads);
  if (dtype == SWA_F16) return nh <= 8 ? launch_split_dims<__half, 1>(a, units, st) : launch_split_dims<__half, 2>(a, units, st);
  if (dtype == SWA_BF16) return nh <= 8 ? launch_split_dims<__nv_bfloat16, 1>(a, units, st) : launch_split_dims<__nv_bfloat16, 2>(a, units, st);
  return nh <= 4 ? launch_split_dims<float, 1>(a, units, st) : nh <= 8 ? launch_split_dims<float, 2>(a, units, st) : launch_split_dims<float, 4>(a, units, st);
}

}  // namespace

extern "C" {

int rope_axes_apply(int32_t dtype, const rope_axes_t* r, int32_t B, int64_t N, int32_t C, const swa_tensor_t* x, const swa_tensor_t* y,
                    int32_t H, const swa_tensor_t* x2, const swa_tensor_t* y2, int32_t H2, int32_t inverse, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (B <= 0 || B > 65535 || N <= 0 || N > INT32_MAX || C <= 0 || H <= 0 || (x2 && H2 <= 0)) return fail(E_SHAPE, "bad batch, tokens, heads or head dim");
  if (int e = check_axes(r, C)) return e;
  if (!r->pos) return fail(E_NULL, "positions are NULL");
  if (int e = check_tensor(x, "x")) return e;
  if (int e = check_tensor(y, "y")) return e;
  if (x2) {
    if (int e = check_tensor(x2, "x2")) return e;
    if (int e = check_tensor(y2, "y2")) return e;
  }
  swa::axes::Args a;
  memset(&a, 0, sizeof(a));
  set_axes(&a, r);
  a.N = (int)N;
  a.sign = inverse ? -1.f : 1.f;
  a.g[0] = swa::axes::Group{swa::make_view(x), swa::make_view(y), H, C, 1, 0, 0};
  if (x2) a.g[1] = swa::axes::Group{swa::make_view(x2), swa::make_view(y2), H2, C, 1, 0, 0};
  const swa_tensor_t* ts[] = {x, y, x2, y2};
  return launch_rotate(a, x2 ? 2 : 1, ts, x2 ? 4 : 2, dtype, B, (cudaStream_t)stream);
}

int kv_append_rope(int32_t dtype, const rope_axes_t* r, int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t d_qk, int32_t d_v,
                   const swa_tensor_t* q, const swa_tensor_t* q_out, const swa_tensor_t* k, const swa_tensor_t* v,
                   const sink_cache_t* cache, const int32_t* new_lens, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (B <= 0 || B > 65535 || Hkv <= 0 || T <= 0 || d_qk <= 0 || d_v <= 0 || (q && Hq <= 0)) return fail(E_SHAPE, "bad batch, tokens, heads or head dim");
  const bool rot = r && r->pos;
  if (rot)
    if (int e = check_axes(r, d_qk)) return e;
  if (int e = check_tensor(k, "k")) return e;
  if (int e = check_tensor(v, "v")) return e;
  if (int e = check_cache(cache)) return e;
  if ((q != nullptr) != (q_out != nullptr)) return fail(E_NULL, "q and q_out go together");
  if (q) {
    if (int e = check_tensor(q, "q")) return e;
    if (int e = check_tensor(q_out, "q_out")) return e;
  }
  swa::axes::Args a;
  memset(&a, 0, sizeof(a));
  if (rot) set_axes(&a, r);
  a.N = T;
  a.sign = 1.f;
  a.page_table = cache->page_table;
  a.seq_lens = cache->seq_lens;
  a.new_lens = new_lens;
  a.max_pages = cache->max_pages;
  a.n_pages = cache->n_pages;
  a.page_size = cache->page_size;
  const swa_tensor_t* ts[6] = {k, &cache->k, v, &cache->v, q, q_out};
  a.g[0] = swa::axes::Group{swa::make_view(k), swa::make_view(&cache->k), Hkv, d_qk, rot, 1, 0};
  a.g[1] = swa::axes::Group{swa::make_view(v), swa::make_view(&cache->v), Hkv, d_v, 0, 1, 0};
  if (q) a.g[2] = swa::axes::Group{swa::make_view(q), swa::make_view(q_out), Hq, d_qk, rot, 0, 0};
  return launch_rotate(a, q ? 3 : 2, ts, q ? 6 : 4, dtype, B, (cudaStream_t)stream);
}

int sink_swa_select(const sink_geom_t* g) {
  if (int e = check_geom(g)) return e;
  return resolve(g, nullptr, 0);
}

int sink_swa_fwd(const sink_geom_t* g, const swa_tensor_t* q, const swa_tensor_t* k, const swa_tensor_t* v, const swa_tensor_t* o,
                 float* lse, int32_t* status, void* stream) {
  if (int e = check_geom(g)) return e;
  if (int e = check_tensor(q, "q")) return e;
  if (int e = check_tensor(k, "k")) return e;
  if (int e = check_tensor(v, "v")) return e;
  if (int e = check_tensor(o, "o")) return e;
  if (!lse) return fail(E_NULL, "lse is NULL");
  const swa_tensor_t* ts[] = {q, k, v, o};
  const int impl = resolve(g, ts, 4);
  if (impl < 0) return impl;
  cudaStream_t st = (cudaStream_t)stream;
  swa::sink::Args a = make_args(g);
  a.q = swa::make_view(q); a.k = swa::make_view(k); a.v = swa::make_view(v); a.o = swa::make_view(o);
  a.lse = lse;
  if (impl == SWA_IMPL_TC) {
    if (swa::sink::tc_fwd(a, g->dtype, status, st)) return fail(E_LAUNCH, "tcgen05 sink forward: %s", swa::sink::tc_error());
    return abi_launched("tcgen05 sink forward");
  }
  if (f32_tiles(g, ts, 4)) return launch_f32<0>(a, nullptr, st);
  return launch_rows<0>(a, g->dtype, st);
}

// The softmax delta: rows of whole 16-byte units, up to 32 of them, or any others.
static int launch_delta(const swa::sink::Args& a, const sink_geom_t* g, const swa_tensor_t* o, const swa_tensor_t* d_o, void* stream) {
  const int e = g->dtype == SWA_F32 ? 4 : 8, units = g->d_v / e;
  auto whole = [&](const swa_tensor_t* t) {
    return t->stride[3] == 1 && (uintptr_t)t->ptr % 16 == 0 && t->stride[0] % e == 0 && t->stride[1] % e == 0 && t->stride[2] % e == 0;
  };
  cudaError_t err = cudaSuccess;
  if (g->d_v % e || units > 32 || !whole(o) || !whole(d_o)) {
    const dim3 grid((a.N + swa::sink::kRowWarps - 1) / swa::sink::kRowWarps, a.Hq, a.B);
    SINK_DISPATCH(g->dtype, err = swa::launch_stream(swa::sink::delta_any_kernel<T>, grid, 32 * swa::sink::kRowWarps, (cudaStream_t)stream, a));
    return launched(err, "sink delta");
  }
  int group = 1;
  while (group < units) group *= 2;
  const int rows = 256 / group * swa::sink::kDeltaRows;
  const dim3 grid((a.N + rows - 1) / rows, a.Hq, a.B);
  SINK_DISPATCH(g->dtype, err = swa::launch_stream(swa::sink::delta_rows_kernel<T>, grid, 256, (cudaStream_t)stream, a, units, group));
  return launched(err, "sink delta");
}

static int64_t delta_bytes(const sink_geom_t* g) { return ((int64_t)g->B * g->Hq * g->N * 4 + 255) / 256 * 256; }

static int64_t part_bytes(const sink_geom_t* g, int impl) {
  return impl == SWA_IMPL_TC ? swa::sink::tc_bwd_scratch(make_args(g)) : f32_shape(g) ? f32_scratch(make_args(g)) : 0;
}

int64_t sink_swa_bwd_scratch(const sink_geom_t* g) {
  if (int e = check_geom(g)) return e;
  const int impl = resolve(g, nullptr, 0);
  if (impl < 0) return impl;
  return delta_bytes(g) + part_bytes(g, impl);
}

int sink_swa_bwd(const sink_geom_t* g, const swa_tensor_t* q, const swa_tensor_t* k, const swa_tensor_t* v, const swa_tensor_t* o,
                 const swa_tensor_t* d_o, const float* lse, const swa_tensor_t* dq, const swa_tensor_t* dk, const swa_tensor_t* dv,
                 void* scratch, int64_t scratch_bytes, int32_t* status, void* stream) {
  if (int e = check_geom(g)) return e;
  const swa_tensor_t* ts[] = {q, k, v, o, d_o, dq, dk, dv};
  const char* names[] = {"q", "k", "v", "o", "do", "dq", "dk", "dv"};
  for (int i = 0; i < 8; ++i)
    if (int e = check_tensor(ts[i], names[i])) return e;
  if (!lse || !scratch) return fail(E_NULL, "lse or scratch is NULL");
  const int impl = resolve(g, ts, 8);
  if (impl < 0) return impl;
  const int64_t need = delta_bytes(g) + part_bytes(g, impl);
  if (scratch_bytes < need || (uintptr_t)scratch % 16) return fail(E_SHAPE, "scratch: %lld bytes on a 16-byte boundary needed", (long long)need);
  cudaStream_t st = (cudaStream_t)stream;
  swa::sink::Args a = make_args(g);
  a.q = swa::make_view(q); a.k = swa::make_view(k); a.v = swa::make_view(v); a.o = swa::make_view(o); a.d_o = swa::make_view(d_o);
  a.dq = swa::make_view(dq); a.dk = swa::make_view(dk); a.dv = swa::make_view(dv);
  a.lse = const_cast<float*>(lse);
  a.delta = (float*)scratch;
  if (int e = launch_delta(a, g, o, d_o, stream)) return e;
  if (impl == SWA_IMPL_TC) {
    int launches = 0;
    if (swa::sink::tc_bwd(a, g->dtype, (char*)scratch + delta_bytes(g), status, st, &launches))
      return fail(E_LAUNCH, "tcgen05 sink backward: %s", swa::sink::tc_error());
    for (int i = 0; i < launches; ++i)
      if (int e = abi_launched("tcgen05 sink backward")) return e;
    return 0;
  }
  if (f32_tiles(g, ts, 8)) {
    if (int e = launch_f32<1>(a, nullptr, st)) return e;
    return launch_f32<2>(a, (float*)((char*)scratch + delta_bytes(g)), st);
  }
  if (int e = launch_rows<1>(a, g->dtype, st)) return e;
  return launch_rows<2>(a, g->dtype, st);
}

int sink_swa_decode(int32_t dtype, int32_t B, int32_t Hq, int32_t Hkv, int32_t d_qk, int32_t d_v, int32_t window, int32_t n_sink,
                    float sm_scale, int32_t impl, const swa_tensor_t* q, const sink_cache_t* cache, const swa_tensor_t* o, void* stream) {
  if (int e = check_dtype(dtype)) return e;
  if (int e = check_heads(B, Hq, Hkv)) return e;
  if (d_qk <= 0 || d_v <= 0 || d_qk > swa::sink::kMaxDim || d_v > swa::sink::kMaxDim)
    return fail(E_SHAPE, "head dims must be in [1, %d]", swa::sink::kMaxDim);
  if (window < 1) return fail(E_SHAPE, "window must be at least 1 (a token sees itself)");
  if (n_sink < 0 || n_sink > SINK_MAX_SINKS) return fail(E_SHAPE, "n_sink must be in [0, %d]", SINK_MAX_SINKS);
  if (impl < SWA_IMPL_AUTO || impl > SWA_IMPL_TC) return fail(E_IMPL, "unknown impl %d", impl);
  if (int e = check_tensor(q, "q")) return e;
  if (int e = check_tensor(o, "o")) return e;
  if (int e = check_cache(cache)) return e;
  swa::sink::DecodeArgs a;
  memset(&a, 0, sizeof(a));
  a.q = swa::make_view(q); a.o = swa::make_view(o); a.k = swa::make_view(&cache->k); a.v = swa::make_view(&cache->v);
  a.page_table = cache->page_table; a.seq_lens = cache->seq_lens;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.G = Hq / Hkv; a.dqk = d_qk; a.dv = d_v; a.W = window; a.ns = n_sink;
  a.max_pages = cache->max_pages; a.n_pages = cache->n_pages; a.page_size = cache->page_size;
  a.c2 = sm_scale * swa::kLog2e;
  cudaStream_t st = (cudaStream_t)stream;
  const char* why = split_unsupported(dtype, a);
  if (impl == SWA_IMPL_TC && (why || dtype == SWA_F32)) return fail(E_IMPL, "tensor-core path unavailable: %s", why ? why : "fp32");
  if (!why && impl != SWA_IMPL_SIMT) return launched(launch_split(dtype, a, st), "sink decode split");
  const dim3 grid((Hq + swa::sink::kRowWarps - 1) / swa::sink::kRowWarps, B);
  cudaError_t e = cudaSuccess;
  SINK_DISPATCH(dtype, e = swa::launch_pdl(swa::sink::decode_rows_kernel<T>, grid, 32 * swa::sink::kRowWarps, 0, st, a));
  return launched(e, "sink decode");
}

}  // extern "C"
