/*
 * swa_sequence.h -- C ABI of the operators for token sequences: rotary positions with several axes, attention with a sliding
 * window and sink tokens, and the paged cache that serves both.  Same library and conventions as swa2d.h: device pointers and
 * element strides, work enqueued on `stream`, 0 = enqueued, negative = refused before any launch (swa_last_error()).
 * What a call writes shares no memory with what it reads.
 *
 * Head dims: the CUDA-core kernels take up to 256, the tensor-core kernels multiples of 8 up to 128 in fp16 / bf16.
 */
#ifndef SWA_SEQUENCE_H_
#define SWA_SEQUENCE_H_

#include "swa2d.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ROPE_MAX_AXES 4
#define SINK_MAX_SINKS 1024

typedef struct {
  const int32_t* pos;               /* element [b, a, n] at b * pos_stride[0] + a * pos_stride[1] + n; NULL: no rotation  */
  int64_t pos_stride[2];            /* pos_stride[0] = 0: the batch shares its positions                                  */
  int32_t n_axes;                   /* 1 .. ROPE_MAX_AXES                                                                 */
  int32_t n_pairs[ROPE_MAX_AXES];   /* rotated pairs of each axis; 2 * sum <= head dim                                    */
  int32_t max_pos[ROPE_MAX_AXES];   /* rows of each table; a position behind the last row takes the last row, a negative
                                       one is not rotated on that axis                                                    */
  const float* cs[ROPE_MAX_AXES];   /* (cos, sin) tables [max_pos, n_pairs, 2] fp32                                       */
} rope_axes_t;

/* y = rotation of x by the positions (`inverse`: by their negatives, the gradient); x, y [B, H, N, C].  x2 / y2: a second
 * pair of H2 heads in the same launch, or NULL.  x and y must not overlap. */
int rope_axes_apply(int32_t dtype, const rope_axes_t* r, int32_t B, int64_t N, int32_t C, const swa_tensor_t* x, const swa_tensor_t* y,
                    int32_t H, const swa_tensor_t* x2, const swa_tensor_t* y2, int32_t H2, int32_t inverse, void* stream);

/* Attention of a token sequence: q [B, Hq, N, d_qk], k [B, Hkv, N, d_qk], v [B, Hkv, N, d_v], Hq a multiple of Hkv.  Token i sees
 * token j if j <= i and (j > i - window or j < n_sink).  lens (device int32 [B], or NULL: all N): tokens of each sequence; rows
 * behind its end are not read as keys, their outputs and gradients are zero, their lse -inf. */
typedef struct {
  int32_t dtype, B, Hq, Hkv, N, d_qk, d_v, window, n_sink;
  float sm_scale;
  int32_t impl;                     /* swa_impl_t */
  const int32_t* lens;
} sink_geom_t;

/* SWA_IMPL_SIMT or SWA_IMPL_TC: the kernels that run this shape; negative: refused. */
int sink_swa_select(const sink_geom_t* g);
/* lse [B, Hq, N] fp32, base 2. */
int sink_swa_fwd(const sink_geom_t* g, const swa_tensor_t* q, const swa_tensor_t* k, const swa_tensor_t* v, const swa_tensor_t* o,
                 float* lse, int32_t* status, void* stream);
/* Bytes of device memory sink_swa_bwd needs as scratch (16-byte aligned); negative: refused. */
int64_t sink_swa_bwd_scratch(const sink_geom_t* g);
int sink_swa_bwd(const sink_geom_t* g, const swa_tensor_t* q, const swa_tensor_t* k, const swa_tensor_t* v, const swa_tensor_t* o,
                 const swa_tensor_t* d_o, const float* lse, const swa_tensor_t* dq, const swa_tensor_t* dk, const swa_tensor_t* dv,
                 void* scratch, int64_t scratch_bytes, int32_t* status, void* stream);

/* A paged cache: k [n_pages, Hkv, page_size, d_qk], v [n_pages, Hkv, page_size, d_v] (any strides), page_table int32
 * [B, max_pages] contiguous: position p of sequence b lies in slot p % page_size of page page_table[b][p / page_size].  seq_lens int32 [B]:
 * tokens of each sequence, those of the call included.  A page number outside [0, n_pages) is no page: nothing is written to it and
 * nothing of it is seen; so pages that neither window nor sinks reach any more may be given back. */
typedef struct {
  swa_tensor_t k, v;
  const int32_t* page_table;
  const int32_t* seq_lens;
  int32_t n_pages, page_size, max_pages;
} sink_cache_t;

/* k, v [B, Hkv, T, .]: the last new_lens[b] (NULL: T) positions of sequence b, k rotated, v as it is; rows behind new_lens[b] are not
 * read.  q [B, Hq, T, d_qk] -> q_out, rotated (both NULL: none).  r->pos NULL: nothing is rotated. */
int kv_append_rope(int32_t dtype, const rope_axes_t* r, int32_t B, int32_t Hq, int32_t Hkv, int32_t T, int32_t d_qk, int32_t d_v,
                   const swa_tensor_t* q, const swa_tensor_t* q_out, const swa_tensor_t* k, const swa_tensor_t* v,
                   const sink_cache_t* cache, const int32_t* new_lens, void* stream);

/* One new token per sequence: q [B, Hq, 1, d_qk] at position seq_lens[b] - 1, o [B, Hq, 1, d_v]; a sequence of no tokens gives
 * zeros. */
int sink_swa_decode(int32_t dtype, int32_t B, int32_t Hq, int32_t Hkv, int32_t d_qk, int32_t d_v, int32_t window, int32_t n_sink,
                    float sm_scale, int32_t impl, const swa_tensor_t* q, const sink_cache_t* cache, const swa_tensor_t* o, void* stream);

#ifdef __cplusplus
}
#endif

#endif  /* SWA_SEQUENCE_H_ */
