// tcgen05 kernels of the attention with a sliding window and sink tokens: interface used by the C ABI.
#pragma once

#include "sink_rows.cuh"

namespace swa {
namespace sink {

// nullptr when the tensor-core kernels take this call, else the reason they do not.  `ts` may be null (shape only).
const char* tc_unsupported(const sink_geom_t* g, const swa_tensor_t* const* ts, int n);
const char* tc_error();
int tc_fwd(const Args& a, int dtype, int32_t* status, cudaStream_t st);
// Bytes of scratch behind the softmax delta.
int64_t tc_bwd_scratch(const Args& a);
int tc_bwd(const Args& a, int dtype, void* scratch, int32_t* status, cudaStream_t st, int* launches);

}  // namespace sink
}  // namespace swa
