// Host side of the tcgen05 kernels for attention with a sliding window and sink tokens.
#include "sink_tc.cuh"

namespace swa {
namespace sink {

const char* tc_unsupported(const sink_geom_t*, const swa_tensor_t* const*, int) { return "not built"; }
const char* tc_error() { return ""; }
int tc_fwd(const Args&, int, int32_t*, cudaStream_t) { return -1; }
int64_t tc_bwd_scratch(const Args&) { return 0; }
int tc_bwd(const Args&, int, void*, int32_t*, cudaStream_t, int*) { return -1; }

}  // namespace sink
}  // namespace swa
