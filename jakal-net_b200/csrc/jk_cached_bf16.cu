// Propagation over a paged cache, bf16 (a unit of its own, so that the types compile in parallel).
#include "jk_cached.cuh"

namespace jk {
namespace cached {

int launch_bf16(const Args& a, const Maps& maps, const Shape& s, int64_t units, cudaStream_t stream) { return launch<__nv_bfloat16>(a, maps, s, units, stream); }

}  // namespace cached

JK_ERROR_READER(read_error_cached_bf16)

}  // namespace jk
