// The grouped products' kernels for bf16 (a file a type: they compile side by side).
#include "grouped_kernels.cuh"

namespace gsb {
namespace grouped {

template int forward<__nv_bfloat16>(
    int, const Shape&, const WaitArgs&, const void*, const int32_t*, const int32_t*, const void*,
    const void*, void*, cudaStream_t);
template int backward<__nv_bfloat16>(
    const gs_grouped_params*, const Shape&, const WaitArgs&, const void*, const int32_t*,
    const int32_t*, const void*, const void*, const void*, void*, void*, void*, float*,
    cudaStream_t);

}  // namespace grouped
}  // namespace gsb
