// The grouped products' kernels for fp16 (a file a type: they compile side by side).
#include "grouped_kernels.cuh"

namespace gsb {
namespace grouped {

template int forward<__half>(
    int, const Shape&, const WaitArgs&, const void*, const int32_t*, const int32_t*, const void*,
    const void*, void*, cudaStream_t);
template int backward<__half>(
    const gs_grouped_params*, const Shape&, const WaitArgs&, const void*, const int32_t*,
    const int32_t*, const void*, const void*, const void*, void*, void*, void*, float*,
    cudaStream_t);

}  // namespace grouped
}  // namespace gsb
