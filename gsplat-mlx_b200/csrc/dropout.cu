// Dropout with a mask from a counter-based generator that is never stored:
//
//   word(i) = Philox4x32-7(key = seed, counter = (i / 4, step))[i % 4]
//   y[i]    = word(i) >= p 2^32 ? x[i] / (1 - p) : 0
//
// with i the row (whole Gaussians) or the value's place.  The backward is the
// same map on v_y, so nothing but (seed, step) is kept between the two.
//
// Philox4x32 is the counter-based generator of Salmon, Moraes, Dror and Shaw,
// "Parallel random numbers: as easy as 1, 2, 3" (SC'11); 7 rounds are the
// fewest that the paper reports as passing BigCrush.  One call yields the
// decisions of four indexes.
//
// HBM-bound: x read once, y written once, 16 bytes a thread and access.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cmath>

#include "common.cuh"

namespace gsb {
namespace {

struct Draw {
  uint32_t k0, k1;      // the seed
  uint64_t step;        // + *step_device
  const int64_t* step_device;
  uint64_t threshold;   // p 2^32: a word below it drops
  float scale;          // 1 / (1 - p)
};

__device__ __forceinline__ uint64_t draw_step(const Draw& d) {
  return d.step + (d.step_device ? (uint64_t)__ldg(d.step_device) : 0ull);
}

__device__ __forceinline__ uint4 philox7(uint64_t block, uint64_t step, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32);
  uint32_t c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint32_t keep_bits(const uint4& w, uint64_t t) {
  return (w.x >= t ? 1u : 0u) | (w.y >= t ? 2u : 0u) | (w.z >= t ? 4u : 0u) | (w.w >= t ? 8u : 0u);
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// The first right form: a thread per value.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(int64_t total, int64_t width, bool by_row,
                                                      Draw d, const T* x, T* y) {
  const uint64_t step = draw_step(d);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t at = by_row ? i / width : i;
    const uint32_t keep = keep_bits(philox7((uint64_t)at >> 2, step, d.k0, d.k1), d.threshold);
    y[i] = (keep >> (at & 3)) & 1 ? from_f<T>(to_f(x[i]) * d.scale) : from_f<T>(0.0f);
  }
}

template <typename T>
int launch(const gs_dropout_params& p, const Draw& d, const void* x, void* y, cudaStream_t s) {
  const int64_t total = p.rows * p.width;
  dropout_kernel<T><<<grid_for(total, 256), 256, 0, s>>>(total, p.width, p.by_row != 0, d,
                                                        static_cast<const T*>(x),
                                                        static_cast<T*>(y));
  return launch_status("dropout");
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int gs_dropout(const gs_dropout_params* p, const void* x, const int64_t* step_device,
                          void* y, gs_stream_t stream) {
  if (!p || p->rows < 0 || p->width < 0) return invalid("dropout: bad params");
  if (!(p->p >= 0.0 && p->p <= 1.0)) return invalid("dropout: p outside [0, 1]");
  if (p->dtype < GS_F32 || p->dtype > GS_F16) return invalid("dropout: unknown dtype");
  if (p->width > 0 && p->rows > (INT64_MAX >> 3) / p->width)
    return invalid("dropout: rows * width too large");
  if (p->by_row && p->width >= (int64_t(1) << 24))
    return invalid("dropout: rows of 2^24 values or more are not dropped as a whole");
  if (p->rows == 0 || p->width == 0) return GS_OK;
  if (!x || !y) return invalid("dropout: missing buffer");
  Draw d;
  d.k0 = static_cast<uint32_t>(p->seed);
  d.k1 = static_cast<uint32_t>(p->seed >> 32);
  d.step = p->step;
  d.step_device = step_device;
  d.threshold = static_cast<uint64_t>(std::nearbyint(p->p * 4294967296.0));
  d.scale = p->p < 1.0 ? static_cast<float>(1.0 / (1.0 - p->p)) : 0.0f;
  cudaStream_t s = as_stream(stream);
  if (p->dtype == GS_F32) return launch<float>(*p, d, x, y, s);
  if (p->dtype == GS_BF16) return launch<__nv_bfloat16>(*p, d, x, y, s);
  return launch<__half>(*p, d, x, y, s);
}
