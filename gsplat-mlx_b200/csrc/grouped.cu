// Products of ragged groups of rows with one weight matrix per group (a
// learned layer per camera over the packed rows, which are sorted by camera):
//
//   y[r]   = act(W[g] x[id(r)] + b[g])           off[g] <= r < off[g + 1]
//   v_z[r] = v_y[r] act'(y[r])
//   v_x[id(r)] += W[g]^T v_z[r],  v_W[g] = sum v_z[r] x[id(r)]^T,  v_b[g] = sum v_z[r]
//
// A row's group is found by binary search over the offsets; the search's
// invariant off[g] <= r < off[g + 1] holds for the pair that it ends at even
// where the offsets do not ascend, so no index leaves its buffer.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace gsb {
namespace {

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

struct Shape {
  int64_t R, n;
  int G, K, M;
};

// The group of row r: -1 in front of the first, G behind the last.
__device__ __forceinline__ int group_of(const int32_t* __restrict__ off, int G, int64_t r) {
  if (r < __ldg(off)) return -1;
  if (r >= __ldg(off + G)) return G;
  int lo = 0, hi = G;  // off[lo] <= r < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(off + mid) <= r) lo = mid; else hi = mid;
  }
  return lo;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == GS_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN passes
  if (ACT == GS_ACT_SIGMOID) return 1.0f / (1.0f + expf(-z));
  return z;
}
// v_z from v and the activated y
template <int ACT>
__device__ __forceinline__ float through(float v, float y) {
  if (ACT == GS_ACT_RELU) return y > 0.0f ? v : 0.0f;
  if (ACT == GS_ACT_SIGMOID) return v * y * (1.0f - y);
  return v;
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) fwd_kernel(Shape s, const T* __restrict__ x,
                                                  const int32_t* __restrict__ ids,
                                                  const int32_t* __restrict__ off,
                                                  const T* __restrict__ w,
                                                  const T* __restrict__ b, T* __restrict__ y) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < s.R * s.M;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / s.M;
    const int m = (int)(i - r * s.M);
    const int g = group_of(off, s.G, r);
    if (g < 0 || g >= s.G) {
      y[i] = from_f<T>(0.0f);
      continue;
    }
    const int64_t at = ids ? ids[r] : r;
    float acc = 0.0f;
    if (at >= 0 && at < s.n)
      for (int k = 0; k < s.K; ++k)
        acc = fmaf(to_f(x[at * s.K + k]), to_f(w[((int64_t)g * s.M + m) * s.K + k]), acc);
    if (b) acc += to_f(b[(int64_t)g * s.M + m]);
    y[i] = from_f<T>(activate<ACT>(acc));
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) bwd_x_kernel(Shape s, const int32_t* __restrict__ ids,
                                                    const int32_t* __restrict__ off,
                                                    const T* __restrict__ w,
                                                    const T* __restrict__ y,
                                                    const T* __restrict__ vy,
                                                    float* __restrict__ sum, T* __restrict__ vx) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < s.R * s.K;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / s.K;
    const int k = (int)(i - r * s.K);
    const int g = group_of(off, s.G, r);
    float acc = 0.0f;
    if (g >= 0 && g < s.G)
      for (int m = 0; m < s.M; ++m) {
        const float v = through<ACT>(to_f(vy[r * s.M + m]), ACT ? to_f(y[r * s.M + m]) : 0.0f);
        acc = fmaf(v, to_f(w[((int64_t)g * s.M + m) * s.K + k]), acc);
      }
    if (!ids) {
      vx[i] = from_f<T>(acc);
    } else if (g >= 0 && g < s.G) {
      const int64_t at = ids[r];
      if (at >= 0 && at < s.n) atomicAdd(sum + at * s.K + k, acc);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) round_kernel(int64_t n, const float* __restrict__ a,
                                                    T* __restrict__ b) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    b[i] = from_f<T>(a[i]);
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) bwd_w_kernel(Shape s, const T* __restrict__ x,
                                                    const int32_t* __restrict__ ids,
                                                    const int32_t* __restrict__ off,
                                                    const T* __restrict__ y,
                                                    const T* __restrict__ vy, T* __restrict__ vw,
                                                    T* __restrict__ vb) {
  const int64_t each = (int64_t)s.M * (s.K + 1);
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < s.G * each;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int g = (int)(i / each);
    const int m = (int)((i - g * each) / (s.K + 1));
    const int k = (int)((i - g * each) % (s.K + 1));
    const int64_t r0 = max((int64_t)off[g], (int64_t)0), r1 = min((int64_t)off[g + 1], s.R);
    float acc = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
      const float v = through<ACT>(to_f(vy[r * s.M + m]), ACT ? to_f(y[r * s.M + m]) : 0.0f);
      if (k == s.K) {
        acc += v;
        continue;
      }
      const int64_t at = ids ? ids[r] : r;
      if (at >= 0 && at < s.n) acc = fmaf(v, to_f(x[at * s.K + k]), acc);
    }
    if (k < s.K) {
      if (vw) vw[((int64_t)g * s.M + m) * s.K + k] = from_f<T>(acc);
    } else if (vb) {
      vb[(int64_t)g * s.M + m] = from_f<T>(acc);
    }
  }
}

__global__ void __launch_bounds__(256) offsets_kernel(int64_t n, const int32_t* __restrict__ ids,
                                                      int G, int32_t* __restrict__ off) {
  for (int g = blockIdx.x * blockDim.x + threadIdx.x; g <= G; g += gridDim.x * blockDim.x) {
    int64_t lo = 0, hi = n;  // ids below g end in [lo, hi]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (__ldg(ids + mid) < g) lo = mid + 1; else hi = mid;
    }
    off[g] = (int32_t)lo;
  }
}

template <typename T, int ACT>
int run_fwd(const Shape& s, const void* x, const int32_t* ids, const int32_t* off, const void* w,
            const void* b, void* y, cudaStream_t st) {
  fwd_kernel<T, ACT><<<grid_for(s.R * s.M, 256), 256, 0, st>>>(
      s, static_cast<const T*>(x), ids, off, static_cast<const T*>(w), static_cast<const T*>(b),
      static_cast<T*>(y));
  return launch_status("grouped_linear_fwd");
}

template <typename T, int ACT>
int run_bwd(const Shape& s, bool shared, const void* x, const int32_t* ids, const int32_t* off, const void* w,
            const void* y, const void* vy, void* vx, void* vw, void* vb, void* ws,
            cudaStream_t st) {
  if (vx) {
    float* sum = sizeof(T) == 4 ? static_cast<float*>(vx) : static_cast<float*>(ws);
    if (shared && cudaMemsetAsync(sum, 0, sizeof(float) * s.n * s.K, st) != cudaSuccess)
      return launch_status("grouped_linear_bwd");
    if (s.R > 0)
      bwd_x_kernel<T, ACT><<<grid_for(s.R * s.K, 256), 256, 0, st>>>(
          s, ids, off, static_cast<const T*>(w), static_cast<const T*>(y),
          static_cast<const T*>(vy), sum, static_cast<T*>(vx));
    if (shared && sizeof(T) == 2 && s.n > 0)
      round_kernel<T><<<grid_for(s.n * s.K, 256), 256, 0, st>>>(s.n * s.K, sum,
                                                                static_cast<T*>(vx));
  }
  if (vw || vb)
    bwd_w_kernel<T, ACT><<<grid_for((int64_t)s.G * s.M * (s.K + 1), 256), 256, 0, st>>>(
        s, static_cast<const T*>(x), ids, off, static_cast<const T*>(y),
        static_cast<const T*>(vy), static_cast<T*>(vw), static_cast<T*>(vb));
  return launch_status("grouped_linear_bwd");
}

// Calls f<T, ACT>(args...) for the params' dtype and activation.
#define GROUPED_DISPATCH(p, f, ...)                                                    \
  switch ((p)->dtype * 3 + (p)->activation) {                                          \
    case 0: return f<float, GS_ACT_NONE>(__VA_ARGS__);                                 \
    case 1: return f<float, GS_ACT_RELU>(__VA_ARGS__);                                 \
    case 2: return f<float, GS_ACT_SIGMOID>(__VA_ARGS__);                              \
    case 3: return f<__nv_bfloat16, GS_ACT_NONE>(__VA_ARGS__);                         \
    case 4: return f<__nv_bfloat16, GS_ACT_RELU>(__VA_ARGS__);                         \
    case 5: return f<__nv_bfloat16, GS_ACT_SIGMOID>(__VA_ARGS__);                      \
    case 6: return f<__half, GS_ACT_NONE>(__VA_ARGS__);                                \
    case 7: return f<__half, GS_ACT_RELU>(__VA_ARGS__);                                \
    default: return f<__half, GS_ACT_SIGMOID>(__VA_ARGS__);                            \
  }

int bad_params(const gs_grouped_params* p) {
  if (!p || p->rows < 0 || p->n < 0 || p->groups < 1 || p->in_features < 1 ||
      p->out_features < 1)
    return invalid("grouped_linear: bad params");
  if (p->rows >= INT32_MAX || p->n >= INT32_MAX)
    return invalid("grouped_linear: 2^31 rows or more");
  if (!p->use_row_ids && p->n != p->rows)
    return invalid("grouped_linear: x has another number of rows");
  if (p->dtype < GS_F32 || p->dtype > GS_F16) return invalid("grouped_linear: unknown dtype");
  if (p->activation < GS_ACT_NONE || p->activation > GS_ACT_SIGMOID)
    return invalid("grouped_linear: unknown activation");
  return GS_OK;
}

}  // namespace
}  // namespace gsb

using namespace gsb;

extern "C" int gs_group_offsets(int64_t n, const int32_t* sorted_ids, int32_t groups,
                                int32_t* offsets, gs_stream_t stream) {
  if (n < 0 || n >= INT32_MAX || groups < 0 || groups == INT32_MAX)
    return invalid("group_offsets: bad size");
  if ((n > 0 && !sorted_ids) || !offsets) return invalid("group_offsets: missing buffer");
  offsets_kernel<<<grid_for((int64_t)groups + 1, 256), 256, 0, as_stream(stream)>>>(
      n, sorted_ids, groups, offsets);
  return launch_status("group_offsets");
}

extern "C" int gs_grouped_linear_fwd(const gs_grouped_params* p, const void* x,
                                     const int32_t* row_ids, const int32_t* offsets,
                                     const void* weights, const void* biases, void* y,
                                     gs_stream_t stream) {
  if (int rc = bad_params(p)) return rc;
  if (p->rows == 0) return GS_OK;
  if ((p->n > 0 && !x) || !offsets || !weights || !y || (p->use_row_ids && !row_ids))
    return invalid("grouped_linear: missing buffer");
  if (!p->use_row_ids) row_ids = nullptr;
  const Shape s{p->rows, p->n, p->groups, p->in_features, p->out_features};
  GROUPED_DISPATCH(p, run_fwd, s, x, row_ids, offsets, weights, biases, y, as_stream(stream));
}

extern "C" size_t gs_grouped_linear_bwd_workspace_size(const gs_grouped_params* p) {
  if (bad_params(p) != GS_OK) return 0;
  return p->use_row_ids && p->dtype != GS_F32 ? sizeof(float) * (size_t)p->n * p->in_features : 0;
}

extern "C" int gs_grouped_linear_bwd(const gs_grouped_params* p, const void* x,
                                     const int32_t* row_ids, const int32_t* offsets,
                                     const void* weights, const void* y, const void* v_y,
                                     void* v_x, void* v_weights, void* v_biases, void* workspace,
                                     size_t workspace_bytes, gs_stream_t stream) {
  if (int rc = bad_params(p)) return rc;
  if (!v_x && !v_weights && !v_biases) return GS_OK;
  if (!offsets || !weights || (p->n > 0 && !x) ||
      (p->rows > 0 && (!v_y || (p->activation != GS_ACT_NONE && !y) ||
                       (p->use_row_ids && !row_ids))))
    return invalid("grouped_linear: missing buffer");
  const size_t need = gs_grouped_linear_bwd_workspace_size(p);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    set_error("grouped_linear: workspace of %zu bytes needed", need);
    return GS_ERR_WORKSPACE;
  }
  if (!p->use_row_ids) row_ids = nullptr;
  const Shape s{p->rows, p->n, p->groups, p->in_features, p->out_features};
  GROUPED_DISPATCH(p, run_bwd, s, p->use_row_ids != 0, x, row_ids, offsets, weights, y, v_y, v_x, v_weights, v_biases,
                   workspace, as_stream(stream));
}
