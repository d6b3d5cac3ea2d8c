// Entries of the grouped products (the kernels: grouped_kernels.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cstring>
#include <mutex>

#include "grouped.cuh"

namespace gsb {
namespace grouped {

Plan plan_of(const gs_grouped_params* p) {  // one CTA an SM, or two
  Plan q;
  const int wanted = p->wanted ? p->wanted : GS_WANT_V_X | GS_WANT_V_WEIGHTS | GS_WANT_V_BIASES;
  const bool sums = wanted & (GS_WANT_V_WEIGHTS | GS_WANT_V_BIASES);
  q.nt = p->out_features > 64 ? 128 : 64;
  q.kt = (int)ceil_div(p->in_features, 128);
  q.mt = (int)ceil_div(p->out_features, q.nt);
  const int64_t tiles = ceil_div(p->rows, kTile);
  q.narrow = is_narrow(p->in_features, p->out_features, p->dtype, true);
  // Rows of 16-bit values that are no whole chunks: a copy of them costs a
  // fraction of what taking them apart by single values does (200 k rows 77-45:
  // 223 -> 96 us).
  q.kp = p->in_features, q.mp = p->out_features;
  const int k8 = (int)ceil_div(q.kp, 8) * 8, m8 = (int)ceil_div(q.mp, 8) * 8;
  q.padded = p->dtype != GS_F32 && p->n > 0 && !q.narrow && !dims_fit_both(q.kp, q.mp) &&
             dims_fit_both(k8, m8);
  if (q.padded) q.kp = k8, q.mp = m8;
  const bool two = q.narrow || (p->dtype != GS_F32 && !dims_fit_both(q.kp, q.mp));
  int64_t n = (int64_t)sm_count() * (two ? 2 : 1) / ((int64_t)q.kt * q.mt);
  n = n < 1 ? 1 : n > tiles ? tiles : n;
  q.parts = (int)n;
  q.copies = p->dtype == GS_F32 && !q.narrow ? kBiasCopies32 : 1;
  q.part_floats = sums ? ((size_t)q.parts + p->groups) * q.mp * ((size_t)q.kp + q.copies) : 0;
  q.sum_floats = wanted & GS_WANT_V_X && p->use_row_ids && p->dtype != GS_F32
                     ? (size_t)p->n * p->in_features : 0;
  q.part_floats = (q.part_floats + 63) / 64 * 64;  // the sums start on 256 bytes
  q.sum_floats = (q.sum_floats + 63) / 64 * 64;
  const bool copies = q.padded && sums;
  q.pad_x = copies ? (size_t)p->n * q.kp : 0;
  q.pad_w = copies ? (size_t)p->groups * q.mp * q.kp : 0;
  q.pad_v = copies ? (size_t)p->rows * q.mp : 0;
  return q;
}

namespace {

__global__ void __launch_bounds__(256) offsets_kernel(int64_t n, const int32_t* __restrict__ ids,
                                                      int G, int32_t* __restrict__ off) {
  for (int64_t g = blockIdx.x * blockDim.x + threadIdx.x; g <= G;
       g += gridDim.x * blockDim.x) {  // past 2^31 where G is next to it
    int64_t lo = 0, hi = n;  // ids below g end in [lo, hi]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (__ldg(ids + mid) < g) lo = mid + 1; else hi = mid;
    }
    off[g] = (int32_t)lo;
  }
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// f of a value of the params' type.
template <typename F>
int by_type(int dtype, F f) {
  return dtype == GS_F32 ? f(float()) : dtype == GS_BF16 ? f(__nv_bfloat16()) : f(__half());
}

// The word of the current device that says that a wait of a call without a word of
// its own gave up: in pinned host memory, so that the host reads it without
// waiting for the device.
int device_word(uint32_t** word) {
  static std::mutex mutex;
  static uint32_t* words = nullptr;  // a cache line for each device
  constexpr int kDevices = 64, kApart = 32;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return launch_status("grouped_linear");
  if (dev < 0 || dev >= kDevices) return invalid("grouped_linear: device index past 63");
  std::lock_guard<std::mutex> lock(mutex);
  if (!words) {
    // the current stream may be recording a graph, of which this is no part
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    void* p = nullptr;
    const cudaError_t e = cudaHostAlloc(&p, kDevices * kApart * sizeof(uint32_t),
                                        cudaHostAllocPortable | cudaHostAllocMapped);
    cudaThreadExchangeStreamCaptureMode(&mode);
    if (e != cudaSuccess) return launch_status("grouped_linear");
    std::memset(p, 0, kDevices * kApart * sizeof(uint32_t));
    words = static_cast<uint32_t*>(p);
  }
  *word = words + dev * kApart;
  return GS_OK;
}

int gave_up(const char* more) {
  set_error("grouped_linear: a wait inside a kernel gave up: its call's results are void%s", more);
  return GS_ERR_DEVICE;
}

// Where a call's waits report to, and how long they are.
int waits_of(const gs_grouped_params* p, WaitArgs* w) {
  w->limit = p->wait_selftest ? 0 : kWaitLimit;
  w->status = p->status;
  if (p->status) return GS_OK;
  if (int rc = device_word(&w->status)) return rc;
  return __atomic_load_n(w->status, __ATOMIC_ACQUIRE)
             ? gave_up("; refused until gs_grouped_linear_check has reported it") : GS_OK;
}

// Rows are counted in 32 bits, some tiles past the last.
constexpr int64_t kRowsMost = INT32_MAX - 4096;
constexpr int32_t kFeaturesMost = 16384;  // 128 x 256 tiles of weights: a grid's second side

int bad_params(const gs_grouped_params* p) {
  if (!p || p->rows < 0 || p->n < 0 || p->groups < 1 || p->in_features < 1 ||
      p->out_features < 1)
    return invalid("grouped_linear: bad params");
  if (p->groups == INT32_MAX) return invalid("grouped_linear: 2^31 - 1 groups or more");
  if (p->rows > kRowsMost || p->n > kRowsMost)
    return invalid("grouped_linear: 2^31 - 4096 rows or more");
  if (!p->use_row_ids && p->n != p->rows)
    return invalid("grouped_linear: x has another number of rows");
  if (p->in_features > kFeaturesMost || p->out_features > kFeaturesMost)
    return invalid("grouped_linear: more than 16384 features");
  if (p->dtype < GS_F32 || p->dtype > GS_F16) return invalid("grouped_linear: unknown dtype");
  if (p->activation < GS_ACT_NONE || p->activation > GS_ACT_SIGMOID)
    return invalid("grouped_linear: unknown activation");
  if (p->wanted & ~(GS_WANT_V_X | GS_WANT_V_WEIGHTS | GS_WANT_V_BIASES))
    return invalid("grouped_linear: unknown gradient wanted");
  return GS_OK;
}

}  // namespace
}  // namespace grouped
}  // namespace gsb

using namespace gsb;
using namespace gsb::grouped;

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
  WaitArgs waits;
  if (int rc = waits_of(p, &waits)) return rc;
  cudaStream_t st = as_stream(stream);
  return by_type(p->dtype, [&](auto type) {
    return forward<decltype(type)>(p->activation, s, waits, x, row_ids, offsets, weights, biases, y,
                                   st);
  });
}

extern "C" size_t gs_grouped_linear_bwd_workspace_size(const gs_grouped_params* p) {
  if (bad_params(p) != GS_OK) return 0;
  const Plan q = plan_of(p);
  return sizeof(float) * (q.part_floats + q.sum_floats) +
         2 * (q.pad_x + q.pad_w + q.pad_v * (p->activation == GS_ACT_NONE ? 1 : 2));
}

extern "C" int gs_grouped_linear_bwd(const gs_grouped_params* p, const void* x,
                                     const int32_t* row_ids, const int32_t* offsets,
                                     const void* weights, const void* y, const void* v_y,
                                     void* v_x, void* v_weights, void* v_biases, void* workspace,
                                     size_t workspace_bytes, gs_stream_t stream) {
  if (int rc = bad_params(p)) return rc;
  if (!v_x && !v_weights && !v_biases) return GS_OK;
  const int given = (v_x ? GS_WANT_V_X : 0) | (v_weights ? GS_WANT_V_WEIGHTS : 0) |
                    (v_biases ? GS_WANT_V_BIASES : 0);
  if (p->wanted && given & ~p->wanted)
    return invalid("grouped_linear: a gradient that wanted does not name");
  if (!offsets || !weights || (p->n > 0 && !x) ||
      (p->rows > 0 && (!v_y || (p->activation != GS_ACT_NONE && !y) ||
                       (p->use_row_ids && !row_ids))))
    return invalid("grouped_linear: missing buffer");
  const size_t need = gs_grouped_linear_bwd_workspace_size(p);
  if (need > 0 && (!workspace || workspace_bytes < need || !on16(workspace))) {
    set_error("grouped_linear: a workspace of %zu bytes on a 16-byte boundary is needed", need);
    return GS_ERR_WORKSPACE;
  }
  if (!p->use_row_ids) row_ids = nullptr;
  const Shape s{p->rows, p->n, p->groups, p->in_features, p->out_features};
  WaitArgs waits;
  if (int rc = waits_of(p, &waits)) return rc;
  cudaStream_t st = as_stream(stream);
  return by_type(p->dtype, [&](auto type) {
    return backward<decltype(type)>(p, s, waits, x, row_ids, offsets, weights, y, v_y, v_x,
                                    v_weights, v_biases, static_cast<float*>(workspace), st);
  });
}

extern "C" int gs_grouped_linear_check(gs_stream_t stream) {
  if (cudaStreamSynchronize(as_stream(stream)) != cudaSuccess)
    return launch_status("grouped_linear_check");
  uint32_t* word = nullptr;
  if (int rc = device_word(&word)) return rc;
  if (!__atomic_exchange_n(word, 0u, __ATOMIC_ACQ_REL)) return GS_OK;
  return gave_up("");
}
