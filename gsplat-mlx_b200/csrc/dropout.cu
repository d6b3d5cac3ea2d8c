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
// HBM-bound: x read once (dropped rows not at all), y written once, 16 bytes a
// thread and access.  Of copy bandwidth (6548 GB/s measured): whole rows of 48
// fp32 values, 3 M of them, 160 us, 6.49 TB/s; single bf16 values, 128 M of
// them, 84 us, 6.07 TB/s (14.7 instructions a value, the multiply and the
// logic pipes at 60% each: the generator costs 28 of the ~59 of four values),
// and 31 us, 5.3 TB/s for 40 M, where the ramp shows.
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
  uint32_t threshold;   // p 2^32: a word below it drops
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

__device__ __forceinline__ uint32_t keep_bits(const uint4& w, uint32_t t) {
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

// N values at p as one access of N sizeof(T) bytes (1 to 16).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T>
__device__ __forceinline__ T dropped(T x, bool keep, float scale) {
  return keep ? from_f<T>(to_f(x) * scale) : from_f<T>(0.0f);
}

// A decision per value (or rows of one value): a thread takes 16 bytes at a
// time, kUnroll times a block's width apart, all loaded before the first is
// used (twice instead of four times: 33 against 31 us at 37 M fp16 values).
// E = 1 is for buffers that do not start on 16 bytes.
constexpr int kUnroll = 4;

// Two values at a time: the 16-bit types convert in pairs.
__device__ __forceinline__ float2 pair_f(const float* v) { return make_float2(v[0], v[1]); }
__device__ __forceinline__ float2 pair_f(const __nv_bfloat16* v) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v));
}
__device__ __forceinline__ float2 pair_f(const __half* v) {
  return __half22float2(*reinterpret_cast<const __half2*>(v));
}
__device__ __forceinline__ void set_pair(float* v, float a, float b) { v[0] = a, v[1] = b; }
__device__ __forceinline__ void set_pair(__nv_bfloat16* v, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(v) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void set_pair(__half* v, float a, float b) {
  *reinterpret_cast<__half2*>(v) = __floats2half2_rn(a, b);
}

template <typename T, int W>
__device__ __forceinline__ void drop_pack(Pack<T, W>& v, uint64_t block, uint64_t step,
                                          const Draw& d) {
#pragma unroll
  for (int q = 0; q < W / 4; ++q) {
    const uint4 w = philox7(block + q, step, d.k0, d.k1);
    const float2 a = pair_f(&v.v[q * 4]), b = pair_f(&v.v[q * 4 + 2]);
    set_pair(&v.v[q * 4], w.x >= d.threshold ? a.x * d.scale : 0.0f,
             w.y >= d.threshold ? a.y * d.scale : 0.0f);
    set_pair(&v.v[q * 4 + 2], w.z >= d.threshold ? b.x * d.scale : 0.0f,
             w.w >= d.threshold ? b.y * d.scale : 0.0f);
  }
}

template <typename T, int E>
__global__ void __launch_bounds__(256) values_kernel(int64_t total, Draw d, const T* x, T* y) {
  const uint64_t step = draw_step(d);
  // E >= 4: packs of E; E == 1: four single values of one generator call
  constexpr int W = E >= 4 ? E : 4;
  const int64_t base = (int64_t)blockIdx.x * (256 * kUnroll * W);
  Pack<T, W> in[kUnroll];
  if (E >= 4 && base + 256 * kUnroll * W <= total) {
    const int64_t i = base + threadIdx.x * W;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      in[u] = *reinterpret_cast<const Pack<T, W>*>(x + i + u * 256 * W);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      drop_pack<T, W>(in[u], (uint64_t)(i + u * 256 * W) / 4, step, d);
      *reinterpret_cast<Pack<T, W>*>(y + i + u * 256 * W) = in[u];
    }
    return;
  }
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t i = base + (int64_t)(u * 256 + threadIdx.x) * W;
    if (i >= total) return;
    const int n = (int)min((int64_t)W, total - i);
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < n) in[0].v[e] = x[i + e];
    drop_pack<T, W>(in[0], (uint64_t)i / 4, step, d);
#pragma unroll
    for (int e = 0; e < W; ++e)
      if (e < n) y[i + e] = in[0].v[e];
  }
}

// A decision per row.  A warp draws the 128 decisions of a block of rows with
// one generator call per lane and holds them as four ballots; it then streams
// one part of the block's values (kUnroll2 packs a lane), reading only packs
// that keep something.  STRADDLE: packs may lie across rows (width not a
// multiple of E).
constexpr int kUnroll2 = 8;

template <typename T, int E, bool STRADDLE>
__global__ void __launch_bounds__(256) rows_kernel(int64_t rows, uint32_t width, uint32_t parts,
                                                   Draw d, const T* x, T* y) {
  const int lane = threadIdx.x & 31;
  const int64_t warp = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int64_t block = warp / parts;
  const uint32_t part = (uint32_t)(warp - block * parts);
  const int64_t row0 = block * 128;
  if (row0 >= rows) return;
  const uint32_t keep4 =
      keep_bits(philox7((uint64_t)row0 / 4 + lane, draw_step(d), d.k0, d.k1), d.threshold);
  uint32_t keep[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) keep[i] = __ballot_sync(0xffffffffu, (keep4 >> i) & 1);
  auto kept = [&](uint32_t r) {  // row row0 + r
    const uint32_t a = r & 1 ? keep[1] : keep[0], b = r & 1 ? keep[3] : keep[2];
    return ((r & 2 ? b : a) >> ((r >> 2) & 31)) & 1;
  };
  const uint32_t values = (uint32_t)min((int64_t)128, rows - row0) * width;  // below 2^31
  x += row0 * width;
  y += row0 * width;
  const uint32_t at = (part * kUnroll2 * 32 + lane) * E;
  Pack<T, E> in[kUnroll2];
  uint32_t bits[kUnroll2];
#pragma unroll
  for (int u = 0; u < kUnroll2; ++u) {
    const uint32_t i = at + u * 32 * E;
    bits[u] = 0;
    if (i >= values) continue;
    uint32_t r = i / width;
    if (!STRADDLE) {
      bits[u] = kept(r) ? (1u << E) - 1 : 0;
    } else {
      uint32_t c = i - r * width;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        bits[u] |= kept(r) << e;
        if (++c == width) c = 0, ++r;
      }
    }
    if (i + E <= values) {
      if (bits[u]) in[u] = *reinterpret_cast<const Pack<T, E>*>(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < values) in[u].v[e] = x[i + e];
    }
  }
#pragma unroll
  for (int u = 0; u < kUnroll2; ++u) {
    const uint32_t i = at + u * 32 * E;
    if (i >= values) break;
#pragma unroll
    for (int e = 0; e < E; ++e)
      in[u].v[e] = dropped(in[u].v[e], (bits[u] >> e) & 1, d.scale);
    if (i + E <= values) {
      *reinterpret_cast<Pack<T, E>*>(y + i) = in[u];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < values) y[i + e] = in[u].v[e];
    }
  }
}

template <typename T, int E>
int launch_as(const gs_dropout_params& p, const Draw& d, const T* x, T* y, cudaStream_t s) {
  if (!p.by_row || p.width == 1) {
    const int64_t total = p.rows * p.width;
    const int64_t blocks = ceil_div(total, 256 * kUnroll * (E >= 4 ? E : 4));
    if (blocks > INT32_MAX) return invalid("dropout: rows * width too large");
    values_kernel<T, E><<<(unsigned)blocks, 256, 0, s>>>(total, d, x, y);
  } else {
    const int64_t parts = ceil_div(128 * p.width, 32 * kUnroll2 * E);
    const int64_t blocks = ceil_div(ceil_div(p.rows, 128) * parts, 8);
    if (blocks > INT32_MAX) return invalid("dropout: rows * width too large");
    if (p.width % E == 0)
      rows_kernel<T, E, false><<<(unsigned)blocks, 256, 0, s>>>(p.rows, (uint32_t)p.width,
                                                                (uint32_t)parts, d, x, y);
    else
      rows_kernel<T, E, true><<<(unsigned)blocks, 256, 0, s>>>(p.rows, (uint32_t)p.width,
                                                               (uint32_t)parts, d, x, y);
  }
  return launch_status("dropout");
}

template <typename T>
int launch(const gs_dropout_params& p, const Draw& d, const void* x, void* y, cudaStream_t s) {
  const bool wide = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
  const T* xt = static_cast<const T*>(x);
  T* yt = static_cast<T*>(y);
  return wide ? launch_as<T, 16 / sizeof(T)>(p, d, xt, yt, s) : launch_as<T, 1>(p, d, xt, yt, s);
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
  cudaStream_t s = as_stream(stream);
  const double threshold = std::nearbyint(p->p * 4294967296.0);
  if (threshold >= 4294967296.0) {  // no word reaches it: everything is dropped
    const size_t size = (p->dtype == GS_F32 ? 4 : 2) * (size_t)(p->rows * p->width);
    if (cudaMemsetAsync(y, 0, size, s) != cudaSuccess) return launch_status("dropout");
    return GS_OK;
  }
  d.threshold = static_cast<uint32_t>(threshold);
  d.scale = static_cast<float>(1.0 / (1.0 - p->p));
  if (p->dtype == GS_F32) return launch<float>(*p, d, x, y, s);
  if (p->dtype == GS_BF16) return launch<__nv_bfloat16>(*p, d, x, y, s);
  return launch<__half>(*p, d, x, y, s);
}
