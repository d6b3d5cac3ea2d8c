// What the grouped products' entries (grouped.cu) and their kernels for each
// type (grouped_kernels.cuh) share.
#pragma once

#include "common.cuh"

namespace gsb {
namespace grouped {

struct Shape {
  int64_t R, n;
  int G, K, M;
};

constexpr int kTile = 128;        // rows of a tile: the lanes of an accumulator
constexpr int kBiasCopies32 = 4;  // partial sums of v_b: front groups x halves

constexpr uint32_t kWaitLimit = 1u << 18;  // polls of 4 us: a second
struct WaitArgs {
  uint32_t limit;
  uint32_t* status;
};

// Few outputs of rows of up to 32 chunks; the backward has to hold a lane's
// weights and sums in registers.
inline bool is_narrow(int K, int M, int dtype, bool backward) {
  const int e = dtype == GS_F32 ? 4 : 8;
  return M <= (backward && dtype != GS_F32 ? 4 : 8) && K <= 32 * e;
}

inline bool dims_fit_both(int K, int M) { return K <= 128 && M <= 128 && K % 8 == 0 && M % 8 == 0; }

// The backward's launches and its scratch: parts of the weight sums, then
// the fp32 sums of shared rows for the 16-bit types.
struct Plan {
  int nt, kt, mt, parts;
  int copies;  // of v_b's sums in a place
  bool narrow;
  bool padded;  // 16-bit rows are copied to whole chunks first
  int kp, mp;   // K and M as the kernels see them
  size_t part_floats, sum_floats;
  size_t pad_x, pad_w, pad_v;  // 16-bit values of the copies
};

Plan plan_of(const gs_grouped_params* p);

// The forward, and the backward with its join, of one type; activation is the
// params'.
template <typename T>
int forward(int activation, const Shape& s, const WaitArgs& waits, const void* x,
            const int32_t* ids, const int32_t* off, const void* w, const void* b, void* y,
            cudaStream_t st);
template <typename T>
int backward(const gs_grouped_params* prm, const Shape& s, const WaitArgs& waits, const void* x,
             const int32_t* ids, const int32_t* off, const void* w, const void* y, const void* vy,
             void* vx, void* vw, void* vb, float* ws, cudaStream_t st);

}  // namespace grouped
}  // namespace gsb
