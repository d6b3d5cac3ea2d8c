// Products of ragged groups of rows with one weight matrix per group (a
// learned layer per camera over the packed rows, which are sorted by camera):
//
//   y[r]   = act(W[g] x[id(r)] + b[g])           off[g] <= r < off[g + 1]
//   v_z[r] = v_y[r] act'(y[r])
//   v_x[id(r)] += W[g]^T v_z[r],  v_W[g] = sum v_z[r] x[id(r)]^T,  v_b[g] = sum v_z[r]
//
// A row's group is found by a search over the offsets whose invariant
// off[g] <= r < off[g + 1] holds for the pair that it ends at even where the
// offsets do not ascend, so every run of rows has one row at least and no
// index leaves its buffer.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <type_traits>

#include "grouped.cuh"
#include "tcgen05.cuh"

namespace gsb {
namespace grouped {
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

// The group of row r: -1 in front of the first, G behind the last.  Called by
// whole warps with the same r: a step of the search looks at 32 places.
__device__ __forceinline__ int group_of(const int32_t* __restrict__ off, int G, int r) {
  const int lane = threadIdx.x & 31;
  const int first = __ldg(off), last = __ldg(off + G);
  uint32_t lo = 0, hi = G;  // off[lo] <= r < off[hi]
  while (hi - lo > 1) {
    const uint32_t step = (hi - lo + 31) / 32, at = lo + lane * step;  // up to 2^31 + 30
    const uint32_t below = __ballot_sync(0xffffffffu, at < hi && __ldg(off + at) <= r);
    // the places where the row is above one and below the next
    const int i = below == 0xffffffffu ? 31 : max(__ffs(~below) - 2, 0);
    lo += i * step;
    hi = min(hi, lo + step);
  }
  return r < first ? -1 : r >= last ? G : (int)lo;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
  if (ACT == GS_ACT_RELU) {  // NaN passes
    float r;
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(z));
    return r;
  }
  if (ACT == GS_ACT_SIGMOID) return __fdividef(1.0f, 1.0f + expf(-z));
  return z;
}
// v_z from v and the activated y
template <int ACT>
__device__ __forceinline__ float through(float v, float y) {
  if (ACT == GS_ACT_RELU) return y > 0.0f ? v : 0.0f;
  if (ACT == GS_ACT_SIGMOID) return v * y * (1.0f - y);
  return v;
}

// ------------------------------------------------------------ tensor-core tiles
//
// Operands in 16 bits go to the tensor core as they are.  An fp32 value goes
// as two tf32 parts, x = hi + lo to 2^-22 |x|; the products hi hi are summed
// in one accumulator and the three others in a second, which are added in
// fp32 when the sum is read.  A product is off by up to 3 2^-22: sums of a few are
// off by two to three times what fp32 multiply-adds would be, longer ones by
// no more.  (A NaN all of whose payload lies in the 13 low bits counts as an
// infinity.)  Where the first accumulator is not finite it is the result: the
// second has inf - inf and inf * 0 there, and is not finite only where the first is
// not.  v_z of the sigmoid in 16 bits goes as two parts in the same manner, so that it is not
// rounded to 16 bits on its way.  fp16 ends at 2^-24, next to the gradients of a
// mean over an image, so its second part is held times 2^11 (it is at most 2^4:
// half a step of the first) and what it gives is scaled back where the sums are
// joined: v_z is carried to 2^-22 of itself and to 2^-36.  bf16 has fp32's range.
//
// Waits are for the CTA's own copies, MMAs and warps, and are bounded.  A warp
// whose wait gives up says so in *status and to the CTA's other warps, which
// then give up their next wait that does not end at once.  From then on it sends
// no copies, issues no MMAs and arrives nowhere, so that no barrier moves on by
// what was not done: it leaves its loops, or walks on to the named barriers at
// which other warps meet it.  Whoever sent bulk copies or MMAs waits for those
// (with a limit of its own) before the CTA gives its memory back.  The results
// are void.  A test sets the limit to 0: then the barriers of what arrives expect
// one arrival that nobody makes.
constexpr uint32_t kDrainLimit = 1u << 12;  // for what takes microseconds

// False for the whole warp where the wait gave up.
__device__ __forceinline__ bool waited(uint32_t bar, uint32_t parity, const WaitArgs& p,
                                       uint32_t* stop) {
  if (tc::bar_wait(bar, parity & 1, p.limit, stop)) return true;
  *static_cast<volatile uint32_t*>(stop) = 1;
  *static_cast<volatile uint32_t*>(p.status) = 1;
  return false;
}
// A wait of a role that leaves its loops where one gives up.
#define WAIT_OR(done, bar, parity) \
  if (!waited(bar, parity, p.waits, &s_stop)) goto done

__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  tc::bar_wait(bar, parity & 1, kDrainLimit, nullptr);
}
// The last of `sent` copies into a ring of slots, those that may be under way.
template <typename Full>
__device__ __forceinline__ void drain_ring(int sent, int slots, Full full) {
  for (int i = max(sent - slots, 0); i < sent; ++i) drain(full(i % slots), i / slots);
}

template <typename T> struct Mma;
template <> struct Mma<float> {
  static constexpr bool TF32 = true;
  static constexpr uint32_t format = tc::kTF32;
};
template <> struct Mma<__nv_bfloat16> {
  static constexpr bool TF32 = false;
  static constexpr uint32_t format = tc::kBF16;
};
template <> struct Mma<__half> {
  static constexpr bool TF32 = false;
  static constexpr uint32_t format = tc::kF16;
};

constexpr int kThreads = 256;
constexpr int kPanel = kTile * 128;  // bytes of 128 operand rows, 128 bytes deep
constexpr int kSlotsMost = 6;        // panels of a ring

// The values of one 16-byte chunk.
template <typename T>
union Chunk {
  static constexpr int E = 16 / sizeof(T);
  uint4 q;
  T v[E];
  __device__ Chunk() {}
};

// Where chunk c of operand row r lies in its panel.
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
}

// What the second part of a value in 16 bits is held times.
template <typename T> constexpr float kLowScale = 1.0f;
template <> constexpr float kLowScale<__half> = 2048.0f;

// Sums of the first parts joined with those of the second.
template <typename T>
__device__ __forceinline__ void join_parts(float (&v)[16], const float (&u)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (fabsf(v[i]) < INFINITY) v[i] = fmaf(u[i], 1.0f / kLowScale<T>, v[i]);
}

// Writes f[0..E) as one operand chunk: one part, or two at a panel's distance.
template <typename T, bool SPLIT>
__device__ __forceinline__ void put_chunk(char* at, ptrdiff_t lo_offset, const float* f) {
  Chunk<T> hi, lo;
#pragma unroll
  for (int e = 0; e < Chunk<T>::E; ++e) {
    hi.v[e] = from_f<T>(f[e]);
    if (SPLIT && sizeof(T) == 2) lo.v[e] = from_f<T>((f[e] - to_f(hi.v[e])) * kLowScale<T>);
  }
  *reinterpret_cast<uint4*>(at) = hi.q;
  if constexpr (sizeof(T) == 4) put_low(at + lo_offset, hi);
  else if (SPLIT) *reinterpret_cast<uint4*>(at + lo_offset) = lo.q;
}

// The low part of a chunk of fp32 operands whose upper parts the tensor core
// takes from the values themselves: x without its 13 low bits; the rest is
// exact, has 13 bits, and is rounded to the 11 of a tf32 operand (the
// addition; the bits behind are ignored), which leaves 2^-22 |x|.
__device__ __forceinline__ void put_low(char* at, const Chunk<float>& x) {
  Chunk<float> lo;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float hi = __uint_as_float(__float_as_uint(x.v[e]) & 0xFFFFE000u);
    lo.v[e] = __uint_as_float(__float_as_uint(x.v[e] - hi) + 0x1000u);
  }
  *reinterpret_cast<uint4*>(at) = lo.q;
}

// E values from p: one access, or one by one where p is not aligned or fewer
// than E are there.  What is not there is zero.
template <typename T, bool WIDE>
__device__ __forceinline__ uint4 get_chunk(const T* __restrict__ p, int there) {
  Chunk<T> c;
  if (WIDE) {
    c.q = there > 0 ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0, 0, 0, 0);
  } else {
#pragma unroll
    for (int e = 0; e < Chunk<T>::E; ++e) c.v[e] = e < there ? p[e] : from_f<T>(0.0f);
  }
  return c.q;
}

// The place of a ring of buffers that is next, and how often it went round:
// the phase of the place's barriers.
struct Ring {
  int slots, slot, turn;
  __device__ __forceinline__ explicit Ring(int n) : slots(n), slot(0), turn(0) {}
  __device__ __forceinline__ void next() {
    if (++slot == slots) slot = 0, ++turn;
  }
  // the place `n` <= slots before, and its last phase
  __device__ __forceinline__ int slot_before(int n) const {
    return slot >= n ? slot - n : slot - n + slots;
  }
  __device__ __forceinline__ int turn_before(int n) const { return slot >= n ? turn : turn - 1; }
};

// Consecutive rows of one group, at most `most` of them, up to `end`.
struct Run {
  int row;
  int n;      // 0: no rows are left
  int g;      // -1 or G: outside every group
  int group_end;
};

__device__ __forceinline__ Run run_from(const int32_t* __restrict__ off, int G, int row, int end,
                                        int most, Run prev) {
  Run t;
  t.row = row;
  t.g = prev.g;
  t.group_end = prev.group_end;
  if (row >= end) {
    t.n = 0;
    return t;
  }
  if (row >= t.group_end) {
    t.g = group_of(off, G, row);
    const int stop = t.g < 0 ? __ldg(off) : t.g < G ? __ldg(off + t.g + 1) : end;
    t.group_end = min(stop, end);
  }
  t.n = min(most, t.group_end - row);
  return t;
}

// The tiles of kTile rows are dealt to `parts` CTAs in order: CTA b has the
// tiles [T b / parts, T (b + 1) / parts).
__host__ __device__ __forceinline__ int64_t first_tile(int64_t tiles, int parts, int b) {
  return tiles * b / parts;
}

struct RowsArgs {
  Shape s;                 // R, n, G and K, M as the caller gave them
  const void* a;           // rows that are multiplied: x, or v_y
  const void* y;           // backward through an activation
  const int32_t* ids;
  const int32_t* off;
  const void* w;
  const void* bias;
  void* out;
  int depth, width;        // K, M; the backward's M, K
  int nt;                  // columns of a CTA's tile: a multiple of 32
  int panels;              // of `depth`
  int resident;            // all weight panels of the tile stay in shared memory
  int slots;               // panels of rows that are in flight or in use
  int wide_w, wide_out;    // 16-byte accesses are aligned
  WaitArgs waits;
};

enum { kForward, kBackward, kScatter };

template <typename T, int ACT, int MODE, bool SPLIT>
struct RowsLayout {
  static constexpr bool kY = MODE != kForward && ACT != GS_ACT_NONE;  // y is read too
  static constexpr int kTerms = SPLIT || sizeof(T) == 4 ? 2 : 1;      // parts of a row value
  static constexpr int kWTerms = sizeof(T) == 4 ? 2 : 1;              // of a weight
  // low parts of two panels; with y they take the place of the panel's y
  static constexpr int kLow = kTerms == 2 && !kY ? 2 * kPanel : 0;
  static constexpr int kStage = 8 * 2048;                             // the warps' results
  static int smem(const RowsArgs& p) {
    return 1024 + kLow + kStage + p.slots * kPanel * (kY ? 2 : 1) +
           (p.resident ? p.panels : 1) * kWTerms * p.nt * 128;
  }
  // two accumulators (of two parts), so that one is read while the next
  // tile's is made
  static int columns(int nt) {
    int c = 32;
    while (c < 2 * nt * kTerms) c *= 2;
    return c;
  }
};

// Eight sums as a chunk of 16-bit results; two convert in one instruction.
template <typename T>
__device__ __forceinline__ uint4 round_chunk(const float* v) {
  uint4 q;
  uint32_t* const r = &q.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __half>::value)
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
    else
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r[i]) : "f"(v[2 * i + 1]), "f"(v[2 * i]));
  }
  return q;
}

// One chunk of a row on its way to shared memory: `there` values from p (none
// where there <= 0), zeros behind them.  WIDE: 16 bytes at once.  Else by
// single fp32 values, or, for 16-bit rows off the boundary, through
// registers.
template <typename T, bool WIDE>
__device__ __forceinline__ void send_chunk(char* to, const T* __restrict__ p, int there) {
  constexpr int E = Chunk<T>::E;
  if (there <= 0) {
    *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
  } else if constexpr (WIDE) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                 ::"r"(tc::smem_addr(to)), "l"(p) : "memory");
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;"
                   ::"r"(tc::smem_addr(to + 4 * e)), "l"(e < there ? p + e : p),
                   "r"(e < there ? 4 : 0) : "memory");
  } else {
    *reinterpret_cast<uint4*>(to) = get_chunk<T, false>(p, there);
  }
}
// The same for 16 bytes at once, with zeros copied, too: the barrier that counts
// the copies covers them.
__device__ __forceinline__ void send_or_zero(char* to, const void* p, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
               ::"r"(tc::smem_addr(to)), "l"(p), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void send_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last `n` groups have arrived.
__device__ __forceinline__ void arrived(int n) {
  if (n >= 4) asm volatile("cp.async.wait_group 4;" ::: "memory");
  else if (n == 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Which piece of a depth an accumulator holds.
enum { kWhole, kFirst, kMiddle, kLast };

// A warp's 32 lanes of an accumulator (columns of its half), 64 bytes of
// results at a time: through `stage`, the warp's own 2 KB of shared memory, and
// in pieces of rows to `out_rows`.  into: the row that lane's row is added to
// (kScatter).  A tile that is not live gives zeros.  Of a depth in pieces (fp32)
// the sums so far wait in the place of the result.
template <typename T, int ACT, int MODE, int TERMS>
__device__ __forceinline__ void take_results(bool live, uint32_t acc, int second, int half,
                                             int rows, int cols, const float* my_bias, int into,
                                             char* stage, void* out_rows, int row, int pitch,
                                             int n0, int wide_out, int part = kWhole) {
  constexpr bool BACK = MODE != kForward;
  constexpr int OB = MODE == kScatter ? 4 : sizeof(T);  // bytes of a result
  constexpr int OE = 16 / OB, SC = 64 / OB;             // results in 16 and in 64 bytes
  constexpr bool PIECES = sizeof(T) == 4 && MODE != kScatter;
  const int lane = threadIdx.x & 31;
  auto stage_at = [&](int r, int c) { return stage + r * 64 + ((c ^ ((r >> 1) & 3)) << 4); };
  for (int c0 = half * SC; c0 < cols; c0 += 2 * SC) {
    const int width = min(SC, cols - c0);  // columns here
    if constexpr (PIECES) {
      if (part == kMiddle || part == kLast) {  // the sums so far, written with the piece before
        const float* const from = static_cast<const float*>(out_rows) + (int64_t)row * pitch + n0 + c0;
        if (wide_out) {
          const int c = lane & 3;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if ((lane >> 2) + 8 * i < rows && c * 4 < width)
              *reinterpret_cast<float4*>(stage_at((lane >> 2) + 8 * i, c)) =
                  *reinterpret_cast<const float4*>(from + (int64_t)((lane >> 2) + 8 * i) * pitch + c * 4);
        } else {
          for (int i = lane; i < rows * width; i += 32) {
            const int r = i / width, e = i - r * width;
            reinterpret_cast<float*>(stage_at(r, e / 4))[e % 4] = from[(int64_t)r * pitch + e];
          }
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int h = 0; h < SC / 16; ++h) {
      if (h * 16 >= width) break;
      float v[16];
      if (live) {
        tc::load16(acc + c0 + h * 16, v);
        if (TERMS == 2) {
          float u[16];
          tc::load16(acc + second + c0 + h * 16, u);
          join_parts<T>(v, u);
        }
      }
      if constexpr (PIECES) {
        if (part == kMiddle || part == kLast) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float4 s = *reinterpret_cast<const float4*>(stage_at(lane, h * 4 + k));
            v[k * 4] += s.x, v[k * 4 + 1] += s.y, v[k * 4 + 2] += s.z, v[k * 4 + 3] += s.w;
          }
        }
      }
      if (!live) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.0f;
      } else if (!BACK && (!PIECES || part == kWhole || part == kLast)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (ACT == GS_ACT_SIGMOID && h * 16 + k * 4 >= width) break;  // 20 instructions each
          const float4 b = *reinterpret_cast<const float4*>(my_bias + c0 + h * 16 + k * 4);
          v[k * 4] = activate<ACT>(v[k * 4] + b.x);
          v[k * 4 + 1] = activate<ACT>(v[k * 4 + 1] + b.y);
          v[k * 4 + 2] = activate<ACT>(v[k * 4 + 2] + b.z);
          v[k * 4 + 3] = activate<ACT>(v[k * 4 + 3] + b.w);
        }
      }
#pragma unroll
      for (int c = 0; c < 16 / OE; ++c) {
        char* const to = stage_at(lane, h * (16 / OE) + c);
        if constexpr (OB == 4)
          *reinterpret_cast<float4*>(to) =
              make_float4(v[c * OE], v[c * OE + 1], v[c * OE + 2], v[c * OE + 3]);
        else
          *reinterpret_cast<uint4*>(to) = round_chunk<T>(v + c * OE);
      }
    }
    __syncwarp();
    const int c = lane & 3;
    if constexpr (MODE == kScatter) {
      float* const sum = static_cast<float*>(out_rows);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (lane >> 2) + 8 * i;
        const int32_t to_row = __shfl_sync(0xffffffffu, into, r);
        if (to_row < 0 || c * 4 >= width) continue;
        float* const to = sum + (int64_t)to_row * pitch + n0 + c0 + c * 4;
        const float4 v = *reinterpret_cast<const float4*>(stage_at(r, c));
        if (wide_out) {
          asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                       ::"l"(to), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w) : "memory");
        } else {
          atomicAdd(to, v.x);
          if (c * 4 + 1 < width) atomicAdd(to + 1, v.y);
          if (c * 4 + 2 < width) atomicAdd(to + 2, v.z);
          if (c * 4 + 3 < width) atomicAdd(to + 3, v.w);
        }
      }
    } else {
      T* const out = static_cast<T*>(out_rows) + (int64_t)row * pitch + n0 + c0;
      if (wide_out) {
        if (c * OE < width) {
          T* to = out + (int64_t)(lane >> 2) * pitch + c * OE;
          const int64_t down = (int64_t)8 * pitch;
#pragma unroll
          for (int i = 0; i < 4; ++i, to += down)
            if ((lane >> 2) + 8 * i < rows)
              *reinterpret_cast<uint4*>(to) =
                  *reinterpret_cast<const uint4*>(stage_at((lane >> 2) + 8 * i, c));
        }
      } else if (pitch <= SC) {  // whole rows: one run of memory
        const int total = rows * width;
        for (int i = lane; i < total; i += 32) {
          const int r = i / width, e = i - r * width;
          out[i] = reinterpret_cast<const T*>(stage_at(r, e / OE))[e % OE];
        }
      } else {
        constexpr int LR = 32 / SC;  // rows that the lanes cover
        const int e = lane & (SC - 1);
        if (e < width)
          for (int r = lane / SC; r < rows; r += LR)
            out[(int64_t)r * pitch + e] =
                reinterpret_cast<const T*>(stage_at(r, e / OE))[e % OE];
      }
    }
    __syncwarp();
  }
}

// out[row] = f(rows a, weights of the row's group): the forward, and v_x.
//
// One CTA an SM streams consecutive 128-row tiles, a panel (128 bytes of
// depth) at a time, through a ring of `slots` panels.  One warp has the
// panels filled by TMA, or two gather rows by asynchronous copies; rows off
// the 16-byte boundary the eight front warps copy.  These make
// operands of the panels, another warp issues the MMAs, and the eight back
// warps take a tile's accumulator while the next tile's is made.  16-bit rows
// are multiplied as they arrive; of fp32 rows the tensor core reads the upper
// part itself (it ignores the 13 low bits) and the low part is written beside;
// the backward through an activation rewrites the panel as v_z.  The group's
// weights are staged once per group, and stay.
//
// Bound by HBM for 16-bit rows: 2 M rows 128-128 bf16 forward 182 us, 5.6 TB/s of
// a copy's 6.5; v_x of 1.2 M rows 64-64 fp32, gathered, 6.1 TB/s of DRAM traffic
// (the sums' lines are read and written).  fp32 forwards wait: 600 k rows 128-128
// take 203 us, where HBM needs 94 and the four MMAs a step 66 (with the copies and
// low parts shared memory is busy for 89): only two panels of low parts are in
// flight.  A form that ran a tile's loads, MMAs and results one after the other,
// two CTAs an SM, took 284 us of the first.
//
// How rows arrive: by TMA; gathered, by two warps' copies; by copies of the
// front warps.  (TMA's four-row gathers took 19 cycles a 128-byte row, 49 us
// where the copies take 40: 316 k rows 64-64 fp32.)
enum { kTma, kGather, kCopy };

// Panels of fp32 rows that go through one accumulator: 256 features, 32 steps,
// of which each cuts the sum to fp32 (16384 features of one sign were 1.2e-4 low in
// one).  16-bit rows keep one: the 1024 steps of 16384 features lose 1e-4 of a sum
// of one sign, a fifth of fp16's own rounding.
constexpr int kPieceDepth = 8;
constexpr int kLoaders = 64;                          // threads of the gathering warps
constexpr int kCta = 2 * kThreads + 64 + kLoaders;    // front, back, MMA, TMA, gathers

template <typename T, int ACT, int MODE, int LOAD, bool WIDE, bool SPLIT>
__global__ void __launch_bounds__(LOAD == kGather ? kCta : kCta - kLoaders, 1)
    rows_mma_kernel(RowsArgs p, int columns, const __grid_constant__ CUtensorMap map_a,
                    const __grid_constant__ CUtensorMap map_y) {
  using L = RowsLayout<T, ACT, MODE, SPLIT>;
  constexpr int E = Chunk<T>::E;
  constexpr int DP = 128 / sizeof(T);   // depth of a panel
  constexpr int STEP = 32 / sizeof(T);  // depth of an MMA
  constexpr bool BACK = MODE != kForward;
  constexpr bool kPieces = sizeof(T) == 4;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t s_bars[3 * kSlotsMost + 6];
  __shared__ uint32_t s_tmem, s_stop;
  __shared__ __align__(16) float s_bias[8][kTile];
  char* const s_low = smem_raw + (1024 - (tc::smem_addr(smem_raw) & 1023)) % 1024;
  char* const s_stage = s_low + L::kLow;
  char* const s_rows = s_stage + L::kStage;
  char* const s_y = s_rows + p.slots * kPanel;
  char* const s_w = s_y + (L::kY ? p.slots * kPanel : 0);
  const uint32_t bar0 = tc::smem_addr(s_bars);
  auto full = [&](int i) { return bar0 + 8 * i; };                       // a slot has its rows
  auto free_ = [&](int i) { return bar0 + 8 * (kSlotsMost + i); };       // its MMAs are done
  auto ready = [&](int i) { return bar0 + 8 * (2 * kSlotsMost + i); };   // it has operands
  auto made = [&](int i) { return bar0 + 8 * (3 * kSlotsMost + i); };    // an accumulator is
  auto taken = [&](int i) { return bar0 + 8 * (3 * kSlotsMost + 2 + i); };
  const uint32_t weighed = bar0 + 8 * (3 * kSlotsMost + 4);              // the weights are there
  const uint32_t drained = bar0 + 8 * (3 * kSlotsMost + 5);              // all MMAs are done
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // known to be uniform
  const int n0 = blockIdx.y * p.nt;
  const int cols = min(p.nt, p.width - n0);
  const int wbytes = p.nt * 128;  // of a weight panel's part

  if (warp == 0) tc::alloc(&s_tmem, columns);
  if (threadIdx.x == 32) {
    const int none = p.waits.limit == 0;
    for (int i = 0; i < p.slots; ++i) {
      tc::bar_init(full(i), (LOAD == kGather ? kLoaders : 1) + none);
      tc::bar_init(free_(i), 1);
      tc::bar_init(ready(i), 8 + none);
    }
    tc::bar_init(weighed, 8);
    tc::bar_init(drained, 1);
    s_stop = 0;
    for (int i = 0; i < 2; ++i) {
      tc::bar_init(made(i), 1);
      tc::bar_init(taken(i), 8);
    }
    tc::bar_init_done();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  bool alive = true;  // no wait of this warp gave up
  auto wait = [&](uint32_t bar, uint32_t parity) {
    alive = alive && waited(bar, parity, p.waits, &s_stop);
  };

  const int64_t tiles = (p.s.R + kTile - 1) / kTile;
  const int end = (int)min(p.s.R, first_tile(tiles, gridDim.x, blockIdx.x + 1) * kTile);
  Run none;
  none.row = (int)(first_tile(tiles, gridDim.x, blockIdx.x) * kTile);
  none.n = 0, none.g = -1, none.group_end = 0;
  // the rows behind t that belong together
  auto after = [&](const Run& t) { return run_from(p.off, p.s.G, t.row + t.n, end, INT_MAX, t); };
  auto after_live = [&](Run t) {  // rows outside every group are the back's alone
    t = after(t);
    while (t.n > 0 && (t.g < 0 || t.g >= p.s.G)) t = after(t);
    return t;
  };
  auto steps_of = [&](int j) { return (min(DP, p.depth - j * DP) + STEP - 1) / STEP; };
  // the front makes operands of the panels; else they are multiplied as they are
  constexpr bool kWork = LOAD != kTma || L::kTerms == 2 || L::kY;

  if (warp == 17) {
    // ------------------------------------------------------------- TMA
    if (LOAD == kTma) {
      Ring ring(p.slots);
      int sent = 0;
      for (Run cur = after_live(none); cur.n > 0; cur = after_live(cur))
        for (int i = 0; i < cur.n; i += kTile)
          for (int j = 0; j < p.panels; ++j, ring.next()) {
            const int slot = ring.slot;
            if (ring.turn > 0) WAIT_OR(sent_all, free_(slot), ring.turn - 1);
            if (tc::elected()) {
              const uint32_t to = tc::smem_addr(s_rows + slot * kPanel);
              tc::expect(full(slot), kPanel * (L::kY ? 2 : 1));
              tc::load_box(to, &map_a, j * DP, cur.row + i, full(slot));
              if (L::kY)
                tc::load_box(to + p.slots * kPanel, &map_y, j * DP, cur.row + i, full(slot));
            }
            __syncwarp();
            ++sent;
          }
    sent_all:
      drain_ring(sent, p.slots, full);
    }
  } else if (warp >= 18) {
    // ------------------------------------------------------------- gathers
    if constexpr (LOAD == kGather) {
      const T* const a = static_cast<const T*>(p.a);
      const int lt = threadIdx.x - (kCta - kLoaders), c16 = lt & 7, r8 = lt >> 3;
      constexpr int N = kTile / 8;  // rows of a thread: r8 + 8 i
      Ring ring(p.slots);
      Run ahead = after_live(none);
      int ahead_row = 0, sent = 0, id[N];
      auto read_ids = [&]() {  // no use yet of what is read
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int row = ahead_row + r8 + 8 * i;
          id[i] = -1;
          if (row < ahead.n) id[i] = __ldg(p.ids + ahead.row + row);
        }
      };
      read_ids();
      while (ahead.n > 0) {
        int at[N];
#pragma unroll
        for (int i = 0; i < N; ++i) at[i] = id[i] < p.s.n ? id[i] : -1;
        ahead_row += kTile;
        if (ahead_row >= ahead.n) {
          ahead = after_live(ahead);
          ahead_row = 0;
        }
        read_ids();  // of the next tile
        for (int j = 0; j < p.panels; ++j, ring.next()) {
          const int slot = ring.slot, d = j * DP + c16 * E;
          if (ring.turn > 0) WAIT_OR(gathered, free_(slot), ring.turn - 1);
          if (c16 < 2 * steps_of(j)) {
            char* const to = s_rows + slot * kPanel + chunk_at(r8, c16);  // r & 7 is r8
            const T* const ad = d < p.depth ? a + d : a;
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const bool there = at[i] >= 0 && d < p.depth;
              send_or_zero(to + 1024 * i, there ? ad + (int64_t)at[i] * p.depth : a, there);
            }
          }
          tc::arrive_copied(full(slot));
          ++sent;
        }
      }
    gathered:
      arrived(0);
      drain_ring(sent, p.slots, full);
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------- MMAs
    const uint32_t idesc = tc::instr_desc(Mma<T>::format, (cols + 15) / 16 * 16);
    const uint32_t leader = tc::elected();
    Ring ring(p.slots);
    int stagings = 0, q = 0, t = 0;
    for (Run cur = after_live(none); cur.n > 0; cur = after_live(cur))
    for (int row = 0; row < cur.n; row += kTile, t += kPieces ? 0 : 1) {
      int held = 0;  // panels in the accumulator
      for (int j = 0; j < p.panels; ++j, ++q, ring.next()) {
        const int slot = ring.slot;
        if (row + j == 0 || !p.resident) WAIT_OR(mma_done, weighed, stagings++);
        WAIT_OR(mma_done, kWork ? ready(slot) : full(slot), ring.turn);
        if ((kPieces ? held : j) == 0 && t > 1) WAIT_OR(mma_done, taken(t & 1), (t >> 1) - 1);
        tc::fence_after_sync();
        const int steps = steps_of(j);
        const uint32_t acc = tmem + (t & 1) * p.nt * L::kTerms;
        const uint64_t da = tc::smem_desc(tc::smem_addr(s_rows + slot * kPanel));
        const uint64_t dl = tc::smem_desc(
            tc::smem_addr(L::kY ? s_y + slot * kPanel : s_low + (q & 1) * kPanel));
        const uint64_t dw =
            tc::smem_desc(tc::smem_addr(s_w + (p.resident ? j : 0) * L::kWTerms * wbytes));
        const uint64_t lo_w = wbytes >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i >= steps) break;
          const uint64_t step = 2 * i;  // 32 bytes
          const bool more = (kPieces ? held : j) > 0 || i > 0;
          if (L::kTerms == 2) {
            tc::mma<Mma<T>::TF32>(leader, acc + p.nt, dl + step, dw + step, idesc, more);
            if (L::kWTerms == 2) {
              tc::mma<Mma<T>::TF32>(leader, acc + p.nt, da + step, dw + lo_w + step, idesc, true);
              tc::mma<Mma<T>::TF32>(leader, acc + p.nt, dl + step, dw + lo_w + step, idesc, true);
            }
          }
          tc::mma<Mma<T>::TF32>(leader, acc, da + step, dw + step, idesc, more);
        }
        tc::commit(leader, free_(slot));
        if constexpr (!kPieces) {
          if (j + 1 == p.panels) tc::commit(leader, made(t & 1));
        } else if (++held == kPieceDepth || j + 1 == p.panels) {
          tc::commit(leader, made(t & 1));
          ++t;
          held = 0;
        }
      }
    }
    // every MMA is done before the memory goes
  mma_done:
    tc::commit(leader, drained);
    drain(drained, 0);
  } else if (warp < 8) {
    // ------------------------------------------------------------ front warps
    const int tid = threadIdx.x;
    const T* const a = static_cast<const T*>(p.a);
    const T* const y = static_cast<const T*>(p.y);
    const T* const w = static_cast<const T*>(p.w);
    const int c16 = tid & 7, r16 = tid >> 3;  // this thread's chunk, and its rows r16 + 32 i
    const uint32_t o16 = chunk_at(r16, c16);  // + 4096 i in a panel

    // The panel that is copied next: panel ahead_j of the rows at[], into slot
    // `ahead_s`; id[] are the rows of the tile after, from `behind_row` of
    // `behind` on, as they were read.
    Run behind = none;
    int behind_row = 0, ahead_j = 0, ahead_s = 0, at[4], id[4];
    bool ahead = false;  // there is something to copy
    auto move_on = [&]() {
#pragma unroll
      for (int i = 0; i < 4; ++i) at[i] = id[i] < p.s.n || BACK ? id[i] : -1;
      ahead = behind.n > 0;
      behind_row += kTile;
      if (behind_row >= behind.n) {
        behind = after_live(behind);
        behind_row = 0;
      }
      // (no use of what is read here: it is on its way for a tile's time)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = behind_row + r16 + 32 * i;
        id[i] = -1;
        if (row < behind.n) {
          if (p.ids && !BACK) id[i] = __ldg(p.ids + behind.row + row);
          else id[i] = behind.row + row;
        }
      }
    };
    auto send = [&]() {
      if (ahead) {
        if (c16 < 2 * steps_of(ahead_j)) {
          const int d = ahead_j * DP + c16 * E;
          const uint32_t to = ahead_s * kPanel + o16;
          const T* const ad = a + d;
          const T* const yd = L::kY ? y + d : nullptr;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int there = at[i] >= 0 ? p.depth - d : 0;
            const int64_t from = (int64_t)at[i] * p.depth;
            send_chunk<T, WIDE>(s_rows + to + 4096 * i, ad + from, there);
            if (L::kY) send_chunk<T, WIDE>(s_y + to + 4096 * i, yd + from, there);
          }
        }
        ahead_s = ahead_s + 1 == p.slots ? 0 : ahead_s + 1;
        if (++ahead_j == p.panels) {
          ahead_j = 0;
          move_on();
        }
      }
      send_done();  // also where nothing is left, to keep the count
    };

    // weight panels [j0, j1) of group g: rows n (columns of the result) x depth
    const int wlog = p.nt > 64 ? 7 : p.nt > 32 ? 6 : 5;
    auto stage_weights = [&](int g, int j0, int j1) {
      const T* const wg = w + (int64_t)g * p.s.M * p.s.K;
      const int units = (j1 - j0) * 8 << wlog;
      for (int u0 = tid; u0 < units; u0 += 4 * kThreads) {  // four loads in flight
        Chunk<T> q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int u = u0 + i * kThreads;
          if (!BACK) {  // chunks of a weight row
            const int c = u & 7, n = (u >> 3) & ((1 << wlog) - 1), j = u >> (3 + wlog);
            const int d = (j0 + j) * DP + c * E;
            const int there = u < units && n < cols ? p.depth - d : 0;
            const T* const from = wg + (there > 0 ? (int64_t)(n0 + n) * p.depth + d : 0);
            q[i].q = p.wide_w ? get_chunk<T, true>(from, there) : get_chunk<T, false>(from, there);
          } else {      // down a weight column; neighbours are neighbouring threads'
            const int n = u & ((1 << wlog) - 1), c = (u >> wlog) & 7, j = u >> (3 + wlog);
            const int d = (j0 + j) * DP + c * E;
            const bool in = u < units && n < cols;
#pragma unroll
            for (int e = 0; e < E; ++e)
              q[i].v[e] = in && d + e < p.depth ? wg[(int64_t)(d + e) * p.width + n0 + n]
                                                : from_f<T>(0.0f);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int u = u0 + i * kThreads;
          const int c = BACK ? (u >> wlog) & 7 : u & 7, j = u >> (3 + wlog);
          const int n = (BACK ? u : u >> 3) & ((1 << wlog) - 1);
          if (u < units && n < p.nt) {
            char* const to = s_w + j * L::kWTerms * wbytes + chunk_at(n, c);
            *reinterpret_cast<uint4*>(to) = q[i].q;
            if constexpr (sizeof(T) == 4) put_low(to + wbytes, q[i]);
          }
        }
      }
    };

    // A slot is filled again `lag` panels after its own, when its MMAs are
    // long done.
    const int lag = p.slots > 2 ? 2 : 1;
    if (LOAD == kCopy) {
#pragma unroll
      for (int i = 0; i < 4; ++i) id[i] = -1;
      move_on();
      move_on();
      for (int i = lag; i < p.slots; ++i) send();
    }
    Ring ring(p.slots);
    int q = 0;
    for (Run cur = after_live(none); cur.n > 0; cur = after_live(cur)) {
      if (p.resident) {
        // every MMA of the group before is done
        if (q > 0) WAIT_OR(fronted, free_(ring.slot_before(1)), ring.turn_before(1));
        stage_weights(cur.g, 0, p.panels);
        tc::fence_smem();
        __syncwarp();
        if (lane == 0) tc::arrive(weighed);
      }
      for (int row = 0; row < cur.n; row += kTile)
      for (int j = 0; j < p.panels; ++j, ++q, ring.next()) {
        const int slot = ring.slot;
        if (!p.resident) {
          if (q > 0) WAIT_OR(fronted, free_(ring.slot_before(1)), ring.turn_before(1));
          stage_weights(cur.g, j, j + 1);
          tc::fence_smem();
          __syncwarp();
          if (lane == 0) tc::arrive(weighed);
        }
        if (kWork) {
          // the panel `lag` before is done with: its slot, and its low parts
          if (q >= lag) WAIT_OR(fronted, free_(ring.slot_before(lag)), ring.turn_before(lag));
          if (LOAD == kCopy) {
            send();
            arrived(p.slots - lag);
          } else {
            WAIT_OR(fronted, full(slot), ring.turn);
          }
          if ((L::kTerms == 2 || L::kY) && c16 < 2 * steps_of(j)) {
            char* const here = s_rows + slot * kPanel;
            char* const low = L::kY ? s_y + slot * kPanel : s_low + (q & 1) * kPanel;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t o = o16 + 4096 * i;
              Chunk<T> v;
              v.q = *reinterpret_cast<const uint4*>(here + o);
              if constexpr (L::kY) {
                Chunk<T> z;
                z.q = *reinterpret_cast<const uint4*>(low + o);
                float f[E];
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = through<ACT>(to_f(v.v[e]), to_f(z.v[e]));
                put_chunk<T, SPLIT>(here + o, low - here, f);
              } else if constexpr (sizeof(T) == 4) {
                put_low(low + o, v);
              }
            }
          }
          tc::fence_smem();
          __syncwarp();
          if (lane == 0) tc::arrive(ready(slot));
        } else {
          // keeps pace: a barrier says whether its last phase is over, not
          // which one that is
          WAIT_OR(fronted, free_(slot), ring.turn);
        }
      }
    }
  fronted:
    if (LOAD == kCopy) arrived(0);
  } else {
    // ------------------------------------------------------------- back warps
    const T* const bias = static_cast<const T*>(p.bias);
    const int bw = warp - 8, row0 = (bw & 3) * 32;  // lanes of the accumulator
    float* const my_bias = s_bias[bw];
    int biased = -1, t = 0;
    for (Run cur = after(none); cur.n > 0; cur = after(cur))
    for (int row = cur.row; row < cur.row + cur.n; row += kTile) {
      const bool live = cur.g >= 0 && cur.g < p.s.G;
      const int rows = min(32, cur.row + cur.n - row - row0);
      int32_t into = -1;  // where lane's row is added up
      if (MODE == kScatter && live && lane < rows) into = __ldg(p.ids + row + row0 + lane);
      if (live && !BACK && cur.g != biased) {
        __syncwarp();
        for (int i = lane; i < p.nt; i += 32)
          my_bias[i] = bias && i < cols ? to_f(bias[(int64_t)cur.g * p.s.M + n0 + i]) : 0.0f;
        __syncwarp();
        biased = cur.g;
      }
      auto take = [&](int part) {
        const uint32_t acc = tmem + (t & 1) * p.nt * L::kTerms + ((uint32_t)row0 << 16);
        if (live) {
          wait(made(t & 1), t >> 1);
          if (!alive) return;
          tc::fence_after_sync();
        }
        if (into >= p.s.n) into = -1;
        take_results<T, ACT, MODE, L::kTerms>(live, acc, p.nt, bw >> 2, rows, cols, my_bias, into,
                                              s_stage + bw * 2048, p.out,
                                              MODE == kScatter ? 0 : row + row0, p.width,
                                              n0, p.wide_out, part);
        if (live) {
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::arrive(taken(t & 1));
          ++t;
        }
      };
      if (kPieces && live && p.panels > kPieceDepth) {
        for (int left = p.panels; left > 0; left -= kPieceDepth)
          take(left == p.panels ? kFirst : left > kPieceDepth ? kMiddle : kLast);
      } else {
        take(kWhole);
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::dealloc(tmem, columns);
}

// ---------------------------------------------------------- v_weights, v_biases
struct WeightArgs {
  Shape s;
  const void* x;
  const void* y;
  const void* vy;
  const int32_t* ids;
  const int32_t* off;
  float* part;       // [parts + G][M * K + M x copies of v_b]
  int kt, mt;        // tiles of K (128) and M (NT)
  int wide_x, wide_y;
  int biases;
  WaitArgs waits;
};

// The first piece of a sum is written, the others are added without waiting
// for what is there.  No other thread has the sum, so the order of the
// additions is the pieces'.
__device__ __forceinline__ void add_to(float* at, float v, bool first) {
  if (first) *at = v;
  else atomicAdd(at, v);
}
// A lane's 16 sums of an accumulator (`there` of them are wanted) to its column of
// the CTA's place, `pitch` floats apart.
__device__ __forceinline__ void add_piece(float* at, int pitch, int there, const float (&v)[16],
                                          bool first) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    if (i >= there) break;
    add_to(at + (int64_t)i * pitch, v[i], first);
  }
}

// v_W[g] (as K lanes x M columns) = sum over g's rows of x[r]^T v_z[r], of
// 16-bit rows that the kernel for the whole backward does not take: off the 16-byte
// boundary, or more than 128 features.
//
// The rows are the depth here, and both operands are staged transposed: a
// thread takes eight rows' chunks of the same eight columns and writes their
// columns as chunks.  A CTA sums the rows of its consecutive tiles; what it
// has at the end of a group goes to its own place in `part` (CTA b and group
// g: place b + g; both only ever grow), and the places of a group are added
// in order by another kernel, so the sums have a fixed order.  So does what it
// has after every kPiecePanels panels, since the tensor core cuts sums to fp32:
// 600 k rows 200-130 of one sign were 5e-5 low without that.
constexpr int kPiecePanels = 8;

template <typename T, int ACT, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 2)
    weights_mma_kernel(WeightArgs p, int columns) {
  constexpr int E = Chunk<T>::E;
  constexpr int DP = 128 / sizeof(T);
  constexpr int STEP = 32 / sizeof(T);
  constexpr int VTERMS = SPLIT ? 2 : 1;
  constexpr int VPANEL = NT * 128;
  extern __shared__ char smem_raw[];
  __shared__ uint64_t s_bars[2];
  __shared__ uint32_t s_tmem, s_stop;
  __shared__ int32_t s_ids[4][DP];
  char* const s_x = smem_raw + (1024 - (tc::smem_addr(smem_raw) & 1023)) % 1024;
  char* const s_v = s_x + kPanel;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int k0 = (blockIdx.y % p.kt) * 128, m0 = (blockIdx.y / p.kt) * NT;
  const int kn = min(128, p.s.K - k0), mn = min(NT, p.s.M - m0);
  const T* const x = static_cast<const T*>(p.x);
  const T* const y = static_cast<const T*>(p.y);
  const T* const vy = static_cast<const T*>(p.vy);

  if (warp == 0) tc::alloc(&s_tmem, columns);
  if (tid == 0) {
    tc::bar_init(tc::smem_addr(s_bars), p.waits.limit == 0 ? 2 : 1);
    tc::bar_init(tc::smem_addr(s_bars + 1), 1);
    s_stop = 0;
    tc::bar_init_done();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem, bar = tc::smem_addr(s_bars), drained = bar + 8;
  const uint32_t idesc = tc::instr_desc(Mma<T>::format, (mn + 15) / 16 * 16);
  uint32_t phase = 0;
  bool alive = true;  // no wait of this warp gave up
  auto wait_mma = [&]() {
    alive = alive && waited(bar, phase, p.waits, &s_stop);
    phase ^= 1;
    tc::fence_after_sync();
  };

  // This thread's blocks of E rows x E columns: eight neighbouring threads
  // have the panel's eight row blocks of the same columns, so that their
  // writes of a column go to eight different chunks of one operand row.
  const int x_units = 8 * ((kn + E - 1) / E), v_units = 8 * ((mn + E - 1) / E);
  const int vu = (tid + kThreads - x_units % kThreads) % kThreads;
  const bool has_x = tid < x_units, has_v = vu < v_units;
  const int rb = (tid & 7) * E;                 // first row of either block
  const int xc = (tid >> 3) * E, vc = (vu >> 3) * E;
  uint4 rx[E], ry[ACT ? E : 1];  // a thread has a block of x or one of v_y
  float bsum[E];
#pragma unroll
  for (int e = 0; e < E; ++e) bsum[e] = 0.0f;

  const int64_t tiles = (p.s.R + kTile - 1) / kTile;
  const int end = (int)min(p.s.R, first_tile(tiles, gridDim.x, blockIdx.x + 1) * kTile);
  auto next_run = [&](Run t) {  // skips rows outside every group
    Run n = run_from(p.off, p.s.G, t.row + t.n, end, DP, t);
    while (n.n > 0 && (n.g < 0 || n.g >= p.s.G))
      n = run_from(p.off, p.s.G, n.group_end, end, DP, n);
    return n;
  };
  Run none;
  none.row = (int)(first_tile(tiles, gridDim.x, blockIdx.x) * kTile);
  none.n = 0, none.g = -1, none.group_end = 0;
  Run cur = next_run(none);
  Run nxt = next_run(cur);
  auto id_of = [&](const Run& t, int i) {
    return p.ids && i < t.n ? __ldg(p.ids + t.row + i) : -1;
  };
  auto load_run = [&](const Run& t, int k) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const bool in = rb + i < t.n;
      if (has_x) {
        int at = t.row + rb + i;
        bool ok = in;
        if (p.ids) {
          at = s_ids[k & 3][rb + i];
          ok = at >= 0 && at < p.s.n;
        }
        const T* const from = x + (ok ? (int64_t)at * p.s.K + k0 + xc : 0);
        const int there = ok ? kn - xc : 0;
        rx[i] = p.wide_x ? get_chunk<T, true>(from, there) : get_chunk<T, false>(from, there);
      }
      if (has_v) {
        const int64_t from = in ? (int64_t)(t.row + rb + i) * p.s.M + m0 + vc : 0;
        const int there = in ? mn - vc : 0;
        rx[i] = p.wide_y ? get_chunk<T, true>(vy + from, there) : get_chunk<T, false>(vy + from, there);
        if (ACT)
          ry[ACT ? i : 0] = p.wide_y ? get_chunk<T, true>(y + from, there)
                                     : get_chunk<T, false>(y + from, there);
      }
    }
  };

  constexpr int HALF = NT / 2;  // columns of a warp's half of the accumulators
  if (tid < DP) s_ids[0][tid] = id_of(cur, tid);
  int next_id = tid < DP ? id_of(nxt, tid) : -1;
  __syncthreads();
  if (cur.n > 0) load_run(cur, 0);
  int pending = 0;              // panels in the accumulators
  bool first = true;            // none of the group have left them yet

  for (int k = 0; cur.n > 0; ++k) {
    if (pending > 0) wait_mma();  // the panels' memory is free again
    if (has_x) {
#pragma unroll
      for (int c = 0; c < E; ++c) {
        Chunk<T> raw;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          Chunk<T> q;
          q.q = rx[i];
          raw.v[i] = q.v[c];
        }
        *reinterpret_cast<uint4*>(s_x + chunk_at(xc + c, tid & 7)) = raw.q;
      }
    }
    if (has_v) {
#pragma unroll
      for (int c = 0; c < E; ++c) {
        float f[E];
#pragma unroll
        for (int i = 0; i < E; ++i) {
          Chunk<T> q, o;
          q.q = rx[i];
          if (ACT) o.q = ry[ACT ? i : 0];
          f[i] = through<ACT>(to_f(q.v[c]), ACT ? to_f(o.v[c]) : 0.0f);
          bsum[c] += f[i];
        }
        put_chunk<T, SPLIT>(s_v + chunk_at(vc + c, tid & 7), VPANEL, f);
      }
    }
    if (tid < DP) s_ids[(k + 1) & 3][tid] = next_id;
    tc::fence_smem();
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 0) {
      tc::fence_after_sync();
      const uint32_t elect = tc::elected(), leader = alive ? elect : 0;
      const uint64_t dx = tc::smem_desc(tc::smem_addr(s_x)), dv = tc::smem_desc(tc::smem_addr(s_v));
      const int steps = (cur.n + STEP - 1) / STEP;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= steps) break;
        const uint64_t at = 2 * i;
        const bool more = pending > 0 || i > 0;
        if (VTERMS == 2)
          tc::mma<false>(leader, tmem + NT, dx + at, dv + (VPANEL >> 4) + at, idesc, more);
        tc::mma<false>(leader, tmem, dx + at, dv + at, idesc, more);
      }
      tc::commit(leader, bar);
    }
    ++pending;
    Run after = nxt;
    if (nxt.n > 0) {
      load_run(nxt, k + 1);
      after = next_run(nxt);
      if (tid < DP) next_id = id_of(after, tid);
    }
    const bool last = nxt.n == 0 || nxt.g != cur.g;  // of the group
    if (last || pending == kPiecePanels) {  // the sums to their place
      wait_mma();
      float* const to = p.part + (int64_t)(blockIdx.x + cur.g) * ((int64_t)p.s.M * (p.s.K + 1));
      const int kk = (warp & 3) * 32 + lane;
#pragma unroll
      for (int c = 0; c < HALF; c += 16) {
        float v[16];
        const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16) + (warp >> 2) * HALF + c;
        tc::load16(from, v);
        if (SPLIT) {
          float u[16];
          tc::load16(from + NT, u);
          join_parts<T>(v, u);
        }
        const int m = (warp >> 2) * HALF + c;
        if (kk < kn)
          add_piece(to + (int64_t)(m0 + m) * p.s.K + k0 + kk, p.s.K, mn - m, v, first);
      }
#pragma unroll
      for (int e = 0; e < E; ++e) {
        float b = bsum[e];
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) b += __shfl_xor_sync(0xffffffffu, b, o);
        if (has_v && p.biases && k0 == 0 && (tid & 7) == 0 && vc + e < mn)
          add_to(to + (int64_t)p.s.M * p.s.K + m0 + vc + e, b, first);
        bsum[e] = 0.0f;
      }
      pending = 0;
      first = last;
      tc::fence_before_sync();
      __syncthreads();
    }
    cur = nxt;
    nxt = after;
  }
  if (warp == 0) {
    tc::commit(tc::elected(), drained);
    drain(drained, 0);
    tc::dealloc(tmem, columns);
  }
}

// v_W and v_b of fp32 rows.
//
// Depth runs over rows here and tf32 operands are K-major, so what arrives as
// 32 rows x 32 columns boxes (TMA; copies where rows are gathered or off the
// boundary) is transposed on its way to the operands: a thread reads a 4 x 4
// block as four chunks and writes its columns as chunks of the values (of
// which the tensor core takes the upper part) and of their low parts.  The
// eight lanes of an access take the diagonal blocks (column block l, row
// block l ^ p), which keeps both the reads and the writes free of conflicts in
// the swizzled panels.  Two groups of four front warps take every second
// panel of 32 rows, with operand memory of its own for one or two of them.
//
// The tensor core cuts a sum to fp32 at each addition; left to itself that
// was 2e-5 of the result after 8000 rows.  So every kFlush panels the MMAs
// change accumulators, and the back warps add the finished one to sums that
// they hold in registers.
//
// 1.2 M gathered rows 64-64: 212 us with the join, 4.4 TB/s.  The MMAs (16 a panel,
// 48 cycles each), the transposition and the copies share the shared memory's 128
// bytes a cycle: about 1400 of the 1500 cycles that a panel takes.  More than 64
// outputs spill: the back warps' sums do not all fit a thread's 96 registers.
constexpr int kFlush = 4;
constexpr int kRows32 = 32;
constexpr int kBox = kRows32 * 128;
constexpr int kBars32 = 29;

struct Weight32Args {
  Shape s;
  const float* x;
  const float* y;
  const float* vy;
  const int32_t* ids;
  const int32_t* off;
  float* part;         // as in WeightArgs, with kBiasCopies32 rows of v_b
  int kt;              // tiles of K (128)
  int kx, mx;          // boxes of a K tile and of an M tile
  int slots;           // panels of boxes; even with copies, and at least `sets`
  int sets;            // of operands: 2 or 4
  int x_mode, v_mode;  // 0: TMA, 1: gathered, 2: the front's copies of 4 bytes
  int biases;
  WaitArgs waits;
};

template <int ACT, int NT>
__global__ void __launch_bounds__(kCta, 1)
    weights32_kernel(Weight32Args p, const __grid_constant__ CUtensorMap map_x,
                     const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ CUtensorMap map_y) {
  constexpr bool HAS_Y = ACT != GS_ACT_NONE;
  extern __shared__ __align__(1024) char smem_raw[];
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int K = p.s.K, M = p.s.M;
  const int k0 = (blockIdx.y % p.kt) * 128, m0 = (blockIdx.y / p.kt) * NT;
  const int kn = min(128, K - k0), mn = min(NT, M - m0);
  const int boxes = p.kx + p.mx;                          // x's, then v_y's
  const int slot_bytes = (boxes + (HAS_Y ? p.mx : 0)) * kBox;  // then y's
  // operands: sets of values and low parts of x, of v_z.  An MMA reads
  // 128 rows of x's whatever kn is: what lies behind goes to unused lanes.
  const int set_bytes = 2 * boxes * kBox;
  char* const s_sets = smem_raw;
  char* const s_slots = s_sets + p.sets * set_bytes;
  uint64_t* const s_bars = reinterpret_cast<uint64_t*>(s_slots + p.slots * slot_bytes);
  uint32_t& s_tmem = *reinterpret_cast<uint32_t*>(s_bars + kBars32);
  uint32_t& s_stop = (&s_tmem)[1];
  const uint32_t bar0 = tc::smem_addr(s_bars);
  auto full = [&](int i) { return bar0 + 8 * i; };          // TMA's boxes are there
  auto free_ = [&](int i) { return bar0 + 8 * (8 + i); };   // and have been read
  auto ready = [&](int i) { return bar0 + 8 * (16 + i); };  // operands
  auto spent = [&](int i) { return bar0 + 8 * (20 + i); };
  auto made = [&](int i) { return bar0 + 8 * (24 + i); };   // accumulators
  auto taken = [&](int i) { return bar0 + 8 * (26 + i); };
  const uint32_t drained = bar0 + 8 * 28;
  const int log_sets = p.sets == 4 ? 2 : 1;
  const int tma_boxes = (p.x_mode == 0 ? p.kx : 0) + (p.v_mode == 0 ? p.mx * (HAS_Y ? 2 : 1) : 0);
  const bool sent = tma_boxes > 0 || p.x_mode == 1;  // by other than the front warps
  if (warp == 0) tc::alloc(&s_tmem, 4 * NT);
  if (threadIdx.x == 32) {
    const int none = p.waits.limit == 0;
    for (int i = 0; i < 8; ++i) {
      tc::bar_init(full(i),
                   max((tma_boxes > 0 ? 1 : 0) + (p.x_mode == 1 ? kLoaders : 0), 1) + none);
      tc::bar_init(free_(i), 4);
    }
    for (int i = 0; i < 4; ++i) {
      tc::bar_init(ready(i), 4 + none);
      tc::bar_init(spent(i), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::bar_init(made(i), 1);
      tc::bar_init(taken(i), 8);
    }
    tc::bar_init(drained, 1);
    s_stop = 0;
    tc::bar_init_done();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  bool alive = true;  // no wait of this warp gave up
  auto wait = [&](uint32_t bar, uint32_t parity) {
    alive = alive && waited(bar, parity, p.waits, &s_stop);
  };

  const int64_t tiles = (p.s.R + kTile - 1) / kTile;
  const int end = (int)min(p.s.R, first_tile(tiles, gridDim.x, blockIdx.x + 1) * kTile);
  Run none;
  none.row = (int)(first_tile(tiles, gridDim.x, blockIdx.x) * kTile);
  none.n = 0, none.g = -1, none.group_end = 0;
  // all of this CTA's rows of the next group; rows outside every group are
  // skipped
  auto after = [&](Run t) {
    t = run_from(p.off, p.s.G, t.row + t.n, end, INT_MAX, t);
    while (t.n > 0 && (t.g < 0 || t.g >= p.s.G))
      t = run_from(p.off, p.s.G, t.group_end, end, INT_MAX, t);
    return t;
  };

  if (warp == 17) {
    // ------------------------------------------------------------- TMA
    if (tma_boxes > 0) {
      Ring ring(p.slots);
      int panels = 0;
      for (Run cur = after(none); cur.n > 0; cur = after(cur))
        for (int row = cur.row; row < cur.row + cur.n; row += kRows32, ring.next()) {
          const int slot = ring.slot;
          if (ring.turn > 0) WAIT_OR(sent_all, free_(slot), ring.turn - 1);
          if (tc::elected()) {
            const uint32_t to = tc::smem_addr(s_slots + slot * slot_bytes);
            tc::expect(full(slot), tma_boxes * kBox);
            if (p.x_mode == 0)
              for (int j = 0; j < p.kx; ++j)
                tc::load_box(to + j * kBox, &map_x, k0 + j * 32, row, full(slot));
            if (p.v_mode == 0)
              for (int j = 0; j < p.mx; ++j) {
                tc::load_box(to + (p.kx + j) * kBox, &map_v, m0 + j * 32, row, full(slot));
                if (HAS_Y)
                  tc::load_box(to + (boxes + j) * kBox, &map_y, m0 + j * 32, row, full(slot));
              }
          }
          __syncwarp();
          ++panels;
        }
    sent_all:
      drain_ring(panels, p.slots, full);
    }
  } else if (warp >= 18) {
    // ------------------------------------------------------------- gathers
    if (p.x_mode == 1) {
      const int lt = threadIdx.x - (kCta - kLoaders), c16 = lt & 7, r8 = lt >> 3;
      Ring ring(p.slots);
      Run ahead = after(none);
      int panels = 0, ahead_row = 0, id[2][4];  // rows r8 + 8 i of the next two panels
      auto read_ids = [&](int (&to)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = ahead_row + r8 + 8 * i;
          to[i] = -1;
          if (row < ahead.n) to[i] = __ldg(p.ids + ahead.row + row);
        }
        ahead_row += kRows32;
        if (ahead_row >= ahead.n) {
          ahead = after(ahead);
          ahead_row = 0;
        }
      };
      read_ids(id[0]);
      read_ids(id[1]);
      for (Run cur = after(none); cur.n > 0; cur = after(cur))
        for (int left = cur.n; left > 0; left -= kRows32, ring.next()) {
          const int slot = ring.slot;
          int at[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            at[i] = id[0][i] < p.s.n ? id[0][i] : -1;
            id[0][i] = id[1][i];
          }
          read_ids(id[1]);
          if (ring.turn > 0) WAIT_OR(gathered, free_(slot), ring.turn - 1);
          char* const to = s_slots + slot * slot_bytes + chunk_at(r8, c16);
          for (int j = 0; j < p.kx; ++j) {
            const int k = j * 32 + c16 * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool there = at[i] >= 0 && k < kn;
              send_or_zero(to + j * kBox + 1024 * i,
                           there ? p.x + (int64_t)at[i] * K + k0 + k : p.x, there);
            }
          }
          tc::arrive_copied(full(slot));
          ++panels;
        }
    gathered:
      arrived(0);
      drain_ring(panels, p.slots, full);
    }
  } else if (warp == 16) {
    // ------------------------------------------------------------- MMAs
    const uint32_t idesc = tc::instr_desc(tc::kTF32, (mn + 15) / 16 * 16);
    const uint32_t leader = tc::elected();
    int q = 0, held = 0, sums = 0;
    for (Run cur = after(none); cur.n > 0; cur = after(cur))
    for (int left = cur.n; left > 0; left -= kRows32, ++q) {
      const int set = q & (p.sets - 1), buf = sums & 1;
      WAIT_OR(mma_done, ready(set), q >> log_sets);
      if (held == 0 && sums > 1) WAIT_OR(mma_done, taken(buf), (sums >> 1) - 1);
      tc::fence_after_sync();
      const uint32_t x_at = tc::smem_addr(s_sets + set * set_bytes);
      const uint64_t xh = tc::smem_desc(x_at), xl = tc::smem_desc(x_at + p.kx * kBox);
      const uint32_t v_at = x_at + 2 * p.kx * kBox;
      const uint64_t vh = tc::smem_desc(v_at), vl = tc::smem_desc(v_at + p.mx * kBox);
      const uint32_t acc = tmem + buf * 2 * NT;
      const int steps = (left + 7) / 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= steps) break;
        const uint64_t at = 2 * i;
        const bool more = held > 0 || i > 0;
        tc::mma<true>(leader, acc + NT, xl + at, vl + at, idesc, more);
        tc::mma<true>(leader, acc + NT, xl + at, vh + at, idesc, true);
        tc::mma<true>(leader, acc + NT, xh + at, vl + at, idesc, true);
        tc::mma<true>(leader, acc, xh + at, vh + at, idesc, more);
      }
      tc::commit(leader, spent(set));
      if (++held == kFlush || left <= kRows32) {
        tc::commit(leader, made(buf));
        ++sums;
        held = 0;
      }
    }
  mma_done:
    tc::commit(leader, drained);  // every MMA is done before the memory goes
    drain(drained, 0);
  } else if (warp < 8) {
    // ------------------------------------------------------------ front warps
    const int fg = warp >> 2, tid = threadIdx.x & 127;
    const bool copies = p.x_mode == 2 || p.v_mode == 2;
    const int own = p.slots / 2;  // with copies: this group's slots
    // copies: rows r16 and r16 + 16, chunk c16, of every box
    const int r16 = tid >> 3, c16 = tid & 7;
    Run ahead = none;           // the rows that are copied next: from ahead_row on
    int ahead_row = 0, ahead_i = 0, id[2];
    auto forward = [&](int panels) {  // moves on, to this group's next panel
      for (; panels > 0 && ahead.n > 0; --panels) {
        ahead_row += kRows32;
        if (ahead_row >= ahead.row + ahead.n) {
          ahead = after(ahead);
          ahead_row = ahead.row;
        }
      }
      // (no use of what is read here: it is on its way until the next copies)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = ahead_row + r16 + 16 * i;
        id[i] = -1;
        if (row < ahead.row + ahead.n) {
          if (p.ids) id[i] = __ldg(p.ids + row);
          else id[i] = row;
        }
      }
    };
    auto send = [&]() {
      if (ahead.n > 0) {
        char* const to = s_slots + (2 * ahead_i + fg) * slot_bytes;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = r16 + 16 * i;
          const uint32_t o = chunk_at(row, c16);
          if (p.x_mode == 2) {
            const bool ok = id[i] >= 0 && id[i] < p.s.n;
            const float* const from = p.x + (ok ? (int64_t)id[i] * K + k0 + c16 * 4 : 0);
            for (int j = 0; j < p.kx; ++j) {
              const int there = ok ? kn - j * 32 - c16 * 4 : 0;
              send_chunk<float, false>(to + j * kBox + o, from + j * 32, there);
            }
          }
          if (p.v_mode == 2) {
            const bool ok = ahead_row + row < ahead.row + ahead.n;
            const int64_t from = ok ? (int64_t)(ahead_row + row) * M + m0 + c16 * 4 : 0;
            for (int j = 0; j < p.mx; ++j) {
              const int there = ok ? mn - j * 32 - c16 * 4 : 0;
              send_chunk<float, false>(to + (p.kx + j) * kBox + o, p.vy + from + j * 32, there);
              if (HAS_Y)
                send_chunk<float, false>(to + (boxes + j) * kBox + o, p.y + from + j * 32, there);
            }
          }
        }
        ahead_i = ahead_i + 1 == own ? 0 : ahead_i + 1;
        forward(2);
      }
      send_done();
    };
    if (copies) {
      ahead = after(none);
      ahead_row = ahead.row;
      forward(fg);
      for (int i = 1; i < own; ++i) send();
    }
    // this thread's 4 x 4 blocks: of boxes 2 it + (tid >> 6)
    const int l = tid & 7, c = l, rg = l ^ ((tid >> 3) & 7);
    constexpr int ITS = (4 + NT / 32) / 2;
    float db[ITS][4];
#pragma unroll
    for (int it = 0; it < ITS; ++it)
#pragma unroll
      for (int j = 0; j < 4; ++j) db[it][j] = 0.0f;
    Ring ring(p.slots);
    int q = 0, left = 0;
    Run cur;
    for (cur = after(none); cur.n > 0; cur = after(cur)) {
      for (left = cur.n; left > 0; left -= kRows32, ++q, ring.next()) {
        if ((q & 1) != fg) continue;
        const int slot = ring.slot;
        if (copies) {
          if (own > 1) {
            arrived(own - 2);
            tc::bar_sync(1 + fg, 128);  // everyone's copies, and nobody in the panel before
            send();
          } else {
            tc::bar_sync(1 + fg, 128);
            send();
            arrived(0);
            tc::bar_sync(1 + fg, 128);
          }
        }
        // (first: it says that all panels up to the one `sets` <= `slots` before
        // have been through their slots, so that the slot's barrier is at this
        // panel)
        const int at_set = q & (p.sets - 1);
        if (q >= p.sets) WAIT_OR(walk, spent(at_set), (q >> log_sets) - 1);
        if (sent) WAIT_OR(walk, full(slot), ring.turn);
        const char* const from = s_slots + slot * slot_bytes;
        char* const set = s_sets + at_set * set_bytes;
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const int b = 2 * it + (tid >> 6);
          if (b < boxes) {
            const bool is_v = b >= p.kx;
            Chunk<float> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int row = 4 * rg + i;
              v[i].q = row < left
                           ? *reinterpret_cast<const uint4*>(from + b * kBox + chunk_at(row, c))
                           : make_uint4(0, 0, 0, 0);
            }
            if (is_v) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int row = 4 * rg + i;
                if (HAS_Y) {
                  Chunk<float> z;
                  z.q = *reinterpret_cast<const uint4*>(from + (b + p.mx) * kBox + chunk_at(row, c));
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    v[i].v[j] = row < left ? through<ACT>(v[i].v[j], z.v[j]) : 0.0f;
                }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
                db[it][j] += (v[0].v[j] + v[1].v[j]) + (v[2].v[j] + v[3].v[j]);
            }
            // values, and as many bytes behind all of them their low parts
            char* const to = set + (is_v ? (p.kx + b) * kBox : b * kBox);
            const int low = (is_v ? p.mx : p.kx) * kBox;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              Chunk<float> t;
#pragma unroll
              for (int i = 0; i < 4; ++i) t.v[i] = v[i].v[j];
              char* const at = to + chunk_at(4 * c + j, rg);
              *reinterpret_cast<uint4*>(at) = t.q;
              put_low(at + low, t);
            }
          }
          asm volatile("" ::: "memory");  // one block at a time: registers
        }
        tc::fence_smem();
        __syncwarp();
        if (lane == 0) {
          tc::arrive(ready(at_set));
          if (sent) tc::arrive(free_(slot));
        }
      }
      if (p.biases && k0 == 0) {  // v_b: this front group's and half's share
        float* const to = p.part + (int64_t)(blockIdx.x + cur.g) * M * (K + kBiasCopies32) +
                          (int64_t)M * K + (int64_t)(2 * fg + ((tid >> 5) & 1)) * M + m0;
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const int col = (2 * it + (tid >> 6) - p.kx) * 32 + c * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float b = db[it][j];
            b += __shfl_xor_sync(0xffffffffu, b, 8);
            b += __shfl_xor_sync(0xffffffffu, b, 16);
            if (lane < 8 && col >= 0 && col + j < mn) to[col + j] = b;
          }
        }
      }
#pragma unroll
      for (int it = 0; it < ITS; ++it)
#pragma unroll
        for (int j = 0; j < 4; ++j) db[it][j] = 0.0f;
    }
  walk:
    // behind a wait that gave up: the group's other warps still meet this one
    while (copies && cur.n > 0) {
      left -= kRows32, ++q;
      if (left <= 0) cur = after(cur), left = cur.n;
      if (cur.n > 0 && (q & 1) == fg)
        for (int i = own > 1 ? 1 : 0; i < 2; ++i) tc::bar_sync(1 + fg, 128);
    }
    if (copies) arrived(0);
  } else {
    // ------------------------------------------------------------- back warps
    constexpr int HALF = NT / 2;
    const int bw = warp - 8, row0 = (bw & 3) * 32, c0 = (bw >> 2) * HALF;
    float acc[HALF];
#pragma unroll
    for (int i = 0; i < HALF; ++i) acc[i] = 0.0f;
    int sums = 0;
    for (Run cur = after(none); cur.n > 0; cur = after(cur))
      for (int left = cur.n; left > 0; left -= kFlush * kRows32) {
        const int buf = sums & 1;
        WAIT_OR(taken_all, made(buf), sums >> 1);
        tc::fence_after_sync();
#pragma unroll
        for (int c = 0; c < HALF; c += 16) {
          if (c0 + c >= mn) break;
          float v[16], u[16];
          const uint32_t from = tmem + buf * 2 * NT + ((uint32_t)row0 << 16) + c0 + c;
          tc::load16(from, v);
          tc::load16(from + NT, u);
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c + i] += fabsf(v[i]) < INFINITY ? v[i] + u[i] : v[i];
        }
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::arrive(taken(buf));
        ++sums;
        if (left <= kFlush * kRows32) {
          float* const to = p.part + (int64_t)(blockIdx.x + cur.g) * M * (K + kBiasCopies32) +
                            (int64_t)(m0 + c0) * K + k0 + row0 + lane;
#pragma unroll
          for (int i = 0; i < HALF; ++i) {
            if (row0 + lane < kn && c0 + i < mn) to[(int64_t)i * K] = acc[i];
            acc[i] = 0.0f;
          }
        }
      }
  taken_all:;
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::dealloc(tmem, 4 * NT);
}

// ------------------------------------------------- the whole backward, 16 bits
struct BothArgs {
  Shape s;
  const int32_t* ids;
  const int32_t* off;
  const void* w;
  void* vx;          // v_x, its fp32 sums with SHARED, or NULL: not wanted
  float* part;       // as in WeightArgs
  int pk, pm;        // panels (64 columns) of K and M: 1 or 2
  int slots, ys;     // tiles of v_y and x, and panels of y, in shared memory
  int biases;
  int vx_width;      // columns of v_x: K, or fewer where K was padded
  int wide_out;
  WaitArgs waits;
};

// Rows of K and M of up to 128 features, on 16-byte boundaries: v_y, y and x
// are read once for v_x, v_W and v_b together.  A tile is 128 rows; v_y's
// panels are rewritten as v_z and multiplied twice from where they lie: with
// rows as lanes and the weights (v_x), and with rows as depth and x (v_W: both
// operands are "MN-major" then, as the weights are in the first product), so
// nothing is transposed.  The roles of the warps are those of the rows kernel.
// HBM-bound: 2 M rows 128-128 bf16, relu, 340 us with the join, 6.0 TB/s; v_x and
// v_W by kernels of their own took 1107 us.
//
// v_W's accumulator is added to the CTA's place in `part` at the end of a
// group, and every kPiece tiles: the tensor core cuts sums to fp32 instead of
// rounding them, by 3 2^-25 of a growing sum at each of a tile's 8 steps.  With 32
// tiles sums of one sign were 2.5e-5 low, with 4 they are 3e-6; the 2 M rows take
// 340 us instead of 336 (in a long run, which power bounds, 361 instead of 350).
// Another accumulator is filled meanwhile where v_z has one part.
constexpr int kPiece = 4;
constexpr int kBothBars = 30;

template <typename T, int ACT, bool SHARED>
__global__ void __launch_bounds__(2 * kThreads + 64, 1)
    both_mma_kernel(BothArgs p, int columns, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ CUtensorMap map_y,
                    const __grid_constant__ CUtensorMap map_x) {
  constexpr int TERMS = ACT == GS_ACT_SIGMOID ? 2 : 1;  // parts of v_z
  constexpr int NBUF = TERMS == 2 ? 1 : 2;              // accumulators of v_x, and of v_W
  constexpr bool HAS_Y = ACT != GS_ACT_NONE;
  // all of it dynamic: the panels have to start on 1024 bytes, with nothing lost
  extern __shared__ __align__(1024) char smem_raw[];
  const int lane = threadIdx.x & 31;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int K = p.s.K, M = p.s.M;
  const int nk = (K + 31) / 32 * 32, nm = (M + 31) / 32 * 32;
  const int tile_bytes = (p.pm + p.pk) * kPanel;
  char* const s_tiles = smem_raw;              // v_z's panels, then x's
  char* const s_y = s_tiles + p.slots * tile_bytes;
  char* const s_w = s_y + p.ys * kPanel;
  char* const s_stage = s_w + p.pk * kPanel;
  float (*const s_db)[64] = reinterpret_cast<float (*)[64]>(s_stage + 8 * 2048);
  uint64_t* const s_bars = reinterpret_cast<uint64_t*>(s_db + 8);
  uint32_t& s_tmem = *reinterpret_cast<uint32_t*>(s_bars + kBothBars);
  uint32_t& s_stop = (&s_tmem)[1];
  const uint32_t bar0 = tc::smem_addr(s_bars);
  auto full = [&](int i) { return bar0 + 8 * i; };
  auto free_ = [&](int i) { return bar0 + 8 * (4 + i); };
  auto ready = [&](int i) { return bar0 + 8 * (8 + i); };
  auto y_full = [&](int i) { return bar0 + 8 * (12 + i); };
  auto y_free = [&](int i) { return bar0 + 8 * (16 + i); };
  auto made = [&](int i) { return bar0 + 8 * (20 + i); };
  auto taken = [&](int i) { return bar0 + 8 * (22 + i); };
  auto sum_made = [&](int i) { return bar0 + 8 * (24 + i); };
  auto sum_taken = [&](int i) { return bar0 + 8 * (26 + i); };
  const uint32_t weighed = bar0 + 8 * 28, drained = bar0 + 8 * 29;

  if (warp == 0) tc::alloc(&s_tmem, columns);
  if (threadIdx.x == 32) {
    for (int i = 0; i < 4; ++i) {
      tc::bar_init(full(i), p.waits.limit == 0 ? 2 : 1);
      tc::bar_init(free_(i), 1);
      tc::bar_init(ready(i), 8);
      tc::bar_init(y_full(i), 1);
      tc::bar_init(y_free(i), TERMS == 2 ? 1 : 8);  // the low parts of v_z lie there
    }
    for (int i = 0; i < 2; ++i) {
      tc::bar_init(made(i), 1);
      tc::bar_init(taken(i), 8);
      tc::bar_init(sum_made(i), 1);
      tc::bar_init(sum_taken(i), 8);
    }
    tc::bar_init(weighed, 8);
    tc::bar_init(drained, 1);
    s_stop = 0;
    tc::bar_init_done();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem, sum_acc = tmem + NBUF * TERMS * nk;

  const int64_t tiles = (p.s.R + kTile - 1) / kTile;
  const int end = (int)min(p.s.R, first_tile(tiles, gridDim.x, blockIdx.x + 1) * kTile);
  Run none;
  none.row = (int)(first_tile(tiles, gridDim.x, blockIdx.x) * kTile);
  none.n = 0, none.g = -1, none.group_end = 0;
  auto after = [&](const Run& t) { return run_from(p.off, p.s.G, t.row + t.n, end, INT_MAX, t); };
  auto after_live = [&](Run t) {
    t = after(t);
    while (t.n > 0 && (t.g < 0 || t.g >= p.s.G)) t = after(t);
    return t;
  };

  if (warp == 17) {
    // ------------------------------------------------------------- TMA
    Ring ring(p.slots), y_ring(p.ys);
    int sent = 0, y_sent = 0, id[4];
    auto read_ids = [&](const Run& t, int row) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        id[i] = -1;
        if (row + 4 * lane + i < t.row + t.n) id[i] = __ldg(p.ids + row + 4 * lane + i);
      }
    };
    for (Run cur = after_live(none); cur.n > 0; cur = after_live(cur))
    for (int row = cur.row; row < cur.row + cur.n; row += kTile, ring.next()) {
      const int slot = ring.slot;
      int rows[4];  // gathered rows of x: four a lane, read a tile ahead
      if (SHARED) {
        if (row == cur.row) read_ids(cur, row);
#pragma unroll
        for (int i = 0; i < 4; ++i) rows[i] = id[i];
        read_ids(cur, row + kTile);
      }
      if (ring.turn > 0) WAIT_OR(sent_all, free_(slot), ring.turn - 1);
      if (tc::elected()) {
        const uint32_t to = tc::smem_addr(s_tiles + slot * tile_bytes);
        tc::expect(full(slot), tile_bytes);
        for (int j = 0; j < p.pm; ++j)
          tc::load_box(to + j * kPanel, &map_v, j * 64, row, full(slot));
        if (!SHARED)
          for (int j = 0; j < p.pk; ++j)
            tc::load_box(to + (p.pm + j) * kPanel, &map_x, j * 64, row, full(slot));
      }
      __syncwarp();
      for (int j = 0; SHARED && j < p.pk; ++j)
        tc::load_rows4(tc::smem_addr(s_tiles + slot * tile_bytes) + (p.pm + j) * kPanel + lane * 512,
                       &map_x, j * 64, rows, full(slot));
      __syncwarp();
      ++sent;
      for (int j = 0; HAS_Y && j < p.pm; ++j, y_ring.next()) {
        const int ys = y_ring.slot;
        if (y_ring.turn > 0) WAIT_OR(sent_all, y_free(ys), y_ring.turn - 1);
        if (tc::elected()) {
          tc::expect(y_full(ys), kPanel);
          tc::load_box(tc::smem_addr(s_y + ys * kPanel), &map_y, j * 64, row, y_full(ys));
        }
        __syncwarp();
        ++y_sent;
      }
    }
  sent_all:
    drain_ring(sent, p.slots, full);
    if (HAS_Y) drain_ring(y_sent, p.ys, y_full);
  } else if (warp == 16) {
    // ------------------------------------------------------------- MMAs
    const uint32_t by_rows = tc::instr_desc(Mma<T>::format, (K + 15) / 16 * 16) | tc::kMnMajorB;
    const uint32_t by_sums = tc::instr_desc(Mma<T>::format, (M + 15) / 16 * 16) |
                             tc::kMnMajorA | tc::kMnMajorB;
    const uint32_t leader = tc::elected();
    const uint32_t k_blocks = p.pk > 1 ? kPanel : 0;  // to the next 64 columns
    const int steps = (M + 15) / 16;
    Ring ring(p.slots);
    int stagings = 0, ys = 0, t = 0, piece = 0, sums = 0;
    for (Run cur = after_live(none); cur.n > 0; cur = after_live(cur))
    for (int left = cur.n; left > 0; left -= kTile, ++t, ring.next()) {
      const int slot = ring.slot;
      char* const vz = s_tiles + slot * tile_bytes;
      const uint32_t v_at = tc::smem_addr(vz), x_at = v_at + p.pm * kPanel;
      const uint32_t low_at = tc::smem_addr(s_y + ys * kPanel);  // whole tiles: ys % pm == 0
      WAIT_OR(mma_done, ready(slot), ring.turn);
      if (p.vx) {
        if (left == cur.n) WAIT_OR(mma_done, weighed, stagings++);
        const int buf = NBUF == 2 ? t & 1 : 0;
        if (t >= NBUF) WAIT_OR(mma_done, taken(buf), t / NBUF - 1);
        tc::fence_after_sync();
        const uint32_t acc = tmem + buf * TERMS * nk;
        for (int i = 0; i < steps; ++i) {  // 16 of M: 32 bytes of a row, 16 rows of weights
          const uint32_t at = (i >> 2) * kPanel + (i & 3) * 32;
          const uint64_t dw = tc::smem_desc_mn(tc::smem_addr(s_w) + i * 2048, k_blocks);
          tc::mma<false>(leader, acc, tc::smem_desc(v_at + at), dw, by_rows, i > 0);
          if (TERMS == 2)
            tc::mma<false>(leader, acc + nk, tc::smem_desc(low_at + at), dw, by_rows, i > 0);
        }
        tc::commit(leader, made(buf));
      }
      const int sum_buf = NBUF == 2 ? sums & 1 : 0;
      if (piece == 0 && sums >= NBUF) WAIT_OR(mma_done, sum_taken(sum_buf), sums / NBUF - 1);
      tc::fence_after_sync();
      const uint32_t sum = sum_acc + sum_buf * nm;
#pragma unroll
      for (int i = 0; i < 8; ++i) {        // 16 rows
        const uint64_t dx = tc::smem_desc_mn(x_at + i * 2048, k_blocks);
        tc::mma<false>(leader, sum, dx, tc::smem_desc_mn(v_at + i * 2048, kPanel), by_sums,
                       piece > 0 || i > 0);
        if (TERMS == 2)
          tc::mma<false>(leader, sum + nm, dx, tc::smem_desc_mn(low_at + i * 2048, kPanel),
                         by_sums, piece > 0 || i > 0);
      }
      tc::commit(leader, free_(slot));
      for (int j = 0; TERMS == 2 && j < p.pm; ++j) tc::commit(leader, y_free(ys + j));
      if (++piece == kPiece || left <= kTile) {
        tc::commit(leader, sum_made(sum_buf));
        ++sums;
        piece = 0;
      }
      ys = ys + p.pm >= p.ys ? 0 : ys + p.pm;
    }
  mma_done:
    tc::commit(leader, drained);  // every MMA is done before the memory goes
    drain(drained, 0);
  } else if (warp < 8) {
    // ------------------------------------------------------------ front warps
    const int tid = threadIdx.x;
    const T* const w = static_cast<const T*>(p.w);
    const int c16 = tid & 7, r16 = tid >> 3;
    const uint32_t o16 = chunk_at(r16, c16);
    auto stage_weights = [&](int g) {  // rows of M, as they are
      const T* const wg = w + (int64_t)g * M * K;
      uint4 q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int m = r16 + 32 * (i & 3), c = (i >> 2) * 64 + c16 * 8;
        const bool in = m < M && c < K;
        q[i] = get_chunk<T, true>(in ? wg + (int64_t)m * K + c : wg, in);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >> 2 < p.pk)
          *reinterpret_cast<uint4*>(s_w + (i >> 2) * kPanel + o16 + 4096 * (i & 3)) = q[i];
    };
    float db[2][8];
#pragma unroll
    for (int i = 0; i < 16; ++i) db[i >> 3][i & 7] = 0.0f;
    Ring ring(p.slots), y_ring(p.ys);
    int t = 0;
    Run cur;
    for (cur = after_live(none); cur.n > 0; cur = after_live(cur))
    for (int left = cur.n; left > 0; left -= kTile, ++t, ring.next()) {
      const int slot = ring.slot;
      if (p.vx && left == cur.n) {
        if (t > 0) WAIT_OR(walk, free_(ring.slot_before(1)), ring.turn_before(1));
        stage_weights(cur.g);
        tc::fence_smem();
        __syncwarp();
        if (lane == 0) tc::arrive(weighed);
      }
      WAIT_OR(walk, full(slot), ring.turn);
      char* const vz = s_tiles + slot * tile_bytes;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (j >= p.pm) break;
        const int ys = y_ring.slot;
        char* const yt = s_y + ys * kPanel - j * kPanel;
        if (HAS_Y) WAIT_OR(walk, y_full(ys), y_ring.turn);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t o = j * kPanel + o16 + 4096 * i;
          const bool in = r16 + 32 * i < left;  // rows behind are another group's
          Chunk<T> v, z;
          v.q = *reinterpret_cast<const uint4*>(vz + o);
          if (HAS_Y) z.q = *reinterpret_cast<const uint4*>(yt + o);
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = in ? through<ACT>(to_f(v.v[e]), HAS_Y ? to_f(z.v[e]) : 0.0f) : 0.0f;
            db[j][e] += f[e];
          }
          if (TERMS == 2) {
            put_chunk<T, true>(vz + o, yt - vz, f);
          } else if (HAS_Y || !in) {  // exact: v_y or 0
            *reinterpret_cast<uint4*>(vz + o) = round_chunk<T>(f);
          }
        }
        if (HAS_Y) {
          if (TERMS == 1) {
            tc::fence_smem();  // read before TMA writes there again
            __syncwarp();
            if (lane == 0) tc::arrive(y_free(ys));
          }
          y_ring.next();
        }
      }
      if (!SHARED && left < kTile) {  // nor may what x has there be multiplied, even by zeros
        for (int i = 0; i < 4; ++i)
          if (r16 + 32 * i >= left)
            for (int j = 0; j < p.pk; ++j)
              *reinterpret_cast<uint4*>(vz + (p.pm + j) * kPanel + o16 + 4096 * i) =
                  make_uint4(0, 0, 0, 0);
      }
      tc::fence_smem();
      __syncwarp();
      if (lane == 0) tc::arrive(ready(slot));
      if (left <= kTile) {  // the group's v_b, summed in a fixed order
        if (p.biases) {
          float* const to = p.part + (int64_t)(blockIdx.x + cur.g) * ((int64_t)M * (K + 1)) +
                            (int64_t)M * K;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              float b = db[j][e];
              b += __shfl_xor_sync(0xffffffffu, b, 8);
              b += __shfl_xor_sync(0xffffffffu, b, 16);
              if (lane < 8) s_db[warp][lane * 8 + e] = b;
            }
            tc::bar_sync(1, kThreads);
            if (tid < 64 && j * 64 + tid < M) {
              float b = 0.0f;
#pragma unroll
              for (int i = 0; i < 8; ++i) b += s_db[i][tid];
              to[j * 64 + tid] = b;
            }
            tc::bar_sync(1, kThreads);
          }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) db[i >> 3][i & 7] = 0.0f;
      }
    }
  walk:
    // behind a wait that gave up: the other front warps still meet this one
    for (; p.biases && cur.n > 0; cur = after_live(cur))
      for (int i = 0; i < 4; ++i) tc::bar_sync(1, kThreads);
  } else {
    // ------------------------------------------------------------- back warps
    constexpr int MODE = SHARED ? kScatter : kBackward;
    const int bw = warp - 8, row0 = (bw & 3) * 32;
    int t = 0, piece = 0, sums = 0;
    bool first = true;  // of the group
    for (Run cur = after(none); cur.n > 0; cur = after(cur))
    for (int left = cur.n; left > 0; left -= kTile) {
      const bool live = cur.g >= 0 && cur.g < p.s.G;
      const int row = cur.row + cur.n - left + row0;  // this warp's first
      const int rows = min(32, left - row0), buf = NBUF == 2 ? t & 1 : 0;
      if (p.vx) {
        int into = -1;
        if (SHARED && live && lane < rows) into = __ldg(p.ids + row + lane);
        if (live) {
          WAIT_OR(taken_all, made(buf), t / NBUF);
          tc::fence_after_sync();
        }
        if (into >= p.s.n) into = -1;
        if (!SHARED || live)
          take_results<T, ACT, MODE, TERMS>(live, tmem + buf * TERMS * nk + ((uint32_t)row0 << 16),
                                            nk, bw >> 2, rows, p.vx_width, nullptr, into,
                                            s_stage + bw * 2048, p.vx, SHARED ? 0 : row,
                                            p.vx_width, 0, p.wide_out);
        if (live) {
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::arrive(taken(buf));
        }
      }
      if (live) {
        ++t;
        const bool last = left <= kTile;
        if (++piece == kPiece || last) {
          const int sum_buf = NBUF == 2 ? sums & 1 : 0;
          WAIT_OR(taken_all, sum_made(sum_buf), sums / NBUF);
          tc::fence_after_sync();
          const uint32_t sum = sum_acc + sum_buf * nm + ((uint32_t)row0 << 16);
          float* const to = p.part + (int64_t)(blockIdx.x + cur.g) * ((int64_t)M * (K + 1));
          const int kk = row0 + lane;
          for (int c0 = (bw >> 2) * 16; c0 < M; c0 += 32) {
            float v[16];
            tc::load16(sum + c0, v);
            if (TERMS == 2) {
              float u[16];
              tc::load16(sum + nm + c0, u);
              join_parts<T>(v, u);
            }
            if (kk < K) add_piece(to + (int64_t)c0 * K + kk, K, M - c0, v, first);
          }
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::arrive(sum_taken(sum_buf));
          ++sums;
          piece = 0;
          first = last;
        }
      }
    }
  taken_all:;
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 0) tc::dealloc(tmem, columns);
}

// v_W and v_b of a group: the places of the CTAs that had rows of it, in
// order; a place has mp x kp sums, of which M x K are wanted, and `copies`
// rows of mp sums.  A block takes 256 / SHARES values; its warps take a share of the
// places each, and the shares are added in order.
template <typename T, int SHARES>
__global__ void __launch_bounds__(256) join_kernel(Shape s, int kp, int mp, int parts, int copies,
                                                   const int32_t* __restrict__ off,
                                                   const float* __restrict__ part,
                                                   T* __restrict__ vw, T* __restrict__ vb) {
  constexpr int VALUES = 256 / SHARES;
  __shared__ float s_sum[SHARES][VALUES];
  const int share = threadIdx.x / VALUES, at = threadIdx.x % VALUES;
  const int64_t mk = (int64_t)s.M * s.K, each = mk + s.M;
  const int64_t sums = (int64_t)mp * kp, place = sums + (int64_t)copies * mp;
  const int64_t i = (int64_t)blockIdx.x * VALUES + at;
  const int64_t in_place = i >= mk ? sums + (i - mk) : kp == s.K ? i : i / s.K * kp + i % s.K;
  const int64_t tiles = (s.R + kTile - 1) / kTile;
  auto part_of = [&](int64_t r) { return (int)(((r / kTile + 1) * parts - 1) / tiles); };
  for (int64_t g = blockIdx.y; g < s.G; g += gridDim.y) {
    const int64_t r0 = max((int64_t)__ldg(off + g), (int64_t)0);
    const int64_t r1 = min((int64_t)__ldg(off + g + 1), s.R);
    float sum = 0.0f;
    if (r0 < r1 && i < each) {
      const int b0 = part_of(r0), n = part_of(r1 - 1) - b0 + 1;
      const int from = n * share / SHARES, to = n * (share + 1) / SHARES;
      const float* p = part + (b0 + g + from) * place + in_place;
      if (i < mk) {
#pragma unroll 8
        for (int b = from; b < to; ++b, p += place) sum += __ldg(p);
      } else {
        for (int b = from; b < to; ++b, p += place)
          for (int c = 0; c < copies; ++c) sum += __ldg(p + (int64_t)c * mp);
      }
    }
    if (SHARES > 1) {
      __syncthreads();
      s_sum[share][at] = sum;
      __syncthreads();
#pragma unroll
      for (int w = 1; w < SHARES; ++w) sum += share == 0 ? s_sum[w][at] : 0.0f;
    }
    if (share == 0 && i < each) {
      if (i < mk) {
        if (vw) vw[g * mk + i] = from_f<T>(sum);
      } else if (vb) {
        vb[g * s.M + (i - mk)] = from_f<T>(sum);
      }
    }
  }
}

// --------------------------------------------------------- few outputs (colours)
//
// Up to 8 outputs (a colour has 3) and rows of up to 512 bytes: a tensor-core
// tile would be nearly all padding (32-3 fp32: 16 MMAs of 128 x 16 a panel took
// 1000 cycles, the panel's 16 KB come in 370).  Here `lpr` neighbouring lanes
// take a row, 16 bytes each; a lane keeps its columns of the group's weights
// in registers, and of v_W's sums in the backward, which does all of its parts
// in the one pass.  A warp has 16 / MP rows per lane in flight.
//
// 4 M gathered rows 32-3 fp32: 127 us (as tensor-core tiles 278).  The 128-byte row
// reads alone take 94 us, 5.4 TB/s; the rest is that a warp loads and uses its
// rows in the same turn, with nothing under way while it adds up (7% fewer
// instructions changed nothing).  Its backward, 1.2 M rows: 163 us.
struct NarrowArgs {
  Shape s;
  const void* x;
  const int32_t* ids;
  const int32_t* off;
  const void* w;
  const void* bias;
  void* y;             // written by the forward, read by the backward
  const void* vy;
  void* vx;            // v_x, its fp32 sums with row ids, or NULL
  float* part;         // as in WeightArgs, or NULL
  int lpr;             // a power of two
  int act;
};

__device__ __forceinline__ float activate_as(int act, float z) {
  return act == GS_ACT_RELU ? activate<GS_ACT_RELU>(z)
                            : act == GS_ACT_SIGMOID ? activate<GS_ACT_SIGMOID>(z) : z;
}
__device__ __forceinline__ float through_as(int act, float v, float y) {
  return act == GS_ACT_RELU ? through<GS_ACT_RELU>(v, y)
                            : act == GS_ACT_SIGMOID ? through<GS_ACT_SIGMOID>(v, y) : v;
}

// The spans of this CTA's rows that belong together, and this lane's place.
#define NARROW_SETUP                                                                        \
  constexpr int E = Chunk<T>::E, U = 16 / MP;                                               \
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;                               \
  const int K = p.s.K, M = p.s.M;                                                           \
  const int c = lane & (p.lpr - 1), rg = lane / p.lpr, set = 32 / p.lpr; /* rows at once */ \
  const T* const x = static_cast<const T*>(p.x);                                            \
  const T* const w = static_cast<const T*>(p.w);                                            \
  const int there = K - c * E; /* columns of this lane: none, some or E */                  \
  const int64_t tiles = (p.s.R + kTile - 1) / kTile;                                        \
  const int end = (int)min(p.s.R, first_tile(tiles, gridDim.x, blockIdx.x + 1) * kTile);    \
  Run none;                                                                                 \
  none.row = (int)(first_tile(tiles, gridDim.x, blockIdx.x) * kTile);                       \
  none.n = 0, none.g = -1, none.group_end = 0;                                              \
  auto after = [&](const Run& t) {                                                          \
    return run_from(p.off, p.s.G, t.row + t.n, end, INT_MAX, t);                            \
  };                                                                                        \
  float wk[MP][E];                                                                          \
  auto read_weights = [&](int g) {                                                          \
    _Pragma("unroll") for (int m = 0; m < MP; ++m) {                                        \
      Chunk<T> q;                                                                           \
      q.q = get_chunk<T, WIDE>(w + ((int64_t)g * M + (m < M ? m : 0)) * K +                 \
                                   (there > 0 ? c * E : 0), m < M ? there : 0);             \
      _Pragma("unroll") for (int e = 0; e < E; ++e) wk[m][e] = to_f(q.v[e]);                \
    }                                                                                       \
  };                                                                                        \
  int id[U];                                                                                \
  auto read_ids = [&](int r, int stop) { /* no use of what is read yet */                   \
    _Pragma("unroll") for (int u = 0; u < U; ++u) {                                         \
      const int row = r + u * set + rg;                                                     \
      id[u] = -1;                                                                           \
      if (row < stop) {                                                                     \
        if (p.ids) id[u] = __ldg(p.ids + row);                                              \
        else id[u] = row;                                                                   \
      }                                                                                     \
    }                                                                                       \
  };

// A lane keeps H of its 2 H values, with the partner's share of them.
template <int H>
__device__ __forceinline__ void hand_over(float (&v)[16], bool up, int o) {
#pragma unroll
  for (int i = 0; i < H; ++i) {
    const float mine = up ? v[i + H] : v[i];
    v[i] = mine + __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + H], o);
  }
}

template <typename T, int MP, bool WIDE>
__global__ void __launch_bounds__(256, MP == 4 && sizeof(T) == 4 ? 4 : 2)
    narrow_fwd_kernel(NarrowArgs p) {
  NARROW_SETUP
  const T* const bias = static_cast<const T*>(p.bias);
  T* const y = static_cast<T*>(p.y);
  // A row's lanes end up with 16 / lpr of its U x MP values each: lane c with
  // those from c 16 / lpr on, n of them (of 32 lanes every second has one).
  const int n = p.lpr > 16 ? 1 - (lane & 1) : 16 / p.lpr;
  const int first = p.lpr > 16 ? c >> 1 : c * (16 / p.lpr);
  const int m0 = first % MP, u0 = first / MP;
  for (Run cur = after(none); cur.n > 0; cur = after(cur)) {
    const int stop = cur.row + cur.n;
    if (cur.g < 0 || cur.g >= p.s.G) {
      for (int64_t i = (int64_t)cur.row * M + threadIdx.x; i < (int64_t)stop * M; i += 256)
        y[i] = from_f<T>(0.0f);
      continue;
    }
    read_weights(cur.g);
    float b[MP];  // of the values that this lane ends up with
#pragma unroll
    for (int i = 0; i < MP; ++i) {
      const int m = n < MP ? m0 + i : i;
      b[i] = bias && m < M ? to_f(__ldg(bias + (int64_t)cur.g * M + m)) : 0.0f;
    }
    int r = cur.row + warp * U * set;
    read_ids(r, stop);
    for (; r < stop; r += 8 * U * set) {
      Chunk<T> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const bool ok = id[u] >= 0 && id[u] < p.s.n && there > 0;
        q[u].q = get_chunk<T, WIDE>(x + (ok ? (int64_t)id[u] * K + c * E : 0), ok ? there : 0);
      }
      read_ids(r + 8 * U * set, stop);
      float v[16];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int m = 0; m < MP; ++m) {
          float a = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) a = fmaf(to_f(q[u].v[e]), wk[m][e], a);
          v[u * MP + m] = a;
        }
      // The row's lanes add up their parts; each step a lane hands half of its
      // values to the partner and adds the partner's other half.
      if (p.lpr > 1) hand_over<8>(v, lane & (p.lpr >> 1), p.lpr >> 1);
      if (p.lpr > 2) hand_over<4>(v, lane & (p.lpr >> 2), p.lpr >> 2);
      if (p.lpr > 4) hand_over<2>(v, lane & (p.lpr >> 3), p.lpr >> 3);
      if (p.lpr > 8) hand_over<1>(v, lane & (p.lpr >> 4), p.lpr >> 4);
      if (p.lpr > 16) v[0] += __shfl_xor_sync(0xffffffffu, v[0], 1);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (i >= n) break;
        // (n values of one row, or whole rows)
        const int m = n < MP ? m0 + i : i % MP, row = r + (u0 + i / MP) * set + rg;
        if (m < M && row < stop)
          y[(int64_t)row * M + m] = from_f<T>(activate_as(p.act, v[i] + b[i % MP]));
      }
    }
  }
}

// E values to p, `there` of them.
template <typename T, bool WIDE>
__device__ __forceinline__ void set_chunk(T* p, const float* f, int there) {
  constexpr int E = Chunk<T>::E;
  if (WIDE) {
    if (there > 0) {
      if constexpr (E == 4)
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
      else
        *reinterpret_cast<uint4*>(p) = round_chunk<T>(f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < there) p[e] = from_f<T>(f[e]);
  }
}

template <typename T, int MP, bool WIDE>
__global__ void __launch_bounds__(256, 2) narrow_bwd_kernel(NarrowArgs p) {
  NARROW_SETUP
  __shared__ float s_part[8][32];
  const T* const y = static_cast<const T*>(p.y);
  const T* const vy = static_cast<const T*>(p.vy);
  for (Run cur = after(none); cur.n > 0; cur = after(cur)) {
    const int stop = cur.row + cur.n;
    if (cur.g < 0 || cur.g >= p.s.G) {
      if (p.vx && !p.ids)
        for (int64_t i = (int64_t)cur.row * K + threadIdx.x; i < (int64_t)stop * K; i += 256)
          static_cast<T*>(p.vx)[i] = from_f<T>(0.0f);
      continue;
    }
    read_weights(cur.g);
    float sum[MP][E], db[MP];
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      db[m] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) sum[m][e] = 0.0f;
    }
    int r = cur.row + warp * U * set;
    read_ids(r, stop);
    for (; r < stop; r += 8 * U * set) {
      Chunk<T> q[U];
      float vz[U][MP];
      bool ok[U];
      int64_t to[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int row = r + u * set + rg;
        ok[u] = id[u] >= 0 && id[u] < p.s.n && there > 0;
        to[u] = ok[u] ? (int64_t)id[u] * K + c * E : 0;
        if (p.part) q[u].q = get_chunk<T, WIDE>(x + to[u], ok[u] ? there : 0);
#pragma unroll
        for (int m = 0; m < MP; ++m) {
          const bool in = m < M && row < stop;
          const int64_t at = in ? (int64_t)row * M + m : 0;
          vz[u][m] = in ? to_f(vy[at]) : 0.0f;
          if (p.act) vz[u][m] = in ? through_as(p.act, vz[u][m], to_f(y[at])) : 0.0f;
        }
      }
      read_ids(r + 8 * U * set, stop);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p.vx && ok[u]) {
          float f[E];
#pragma unroll
          for (int e = 0; e < E; ++e) {
            f[e] = 0.0f;
#pragma unroll
            for (int m = 0; m < MP; ++m) f[e] = fmaf(vz[u][m], wk[m][e], f[e]);
          }
          if (!p.ids) {
            set_chunk<T, WIDE>(static_cast<T*>(p.vx) + to[u], f, there);
          } else {
            float* const at = static_cast<float*>(p.vx) + to[u];
#pragma unroll
            for (int e = 0; e < E; e += 4) {
              if (WIDE) {  // 16 bytes of T: K is a multiple of 4, and the sums are aligned
                asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};"
                             ::"l"(at + e), "f"(f[e]), "f"(f[e + 1]), "f"(f[e + 2]), "f"(f[e + 3])
                             : "memory");
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (e + i < there) atomicAdd(at + e + i, f[e + i]);
              }
            }
          }
        }
      }
      if (p.part) {  // these rows first: a long sum takes a quarter of the additions
#pragma unroll
        for (int m = 0; m < MP; ++m) {
          float b = vz[0][m];
#pragma unroll
          for (int u = 1; u < U; ++u) b += vz[u][m];
          db[m] += b;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            float a = vz[0][m] * to_f(q[0].v[e]);
#pragma unroll
            for (int u = 1; u < U; ++u) a = fmaf(vz[u][m], to_f(q[u].v[e]), a);
            sum[m][e] += a;
          }
        }
      }
    }
    if (!p.part) continue;
    // over the warp's rows, then over the warps, in order
    float* const place = p.part + (int64_t)(blockIdx.x + cur.g) * ((int64_t)M * (K + 1));
#pragma unroll
    for (int m = 0; m < MP; ++m) {
      if (m >= M) break;
#pragma unroll
      for (int e = 0; e <= E; ++e) {  // E: v_b
        float a = e < E ? sum[m][e < E ? e : 0] : db[m];
        for (int o = p.lpr; o < 32; o <<= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        __syncthreads();
        s_part[warp][lane] = a;
        __syncthreads();
        if (warp == 0 && rg == 0) {
#pragma unroll
          for (int i = 1; i < 8; ++i) a += s_part[i][lane];
          if (e < E && e < there) place[(int64_t)m * K + c * E + e] = a;
          if (e == E && c == 0) place[(int64_t)M * K + m] = a;
        }
      }
    }
  }
}

// 16-bit rows of `width` values, `rows` of each `groups`, to rows of `wide`
// (a multiple of 8), `tall` of each group: what is added is zero.
template <typename T>
__global__ void __launch_bounds__(256) pad_kernel(int64_t groups, int64_t rows, int64_t tall,
                                                  int width, int wide, const T* __restrict__ a,
                                                  T* __restrict__ b) {
  const int chunks = wide / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < groups * tall * chunks;
       i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / chunks, g = groups > 1 ? row / tall : 0;
    const int c = (int)(i - row * chunks) * 8;
    const bool in = row - g * tall < rows;
    const int64_t from = in ? (row - g * (tall - rows)) * width + c : 0;
    reinterpret_cast<uint4*>(b)[i] = get_chunk<T, false>(a + from, in ? width - c : 0);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) round_kernel(int64_t n, const float* __restrict__ a,
                                                    T* __restrict__ b) {
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    b[i] = from_f<T>(a[i]);
}

// ------------------------------------------------------------------- host side
bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Dynamic shared memory of a CTA that has an SM to itself, beside its static
// arrays.
constexpr int kSmemMost = 227 * 1024 - 5120;

// Lets a kernel use `bytes` of dynamic shared memory on the current device; asked once for
// each kernel (the instantiation is the kernel's own) and device.
template <auto kernel, int bytes = kSmemMost>
int allow_smem() {
  static bool done[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
    return launch_status("grouped_linear");
  if (!done[dev]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        cudaSuccess)
      return launch_status("grouped_linear");
    done[dev] = true;
  }
  return GS_OK;
}

// A map of rows [n, depth] in boxes of `tall` rows x 128 bytes, swizzled as
// the operands are; what lies outside reads as zeros.
int make_map(CUtensorMap* map, const void* rows, int dtype, int64_t n, int depth,
             int tall = kTile) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                              const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (!encode) {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) !=
            cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      set_error("grouped_linear: no cuTensorMapEncodeTiled in this driver");
      return GS_ERR_CUDA;
    }
    encode = reinterpret_cast<Encode>(f);
  }
  const cuuint64_t es = dtype == GS_F32 ? 4 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)depth, (cuuint64_t)n}, pitch[1] = {depth * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)tall}, ones[2] = {1, 1};
  const CUtensorMapDataType type = dtype == GS_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == GS_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                      : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (encode(map, type, 2, const_cast<void*>(rows), dims, pitch, box, ones,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) !=
      CUDA_SUCCESS) {
    set_error("grouped_linear: rows [%lld, %d] cannot be mapped", (long long)n, depth);
    return GS_ERR_CUDA;
  }
  return GS_OK;
}

template <typename T> constexpr int dtype_of = GS_F32;
template <> constexpr int dtype_of<__nv_bfloat16> = GS_BF16;
template <> constexpr int dtype_of<__half> = GS_F16;

template <typename T, int ACT, int MODE, int LOAD, bool WIDE, bool SPLIT>
int launch_rows(RowsArgs p, cudaStream_t st) {
  using L = RowsLayout<T, ACT, MODE, SPLIT>;
  constexpr auto kernel = rows_mma_kernel<T, ACT, MODE, LOAD, WIDE, SPLIT>;
  if (int rc = allow_smem<kernel>()) return rc;
  p.panels = (int)ceil_div(p.depth, 128 / (int)sizeof(T));
  // The widest tile whose weights stay in shared memory: half the width
  // reads the rows twice, which costs less than staging the weights again
  // for every tile.
  const int widest = p.width >= 128 ? 128 : (int)ceil_div(p.width, 32) * 32;
  p.nt = widest;
  p.slots = 2;
  p.resident = 1;
  while (L::smem(p) > kSmemMost && p.nt > 32) p.nt = (p.nt / 2 + 31) / 32 * 32;
  if (L::smem(p) > kSmemMost) p.resident = 0, p.nt = widest;
  // as many panels in flight as there is room for
  while (p.slots < kSlotsMost) {
    ++p.slots;
    if (L::smem(p) > kSmemMost) {
      --p.slots;
      break;
    }
  }
  const int64_t ny = ceil_div(p.width, p.nt);
  const int64_t tiles = ceil_div(p.s.R, kTile);
  int64_t nx = sm_count() / ny;
  nx = nx < 1 ? 1 : nx > tiles ? tiles : nx;
  CUtensorMap map_a{}, map_y{};
  if (LOAD == kTma) {
    if (int rc = make_map(&map_a, p.a, dtype_of<T>, p.s.R, p.depth)) return rc;
    if (L::kY)
      if (int rc = make_map(&map_y, p.y, dtype_of<T>, p.s.R, p.depth)) return rc;
  }
  kernel<<<dim3((unsigned)nx, (unsigned)ny), LOAD == kGather ? kCta : kCta - kLoaders,
           L::smem(p), st>>>(
      p, L::columns(p.nt), map_a, map_y);
  return launch_status("grouped_linear");
}

template <typename T, int ACT, int MODE, bool SPLIT>
int launch_rows(const RowsArgs& p, cudaStream_t st) {
  const bool wide = p.depth * sizeof(T) % 16 == 0 && on16(p.a) && (!p.y || on16(p.y)) &&
                    p.s.n > 0;  // there is no address in an empty x
  if (!wide) return launch_rows<T, ACT, MODE, kCopy, false, SPLIT>(p, st);
  if constexpr (MODE == kForward)
    if (p.ids) return launch_rows<T, ACT, MODE, kGather, true, SPLIT>(p, st);
  return launch_rows<T, ACT, MODE, kTma, true, SPLIT>(p, st);
}

template <typename T>
int launch_narrow(NarrowArgs p, bool backward, int parts, cudaStream_t st) {
  const int chunks = (int)ceil_div(p.s.K, 16 / (int)sizeof(T));
  p.lpr = 1;
  while (p.lpr < chunks) p.lpr *= 2;
  const bool wide = p.s.K * sizeof(T) % 16 == 0 && on16(p.x) && on16(p.w) && (!p.vx || on16(p.vx));
  const dim3 grid((unsigned)parts);
  if (backward) {
    if (p.s.M <= 4) {
      if (wide) narrow_bwd_kernel<T, 4, true><<<grid, 256, 0, st>>>(p);
      else narrow_bwd_kernel<T, 4, false><<<grid, 256, 0, st>>>(p);
    } else if constexpr (sizeof(T) == 4) {
      if (wide) narrow_bwd_kernel<T, 8, true><<<grid, 256, 0, st>>>(p);
      else narrow_bwd_kernel<T, 8, false><<<grid, 256, 0, st>>>(p);
    }
  } else if (p.s.M <= 4) {
    if (wide) narrow_fwd_kernel<T, 4, true><<<grid, 256, 0, st>>>(p);
    else narrow_fwd_kernel<T, 4, false><<<grid, 256, 0, st>>>(p);
  } else {
    if (wide) narrow_fwd_kernel<T, 8, true><<<grid, 256, 0, st>>>(p);
    else narrow_fwd_kernel<T, 8, false><<<grid, 256, 0, st>>>(p);
  }
  return launch_status("grouped_linear");
}

template <typename T, int ACT>
int run_fwd(const Shape& s, const WaitArgs& waits, const void* x, const int32_t* ids,
            const int32_t* off, const void* w, const void* b, void* y, cudaStream_t st) {
  if (is_narrow(s.K, s.M, dtype_of<T>, false)) {
    NarrowArgs p{};
    p.s = s;
    p.x = x, p.ids = ids, p.off = off, p.w = w, p.bias = b, p.y = y, p.act = ACT;
    const int64_t tiles = ceil_div(s.R, kTile), most =
        (int64_t)sm_count() * (s.M <= 4 && sizeof(T) == 4 ? 4 : 2);
    return launch_narrow<T>(p, false, (int)(tiles < most ? tiles : most), st);
  }
  RowsArgs p{};
  p.s = s;
  p.a = x, p.ids = ids, p.off = off, p.w = w, p.bias = b, p.out = y;
  p.depth = s.K, p.width = s.M;
  p.waits = waits;
  p.wide_w = s.K * sizeof(T) % 16 == 0 && on16(w);
  p.wide_out = s.M * sizeof(T) % 16 == 0 && on16(y);
  return launch_rows<T, ACT, kForward, false>(p, st);
}

template <int ACT, int NT>
int launch_weights32(const Shape& s, const void* x, const void* y, const void* vy,
                     const int32_t* ids, const int32_t* off, float* part, const void* vb,
                     const WaitArgs& waits, const Plan& q, cudaStream_t st) {
  constexpr auto kernel = weights32_kernel<ACT, NT>;
  constexpr int kAll = 227 * 1024;  // this kernel has no static shared memory
  if (int rc = allow_smem<kernel, kAll>()) return rc;
  Weight32Args p{};
  p.s = s;
  p.x = static_cast<const float*>(x), p.y = static_cast<const float*>(y);
  p.vy = static_cast<const float*>(vy), p.ids = ids, p.off = off, p.part = part;
  p.kt = q.kt, p.biases = vb != nullptr, p.waits = waits;
  p.kx = ((s.K < 128 ? s.K : 128) + 31) / 32, p.mx = ((s.M < NT ? s.M : NT) + 31) / 32;
  const bool wide_x = s.K % 4 == 0 && on16(x);
  p.x_mode = wide_x && s.n > 0 ? (ids ? 1 : 0) : 2;
  p.v_mode = s.M % 4 == 0 && on16(vy) && (!y || on16(y)) ? 0 : 2;
  const int set = 2 * (p.kx + p.mx) * kBox, slot = (p.kx + p.mx * (ACT ? 2 : 1)) * kBox;
  const int bars = kBars32 * 8 + 8;
  // an x operand's MMA reads 128 rows from its start on: they lie in the sets
  // and slots behind it
  // Two sets a front group where there is room: the next panel's operands are
  // made while this one's are multiplied (1.2 M rows 64-64: 256 -> 200 us).
  p.sets = (kAll - bars - 4 * set) / slot >= 4 ? 4 : 2;
  const int fixed = p.sets * set + bars;
  p.slots = (kAll - fixed) / slot;
  p.slots = p.slots > 8 ? 8 : p.slots;
  if (p.x_mode == 2 || p.v_mode == 2) p.slots = p.slots / 2 * 2;
  CUtensorMap map_x{}, map_v{}, map_y{};
  if (p.x_mode == 0)
    if (int rc = make_map(&map_x, x, GS_F32, s.n, s.K, kRows32)) return rc;
  if (p.v_mode == 0) {
    if (int rc = make_map(&map_v, vy, GS_F32, s.R, s.M, kRows32)) return rc;
    if (ACT)
      if (int rc = make_map(&map_y, y, GS_F32, s.R, s.M, kRows32)) return rc;
  }
  kernel<<<dim3((unsigned)q.parts, (unsigned)(q.kt * q.mt)), kCta,
           fixed + p.slots * slot, st>>>(p, map_x, map_v, map_y);
  return launch_status("grouped_linear_bwd");
}

template <typename T, int ACT, int NT, bool SPLIT>
int launch_weights(const WeightArgs& p, const Plan& q, cudaStream_t st) {
  constexpr auto kernel = weights_mma_kernel<T, ACT, NT, SPLIT>;
  if (int rc = allow_smem<kernel>()) return rc;
  const int vt = SPLIT ? 2 : 1;
  const int smem = 1024 + kPanel + vt * NT * 128, columns = NT * vt;
  kernel<<<dim3((unsigned)q.parts, (unsigned)(q.kt * q.mt)), kThreads, smem, st>>>(p, columns);
  return launch_status("grouped_linear_bwd");
}

// Whether one kernel can do the whole backward of 16-bit rows.
template <typename T>
bool fits_both(const Shape& s, const void* x, const void* w, const void* y, const void* vy,
               const void* vx) {
  return sizeof(T) == 2 && dims_fit_both(s.K, s.M) && s.R > 0 && s.n > 0 && on16(x) && on16(w) &&
         on16(vy) && (!y || on16(y)) && (!vx || on16(vx));
}

template <typename T, int ACT, bool SHARED>
int launch_both(BothArgs p, const void* x, const void* vy, const void* y, const Plan& q,
                cudaStream_t st) {
  constexpr auto kernel = both_mma_kernel<T, ACT, SHARED>;
  constexpr int kAll = 227 * 1024;  // this kernel has no static shared memory
  if (int rc = allow_smem<kernel, kAll>()) return rc;
  p.pk = p.s.K > 64 ? 2 : 1, p.pm = p.s.M > 64 ? 2 : 1;
  const int terms = ACT == GS_ACT_SIGMOID ? 2 : 1;  // parts of v_z
  // As many tiles as there is room for beside one tile of y, then as many
  // panels of y (whole tiles where the low parts of v_z lie in them).
  p.slots = 2, p.ys = ACT ? p.pm : 0;
  auto smem = [&]() {
    return 8 * 2048 + 2048 + kBothBars * 8 + 8 + kPanel * (p.pk + p.slots * (p.pm + p.pk) + p.ys);
  };
  while (p.slots < 4 && smem() + (p.pm + p.pk) * kPanel <= kAll) ++p.slots;
  const int more = terms == 2 ? p.pm : 1;
  while (ACT && p.ys + more <= 4 && smem() + more * kPanel <= kAll) p.ys += more;
  const int nk = (p.s.K + 31) / 32 * 32, nm = (p.s.M + 31) / 32 * 32;
  int columns = 32;
  while (columns < 2 * nk + 2 * nm) columns *= 2;  // two accumulators, or two parts of one
  CUtensorMap map_v{}, map_y{}, map_x{};
  if (int rc = make_map(&map_v, vy, dtype_of<T>, p.s.R, p.s.M)) return rc;
  if (ACT)
    if (int rc = make_map(&map_y, y, dtype_of<T>, p.s.R, p.s.M)) return rc;
  if (int rc = make_map(&map_x, x, dtype_of<T>, p.s.n, p.s.K, SHARED ? 1 : kTile)) return rc;
  kernel<<<(unsigned)q.parts, 2 * kThreads + 64, smem(), st>>>(p, columns, map_v, map_y, map_x);
  return launch_status("grouped_linear_bwd");
}

template <typename T, int ACT>
int run_bwd(const gs_grouped_params* prm, const Shape& s, const WaitArgs& waits, const void* x,
            const int32_t* ids, const int32_t* off, const void* w, const void* y, const void* vy,
            void* vx, void* vw, void* vb, float* ws, cudaStream_t st) {
  constexpr bool kSplit = sizeof(T) == 2 && ACT == GS_ACT_SIGMOID;
  const Plan q = plan_of(prm);
  if (ACT == GS_ACT_NONE) y = nullptr;
  const bool shared = prm->use_row_ids != 0;
  float* const sum = sizeof(T) == 4 ? static_cast<float*>(vx) : ws + q.part_floats;
  const bool pad = q.padded && (vw || vb) && s.R > 0 && s.n > 0;
  const bool both = pad || (!q.narrow && (vw || vb) && fits_both<T>(s, x, w, y, vy, vx));
  if (q.narrow) {
    if (vx && shared && cudaMemsetAsync(sum, 0, sizeof(float) * s.n * s.K, st) != cudaSuccess)
      return launch_status("grouped_linear_bwd");
    if (s.R > 0) {
      NarrowArgs p{};
      p.s = s;
      p.x = x, p.ids = ids, p.off = off, p.w = w, p.act = ACT, p.vy = vy;
      p.y = const_cast<void*>(y);
      p.vx = !vx ? nullptr : shared ? sum : vx;
      p.part = vw || vb ? ws : nullptr;
      if (int rc = launch_narrow<T>(p, true, q.parts, st)) return rc;
    }
    if (vx && shared && sizeof(T) == 2 && s.n > 0)
      round_kernel<T><<<grid_for(s.n * s.K, 256), 256, 0, st>>>(s.n * s.K, sum,
                                                                static_cast<T*>(vx));
  }
  if constexpr (sizeof(T) == 2) {
    if (both) {
      if (vx && shared && cudaMemsetAsync(sum, 0, sizeof(float) * s.n * s.K, st) != cudaSuccess)
        return launch_status("grouped_linear_bwd");
      BothArgs p{};
      p.s = s;
      p.ids = ids, p.off = off, p.part = ws;
      p.vx = !vx ? nullptr : shared ? sum : vx;
      p.vx_width = s.K, p.waits = waits;
      p.wide_out = s.K * (shared ? 4 : 2) % 16 == 0 && on16(p.vx);
      p.biases = vb != nullptr;
      if (pad) {
        T* const xp = reinterpret_cast<T*>(ws + q.part_floats + q.sum_floats);
        T *const wp = xp + q.pad_x, *const vp = wp + q.pad_w, *const yp = vp + q.pad_v;
        auto copy = [&](int64_t groups, int64_t rows, int64_t tall, int width, int wide,
                        const void* from, T* to) {
          pad_kernel<T><<<grid_for(groups * tall * (wide / 8), 256), 256, 0, st>>>(
              groups, rows, tall, width, wide, static_cast<const T*>(from), to);
        };
        copy(1, s.n, s.n, s.K, q.kp, x, xp);
        copy(s.G, s.M, q.mp, s.K, q.kp, w, wp);
        copy(1, s.R, s.R, s.M, q.mp, vy, vp);
        if (ACT) copy(1, s.R, s.R, s.M, q.mp, y, yp);
        x = xp, w = wp, vy = vp, y = ACT ? yp : nullptr;
        p.s.K = q.kp, p.s.M = q.mp;
      }
      p.w = w;
      const int rc = shared ? launch_both<T, ACT, true>(p, x, vy, y, q, st)
                            : launch_both<T, ACT, false>(p, x, vy, y, q, st);
      if (rc) return rc;
      if (vx && shared && s.n > 0)
        round_kernel<T><<<grid_for(s.n * s.K, 256), 256, 0, st>>>(s.n * s.K, sum,
                                                                  static_cast<T*>(vx));
    }
  }
  if (vx && !both && !q.narrow) {
    if (shared && cudaMemsetAsync(sum, 0, sizeof(float) * s.n * s.K, st) != cudaSuccess)
      return launch_status("grouped_linear_bwd");
    if (s.R > 0) {
      RowsArgs p{};
      p.s = s;
      p.a = vy, p.y = y, p.ids = ids, p.off = off, p.w = w, p.out = shared ? sum : vx;
      p.depth = s.M, p.width = s.K, p.waits = waits;
      const size_t each = shared ? 4 : sizeof(T);
      p.wide_out = s.K * each % 16 == 0 && on16(p.out);
      const int rc = shared ? launch_rows<T, ACT, kScatter, kSplit>(p, st)
                            : launch_rows<T, ACT, kBackward, kSplit>(p, st);
      if (rc) return rc;
    }
    if (shared && sizeof(T) == 2 && s.n > 0)
      round_kernel<T><<<grid_for(s.n * s.K, 256), 256, 0, st>>>(s.n * s.K, sum,
                                                                static_cast<T*>(vx));
  }
  if (vw || vb) {
    if (q.narrow) {
    } else if constexpr (sizeof(T) == 4) {
      if (s.R > 0) {
        const int rc =
            q.nt == 64 ? launch_weights32<ACT, 64>(s, x, y, vy, ids, off, ws, vb, waits, q, st)
                      : launch_weights32<ACT, 128>(s, x, y, vy, ids, off, ws, vb, waits, q, st);
        if (rc) return rc;
      }
    } else if (s.R > 0 && !both) {
      WeightArgs p{};
      p.s = s;
      p.x = x, p.y = y, p.vy = vy, p.ids = ids, p.off = off, p.part = ws;
      p.kt = q.kt, p.mt = q.mt, p.biases = vb != nullptr, p.waits = waits;
      p.wide_x = s.K * sizeof(T) % 16 == 0 && on16(x);
      p.wide_y = s.M * sizeof(T) % 16 == 0 && on16(vy) && (!y || on16(y));
      const int rc = q.nt == 64 ? launch_weights<T, ACT, 64, kSplit>(p, q, st)
                                : launch_weights<T, ACT, 128, kSplit>(p, q, st);
      if (rc) return rc;
    }
    const int64_t each = (int64_t)s.M * (s.K + 1);
    const unsigned gy = s.G < 65535 ? s.G : 65535;
    // a thread a value fills the GPU, or eight warps share a value's places
    // (19 groups 77-45: 20 against 10 us; 32 groups 128-128: 12 against 27)
    if (ceil_div(each, 256) * gy >= 2 * sm_count())
      join_kernel<T, 1><<<dim3((unsigned)ceil_div(each, 256), gy), 256, 0, st>>>(
          s, q.kp, q.mp, q.parts, q.copies, off, ws, static_cast<T*>(vw), static_cast<T*>(vb));
    else
      join_kernel<T, 8><<<dim3((unsigned)ceil_div(each, 32), gy), 256, 0, st>>>(
          s, q.kp, q.mp, q.parts, q.copies, off, ws, static_cast<T*>(vw), static_cast<T*>(vb));
  }
  return launch_status("grouped_linear_bwd");
}

}  // namespace

template <typename T>
int forward(int activation, const Shape& s, const WaitArgs& waits, const void* x,
            const int32_t* ids, const int32_t* off, const void* w, const void* b, void* y,
            cudaStream_t st) {
  if (activation == GS_ACT_NONE)
    return run_fwd<T, GS_ACT_NONE>(s, waits, x, ids, off, w, b, y, st);
  if (activation == GS_ACT_RELU)
    return run_fwd<T, GS_ACT_RELU>(s, waits, x, ids, off, w, b, y, st);
  return run_fwd<T, GS_ACT_SIGMOID>(s, waits, x, ids, off, w, b, y, st);
}

template <typename T>
int backward(const gs_grouped_params* prm, const Shape& s, const WaitArgs& waits, const void* x,
             const int32_t* ids, const int32_t* off, const void* w, const void* y, const void* vy,
             void* vx, void* vw, void* vb, float* ws, cudaStream_t st) {
  if (prm->activation == GS_ACT_NONE)
    return run_bwd<T, GS_ACT_NONE>(prm, s, waits, x, ids, off, w, y, vy, vx, vw, vb, ws, st);
  if (prm->activation == GS_ACT_RELU)
    return run_bwd<T, GS_ACT_RELU>(prm, s, waits, x, ids, off, w, y, vy, vx, vw, vb, ws, st);
  return run_bwd<T, GS_ACT_SIGMOID>(prm, s, waits, x, ids, off, w, y, vy, vx, vw, vb, ws, st);
}

}  // namespace grouped
}  // namespace gsb
