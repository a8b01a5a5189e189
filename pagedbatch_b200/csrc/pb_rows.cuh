// Reading whole logits rows as 16-byte vectors at any alignment, and the sums and launch helpers
// shared by the row-wise operators (top log-probabilities, distillation loss, verification).
#pragma once

#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/pagedbatch_b200.h"
#include "pb_device.cuh"
#include "pb_elem.cuh"

namespace pb {

// A row of V elements seen as nvec aligned 16-byte vectors: vector v holds elements
// [v * EPV - off, (v + 1) * EPV - off), of which those outside [0, V) are not the row's. Only the
// first and the last vector can hold such elements.
template <typename T>
struct RowView {
  static constexpr int EPV = Elem<T>::EPV;
  const T* row;
  int32_t off, V, nvec;
  __device__ RowView(const T* r, int32_t v)
      : row(r), off((int32_t)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T))), V(v) {
    nvec = (off + V + EPV - 1) / EPV;
  }
  __device__ int32_t first(int32_t v) const { return v * EPV - off; }
  __device__ bool whole(int32_t v) const { return first(v) >= 0 && first(v) + EPV <= V; }
};

// Vector v of the row, elements outside it -inf. A whole vector is one 16-byte load; a partial one
// is loaded element by element, so nothing outside the row is read.
template <typename T>
__device__ __noinline__ uint4 part_vec_at(const T* row, int32_t e0, int32_t V) {
  constexpr int EPV = Elem<T>::EPV;
  uint32_t w[4] = {Elem<T>::NEG_INF_WORD, Elem<T>::NEG_INF_WORD, Elem<T>::NEG_INF_WORD, Elem<T>::NEG_INF_WORD};
#pragma unroll
  for (int q = 0; q < EPV; ++q) {
    const int32_t e = e0 + q;
    if (e >= 0 && e < V) {
      if constexpr (EPV == 4) {
        w[q] = __ldg(reinterpret_cast<const uint32_t*>(row) + e);
      } else {
        const uint32_t b = __ldg(reinterpret_cast<const unsigned short*>(row) + e);
        const int sh = (q & 1) * 16;
        w[q >> 1] = (w[q >> 1] & ~(0xFFFFu << sh)) | (b << sh);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A 16-byte load of data that this launch reads once.
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}

template <typename T>
__device__ __forceinline__ uint4 load_vec(const RowView<T>& r, int32_t v) {
  const int32_t e0 = r.first(v);
  if (e0 >= 0 && e0 + Elem<T>::EPV <= r.V) return __ldg(reinterpret_cast<const uint4*>(r.row + e0));
  return part_vec_at<T>(r.row, e0, r.V);
}

// Largest element of a vector as fp32, NaN if it holds one.
template <typename T>
__device__ __forceinline__ float vec_max_nan(uint4 v) {
  return Elem<T>::word_max(Elem<T>::max2(Elem<T>::max2(v.x, v.y), Elem<T>::max2(v.z, v.w)));
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The sum of 2^((x_j - m) c) of some elements, m the largest seen: log2 of the sum of 2^(x_j c) is
// m c + log2(s). The difference is taken before the product, so that rows at the end of the range
// (masks of the type's lowest value) neither overflow nor lose the difference. m starts at the
// lowest finite value, so a set of -inf alone stays an empty sum (s = 0) and not a NaN; a NaN or
// +inf element makes s NaN.
constexpr float LOWEST = -3.402823466e+38f;
struct ExpSum {
  float m, s;
};
__device__ __forceinline__ ExpSum expsum_empty() { return ExpSum{LOWEST, 0.0f}; }
__device__ __forceinline__ ExpSum expsum_join(ExpSum a, ExpSum b, float c) {
  ExpSum r;
  r.m = fmaxf(a.m, b.m);
  r.s = a.s * ex2((a.m - r.m) * c) + b.s * ex2((b.m - r.m) * c);
  return r;
}

// ---- two fp32 operations an instruction (each half rounded as the scalar operation is) ----------

__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// Exponents (x - m) c - l of a vector's elements, in pairs. While |m c| is small, as one fused
// operation x c - RN(m c + l), off by at most 2^-24 (|m c| + |l|) for all elements alike; else the
// difference first, which keeps its precision at any offset and does not overflow.
constexpr float NEAR_ZERO = 64.0f;
struct Exponent {
  float m, c, mc, l;
  __device__ __forceinline__ Exponent(float m_, float c_, float l_ = 0.0f) : m(m_), c(c_), mc(m_ * c_), l(l_) {}
  template <typename T>
  __device__ __forceinline__ void of(uint4 v, uint64_t* e) const {
    constexpr int EPV = Elem<T>::EPV;
    float x[EPV];
    Elem<T>::unpack(v, x);
    const uint64_t c2 = pack2(c, c);
    if (fabsf(mc) <= NEAR_ZERO) {
      const uint64_t n2 = pack2(-(mc + l), -(mc + l));
#pragma unroll
      for (int q = 0; q < EPV / 2; ++q) e[q] = fma2(pack2(x[2 * q], x[2 * q + 1]), c2, n2);
    } else {
      const uint64_t n2 = pack2(-m, -m), l2 = pack2(-l, -l);
#pragma unroll
      for (int q = 0; q < EPV / 2; ++q) e[q] = fma2(add2(pack2(x[2 * q], x[2 * q + 1]), n2), c2, l2);
    }
  }
};

// Largest element of n vectors, NaN if one is.
template <typename T, int N>
__device__ __forceinline__ float vecs_max_nan(const uint4* v) {
  uint4 m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    m.x = Elem<T>::max2(m.x, v[i].x);
    m.y = Elem<T>::max2(m.y, v[i].y);
    m.z = Elem<T>::max2(m.z, v[i].z);
    m.w = Elem<T>::max2(m.w, v[i].w);
  }
  return vec_max_nan<T>(m);
}

// A running sum over vectors, N at a time (one rescale when the maximum grows). The sum is kept as
// two halves, so that additions go in pairs.
struct RunningSum {
  float m;
  uint64_t s;
  __device__ __forceinline__ RunningSum() : m(LOWEST), s(0) {}
  // returns the largest element of the vectors
  template <typename T, int N>
  __device__ __forceinline__ float add(const uint4* v, float c) {
    constexpr int EPV = Elem<T>::EPV;
    const float mx = vecs_max_nan<T, N>(v);
    if (mx > m) {
      const float f = ex2((m - mx) * c);
      s = mul2(s, pack2(f, f));
      m = mx;
    }
    const Exponent ex(m, c);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      uint64_t e[EPV / 2];
      ex.template of<T>(v[j], e);
#pragma unroll
      for (int i = 0; i < EPV / 2; ++i) {
        float lo, hi;
        unpack2(e[i], lo, hi);
        s = add2(s, pack2(ex2(lo), ex2(hi)));
      }
    }
    return mx;
  }
  __device__ __forceinline__ ExpSum total() const {
    float lo, hi;
    unpack2(s, lo, hi);
    return ExpSum{m, lo + hi};
  }
};

// The join of a warp's sums; every lane gets it.
__device__ __forceinline__ ExpSum warp_expsum(ExpSum v, float c) {
  float m = v.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  return ExpSum{m, warp_sum(v.s * ex2((v.m - m) * c))};
}

// The join over the block (NWARP warps), in warp 0's lanes only. `scratch` holds NWARP entries; one
// barrier.
template <int NWARP>
__device__ __forceinline__ ExpSum block_expsum(ExpSum v, float c, ExpSum* scratch) {
  v = warp_expsum(v, c);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x < 32) v = warp_expsum(threadIdx.x < NWARP ? scratch[threadIdx.x] : expsum_empty(), c);
  return v;
}

// ---- segments ---------------------------------------------------------------------------------

// A row is worked on in segments of at most SEG_V vectors for each of a CTA's SEG_T threads: every CTA
// of a grid (rows, segments) takes one, its loads all in flight in registers before anything else is
// done. Small CTAs, SEG_CTAS to an SM, hide each other's latency (40 KB in flight on each SM), and nothing is
// exchanged between them: a launch after this one joins a row's segments. [1024, 128256] bf16 rows are read
// so at 5.7 TB/s, their sums and group keys taken on the way. (Clusters that hold a row in shared memory were
// measured at half this speed: a cluster starts only where all its places are free, and waits for its
// slowest CTA three times a row.)
constexpr int SEG_T = 256;
constexpr int SEG_NW = SEG_T / 32;
constexpr int SEG_V = 8;
constexpr int SEG_CTAS = 5;  // CTAs per SM of the launches that read segments

struct SegPlan {
  int32_t segs, per;  // segments per row, vectors per segment (equal shares of the longest row)
};
inline SegPlan seg_plan(int64_t V, int es, const void* rows, int64_t row_stride) {
  // a row's vectors: exactly, where every row starts on a 16-byte boundary, else the most it can have
  const bool even = reinterpret_cast<uintptr_t>(rows) % 16 == 0 && row_stride * es % 16 == 0;
  const int64_t epv = 16 / es, nvec = even ? (V + epv - 1) / epv : (V + 2 * epv - 2) / epv;
  SegPlan p;
  p.segs = (int32_t)((nvec + SEG_T * SEG_V - 1) / (SEG_T * SEG_V));
  p.per = (int32_t)((nvec + p.segs - 1) / p.segs);
  return p;
}

// This thread's vectors of segment [v0, v1): v0 + i * SEG_T + tid, i < SEG_V; -inf past v1.
template <typename T>
__device__ __forceinline__ void load_segment(const RowView<T>& r, int32_t v0, int32_t v1, uint4* q) {
  constexpr int EPV = Elem<T>::EPV;
  const int32_t mine = v0 + (int32_t)threadIdx.x;
  const T* src = r.row + r.first(mine);
  // vectors [lo, hi) lie whole in the row
  const int32_t lo = r.off ? 1 : 0, hi = (r.off + r.V) / EPV;
  const uint32_t none = Elem<T>::NEG_INF_WORD;
#pragma unroll
  for (int i = 0; i < SEG_V; ++i) {
    const int32_t v = mine + i * SEG_T;
    q[i] = make_uint4(none, none, none, none);
    if (v < v1 && v >= lo && v < hi) q[i] = ld_stream16(src + i * SEG_T * EPV);
  }
  // the row's first and last vector, where it starts or ends inside them
  if (v0 == 0 && threadIdx.x == 0 && r.off) q[0] = part_vec_at<T>(r.row, -r.off, r.V);
  if (v1 == r.nvec && hi < r.nvec && hi >= lo && hi >= mine && ((hi - mine) & (SEG_T - 1)) == 0) {
    const uint4 p = part_vec_at<T>(r.row, r.first(hi), r.V);
#pragma unroll
    for (int i = 0; i < SEG_V; ++i) {
      const bool here = mine + i * SEG_T == hi;
      q[i].x = here ? p.x : q[i].x;
      q[i].y = here ? p.y : q[i].y;
      q[i].z = here ? p.z : q[i].z;
      q[i].w = here ? p.w : q[i].w;
    }
  }
}

// Sum of the segment's exponentials, and its largest element (NaN if one is).
template <typename T>
__device__ __forceinline__ RunningSum sum_segment(const uint4* q, int32_t n, float c, float* largest = nullptr) {
  RunningSum acc;
  float mx = acc.template add<T, 4>(q, c);
  if (n > 6 * SEG_T) mx = max_nan(mx, acc.template add<T, 4>(q + 4, c));  // (no thread has a vector past n)
  else if (n > 4 * SEG_T) mx = max_nan(mx, acc.template add<T, 2>(q + 4, c));
  if (largest) *largest = mx;
  return acc;
}

// The largest element of each 128-byte group (8 vectors side by side, held by 8 lanes) of the segment:
// thread t ends with the largest of group t, vectors group_of(t) to group_of(t) + 7 of the segment. The
// eight lanes' eight words are reduced by halves: four words change hands, then two, then one.
__device__ __forceinline__ int32_t group_of(int32_t t) { return (t & 7) * SEG_T + (t & ~7); }
template <typename T>
__device__ __forceinline__ float group_largest(const uint4* q) {
  static_assert(SEG_V == 8, "eight words for eight lanes");
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = Elem<T>::max2(Elem<T>::max2(q[i].x, q[i].y), Elem<T>::max2(q[i].z, q[i].w));
  const uint32_t lane = threadIdx.x & 7;
#pragma unroll
  for (int half = 4; half > 0; half >>= 1) {
    const bool up = (lane & half) != 0;  // this lane keeps the upper half of the words
#pragma unroll
    for (int i = 0; i < half; ++i) {
      const uint32_t give = up ? w[i] : w[i + half], keep = up ? w[i + half] : w[i];
      w[i] = Elem<T>::max2(keep, __shfl_xor_sync(0xFFFFFFFFu, give, half));
    }
  }
  return Elem<T>::word_max(w[0]);
}

// Start the launch that follows on the stream as soon as this grid's CTAs have all begun (it waits
// for this grid's results with grid_wait), and that wait.
__device__ __forceinline__ void grid_release() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---- host side -------------------------------------------------------------------------------

// Whether an array of elements of `size` bytes can start at p (null: there is none).
inline bool aligned(const void* p, int size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }

inline int elem_size(int dtype) {
  return (dtype == PB_DTYPE_F32) ? 4 : (dtype == PB_DTYPE_BF16 || dtype == PB_DTYPE_F16) ? 2 : 0;
}

// Launch that may begin while the one before it on the stream is still running (the kernel waits for
// it with grid_wait before it reads its results).
template <typename K, typename A>
int launch_after(K kernel, const A& args, dim3 grid, int threads, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) {
    (void)cudaGetLastError();
    return PB_E_LAUNCH;
  }
  return cudaGetLastError() == cudaSuccess ? PB_OK : PB_E_LAUNCH;
}

}  // namespace pb
