// Reading whole logits rows as 16-byte vectors at any alignment, and the block and cluster helpers
// shared by the row-wise operators (top log-probabilities, distillation loss, verification).
#pragma once

#include <cooperative_groups.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <algorithm>
#include <atomic>

#include "../../include/pagedbatch_b200.h"
#include "pb_device.cuh"
#include "pb_elem.cuh"

namespace pb {

namespace cg = cooperative_groups;

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

// Join over a warp, then the block (NWARP warps); every thread gets the result. `scratch` holds
// NWARP entries; contains two barriers.
template <int NWARP>
__device__ __forceinline__ ExpSum block_expsum(ExpSum v, float c, ExpSum* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = v.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  float s = v.s * ex2((v.m - m) * c);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (lane == 0) scratch[warp] = ExpSum{m, s};
  __syncthreads();
  ExpSum r = scratch[0];
#pragma unroll
  for (int w = 1; w < NWARP; ++w) r = expsum_join(r, scratch[w], c);
  __syncthreads();
  return r;
}

// Block sum of one float per thread in a fixed order; every thread gets it. Two barriers.
template <int NWARP>
__device__ __forceinline__ float block_sum(float v, float* scratch) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = scratch[0];
#pragma unroll
  for (int w = 1; w < NWARP; ++w) r += scratch[w];
  __syncthreads();
  return r;
}

template <int NWARP>
__device__ __forceinline__ float block_max(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float r = scratch[0];
#pragma unroll
  for (int w = 1; w < NWARP; ++w) r = fmaxf(r, scratch[w]);
  __syncthreads();
  return r;
}

// Add a vector's elements to a running sum (one rescale when the maximum grows).
template <typename T>
__device__ __forceinline__ void expsum_add(ExpSum& a, const float* x, float c) {
  constexpr int EPV = Elem<T>::EPV;
  float mx = x[0];
#pragma unroll
  for (int q = 1; q < EPV; ++q) mx = fmaxf(mx, x[q]);
  if (mx > a.m) {
    a.s *= ex2((a.m - mx) * c);
    a.m = mx;
  }
  float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
  for (int q = 0; q < EPV; q += 2) {
    s0 += ex2((x[q] - a.m) * c);
    s1 += ex2((x[q + 1] - a.m) * c);
  }
  a.s += s0 + s1;
}

__device__ __forceinline__ void cluster_barrier(int C) {
  if (C == 1) __syncthreads();
  else cg::this_cluster().sync();
}

// ---- host side -------------------------------------------------------------------------------

inline int elem_size(int dtype) {
  return (dtype == PB_DTYPE_F32) ? 4 : (dtype == PB_DTYPE_BF16 || dtype == PB_DTYPE_F16) ? 2 : 0;
}

// SMs of the current device (148 where it cannot be asked), looked up once per device.
inline int device_sms() {
  static std::atomic<int> cache[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = cache[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cache[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Launch of a kernel whose blocks form clusters of C along x, with `smem` bytes of dynamic shared
// memory (the kernel's limit is raised on the current device when that and the kernel's static
// shared memory, at most 24 KB in these kernels, may pass 48 KB).
template <typename K, typename A>
int launch_cluster(K kernel, const A& args, int64_t blocks, int threads, int C, size_t smem, cudaStream_t st) {
  if (smem > 24 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess) {
    (void)cudaGetLastError();
    return PB_E_DEVICE;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args) != cudaSuccess) {
    (void)cudaGetLastError();
    return PB_E_LAUNCH;
  }
  return cudaGetLastError() == cudaSuccess ? PB_OK : PB_E_LAUNCH;
}

}  // namespace pb
