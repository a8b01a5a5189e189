// Distillation from a teacher's top entries: the loss of each row of student logits, and its gradient.
//
// A row has student logits z (V of them), a temperature tau, and K entries (index, teacher value lp);
// entries of index -1 are padding. With y = z / tau and s = softmax(y):
//   renormalised:  t = softmax of the entries' values;   loss = sum_i t_i (log t_i - log s_i)
//   tail bucket:   t_i = exp(lp_i), T = max(0, 1 - sum t), S = the student's mass outside the entries;
//                  loss = sum_i t_i (log t_i - log s_i) + T (log T - log S)
//                  (the last term is left out where S is 0: below 2^-1000)
// and with A = sum t + T (renormalised: T = 0, A = 1):
//   dloss/dz_j = (1 / tau) (A s_j - sum_{i: index_i = j} t_i)     for j among the entries
//              = (1 / tau) (A s_j - T s_j / S)                    for the others
// A row without an entry of weight, and a row whose row weight is 0, has loss 0 and gradient 0.
//
// Forward: one cluster of C CTAs per row, each reading its slice of the row once, with a running
// maximum and sum of exponentials per thread. For the tail bucket the entries are kept out of that
// sum exactly (a bit per element of the slice in shared memory), so S has no cancellation however
// sure the student is. Backward: one pass, z in and dz out, on the statistics of the forward.
// Both are bound by HBM: V * es bytes a row forward, twice that backward.
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int DT = 512;         // threads per CTA
constexpr int DNW = DT / 32;
constexpr int DU = 4;           // vectors each thread has in flight
constexpr int DKMAX = PB_DISTILL_MAX_ENTRIES;     // entries per row
constexpr int DEPT = DKMAX / DT;  // entries per thread
constexpr int64_t DVMAX = PB_DISTILL_MAX_VOCAB;  // logits per row (one bit each in shared memory)

enum : int32_t { D_ROW = 0, D_EMPTY = 1, D_DUP = 2 };  // D_DUP: two entries name one element

// log2 of the student's mass outside the entries below which there is none: logits there of -inf, or
// masked with the type's lowest value.
constexpr float NO_SHARE = -1000.0f;

// What the backward pass needs of a row.
struct alignas(16) RowStats {
  float ref_m, ref_l;  // outside the entries: gradient 2^((z_j - ref_m) c - ref_l) * coef
  float coef;
  float all_m, all_l;  // s_j = 2^((z_j - all_m) c - all_l)
  float mass;          // A
  float norm;          // t_i = exp(lp_i - norm)
  int32_t flags;       // D_*
};

struct DistillArgs {
  const void* z;
  int64_t z_stride;  // elements
  const float* lp;
  int64_t lp_stride;
  const void* idx;
  int64_t idx_stride;
  int32_t idx64;
  int32_t tail;
  const float* weight;  // per row, or null
  float* loss;          // forward: [n]
  RowStats* stats;      // [n]
  const float* grad;    // backward: incoming gradient, row r at grad[r * grad_stride]
  int64_t grad_stride;
  void* dz;             // backward: [n][V]
  int64_t n;
  int32_t V, K;
  float c, inv_tau;     // log2(e) / tau, 1 / tau
  int32_t chunks;       // backward: CTAs per row
};

__device__ __forceinline__ int64_t entry_index(const DistillArgs& a, int64_t row, int i) {
  const int64_t at = row * a.idx_stride + i;
  return a.idx64 ? __ldg(static_cast<const long long*>(a.idx) + at) : (int64_t)__ldg(static_cast<const int*>(a.idx) + at);
}

struct FwdShared {
  ExpSum red[DNW];
  float fred[DNW];
  ExpSum pub_rest, pub_mem;  // this CTA's sums: outside the entries, over its distinct entries
  float pub_dot;             // this CTA's part of sum t (log t - log s)
};

template <typename T, bool TAIL>
__global__ void __launch_bounds__(DT, 2) distill_forward_kernel(DistillArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  extern __shared__ __align__(16) uint32_t mask[];  // a bit per element of the slice: an entry's
  __shared__ FwdShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.z) + row * a.z_stride, a.V);
  const int32_t v0 = (int32_t)((int64_t)rv.nvec * rank / C), v1 = (int32_t)((int64_t)rv.nvec * (rank + 1) / C);
  const int32_t words = ((v1 - v0) * EPV + 31) / 32;

  for (int32_t w = tid; w < words; w += DT) mask[w] = 0;

  // this thread's entries
  int32_t ix[DEPT];
  float lp[DEPT];
  bool bad = false, any = false;
  float mx = -INFINITY;
#pragma unroll
  for (int j = 0; j < DEPT; ++j) {
    const int i = tid + j * DT;
    ix[j] = -1;
    lp[j] = -INFINITY;
    if (i < a.K) {
      const int64_t e = entry_index(a, row, i);
      if (e < -1 || e >= a.V) bad = true;
      else if (e >= 0) {
        ix[j] = (int32_t)e;
        lp[j] = __ldg(a.lp + row * a.lp_stride + i);
        any = true;
        mx = fmaxf(mx, lp[j]);
      }
    }
  }
  // the entries' probabilities: t_i = exp(lp_i - norm)
  float norm = 0.0f;
  if (!TAIL) {
    mx = block_max<DNW>(mx, sh.fred);
    norm = (mx == -INFINITY) ? 0.0f : mx;
  }
  float t[DEPT], part = 0.0f;
#pragma unroll
  for (int j = 0; j < DEPT; ++j) {
    t[j] = (ix[j] >= 0) ? expf(lp[j] - norm) : 0.0f;
    part += t[j];
  }
  float sum_t = block_sum<DNW>(part, sh.fred);
  const bool row_bad = __syncthreads_or(bad) != 0;
  const bool row_any = __syncthreads_or(any) != 0;
  // no entry, or (renormalised) none of any weight: a padded row
  const float wt = a.weight ? __ldg(a.weight + row) : 1.0f;
  const bool empty = !row_bad && (wt == 0.0f || !row_any || (!TAIL && sum_t == 0.0f));
  if (empty) {  // the whole cluster: every CTA sees the same entries
    if (rank == 0 && tid == 0) {
      a.loss[row] = 0.0f;
      a.stats[row] = RowStats{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, D_EMPTY};
    }
    return;
  }
  if (!TAIL) {
    norm += logf(sum_t);
    const float inv = 1.0f / sum_t;
#pragma unroll
    for (int j = 0; j < DEPT; ++j) t[j] *= inv;
  }

  // mark the slice's entries; the first to mark an element owns it (its term of the student's sum
  // counts once, however many entries name it)
  float z[DEPT];
  bool own[DEPT], mine[DEPT], dup = false;
#pragma unroll
  for (int j = 0; j < DEPT; ++j) {
    mine[j] = own[j] = false;
    z[j] = 0.0f;
    if (ix[j] >= 0) {
      const int32_t v = (ix[j] + rv.off) / EPV;
      if (v >= v0 && v < v1) {
        mine[j] = true;
        const uint32_t b = (uint32_t)(ix[j] + rv.off - v0 * EPV);
        own[j] = !((atomicOr(&mask[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u);
        dup |= !own[j];
        z[j] = Elem<T>::ld(rv.row + ix[j]);
      }
    }
  }
  // (this barrier also ends the marking)
  const bool row_dup = __syncthreads_or(dup) != 0;

  // the slice: a running maximum and sum of 2^(z c)
  ExpSum acc = expsum_empty();
  for (int32_t vb = v0; vb < v1; vb += DT * DU) {
    uint4 q[DU];
#pragma unroll
    for (int u = 0; u < DU; ++u) {
      const int32_t v = vb + u * DT + tid;
      if (v < v1) q[u] = load_vec(rv, v);
    }
#pragma unroll
    for (int u = 0; u < DU; ++u) {
      const int32_t v = vb + u * DT + tid;
      if (v < v1) {
        float x[EPV];
        Elem<T>::unpack(q[u], x);
        if constexpr (TAIL) {
          const int32_t b = (v - v0) * EPV;
          uint32_t bits = (mask[b >> 5] >> (b & 31)) & ((1u << EPV) - 1u);
          if (bits) {
#pragma unroll
            for (int e = 0; e < EPV; ++e)
              if ((bits >> e) & 1u) x[e] = -INFINITY;
          }
        }
        expsum_add<T>(acc, x, a.c);
      }
    }
  }
  ExpSum rest = block_expsum<DNW>(acc, a.c, sh.red);
  ExpSum mem = expsum_empty();
  if constexpr (TAIL) {
#pragma unroll
    for (int j = 0; j < DEPT; ++j)
      if (own[j]) {
        // (a NaN or +inf logit makes the sum NaN, as in the stream)
        const float m = fmaxf(LOWEST, z[j]);
        mem = expsum_join(mem, ExpSum{m, ex2((z[j] - m) * a.c)}, a.c);
      }
    mem = block_expsum<DNW>(mem, a.c, sh.red);
  }
  if (tid == 0) {
    sh.pub_rest = rest;
    sh.pub_mem = mem;
  }
  cluster_barrier(C);
  if (C > 1) {
    rest = cluster.map_shared_rank(&sh, 0)->pub_rest;
    mem = cluster.map_shared_rank(&sh, 0)->pub_mem;
    for (int r = 1; r < C; ++r) {
      rest = expsum_join(rest, cluster.map_shared_rank(&sh, r)->pub_rest, a.c);
      if (TAIL) mem = expsum_join(mem, cluster.map_shared_rank(&sh, r)->pub_mem, a.c);
    }
  }
  const ExpSum all = TAIL ? expsum_join(rest, mem, a.c) : rest;
  const float all_l = log2f(all.s);

  // sum t (log t - log s) over the slice's entries
  constexpr float LN2 = 0.6931471805599453f;
  float dot = 0.0f;
#pragma unroll
  for (int j = 0; j < DEPT; ++j) {
    if (mine[j] && t[j] != 0.0f) {  // (NaN counts)
      dot += t[j] * ((lp[j] - norm) - ((z[j] - all.m) * a.inv_tau - all_l * LN2));
    }
  }
  dot = block_sum<DNW>(dot, sh.fred);
  bool any_dup = row_dup;
  if (C > 1) {
    if (tid == 0) {
      sh.pub_dot = dot;
      sh.fred[0] = row_dup ? 1.0f : 0.0f;
    }
    cluster_barrier(C);
    if (rank == 0 && tid == 0) {
      for (int r = 1; r < C; ++r) {
        dot += cluster.map_shared_rank(&sh, r)->pub_dot;
        any_dup |= cluster.map_shared_rank(&sh, r)->fred[0] != 0.0f;
      }
    }
  }
  if (rank == 0 && tid == 0) {
    float loss = dot;
    RowStats st;
    st.ref_m = st.all_m = all.m;
    st.ref_l = st.all_l = all_l;
    st.coef = st.mass = 1.0f;
    st.norm = norm;
    st.flags = any_dup ? D_DUP : D_ROW;
    if (TAIL) {
      const float rest_l = log2f(rest.s);
      const float log2_share = (rest.m - all.m) * a.c + (rest_l - all_l);  // log2 S
      float tm = 1.0f - sum_t;
      tm = (tm < 0.0f || log2_share < NO_SHARE) ? 0.0f : tm;  // (NaN stays)
      st.coef = st.mass = sum_t + tm;
      if (tm != 0.0f) {
        loss += tm * (logf(tm) - log2_share * LN2);
        st.ref_m = rest.m;
        st.ref_l = rest_l;
        st.coef = st.mass * exp2f(log2_share) - tm;
      }
    }
    if (row_bad || all.s == 0.0f) loss = st.all_l = st.ref_l = NAN;  // an index out of range; no student mass at all
    a.loss[row] = loss * wt;
    a.stats[row] = st;
  }
  if (C > 1) cluster.sync();  // shared memory stays until rank 0 has read it
}

template <typename T>
__device__ __forceinline__ T narrow(float x);
template <>
__device__ __forceinline__ float narrow<float>(float x) { return x; }
// round to nearest even: half a unit of the gradient's own type, as any product of torch in that type
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half narrow<__half>(float x) { return __float2half_rn(x); }

template <typename T>
__device__ __forceinline__ uint4 pack_vec(const float* x) {
  if constexpr (Elem<T>::EPV == 4) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      } else {
        const __half2 p = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// CTA (row, chunk): the gradient of the row's vectors [v0, v1), then the entries among them.
template <typename T>
__global__ void __launch_bounds__(DT, 2) distill_backward_kernel(DistillArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  const int64_t row = blockIdx.x / a.chunks;
  const int chunk = (int)(blockIdx.x - row * a.chunks);
  const int tid = threadIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.z) + row * a.z_stride, a.V);
  T* out = static_cast<T*>(a.dz) + row * (int64_t)a.V;
  const bool together = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(rv.row)) & 15) == 0;
  const int32_t v0 = (int32_t)((int64_t)rv.nvec * chunk / a.chunks),
                v1 = (int32_t)((int64_t)rv.nvec * (chunk + 1) / a.chunks);
  const RowStats st = a.stats[row];
  float g = __ldg(a.grad + row * a.grad_stride) * a.inv_tau;
  if (a.weight) g *= __ldg(a.weight + row);
  const bool zero = (st.flags & D_EMPTY) || g == 0.0f;
  const float gc = g * st.coef;

  auto put = [&](int32_t v, const float* x) {
    const int32_t e0 = rv.first(v);
    if (together && rv.whole(v)) {
      *reinterpret_cast<uint4*>(out + e0) = pack_vec<T>(x);
    } else {
#pragma unroll
      for (int q = 0; q < EPV; ++q)
        if (e0 + q >= 0 && e0 + q < a.V) out[e0 + q] = narrow<T>(x[q]);
    }
  };
  if (zero) {
    float x[EPV];
#pragma unroll
    for (int q = 0; q < EPV; ++q) x[q] = 0.0f;
    for (int32_t v = v0 + tid; v < v1; v += DT) put(v, x);
    return;
  }
  for (int32_t vb = v0; vb < v1; vb += DT * DU) {
    uint4 in[DU];
#pragma unroll
    for (int u = 0; u < DU; ++u) {
      const int32_t v = vb + u * DT + tid;
      if (v < v1) in[u] = load_vec(rv, v);
    }
#pragma unroll
    for (int u = 0; u < DU; ++u) {
      const int32_t v = vb + u * DT + tid;
      if (v < v1) {
        float x[EPV];
        Elem<T>::unpack(in[u], x);
#pragma unroll
        for (int q = 0; q < EPV; ++q) x[q] = ex2(fmaf(x[q] - st.ref_m, a.c, -st.ref_l)) * gc;
        put(v, x);
      }
    }
  }
  __syncthreads();  // the entries' elements are written again, after the stream's
  for (int i = tid; i < a.K; i += DT) {
    const int64_t e = entry_index(a, row, i);
    if (e < 0 || e >= a.V) continue;
    const int32_t v = ((int32_t)e + rv.off) / EPV;
    if (v < v0 || v >= v1) continue;
    float t = 0.0f;
    if (st.flags & D_DUP) {  // every entry that names e writes the same sum, taken in entry order
      for (int j = 0; j < a.K; ++j)
        if (entry_index(a, row, j) == e) t += expf(__ldg(a.lp + row * a.lp_stride + j) - st.norm);
    } else {
      t = expf(__ldg(a.lp + row * a.lp_stride + i) - st.norm);
    }
    const float s = ex2(fmaf(Elem<T>::ld(rv.row + e) - st.all_m, a.c, -st.all_l));
    out[e] = narrow<T>((st.mass * s - t) * g);
  }
}

// CTAs per row: enough to give every SM two, with slices of at least 8 KB.
int cluster_for(int64_t n, int64_t bytes) {
  const int64_t want = 2 * (int64_t)device_sms();
  int C = 1;
  while (C < 8 && n * C < want && bytes / (2 * C) >= 8192) C <<= 1;
  return C;
}

size_t mask_bytes(int64_t V, int es, int C) {
  const int64_t epv = 16 / es, nvec = (V + 2 * epv - 2) / epv;  // the most vectors a row of any alignment has
  return (size_t)(((nvec + C - 1) / C * epv + 31) / 32 * 4);
}

template <typename T>
int forward(const DistillArgs& a, cudaStream_t st) {
  const int C = cluster_for(a.n, (int64_t)a.V * sizeof(T));
  const size_t smem = mask_bytes(a.V, sizeof(T), C);
  return a.tail ? launch_cluster(distill_forward_kernel<T, true>, a, a.n * C, DT, C, smem, st)
                : launch_cluster(distill_forward_kernel<T, false>, a, a.n * C, DT, C, smem, st);
}

template <typename T>
int backward(DistillArgs a, cudaStream_t st) {
  // chunks of a row: CTAs of at least 4 vectors a thread, unless the rows alone cannot fill the SMs
  a.chunks = cluster_for(a.n, (int64_t)a.V * sizeof(T));
  return launch_cluster(distill_backward_kernel<T>, a, a.n * a.chunks, DT, 1, 0, st);
}

int check(const DistillArgs& a, int es, int64_t vocab, float temperature) {
  if (a.n < 0 || vocab <= 0 || a.K < 1 || a.K > DKMAX) return PB_E_INVALID;
  if (vocab > DVMAX) return PB_E_TOO_LARGE;
  if (!(temperature >= 0x1p-20f && temperature <= 0x1p20f)) return PB_E_INVALID;
  if (!es) return PB_E_INVALID;
  if (a.n == 0) return PB_OK;
  if (!a.z || !a.lp || !a.idx || !a.stats) return PB_E_INVALID;
  if (a.n > (int64_t)(0x7FFFFFFF / 8)) return PB_E_INVALID;
  if (a.z_stride < 0 || a.lp_stride < 0 || a.idx_stride < 0) return PB_E_INVALID;
  if (reinterpret_cast<uintptr_t>(a.z) % es) return PB_E_INVALID;
  if (reinterpret_cast<uintptr_t>(a.stats) & 15) return PB_E_INVALID;
  if ((reinterpret_cast<uintptr_t>(a.idx) % (a.idx64 ? 8 : 4)) || (reinterpret_cast<uintptr_t>(a.lp) & 3))
    return PB_E_INVALID;
  return PB_OK;
}

}  // namespace

extern "C" {

int64_t pb_distill_stats_bytes(int64_t n_rows) { return n_rows < 0 ? PB_E_INVALID : n_rows * (int64_t)sizeof(RowStats); }

int pb_distill_forward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                       const float* teacher, int64_t teacher_stride, const void* indices, int64_t index_stride,
                       int index_bytes, int32_t n_entries, float temperature, int tail, const float* row_weight,
                       float* out_loss, void* out_stats, void* stream) {
  const int es = elem_size(dtype);
  if (index_bytes != 4 && index_bytes != 8) return PB_E_INVALID;
  DistillArgs a = {};
  a.z = logits;
  a.z_stride = row_stride;
  a.lp = teacher;
  a.lp_stride = teacher_stride;
  a.idx = indices;
  a.idx_stride = index_stride;
  a.idx64 = index_bytes == 8;
  a.tail = tail != 0;
  a.weight = row_weight;
  a.loss = out_loss;
  a.stats = static_cast<RowStats*>(out_stats);
  a.n = n_rows;
  a.V = (int32_t)vocab;
  a.K = n_entries;
  const int rc = check(a, es, vocab, temperature);
  if (rc != PB_OK || n_rows == 0) return rc;
  if (!out_loss) return PB_E_INVALID;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = 1.0f / temperature;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return forward<float>(a, st);
  if (dtype == PB_DTYPE_BF16) return forward<__nv_bfloat16>(a, st);
  return forward<__half>(a, st);
}

int pb_distill_backward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                        const float* teacher, int64_t teacher_stride, const void* indices, int64_t index_stride,
                        int index_bytes, int32_t n_entries, float temperature, const float* row_weight,
                        const void* stats, const float* grad_loss, int64_t grad_stride, void* out_grad, void* stream) {
  const int es = elem_size(dtype);
  if (index_bytes != 4 && index_bytes != 8) return PB_E_INVALID;
  DistillArgs a = {};
  a.z = logits;
  a.z_stride = row_stride;
  a.lp = teacher;
  a.lp_stride = teacher_stride;
  a.idx = indices;
  a.idx_stride = index_stride;
  a.idx64 = index_bytes == 8;
  a.weight = row_weight;
  a.stats = const_cast<RowStats*>(static_cast<const RowStats*>(stats));
  a.grad = grad_loss;
  a.grad_stride = grad_stride;
  a.dz = out_grad;
  a.n = n_rows;
  a.V = (int32_t)vocab;
  a.K = n_entries;
  const int rc = check(a, es, vocab, temperature);
  if (rc != PB_OK || n_rows == 0) return rc;
  if (!grad_loss || !out_grad || grad_stride < 0) return PB_E_INVALID;
  if (reinterpret_cast<uintptr_t>(out_grad) % es) return PB_E_INVALID;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = 1.0f / temperature;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return backward<float>(a, st);
  if (dtype == PB_DTYPE_BF16) return backward<__nv_bfloat16>(a, st);
  return backward<__half>(a, st);
}

}  // extern "C"
