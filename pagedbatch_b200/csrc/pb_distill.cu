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
// Forward, two launches: part_kernel reads every row once, a CTA per segment of it, with a running
// maximum and sum of exponentials; finish_kernel, one warp per row, joins the segments and takes the
// loss from the row's entries. For the tail bucket the entries are kept out of the sums exactly (a bit
// per element of the segment in shared memory), so S has no cancellation however sure the student is.
// Backward: one launch, z in and dz out, on the statistics of the forward. Both passes are bound by
// HBM: V * es bytes a row forward, twice that backward. [4096, 128256] bf16 with a tail, summed: 557 us of launches
// back to back (a captured step; one call by itself 606 us, as the host starts each half),
// floor 326 us if the backward pass found the logits on chip, 488 us as they are read twice. (A persistent
// kernel that takes both passes over a few rows at a time, the second from L2, took 570 us: its halves wait
// for one another.)
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int DKMAX = PB_DISTILL_MAX_ENTRIES;    // entries per row
constexpr int64_t DVMAX = PB_DISTILL_MAX_VOCAB;  // logits per row
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

// What a segment adds to its row.
struct Part {
  ExpSum rest, mem;  // sums outside the entries, over the segment's distinct entries
  int32_t dup, pad;  // two entries name one of its elements
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
  Part* parts;          // [n][segs]
  const float* grad;    // backward: incoming gradient, row r at grad[r * grad_stride]
  int64_t grad_stride;
  void* dz;             // backward: [n][V]
  int64_t n;
  int32_t V, K;
  float c, inv_tau;     // log2(e) / tau, 1 / tau
  SegPlan seg;
};

__device__ __forceinline__ int64_t entry_index(const DistillArgs& a, int64_t row, int i) {
  const int64_t at = row * a.idx_stride + i;
  return a.idx64 ? __ldg(static_cast<const long long*>(a.idx) + at) : (int64_t)__ldg(static_cast<const int*>(a.idx) + at);
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

// Element x of a vector, from the word that holds it.
template <typename T>
__device__ __forceinline__ float word_elem(uint32_t v, int x) {
  if constexpr (Elem<T>::EPV == 4) return __uint_as_float(v);
  else return Elem<T>::elem(make_uint4(v, 0u, 0u, 0u), x & 1);
}

// A row's gradient: where it goes, and its scale g.
template <typename T>
struct GradRow {
  static constexpr int EPV = Elem<T>::EPV;
  const DistillArgs& a;
  const RowView<T>& rv;
  const RowStats& st;
  int64_t row;
  T* out;
  bool together;  // the row and its gradient lie alike on 16-byte boundaries
  float g;
  __device__ GradRow(const DistillArgs& a_, const RowView<T>& rv_, const RowStats& st_, int64_t row_, float g_)
      : a(a_), rv(rv_), st(st_), row(row_), g(g_) {
    out = static_cast<T*>(a.dz) + row * (int64_t)a.V;
    together = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(rv.row)) & 15) == 0;
  }
  __device__ __forceinline__ void put(int32_t v, const float* x) const {
    const int32_t e0 = rv.first(v);
    if (together && rv.whole(v)) {
      __stcs(reinterpret_cast<uint4*>(out + e0), pack_vec<T>(x));
    } else {
#pragma unroll
      for (int q = 0; q < EPV; ++q)
        if (e0 + q >= 0 && e0 + q < a.V) out[e0 + q] = narrow<T>(x[q]);
    }
  }
  __device__ __forceinline__ void put_zero(int32_t v) const {
    float x[EPV];
#pragma unroll
    for (int q = 0; q < EPV; ++q) x[q] = 0.0f;
    put(v, x);
  }
  // the elements of vector v as if none were an entry
  __device__ __forceinline__ void put_rest(int32_t v, uint4 in, const Exponent& ex) const {
    const float gc = g * st.coef;
    float x[EPV];
    uint64_t e[EPV / 2];
    ex.template of<T>(in, e);
    const uint64_t g2 = pack2(gc, gc);
#pragma unroll
    for (int i = 0; i < EPV / 2; ++i) {
      float lo, hi;
      unpack2(e[i], lo, hi);
      unpack2(mul2(pack2(ex2(lo), ex2(hi)), g2), x[2 * i], x[2 * i + 1]);
    }
    put(v, x);
  }
  // entry i, which names element e
  __device__ __forceinline__ void put_entry(int i, int64_t e) const {
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
};

// CTA (row, segment): the sums of the segment's exponentials. [4096, 128256] bf16 with a tail (1.05 GB) in
// 207 us, 5.1 TB/s: no more loads are issued while the entries are marked. (Entries matched by each warp for
// itself, without the marks, took a quarter longer; four CTAs to an SM without spilled registers, 5%.)
template <typename T, bool TAIL>
__global__ void __launch_bounds__(SEG_T, SEG_CTAS) part_kernel(DistillArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ uint32_t mask[SEG_T * SEG_V * EPV / 32];  // a bit per element of the segment: an entry's
  __shared__ uint32_t marked[SEG_T];                   // by thread: a bit per vector that holds an entry
  __shared__ Part warps[SEG_NW];
  __shared__ int32_t any_dup;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowView<T> rv(static_cast<const T*>(a.z) + row * a.z_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  load_segment(rv, v0, v1, q);
  grid_release();

  // mark the segment's entries, while its vectors are on their way
  const int32_t first = rv.first(v0), e0 = max(0, first), e1 = min(a.V, rv.first(v1));
  auto place = [&](int i) -> int32_t {  // of entry i in the segment's vectors, or -1
    const int64_t e = entry_index(a, row, i);
    return e >= e0 && e < e1 ? (int32_t)e - first : -1;
  };
  int32_t b = tid < a.K ? place(tid) : -1;
#pragma unroll
  for (int w = tid; w < SEG_T * SEG_V * EPV / 32; w += SEG_T) mask[w] = 0;
  marked[tid] = 0;
  if (tid == 0) any_dup = 0;
  __syncthreads();
  for (int i = tid; i < a.K; i += SEG_T) {
    if (i != tid) b = place(i);
    if (b < 0) continue;
    if ((atomicOr(&mask[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1u) any_dup = 1;
    else if (TAIL) atomicOr(&marked[b / EPV % SEG_T], 1u << (b / EPV / SEG_T));
  }
  __syncthreads();
  // the entries' elements, each once however many entries name it, leave the vectors for a sum of their own
  ExpSum mem = expsum_empty();
  if constexpr (TAIL) {
    uint32_t mk = marked[tid];
    if (mk) {
#pragma unroll
      for (int i = 0; i < SEG_V; ++i) {
        if (!((mk >> i) & 1u)) continue;
        const uint32_t at = (uint32_t)(tid + i * SEG_T) * EPV, bits = mask[at >> 5] >> (at & 31) & ((1u << EPV) - 1u);
        uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll 1
        for (uint32_t left = bits; left; left &= left - 1) {
          const int x = __ffs(left) - 1, word = (EPV == 4) ? x : x >> 1;
          const uint32_t part = (EPV == 4) ? 0xFFFFFFFFu : 0xFFFFu << (16 * (x & 1));
          uint32_t v = w[0];
#pragma unroll
          for (int j = 1; j < 4; ++j) v = word == j ? w[j] : v;
          // (a NaN or +inf logit makes the sum NaN, as in the stream)
          const float z = word_elem<T>(v, x), m = fmaxf(LOWEST, z);
          mem = expsum_join(mem, ExpSum{m, ex2((z - m) * a.c)}, a.c);
          v = (v & ~part) | (Elem<T>::NEG_INF_WORD & part);
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = word == j ? v : w[j];
        }
        q[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  const ExpSum rest = warp_expsum(sum_segment<T>(q, v1 - v0, a.c).total(), a.c);
  if (TAIL) mem = warp_expsum(mem, a.c);
  if (lane == 0) warps[warp] = Part{rest, mem, 0, 0};
  __syncthreads();
  if (warp != 0) return;
  Part p = lane < SEG_NW ? warps[lane] : Part{expsum_empty(), expsum_empty(), 0, 0};
  p.rest = warp_expsum(p.rest, a.c);
  if (TAIL) p.mem = warp_expsum(p.mem, a.c);
  p.dup = any_dup;
  if (lane == 0) a.parts[row * a.seg.segs + blockIdx.y] = p;
}

// One warp per row: joins the row's segments, takes the loss from its entries, and leaves what the
// backward pass needs. Its loads of entries go ahead of the wait for the segments. 10 us for 4096 rows.
template <typename T, bool TAIL>
__global__ void __launch_bounds__(256) finish_kernel(DistillArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.n) return;
  const float wt = a.weight ? __ldg(a.weight + row) : 1.0f;
  const T* zr = static_cast<const T*>(a.z) + row * a.z_stride;

  // the entries: sum of exp(value - top) (the tail's are probabilities as they are: top is 0). The
  // first FIRST are kept in registers, with their logits, and loaded together.
  constexpr int FIRST = 128, PER = FIRST / 32;
  int32_t ix[PER];
  float val[PER], z[PER];
  bool any = false, bad = false;
  float top = -INFINITY, sum = 0.0f;
  auto look = [&](int64_t e, float lp) {
    bad |= e < -1 || e >= a.V;
    if (e >= 0) {
      any = true;
      top = max_nan(top, lp);
    }
  };
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int i = lane + 32 * j;
    const int64_t e = i < a.K ? entry_index(a, row, i) : -1;
    val[j] = i < a.K ? __ldg(a.lp + row * a.lp_stride + i) : 0.0f;
    look(e, val[j]);
    ix[j] = e >= 0 && e < a.V ? (int32_t)e : -1;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) z[j] = ix[j] >= 0 ? Elem<T>::ld(zr + ix[j]) : 0.0f;
  for (int i = FIRST + lane; i < a.K; i += 32) look(entry_index(a, row, i), __ldg(a.lp + row * a.lp_stride + i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (TAIL || top == -INFINITY) top = 0.0f;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (ix[j] >= 0) sum += expf(val[j] - top);
  for (int i = FIRST + lane; i < a.K; i += 32)
    if (entry_index(a, row, i) >= 0) sum += expf(__ldg(a.lp + row * a.lp_stride + i) - top);
  sum = warp_sum(sum);
  any = __any_sync(0xFFFFFFFFu, any);
  bad = __any_sync(0xFFFFFFFFu, bad);
  const float norm = TAIL ? 0.0f : top + logf(sum);  // t_i = exp(value_i - norm)

  grid_wait();  // the segments' sums
  // no entry, or (renormalised) none of any weight: a padded row
  if (!bad && (wt == 0.0f || !any || (!TAIL && sum == 0.0f))) {
    if (lane == 0) {
      a.loss[row] = 0.0f;
      a.stats[row] = RowStats{0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, D_EMPTY};
    }
    return;
  }
  ExpSum rest = expsum_empty(), mem = rest;
  int32_t dup = 0;
  for (int s = lane; s < a.seg.segs; s += 32) {
    const Part p = a.parts[row * a.seg.segs + s];
    rest = expsum_join(rest, p.rest, a.c);
    if (TAIL) mem = expsum_join(mem, p.mem, a.c);
    dup |= p.dup;
  }
  rest = warp_expsum(rest, a.c);
  if (TAIL) mem = warp_expsum(mem, a.c);
  dup = __any_sync(0xFFFFFFFFu, dup);
  constexpr float LN2 = 0.6931471805599453f;
  const ExpSum full = TAIL ? expsum_join(rest, mem, a.c) : rest;
  RowStats st;
  st.ref_m = st.all_m = full.m;
  st.ref_l = st.all_l = log2f(full.s);
  st.coef = st.mass = 1.0f;
  st.norm = norm;
  st.flags = dup ? D_DUP : D_ROW;
  float dot = 0.0f;
  auto term = [&](float lp, float zi) {
    const float t = expf(lp - norm);
    if (t != 0.0f)  // (NaN counts)
      dot += t * ((lp - norm) - ((zi - full.m) * a.inv_tau - st.all_l * LN2));
  };
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (ix[j] >= 0) term(val[j], z[j]);
  for (int i = FIRST + lane; i < a.K; i += 32) {
    const int64_t e = entry_index(a, row, i);
    if (e >= 0 && e < a.V) term(__ldg(a.lp + row * a.lp_stride + i), Elem<T>::ld(zr + e));
  }
  float loss = warp_sum(dot);
  if (TAIL) {
    const float rest_l = log2f(rest.s);
    const float log2_share = (rest.m - full.m) * a.c + (rest_l - st.all_l);  // log2 S
    float tm = 1.0f - sum;
    tm = (tm < 0.0f || log2_share < NO_SHARE) ? 0.0f : tm;  // (NaN stays)
    st.coef = st.mass = sum + tm;
    if (tm != 0.0f) {
      loss += tm * (logf(tm) - log2_share * LN2);
      st.ref_m = rest.m;
      st.ref_l = rest_l;
      st.coef = st.mass * exp2f(log2_share) - tm;
    }
  }
  if (bad || full.s == 0.0f) loss = st.all_l = st.ref_l = NAN;  // an index out of range; no student mass at all
  if (lane == 0) {
    a.loss[row] = loss * wt;
    a.stats[row] = st;
  }
}

// CTA (row, segment): the gradient of the segment, then of the entries in it. Bound by HBM: [4096, 128256]
// bf16, 2.1 GB read and written in 345 us, 6.1 TB/s (94% of the measured copy rate).
template <typename T>
__global__ void __launch_bounds__(SEG_T, 4) backward_kernel(DistillArgs a) {
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.z) + row * a.z_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  load_segment(rv, v0, v1, q);
  const RowStats st = a.stats[row];
  float g = __ldg(a.grad + row * a.grad_stride) * a.inv_tau;
  if (a.weight) g *= __ldg(a.weight + row);
  const GradRow<T> grad(a, rv, st, row, g);
  if ((st.flags & D_EMPTY) || g == 0.0f) {
    for (int32_t v = v0 + tid; v < v1; v += SEG_T) grad.put_zero(v);
    return;
  }
  const Exponent ex(st.ref_m, a.c, st.ref_l);
#pragma unroll
  for (int i = 0; i < SEG_V; ++i)
    if (v0 + i * SEG_T + tid < v1) grad.put_rest(v0 + i * SEG_T + tid, q[i], ex);
  __syncthreads();  // the entries' elements are written again, after the stream's
  const int32_t e0 = max(0, rv.first(v0)), e1 = min(a.V, rv.first(v1));
  for (int i = tid; i < a.K; i += SEG_T) {
    const int64_t e = entry_index(a, row, i);
    if (e >= e0 && e < e1) grad.put_entry(i, e);
  }
}

// Sum of the rows' losses, in 64 bits and a fixed order, by one CTA (3 us for 4096).
__global__ void __launch_bounds__(1024) distill_sum_kernel(const float* loss, int64_t n, float* out) {
  __shared__ double part[32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) s += (double)loss[i];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(part[threadIdx.x]);
    if (threadIdx.x == 0) *out = (float)s;
  }
}

template <typename T, bool TAIL>
int forward_as(const DistillArgs& a, cudaStream_t st) {
  part_kernel<T, TAIL><<<dim3((unsigned)a.n, (unsigned)a.seg.segs), SEG_T, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return PB_E_LAUNCH;
  return launch_after(finish_kernel<T, TAIL>, a, dim3((unsigned)((a.n + 7) / 8)), 256, st);
}

template <typename T>
int forward(DistillArgs a, cudaStream_t st) {
  a.seg = seg_plan(a.V, sizeof(T), a.z, a.z_stride);
  return a.tail ? forward_as<T, true>(a, st) : forward_as<T, false>(a, st);
}

template <typename T>
int backward(DistillArgs a, cudaStream_t st) {
  a.seg = seg_plan(a.V, sizeof(T), a.z, a.z_stride);
  backward_kernel<T><<<dim3((unsigned)a.n, (unsigned)a.seg.segs), SEG_T, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? PB_OK : PB_E_LAUNCH;
}

constexpr int64_t stats_bytes(int64_t n) { return n * (int64_t)sizeof(RowStats); }

int check(const DistillArgs& a, int es, int64_t vocab, float temperature) {
  if (a.n < 0 || vocab <= 0 || a.K < 1 || a.K > DKMAX) return PB_E_INVALID;
  if (vocab > DVMAX) return PB_E_TOO_LARGE;
  if (!(temperature >= 0x1p-20f && temperature <= 0x1p20f)) return PB_E_INVALID;
  if (!es) return PB_E_INVALID;
  if (a.n == 0) return PB_OK;
  if (!a.z || !a.lp || !a.idx || !a.stats) return PB_E_INVALID;
  if (a.n > (int64_t)(0x7FFFFFFF / 8)) return PB_E_INVALID;
  if (a.z_stride < 0 || a.lp_stride < 0 || a.idx_stride < 0) return PB_E_INVALID;
  if (!aligned(a.z, es) || !aligned(a.stats, 16) || !aligned(a.idx, a.idx64 ? 8 : 4) || !aligned(a.lp, 4) ||
      !aligned(a.weight, 4) || !aligned(a.loss, 4) || !aligned(a.grad, 4) || !aligned(a.dz, es))
    return PB_E_INVALID;
  return PB_OK;
}

}  // namespace

extern "C" {

int64_t pb_distill_stats_bytes(int64_t n_rows) { return n_rows < 0 ? PB_E_INVALID : stats_bytes(n_rows); }

int64_t pb_distill_ws_bytes(int64_t n_rows, int64_t vocab, int dtype) {
  const int es = elem_size(dtype);
  if (n_rows < 0 || vocab <= 0 || vocab > DVMAX || !es) return PB_E_INVALID;
  return n_rows * seg_plan(vocab, es, nullptr, 1).segs * (int64_t)sizeof(Part)  /* rows of any alignment */;
}

int pb_distill_forward(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
                       const float* teacher, int64_t teacher_stride, const void* indices, int64_t index_stride,
                       int index_bytes, int32_t n_entries, float temperature, int tail, const float* row_weight,
                       float* out_loss, void* out_stats, void* workspace, int64_t ws_bytes, void* stream) {
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
  if (!out_loss || !workspace || !aligned(workspace, 16)) return PB_E_INVALID;
  if (ws_bytes < pb_distill_ws_bytes(n_rows, vocab, dtype)) return PB_E_INVALID;
  a.parts = static_cast<Part*>(workspace);
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
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.inv_tau = 1.0f / temperature;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return backward<float>(a, st);
  if (dtype == PB_DTYPE_BF16) return backward<__nv_bfloat16>(a, st);
  return backward<__half>(a, st);
}

int pb_distill_sum(const float* loss, int64_t n_rows, float* out_sum, void* stream) {
  if (n_rows < 0 || !out_sum || (n_rows && !loss) || !aligned(loss, 4) || !aligned(out_sum, 4)) return PB_E_INVALID;
  distill_sum_kernel<<<1, 1024, 0, static_cast<cudaStream_t>(stream)>>>(loss, n_rows, out_sum);
  return cudaGetLastError() == cudaSuccess ? PB_OK : PB_E_LAUNCH;
}

}  // extern "C"
