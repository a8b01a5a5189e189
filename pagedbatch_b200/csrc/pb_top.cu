// The k largest log-probabilities of each row, with their indices and the row's log-sum-exp: what a
// server returns as log-probabilities and what a teacher records for distillation.
//
//   y_j = x_j / T,  lse = log sum_j exp(y_j),  log p_j = y_j - lse
//   the k largest x in the order (value descending, index ascending), NaN above every value
//   (the sampler's order). A row holding NaN or +inf, or only -inf, has NaN log-probabilities.
//
// Two launches. part_kernel reads every row once, a CTA per segment of it: per thread a running
// maximum and sum of exponentials, and for the CTA the key of the largest value of every 128 bytes (a
// group).
// select_kernel, a CTA per row: a lower bound of the k-th largest value follows from the lanes'
// largest group keys, since each of its 8 warps holds ceil(k / 8) values at or above its
// ceil(k / 8)-th largest lane maximum, so the row holds k at or above the smallest of these. A
// histogram of the group keys above that bound (256 equal steps up to the largest key) raises it to
// the step that k of them reach. Only the groups whose key reaches the raised bound are read again
// (from L2); their values at or above it are the candidates, a little more than k, put in order by
// counting for each the candidates before it, or where they are many by a bitonic network. A row with more
// candidates than the list holds, nearly all of them equal as a mask makes them, has those above that
// value listed and the first of its equals added; any other is selected by bisection over (value, index), as are
// rows of fewer groups than k and more elements than the list (k 223, 587 rows of 13394 bf16: 457 us).
// HBM-bound: V * es bytes a row, and 1/32 of that written as keys. [1024, 128256] bf16, k 128: 77 us, the
// read's floor 41 us; one CTA or cluster a row, which selects while others read, took 187 us.
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int TT = SEG_T;          // threads per CTA
constexpr int TNW = SEG_NW;
constexpr int TKMAX = PB_TOP_MAX;  // largest k
constexpr int TCAP = 2048;         // candidates of a row
constexpr int TRANK = 512;         // candidates ordered by counting
constexpr int TLIST = 1024;        // groups of a row that are read again
static_assert((TKMAX + TNW - 1) / TNW <= 32, "every warp has enough lanes");

struct TopArgs {
  const void* x;
  int64_t row_stride;  // elements
  int64_t n;
  int32_t V, k;
  float c, temperature;  // log2(e) / T
  float* logprob;        // [n][k]
  int32_t* index;        // [n][k]
  float* lse;            // [n]
  SegPlan seg;
  ExpSum* parts;         // workspace: [n][segs]
  uint32_t* keys;        // workspace: [n][segs][TT]
};

struct TopShared {
  ExpSum sum[TNW];
  uint32_t bound[TNW], top[TNW];
  uint32_t hist[TT];                // group keys by step above the bound
  uint32_t steps[TNW];
  uint32_t raised;                  // the bound raised by the histogram
  uint32_t groups;                  // groups listed
  uint32_t n;                       // candidates
  uint32_t cnt[2];                  // bisection counts
  uint32_t group[TLIST];
  alignas(16) uint64_t list[TCAP];  // candidates
};

// c-th largest (1 <= c <= 32) of the warp's 32 values: c rounds of a warp maximum, one copy of the
// maximum removed in each.
__device__ __forceinline__ uint32_t warp_nth_largest(uint32_t v, int c) {
  uint32_t r = 0;
  for (int i = 0; i < c; ++i) {
    r = __reduce_max_sync(0xFFFFFFFFu, v);
    const uint32_t who = __ballot_sync(0xFFFFFFFFu, v == r);
    if ((int)(threadIdx.x & 31) == __ffs(who) - 1) v = 0;
  }
  return r;
}

// Exact selection in one CTA, for rows whose candidates overflow the list: the k-th largest key by
// bisection over the keys, then the largest index taken among its equals by bisection over indices,
// each step one pass over the row. Writes exactly k entries to sh.list.
template <typename T>
__device__ __noinline__ void select_slow(const RowView<T>& rv, int k, TopShared& sh) {
  constexpr int EPV = Elem<T>::EPV;
  const int tid = threadIdx.x;
  int phase = 0;
  auto count = [&](auto&& pred) -> uint32_t {  // elements of the row for which pred(key, index) holds
    if (tid == 0) sh.cnt[phase] = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (int32_t v = tid; v < rv.nvec; v += TT) {
      float x[EPV];
      Elem<T>::unpack(load_vec(rv, v), x);
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        const int32_t e = rv.first(v) + q;
        if (e >= 0 && e < rv.V && pred(key_of(x[q]), (uint32_t)e)) ++mine;
      }
    }
    mine = __reduce_add_sync(0xFFFFFFFFu, mine);
    if ((tid & 31) == 0 && mine) atomicAdd(&sh.cnt[phase], mine);
    __syncthreads();
    const uint32_t r = sh.cnt[phase];
    phase ^= 1;
    return r;
  };
  uint64_t lo = 0, hi = 1ull << 32;  // at least k keys are >= lo, fewer are >= hi
  while (hi - lo > 1) {
    const uint64_t mid = lo + ((hi - lo) >> 1);
    const uint32_t c = count([&](uint32_t key, uint32_t) { return (uint64_t)key >= mid; });
    if (c >= (uint32_t)k) lo = mid;
    else hi = mid;
  }
  const uint32_t kth = (uint32_t)lo;
  const uint32_t above = count([&](uint32_t key, uint32_t) { return key > kth; });
  const uint32_t want = (uint32_t)k - above;  // of the elements equal to kth, those of lowest index
  int32_t a = 0, b = rv.V - 1;                // smallest index i with `want` equals at or below it
  while (a < b) {
    const int32_t mid = a + ((b - a) >> 1);
    const uint32_t c = count([&](uint32_t key, uint32_t e) { return key == kth && e <= (uint32_t)mid; });
    if (c >= want) b = mid;
    else a = mid + 1;
  }
  if (tid == 0) sh.n = 0;
  __syncthreads();
  for (int32_t v = tid; v < rv.nvec; v += TT) {
    float x[EPV];
    Elem<T>::unpack(load_vec(rv, v), x);
#pragma unroll
    for (int q = 0; q < EPV; ++q) {
      const int32_t e = rv.first(v) + q;
      const uint32_t key = key_of(x[q]);
      if (e >= 0 && e < rv.V && (key > kth || (key == kth && e <= a)))
        sh.list[atomicAdd(&sh.n, 1u)] = compose(key, (uint32_t)e);
    }
  }
  __syncthreads();
}

// Lists a group where it is a hit (all lanes of a warp call it).
__device__ __forceinline__ void list_group(TopShared& sh, uint32_t group, bool hit) {
  const uint32_t b = __ballot_sync(0xFFFFFFFFu, hit);
  if (!b) return;
  uint32_t at = 0;
  if ((threadIdx.x & 31) == 0) at = atomicAdd(&sh.groups, (uint32_t)__popc(b));
  at = __shfl_sync(0xFFFFFFFFu, at, 0) + (uint32_t)__popc(b & lanemask_lt());
  if (hit && at < (uint32_t)TLIST) sh.group[at] = group;
}

// Lists the listed groups' values at or above a key. One barrier.
template <typename T>
__device__ __forceinline__ void list_values(const RowView<T>& rv, int32_t per, uint32_t least, TopShared& sh) {
  constexpr int EPV = Elem<T>::EPV;
  constexpr int AHEAD = 4;  // vectors a thread has in flight
  const uint32_t tid = threadIdx.x, groups = sh.groups;
  if (groups <= (uint32_t)TLIST) {
    for (uint32_t i0 = tid; i0 < groups * SEG_V; i0 += TT * AHEAD) {
      uint4 q[AHEAD];
      int32_t v[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        const uint32_t i = i0 + u * TT;
        v[u] = -1;
        if (i < groups * SEG_V) {
          const uint32_t g = sh.group[i / SEG_V];
          const int32_t v0 = (int32_t)(g / TT) * per;
          const int32_t at = v0 + group_of((int32_t)(g % TT)) + (int32_t)(i % SEG_V);
          if (at < min(rv.nvec, v0 + per)) {
            v[u] = at;
            q[u] = load_vec(rv, at);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (v[u] < 0 || key_of(vec_max_nan<T>(q[u])) < least) continue;
        float x[EPV];
        Elem<T>::unpack(q[u], x);
#pragma unroll
        for (int j = 0; j < EPV; ++j) {
          const uint32_t kx = key_of(x[j]);
          const int32_t e = rv.first(v[u]) + j;
          if (kx >= least && e >= 0 && e < rv.V) {
            const uint32_t at = atomicAdd(&sh.n, 1u);
            if (at < (uint32_t)TCAP) sh.list[at] = compose(kx, (uint32_t)e);
          }
        }
      }
    }
  }
  __syncthreads();
}

// The lists once more, for a key above the one that too many values reach: most of those equal it
// (masked values, as a rule). Whether they fit now.
template <typename T>
__device__ __noinline__ bool list_above(const RowView<T>& rv, SegPlan seg, const uint32_t* keys, uint32_t least,
                                        TopShared& sh) {
  __syncthreads();
  if (threadIdx.x == 0) sh.groups = sh.n = 0;
  __syncthreads();
  for (int32_t s = 0; s < seg.segs; ++s)
    list_group(sh, (uint32_t)s * TT + threadIdx.x, __ldcg(keys + (int64_t)s * TT) >= least);
  __syncthreads();
  list_values<T>(rv, seg.per, least, sh);
  return sh.groups <= (uint32_t)TLIST && sh.n <= (uint32_t)TCAP;
}

// Adds to the sh.n listed candidates those of the row's elements of this key that have the lowest
// indices, up to k candidates.
template <typename T>
__device__ __noinline__ void add_equals(const RowView<T>& rv, uint32_t key, uint32_t k, TopShared& sh) {
  constexpr int EPV = Elem<T>::EPV;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t n = sh.n;
  for (int32_t v0 = 0; v0 < rv.nvec && n < k; v0 += TT) {  // (every thread has the same n)
    const int32_t v = v0 + tid, e0 = rv.first(v);
    uint32_t eq = 0;
    if (v < rv.nvec) {
      float x[EPV];
      Elem<T>::unpack(load_vec(rv, v), x);
#pragma unroll
      for (int q = 0; q < EPV; ++q) eq |= (key_of(x[q]) == key && e0 + q >= 0 && e0 + q < rv.V ? 1u : 0u) << q;
    }
    const uint32_t mine = (uint32_t)__popc(eq), incl = warp_incl_scan(mine);
    if (lane == 31) sh.steps[warp] = incl;
    __syncthreads();
    uint32_t at = n + incl - mine;
    for (int w = 0; w < TNW; ++w) {
      if (w < warp) at += sh.steps[w];
      n += sh.steps[w];
    }
    for (; eq && at < k; eq &= eq - 1, ++at) sh.list[at] = compose(key, (uint32_t)(e0 + __ffs(eq) - 1));
    __syncthreads();
  }
}

// CTA (row, segment): the keys of its groups and its sum. Bound by HBM: [1024, 128256] bf16 (263 MB) in 46
// us, 5.8 TB/s (89% of the measured copy rate).
template <typename T>
__global__ void __launch_bounds__(TT, SEG_CTAS) part_kernel(TopArgs a) {
  __shared__ ExpSum scratch[TNW];
  const int64_t row = blockIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  load_segment(rv, v0, v1, q);
  grid_release();
  const int64_t part = row * a.seg.segs + blockIdx.y;
  a.keys[part * TT + threadIdx.x] = key_of(group_largest<T>(q));
  const ExpSum sum = block_expsum<TNW>(sum_segment<T>(q, v1 - v0, a.c).total(), a.c, scratch);
  if (threadIdx.x == 0) a.parts[part] = sum;
}

// A CTA per row, as above. Latency (the keys, the bound, the groups, the order, each after the one before),
// 592 rows at a time: 9 us for 256 rows of k 50, 30 us for 1024 of k 128. (Six CTAs to an SM did not shorten
// it.)
template <typename T>
__global__ void __launch_bounds__(TT, 4) select_kernel(TopArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ TopShared sh;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t segs = a.seg.segs;
  if (tid == 0) sh.groups = sh.n = 0;
  sh.hist[tid] = 0;
  grid_wait();  // the segments' keys and sums
  const uint32_t* keys = a.keys + row * segs * TT + tid;
  constexpr int HELD = 16;  // keys a thread keeps; longer rows' are read twice
  uint32_t key[HELD], lmax = 0;
#pragma unroll
  for (int s = 0; s < HELD; ++s) key[s] = s < segs ? __ldcg(keys + s * TT) : 0u;
  ExpSum sum = expsum_empty();
  for (int32_t s = tid; s < segs; s += TT) {
    const float2 p = __ldcg(reinterpret_cast<const float2*>(a.parts + row * segs + s));
    sum = expsum_join(sum, ExpSum{p.x, p.y}, a.c);
  }
#pragma unroll
  for (int s = 0; s < HELD; ++s) lmax = max(lmax, key[s]);
  for (int32_t s = HELD; s < segs; ++s) lmax = max(lmax, __ldcg(keys + (int64_t)s * TT));
  const uint32_t wb = warp_nth_largest(lmax, (a.k + TNW - 1) / TNW);
  const uint32_t wt = __reduce_max_sync(0xFFFFFFFFu, lmax);
  sum = warp_expsum(sum, a.c);
  if (lane == 0) {
    sh.bound[warp] = wb;
    sh.top[warp] = wt;
    sh.sum[warp] = sum;
  }
  __syncthreads();
  uint32_t bound = sh.bound[0], top = sh.top[0];
#pragma unroll
  for (int w = 1; w < TNW; ++w) {
    bound = min(bound, sh.bound[w]);
    top = max(top, sh.top[w]);
  }
  // raise the bound: group keys at or above it, by step; then the steps from the top until k are held
  // (each group's key is a value of the row, so k values reach the last of these steps)
  const int shift = max(0, 24 - __clz(top - bound));  // the span above the bound in at most TT steps
  auto count_key = [&](uint32_t k) {
    if (k >= bound) atomicAdd(&sh.hist[(k - bound) >> shift], 1u);
  };
#pragma unroll
  for (int s = 0; s < HELD; ++s)
    if (s < segs) count_key(key[s]);
  for (int32_t s = HELD; s < segs; ++s) count_key(__ldcg(keys + (int64_t)s * TT));
  if (warp == 0) {
    sum = warp_expsum(lane < TNW ? sh.sum[lane] : expsum_empty(), a.c);
    if (lane == 0) sh.sum[0] = sum;
  }
  __syncthreads();
  {
    const uint32_t h = sh.hist[TT - 1 - tid];  // from the top step down
    const uint32_t incl = warp_incl_scan(h);
    if (lane == 31) sh.steps[warp] = incl;
    if (tid == 0) sh.raised = bound;
    __syncthreads();
    uint32_t before = incl - h;
    for (int w = 0; w < warp; ++w) before += sh.steps[w];
    if (before < (uint32_t)a.k && before + h >= (uint32_t)a.k) sh.raised = bound + ((uint32_t)(TT - 1 - tid) << shift);
    __syncthreads();
  }
  sum = sh.sum[0];
  bound = sh.raised;

  // the groups that reach the bound, then the values in them that do
#pragma unroll
  for (int s = 0; s < HELD; ++s)
    if (s < segs) list_group(sh, (uint32_t)(s * TT + tid), key[s] >= bound);
  for (int32_t s = HELD; s < segs; ++s) list_group(sh, (uint32_t)(s * TT + tid), __ldcg(keys + (int64_t)s * TT) >= bound);
  __syncthreads();
  list_values<T>(rv, a.seg.per, bound, sh);
  bool fits = sh.groups <= (uint32_t)TLIST && sh.n <= (uint32_t)TCAP;
  if (!fits && bound != 0xFFFFFFFFu) fits = list_above<T>(rv, a.seg, keys, bound + 1, sh);
  constexpr float LN2 = 0.6931471805599453f;
  // NaN or +inf in the row (the sum is NaN then), or nothing above -inf: no distribution
  const float l = (sum.s == 0.0f) ? NAN : log2f(sum.s);
  if (tid == 0) a.lse[row] = sum.m / a.temperature + l * LN2;
  auto put = [&](uint32_t at, uint64_t e) {
    a.logprob[row * a.k + at] = (value_of(comp_key(e)) - sum.m) / a.temperature - l * LN2;
    a.index[row * a.k + at] = (int32_t)comp_idx(e);
  };
  uint32_t n = sh.n;
  if (!fits || n < (uint32_t)a.k) {
    __syncthreads();
    if (!fits) select_slow<T>(rv, a.k, sh);
    else add_equals<T>(rv, bound, (uint32_t)a.k, sh);
    n = (uint32_t)a.k;
  }
  if (n <= (uint32_t)TRANK) {
    // the place of each candidate: the number of those above it (no two are equal)
    if (tid == 0 && (n & 1)) sh.list[n] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += TT) {
      const uint64_t e = sh.list[i];
      uint32_t above = 0;
#pragma unroll 4
      for (uint32_t j = 0; j < n; j += 2) {
        const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(&sh.list[j]);
        above += (o.x > e ? 1u : 0u) + (o.y > e ? 1u : 0u);
      }
      if (above < (uint32_t)a.k) put(above, e);
    }
    return;
  }
  // a bitonic network over the next power of two, padded with zeros (below every entry)
  uint32_t size = 2 * TRANK;
  while (size < n) size <<= 1;
  for (uint32_t i = n + tid; i < size; i += TT) sh.list[i] = 0;
  __syncthreads();
  for (uint32_t k2 = 2; k2 <= size; k2 <<= 1)
    for (uint32_t j = k2 >> 1; j > 0; j >>= 1) {
      for (uint32_t i = tid; i < size / 2; i += TT) {
        const uint32_t p = ((i & ~(j - 1)) << 1) | (i & (j - 1)), p2 = p | j;
        const uint64_t x = sh.list[p], y = sh.list[p2];
        if ((x < y) == ((p & k2) == 0)) {
          sh.list[p] = y;
          sh.list[p2] = x;
        }
      }
      __syncthreads();
    }
  for (int i = tid; i < a.k; i += TT) put(i, sh.list[i]);
}

struct TopPlan {
  SegPlan seg;
  int64_t keys, bytes;  // offset of the keys in the workspace, and its size
};
TopPlan top_plan(int64_t n, int64_t V, int es, const void* rows, int64_t row_stride) {
  TopPlan p;
  p.seg = seg_plan(V, es, rows, row_stride);
  p.keys = (n * p.seg.segs * (int64_t)sizeof(ExpSum) + 255) & ~(int64_t)255;
  p.bytes = p.keys + n * p.seg.segs * TT * 4;
  return p;
}

template <typename T>
int top_run(const TopArgs& a, cudaStream_t st) {
  part_kernel<T><<<dim3((unsigned)a.n, (unsigned)a.seg.segs), TT, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return PB_E_LAUNCH;
  return launch_after(select_kernel<T>, a, dim3((unsigned)a.n), TT, st);
}

}  // namespace

extern "C" {

int64_t pb_top_ws_bytes(int64_t n_rows, int64_t vocab, int dtype) {
  const int es = elem_size(dtype);
  if (n_rows < 0 || vocab <= 0 || !es) return PB_E_INVALID;
  return top_plan(n_rows, vocab, es, nullptr, 1).bytes;  // (rows of any alignment: the most it takes)
}

int pb_top_logprobs(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, int32_t k,
                    float temperature, float* out_logprob, int32_t* out_index, float* out_lse, void* workspace,
                    int64_t ws_bytes, void* stream) {
  const int es = elem_size(dtype);
  if (n_rows < 0 || vocab <= 0 || row_stride < 0 || !es) return PB_E_INVALID;
  if (vocab >= PB_MAX_VOCAB) return PB_E_TOO_LARGE;
  if (k < 1 || k > TKMAX || k > vocab) return PB_E_INVALID;
  if (!(temperature >= 0x1p-20f && temperature <= 0x1p20f)) return PB_E_INVALID;
  if (n_rows == 0) return PB_OK;
  if (!logits || !out_logprob || !out_index || !out_lse) return PB_E_INVALID;
  if (n_rows > (int64_t)(0x7FFFFFFF / 8)) return PB_E_INVALID;
  if (!aligned(logits, es) || !aligned(out_logprob, 4) || !aligned(out_index, 4) || !aligned(out_lse, 4)) return PB_E_INVALID;
  const TopPlan plan = top_plan(n_rows, vocab, es, logits, row_stride);
  if (!workspace || !aligned(workspace, 256) || ws_bytes < plan.bytes) return PB_E_INVALID;
  TopArgs a;
  a.x = logits;
  a.row_stride = row_stride;
  a.n = n_rows;
  a.V = (int32_t)vocab;
  a.k = k;
  a.c = (float)(1.4426950408889634 / (double)temperature);
  a.temperature = temperature;
  a.logprob = out_logprob;
  a.index = out_index;
  a.lse = out_lse;
  a.seg = plan.seg;
  a.parts = static_cast<ExpSum*>(workspace);
  a.keys = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + plan.keys);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return top_run<float>(a, st);
  if (dtype == PB_DTYPE_BF16) return top_run<__nv_bfloat16>(a, st);
  return top_run<__half>(a, st);
}

}  // extern "C"
