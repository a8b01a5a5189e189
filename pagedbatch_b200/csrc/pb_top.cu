// The k largest log-probabilities of each row, with their indices and the row's log-sum-exp: what a
// server returns as log-probabilities and what a teacher records for distillation.
//
//   y_j = x_j / T,  lse = log sum_j exp(y_j),  log p_j = y_j - lse
//   the k largest x in the order (value descending, index ascending), NaN above every value
//   (the sampler's order). A row holding NaN or +inf, or only -inf, has NaN log-probabilities.
//
// One cluster of C CTAs per row reads the row once. Every thread keeps a running maximum and sum of
// exponentials, and the key of the largest value of each run of TU vectors it loads together (its
// groups) in shared memory. A lower bound of the k-th largest value follows from the lanes' largest
// group keys: with W warps in the cluster, each warp's ceil(k / W)-th largest lane maximum is reached
// by that many values of the warp, so the smallest of these over the warps is reached by at least k
// values of the row. Only the groups whose key reaches the bound are read again (from L2); their
// values at or above it are the candidates, a little more than k, sorted in one CTA.
// HBM-bound: V * es bytes a row. A row with more candidates than the list holds (rows of very many
// equal values) is selected by bisection over (value, index) in its first CTA.
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int TT = 512;            // threads per CTA
constexpr int TNW = TT / 32;
constexpr int TU = 4;              // vectors a thread loads together: one group
constexpr int TKMAX = PB_TOP_MAX;   // largest k
constexpr int TCAP = 2048;         // candidates of a row
constexpr int TGROUPS = 16;        // groups a thread keeps; longer slices keep the largest of several

struct TopArgs {
  const void* x;
  int64_t row_stride;  // elements
  int64_t n;
  int32_t V, k;
  float c, temperature;  // log2(e) / T
  float* logprob;        // [n][k]
  int32_t* index;        // [n][k]
  float* lse;            // [n]
};

struct TopShared {
  ExpSum red[TNW];
  uint32_t bound[TNW], top[TNW];
  ExpSum pub_sum;
  uint32_t pub_bound;    // smallest of the CTA's warps' bounds
  uint32_t pub_max;      // largest key
  uint32_t n;            // rank 0: candidates of the row
  uint32_t cnt[2];       // bisection counts
  uint64_t list[TCAP];   // rank 0: candidates
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

template <typename T>
__global__ void __launch_bounds__(TT, 2) top_kernel(TopArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  extern __shared__ __align__(16) uint32_t keys[];  // [groups][TT]: keys of the thread's groups
  __shared__ TopShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)((int64_t)rv.nvec * rank / C), v1 = (int32_t)((int64_t)rv.nvec * (rank + 1) / C);
  const int32_t iters = (v1 - v0 + TT * TU - 1) / (TT * TU);
  const int32_t per = (iters + TGROUPS - 1) / TGROUPS;  // loads that share one kept key

  if (tid == 0) sh.n = 0;
  ExpSum acc = expsum_empty();
  uint32_t lmax = 0, gkey = 0;  // 0: below every key (a thread without vectors)
  for (int32_t it = 0; it < iters; ++it) {
    const int32_t vb = v0 + it * TT * TU + tid;
    uint4 q[TU];
#pragma unroll
    for (int u = 0; u < TU; ++u)
      if (vb + u * TT < v1) q[u] = load_vec(rv, vb + u * TT);
#pragma unroll
    for (int u = 0; u < TU; ++u) {
      if (vb + u * TT < v1) {
        float x[EPV];
        Elem<T>::unpack(q[u], x);
        gkey = max(gkey, key_of(vec_max_nan<T>(q[u])));
        expsum_add<T>(acc, x, a.c);
      }
    }
    if ((it + 1) % per == 0 || it + 1 == iters) {
      keys[(it / per) * TT + tid] = gkey;
      lmax = max(lmax, gkey);
      gkey = 0;
    }
  }

  // the bound of the k-th largest value, from the lanes' largest keys
  const int nth = (a.k + C * TNW - 1) / (C * TNW);
  const uint32_t wb = warp_nth_largest(lmax, nth);
  const uint32_t wm = __reduce_max_sync(0xFFFFFFFFu, lmax);
  if (lane == 0) {
    sh.bound[warp] = wb;
    sh.top[warp] = wm;
  }
  const ExpSum cta = block_expsum<TNW>(acc, a.c, sh.red);
  if (tid == 0) {
    uint32_t b = sh.bound[0], m = sh.top[0];
    for (int w = 1; w < TNW; ++w) {
      b = min(b, sh.bound[w]);
      m = max(m, sh.top[w]);
    }
    sh.pub_sum = cta;
    sh.pub_bound = b;
    sh.pub_max = m;
  }
  cluster_barrier(C);
  TopShared* first = C > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
  ExpSum all = first->pub_sum;
  uint32_t bound = first->pub_bound, mx = first->pub_max;
  for (int r = 1; r < C; ++r) {
    const TopShared* o = cluster.map_shared_rank(&sh, r);
    all = expsum_join(all, o->pub_sum, a.c);
    bound = min(bound, o->pub_bound);
    mx = max(mx, o->pub_max);
  }

  // candidates: values at or above the bound, from the groups whose key reaches it
  for (int32_t g = 0; g * per < iters; ++g) {
    if (keys[g * TT + tid] < bound) continue;
    for (int32_t it = g * per; it < min(iters, (g + 1) * per); ++it) {
      const int32_t vb = v0 + it * TT * TU + tid;
#pragma unroll
      for (int u = 0; u < TU; ++u) {
        const int32_t v = vb + u * TT;
        if (v >= v1) break;
        float x[EPV];
        Elem<T>::unpack(load_vec(rv, v), x);
#pragma unroll
        for (int q = 0; q < EPV; ++q) {
          const uint32_t key = key_of(x[q]);
          const int32_t e = rv.first(v) + q;
          if (key >= bound && e >= 0 && e < a.V) {
            const uint32_t at = atomicAdd(&first->n, 1u);
            if (at < (uint32_t)TCAP) first->list[at] = compose(key, (uint32_t)e);
          }
        }
      }
    }
  }
  cluster_barrier(C);
  if (rank != 0) return;
  uint32_t n = sh.n;
  if (n > (uint32_t)TCAP) {
    __syncthreads();
    select_slow<T>(rv, a.k, sh);
    n = (uint32_t)a.k;
  }
  // sort: a bitonic network over the next power of two, padded with zeros (below every entry)
  uint32_t size = 64;
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
  constexpr float LN2 = 0.6931471805599453f;
  // NaN or +inf in the row (the sum is NaN then), or nothing above -inf: no distribution
  const float l = (all.s == 0.0f) ? NAN : log2f(all.s);
  if (tid == 0) a.lse[row] = all.m / a.temperature + l * LN2;
  for (int i = tid; i < a.k; i += TT) {
    const uint64_t e = sh.list[i];
    a.logprob[row * a.k + i] = (value_of(comp_key(e)) - all.m) / a.temperature - l * LN2;
    a.index[row * a.k + i] = (int32_t)comp_idx(e);
  }
}

int top_cluster(int64_t n, int64_t bytes) {
  const int64_t want = 2 * (int64_t)device_sms();
  int C = 1;
  while (C < 8 && n * C < want && bytes / (2 * C) >= 8192) C <<= 1;
  return C;
}

template <typename T>
int top_run(const TopArgs& a, cudaStream_t st) {
  const int C = top_cluster(a.n, (int64_t)a.V * sizeof(T));
  constexpr int EPV = 16 / (int)sizeof(T);
  const int64_t nvec = ((int64_t)a.V + 2 * EPV - 2) / EPV, slice = (nvec + C - 1) / C;
  const int64_t iters = (slice + TT * TU - 1) / (TT * TU);
  const size_t smem = (size_t)std::min<int64_t>(iters, TGROUPS) * TT * 4;
  return launch_cluster(top_kernel<T>, a, a.n * C, TT, C, smem, st);
}

}  // namespace

extern "C" {

int pb_top_logprobs(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride, int32_t k,
                    float temperature, float* out_logprob, int32_t* out_index, float* out_lse, void* stream) {
  const int es = elem_size(dtype);
  if (n_rows < 0 || vocab <= 0 || row_stride < 0 || !es) return PB_E_INVALID;
  if (vocab >= PB_MAX_VOCAB) return PB_E_TOO_LARGE;
  if (k < 1 || k > TKMAX || k > vocab) return PB_E_INVALID;
  if (!(temperature >= 0x1p-20f && temperature <= 0x1p20f)) return PB_E_INVALID;
  if (n_rows == 0) return PB_OK;
  if (!logits || !out_logprob || !out_index || !out_lse) return PB_E_INVALID;
  if (n_rows > (int64_t)(0x7FFFFFFF / 8)) return PB_E_INVALID;
  if (reinterpret_cast<uintptr_t>(logits) % es) return PB_E_INVALID;
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
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return top_run<float>(a, st);
  if (dtype == PB_DTYPE_BF16) return top_run<__nv_bfloat16>(a, st);
  return top_run<__half>(a, st);
}

}  // extern "C"
