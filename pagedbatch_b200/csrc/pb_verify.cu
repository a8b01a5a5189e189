// Verification of drafted tokens against the target's distribution, from given random numbers.
//
// A sequence owns a run of target rows: one for each of its drafts and one more. Row r's target
// distribution is the sampler's own for the sequence's parameters: weights P_i = q_i on the kept set,
// Z their sum (fixed point, exact). With u the row's random number and d the draft's probability
// (its distribution at the drafted token x, or 1 for a draft without a distribution):
//   accept x     iff  (u * d) * Z < P_x                      (fp64, each product rounded once)
//   first reject:     draw from max(0, P_i - floor(d_i * Z)) (or from P without x)
//   all accepted:     draw from P at the last row
// The draw goes by the random number of the sequence's last row, which no acceptance has looked at
// (given a rejection, the rejected row's own number is no longer uniform).
// A draw takes t = floor(U53 * R / 2^53), R the sum, and the first index (ascending) whose inclusive
// prefix exceeds t; an empty residual is replaced by P. Greedy rows accept the first maximum only.
// Both steps leave every token distributed as the target's own samples are.
//
// Launches, each of which may start while the one before it ends:
//   1. expand_kernel: each row's parameters from its sequence's.
//   2. each row's kept set and its mass, as the sampler's info record describes them. Greedy and small
//      top-k rows: pb_sample_ws. Rows without filters, whose kept set is the whole row: max_kernel, the
//      largest value and a sum of exponentials near the mass, all that most decisions need. Rows
//      with top-p alone: max_kernel, then hist_kernel sums the weights in 512 steps of the key,
//      cut_kernel finds the step in which the mass passes top-p, gather_kernel lists its elements and
//      order_kernel finds the last kept one among them. Every other row (large top-k, a step of too
//      many elements, rejected parameters): the sampler's cluster kernel. Rows of kinds that the caller does not
//      name but allows (PB_VERIFY_REST): pb_sample_ws's or the cluster kernel, whichever is launched.
//   3. decide_kernel: a CTA per sequence finds the first rejected row.
//   4. mass_kernel: that row's mass, where it has no filters.
//   5. weigh_kernel: that row's weights, summed per tile (256 vectors), a CTA per segment.
//   6. draw_kernel: a CTA per sequence finds the draw's tile and its element.
// Weights are exact integers throughout (multiples of 2^-40 below 2^13, which fp64 adds without
// rounding), so no result depends on an order of addition.
#include "pb_internal.h"
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int VT = SEG_T;        // threads per CTA
constexpr int VNW = SEG_NW;
constexpr int SMALL_K = 128;      // largest top_k that pb_sample_ws's two passes settle
constexpr int TILES = SEG_V;     // tiles per segment: tile i holds vectors v0 + i * SEG_T + thread

// A row as the passes over whole rows see it.
enum : int32_t { ROW_SMALL = 0, ROW_WHOLE = 1, ROW_MASS = 2, ROW_OTHER = 3 };  // what settles a row
struct RowMeta {
  float t;           // temperature
  int32_t kind;      // ROW_*
  uint32_t max_key;  // key of its largest value (max_kernel)
  uint32_t listed;   // ROW_MASS: elements of the step where top-p cuts (gather_kernel)
  uint64_t above;    // ... mass above the step
  uint64_t cut;      // ... floor(top_p * mass)
  int32_t step;      // ... the step
  float top_p;
};

constexpr int WEIGH_CTAS = 3 * 148;    // CTAs of weigh_kernel that are on a B200 at once (3 on each SM)
constexpr int STEPS = 512;             // histogram steps of a row's key
constexpr float STEP_SCALE = STEPS / 28.0f;  // keys further than 27.73 below the maximum have no weight
constexpr int LIST = 2048;             // elements order_kernel takes from one step (a row has its vocabulary's at most)

// Sums of one tile of the row a sequence draws from, in units of 2^-40. Where top-p cut among the
// equals of the last kept key, `w` leaves those equals out, `tie_w` is theirs and `ties` counts them.
struct Tile {
  uint64_t w, tie_w;
  int32_t ties, pad;
};

// Where a sequence stopped: EV_TIE is a draft whose row has to be looked at again before it is decided.
enum : int32_t { EV_REJECT = 0, EV_BAD = 1, EV_TIE = 2, EV_LAST = 3 };
struct Decision {
  int64_t row;
  int32_t kind;   // EV_*
  int32_t draws;  // the last token is drawn from the row's weights
};

struct VerifyArgs {
  const void* x;
  int64_t row_stride;            // elements
  int64_t n_rows, n_seqs;
  int32_t V;
  const pb_row_params* params;   // [n_seqs]
  const int32_t* offsets;        // [n_seqs + 1]
  const int64_t* drafts;         // [n_rows]
  const double* uniforms;        // [n_rows]
  const void* probs;             // [n_probs][V], or null
  int64_t probs_stride, n_probs;
  int32_t probs_dtype;
  pb_row_params* rowp;           // workspace: [n_rows], what pb_sample_ws sees
  pb_row_params* rowq;           // workspace: [n_rows], the rows' own
  uint64_t* hist;                // workspace: [n_rows][STEPS] (a batch with ROW_MASS rows)
  uint64_t* list;                // ... [n_rows][list_len]
  int32_t list_len;              // LIST, or the vocabulary where it is smaller
  pb_row_info* info;             // workspace: [n_rows]
  int64_t* tok;                  // workspace: [n_rows], the sampler's tokens (greedy rows' maxima)
  RowMeta* meta;                 // workspace: [n_rows]
  ExpSum* sums;                  // workspace: [n_rows][segs], of ROW_WHOLE rows
  Decision* decision;            // workspace: [n_seqs]
  Tile* tiles;                   // workspace: [n_seqs][segs][TILES]
  SegPlan seg;
  int32_t share;                 // tiles per CTA of weigh_kernel: TILES, or its half, quarter or eighth
  GroupKeys groups;              // of the rows the sampler settled (keys null: none)
  int32_t kinds;                 // PB_VERIFY_* of the batch, as the caller names them
  int32_t rest;                  // what settles rows of other kinds (ROW_SMALL, ROW_OTHER), or -1
  int32_t one_kind;              // ROW_WHOLE or ROW_MASS where every row is of that kind, else -1
  int64_t* out_tokens;           // [n_rows]
  int32_t* out_accepted;         // [n_seqs]
  int32_t* out_status;           // [n_seqs] or null
};

// What settles a row of these parameters.
__device__ __forceinline__ int32_t row_kind(const pb_row_params& p, int32_t V) {
  if (!(p.temperature >= 0.0) || !(p.top_p > 0.0 && p.top_p <= 1.0) || p.top_k < 0) return ROW_OTHER;  // rejected there
  if (p.temperature == 0.0) return ROW_SMALL;
  if (p.top_k > 0 && p.top_k < V) return p.top_k <= SMALL_K ? ROW_SMALL : ROW_OTHER;
  return (float)p.top_p < 1.0f ? ROW_MASS : ROW_WHOLE;
}

// The launches that settle rows of a kind, as the caller names them (the one for other kinds takes top-p's
// too), and what settles a sequence's rows in this call.
__device__ __forceinline__ int32_t takes(int32_t kind) {
  return kind == ROW_SMALL  ? PB_VERIFY_SMALL
         : kind == ROW_WHOLE ? PB_VERIFY_WHOLE
         : kind == ROW_MASS  ? PB_VERIFY_TOPP | PB_VERIFY_OTHER
                             : PB_VERIFY_OTHER;
}
template <bool REST>
__device__ __forceinline__ int32_t settled_as(const VerifyArgs& a, const pb_row_params& p) {
  const int32_t kind = row_kind(p, a.V);
  return REST && !(a.kinds & takes(kind)) ? a.rest : kind;
}

// Each row's parameters, from its sequence's (a binary search over the offsets, which are brought into shared
// memory where they fit: each of its steps waits for the one before), and its records cleared. Latency alone:
// 5 us for 898 rows of 256 sequences.
__global__ void __launch_bounds__(256) expand_kernel(VerifyArgs a) {
  constexpr int HELD = 2048;
  __shared__ int32_t starts[HELD];
  grid_release();
  const bool held = a.n_seqs <= HELD;
  if (held) {
    for (int i = threadIdx.x; i < (int)a.n_seqs; i += 256) starts[i] = __ldg(a.offsets + i);
    __syncthreads();
  }
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= a.n_rows) return;
  int64_t lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before row r
  while (hi - lo > 1) {
    const int64_t mid = lo + ((hi - lo) >> 1);
    if ((int64_t)(held ? starts[mid] : __ldg(a.offsets + mid)) <= r) lo = mid;
    else hi = mid;
  }
  pb_row_params p = a.params[lo];
  p.uniform = 0.0;  // the sampler's own draw is not used
  p.rng = 0;
  const int32_t kind = a.rest >= 0 ? settled_as<true>(a, p) : settled_as<false>(a, p);
  a.meta[r] = RowMeta{(float)p.temperature, kind, 0u, 0u, 0ull, 0ull, 0, (float)p.top_p};
  a.rowq[r] = p;
  // rows of other kinds pass through pb_sample_ws as greedy ones, its cheapest
  if (kind != ROW_SMALL) p.temperature = 0.0, p.top_p = 1.0, p.top_k = 0;
  a.rowp[r] = p;
  pb_row_info* o = a.info + r;
  // until a launch settles the row: the sampler's cluster kernel, or (a kind that no launch is for) none
  o->status = kind == ROW_OTHER && a.rest == ROW_OTHER ? PB_ROW_FALLBACK : PB_ROW_INTERNAL;
  o->z_q = o->kept_q = 0;
  a.tok[r] = -1;
  a.out_tokens[r] = -1;
}

// x / T as the sampler rounds it: IEEE division, or the same value by the exact reciprocal of a
// power of two.
struct Scale {
  float t, inv;
  __device__ explicit Scale(float tf) : t(tf) {
    const uint32_t b = __float_as_uint(tf), e = (b >> 23) & 0xFF;
    inv = ((b & 0x807FFFFFu) != 0 || e < 1 || e > 253) ? 0.0f : __uint_as_float((254u - e) << 23);
  }
  __device__ __forceinline__ float operator()(float x) const {
    return (inv != 0.0f) ? __fmul_rn(x, inv) : __fdiv_rn(x, t);
  }
};

// Raw values below this are surely below the scaled key thr (a few roundings of the quotient apart).
__device__ __forceinline__ float surely_below(uint32_t thr, float tf) {
  if (!(thr > KEY_NEG_INF && thr < KEY_POS_INF)) return -INFINITY;
  const float b = value_of(thr) * tf, r = b - fabsf(b) * 0x1p-20f - 0x1p-100f;
  return (r > -INFINITY) ? r : -INFINITY;
}

// ---- weights ---------------------------------------------------------------------------------

// The sampler's weights of a vector's elements, e^(x / T - m) as exp_weight computes it (before its
// scaling to 2^40), for rows of ordinary values. Every step is the same correctly rounded operation,
// two elements at a time:
//  * x / T: a product with the exact reciprocal of a power of two, else by Markstein's division
//    (IBM J. Res. Dev. 34, 1990): with y = RN(1 / T), two corrections q += (x - q T) y, the remainders
//    exact in one fused operation each, give RN(x / T) while nothing over- or underflows. Values of
//    |x| < 2^-100 (a remainder may lie below the subnormals) or |x / T| < 2^-126 can miss a last bit. They
//    are below 2^-40 of the row's largest, so RN(y - max) is -max all the same and no weight sees it; a
//    comparison with the last kept key does, and rows whose cut is as near to 0 are not `fast` (DrawRow);
//  * keys further than 40 below the maximum, whose weight is below 2^-40, are taken as 40 below it.
struct Weigher {
  float t, recip, inv, m;
  bool fast;  // the row's values are ordinary enough for the packed steps
  static constexpr float MAGIC = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number
  __device__ Weigher(float t_, float m_, float raw_max) : t(t_), m(m_) {
    const Scale s(t_);
    inv = s.inv;
    recip = __frcp_rn(t_);
    const float a = fabsf(raw_max);
    fast = a >= 0x1p-40f && a <= 0x1p60f && t_ >= 0x1p-40f && t_ <= 0x1p40f;
  }
  // weights w and scaled values y of a vector's elements
  template <typename T>
  __device__ __forceinline__ void of(uint4 v, float* w, float* y) const {
    constexpr int EPV = Elem<T>::EPV;
    float x[EPV];
    Elem<T>::unpack(v, x);
    if (!fast) {
      const Scale s(t);
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        y[q] = s(x[q]);
        w[q] = exp_weight(__fsub_rn(y[q], m));
      }
      return;
    }
    const uint64_t m2 = pack2(-m, -m);
#pragma unroll
    for (int q = 0; q < EPV; q += 2) {
      uint64_t k;
      if (inv != 0.0f) {
        k = mul2(pack2(x[q], x[q + 1]), pack2(inv, inv));
      } else {
        // (values below -2^100 have no weight: taken as that, so that -inf divides)
        const uint64_t x2 = pack2(fmaxf(x[q], -0x1p100f), fmaxf(x[q + 1], -0x1p100f)), y2 = pack2(recip, recip), t2 = pack2(-t, -t);
        k = mul2(x2, y2);
        k = fma2(fma2(k, t2, x2), y2, k);
        k = fma2(fma2(k, t2, x2), y2, k);
      }
      unpack2(k, y[q], y[q + 1]);
      float d0, d1;
      unpack2(add2(k, m2), d0, d1);
      d0 = fmaxf(d0, -40.0f), d1 = fmaxf(d1, -40.0f);
      const uint64_t d = pack2(d0, d1);
      // (the product in two scalar operations: a packed product and sum of .rn each were seen joined into
      // one rounding, which takes another n where d log2(e) rounds to a half)
      const uint64_t tn = add2(pack2(__fmul_rn(d0, 0x1.715476p+0f), __fmul_rn(d1, 0x1.715476p+0f)), pack2(MAGIC, MAGIC));
      const uint64_t n = add2(tn, pack2(-MAGIC, -MAGIC));
      uint64_t r = fma2(n, pack2(-0x1.62e43p-1f, -0x1.62e43p-1f), d);
      r = fma2(n, pack2(0x1.05c61p-29f, 0x1.05c61p-29f), r);
      uint64_t p = pack2(0x1.a01a02p-13f, 0x1.a01a02p-13f);
      p = fma2(p, r, pack2(0x1.6c16c2p-10f, 0x1.6c16c2p-10f));
      p = fma2(p, r, pack2(0x1.111112p-7f, 0x1.111112p-7f));
      p = fma2(p, r, pack2(0x1.555556p-5f, 0x1.555556p-5f));
      p = fma2(p, r, pack2(0x1.555556p-3f, 0x1.555556p-3f));
      p = fma2(p, r, pack2(0.5f, 0.5f));
      p = fma2(p, r, pack2(1.0f, 1.0f));
      p = fma2(p, r, pack2(1.0f, 1.0f));
      float p0, p1, n0, n1;
      unpack2(p, p0, p1);
      unpack2(tn, n0, n1);
      // (the low bits of MAGIC + n are n, and MAGIC's own leave the word with the shift)
      w[q] = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(n0) << 23));
      w[q + 1] = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(n1) << 23));
    }
  }
};

// Exact sums of weights floored to multiples of 2^-40: a double of 2^12 has its last place there, so
// adding to it towards minus infinity floors what is added. Room for 4095 weights of 1.
constexpr double GRID = 4096.0;
__device__ __forceinline__ double on_grid(float w) { return __dadd_rd(GRID, (double)w); }  // GRID + floor
__device__ __forceinline__ uint64_t grid_units(double sum) {                               // sum - GRID in 2^-40
  return (uint64_t)__double_as_longlong(sum) & ((1ull << 52) - 1);
}

// Base-2 exponent of a raw difference.
__device__ __forceinline__ float exponent_of(float t) { return __fdiv_rn(1.44269504f, t); }

// Key of the largest value of every row that is summed here, and for ROW_WHOLE rows the segment's sum of
// exponentials in fp32; clears the histograms of the others. Bound by HBM, the sums by issue nearly as much:
// 898 rows of 128256 bf16 (230 MB) in 44 us, 5.3 TB/s (30 us without the sums).
template <typename T>
__global__ void __launch_bounds__(VT, SEG_CTAS) max_kernel(VerifyArgs a) {
  __shared__ uint32_t top[VNW];
  __shared__ ExpSum scratch[VNW];
  grid_release();
  const int64_t row = blockIdx.x;
  if (a.one_kind < 0) {
    grid_wait();
    const int32_t kind = a.meta[row].kind;
    if (kind != ROW_WHOLE && !(kind == ROW_MASS && a.hist)) return;
  }
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  load_segment(rv, v0, v1, q);
  grid_wait();  // expand_kernel has set the keys to 0
  const RowMeta meta = a.meta[row];
  float largest;
  if (meta.kind == ROW_WHOLE && a.sums) {
    const float c = exponent_of(meta.t);
    const ExpSum sum = block_expsum<VNW>(sum_segment<T>(q, v1 - v0, c, &largest).total(), c, scratch);
    if (threadIdx.x == 0) a.sums[row * a.seg.segs + blockIdx.y] = sum;
  } else {
    largest = vecs_max_nan<T, SEG_V>(q);
    if (a.hist && blockIdx.y == 0)
      for (int i = threadIdx.x; i < STEPS; i += VT) a.hist[row * STEPS + i] = 0;
  }
  uint32_t k = __reduce_max_sync(0xFFFFFFFFu, key_of(largest));
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = k;
  __syncthreads();
  if (threadIdx.x < 32) {
    k = __reduce_max_sync(0xFFFFFFFFu, threadIdx.x < VNW ? top[threadIdx.x] : 0u);
    if (threadIdx.x == 0) atomicMax(&a.meta[row].max_key, k);
  }
}

// What is known of a ROW_WHOLE row's mass Z (in 2^-40, as the sampler rounds it) from its segments' sums:
// lo <= Z <= hi. With u = 2^-24 and M the largest key, Z differs from the sum S of e^((x - max) / T) by
//   a weight's key, its distance and its exponential:  S u (2 |M| + 58)
//   its floor, or its absence beyond 27.73:            2^-40 an element
// and the fp32 sums from S, elements below 2^-40 of the largest left aside, by at most u S times
//   132 for an element (its exponent, 40 at most: 64 and 40 for the two roundings, 80 for the factor c, all by
//   ln 2; 4 for ex2), 33 for a thread's additions, 5 for a warp's and 5 for a block's, 2 for each segment,
//   and 116 for each change of the largest value: two in a thread, one in the warp, one in the block, one here
// which is below 1000 u S + 2 segs u S. A sum that is not finite, or a temperature near the ends of the
// range, tells nothing: hi is infinite.
struct Mass {
  double lo, hi;
};
__device__ __forceinline__ Mass mass_near(const VerifyArgs& a, int64_t row, float t, float raw_max, float m) {
  const float c = exponent_of(t);
  float s = 0.0f;
  for (int32_t i = 0; i < a.seg.segs; ++i) {
    const float2 p = __ldcg(reinterpret_cast<const float2*>(a.sums + row * a.seg.segs + i));
    s += p.y * ex2((p.x - raw_max) * c);
  }
  const double off = 0x1p-24 * (1000.0 + 2.1 * (double)fabsf(m) + 2.0 * a.seg.segs), sum = (double)s * 0x1p40;
  if (!(s < INFINITY) || !(off < 0.25) || !(t >= 0x1p-20f && t <= 0x1p20f)) return Mass{0.0, INFINITY};
  const double few = 1.1 * (double)a.V;
  return Mass{sum * (1.0 - off) - few, sum * (1.0 + off) + few};
}

// The mass of the rows that sequences draw a residual from: the sum of the row's weights, a CTA per segment.
// Bound by issue and the FMA pipe, not by memory: 18 instructions a 32 elements (the exponential's polynomial
// in pairs, the exact sums), 256 rows of 128256 bf16 in 18 us. (Scalar arithmetic took longer: 233 us a call
// against 209 us. The masses of all 898 rows, before the decisions and instead of the near sums: 88 us.)
template <typename T>
__global__ void __launch_bounds__(VT, 4) mass_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ uint64_t part[VNW];
  grid_release();
  grid_wait();  // the decisions
  const Decision d = a.decision[blockIdx.x];
  if (!d.draws || d.kind != EV_REJECT) return;
  const RowMeta meta = a.meta[d.row];
  if (meta.kind != ROW_WHOLE) return;
  const RowView<T> rv(static_cast<const T*>(a.x) + d.row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  load_segment(rv, v0, v1, q);
  const float raw = value_of(meta.max_key);
  const Weigher weigh(meta.t, Scale(meta.t)(raw), raw);
  double s0 = GRID, s1 = GRID;  // (at most SEG_V * EPV weights of 1 in both)
#pragma unroll
  for (int i = 0; i < SEG_V; ++i) {
    if (i * SEG_T >= v1 - v0) break;
    float w[EPV], y[EPV];
    weigh.template of<T>(q[i], w, y);  // elements outside the row are -inf: no weight
#pragma unroll
    for (int j = 0; j < EPV; j += 2) {
      s0 = __dadd_rd(s0, (double)w[j]);
      s1 = __dadd_rd(s1, (double)w[j + 1]);
    }
  }
  uint64_t z = warp_sum(grid_units(s0) + grid_units(s1));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = z;
  __syncthreads();
  if (threadIdx.x < 32) {
    z = warp_sum(threadIdx.x < VNW ? part[threadIdx.x] : 0ull);
    if (threadIdx.x == 0) {  // (whole numbers: the order of the segments does not matter)
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.info[d.row].z_q), (unsigned long long)z);
      atomicAdd(reinterpret_cast<unsigned long long*>(&a.info[d.row].kept_q), (unsigned long long)z);
    }
  }
}

// The mass of one row, by one CTA: for the few drafts that mass_near's bounds do not settle.
template <typename T>
__device__ __noinline__ uint64_t mass_of(const RowView<T>& rv, float t, float m, float raw, uint64_t* scan) {
  constexpr int EPV = Elem<T>::EPV;
  const Weigher weigh(t, m, raw);
  uint64_t z = 0;
  for (int32_t v = threadIdx.x; v < rv.nvec; v += VT) {
    float w[EPV], y[EPV];
    weigh.template of<T>(load_vec(rv, v), w, y);
    double s = GRID;
#pragma unroll
    for (int j = 0; j < EPV; ++j) s = __dadd_rd(s, (double)w[j]);
    z += grid_units(s);
  }
  uint64_t total;
  block_excl_scan<uint64_t, VT>(z, scan, &total);
  return total;
}

// ---- top-p alone -----------------------------------------------------------------------------

// Step in its row's histogram of a key d below the largest (d = RN(y - m), not below -28): the whole number
// next to -d * STEP_SCALE, which does not fall as the key falls.
__device__ __forceinline__ int32_t step_of(float d) {
  return __float_as_int(__fmaf_rn(d, -STEP_SCALE, Weigher::MAGIC)) - __float_as_int(Weigher::MAGIC);
}

// lo[0] + 2^32 lo[STEPS] += u, in shared memory (nothing for u = 0; a carry is rare).
__device__ __forceinline__ void add_to_step(uint32_t* lo, uint64_t u) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(lo);
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      ".reg .u32 l, h, old;\n"
      "mov.b64 {l, h}, %1;\n"
      "mov.u32 old, 0;\n"
      "setp.ne.u64 p, %1, 0;\n"
      "@p atom.shared.add.u32 old, [%0], l;\n"
      "add.cc.u32 l, old, l;\n"
      "addc.u32 h, h, 0;\n"
      "setp.ne.u32 q, h, 0;\n"
      "@q red.shared.add.u32 [%0 + %2], h;\n"
      "}\n" ::"r"(at), "l"(u), "n"(STEPS * 4)
      : "memory");
}

// Sums of the weights of every ROW_MASS row, by step: shared-memory atomics for the segment, then one
// global atomic a step that holds weight (whole numbers: no order shows). Bound by issue: about 36
// instructions a 32 elements, 256 rows of 49152 bf16 in 24 us. (With the cut found by the sampler's cluster kernel, a
// cluster's repeated sums over its row, the whole call took 238 us instead of 139 us.)
template <typename T>
__global__ void __launch_bounds__(VT, 3) hist_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ uint32_t lo[2 * STEPS];  // 64-bit sums: low words, then high words
  grid_release();
  const int64_t row = a.n_rows - 1 - blockIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)(gridDim.y - 1 - blockIdx.y) * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  if (a.one_kind == ROW_MASS) load_segment(rv, v0, v1, q);
  for (int i = threadIdx.x; i < 2 * STEPS; i += VT) lo[i] = 0;
  grid_wait();  // the rows' largest values
  const RowMeta meta = a.meta[row];
  if (meta.kind != ROW_MASS) return;
  if (a.one_kind != ROW_MASS) load_segment(rv, v0, v1, q);
  const float raw = value_of(meta.max_key), m = Scale(meta.t)(raw);
  const uint32_t sk = key_of(m);
  if (meta.max_key == 0xFFFFFFFFu || sk >= KEY_POS_INF || sk <= KEY_NEG_INF) return;  // (no distribution)
  const Weigher weigh(meta.t, m, raw);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < SEG_V; ++i) {
    if (i * SEG_T >= v1 - v0) break;
    float w[EPV], y[EPV];
    weigh.template of<T>(q[i], w, y);
#pragma unroll
    for (int j = 0; j < EPV; ++j) {
      // (below -28 there is no weight and nothing is added: the address is any)
      const int32_t s = step_of(fmaxf(__fsub_rn(y[j], m), -27.75f));
      add_to_step(lo + s, grid_units(on_grid(w[j])));
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < STEPS; i += VT) {
    const unsigned long long u = (uint64_t)lo[STEPS + i] << 32 | lo[i];
    if (u) atomicAdd(reinterpret_cast<unsigned long long*>(a.hist + row * STEPS + i), u);
  }
}

// The step in which a ROW_MASS row's mass passes top-p: the last one that holds weight and has at most
// floor(top_p * mass) above it. All weights of the steps above it are kept, none of those below. Latency
// alone: 3 us.
__global__ void __launch_bounds__(VT) cut_kernel(VerifyArgs a) {
  __shared__ uint64_t scan[VNW + 1];
  __shared__ int32_t last;
  grid_release();
  const int64_t row = blockIdx.x;
  if (threadIdx.x == 0) last = 0;
  grid_wait();
  const RowMeta meta = a.meta[row];
  if (meta.kind != ROW_MASS) return;
  const float m = Scale(meta.t)(value_of(meta.max_key));
  const uint32_t sk = key_of(m);
  if (meta.max_key == 0xFFFFFFFFu || sk >= KEY_POS_INF || sk <= KEY_NEG_INF) {
    if (threadIdx.x == 0) a.info[row].status = PB_ROW_NONFINITE;
    return;
  }
  constexpr int PER = STEPS / VT;
  const uint64_t* h = a.hist + row * STEPS + threadIdx.x * PER;
  uint64_t v[PER], sum = 0, z;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += v[i] = __ldcg(h + i);
  uint64_t above = block_excl_scan<uint64_t, VT>(sum, scan, &z);
  const uint64_t cut = mul_floor(meta.top_p, z), first = above;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (v[i] && above <= cut) atomicMax(&last, (int32_t)threadIdx.x * PER + i);
    above += v[i];
  }
  __syncthreads();
  if ((int32_t)threadIdx.x == last / PER) {
    above = first;
    for (int i = 0; i < last % PER; ++i) above += v[i];
    RowMeta* o = a.meta + row;
    o->above = above;
    o->cut = cut;
    o->step = last;
    o->listed = 0;
    a.info[row].z_q = z;
    a.info[row].max_key = m;
  }
}

// The elements of that step, in any order, listed by each CTA for itself and then added to the row's list. A vector is left after one comparison of its largest element;
// elements surely outside the step by their raw values after two. 256 rows of 49152 bf16 in 14 us, the rows
// from L2, bound by issue.
template <typename T>
__global__ void __launch_bounds__(VT, 4) gather_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ uint64_t list[LIST];
  __shared__ uint32_t found, base;
  grid_release();
  const int64_t row = blockIdx.x;
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(rv.nvec, v0 + a.seg.per);
  uint4 q[SEG_V];
  if (a.one_kind == ROW_MASS) load_segment(rv, v0, v1, q);
  grid_wait();
  const RowMeta meta = a.meta[row];
  if (meta.kind != ROW_MASS || a.info[row].status == PB_ROW_NONFINITE) return;
  if (a.one_kind != ROW_MASS) load_segment(rv, v0, v1, q);
  const Scale scaled(meta.t);
  const float m = a.info[row].max_key;
  if (threadIdx.x == 0) found = 0;
  __syncthreads();
  // raw values that are surely below the step, or above it
  const float raw_lo = surely_below(key_of(m - ((float)meta.step + 1.0f) / STEP_SCALE), meta.t);
  const float above = (m - ((float)meta.step - 1.0f) / STEP_SCALE) * meta.t;
  const float raw_hi = above + fabsf(above) * 0x1p-20f + 0x1p-100f;  // (NaN or infinite: no bound)
#pragma unroll
  for (int i = 0; i < SEG_V; ++i) {
    if (!(vec_max_nan<T>(q[i]) >= raw_lo)) continue;
    float x[EPV];
    Elem<T>::unpack(q[i], x);
    uint32_t near = 0;
#pragma unroll
    for (int j = 0; j < EPV; ++j) near |= (x[j] >= raw_lo && !(x[j] > raw_hi) ? 1u : 0u) << j;
    const int32_t e0 = rv.first(v0 + i * SEG_T + (int32_t)threadIdx.x);
    while (near) {
      const int j = __ffs(near) - 1;
      near &= near - 1;
      const float y = scaled(Elem<T>::elem(q[i], j));
      if (e0 + j < 0 || e0 + j >= a.V || !weight_q(y, m) || step_of(__fsub_rn(y, m)) != meta.step) continue;
      const uint32_t at = atomicAdd(&found, 1u);
      if (at < (uint32_t)LIST) list[at] = compose(key_of(y), (uint32_t)(e0 + j));
    }
  }
  __syncthreads();
  const uint32_t n = found;
  if (threadIdx.x == 0 && n) base = atomicAdd(&a.meta[row].listed, n);
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n && base + i < (uint32_t)a.list_len; i += VT) a.list[row * a.list_len + base + i] = list[i];
}

// The last kept element among them, in the order (key descending, index ascending): what the row's
// record needs. Rows of other kinds, and steps of more elements than the list holds (or none: no step
// was looked for), are left to the sampler. Latency: a bitonic network over the list, 11 us for lists of
// several hundred.
__global__ void __launch_bounds__(VT) order_kernel(VerifyArgs a) {
  __shared__ uint64_t list[LIST];
  __shared__ uint64_t scan[VNW + 1];
  __shared__ int32_t kept;
  __shared__ uint64_t kept_q;
  grid_wait();
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  const RowMeta meta = a.meta[row];
  pb_row_info* o = a.info + row;
  if (meta.kind == ROW_OTHER || (meta.kind == ROW_MASS && o->status != PB_ROW_NONFINITE && (meta.listed == 0 || meta.listed > (uint32_t)a.list_len))) {
    if (tid == 0) o->status = PB_ROW_FALLBACK;
    return;
  }
  if (meta.kind != ROW_MASS || o->status == PB_ROW_NONFINITE) return;
  const int32_t n = (int32_t)meta.listed;
  uint32_t size = 2;
  while (size < (uint32_t)n) size <<= 1;
  for (uint32_t i = tid; i < size; i += VT) list[i] = i < (uint32_t)n ? __ldcg(a.list + row * a.list_len + i) : 0ull;
  if (tid == 0) kept = 0, kept_q = 0;
  __syncthreads();
  for (uint32_t k = 2; k <= size; k <<= 1)
    for (uint32_t j = k >> 1; j > 0; j >>= 1) {
      for (uint32_t i = tid; i < size / 2; i += VT) {
        const uint32_t p = ((i & ~(j - 1)) << 1) | (i & (j - 1)), p2 = p | j;
        const uint64_t x = list[p], y = list[p2];
        if ((x < y) == ((p & k) == 0)) {
          list[p] = y;
          list[p2] = x;
        }
      }
      __syncthreads();
    }
  // kept: those whose exclusive prefix of the mass is at most the cut (a prefix of the list)
  const float m = o->max_key;
  uint64_t base = meta.above;
  for (int32_t i0 = 0; i0 < n; i0 += VT) {
    const int32_t i = i0 + tid;
    const uint64_t q = i < n ? weight_q(value_of(comp_key(list[i])), m) : 0;
    uint64_t total;
    const uint64_t before = base + block_excl_scan<uint64_t, VT>(q, scan, &total);
    if (i < n && before <= meta.cut) {
      atomicMax(&kept, i + 1);
      atomicMax(reinterpret_cast<unsigned long long*>(&kept_q), (unsigned long long)(before + q));
    }
    base += total;
  }
  __syncthreads();
  if (tid == 0) {
    const uint32_t thr = comp_key(list[kept - 1]);
    int32_t first = kept - 1;
    while (first > 0 && comp_key(list[first - 1]) == thr) --first;
    o->thr_key = thr;
    o->n_tie_kept = kept - first;
    o->kept_count = 0;  // (not needed here)
    o->status = PB_ROW_OK;
    o->flags = PB_PATH_LARGE;
    o->kept_q = kept_q;
  }
}

// ---- deciding --------------------------------------------------------------------------------

__device__ __forceinline__ float prob_at(const VerifyArgs& a, int64_t d, int64_t i) {
  const int64_t at = d * a.probs_stride + i;
  if (a.probs_dtype == PB_DTYPE_F32) return __ldg(static_cast<const float*>(a.probs) + at);
  if (a.probs_dtype == PB_DTYPE_BF16) return Elem<__nv_bfloat16>::ld(static_cast<const __nv_bfloat16*>(a.probs) + at);
  return Elem<__half>::ld(static_cast<const __half*>(a.probs) + at);
}

// The row a sequence draws its last token from, and the weights of its elements.
template <typename T>
struct DrawRow {
  static constexpr int EPV = Elem<T>::EPV;
  const VerifyArgs& a;
  RowView<T> rv;
  pb_row_info f;
  Scale scaled;
  Weigher weigh;
  double z;          // mass, in the weights' own scale
  float d_most;      // draft probabilities above this take all of any weight, and stay on the grid below
  int64_t dx, drow;  // the rejected draft; its row of draft_probs
  bool residual, dist, cut_ties, whole;
  float raw_lo, thr;  // raw values below raw_lo have no weight (a key's order is its value's: the row holds no NaN)
  __device__ DrawRow(const VerifyArgs& a_, int64_t seq, const Decision& d, float tf, const pb_row_info& f_)
      : a(a_), rv(static_cast<const T*>(a_.x) + d.row * a_.row_stride, a_.V), f(f_), scaled(tf),
        weigh(tf, f_.max_key, f_.max_key * tf) {
    residual = d.kind == EV_REJECT;
    dx = residual ? a.drafts[d.row] : -1;
    drow = d.row - seq;
    dist = residual && a.probs && drow >= 0 && drow < a.n_probs;
    cut_ties = f.kept_q != f.z_q;
    whole = f.thr_key == 0;
    // (a key more than 28 below the largest has no weight, kept or not: masked values among a top-k)
    raw_lo = fmaxf(surely_below(f.thr_key, tf), surely_below(key_of(f.max_key - 28.0f), tf));
    thr = value_of(f.thr_key);
    // (the quotients that the packed steps may miss are below 2^-60, as T >= 2^-40)
    if (fabsf(thr) < 0x1p-59f) weigh.fast = false;
    z = __ull2double_rn(f.kept_q) * 0x1p-40;
    d_most = 2048.0f / (float)z;  // (anywhere between 1 / Z and 4095 / Z would do)
  }
  // The draft's probabilities of a whole vector, where they can be loaded as vectors of their own.
  __device__ __forceinline__ bool packed_probs(int32_t v) const {
    return dist && a.probs_dtype == PB_DTYPE_F32 && rv.whole(v) &&
           (reinterpret_cast<uintptr_t>(static_cast<const float*>(a.probs) + drow * a.probs_stride + rv.first(v)) & 15) == 0;
  }
  __device__ __forceinline__ void load_probs(int32_t v, float4* d) const {
    const float4* p = reinterpret_cast<const float4*>(static_cast<const float*>(a.probs) + drow * a.probs_stride + rv.first(v));
#pragma unroll
    for (int q = 0; q < EPV / 4; ++q) d[q] = __ldg(p + q);
  }
  // GRID + floor(d * Z): NaN and what is below 0 take nothing. (Beyond the grid the floor is coarser,
  // and more than any weight all the same.)
  __device__ __forceinline__ double taken_by(float d) const {
    return __dadd_rd(GRID, __dmul_rn((double)fmaxf(d, 0.0f), z));
  }
  // max(p - taken, 0), by the sign bit of the difference (exact where it is not negative)
  static __device__ __forceinline__ double leaves(double p, double taken) {
    const long long r = __double_as_longlong(p - taken);
    return __longlong_as_double(r & ~(r >> 63));
  }
  // Weights of vector v (elements q4): target, or what the draft's distribution leaves of it, in the
  // grid's scale. `eq` gets a bit per element whose key equals the last kept one, where top-p cut
  // there. `have`: its draft probabilities are in d.
  __device__ __forceinline__ void of(int32_t v, uint4 q4, bool target, bool have, const float4* d4, double* r,
                                     uint32_t& eq) const {
    eq = 0;
#pragma unroll
    for (int q = 0; q < EPV; ++q) r[q] = 0.0;
    if (!(vec_max_nan<T>(q4) >= raw_lo)) return;
    const int32_t e0 = rv.first(v);
    float w[EPV], y[EPV];
    weigh.template of<T>(q4, w, y);
    uint32_t some = (1u << EPV) - 1u;  // elements of weight
    if (!rv.whole(v)) {
#pragma unroll
      for (int q = 0; q < EPV; ++q)
        if (e0 + q < 0 || e0 + q >= a.V) some &= ~(1u << q);
    }
    if (!whole) {
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        if (!(y[q] >= thr)) some &= ~(1u << q);
        if (cut_ties && y[q] == thr) eq |= 1u << q;
      }
      eq &= some;
    }
    if (!some) return;
    float d[EPV];
    if (dist && !target) {
      if (have) {
#pragma unroll
        for (int q = 0; q < EPV; q += 4) {
          d[q] = d4[q / 4].x;
          d[q + 1] = d4[q / 4].y;
          d[q + 2] = d4[q / 4].z;
          d[q + 3] = d4[q / 4].w;
        }
      } else {
#pragma unroll
        for (int q = 0; q < EPV; ++q) d[q] = ((some >> q) & 1u) ? prob_at(a, drow, e0 + q) : 0.0f;
      }
    }
    if (dist && !target && some == (1u << EPV) - 1u) {  // the common case, without selections
#pragma unroll
      for (int q = 0; q < EPV; ++q) r[q] = leaves(on_grid(w[q]), taken_by(d[q]));
      return;
    }
#pragma unroll
    for (int q = 0; q < EPV; ++q) {
      const double p = on_grid(w[q]);
      double taken = GRID;
      if (!target) {
        if (dist) taken = taken_by(d[q]);
        else if (residual && e0 + q == dx) taken = p;
      }
      if ((some >> q) & 1u) r[q] = leaves(p, taken);
    }
  }
};

// A sum below 2^12 in units of 2^-40.
__device__ __forceinline__ uint64_t units(double sum) { return grid_units(sum + GRID); }

// Exclusive prefix over the block of one value per thread, and their sum.
template <typename U>
__device__ __forceinline__ U block_prefix(U v, U* scratch, U* total) {
  return block_excl_scan<U, VT>(v, scratch, total);
}

// A thread's run of consecutive 128-byte groups of a row, looked through by their keys: f(v, vector)
// for every vector, in index order, of the groups whose largest value may reach raw_lo.
template <typename T, typename F>
__device__ __forceinline__ void each_near(const GroupKeys& g, const RowView<T>& rv, int64_t row, float raw_lo, F&& f) {
  constexpr int GV = 8;  // vectors of a group (such rows start on a 16-byte boundary)
  const int32_t run = ((g.groups + VT - 1) / VT + 3) & ~3;
  const int32_t g0 = (int32_t)threadIdx.x * run, g1 = min(g.groups, g0 + run);
  const uint32_t lo = key_of(raw_lo);
  const uint32_t* keys = g.keys + row * g.stride;
  for (int32_t k0 = g0; k0 < g1; k0 += 16) {  // 16 keys at a time (a row's keys have room for whole fours)
    uint4 k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k[i] = make_uint4(0u, 0u, 0u, 0u);
      if (k0 + 4 * i < g1) k[i] = __ldcg(reinterpret_cast<const uint4*>(keys + k0 + 4 * i));
    }
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      hits |= (k[i].x >= lo ? 1u : 0u) << (4 * i);
      hits |= (k[i].y >= lo ? 1u : 0u) << (4 * i + 1);
      hits |= (k[i].z >= lo ? 1u : 0u) << (4 * i + 2);
      hits |= (k[i].w >= lo ? 1u : 0u) << (4 * i + 3);
    }
    const int32_t left = g1 - k0;
    if (left < 16) hits &= (1u << left) - 1u;  // (keys past the row's groups were never written)
    while (hits) {
      const int32_t v0 = (k0 + __ffs(hits) - 1) * GV;
      hits &= hits - 1;
      uint4 q[GV];
#pragma unroll
      for (int j = 0; j < GV; ++j) {
        const uint32_t none = Elem<T>::NEG_INF_WORD;
        q[j] = make_uint4(none, none, none, none);
        if (v0 + j < rv.nvec) q[j] = load_vec(rv, v0 + j);
      }
#pragma unroll
      for (int j = 0; j < GV; ++j)
        if (vec_max_nan<T>(q[j]) >= raw_lo) f(v0 + j, q[j]);
    }
  }
}

constexpr int NEAR_CAP = 256;   // listed elements of a row drawn from by one CTA
constexpr int NEAR_GROUPS = 512;  // ... and the groups they are looked for in
struct NearShared {
  uint64_t scan[VNW + 1];
  uint32_t tscan[VNW + 1];
  uint32_t n, groups;
  int32_t group[NEAR_GROUPS];
  int32_t index[NEAR_CAP], sorted[NEAR_CAP];
  float value[NEAR_CAP], sorted_value[NEAR_CAP];
  int32_t found;
  bool none;
};

// The values of a row at or above raw_lo (finite), by its group keys: the CTA lists the groups whose
// largest value is, then the values, in any order. Returns their number, or -1 where a list is too
// short for the row. (Few instructions, each run once: one CTA a sequence waits for code as for data.)
template <typename T>
__device__ int32_t list_near(const RowView<T>& rv, const GroupKeys& g, int64_t at_row, float raw_lo, NearShared& sh) {
  constexpr int EPV = Elem<T>::EPV;
  const int tid = threadIdx.x;
  if (tid == 0) sh.n = sh.groups = 0;
  __syncthreads();
  constexpr int GV = 8;  // vectors of a group (such rows start on a 16-byte boundary)
  const uint32_t lo = key_of(raw_lo);
  const uint32_t* keys = g.keys + at_row * g.stride;
  for (int32_t k0 = tid; k0 < g.groups; k0 += VT * 16) {
    uint32_t hits = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (k0 + i * VT < g.groups) hits |= (__ldcg(keys + k0 + i * VT) >= lo ? 1u : 0u) << i;
    while (hits) {
      const uint32_t at = atomicAdd(&sh.groups, 1u);
      if (at < (uint32_t)NEAR_GROUPS) sh.group[at] = k0 + (__ffs(hits) - 1) * VT;
      hits &= hits - 1;
    }
  }
  __syncthreads();
  const int32_t nv = (int32_t)min(sh.groups, (uint32_t)NEAR_GROUPS) * GV;
  if (sh.groups > (uint32_t)NEAR_GROUPS) return -1;
  constexpr int AHEAD = 4;  // vectors a thread has in flight
  for (int32_t i0 = tid; i0 < nv; i0 += VT * AHEAD) {
    uint4 q[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int32_t i = i0 + u * VT, v = i < nv ? sh.group[i / GV] * GV + i % GV : rv.nvec;
      const uint32_t none_word = Elem<T>::NEG_INF_WORD;
      q[u] = make_uint4(none_word, none_word, none_word, none_word);
      if (v < rv.nvec) q[u] = load_vec(rv, v);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (!(vec_max_nan<T>(q[u]) >= raw_lo)) continue;
      const int32_t i = i0 + u * VT, e0 = rv.first(sh.group[i / GV] * GV + i % GV);
#pragma unroll 1
      for (int j = 0; j < EPV; ++j) {
        const float x = Elem<T>::elem(q[u], j);
        if (!(x >= raw_lo)) continue;  // (elements past the row are -inf, and raw_lo is finite)
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < (uint32_t)NEAR_CAP) {
          sh.index[at] = e0 + j;
          sh.value[at] = x;
        }
      }
    }
  }
  __syncthreads();
  return sh.n <= (uint32_t)NEAR_CAP ? (int32_t)sh.n : -1;
}

// The draw over a row whose group keys are known, for rows with few values near the kept ones (as all
// but odd rows of top-k have): the listed values are put in index order by counting, then one warp
// weighs them, which needs no more barriers. Returns the token (every thread), -1 where there is no
// weight at all; false in *fits where the list is too short for the row.
template <typename T>
__device__ int32_t draw_listed(const DrawRow<T>& row, const GroupKeys& g, int64_t at_row, uint64_t u53, NearShared& sh,
                               bool* fits, bool* none) {
  constexpr int PER = NEAR_CAP / 32;
  const int tid = threadIdx.x;
  const int32_t n = list_near(row.rv, g, at_row, row.raw_lo, sh);
  *none = false;
  *fits = n >= 0;
  if (n < 0) return -1;
  if (tid < n) {
    const int32_t e = sh.index[tid];
    int32_t before = 0;
    for (int32_t j = 0; j < n; ++j) before += sh.index[j] < e ? 1 : 0;
    sh.sorted[before] = e;
    sh.sorted_value[before] = sh.value[tid];
  }
  __syncthreads();
  if (tid < 32) {
    // entries lane * per .. of the list: target weights, equals of the last kept key, what is left
    const int32_t per = (n + 31) / 32, i0 = tid * per;
    uint64_t p[PER], r[PER];
    float d[PER];
    uint32_t eq = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      p[j] = r[j] = 0;
      d[j] = 0.0f;
      if (j < per && i0 + j < n && row.dist) d[j] = prob_at(row.a, row.drow, sh.sorted[i0 + j]);
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j < per && i0 + j < n) {
        const float y = row.scaled(sh.sorted_value[i0 + j]);
        if (y >= row.thr) p[j] = weight_q(y, row.f.max_key);
        if (row.cut_ties && y == row.thr) eq |= 1u << j;
      }
    if (row.cut_ties) {
      const uint32_t mine = (uint32_t)__popc(eq);
      uint32_t before = warp_incl_scan(mine) - mine;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if ((eq >> j) & 1u) {
          if (before >= (uint32_t)row.f.n_tie_kept) p[j] = 0;
          ++before;
        }
    }
    uint64_t sum = 0, all = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (p[j]) {
        uint64_t taken = 0;
        // (NaN is 0 before the bound, which would take all of the weight in its place)
        if (row.dist) taken = grid_units(row.taken_by(fminf(fmaxf(d[j], 0.0f), row.d_most)));
        else if (row.residual && sh.sorted[i0 + j] == row.dx) taken = p[j];
        r[j] = p[j] > taken ? p[j] - taken : 0;
      }
      sum += r[j];
      all += p[j];
    }
    uint64_t incl = warp_incl_scan(sum), total = __shfl_sync(0xFFFFFFFFu, incl, 31);
    const bool target = total == 0;  // an empty residual: drawn from the target itself
    if (target) {
      sum = all;
      incl = warp_incl_scan(sum);
      total = __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
    if (tid == 0) {
      sh.found = -1;
      sh.none = total == 0;
    }
    __syncwarp();
    const uint64_t want = scale_u53(u53, total);
    uint64_t run = incl - sum;
    if (run <= want && want < incl) {
      int32_t found = -1;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        run += target ? p[j] : r[j];
        if (found < 0 && run > want) found = sh.sorted[i0 + j];
      }
      sh.found = found;
    }
  }
  __syncthreads();
  *none = sh.none;
  return sh.found;
}

// The same draw for rows of any number of such values (very many equal ones): the runs are looked
// through again for every sum.
template <typename T>
__device__ __noinline__ int32_t draw_near(const DrawRow<T>& row, const GroupKeys& g, int64_t at_row, uint64_t u53,
                                          NearShared& sh, bool* none) {
  constexpr int EPV = Elem<T>::EPV;
  uint32_t base = 0;  // equals of the last kept key before this thread's run
  if (row.cut_ties) {
    uint32_t n = 0, total;
    each_near<T>(g, row.rv, at_row, row.raw_lo, [&](int32_t v, uint4 q) {
      double r[EPV];
      uint32_t eq;
      row.of(v, q, true, false, nullptr, r, eq);
      n += (uint32_t)__popc(eq);
    });
    base = block_prefix(n, sh.tscan, &total);
  }
  const uint32_t keep = (uint32_t)row.f.n_tie_kept;
  // f(first element, weights) of this thread's vectors, equals that were cut without weight
  auto weights = [&](bool target, auto&& f) {
    uint32_t at = base;
    each_near<T>(g, row.rv, at_row, row.raw_lo, [&](int32_t v, uint4 q) {
      double r[EPV];
      uint32_t eq;
      row.of(v, q, target, false, nullptr, r, eq);
      if (eq) {
#pragma unroll
        for (int j = 0; j < EPV; ++j)
          if ((eq >> j) & 1u) {
            if (at >= keep) r[j] = 0.0;
            ++at;
          }
      }
      f(row.rv.first(v), r);
    });
  };
  bool target = false;
  uint64_t mine, total, before;
  while (true) {
    mine = 0;
    weights(target, [&](int32_t, const double* r) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) mine += units(r[j]);
    });
    before = block_prefix(mine, sh.scan, &total);
    if (total || target) break;
    target = true;  // an empty residual: drawn from the target itself
  }
  *none = total == 0;
  const uint64_t want = scale_u53(u53, total);
  int32_t found = -1;
  if (before <= want && want < before + mine) {
    uint64_t run = before;
    weights(target, [&](int32_t e0, const double* r) {
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        run += units(r[j]);
        if (found < 0 && run > want) found = e0 + j;
      }
    });
  }
  return found;
}

// A CTA per sequence: the first row that is not accepted, its accepted tokens, and for sequences whose
// rows' group keys are known the draw. Latency: 10 us for 256 sequences without draws here, 15 us for 64
// that draw from their top-k rows (the groups' list, their values, the weights: each waits for the one
// before). With the draws left to weigh_kernel and draw_kernel that call took 106 us instead of 65 us. REST: rows
// of kinds that are not named may occur. (One kernel for both took 1.4 us more.)
template <typename T, bool REST>
__global__ void __launch_bounds__(VT, 2) decide_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ struct {
    int32_t event;
    uint32_t cnt[1];
  } sh;
  __shared__ NearShared near_sh;
  grid_release();
  const int64_t seq = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t R = a.n_rows;
  const int64_t lo = min(max((int64_t)a.offsets[seq], (int64_t)0), R);
  const int64_t hi = min(max((int64_t)a.offsets[seq + 1], lo), R);
  const pb_row_params p = a.params[seq];
  const bool greedy = p.temperature == 0.0;
  const float tf = (float)p.temperature;
  const Scale scaled(tf);
  // what a draft's row needs of the inputs, loaded before the records are waited for (the first VT
  // drafts of a sequence; later ones, which hardly exist, load theirs when they are looked at)
  struct Draft {
    int64_t x;
    double u;
    float logit, prob;
  };
  auto draft_of = [&](int64_t r) -> Draft {
    Draft d{-1, 0.0, 0.0f, 1.0f};
    if (r >= hi) return d;
    d.u = a.uniforms[r];
    if (r == hi - 1) return d;
    d.x = a.drafts[r];
    if (greedy || d.x < 0 || d.x >= a.V) return d;
    d.logit = Elem<T>::ld(static_cast<const T*>(a.x) + r * a.row_stride + d.x);
    if (a.probs) {
      const int64_t at = r - seq;
      d.prob = (at >= 0 && at < a.n_probs) ? prob_at(a, at, d.x) : NAN;
    }
    return d;
  };
  const Draft first = draft_of(lo + tid);
  // whether a launch settles rows of this kind
  const int32_t row_is = settled_as<REST>(a, p);
  const bool settled = REST || (a.kinds & takes(row_is)) != 0;
  const double u_draw = lo < hi ? a.uniforms[hi - 1] : 0.0;
  grid_wait();  // the rows' records
  if (lo >= hi) {  // a sequence without rows
    if (tid == 0) {
      a.out_accepted[seq] = 0;
      if (a.out_status) a.out_status[seq] = PB_ROW_BAD_PARAMS;
      a.decision[seq] = Decision{0, EV_BAD, 0};
    }
    return;
  }

  // a row's record; that of a ROW_WHOLE row, without its mass, from its largest value (every key is above
  // thr_key)
  auto record = [&](int64_t r) -> pb_row_info {
    pb_row_info f = a.info[r];
    if (row_is == ROW_WHOLE && settled) {
      const uint32_t raw = a.meta[r].max_key, m = key_of(scaled(value_of(raw)));
      f.status = raw != 0xFFFFFFFFu && m < KEY_POS_INF && m > KEY_NEG_INF ? PB_ROW_OK : PB_ROW_NONFINITE;
      f.max_key = value_of(m);
      f.thr_key = 0;
      f.n_tie_kept = 0;
      f.z_q = f.kept_q = 0;  // (mass_kernel adds them)
    }
    return f;
  };

  // the first row that is not accepted
  int64_t from = lo, stop = hi - 1;
  int32_t kind = EV_LAST;
  while (true) {
    if (tid == 0) sh.event = 0x7FFFFFFF;
    __syncthreads();
    for (int64_t r = from + tid; r < hi; r += VT) {
      const pb_row_info f = record(r);
      const Draft d = r == lo + tid ? first : draft_of(r);
      int32_t ev = -1;
      if (!settled || f.status != PB_ROW_OK) {
        ev = EV_BAD;
      } else if (!greedy && !(d.u >= 0.0 && d.u < 1.0)) {
        ev = EV_BAD;
      } else if (r == hi - 1) {
        ev = EV_LAST;
      } else {
        bool ok = false;
        if (d.x >= 0 && d.x < a.V) {  // (a draft outside the vocabulary has no mass: rejected)
          if (greedy) {
            ok = d.x == a.tok[r];
          } else {
            const float y = scaled(d.logit);
            const uint32_t key = key_of(y);
            bool kept = key > f.thr_key;
            if (key == f.thr_key) {
              // equals of the last kept key: all of them, or (cut by top-p) those of lowest index
              if (f.kept_q == f.z_q) kept = true;
              else ev = EV_TIE;
            }
            const uint64_t px = (kept || ev == EV_TIE) ? weight_q(y, f.max_key) : 0;
            const double want = a.probs ? __dmul_rn(d.u, (double)d.prob) : d.u, p = __ull2double_rn(px);
            if (want < 0.0) {  // below any weight, be it 0
              ok = true;
              ev = -1;
            } else if (row_is == ROW_WHOLE) {
              // (what fp64's own roundings add is far below the bounds' slack)
              const Mass z = mass_near(a, r, tf, value_of(a.meta[r].max_key), f.max_key);
              ok = want * z.lo < p;
              if (ok && !(want * z.hi < p)) ev = EV_TIE;
            } else {
              ok = __dmul_rn(want, __ull2double_rn(f.kept_q)) < p;
              if (ev == EV_TIE && !ok) ev = EV_REJECT;  // rejected either way
            }
          }
        }
        if (ev < 0 && !ok) ev = EV_REJECT;
      }
      // the first event of the sequence: rows in the high bits, its kind below
      if (ev >= 0) atomicMin(&sh.event, (int32_t)((r - lo) << 2 | ev));
    }
    __syncthreads();
    const int32_t e = sh.event;
    __syncthreads();
    kind = e & 3;
    stop = lo + (e >> 2);
    if (kind != EV_TIE) break;
    if (row_is == ROW_WHOLE) {
      const float raw = value_of(a.meta[stop].max_key), m = scaled(raw);
      const RowView<T> row(static_cast<const T*>(a.x) + stop * a.row_stride, a.V);
      const uint64_t z = mass_of<T>(row, tf, m, raw, near_sh.scan);
      const Draft d = draft_of(stop);
      const double want = a.probs ? __dmul_rn(d.u, (double)d.prob) : d.u;
      if (!(__dmul_rn(want, __ull2double_rn(z)) < __ull2double_rn(weight_q(scaled(d.logit), m)))) {
        kind = EV_REJECT;
        break;
      }
      from = stop + 1;  // accepted
      continue;
    }
    // rank of the draft among the equals of the last kept key, in index order
    const pb_row_info f = a.info[stop];
    const int32_t x = (int32_t)a.drafts[stop];
    const RowView<T> rv(static_cast<const T*>(a.x) + stop * a.row_stride, a.V);
    if (tid == 0) sh.cnt[0] = 0;
    __syncthreads();
    uint32_t before = 0;
    const float lo_raw = surely_below(f.thr_key, tf);
    const bool keyed = a.groups.keys && row_is == ROW_SMALL;
    const int32_t near = keyed && lo_raw > -INFINITY ? list_near(rv, a.groups, stop, lo_raw, near_sh) : -1;
    if (near >= 0) {
      if (tid < near) before = near_sh.index[tid] < x && key_of(scaled(near_sh.value[tid])) == f.thr_key;
    } else if (keyed) {
      each_near<T>(a.groups, rv, stop, lo_raw, [&](int32_t v, uint4 q4) {
        float y[EPV];
        Elem<T>::unpack(q4, y);
#pragma unroll
        for (int q = 0; q < EPV; ++q)
          if (rv.first(v) + q < x && key_of(scaled(y[q])) == f.thr_key) ++before;
      });
    } else
    for (int32_t v0 = tid; v0 < rv.nvec && rv.first(v0) < x; v0 += VT * SEG_V) {
      uint4 q4[SEG_V];
#pragma unroll
      for (int u = 0; u < SEG_V; ++u) {
        const uint32_t none = Elem<T>::NEG_INF_WORD;
        q4[u] = make_uint4(none, none, none, none);
        if (v0 + u * VT < rv.nvec && rv.first(v0 + u * VT) < x) q4[u] = load_vec(rv, v0 + u * VT);
      }
#pragma unroll
      for (int u = 0; u < SEG_V; ++u) {
        if (!(vec_max_nan<T>(q4[u]) >= lo_raw)) continue;
        float y[EPV];
        Elem<T>::unpack(q4[u], y);
#pragma unroll
        for (int q = 0; q < EPV; ++q) {
          const int32_t i = rv.first(v0 + u * VT) + q;
          if (i >= 0 && i < x && key_of(scaled(y[q])) == f.thr_key) ++before;
        }
      }
    }
    before = __reduce_add_sync(0xFFFFFFFFu, before);
    if (lane == 0 && before) atomicAdd(&sh.cnt[0], before);
    __syncthreads();
    const bool kept = sh.cnt[0] < (uint32_t)f.n_tie_kept;
    __syncthreads();
    if (!kept) {
      kind = EV_REJECT;
      break;
    }
    from = stop + 1;  // accepted
  }
  if (kind == EV_REJECT && !greedy && !(u_draw >= 0.0 && u_draw < 1.0)) kind = EV_BAD;

  for (int64_t r = lo + tid; r < stop; r += VT) a.out_tokens[r] = a.drafts[r];
  if (tid == 0) {
    a.out_accepted[seq] = (int32_t)(stop - lo);
    const pb_row_info f = record(stop);
    if (row_is == ROW_WHOLE && settled) a.info[stop] = f;
    int32_t st = PB_ROW_OK;
    if (!settled) st = PB_ROW_INTERNAL;
    else if (kind == EV_BAD) st = f.status != PB_ROW_OK ? f.status : PB_ROW_BAD_UNIFORM;
    if (a.out_status) a.out_status[seq] = st;
    if (greedy && kind != EV_BAD) a.out_tokens[stop] = a.tok[stop];
  }
  // the last token: here, where the row's group keys are known, else by the launches that follow
  const bool draws = !greedy && kind != EV_BAD, here = a.groups.keys && row_is == ROW_SMALL;
  if (tid == 0) a.decision[seq] = Decision{stop, kind, draws && !here};
  if (draws && here) {
    const DrawRow<T> row(a, seq, Decision{stop, kind, 1}, tf, a.info[stop]);
    const uint64_t u53 = (uint64_t)(u_draw * 0x1p53);
    bool fits = false, none = false;
    int32_t found = -1;
    if (row.raw_lo > -INFINITY) found = draw_listed<T>(row, a.groups, stop, u53, near_sh, &fits, &none);
    if (!fits) found = draw_near<T>(row, a.groups, stop, u53, near_sh, &none);
    if (found >= 0 && (!fits || tid == 0)) a.out_tokens[stop] = found;
    if (none && tid == 0 && a.out_status) a.out_status[seq] = PB_ROW_INTERNAL;
  }
}

// ---- drawing ---------------------------------------------------------------------------------

// CTA (sequence, segment, share): the sums of a share of the segment's tiles. Every thread leaves its own
// sum of each tile in shared memory; the warps then take a tile each. 256 rows of 128256 bf16 with their
// fp32 draft probabilities (197 MB) in 53 us, 3.7 TB/s, bound by issue: 40 instructions a 32 elements (the
// weights, and a product and four sums of fp64).
template <typename T>
__global__ void __launch_bounds__(VT, 3) weigh_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  static_assert(TILES == VNW, "a warp per tile");
  __shared__ double part[TILES][VT], tie_part[TILES][VT];
  __shared__ uint8_t ties[TILES][VT];
  grid_release();
  grid_wait();
  const int64_t seq = blockIdx.x;
  const Decision d = a.decision[seq];
  if (!d.draws) return;
  const pb_row_info f = a.info[d.row];
  const DrawRow<T> row(a, seq, d, (float)a.params[seq].temperature, f);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t v0 = (int32_t)blockIdx.y * a.seg.per, v1 = min(row.rv.nvec, v0 + a.seg.per);
  const int32_t t0 = (int32_t)blockIdx.z * a.share, t1 = t0 + a.share;
  // one vector (and its draft probabilities) is on its way while the one before it is weighed
  const uint32_t none = Elem<T>::NEG_INF_WORD;
  const uint4 nothing = make_uint4(none, none, none, none);
  uint4 next = nothing;
  float4 next_d[EPV / 4];
  bool next_have = false;
  auto fetch = [&](int i) {
    const int32_t v = v0 + i * SEG_T + tid;
    next = nothing;
    next_have = false;
    if (i < t1 && v < v1) {
      next = load_vec(row.rv, v);
      next_have = row.packed_probs(v);
      if (next_have) row.load_probs(v, next_d);
    }
  };
  fetch(t0);
#pragma unroll 1
  for (int i = t0; i < t1; ++i) {
    const uint4 qi = next;
    float4 di[EPV / 4];
#pragma unroll
    for (int j = 0; j < EPV / 4; ++j) di[j] = next_d[j];
    const bool have = next_have;
    fetch(i + 1);
    double sum = 0.0, tsum = 0.0;
    uint32_t eq = 0;
    const int32_t at = v0 + i * SEG_T + tid, e0 = row.rv.first(at);
    const bool simple = at < v1 && row.whole && row.rv.whole(at);  // every element of the vector counts
    if (simple && have) {
      float w[EPV], y[EPV];
      row.weigh.template of<T>(qi, w, y);
#pragma unroll
      for (int j = 0; j < EPV; j += 4) {
        sum += row.leaves(on_grid(w[j]), row.taken_by(di[j / 4].x));
        sum += row.leaves(on_grid(w[j + 1]), row.taken_by(di[j / 4].y));
        sum += row.leaves(on_grid(w[j + 2]), row.taken_by(di[j / 4].z));
        sum += row.leaves(on_grid(w[j + 3]), row.taken_by(di[j / 4].w));
      }
    } else if (simple && !row.dist && !(row.dx >= e0 && row.dx < e0 + EPV)) {
      float w[EPV], y[EPV];
      row.weigh.template of<T>(qi, w, y);
      double s0 = GRID, s1 = GRID;
#pragma unroll
      for (int j = 0; j < EPV; j += 2) {
        s0 = __dadd_rd(s0, (double)w[j]);
        s1 = __dadd_rd(s1, (double)w[j + 1]);
      }
      sum = (s0 - GRID) + (s1 - GRID);
    } else if (at < v1) {
      double r[EPV];
      row.of(at, qi, false, have, di, r, eq);
#pragma unroll
      for (int j = 0; j < EPV; ++j) {
        if ((eq >> j) & 1u) tsum += r[j];
        else sum += r[j];
      }
    }
    part[i][tid] = sum;
    if (row.cut_ties) {
      tie_part[i][tid] = tsum;
      ties[i][tid] = (uint8_t)__popc(eq);
    }
  }
  __syncthreads();
  if (warp < t0 || warp >= t1) return;
  Tile t{0, 0, 0, 0};
  double sum = 0.0, tsum = 0.0;  // (64 weights of at most 1)
#pragma unroll
  for (int j = 0; j < VT / 32; ++j) {
    sum += part[warp][j * 32 + lane];
    if (row.cut_ties) {
      tsum += tie_part[warp][j * 32 + lane];
      t.ties += ties[warp][j * 32 + lane];
    }
  }
  t.w = warp_sum(units(sum));
  if (row.cut_ties) {
    t.tie_w = warp_sum(units(tsum));
    t.ties = __reduce_add_sync(0xFFFFFFFFu, t.ties);
  }
  if (lane == 0) a.tiles[(seq * a.seg.segs + blockIdx.y) * TILES + warp] = t;
}

struct DrawShared {
  uint64_t scan[VNW + 1];
  uint32_t tscan[VNW + 1];
  uint64_t left;     // the draw's number within its tile
  int32_t tile;      // the draw's tile
  uint32_t before;   // equals of the last kept key before it
  int32_t cut;       // the tile in which the kept equals end
  uint32_t cut_before;
};

// The draw: one CTA per sequence. Tiles are in index order, so are a tile's vectors over the threads. Only
// the draw's own tile is weighed again. Latency: 8 us for 256 sequences of 128256 tokens, 12 us where top-p
// cut between equals.
template <typename T>
__global__ void __launch_bounds__(VT, 2) draw_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ DrawShared sh;
  grid_wait();
  const int64_t seq = blockIdx.x;
  const Decision d = a.decision[seq];
  if (!d.draws) return;
  const int tid = threadIdx.x;
  const pb_row_info f = a.info[d.row];
  const DrawRow<T> row(a, seq, d, (float)a.params[seq].temperature, f);
  const int32_t nt = a.seg.segs * TILES;
  const Tile* tiles = a.tiles + seq * nt;
  const uint32_t keep = (uint32_t)f.n_tie_kept;
  const int64_t last = min((int64_t)a.offsets[seq + 1], a.n_rows) - 1;
  const uint64_t u53 = (uint64_t)(a.uniforms[last] * 0x1p53);

  // this thread's vector of tile k, its weights (those equals that were cut have none), and their sum;
  // `before`: equals before the tile
  auto tile_weights = [&](int32_t k, bool target, uint32_t before, double* r) -> uint64_t {
    const int32_t v0 = (k / TILES) * a.seg.per, v1 = min(row.rv.nvec, v0 + a.seg.per);
    const int32_t v = v0 + (k % TILES) * SEG_T + tid;
    uint32_t eq = 0;
#pragma unroll
    for (int q = 0; q < EPV; ++q) r[q] = 0.0;
    if (v < v1) row.of(v, load_vec(row.rv, v), target, false, nullptr, r, eq);
    if (row.cut_ties) {
      uint32_t total;
      uint32_t at = before + block_excl_scan<uint32_t, VT>((uint32_t)__popc(eq), sh.tscan, &total);
#pragma unroll
      for (int q = 0; q < EPV; ++q)
        if ((eq >> q) & 1u) {
          if (at >= keep) r[q] = 0.0;
          ++at;
        }
    }
    double s = 0.0;
#pragma unroll
    for (int q = 0; q < EPV; ++q) s += r[q];
    return units(s);
  };
  if (tid == 0) sh.tile = sh.cut = -1;
  __syncthreads();
  // a tile's weight comes from its record, but for the one in which the kept equals end: that is weighed again
  uint64_t cut_w = 0;
  if (row.cut_ties) {
    uint32_t base = 0;
    for (int32_t k0 = 0; k0 < nt; k0 += VT) {
      const uint32_t n = k0 + tid < nt ? (uint32_t)__ldcg(&tiles[k0 + tid].ties) : 0u;
      uint32_t total;
      const uint32_t at = base + block_excl_scan<uint32_t, VT>(n, sh.tscan, &total);
      if (at < keep && at + n > keep) {
        sh.cut = k0 + tid;
        sh.cut_before = at;
      }
      base += total;
    }
    __syncthreads();
    if (sh.cut >= 0) {
      double r[EPV];
      const uint64_t s = tile_weights(sh.cut, false, sh.cut_before, r);
      block_excl_scan<uint64_t, VT>(s, sh.scan, &cut_w);
    }
  }
  const int32_t cut = sh.cut;
  // over the tiles in order: the total, then the tile whose inclusive prefix first exceeds the target
  auto walk = [&](bool find, uint64_t target) -> uint64_t {
    uint64_t run = 0;
    uint32_t base = 0;
    for (int32_t k0 = 0; k0 < nt; k0 += VT) {
      const int32_t k = k0 + tid;
      uint64_t w = 0;
      uint32_t n = 0, before = 0, total_n = 0;
      Tile t{0, 0, 0, 0};
      if (k < nt) {
        t.w = __ldcg(&tiles[k].w);
        if (row.cut_ties) {
          t.tie_w = __ldcg(&tiles[k].tie_w);
          t.ties = __ldcg(&tiles[k].ties);
        }
      }
      if (row.cut_ties) {
        n = (uint32_t)t.ties;
        before = base + block_excl_scan<uint32_t, VT>(n, sh.tscan, &total_n);
        base += total_n;
      }
      w = (k == cut) ? cut_w : t.w + (before + n <= keep ? t.tie_w : 0ull);
      uint64_t total;
      const uint64_t at = run + block_excl_scan<uint64_t, VT>(w, sh.scan, &total);
      if (find && at <= target && target < at + w) {
        sh.tile = k;
        sh.left = target - at;
        sh.before = before;
      }
      run += total;
      if (find && target < run) break;
    }
    __syncthreads();
    return run;
  };
  uint64_t total = walk(false, 0);
  const bool target = total == 0;  // an empty residual: drawn from the target itself
  if (!target) {
    walk(true, scale_u53(u53, total));
  } else {
    // (rare: tile by tile, the target's weights anew)
    const uint64_t want = scale_u53(u53, f.kept_q);
    uint64_t run = 0;
    uint32_t before = 0;
    for (int32_t k = 0; k < nt; ++k) {
      double r[EPV];
      uint64_t w;
      block_excl_scan<uint64_t, VT>(tile_weights(k, true, before, r), sh.scan, &w);
      if (want < run + w) {
        if (tid == 0) {
          sh.tile = k;
          sh.left = want - run;
          sh.before = before;
        }
        break;
      }
      run += w;
      if (row.cut_ties) before += (uint32_t)__ldcg(&tiles[k].ties);
    }
    __syncthreads();
  }
  const int32_t tile = sh.tile;
  if (tile < 0) {  // no mass at all: the row's record and its weights disagree
    if (tid == 0 && a.out_status) a.out_status[seq] = PB_ROW_INTERNAL;
    return;
  }
  double r[EPV];
  const uint64_t s = tile_weights(tile, target, sh.before, r);
  uint64_t whole;
  uint64_t run = block_excl_scan<uint64_t, VT>(s, sh.scan, &whole);
  const uint64_t left = sh.left;
  if (run <= left && left < run + s) {
    const int32_t v0 = (tile / TILES) * a.seg.per, v = v0 + (tile % TILES) * SEG_T + tid;
    int32_t found = -1;
#pragma unroll
    for (int q = 0; q < EPV; ++q) {
      run += units(r[q]);
      if (found < 0 && run > left) found = row.rv.first(v) + q;
    }
    a.out_tokens[d.row] = found;
  }
}

constexpr int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

constexpr int64_t list_len(int64_t vocab) { return vocab < LIST ? vocab : LIST; }

struct VerifyPlan {
  int64_t rowp, rowq, info, tok, meta, decision, tiles, sums, hist, list, sampler, bytes;  // offsets in the workspace, its size
};
VerifyPlan verify_plan(int64_t n_rows, int64_t n_seqs, int64_t vocab, int dtype, int kinds) {
  const SegPlan seg = seg_plan(vocab, elem_size(dtype), nullptr, 1);  // (rows of any alignment: the most segments)
  VerifyPlan v;
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t from = at;
    at += up256(bytes);
    return from;
  };
  v.rowp = take(n_rows * (int64_t)sizeof(pb_row_params));
  v.rowq = take(n_rows * (int64_t)sizeof(pb_row_params));
  v.info = take(n_rows * (int64_t)sizeof(pb_row_info));
  v.tok = take(n_rows * 8);
  v.meta = take(n_rows * (int64_t)sizeof(RowMeta));
  v.decision = take(n_seqs * (int64_t)sizeof(Decision));
  v.tiles = take(n_seqs * seg.segs * TILES * (int64_t)sizeof(Tile));
  v.sums = take(kinds & PB_VERIFY_WHOLE ? n_rows * seg.segs * (int64_t)sizeof(ExpSum) : 0);
  v.hist = take(kinds & PB_VERIFY_TOPP ? n_rows * STEPS * 8 : 0);
  v.list = take(kinds & PB_VERIFY_TOPP ? n_rows * list_len(vocab) * 8 : 0);
  v.sampler = at;
  v.bytes = at + (kinds & PB_VERIFY_SMALL ? pb_sample_ws_bytes(n_rows, vocab, dtype) : 0);
  return v;
}

template <typename T>
int verify_run(VerifyArgs a, int dtype, int named, uint8_t* ws, const VerifyPlan& plan, cudaStream_t st) {
  const int kinds = named & PB_VERIFY_ANY;
  a.rowp = reinterpret_cast<pb_row_params*>(ws + plan.rowp);
  a.rowq = reinterpret_cast<pb_row_params*>(ws + plan.rowq);
  a.info = reinterpret_cast<pb_row_info*>(ws + plan.info);
  a.tok = reinterpret_cast<int64_t*>(ws + plan.tok);
  a.meta = reinterpret_cast<RowMeta*>(ws + plan.meta);
  a.decision = reinterpret_cast<Decision*>(ws + plan.decision);
  a.tiles = reinterpret_cast<Tile*>(ws + plan.tiles);
  if (kinds & PB_VERIFY_WHOLE) a.sums = reinterpret_cast<ExpSum*>(ws + plan.sums);
  if (kinds & PB_VERIFY_TOPP) {
    a.hist = reinterpret_cast<uint64_t*>(ws + plan.hist);
    a.list = reinterpret_cast<uint64_t*>(ws + plan.list);
    a.list_len = (int32_t)list_len(a.V);
  }
  a.seg = seg_plan(a.V, sizeof(T), a.x, a.row_stride);
  a.kinds = kinds;
  // rows of kinds that are not named: by the cluster kernel where it is launched, else by the sampler's launches
  // (which settle any row) where they are
  const bool general = (kinds & (PB_VERIFY_TOPP | PB_VERIFY_OTHER)) != 0;
  a.rest = !(named & PB_VERIFY_REST) ? -1 : !general && (kinds & PB_VERIFY_SMALL) ? ROW_SMALL : ROW_OTHER;
  a.one_kind = kinds == PB_VERIFY_WHOLE ? ROW_WHOLE : kinds == PB_VERIFY_TOPP ? ROW_MASS : -1;
  const dim3 rows((unsigned)a.n_rows, (unsigned)a.seg.segs), each_row((unsigned)a.n_rows);
  const dim3 seqs((unsigned)a.n_seqs), parts((unsigned)a.n_seqs, (unsigned)a.seg.segs);
  auto fallback = [&] { return sample_fallback_rows(a.x, dtype, a.n_rows, a.V, a.row_stride, a.rowq, a.tok, a.info, st); };
  expand_kernel<<<(unsigned)((a.n_rows + 255) / 256), 256, 0, st>>>(a);
  int rc = cudaGetLastError() == cudaSuccess ? PB_OK : PB_E_LAUNCH;
  if (rc == PB_OK && (kinds & PB_VERIFY_SMALL)) {
    // the two-pass launch where the rows suit it, else pb_sample's own launches (the workspace's other
    // launch cuts rows into pieces for large batches: 72 rows of 50021 fp16 take it 31 us, these 27 us)
    a.groups = sample_ws_keys(a.x, dtype, a.n_rows, a.V, a.row_stride, ws + plan.sampler, plan.bytes - plan.sampler);
    if (!a.groups.keys)
      rc = pb_sample(a.x, dtype, a.n_rows, a.V, a.row_stride, nullptr, a.rowp, a.tok, a.info, nullptr, st);
    else if (a.rest == ROW_SMALL)  // (rows of any kind, perhaps none that pb_sample_ws's launches wait for)
      rc = sample_ws_in_turn(a.x, dtype, a.n_rows, a.V, a.row_stride, a.rowp, a.tok, a.info, ws + plan.sampler, st);
    else
      rc = pb_sample_ws(a.x, dtype, a.n_rows, a.V, a.row_stride, nullptr, a.rowp, a.tok, a.info, nullptr, ws + plan.sampler,
                        plan.bytes - plan.sampler, st);
  }
  // (before the pass over whole rows, which the launches after it overlap with)
  if (rc == PB_OK && a.rest == ROW_OTHER && !general) rc = fallback();
  if (rc == PB_OK && (kinds & (PB_VERIFY_WHOLE | PB_VERIFY_TOPP))) rc = launch_after(max_kernel<T>, a, rows, VT, st);
  if (rc == PB_OK && (kinds & PB_VERIFY_TOPP)) {
    rc = launch_after(hist_kernel<T>, a, rows, VT, st);
    if (rc == PB_OK) rc = launch_after(cut_kernel, a, each_row, VT, st);
    if (rc == PB_OK) rc = launch_after(gather_kernel<T>, a, rows, VT, st);
  }
  if (rc == PB_OK && general) {
    rc = launch_after(order_kernel, a, each_row, VT, st);
    if (rc == PB_OK) rc = fallback();
  }
  if (rc == PB_OK) rc = launch_after(a.rest >= 0 ? decide_kernel<T, true> : decide_kernel<T, false>, a, seqs, VT, st);
  // (a batch whose every sequence draws in decide_kernel needs no more)
  if (rc != PB_OK || (kinds == PB_VERIFY_SMALL && a.groups.keys)) return rc;
  if (kinds & PB_VERIFY_WHOLE) rc = launch_after(mass_kernel<T>, a, parts, VT, st);
  // few sequences: a segment's tiles shared between more CTAs, as long as all of them run at once (64
  // sequences of 49152 bf16 with draft probabilities: 14.6 us against 18 us unshared, 16 mixed ones of
  // fp16: 6.3 us against 12.9 us)
  a.share = TILES;
  while (a.share > 1 && 2 * a.n_seqs * a.seg.segs * (TILES / a.share) <= WEIGH_CTAS) a.share /= 2;
  if (rc == PB_OK) rc = launch_after(weigh_kernel<T>, a, dim3(parts.x, parts.y, TILES / a.share), VT, st);
  if (rc == PB_OK) rc = launch_after(draw_kernel<T>, a, seqs, VT, st);
  return rc;
}

// 0, or some kinds with or without PB_VERIFY_REST.
bool kinds_ok(int kinds) { return kinds == 0 || (kinds > 0 && kinds <= (PB_VERIFY_ANY | PB_VERIFY_REST) && (kinds & PB_VERIFY_ANY)); }

}  // namespace

extern "C" {

int64_t pb_verify_ws_bytes(int64_t n_rows, int64_t n_seqs, int64_t vocab, int dtype, int kinds) {
  if (n_rows < 0 || n_seqs < 0 || vocab <= 0 || !elem_size(dtype) || !kinds_ok(kinds)) return PB_E_INVALID;
  return verify_plan(n_rows, n_seqs, vocab, dtype, kinds ? kinds : PB_VERIFY_ANY).bytes;
}

int pb_verify(const void* logits, int dtype, int64_t n_rows, int64_t vocab, int64_t row_stride,
              const pb_row_params* params, int64_t n_seqs, const int32_t* row_offsets, const int64_t* drafts,
              const double* uniforms, const void* draft_probs, int probs_dtype, int64_t n_probs, int64_t probs_stride,
              int kinds, int64_t* out_tokens, int32_t* out_accepted, int32_t* out_status, void* workspace,
              int64_t ws_bytes, void* stream) {
  const int es = elem_size(dtype);
  if (n_rows < 0 || n_seqs < 0 || n_probs < 0 || vocab <= 0 || row_stride < vocab || !es) return PB_E_INVALID;
  if (vocab >= PB_MAX_VOCAB) return PB_E_TOO_LARGE;
  if (n_rows == 0 && n_seqs == 0) return PB_OK;
  if (n_rows == 0 || n_seqs == 0) return PB_E_INVALID;
  if (!logits || !params || !row_offsets || !drafts || !uniforms || !out_tokens || !out_accepted || !workspace)
    return PB_E_INVALID;
  if (n_rows > (1 << 28) || n_seqs > n_rows) return PB_E_INVALID;
  if (!aligned(logits, es) || !aligned(params, 8) || !aligned(row_offsets, 4) || !aligned(drafts, 8) ||
      !aligned(uniforms, 8) || !aligned(out_tokens, 8) || !aligned(out_accepted, 4) || !aligned(out_status, 4))
    return PB_E_INVALID;
  if (draft_probs) {
    const int ps = elem_size(probs_dtype);
    if (!ps || probs_stride < vocab || !aligned(draft_probs, ps)) return PB_E_INVALID;
  }
  if (!kinds_ok(kinds)) return PB_E_INVALID;
  const int k = kinds ? kinds : PB_VERIFY_ANY;
  const VerifyPlan plan = verify_plan(n_rows, n_seqs, vocab, dtype, k);
  if (!aligned(workspace, 256) || ws_bytes < plan.bytes) return PB_E_INVALID;
  VerifyArgs a = {};
  a.x = logits;
  a.row_stride = row_stride;
  a.n_rows = n_rows;
  a.n_seqs = n_seqs;
  a.V = (int32_t)vocab;
  a.params = params;
  a.offsets = row_offsets;
  a.drafts = drafts;
  a.uniforms = uniforms;
  a.probs = draft_probs;
  a.probs_dtype = probs_dtype;
  a.probs_stride = probs_stride;
  a.n_probs = n_probs;
  a.out_tokens = out_tokens;
  a.out_accepted = out_accepted;
  a.out_status = out_status;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return verify_run<float>(a, dtype, k, ws, plan, st);
  if (dtype == PB_DTYPE_BF16) return verify_run<__nv_bfloat16>(a, dtype, k, ws, plan, st);
  return verify_run<__half>(a, dtype, k, ws, plan, st);
}

}  // extern "C"
