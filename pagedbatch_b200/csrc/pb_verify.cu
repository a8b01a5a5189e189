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
//   1. expand: each row's parameters from its sequence's.
//   2. the sampler over the rows (its info record describes the kept set and its mass); rows without
//      top-k and top-p, whose kept set is the whole row, are summed by mass_kernel instead.
//   3. pick: one cluster per sequence finds the first rejected row and draws the last token from it.
#include "pb_rows.cuh"

using namespace pb;

namespace {

constexpr int VT = 512;          // threads per CTA
constexpr int VNW = VT / 32;
constexpr int VSTEPS = 64;       // parts of a warp's share of a row whose sums are kept for the draw

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
  int32_t sampler_runs, mass_runs;
  pb_row_params* rowp;           // workspace: [n_rows]
  pb_row_info* info;             // workspace: [n_rows]
  int64_t* tok;                  // workspace: [n_rows], the sampler's tokens (greedy rows' maxima)
  int64_t* out_tokens;           // [n_rows]
  int32_t* out_accepted;         // [n_seqs]
  int32_t* out_status;           // [n_seqs] or null
};

// Rows whose kept set is the whole row: valid parameters, no greedy, no top-k, no top-p.
__device__ __forceinline__ bool whole_row(const pb_row_params& p, int32_t V) {
  const bool ok = p.temperature > 0.0 && p.top_p > 0.0 && p.top_p <= 1.0 && p.top_k >= 0;
  return ok && !(p.top_k > 0 && p.top_k < V) && !((float)p.top_p < 1.0f);
}

__global__ void __launch_bounds__(256) expand_kernel(VerifyArgs a) {
  const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (r >= a.n_rows) return;
  int64_t lo = 0, hi = a.n_seqs;  // the last sequence that starts at or before row r
  while (hi - lo > 1) {
    const int64_t mid = lo + ((hi - lo) >> 1);
    if ((int64_t)a.offsets[mid] <= r) lo = mid;
    else hi = mid;
  }
  pb_row_params p = a.params[lo];
  p.uniform = 0.0;  // the sampler's own draw is not used
  p.rng = 0;
  // mass_kernel sums these; the sampler passes over them as greedy rows, its cheapest kind
  if (a.mass_runs && a.sampler_runs && whole_row(p, a.V)) p.temperature = 0.0;
  a.rowp[r] = p;
  a.info[r].status = PB_ROW_INTERNAL;  // until a launch settles the row
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

struct MassShared {
  uint32_t top[VNW];
  uint64_t sum[VNW];
  uint32_t pub_max;
  uint64_t pub_sum;
};

// Mass of a whole row: the largest scaled key, then the sum of the fixed-point weights. One cluster
// per row; the second pass reads its slice from L2.
template <typename T>
__global__ void __launch_bounds__(VT, 2) mass_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ MassShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / C;
  const int tid = threadIdx.x;
  int64_t lo = 0, hi = a.n_seqs;
  while (hi - lo > 1) {
    const int64_t mid = lo + ((hi - lo) >> 1);
    if ((int64_t)a.offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  const pb_row_params p = a.params[lo];
  if (!whole_row(p, a.V)) return;  // the whole cluster leaves
  const Scale scaled((float)p.temperature);
  const RowView<T> rv(static_cast<const T*>(a.x) + row * a.row_stride, a.V);
  const int32_t v0 = (int32_t)((int64_t)rv.nvec * rank / C), v1 = (int32_t)((int64_t)rv.nvec * (rank + 1) / C);
  uint32_t mk = 0;
  for (int32_t v = v0 + tid; v < v1; v += VT) mk = max(mk, key_of(vec_max_nan<T>(load_vec(rv, v))));
  mk = __reduce_max_sync(0xFFFFFFFFu, mk);
  if ((tid & 31) == 0) sh.top[tid >> 5] = mk;
  __syncthreads();
  mk = 0;
  for (int w = 0; w < VNW; ++w) mk = max(mk, sh.top[w]);
  if (C > 1) {
    if (tid == 0) sh.pub_max = mk;
    cluster.sync();
    for (int r = 0; r < C; ++r) mk = max(mk, cluster.map_shared_rank(&sh, r)->pub_max);
  }
  const float m = scaled(value_of(mk));
  const uint32_t sk = key_of(m);
  const bool ok = mk != 0xFFFFFFFFu && sk < KEY_POS_INF && sk > KEY_NEG_INF;
  uint64_t z = 0;
  if (ok) {
    for (int32_t v = v0 + tid; v < v1; v += VT) {
      float x[EPV];
      Elem<T>::unpack(load_vec(rv, v), x);
#pragma unroll
      for (int q = 0; q < EPV; ++q) z += weight_q(scaled(x[q]), m);  // elements outside the row are -inf: 0
    }
  }
  z = warp_sum(z);
  if ((tid & 31) == 0) sh.sum[tid >> 5] = z;
  __syncthreads();
  z = 0;
  for (int w = 0; w < VNW; ++w) z += sh.sum[w];
  if (C > 1) {
    if (tid == 0) sh.pub_sum = z;
    cluster.sync();
    if (rank == 0 && tid == 0)
      for (int r = 1; r < C; ++r) z += cluster.map_shared_rank(&sh, r)->pub_sum;
  }
  if (rank == 0 && tid == 0) {
    pb_row_info* o = a.info + row;
    o->thr_key = 0;  // every key is above it
    o->n_tie_kept = 0;
    o->kept_count = a.V;
    o->status = ok ? PB_ROW_OK : PB_ROW_NONFINITE;
    o->max_key = m;
    o->flags = PB_PATH_LARGE;
    o->z_q = z;
    o->kept_q = z;
  }
  if (C > 1) cluster.sync();
}

// ---- pick ----------------------------------------------------------------------------------------

struct PickShared {
  uint64_t res[VNW][VSTEPS], all[VNW][VSTEPS];  // sums of a warp's parts: residual, target
  uint64_t wres[VNW], wall[VNW];
  uint32_t wtie[VNW];
  uint32_t ctie;
  int32_t event, kind;
  // rank 0's decision
  int32_t owner, use_all;  // cluster-wide warp that holds the draw, which sums it goes by
  uint64_t left;           // the draw's target inside that warp
  uint32_t cnt[2];
};

enum : int32_t { EV_REJECT = 0, EV_BAD = 1, EV_TIE = 2, EV_LAST = 3 };

__device__ __forceinline__ float prob_at(const VerifyArgs& a, int64_t d, int64_t i) {
  const int64_t at = d * a.probs_stride + i;
  if (a.probs_dtype == PB_DTYPE_F32) return __ldg(static_cast<const float*>(a.probs) + at);
  if (a.probs_dtype == PB_DTYPE_BF16) return Elem<__nv_bfloat16>::ld(static_cast<const __nv_bfloat16*>(a.probs) + at);
  return Elem<__half>::ld(static_cast<const __half*>(a.probs) + at);
}

// What the draft's distribution takes of a target weight of mass scale zd: floor(d * Z), 0 for d <= 0
// or NaN (fp64: d has at most 24 bits and Z is rounded to 53, one rounding of the product).
__device__ __forceinline__ uint64_t taken_of(float d, double zd) {
  if (!(d > 0.0f)) return 0;
  const double t = __dmul_rn((double)d, zd);
  return (t >= 0x1p63) ? ~0ull : (uint64_t)t;
}

template <typename T>
__global__ void __launch_bounds__(VT, 2) pick_kernel(VerifyArgs a) {
  constexpr int EPV = Elem<T>::EPV;
  __shared__ PickShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t seq = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t R = a.n_rows;
  const int64_t lo = min(max((int64_t)a.offsets[seq], (int64_t)0), R);
  const int64_t hi = min(max((int64_t)a.offsets[seq + 1], lo), R);
  if (lo >= hi) {  // a sequence without rows (the whole cluster leaves)
    if (rank == 0 && tid == 0) {
      a.out_accepted[seq] = 0;
      if (a.out_status) a.out_status[seq] = PB_ROW_BAD_PARAMS;
    }
    return;
  }
  const pb_row_params p = a.params[seq];
  const bool greedy = p.temperature == 0.0;
  const float tf = (float)p.temperature;
  const Scale scaled(tf);

  // Every CTA of the cluster finds the first row that is not accepted, by the same steps.
  int64_t from = lo, stop = hi - 1;
  int32_t kind = EV_LAST;
  while (true) {
    if (tid == 0) {
      sh.event = 0x7FFFFFFF;
      sh.kind = EV_LAST;
    }
    __syncthreads();
    for (int64_t r = from + tid; r < hi; r += VT) {
      const pb_row_info f = a.info[r];
      int32_t ev = -1;
      if (f.status != PB_ROW_OK) {
        ev = EV_BAD;
      } else if (!greedy && !(a.uniforms[r] >= 0.0 && a.uniforms[r] < 1.0)) {
        ev = EV_BAD;
      } else if (r == hi - 1) {
        ev = EV_LAST;
      } else {
        const int64_t x = a.drafts[r];
        bool ok = false;
        if (x >= 0 && x < a.V) {  // (a draft outside the vocabulary has no mass: rejected)
          if (greedy) {
            ok = x == a.tok[r];
          } else {
            const float y = scaled(Elem<T>::ld(static_cast<const T*>(a.x) + r * a.row_stride + x));
            const uint32_t key = key_of(y);
            bool kept = key > f.thr_key;
            if (key == f.thr_key) {
              // equals of the last kept key: all of them, or (cut by top-p) those of lowest index
              if (f.kept_q == f.z_q) kept = true;
              else ev = EV_TIE;
            }
            const uint64_t px = (kept || ev == EV_TIE) ? weight_q(y, f.max_key) : 0;
            double want = a.uniforms[r];
            if (a.probs) {
              const int64_t d = r - seq;
              want = (d >= 0 && d < a.n_probs) ? __dmul_rn(want, (double)prob_at(a, d, x)) : NAN;
            }
            ok = __dmul_rn(want, __ull2double_rn(f.kept_q)) < __ull2double_rn(px);
            if (ev == EV_TIE && !ok) ev = EV_REJECT;  // rejected either way
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
    // rank of the draft among the equals of the last kept key, in index order
    const pb_row_info f = a.info[stop];
    const int32_t x = (int32_t)a.drafts[stop];
    const RowView<T> rv(static_cast<const T*>(a.x) + stop * a.row_stride, a.V);
    if (tid == 0) sh.cnt[0] = 0;
    __syncthreads();
    uint32_t before = 0;
    for (int32_t v = tid; v < rv.nvec && rv.first(v) < x; v += VT) {
      float y[EPV];
      Elem<T>::unpack(load_vec(rv, v), y);
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        const int32_t i = rv.first(v) + q;
        if (i >= 0 && i < x && key_of(scaled(y[q])) == f.thr_key) ++before;
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
  const double u_draw = a.uniforms[hi - 1];
  if (kind == EV_REJECT && !greedy && !(u_draw >= 0.0 && u_draw < 1.0)) kind = EV_BAD;

  if (rank == 0) {
    for (int64_t r = lo + tid; r < stop; r += VT) a.out_tokens[r] = a.drafts[r];
    if (tid == 0) {
      a.out_accepted[seq] = (int32_t)(stop - lo);
      int32_t st = PB_ROW_OK;
      if (kind == EV_BAD) st = a.info[stop].status != PB_ROW_OK ? a.info[stop].status : PB_ROW_BAD_UNIFORM;
      if (a.out_status) a.out_status[seq] = st;
      if (greedy && kind != EV_BAD) a.out_tokens[stop] = a.tok[stop];
    }
  }
  if (greedy || kind == EV_BAD) return;

  // ---- the last token: a draw over row `stop` in index order ----
  const pb_row_info f = a.info[stop];
  const float m = f.max_key;
  const uint32_t thr = f.thr_key;
  const double zd = __ull2double_rn(f.kept_q);
  const bool residual = kind == EV_REJECT;
  const int64_t dx = residual ? a.drafts[stop] : -1;
  const int64_t drow = stop - seq;
  const bool dist = residual && a.probs && drow >= 0 && drow < a.n_probs;
  const bool cut_ties = f.kept_q != f.z_q;
  // raw values below this are surely below the last kept key (two roundings of the quotient apart)
  float raw_lo = -INFINITY;
  if (thr > KEY_NEG_INF && thr < KEY_POS_INF) {
    const float b = value_of(thr) * tf;
    raw_lo = b - fabsf(b) * 0x1p-20f - 0x1p-100f;
    if (!(raw_lo > -INFINITY)) raw_lo = -INFINITY;
  }
  const RowView<T> rv(static_cast<const T*>(a.x) + stop * a.row_stride, a.V);
  const int gw = rank * VNW + warp, GW = C * VNW;
  const int32_t v0 = (int32_t)((int64_t)rv.nvec * gw / GW), v1 = (int32_t)((int64_t)rv.nvec * (gw + 1) / GW);
  // the warp's share in parts of `step` vectors (a multiple of 32), at most VSTEPS of them
  const int32_t step = (((v1 - v0) + VSTEPS - 1) / VSTEPS + 31) & ~31;

  // equals of the last kept key before this warp's share, where top-p cut among them
  uint32_t tie_base = 0;
  if (cut_ties) {
    uint32_t c = 0;
    for (int32_t v = v0 + lane; v < v1; v += 32) {
      const uint4 q4 = load_vec(rv, v);
      if (!(vec_max_nan<T>(q4) >= raw_lo)) continue;
      float y[EPV];
      Elem<T>::unpack(q4, y);
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        const int32_t i = rv.first(v) + q;
        if (i >= 0 && i < a.V && key_of(scaled(y[q])) == thr) ++c;
      }
    }
    c = __reduce_add_sync(0xFFFFFFFFu, c);
    if (lane == 0) sh.wtie[warp] = c;
    __syncthreads();
    if (tid == 0) {
      uint32_t s = 0;
      for (int w = 0; w < VNW; ++w) s += sh.wtie[w];
      sh.ctie = s;
    }
    cluster_barrier(C);
    for (int r = 0; r < rank; ++r) tie_base += cluster.map_shared_rank(&sh, r)->ctie;
    for (int w = 0; w < warp; ++w) tie_base += sh.wtie[w];
  }

  // the weights of vector v (all lanes of the warp call together, lanes side by side): target and
  // residual; `ties` counts the equals before it
  auto weigh = [&](int32_t v, bool in, uint32_t& ties, uint64_t* P, uint64_t* r) {
#pragma unroll
    for (int q = 0; q < EPV; ++q) P[q] = r[q] = 0;
    uint4 q4 = make_uint4(0u, 0u, 0u, 0u);
    if (in) {
      q4 = load_vec(rv, v);
      in = vec_max_nan<T>(q4) >= raw_lo;
    }
    uint32_t eq = 0;  // a bit per element equal to the last kept key
    float y[EPV];
    if (in) {
      Elem<T>::unpack(q4, y);
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        const int32_t i = rv.first(v) + q;
        y[q] = scaled(y[q]);
        const uint32_t key = key_of(y[q]);
        if (i >= 0 && i < a.V) {
          if (key >= thr) P[q] = weight_q(y[q], m);
          if (key == thr) eq |= 1u << q;
        }
      }
    }
    if (cut_ties && __any_sync(0xFFFFFFFFu, eq != 0)) {
      const uint32_t mine = (uint32_t)__popc(eq), incl = warp_incl_scan(mine);
      uint32_t at = ties + incl - mine;
#pragma unroll
      for (int q = 0; q < EPV; ++q)
        if ((eq >> q) & 1u) {
          if (at >= (uint32_t)f.n_tie_kept) P[q] = 0;
          ++at;
        }
      ties += __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
    if (in) {
#pragma unroll
      for (int q = 0; q < EPV; ++q) {
        const int64_t i = rv.first(v) + q;
        if (P[q]) {
          uint64_t t = 0;
          if (dist) t = taken_of(prob_at(a, drow, i), zd);
          else if (residual && i == dx) t = P[q];
          r[q] = (P[q] > t) ? P[q] - t : 0;
        }
      }
    }
  };

  uint64_t sum_r = 0, sum_p = 0;
  uint32_t ties = tie_base;
  for (int s = 0; s < VSTEPS; ++s) {
    uint64_t sr = 0, sp = 0;
    const int32_t vs = v0 + s * step;
    if (vs < v1) {
      for (int32_t vb = vs; vb < min(vs + step, v1); vb += 32) {
        uint64_t P[EPV], r[EPV];
        weigh(vb + lane, vb + lane < v1, ties, P, r);
#pragma unroll
        for (int q = 0; q < EPV; ++q) {
          sp += P[q];
          sr += r[q];
        }
      }
      sr = warp_sum(sr);
      sp = warp_sum(sp);
    }
    if (lane == 0) {
      sh.res[warp][s] = sr;
      sh.all[warp][s] = sp;
    }
    sum_r += sr;
    sum_p += sp;
  }
  if (lane == 0) {
    sh.wres[warp] = sum_r;
    sh.wall[warp] = sum_p;
  }
  cluster_barrier(C);
  if (rank == 0 && tid == 0) {
    uint64_t tr = 0, tp = 0;
    for (int r = 0; r < C; ++r) {
      const PickShared* o = C > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
      for (int w = 0; w < VNW; ++w) {
        tr += o->wres[w];
        tp += o->wall[w];
      }
    }
    const int use_all = tr == 0;
    uint64_t t = scale_u53((uint64_t)(u_draw * 0x1p53), use_all ? tp : tr);
    int owner = -1;
    for (int r = 0; r < C && owner < 0; ++r) {
      const PickShared* o = C > 1 ? cluster.map_shared_rank(&sh, r) : &sh;
      for (int w = 0; w < VNW; ++w) {
        const uint64_t c = use_all ? o->wall[w] : o->wres[w];
        if (t < c) {
          owner = r * VNW + w;
          break;
        }
        t -= c;
      }
    }
    sh.owner = owner;
    sh.use_all = use_all;
    sh.left = t;
    if (owner < 0) {  // no mass at all: the row's record and its weights disagree
      if (a.out_status) a.out_status[seq] = PB_ROW_INTERNAL;
    }
  }
  cluster_barrier(C);
  const PickShared* d0 = C > 1 ? cluster.map_shared_rank(&sh, 0) : &sh;
  const int owner = d0->owner;
  const bool use_all = d0->use_all != 0;
  uint64_t left = d0->left;
  if (owner == gw) {
    int s = 0;
    for (; s < VSTEPS; ++s) {
      const uint64_t c = use_all ? sh.all[warp][s] : sh.res[warp][s];
      if (left < c) break;
      left -= c;
    }
    // equals of the last kept key in the parts before
    uint32_t before = tie_base;
    if (cut_ties) {
      uint32_t c = 0;
      for (int32_t v = v0 + lane; v < min(v0 + s * step, v1); v += 32) {
        float y[EPV];
        Elem<T>::unpack(load_vec(rv, v), y);
#pragma unroll
        for (int q = 0; q < EPV; ++q) {
          const int32_t i = rv.first(v) + q;
          if (i >= 0 && i < a.V && key_of(scaled(y[q])) == thr) ++c;
        }
      }
      before += __reduce_add_sync(0xFFFFFFFFu, c);
    }
    int64_t found = -1;
    for (int32_t vb = v0 + s * step; vb < v1; vb += 32) {
      uint64_t P[EPV], r[EPV], c = 0;
      weigh(vb + lane, vb + lane < v1, before, P, r);
#pragma unroll
      for (int q = 0; q < EPV; ++q) c += use_all ? P[q] : r[q];
      const uint64_t incl = warp_incl_scan(c), total = __shfl_sync(0xFFFFFFFFu, incl, 31);
      const uint32_t hit = __ballot_sync(0xFFFFFFFFu, incl > left);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          uint64_t run = incl - c;
#pragma unroll
          for (int q = 0; q < EPV; ++q) {
            run += use_all ? P[q] : r[q];
            if (found < 0 && run > left) found = rv.first(vb + lane) + q;
          }
          a.out_tokens[stop] = found;
        }
        break;
      }
      left -= total;
    }
  }
  if (C > 1) cluster.sync();  // rank 0's decision stays until every CTA has read it
}

int verify_cluster(int64_t n, int64_t bytes) {
  const int64_t want = 2 * (int64_t)device_sms();
  int C = 1;
  while (C < 8 && n * C < want && bytes / (2 * C) >= 8192) C <<= 1;
  return C;
}

constexpr int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }

struct VerifyPlan {
  int64_t rowp, info, tok, sampler, bytes;  // offsets in the workspace, and its size
};
VerifyPlan verify_plan(int64_t n_rows, int64_t vocab, int dtype) {
  VerifyPlan v;
  v.rowp = 0;
  v.info = up256(n_rows * (int64_t)sizeof(pb_row_params));
  v.tok = v.info + up256(n_rows * (int64_t)sizeof(pb_row_info));
  v.sampler = v.tok + up256(n_rows * 8);
  v.bytes = v.sampler + pb_sample_ws_bytes(n_rows, vocab, dtype);
  return v;
}

template <typename T>
int verify_run(VerifyArgs a, int dtype, int kinds, uint8_t* ws, const VerifyPlan& plan, cudaStream_t st) {
  a.rowp = reinterpret_cast<pb_row_params*>(ws + plan.rowp);
  a.info = reinterpret_cast<pb_row_info*>(ws + plan.info);
  a.tok = reinterpret_cast<int64_t*>(ws + plan.tok);
  a.sampler_runs = (kinds & (PB_VERIFY_SMALL | PB_VERIFY_OTHER)) != 0;
  a.mass_runs = (kinds & PB_VERIFY_WHOLE) != 0;
  expand_kernel<<<(unsigned)((a.n_rows + 255) / 256), 256, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return PB_E_LAUNCH;
  int rc = PB_OK;
  if (a.sampler_runs) {
    // rows that pb_sample_ws's two passes settle themselves go through it, a batch with others
    // through pb_sample (the same choice as for sampling)
    if (!(kinds & PB_VERIFY_OTHER))
      rc = pb_sample_ws(a.x, dtype, a.n_rows, a.V, a.row_stride, nullptr, a.rowp, a.tok, a.info, nullptr,
                        ws + plan.sampler, plan.bytes - plan.sampler, st);
    else
      rc = pb_sample(a.x, dtype, a.n_rows, a.V, a.row_stride, nullptr, a.rowp, a.tok, a.info, nullptr, st);
    if (rc != PB_OK) return rc;
  }
  if (a.mass_runs) {
    const int C = verify_cluster(a.n_rows, (int64_t)a.V * sizeof(T));
    rc = launch_cluster(mass_kernel<T>, a, a.n_rows * C, VT, C, 0, st);
    if (rc != PB_OK) return rc;
  }
  const int C = verify_cluster(a.n_seqs, (int64_t)a.V * sizeof(T));
  return launch_cluster(pick_kernel<T>, a, a.n_seqs * C, VT, C, 0, st);
}

}  // namespace

extern "C" {

int64_t pb_verify_ws_bytes(int64_t n_rows, int64_t vocab, int dtype) {
  if (n_rows < 0 || vocab <= 0 || !elem_size(dtype)) return PB_E_INVALID;
  return verify_plan(n_rows, vocab, dtype).bytes;
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
  if (reinterpret_cast<uintptr_t>(logits) % es) return PB_E_INVALID;
  if (draft_probs) {
    const int ps = elem_size(probs_dtype);
    if (!ps || probs_stride < vocab || reinterpret_cast<uintptr_t>(draft_probs) % ps) return PB_E_INVALID;
  }
  if (kinds < 0 || kinds > PB_VERIFY_ANY) return PB_E_INVALID;
  const VerifyPlan plan = verify_plan(n_rows, vocab, dtype);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) || ws_bytes < plan.bytes) return PB_E_INVALID;
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
  const int k = kinds ? kinds : PB_VERIFY_ANY;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == PB_DTYPE_F32) return verify_run<float>(a, dtype, k, ws, plan, st);
  if (dtype == PB_DTYPE_BF16) return verify_run<__nv_bfloat16>(a, dtype, k, ws, plan, st);
  return verify_run<__half>(a, dtype, k, ws, plan, st);
}

}  // extern "C"
