// logit_loss.cu — losses of post-training on rows of logits and their
// gradients (sm_100a): the clipped policy loss with a KL term and the
// preference loss on paired sequences.
//
// For a row with scaled logits z = scale * x and label y:
//   lse = log sum exp z,  logp = z_y - lse.
// Policy: r = exp(logp - old), l1 = -r A, l2 = -clip(r, lo, hi) A, d = ref - logp,
//   kl = exp(d) - d - 1,  loss = max(l1, l2) + beta kl,
//   g = dloss/dlogp = (l2 > l1 ? 0 : -r A) + beta (1 - exp(d)).
// Preference: S_s = sum over the sequence's rows of logp - ref, m = beta (S_chosen - S_rejected),
//   loss = (1 - e) softplus(-m) + e softplus(m),
//   g = +-beta (e sigmoid(m) - (1 - e) sigmoid(-m)) on the chosen / rejected rows.
// Both: dlogits[c] = dloss g scale ([c == y] - exp(z_c - lse)).
//
// A row is left out when its label is the ignored index or no column (and, for
// preferences, when it lies in no sequence): its logits are not read, its
// results and gradients are 0.
//
// Statistics: with c = scale log2(e) and m the running extreme (the largest x, or
// the smallest for a negative scale), an online sum of 2^(x c - R) per thread,
// R = m c as rounded; x c - R is one fma. What R lost is put back at the end,
// in 64 bits once per row: logp = scale (x_y - m) - ln s, lse = scale m + ln s.
// Where |R| is 2^23 or more (a row masked with the type's lowest value
// throughout), 2^((x - m) c) is summed instead, which is right for any size. c has
// two float32 parts: rounded to one it would shift every lse of a call in the
// same direction (some 5e-7), which a sum over a sequence's rows adds up. Both
// parts have one sign, so that a logit of -inf gives -inf and not NaN.
#include "common.cuh"
#include "pipe.cuh"

namespace dslpg {

struct LossRows {
  const void* x;
  const void* labels;
  int64_t M, N, ld, ignored;
  int label64;
  double scale;
  float scale_f, sign;  // scale as float32; 1 or -1
  float c_hi, c_lo;     // scale * log2(e) in two parts of one sign
  int tpr, rpc;         // threads of a row, rows of a CTA
};

struct PolicyTerms {
  const float *old_logp, *adv, *ref;
  int64_t old_stride, adv_stride, ref_stride;
  float lo, hi, kl_coef;
};

struct PairTerms {
  const void* starts;
  int starts64;
  int64_t pairs;
  const float* ref;
  int64_t ref_stride;
  float beta, smoothing;
};

struct LossOut {
  float *loss, *logp, *lse, *kl;
};

struct GradOut {
  const float* dloss;
  int64_t dloss_stride;
  const float* lse;        // backward: the forward's
  const float* log_ratio;  // preference backward
  void* dx;
  int64_t ldo;
};

// Sequence bound s of a preference batch, kept inside the rows.
DSLPG_DEV int64_t start_at(const PairTerms& p, int64_t s, int64_t rows) {
  const int64_t v = p.starts64 ? static_cast<const int64_t*>(p.starts)[s]
                               : static_cast<int64_t>(static_cast<const int32_t*>(p.starts)[s]);
  return v < 0 ? 0 : (v > rows ? rows : v);
}

// Column of row r's label, or -1 when the row is left out.
DSLPG_DEV int64_t label_col(const LossRows& a, int64_t r) {
  const int64_t y = a.label64 ? static_cast<const int64_t*>(a.labels)[r]
                              : static_cast<int64_t>(static_cast<const int32_t*>(a.labels)[r]);
  return (y == a.ignored || y < 0 || y >= a.N) ? -1 : y;
}

// The row's sequence (the last one that starts at or before r), or -1 outside all of them.
DSLPG_DEV int64_t sequence_of(const PairTerms& p, int64_t r, int64_t rows) {
  const int64_t n = 2 * p.pairs;
  if (r < start_at(p, 0, rows) || r >= start_at(p, n, rows)) return -1;
  int64_t lo = 0, hi = n;  // starts[lo] <= r < starts[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (start_at(p, mid, rows) <= r) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr float kPlainR = 8388608.f;  // 2^23

// log2 of what a sum against the extreme m0 is multiplied with to be one against
// m1 >= m0 (extremes as sign * x, ca = |c|).
DSLPG_DEV float rebase_log2(float m0, float m1, float ca) {
  const float r0 = m0 * ca, r1 = m1 * ca;
  return fmaxf(fabsf(r0), fabsf(r1)) < kPlainR ? r0 - r1 : (m0 - m1) * ca;
}

// Online statistics of one thread: m = the largest sign * x, s the sum.
struct Stat {
  float m = kNegInf, s = 0.f;
  DSLPG_DEV void rebase(float nm, const LossRows& a) {
    if (m != nm && m != kNegInf) s *= ex2(rebase_log2(m, nm, fabsf(a.c_hi)));  // s is 0 while m = -inf
    m = nm;
  }
};

// One logit.
DSLPG_DEV void fold_value(Stat& st, float x, const LossRows& a) {
  const float nm = max_nan(st.m, x * a.sign);
  if (nm == kNegInf) return;  // nothing but -inf so far
  st.rebase(nm, a);
  const float r = nm * fabsf(a.c_hi);
  const float y = fabsf(r) < kPlainR ? x : x - nm * a.sign;
  st.s += ex2(fmaf(y, a.c_lo, fmaf(y, a.c_hi, fabsf(r) < kPlainR ? -r : 0.f)));
}

// NV vectors of logits, all valid. PACKED: two to an instruction (fma.f32x2),
// which the forward kernel gains by (201 us against 208 for the batch below, at
// 3 CTAs an SM); the fused one, at 64 registers a thread, spills with it.
template <typename T, int NV, bool PACKED>
DSLPG_DEV void fold_rows(Stat& st, const Vec16 (&v)[NV], const LossRows& a) {
  constexpr int E = Elt<T>::kPerVec;
  const float ext = (a.sign >= 0.f) ? RawExtreme<T, NV, false>::run(v) : RawExtreme<T, NV, true>::run(v);
  const float nm = max_nan(st.m, ext * a.sign);
  if (nm == kNegInf) return;
  const float r = nm * fabsf(a.c_hi), m = nm * a.sign;
  float acc[2] = {0.f, 0.f};
  if (!(fabsf(r) < kPlainR)) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[E];
      unpack<T>(v[k], x);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e & 1] += ex2(fmaf(x[e] - m, a.c_lo, (x[e] - m) * a.c_hi));
    }
  } else if constexpr (PACKED) {
    const f32x2 hi = pk2(a.c_hi, a.c_hi), lo = pk2(a.c_lo, a.c_lo), neg = pk2(-r, -r);
    f32x2 sum[2] = {pk2(0.f, 0.f), pk2(0.f, 0.f)};
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int p = 0; p < E / 2; ++p) {
        const f32x2 x = unpack_pair<T>(v[k], p);
        float d0, d1;
        upk2(fma2(x, lo, fma2(x, hi, neg)), d0, d1);
        sum[p & 1] = add2(sum[p & 1], pk2(ex2(d0), ex2(d1)));
      }
    acc[0] = hsum2(add2(sum[0], sum[1]));
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      float x[E];
      unpack<T>(v[k], x);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e & 1] += ex2(fmaf(x[e], a.c_lo, fmaf(x[e], a.c_hi, -r)));
    }
  }
  st.rebase(nm, a);
  st.s += acc[0] + acc[1];
}

// A thread's sum against the row's extreme.
DSLPG_DEV float merged(const Stat& st, float gm, const LossRows& a) {
  return (st.m == gm || st.m == kNegInf) ? st.s : st.s * ex2(rebase_log2(st.m, gm, fabsf(a.c_hi)));
}

// A row's merged statistics. Where the extreme is not finite, all of it is NaN.
struct RowStat {
  float m, r;     // the extreme x itself; m c as rounded
  float log2_sum;  // of the sum as it was formed
  double log2_s;  // of the sum of 2^((x - m) c)
  DSLPG_DEV RowStat(float gm, float gs, const LossRows& a) : m(gm * a.sign), r(gm * fabsf(a.c_hi)) {
    log2_sum = fabsf(gm) < kPosInf ? log2f(gs) : __builtin_nanf("");
    log2_s = log2_sum;
    if (fabsf(r) < kPlainR) {
      const double c = static_cast<double>(a.c_hi) + static_cast<double>(a.c_lo);
      log2_s += static_cast<double>(r) - static_cast<double>(m) * c;
    }
  }
  DSLPG_DEV double ln_s() const { return 0.69314718055994530942 * log2_s; }
  DSLPG_DEV double lse(const LossRows& a) const { return a.scale * static_cast<double>(m) + ln_s(); }
  DSLPG_DEV double logp(const LossRows& a, float xl) const {
    const double v = a.scale * (static_cast<double>(xl) - static_cast<double>(m)) - ln_s();
    return v > 0.0 ? 0.0 : v;  // rounding may leave the only column with a probability 1e-8 above 0
  }
};

struct PolicyRow {
  float loss, kl, g;  // g: dloss / dlogp
};

DSLPG_DEV PolicyRow policy_row(const PolicyTerms& p, float old_logp, float adv, float ref, double logp) {
  float ratio = expf(static_cast<float>(logp - static_cast<double>(old_logp)));
  if (adv == 0.f && ratio == kPosInf) ratio = 1.f;  // r A is 0 at A = 0 for any r, also one beyond float32
  const float l1 = -ratio * adv, l2 = -fminf(fmaxf(ratio, p.lo), p.hi) * adv;
  PolicyRow o{max_nan(l1, l2), 0.f, l2 > l1 ? 0.f : l1};
  if (p.ref != nullptr) {
    const float d = static_cast<float>(static_cast<double>(ref) - logp);
    const float e = expm1f(d);
    // exp(d) - d - 1; its power series near 0, where the difference cancels (|d| < 1/4: the first term left out is
    // below 2e-8 of the sum). At d = inf (logp = -inf) it is inf, not inf - inf.
    o.kl = fabsf(d) < 0.25f
               ? d * d * (0.5f + d * (1.f / 6 + d * (1.f / 24 + d * (1.f / 120 + d * (1.f / 720 + d * (1.f / 5040))))))
               : (d == kPosInf ? d : e - d);
    if (p.kl_coef != 0.f) {
      o.loss += p.kl_coef * o.kl;
      o.g -= p.kl_coef * e;
    }
  }
  return o;
}

DSLPG_DEV PolicyRow policy_row(const PolicyTerms& p, int64_t r, double logp) {
  return policy_row(p, p.old_logp[r * p.old_stride], p.adv[r * p.adv_stride],
                    p.ref != nullptr ? p.ref[r * p.ref_stride] : 0.f, logp);
}

// dloss g of a preference row in sequence `seq` (chosen ones first).
DSLPG_DEV float pair_slope(const PairTerms& p, const float* log_ratio, int64_t seq) {
  const bool chosen = seq < p.pairs;
  const int64_t k = chosen ? seq : seq - p.pairs;
  const float m = p.beta * (log_ratio[k] - log_ratio[p.pairs + k]);
  const float up = 1.f / (1.f + expf(-m)), down = 1.f / (1.f + expf(m));  // sigmoid(m), sigmoid(-m)
  const float slope = p.beta * (p.smoothing * up - (1.f - p.smoothing) * down);
  return chosen ? slope : -slope;
}

enum LossKind : int { kPolicy = 0, kPair = 1 };

// A stretch of n elements from p on as vectors: `head` elements up to the next
// 16-byte boundary, `vecs` vectors, and `tail` elements.
template <typename T> struct Stretch {
  int head, vecs, tail;
  DSLPG_DEV Stretch(const T* p, int64_t n) {
    constexpr int E = Elt<T>::kPerVec;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15) / static_cast<int>(sizeof(T));
    const int64_t h = off ? E - off : 0;
    head = static_cast<int>(h < n ? h : n);
    vecs = static_cast<int>((n - head) / E);
    tail = static_cast<int>(n - head - static_cast<int64_t>(vecs) * E);
  }
};

// Fold elements [0, n) from xr on with `tpr` threads, this one being t: 16-byte
// vectors, the next ones loaded before this step's arithmetic, and the elements
// before the first and behind the last whole vector, one a thread.
template <typename T, int U, bool PACKED, class Load>
DSLPG_DEV void fold_row(Stat& st, const T* xr, int64_t n, const LossRows& a, int t, int tpr, Load ld) {
  constexpr int E = Elt<T>::kPerVec;
  const Stretch<T> w(xr, n);
  const T* body = xr + w.head;
  const int stride = U * tpr;
  auto load = [&](Vec16 (&dst)[U], int j0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u * tpr;
      dst[u] = Vec16{{0u, 0u, 0u, 0u}};
      if (j < w.vecs) dst[u] = ld(body + static_cast<int64_t>(j) * E);
    }
  };
  Vec16 nx[U];
  load(nx, t);
  if (t < w.head + w.tail) {
    fold_value(st, to_f(t < w.head ? xr[t] : xr[n - w.tail + (t - w.head)]), a);
  }
  for (int j0 = t; j0 < w.vecs; j0 += stride) {
    Vec16 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = nx[u];
    if (j0 + stride < w.vecs) load(nx, j0 + stride);
    if (j0 + (U - 1) * tpr < w.vecs) {
      fold_rows<T, U, PACKED>(st, v, a);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (j0 + u * tpr < w.vecs) {
          const Vec16 one[1] = {v[u]};
          fold_rows<T, 1, PACKED>(st, one, a);
        }
      }
    }
  }
}

// The results of a row that counts, or of one that is left out.
template <int KIND>
DSLPG_DEV void write_row(const LossRows& a, const PolicyTerms& pol, const LossOut& o, int64_t r, bool counts, float xl,
                         const RowStat& rs) {
  double logp = 0.0, lse = 0.0;
  PolicyRow p{0.f, 0.f, 0.f};
  if (counts) {
    lse = rs.lse(a);
    logp = rs.logp(a, xl);
    if constexpr (KIND == kPolicy) p = policy_row(pol, r, logp);
  }
  o.logp[r] = static_cast<float>(logp);
  o.lse[r] = static_cast<float>(lse);
  if constexpr (KIND == kPolicy) {
    o.loss[r] = p.loss;
    o.kl[r] = p.kl;
  }
}

template <int KIND> DSLPG_DEV int64_t counted_col(const LossRows& a, const PairTerms& pair, int64_t r) {
  int64_t col = label_col(a, r);
  if constexpr (KIND == kPair)
    if (col >= 0 && sequence_of(pair, r, a.M) < 0) col = -1;
  return col;
}

// Row statistics: `tpr` threads a row. HBM-bound: bf16 [6000, 128256] with 1500
// rows left out takes 188 us (6.14 TB/s of 6.51 measured) in a loop over one batch,
// 202 over three in turn, with 4 loads in flight a thread and 4 CTAs an SM; in the
// loop 3 CTAs 202, 5 193; 2, 3, 6 and 8 loads 197, 194, 223, 221.
// A CTA a row, handed out by the hardware: shared out evenly beforehand, rows that
// are left out leave some CTAs with less than others (261 us). Writes the row's losses (policy) or its
// logp and lse (preferences; pair_kernel then sums them).
template <int KIND, typename T>
__global__ void __launch_bounds__(256, 4) loss_rows_kernel(const __grid_constant__ LossRows a,
                                                           const __grid_constant__ PolicyTerms pol,
                                                           const __grid_constant__ PairTerms pair, const LossOut o) {
  __shared__ float red[2][32];
  const int g = threadIdx.x / a.tpr, t = threadIdx.x - g * a.tpr;
  const int nw = a.tpr >> 5, first_warp = g * nw;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.rpc;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.rpc; base < a.M; base += step) {
    const int64_t r = base + g;
    const int64_t col = r < a.M ? counted_col<KIND>(a, pair, r) : -1;
    const T* xr = static_cast<const T*>(a.x) + r * a.ld;
    Stat st;
    float xl = 0.f;
    if (col >= 0) {
      if (t == 0) xl = to_f(xr[col]);
      fold_row<T, 4, true>(st, xr, a.N, a, t, a.tpr, [](const void* p) { return ld_stream(p); });
    }
    const float gm = group_reduce<MaxOp>(st.m, red[0], nw, first_warp);
    const float gs = group_reduce<SumOp>(merged(st, gm, a), red[1], nw, first_warp);
    if (t == 0 && r < a.M) write_row<KIND>(a, pol, o, r, col >= 0, xl, RowStat(gm, gs, a));
  }
}

// The same for few long rows: a cluster of CTAs a row, each folding a stretch of
// it; their statistics meet in distributed shared memory.
template <int KIND, typename T>
__global__ void __launch_bounds__(512) loss_split_kernel(const __grid_constant__ LossRows a,
                                                         const __grid_constant__ PolicyTerms pol,
                                                         const __grid_constant__ PairTerms pair, const LossOut o) {
  __shared__ float red[2][32];
  __shared__ float slots[2];
  namespace cg = cooperative_groups;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int64_t r = blockIdx.x / C;
  const int64_t col = counted_col<KIND>(a, pair, r);
  ClusterReducer rd{slots, red, 0, C};
  Stat st;
  float xl = 0.f;
  if (col >= 0) {
    const T* xr = static_cast<const T*>(a.x) + r * a.ld;
    const int64_t part = ((a.N + C - 1) / C + 63) & ~63ll, lo = part * rank, n = lo + part < a.N ? part : a.N - lo;
    if (threadIdx.x == 0 && rank == 0) xl = to_f(xr[col]);
    if (n > 0) fold_row<T, 4, true>(st, xr + lo, n, a, threadIdx.x, blockDim.x, [](const void* p) { return ld_stream(p); });
  }
  const float gm = rd.template reduce<MaxOp>(st.m);
  const float gs = rd.template reduce<SumOp>(merged(st, gm, a));
  if (rank == 0 && threadIdx.x == 0) write_row<KIND>(a, pol, o, r, col >= 0, xl, RowStat(gm, gs, a));
  cl.sync();  // no CTA leaves while another may still read its slots
}

DSLPG_DEV double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

// One CTA a pair: the two sequences' sums of logp - ref (64 bits, in a fixed
// order), their margin and the pair's loss.
__global__ void __launch_bounds__(256) pair_kernel(const LossRows a, const PairTerms p, const float* logp, float* loss,
                                                   float* log_ratio) {
  __shared__ double part[2][8];
  wait_for_primary();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t k = blockIdx.x; k < p.pairs; k += gridDim.x) {
    for (int side = 0; side < 2; ++side) {
      const int64_t s = k + side * p.pairs;
      const int64_t lo = start_at(p, s, a.M), hi = start_at(p, s + 1, a.M);
      double sum = 0.0;
      for (int64_t r = lo + threadIdx.x; r < hi; r += blockDim.x)
        if (label_col(a, r) >= 0) sum += static_cast<double>(logp[r]) - static_cast<double>(p.ref[r * p.ref_stride]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) part[side][warp] = sum;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      double t[2] = {0.0, 0.0};
      for (int side = 0; side < 2; ++side) {
        for (int w = 0; w < 8; ++w) t[side] += part[side][w];
        log_ratio[k + side * p.pairs] = static_cast<float>(t[side]);
      }
      const double m = static_cast<double>(p.beta) * (t[0] - t[1]), e = p.smoothing;
      // a term of weight 0 is left out: an infinite margin would make it NaN
      const double up = e < 1.0 ? (1.0 - e) * softplus(-m) : 0.0, down = e > 0.0 ? e * softplus(m) : 0.0;
      loss[k] = static_cast<float>(up + down);
    }
    __syncthreads();
  }
}

// dlogits[c] = k1 p with k1 = -dloss g scale; p = 2^(x c + off), or 2^((x + shift) c + off) where `far`: where off
// would be so large (beyond kNear) that its rounding shows.
struct GradTerms {
  float k1, c, off, shift;
  bool far;
};
constexpr float kNear = 64.f;

template <typename T, bool FAR> DSLPG_DEV void grad_vec(const Vec16& v, const GradTerms& gt, T* dst) {
  constexpr int E = Elt<T>::kPerVec;
  float x[E];
  unpack<T>(v, x);
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = gt.k1 * ex2(fmaf(FAR ? x[e] + gt.shift : x[e], gt.c, gt.off));
  StoreOut<T, E>::run(dst, x);
}

template <typename T> DSLPG_DEV void grad_one(const T* x, T* y, const GradTerms& gt) {
  *y = from_f<T>(gt.k1 * ex2(fmaf(gt.far ? to_f(*x) + gt.shift : to_f(*x), gt.c, gt.off)));
}

// 16 bytes from any element on: the two vectors around them, shifted together.
// `s`: their distance from a 16-byte boundary (the same for a whole row).
DSLPG_DEV Vec16 shifted_vec(const Vec16& lo, const Vec16& hi, int s) {
  uint32_t w[8] = {lo.w[0], lo.w[1], lo.w[2], lo.w[3], hi.w[0], hi.w[1], hi.w[2], hi.w[3]};
  if (s & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (s & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  Vec16 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v.w[i] = __funnelshift_r(w[i], w[i + 1], (s & 3) * 8);
  return v;
}

// dlogits of elements [0, n) by `nt` threads, this one being t, then the label
// column (col, if in there): k1 expm1(logp). Vectors are those of the output; the
// logits' may lie at another distance from a 16-byte boundary (rows of odd
// length). Where they lie at the same one (SAME: in every row), the next chunk's
// loads are issued before this chunk's arithmetic; elsewhere two vectors are read
// for each one written, two at a time, with nothing ahead (126 registers already):
// fp16 [2048, 32001] in rows 32064 apart 81 us, [2048, 32000] 50.
template <typename T, int U, bool SAME, bool FAR>
DSLPG_DEV void grad_row_as(const T* xr, T* yr, int64_t n, const GradTerms& gt, double logp, int64_t col, int t, int nt) {
  constexpr int E = Elt<T>::kPerVec;
  const Stretch<T> w(yr, n);
  const T* xb = xr + w.head;
  T* yb = yr + w.head;
  const int s = SAME ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(xb) & 15);
  if (s == 0) {
    auto load = [&](Vec16 (&dst)[U], int j0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * nt;
        dst[u] = Vec16{{0u, 0u, 0u, 0u}};
        if (j < w.vecs) dst[u] = ld_stream(xb + static_cast<int64_t>(j) * E);
      }
    };
    Vec16 nx[U];
    load(nx, t);
    for (int j0 = t; j0 < w.vecs; j0 += U * nt) {
      Vec16 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = nx[u];
      if (j0 + U * nt < w.vecs) load(nx, j0 + U * nt);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * nt;
        if (j < w.vecs) grad_vec<T, FAR>(v[u], gt, yb + static_cast<int64_t>(j) * E);
      }
    }
  } else if constexpr (!SAME) {
    // a vector whose two neighbours do not both lie inside the row (its first and last ones) is done element by element
    const uintptr_t x_lo = reinterpret_cast<uintptr_t>(xr), x_hi = reinterpret_cast<uintptr_t>(xr + n);
    for (int j0 = t; j0 < w.vecs; j0 += 2 * nt) {
      Vec16 lo[2], hi[2];
      bool inside[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u * nt;
        const uintptr_t at = reinterpret_cast<uintptr_t>(xb + static_cast<int64_t>(j) * E) - s;
        inside[u] = j < w.vecs && at >= x_lo && at + 32 <= x_hi;
        if (inside[u]) {
          lo[u] = ld_keep(reinterpret_cast<const void*>(at));
          hi[u] = ld_keep(reinterpret_cast<const void*>(at + 16));
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = j0 + u * nt;
        if (j >= w.vecs) continue;
        const int64_t c = static_cast<int64_t>(j) * E;
        if (inside[u]) {
          grad_vec<T, FAR>(shifted_vec(lo[u], hi[u], s), gt, yb + c);
        } else {
          for (int e = 0; e < E; ++e) grad_one(xb + c + e, yb + c + e, gt);
        }
      }
    }
  }
  if (t < w.head + w.tail) {
    const int64_t c = t < w.head ? t : n - w.tail + (t - w.head);
    grad_one(xr + c, yr + c, gt);
  }
  // the label column, rewritten by the thread that wrote its vector or element
  if (col >= 0 && col < n) {
    int64_t owner;
    if (col < w.head) owner = col;
    else if (col >= n - w.tail) owner = w.head + (col - (n - w.tail));
    else owner = (col - w.head) / E % nt;
    if (owner == t) yr[col] = from_f<T>(gt.k1 * expm1f(static_cast<float>(logp)));
  }
}

// (`far`: one vector at a time, to keep the registers of the other loop. It begins at |lse| of 44 and costs: bf16
// [4096, 128256] with lse near 60 448 us, near 16 316.)
template <typename T, int U, bool SAME>
DSLPG_DEV void grad_row(const T* xr, T* yr, int64_t n, const GradTerms& gt, double logp, int64_t col, int t, int nt) {
  if (gt.far) grad_row_as<T, 1, SAME, true>(xr, yr, n, gt, logp, col, t, nt);
  else grad_row_as<T, U, SAME, false>(xr, yr, n, gt, logp, col, t, nt);
}

template <typename T> DSLPG_DEV void zero_row(T* yr, int64_t n, int t, int nt) {
  constexpr int E = Elt<T>::kPerVec;
  const Stretch<T> w(yr, n);
  for (int j = t; j < w.vecs; j += nt) st_stream(yr + w.head + static_cast<int64_t>(j) * E, Vec16{{0u, 0u, 0u, 0u}});
  if (t < w.head + w.tail) yr[t < w.head ? t : n - w.tail + (t - w.head)] = from_f<T>(0.f);
}

// Of a row whose statistics are known, dl = its dloss: p = 2^(x c - (R + log2 sum)), or 2^((x - m) c - log2 s).
DSLPG_DEV GradTerms grad_terms(const RowStat& rs, const LossRows& a, float dl, float g) {
  const float k1 = -(dl * g) * a.scale_f, off = rs.r + rs.log2_sum;
  const bool far = !(fabsf(off) <= kNear && fabsf(rs.r) <= kNear);
  return GradTerms{k1, a.c_hi, far ? -static_cast<float>(rs.log2_s) : -off, -rs.m, far};
}

// Beyond this a float32 lse no longer tells the row's probabilities to 2e-5 (a
// row masked with the type's lowest value throughout has lse = -3e38 + ln N).
constexpr float kLseTrusted = 256.f;

// The gradient alone, from the forward's lse: `tpr` threads a row, or (few long
// rows) gridDim.y CTAs a row, each a stretch of its columns; read once and
// written once. HBM-bound: 158 us for bf16 [2100, 128256] with 552 rows left out
// (5.93 TB/s). Rows whose lse is beyond kLseTrusted have their statistics formed
// again.
template <int KIND, typename T, bool SAME>
__global__ void __launch_bounds__(256) loss_bwd_kernel(const __grid_constant__ LossRows a,
                                                       const __grid_constant__ PolicyTerms pol,
                                                       const __grid_constant__ PairTerms pair, const GradOut o) {
  __shared__ float red[2][32];
  const int g0 = threadIdx.x / a.tpr, t = threadIdx.x - g0 * a.tpr;
  const int nw = a.tpr >> 5, first_warp = g0 * nw;
  const int64_t part = ((a.N + gridDim.y - 1) / gridDim.y + 63) & ~63ll, lo = part * blockIdx.y;
  const int64_t n = lo + part < a.N ? part : a.N - lo;
  const int64_t step = static_cast<int64_t>(gridDim.x) * a.rpc;
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * a.rpc; base < a.M; base += step) {
    const int64_t r = base + g0;
    int64_t col = -1, seq = 0;
    if (r < a.M) {
      col = label_col(a, r);
      if (KIND == kPair && col >= 0 && (seq = sequence_of(pair, r, a.M)) < 0) col = -1;
    }
    T* yr = static_cast<T*>(o.dx) + r * o.ldo + lo;
    const T* xr = static_cast<const T*>(a.x) + r * a.ld;
    float lse = 0.f, xl = 0.f;
    if (col >= 0) {
      lse = o.lse[r];
      xl = to_f(xr[col]);
    }
    double logp = static_cast<double>(xl) * a.scale - static_cast<double>(lse);
    // p = 2^(x c - lse log2(e)), or 2^((x - lse / scale) c) (at scale 0 the row is uniform)
    const double off = -1.4426950408889634074 * static_cast<double>(lse);
    GradTerms gt{0.f, a.c_hi, static_cast<float>(off), 0.f, fabs(off) > static_cast<double>(kNear) && a.scale != 0.0};
    if (gt.far) {
      gt.shift = -static_cast<float>(static_cast<double>(lse) / a.scale);
      gt.off = 0.f;
    }
    const bool again = !(fabsf(lse) <= kLseTrusted);
    if (__syncthreads_or(again)) {  // the CTA's rows together: the reductions have barriers
      Stat st;
      if (again) fold_row<T, 1, true>(st, xr, a.N, a, t, a.tpr, [](const void* p) { return ld_stream(p); });
      const float gm = group_reduce<MaxOp>(st.m, red[0], nw, first_warp);
      const float gs = group_reduce<SumOp>(merged(st, gm, a), red[1], nw, first_warp);
      if (again) {
        const RowStat rs(gm, gs, a);
        logp = rs.logp(a, xl);
        gt = grad_terms(rs, a, 0.f, 0.f);
      }
    }
    if (r >= a.M || n <= 0) continue;
    if (col < 0) {
      zero_row<T>(yr, n, t, a.tpr);
      continue;
    }
    float g, dl;
    if constexpr (KIND == kPolicy) {
      g = policy_row(pol, r, logp).g;
      dl = o.dloss[r * o.dloss_stride];
    } else {
      g = pair_slope(pair, o.log_ratio, seq);
      dl = o.dloss[(seq < pair.pairs ? seq : seq - pair.pairs) * o.dloss_stride];
    }
    gt.k1 = -(dl * g) * a.scale_f;
    grad_row<T, 4, SAME>(xr + lo, yr, n, gt, logp, col - lo, t, a.tpr);
  }
}

// Loss and gradient in one kernel, any row: a CTA a row, whose second reading
// comes from L2 while the rows in flight, one an SM, fit there (38 MB for 16-bit
// rows of 128256, 76 MB in fp32; the first reading marks its lines to stay, and
// nothing demotes them). Rows are taken NT at a time: of the counted
// ones among them, and of the left-out ones, CTA k does every G-th by their
// number, so that none gets more of either kind than another.
// Bound by instructions and latency: one pass of a row at a time is on an SM, so its
// reading of HBM and its writing take turns. bf16 [8192, 128256] with 1024 rows left
// out takes 812 us (floor 605); 768 threads 835, two CTAs of 512 827, a quarter of
// the exponentials on the FMA pipe 817. A row kept in the shared memory of a
// cluster (bulk copies, one read) was slower, 868 us: the ring holds 1.6 such rows
// an SM, too little to cover the loads, the exchange of statistics and the gradient
// behind one another.
template <typename T, int NT, bool SAME>
__global__ void __launch_bounds__(NT, 1) policy_two_pass_kernel(const __grid_constant__ LossRows a,
                                                                const __grid_constant__ PolicyTerms pol,
                                                                const LossOut o, const GradOut go) {
  __shared__ float red[2][32];
  __shared__ int in_warp[32];
  __shared__ int list_row[2][NT], list_col[NT];
  constexpr int nw = NT / 32;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int64_t G = gridDim.x;
  int64_t seen[2] = {0, 0};  // left-out and counted rows before the present ones
  for (int64_t base = 0; base < a.M; base += NT) {
    const int64_t mine = base + t;
    const int64_t label = mine < a.M ? label_col(a, mine) : -1;
    const bool counted = label >= 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, counted);
    if (lane == 0) in_warp[warp] = __popc(mask);
    __syncthreads();
    int before = lane < nw && lane < warp ? in_warp[lane] : 0, total = lane < nw ? in_warp[lane] : 0;
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, k);
      total += __shfl_xor_sync(0xffffffffu, total, k);
    }
    before += __popc(mask & ((1u << lane) - 1u));  // counted rows of this block before mine
    const int rows = static_cast<int>(a.M - base < NT ? a.M - base : NT);
    // the first of CTA k's numbers from seen[kind] on, and how many of the block's rows have one
    int64_t first[2] = {0, 0};
    int count[2] = {0, 0};
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const int64_t n = kind ? total : rows - total;
      first[kind] = seen[kind] + (static_cast<int64_t>(blockIdx.x) + G - seen[kind] % G) % G;
      const int64_t ahead = seen[kind] + n - first[kind];
      count[kind] = ahead > 0 ? static_cast<int>((ahead + G - 1) / G) : 0;
    }
    if (mine < a.M) {
      const int64_t number = counted ? seen[1] + before - first[1] : seen[0] + (t - before) - first[0];
      if (number >= 0 && number % G == 0) {
        list_row[counted][number / G] = t;
        if (counted) list_col[number / G] = static_cast<int>(label);
      }
    }
    __syncthreads();
    seen[0] += rows - total;
    seen[1] += total;
    for (int n = 0; n < count[1]; ++n) {
      const int64_t r = base + list_row[1][n];
      const int col = list_col[n];
      const T* xr = static_cast<const T*>(a.x) + r * a.ld;
      const float xl = to_f(xr[col]), dl = go.dloss[r * go.dloss_stride];
      uint64_t keep;
      asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(keep));
      Stat st;
      fold_row<T, 4, false>(st, xr, a.N, a, t, NT, [&](const void* p) {
        Vec16 v;
        asm volatile("ld.global.nc.L1::no_allocate.L2::cache_hint.v4.u32 {%0,%1,%2,%3}, [%4], %5;"
                     : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3])
                     : "l"(p), "l"(keep));
        return v;
      });
      const float gm = group_reduce<MaxOp>(st.m, red[0], nw, 0);
      const float gs = group_reduce<SumOp>(merged(st, gm, a), red[1], nw, 0);
      const RowStat rs(gm, gs, a);
      if (t == 0) write_row<kPolicy>(a, pol, o, r, true, xl, rs);
      const double logp = rs.logp(a, xl);
      grad_row<T, 2, SAME>(xr, static_cast<T*>(go.dx) + r * go.ldo, a.N, grad_terms(rs, a, dl, policy_row(pol, r, logp).g),
                     logp, col, t, NT);
    }
    for (int n = 0; n < count[0]; ++n) {
      const int64_t r = base + list_row[0][n];
      zero_row<T>(static_cast<T*>(go.dx) + r * go.ldo, a.N, t, NT);
      if (t == 0) o.loss[r] = o.logp[r] = o.lse[r] = o.kl[r] = 0.f;
    }
    __syncthreads();  // the lists are written again
  }
}

// Loss and gradient of rows that their threads hold (NV vectors a thread, 16-byte
// rows): read once, written once. In registers, but for 8 vectors of fp32, of which
// 128 bytes lie in local memory ([2048, 8192] 37.8 us of a floor of 19.6).
template <typename T, int NV>
__global__ void __launch_bounds__(512) policy_short_kernel(const __grid_constant__ LossRows a,
                                                           const __grid_constant__ PolicyTerms pol, const LossOut o,
                                                           const GradOut go) {
  constexpr int E = Elt<T>::kPerVec;
  __shared__ float red[2][32];
  const int g = threadIdx.x / a.tpr, t = threadIdx.x - g * a.tpr;
  const int nw = a.tpr >> 5, first_warp = g * nw;
  const int vecs = static_cast<int>(a.N / E);
  const int64_t r = static_cast<int64_t>(blockIdx.x) * a.rpc + g;
  const int64_t col = r < a.M ? label_col(a, r) : -1;
  const T* xr = static_cast<const T*>(a.x) + r * a.ld;
  T* yr = static_cast<T*>(go.dx) + r * go.ldo;
  Vec16 v[NV];
  float xl = 0.f, dl = 0.f;
  Stat st;
  if (col >= 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      v[k] = Vec16{{0u, 0u, 0u, 0u}};
      if (t + k * a.tpr < vecs) v[k] = ld_stream(xr + static_cast<int64_t>(t + k * a.tpr) * E);
    }
    xl = to_f(xr[col]);
    dl = go.dloss[r * go.dloss_stride];
    if (t + (NV - 1) * a.tpr < vecs) {
      fold_rows<T, NV, true>(st, v, a);
    } else {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        if (t + k * a.tpr < vecs) {
          const Vec16 one[1] = {v[k]};
          fold_rows<T, 1, true>(st, one, a);
        }
      }
    }
  }
  const float gm = group_reduce<MaxOp>(st.m, red[0], nw, first_warp);
  const float gs = group_reduce<SumOp>(merged(st, gm, a), red[1], nw, first_warp);
  if (r >= a.M) return;
  const RowStat rs(gm, gs, a);
  if (t == 0) write_row<kPolicy>(a, pol, o, r, col >= 0, xl, rs);
  if (col < 0) {
    zero_row<T>(yr, a.N, t, a.tpr);
    return;
  }
  const double logp = rs.logp(a, xl);
  const GradTerms gt = grad_terms(rs, a, dl, policy_row(pol, r, logp).g);
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if (t + k * a.tpr < vecs) {
      T* y = yr + static_cast<int64_t>(t + k * a.tpr) * E;
      if (gt.far) grad_vec<T, true>(v[k], gt, y);
      else grad_vec<T, false>(v[k], gt, y);
    }
  if (static_cast<int>(col / E % a.tpr) == t) yr[col] = from_f<T>(gt.k1 * expm1f(static_cast<float>(logp)));
}

namespace {

// Threads of a row: about 16 vectors each, a warp at least, `most` at most.
template <typename T> void set_threads(LossRows& a, int64_t n, int most) {
  const int64_t want = (n / Elt<T>::kPerVec + 15) / 16;
  a.tpr = static_cast<int>(want >= most ? most : (want + 31) / 32 * 32);
  if (a.tpr < 32) a.tpr = 32;
  a.rpc = a.tpr >= 256 ? 1 : 256 / a.tpr;
}

int ctas_of(const LossRows& a) {  // a CTA for each of its rows: the hardware hands them out as SMs become free
  const int64_t n = (a.M + a.rpc - 1) / a.rpc;
  return static_cast<int>(n < 0x7fffffff ? n : 0x7fffffff);
}

// Whether a row's logits and its gradients lie at the same distance from a 16-byte boundary, in every row.
template <typename T> bool same_phase(const LossRows& a, const GradOut& o) {
  const uintptr_t apart = reinterpret_cast<uintptr_t>(a.x) - reinterpret_cast<uintptr_t>(o.dx);
  return apart % 16 == 0 && (a.ld - o.ldo) * static_cast<int64_t>(sizeof(T)) % 16 == 0;
}

constexpr int64_t kSplitBytes = 32 * 1024;  // a CTA's stretch of a split row, at least

template <int KIND, typename T>
cudaError_t launch_rows(LossRows a, const PolicyTerms& pol, const PairTerms& pair, const LossOut& o, cudaStream_t st) {
  // few long rows: a cluster of up to 8 CTAs each
  const int64_t bytes = a.N * static_cast<int64_t>(sizeof(T));
  int C = 1;
  while (C < 8 && a.M * C * 2 <= sm_count() && bytes / (C * 2) >= kSplitBytes) C *= 2;
  if (C > 1) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(C);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(a.M * C));
    cfg.blockDim = dim3(512);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, loss_split_kernel<KIND, T>, a, pol, pair, o);
  }
  set_threads<T>(a, a.N, 256);
  loss_rows_kernel<KIND, T><<<ctas_of(a), a.tpr * a.rpc, 0, st>>>(a, pol, pair, o);
  return cudaGetLastError();
}

template <int KIND, typename T>
cudaError_t launch_bwd(LossRows a, const PolicyTerms& pol, const PairTerms& pair, const GradOut& o, cudaStream_t st) {
  const int64_t bytes = a.N * static_cast<int64_t>(sizeof(T));
  int split = 1;
  while (split < 32 && a.M * split * 2 <= sm_count() * 4 && bytes / (split * 2) >= kSplitBytes / 2) split *= 2;
  set_threads<T>(a, (a.N + split - 1) / split, 256);
  const dim3 grid(ctas_of(a), split);
  if (same_phase<T>(a, o)) loss_bwd_kernel<KIND, T, true><<<grid, a.tpr * a.rpc, 0, st>>>(a, pol, pair, o);
  else loss_bwd_kernel<KIND, T, false><<<grid, a.tpr * a.rpc, 0, st>>>(a, pol, pair, o);
  return cudaGetLastError();
}

template <typename T, int NV>
cudaError_t launch_short(LossRows a, const PolicyTerms& pol, const LossOut& o, const GradOut& go, cudaStream_t st) {
  const int64_t want = (a.N / Elt<T>::kPerVec + NV - 1) / NV;
  a.tpr = static_cast<int>((want + 31) / 32 * 32);
  a.rpc = a.tpr >= 128 ? 1 : 128 / a.tpr;
  policy_short_kernel<T, NV><<<ctas_of(a), a.tpr * a.rpc, 0, st>>>(a, pol, o, go);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch_fused(LossRows a, const PolicyTerms& pol, const LossOut& o, const GradOut& go, cudaStream_t st) {
  constexpr int E = Elt<T>::kPerVec;
  const bool vec = kernel_path() != DSLPG_PATH_STREAM && aligned(a.x, 16) && aligned(go.dx, 16) && a.N % E == 0 &&
                   a.ld % E == 0 && go.ldo % E == 0;
  const int64_t vecs = a.N / E;
  if (vec && vecs <= 2 * 128) return launch_short<T, 2>(a, pol, o, go, st);
  if (vec && vecs <= 8 * 512) return launch_short<T, 8>(a, pol, o, go, st);
  // Both passes in one kernel pay where a CTA has one row (the second launch is saved), and for many long rows, whose
  // second reading then comes from L2. Elsewhere the forward and the backward kernel follow one another: of many shorter
  // rows an SM has several in flight there, and of few long ones several SMs share each. One kernel / two, in us, bf16:
  // [300, 1001] 8.4 / 9.7, [600, 1001] 12.4 / 10.3, [40000, 1001] 851 / 97; [148, 9001] 10.4 / 12.4, [10000, 9001]
  // 305 / 117; [6000, 48001] 319 / 289, [6000, 64001] 369 / 370, [6000, 96001] 495 / 539, [8192, 128256] 817 / 924;
  // [8, 2^20] 94 / 21, [74, 128256] 23.4 / 19.9, [100, 128256] 24.7 / 27.3; fp32 [2000, 28001] 124 / 120, [2000, 32001]
  // 128 / 135, [64, 128256] 37 / 29, [148, 128256] 44 / 57.
  const bool small = vecs <= 4 * 256, longer = a.N * static_cast<int64_t>(sizeof(T)) >= 112 * 1024;
  const int64_t sms = sm_count();
  if (longer ? 2 * a.M <= sms : a.M > (small ? 2 * sms : sms)) {
    if (cudaError_t e = launch_rows<kPolicy, T>(a, pol, PairTerms{}, o, st)) return e;
    GradOut from = go;
    from.lse = o.lse;
    return launch_bwd<kPolicy, T>(a, pol, PairTerms{}, from, st);
  }
  const int grid = static_cast<int>(small || a.M < sms ? a.M : sms);  // one CTA of 1024 threads an SM
  auto launch = [&](auto few, auto large) {
    if (small) few<<<grid, 128, 0, st>>>(a, pol, o, go);
    else large<<<grid, 1024, 0, st>>>(a, pol, o, go);
  };
  if (same_phase<T>(a, go)) launch(&policy_two_pass_kernel<T, 128, true>, &policy_two_pass_kernel<T, 1024, true>);
  else launch(&policy_two_pass_kernel<T, 128, false>, &policy_two_pass_kernel<T, 1024, false>);
  return cudaGetLastError();
}

enum Way { kFwd, kBwd, kFwdBwd };

template <int KIND, typename T>
cudaError_t launch_way(Way way, const LossRows& a, const PolicyTerms& pol, const PairTerms& pair, const LossOut& o,
                       const GradOut& go, cudaStream_t st) {
  if (way == kFwd) return launch_rows<KIND, T>(a, pol, pair, o, st);
  if (way == kBwd) return launch_bwd<KIND, T>(a, pol, pair, go, st);
  if constexpr (KIND == kPolicy) return launch_fused<T>(a, pol, o, go, st);
  return cudaErrorNotSupported;
}

template <int KIND>
cudaError_t dispatch(Way way, int dt, const LossRows& a, const PolicyTerms& pol, const PairTerms& pair,
                     const LossOut& o, const GradOut& go, cudaStream_t st) {
  switch (dt) {
    case DSLPG_F32: return launch_way<KIND, float>(way, a, pol, pair, o, go, st);
    case DSLPG_F16: return launch_way<KIND, __half>(way, a, pol, pair, o, go, st);
    default: return launch_way<KIND, __nv_bfloat16>(way, a, pol, pair, o, go, st);
  }
}

bool finite(double v) { return v - v == 0.0; }

// c's first part has to be a normal float32, and its second one (2^-24 of it, or 2^-126 in place of 0) small beside it.
bool scale_ok(double v) { return v == 0.0 || (fabs(v) >= 1e-30 && fabs(v) <= 1e30); }

int rows_args(LossRows& a, const dslpg_logit_rows* h) {
  if (!h) return DSLPG_ERR_NULL_POINTER;
  if (!is_float_dtype(h->logits_dtype) || (h->labels_dtype != DSLPG_I32 && h->labels_dtype != DSLPG_I64))
    return DSLPG_ERR_BAD_DTYPE;
  if (h->n_rows < 0 || h->n_cols < 1 || h->n_cols > (1ll << 30) || h->row_stride < h->n_cols) return DSLPG_ERR_BAD_SHAPE;
  if (!scale_ok(h->logit_scale)) return DSLPG_ERR_BAD_ARGUMENT;
  if (h->n_rows > 0 && (!h->logits || !h->labels)) return DSLPG_ERR_NULL_POINTER;
  a.x = h->logits;
  a.labels = h->labels;
  a.M = h->n_rows;
  a.N = h->n_cols;
  a.ld = h->row_stride;
  a.ignored = h->ignored_index;
  a.label64 = h->labels_dtype == DSLPG_I64 ? 1 : 0;
  a.scale = h->logit_scale;
  const double c = h->logit_scale * 1.4426950408889634074;  // log2(e)
  a.scale_f = static_cast<float>(h->logit_scale);
  a.sign = h->logit_scale < 0 ? -1.f : 1.f;
  a.c_hi = static_cast<float>(c);
  if (fabs(static_cast<double>(a.c_hi)) > fabs(c)) a.c_hi = nextafterf(a.c_hi, 0.f);
  a.c_lo = static_cast<float>(c - static_cast<double>(a.c_hi));
  if (a.c_lo == 0.f && a.c_hi != 0.f) a.c_lo = copysignf(1.17549435e-38f, a.c_hi);
  return DSLPG_OK;
}

int policy_args(PolicyTerms& p, const dslpg_policy_terms* h, int64_t rows) {
  if (!h) return DSLPG_ERR_NULL_POINTER;
  if (rows > 0 && (!h->old_logp || !h->advantages)) return DSLPG_ERR_NULL_POINTER;
  if (h->old_stride < 0 || h->advantages_stride < 0 || h->ref_stride < 0) return DSLPG_ERR_BAD_SHAPE;
  if (!(h->clip_low >= 0.f && h->clip_low <= 1.f) || !(h->clip_high >= 0.f) || !finite(h->kl_coef))
    return DSLPG_ERR_BAD_ARGUMENT;
  p.old_logp = h->old_logp;
  p.adv = h->advantages;
  p.ref = h->ref_logp;
  p.old_stride = h->old_stride;
  p.adv_stride = h->advantages_stride;
  p.ref_stride = h->ref_stride;
  p.lo = 1.f - h->clip_low;
  p.hi = 1.f + h->clip_high;
  p.kl_coef = h->kl_coef;
  return DSLPG_OK;
}

int pair_args(PairTerms& p, const dslpg_pair_terms* h, int64_t rows, bool fwd) {
  if (!h) return DSLPG_ERR_NULL_POINTER;
  if (h->starts_dtype != DSLPG_I32 && h->starts_dtype != DSLPG_I64) return DSLPG_ERR_BAD_DTYPE;
  if (h->n_pairs < 1 || h->n_pairs > (1ll << 30) || h->ref_stride < 0) return DSLPG_ERR_BAD_SHAPE;
  if (!h->seq_starts || (fwd && rows > 0 && !h->ref_logp)) return DSLPG_ERR_NULL_POINTER;
  if (!finite(h->beta) || !(h->smoothing >= 0.f && h->smoothing <= 1.f)) return DSLPG_ERR_BAD_ARGUMENT;
  p.starts = h->seq_starts;
  p.starts64 = h->starts_dtype == DSLPG_I64 ? 1 : 0;
  p.pairs = h->n_pairs;
  p.ref = h->ref_logp;
  p.ref_stride = h->ref_stride;
  p.beta = h->beta;
  p.smoothing = h->smoothing;
  return DSLPG_OK;
}

}  // namespace

}  // namespace dslpg

using namespace dslpg;

extern "C" int dslpg_policy_loss_fwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms, float* loss,
                                     float* logp, float* lse, float* kl, cudaStream_t stream) {
  LossRows a{};
  PolicyTerms p{};
  if (int rc = rows_args(a, rows)) return rc;
  if (int rc = policy_args(p, terms, a.M)) return rc;
  if (a.M == 0) return DSLPG_OK;
  if (!loss || !logp || !lse || !kl) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(
      dispatch<kPolicy>(kFwd, rows->logits_dtype, a, p, PairTerms{}, LossOut{loss, logp, lse, kl}, GradOut{}, stream));
}

extern "C" int dslpg_policy_loss_bwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms, const float* dloss,
                                     int64_t dloss_stride, const float* lse, void* dlogits, int64_t dlogits_row_stride,
                                     cudaStream_t stream) {
  LossRows a{};
  PolicyTerms p{};
  if (int rc = rows_args(a, rows)) return rc;
  if (int rc = policy_args(p, terms, a.M)) return rc;
  if (dloss_stride < 0 || dlogits_row_stride < a.N) return DSLPG_ERR_BAD_SHAPE;
  if (a.M == 0) return DSLPG_OK;
  if (!dloss || !lse || !dlogits) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch<kPolicy>(kBwd, rows->logits_dtype, a, p, PairTerms{}, LossOut{},
                                            GradOut{dloss, dloss_stride, lse, nullptr, dlogits, dlogits_row_stride},
                                            stream));
}

extern "C" int dslpg_policy_loss_fwd_bwd(const dslpg_logit_rows* rows, const dslpg_policy_terms* terms,
                                         const float* dloss, int64_t dloss_stride, float* loss, float* logp, float* lse,
                                         float* kl, void* dlogits, int64_t dlogits_row_stride, cudaStream_t stream) {
  LossRows a{};
  PolicyTerms p{};
  if (int rc = rows_args(a, rows)) return rc;
  if (int rc = policy_args(p, terms, a.M)) return rc;
  if (dloss_stride < 0 || dlogits_row_stride < a.N) return DSLPG_ERR_BAD_SHAPE;
  if (a.M == 0) return DSLPG_OK;
  if (!dloss || !loss || !logp || !lse || !kl || !dlogits) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch<kPolicy>(kFwdBwd, rows->logits_dtype, a, p, PairTerms{}, LossOut{loss, logp, lse, kl},
                                            GradOut{dloss, dloss_stride, nullptr, nullptr, dlogits, dlogits_row_stride},
                                            stream));
}

extern "C" int dslpg_preference_loss_fwd(const dslpg_logit_rows* rows, const dslpg_pair_terms* terms, float* loss,
                                         float* log_ratio, float* logp, float* lse, cudaStream_t stream) {
  LossRows a{};
  PairTerms p{};
  if (int rc = rows_args(a, rows)) return rc;
  if (int rc = pair_args(p, terms, a.M, true)) return rc;
  if (!loss || !log_ratio || (a.M > 0 && (!logp || !lse))) return DSLPG_ERR_NULL_POINTER;
  if (a.M > 0) {
    const cudaError_t e = dispatch<kPair>(kFwd, rows->logits_dtype, a, PolicyTerms{}, p,
                                          LossOut{nullptr, logp, lse, nullptr}, GradOut{}, stream);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  const int grid = static_cast<int>(p.pairs < 65535 ? p.pairs : 65535);
  return static_cast<int>(
      launch_dependent(pair_kernel, dim3(grid), 256, stream, a, p, static_cast<const float*>(logp), loss, log_ratio));
}

extern "C" int dslpg_preference_loss_bwd(const dslpg_logit_rows* rows, const dslpg_pair_terms* terms,
                                         const float* dloss, int64_t dloss_stride, const float* lse,
                                         const float* log_ratio, void* dlogits, int64_t dlogits_row_stride,
                                         cudaStream_t stream) {
  LossRows a{};
  PairTerms p{};
  if (int rc = rows_args(a, rows)) return rc;
  if (int rc = pair_args(p, terms, a.M, false)) return rc;
  if (dloss_stride < 0 || dlogits_row_stride < a.N) return DSLPG_ERR_BAD_SHAPE;
  if (a.M == 0) return DSLPG_OK;
  if (!dloss || !lse || !log_ratio || !dlogits) return DSLPG_ERR_NULL_POINTER;
  return static_cast<int>(dispatch<kPair>(kBwd, rows->logits_dtype, a, PolicyTerms{}, p, LossOut{},
                                          GradOut{dloss, dloss_stride, lse, log_ratio, dlogits, dlogits_row_stride},
                                          stream));
}
