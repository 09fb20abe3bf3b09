// Fine-tuning losses over logits, forward and gradient: the clipped policy
// loss with a KL term, and the preference loss over pairs of sequences.
//
// Both are functions of the target's log-probability in each row of logits,
//   lp = x[target] - max(x) - log(sum_j exp(x_j - max(x))),  j < V,
// with d(lp)/d(x_j) = [j = target] - softmax(x)_j, so the gradient of either
// loss is one coefficient c = d(loss)/d(lp) per row times that difference.
// Rows of weight zero (prompts, padding) take no part; their gradient is zero.
//
// Memory bounds both. The policy loss is independent from row to row, so one
// kernel (row_kernel) reads each row once, keeps it in shared memory while its
// sum forms, and writes the gradient from there: 16 x 1024 rows of 50257 bf16
// logits, half of them live, in 425 us, 5.8 TB/s of the 2.47 GB it cannot do
// without (a copy of the kernel without its arithmetic takes as long). The
// preference loss needs the sums over whole sequences before the first gradient:
// row_kernel leaves each row's (max, sum), preference_pair_kernel forms the
// losses and every row's coefficient, and row_gradient_kernel streams the logits
// a second time: 8 pairs of 1024 positions in 598 us, 5.5 TB/s of 3.30 GB. A few
// long rows take that second way for the policy loss too. Of two variants that a
// comment compares, both were measured with the rest of the kernel as it was then.
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "ptx.cuh"
#include "runtime.h"
#include "vec8.cuh"

namespace llmk {
namespace {

template <typename T>
constexpr int vec_elems() {  // elements of a 16-byte vector
  return 16 / static_cast<int>(sizeof(T));
}

// The maximum of a row, or of part of one, the sum of exp(x - max), and (whole
// rows) the target's logit. The sum is a double: what corrects it is less than
// half a step of fp32.
struct __align__(16) RowSum {
  double s;
  float m, xt;
};

// What the gradient of a row is made of.
struct __align__(16) RowCoef {
  float max;
  float scale;  // c / sum
  float c;      // d(loss) / d(lp), dscale included; 0: the row's gradient is 0
  int target;
};

__device__ __forceinline__ float warp_max_f(float v) {  // of the values that are not NaN
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The reference point of exp(x - m): a slice or row of nothing but -inf has
// sum 0 (or NaN, when it holds one), not exp(-inf + inf).
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.f : m; }

// A row's sum from its slots, given its target's logit (NaN for a target outside
// [0, V)). The loads do not wait for one another.
constexpr int kMaxParts = 16;
__device__ __forceinline__ RowSum fold_slots(const RowSum* __restrict__ slots, long long row, int rows, int nslots, float xt) {
  if (nslots == 1) {
    RowSum t = slots[row];
    t.xt = xt;
    return t;
  }
  RowSum p[kMaxParts];
#pragma unroll
  for (int k = 0; k < kMaxParts; ++k) p[k] = k < nslots ? slots[static_cast<long long>(k) * rows + row] : RowSum{0.0, -INFINITY, 0.f};
  float M = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMaxParts; ++k) M = fmaxf(M, p[k].m);
  const float ref = finite_max(M);
  double S = 0.0;
#pragma unroll
  for (int k = 0; k < kMaxParts; ++k) S += p[k].s * static_cast<double>(expf(p[k].m - ref));
  return RowSum{S, M, xt};
}
__device__ __forceinline__ double logp_of(const RowSum& t) {
  return static_cast<double>(t.xt) - static_cast<double>(t.m) - log(t.s);
}

// The policy loss of one live row. With rho = exp(lp - old), A the advantage and
// d = ref - lp: loss = w (-min(rho A, clamp(rho) A) + kl_coef (exp(d) - d - 1)).
// The clipped branch has no gradient; where both products are equal (rho inside
// the bounds, or on one) the unclipped one counts. In 64 bits: exp(d) - 1 and
// exp(d) - d - 1 are differences of nearly equal numbers for a policy close to
// its reference, and rho against a bound decides between two gradients.
struct PolicyRow {
  float adv, old, ref;
  int target;
};
__device__ __forceinline__ PolicyRow policy_row_load(const PolicyArgs& a, long long row) {
  PolicyRow r;
  r.adv = a.advantages[row];
  r.old = a.old_logps ? a.old_logps[row] : 0.f;
  r.ref = a.ref_logps ? a.ref_logps[row] : 0.f;
  r.target = a.targets[row];
  return r;
}
// -min(rho A, clamp(rho) A) and its derivative by lp. The loss and the gradient
// take rho = exp(xt - max - old) / sum from the same operations, so that they
// decide alike.
struct PolicyTerm {
  double loss, slope;
};
__device__ __forceinline__ PolicyTerm policy_term(const PolicyArgs& a, double A, double rho) {
  const double lo = 1.0 - static_cast<double>(a.clip_low), hi = 1.0 + static_cast<double>(a.clip_high);
  const double clamped = rho < lo ? lo : (rho > hi ? hi : rho);
  const double s1 = A == 0.0 ? 0.0 : rho * A, s2 = clamped * A;
  return s1 > s2 ? PolicyTerm{-s2, 0.0} : PolicyTerm{-s1, -s1};
}
__device__ __forceinline__ double target_offset(const RowSum& t) {  // lp + log(sum)
  return static_cast<double>(t.xt) - static_cast<double>(t.m);
}
// Writes the row's outputs and returns d(loss)/d(lp) with weight and dscale.
__device__ __forceinline__ double policy_row(const PolicyArgs& a, const PolicyRow& r, long long row, float w, const RowSum& t) {
  const double lp = logp_of(t);
  const double rho = a.old_logps ? exp(target_offset(t) - static_cast<double>(r.old)) * (1.0 / t.s) : 1.0;
  const PolicyTerm term = policy_term(a, r.adv, rho);
  double loss = term.loss, g = term.slope;
  if (isnan(lp)) loss = g = lp;  // also where rho does not carry it
  if (a.ref_logps) {
    const double d = static_cast<double>(r.ref) - lp;
    const double e = expm1(d);
    const double kl = isinf(e) ? e : e - d;
    if (a.kls) a.kls[row] = static_cast<float>(kl);
    if (a.kl_coef != 0.f) {
      loss += static_cast<double>(a.kl_coef) * kl;
      g -= static_cast<double>(a.kl_coef) * e;
    }
  }
  a.losses[row] = static_cast<float>(w * loss);
  if (a.logps) a.logps[row] = static_cast<float>(lp);
  return g * w * a.dscale;
}
// The coefficient alone, by a whole warp, while the row's other warps wait: no
// logarithm, since exp(d) = exp(ref - xt + max) sum, and one exponential for both
// terms, of lane 0 for rho and of the others for the KL term.
__device__ __forceinline__ double policy_coef(const PolicyArgs& a, const PolicyRow& r, float w, const RowSum& t, double inv_s, int lane) {
  const double x = target_offset(t);
  double rho = 1.0, e = 0.0;
  if (a.old_logps || a.kl_coef != 0.f) {
    const double v = exp(lane == 0 ? x - static_cast<double>(r.old) : static_cast<double>(r.ref) - x);
    if (a.old_logps) rho = __shfl_sync(0xffffffffu, v, 0) * inv_s;
    e = __shfl_sync(0xffffffffu, v, 1) * t.s - 1.0;
  }
  double g = policy_term(a, r.adv, rho).slope;
  if (a.kl_coef != 0.f) g -= static_cast<double>(a.kl_coef) * e;
  return isnan(x) || isnan(t.s) ? static_cast<double>(NAN) : g * w * a.dscale;
}
__device__ __forceinline__ void policy_row_masked(const PolicyArgs& a, long long row) {
  a.losses[row] = 0.f;
  if (a.kls) a.kls[row] = 0.f;
  if (a.logps) a.logps[row] = 0.f;
}

// One 16-byte vector.
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack_vec(const uint4& u, float (&v)[4]) {
  v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y); v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
}
template <typename T>
__device__ __forceinline__ float max_vec(const uint4& u, const uint4& w) {
  if constexpr (sizeof(T) == 2) {
    auto h = [](const uint32_t& v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    const __nv_bfloat162 m = __hmax2(__hmax2(__hmax2(h(u.x), h(u.y)), __hmax2(h(u.z), h(u.w))),
                                     __hmax2(__hmax2(h(w.x), h(w.y)), __hmax2(h(w.z), h(w.w))));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    auto f = [](uint32_t v) { return __uint_as_float(v); };
    return fmaxf(fmaxf(fmaxf(f(u.x), f(u.y)), fmaxf(f(u.z), f(u.w))), fmaxf(fmaxf(f(w.x), f(w.y)), fmaxf(f(w.z), f(w.w))));
  }
}
template <typename T>
__device__ __forceinline__ float max_vec(const uint4& u) {
  return max_vec<T>(u, u);
}
// The elements from `keep` on replaced by -inf.
template <typename T>
__device__ __forceinline__ uint4 cut_vec(const uint4& u, int keep) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 2) {
      if (2 * i >= keep) w[i] = 0xff80ff80u;
      else if (2 * i + 1 >= keep) w[i] = (w[i] & 0xffffu) | 0xff800000u;
    } else {
      if (i >= keep) w[i] = 0xff800000u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Sum of exp(x - ref) over a vector as a packed pair of sums; *first: its first
// element's term. The differences, products and sums run two to an instruction.
template <typename T>
__device__ __forceinline__ uint64_t sum_exp_vec(const uint4& u, uint64_t neg_ref, float* first) {
  constexpr int kP = vec_elems<T>() / 2;
  const uint64_t l = f2_pack(kLog2e, kLog2e);
  float v[2 * kP];
  unpack_vec(u, v);
  uint64_t e[kP];
#pragma unroll
  for (int j = 0; j < kP; ++j) {
    float a, b;
    f2_unpack(f2_mul(f2_add(f2_pack(v[2 * j], v[2 * j + 1]), neg_ref), l), a, b);
    a = ex2_approx(a), b = ex2_approx(b);
    if (j == 0) *first = a;
    e[j] = f2_pack(a, b);
  }
#pragma unroll
  for (int n = kP / 2; n > 0; n >>= 1)
#pragma unroll
    for (int j = 0; j < n; ++j) e[j] = f2_add(e[j], e[j + n]);
  return e[0];
}
template <typename T>
__device__ __forceinline__ float first_elem(const uint4& u) {
  return __uint_as_float(sizeof(T) == 2 ? u.x << 16 : u.x);
}

// A warp's running maximum and sum of exp(x - m). m starts as the maximum over
// the warp's first vectors and, in a lane, follows a value more than 10 above it:
// the terms stay far inside fp32's range, and a lane that raises m is rare (at
// every new maximum: evaluation of 8 x 1024 rows 137 against 131 us).
// ex2.approx is 5e-8 low on average (measured), and the fp32 product by log2 e
// moves a term by its distance from m times 1.3e-8. A sum over a vocabulary keeps
// the mean of that while the rounding errors cancel, and a preference loss adds
// such sums over a thousand positions. Two things hold that mean at 1.2e-8 of a
// row's log-probability, for logits spread by 0.1 to 4 and for one that stands 2
// to 15 above the others, in vocabularies of 1000 to 50257. The row's maximum is
// taken out of its lane's sum at the end and counts exactly 1 (7e-8 with it left
// in, where it stands out). And one term in 8 to 32 is also computed by expf, and
// the sum of the others is corrected by what those terms differ by (1.9e-8
// without; evaluation 131 against 126 us, the gradient 425 against 431 us). The
// terms on the FMA units instead, by a polynomial, are as exact but slower: 185
// against 174 us (evaluation at that time) with an eighth of them there.
struct WarpSum {
  float top, m, s;
  float part, off;  // the terms computed twice: their sum, and what it lacks
};
struct RunningSum {
  float top = -INFINITY, m = -INFINITY, m0 = -INFINITY;
  uint64_t s = 0;  // two sums
  float part = 0.f, off = 0.f;
  __device__ __forceinline__ void start(float vm) { m = m0 = warp_max_f(vm); }
  __device__ __forceinline__ float raise(float vm) {
    top = fmaxf(top, vm);
    if (!(vm <= m + 10.f)) {
      const float f = expf(m - vm);
      s = f2_mul(s, f2_pack(f, f)), part *= f, off *= f;
      m = vm;
    }
    return finite_max(m);
  }
  __device__ __forceinline__ void twice(float x, float ref, float e) {
    part += e;
    off += expf(x - ref) - e;
  }
  template <typename T>
  __device__ __forceinline__ void add(const uint4& u) {
    const float ref = raise(max_vec<T>(u));
    const uint64_t r = f2_pack(-ref, -ref);
    float e;
    s = f2_add(s, sum_exp_vec<T>(u, r, &e));
    twice(first_elem<T>(u), ref, e);
  }
  template <typename T>
  __device__ __forceinline__ void add(const uint4& u, const uint4& w) {
    const float ref = raise(max_vec<T>(u, w));
    const uint64_t r = f2_pack(-ref, -ref);
    float e, unused;
    s = f2_add(s, f2_add(sum_exp_vec<T>(u, r, &e), sum_exp_vec<T>(w, r, &unused)));
    twice(first_elem<T>(u), ref, e);
  }
  template <typename T>
  __device__ __forceinline__ void add(const uint4& a, const uint4& b, const uint4& c, const uint4& d) {
    const float ref = raise(fmaxf(max_vec<T>(a, b), max_vec<T>(c, d)));
    const uint64_t r = f2_pack(-ref, -ref);
    float e, unused;
    s = f2_add(s, f2_add(f2_add(sum_exp_vec<T>(a, r, &e), sum_exp_vec<T>(b, r, &unused)),
                         f2_add(sum_exp_vec<T>(c, r, &unused), sum_exp_vec<T>(d, r, &unused))));
    twice(first_elem<T>(a), ref, e);
  }
  // The warp's vectors x[0, full), and x[full] cut after `keep` elements when
  // there is one. kWide: four vectors a step, where the registers are there for it.
  template <typename T, bool kWide>
  __device__ __forceinline__ void add_all(const uint4* x, int full, bool partial, int keep, int lane) {
    int i = lane;
    if constexpr (kWide)
      for (; i + 96 < full; i += 128) add<T>(x[i], x[i + 32], x[i + 64], x[i + 96]);
    for (; i + 32 < full; i += 64) add<T>(x[i], x[i + 32]);
    if (i < full) add<T>(x[i]);
    if (partial && lane == 0) add<T>(cut_vec<T>(x[full], keep));
  }
  // The warp's sums, at one m, without the term of its maximum: a value up to 10
  // above m had it off by up to 2e-7, while it is exp(top - m) to be joined.
  __device__ __forceinline__ WarpSum join(int lane) const {
    float s0, s1;
    f2_unpack(s, s0, s1);
    WarpSum w{warp_max_f(top), m0, s0 + s1, part, off};
    const unsigned holders = __ballot_sync(0xffffffffu, top == w.top);
    if (lane == __ffs(holders) - 1) w.s -= ex2_approx((top - finite_max(m)) * kLog2e);  // as sum_exp_vec has it
    if (__any_sync(0xffffffffu, m != m0)) {  // also where m is NaN
      w.m = warp_max_f(m);
      const float f = expf(m - finite_max(w.m));
      w.s *= f, w.part *= f, w.off *= f;
    }
    w.s = warp_sum_f(w.s), w.part = warp_sum_f(w.part), w.off = warp_sum_f(w.off);
    return w;
  }
};

// The same over a warp's only chunk by expf, added in 64 bits, with nothing to
// correct: `off` is what `s` rounds away, `part` 0.
template <typename T>
__device__ __forceinline__ WarpSum exact_sum(const uint4* x, int full, bool partial, int keep, int lane) {
  float top = -INFINITY;
  for (int i = lane; i < full; i += 32) top = fmaxf(top, max_vec<T>(x[i]));
  if (partial && lane == 0) top = fmaxf(top, max_vec<T>(cut_vec<T>(x[full], keep)));
  top = warp_max_f(top);
  const float ref = finite_max(top);
  double s = 0.0;
  auto add = [&](const uint4& u) {
    float v[vec_elems<T>()];
    unpack_vec(u, v);
#pragma unroll
    for (int j = 0; j < vec_elems<T>(); ++j) s += static_cast<double>(expf(v[j] - ref));
  };
  for (int i = lane; i < full; i += 32) add(x[i]);
  if (partial && lane == 0) add(cut_vec<T>(x[full], keep));
  s = warp_sum_d(s);
  const float high = static_cast<float>(s);
  return WarpSum{top, top, high, 0.f, static_cast<float>(s - static_cast<double>(high))};
}

// A row's sum at its maximum M: `tops` terms that are exactly 1, and the sum of all
// others from terms of ex2.approx. `off / part` is what those lack; expf itself is
// 6e-9 high on average, in the terms computed twice and in the warps' factors. No
// term up to 25 below the reference is off by more than 5e-7; a larger quotient
// comes from terms that are next to nothing (where ex2.approx flushes to zero and
// expf does not) and says nothing about the others.
__device__ __forceinline__ RowSum corrected(float M, int tops, float sum, float part, float off) {
  const double s = sum, lack = fminf(fmaxf(off / part, -2e-6f), 2e-6f);
  return RowSum{tops + (part > 0.f ? s + s * (lack - 1.2e-8) : s), M, 0.f};
}
// A row's sum from one warp's, or from several (lanes >= count: none); the same
// in every lane.
__device__ __forceinline__ RowSum fold_exact(const WarpSum* sums, int count, int lane) {
  WarpSum w{-INFINITY, -INFINITY, 0.f, 0.f, 0.f};
  if (lane < count) w = sums[lane];
  const float M = warp_max_f(w.top);
  const double f = exp(static_cast<double>(w.top) - static_cast<double>(finite_max(M)));
  return RowSum{warp_sum_d((static_cast<double>(w.s) + static_cast<double>(w.off)) * f), M, 0.f};
}
__device__ __forceinline__ RowSum fold_warp(const WarpSum& w) {
  const float f = expf(w.m - finite_max(w.top));
  return corrected(w.top, w.top == -INFINITY ? 0 : 1, w.s * f, w.part, w.off);
}
__device__ __forceinline__ RowSum fold_warps(const WarpSum* sums, int count, int lane) {
  WarpSum w{-INFINITY, -INFINITY, 0.f, 0.f, 0.f};
  if (lane < count) w = sums[lane];
  const float M = warp_max_f(w.top);
  const float f = expf(w.m - finite_max(M));
  const int tops = M == -INFINITY ? 0 : __popc(__ballot_sync(0xffffffffu, w.top == M));
  const float others = w.top == M ? 0.f : expf(w.top - M);
  const float S = warp_sum_f(w.s * f + others), P = warp_sum_f(w.part * f), D = warp_sum_f(w.off * f);
  return corrected(M, tops, S, P, D);
}

// -exp(x - max) scale over a vector: the gradient everywhere but at the target.
template <typename T>
struct RowGradient {
  float max, scale;
  float k;  // 16-bit output: log2 |scale|, folded into the exponent
  __device__ __forceinline__ explicit RowGradient(const RowCoef& c) : max(c.max), scale(c.scale), k(0.f) {
    if constexpr (sizeof(T) == 2) k = log2f(fabsf(scale));
  }
  // kMode, 16-bit output: 0 any row; 1 and 2 rows of |max| < 512 and of positive
  // or negative scale, where x log2 e - max log2 e in one rounding is off by at
  // most 2^-14 relative, far inside the 2^-8 the result is rounded by.
  template <int kMode>
  __device__ __forceinline__ uint4 of(const uint4& u) const {
    constexpr int kV = vec_elems<T>();
    float v[kV];
    unpack_vec(u, v);
    if constexpr (sizeof(T) == 2) {
      const float c = fmaf(-max, kLog2e, k);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint64_t x = f2_pack(v[2 * i], v[2 * i + 1]);
        if (kMode == 0) x = f2_add(x, f2_pack(-max, -max));
        float a[2];
        f2_unpack(f2_fma(x, f2_pack(kLog2e, kLog2e), kMode ? f2_pack(c, c) : f2_pack(k, k)), a[0], a[1]);
        a[0] = ex2_approx(a[0]), a[1] = ex2_approx(a[1]);
        if (kMode == 2 || (kMode == 0 && !(scale > 0.f))) w[i] = pack_bf16x2(a[0], a[1]);
        else w[i] = pack_bf16x2(-a[0], -a[1]);
      }
      return make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      const uint64_t m = f2_pack(-max, -max), l = f2_pack(kLog2e, kLog2e), sc = f2_pack(-scale, -scale);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        float a, b;
        f2_unpack(f2_mul(f2_add(f2_pack(v[j], v[j + 1]), m), l), a, b);
        f2_unpack(f2_mul(f2_pack(ex2_approx(a), ex2_approx(b)), sc), v[j], v[j + 1]);
      }
      return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    }
  }
  template <int kMode>
  __device__ __forceinline__ void store_full(uint4* d, const uint4* x, int full, int lane) const {
    int i = lane;
    for (; i + 32 < full; i += 64) {
      const uint4 a = x[i], b = x[i + 32];
      d[i] = of<kMode>(a);
      d[i + 32] = of<kMode>(b);
    }
    if (i < full) d[i] = of<kMode>(x[i]);
  }
  // `n` vectors of a row, the first of them number v0, by one warp; the row's
  // last, partly live vector gets zeros in its padding.
  __device__ __forceinline__ void store(T* row, const uint4* x, int v0, int n, int V, int lane) const {
    uint4* d = reinterpret_cast<uint4*>(row) + v0;
    const int full = min(n, V / vec_elems<T>() - v0);
    if (sizeof(T) == 2 && fabsf(max) < 512.f) {
      if (scale > 0.f) store_full<1>(d, x, full, lane);
      else store_full<2>(d, x, full, lane);
    } else {
      store_full<0>(d, x, full, lane);
    }
    if (full < n && lane == 0) {
      const uint4 o = of<0>(x[full]);
      uint32_t w[4] = {o.x, o.y, o.z, o.w};
      const int keep = V % vec_elems<T>();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 2) w[j] &= 2 * j >= keep ? 0u : (2 * j + 1 >= keep ? 0x0000ffffu : 0xffffffffu);
        else w[j] &= j >= keep ? 0u : 0xffffffffu;
      }
      d[full] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  __device__ __forceinline__ float at_target(float x, float c) const { return c - expf(x - max) * scale; }
};

// Zeros over 16-byte vectors.
__device__ __forceinline__ void zero_vecs(void* d, int n, int thread, int threads) {
  for (int i = thread; i < n; i += threads) static_cast<uint4*>(d)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// A warp's own ring of chunks in shared memory. Lane 0 issues the bulk copies;
// the warp that reads a chunk is the one that gives its place to the next copy,
// so a __syncwarp is all the hand-over there is.
constexpr int kMaxStages = 8;
struct WarpRing {
  uint8_t* base;
  uint64_t* bars;
  int stages, stage_bytes;
  int in = 0, out = 0, loading = 0;
  uint32_t out_phase = 0;
  unsigned int* status;
  volatile int* abort_flag;
  __device__ __forceinline__ void load(const void* src, int bytes, int lane) {
    if (lane == 0) {
      mbar_arrive_expect_tx(bars + in, bytes);
      bulk_load_1d(base + static_cast<size_t>(in) * stage_bytes, src, bytes, bars + in);
    }
    if (++in == stages) in = 0;
    ++loading;
  }
  // Waits for the next chunk; false when the wait was given up.
  __device__ __forceinline__ bool wait(int site) {
    return __all_sync(0xffffffffu, mbar_wait(bars + out, out_phase, status, abort_flag, site));
  }
  __device__ __forceinline__ const uint4* chunk() const {
    return reinterpret_cast<const uint4*>(base + static_cast<size_t>(out) * stage_bytes);
  }
  __device__ __forceinline__ void step() {
    --loading;
    if (++out == stages) out = 0, out_phase ^= 1u;
  }
  // After a wait that was given up: every copy under way lands before the warp
  // leaves.
  __device__ __forceinline__ void drain() {
    for (; loading > 0; step()) mbar_wait(bars + out, out_phase, status, nullptr, 7);
  }
};

// A place in a grid of items x parts, walked with a fixed stride: no division on
// the way.
struct UnitWalk {
  int item, part;
  int items, parts, step_part, step_item;
  __device__ __forceinline__ UnitWalk(int first, int stride, int items_, int parts_)
      : item(first / parts_), part(first % parts_), items(items_), parts(parts_), step_part(stride % parts_),
        step_item(stride / parts_) {}
  __device__ __forceinline__ bool valid() const { return item < items; }
  __device__ __forceinline__ void next() {
    item += step_item;
    part += step_part;
    if (part >= parts) part -= parts, ++item;
  }
};

// A CTA's units, those of live rows and those of masked ones apart.
constexpr int kMaxItems = 2048;  // units of one CTA in one launch
constexpr int kRowWarps = 24;
constexpr int kRowThreads = 32 * kRowWarps;
struct RowList {
  uint16_t items[kMaxItems];  // the live ones from the front, the masked ones from the back
  uint8_t masked[kMaxItems];
  int count;
  // Called by the whole CTA with its n rows' flags; returns the number of live
  // ones. Up to 32 rows every warp sorts for itself, and nobody waits.
  template <typename F>
  __device__ __forceinline__ int sort(int n, F is_masked) {
    if (n <= 32) {
      const int lane = threadIdx.x & 31;
      const bool is_live = lane < n && !is_masked(lane);
      const unsigned all = __ballot_sync(0xffffffffu, is_live);
      const int at = __popc(all & ((1u << lane) - 1u));
      if (is_live) items[at] = static_cast<uint16_t>(lane);  // the same values from every warp
      else if (lane < n) items[n - 1 - (lane - at)] = static_cast<uint16_t>(lane);
      __syncwarp();
      return __popc(all);
    }
    for (int i = threadIdx.x; i < n; i += kRowThreads) masked[i] = is_masked(i);
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int k = 0;
      for (int i0 = 0; i0 < n; i0 += 32) {
        const int i = i0 + lane;
        const bool is_live = i < n && !masked[i];
        const unsigned all = __ballot_sync(0xffffffffu, is_live);
        const int at = k + __popc(all & ((1u << lane) - 1u));
        if (is_live) items[at] = static_cast<uint16_t>(i);
        else if (i < n) items[n - 1 - (i - at)] = static_cast<uint16_t>(i);
        k += __popc(all);
      }
      if (lane == 0) count = k;
    }
    __syncthreads();
    return count;
  }
  __device__ __forceinline__ int live(int i) const { return items[i]; }
  __device__ __forceinline__ int dead(int i, int n) const { return items[n - 1 - i]; }
};

// kRowLong: kRowGrad for rows that do not fit their group's rings.
enum RowMode { kRowGrad, kRowLong, kRowEval, kRowStats };

// How row_kernel shares the work out. A unit is a row, or (kRowStats) one of
// `parts` parts of it, of `vecs` vectors, summed by expf (`exact`) or by
// ex2.approx; a launch covers units [unit0, unit1) of
// rows * parts, CTA b those at unit0 + b, unit0 + b + grid, ...; `group` warps
// take a unit, each `seg` vectors of it, through its ring in chunks of `sub`.
struct RowJob {
  RowSum* slots;
  const float* weights;
  int rows, V, ld;
  unsigned unit0, unit1;
  int parts, vecs, group, seg, sub, stages;
  bool exact;
  unsigned int* status;
};

// One pass over the rows, one persistent CTA of 24 warps per SM (16 warps: 465
// against 455 us at 16 x 1024 rows, evaluation 227 against 206 us; a copy warp
// and a scalar warp beside 16 consumer warps, a barrier per 8 KB chunk: 582 and
// 312 us). Groups of warps take one row each: pass A waits for the warp's chunks
// as they arrive and folds them into its running sum; the group's first warp
// joins the sums and forms the row's coefficient; in kRowGrad the chunks stay in
// shared memory until pass B has written the gradient from them, so the logits
// are read from memory once, and each chunk's place is then refilled with the
// group's next row. In kRowLong the first chunks give up their places in pass A
// and come again, from L2 (148 rows are on their way), after the ones that stayed:
// 4096 rows of 131072, half live, in 312 us; by two kernels over all rows 406.
// Masked rows take no chunk. Each unit's (max, sum) goes to its
// slot, planes of `rows`. A wait that is given up (the device status says so)
// ends the work, not the barriers: the group's warps still meet.
template <typename T, int kMode, bool kExact>
__global__ void __launch_bounds__(kRowThreads, 1) row_kernel(T* dlogits, const T* logits, RowJob job, PolicyArgs args) {
  constexpr int kV = vec_elems<T>();
  constexpr bool kGrad = kMode == kRowGrad || kMode == kRowLong;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRowWarps * kMaxStages];
  __shared__ WarpSum sums[2][kRowWarps];
  __shared__ RowCoef coef[kRowWarps];
  __shared__ RowList todo;
  __shared__ int abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (kMode == kRowStats) grid_release();
  const unsigned first = job.unit0 + blockIdx.x;
  const int n_items = static_cast<int>((job.unit1 - first + gridDim.x - 1) / gridDim.x);
  auto unit_of = [&](int item) { return first + static_cast<unsigned>(item) * gridDim.x; };
  auto row_of = [&](int item) {
    const unsigned u = unit_of(item);
    return static_cast<long long>(kMode == kRowStats && job.parts > 1 ? u / static_cast<unsigned>(job.parts) : u);
  };
  auto part_of = [&](int item) {
    return kMode == kRowStats && job.parts > 1 ? static_cast<int>(unit_of(item) % static_cast<unsigned>(job.parts)) : 0;
  };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRowWarps * kMaxStages; ++i) mbar_init(bars + i, 1);
    abort_word = 0;
    fence_mbar_init();
  }
  const int live = todo.sort(n_items, [&](int i) { return job.weights && job.weights[row_of(i)] == 0.f; });
  __syncthreads();
  const int G = job.group, group = warp / G, gw = warp - group * G;
  const int groups = kRowWarps / G;
  auto meet = [&] {
    if (G == 1) __syncwarp();
    else named_barrier_sync(1 + group, G * 32);
  };
  WarpRing ring{smem + static_cast<size_t>(warp) * job.stages * job.sub * 16, bars + warp * kMaxStages, job.stages,
                job.sub * 16};
  ring.status = job.status;
  ring.abort_flag = &abort_word;
  const int row_vecs = (job.V + kV - 1) / kV;
  // this warp's vectors of part `part` of a row: the first one's number in the
  // row, and how many
  auto my_first = [&](int part) { return part * job.vecs + gw * job.seg; };
  auto my_count = [&](int part) {
    return max(0, min(job.seg, min(job.vecs, row_vecs - part * job.vecs) - gw * job.seg));
  };

  // Vectors of a segment of n that pass B finds no more in the ring.
  auto lost = [&](int n) { return max(0, (n + job.sub - 1) / job.sub - job.stages) * job.sub; };

  // The copies run ahead of the work by what the ring holds: `ahead` is the
  // live item they are at, `done` of its `count` vectors are loaded or on their
  // way, and the first `again` are to be loaded a second time.
  int ahead = group, done = 0, count = 0, again = 0;
  const uint4* src = nullptr;
  auto open_ahead = [&] {
    if (ahead >= live) return;
    const int item = todo.live(ahead), part = part_of(item);
    done = 0;
    count = my_count(part);
    if (kMode == kRowLong) again = lost(count);
    src = reinterpret_cast<const uint4*>(logits + row_of(item) * job.ld) + my_first(part);
  };
  open_ahead();
  auto load_next = [&] {
    while (ahead < live && done >= count) {
      if (kMode == kRowLong && again > 0) done = 0, count = again, again = 0;
      else ahead += groups, open_ahead();
    }
    if (ahead >= live) return;
    ring.load(src + done, min(job.sub, count - done) * 16, lane);
    done += job.sub;
  };
  for (int i = 0; i < job.stages; ++i) load_next();

  // Masked rows are written between the live ones, in proportion: reads and
  // writes stay mixed.
  int zeroed = group;
  auto zero_rows = [&](int up_to) {
    for (; zeroed < min(up_to, n_items - live); zeroed += groups)
      zero_vecs(dlogits + row_of(todo.dead(zeroed, n_items)) * job.ld, job.ld / kV, gw * 32 + lane, G * 32);
  };
  const float per_live = live > 0 ? static_cast<float>(n_items - live) / static_cast<float>(live) : 0.f;

  bool ok = true;
  int k = 0;  // units so far
  for (int at = group; at < live; at += groups) {
    const int part = part_of(todo.live(at));
    const long long row = row_of(todo.live(at));
    const int v0 = my_first(part), n = my_count(part);
    PolicyRow r{};
    float xt = 0.f, weight = 1.f;
    if (kMode != kRowStats && gw == 0) {  // ahead of their use
      r = policy_row_load(args, row);
      if (job.weights) weight = job.weights[row];
      xt = r.target >= 0 && r.target < job.V ? elem_to_float(logits[row * job.ld + r.target]) : NAN;
    }
    RunningSum run;
    WarpSum sum{-INFINITY, -INFINITY, 0.f, 0.f, 0.f};
    const int gone = kMode == kRowGrad ? 0 : (kMode == kRowLong ? lost(n) : n);  // what lies before is given up as it is read
    int out0 = ring.out, loading0 = ring.loading;
    uint32_t phase0 = ring.out_phase;
    for (int c = 0; c < n; c += job.sub) {
      if (kMode == kRowLong && c == gone) out0 = ring.out, phase0 = ring.out_phase, loading0 = ring.loading;
      ok = ok && ring.wait(4);
      const int nc = min(job.sub, n - c);
      if (!ok) break;
      const uint4* x = ring.chunk();
      const int full = min(nc, job.V / kV - v0 - c);
      if constexpr (kExact) {
        sum = exact_sum<T>(x, full, full < nc, job.V % kV, lane);
      } else {
        if (c == 0) run.start(lane < full ? max_vec<T>(x[lane]) : -INFINITY);
        run.add_all<T, !kGrad || sizeof(T) == 4>(x, full, full < nc, job.V % kV, lane);
      }
      ring.step();
      if (c < gone) {
        __syncwarp();
        load_next();
      }
    }
    if constexpr (!kExact) sum = run.join(lane);
    // Two sets of sums: a set is rewritten two rows on, and between lies a
    // meeting that the group's first warp reaches only after reading it.
    if (G > 1 || kExact) {
      if (lane == 0) sums[k & 1][warp] = sum;
      meet();
    }
    if (gw == 0) {
      RowSum t = kExact ? fold_exact(&sums[k & 1][warp], G, lane)
                           : (G > 1 ? fold_warps(&sums[k & 1][warp], G, lane) : fold_warp(sum));
      t.xt = xt;
      if (lane == 0) job.slots[static_cast<long long>(part) * job.rows + row] = t;
      if (kGrad) {
        const double inv_s = 1.0 / t.s, c = policy_coef(args, r, weight, t, inv_s, lane);
        if (lane == 0) coef[warp] = RowCoef{finite_max(t.m), static_cast<float>(c * inv_s), static_cast<float>(c), r.target};
      }
    }
    ++k;
    if (kGrad) {
      meet();
      const RowCoef rc = coef[group * G];
      T* d = dlogits + row * job.ld;
      // back over the same chunks, then over those that come again
      if (ok) ring.out = out0, ring.out_phase = phase0, ring.loading = loading0;
      const int kept = kMode == kRowLong ? (n + job.sub - 1) / job.sub * job.sub - gone : n;
      if (ok && rc.c == 0.f) {
        zero_vecs(reinterpret_cast<uint4*>(d) + v0, n, lane, 32);
        for (int i = 0; i < n; i += job.sub) {
          if (kMode == kRowLong) {
            if (i >= kept) ok = ok && ring.wait(5);
            if (!ok) break;
          }
          ring.step();
          load_next();
        }
      } else if (ok) {
        const RowGradient<T> g(rc);
        float value = 0.f;  // the gradient at the target
        bool target_here = false;
        for (int i = 0; i < n; i += job.sub) {
          const int c = kMode == kRowGrad ? i : (i < kept ? gone + i : i - kept);
          if (kMode == kRowLong) {
            if (i >= kept) ok = ok && ring.wait(5);
            if (!ok) break;
          }
          const int nc = min(job.sub, n - c);
          g.store(d, ring.chunk(), v0 + c, nc, job.V, lane);
          const int t = rc.target - (v0 + c) * kV;
          if (t >= 0 && t < nc * kV && rc.target < job.V) {
            target_here = true;
            value = g.at_target(elem_to_float(reinterpret_cast<const T*>(ring.chunk())[t]), rc.c);
          }
          ring.step();
          __syncwarp();
          load_next();
        }
        if (target_here && lane == 0) elem_store(d + rc.target, value);
      }
      if (gw == G - 1) zero_vecs(reinterpret_cast<uint4*>(d) + row_vecs, job.ld / kV - row_vecs, lane, 32);
      zero_rows(static_cast<int>(static_cast<float>(at + 1) * per_live));
    }
  }
  if (kGrad) zero_rows(n_items);
  ring.drain();
  if (kMode == kRowStats) return;
  // The losses of this CTA's rows, in 64 bits, a row a thread: beside the passes
  // they would hold up a group for 2000 cycles a row.
  __syncthreads();
  for (int i = threadIdx.x; i < n_items; i += kRowThreads) {
    const long long row = row_of(i);
    const float weight = job.weights ? job.weights[row] : 1.f;
    const RowSum t = job.slots[row];  // all loads at once, for nothing in masked rows
    const PolicyRow r = policy_row_load(args, row);
    if (weight == 0.f) policy_row_masked(args, row);
    else policy_row(args, r, row, weight, t);
  }
}

// The policy loss from slots, one thread a row.
template <typename T>
__global__ void __launch_bounds__(128) policy_rows_kernel(RowCoef* __restrict__ coefs, const RowSum* __restrict__ slots,
                                                          const T* __restrict__ logits, PolicyArgs a, int rows, int V,
                                                          int ld, int nslots) {
  grid_release();
  grid_wait();
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const float w = a.weights ? a.weights[row] : 1.f;
  const PolicyRow r = policy_row_load(a, row);
  const RowSum t = fold_slots(slots, row, rows, nslots,
                              r.target >= 0 && r.target < V ? elem_to_float(logits[row * ld + r.target]) : NAN);
  if (w == 0.f) {
    policy_row_masked(a, row);
    if (coefs) coefs[row] = RowCoef{0.f, 0.f, 0.f, -1};
    return;
  }
  const double c = policy_row(a, r, row, w, t);
  if (coefs) coefs[row] = RowCoef{finite_max(t.m), static_cast<float>(c / t.s), static_cast<float>(c), r.target};
}

// The preference loss from slots, one CTA per pair p (sequence p is the chosen
// one, pairs + p the rejected one): L = sum_t w lp over each sequence, h =
// beta ((L_c - R_c) - (L_r - R_r)), loss = (1 - e) log(1 + exp(-h)) + e log(1 +
// exp(h)). The sums run in a fixed order in 64 bits.
// kEarly: the kernel before only writes slots and began after all before it (a
// plain launch), so that this one may read its other inputs while that one runs
// (8 pairs of 1024: 602 -> 598 us, 2 of 64: 21.9 -> 20.8 us).
constexpr int kPairThreads = 1024;
template <typename T, bool kEarly>
__global__ void __launch_bounds__(kPairThreads) preference_pair_kernel(RowCoef* __restrict__ coefs,
                                                                       RowSum* __restrict__ slots,
                                                                       const T* __restrict__ logits, PreferenceArgs a,
                                                                       int pairs, int Tlen, int V, int ld, int nslots) {
  constexpr int kSide = kPairThreads / 2;  // threads of a sequence
  __shared__ double red[2][kSide / 32];
  grid_release();
  const int pair = blockIdx.x, rows = 2 * pairs * Tlen;
  const int lane = threadIdx.x & 31, side = threadIdx.x / kSide, first = threadIdx.x % kSide;
  const long long row0 = static_cast<long long>(side * pairs + pair) * Tlen;
  float w = 0.f, xt = NAN;
  int target = -1;
  auto fetch = [&](int t) {
    if (t >= Tlen) return;
    w = a.weights ? a.weights[row0 + t] : 1.f;
    target = a.targets[row0 + t];
    xt = target >= 0 && target < V ? elem_to_float(logits[(row0 + t) * ld + target]) : NAN;
  };
  if (kEarly) fetch(first);
  grid_wait();
  // before the barrier that the outputs come after: rewards may be ref_logps, and
  // so may logps where a sequence is one row (elsewhere their sizes differ)
  const float ref0 = a.ref_logps ? a.ref_logps[pair] : 0.f, ref1 = a.ref_logps ? a.ref_logps[pairs + pair] : 0.f;
  double sum = 0.0;
  RowCoef mine{0.f, 0.f, 0.f, -1};  // of the thread's first row; the others' wait in memory
  float logp = 0.f;                 // as well
  for (int t = first; t < Tlen; t += kSide) {
    const long long row = row0 + t;
    if (!kEarly || t != first) fetch(t);
    const RowSum f = fold_slots(slots, row, rows, nslots, xt);
    const double lp = w != 0.f ? logp_of(f) : 0.0;
    if (w != 0.f) sum += static_cast<double>(w) * lp;
    const RowCoef c{finite_max(f.m), static_cast<float>(1.0 / f.s), w, target};
    if (t == first) {
      mine = c;
      logp = static_cast<float>(lp);
    } else {
      if (coefs) coefs[row] = c;
      if (a.logps) a.logps[row] = static_cast<float>(lp);
    }
  }
  sum = warp_sum_d(sum);
  if (lane == 0) red[side][first / 32] = sum;
  __syncthreads();
  if (a.logps && first < Tlen) a.logps[row0 + first] = logp;
  const double L0 = warp_sum_d(lane < kSide / 32 ? red[0][lane] : 0.0), L1 = warp_sum_d(lane < kSide / 32 ? red[1][lane] : 0.0);
  const double beta = a.beta, eps = a.smoothing;
  const double rc = beta * (L0 - static_cast<double>(ref0)), rr = beta * (L1 - static_cast<double>(ref1));
  const double h = rc - rr;
  // log(1 + exp(+-h)) and both sigmoids from exp(-|h|), which does not overflow
  const double e = exp(-fabs(h));
  if (threadIdx.x == kPairThreads - 1) {  // of a warp that seldom has rows
    const double t = log1p(e), up = (h > 0.0 ? h : 0.0) + t, down = (h < 0.0 ? -h : 0.0) + t;
    a.losses[pair] = static_cast<float>(isnan(h) ? h : (1.0 - eps) * down + (eps != 0.0 ? eps * up : 0.0));
    if (a.rewards) {
      a.rewards[pair] = static_cast<float>(rc);
      a.rewards[pairs + pair] = static_cast<float>(rr);
    }
  }
  if (!coefs) return;
  const double near = 1.0 / (1.0 + e), far = e * near;  // the sigmoids of |h| and -|h|
  const double slope = beta * static_cast<double>(a.dscale) * (h > 0.0 ? eps * near - (1.0 - eps) * far : eps * far - (1.0 - eps) * near);
  for (int t = first; t < Tlen; t += kSide) {
    RowCoef c = t == first ? mine : coefs[row0 + t];
    if (c.c == 0.f) {
      c = RowCoef{0.f, 0.f, 0.f, -1};
    } else {
      c.c = static_cast<float>((side ? -slope : slope) * c.c);
      c.scale *= c.c;
    }
    coefs[row0 + t] = c;
  }
}

// The gradient from each row's coefficient: a persistent pass, each warp taking
// units of up to `sub` vectors of a row through its own ring. Neighbouring CTAs
// take neighbouring units, so that the whole GPU works on one stretch of memory
// at a time (units by rows of a CTA's own: 442 against 429 us). Rows of
// coefficient 0 are written without being read. Last rows first: the pass before
// has left those in L2. dlogits may be the logits: a unit is read whole before
// any of it is written, and by its own warp only.
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 1) row_gradient_kernel(T* dlogits, const T* logits,
                                                                      const RowCoef* __restrict__ coefs, int rows, int V,
                                                                      int ld, int sub, int stages, unsigned int* status) {
  constexpr int kV = vec_elems<T>();
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kRowWarps * kMaxStages];
  __shared__ int abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRowWarps * kMaxStages; ++i) mbar_init(bars + i, 1);
    abort_word = 0;
    fence_mbar_init();
  }
  __syncthreads();
  grid_wait();
  WarpRing ring{smem + static_cast<size_t>(warp) * stages * sub * 16, bars + warp * kMaxStages, stages, sub * 16};
  ring.status = status;
  ring.abort_flag = &abort_word;
  const int row_vecs = ld / kV;
  UnitWalk at(warp * gridDim.x + blockIdx.x, gridDim.x * kRowWarps, rows, (row_vecs + sub - 1) / sub);
  UnitWalk ahead = at;
  auto row_of = [&](const UnitWalk& u) { return static_cast<long long>(rows - 1 - u.item); };
  auto coef_of = [&](const UnitWalk& u) { return u.valid() ? coefs[row_of(u)] : RowCoef{0.f, 0.f, 0.f, -1}; };
  float ahead_c = coef_of(ahead).c;
  auto load_next = [&] {
    while (ahead.valid() && ahead_c == 0.f) ahead.next(), ahead_c = coef_of(ahead).c;
    if (!ahead.valid()) return;
    const int v0 = ahead.part * sub;
    ring.load(reinterpret_cast<const uint4*>(logits + row_of(ahead) * ld) + v0, min(sub, row_vecs - v0) * 16, lane);
    ahead.next();
    ahead_c = coef_of(ahead).c;
  };
  for (int i = 0; i < stages; ++i) load_next();
  bool ok = true;
  RowCoef next = coef_of(at);
  while (at.valid()) {
    const UnitWalk u = at;
    const RowCoef rc = next;
    at.next();
    next = coef_of(at);
    const int v0 = u.part * sub, n = min(sub, row_vecs - v0);
    T* d = dlogits + row_of(u) * ld;
    if (rc.c == 0.f) {
      zero_vecs(reinterpret_cast<uint4*>(d) + v0, n, lane, 32);
      continue;
    }
    ok = ok && ring.wait(6);
    if (ok) {
      const RowGradient<T> g(rc);
      const int inside = max(0, min(n, (V + kV - 1) / kV - v0));
      if (inside > 0) g.store(d, ring.chunk(), v0, inside, V, lane);
      zero_vecs(reinterpret_cast<uint4*>(d) + v0 + inside, n - inside, lane, 32);
      const int t = rc.target - v0 * kV;
      const bool here = t >= 0 && t < n * kV;
      const float x = here ? elem_to_float(reinterpret_cast<const T*>(ring.chunk())[t]) : 0.f;
      __syncwarp();
      if (here && rc.target < V && lane == 0) elem_store(d + rc.target, g.at_target(x, rc.c));
      ring.step();
      load_next();
    }
  }
  ring.drain();
}

// Parts a row is cut into when only its sum is wanted and there are few rows:
// four units for every SM, of 256 vectors of bf16 at least.
int parts_of(long long rows, int V) {
  const long long want = (4LL * num_sms() + rows - 1) / rows;
  return static_cast<int>(std::max(1LL, std::min<long long>({want, kMaxParts, (V + 2047LL) / 2048})));
}

// Scratch of `rows` rows of `Vp` columns: the slot planes, then one RowCoef per
// row.
size_t slots_bytes(long long rows, int Vp) {
  return static_cast<size_t>(parts_of(rows, Vp)) * rows * sizeof(RowSum);
}
size_t loss_workspace(long long rows, int Vp) { return slots_bytes(rows, Vp) + static_cast<size_t>(rows) * sizeof(RowCoef); }

int check_rows(const char* what, void* dlogits, const void* logits, llmk_dtype dtype, long long rows, int V, int Vp,
               const void* workspace, size_t workspace_bytes) {
  if (V <= 0 || Vp < V) return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": bad vocabulary size");
  if (rows > (1 << 30)) return fail(LLMK_ERR_UNSUPPORTED, std::string(what) + ": more than 2^30 rows");
  if (dtype != LLMK_F32 && dtype != LLMK_BF16) return fail(LLMK_ERR_UNSUPPORTED, std::string(what) + ": fp32 or bf16");
  if (Vp % 8 || !aligned16(logits) || !aligned16(dlogits))
    return fail(LLMK_ERR_UNSUPPORTED, std::string(what) + ": Vp % 8, 16-byte alignment");
  if (dlogits && dlogits != logits) {
    const size_t bytes = static_cast<size_t>(rows) * Vp * (dtype == LLMK_BF16 ? 2 : 4);
    const uintptr_t a = reinterpret_cast<uintptr_t>(dlogits), b = reinterpret_cast<uintptr_t>(logits);
    if (a < b + bytes && b < a + bytes)
      return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": dlogits overlaps logits without being the same buffer");
  }
  if (!workspace || !aligned16(workspace) || workspace_bytes < loss_workspace(rows, Vp))
    return fail(LLMK_ERR_WORKSPACE, std::string(what) + ": workspace missing or too small");
  return LLMK_OK;
}

// Opts a kernel into its dynamic shared memory, once per device.
template <typename K>
int allow_smem(K kernel, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  LLMK_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && done[dev]) return LLMK_OK;
  LLMK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
  if (dev < 64) done[dev] = true;
  return LLMK_OK;
}

int div_up(long long a, long long b) { return static_cast<int>((a + b - 1) / b); }

// Bytes of shared memory that a warp's ring may take: all of them and the static
// part fit the 227 KB of an SM.
constexpr int kWarpRingBytes = 9216;

// Fills in group, seg, sub and stages for units of job.vecs vectors; returns
// whether a unit fits its group's rings.
//
// Of the groups whose rings hold a unit `times` over, the one that is through
// first, in rounds of units on all SMs: a unit costs its warps their share of the
// vectors and as much again as 300 vectors for the joining of their sums (from
// times of 320 to 16384 rows). times: 1 where a unit stays in the rings. Where it
// streams through them, larger units in smaller groups leave more groups to work
// while one joins, down to a fifth in bf16, where instructions count as much as
// HBM (8192 rows of 50257 133 us, by groups of half a unit 145; 4096 of 131072
// 178 against 222), and a half in fp32, where HBM does (1500 pair rows 242 us, 258
// by smaller groups). Chunks are as large as a ring of two allows: each costs a
// wait, a copy and a start of the loops (192 vectors instead of 288: 8192 rows of
// 20000 149 against 136 us, evaluation of 50257 149 against 141; 96: 166 us).
constexpr int kWarpVecs = kWarpRingBytes / 16;
template <typename T>
constexpr int kStream = sizeof(T) == 2 ? 5 : 2;
bool share_out(RowJob* job, int times) {
  const long long units = static_cast<long long>(job->rows) * job->parts;
  static const int kGroups[] = {1, 2, 3, 4, 6, 8, 12, 24};  // the divisors of kRowWarps
  long long best = 0;
  job->group = 0;
  for (int group : kGroups) {
    if (group < kRowWarps && job->vecs > group * times * kWarpVecs) continue;
    if (job->group && job->vecs <= 32 * job->group) break;
    const long long at_once = static_cast<long long>(num_sms()) * (kRowWarps / group);
    const long long cost = (units + at_once - 1) / at_once * (div_up(job->vecs, group) + 300);
    if (!job->group || cost < best) job->group = group, best = cost;
  }
  job->seg = div_up(job->vecs, job->group);
  const int chunks = std::min(div_up(job->seg, kWarpVecs / 2), 2);
  job->sub = std::min(div_up(div_up(job->seg, chunks), 32) * 32, kWarpVecs / 2);
  job->stages = std::min(kMaxStages, kWarpVecs / job->sub);
  // One round of a few vectors: sums by expf and in 64 bits cost 0.1 to 0.9 us there
  // (148 rows of 500 to 20000; 73 us of 132 in 8192 rows of 50257), and single rows
  // of few terms, whose rounding errors do not average out, need them: KL estimates
  // of one row of 1572 were 2e-6 off, and are 2e-7.
  job->exact = job->seg <= 128 && units <= static_cast<long long>(num_sms()) * (kRowWarps / job->group);
  return job->stages * job->sub >= job->seg;
}

template <typename T, int kMode, bool kExact = false>
int launch_rows(void* dlogits, const void* logits, const RowJob& job, const PolicyArgs& a, cudaStream_t s) {
  if constexpr (!kExact && kMode != kRowLong) {
    if (job.exact) return launch_rows<T, kMode, true>(dlogits, logits, job, a, s);
  }
  static bool done[64] = {};
  LLMK_TRY(allow_smem(row_kernel<T, kMode, kExact>, kRowWarps * kWarpRingBytes, done));
  const size_t smem = static_cast<size_t>(kRowWarps) * job.stages * job.sub * 16;
  const long long units = static_cast<long long>(job.rows) * job.parts, most = static_cast<long long>(num_sms()) * kMaxItems;
  for (long long u = 0; u < units; u += most) {
    RowJob now = job;
    now.unit0 = static_cast<unsigned>(u);
    now.unit1 = static_cast<unsigned>(std::min(units, u + most));
    row_kernel<T, kMode, kExact><<<static_cast<int>(std::min<long long>(now.unit1 - now.unit0, num_sms())), kRowThreads, smem, s>>>(
        static_cast<T*>(dlogits), static_cast<const T*>(logits), now, a);
    count_launch();
  }
  LLMK_CUDA(cudaGetLastError());
  return LLMK_OK;
}

template <typename T>
RowJob row_job(const float* weights, int rows, int V, int Vp) {
  RowJob job{};
  job.weights = weights;
  job.rows = rows, job.V = V, job.ld = Vp;
  job.parts = 1;
  job.vecs = div_up(V, vec_elems<T>());
  job.status = device_status_ptr();
  return job;
}

// Slots of every live row; returns the number of planes through *nslots.
template <typename T>
int launch_slots(RowSum* slots, int* nslots, const void* logits, const float* weights, int rows, int V, int Vp, cudaStream_t s) {
  RowJob job = row_job<T>(weights, rows, V, Vp);
  const int all = job.vecs;
  job.slots = slots;
  job.vecs = div_up(all, parts_of(rows, V));
  job.parts = *nslots = div_up(all, job.vecs);  // rounding up may leave the last part empty
  share_out(&job, kStream<T>);
  return launch_rows<T, kRowStats>(nullptr, logits, job, PolicyArgs{}, s);
}

template <typename T>
int launch_gradient(void* dlogits, const void* logits, const RowCoef* coefs, int rows, int V, int Vp, cudaStream_t s) {
  static bool done[64] = {};
  LLMK_TRY(allow_smem(row_gradient_kernel<T>, kRowWarps * kWarpRingBytes, done));
  const int vecs = Vp / vec_elems<T>(), chunks = div_up(vecs, 192), sub = div_up(div_up(vecs, chunks), 32) * 32;
  const int stages = std::min(kMaxStages, kWarpRingBytes / (sub * 16));
  const long long units = static_cast<long long>(rows) * div_up(vecs, sub);
  LLMK_CUDA(launch_after(row_gradient_kernel<T>, static_cast<int>(std::min<long long>(units, num_sms())), kRowThreads,
                         static_cast<size_t>(kRowWarps) * stages * sub * 16, s, static_cast<T*>(dlogits),
                         static_cast<const T*>(logits), coefs, rows, V, Vp, sub, stages, device_status_ptr()));
  count_launch();
  return LLMK_OK;
}

template <typename T>
int policy_loss(void* dlogits, const void* logits, const PolicyArgs& a, int rows, int V, int Vp, void* workspace,
                cudaStream_t s) {
  RowJob job = row_job<T>(a.weights, rows, V, Vp);
  job.slots = static_cast<RowSum*>(workspace);
  if (!dlogits) {
    share_out(&job, kStream<T>);
    return launch_rows<T, kRowEval>(nullptr, logits, job, a, s);
  }
  // Rows that take more than half an SM each, and for at most half the SMs: three
  // kernels over parts of rows on all SMs are faster (16 rows of 131072 bf16: 11.3
  // against 19.4 us, 64: 16.0 against 19.9, 96: 21.2 against 21.1; 64 of 100000:
  // 14.5 against 16.0, 96: 17.4 against 16.5; 64 of 50257: the same).
  if (job.vecs <= kRowWarps / 2 * kWarpVecs || 2 * rows > num_sms()) {
    const bool fits = share_out(&job, 1);
    return fits ? launch_rows<T, kRowGrad>(dlogits, logits, job, a, s) : launch_rows<T, kRowLong>(dlogits, logits, job, a, s);
  }
  RowSum* slots = job.slots;
  auto* coefs = reinterpret_cast<RowCoef*>(static_cast<char*>(workspace) + slots_bytes(rows, Vp));
  int nslots = 0;
  LLMK_TRY(launch_slots<T>(slots, &nslots, logits, a.weights, rows, V, Vp, s));
  LLMK_CUDA(launch_after(policy_rows_kernel<T>, div_up(rows, 128), 128, 0, s, coefs, slots,
                         static_cast<const T*>(logits), a, rows, V, Vp, nslots));
  count_launch();
  return launch_gradient<T>(dlogits, logits, coefs, rows, V, Vp, s);
}

template <typename T>
int preference_loss(void* dlogits, const void* logits, const PreferenceArgs& a, int pairs, int Tlen, int V, int Vp,
                    void* workspace, cudaStream_t s) {
  const int rows = 2 * pairs * Tlen;
  auto* slots = static_cast<RowSum*>(workspace);
  auto* coefs = dlogits ? reinterpret_cast<RowCoef*>(static_cast<char*>(workspace) + slots_bytes(rows, Vp)) : nullptr;
  int nslots = 0;
  LLMK_TRY(launch_slots<T>(slots, &nslots, logits, a.weights, rows, V, Vp, s));
  LLMK_CUDA(launch_after(preference_pair_kernel<T, true>, pairs, kPairThreads, 0, s, coefs, slots,
                         static_cast<const T*>(logits), a, pairs, Tlen, V, Vp, nslots));
  count_launch();
  return dlogits ? launch_gradient<T>(dlogits, logits, coefs, rows, V, Vp, s) : LLMK_OK;
}

bool bad_nonneg(float v) { return !(v >= 0.f) || std::isinf(v); }

// A slot's sum from the lm_head GEMM's epilogue, whose terms are 2^(x log2 e - c)
// with c = max log2 e rounded: what the rounding adds to every exponent, up to 2e-6
// at logits of 40, is known exactly and leaves the sum again. 16-bit logits have
// few maxima, so that it would not average out over rows (their log-probabilities
// around -40 were 2.6e-7 off on average). Of fp32 logits, the terms of a slot's
// first half carry it twice, the one that is their own maximum's among them, and
// keep one.
__device__ __forceinline__ float slot_sum(const float2& p) {
  const float c = __fmul_rn(p.x, kLog2e);
  const float added = fmaf(p.x, kLog2e, -c);
  return p.x == -INFINITY ? p.y : fmaf(-p.y, added * 0.69314718f, p.y);
}

// From the slots' (max, sum exp(x - max)), one of every 64 columns in planes of
// `rows`: block = 8 rows, 32 threads a row fold a 32nd of the slots each, and one
// joins them in a fixed order.
constexpr int kFoldRows = 8, kFoldGroups = 32;
template <typename T>
__global__ void __launch_bounds__(kFoldRows* kFoldGroups) rowstats_fold_kernel(RowSum* __restrict__ sums,
                                                                              const float2* __restrict__ stats,
                                                                              const T* __restrict__ logits,
                                                                              const int* __restrict__ targets, int rows,
                                                                              int V, int ld, int nslots) {
  __shared__ float2 part[kFoldGroups][kFoldRows];
  grid_release();
  grid_wait();
  const int r = threadIdx.x % kFoldRows, g = threadIdx.x / kFoldRows;
  const long long row = static_cast<long long>(blockIdx.x) * kFoldRows + r;
  float m = -INFINITY, s = 0.f;
  if (row < rows) {
    for (int k = g; k < nslots; k += kFoldGroups) {
      const float2 p = stats[static_cast<long long>(k) * rows + row];
      const float top = fmaxf(m, p.x), ref = finite_max(top);
      s = s * expf(m - ref) + slot_sum(p) * expf(p.x - ref);
      m = top;
    }
  }
  part[g][r] = make_float2(m, s);
  __syncthreads();
  if (g != 0 || row >= rows) return;
  float M = -INFINITY;
  for (int i = 0; i < kFoldGroups; ++i) M = fmaxf(M, part[i][r].x);
  double S = 0.0;
  for (int i = 0; i < kFoldGroups; ++i) S += static_cast<double>(part[i][r].y) * static_cast<double>(expf(part[i][r].x - finite_max(M)));
  const int t = targets[row];
  sums[row] = RowSum{S, M, t >= 0 && t < V ? elem_to_float(logits[row * ld + t]) : NAN};
}

__global__ void __launch_bounds__(256) logps_kernel(float* __restrict__ logps, const RowSum* __restrict__ sums, int rows) {
  grid_wait();
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const RowSum t = sums[row];
  logps[row] = static_cast<float>(logp_of(t));
}

__global__ void __launch_bounds__(1024) sum_losses_kernel(float* __restrict__ out, const float* __restrict__ x, int n, float div) {
  __shared__ double red[32];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) s += x[i];
  s = warp_sum_d(s);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  s = warp_sum_d(red[threadIdx.x]);
  if (threadIdx.x == 0) *out = static_cast<float>(s / div);
}

template <typename T>
int launch_fold(RowSum* sums, const float2* stats, const void* logits, const int* targets, int rows, int V, int ld, cudaStream_t s) {
  LLMK_CUDA(launch_after(rowstats_fold_kernel<T>, div_up(rows, kFoldRows), kFoldRows * kFoldGroups, 0, s, sums, stats,
                         static_cast<const T*>(logits), targets, rows, V, ld, div_up(ld, 64)));
  count_launch();
  return LLMK_OK;
}

struct Scratch {
  RowSum* sums;
  RowCoef* coefs;
};
Scratch split(void* scratch, int rows) {
  auto* sums = static_cast<RowSum*>(scratch);
  return {sums, reinterpret_cast<RowCoef*>(sums + rows)};
}

template <typename T>
int policy_finish_t(void* logits, const float2* stats, const PolicyArgs& a, int rows, int V, int ld, int backward,
                    void* scratch, cudaStream_t s) {
  const Scratch w = split(scratch, rows);
  LLMK_TRY(launch_fold<T>(w.sums, stats, logits, a.targets, rows, V, ld, s));
  RowCoef* coefs = backward ? w.coefs : nullptr;
  LLMK_CUDA(launch_after(policy_rows_kernel<T>, div_up(rows, 128), 128, 0, s, coefs, w.sums,
                         static_cast<const T*>(logits), a, rows, V, ld, 1));
  count_launch();
  return backward ? launch_gradient<T>(logits, logits, w.coefs, rows, V, ld, s) : LLMK_OK;
}

template <typename T>
int preference_finish_t(void* logits, const float2* stats, const PreferenceArgs& a, int pairs, int Tlen, int V, int ld,
                        int backward, void* scratch, cudaStream_t s) {
  const int rows = 2 * pairs * Tlen;
  const Scratch w = split(scratch, rows);
  LLMK_TRY(launch_fold<T>(w.sums, stats, logits, a.targets, rows, V, ld, s));
  RowCoef* coefs = backward ? w.coefs : nullptr;
  LLMK_CUDA(launch_after(preference_pair_kernel<T, false>, pairs, kPairThreads, 0, s, coefs, w.sums,
                         static_cast<const T*>(logits), a, pairs, Tlen, V, ld, 1));
  count_launch();
  return backward ? launch_gradient<T>(logits, logits, w.coefs, rows, V, ld, s) : LLMK_OK;
}

}  // namespace

int policy_finish(void* logits, llmk_dtype dtype, const float2* stats, const PolicyArgs& a, int rows, int V, int ld,
                  int backward, void* scratch, cudaStream_t s) {
  return dtype == LLMK_BF16 ? policy_finish_t<__nv_bfloat16>(logits, stats, a, rows, V, ld, backward, scratch, s)
                            : policy_finish_t<float>(logits, stats, a, rows, V, ld, backward, scratch, s);
}

int preference_finish(void* logits, llmk_dtype dtype, const float2* stats, const PreferenceArgs& a, int pairs, int T, int V,
                      int ld, int backward, void* scratch, cudaStream_t s) {
  return dtype == LLMK_BF16
             ? preference_finish_t<__nv_bfloat16>(logits, stats, a, pairs, T, V, ld, backward, scratch, s)
             : preference_finish_t<float>(logits, stats, a, pairs, T, V, ld, backward, scratch, s);
}

int logps_finish(float* logps, const void* logits, llmk_dtype dtype, const float2* stats, const int* targets, int rows, int V,
                 int ld, void* scratch, cudaStream_t s) {
  const Scratch w = split(scratch, rows);
  if (dtype == LLMK_BF16) LLMK_TRY(launch_fold<__nv_bfloat16>(w.sums, stats, logits, targets, rows, V, ld, s));
  else LLMK_TRY(launch_fold<float>(w.sums, stats, logits, targets, rows, V, ld, s));
  LLMK_CUDA(launch_after(logps_kernel, div_up(rows, 256), 256, 0, s, logps, w.sums, rows));
  count_launch();
  return LLMK_OK;
}

int sum_losses(float* out, const float* x, int n, float div, cudaStream_t s) {
  sum_losses_kernel<<<1, 1024, 0, s>>>(out, x, n, div);
  count_launch();
  LLMK_CUDA(cudaGetLastError());
  return LLMK_OK;
}

int check_policy(const char* what, const PolicyArgs& a, int rows) {
  const std::string w = what;
  if (!a.losses || !a.targets || !a.advantages || rows <= 0)
    return fail(LLMK_ERR_INVALID_ARG, w + ": null operand or no rows");
  if (bad_nonneg(a.clip_low) || bad_nonneg(a.clip_high) || a.clip_low > 1.f || !std::isfinite(a.kl_coef) ||
      !std::isfinite(a.dscale))
    return fail(LLMK_ERR_INVALID_ARG, w + ": clip_low in [0, 1], clip_high >= 0, finite kl_coef and dscale");
  if (!a.ref_logps && (a.kl_coef != 0.f || a.kls))
    return fail(LLMK_ERR_INVALID_ARG, w + ": the KL term needs ref_logps");
  return LLMK_OK;
}

int check_preference(const char* what, const PreferenceArgs& a, int pairs, int T) {
  const std::string w = what;
  if (!a.losses || !a.targets || pairs <= 0 || T <= 0)
    return fail(LLMK_ERR_INVALID_ARG, w + ": null operand, no pairs or no positions");
  if (!(a.beta > 0.f) || std::isinf(a.beta) || !(a.smoothing >= 0.f) || a.smoothing > 1.f || !std::isfinite(a.dscale))
    return fail(LLMK_ERR_INVALID_ARG, w + ": beta > 0, label_smoothing in [0, 1], finite dscale");
  return LLMK_OK;
}

}  // namespace llmk

using namespace llmk;

extern "C" {

size_t llmk_policy_loss_workspace(int rows, int Vp) { return rows <= 0 || Vp <= 0 ? 0 : loss_workspace(rows, Vp); }

int llmk_policy_loss(float* losses, float* kls, float* logps, void* dlogits, const void* logits, llmk_dtype dtype,
                     const int* targets, const float* weights, const float* advantages, const float* old_logps,
                     const float* ref_logps, int rows, int V, int Vp, float clip_low, float clip_high, float kl_coef,
                     float dscale, void* workspace, size_t workspace_bytes, void* stream) {
  const PolicyArgs a{losses, kls, logps, targets, weights, advantages, old_logps, ref_logps, clip_low, clip_high, kl_coef, dscale};
  if (!logits) return fail(LLMK_ERR_INVALID_ARG, "policy_loss: null operand or no rows");
  LLMK_TRY(check_policy("policy_loss", a, rows));
  LLMK_TRY(check_rows("policy_loss", dlogits, logits, dtype, rows, V, Vp, workspace, workspace_bytes));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == LLMK_BF16 ? policy_loss<__nv_bfloat16>(dlogits, logits, a, rows, V, Vp, workspace, s)
                            : policy_loss<float>(dlogits, logits, a, rows, V, Vp, workspace, s);
}

size_t llmk_preference_loss_workspace(int pairs, int T, int Vp) {
  return pairs <= 0 || T <= 0 || Vp <= 0 ? 0 : loss_workspace(2LL * pairs * T, Vp);
}

int llmk_preference_loss(float* losses, float* rewards, float* logps, void* dlogits, const void* logits, llmk_dtype dtype,
                         const int* targets, const float* weights, const float* ref_logps, int pairs, int T, int V,
                         int Vp, float beta, float label_smoothing, float dscale, void* workspace,
                         size_t workspace_bytes, void* stream) {
  const PreferenceArgs a{losses, rewards, logps, targets, weights, ref_logps, beta, label_smoothing, dscale};
  if (!logits) return fail(LLMK_ERR_INVALID_ARG, "preference_loss: null operand, no pairs or no positions");
  LLMK_TRY(check_preference("preference_loss", a, pairs, T));
  LLMK_TRY(check_rows("preference_loss", dlogits, logits, dtype, 2LL * pairs * T, V, Vp, workspace, workspace_bytes));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == LLMK_BF16 ? preference_loss<__nv_bfloat16>(dlogits, logits, a, pairs, T, V, Vp, workspace, s)
                            : preference_loss<float>(dlogits, logits, a, pairs, T, V, Vp, workspace, s);
}

}  // extern "C"
