// Fine-tuning losses over logits, forward and gradient: the clipped policy
// loss with a KL term, and the preference loss over pairs of sequences.
//
// Both are functions of the target's log-probability in each row of logits,
//   lp = x[target] - max(x) - log(sum_j exp(x_j - max(x))),  j < V,
// with d(lp)/d(x_j) = [j = target] - softmax(x)_j, so the gradient of either
// loss is one coefficient c = d(loss)/d(lp) per row times that difference.
// Three steps, for both:
//   1. row_slots_kernel: (max, sum exp(x - max)) of every 16 KB slice of a row;
//   2. one thread per row folds the slices, forms lp and the loss's terms in
//      64 bits, and leaves the row's (max, c / sum, c, target);
//   3. row_gradient_kernel: dlogits = [j = target] c - exp(x - max) c / sum.
// Rows of weight zero (prompts, padding) are not read; their gradient is zero.
#include <algorithm>
#include <climits>
#include <cmath>
#include <string>

#include "ptx.cuh"
#include "runtime.h"
#include "vec8.cuh"

namespace llmk {
namespace {

constexpr int kSliceBytes = 16384;
constexpr int kThreads = 256;

template <typename T>
constexpr int slice_elems() {
  return kSliceBytes / static_cast<int>(sizeof(T));
}

// What step 3 needs to know of a row.
struct __align__(16) RowCoef {
  float max;
  float scale;  // c / sum
  float c;      // d(loss) / d(lp), dscale included; 0: the row's gradient is 0
  int target;
};

__device__ __forceinline__ float warp_max_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
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

// Step 1. Slots lie in planes, slots[slot * rows + row], so that step 2's
// neighbouring threads read neighbouring rows.
template <typename T>
__global__ void __launch_bounds__(kThreads) row_slots_kernel(float2* __restrict__ slots, const T* __restrict__ logits,
                                                             const float* __restrict__ weights, int rows, int V, int ld,
                                                             int nslots) {
  constexpr int kPer = slice_elems<T>() / (kThreads * 8);
  __shared__ float red_m[kThreads / 32], red_s[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long units = static_cast<long long>(rows) * nslots;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long row = u / nslots;
    const int slot = static_cast<int>(u - row * nslots);
    if (weights && weights[row] == 0.f) continue;
    const int c0 = slot * slice_elems<T>();
    const T* x = logits + row * ld + c0;
    const int n = min(slice_elems<T>(), V - c0);
    float v[kPer][8];
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int e = (k * kThreads + threadIdx.x) * 8;
      if (e < n) {
        load8v(x + e, v[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (e + j >= n) v[k][j] = -INFINITY;
          m = fmaxf(m, v[k][j]);
        }
      }
    }
    m = warp_max_f(m);
    if (lane == 0) red_m[warp] = m;
    __syncthreads();
    float M = red_m[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) M = fmaxf(M, red_m[w]);
    const float ref = finite_max(M);
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int e = (k * kThreads + threadIdx.x) * 8;
      if (e < n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s += expf(v[k][j] - ref);
      }
    }
    s = warp_sum_f(s);
    if (lane == 0) red_s[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      float S = 0.f;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) S += red_s[w];
      slots[static_cast<long long>(slot) * rows + row] = make_float2(M, S);
    }
  }
}

// max and sum of a row from its slots.
__device__ __forceinline__ void fold_slots(const float2* __restrict__ slots, long long row, int rows, int nslots, float* m,
                                           double* s) {
  float M = -INFINITY;
  for (int k = 0; k < nslots; ++k) M = fmaxf(M, slots[static_cast<long long>(k) * rows + row].x);
  const float ref = finite_max(M);
  double S = 0.0;
  for (int k = 0; k < nslots; ++k) {
    const float2 p = slots[static_cast<long long>(k) * rows + row];
    S += static_cast<double>(p.y * expf(p.x - ref));
  }
  *m = M;
  *s = S;
}

// lp of a row; NaN for a target outside [0, V).
template <typename T>
__device__ __forceinline__ double target_logp(const T* logits, long long row, int ld, int V, int target, float m, double s) {
  if (target < 0 || target >= V) return static_cast<double>(NAN);
  return static_cast<double>(elem_to_float(logits[row * ld + target])) - static_cast<double>(m) - log(s);
}

struct PolicyArgs {
  float *losses, *kls, *logps;
  const int* targets;
  const float *weights, *advantages, *old_logps, *ref_logps;
  float clip_low, clip_high, kl_coef, dscale;
};

// Step 2 of the policy loss. With rho = exp(lp - old), A the advantage and
// d = ref - lp: loss = w (-min(rho A, clamp(rho) A) + kl_coef (exp(d) - d - 1)).
// The clipped branch has no gradient; where both are equal (rho inside the
// bounds, or on one) the unclipped one counts.
template <typename T>
__global__ void __launch_bounds__(128) policy_rows_kernel(RowCoef* __restrict__ coefs, const float2* __restrict__ slots,
                                                          const T* __restrict__ logits, PolicyArgs a, int rows, int V,
                                                          int ld, int nslots) {
  const long long row = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (row >= rows) return;
  const float w = a.weights ? a.weights[row] : 1.f;
  if (w == 0.f) {
    a.losses[row] = 0.f;
    if (a.kls) a.kls[row] = 0.f;
    if (a.logps) a.logps[row] = 0.f;
    if (coefs) coefs[row] = RowCoef{0.f, 0.f, 0.f, -1};
    return;
  }
  float m;
  double s;
  fold_slots(slots, row, rows, nslots, &m, &s);
  const int target = a.targets[row];
  const double lp = target_logp(logits, row, ld, V, target, m, s);
  const double A = a.advantages[row];
  const double rho = a.old_logps ? exp(lp - static_cast<double>(a.old_logps[row])) : 1.0;
  const double lo = 1.0 - static_cast<double>(a.clip_low), hi = 1.0 + static_cast<double>(a.clip_high);
  const double clamped = rho < lo ? lo : (rho > hi ? hi : rho);
  const double s1 = A == 0.0 ? 0.0 : rho * A, s2 = clamped * A;
  double loss = s1 > s2 ? -s2 : -s1;
  double g = s1 > s2 ? 0.0 : -s1;
  if (!a.old_logps && isnan(lp)) loss = g = lp;
  if (a.ref_logps) {
    const double d = static_cast<double>(a.ref_logps[row]) - lp;
    const double e = expm1(d);
    const double kl = e - d;
    if (a.kls) a.kls[row] = static_cast<float>(kl);
    if (a.kl_coef != 0.f) {
      loss += static_cast<double>(a.kl_coef) * kl;
      g -= static_cast<double>(a.kl_coef) * e;
    }
  }
  a.losses[row] = static_cast<float>(w * loss);
  if (a.logps) a.logps[row] = static_cast<float>(lp);
  if (coefs) {
    const double c = g * w * a.dscale;
    coefs[row] = RowCoef{finite_max(m), static_cast<float>(c / s), static_cast<float>(c), target};
  }
}

struct PreferenceArgs {
  float *losses, *rewards, *logps;
  const int* targets;
  const float *weights, *ref_logps;
  float beta, smoothing, dscale;
};

// log(1 + exp(v)) without overflow.
__device__ __forceinline__ double softplus_d(double v) { return (v > 0.0 ? v : 0.0) + log1p(exp(-fabs(v))); }

// Step 2 of the preference loss, one CTA per pair p (sequence p is the chosen
// one, pairs + p the rejected one): L = sum_t w lp over each sequence, h =
// beta ((L_c - R_c) - (L_r - R_r)), loss = (1 - e) log(1 + exp(-h)) + e log(1 +
// exp(h)). The sums run in a fixed order in 64 bits.
constexpr int kPairThreads = 1024;
template <typename T>
__global__ void __launch_bounds__(kPairThreads) preference_pair_kernel(RowCoef* __restrict__ coefs,
                                                                       float2* __restrict__ slots,
                                                                       const T* __restrict__ logits, PreferenceArgs a,
                                                                       int pairs, int Tlen, int V, int ld, int nslots) {
  __shared__ double red[2][kPairThreads / 32];
  const int pair = blockIdx.x, rows = 2 * pairs * Tlen;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double sum[2] = {0.0, 0.0};
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long row0 = static_cast<long long>(side * pairs + pair) * Tlen;
    for (int t = threadIdx.x; t < Tlen; t += kPairThreads) {
      const long long row = row0 + t;
      const float w = a.weights ? a.weights[row] : 1.f;
      double lp = 0.0;
      if (w != 0.f) {
        float m;
        double s;
        fold_slots(slots, row, rows, nslots, &m, &s);
        lp = target_logp(logits, row, ld, V, a.targets[row], m, s);
        sum[side] += static_cast<double>(w) * lp;
        // kept for the second loop, which this thread runs over the same rows
        if (coefs) coefs[row] = RowCoef{finite_max(m), static_cast<float>(1.0 / s), 0.f, a.targets[row]};
      }
      if (a.logps) a.logps[row] = static_cast<float>(lp);
    }
    sum[side] = warp_sum_d(sum[side]);
    if (lane == 0) red[side][warp] = sum[side];
  }
  __syncthreads();
  double L[2] = {0.0, 0.0};
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int k = 0; k < kPairThreads / 32; ++k) L[side] += red[side][k];
  const double beta = a.beta, e = a.smoothing;
  const double rc = beta * (L[0] - (a.ref_logps ? static_cast<double>(a.ref_logps[pair]) : 0.0));
  const double rr = beta * (L[1] - (a.ref_logps ? static_cast<double>(a.ref_logps[pairs + pair]) : 0.0));
  const double h = rc - rr;
  if (threadIdx.x == 0) {
    a.losses[pair] = static_cast<float>((1.0 - e) * softplus_d(-h) + e * softplus_d(h));
    if (a.rewards) {
      a.rewards[pair] = static_cast<float>(rc);
      a.rewards[pairs + pair] = static_cast<float>(rr);
    }
  }
  if (!coefs) return;
  const double slope = beta * static_cast<double>(a.dscale) * (e / (1.0 + exp(-h)) - (1.0 - e) / (1.0 + exp(h)));
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const long long row0 = static_cast<long long>(side * pairs + pair) * Tlen;
    for (int t = threadIdx.x; t < Tlen; t += kPairThreads) {
      const long long row = row0 + t;
      const float w = a.weights ? a.weights[row] : 1.f;
      if (w == 0.f) {
        coefs[row] = RowCoef{0.f, 0.f, 0.f, -1};
      } else {
        RowCoef rcf = coefs[row];
        rcf.c = static_cast<float>((side ? -slope : slope) * w);
        rcf.scale *= rcf.c;
        coefs[row] = rcf;
      }
    }
  }
}

// Step 3. dlogits may be the logits: every thread writes only what it read.
template <typename T>
__global__ void __launch_bounds__(kThreads) row_gradient_kernel(T* dlogits, const T* logits,
                                                                const RowCoef* __restrict__ coefs, int rows, int V,
                                                                int ld, int nslots) {
  constexpr int kPer = slice_elems<T>() / (kThreads * 8);
  const long long units = static_cast<long long>(rows) * nslots;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const long long row = u / nslots;
    const int c0 = static_cast<int>(u - row * nslots) * slice_elems<T>();
    const int n = min(slice_elems<T>(), ld - c0);
    const RowCoef rc = coefs[row];
    const T* x = logits + row * ld + c0;
    T* d = dlogits + row * ld + c0;
    if (rc.c == 0.f) {
      const float zero[8] = {};
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int e = (k * kThreads + threadIdx.x) * 8;
        if (e < n) store8v(d + e, zero);
      }
      continue;
    }
    float v[kPer][8];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int e = (k * kThreads + threadIdx.x) * 8;
      if (e < n) load8v(x + e, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int e = (k * kThreads + threadIdx.x) * 8, c = c0 + e;
      if (e < n) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float g = -expf(v[k][j] - rc.max) * rc.scale;
          if (c + j == rc.target) g += rc.c;
          v[k][j] = c + j < V ? g : 0.f;
        }
        store8v(d + e, v[k]);
      }
    }
  }
}

template <typename T>
int slots_of(int cols) {
  return (cols + slice_elems<T>() - 1) / slice_elems<T>();
}

int grid_of(long long units) { return static_cast<int>(std::min<long long>(units, num_sms() * 8LL)); }

// Scratch of `rows` rows of `Vp` columns: the slot planes (at the fp32 slot
// count, the larger one), then one RowCoef per row.
size_t slots_bytes(long long rows, int Vp) {
  return (static_cast<size_t>(slots_of<float>(Vp)) * rows * sizeof(float2) + 15) / 16 * 16;
}
size_t loss_workspace(long long rows, int Vp) { return slots_bytes(rows, Vp) + static_cast<size_t>(rows) * sizeof(RowCoef); }

int check_rows(const char* what, void* dlogits, const void* logits, llmk_dtype dtype, long long rows, int V, int Vp,
               const void* workspace, size_t workspace_bytes) {
  if (V <= 0 || Vp < V) return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": bad vocabulary size");
  if (rows > INT_MAX) return fail(LLMK_ERR_UNSUPPORTED, std::string(what) + ": more than 2^31 - 1 rows");
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

template <typename T>
int launch_slots(float2* slots, const void* logits, const float* weights, int rows, int V, int Vp, cudaStream_t s) {
  const int n = slots_of<T>(V);
  row_slots_kernel<T><<<grid_of(static_cast<long long>(rows) * n), kThreads, 0, s>>>(
      slots, static_cast<const T*>(logits), weights, rows, V, Vp, n);
  count_launch();
  LLMK_CUDA(cudaGetLastError());
  return LLMK_OK;
}

template <typename T>
int launch_gradient(void* dlogits, const void* logits, const RowCoef* coefs, int rows, int V, int Vp, cudaStream_t s) {
  const int n = slots_of<T>(Vp);
  row_gradient_kernel<T><<<grid_of(static_cast<long long>(rows) * n), kThreads, 0, s>>>(
      static_cast<T*>(dlogits), static_cast<const T*>(logits), coefs, rows, V, Vp, n);
  count_launch();
  LLMK_CUDA(cudaGetLastError());
  return LLMK_OK;
}

template <typename T>
int policy_loss(void* dlogits, const void* logits, const PolicyArgs& a, int rows, int V, int Vp, void* workspace,
                cudaStream_t s) {
  auto* slots = static_cast<float2*>(workspace);
  auto* coefs = dlogits ? reinterpret_cast<RowCoef*>(static_cast<char*>(workspace) + slots_bytes(rows, Vp)) : nullptr;
  LLMK_TRY(launch_slots<T>(slots, logits, a.weights, rows, V, Vp, s));
  policy_rows_kernel<T><<<static_cast<int>((rows + 127LL) / 128), 128, 0, s>>>(coefs, slots, static_cast<const T*>(logits), a, rows, V, Vp,
                                                           slots_of<T>(V));
  count_launch();
  LLMK_CUDA(cudaGetLastError());
  return dlogits ? launch_gradient<T>(dlogits, logits, coefs, rows, V, Vp, s) : LLMK_OK;
}

template <typename T>
int preference_loss(void* dlogits, const void* logits, const PreferenceArgs& a, int pairs, int Tlen, int V, int Vp,
                    void* workspace, cudaStream_t s) {
  const int rows = 2 * pairs * Tlen;
  auto* slots = static_cast<float2*>(workspace);
  auto* coefs = dlogits ? reinterpret_cast<RowCoef*>(static_cast<char*>(workspace) + slots_bytes(rows, Vp)) : nullptr;
  LLMK_TRY(launch_slots<T>(slots, logits, a.weights, rows, V, Vp, s));
  preference_pair_kernel<T><<<pairs, kPairThreads, 0, s>>>(coefs, slots, static_cast<const T*>(logits), a, pairs, Tlen, V,
                                                           Vp, slots_of<T>(V));
  count_launch();
  LLMK_CUDA(cudaGetLastError());
  return dlogits ? launch_gradient<T>(dlogits, logits, coefs, rows, V, Vp, s) : LLMK_OK;
}

bool bad_nonneg(float v) { return !(v >= 0.f) || std::isinf(v); }

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" {

size_t llmk_policy_loss_workspace(int rows, int Vp) { return rows <= 0 || Vp <= 0 ? 0 : loss_workspace(rows, Vp); }

int llmk_policy_loss(float* losses, float* kls, float* logps, void* dlogits, const void* logits, llmk_dtype dtype,
                     const int* targets, const float* weights, const float* advantages, const float* old_logps,
                     const float* ref_logps, int rows, int V, int Vp, float clip_low, float clip_high, float kl_coef,
                     float dscale, void* workspace, size_t workspace_bytes, void* stream) {
  if (!losses || !logits || !targets || !advantages || rows <= 0)
    return fail(LLMK_ERR_INVALID_ARG, "policy_loss: null operand or no rows");
  if (bad_nonneg(clip_low) || bad_nonneg(clip_high) || clip_low > 1.f || !std::isfinite(kl_coef) || !std::isfinite(dscale))
    return fail(LLMK_ERR_INVALID_ARG, "policy_loss: clip_low in [0, 1], clip_high >= 0, finite kl_coef and dscale");
  if (!ref_logps && (kl_coef != 0.f || kls))
    return fail(LLMK_ERR_INVALID_ARG, "policy_loss: the KL term needs ref_logps");
  LLMK_TRY(check_rows("policy_loss", dlogits, logits, dtype, rows, V, Vp, workspace, workspace_bytes));
  const PolicyArgs a{losses, kls, logps, targets, weights, advantages, old_logps, ref_logps, clip_low, clip_high, kl_coef, dscale};
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
  if (!losses || !logits || !targets || pairs <= 0 || T <= 0)
    return fail(LLMK_ERR_INVALID_ARG, "preference_loss: null operand, no pairs or no positions");
  if (!(beta > 0.f) || std::isinf(beta) || !(label_smoothing >= 0.f) || label_smoothing > 1.f || !std::isfinite(dscale))
    return fail(LLMK_ERR_INVALID_ARG, "preference_loss: beta > 0, label_smoothing in [0, 1], finite dscale");
  LLMK_TRY(check_rows("preference_loss", dlogits, logits, dtype, 2LL * pairs * T, V, Vp, workspace, workspace_bytes));
  const PreferenceArgs a{losses, rewards, logps, targets, weights, ref_logps, beta, label_smoothing, dscale};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == LLMK_BF16 ? preference_loss<__nv_bfloat16>(dlogits, logits, a, pairs, T, V, Vp, workspace, s)
                            : preference_loss<float>(dlogits, logits, a, pairs, T, V, Vp, workspace, s);
}

}  // extern "C"
