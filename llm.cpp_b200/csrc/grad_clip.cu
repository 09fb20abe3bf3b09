// Global gradient norm over many tensors, and clipping.
//
//   norm = |scale| sqrt(sum over all tensors of g^2),
//   out = g min(1, max_norm / (norm + 1e-6)).
//
// One launch covers every tensor: the tensors' addresses, sizes and types ride
// in the kernel's parameter block (so a captured graph replays them, and no
// table has to be uploaded), cut into units of kUnit elements that a fixed
// grid walks (every thread with four 16- or 32-byte loads under way). Each CTA
// leaves one 64-bit partial sum; the next kernel adds the partials in one order,
// so the result does not depend on timing and every CTA sees the same clipping
// factor. Squares are summed in fp32 over the 33
// elements a thread has of a unit, then in 64 bits; where they leave the fp32
// range (|g| above 1e19, or all below 1e-13), the thread adds them again in 64
// bits.
#include <algorithm>
#include <climits>
#include <cmath>
#include <new>
#include <string>
#include <vector>

#include "ptx.cuh"
#include "runtime.h"
#include "vec8.cuh"

namespace llmk {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;                    // vectors of 8 elements a thread holds
constexpr int kUnit = kThreads * 8 * kPer;  // elements of one unit
constexpr int kCtasPerSm = 4;

struct TensorRef {
  const void* in;
  void* out;
  long long n;
  int unit0;  // first unit of this tensor
  short in_dtype, out_dtype;
};
template <int kCap>
struct TensorTable {
  TensorRef t[kCap];
  int count, units;
};

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same value in every thread, in a fixed order.
__device__ __forceinline__ double block_sum_d(double v, double* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_sum_d(v);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) s += red[w];
  return s;
}

// The tensor that unit u belongs to (the last one whose unit0 is <= u; empty
// tensors share their successor's unit0 and are never chosen).
template <int kCap>
__device__ __forceinline__ int find_tensor(const TensorTable<kCap>& tab, int u) {
  int lo = 0, hi = tab.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tab.t[mid].unit0 <= u) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Elements in front of the first 16-byte boundary at or after p.
template <typename T>
__device__ __forceinline__ int head_of(const T* p) {
  return static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
}

// Eight elements as they lie in memory, loaded before they are needed: `load`
// is only the loads, so that a thread's kPer of them are under way together.
template <typename T>
struct Raw {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void values(float (&v)[8]) const { load8v(reinterpret_cast<const T*>(u), v); }
};

// What a unit's n elements from g on are made of: up to 7 in front of the first
// 16-byte boundary, nv vectors of 8, up to 7 behind. Thread x < head has element
// x of the front, thread 8 + x element x of the back.
template <typename T>
struct UnitShape {
  int head, nv, tail;
  __device__ __forceinline__ UnitShape(const T* g, int n) : head(min(n, head_of(g))), nv((n - head) / 8), tail(n - head - nv * 8) {}
  // This thread's element outside the vectors, -1 for none.
  __device__ __forceinline__ int edge() const {
    const int x = threadIdx.x;
    return x < head ? x : (x >= 8 && x < 8 + tail ? head + 8 * nv + x - 8 : -1);
  }
};

// This thread's vectors of a unit: all but the last are there in every thread
// unless the unit is a short one.
template <typename T>
__device__ __forceinline__ void load_unit(Raw<T> (&r)[kPer], const T* a, int nv) {
  const int x = threadIdx.x;
  if (nv >= (kPer - 1) * kThreads) {
#pragma unroll
    for (int q = 0; q < kPer - 1; ++q) r[q].load(a + 8 * (q * kThreads + x));
  } else {
#pragma unroll
    for (int q = 0; q < kPer - 1; ++q) {
      if (q * kThreads + x < nv) r[q].load(a + 8 * (q * kThreads + x));
      else r[q].clear();
    }
  }
  const int last = (kPer - 1) * kThreads + x;
  if (last < nv) r[kPer - 1].load(a + 8 * last);
  else r[kPer - 1].clear();
}

template <typename T>
__device__ __forceinline__ double unit_squares(const T* g, int n) {
  const UnitShape<T> shape(g, n);
  Raw<T> r[kPer];
  load_unit(r, g + shape.head, shape.nv);
  const int x = shape.edge();
  const float e = x >= 0 ? elem_to_float(g[x]) : 0.f;
  float s = e * e;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    float v[8];
    r[q].values(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(v[j], v[j], s);
  }
  // fp32 squares are exact enough while no sum overflows and none that matters
  // underflows; else the thread adds them again in 64 bits
  if (s > 1e-24f && s < INFINITY) return static_cast<double>(s);
  double d = static_cast<double>(e) * static_cast<double>(e);
#pragma unroll 1
  for (int i = threadIdx.x; i < shape.nv; i += kThreads) {
    for (int j = 0; j < 8; ++j) {
      const double v = elem_to_float(g[shape.head + 8 * i + j]);
      d = fma(v, v, d);
    }
  }
  return d;
}

template <int kCap>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) grad_squares_kernel(double* __restrict__ partial,
                                                                const __grid_constant__ TensorTable<kCap> tab) {
  __shared__ double red[kThreads / 32];
  double sum = 0.0;
  // from the end: what is read again next (to be scaled, or by AdamW) is read
  // from the front, and finds the last units read here in L2
  for (int u = tab.units - 1 - static_cast<int>(blockIdx.x); u >= 0; u -= static_cast<int>(gridDim.x)) {
    const TensorRef& t = tab.t[find_tensor(tab, u)];
    const long long e0 = static_cast<long long>(u - t.unit0) * kUnit;
    const int n = static_cast<int>(min(static_cast<long long>(kUnit), t.n - e0));
    if (t.in_dtype == LLMK_F32) sum += unit_squares(static_cast<const float*>(t.in) + e0, n);
    else if (t.in_dtype == LLMK_BF16) sum += unit_squares(static_cast<const __nv_bfloat16*>(t.in) + e0, n);
    else sum += unit_squares(static_cast<const __half*>(t.in) + e0, n);
  }
  sum = block_sum_d(sum, red);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// |scale| sqrt(sum of the partials), the same in every thread.
__device__ __forceinline__ float norm_of(const double* __restrict__ partial, int n, float scale, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) s += partial[i];
  return static_cast<float>(fabs(static_cast<double>(scale)) * sqrt(block_sum_d(s, red)));
}

__global__ void __launch_bounds__(kThreads) grad_norm_kernel(float* __restrict__ norm, const double* __restrict__ partial,
                                                             int n, float scale) {
  __shared__ double red[kThreads / 32];
  grid_wait();
  const float v = norm_of(partial, n, scale, red);
  if (threadIdx.x == 0) *norm = v;
}

template <typename In, typename Out>
__device__ __forceinline__ void unit_scale(Out* out, const In* g, int n, float k) {
  if (static_cast<const void*>(out) == static_cast<const void*>(g) && k == 1.f) return;  // nothing changes
  const UnitShape<In> shape(g, n);
  Out* o = out + shape.head;
  const bool wide = (reinterpret_cast<uintptr_t>(o) & 15) == 0;
  Raw<In> r[kPer];  // every load ahead of the first store: out may be g, which keeps the compiler from moving them
  load_unit(r, g + shape.head, shape.nv);
  const int x = shape.edge();
  if (x >= 0) elem_store(out + x, elem_to_float(g[x]) * k);
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int i = q * kThreads + threadIdx.x;
    if (i >= shape.nv) break;
    float v[8];
    r[q].values(v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= k;
    if (wide) {
      store8v(o + 8 * i, v);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) elem_store(o + 8 * i + j, v[j]);
    }
  }
}

// partials = 0: the norm is there already.
template <int kCap>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) grad_scale_kernel(float* __restrict__ norm, const double* __restrict__ partial,
                                                              int partials, float max_norm,
                                                              const __grid_constant__ TensorTable<kCap> tab) {
  __shared__ double red[kThreads / 32];
  grid_wait();  // not released early: the blocks set up would take room from the sums (250 -> 276 us)
  const float v = partials ? norm_of(partial, partials, 1.f, red) : *norm;
  if (partials && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float q = max_norm / (v + 1e-6f);
  const float k = q > 1.f ? 1.f : q;  // NaN stays NaN
  for (int u = blockIdx.x; u < tab.units; u += gridDim.x) {
    const TensorRef& t = tab.t[find_tensor(tab, u)];
    const long long e0 = static_cast<long long>(u - t.unit0) * kUnit;
    const int n = static_cast<int>(min(static_cast<long long>(kUnit), t.n - e0));
    if (t.in_dtype == LLMK_F32) {
      unit_scale(static_cast<float*>(t.out) + e0, static_cast<const float*>(t.in) + e0, n, k);
    } else if (t.in_dtype == LLMK_BF16) {
      const auto* g = static_cast<const __nv_bfloat16*>(t.in) + e0;
      if (t.out_dtype == LLMK_F32) unit_scale(static_cast<float*>(t.out) + e0, g, n, k);
      else unit_scale(static_cast<__nv_bfloat16*>(t.out) + e0, g, n, k);
    } else {
      const auto* g = static_cast<const __half*>(t.in) + e0;
      if (t.out_dtype == LLMK_F32) unit_scale(static_cast<float*>(t.out) + e0, g, n, k);
      else unit_scale(static_cast<__half*>(t.out) + e0, g, n, k);
    }
  }
}

size_t elem_size(llmk_dtype t) { return t == LLMK_F32 ? 4 : 2; }
bool known(llmk_dtype t) { return t == LLMK_F32 || t == LLMK_BF16 || t == LLMK_F16; }

constexpr int kMaxTable = 1000;  // 32,000 of the 32,764 parameter bytes of a launch

int partials_of_table() { return num_sms() * kCtasPerSm; }

// Whether any range that is written meets another range (a tensor listed twice,
// an `out` inside another tensor): its result would depend on timing.
bool ranges_meet(const llmk_tensor* tensors, int count) {
  struct Range {
    uintptr_t begin, end;
    bool written;
  };
  std::vector<Range> r;
  r.reserve(2 * static_cast<size_t>(count));
  for (int i = 0; i < count; ++i) {
    const llmk_tensor& t = tensors[i];
    if (t.n == 0) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(t.data), b = reinterpret_cast<uintptr_t>(t.out);
    r.push_back({b, b + t.n * elem_size(t.out_dtype), true});
    if (a != b || t.dtype != t.out_dtype) r.push_back({a, a + t.n * elem_size(t.dtype), false});
  }
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.begin < y.begin; });
  uintptr_t end_any = 0, end_written = 0;
  for (const Range& x : r) {
    if (x.begin < (x.written ? end_any : end_written)) return true;
    end_any = std::max(end_any, x.end);
    if (x.written) end_written = std::max(end_written, x.end);
  }
  return false;
}

int check_tensors(const char* what, const llmk_tensor* tensors, int count, bool writes) {
  if (!tensors || count <= 0) return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": no tensors");
  for (int i = 0; i < count; ++i) {
    const llmk_tensor& t = tensors[i];
    auto refuse = [&](int code, const char* why) {
      return fail(code, std::string(what) + ": tensor " + std::to_string(i) + ": " + why);
    };
    if (t.n < 0 || (t.n > 0 && (!t.data || (writes && !t.out)))) return refuse(LLMK_ERR_INVALID_ARG, "null or negative size");
    if (!known(t.dtype) || (writes && t.out_dtype != t.dtype && t.out_dtype != LLMK_F32))
      return refuse(LLMK_ERR_UNSUPPORTED, "fp32, bf16 or fp16, written in its own type or as fp32");
    if (reinterpret_cast<uintptr_t>(t.data) % elem_size(t.dtype) ||
        (writes && reinterpret_cast<uintptr_t>(t.out) % elem_size(t.out_dtype)))
      return refuse(LLMK_ERR_UNSUPPORTED, "not aligned to its elements");
    if (t.n > static_cast<long long>(kUnit) * (INT_MAX / 2)) return refuse(LLMK_ERR_UNSUPPORTED, "too large");
  }
  if (writes && ranges_meet(tensors, count))
    return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": a written tensor overlaps another one");
  return LLMK_OK;
}

// Tables of the given tensors, one launch each: at most kMaxTable tensors and
// INT_MAX / 2 units.
struct Span {
  int first, count, units;
};
std::vector<Span> spans_of(const llmk_tensor* tensors, int count) {
  std::vector<Span> out;
  Span s{0, 0, 0};
  for (int i = 0; i < count; ++i) {
    const long long units = (tensors[i].n + kUnit - 1) / kUnit;
    if (s.count == kMaxTable || s.units + units > INT_MAX / 2) {
      out.push_back(s);
      s = Span{i, 0, 0};
    }
    s.count += 1;
    s.units += static_cast<int>(units);
  }
  out.push_back(s);
  return out;
}

int grid_of(const Span& s) { return std::max(1, std::min(s.units, partials_of_table())); }

template <int kCap>
void fill(TensorTable<kCap>* tab, const llmk_tensor* tensors, const Span& s) {
  int unit = 0;
  for (int i = 0; i < s.count; ++i) {
    const llmk_tensor& t = tensors[s.first + i];
    tab->t[i] = TensorRef{t.data, t.out, t.n, unit, static_cast<short>(t.dtype), static_cast<short>(t.out_dtype)};
    unit += static_cast<int>((t.n + kUnit - 1) / kUnit);
  }
  tab->count = s.count;
  tab->units = s.units;
}

// f(table) with the smallest of four table capacities that holds the span: a
// launch copies its whole parameter block.
template <typename F>
void with_table(const llmk_tensor* tensors, const Span& s, F f) {
  if (s.count <= 4) {
    TensorTable<4> tab;
    fill(&tab, tensors, s);
    f(tab);
  } else if (s.count <= 40) {
    TensorTable<40> tab;
    fill(&tab, tensors, s);
    f(tab);
  } else if (s.count <= 160) {
    TensorTable<160> tab;
    fill(&tab, tensors, s);
    f(tab);
  } else {
    TensorTable<kMaxTable> tab;
    fill(&tab, tensors, s);
    f(tab);
  }
}

template <int kCap>
cudaError_t launch_squares_of(int grid, cudaStream_t s, double* partial, const TensorTable<kCap>& tab) {
  void* args[] = {&partial, const_cast<TensorTable<kCap>*>(&tab)};
  return cudaLaunchKernel(reinterpret_cast<const void*>(&grad_squares_kernel<kCap>), dim3(grid), dim3(kThreads), args, 0, s);
}

// Squares of every tensor, their number of partials to *partials. A launch that
// is refused ends the call: what follows would scale by what the workspace held.
int launch_squares(int* partials, double* partial, const llmk_tensor* tensors, const std::vector<Span>& spans, cudaStream_t s) {
  int n = 0;
  for (const Span& sp : spans) n += grid_of(sp);
  int at = n;
  for (auto sp = spans.rbegin(); sp != spans.rend(); ++sp) {
    const int grid = grid_of(*sp);
    at -= grid;
    cudaError_t e = cudaSuccess;
    with_table(tensors, *sp, [&](const auto& tab) { e = launch_squares_of(grid, s, partial + at, tab); });
    LLMK_TRY(cuda_check(e, "grad_squares_kernel"));
    count_launch();
  }
  *partials = n;
  return LLMK_OK;
}

template <int kCap>
cudaError_t launch_scale(int grid, cudaStream_t s, float* norm, const double* partial, int partials, float max_norm,
                         const TensorTable<kCap>& tab) {
  return launch_after(grad_scale_kernel<kCap>, grid, kThreads, 0, s, norm, partial, partials, max_norm, tab);
}

size_t workspace_of(const std::vector<Span>& spans) {
  size_t n = 0;
  for (const Span& s : spans) n += grid_of(s);
  return n * sizeof(double);
}

int check_workspace(const char* what, const std::vector<Span>& spans, const void* ws, size_t bytes) {
  if (!ws || !aligned16(ws) || bytes < workspace_of(spans))
    return fail(LLMK_ERR_WORKSPACE, std::string(what) + ": workspace missing or too small");
  return LLMK_OK;
}

// The host side keeps a list of spans; a caller in C gets a status, not an
// exception, when there is no memory for it.
template <typename F>
int no_throw(F f) {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return LLMK_ERR_INVALID_ARG;
  }
}

// Whether [p, p + bytes) meets a tensor that is read, or (writes) written.
bool meets(const void* p, size_t bytes, const llmk_tensor* tensors, int count, bool writes) {
  const uintptr_t begin = reinterpret_cast<uintptr_t>(p), end = begin + bytes;
  auto meet = [&](const void* t, size_t n) {
    const uintptr_t b = reinterpret_cast<uintptr_t>(t);
    return n > 0 && begin < b + n && b < end;
  };
  for (int i = 0; i < count; ++i) {
    const llmk_tensor& t = tensors[i];
    if (meet(t.data, t.n * elem_size(t.dtype)) || (writes && meet(t.out, t.n * elem_size(t.out_dtype)))) return true;
  }
  return false;
}

// The partial sums are written while the tensors are read; clipping reads the norm
// while it writes tensors, and its first block writes it while the others read the
// partial sums.
int check_scratch(const char* what, const float* norm, const void* workspace, size_t bytes, const llmk_tensor* tensors, int count,
                  bool writes) {
  if (meets(workspace, bytes, tensors, count, writes) || (writes && meets(norm, sizeof(float), tensors, count, true)))
    return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": norm or workspace overlaps a tensor");
  const uintptr_t n = reinterpret_cast<uintptr_t>(norm), w = reinterpret_cast<uintptr_t>(workspace);
  if (writes && n < w + bytes && w < n + sizeof(float))
    return fail(LLMK_ERR_INVALID_ARG, std::string(what) + ": norm overlaps the workspace");
  return LLMK_OK;
}

int grad_norm(float* norm, const llmk_tensor* tensors, int count, float scale, void* workspace, size_t workspace_bytes,
              cudaStream_t s) {
  if (!norm || !std::isfinite(scale)) return fail(LLMK_ERR_INVALID_ARG, "grad_norm: null norm or bad scale");
  LLMK_TRY(check_tensors("grad_norm", tensors, count, false));
  const auto spans = spans_of(tensors, count);
  LLMK_TRY(check_workspace("grad_norm", spans, workspace, workspace_bytes));
  LLMK_TRY(check_scratch("grad_norm", norm, workspace, workspace_of(spans), tensors, count, false));
  auto* partial = static_cast<double*>(workspace);
  int n = 0;
  LLMK_TRY(launch_squares(&n, partial, tensors, spans, s));
  LLMK_CUDA(launch_after(grad_norm_kernel, 1, kThreads, 0, s, norm, partial, n, scale));
  count_launch();
  return LLMK_OK;
}

int clip_grad_norm(float* norm, const llmk_tensor* tensors, int count, float max_norm, void* workspace,
                   size_t workspace_bytes, cudaStream_t s) {
  if (!norm || !(max_norm > 0.f)) return fail(LLMK_ERR_INVALID_ARG, "clip_grad_norm: null norm, or max_norm not above 0");
  LLMK_TRY(check_tensors("clip_grad_norm", tensors, count, true));
  const auto spans = spans_of(tensors, count);
  LLMK_TRY(check_workspace("clip_grad_norm", spans, workspace, workspace_bytes));
  LLMK_TRY(check_scratch("clip_grad_norm", norm, workspace, workspace_of(spans), tensors, count, true));
  auto* partial = static_cast<double*>(workspace);
  int n = 0;
  LLMK_TRY(launch_squares(&n, partial, tensors, spans, s));
  // Many units: a block for each, in order, streams faster than a fixed grid that
  // walks them (124M bf16 gradients 128 -> 122 us, fp32 267 -> 237 us), but its
  // prologue cannot be the sum of the partials. Few: one launch less counts.
  long long units = 0;
  for (const Span& sp : spans) units += sp.units;
  const bool many = units >= 2048;
  if (many) {
    LLMK_CUDA(launch_after(grad_norm_kernel, 1, kThreads, 0, s, norm, partial, n, 1.f));
    count_launch();
  }
  for (const Span& sp : spans) {
    cudaError_t e = cudaSuccess;
    const int grid = many ? std::max(1, sp.units) : grid_of(sp);
    with_table(tensors, sp, [&](const auto& tab) { e = launch_scale(grid, s, norm, partial, many ? 0 : n, max_norm, tab); });
    LLMK_CUDA(e);
    count_launch();
  }
  return LLMK_OK;
}

}  // namespace
}  // namespace llmk

using namespace llmk;

extern "C" {

size_t llmk_grad_norm_workspace(const llmk_tensor* tensors, int count) {
  if (!tensors || count <= 0) return 0;
  size_t bytes = 0;
  return no_throw([&] { return bytes = workspace_of(spans_of(tensors, count)), LLMK_OK; }) == LLMK_OK ? bytes : 0;
}

int llmk_grad_norm(float* norm, const llmk_tensor* tensors, int count, float scale, void* workspace,
                   size_t workspace_bytes, void* stream) {
  return no_throw([&] {
    return grad_norm(norm, tensors, count, scale, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}

int llmk_clip_grad_norm(float* norm, const llmk_tensor* tensors, int count, float max_norm, void* workspace,
                        size_t workspace_bytes, void* stream) {
  return no_throw([&] {
    return clip_grad_norm(norm, tensors, count, max_norm, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
