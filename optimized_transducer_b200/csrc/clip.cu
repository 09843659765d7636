// The norm of all gradients of a model together, and clipping by it:
//
//   norm = (sum over all tensors and elements of |g|^p)^(1/p),   p = 1, 2 or infinity
//   out  = g * min(1, max_norm / (norm + 1e-6))
//
// The step between a loss's backward pass and the optimizer; the reference leaves it to
// torch.nn.utils.clip_grad_norm_, whose definition this is (the 1e-6 included).
//
// Two launches for up to kLargeTable tensors: norm_kernel reads every gradient once and
// leaves one partial sum per block, in double; apply_kernel's blocks add those partials, in
// a fixed order, each for itself, and scale the gradients.  Nothing waits on a counter, no
// sum depends on the order in which blocks run, and when the factor is 1 and the gradients
// stay where they are apply_kernel ends there.  Bound by HBM: one read for the norm, one
// read (from L2 what still is there: it runs over the tensors backwards) and one write for
// the clipping.  400 M float gradients into other buffers: 0.81 ms for 4.8 GB, 5.9 TB/s; 90 M
// bfloat16 in 600 tensors into float buffers: 0.14 ms.
//
// The tensors' pointers travel as kernel arguments, so a call copies nothing to the device
// and a captured call replays with the pointers it was captured with.
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <new>
#include <vector>

#include "ot_common.cuh"

namespace otb {

namespace {

constexpr int kClipThreads = 256;
constexpr int kClipBlocksPerSm = 8;
constexpr int kSmallTable = 48, kLargeTable = 1000;  // 32 bytes per tensor; kernel arguments end at 32 764 bytes

enum : uint8_t { kF32 = 0, kF64 = 1, kBf16 = 2, kF16 = 3 };

struct ClipTensor {
  const void *grad;
  void *out;
  uint64_t count_and_types;  // count << 8 | type of out << 4 | type of grad
  uint32_t first_chunk;      // chunks of the tensors before this one
  uint32_t pad;
};

template <int kMax> struct ClipTable {
  int tensors;
  uint32_t chunks;
  int64_t chunk;  // elements per chunk
  ClipTensor t[kMax];
};
static_assert(sizeof(ClipTable<kLargeTable>) + 128 <= 32764, "the table must fit the kernel arguments");

// The tensor that chunk c lies in: the last one whose first chunk is not behind c.
template <int kMax> __device__ __forceinline__ int find_tensor(const ClipTable<kMax> &tab, uint32_t c) {
  int lo = 0, hi = tab.tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].first_chunk <= c) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T> struct Vec16 { T v[16 / sizeof(T)]; };
template <typename T> __device__ __forceinline__ Vec16<T> load16(const T *p) {
  const uint4 a = *reinterpret_cast<const uint4 *>(p);
  Vec16<T> r;
  memcpy(&r, &a, 16);
  return r;
}

template <typename T> __device__ __forceinline__ auto widen(T x) { return to_float(x); }
template <> __device__ __forceinline__ auto widen(double x) { return x; }

// Running sum of |g|^p of one thread (p = 1, 2), or the largest |g|.  16- and 32-bit
// elements are summed in float over one group of vectors at a time and the group's sum goes
// to a double; a group whose float sum overflowed, or is so small that squares may have been
// lost, is taken again in double, so the norm is right wherever it is representable.
template <int kNorm> struct Gather {
  double sum = 0.0;
  uint32_t top = 0u;      // kNorm == 0: bits of |g| order as integers do, NaN above infinity
  double top64 = 0.0;     // ... of 64-bit elements; a NaN stays
  __device__ __forceinline__ static float term(float x) { return kNorm == 2 ? x * x : fabsf(x); }
  __device__ __forceinline__ static double term(double x) { return kNorm == 2 ? x * x : fabs(x); }
  template <int N> __device__ __forceinline__ void group(const float (&x)[N]) {
    if constexpr (kNorm == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    } else {
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < N; ++i) s[i & 3] = kNorm == 2 ? fmaf(x[i], x[i], s[i & 3]) : s[i & 3] + fabsf(x[i]);
      const float all = (s[0] + s[1]) + (s[2] + s[3]);
      if (all < 3e38f && (kNorm == 1 || all > 1e-24f)) {
        sum += (double)all;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) sum += term((double)x[i]);
      }
    }
  }
  template <int N> __device__ __forceinline__ void group(const double (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (kNorm == 0) top64 = fabs(x[i]) > top64 || x[i] != x[i] ? fabs(x[i]) : top64;
      else sum += term(x[i]);
    }
  }
  __device__ __forceinline__ double result() const {
    if constexpr (kNorm == 0) {
      const double a = (double)__uint_as_float(top);
      if (a != a || top64 != top64) return __longlong_as_double(0x7ff8000000000000LL);
      return fmax(a, top64);
    }
    return sum;
  }
};

// p = 1, 2: a + b; p = infinity: the larger one, a NaN if there is one.
template <int kNorm> __device__ __forceinline__ double join(double a, double b) {
  if constexpr (kNorm == 0) return a != a ? a : (b > a || b != b ? b : a);
  return a + b;
}

template <int kNorm, typename T>
__device__ __forceinline__ void gather_chunk(Gather<kNorm> &g, const T *p, int64_t n) {
  using W = decltype(widen(T{}));
  constexpr int kPer = 16 / sizeof(T);
  const int64_t off = (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int64_t)sizeof(T);
  const int head = (int)(off < n ? off : n);
  const int64_t vecs = (n - head) / kPer;
  const int tail = (int)(n - head - vecs * kPer);
  if ((int)threadIdx.x < head) { const W x[1] = {widen(p[threadIdx.x])}; g.group(x); }
  const T *body = p + head;
  constexpr int kUnroll = 4;
  int64_t i = threadIdx.x;
  for (; i + (kUnroll - 1) * kClipThreads < vecs; i += kUnroll * kClipThreads) {
    Vec16<T> v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = load16(body + (i + u * kClipThreads) * kPer);
    W x[kUnroll * kPer];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int k = 0; k < kPer; ++k) x[u * kPer + k] = widen(v[u].v[k]);
    g.group(x);
  }
  for (; i < vecs; i += kClipThreads) {
    const Vec16<T> v = load16(body + i * kPer);
    W x[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) x[k] = widen(v.v[k]);
    g.group(x);
  }
  if ((int)threadIdx.x < tail) { const W x[1] = {widen(body[vecs * kPer + threadIdx.x])}; g.group(x); }
}

template <int kNorm, int kMax>
__global__ void __launch_bounds__(kClipThreads)
norm_kernel(const __grid_constant__ ClipTable<kMax> tab, double *__restrict__ partial) {
  __shared__ double s[kClipThreads / 32];
  pdl_wait();
  pdl_trigger();
  Gather<kNorm> g;
  for (uint32_t c = blockIdx.x; c < tab.chunks; c += gridDim.x) {
    const ClipTensor &t = tab.t[find_tensor(tab, c)];
    const int64_t at = (int64_t)(c - t.first_chunk) * tab.chunk;
    const int64_t n = min(tab.chunk, (int64_t)(t.count_and_types >> 8) - at);
    switch (t.count_and_types & 15) {
      case kF64: gather_chunk(g, static_cast<const double *>(t.grad) + at, n); break;
      case kBf16: gather_chunk(g, static_cast<const __nv_bfloat16 *>(t.grad) + at, n); break;
      case kF16: gather_chunk(g, static_cast<const __half *>(t.grad) + at, n); break;
      default: gather_chunk(g, static_cast<const float *>(t.grad) + at, n);
    }
  }
  double v = g.result();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<kNorm>(v, __shfl_xor_sync(kFull, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kClipThreads / 32; ++w) v = join<kNorm>(v, s[w]);
    partial[blockIdx.x] = v;
  }
}

// The norm from the partials, the same bits in every block that asks.
template <int kNorm>
__device__ __forceinline__ double total_norm(const double *__restrict__ partial, int partials) {
  __shared__ double s[kClipThreads / 32];
  double v = 0.0;
  for (int i = threadIdx.x; i < partials; i += kClipThreads) v = join<kNorm>(v, partial[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = join<kNorm>(v, __shfl_xor_sync(kFull, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kClipThreads / 32; ++w) v = join<kNorm>(v, s[w]);
  return kNorm == 2 ? sqrt(v) : v;
}

template <int kNorm>
__global__ void __launch_bounds__(kClipThreads)
finish_norm_kernel(const double *__restrict__ partial, int partials, float *norm_out) {
  pdl_wait();
  pdl_trigger();
  const double norm = total_norm<kNorm>(partial, partials);
  if (threadIdx.x == 0) *norm_out = (float)norm;
}

template <typename O, typename W> __device__ __forceinline__ O narrow(W x) { return (O)(float)x; }
template <> __device__ __forceinline__ double narrow<double, double>(double x) { return x; }
template <> __device__ __forceinline__ double narrow<double, float>(float x) { return (double)x; }
template <> __device__ __forceinline__ float narrow<float, double>(double x) { return (float)x; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16, double>(double x) { return __double2bfloat16(x); }
template <> __device__ __forceinline__ __half narrow<__half, double>(double x) { return __double2half(x); }

// out = g * factor in the wider of float and the element's type, rounded once.  Vectors of
// kPer elements: 16 bytes of the wider of the two types, when both sides are aligned for
// them behind the same head; single elements otherwise.
template <typename T, typename O>
__device__ __forceinline__ void scale_chunk(const T *p, O *out, int64_t n, double factor64) {
  using W = decltype(widen(T{}));
  const W factor = (W)factor64;
  constexpr int kPer = 16 / (sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O));
  struct alignas(sizeof(T) * kPer) In { T v[kPer]; };
  struct alignas(sizeof(O) * kPer) Out { O v[kPer]; };
  int64_t head = (int64_t)((sizeof(In) - (reinterpret_cast<uintptr_t>(p) % sizeof(In))) % sizeof(In)) / (int64_t)sizeof(T);
  if (head > n) head = n;
  const bool vec = reinterpret_cast<uintptr_t>(out + head) % sizeof(Out) == 0;
  if (!vec) head = n;
  for (int64_t i = threadIdx.x; i < head; i += kClipThreads) out[i] = narrow<O>(widen(p[i]) * factor);
  if (!vec) return;
  const int64_t vecs = (n - head) / kPer;
  const In *src = reinterpret_cast<const In *>(p + head);
  Out *dst = reinterpret_cast<Out *>(out + head);
  constexpr int kUnroll = 4;
  int64_t i = threadIdx.x;
  for (; i + (kUnroll - 1) * kClipThreads < vecs; i += kUnroll * kClipThreads) {
    In v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = src[i + u * kClipThreads];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      Out o;
#pragma unroll
      for (int k = 0; k < kPer; ++k) o.v[k] = narrow<O>(widen(v[u].v[k]) * factor);
      dst[i + u * kClipThreads] = o;
    }
  }
  for (; i < vecs; i += kClipThreads) {
    const In v = src[i];
    Out o;
#pragma unroll
    for (int k = 0; k < kPer; ++k) o.v[k] = narrow<O>(widen(v.v[k]) * factor);
    dst[i] = o;
  }
  for (int64_t k = head + vecs * kPer + threadIdx.x; k < n; k += kClipThreads) out[k] = narrow<O>(widen(p[k]) * factor);
}

template <typename T>
__device__ __forceinline__ void scale_to(const T *p, const ClipTensor &t, int64_t at, int64_t n, double factor) {
  switch ((t.count_and_types >> 4) & 15) {
    case kF64: scale_chunk(p + at, static_cast<double *>(t.out) + at, n, factor); break;
    case kBf16: scale_chunk(p + at, static_cast<__nv_bfloat16 *>(t.out) + at, n, factor); break;
    case kF16: scale_chunk(p + at, static_cast<__half *>(t.out) + at, n, factor); break;
    default: scale_chunk(p + at, static_cast<float *>(t.out) + at, n, factor);
  }
}

template <int kNorm, int kMax>
__global__ void __launch_bounds__(kClipThreads)
apply_kernel(const __grid_constant__ ClipTable<kMax> tab, const double *__restrict__ partial, int partials,
             double max_norm, bool in_place, float *norm_out) {
  pdl_wait();
  pdl_trigger();
  const double norm = total_norm<kNorm>(partial, partials);
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  // a NaN norm makes the factor a NaN, an infinite one makes it 0
  const double ratio = max_norm / (norm + 1e-6);
  const double factor = ratio >= 1.0 ? 1.0 : ratio;  // rounded to float where the elements are
  if (in_place && factor == 1.0) return;
  for (uint32_t i = blockIdx.x; i < tab.chunks; i += gridDim.x) {
    const uint32_t c = tab.chunks - 1 - i;  // what the norm pass read last is still in L2
    const ClipTensor &t = tab.t[find_tensor(tab, c)];
    const int64_t at = (int64_t)(c - t.first_chunk) * tab.chunk;
    const int64_t n = min(tab.chunk, (int64_t)(t.count_and_types >> 8) - at);
    switch (t.count_and_types & 15) {
      case kF64: scale_to(static_cast<const double *>(t.grad), t, at, n, factor); break;
      case kBf16: scale_to(static_cast<const __nv_bfloat16 *>(t.grad), t, at, n, factor); break;
      case kF16: scale_to(static_cast<const __half *>(t.grad), t, at, n, factor); break;
      default: scale_to(static_cast<const float *>(t.grad), t, at, n, factor);
    }
  }
}

int fail(int code, const char *fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  set_last_error(msg);
  return code;
}

int type_code(int32_t type) {
  switch (type) {
    case 0: return kF32;
    case OT_B200_FP64: return kF64;
    case OT_B200_BF16: return kBf16;
    case OT_B200_FP16: return kF16;
    default: return -1;
  }
}
size_t type_size(int code) { return code == kF32 ? 4 : (code == kF64 ? 8 : 2); }

struct Span {
  uintptr_t begin, end;
  bool written;
};

// Whether something that the call writes overlaps something else that it reads or writes.
bool overlapping(std::vector<Span> &spans) {
  std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;
  for (const Span &s : spans) {
    if (s.begin < (s.written ? any : written)) return true;
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return false;
}

int max_blocks() { return kClipBlocksPerSm * sm_count(); }

// One table's worth of tensors.
template <int kNorm, int kMax>
cudaError_t launch_norm(const ClipTable<kMax> &tab, double *partial, int *blocks, cudaStream_t s) {
  *blocks = (int)std::min<int64_t>(tab.chunks, max_blocks());
  return launch_pdl(norm_kernel<kNorm, kMax>, (unsigned)*blocks, (unsigned)kClipThreads, 0, s, tab, partial);
}

template <int kMax>
void fill(ClipTable<kMax> &tab, const std::vector<ClipTensor> &all, size_t from, size_t to) {
  int64_t total = 0;
  for (size_t i = from; i < to; ++i) total += (int64_t)(all[i].count_and_types >> 8);
  // chunks small enough that a small model fills the device, large enough that a block
  // seldom looks a tensor up
  int64_t chunk = (total / (2 * (int64_t)max_blocks()) + 1023) / 1024 * 1024;
  tab.chunk = std::min<int64_t>(std::max<int64_t>(chunk, 2048), 65536);
  tab.tensors = (int)(to - from);
  uint32_t chunks = 0;
  for (size_t i = from; i < to; ++i) {
    tab.t[i - from] = all[i];
    tab.t[i - from].first_chunk = chunks;
    chunks += (uint32_t)(((int64_t)(all[i].count_and_types >> 8) + tab.chunk - 1) / tab.chunk);
  }
  tab.chunks = chunks;
}

template <int kNorm, int kMax>
cudaError_t run_tables(const std::vector<ClipTensor> &all, double *partial, bool apply, bool in_place, double max_norm,
                       float *norm_out, cudaStream_t s) {
  ClipTable<kMax> tab;
  int used = 0;
  for (size_t from = 0; from < all.size(); from += kMax) {
    const size_t to = std::min(all.size(), from + kMax);
    fill(tab, all, from, to);
    int blocks = 0;
    const cudaError_t e = launch_norm<kNorm, kMax>(tab, partial + used, &blocks, s);
    if (e != cudaSuccess) return e;
    used += blocks;
  }
  if (!apply || all.empty())
    return launch_pdl(finish_norm_kernel<kNorm>, 1u, (unsigned)kClipThreads, 0, s, (const double *)partial, used, norm_out);
  for (size_t to = all.size(); to > 0;) {  // the last table first: its end is what L2 holds
    const size_t from = (to - 1) / kMax * kMax;
    if (all.size() > kMax) fill(tab, all, from, to);
    const cudaError_t e = launch_pdl(apply_kernel<kNorm, kMax>, (unsigned)std::min<int64_t>(tab.chunks, max_blocks()),
                                     (unsigned)kClipThreads, 0, s, tab, (const double *)partial, used, max_norm, in_place,
                                     from == 0 ? norm_out : (float *)nullptr);
    if (e != cudaSuccess) return e;
    to = from;
  }
  return cudaSuccess;
}

template <int kNorm>
cudaError_t run_norm(const std::vector<ClipTensor> &all, double *partial, bool apply, bool in_place, double max_norm,
                     float *norm_out, cudaStream_t s) {
  if (all.size() <= (size_t)kSmallTable) return run_tables<kNorm, kSmallTable>(all, partial, apply, in_place, max_norm, norm_out, s);
  return run_tables<kNorm, kLargeTable>(all, partial, apply, in_place, max_norm, norm_out, s);
}

int clip(int32_t n, const void *const *grads, const int64_t *counts, const int32_t *types, void *const *outs,
         const int32_t *out_types, int32_t norm_kind, int32_t apply, double max_norm, void *d_workspace,
         uint64_t workspace_bytes, float *d_norm, void *stream) {
  if (n < 0 || (n > 0 && (!grads || !counts || !types)) || !d_norm)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: NULL pointer or a negative number of tensors");
  if ((outs == nullptr) != (out_types == nullptr) || (outs && !apply))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: outs and out_types come together, and with apply only");
  if (norm_kind != OT_B200_NORM_INF && norm_kind != OT_B200_NORM_1 && norm_kind != OT_B200_NORM_2)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: unknown norm");
  if (apply && !(max_norm >= 0.0))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: max_norm must not be negative or a NaN");
  uint64_t need = 0;
  const int rc = ot_b200_clip_workspace_bytes(n, &need);
  if (rc) return rc;
  if (!d_workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(d_workspace) % 8 != 0)
    return fail(OT_B200_ERR_WORKSPACE, "ot_b200_clip_gradients: workspace missing, misaligned or smaller than %llu bytes", (unsigned long long)need);
  std::vector<ClipTensor> all;
  std::vector<Span> spans;
  all.reserve((size_t)n);
  spans.reserve(2 * (size_t)n);
  bool in_place = true;
  for (int32_t i = 0; i < n; ++i) {
    const int t = type_code(types[i]), o = outs ? type_code(out_types[i]) : t;
    if (t < 0 || o < 0) return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: tensor %d has an unknown type", i);
    if (counts[i] < 0 || counts[i] >= ((int64_t)1 << 46))
      return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: tensor %d has a count out of range", i);
    if (counts[i] == 0) continue;
    void *out = outs ? outs[i] : const_cast<void *>(grads[i]);
    const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i]), b = reinterpret_cast<uintptr_t>(out);
    if (!a || !b || a % type_size(t) || b % type_size(o))
      return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: tensor %d is NULL or not aligned to its type", i);
    const bool same = a == b && t == o;
    in_place = in_place && same;
    spans.push_back(Span{a, a + counts[i] * type_size(t), apply && same});
    if (!same) spans.push_back(Span{b, b + counts[i] * type_size(o), true});
    all.push_back(ClipTensor{grads[i], out, (uint64_t)counts[i] << 8 | (uint64_t)o << 4 | (uint64_t)t, 0u, 0u});
  }
  if (apply && overlapping(spans))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: tensors overlap (one is listed twice, or an output lies over another tensor)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  double *partial = static_cast<double *>(d_workspace);
  cudaError_t e;
  if (norm_kind == OT_B200_NORM_2) e = run_norm<2>(all, partial, apply != 0, in_place, max_norm, d_norm, s);
  else if (norm_kind == OT_B200_NORM_1) e = run_norm<1>(all, partial, apply != 0, in_place, max_norm, d_norm, s);
  else e = run_norm<0>(all, partial, apply != 0, in_place, max_norm, d_norm, s);
  if (e != cudaSuccess) return fail(OT_B200_ERR_CUDA, "ot_b200_clip_gradients: %s", cudaGetErrorString(e));
  return OT_B200_OK;
}

}  // namespace

}  // namespace otb

using namespace otb;

extern "C" {

int ot_b200_clip_workspace_bytes(int32_t n, uint64_t *bytes_out) {
  if (n < 0 || !bytes_out) return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_workspace_bytes: n is negative or bytes_out NULL");
  const uint64_t tables = ((uint64_t)n + kLargeTable - 1) / kLargeTable;
  *bytes_out = (tables > 0 ? tables : 1) * (uint64_t)max_blocks() * sizeof(double);
  return OT_B200_OK;
}

int ot_b200_clip_gradients(int32_t n, const void *const *grads, const int64_t *counts, const int32_t *types,
                           void *const *outs, const int32_t *out_types, int32_t norm_kind, int32_t apply,
                           double max_norm, void *d_workspace, uint64_t workspace_bytes, float *d_norm, void *stream) {
  try {
    return clip(n, grads, counts, types, outs, out_types, norm_kind, apply, max_norm, d_workspace, workspace_bytes, d_norm, stream);
  } catch (const std::exception &) {
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_clip_gradients: no host memory for the tensors' table");
  }
}

}  // extern "C"
