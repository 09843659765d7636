// One symbol per row of logits, drawn with a given uniform number from the softmax at a
// temperature, after top-k, top-p and min-p:
//
//   w_i = exp((x_i - max x) / temperature)
//   top_k   keeps the k largest logits
//   top_p   keeps, of what is left, every i with  sum of w before i  <  top_p * sum of w
//   min_p   keeps, of what is left, every i with  w_i >= min_p
//   token   the first index, in index order, at which the kept w sum to more than u * (their sum)
//
// "Before" is the order of falling logits, the lower index first among equal ones; every
// filter keeps a prefix of that order, and its first element always.  The reference has
// no counterpart: decoding lies outside its loss.
//
// Whole numbers have to come out right, so the answer is DEFINED in 64 bits.  The work is
// done in float: the float sum of any subset of the w is off by at most
//     eps * (sum of w)
// where a row of up to 1024 has eps = (3 ln V + n + 6) * 2^-24: 2^-24 per unit of the
// exponent's argument from the subtraction, the factor and the product, sum w_i |ln w_i|
// <= ln V * sum w_i, ex2.approx is good to 2^-22, and n additions lie on the longest path.
// In wider rows more sums come close to each other: there the argument is carried in two
// floats and sums of four weights are added in double, so eps = 9 * 2^-24.  A
// comparison of two such sums that is closer than twice that is made again with double sums
// (few rows at 500 symbols, most at 100 000).  Nothing is sorted: a filter's border is a
// logit, found by bisection on the values and then between the logits that are still in
// question.
#include <cooperative_groups.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

#include "ot_common.cuh"

namespace cg = cooperative_groups;

namespace otb {

namespace {

struct SampleArgs {
  const void *logits;
  int64_t stride;        // elements from one row to the next
  int64_t rows;
  int V;
  const float *u;
  const float *temperature, *top_p, *min_p;  // one value per row, or NULL: the scalar below
  const int32_t *top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  float eps;
  bool vec;              // four logits may be loaded at once, and V is a multiple of four
  int32_t *token;
  float *logprob;
};

constexpr float kLeastNormal = 1.17549435e-38f;  // 2^-126

__device__ __forceinline__ float inf_f() { return __int_as_float(0x7f800000); }

__device__ __forceinline__ float warp_max_f(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_min_f(float v) {
  float r;
  asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// What one pass over the row yields: a sum, a count, the least and the largest of the
// logits that the pass asks for.
enum { kSum = 1, kCount = 2, kEnds = 4 };
template <typename A> struct Pass {
  A sum;
  int count;
  float least, most;
};

// The threads that share a row: kWarps warps of one block, or of each of kCtas blocks of a
// cluster.  Reductions and searches give every thread the same answer, in a fixed order of
// additions.  The scratch is used in two halves in turn, so one barrier per reduction will do.
template <int kWarps, int kCtas> struct Team {
  using Sum = typename std::conditional<kWarps == 1, float, double>::type;
  struct Scratch {
    Pass<double> warp_part[2][kWarps];
    Pass<double> cta_part[2][kCtas];
    double table[16][kWarps];
    int index;
    double before, upto;
    struct { int index; double before, upto; } found[2][kCtas];
  };
  Scratch &s;
  int half = 0;
  __device__ explicit Team(Scratch &scratch) : s(scratch) {}

  // kWhat: which fields are asked for (kSum, kCount, kEnds); the others come back unreduced.
  template <int kWhat, typename A> __device__ __forceinline__ static Pass<A> across(Pass<A> p) {
    if (kWhat & kSum) p.sum = warp_sum(p.sum);
    if (kWhat & kCount) p.count = __reduce_add_sync(kFull, p.count);
    if (kWhat & kEnds) {
      p.least = warp_min_f(p.least);
      p.most = warp_max_f(p.most);
    }
    return p;
  }
  // The same over kN entries (a power of two) that a reduction has left in shared memory.
  // Lane l takes entry l modulo kN, so a sum needs log2(kN) exchanges and every lane has it.
  template <int kWhat, typename A, int kN> __device__ __forceinline__ static Pass<A> over(const Pass<double> (&part)[kN]) {
    const int lane = threadIdx.x & 31;
    const Pass<double> &t = part[lane % kN];
    Pass<A> p{A(0), 0, 0.f, 0.f};
    if (kWhat & kSum) {
      p.sum = (A)t.sum;
#pragma unroll
      for (int o = kN / 2; o > 0; o >>= 1) p.sum += __shfl_xor_sync(kFull, p.sum, o);
    }
    if (kWhat & kCount) p.count = __reduce_add_sync(kFull, lane < kN ? t.count : 0);
    if (kWhat & kEnds) {
      p.least = warp_min_f(t.least);
      p.most = warp_max_f(t.most);
    }
    return p;
  }
  template <int kWhat, typename A> __device__ __forceinline__ Pass<A> reduce(Pass<A> p) {
    p = across<kWhat>(p);
    if constexpr (kWarps > 1) {
      half ^= 1;
      if ((threadIdx.x & 31) == 0) s.warp_part[half][threadIdx.x >> 5] = Pass<double>{(double)p.sum, p.count, p.least, p.most};
      __syncthreads();
      p = over<kWhat, A>(s.warp_part[half]);
    }
    if constexpr (kCtas > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (threadIdx.x < kCtas)
        *cluster.map_shared_rank(&s.cta_part[half][cluster.block_rank()], threadIdx.x) = Pass<double>{(double)p.sum, p.count, p.least, p.most};
      cluster.sync();
      p = over<kWhat, A>(s.cta_part[half]);
    }
    return p;
  }

  __device__ __forceinline__ float max_with_nan(float v) {
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(v) : "f"(v));
    if constexpr (kWarps > 1) {  // as a count and a maximum: the reduction of several warps drops a NaN
      const Pass<float> p = reduce<kCount | kEnds>(Pass<float>{0.f, v != v ? 1 : 0, 0.f, v});
      return p.count ? __int_as_float(0x7fffffff) : p.most;
    }
    return v;
  }

  // The first element, in index order, at which the running sum of value(x, w) exceeds
  // `target`: its index, and the sums before and after it.  Index -1 when there is none.
  // Element e = 4 j + q of thread t has the index first + 4 (j * threads + t) + q.
  template <typename A> struct Found { int index; A before, upto; };

  // kRolled: value() is costly and few rows ask for it, so the loop is not unrolled, and
  // `target` is a fraction of the sum of all values.
  template <int J, typename A, bool kRolled = false, typename F>
  __device__ __forceinline__ Found<A> locate(A target, int first, const float (&x)[4 * J], const float (&w)[4 * J], F value) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    A part[J];
    if constexpr (kRolled) {
      float copy[4 * J];
#pragma unroll
      for (int e = 0; e < 4 * J; ++e) copy[e] = x[e];
#pragma unroll 1
      for (int j = 0; j < J; ++j)
        part[j] = (value(copy[4 * j], 0.f) + value(copy[4 * j + 1], 0.f)) + (value(copy[4 * j + 2], 0.f) + value(copy[4 * j + 3], 0.f));
      A all = A(0);
#pragma unroll
      for (int j = 0; j < J; ++j) all += part[j];
      target = target * reduce<kSum>(Pass<A>{all, 0, 0.f, 0.f}).sum;
    } else {
#pragma unroll
     for (int j = 0; j < J; ++j) {
      auto v = value(x[4 * j], w[4 * j]);
#pragma unroll
      for (int q = 1; q < 4; ++q) v += value(x[4 * j + q], w[4 * j + q]);
      part[j] = (A)v;
     }
    }
    Found<A> f{-1, A(0), A(0)};
    if constexpr (kWarps == 1) {
      A base = A(0), start = A(0);
      int chunk = -1;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const A all = warp_sum(part[j]);
        if (chunk < 0 && base + all > target) { chunk = j; start = base; }
        base += all;
      }
      if (chunk >= 0) f = inside<J>(chunk, start, part, target, first, 0, x, w, value);
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const A all = warp_sum(part[j]);
        if (lane == 0) s.table[j][warp] = (double)all;
      }
      if (threadIdx.x == 0) s.index = -1;
      __syncthreads();
      // every warp walks the table; the one whose entry holds the border looks inside
      A base = A(0);
      if constexpr (kCtas > 1) {  // the sums of the blocks before this one
        A mine = A(0);
        for (int e = 0; e < J * kWarps; ++e) mine += (A)s.table[e / kWarps][e % kWarps];
        half ^= 1;
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x < kCtas)
          cluster.map_shared_rank(&s.cta_part[half][cluster.block_rank()], threadIdx.x)->sum = (double)mine;
        cluster.sync();
        for (int c = 0; c < (int)cluster.block_rank(); ++c) base += (A)s.cta_part[half][c].sum;
      }
      for (int e0 = 0; e0 < J * kWarps; e0 += 32) {
        const int e = e0 + lane;
        A run = e < J * kWarps ? (A)s.table[e / kWarps][e % kWarps] : A(0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const A up = __shfl_up_sync(kFull, run, o);
          if (lane >= o) run += up;
        }
        const unsigned hit = __ballot_sync(kFull, base + run > target);
        if (hit) {
          const int l = __ffs(hit) - 1;
          const A upto_l = __shfl_sync(kFull, run, l > 0 ? l - 1 : 0);
          const int where = e0 + l;
          if (where < J * kWarps && where % kWarps == warp) {
            const A b = base + (l > 0 ? upto_l : A(0));
            f = inside<J>(where / kWarps, b, part, target, first, warp, x, w, value);
            if (lane == 0) { s.index = f.index; s.before = (double)f.before; s.upto = (double)f.upto; }
          }
          break;
        }
        base += __shfl_sync(kFull, run, 31);
      }
      __syncthreads();
      f = Found<A>{s.index, (A)s.before, (A)s.upto};
      if constexpr (kCtas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x < kCtas) {
          auto *there = cluster.map_shared_rank(&s.found[half][cluster.block_rank()], threadIdx.x);
          there->index = f.index;
          there->before = (double)f.before;
          there->upto = (double)f.upto;
        }
        cluster.sync();
        f.index = -1;
        for (int c = 0; c < kCtas; ++c)
          if (f.index < 0 && s.found[half][c].index >= 0)
            f = Found<A>{s.found[half][c].index, (A)s.found[half][c].before, (A)s.found[half][c].upto};
      }
      __syncthreads();  // table and index may be written again
    }
    return f;
  }

  // The element of chunk j of one warp at which base + the running sum exceeds target.
  template <int J, typename A, typename F>
  __device__ __forceinline__ Found<A> inside(int j, A base, const A (&part)[J], A target, int first, int warp,
                                             const float (&x)[4 * J], const float (&w)[4 * J], F value) {
    const int lane = threadIdx.x & 31;
    A run = A(0);
    float xs[4], ws[4];
#pragma unroll
    for (int i = 0; i < J; ++i)
      if (i == j) {
        run = part[i];
#pragma unroll
        for (int q = 0; q < 4; ++q) { xs[q] = x[4 * i + q]; ws[q] = w[4 * i + q]; }
      }
    // the scan's order of additions may fall short of the chunk's sum by a rounding: then
    // the last lane that has any weight
    const unsigned any = __ballot_sync(kFull, run > A(0));
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const A up = __shfl_up_sync(kFull, run, o);
      if (lane >= o) run += up;
    }
    const unsigned hit = __ballot_sync(kFull, base + run > target);
    A before_lane = __shfl_up_sync(kFull, run, 1);
    if (lane == 0) before_lane = A(0);
    const int l = hit ? __ffs(hit) - 1 : 31 - __clz(any | 1u);
    A c = base + before_lane, before = c;
    int at = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const A v = (A)value(xs[q], ws[q]);
      if (v > A(0) && (q == 0 || !(c > target))) { before = c; c += v; at = q; }
    }
    Found<A> f;
    f.index = __shfl_sync(kFull, first + 4 * ((j * kWarps + warp) * 32 + lane) + at, l);
    f.before = __shfl_sync(kFull, before, l);
    f.upto = __shfl_sync(kFull, c, l);
    return f;
  }
};

// Between a < b in the order of the floats' bits: bisection by value is quick where the
// logits are spread evenly, this one bounds the number of steps where they are not.
__device__ __forceinline__ float middle_by_bits(float a, float b) {
  const auto key = [](float x) { const int i = __float_as_int(x); return i >= 0 ? i : (int)0x80000000 - i; };
  const int ka = key(a), kb = key(b);
  const int k = (int)(((int64_t)ka + kb) >> 1);
  return __int_as_float(k >= 0 ? k : (int)0x80000000 - k);
}

// exp(x) for x <= 0 in double, to a few units of its last place: x = k ln 2 + r with
// |r| <= ln 2 / 2, the Taylor series of e^r to the 13th power (the next term is below 2^-57),
// and 2^k by the exponent field, in two factors where the result is below the normal numbers.
__device__ __forceinline__ double exp_below_zero(double x) {
  if (x < -746.0) return 0.0;
  const double k = rint(x * 1.4426950408889634074);
  double r = fma(k, -0.693147180559945309417, x);       // ln 2 rounded to double ...
  r = fma(k, -2.3190468138462996e-17, r);               // ... and what the rounding left out
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  const int whole = (int)k, first = max(whole, -1000);
  return __longlong_as_double(__double_as_longlong(p) + ((long long)first << 52)) * __longlong_as_double((long long)(1023 + whole - first) << 52);
}

// The weight in 64 bits.  Few rows ask for it, so where it is taken for every element the
// loop runs over groups of four (independent of each other: one waits while the next is
// worked on) and is not unrolled further; single elements make a call.
__device__ __forceinline__ double exact_weight(float x, float top, double inverse_t) {
  return x > -inf_f() ? exp_below_zero(((double)x - (double)top) * inverse_t) : 0.0;
}
__device__ __noinline__ double exact_weight_call(float x, float top, double inverse_t) { return exact_weight(x, top, inverse_t); }

// A row lives in the registers of its threads, 4 J logits and their weights in each, so HBM is
// read once; what bounds the kernel is the work on a row.  80 000 rows of 500 (float, 160 MB):
// 53 us without a filter, 157 us with top-p (about 1 900 instructions per row; the issue slots
// are 85 % used), 24 us would be the read.  A few rows are bound by the chain of a search's
// steps (a comparison per logit, then a reduction: 350 cycles in a warp, 600 in a block, 1.5 us
// in a cluster): 256 x 5000 with all filters 25 us, 16 x 100003 with top-p and min-p 49 - 72 us
// (over a dozen sets of inputs: by how often the slowest row asks for its sums in double).
// Tried and slower: four or eight pivots per step (the instructions grow faster than the
// steps fall: 256 x 5000 46 us with eight), pivots by the secant of the logarithm of what lies
// below (one end of the bracket stays put), a bisection that keeps both ends on logits from
// the start (twice the instructions per step).
template <typename T, int kWarps, int kCtas, int J, int kRowsPerBlock>
__global__ void __launch_bounds__(kWarps * 32 * kRowsPerBlock, kWarps == 1 ? (J <= 4 ? 8 : 4) : (kWarps == 8 ? 2 : 1))
sample_kernel(const SampleArgs a) {
  constexpr int E = 4 * J;
  using TeamT = Team<kWarps, kCtas>;
  __shared__ typename TeamT::Scratch scratch[kWarps == 1 ? 1 : kRowsPerBlock];
  TeamT team(scratch[0]);
  const int tid = kWarps == 1 ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t row = kWarps == 1 ? (int64_t)blockIdx.x * kRowsPerBlock + (threadIdx.x >> 5) : (int64_t)(blockIdx.x / kCtas);
  int first = 0;
  if constexpr (kCtas > 1) first = (int)cg::this_cluster().block_rank() * (E * kWarps * 32);
  if constexpr (kCtas > 1) cg::this_cluster().sync();  // every block runs before its shared memory is written from another
  pdl_wait();
  pdl_trigger();
  if (row >= a.rows) return;

  float x[E];
  const T *src = static_cast<const T *>(a.logits) + row * a.stride;
  if (a.vec) {
    // groups of four lie inside the row or outside; all loads are requested before one is used
    typename Raw4<T>::type raw[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int at = first + 4 * (j * kWarps * 32 + tid);
      raw[j] = typename Raw4<T>::type{};
      if (at < a.V) raw[j] = load4(src + at);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float f[4];
      convert4<T>(raw[j], f);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[4 * j + q] = first + 4 * (j * kWarps * 32 + tid) < a.V ? f[q] : -inf_f();
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int at = first + 4 * ((e >> 2) * kWarps * 32 + tid) + (e & 3);
      x[e] = at < a.V ? to_float(__ldg(src + at)) : -inf_f();
    }
  }
  const float u = __ldg(a.u + row);
  const float temperature = a.temperature ? __ldg(a.temperature + row) : a.temperature_all;
  const float top_p = a.top_p ? __ldg(a.top_p + row) : a.top_p_all;
  const float min_p = a.min_p ? __ldg(a.min_p + row) : a.min_p_all;
  const int top_k = a.top_k ? __ldg(a.top_k + row) : a.top_k_all;

  // the largest logit; a NaN anywhere makes it a NaN
  float most = -inf_f();
#pragma unroll
  for (int e = 0; e < E; ++e) asm("max.NaN.f32 %0, %1, %2;" : "=f"(most) : "f"(most), "f"(x[e]));
  const float top = team.max_with_nan(most);
  // (the comparisons are false for a NaN too)
  const bool valid = top < inf_f() && top > -inf_f() && temperature >= 0.f && temperature <= 1e6f && top_p == top_p &&
                     min_p == min_p && u >= 0.f && u <= 1.f;
  const bool writer = tid == 0 && first == 0;
  if (!valid) {
    if (writer) { a.token[row] = -1; a.logprob[row] = __int_as_float(0x7fffffff); }
    if constexpr (kCtas > 1) cg::this_cluster().sync();
    return;
  }
  if (temperature == 0.f || top_p <= 0.f || min_p > 1.f || top_k == 1) {  // only the first element is left
    const auto is_top = [&](float y, float) { return y == top ? 1 : 0; };
    const auto f = team.template locate<J, int>(0, first, x, x, is_top);
    if (writer) { a.token[row] = f.index; a.logprob[row] = 0.f; }
    if constexpr (kCtas > 1) cg::this_cluster().sync();
    return;
  }

  const double inverse_t = 1.0 / (double)temperature;
  const double factor64 = fmin(1.4426950408889634074 * inverse_t, 3e38);  // exponent = (x - max) * factor
  const float factor = (float)factor64, lowest = -200.f / factor;         // 2^-200 is 0 in float
  const float factor_rest = (float)(factor64 - (double)factor);
  const auto weight = [&](float y) {
    const float d0 = y - top, d = fmaxf(d0, lowest), t = d * factor;
    if constexpr (kWarps == 1) return ex2_approx(t);
    // what the roundings of the subtraction, the factor and the product left out
    const float b = d0 - y, lost = d0 >= lowest ? (y - (d0 - b)) - (top + b) : 0.f;
    const float rest = fmaf(lost, factor, fmaf(d, factor_rest, fmaf(d, factor, -t)));
    const float v = ex2_approx(t);
    return fmaf(v * 0.6931471805599453f, rest, v);
  };
  const auto exact = [&](float y) { return exact_weight_call(y, top, inverse_t); };
  float w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = weight(x[e]);
  if (temperature < kLeastNormal) {  // 1 / temperature is no float: such a row's weights come from double
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = (float)exact(x[e]);
  }
  // The sum of f over the thread's elements: in wide rows fours in float, those in double
  using S = typename TeamT::Sum;
  const auto sum_of = [&](auto f) {
    if constexpr (kWarps == 1) {
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) c[e & 3] += f(e);
      return (c[0] + c[1]) + (c[2] + c[3]);
    } else {
      double c = 0.0;
#pragma unroll
      for (int j = 0; j < J; ++j) c += (double)((f(4 * j) + f(4 * j + 1)) + (f(4 * j + 2) + f(4 * j + 3)));
      return c;
    }
  };
  const auto sum_above = [&](float border) {
    if constexpr (kWarps == 1) {  // (one predicated addition per element, four chains)
      float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > border) c[e & 3] += w[e];
      return (c[0] + c[1]) + (c[2] + c[3]);
    } else {
      return sum_of([&](int e) { return x[e] > border ? w[e] : 0.f; });
    }
  };
  const auto least_finite = [&]() {
    Pass<float> r{0.f, 0, inf_f(), 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) r.least = x[e] > -inf_f() ? fminf(r.least, x[e]) : r.least;
    return team.template reduce<kEnds>(r).least;
  };
  // All weights, and those of the logits above `border`, in double.  The loop is not unrolled:
  // few rows come here, and the code of the others should stay small.
  const auto exact_sums = [&](float border, double &above) {
    float copy[E];
#pragma unroll
    for (int e = 0; e < E; ++e) copy[e] = x[e];
    double all = 0.0, part = 0.0;
#pragma unroll 1
    for (int j = 0; j < J; ++j) {
      double v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = exact_weight(copy[4 * j + q], top, inverse_t);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        all += v[q];
        if (copy[4 * j + q] > border) part += v[q];
      }
    }
    above = team.template reduce<kSum>(Pass<double>{part, 0, 0.f, 0.f}).sum;
    return team.template reduce<kSum>(Pass<double>{all, 0, 0.f, 0.f}).sum;
  };
  const auto drop = [&](int e) { x[e] = -inf_f(); w[e] = 0.f; };
  const auto index = [&](int e) { return first + 4 * ((e >> 2) * kWarps * 32 + tid) + (e & 3); };

  // Keeps the logits above `border` and the first `ties` (by index) of the `equal` that are the border.
  const auto cut = [&](float border, int ties, int equal) {
    if (ties < equal) {
      const auto is_border = [&](float y, float) { return y == border ? 1 : 0; };
      const int last = team.template locate<J, int>(ties - 1, first, x, x, is_border).index;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] == border && index(e) > last) drop(e);
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] < border) drop(e);
  };
  const auto equal_to = [&](float y) {
    Pass<float> c{0.f, 0, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) c.count += x[e] == y;
    return team.template reduce<kCount>(c).count;
  };
  // How many logits lie in (lo, hi], or [lo, hi] if not `open`, the least and the largest of them.
  const auto between = [&](float lo, float hi, bool open) {
    const float from = open ? lo : -inf_f();  // not open: lo is the least of all
    Pass<float> q{0.f, 0, inf_f(), -inf_f()};
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] > from && x[e] <= hi) { ++q.count; q.least = fminf(q.least, x[e]); q.most = fmaxf(q.most, x[e]); }
    return team.template reduce<kCount | kEnds>(q);
  };
  const auto middle = [&](float lo, float hi, int step) {
    float m = step < 24 ? 0.5f * lo + 0.5f * hi : middle_by_bits(lo, hi);
    return m < hi && m >= lo ? m : lo;
  };

  constexpr int kSteps = 16;  // of a search by value; the search between logits that follows ends by itself

  float least = -inf_f();  // of the logits that top-k kept
  int live = 0;
  if (top_k > 0 && top_k < a.V) {
    Pass<float> r{0.f, 0, inf_f(), 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] > -inf_f()) { ++r.count; r.least = fminf(r.least, x[e]); }
    r = team.template reduce<kCount | kEnds>(r);
    least = r.least;
    live = r.count;
  }
  if (top_k > 0 && top_k < live) {
    // border: the logit with fewer than k above it and k at or above it
    float lo = least, hi = top, found = 0.f;  // found: a border at or above which exactly k lie
    int above = 0, at_lo = live;              // logits above hi, and at or above lo
    bool split = false;
    bool open = false;                        // lo itself no longer counts
    for (int step = 0; step < kSteps && at_lo - above > 1 && hi - lo < 1e30f && !split; ++step) {
      const float mid = 0.5f * lo + 0.5f * hi;
      if (!(mid > lo && mid < hi)) break;
      int c[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) c[e & 1] += x[e] > mid;
      const int n = team.template reduce<kCount>(Pass<float>{0.f, c[0] + c[1], 0.f, 0.f}).count;
      if (n >= top_k) { lo = mid; at_lo = n; open = true; } else { hi = mid; above = n; }
      split = open && at_lo == top_k;
      found = lo;
    }
    if (split) {  // exactly k logits above lo
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(x[e] > found)) drop(e);
      least = least_finite();
    } else {
      // the logits still in question, from least to most; then bisection between them
      Pass<float> r = between(lo, hi, open);
      lo = r.least;
      hi = r.most;
      for (int step = 0; lo < hi; ++step) {
        const float mid = middle(lo, hi, step);
        Pass<float> b{0.f, 0, inf_f(), -inf_f()};
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (x[e] > mid) { ++b.count; b.least = fminf(b.least, x[e]); }
          else b.most = fmaxf(b.most, x[e]);
        }
        b = team.template reduce<kCount | kEnds>(b);
        if (b.count >= top_k) lo = b.least; else { hi = b.most; above = b.count; }
      }
      cut(hi, top_k - above, r.count == 1 ? 1 : equal_to(hi));
      least = hi;
    }
  }

  if (top_p < 1.f) {
    const S total = team.template reduce<kSum>(Pass<S>{sum_of([&](int e) { return w[e]; }), 0, 0.f, 0.f}).sum;
    const S goal = (S)top_p * total, near = (S)(2.f * a.eps) * total;
    // border: the logit with less than `goal` above it and at least that at or above it
    float lo = least, hi = top;
    S above = S(0), at_lo = total;
    bool open = false;  // lo itself no longer counts
    if (S(1) - goal > near) {
      lo = nextafterf(top, -inf_f());  // the largest alone weighs enough: nothing else is in question
      at_lo = S(0);
      open = true;
    } else {
      // V logits of weight (1 - top_p) * sum / (2 V) each would not weigh what top_p leaves:
      // the border lies above them (and a step down, for the rounding of this sum, which may be
      // coarse beside the temperature)
      const float floor_x = top + temperature * logf((1.f - top_p) * (float)total / (2.f * (float)a.V));
      lo = fmaxf(least, nextafterf(floor_x, -inf_f()));
      open = lo > least;
    }
    // First by value, as far as these sums decide; (at_lo - above) / w(hi) is about the number
    // of logits left between.
    for (int step = 0; step < kSteps && hi - lo < 1e30f && (float)(at_lo - above) > 1.5f * weight(hi); ++step) {
      const float mid = 0.5f * lo + 0.5f * hi;
      if (!(mid > lo && mid < hi)) break;
      const S n = team.template reduce<kSum>(Pass<S>{sum_above(mid), 0, 0.f, 0.f}).sum;
      if (n >= goal + near) { lo = mid; at_lo = n; open = true; }   // surely enough above it
      else if (n <= goal - near) { hi = mid; above = n; }           // surely not
      else break;
    }
    // Then between the logits that are left, from the least to the largest of them.
    const Pass<float> q = between(lo, hi, open);
    lo = q.least;
    hi = q.most;
    for (int step = 0; lo < hi; ++step) {
      const float mid = middle(lo, hi, step);
      Pass<S> s{sum_above(mid), 0, inf_f(), -inf_f()};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (x[e] > mid) s.least = fminf(s.least, x[e]);
        else s.most = fmaxf(s.most, x[e]);
      }
      s = team.template reduce<kSum | kEnds>(s);
      bool enough = s.sum >= goal;
      if ((s.sum > goal ? s.sum - goal : goal - s.sum) <= near) {
        double above64;
        const double goal64 = (double)top_p * exact_sums(mid, above64);
        enough = above64 >= goal64;
      }
      if (enough) lo = s.least; else { hi = s.most; above = s.sum; }
    }
    const int equal = q.count == 1 ? 1 : equal_to(hi);
    int ties = 1;
    if (equal > 1) {
      // the i-th of the border's equals stays while above + i * w < goal
      const S wb = (S)weight(hi), n = ceil((goal - above) / wb);
      ties = (int)fmin(fmax(n, S(1)), (S)equal);
      const S at = above + (S)ties * wb - goal;
      if (temperature < kLeastNormal || !(wb > S(0)) || fabs(at) <= near || (ties > 1 && fabs(at - wb) <= near)) {
        double above64;
        const double goal64 = (double)top_p * exact_sums(hi, above64), wb64 = exact(hi);
        double m = ceil((goal64 - above64) / wb64);
        m = fmin(fmax(m, 1.0), (double)equal);  // a NaN (0 / 0) becomes 1
        if (m > 1.0 && above64 + (m - 1.0) * wb64 >= goal64) m -= 1.0;
        else if (m < (double)equal && above64 + m * wb64 < goal64) m += 1.0;
        ties = (int)m;
      }
    }
    cut(hi, ties, equal);
  }

  if (min_p > 0.f) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (x[e] == -inf_f()) continue;
      bool keep = w[e] >= min_p;
      // the weight's own relative error: (3 |ln w| + 4) * 2^-24, below 2^-16 down to 2^-126
      if (fabsf(w[e] - min_p) <= 1.6e-5f * min_p || min_p < 1e-35f) keep = exact(x[e]) >= (double)min_p;
      if (!keep) drop(e);
    }
  }

  const S sum = team.template reduce<kSum>(Pass<S>{sum_of([&](int e) { return w[e]; }), 0, 0.f, 0.f}).sum;
  const S goal = (S)u * sum, near = (S)(2.f * a.eps) * sum;
  const auto value = [](float, float v) { return v; };
  const auto f = team.template locate<J, S>(goal, first, x, w, value);
  int token = f.index;
  if (token < 0 || f.upto - goal <= near || goal - f.before <= near) {
    const auto value64 = [&](float y, float) { return exact_weight(y, top, inverse_t); };
    // u = 1 asks for the last: two orders of adding the same doubles may differ by a
    // rounding, which is far below the 2^-24 that any other u stays away from the total
    token = u < 1.f ? team.template locate<J, double, true>((double)u, first, x, w, value64).index : -1;
    if (token < 0) {  // the last that has any weight (indices stay below 2^24: exact in float)
      Pass<float> last{0.f, 0, 0.f, -1.f};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (exact(x[e]) > 0.0) last.most = fmaxf(last.most, (float)index(e));
      token = (int)team.template reduce<kEnds>(last).most;
    }
  }
  if (tid == 0 && first == 0) {
    const float xt = to_float(src[token]);
    a.token[row] = token;
    a.logprob[row] = (xt - top) / temperature - logf((float)sum);
  }
  if constexpr (kCtas > 1) cg::this_cluster().sync();  // no block leaves while another reads its shared memory
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

template <typename T, int kWarps, int kCtas, int J, int kRowsPerBlock>
cudaError_t launch(SampleArgs a, cudaStream_t s) {
  // additions on the longest path of a warp's row: J in a chain, 2 to join four, 5 in the warp, and u * sum
  const float ulp = 5.9604645e-8f;
  a.eps = kWarps == 1 ? (3.f * logf((float)a.V + 2.f) + (J + 2 + 5 + 1) + 6) * ulp : 9.f * ulp;
  cudaLaunchConfig_t cfg = {};
  const int64_t blocks = kWarps == 1 ? (a.rows + kRowsPerBlock - 1) / kRowsPerBlock : a.rows * kCtas;
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWarps * 32 * kRowsPerBlock);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCtas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kCtas > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T, kWarps, kCtas, J, kRowsPerBlock>, a);
}

// A row that fits the registers of a warp stays with one warp; wider ones take a block, and
// the widest a cluster of eight, whose blocks hold a piece of the row each.  The rule: the
// narrowest form that holds the row.  At every width and number of rows measured it is the
// fastest, because a step's instructions grow with the logits per thread and its barrier with
// the warps; a form more than the row needs costs (us, float, top-p 0.9, the row's own form and
// the next wider one; a few rows without a filter take 5 in both):
//     V = 128     40 000 rows    44   69      V = 6144     4096 rows   186   351
//     V = 512     40 000 rows    80  134      V = 8192     4096 rows   359   470
//     V = 1024    40 000 rows   146 1266      V = 16384     256 rows    50   456
//     V = 4096      4096 rows   154  178      V = 64000     256 rows   519   629
//     V = 5000 (the 6144 form)  4096 rows 182 345, 16 rows 12.4 14.5
//     V = 130000    256 rows    702 1397
// So 16 385 columns cost nine times what 16 384 do: a cluster of eight for a row that three
// blocks would hold.
template <typename T> cudaError_t launch_by_width(const SampleArgs &a, cudaStream_t s) {
  if (a.V <= 128) return launch<T, 1, 1, 1, 4>(a, s);
  if (a.V <= 512) return launch<T, 1, 1, 4, 4>(a, s);
  if (a.V <= 1024) return launch<T, 1, 1, 8, 4>(a, s);
  if (a.V <= 4096) return launch<T, 8, 1, 4, 1>(a, s);
  if (a.V <= 6144) return launch<T, 8, 1, 6, 1>(a, s);
  if (a.V <= 8192) return launch<T, 16, 1, 4, 1>(a, s);
  if (a.V <= 16384) return launch<T, 16, 1, 8, 1>(a, s);
  if (a.V <= 65536) return launch<T, 16, 8, 4, 1>(a, s);
  if (a.V <= 131072) return launch<T, 16, 8, 8, 1>(a, s);
  return launch<T, 16, 8, 16, 1>(a, s);
}

}  // namespace

}  // namespace otb

using namespace otb;

extern "C" int ot_b200_sample(const void *d_logits, int64_t rows, int32_t V, int64_t row_stride, uint32_t flags,
                              const float *d_uniforms, const float *d_temperature, float temperature,
                              const int32_t *d_top_k, int32_t top_k, const float *d_top_p, float top_p,
                              const float *d_min_p, float min_p, int32_t *d_tokens, float *d_logprobs, void *stream) {
  const uint32_t types = flags & (OT_B200_BF16 | OT_B200_FP16);
  if ((flags & ~(OT_B200_BF16 | OT_B200_FP16)) || (types & (types - 1)))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_sample: flags may hold one of OT_B200_BF16 and OT_B200_FP16");
  if (!d_logits || !d_uniforms || !d_tokens || !d_logprobs)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_sample: NULL pointer");
  if (rows <= 0 || V <= 0 || V > OT_B200_SAMPLE_MAX_V || (rows > 1 && row_stride < V))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_sample: rows must be positive, V in 1..%d, row_stride >= V", OT_B200_SAMPLE_MAX_V);
  if (!d_temperature && !(temperature >= 0.f && temperature <= 1e6f))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_sample: the temperature must be in [0, 1e6]");
  if ((!d_top_p && top_p != top_p) || (!d_min_p && min_p != min_p))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_sample: top_p and min_p must be numbers");
  SampleArgs a;
  a.logits = d_logits;
  a.stride = row_stride;
  a.rows = rows;
  a.V = V;
  a.u = d_uniforms;
  a.temperature = d_temperature;
  a.top_p = d_top_p;
  a.min_p = d_min_p;
  a.top_k = d_top_k;
  a.temperature_all = temperature;
  a.top_p_all = top_p;
  a.min_p_all = min_p;
  a.top_k_all = top_k;
  const size_t es = types ? 2 : 4;
  a.vec = reinterpret_cast<uintptr_t>(d_logits) % (4 * es) == 0 && (rows == 1 || row_stride % 4 == 0) && V % 4 == 0;
  a.token = d_tokens;
  a.logprob = d_logprobs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (types == OT_B200_BF16) e = launch_by_width<__nv_bfloat16>(a, s);
  else if (types == OT_B200_FP16) e = launch_by_width<__half>(a, s);
  else e = launch_by_width<float>(a, s);
  if (e != cudaSuccess) return fail(OT_B200_ERR_CUDA, "ot_b200_sample: %s", cudaGetErrorString(e));
  return OT_B200_OK;
}
