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
// done in float: with E logits per thread the float sum of any subset of the w is off by
// at most
//     eps * (sum of w),   eps = (3 ln V + E + 24) * 2^-24
// (3 * 2^-24 per unit of the exponent's argument from the subtraction, the factor and the
// product, and sum w_i |ln w_i| <= ln V * sum w_i; 2^-22 from ex2.approx; one rounding per
// addition on the longest path), and a comparison of two such sums that is closer than
// twice that is made again with double sums.  Nothing is sorted: a filter's border is a
// logit, found by bisection between the logits that are still in question.
#include <cooperative_groups.h>
#include <math.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

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
  template <int kWhat, typename A> __device__ __forceinline__ Pass<A> reduce(Pass<A> p) {
    if (kWhat & kSum) p.sum = warp_sum(p.sum);
    if (kWhat & kCount) p.count = __reduce_add_sync(kFull, p.count);
    if (kWhat & kEnds) {
      p.least = warp_min_f(p.least);
      p.most = warp_max_f(p.most);
    }
    if constexpr (kWarps > 1) {
      const int warp = threadIdx.x >> 5;
      half ^= 1;
      if ((threadIdx.x & 31) == 0) s.warp_part[half][warp] = Pass<double>{(double)p.sum, p.count, p.least, p.most};
      __syncthreads();
      Pass<double> t = s.warp_part[half][0];
      A sum = (A)t.sum;
#pragma unroll 8
      for (int w = 1; w < kWarps; ++w) {
        const Pass<double> o = s.warp_part[half][w];
        sum += (A)o.sum;
        t.count += o.count;
        t.least = fminf(t.least, o.least);
        t.most = fmaxf(t.most, o.most);
      }
      p = Pass<A>{sum, t.count, t.least, t.most};
    }
    if constexpr (kCtas > 1) {
      cg::cluster_group cluster = cg::this_cluster();
      if (threadIdx.x < kCtas) {
        Pass<double> *there = cluster.map_shared_rank(&s.cta_part[half][cluster.block_rank()], threadIdx.x);
        *there = Pass<double>{(double)p.sum, p.count, p.least, p.most};
      }
      cluster.sync();
      Pass<double> t = s.cta_part[half][0];
      A sum = (A)t.sum;
#pragma unroll
      for (int c = 1; c < kCtas; ++c) {
        const Pass<double> o = s.cta_part[half][c];
        sum += (A)o.sum;
        t.count += o.count;
        t.least = fminf(t.least, o.least);
        t.most = fmaxf(t.most, o.most);
      }
      p = Pass<A>{sum, t.count, t.least, t.most};
    }
    return p;
  }

  // The first element, in index order, at which the running sum of value(x, w) exceeds
  // `target`: its index, and the sums before and after it.  Index -1 when there is none.
  // Element e = 4 j + q of thread t has the index first + 4 (j * threads + t) + q.
  template <typename A> struct Found { int index; A before, upto; };

  template <int J, typename A, typename F>
  __device__ __forceinline__ Found<A> locate(A target, int first, const float (&x)[4 * J], const float (&w)[4 * J], F value) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    A part[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      A v = A(0);
#pragma unroll
      for (int q = 0; q < 4; ++q) v += value(x[4 * j + q], w[4 * j + q]);
      part[j] = v;
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
      const A v = value(xs[q], ws[q]);
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

// The weight in 64 bits; a call, because few rows need it and it would be inlined once per element.
__device__ __noinline__ double exact_weight(float x, float top, float temperature) {
  return x > -inf_f() ? exp(((double)x - (double)top) / (double)temperature) : 0.0;
}

template <typename T, int kWarps, int kCtas, int J, int kRowsPerBlock>
__global__ void __launch_bounds__(kWarps * 32 * kRowsPerBlock)
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

  // largest logit, least finite one, how many are not -inf; a NaN counts as +inf
  Pass<float> p{0.f, 0, inf_f(), -inf_f()};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (x[e] != x[e]) x[e] = inf_f();
    if (x[e] > -inf_f()) { ++p.count; p.least = fminf(p.least, x[e]); }
    p.most = fmaxf(p.most, x[e]);
  }
  p = team.template reduce<kCount | kEnds>(p);
  const float top = p.most;
  float least = p.least;
  const int live = p.count;
  // (the negations are false for a NaN too)
  const bool valid = top < inf_f() && live > 0 && temperature >= 0.f && temperature <= 1e6f && top_p == top_p &&
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

  const float factor = (float)(1.4426950408889634074 / (double)temperature);
  const auto weight = [&](float y) { const float d = y - top; return d == 0.f ? 1.f : ex2_approx(d * factor); };
  const auto exact = [&](float y) { return exact_weight(y, top, temperature); };
  float w[E];
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = weight(x[e]);
  const auto drop = [&](int e) { x[e] = -inf_f(); w[e] = 0.f; };
  const auto index = [&](int e) { return first + 4 * ((e >> 2) * kWarps * 32 + tid) + (e & 3); };

  // Keeps the logits above `border` and the first `ties` (by index) of the `equal` that are the border.
  const auto cut = [&](float border, int ties, int equal) {
    int last = 0x7fffffff;
    if (ties < equal) {
      const auto is_border = [&](float y, float) { return y == border ? 1 : 0; };
      last = team.template locate<J, int>(ties - 1, first, x, x, is_border).index;
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] < border || (x[e] == border && index(e) > last)) drop(e);
  };
  const auto middle = [&](float lo, float hi, int step) {
    float m = step < 24 ? 0.5f * lo + 0.5f * hi : middle_by_bits(lo, hi);
    return m < hi && m >= lo ? m : lo;
  };

  if (top_k > 0 && top_k < live) {
    // border: the logit with fewer than k above it and k at or above it; always in [lo, hi]
    float lo = least, hi = top;
    int above = 0;  // logits above hi
    bool split = false;
    for (int step = 0; lo < hi && !split; ++step) {
      const float mid = middle(lo, hi, step);
      Pass<float> r{0.f, 0, inf_f(), -inf_f()};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (x[e] > mid) { ++r.count; r.least = fminf(r.least, x[e]); }
        else r.most = fmaxf(r.most, x[e]);
      }
      r = team.template reduce<kCount | kEnds>(r);
      if (r.count >= top_k) lo = r.least; else { hi = r.most; above = r.count; }
      split = r.count == top_k;
    }
    if (split) {  // exactly k logits at or above lo
      cut(lo, 1, 1);
      least = lo;
    } else {
      Pass<float> r{0.f, 0, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) r.count += x[e] == hi;
      r = team.template reduce<kCount>(r);
      cut(hi, top_k - above, r.count);
      least = hi;
    }
  }

  if (top_p < 1.f) {
    Pass<float> r{0.f, 0, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) r.sum += w[e];
    r = team.template reduce<kSum>(r);
    const float goal = top_p * r.sum, near = 2.f * a.eps * r.sum;
    double goal64 = -1.0;  // taken only when a comparison needs it
    const auto exact_sum_above = [&](float border) {
      Pass<double> d{0.0, 0, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x[e] > border) d.sum += exact(x[e]);
      return team.template reduce<kSum>(d).sum;
    };
    // border: the logit with less than `goal` above it and at least that at or above it
    float lo = least, hi = top, above = 0.f;
    for (int step = 0; lo < hi; ++step) {
      const float mid = middle(lo, hi, step);
      Pass<float> s{0.f, 0, inf_f(), -inf_f()};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (x[e] > mid) { s.sum += w[e]; s.least = fminf(s.least, x[e]); }
        else s.most = fmaxf(s.most, x[e]);
      }
      s = team.template reduce<kSum | kEnds>(s);
      bool enough = s.sum >= goal;
      if (fabsf(s.sum - goal) <= near) {
        if (goal64 < 0.0) goal64 = (double)top_p * exact_sum_above(-inf_f());
        enough = exact_sum_above(mid) >= goal64;
      }
      if (enough) lo = s.least; else { hi = s.most; above = s.sum; }
    }
    Pass<float> c{0.f, 0, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) c.count += x[e] == hi;
    c = team.template reduce<kCount>(c);
    int ties = 1;
    if (c.count > 1) {
      // the i-th of the border's equals stays while above + i * w < goal
      const float wb = weight(hi);
      const float n = ceilf((goal - above) / wb);
      ties = (int)fminf(fmaxf(n, 1.f), (float)c.count);
      const float at = above + (float)ties * wb;
      if (fabsf(at - goal) <= near || (ties > 1 && fabsf(at - wb - goal) <= near) || !(wb > 0.f)) {
        if (goal64 < 0.0) goal64 = (double)top_p * exact_sum_above(-inf_f());
        const double above64 = exact_sum_above(hi), wb64 = exact(hi);
        double m = ceil((goal64 - above64) / wb64);
        m = fmin(fmax(m, 1.0), (double)c.count);  // a NaN (0 / 0) becomes 1
        if (m > 1.0 && above64 + (m - 1.0) * wb64 >= goal64) m -= 1.0;
        else if (m < (double)c.count && above64 + m * wb64 < goal64) m += 1.0;
        ties = (int)m;
      }
    }
    cut(hi, ties, c.count);
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

  Pass<float> z{0.f, 0, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < E; ++e) z.sum += w[e];
  z = team.template reduce<kSum>(z);
  const float goal = u * z.sum, near = 2.f * a.eps * z.sum;
  const auto value = [](float, float v) { return v; };
  const auto f = team.template locate<J, float>(goal, first, x, w, value);
  int token = f.index;
  if (token < 0 || f.upto - goal <= near || goal - f.before <= near) {
    Pass<double> d{0.0, 0, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < E; ++e) d.sum += exact(x[e]);
    const double total = team.template reduce<kSum>(d).sum;
    const auto value64 = [&](float y, float) { return exact(y); };
    // u = 1 asks for the last: two orders of adding the same doubles may differ by a
    // rounding, which is far below the 2^-24 that any other u stays away from the total
    token = u < 1.f ? team.template locate<J, double>((double)u * total, first, x, w, value64).index : -1;
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
    a.logprob[row] = (xt - top) / temperature - logf(z.sum);
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
  a.eps = (3.f * logf((float)a.V + 2.f) + 4 * J + 24) * 5.9604645e-8f;
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
// the widest a cluster of eight, whose blocks hold a piece of the row each.
template <typename T> cudaError_t launch_by_width(const SampleArgs &a, cudaStream_t s) {
  if (a.V <= 128) return launch<T, 1, 1, 1, 4>(a, s);
  if (a.V <= 512) return launch<T, 1, 1, 4, 4>(a, s);
  if (a.V <= 1024) return launch<T, 1, 1, 8, 4>(a, s);
  if (a.V <= 4096) return launch<T, 8, 1, 4, 1>(a, s);
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
