// The joiner's output projection in 8-bit floating point (e4m3) with one float scale
// for every block of 128 elements along the contraction:
//
//   out[m, n] = sum_kb sa[m, kb] * sb[n / 128, kb] * ( sum_{k in block kb} a[m, k] * b[n, k] )  (+ bias[n])
//
// a (M, K) has blocks of 1 x 128, b (N, K) blocks of 128 x 128.  Three products of a
// training step have this form, each with both operands stored along the contraction:
//   logits = x * W^T       a = x (rows, D)         b = W (V, D)
//   dX     = dY * W        a = dY (rows, V)        b = W^T (D, V)
//   dW     = dY^T * X      a = dY^T (V, rows)      b = X^T (D, rows)
// so the quantiser below writes a tile plain, transposed, or both from one read.  The
// reference has no counterpart: it takes the logits as they are
// (optimized_transducer/csrc/transducer-loss.h:60-63).
//
// Scales.  quantize_kernel takes the smallest power of two s with max|x| / s <= 448 (the
// largest e4m3 value), 2^-126 at least, 1 for a block of zeros: x / s is then exact but
// for the rounding to e4m3 itself, which is off by at most max(2^-4 |x|, 2^-10 s): e4m3 is a
// floating-point type down to 2^-6 and has steps of 2^-9 below, so what is less than 2^-6 s
// (some 2^-14 of the block's largest) loses bits and what is less than 2^-10 s becomes 0.  A
// scale that is not a power of two would round the larger ones no less; it could move that
// border down by up to a factor of two.  A block that holds an infinity or a NaN gets
// the scale NaN: every product with it is NaN, as it would be without the quantiser.  The
// product takes any float scales (a checkpoint's).
#include <cuda_fp8.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>

#include "ot_common.cuh"
#include "tensor_core.cuh"

namespace otb {

namespace {

constexpr int kScaleBlock = 128;  // elements of the contraction that share a scale
constexpr int kQuantThreads = 256;
constexpr int kQuantRows = kScaleBlock / (kQuantThreads / 32);  // rows of a tile per warp

int fail(int code, const char *fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  set_last_error(msg);
  return code;
}

// ---------------------------------------------------------------------------
// quantisation
// ---------------------------------------------------------------------------
// Scale of a block whose largest magnitude has the float bits `top` (bits of |x| order as
// unsigned integers do, NaN above infinity), and its reciprocal; both exact.
__device__ __forceinline__ float block_scale(uint32_t top, float &inverse) {
  if (top == 0u) { inverse = 1.f; return 1.f; }
  if (top >= 0x7f800000u) { inverse = __int_as_float(0x7fffffff); return inverse; }
  // |x| = f * 2^(e - 127) with 1 <= f < 2; 448 = 1.75 * 2^8
  int k = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k < -126 ? -126 : k;
  inverse = __int_as_float((127 - k) << 23);
  return __int_as_float((127 + k) << 23);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

enum { kNone = 0, kRowBlocks = 1, kSquareBlocks = 2, kColumnBlocks = 1 };

struct QuantArgs {
  int64_t rows, ld;     // ld: elements from one row of x to the next
  int cols, col_tiles;
  bool vec;             // four columns may be loaded at once, and their number is a multiple of four
  uint8_t *q;           // (rows, cols), rows q_pitch bytes apart
  int64_t q_pitch;
  float *scale;         // kRowBlocks: [column tile][row]; kSquareBlocks: [row tile][column tile]
  uint8_t *qt;          // (cols, rows), rows qt_pitch bytes apart
  int64_t qt_pitch;
  float *scale_t;       // kColumnBlocks: [row tile][column]; kSquareBlocks: [column tile][row tile]
  int64_t row_tiles;
  float *column_sums;   // [row tile][column], or NULL
};

// A lane's four elements of one row as they were loaded.
template <typename T> struct Quad {
  typename Raw4<T>::type raw;
  __device__ __forceinline__ void clear() { raw = typename Raw4<T>::type{}; }
  __device__ __forceinline__ void set(int j, T x) {
    T t[4];
    memcpy(t, &raw, sizeof(raw));
    t[j] = x;
    memcpy(&raw, t, sizeof(raw));
  }
  // Makes the compiler forget what it converted so far: in 16 bits converting again costs an
  // instruction, keeping 64 floats alive from one pass over the tile to the next costs spills.
  __device__ __forceinline__ void forget() {
    if constexpr (sizeof(T) == 2) asm volatile("" : "+r"(raw.x), "+r"(raw.y));
  }
  __device__ __forceinline__ float at(int j) const {
    T t[4];
    memcpy(t, &raw, sizeof(raw));
    return to_float(t[j]);
  }
  // Bits of |x| of the four, of the largest; bits of |x| order as unsigned integers do, also
  // those of the 16-bit types, so two of these are compared at a time.
  __device__ __forceinline__ uint32_t top() const {
    if constexpr (sizeof(T) == 4) {
      return max(max(abs_bits(at(0)), abs_bits(at(1))), max(abs_bits(at(2)), abs_bits(at(3))));
    } else {
      uint32_t w[2];
      memcpy(w, &raw, 8);
      const uint32_t m = __vmaxu2(w[0] & 0x7fff7fffu, w[1] & 0x7fff7fffu);
      return widen(max(m & 0xffffu, m >> 16));
    }
  }
  // ... and of the largest of each of the four columns of a lane's rows.
  __device__ __forceinline__ static void column_tops(const Quad (&v)[kQuantRows], uint32_t (&top)[4]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        top[j] = 0u;
#pragma unroll
        for (int i = 0; i < kQuantRows; ++i) top[j] = max(top[j], abs_bits(v[i].at(j)));
      }
    } else {
      uint32_t m[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < kQuantRows; ++i) {
        uint32_t w[2];
        memcpy(w, &v[i].raw, 8);
        m[0] = __vmaxu2(m[0], w[0] & 0x7fff7fffu);
        m[1] = __vmaxu2(m[1], w[1] & 0x7fff7fffu);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) top[j] = widen((j & 1) ? m[j >> 1] >> 16 : m[j >> 1] & 0xffffu);
    }
  }
  // Float bits of |x| from the bits of the element type's |x|.
  __device__ __forceinline__ static uint32_t widen(uint32_t bits) {
    if constexpr (sizeof(T) == 4) {
      return bits;
    } else {
      const uint16_t b = (uint16_t)bits;
      T t;
      memcpy(&t, &b, 2);
      return __float_as_uint(to_float(t));
    }
  }
};

// One block per 128 x 128 tile of x; a warp holds 16 rows, a lane four columns of each, in
// registers and in the type they have (half the registers in 16 bits: three blocks per SM
// instead of one), so the tile is read once whatever is written: bytes along the rows
// (kPlain), transposed bytes (kTrans), and the tile's column sums.  Bound by HBM (sizeof(T)
// bytes read and one or two written per element) and, with everything asked for, by
// instruction issue: 116 250 x 512 bfloat16 along the rows 34 us = 5.3 TB/s; 116 250 x 5000 along
// rows and columns with sums 496 us = 4.7 TB/s (26 instructions per element with every lane
// working out every row's scale and float column maxima: 583 us).
template <typename T, int kPlain, int kTrans, bool kSums>
__global__ void __launch_bounds__(kQuantThreads, sizeof(T) == 2 ? 3 : 2)
quantize_kernel(const T *__restrict__ x, const QuantArgs a) {
  __shared__ __align__(16) uint32_t top_s[8][kScaleBlock];   // column maxima of each warp (or one word per warp)
  __shared__ __align__(16) float sum_s[kSums ? 8 : 1][kScaleBlock];
  __shared__ __align__(16) float inv_s[kScaleBlock];
  __shared__ __align__(16) uint8_t tile_s[kTrans != kNone ? kScaleBlock * kScaleBlock : 16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rt = blockIdx.x / (uint32_t)a.col_tiles;
  const int ct = (int)(blockIdx.x - rt * (uint32_t)a.col_tiles);
  const int64_t row0 = (int64_t)rt * kScaleBlock + warp * kQuantRows;
  const int col0 = ct * kScaleBlock, col = col0 + 4 * lane;
  const int rows_here = (int)min((int64_t)kQuantRows, max((int64_t)0, a.rows - row0));
  pdl_wait();
  pdl_trigger();

  Quad<T> v[kQuantRows];
  const T *p = x + row0 * a.ld + col;
  if (a.vec) {
    // groups of four lie inside a row or outside; all loads are requested before one is used
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) {
      v[i].clear();
      if (i < rows_here && col < a.cols) v[i].raw = load4(p + i * a.ld);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) {
      v[i].clear();
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i < rows_here && col + j < a.cols) v[i].set(j, p[i * a.ld + j]);
    }
  }

  if constexpr (kPlain == kRowBlocks) {
    // every lane learns every row's maximum, lane i works out the scale of row i
    uint32_t my_top = 0u;
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) {
      const uint32_t top = __reduce_max_sync(kFull, v[i].top());
      if (lane == i) my_top = top;
    }
    float my_inv;
    const float my_scale = block_scale(my_top, my_inv);
    if (lane < rows_here) a.scale[(int64_t)ct * a.rows + row0 + lane] = my_scale;
    uint8_t *q = a.q + row0 * a.q_pitch + col;
    const int rows_stored = col < a.cols ? rows_here : 0;  // the pitch is a multiple of 16: a word stays inside its row
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) {
      const float inv = __shfl_sync(kFull, my_inv, i);
      const uint32_t word = pack4(v[i].at(0) * inv, v[i].at(1) * inv, v[i].at(2) * inv, v[i].at(3) * inv);
      if (i < rows_stored) *reinterpret_cast<uint32_t *>(q) = word;
      q += a.q_pitch;
    }
  }
  float square_inv = 0.f;
  if constexpr (kPlain == kSquareBlocks || kTrans == kSquareBlocks) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) top = max(top, v[i].top());
    top = __reduce_max_sync(kFull, top);
    if (lane == 0) top_s[0][warp] = top;
    __syncthreads();
    top = 0u;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max(top, top_s[0][w]);
    const float s = block_scale(top, square_inv);
    if (threadIdx.x == 0) {
      if (kPlain == kSquareBlocks) a.scale[(int64_t)rt * a.col_tiles + ct] = s;
      if (kTrans == kSquareBlocks) a.scale_t[(int64_t)ct * a.row_tiles + rt] = s;
    }
    if (kPlain == kSquareBlocks) {
      uint8_t *q = a.q + row0 * a.q_pitch + col;
#pragma unroll
      for (int i = 0; i < kQuantRows; ++i)
        if (i < rows_here && col < a.cols)
          *reinterpret_cast<uint32_t *>(q + i * a.q_pitch) =
              pack4(v[i].at(0) * square_inv, v[i].at(1) * square_inv, v[i].at(2) * square_inv, v[i].at(3) * square_inv);
    }
  }
#pragma unroll
  for (int i = 0; i < kQuantRows; ++i) v[i].forget();
  if constexpr (kTrans == kColumnBlocks || kSums) {
    if constexpr (kTrans == kColumnBlocks) {
      uint32_t top[4];
      Quad<T>::column_tops(v, top);
      *reinterpret_cast<uint4 *>(&top_s[warp][4 * lane]) = make_uint4(top[0], top[1], top[2], top[3]);
    }
    if constexpr (kSums) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kQuantRows; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] += v[i].at(j);
      *reinterpret_cast<float4 *>(&sum_s[warp][4 * lane]) = make_float4(sum[0], sum[1], sum[2], sum[3]);
    }
    __syncthreads();
    if (threadIdx.x < kScaleBlock) {
      const int c = threadIdx.x;
      if (kTrans == kColumnBlocks) {
        uint32_t top = 0u;
#pragma unroll
        for (int w = 0; w < 8; ++w) top = max(top, top_s[w][c]);
        float inv;
        const float s = block_scale(top, inv);
        inv_s[c] = inv;
        if (col0 + c < a.cols) a.scale_t[(int64_t)rt * a.cols + col0 + c] = s;
      }
      if (kSums) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) sum += sum_s[w][c];
        if (col0 + c < a.cols) a.column_sums[(int64_t)rt * a.cols + col0 + c] = sum;
      }
    }
    __syncthreads();
  }
  if constexpr (kTrans != kNone) {
    // A lane's 16 rows of one column are 16 consecutive bytes of the transposed tile.  The
    // 16-byte pieces of a column are permuted by the column's group of four, so that the
    // eight lanes of a store phase (columns four apart) hit different banks.
#pragma unroll
    for (int i = 0; i < kQuantRows; ++i) v[i].forget();
    __align__(16) float inv_of[4] = {square_inv, square_inv, square_inv, square_inv};
    if (kTrans == kColumnBlocks) *reinterpret_cast<float4 *>(inv_of) = *reinterpret_cast<const float4 *>(inv_s + 4 * lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float inv = inv_of[j];
      uint32_t w[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        w[k] = pack4(v[4 * k].at(j) * inv, v[4 * k + 1].at(j) * inv, v[4 * k + 2].at(j) * inv, v[4 * k + 3].at(j) * inv);
      *reinterpret_cast<uint4 *>(tile_s + (4 * lane + j) * kScaleBlock + 16 * (warp ^ (lane & 7))) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();
#pragma unroll
    for (int i = threadIdx.x; i < kScaleBlock * 8; i += kQuantThreads) {
      const int c = i >> 3, piece = i & 7;
      const int64_t at = (int64_t)rt * kScaleBlock + 16 * piece;
      if (col0 + c < a.cols && at < a.qt_pitch)
        *reinterpret_cast<uint4 *>(a.qt + (int64_t)(col0 + c) * a.qt_pitch + at) =
            *reinterpret_cast<const uint4 *>(tile_s + c * kScaleBlock + 16 * (piece ^ ((c >> 2) & 7)));
    }
  }
}

// Column sums from the tiles' partial sums, in a fixed order: a block adds the partials of
// 8 columns with 32 threads each, then the 32 sums by a tree.
__global__ void __launch_bounds__(256)
column_sum_kernel(const float *__restrict__ part, int64_t row_tiles, int cols, float *__restrict__ out) {
  __shared__ float s[32][9];
  pdl_wait();
  pdl_trigger();
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3;
  const int col = blockIdx.x * 8 + c;
  float sum = 0.f;
  if (col < cols)
    for (int64_t r = g; r < row_tiles; r += 32) sum += __ldg(part + r * cols + col);
  s[g][c] = sum;
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) {
    if (g < o) s[g][c] += s[g + o][c];
    __syncthreads();
  }
  if (g == 0 && col < cols) out[col] = s[0][c];
}

// ---------------------------------------------------------------------------
// the product
// ---------------------------------------------------------------------------
constexpr int kTileM = 128;                      // rows per tile = TMEM lanes
constexpr int kMmaK = 32;                        // K of one tcgen05.mma for 8-bit operands
constexpr uint32_t kBytesA = kTileM * kScaleBlock;
constexpr int kStagedBytes = 32 * 128;           // a warp's staging tile: 32 rows of 128 bytes in the 128-byte swizzle

// Columns per tile: 256, 128 or 64.  An epilogue warp owns 32 rows x `columns` columns.
template <int kTileN> struct Shape {
  static constexpr int columns = kTileN == 256 ? 128 : 64;
  static constexpr int epilogue_warps = 4 * kTileN / columns;
  static constexpr int threads = 128 + 32 * epilogue_warps;  // one warpgroup for the two control warps
  // Registers per thread of the widest tile: a launch of 384 threads gives each 168, of which the
  // control warps need 56 at most and the epilogue's 128 sums and 64 values on their way more:
  // 128 * 56 + 256 * 224 = 384 * 168.
  static constexpr bool split_registers = kTileN == 256;
  static constexpr uint32_t stage_bytes = kBytesA + kTileN * kScaleBlock;
  static constexpr int ring = kTileN == 256 ? 3 : (kTileN == 128 ? 4 : 6);
  static constexpr int accumulators = kTileN == 256 ? 2 : 4;
  static constexpr int staged_tiles = columns / 64;  // tiles per warp: its columns in 16 bits, half of them in float
  static constexpr uint32_t tmem_columns = accumulators * kTileN;
  static constexpr size_t smem = 1024 + (size_t)ring * stage_bytes + (size_t)epilogue_warps * staged_tiles * kStagedBytes;
  // kind::f8f6f4: float accumulator (bits [4,6) = 1), e4m3 A and B (0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24
  static constexpr uint32_t instr = (1u << 4) | ((uint32_t)(kTileN >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
};

__device__ __forceinline__ void mma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t instr, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(instr), "r"(accumulate)
      : "memory");
}

// Rounds two floats to a pair of 16-bit values (not called for float).
template <typename T> __device__ __forceinline__ uint32_t round_pair(float a, float b) { return Pair16<T>::round(a, b); }

// Where 16-byte piece `piece` of row `row` of a staging tile lies (128-byte swizzle: what a
// TMA store expects; also, a warp that writes or reads a column of pieces hits every bank once).
__device__ __forceinline__ int staged_at(int row, int piece) { return row * 128 + ((piece ^ (row & 7)) << 4); }

// Copies a staged tile to rows of out that are `pitch` bytes apart, in units of sizeof(U)
// bytes: a store instruction covers whole 128-byte pieces of rows.
template <typename U>
__device__ __forceinline__ void store_staged(const unsigned char *staged, unsigned char *out, int64_t pitch, int rows, int bytes, int lane) {
  constexpr int kUnits = 128 / sizeof(U);                // units per row
  constexpr int kRows = kUnits >= 32 ? 1 : 32 / kUnits;  // rows per instruction
#pragma unroll
  for (int u0 = 0; u0 < kUnits; u0 += 32) {
    const int unit = u0 + lane % kUnits, r0 = lane / kUnits, byte = unit * (int)sizeof(U);
    if (byte < bytes) {
      unsigned char *dst = out + r0 * pitch + byte;
#pragma unroll 4
      for (int r = r0; r < rows; r += kRows, dst += kRows * pitch)
        *reinterpret_cast<U *>(dst) = *reinterpret_cast<const U *>(staged + staged_at(r, byte >> 4) + (byte & 15));
    }
  }
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, const void *src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
               ::"l"(map), "r"(smem_u32(src)), "r"(c0), "r"(c1) : "memory");
}

struct MatmulArgs {
  const float *sa;      // [K block][M]
  const float *sb;      // [N / 128][K block]
  const float *bias;    // [N] or NULL
  unsigned char *out;   // (M, N); pieces of K: (splits, out_rows, N) partial sums
  int64_t M, out_rows;
  int N, k_blocks, n_tiles, splits;
  uint32_t tiles;
  int unit;             // bytes per store, the largest of 8, 4, 2 that divides the rows' pitch and the base; 0: TMA stores (16 bytes do)
  int32_t *sticky;      // error record, or NULL
  int32_t seq;
  int wait_limit;       // polls of a barrier before a wait gives up
};

// True for one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

// Where the roles of a CTA meet, each at the end of its own branch.
__device__ __forceinline__ void meet_in_cta() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  asm volatile("bar.sync 0;" ::: "memory");
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

template <int kTileN> struct MatmulShared {
  uint64_t full[Shape<kTileN>::ring];          // TMA -> MMA
  uint64_t empty[Shape<kTileN>::ring];         // MMA -> TMA
  uint64_t acc_full[Shape<kTileN>::accumulators];   // MMA -> epilogue: one K block's product is complete
  uint64_t acc_empty[Shape<kTileN>::accumulators];  // epilogue -> MMA, one arrival per warp: 256 of them took as long as the block's MMAs
  uint64_t drained;                            // every MMA issued so far has completed (after an abort)
  uint32_t tmem_base;
  int never;
  volatile int abort;                          // a wait ran out: every role leaves its loop
  alignas(16) float bias[Shape<kTileN>::epilogue_warps][Shape<kTileN>::columns];  // read as float4
};

// One CTA per SM, persistent over (row tile, column tile, piece of K).  The scales change
// with every K block, so a block's product is complete in tensor memory on its own (four
// MMAs of K = 32) and the epilogue adds it, scaled, to sums held in registers in float:
// one multiply-add per element and K block, which runs while the tensor cores work on the
// next block's product.
//   warp 0   TMA producer: a (128 x 128) and b (kTileN x 128) boxes into the ring
//   warp 1   MMA issuer
//   warps 4..  epilogue: warp % 4 picks the TMEM lanes (rows), the rest the columns
// Measured (116 250 rows): logits from D = 512 to V = 5000 470-530 us, dX (V -> D) 350 us =
// 1.7 PFLOP/s, dW 373 us.  A K block takes about 1 150 cycles, of which the epilogue is busy for
// 990, and the SMs' clock falls to 1.5 - 1.7 GHz under this load; sixteen epilogue warps of 64
// columns, a leaner wait and other depths of the reads all came out within 3 % of this form.
// A wait that runs out raises the CTA's abort flag and every role leaves its loop.  Whichever
// role that was, and however far the others had come (the producer runs a ring ahead, and
// leaves without a wait when its K blocks fit the ring), they all look at the flag once more
// behind the barrier where they meet: the producer then waits (bounded) for its copies in
// flight and writes the record of the failure to `sticky`, the issuer waits for its MMAs in
// flight, and the epilogue fills the CTA's tiles with NaN.
//
// kLimited: the waits on other roles end after g.wait_limit polls, for tests of the way out.  A
// limit known to the compiler is worth the second instantiation: as a kernel argument it cost
// every wait a load and a comparison (40 007 x 512 x 500, forward and backward: 123.8 -> 124.9 us).
template <int kTileN, typename OutT, bool kLimited>
__global__ void __launch_bounds__(Shape<kTileN>::threads, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                  const __grid_constant__ CUtensorMap map_out, const MatmulArgs g) {
  using S = Shape<kTileN>;
  constexpr int R = S::ring, B = S::accumulators;
  const int limit = kLimited ? g.wait_limit : kSpinLimit;
  extern __shared__ __align__(1024) unsigned char ring_mem[];
  __shared__ MatmulShared<kTileN> sh;
  const int warp = __shfl_sync(kFull, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // one value per warp, for the compiler too
  unsigned char *ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(ring_mem) + 1023) & ~uintptr_t(1023));
  unsigned char *staging = ring + (size_t)R * S::stage_bytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < R; ++i) { mbar_init(&sh.full[i], 1); mbar_init(&sh.empty[i], 1); }
    for (int i = 0; i < B; ++i) { mbar_init(&sh.acc_full[i], 1); mbar_init(&sh.acc_empty[i], S::epilogue_warps); }
    mbar_init(&sh.drained, 1);
    sh.abort = 0;
    sh.never = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  pdl_wait();  // before the allocation: a predecessor's blocks may still hold tensor memory
  pdl_trigger();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&sh.tmem_base)), "r"(S::tmem_columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = sh.tmem_base;

  // tile -> (piece of K, row tile, column tile), the column tile fastest: the row tile's
  // bytes are read once from HBM and again from L2
  struct Place { int nt, mt, sp, k0, k1; };
  const auto place = [&](uint32_t tile) {
    const uint32_t rest = tile / (uint32_t)g.n_tiles;
    Place p;
    p.nt = (int)(tile - rest * (uint32_t)g.n_tiles);
    p.mt = (int)rest;
    p.sp = 0;
    p.k0 = 0;
    p.k1 = g.k_blocks;
    if (g.splits > 1) {
      p.mt = (int)(rest / (uint32_t)g.splits);
      p.sp = (int)rest - p.mt * g.splits;
      p.k0 = (int)((int64_t)g.k_blocks * p.sp / g.splits);
      p.k1 = (int)((int64_t)g.k_blocks * (p.sp + 1) / g.splits);
    }
    return p;
  };

  // The two control warps run their loops with all lanes and let one issue: stage indices,
  // barrier addresses and descriptors then live in uniform registers, where the MMAs want them.
  // (With one lane in the loop the issue of a block's MMAs took 740 cycles, more than the MMAs.)
  if (warp < 4) {
  if constexpr (S::split_registers) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  if (warp == 0) {
    int s = 0;           // stage
    uint32_t phase = 1;  // parity of the wait for it; the first round finds the stages empty
    uint32_t issued = 0;
    bool dead = false;
    for (uint32_t tile = blockIdx.x; tile < g.tiles && !dead; tile += gridDim.x) {
      const Place p = place(tile);
      for (int kb = p.k0; kb < p.k1; ++kb) {
        if (issued >= (uint32_t)R) {
          dead = !__all_sync(kFull, mbar_wait(&sh.empty[s], phase, &sh.abort, limit));
          if (dead) { sh.abort = 1; break; }
        }
        unsigned char *a = ring + (size_t)s * S::stage_bytes;
        if (elect_one()) {
          mbar_expect_tx(&sh.full[s], S::stage_bytes);
          // what lies beyond either matrix is filled with zeros by the copy
          tma_load_2d(a, &map_a, kb * kScaleBlock, p.mt * kTileM, &sh.full[s]);
          tma_load_2d(a + kBytesA, &map_b, kb * kScaleBlock, p.nt * kTileN, &sh.full[s]);
        }
        __syncwarp();
        ++issued;
        if (++s == R) { s = 0; phase ^= 1; }
      }
    }
    meet_in_cta();
    if (sh.abort) {
      const volatile int *never = &sh.never;  // the flag itself must not end this wait
      for (uint32_t j = (issued > (uint32_t)R ? issued - R : 0); j < issued; ++j) mbar_wait(&sh.full[j % R], (j / R) & 1, never);
      if (lane == 0 && g.sticky != nullptr) {
        volatile int32_t *r = g.sticky;
        r[1] = 0;
        r[2] = g.seq;
        __threadfence_system();
        r[0] = OT_B200_COPY_TIMEOUT;
      }
    }
  } else if (warp == 1) {
    int s = 0, buf = 0;
    uint32_t full_phase = 0, free_phase = 1, blocks = 0;
    const uint64_t desc_a = smem_desc(smem_u32(ring)), desc_b = smem_desc(smem_u32(ring) + kBytesA);
    bool dead = false;
    for (uint32_t tile = blockIdx.x; tile < g.tiles && !dead; tile += gridDim.x) {
      const Place p = place(tile);
      for (int kb = p.k0; kb < p.k1; ++kb, ++blocks) {
        bool ok = true;
        if (blocks >= (uint32_t)B) ok = mbar_wait(&sh.acc_empty[buf], free_phase, &sh.abort, limit);
        ok = ok && mbar_wait(&sh.full[s], full_phase, &sh.abort, limit);
        dead = !__all_sync(kFull, ok);
        if (dead) { sh.abort = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t step = (uint64_t)((uint32_t)s * (S::stage_bytes >> 4));
        const uint32_t d = tmem + (uint32_t)(buf * kTileN);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kScaleBlock / kMmaK; ++k)  // 32 bytes further along K inside the swizzle row
            mma_f8(d, desc_a + step + (uint64_t)(k * 2), desc_b + step + (uint64_t)(k * 2), S::instr, k != 0);
          mma_commit(&sh.empty[s]);
          mma_commit(&sh.acc_full[buf]);
        }
        __syncwarp();
        if (++s == R) { s = 0; full_phase ^= 1; }
        if (++buf == B) { buf = 0; free_phase ^= 1; }
      }
    }
    meet_in_cta();
    if (sh.abort && blocks > 0) {  // the MMAs in flight still read shared memory and write tensor memory
      if (elect_one()) mma_commit(&sh.drained);
      __syncwarp();
      mbar_wait(&sh.drained, 0, &sh.never);
    }
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::tmem_columns) : "memory");
  } else {
    meet_in_cta();
  }
  } else {
    if constexpr (S::split_registers) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int quarter = warp & 3;
    const int part = (warp - 4) >> 2;
    constexpr int kCols = S::columns;
    unsigned char *staging_tiles = staging + (size_t)(warp - 4) * S::staged_tiles * kStagedBytes;
    float *bias_s = sh.bias[warp - 4];
    uint32_t it = 0;
    bool dead = false;  // the same for all lanes: the reads of tensor memory are warp-wide
    // The scales of the next K block and the bias of the next tile are requested one block
    // ahead, across tiles: a load's latency is longer than a block's multiply-adds.
    const float *sa = nullptr, *sb = nullptr;
    float sa_next = 0.f, sb_next = 0.f, bias_next[kCols / 32];
    const auto aim = [&](const Place &p) {
      const int64_t row = (int64_t)p.mt * kTileM + quarter * 32 + lane;
      const int col0 = p.nt * kTileN + part * kCols;
      sa = g.sa + (int64_t)p.k0 * g.M + (row < g.M ? row : 0);
      sb = g.sb + (int64_t)min(col0 / kScaleBlock, (g.N - 1) / kScaleBlock) * g.k_blocks + p.k0;
      sa_next = __ldg(sa);
      sb_next = __ldg(sb);
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) {
        const int c = col0 + 32 * i + lane;
        bias_next[i] = (g.bias != nullptr && c < g.N) ? __ldg(g.bias + c) : 0.f;
      }
    };
    uint32_t tile = blockIdx.x;
    Place p = place(tile);
    if (tile < g.tiles) aim(p);
    while (tile < g.tiles) {
      const int64_t row0 = (int64_t)p.mt * kTileM + quarter * 32;
      const int col0 = p.nt * kTileN + part * kCols;
      const int sp = p.sp, blocks = p.k1 - p.k0;
      tile += gridDim.x;
      if (tile < g.tiles) p = place(tile);
      __syncwarp();  // the previous tile's bias has been read
#pragma unroll
      for (int i = 0; i < kCols / 32; ++i) bias_s[32 * i + lane] = bias_next[i];
      __syncwarp();
      float acc[kCols];  // starts as the bias
#pragma unroll
      for (int i = 0; i < kCols / 4; ++i) {
        const float4 v = reinterpret_cast<const float4 *>(bias_s)[i];
        acc[4 * i] = v.x; acc[4 * i + 1] = v.y; acc[4 * i + 2] = v.z; acc[4 * i + 3] = v.w;
      }
      for (int kb = 0; kb < blocks; ++kb, ++it) {
        const int buf = it % B;
        const float sa_now = sa_next, sb_now = sb_next;
        if (kb + 1 < blocks) {
          sa += g.M;
          ++sb;
          sa_next = __ldg(sa);
          sb_next = __ldg(sb);
        } else if (tile < g.tiles) {
          aim(p);
        }
        dead = !__all_sync(kFull, mbar_wait(&sh.acc_full[buf], (it / B) & 1, &sh.abort, limit));
        if (dead) { sh.abort = 1; break; }
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        float s;  // volatile: stays behind the wait.  Left to the compiler the product moved up to where its
                  // factors are loaded, and every block waited for that load: 460 of 1200 cycles
        asm volatile("mul.f32 %0, %1, %2;" : "=f"(s) : "f"(sa_now), "f"(sb_now));
        const uint32_t taddr = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * kTileN + part * kCols);
        uint32_t r[2][32];
        tmem_load_32_issue(taddr, r[0]);
#pragma unroll
        for (int c = 0; c < kCols / 32; ++c) {
          tmem_load_32_wait(r[c & 1]);
          if (c + 1 < kCols / 32) {
            tmem_load_32_issue(taddr + 32 * (c + 1), r[(c + 1) & 1]);
          } else {  // the last read has landed: the accumulator goes back
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.acc_empty[buf]);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) acc[32 * c + i] = fmaf(s, __uint_as_float(r[c & 1][i]), acc[32 * c + i]);
        }
      }
      if (dead) break;
      // rows leave through the warp's staging tiles, 128 bytes of each in one tile
      constexpr int kChunk = 128 / (int)sizeof(OutT);
      constexpr int kChunks = kCols / kChunk;
      const int rows_here = (int)min((int64_t)32, g.M - row0);
      const int64_t pitch = (int64_t)g.N * sizeof(OutT);
      unsigned char *out = g.out + ((int64_t)sp * g.out_rows + row0) * pitch + (int64_t)col0 * sizeof(OutT);
#pragma unroll
      for (int c0 = 0; c0 < kChunks; c0 += S::staged_tiles) {
        if (rows_here <= 0) break;
        if (g.unit == 0) {  // the stores that used the tiles have read them
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
#pragma unroll
        for (int k = 0; k < S::staged_tiles && c0 + k < kChunks; ++k)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint4 w;
            if constexpr (sizeof(OutT) == 4) {
              const float *v = acc + 32 * (c0 + k) + 4 * i;
              w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
            } else {
              const float *v = acc + 64 * (c0 + k) + 8 * i;
              w = make_uint4(round_pair<OutT>(v[0], v[1]), round_pair<OutT>(v[2], v[3]), round_pair<OutT>(v[4], v[5]), round_pair<OutT>(v[6], v[7]));
            }
            *reinterpret_cast<uint4 *>(staging_tiles + k * kStagedBytes + staged_at(lane, i)) = w;
          }
        if (g.unit == 0) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (g.unit == 0) {
          // what lies beyond the matrix is not written
          if (lane == 0) {
#pragma unroll
            for (int k = 0; k < S::staged_tiles && c0 + k < kChunks; ++k)
              if (col0 + (c0 + k) * kChunk < g.N)
                tma_store_2d(&map_out, staging_tiles + k * kStagedBytes, col0 + (c0 + k) * kChunk, (int)(sp * g.out_rows + row0));
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else {
#pragma unroll
          for (int k = 0; k < S::staged_tiles && c0 + k < kChunks; ++k) {
            const unsigned char *staged = staging_tiles + k * kStagedBytes;
            unsigned char *dst = out + (c0 + k) * 128;
            const int bytes = min(128, (g.N - col0) * (int)sizeof(OutT) - (c0 + k) * 128);
            if (bytes <= 0) break;  // warp-uniform
            if (g.unit == 8) store_staged<uint2>(staged, dst, pitch, rows_here, bytes, lane);
            else if (g.unit == 4) store_staged<uint32_t>(staged, dst, pitch, rows_here, bytes, lane);
            else store_staged<uint16_t>(staged, dst, pitch, rows_here, bytes, lane);
          }
          __syncwarp();
        }
      }
    }
    if (g.unit == 0 && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    meet_in_cta();
    if (sh.abort) {
      for (tile = blockIdx.x; tile < g.tiles; tile += gridDim.x) {
        p = place(tile);
        const int64_t row0 = (int64_t)p.mt * kTileM;
        const int rows = (int)min((int64_t)kTileM, g.M - row0), cols = min(kTileN, g.N - p.nt * kTileN);
        OutT *out = reinterpret_cast<OutT *>(g.out) + ((int64_t)p.sp * g.out_rows + row0) * g.N + p.nt * kTileN;
        for (int i = threadIdx.x - 128; i < rows * cols; i += 32 * S::epilogue_warps)
          out[(int64_t)(i / cols) * g.N + i % cols] = (OutT)__int_as_float(0x7fffffff);
      }
    }
  }
}

// out = sum over the pieces of K (in their order) + bias, rounded once.
template <typename OutT>
__global__ void __launch_bounds__(256)
split_sum_kernel(const float *__restrict__ part, int splits, int64_t stride, int64_t count, int N, const float *__restrict__ bias, OutT *__restrict__ out) {
  pdl_wait();
  pdl_trigger();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float sum = bias != nullptr ? __ldg(bias + i % N) : 0.f;
    for (int s = 0; s < splits; ++s) sum += __ldg(part + (int64_t)s * stride + i);
    out[i] = (OutT)sum;
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
struct MatmulPlan { int tile_n, splits; };

// Rows of one piece's partial sums: whole row tiles, so that a store never reaches the next piece's.
int64_t whole_tiles(int64_t M) { return (M + kTileM - 1) / kTileM * kTileM; }

// Columns per tile: the widest tile that still gives every SM a tile of its own (per K
// block a wide tile reads fewer bytes of shared memory per product); a narrower N wants no
// wider tile.  Pieces of K, when K is long (dW: K is the number of rows): as many as make
// the shortest of the times below, where a K block of a 256-column tile takes 0.4 us and the
// pieces' sums are written and read once at 4 TB/s, behind one more launch (80 tiles of 909
// blocks on 148 SMs: 538 us in one piece, 330 in five).
MatmulPlan plan_matmul(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t mt = (M + kTileM - 1) / kTileM, kb = (K + kScaleBlock - 1) / kScaleBlock;
  const bool long_k = kb >= 32;
  int tile_n = 256;
  while (tile_n > 64 && (N <= tile_n / 2 || (!long_k && mt * ((N + tile_n - 1) / tile_n) < sms))) tile_n /= 2;
  const int64_t tiles = mt * ((N + tile_n - 1) / tile_n);
  int splits = 1;
  if (long_k && tiles < 2 * sms) {
    double best = 1e300;
    for (int s = 1; s <= kb / 8 && s <= 2 * sms; ++s) {
      const double blocks = (double)((tiles * s + sms - 1) / sms) * (double)((kb + s - 1) / s);
      const double us = blocks * 0.4 * tile_n / 256 + (s > 1 ? 3.0 + s * (double)whole_tiles(M) * N * 8 / 4e6 : 0.0);
      if (us < 0.98 * best) { best = us; splits = s; }
    }
  }
  return {tile_n, splits};
}

template <int kTileN, typename OutT, bool kLimited>
cudaError_t launch_matmul_limited(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo, const MatmulArgs &g, cudaStream_t s) {
  static SmemGrant grant;
  const cudaError_t e = grant.ensure(fp8_matmul_kernel<kTileN, OutT, kLimited>, Shape<kTileN>::smem);
  if (e != cudaSuccess) return e;
  const int sms = sm_count();
  const unsigned grid = g.tiles < (unsigned)sms ? g.tiles : (unsigned)sms;
  return launch_pdl(fp8_matmul_kernel<kTileN, OutT, kLimited>, grid, (unsigned)Shape<kTileN>::threads, Shape<kTileN>::smem, s, ma, mb, mo, g);
}

template <int kTileN, typename OutT>
cudaError_t launch_matmul(const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo, const MatmulArgs &g, cudaStream_t s) {
  if (g.wait_limit < kSpinLimit) return launch_matmul_limited<kTileN, OutT, true>(ma, mb, mo, g, s);
  return launch_matmul_limited<kTileN, OutT, false>(ma, mb, mo, g, s);
}

template <typename OutT>
cudaError_t launch_matmul_n(int tile_n, const CUtensorMap &ma, const CUtensorMap &mb, const CUtensorMap &mo, const MatmulArgs &g, cudaStream_t s) {
  if (tile_n == 256) return launch_matmul<256, OutT>(ma, mb, mo, g, s);
  if (tile_n == 128) return launch_matmul<128, OutT>(ma, mb, mo, g, s);
  return launch_matmul<64, OutT>(ma, mb, mo, g, s);
}

template <typename OutT>
cudaError_t launch_split_sum(const float *part, int splits, int64_t stride, int64_t count, int N, const float *bias, void *out, cudaStream_t s) {
  const int64_t blocks = (count + 255) / 256;
  return launch_pdl(split_sum_kernel<OutT>, (unsigned)std::min<int64_t>(blocks, 16 * (int64_t)sm_count()), 256u, 0, s,
                    part, splits, stride, count, N, bias, static_cast<OutT *>(out));
}

template <typename T>
cudaError_t launch_quantize(const void *x, const QuantArgs &a, int plain, int trans, cudaStream_t s) {
  const unsigned grid = (unsigned)(a.row_tiles * a.col_tiles);
  const T *p = static_cast<const T *>(x);
  const bool sums = a.column_sums != nullptr;
#define OTB_QUANT(P, R, S) \
  if (plain == P && trans == R && sums == S) return launch_pdl(quantize_kernel<T, P, R, S>, grid, (unsigned)kQuantThreads, 0, s, p, a)
  OTB_QUANT(kRowBlocks, kNone, false);
  OTB_QUANT(kRowBlocks, kSquareBlocks, false);
  OTB_QUANT(kSquareBlocks, kNone, false);
  OTB_QUANT(kSquareBlocks, kSquareBlocks, false);
  OTB_QUANT(kRowBlocks, kColumnBlocks, false);
  OTB_QUANT(kRowBlocks, kColumnBlocks, true);
#undef OTB_QUANT
  return cudaErrorInvalidValue;
}

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

}  // namespace otb

using namespace otb;

extern "C" {

int ot_b200_fp8_quantize(const void *d_x, int64_t rows, int32_t cols, int64_t row_stride, uint32_t flags, int32_t mode,
                         void *d_q, int64_t q_pitch, float *d_scale, void *d_qt, int64_t qt_pitch, float *d_scale_t,
                         float *d_partial_sums, float *d_column_sums, void *stream) {
  const uint32_t types = flags & (OT_B200_BF16 | OT_B200_FP16);
  if ((flags & ~(OT_B200_BF16 | OT_B200_FP16)) || (types & (types - 1)))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: flags may hold one of OT_B200_BF16 and OT_B200_FP16");
  if (!d_x || rows <= 0 || cols <= 0 || rows > INT32_MAX || row_stride < cols)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: x is NULL or its sizes are not 1..2^31-1, or row_stride < cols");
  if (mode < OT_B200_FP8_ROWS || mode > OT_B200_FP8_ROWS_AND_COLUMNS)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: unknown mode %d", mode);
  const bool with_t = mode == OT_B200_FP8_ROWS_AND_SQUARES || mode == OT_B200_FP8_SQUARES_BOTH || mode == OT_B200_FP8_ROWS_AND_COLUMNS;
  const int64_t need = ((int64_t)cols + 15) / 16 * 16, need_t = (rows + 15) / 16 * 16;
  if (!d_q || !d_scale || !aligned16(d_q) || q_pitch % 16 != 0 || q_pitch < need)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: q and scale must be non-NULL, q 16-byte aligned, its pitch a multiple of 16 of at least cols");
  if (with_t && (!d_qt || !d_scale_t || !aligned16(d_qt) || qt_pitch % 16 != 0 || qt_pitch < need_t ||
                 qt_pitch > (rows + kScaleBlock - 1) / kScaleBlock * kScaleBlock))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: qt and scale_t must be non-NULL, qt 16-byte aligned, its pitch a multiple of 16 from rows to rows rounded up to 128");
  if ((d_partial_sums == nullptr) != (d_column_sums == nullptr) || (d_column_sums && mode != OT_B200_FP8_ROWS_AND_COLUMNS))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: column sums come with mode OT_B200_FP8_ROWS_AND_COLUMNS and both of their buffers");
  QuantArgs a;
  a.rows = rows;
  a.ld = row_stride;
  a.cols = cols;
  a.col_tiles = (cols + kScaleBlock - 1) / kScaleBlock;
  a.row_tiles = (rows + kScaleBlock - 1) / kScaleBlock;
  if (a.row_tiles * a.col_tiles > INT32_MAX)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_quantize: more than 2^31 - 1 blocks of 128 x 128");
  const size_t es = types ? 2 : 4;
  a.vec = reinterpret_cast<uintptr_t>(d_x) % (4 * es) == 0 && row_stride % 4 == 0 && cols % 4 == 0;
  a.q = static_cast<uint8_t *>(d_q);
  a.q_pitch = q_pitch;
  a.scale = d_scale;
  a.qt = static_cast<uint8_t *>(d_qt);
  a.qt_pitch = qt_pitch;
  a.scale_t = d_scale_t;
  a.column_sums = d_partial_sums;
  const int plain = (mode == OT_B200_FP8_SQUARES || mode == OT_B200_FP8_SQUARES_BOTH) ? kSquareBlocks : kRowBlocks;
  const int trans = !with_t ? kNone : (mode == OT_B200_FP8_ROWS_AND_COLUMNS ? kColumnBlocks : kSquareBlocks);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (types == OT_B200_BF16) e = launch_quantize<__nv_bfloat16>(d_x, a, plain, trans, s);
  else if (types == OT_B200_FP16) e = launch_quantize<__half>(d_x, a, plain, trans, s);
  else e = launch_quantize<float>(d_x, a, plain, trans, s);
  if (e == cudaSuccess && d_column_sums)
    e = launch_pdl(column_sum_kernel, (unsigned)((cols + 7) / 8), 256u, 0, s, (const float *)d_partial_sums, a.row_tiles, (int)cols, d_column_sums);
  if (e != cudaSuccess) return fail(OT_B200_ERR_CUDA, "ot_b200_fp8_quantize: %s", cudaGetErrorString(e));
  return OT_B200_OK;
}

int ot_b200_fp8_matmul_workspace_bytes(int64_t M, int64_t N, int64_t K, uint64_t *bytes_out) {
  if (!bytes_out || M <= 0 || N <= 0 || K <= 0 || M > INT32_MAX || N > INT32_MAX || K > INT32_MAX)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: sizes must be 1..2^31-1");
  const MatmulPlan p = plan_matmul(M, N, K, sm_count());
  *bytes_out = p.splits > 1 ? (uint64_t)p.splits * whole_tiles(M) * N * sizeof(float) : 0;
  return OT_B200_OK;
}

// Which error record a call writes to, or none: what begin_reported_call found.  An entry point
// of several launches asks before the first of them.
struct Report {
  int32_t *sticky = nullptr;
  int32_t seq = 0;
};

// The product; `report` NULL: it asks for the error record itself.
static int matmul(const void *d_a, int64_t a_pitch, const float *d_scale_a, const void *d_b, int64_t b_pitch,
                  const float *d_scale_b, const float *d_bias, int64_t M, int64_t N, int64_t K, uint32_t flags,
                  void *d_workspace, uint64_t workspace_bytes, void *d_out, const Report *report, void *stream) {
  const uint32_t types = flags & (OT_B200_BF16 | OT_B200_FP16);
  if ((flags & ~(OT_B200_BF16 | OT_B200_FP16 | OT_B200_REPORT_ERRORS)) || (types & (types - 1)))
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: flags may hold one of OT_B200_BF16 and OT_B200_FP16, and OT_B200_REPORT_ERRORS");
  if (!d_a || !d_b || !d_scale_a || !d_scale_b || !d_out)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: NULL pointer");
  if (!aligned16(d_a) || !aligned16(d_b) || a_pitch % 16 != 0 || b_pitch % 16 != 0 || a_pitch < K || b_pitch < K)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: operands must be 16-byte aligned, their pitches multiples of 16 of at least K");
  uint64_t need = 0;
  const int rc = ot_b200_fp8_matmul_workspace_bytes(M, N, K, &need);
  if (rc) return rc;
  const size_t es = types ? 2 : 4;
  if (reinterpret_cast<uintptr_t>(d_out) % es != 0)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: out is not aligned to its type");
  if (need > 0 && (!d_workspace || workspace_bytes < need || !aligned16(d_workspace)))
    return fail(OT_B200_ERR_WORKSPACE, "ot_b200_fp8_matmul: workspace missing, misaligned or smaller than %llu bytes", (unsigned long long)need);
  MatmulArgs g;
  g.wait_limit = wait_limit();
  if (report != nullptr) {
    g.sticky = report->sticky;
    g.seq = report->seq;
  } else {
    const int begun = begin_reported_call(flags, &g.sticky, &g.seq);
    if (begun) return begun;
  }
  const MatmulPlan p = plan_matmul(M, N, K, sm_count());
  CUtensorMap ma, mb;
  if (!make_tensor_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, d_a, (uint64_t)M, (uint64_t)K, (uint64_t)a_pitch, kTileM, kScaleBlock) ||
      !make_tensor_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, d_b, (uint64_t)N, (uint64_t)K, (uint64_t)b_pitch, (uint32_t)p.tile_n, kScaleBlock))
    return fail(OT_B200_ERR_CUDA, "ot_b200_fp8_matmul: the driver's tensor-map encoder is not available or refused the operands");
  g.sa = d_scale_a;
  g.sb = d_scale_b;
  g.M = M;
  g.N = (int)N;
  g.k_blocks = (int)((K + kScaleBlock - 1) / kScaleBlock);
  g.n_tiles = (int)((N + p.tile_n - 1) / p.tile_n);
  g.splits = p.splits;
  const int64_t tiles = (M + kTileM - 1) / kTileM * g.n_tiles * p.splits;
  if (tiles > INT32_MAX) return fail(OT_B200_ERR_ARGUMENT, "ot_b200_fp8_matmul: more than 2^31 - 1 tiles");
  g.tiles = (uint32_t)tiles;
  const bool split = p.splits > 1;
  g.bias = split ? nullptr : d_bias;
  g.out = static_cast<unsigned char *>(split ? d_workspace : d_out);
  g.out_rows = split ? whole_tiles(M) : M;
  const size_t out_es = split ? sizeof(float) : es;
  const uint64_t where = reinterpret_cast<uintptr_t>(g.out) | (uint64_t)(N * out_es);
  g.unit = where % 16 == 0 ? 0 : (where % 8 == 0 ? 8 : (where % 4 == 0 ? 4 : 2));
  CUtensorMap mo;
  memset(&mo, 0, sizeof(mo));
  // (stores in float are split over 32 columns, in 16 bits over 64: 128 bytes)
  if (g.unit == 0 &&
      !make_tensor_map(&mo, out_es == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, g.out,
                       (uint64_t)(p.splits * g.out_rows), (uint64_t)N, (uint64_t)(N * out_es), 32, (uint32_t)(128 / out_es)))
    g.unit = 8;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (split || types == 0) e = launch_matmul_n<float>(p.tile_n, ma, mb, mo, g, s);
  else if (types == OT_B200_BF16) e = launch_matmul_n<__nv_bfloat16>(p.tile_n, ma, mb, mo, g, s);
  else e = launch_matmul_n<__half>(p.tile_n, ma, mb, mo, g, s);
  if (e == cudaSuccess && split) {
    const float *part = static_cast<const float *>(d_workspace);
    if (types == 0) e = launch_split_sum<float>(part, p.splits, g.out_rows * N, M * N, (int)N, d_bias, d_out, s);
    else if (types == OT_B200_BF16) e = launch_split_sum<__nv_bfloat16>(part, p.splits, g.out_rows * N, M * N, (int)N, d_bias, d_out, s);
    else e = launch_split_sum<__half>(part, p.splits, g.out_rows * N, M * N, (int)N, d_bias, d_out, s);
  }
  if (e != cudaSuccess) return fail(OT_B200_ERR_CUDA, "ot_b200_fp8_matmul: %s", cudaGetErrorString(e));
  return OT_B200_OK;
}

int ot_b200_fp8_matmul(const void *d_a, int64_t a_pitch, const float *d_scale_a, const void *d_b, int64_t b_pitch,
                       const float *d_scale_b, const float *d_bias, int64_t M, int64_t N, int64_t K, uint32_t flags,
                       void *d_workspace, uint64_t workspace_bytes, void *d_out, void *stream) {
  return matmul(d_a, a_pitch, d_scale_a, d_b, b_pitch, d_scale_b, d_bias, M, N, K, flags, d_workspace, workspace_bytes, d_out,
                nullptr, stream);
}

// Bytes from row to row of a quantised matrix: whole cache lines, so that the 128 bytes of a
// row that one TMA box takes lie in one line and not in two.
static int64_t row_pitch(int64_t n) { return (n + 127) / 128 * 128; }

// x in e4m3, its scales, and the product's own workspace, one behind the other.
static void joiner_layout(int64_t rows, int64_t D, uint64_t *scale_off, uint64_t *product_off) {
  const auto align = [](uint64_t n) { return (n + 255) & ~uint64_t(255); };
  *scale_off = align((uint64_t)rows * row_pitch(D));
  *product_off = *scale_off + align((uint64_t)rows * ((D + kScaleBlock - 1) / kScaleBlock) * sizeof(float));
}

int ot_b200_joiner_logits_workspace_bytes(int64_t rows, int32_t D, int32_t V, uint64_t *bytes_out) {
  uint64_t product = 0, scale_off, product_off;
  const int rc = ot_b200_fp8_matmul_workspace_bytes(rows, V, D, &product);
  if (rc) return rc;
  joiner_layout(rows, D, &scale_off, &product_off);
  *bytes_out = product_off + product;
  return OT_B200_OK;
}

int ot_b200_joiner_logits(const void *d_x, int64_t rows, int32_t D, int64_t row_stride, uint32_t x_flags, const void *d_w,
                          int64_t w_pitch, const float *d_w_scale, int32_t V, const float *d_bias, uint32_t out_flags,
                          void *d_workspace, uint64_t workspace_bytes, void *d_out, void *stream) {
  uint64_t need = 0, scale_off, product_off;
  int rc = ot_b200_joiner_logits_workspace_bytes(rows, D, V, &need);
  if (rc) return rc;
  if (!d_workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(d_workspace) % 256 != 0)
    return fail(OT_B200_ERR_WORKSPACE, "ot_b200_joiner_logits: workspace missing, not 256-byte aligned or smaller than %llu bytes", (unsigned long long)need);
  Report report;
  rc = begin_reported_call(out_flags, &report.sticky, &report.seq);
  if (rc) return rc;
  joiner_layout(rows, D, &scale_off, &product_off);
  char *ws = static_cast<char *>(d_workspace);
  const int64_t pitch = row_pitch(D);
  float *scale = reinterpret_cast<float *>(ws + scale_off);
  rc = ot_b200_fp8_quantize(d_x, rows, D, row_stride, x_flags, OT_B200_FP8_ROWS, ws, pitch, scale, nullptr, 0, nullptr, nullptr, nullptr, stream);
  if (rc) return rc;
  return matmul(ws, pitch, scale, d_w, w_pitch, d_w_scale, d_bias, rows, V, D, out_flags, ws + product_off,
                workspace_bytes - product_off, d_out, &report, stream);
}

// The training form's buffers, one behind the other (0 bytes where a gradient is not asked for).
namespace {
struct TrainLayout {
  // kept from the forward to the backward call: W^T and X^T in blocks of 128 x 128
  uint64_t wt = 0, wt_scale = 0, xt = 0, xt_scale = 0, saved = 0;
  // forward scratch
  uint64_t w = 0, w_scale = 0, x = 0, x_scale = 0, f_product = 0, forward = 0;
  // backward scratch: the gradient of the logits along its rows and along its columns
  uint64_t g = 0, g_scale = 0, gt = 0, gt_scale = 0, sums = 0, b_product = 0, backward = 0;
};

int train_layout(int64_t rows, int64_t D, int64_t V, int need_x, int need_w, int need_b, TrainLayout *t) {
  uint64_t p = 0, px = 0, pw = 0;
  int rc = ot_b200_fp8_matmul_workspace_bytes(rows, V, D, &p);
  if (!rc && need_x) rc = ot_b200_fp8_matmul_workspace_bytes(rows, D, V, &px);
  if (!rc && need_w) rc = ot_b200_fp8_matmul_workspace_bytes(V, D, rows, &pw);
  if (rc) return rc;
  const auto put = [](uint64_t *at, uint64_t *end, uint64_t bytes) {
    *at = *end;
    *end = (*end + bytes + 255) & ~uint64_t(255);
  };
  const auto blocks = [](int64_t n) { return (uint64_t)((n + kScaleBlock - 1) / kScaleBlock); };
  put(&t->wt, &t->saved, need_x ? (uint64_t)D * row_pitch(V) : 0);
  put(&t->wt_scale, &t->saved, need_x ? blocks(D) * blocks(V) * 4 : 0);
  put(&t->xt, &t->saved, need_w ? (uint64_t)D * row_pitch(rows) : 0);
  put(&t->xt_scale, &t->saved, need_w ? blocks(D) * blocks(rows) * 4 : 0);
  put(&t->w, &t->forward, (uint64_t)V * row_pitch(D));
  put(&t->w_scale, &t->forward, blocks(V) * blocks(D) * 4);
  put(&t->x, &t->forward, (uint64_t)rows * row_pitch(D));
  put(&t->x_scale, &t->forward, (uint64_t)rows * blocks(D) * 4);
  put(&t->f_product, &t->forward, p);
  put(&t->g, &t->backward, (uint64_t)rows * row_pitch(V));
  put(&t->g_scale, &t->backward, (uint64_t)rows * blocks(V) * 4);
  put(&t->gt, &t->backward, (need_w || need_b) ? (uint64_t)V * row_pitch(rows) : 0);
  put(&t->gt_scale, &t->backward, (need_w || need_b) ? (uint64_t)V * blocks(rows) * 4 : 0);
  put(&t->sums, &t->backward, need_b ? blocks(rows) * (uint64_t)V * 4 : 0);
  put(&t->b_product, &t->backward, px > pw ? px : pw);
  return OT_B200_OK;
}

int check_train_buffers(const char *who, const TrainLayout &t, const void *saved, uint64_t saved_bytes, const void *workspace,
                        uint64_t workspace_bytes, uint64_t need) {
  if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 != 0 || (t.saved && (!saved || reinterpret_cast<uintptr_t>(saved) % 256 != 0)))
    return fail(OT_B200_ERR_WORKSPACE, "%s: a buffer is missing or not 256-byte aligned", who);
  if (workspace_bytes < need || saved_bytes < t.saved)
    return fail(OT_B200_ERR_WORKSPACE, "%s: the workspace has fewer than %llu bytes or the saved buffer fewer than %llu", who,
                (unsigned long long)need, (unsigned long long)t.saved);
  return OT_B200_OK;
}
}  // namespace

int ot_b200_joiner_train_bytes(int64_t rows, int32_t D, int32_t V, int32_t need_x, int32_t need_w, int32_t need_b,
                               uint64_t *saved_out, uint64_t *forward_out, uint64_t *backward_out) {
  if (!saved_out || !forward_out || !backward_out)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_joiner_train_bytes: NULL output");
  TrainLayout t;
  const int rc = train_layout(rows, D, V, need_x, need_w, need_b, &t);
  if (rc) return rc;
  *saved_out = t.saved;
  *forward_out = t.forward;
  *backward_out = t.backward;
  return OT_B200_OK;
}

int ot_b200_joiner_train_forward_sized(const void *d_x, int64_t rows, int32_t D, int64_t x_stride, uint32_t x_flags, const void *d_w,
                                       int32_t V, int64_t w_stride, uint32_t w_flags, const float *d_bias, uint32_t out_flags,
                                       int32_t need_x, int32_t need_w, void *d_saved, uint64_t saved_bytes, void *d_workspace,
                                       uint64_t workspace_bytes, void *d_out, void *stream) {
  TrainLayout t;
  int rc = train_layout(rows, D, V, need_x, need_w, 0, &t);
  if (rc) return rc;
  rc = check_train_buffers("ot_b200_joiner_train_forward", t, d_saved, saved_bytes, d_workspace, workspace_bytes, t.forward);
  if (rc) return rc;
  Report report;
  rc = begin_reported_call(out_flags, &report.sticky, &report.seq);
  if (rc) return rc;
  char *ws = static_cast<char *>(d_workspace), *saved = static_cast<char *>(d_saved);
  const auto at = [](char *base, uint64_t off) { return reinterpret_cast<float *>(base + off); };
  rc = ot_b200_fp8_quantize(d_w, V, D, w_stride, w_flags, need_x ? OT_B200_FP8_SQUARES_BOTH : OT_B200_FP8_SQUARES,
                            ws + t.w, row_pitch(D), at(ws, t.w_scale), need_x ? saved + t.wt : nullptr,
                            need_x ? row_pitch(V) : 0, need_x ? at(saved, t.wt_scale) : nullptr, nullptr, nullptr, stream);
  if (!rc)
    rc = ot_b200_fp8_quantize(d_x, rows, D, x_stride, x_flags, need_w ? OT_B200_FP8_ROWS_AND_SQUARES : OT_B200_FP8_ROWS,
                              ws + t.x, row_pitch(D), at(ws, t.x_scale), need_w ? saved + t.xt : nullptr,
                              need_w ? row_pitch(rows) : 0, need_w ? at(saved, t.xt_scale) : nullptr, nullptr, nullptr, stream);
  if (!rc)
    rc = matmul(ws + t.x, row_pitch(D), at(ws, t.x_scale), ws + t.w, row_pitch(D), at(ws, t.w_scale), d_bias, rows, V, D, out_flags,
                ws + t.f_product, t.forward - t.f_product, d_out, &report, stream);
  return rc;
}

int ot_b200_joiner_train_backward_sized(const void *d_g, int64_t rows, int32_t V, int64_t g_stride, uint32_t g_flags, int32_t D,
                                        const void *d_saved, uint64_t saved_bytes, void *d_gx, uint32_t x_flags, void *d_gw,
                                        uint32_t w_flags, float *d_gb, uint32_t flags, void *d_workspace, uint64_t workspace_bytes,
                                        void *stream) {
  TrainLayout t;
  int rc = train_layout(rows, D, V, d_gx != nullptr, d_gw != nullptr, d_gb != nullptr, &t);
  if (rc) return rc;
  rc = check_train_buffers("ot_b200_joiner_train_backward", t, d_saved, saved_bytes, d_workspace, workspace_bytes, t.backward);
  if (rc) return rc;
  if (flags & ~OT_B200_REPORT_ERRORS)
    return fail(OT_B200_ERR_ARGUMENT, "ot_b200_joiner_train_backward: flags may hold OT_B200_REPORT_ERRORS");
  Report report;
  rc = begin_reported_call(flags, &report.sticky, &report.seq);
  if (rc) return rc;
  char *ws = static_cast<char *>(d_workspace), *saved = static_cast<char *>(const_cast<void *>(d_saved));
  const auto at = [](char *base, uint64_t off) { return reinterpret_cast<float *>(base + off); };
  const bool columns = d_gw || d_gb;
  rc = ot_b200_fp8_quantize(d_g, rows, V, g_stride, g_flags, columns ? OT_B200_FP8_ROWS_AND_COLUMNS : OT_B200_FP8_ROWS, ws + t.g,
                            row_pitch(V), at(ws, t.g_scale), columns ? ws + t.gt : nullptr, columns ? row_pitch(rows) : 0,
                            columns ? at(ws, t.gt_scale) : nullptr, d_gb ? at(ws, t.sums) : nullptr, d_gb, stream);
  if (!rc && d_gx)
    rc = matmul(ws + t.g, row_pitch(V), at(ws, t.g_scale), saved + t.wt, row_pitch(V), at(saved, t.wt_scale), nullptr, rows, D, V,
                x_flags | flags, ws + t.b_product, t.backward - t.b_product, d_gx, &report, stream);
  if (!rc && d_gw)
    rc = matmul(ws + t.gt, row_pitch(rows), at(ws, t.gt_scale), saved + t.xt, row_pitch(rows), at(saved, t.xt_scale), nullptr, V, D, rows,
                w_flags | flags, ws + t.b_product, t.backward - t.b_product, d_gw, &report, stream);
  return rc;
}

int ot_b200_joiner_train_forward(const void *d_x, int64_t rows, int32_t D, int64_t x_stride, uint32_t x_flags, const void *d_w,
                                 int32_t V, int64_t w_stride, uint32_t w_flags, const float *d_bias, uint32_t out_flags,
                                 int32_t need_x, int32_t need_w, void *d_saved, void *d_workspace, void *d_out, void *stream) {
  return ot_b200_joiner_train_forward_sized(d_x, rows, D, x_stride, x_flags, d_w, V, w_stride, w_flags, d_bias, out_flags, need_x, need_w,
                                            d_saved, UINT64_MAX, d_workspace, UINT64_MAX, d_out, stream);
}

int ot_b200_joiner_train_backward(const void *d_g, int64_t rows, int32_t V, int64_t g_stride, uint32_t g_flags, int32_t D,
                                  const void *d_saved, void *d_gx, uint32_t x_flags, void *d_gw, uint32_t w_flags, float *d_gb,
                                  uint32_t flags, void *d_workspace, void *stream) {
  return ot_b200_joiner_train_backward_sized(d_g, rows, V, g_stride, g_flags, D, d_saved, UINT64_MAX, d_gx, x_flags, d_gw, w_flags, d_gb,
                                             flags, d_workspace, UINT64_MAX, stream);
}

}  // extern "C"
