// cross_entropy.hip -- the loss of supervised training over a large
// vocabulary, with the gradients of the states and of the table, without
// keeping the logits.
//
//   l[t, v] = sum_h x[t, h] w[v, h],   lse[t] = log sum_v exp l[t, v]
//   loss    = sum_t r[t] ((1 - s)(lse - l[t, y]) + s (lse - mean_v l))
//   g[t, v] = exp(l - lse) - (1 - s)[v = y] - s / V
//   dx[t]   = r[t] sum_v g[t, v] w[v],   dw[v] = sum_t r[t] g[t, v] x[t]
//
// The rows' statistics take a first product, whose tiles leave a maximum, a
// sum of exponentials and a sum of logits a row.  Then the vocabulary goes in
// pieces: the logits of a piece are made again, their slopes g are stored in 16
// bits (of a size that the last level's cache holds), and two products take
// them to dx, whose sums over the pieces stay in 32 bits, and to dw.  Four
// products where a stored [rows, vocab] would need three.
//
// r[t] = m 2^e, m in [1, 2).  g is stored times m, so that its rounding is
// relative to itself also in float16 (there times 2^14: |g m| < 2, and what is
// below 2^-28 of it loses digits that no sum keeps); dx is multiplied by 2^e at
// its end, and dw takes rows of x times 2^(e - the largest e), which is exact
// but for parts that the largest row's swallow.  A row without a target, or of
// weight 0, has g = 0 and such an x of 0, whatever its x holds.
#include <algorithm>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, __bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 x 16 tile by 32: lane l gives 8 of row l % 16 of either operand, from
// column 8 (l / 16) on; it gets rows 4 (l / 16) ... + 3 of column l % 16.

// What g is stored times, beside m.
template <typename T>
constexpr float kUp = 1.0f;
template <>
constexpr float kUp<_Float16> = 16384.0f;

struct Args {
  const void* x;
  const void* weight;
  const int32_t* target;
  const float* row_weight;
  void* dx;
  void* dweight;
  float* loss;
  float* logp;
  int64_t x_stride, weight_stride, dx_stride, dweight_stride;
  uint32_t rows, rows64, hidden, hidden64, vocab, tiles;  // (up to whole 64s); token tiles of the statistics
  float smoothing;
  // workspace
  float* mant;      // [rows64]: m, 0 without a target
  float* power;     // [rows64]: 2^e
  float* largest;   // 2^(the largest e)
  float* part;      // [3][tiles][rows64]: max, sum of exponentials, sum of logits
  float* picked;    // [rows64]: the target's logit
  float* top;       // [rows64]: max
  float* logsum;    // [rows64]: lse - max
  float* terms;     // [rows64]: of the loss
  void* xs;         // [rows64][hidden64]: x times 2^(e - largest)
  void* slopes;     // [rows64][piece]
  float* dxs;       // [splits][rows64][hidden64]
  // a piece of the vocabulary
  uint32_t piece, first, splits, split_steps;  // tokens of it; its first; parts of dx and their steps of 64
};

// --- rows -------------------------------------------------------------------

__device__ __forceinline__ int exponent_of(const Args& a, uint32_t t, float* m) {
  const float r = a.row_weight[t];
  *m = a.target[t] < 0 ? 0.0f : r;
  if (*m == 0.0f || !(fabsf(r) < INFINITY)) return -1000;  // as it is
  int e;
  *m = 2.0f * frexpf(r, &e);
  return e - 1;
}

// A wave a row.
template <typename T>
__global__ void __launch_bounds__(256) xent_rows(Args a) {
  __shared__ int biggest[4];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int big = -1000;
  for (uint32_t t = tid; t < a.rows; t += 256) {
    float m;
    big = max(big, exponent_of(a, t, &m));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) big = max(big, __shfl_xor(big, d, 64));
  if (lane == 0) biggest[wave] = big;
  __syncthreads();
  big = max(max(biggest[0], biggest[1]), max(biggest[2], biggest[3]));
  if (big == -1000) big = 0;
  const uint32_t t = blockIdx.x * 4 + wave;
  float m = 0.0f;
  int e = t < a.rows ? exponent_of(a, t, &m) : 0;
  if (e == -1000) e = m == 0.0f ? 0 : big;
  if (lane == 0) {
    a.mant[t] = m;
    a.power[t] = ldexpf(1.0f, e);
    if (t == 0) *a.largest = ldexpf(1.0f, big);
  }
  if (!a.dweight) return;
  const T* row = (const T*)a.x + (int64_t)min(t, a.rows - 1) * a.x_stride;
  for (uint32_t k = lane * 8; k < a.hidden64; k += 512) {
    u32x4 v{};
    if (m != 0.0f) {
      v = load_row_vec(row, k, a.hidden, (T)0.0f);
      if (e != big) {
        float f[8];
        to_float<T>(v, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = ldexpf(f[i], e - big);
        v = from_float<T>(f);
      }
    }
    ((u32x4*)a.xs)[((uint64_t)t * a.hidden64 + k) / 8] = v;
  }
}

// 64 rows by 16 waves, which take the tiles in turn.
__global__ void __launch_bounds__(1024) xent_join(Args a) {
  __shared__ float sm[16][64], ss[16][64], sl[16][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = blockIdx.x * 64 + lane;
  const uint64_t each = (uint64_t)a.tiles * a.rows64;
  MaxSum p{-INFINITY, 0.0f};
  float l = 0.0f;
#pragma unroll 4
  for (uint32_t i = wave; i < a.tiles; i += 16) {
    const uint64_t at = (uint64_t)i * a.rows64 + t;
    p = merge(p, MaxSum{a.part[at], a.part[each + at]});
    l += a.part[2 * each + at];
  }
  sm[wave][lane] = p.m;
  ss[wave][lane] = p.s;
  sl[wave][lane] = l;
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int w = 1; w < 16; ++w) {
    p = merge(p, MaxSum{sm[w][lane], ss[w][lane]});
    l += sl[w][lane];
  }
  const int32_t y = t < a.rows ? a.target[t] : -1;
  const float base = exp_base(p.m);
  float ls = logf(p.s);
  float at = y >= 0 && (uint32_t)y < a.vocab ? a.picked[t] - base : NAN;
  if (y >= 0 && (uint32_t)y >= a.vocab) ls = NAN;  // and with it the row's slopes
  a.top[t] = base;
  a.logsum[t] = ls;
  float term = 0.0f;
  if (y >= 0) {
    a.logp[t] = at - ls;
    const float r = a.row_weight[t];
    term = (1.0f - a.smoothing) * (ls - at);
    if (a.smoothing != 0.0f) term += a.smoothing * (ls - (l / (float)a.vocab - base));
    term = r == 0.0f ? 0.0f : r * term;
  } else if (t < a.rows) {
    a.logp[t] = 0.0f;
  }
  a.terms[t] = term;
}

__global__ void __launch_bounds__(1024) xent_loss(Args a) {
  __shared__ float waves[16];
  float sum = 0.0f;
  for (uint32_t t = threadIdx.x; t < a.rows; t += 1024) sum += a.terms[t];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  sum = 0.0f;
  for (int w = 0; w < 16; ++w) sum += waves[w];
  *a.loss = sum;
}

// No rows: a table's gradient of zeros.
template <typename T>
__global__ void __launch_bounds__(256) xent_nothing(Args a) {
  T* row = (T*)a.dweight + (int64_t)blockIdx.x * a.dweight_stride;
  for (uint32_t h = threadIdx.x; h < a.hidden; h += 256) row[h] = (T)0.0f;
}

// dx from its parts; a wave a row.
template <typename T>
__global__ void __launch_bounds__(256) xent_states(Args a) {
  const uint32_t lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= a.rows) return;
  const bool none = a.mant[t] == 0.0f;
  const float f = a.power[t] * (1.0f / kUp<T>);
  const uint64_t each = (uint64_t)a.rows64 * a.hidden64;
  for (uint32_t h = lane * 8; h < a.hidden; h += 512) {
    float y[8] = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
      const float* p = a.dxs + s * each + (uint64_t)t * a.hidden64 + h;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] += p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = none ? 0.0f : y[i] * f;
    T* out = (T*)a.dx + (int64_t)t * a.dx_stride + h;
    if (h + 8 <= a.hidden) store_vec(out, from_float<T>(y));
    else store_part(out, (int)(a.hidden - h), from_float<T>(y));
  }
}

// --- products ---------------------------------------------------------------
// Every product is out[j, i] = sum_k P[i, k] Q[j, k] with i along the outputs'
// rows.  An operand lies by k (a row for each i, its k side by side) or across
// it (a row for each k): then LDS holds it as it lies and the matrix operands
// are read transposed, four k of 16 columns an instruction.
enum Kind { kStats, kSlopes, kStates, kTable };

struct Operand {
  const void* base;
  int64_t stride;
  uint32_t rows, columns;  // rows past the end: the last; columns: zero
};

// Any alignment: operands pass registers on their way to LDS, no step ahead.
// Block: 128 of i by 64 of j; wave w has 32 w ... of i, and all of j.
constexpr int kBM = 64, kBN = 128, kBK = 64, kThreads = 256;

template <typename T, bool kAcross, int kB>
struct Stage {
  static constexpr int kRows = kAcross ? kBK : kB, kCols = (kAcross ? kB : kBK) / 8;  // in vectors
  static constexpr int kPitch = kAcross ? kCols + 2 : kCols;
  static constexpr int kVecs = kRows * kPitch, kTurns = kRows * kCols / kThreads;

  static __device__ __forceinline__ void load(const Operand& o, uint32_t i0, uint32_t k0, u32x4 (&r)[kTurns]) {
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const uint32_t at = t * kThreads + threadIdx.x, row = at / kCols, c = at % kCols * 8;
      const T* p = (const T*)o.base + (int64_t)min((kAcross ? k0 : i0) + row, o.rows - 1) * o.stride;
      r[t] = load_row_vec(p, (kAcross ? i0 : k0) + c, o.columns, (T)0.0f);
    }
  }
  static __device__ __forceinline__ void store(u32x4* st, const u32x4 (&r)[kTurns]) {
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
      const uint32_t at = t * kThreads + threadIdx.x, row = at / kCols, c = at % kCols;
      st[row * kPitch + (kAcross ? c : c ^ (row & 7))] = r[t];
    }
  }
  // columns 32 kk + 8 (l / 16) ... + 7 of k, row (16 sub + l % 16) of i
  static __device__ __forceinline__ u32x4 read(const u32x4* st, uint32_t sub, int kk) {
    const uint32_t lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
    if (!kAcross) return st[(sub * 16 + col) * kPitch + ((kk * 4 + q) ^ (col & 7))];
    const char* p = (const char*)(st + (kk * 32 + q * 8 + (col >> 2)) * kPitch) + sub * 32 + (col & 3) * 8;
    union {
      s16x4 h[2];
      u32x4 v;
    } u;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      u.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(p + i * 4 * kPitch * 16));
    return u.v;
  }
};

// What a product leaves.  The wave's i are i0 ..., 16 kN of them, its j j0 ...;
// a lane has four neighbouring i of row j.
template <typename T, Kind kKind, int kN, int kM, int kWaves>
__device__ __forceinline__ void finish(const Args& a, uint32_t tile, uint32_t i0, uint32_t j0, uint32_t split,
                                       f32x4 (&acc)[kN][kM], float (*joined)[3][16 * kM], uint32_t wave) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  if constexpr (kKind == kStats) {
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      const uint32_t t = j0 + s * 16 + col;
      const int32_t y = t < a.rows ? a.target[t] : -1;
      MaxSum p{-INFINITY, 0.0f};
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        float l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t tok = i0 + v * 16 + q * 4 + e;
          l[e] = tok < a.vocab ? acc[v][s][e] : -INFINITY;
          if (tok < a.vocab) sum += l[e];
          if ((int32_t)tok == y && tok < a.vocab) a.picked[t] = l[e];
        }
        add_terms(p, l);
      }
#pragma unroll
      for (int d = 16; d < 64; d *= 2) {
        p = merge(p, MaxSum{__shfl_xor(p.m, d, 64), __shfl_xor(p.s, d, 64)});
        sum += __shfl_xor(sum, d, 64);
      }
      if (q == 0) {
        joined[wave][0][s * 16 + col] = p.m;
        joined[wave][1][s * 16 + col] = p.s;
        joined[wave][2][s * 16 + col] = sum;
      }
    }
    __syncthreads();
    const uint64_t each = (uint64_t)a.tiles * a.rows64;
    for (uint32_t j = threadIdx.x; j < 16 * kM; j += blockDim.x) {
      MaxSum p{joined[0][0][j], joined[0][1][j]};
      float sum = joined[0][2][j];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        p = merge(p, MaxSum{joined[w][0][j], joined[w][1][j]});
        sum += joined[w][2][j];
      }
      const uint64_t at = (uint64_t)tile * a.rows64 + j0 + j;
      a.part[at] = p.m;
      a.part[each + at] = p.s;
      a.part[2 * each + at] = sum;
    }
  }
  if constexpr (kKind == kSlopes) {
    const float even = a.smoothing / (float)a.vocab, own = 1.0f - a.smoothing;
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      const uint32_t t = j0 + s * 16 + col;
      const int32_t y = t < a.rows ? a.target[t] : -1;
      const float m = a.mant[t] * kUp<T>, top = a.top[t], ls = a.logsum[t];
      T* row = (T*)a.slopes + (uint64_t)t * a.piece + (i0 - a.first);
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        union {
          uint2 u;
          T g[4];
        } o;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t tok = i0 + v * 16 + q * 4 + e;
          float g = exp_term(acc[v][s][e] - top, ls) - even;
          if ((int32_t)tok == y) g -= own;
          o.g[e] = (T)(m != 0.0f && tok < a.vocab ? g * m : 0.0f);
        }
        *(uint2*)(row + v * 16 + q * 4) = o.u;
      }
    }
  }
  if constexpr (kKind == kStates) {
#pragma unroll
    for (int s = 0; s < kM; ++s)
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        const uint32_t h = i0 + v * 16 + q * 4;
        if (h >= a.hidden64) continue;
        f32x4* to = (f32x4*)(a.dxs + ((uint64_t)split * a.rows64 + j0 + s * 16 + col) * a.hidden64 + h);
        *to = a.first ? *to + acc[v][s] : acc[v][s];
      }
  }
  if constexpr (kKind == kTable) {
    const float f = *a.largest * (1.0f / kUp<T>);
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      const uint32_t tok = a.first + j0 + s * 16 + col;
      if (tok >= a.vocab) continue;
      T* row = (T*)a.dweight + (int64_t)tok * a.dweight_stride;
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        const uint32_t h = i0 + v * 16 + q * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (h + e < a.hidden) row[h + e] = (T)(acc[v][s][e] * f);
      }
    }
  }
}

template <typename T, Kind kKind>
__global__ void __launch_bounds__(kThreads) xent_product(Args a) {
  using P = Stage<T, kKind >= kStates, kBN>;
  using Q = Stage<T, kKind == kTable, kBM>;
  __shared__ u32x4 ps[P::kVecs], qs[Q::kVecs];
  __shared__ float joined[4][3][kBM];
  const uint32_t wave = threadIdx.x >> 6;
  // tiles of i, j and, for dx, of k
  const uint32_t js = kKind == kTable ? a.piece / kBM : a.rows64 / kBM;
  const uint32_t tj = blockIdx.x % js, rest = blockIdx.x / js;
  uint32_t ti = rest, split = 0, k0 = 0, k1;
  Operand po, qo;
  if (kKind == kStats || kKind == kSlopes) {
    po = Operand{a.weight, a.weight_stride, a.vocab, a.hidden};
    qo = Operand{a.x, a.x_stride, a.rows, a.hidden};
    k1 = a.hidden64;
  } else if (kKind == kStates) {
    ti = rest % ((a.hidden64 + kBN - 1) / kBN);
    split = rest / ((a.hidden64 + kBN - 1) / kBN);
    const uint32_t last = a.vocab - 1 - a.first;  // (columns of g past the vocabulary are zero)
    po = Operand{(const T*)a.weight + (int64_t)a.first * a.weight_stride, a.weight_stride, last + 1, a.hidden};
    qo = Operand{a.slopes, a.piece, a.rows64, a.piece};
    k0 = split * a.split_steps * kBK;
    k1 = min(k0 + a.split_steps * kBK, a.piece);
  } else {
    po = Operand{a.xs, a.hidden64, a.rows64, a.hidden64};
    qo = Operand{a.slopes, a.piece, a.rows64, a.piece};
    k1 = a.rows64;
  }
  const uint32_t i0 = ti * kBN + (kKind == kSlopes ? a.first : 0), j0 = tj * kBM;
  f32x4 acc[2][kBM / 16] = {};
  for (uint32_t k = k0; k < k1; k += kBK) {
    u32x4 pr[P::kTurns], qr[Q::kTurns];
    P::load(po, i0, k, pr);
    Q::load(qo, j0, k, qr);
    __syncthreads();
    P::store(ps, pr);
    Q::store(qs, qr);
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kBK / 32; ++kk) {
      u32x4 pf[2], qf[kBM / 16];
#pragma unroll
      for (int i = 0; i < 2; ++i) pf[i] = P::read(ps, wave * 2 + i, kk);
#pragma unroll
      for (int j = 0; j < kBM / 16; ++j) qf[j] = Q::read(qs, j, kk);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kBM / 16; ++j) acc[i][j] = mfma(pf[i], qf[j], acc[i][j], T{});
    }
  }
  finish<T, kKind, 2, kBM / 16, 4>(a, ti, i0 + wave * 32, j0, split, acc, joined, wave);
}

// --- plan -------------------------------------------------------------------

constexpr uint32_t kCUs = 256;

struct Plan {
  uint64_t mant, power, largest, part, picked, top, logsum, terms, xs, slopes, dxs, bytes;
  uint32_t rows64, hidden64, tiles, piece, splits, split_steps;
};

Plan plan(const ft_cross_entropy_loss_args& a) {
  Plan p{};
  Arena ar;
  p.rows64 = (uint32_t)round_up(a.rows, 64);
  p.hidden64 = (uint32_t)round_up(a.hidden, 64);
  p.tiles = (a.vocab + kBN - 1) / kBN;
  const uint64_t r = p.rows64;
  p.mant = ar.take(r * 4);
  p.power = ar.take(r * 4);
  p.largest = ar.take(4);
  p.part = ar.take(3 * r * p.tiles * 4);
  p.picked = ar.take(r * 4);
  p.top = ar.take(r * 4);
  p.logsum = ar.take(r * 4);
  p.terms = ar.take(r * 4);
  if (a.dx || a.dweight) {
    // a piece's slopes: up to 128 MB, half of the last level's cache
    const uint64_t whole = round_up(a.vocab, 256);
    p.piece = (uint32_t)std::min(whole, std::max<uint64_t>(256, (128ull << 20) / std::max<uint64_t>(64, r) / 512 * 256));
    p.slopes = ar.take(r * p.piece * 2);
  }
  if (a.dweight) p.xs = ar.take(r * p.hidden64 * 2);
  if (a.dx) {
    // as many parts of the sum over tokens as fill the chip
    const uint64_t tiles = std::max<uint64_t>(1, r / kBM * ((p.hidden64 + kBN - 1) / kBN));
    const uint32_t steps = p.piece / kBK;
    const uint64_t want = std::max<uint64_t>(1, 2 * kCUs / tiles);
    p.split_steps = (uint32_t)std::max<uint64_t>(4, (steps + want - 1) / want);
    p.splits = (steps + p.split_steps - 1) / p.split_steps;
    p.dxs = ar.take((uint64_t)p.splits * r * p.hidden64 * 4);
  }
  p.bytes = ar.used;
  return p;
}

template <typename T>
hipError_t launch(Args a, hipStream_t s) {
  if (a.rows == 0) {
    const hipError_t e = start(xent_loss, 1, 1024, s, a);
    return e == hipSuccess && a.dweight ? start(xent_nothing<T>, a.vocab, 256, s, a) : e;
  }
  hipError_t e = start(xent_rows<T>, a.rows64 / 4, 256, s, a);
  if (e != hipSuccess) return e;
  const uint64_t js = a.rows64 / kBM;
  e = start(xent_product<T, kStats>, a.tiles * js, kThreads, s, a);
  if (e != hipSuccess) return e;
  e = start(xent_join, a.rows64 / 64, 1024, s, a);
  if (e != hipSuccess) return e;
  e = start(xent_loss, 1, 1024, s, a);
  if (e != hipSuccess || !(a.dx || a.dweight)) return e;
  const uint64_t hs = (a.hidden64 + kBN - 1) / kBN;
  for (a.first = 0; a.first < a.vocab; a.first += a.piece) {
    e = start(xent_product<T, kSlopes>, a.piece / kBN * js, kThreads, s, a);
    if (e != hipSuccess) return e;
    if (a.dx) {
      e = start(xent_product<T, kStates>, hs * js * a.splits, kThreads, s, a);
      if (e != hipSuccess) return e;
    }
    if (a.dweight) {
      e = start(xent_product<T, kTable>, hs * (a.piece / kBM), kThreads, s, a);
      if (e != hipSuccess) return e;
    }
  }
  if (!a.dx) return hipSuccess;
  return start(xent_states<T>, (a.rows + 3) / 4, 256, s, a);
}

}  // namespace

uint64_t cross_entropy_loss_workspace(const ft_cross_entropy_loss_args& a) { return plan(a).bytes; }

hipError_t launch_cross_entropy_loss(const ft_cross_entropy_loss_args& q, uint8_t* ws, hipStream_t s) {
  const Plan p = plan(q);
  Args a{};
  a.x = q.x;
  a.weight = q.weight;
  a.target = q.target;
  a.row_weight = q.row_weight;
  a.dx = q.dx;
  a.dweight = q.dweight;
  a.loss = q.loss;
  a.logp = q.logp;
  a.x_stride = q.x_stride;
  a.weight_stride = q.weight_stride;
  a.dx_stride = q.dx_stride;
  a.dweight_stride = q.dweight_stride;
  a.rows = (uint32_t)q.rows;
  a.rows64 = p.rows64;
  a.hidden = q.hidden;
  a.hidden64 = p.hidden64;
  a.vocab = q.vocab;
  a.tiles = p.tiles;
  a.smoothing = q.smoothing;
  a.mant = (float*)(ws + p.mant);
  a.power = (float*)(ws + p.power);
  a.largest = (float*)(ws + p.largest);
  a.part = (float*)(ws + p.part);
  a.picked = (float*)(ws + p.picked);
  a.top = (float*)(ws + p.top);
  a.logsum = (float*)(ws + p.logsum);
  a.terms = (float*)(ws + p.terms);
  a.xs = ws + p.xs;
  a.slopes = ws + p.slopes;
  a.dxs = (float*)(ws + p.dxs);
  a.piece = p.piece;
  a.splits = p.splits;
  a.split_steps = p.split_steps;
  return q.dtype == FT_BF16 ? launch<__bf16>(a, s) : launch<_Float16>(a, s);
}

}  // namespace fto
