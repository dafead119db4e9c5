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
// Launches: the statistics (xent_tile or xent_product, kStats), their join with
// the rows' factors and scaled states (xent_rows), then for each piece the
// slopes and the two gradients' products, at last dx from its parts
// (xent_states).  For few rows: xent_few twice, xent_states.
//
// Many rows are bound by the matrix cores (4,096 rows x 262,144 x 1,024 bf16: 7.7
// ms, 1.14 PFLOP/s over the four products, where the library's four take 8.75),
// few by the table's way from and to memory (10 rows of these sizes: 303 us for
// two reads and a write of 537 MB, 5.3 TB/s); one key's 8 rows x 32,768 x 512 take
// 37 us, three launches.
//
// r[t] = m 2^e, m in [1, 2).  g is stored times m, so that its rounding is
// relative to itself also in float16 (there times 2^14: |g m| < 2, and what is
// below 2^-28 of it loses digits that no sum keeps), and times a factor within
// 2^-8 of 1 by which the target's slope, the largest as a rule, is one of the
// type's numbers.  dx is multiplied by r over both at its end; dw takes rows of
// x times that over 2^(the largest e), rounded to x's type.  So dx has about
// its own rounding alone, and dw that and x's.  A row without a target, or of
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
  float* factor;    // [rows64]: what slopes are stored times, 0 without a target
  float* power;     // [rows64]: r over it
  float* largest;   // 2^(the largest e)
  float* part;      // [3][tiles][rows64]: c, s, sum of logits
  float* picked;    // [rows64]: the target's logit
  float* top;       // [rows64]: c
  float* logsum;    // [rows64]: log2 s
  float* terms;     // [rows64]: of the loss
  void* xs;         // [rows64][hidden64]: x times 2^(e - largest)
  void* slopes;     // [rows64][slope_stride]
  float* dxs;       // [splits][rows64][hidden64]
  // a piece of the vocabulary
  uint32_t piece, first, width;  // most tokens of it; its first; its tokens up to whole 256s
  uint32_t slope_stride;  // of the slopes' rows
  uint32_t splits, split_steps;  // parts of dx and their steps of 64
  uint64_t split_stride;
  uint32_t tiled;    // rows that the tiles cover
  uint32_t prepare;  // workgroups in front of the statistics' that prepare rows
};

// A part of a row's statistics is (c, s): s = sum of 2^(l log2 e - c), c the
// part's largest l, times log2 e in 32 bits (0 where that is -infinity).  The
// product and the difference are one fused step, so a term's exponent is
// rounded once, relative to itself.  A NaN or +infinity makes s NaN.
struct Part {
  float c, s;
};
__device__ __forceinline__ float power_of(float l, float c) { return exp2_raw(__builtin_fmaf(l, kLog2e, -c)); }
__device__ __forceinline__ Part join(Part a, Part b) {
  // (a part of nothing has s = 0 and takes no part in c)
  const float c = a.s == 0.0f ? b.c : b.s == 0.0f ? a.c : fmaxf(a.c, b.c);
  return Part{c, (a.s == 0.0f ? 0.0f : a.s * exp2_raw(a.c - c)) + (b.s == 0.0f ? 0.0f : b.s * exp2_raw(b.c - c))};
}

// --- rows -------------------------------------------------------------------

__device__ __forceinline__ int exponent_of(const Args& a, uint32_t t, float* m) {
  const float r = a.row_weight[t];
  *m = a.target[t] < 0 ? 0.0f : r;
  if (*m == 0.0f || !(fabsf(r) < INFINITY)) return -1000;  // as it is
  int e;
  *m = 2.0f * frexpf(r, &e);
  return e - 1;
}

// The target's slope over r, as the slopes' product makes it.
__device__ __forceinline__ float target_slope(const Args& a, uint32_t t) {
  const float even = a.smoothing / (float)a.vocab, own = 1.0f - a.smoothing;
  return exp2_raw(__builtin_fmaf(a.picked[t], kLog2e, -a.top[t]) - a.logsum[t]) - even - own;
}

// Rows' factors and, for the table's gradient, their scaled states: a wave of
// kWaves a row.  kFit (past the statistics): a row's slopes are stored times a
// factor next to m for which the target's, the largest as a rule, has no
// rounding; dx is divided by it in 32 bits, the states in their type.
template <typename T, int kWaves, bool kFit>
__device__ __forceinline__ void prepare_rows(const Args& a, uint32_t block) {
  __shared__ int biggest[kWaves];
  const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int big = -1000;
  for (uint32_t t = tid; t < a.rows; t += 64 * kWaves) {
    float m;
    big = max(big, exponent_of(a, t, &m));
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) big = max(big, __shfl_xor(big, d, 64));
  if (lane == 0) biggest[wave] = big;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) big = max(big, biggest[w]);
  if (big == -1000) big = 0;
  const uint32_t t = block * kWaves + wave;
  float m = 0.0f;
  int e = t < a.rows ? exponent_of(a, t, &m) : 0;
  if (e == -1000) e = m == 0.0f ? 0 : big;
  float times = m * kUp<T>, back = 1.0f;  // m = times back / kUp
  if (kFit && m != 0.0f && fabsf(m) < INFINITY) {
    const float g = (uint32_t)a.target[t] < a.vocab ? target_slope(a, t) : NAN;
    // (one that is far below the others is left alone; so is NaN)
    const float fit = (float)(T)(g * times);
    if (fabsf(fit) > 0x1p-10f && fabsf(fit) < INFINITY) {
      back = times;
      times = fit / g;
      back /= times;
    }
  }
  if (lane == 0) {
    a.factor[t] = times;
    a.power[t] = ldexpf(back * (1.0f / kUp<T>), e);
    if (t == 0) *a.largest = ldexpf(1.0f, big);
  }
  if (!a.dweight) return;
  const T* row = (const T*)a.x + (int64_t)min(t, a.rows - 1) * a.x_stride;
  for (uint32_t k = lane * 8; k < a.hidden64; k += 512) {
    u32x4 v{};
    if (m != 0.0f) {
      v = load_row_vec(row, k, a.hidden, (T)0.0f);
      if (e != big || back != 1.0f) {
        float f[8];
        to_float<T>(v, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = ldexpf(f[i] * back, e - big);
        v = from_float<T>(f);
      }
    }
    ((u32x4*)a.xs)[((uint64_t)t * a.hidden64 + k) / 8] = v;
  }
  // rows behind the last tile's, which the table's product reads too
  if (t >= a.tiled)
    for (uint32_t k = lane * 8; k < a.piece; k += 512) ((u32x4*)a.slopes)[((uint64_t)t * a.slope_stride + k) / 8] = u32x4{};
}
// 16 rows, by 64 parts of the tiles, through 12 KB of LDS: c and log2 s go to
// `top` and `logsum`, the rows' scores and terms, where `write`, to memory.
__device__ __forceinline__ void join_rows(const Args& a, uint32_t first, float (*lds)[64][16], float* top,
                                          float* logsum, bool write) {
  float(*sc)[16] = lds[0], (*ss)[16] = lds[1], (*sl)[16] = lds[2];
  const uint32_t row = threadIdx.x & 15, from = threadIdx.x >> 4, t = first + row;
  const uint64_t each = (uint64_t)a.tiles * a.rows64;
  Part p{0.0f, 0.0f};
  float l = 0.0f;
  for (uint32_t i = from; i < a.tiles; i += 64 * 8) {
    float c[8], s[8], sum[8];  // (their loads together)
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool in = i + u * 64 < a.tiles;
      const uint64_t at = (uint64_t)min(i + u * 64, a.tiles - 1) * a.rows64 + t;
      c[u] = a.part[at];
      s[u] = in ? a.part[each + at] : 0.0f;
      sum[u] = in ? a.part[2 * each + at] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      p = join(p, Part{c[u], s[u]});
      l += sum[u];
    }
  }
  sc[from][row] = p.c;
  ss[from][row] = p.s;
  sl[from][row] = l;
  __syncthreads();
  if (from >= 4) return;  // a wave joins 16 parts a lane, then its lanes'
#pragma unroll
  for (uint32_t w = 4; w < 64; w += 4) {
    p = join(p, Part{sc[from + w][row], ss[from + w][row]});
    l += sl[from + w][row];
  }
#pragma unroll
  for (int d = 16; d < 64; d *= 2) {
    const Part other{__shfl_xor(p.c, d, 64), __shfl_xor(p.s, d, 64)};
    const float more = __shfl_xor(l, d, 64);
    p = join(p, other);
    l += more;
  }
  if (from > 0) return;
  // (in 64 bits: a score near 0 is a difference of near numbers)
  constexpr double kLn2 = 0.693147180559945309;
  const int32_t y = t < a.rows ? a.target[t] : -1;
  const bool there = y >= 0 && (uint32_t)y < a.vocab;
  // (a target out of range: NaN, and with it the row's slopes)
  const double ls = y < 0 || there ? log2((double)p.s) : (double)NAN;
  const float at = there ? (float)((((double)a.picked[t] * (double)kLog2e - (double)p.c) - ls) * kLn2) : NAN;
  top[row] = p.c;
  logsum[row] = (float)ls;
  if (!write) return;
  float term = 0.0f;
  if (y >= 0) {
    a.logp[t] = at;
    const float r = a.row_weight[t];
    term = (1.0f - a.smoothing) * -at;
    if (a.smoothing != 0.0f)
      term += a.smoothing * (float)((ls - ((double)(l / (float)a.vocab) * (double)kLog2e - (double)p.c)) * kLn2);
    term = r == 0.0f ? 0.0f : r * term;
  } else if (t < a.rows) {
    a.logp[t] = 0.0f;
  }
  a.terms[t] = term;
}

// In 1024 parts, whatever the workgroup: the same sum from every launch.
__device__ __forceinline__ void add_loss(const Args& a) {
  __shared__ float waves[16];
  const uint32_t lane = threadIdx.x & 63;
  for (uint32_t w = threadIdx.x >> 6; w < 16; w += blockDim.x >> 6) {
    float sum = 0.0f;
    for (uint32_t t = w * 64 + lane; t < a.rows; t += 1024) sum += a.terms[t];
    sum = wave_sum(sum);
    if (lane == 0) waves[w] = sum;
  }
  __syncthreads();
  if (threadIdx.x) return;
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 16; ++w) sum += waves[w];
  *a.loss = sum;
}
__global__ void __launch_bounds__(1024) xent_loss(Args a) { add_loss(a); }
// Up to 16 rows: their loss too.
__global__ void __launch_bounds__(1024) xent_join(Args a) {
  __shared__ float lds[3][64][16];
  join_rows(a, blockIdx.x * 16, lds, a.top + blockIdx.x * 16, a.logsum + blockIdx.x * 16, true);
  if (a.rows > 16) return;
  __syncthreads();
  add_loss(a);
}
// And the rows' factors and scaled states, of all rows up to whole 64s.
template <typename T>
__global__ void __launch_bounds__(1024) xent_rows(Args a) {
  __shared__ float lds[3][64][16];
  if (blockIdx.x * 16 < a.rows)
    join_rows(a, blockIdx.x * 16, lds, a.top + blockIdx.x * 16, a.logsum + blockIdx.x * 16, true);
  __syncthreads();
  prepare_rows<T, 16, true>(a, blockIdx.x);
}

// No rows: a table's gradient of zeros.
template <typename T>
__global__ void __launch_bounds__(256) xent_nothing(Args a) {
  T* row = (T*)a.dweight + (int64_t)blockIdx.x * a.dweight_stride;
  for (uint32_t h = threadIdx.x; h < a.hidden; h += 256) row[h] = (T)0.0f;
}

// dx from its parts: 64 columns of a row a wave (kWave, up to 16 parts) or a
// workgroup, and turn; 16 lanes a part.  The first workgroup adds up the loss
// where another launch does not.  4 parts of 4,096 rows x 1,024: 22 us by waves,
// 33 by workgroups of one.
constexpr uint32_t kStatesGrid = 1 << 20;
template <typename T, bool kLoss, bool kWave>
__global__ void __launch_bounds__(1024) xent_states(Args a) {
  __shared__ f32x4 waves[16][16];
  const uint32_t tid = threadIdx.x, lane = tid & 15, wave = tid >> 6;
  const uint32_t part = kWave ? tid >> 4 & 3 : tid >> 4, parts = kWave ? 4 : blockDim.x / 16;
  const uint32_t panels = a.hidden64 / 64, each = kWave ? blockDim.x / 64 : 1;
  if (kLoss && blockIdx.x == 0) add_loss(a);
  const uint64_t units = (uint64_t)a.rows * panels;
  for (uint64_t unit = (uint64_t)blockIdx.x * each + (kWave ? wave : 0); unit < units; unit += (uint64_t)gridDim.x * each) {
    const uint32_t t = (uint32_t)(unit / panels), h = ((uint32_t)(unit % panels) * 16 + lane) * 4;
    const float* p = a.dxs + (uint64_t)t * a.hidden64 + h;
    f32x4 y{};
#pragma unroll 4
    for (uint32_t s = part; s < a.splits; s += parts) y += *(const f32x4*)(p + s * a.split_stride);
#pragma unroll
    for (int d = 16; d < 64; d *= 2)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += __shfl_xor(y[e], d, 64);
    if (!kWave) {
      __syncthreads();  // (the turn before has read its sums)
      if ((tid & 63) < 16) waves[wave][lane] = y;
      __syncthreads();
      if (wave > 0) continue;
      for (uint32_t w = 1; w < parts / 4; ++w) y += waves[w][lane];
    }
    if ((tid & 63) >= 16) continue;
    const bool none = a.factor[t] == 0.0f;
    const float f = a.power[t];
    T* out = (T*)a.dx + (int64_t)t * a.dx_stride + h;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (h + e < a.hidden) out[e] = (T)(none ? 0.0f : y[e] * f);
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

// Any alignment: operands pass registers on their way to LDS, no step ahead
// (4,096 rows x 262,144 x 1,024: 14.2 ms where xent_tile takes 7.9).
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

// What a product leaves.  The wave's i are i0 ..., 16 kN of them, its j jb + jw
// ..., 16 kM of the workgroup's kB; a lane has four neighbouring i of row j.
// Waves wn = 0 ... kWaves - 1 have other i of the same j.
// A wave's LDS `mine` (or none) takes 16 rows of numbers of 16 bits, so that
// they are stored by whole lines.
template <int kN>
constexpr int kStored = 16 * (kN * 32 + 16);  // bytes

// Rows r of 16 kN numbers, of which a lane has o[v], numbers 16 v + 4 q ... of
// row `col`; to(r, c) is where row r's from c on lie, or null.
template <int kN, typename To>
__device__ __forceinline__ void store_rows(const uint2 (&o)[kN], char* mine, uint32_t lane, To&& to) {
  constexpr int kRow = kN * 32 + 16, kPer = kN * 2;  // bytes, pieces of 16
  const uint32_t col = lane & 15, q = lane >> 4;
#pragma unroll
  for (int v = 0; v < kN; ++v) *(uint2*)(mine + col * kRow + v * 32 + q * 8) = o[v];
  asm volatile("" ::: "memory");  // (a wave's LDS accesses are in order)
#pragma unroll
  for (int p = 0; p < 16 * kPer / 64; ++p) {
    const uint32_t at = p * 64 + lane, r = at / kPer, c = at % kPer * 8;
    const u32x4 v = *(const u32x4*)(mine + r * kRow + c * 2);
    to(r, c, v);
  }
  asm volatile("" ::: "memory");
}

template <typename T, Kind kKind, int kN, int kM, int kWaves, int kB, bool kLines, bool kPast>
__device__ __forceinline__ void finish(const Args& a, uint32_t tid, uint32_t tile, uint32_t i0, uint32_t jb,
                                       uint32_t jw, uint32_t wn, uint32_t split, f32x4 (&acc)[kN][kM],
                                       float (*joined)[3][kB], char* mine) {
  const uint32_t lane = tid & 63, col = lane & 15, q = lane >> 4, j0 = jb + jw;
  if constexpr (kKind == kStats) {
    const bool inside = i0 + 16 * kN <= a.vocab;
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      const uint32_t t = j0 + s * 16 + col;
      float sum = 0.0f, total = 0.0f, big = -INFINITY;
      // the target, in one tile of many
      const uint32_t y = (t < a.rows ? (uint32_t)a.target[t] : ~0u) - i0;
      if (__ballot(y < 16 * kN)) {
#pragma unroll
        for (int v = 0; v < kN; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (y == v * 16 + q * 4 + e && i0 + y < a.vocab) a.picked[t] = acc[v][s][e];
      }
      if (!inside) {  // (tokens past the vocabulary add 0 to the sum of logits)
#pragma unroll
        for (int v = 0; v < kN; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i0 + v * 16 + q * 4 + e >= a.vocab) acc[v][s][e] = 0.0f;
      }
      if (a.smoothing != 0.0f) {
#pragma unroll
        for (int v = 0; v < kN; ++v) total += (acc[v][s][0] + acc[v][s][1]) + (acc[v][s][2] + acc[v][s][3]);
      }
      if (!inside) {
#pragma unroll
        for (int v = 0; v < kN; ++v)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i0 + v * 16 + q * 4 + e >= a.vocab) acc[v][s][e] = -INFINITY;
      }
#pragma unroll
      for (int v = 0; v < kN; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) big = fmaxf(big, acc[v][s][e]);
#pragma unroll
      for (int d = 16; d < 64; d *= 2) big = fmaxf(big, __shfl_xor(big, d, 64));
      const float c = big == -INFINITY ? 0.0f : big * kLog2e;
#pragma unroll
      for (int v = 0; v < kN; ++v)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += power_of(acc[v][s][e], c);
#pragma unroll
      for (int d = 16; d < 64; d *= 2) {
        sum += __shfl_xor(sum, d, 64);
        total += __shfl_xor(total, d, 64);
      }
      if (q == 0) {
        joined[wn][0][jw + s * 16 + col] = c;
        joined[wn][1][jw + s * 16 + col] = sum;
        joined[wn][2][jw + s * 16 + col] = total;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    const uint64_t each = (uint64_t)a.tiles * a.rows64;
    for (uint32_t j = tid; j < kB && jb + j < a.rows64; j += blockDim.x) {
      Part p{joined[0][0][j], joined[0][1][j]};
      float sum = joined[0][2][j];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) {
        p = join(p, Part{joined[w][0][j], joined[w][1][j]});
        sum += joined[w][2][j];
      }
      const uint64_t at = (uint64_t)tile * a.rows64 + jb + j;
      a.part[at] = p.c;
      a.part[each + at] = p.s;
      a.part[2 * each + at] = sum;
    }
  }
  if constexpr (kKind == kSlopes) {
    const float even = a.smoothing / (float)a.vocab, own = 1.0f - a.smoothing;
    const bool inside = i0 + 16 * kN <= a.vocab;
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      if (j0 + s * 16 >= a.rows64) break;
      const uint32_t t = j0 + s * 16 + col;
      const uint32_t y = (t < a.rows ? (uint32_t)a.target[t] : ~0u) - i0;
      const float m = a.factor[t], c = a.top[t], ls = a.logsum[t];
      const bool hit = __ballot(y < 16 * kN) != 0;  // (a target in one tile of many)
      union {
        uint2 u;
        T g[4];
      } o;
      uint2 all[kN];
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        float g[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          g[e] = (exp2_raw(__builtin_fmaf(acc[v][s][e], kLog2e, -c) - ls) - even) * m;
        if (hit) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (y == v * 16 + q * 4 + e)
              g[e] = (exp2_raw(__builtin_fmaf(acc[v][s][e], kLog2e, -c) - ls) - even - own) * m;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (!inside && i0 + v * 16 + q * 4 + e >= a.vocab) g[e] = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.g[e] = (T)g[e];
        all[v] = m == 0.0f ? uint2{0, 0} : o.u;
      }
      T* first = (T*)a.slopes + (i0 - a.first);
      if constexpr (kLines) {
        store_rows<kN>(all, mine, lane, [&](uint32_t r, uint32_t c, u32x4 v) {
          *(u32x4*)(first + (uint64_t)(j0 + s * 16 + r) * a.slope_stride + c) = v;
        });
        __builtin_amdgcn_sched_barrier(0);
      } else {
#pragma unroll
        for (int v = 0; v < kN; ++v) *(uint2*)(first + (uint64_t)t * a.slope_stride + v * 16 + q * 4) = all[v];
      }
    }
  }
  if constexpr (kKind == kStates) {
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      if (j0 + s * 16 >= a.rows64) break;
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        const uint32_t h = i0 + v * 16 + q * 4;
        if (h >= a.hidden64) continue;
        f32x4* to = (f32x4*)(a.dxs + split * a.split_stride + (uint64_t)(j0 + s * 16 + col) * a.hidden64 + h);
        *to = a.first ? *to + acc[v][s] : acc[v][s];
      }
    }
  }
  if constexpr (kKind == kTable) {
    const float f = *a.largest * (1.0f / kUp<T>);
#pragma unroll
    for (int s = 0; s < kM; ++s) {
      union {
        uint2 u;
        T e[4];
      } o;
      uint2 all[kN];
#pragma unroll
      for (int v = 0; v < kN; ++v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o.e[e] = (T)(acc[v][s][e] * f);
        all[v] = o.u;
      }
      const uint32_t tok = a.first + j0 + s * 16;
      if constexpr (kLines) {
        store_rows<kN>(all, mine, lane, [&](uint32_t r, uint32_t c, u32x4 v) {
          if (tok + r < a.vocab && i0 + c < a.hidden)  // (whole lines of columns)
            store_to<kPast>((T*)a.dweight + (int64_t)(tok + r) * a.dweight_stride + i0 + c, v);
        });
        __builtin_amdgcn_sched_barrier(0);
      } else if (tok + col < a.vocab) {
        T* row = (T*)a.dweight + (int64_t)(tok + col) * a.dweight_stride;
#pragma unroll
        for (int v = 0; v < kN; ++v) {
          const uint32_t h = i0 + v * 16 + q * 4;
          o.u = all[v];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (h + e < a.hidden) row[h + e] = o.e[e];
        }
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
  const uint32_t js = kKind == kTable ? a.width / kBM : a.rows64 / kBM;
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
    qo = Operand{a.slopes, a.slope_stride, a.rows64, a.piece};
    k0 = split * a.split_steps * kBK;
    k1 = min(k0 + a.split_steps * kBK, a.width);
  } else {
    po = Operand{a.xs, a.hidden64, a.rows64, a.hidden64};
    qo = Operand{a.slopes, a.slope_stride, a.rows64, a.piece};
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
  finish<T, kKind, 2, kBM / 16, 4, kBM, false, false>(a, threadIdx.x, ti, i0 + wave * 32, j0, 0, wave, split, acc, joined,
                                                nullptr);
}

// Operands whose rows are whole lines of 128 bytes: tiles of 256 of i by BM of
// j, steps of 64 of k copied straight to two LDS stages.  The operands of half
// a step are read from LDS during the matrix instructions of the half before,
// so that past a barrier there is work at once.
//
// An operand by k is a line of eight 16-byte columns a row, exchanged by the
// row's number.  One across k has lines of 512 bytes (256 of i) for each k: a
// copy of a wave brings two, whose 32-byte units are exchanged by the row's
// lowest bit, and copies lie 64 bytes more than their length apart, every
// fourth 128 more: a transposed read takes 32 bytes of four rows in 16 lanes,
// and of eight rows in 32, without bank conflicts.
constexpr int kTileBN = 256, kTileThreads = 512;

// 16 bytes a lane, from an offset (a lane's and the wave's) of a buffer to
// the wave's place in LDS.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t whole_buffer(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)0xFFFFFFFFu, 0x00027000);
}
__device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lane, uint32_t wave, void* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, (int)lane,
                                           (int)wave, 0, 0);
}
// All LDS reads of the wave are done, and all its copies but the last n.
template <int n>
__device__ __forceinline__ void wait_copies() {
  asm volatile("" ::: "memory");
  // vmcnt n, lgkmcnt 0, the third counter free
  __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4);
}

// kWhole: across, rows are whole steps.
template <typename T, bool kAcross, int kB, bool kWhole>
struct Lines {
  static constexpr int kTurns = (kB + 63) / 64;  // copies of a wave and step (the last: of some waves)
  static constexpr uint32_t kBytes = kAcross ? 32 * 1088 + 8 * 128 : kB * 128;
  static constexpr int kOffsets = kAcross ? 1 : kTurns;
  static_assert(!kAcross || kB == 256, "lines of 512 bytes");

  const char* base;
  uint32_t line;           // bytes from row to row
  uint32_t left;           // across: rows from base on
  uint32_t off[kOffsets];  // of this lane's copies
  uint32_t at[2];          // this lane's reads: of a step's halves; across: of even and odd subtiles

  // by k: rows i0 ..., from column k0 on; across: columns i0 ..., from row k0 on
  __device__ __forceinline__ void begin(const Operand& o, uint32_t i0, uint32_t k0, uint32_t sub0, uint32_t tid,
                                        uint32_t wave) {
    const uint32_t lane = tid & 63, col = lane & 15, q = lane >> 4;
    line = (uint32_t)o.stride * 2;
    if constexpr (kAcross) {
      const uint32_t row0 = min(k0, o.rows - 1);
      base = (const char*)((const T*)o.base + (int64_t)row0 * o.stride);
      left = o.rows - row0;
      const uint32_t row = 2 * wave + (lane >> 5), piece = (lane & 31) ^ (lane >> 5 << 1);
      // (columns past the end: the last ones, whose products are not stored)
      off[0] = row * line + min(i0 / 8 + piece, o.columns / 8 - 1) * 16;
      const uint32_t r4 = col >> 2, b = r4 & 1;
      at[0] = q * (4 * 1088 + 128) + (r4 >> 1) * 1088 + b * 512 + sub0 * 32 + (col & 3) * 8;
      at[1] = at[0] - b * 32;
      at[0] += b * 32;
    } else {
      base = (const char*)((const T*)o.base + (int64_t)i0 * o.stride + k0);
#pragma unroll
      for (int c = 0; c < kTurns; ++c) {
        const uint32_t row = (c * kTileThreads + tid) / 8;
        off[c] = min(row, o.rows - 1 - i0) * line + ((tid & 7) ^ (row & 7)) * 16;
      }
      at[0] = ((sub0 * 16 + col) * 8 + (q ^ (col & 7))) * 16;
      at[1] = at[0] ^ 64;
    }
    asm volatile("" : "+v"(at[0]), "+v"(at[1]));
  }
  // step k from the first on
  __device__ __forceinline__ void copy(char* st, uint32_t k, uint32_t lane, uint32_t wave) const {
    if constexpr (kAcross) {
      const uint32_t first = kWhole ? k * 64 : min(k * 64, left - 1);
      const __amdgpu_buffer_rsrc_t b = whole_buffer(base + (uint64_t)first * line);
      char* to = st + wave * 1088 + (wave >> 2) * 128;
      if (kWhole || first + 64 <= left) {
#pragma unroll
        for (int c = 0; c < kTurns; ++c) copy_to_lds(b, off[0], c * 16 * line, to + c * (8 * 1088 + 256));
      } else {  // rows past the end: the last one
        const uint32_t row = 2 * wave + (lane >> 5), at = off[0] - row * line;
#pragma unroll
        for (int c = 0; c < kTurns; ++c)
          copy_to_lds(b, min(c * 16 + row, left - first - 1) * line + at, 0, to + c * (8 * 1088 + 256));
      }
    } else {
      const __amdgpu_buffer_rsrc_t b = whole_buffer(base);
#pragma unroll
      for (int c = 0; c < kTurns; ++c)
        if (kB % 64 == 0 || c * 64 + wave * 8 < (uint32_t)kB) copy_to_lds(b, off[c], k * 128, st + (c * 8 + wave) * 1024);
    }
  }
  // subtile sub0 + v, half kk of a step
  __device__ __forceinline__ u32x4 read(const char* st, int v, int kk) const {
    if constexpr (kAcross) {
      const char* p = st + at[v & 1] + (v * 32 + kk * (16 * 1088 + 4 * 128));
      union {
        s16x4 h[2];
        u32x4 v;
      } u;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        u.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p + i * 2 * 1088));
      return u.v;
    } else {
      return *(const u32x4*)(st + at[kk] + v * 2048);
    }
  }
};

// Tile (j, i, split) of n, in turn.  Consecutive workgroups go to the XCDs in
// turn, so each XCD takes a run of tiles; a run goes over four tiles of j at a
// time, then over i: what an XCD runs at once shares operands in its L2.
__device__ __forceinline__ void tile_of(uint32_t block, uint32_t n, uint32_t js, uint32_t is, uint32_t* tj,
                                        uint32_t* ti, uint32_t* split) {
  const uint32_t run = n / 8;
  uint32_t t = block < run * 8 ? (block % 8) * run + block / 8 : block;
  *split = t / (js * is);
  t -= *split * (js * is);
  constexpr uint32_t kGroup = 4;
  const uint32_t g = t / (kGroup * is), in = t - g * kGroup * is;
  const uint32_t width = min(kGroup, js - g * kGroup);
  *ti = in / width;
  *tj = g * kGroup + in % width;
}

template <int kBMs, int kWM>
struct TileShape {
  static constexpr int BM = 16 * kBMs, WM = kWM, WN = 8 / kWM, M = kBMs / WM, N = 16 / WN;
};

// Workgroups take tiles in turn: the next one's first two steps are copied
// before what this one leaves is worked out.  A piece of 16,384 tokens, 4,096
// rows x 1,024 bf16: slopes 142 us (0.97 PFLOP/s; their exponentials and stores are
// not hidden), dx 117 (1.17; 67 MB of its parts read and written), the table's
// gradient 100 (1.37); the statistics of all 262,144 tokens 1.94 ms (1.13).
template <typename T, Kind kKind, typename S, bool kPast = false>
__global__ void __launch_bounds__(kTileThreads) xent_tile(Args a) {
  using P = Lines<T, kKind >= kStates, kTileBN, kKind == kTable>;
  using Q = Lines<T, kKind == kTable, S::BM, true>;
  __shared__ __attribute__((aligned(1024))) char st0[P::kBytes + Q::kBytes], st1[P::kBytes + Q::kBytes];
  __shared__ float joined[kKind == kStats ? S::WN : 1][3][kKind == kStats ? S::BM : 1];
  __shared__ u32x4 stored[kKind == kSlopes || kKind == kTable ? 8 * kStored<S::N> / 16 : 1];
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t wm = wave % S::WM, wn = wave / S::WM;
  const uint32_t js = kKind == kTable ? a.width / S::BM : (a.rows + S::BM - 1) / S::BM;
  const uint32_t is = kKind == kStats    ? a.tiles
                      : kKind == kSlopes ? a.width / kTileBN
                                         : (a.hidden64 + kTileBN - 1) / kTileBN;
  const uint32_t splits = kKind == kStates ? (a.width / 64 + a.split_steps - 1) / a.split_steps : 1;
  const uint32_t tiles = js * is * splits;
  uint32_t tj, ti, split, steps;
  P p;
  Q x;
  const auto copy = [&](char* st, uint32_t i, uint32_t lane) {
    const uint32_t k = min(i, steps - 1);  // (past the end: again, unused)
    p.copy(st, k, lane, wave);
    x.copy(st + P::kBytes, k, lane, wave);
  };
  const auto begin = [&](uint32_t block) {
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // (nothing of this is kept through a tile)
    tile_of(block, tiles, js, is, &tj, &ti, &split);
    Operand po, qo;
    uint32_t k0 = 0;
    if (kKind == kStats || kKind == kSlopes) {
      po = Operand{a.weight, a.weight_stride, a.vocab, a.hidden};
      qo = Operand{a.x, a.x_stride, a.rows, a.hidden};
      steps = a.hidden64 / 64;
    } else if (kKind == kStates) {
      po = Operand{(const T*)a.weight + (int64_t)a.first * a.weight_stride, a.weight_stride, a.vocab - a.first, a.hidden};
      qo = Operand{a.slopes, a.slope_stride, a.rows64, a.piece};
      k0 = split * a.split_steps * 64;
      steps = min(a.split_steps, a.width / 64 - split * a.split_steps);
    } else {
      po = Operand{a.xs, a.hidden64, a.rows64, a.hidden64};
      qo = Operand{a.slopes, a.slope_stride, a.rows64, a.piece};
      steps = a.rows64 / 64;
    }
    p.begin(po, ti * kTileBN + (kKind == kSlopes ? a.first : 0), k0, wn * S::N, tid, wave);
    x.begin(qo, tj * S::BM, k0, wm * S::M, tid, wave);
    copy(st0, 0, tid & 63);
    copy(st1, 1, tid & 63);
  };
  begin(blockIdx.x);
  for (uint32_t block = blockIdx.x;;) {
    f32x4 acc[S::N][S::M] = {};
    // Half a step: the products of w and x, while w and `ahead` take the next
    // half's operands, kk of the stage `next`.  A register of w is free when
    // its products are issued; x has two sets.
    u32x4 w[S::N], x0[S::M], x1[S::M];
    const auto half = [&](const u32x4 (&now)[S::M], u32x4 (&ahead)[S::M], const char* next, int kk) {
#pragma unroll
      for (int v = 0; v < S::N; ++v) {
#pragma unroll
        for (int j = 0; j < S::M; ++j) acc[v][j] = mfma(w[v], now[j], acc[v][j], T{});
        w[v] = p.read(next, v, kk);
        constexpr int kEach = (S::M + S::N - 1) / S::N;
#pragma unroll
        for (int j = v * kEach; j < (v + 1) * kEach && j < S::M; ++j) ahead[j] = x.read(next + P::kBytes, j, kk);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // Step i: w and x0 hold its first half's operands.  At the barrier all of
    // the step has been read, and the next is there.
    const auto step = [&](uint32_t i, char* st, const char* next) {
      half(x0, x1, st, 1);
      wait_copies<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      copy(st, i + 2, threadIdx.x & 63);
      half(x1, x0, next, 0);
    };
    wait_copies<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int v = 0; v < S::N; ++v) w[v] = p.read(st0, v, 0);
#pragma unroll
    for (int j = 0; j < S::M; ++j) x0[j] = x.read(st0 + P::kBytes, j, 0);
    for (uint32_t i = 0;;) {
      step(i, st0, st1);
      if (++i == steps) break;
      step(i, st1, st0);
      if (++i == steps) break;
    }
    wait_copies<0>();
    __syncthreads();
    const uint32_t jb = tj * S::BM, tile = ti, part = split;
    block += gridDim.x;
    const bool more = block < tiles;
    if (more) begin(block);
    uint32_t tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    finish<T, kKind, S::N, S::M, S::WN, S::BM, true, kPast>(
        a, tid, tile, tile * kTileBN + (kKind == kSlopes ? a.first : 0) + wn * S::N * 16, jb, wm * S::M * 16, wn,
        part, acc, (float(*)[3][S::BM])joined, (char*)stored + wave * kStored<S::N>);
    if (!more) break;
  }
}

// Few rows, whose states fit LDS beside a tile of the table: one pass over the
// table leaves both gradients.  A workgroup takes tiles of kTok tokens in turn:
// their logits (the waves share the 16 x 16 tiles and the hidden columns; the
// states are their registers'), slopes by way of LDS, then each wave, for its
// own columns, adds to its sums for dx, which stay in registers to the end, and
// stores its part of the tokens' dweight rows.  The next tile is on its way to
// registers meanwhile.  Rows of the table and of the scaled states lie in LDS
// as they are, their 16-byte columns exchanged by the row's number such that
// eight rows of a column, and two columns of four rows, are free of bank
// conflicts: the logits read the table by k, the gradients read across.  10 rows x
// 262,144 x 1,024 bf16: 208 us for both gradients (5.2 TB/s read and written; 295
// with dweight stored eight bytes a lane), 112 us for dx alone, 87 for the
// statistics.
constexpr uint32_t kFewBytes = 65536;  // of the states, and of a tile
constexpr int kFewThreads = 1024;

// kStats: the pass before it, for the rows' statistics: each workgroup's own,
// held by lanes (a row, and the tokens 4 q ... of a subtile) to the end.
template <typename T, int kR, int kTok, bool kStats, bool kPast>
__global__ void __launch_bounds__(kFewThreads) xent_few(Args a) {
  if constexpr (kStats) {
    if (blockIdx.x < a.prepare) {
      prepare_rows<T, 16, false>(a, blockIdx.x);
      return;
    }
  }
  const uint32_t block = blockIdx.x - (kStats ? a.prepare : 0), blocks = gridDim.x - (kStats ? a.prepare : 0);
  constexpr int kTiles = kR * kTok / 16, kSplits = 16 / kTiles;  // 16 x 16 tiles of logits, waves for one
  constexpr int kColumns = 32768 / kTok;                         // the most
  constexpr int kSubs = kColumns / 256, kX = kColumns / 32 / kSplits;  // of a wave: 16-column subtiles, steps of 32
  constexpr int kLoads = (int)kFewBytes / 16 / kFewThreads, kPitch = 40, kRowPitch = (kTok < 32 ? 32 : kTok) + 8;
  constexpr int kLine = kSubs == 4 && kR == 1 ? 4 : 2;  // subtiles stored at a time: LDS for more where it is left
  __shared__ u32x4 st[kFewBytes / 16], xl[kStats ? 1 : kR * 16 * kColumns / 8];
  // of a wave: its part of a tile of logits, then the lines that it stores
  __shared__ u32x4 own_lds[16][kStored<kLine> / 16];
  static_assert(kStored<kLine> >= 1024, "a tile's part fits");
  // the slopes as a sum of two of the type, which cost nothing here: 16 of a
  // step's 32 k beside the other 16, or an array each; and some space
  constexpr int kTokenParts = kR == 1 ? 2 : 1, kRowParts = kTok == 16 ? 2 : 1;  // in a step
  __shared__ __attribute__((aligned(16))) T by_token[3 - kTokenParts][kTok][kPitch];
  __shared__ __attribute__((aligned(16))) T by_row[3 - kRowParts][kR * 16][kRowPitch];
  __shared__ float known[4][kR * 16];  // of a row: m, c, log2 s, target
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t vecs = a.hidden / 8, tiles = (a.vocab + kTok - 1) / kTok;
  // this wave's columns: neighbours, so that it stores by lines
  const uint32_t subs = a.hidden / 16, each_subs = (subs + 15) / 16, sub0 = wave * each_subs;
  const uint32_t own_subs = sub0 < subs ? min(each_subs, subs - sub0) : 0;
  const auto swap = [](uint32_t row) { return 2 * (row & 3) + (row >> 2 & 1); };

  // a tile's vectors, of rows past the vocabulary the last's: bytes from the
  // tile's first, and their places in LDS
  const uint32_t line = (uint32_t)a.weight_stride * 2;
  // (eight columns and more a row: the exchange is of a vector's own number)
  uint32_t from[kLoads], swaps = 0;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const uint32_t at = i * kFewThreads + tid, row = at / vecs;
    from[i] = row < (uint32_t)kTok ? row * line + (at - row * vecs) * 16 : ~0u;
    swaps |= swap(row) << (3 * i);
  }
  u32x4 next[kLoads];
  const auto load = [&](uint32_t tile) {
    const char* base = (const char*)a.weight + (uint64_t)tile * kTok * line;
    const uint32_t rows = min((uint32_t)kTok, a.vocab - tile * kTok);
    if (rows == (uint32_t)kTok) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if (from[i] != ~0u)
          next[i] = kPast ? __builtin_nontemporal_load((const u32x4*)(base + from[i])) : *(const u32x4*)(base + from[i]);
    } else {
      uint32_t now = tid;
      asm volatile("" : "+v"(now));
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const uint32_t at = i * kFewThreads + now, row = at / vecs, c = at - row * vecs;
        if (from[i] != ~0u) next[i] = *(const u32x4*)(base + (uint64_t)min(row, rows - 1) * line + c * 16);
      }
    }
  };
  const auto keep = [&]() {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (from[i] != ~0u) st[(i * kFewThreads + tid) ^ (swaps >> (3 * i) & 7)] = next[i];
  };
  uint32_t tile = block;
  load(tile);
  if (!kStats && a.dweight)
    for (uint32_t at = tid; at < kR * 16 * vecs; at += kFewThreads) {
      const uint32_t row = at / vecs, c = at - row * vecs;
      xl[row * vecs + (c ^ swap(row))] = ((const u32x4*)a.xs)[(uint64_t)row * (a.hidden64 / 8) + c];
    }
  // the tile of logits that this wave shares, its steps of the hidden columns,
  // and what a lane knows of its row
  const uint32_t ts = wave % kTiles % (kTok / 16), rs = wave % kTiles / (kTok / 16), t = rs * 16 + col;
  const uint32_t steps = a.hidden / 32, each = (steps + kSplits - 1) / kSplits;
  const uint32_t s0 = min(wave / kTiles * each, steps), s1 = min(s0 + each, steps);
  u32x4 x[kX];
#pragma unroll
  for (int s = 0; s < kX; ++s)
    x[s] = *(const u32x4*)((const T*)a.x + (int64_t)min(t, a.rows - 1) * a.x_stride +
                           (min(s0 + s, steps - 1) * 4 + q) * 8);
  if (tid < kR * 16) {
    if (!kStats) known[0][tid] = a.factor[tid];
    known[3][tid] = __int_as_float(tid < a.rows ? a.target[tid] : -1);
  }
  const float even = a.smoothing / (float)a.vocab, own = 1.0f - a.smoothing;
  const float f = kStats ? 0.0f : *a.largest * (1.0f / kUp<T>);
  // every workgroup joins the statistics for itself (a launch less); the first
  // leaves the scores and the loss
  if (!kStats) {
    for (uint32_t r = 0; r < kR * 16 && r < a.rows; r += 16) {
      join_rows(a, r, (float(*)[64][16])st, known[1] + r, known[2] + r, block == 0);
      __syncthreads();
    }
    if (block == 0) add_loss(a);
  }
  keep();
  f32x4 sum[kSubs][kR] = {};
  Part mine{-INFINITY, 0.0f};
  float total = 0.0f;
  for (; tile < tiles; tile += blocks) {
    load(min(tile + blocks, tiles - 1));
    __syncthreads();
    {
      // (the lane anew here and below, so that addresses are not kept through the
      // loop: there are 128 registers)
      uint32_t now = lane;
      asm volatile("" : "+v"(now));
      const u32x4* wr = st + (ts * 16 + (now & 15)) * vecs;
      const uint32_t q = now >> 4, other = swap(now);
      f32x4 l{};
#pragma unroll
      for (int s = 0; s < kX; ++s)
        if (s0 + s < s1) l = mfma(wr[((s0 + s) * 4 + q) ^ other], x[s], l, T{});
      *(f32x4*)&own_lds[wave][lane] = l;
    }
    __syncthreads();
    if constexpr (kStats) {
      keep();  // (past the barrier all of the tile has been read)
      if (wave < (uint32_t)kTiles) {
        f32x4 l{};
#pragma unroll
        for (int i = 0; i < kSplits; ++i) l += *(const f32x4*)&own_lds[wave + i * kTiles][lane];
        const uint32_t tok = tile * kTok + ts * 16 + q * 4, y = __float_as_uint(known[3][t]) - tok;
        float big = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = tok + e < a.vocab;
          if (y == (uint32_t)e && in) a.picked[t] = l[e];
          total += in ? l[e] : 0.0f;
          if (!in) l[e] = -INFINITY;
          big = fmaxf(big, l[e]);
        }
        if (!(big == -INFINITY)) {
          const float c = fmaxf(mine.c, big * kLog2e);
          mine.s = mine.s == 0.0f ? 0.0f : mine.s * exp2_raw(mine.c - c);
          mine.c = c;
#pragma unroll
          for (int e = 0; e < 4; ++e) mine.s += power_of(l[e], c);
        }
      }
      continue;
    }
    if (wave < (uint32_t)kTiles) {
      const float m = known[0][t], c = known[1][t], ls = known[2][t];
      const int32_t y = __float_as_int(known[3][t]);
      f32x4 l{};
#pragma unroll
      for (int i = 0; i < kSplits; ++i) l += *(const f32x4*)&own_lds[wave + i * kTiles][lane];
      union {
        T e[4];
        uint2 u;
      } o, rest;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t tok = tile * kTok + ts * 16 + q * 4 + e;
        float g = exp2_raw(__builtin_fmaf(l[e], kLog2e, -c) - ls) - even;
        if ((int32_t)tok == y) g -= own;
        g = m != 0.0f && tok < a.vocab ? g * m : 0.0f;
        o.e[e] = (T)g;
        // (an infinity has no rest)
        rest.e[e] = (T)(fabsf((float)o.e[e]) < INFINITY ? g - (float)o.e[e] : 0.0f);
        const uint32_t n = ts * 16 + q * 4 + e;
        by_token[0][n][t] = o.e[e];
        if (kTokenParts == 2) by_token[0][n][16 + t] = rest.e[e];
        else by_token[2 - kTokenParts][n][t] = rest.e[e];
      }
      *(uint2*)&by_row[0][t][ts * 16 + q * 4] = o.u;
      if (kRowParts == 2) *(uint2*)&by_row[0][t][16 + q * 4] = rest.u;
      else *(uint2*)&by_row[2 - kRowParts][t][ts * 16 + q * 4] = rest.u;
    }
    __syncthreads();
    // columns 16 sub ... of rows k0 + 8 q ... of the table or the states, read
    // across (rows behind: these again, for slopes of zero)
    uint32_t now = lane;
    asm volatile("" : "+v"(now));
    const auto across = [&](const u32x4* from, uint32_t rows, uint32_t k0, uint32_t sub) {
      const uint32_t col = now & 15, q = now >> 4;
      union {
        s16x4 h[2];
        u32x4 v;
      } u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t row = (k0 + q * 8 + i * 4 + (col >> 2)) % rows;
        const char* p = (const char*)(from + row * vecs + ((sub * 2 + (col >> 1 & 1)) ^ swap(row))) + (col & 1) * 8;
        u.h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      }
      return u.v;
    };
    if (a.dx) {
#pragma unroll
      for (int k = 0; k < (kTok + 31) / 32; ++k) {
        u32x4 gf[3 - kRowParts][kR];
#pragma unroll
        for (int i = 0; i < 3 - kRowParts; ++i)
#pragma unroll
          for (int r = 0; r < kR; ++r) gf[i][r] = *(const u32x4*)&by_row[i][r * 16 + (now & 15)][k * 32 + (now >> 4) * 8];
#pragma unroll
        for (int j = 0; j < kSubs; ++j) {
          if ((uint32_t)j >= own_subs) break;
          const u32x4 w = across(st, kTok, k * 32, sub0 + j);
#pragma unroll
          for (int i = 0; i < 3 - kRowParts; ++i)
#pragma unroll
            for (int r = 0; r < kR; ++r) sum[j][r] = mfma(w, gf[i][r], sum[j][r], T{});
          if (kSubs > 4 || j % 2) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    __syncthreads();
    keep();
    if (a.dweight) {
#pragma unroll 1
      for (int j0 = 0; j0 < kSubs; j0 += kLine) {
        if ((uint32_t)j0 >= own_subs) break;
        u32x4 xf[kLine];
#pragma unroll
        for (int j = 0; j < kLine; ++j) xf[j] = across(xl, kR * 16, 0, min(sub0 + j0 + j, subs - 1));
#pragma unroll
        for (int i = 0; i < kTok / 16; ++i) {
          const uint32_t tok = tile * kTok + i * 16;
          u32x4 gf[3 - kTokenParts];
#pragma unroll
          for (int p = 0; p < 3 - kTokenParts; ++p)
            gf[p] = *(const u32x4*)&by_token[p][i * 16 + (now & 15)][(now >> 4) * 8];
          uint2 all[kLine];
#pragma unroll
          for (int j = 0; j < kLine; ++j) {
            f32x4 d{};
#pragma unroll
            for (int p = 0; p < 3 - kTokenParts; ++p) d = mfma(xf[j], gf[p], d, T{});
            union {
              T e[4];
              uint2 u;
            } o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.e[e] = (T)(d[e] * f);
            all[j] = o.u;
          }
          store_rows<kLine>(all, (char*)own_lds[wave], now, [&](uint32_t r, uint32_t c, u32x4 v) {
            if (tok + r < a.vocab && j0 * 16 + c < own_subs * 16)
              store_to<kPast>((T*)a.dweight + (int64_t)(tok + r) * a.dweight_stride + (sub0 + j0) * 16 + c, v);
          });
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  if constexpr (kStats) {
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {
      const Part other{__shfl_xor(mine.c, d, 64), __shfl_xor(mine.s, d, 64)};
      const float more = __shfl_xor(total, d, 64);
      mine = join(mine, other);
      total += more;
    }
    float* parts = (float*)&by_row[0][0][0];  // [kTiles][3][16]
    static_assert(sizeof(by_row) >= kTiles * 48 * 4, "the waves' parts fit");
    if (wave < (uint32_t)kTiles && lane < 16) {
      parts[wave * 48 + lane] = mine.c;
      parts[wave * 48 + 16 + lane] = mine.s;
      parts[wave * 48 + 32 + lane] = total;
    }
    __syncthreads();
    if (tid < kR * 16) {
      Part p{0.0f, 0.0f};
      float l = 0.0f;
      for (uint32_t i = 0; i < kTok / 16; ++i) {
        const float* from = parts + (tid / 16 * (kTok / 16) + i) * 48 + tid % 16;
        p = join(p, Part{from[0], from[16]});
        l += from[32];
      }
      const uint64_t each = (uint64_t)a.tiles * a.rows64, at = (uint64_t)block * a.rows64 + tid;
      // (of nothing but -infinity: c is 0)
      a.part[at] = p.c == -INFINITY ? 0.0f : p.c;
      a.part[each + at] = p.s;
      a.part[2 * each + at] = l;
    }
    return;
  }
  if (!a.dx) return;
#pragma unroll
  for (int j = 0; j < kSubs; ++j) {
    if ((uint32_t)j >= own_subs) break;
#pragma unroll
    for (int r = 0; r < kR; ++r)
      *(f32x4*)(a.dxs + block * a.split_stride + (uint64_t)(r * 16 + col) * a.hidden64 + (sub0 + j) * 16 + q * 4) =
          sum[j][r];
  }
}

// --- plan -------------------------------------------------------------------

constexpr uint32_t kCUs = 256;

struct Plan {
  uint64_t factor, power, largest, part, picked, top, logsum, terms, xs, slopes, dxs, bytes;
  uint64_t split_stride;
  uint32_t rows64, hidden64, tiles, piece, slope_stride, splits, split_steps, bm, bn;
  uint32_t few;  // 16-row subtiles of xent_few; 0: other kernels
  bool lines, past;  // past: the caches
};

// The states' and the table's rows are whole lines, and 32-bit offsets reach
// a tile's operands.
bool whole_lines(const ft_cross_entropy_loss_args& a) {
  return a.hidden % 64 == 0 && (uintptr_t)a.x % 16 == 0 && (uintptr_t)a.weight % 16 == 0 &&
         a.x_stride % 8 == 0 && a.weight_stride % 8 == 0 && a.x_stride >= 0 && a.weight_stride >= 0 &&
         a.x_stride < 1 << 22 && a.weight_stride < 1 << 22;
}

Plan plan(const ft_cross_entropy_loss_args& a) {
  Plan p{};
  Arena ar;
  p.rows64 = (uint32_t)round_up(a.rows, 64);
  p.hidden64 = (uint32_t)round_up(a.hidden, 64);
  p.lines = whole_lines(a);
  // Whether the table is read for the last time, and its gradient written, past the
  // caches: 10 and 200 rows on H = 1,024 take 74 and 157 us so, 72 and 157 through
  // them at 100 MB; 95 and 244, 99 and 262 at 150; 169 and 475, 205 and 502 at 300.
  p.past = 2ull * a.vocab * a.hidden > kPastBytes;
  p.bn = p.lines ? kTileBN : kBN;
  p.bm = !p.lines || p.rows64 <= 64 ? 64 : p.rows64 <= 128 ? 128 : 256;
  // Many rows: the tile that leaves the least of them empty, at what a row costs
  // in each (6,720 rows x 65,536 x 1,024, whole tiles of each but 256: 2.68 ms by
  // 224, 2.90 by 192, 2.94 by 160; 4,096 rows x 262,144 x 1,024: 7.91 ms by 256,
  // 8.39 by 224; 777 rows x 50,021 x 768: 304 us by 160, 315 by 192, 331 by 224,
  // 337 by 256).
  if (p.bm == 256) {
    uint64_t least = ~0ull;
    constexpr uint32_t kShapes[4][2] = {{256, 100}, {224, 102}, {192, 107}, {160, 109}};
    for (const auto& shape : kShapes) {
      const uint64_t cost = round_up(a.rows, shape[0]) * shape[1];
      if (cost < least) {
        least = cost;
        p.bm = shape[0];
      }
    }
  }
  p.tiles = (a.vocab + p.bn - 1) / p.bn;
  const uint64_t r = p.rows64;
  if (p.lines && a.rows && a.hidden <= (a.rows <= 16 ? 2048 : a.rows <= 32 ? 512 : 0)) {
    const uint32_t tok = a.hidden <= 512 ? 64 : a.hidden <= 1024 ? 32 : 16;
    p.few = (uint32_t)(a.rows + 15) / 16;
    p.tiles = std::min(kCUs, (a.vocab + tok - 1) / tok);  // workgroups
  }
  p.factor = ar.take(r * 4);
  p.power = ar.take(r * 4);
  p.largest = ar.take(4);
  p.part = ar.take(3 * r * p.tiles * 4);
  p.picked = ar.take(r * 4);
  p.top = ar.take(r * 4);
  p.logsum = ar.take(r * 4);
  p.terms = ar.take(r * 4);
  if ((a.dx || a.dweight) && !p.few) {
    // a piece's slopes: up to 128 MB, half of the last level's cache (512 MB
    // take the same time within 2%)
    const uint64_t most = std::max<uint64_t>(256, (128ull << 20) / std::max<uint64_t>(64, r) / 512 * 256);
    const uint64_t pieces = (a.vocab + most - 1) / most;
    p.piece = (uint32_t)round_up((a.vocab + pieces - 1) / pieces, 256);
    // (rows a line more than a piece apart: not all on the same channels)
    p.slope_stride = p.piece + 64;
    p.slopes = ar.take(r * p.slope_stride * 2);
  }
  if (a.dweight) p.xs = ar.take(r * p.hidden64 * 2);
  if (p.few) {
    p.splits = p.tiles;
    p.split_stride = 16ull * p.few * p.hidden64;
    if (a.dx) p.dxs = ar.take(p.splits * p.split_stride * 4);
  } else if (a.dx) {
    // as many parts of the sum over tokens as fill the chip
    const uint64_t tiles = std::max<uint64_t>(1, (a.rows + p.bm - 1) / p.bm * ((p.hidden64 + p.bn - 1) / p.bn));
    const uint32_t steps = p.piece / kBK;
    const uint64_t want = std::max<uint64_t>(1, (p.lines ? 1 : 2) * kCUs / tiles);
    p.split_steps = (uint32_t)std::max<uint64_t>(4, (steps + want - 1) / want);
    p.splits = (steps + p.split_steps - 1) / p.split_steps;
    p.split_stride = r * p.hidden64;
    p.dxs = ar.take(p.splits * p.split_stride * 4);
  }
  p.bytes = ar.used;
  return p;
}

template <typename T, Kind kKind>
hipError_t product(const Args& a, const Plan& p, hipStream_t s) {
  const uint64_t hs = (a.hidden64 + p.bn - 1) / p.bn;
  const uint64_t js = kKind == kTable ? a.width / (p.lines ? 256 : p.bm) : (a.rows + p.bm - 1) / p.bm;
  const uint64_t blocks = js * (kKind == kStats    ? a.tiles
                                : kKind == kSlopes ? a.width / p.bn
                                : kKind == kStates ? hs * ((a.width / 64 + a.split_steps - 1) / a.split_steps)
                                                   : hs);
  if (!p.lines) return start(xent_product<T, kKind>, blocks, kThreads, s, a);
  if constexpr (kKind != kTable) {
    const uint64_t most = std::min<uint64_t>(blocks, kCUs);
    if (p.bm == 64) return start(xent_tile<T, kKind, TileShape<4, 1>>, most, kTileThreads, s, a);
    if (p.bm == 128) return start(xent_tile<T, kKind, TileShape<8, 2>>, most, kTileThreads, s, a);
    if (p.bm == 160) return start(xent_tile<T, kKind, TileShape<10, 2>>, most, kTileThreads, s, a);
    if (p.bm == 192) return start(xent_tile<T, kKind, TileShape<12, 2>>, most, kTileThreads, s, a);
    if (p.bm == 224) return start(xent_tile<T, kKind, TileShape<14, 2>>, most, kTileThreads, s, a);
  }
  const uint64_t most = std::min<uint64_t>(blocks, kCUs);
  if constexpr (kKind == kTable) {
    if (p.past) return start(xent_tile<T, kKind, TileShape<16, 2>, true>, most, kTileThreads, s, a);
  }
  return start(xent_tile<T, kKind, TileShape<16, 2>>, most, kTileThreads, s, a);
}

template <typename T, bool kStats, bool kPast>
hipError_t few(const Args& a, const Plan& p, uint64_t blocks, hipStream_t s) {
  return p.few == 2         ? start(xent_few<T, 2, 64, kStats, kPast>, blocks, kFewThreads, s, a)
         : a.hidden <= 512  ? start(xent_few<T, 1, 64, kStats, kPast>, blocks, kFewThreads, s, a)
         : a.hidden <= 1024 ? start(xent_few<T, 1, 32, kStats, kPast>, blocks, kFewThreads, s, a)
                            : start(xent_few<T, 1, 16, kStats, kPast>, blocks, kFewThreads, s, a);
}

template <typename T>
hipError_t states(const Args& a, bool loss, hipStream_t s) {
  const uint64_t units = (uint64_t)a.rows * (a.hidden64 / 64);
  const auto most = [](uint64_t blocks) { return std::min<uint64_t>(kStatesGrid, blocks); };
  if (a.splits <= 16)
    return loss ? start(xent_states<T, true, true>, most((units + 3) / 4), 256, s, a)
                : start(xent_states<T, false, true>, most((units + 3) / 4), 256, s, a);
  // (few workgroups: as many loads at once as there are parts)
  const uint32_t threads = (uint32_t)std::min<uint64_t>(units < 1024 ? 1024 : 256, round_up(16 * a.splits, 64));
  return loss ? start(xent_states<T, true, false>, most(units), threads, s, a)
              : start(xent_states<T, false, false>, most(units), threads, s, a);
}

template <typename T>
hipError_t launch(Args a, const Plan& p, hipStream_t s) {
  if (a.rows == 0) {
    const hipError_t e = start(xent_loss, 1, 1024, s, a);
    return e == hipSuccess && a.dweight ? start(xent_nothing<T>, a.vocab, 256, s, a) : e;
  }
  a.tiled = p.few ? a.rows64 : (uint32_t)std::min<uint64_t>(a.rows64, round_up(a.rows, p.bm));
  // a few rows are prepared beside the statistics, and joined with the loss
  const bool grads = a.dx || a.dweight;
  if (p.few && grads) a.prepare = a.rows64 / 16;
  hipError_t e = p.few ? few<T, true, false>(a, p, a.prepare + a.tiles, s) : product<T, kStats>(a, p, s);
  if (e != hipSuccess) return e;
  if (p.few && grads) {
    e = p.past ? few<T, false, true>(a, p, a.splits, s) : few<T, false, false>(a, p, a.splits, s);
    return e == hipSuccess && a.dx ? states<T>(a, false, s) : e;
  }
  e = grads ? start(xent_rows<T>, a.rows64 / 16, 1024, s, a) : start(xent_join, (a.rows + 15) / 16, 1024, s, a);
  if (e != hipSuccess) return e;
  // (the loss: with the rows, with dx, or by itself)
  if (grads ? !a.dx : a.rows > 16) e = start(xent_loss, 1, 1024, s, a);
  if (e != hipSuccess || !grads) return e;
  for (a.first = 0; a.first < a.vocab; a.first += a.piece) {
    a.width = (uint32_t)std::min<uint64_t>(a.piece, round_up(a.vocab - a.first, 256));
    e = product<T, kSlopes>(a, p, s);
    if (e != hipSuccess) return e;
    if (a.dx) {
      e = product<T, kStates>(a, p, s);
      if (e != hipSuccess) return e;
    }
    if (a.dweight) {
      e = product<T, kTable>(a, p, s);
      if (e != hipSuccess) return e;
    }
  }
  if (!a.dx) return hipSuccess;
  return states<T>(a, true, s);
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
  a.factor = (float*)(ws + p.factor);
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
  a.slope_stride = p.slope_stride;
  a.splits = p.splits;
  a.split_steps = p.split_steps;
  a.split_stride = p.split_stride;
  return q.dtype == FT_BF16 ? launch<__bf16>(a, p, s) : launch<_Float16>(a, p, s);
}

}  // namespace fto
