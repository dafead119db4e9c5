// adapter_logits.hip -- logits of a shared vocabulary projection, each row
// with its request's low-rank adapter.
//
//   y[t, v] = sum_h x[t, h] w[v, h] + s_g sum_j z[t, j] up[g, v, j],
//   z[t, j] = sum_h x[t, h] down[g, j, h],  g = adapter[t]
//
// Rows are taken in the order of their adapters (their results do not depend
// on it), so that the 16 rows of a matrix tile have few different ones:
//   logits_order    one workgroup: the rows by adapter
//   logits_shrink   16 rows: z, kept as a sum of 16-bit parts (three bf16 or
//                   two f16 of a row scaled to [1, 2)), 22 bits or more
//   logits_product  a tile of rows x tokens: the product by w, then for each
//                   adapter among the tile's rows the product of z by its up
#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kMaxBins = 8192;  // adapters that logits_order sorts by

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

template <typename T>
constexpr int kParts = 2;
template <>
constexpr int kParts<__bf16> = 3;

struct Args {
  const void* x;
  const void* weight;
  const void* down;
  const void* up;
  int64_t x_stride, weight_stride, down_stride[2], up_stride[2], out_stride;
  uint32_t rows, hidden, vocab, adapters, rank, rank32;  // rank up to whole 32s
  const int32_t* adapter;
  const float* scale;
  void* out;
  // workspace
  int32_t* perm;      // [rows]: the rows by adapter
  int32_t* sorted;    // [rows]: their adapters (-1: none)
  float* zscale;      // [rows]: power of two that z was divided by
  uint16_t* z;        // [rows to whole 16s][kParts][rank32]
  uint32_t* zeros;  // 16 bytes of zeros
  uint32_t row_tiles;
};

// Eight elements of a row from column k on, zero past its end.
template <typename T>
__device__ __forceinline__ u32x4 load_k(const T* row, uint32_t k, uint32_t n) {
  if (k + 8 <= n) return load_vec(row + k);
  return load_part(row + (k < n ? k : 0u), k < n ? (int)(n - k) : 0, (T)0.0f);
}

__global__ void __launch_bounds__(1024) logits_order(Args a) {
  // bin 0: none; 1 + g; the last: out of range
  __shared__ uint32_t at[kMaxBins + 2];
  __shared__ uint32_t waves[16];
  const uint32_t tid = threadIdx.x, bins = a.adapters + 2;
  if (tid < 4) a.zeros[tid] = 0;
  const auto bin = [&](int32_t g) {
    return g < 0 ? 0u : (uint32_t)g < a.adapters ? (uint32_t)g + 1 : bins - 1;
  };
  if (a.adapters > (uint32_t)kMaxBins) {  // as they come
    for (uint32_t i = tid; i < a.rows; i += 1024) {
      a.perm[i] = (int32_t)i;
      a.sorted[i] = max(a.adapter[i], -1);
    }
    return;
  }
  for (uint32_t i = tid; i < bins; i += 1024) at[i] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < a.rows; i += 1024) atomicAdd(&at[bin(a.adapter[i])], 1u);
  __syncthreads();
  // exclusive sums over the bins, neighbours a thread
  const uint32_t each = (bins + 1023) / 1024, b0 = min(tid * each, bins), b1 = min(b0 + each, bins);
  uint32_t sum = 0, t;
  for (uint32_t i = b0; i < b1; ++i) sum += at[i];
  uint32_t front = wave_scan(sum, tid & 63, &t);
  if ((tid & 63) == 0) waves[tid >> 6] = t;
  __syncthreads();
  for (uint32_t w = 0; w < tid >> 6; ++w) front += waves[w];
  for (uint32_t i = b0; i < b1; ++i) {
    const uint32_t n = at[i];
    at[i] = front;
    front += n;
  }
  __syncthreads();
  for (uint32_t i = tid; i < a.rows; i += 1024) {
    const int32_t g = a.adapter[i];
    const uint32_t p = atomicAdd(&at[bin(g)], 1u);
    a.perm[p] = (int32_t)i;
    a.sorted[p] = max(g, -1);
  }
}

// Block b: rows [16 b, 16 b + 16) of the order; the waves share the hidden
// columns and add up in LDS.
template <typename T>
__global__ void __launch_bounds__(256) logits_shrink(Args a) {
  __shared__ float part[4][16][16];     // wave, rank, row
  __shared__ float zs[16][FT_MAX_RANK];  // row, rank
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t r0 = blockIdx.x * 16, n = min(16u, a.rows - r0), col = lane & 15, q = lane >> 4;
  for (uint32_t i = tid; i < 16 * a.rank32; i += 256) zs[i / a.rank32][i % a.rank32] = 0.0f;
  const uint32_t mine = r0 + min(col, n - 1);
  const T* x = (const T*)a.x + (int64_t)a.perm[mine] * a.x_stride;
  __syncthreads();
  for (uint32_t i = 0; i < n;) {
    const int32_t g = a.sorted[r0 + i];
    uint32_t j = i + 1;
    while (j < n && a.sorted[r0 + j] == g) ++j;
    if (g >= 0 && (uint32_t)g < a.adapters) {
      for (uint32_t k0 = 0; k0 < a.rank; k0 += 16) {
        const uint32_t rk = min(k0 + col, a.rank - 1);
        const T* d = (const T*)a.down + (int64_t)g * a.down_stride[0] + (int64_t)rk * a.down_stride[1];
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t h = wave * 32; h < a.hidden; h += 128)
          acc = mfma(load_k(d, h + q * 8, a.hidden), load_k(x, h + q * 8, a.hidden), acc, T{});
#pragma unroll
        for (int e = 0; e < 4; ++e) part[wave][q * 4 + e][col] = acc[e];
        __syncthreads();
        const uint32_t k = tid >> 4, row = tid & 15;
        if (row >= i && row < j && k0 + k < a.rank)
          zs[row][k0 + k] = a.scale[g] * (((part[0][k][row] + part[1][k][row]) + part[2][k][row]) +
                                          part[3][k][row]);
        __syncthreads();
      }
    }
    i = j;
  }
  // 16 threads a row: its power of two, then the parts
  const uint32_t row = tid >> 4, l = tid & 15;
  float big = 0.0f;
  for (uint32_t k = l; k < a.rank; k += 16) big = fmaxf(big, fabsf(zs[row][k]));
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) big = fmaxf(big, __shfl_xor(big, d, 64));
  int e = 0;
  if (big > 0.0f && big < INFINITY) (void)frexpf(big, &e), e -= 1;
  if (l == 0 && row < n) a.zscale[r0 + row] = ldexpf(1.0f, e);
  T* out = (T*)a.z + (uint64_t)(r0 + row) * kParts<T> * a.rank32;
  for (uint32_t k = l; k < a.rank32; k += 16) {
    float v = row < n ? ldexpf(zs[row][k], -e) : 0.0f;
#pragma unroll
    for (int s = 0; s < kParts<T>; ++s) {
      const T h = (T)v;
      out[s * a.rank32 + k] = h;
      const float rest = v - (float)h;
      v = fabsf((float)h) < INFINITY ? rest : 0.0f;
    }
  }
}

// The rows of a tile by their adapters: each run's product of z by its
// adapter's up is added to the rows that have it (not to the others in a
// 16-row tile: their product may hold a NaN of an adapter that is not
// theirs).  The wave's tokens are v0 ... v0 + 16 kN - 1, its rows the
// subtiles s0 ... s0 + kM - 1 of the tile.
template <typename T, int kN, int kM>
__device__ __forceinline__ void add_adapters(const Args& a, const int32_t* ad, const float* zsc,
                                             uint32_t m0, uint32_t rows, uint32_t v0, uint32_t s0,
                                             f32x4 (&acc)[kN][kM]) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  const uint32_t end = min((s0 + kM) * 16, rows);
  for (uint32_t i = s0 * 16; i < end;) {
    const int32_t g = __builtin_amdgcn_readfirstlane(ad[i]);
    uint32_t j = i + 1;
    while (j < end && __builtin_amdgcn_readfirstlane(ad[j]) == g) ++j;
    if (g >= 0 && (uint32_t)g < a.adapters) {
      for (uint32_t k0 = 0; k0 < a.rank32; k0 += 32) {
        u32x4 uf[kN];
#pragma unroll
        for (int v = 0; v < kN; ++v) {
          const uint32_t tok = min(v0 + v * 16 + col, a.vocab - 1);
          uf[v] = load_k((const T*)a.up + (int64_t)g * a.up_stride[0] + (int64_t)tok * a.up_stride[1],
                         k0 + q * 8, a.rank);
        }
#pragma unroll
        for (int s = 0; s < kM; ++s) {
          const uint32_t r0 = (s0 + s) * 16, row = r0 + col;
          if (r0 + 16 <= i || r0 >= j) continue;
          const T* z = (const T*)a.z + (uint64_t)(m0 + row) * kParts<T> * a.rank32 + k0 + q * 8;
          f32x4 d[kN] = {};
#pragma unroll
          for (int part = 0; part < kParts<T>; ++part) {
            const u32x4 zf = load_vec(z + part * a.rank32);
#pragma unroll
            for (int v = 0; v < kN; ++v) d[v] = mfma(uf[v], zf, d[v], T{});
          }
          if (row >= i && row < j) {
            const float f = zsc[row];
#pragma unroll
            for (int v = 0; v < kN; ++v) acc[v][s] += d[v] * f;
          }
        }
      }
    }
    i = j;
  }
}

constexpr int kBK = 64;  // hidden columns of a step: a line of a row

// Any alignment.  Block: rows [64 m, ...) of the order by tokens [128 n,
// ...); wave w has tokens 32 w ... 32 w + 31 of them, and all rows.
constexpr int kBM = 64, kBN = 128, kThreads = 256;
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) logits_product(Args a) {
  __shared__ u32x4 ws[kBN][kBK / 8];  // columns by 8, exchanged within a row
  __shared__ u32x4 xs[kBM][kBK / 8];
  __shared__ int32_t ad[kBM], to[kBM];
  __shared__ float zsc[kBM];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t tm = blockIdx.x % a.row_tiles, tn = blockIdx.x / a.row_tiles;
  const uint32_t m0 = tm * kBM, n0 = tn * kBN;
  const uint32_t rows = min((uint32_t)kBM, a.rows - m0);
  if (tid < kBM) {
    const uint32_t m = m0 + min(tid, rows - 1);
    to[tid] = a.perm[m];
    ad[tid] = tid < rows ? a.sorted[m] : -1;
    zsc[tid] = a.zscale[m];
  }
  __syncthreads();
  f32x4 acc[2][kBM / 16] = {};
  for (uint32_t k0 = 0; k0 < a.hidden; k0 += kBK) {
    u32x4 wr[kBN * kBK / 8 / kThreads], xr[kBM * kBK / 8 / kThreads];
#pragma unroll
    for (int i = 0; i < kBN * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid, v = min(n0 + at / 8, a.vocab - 1);
      wr[i] = load_k((const T*)a.weight + (int64_t)v * a.weight_stride, k0 + at % 8 * 8, a.hidden);
    }
#pragma unroll
    for (int i = 0; i < kBM * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid;
      xr[i] = load_k((const T*)a.x + (int64_t)to[at / 8] * a.x_stride, k0 + at % 8 * 8, a.hidden);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBN * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid, r = at / 8;
      ws[r][(at % 8) ^ (r & 7)] = wr[i];
    }
#pragma unroll
    for (int i = 0; i < kBM * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid, r = at / 8;
      xs[r][(at % 8) ^ (r & 7)] = xr[i];
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kBK / 32; ++kk) {
      u32x4 wf[2], xf[kBM / 16];
#pragma unroll
      for (int i = 0; i < 2; ++i) wf[i] = ws[wave * 32 + i * 16 + col][(kk * 4 + q) ^ (col & 7)];
#pragma unroll
      for (int j = 0; j < kBM / 16; ++j) xf[j] = xs[j * 16 + col][(kk * 4 + q) ^ (col & 7)];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < kBM / 16; ++j) acc[i][j] = mfma(wf[i], xf[j], acc[i][j], T{});
    }
  }
  add_adapters<T, 2, kBM / 16>(a, ad, zsc, m0, rows, n0 + wave * 32, 0, acc);
#pragma unroll
  for (int s = 0; s < kBM / 16; ++s) {
    const uint32_t row = s * 16 + col;
    if (row >= rows) continue;
    O* out = (O*)a.out + (int64_t)to[row] * a.out_stride;
    const bool bad = ad[row] >= 0 && (uint32_t)ad[row] >= a.adapters;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const uint32_t tok = n0 + wave * 32 + v * 16 + q * 4;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok + e < a.vocab) out[tok + e] = (O)(bad ? NAN : acc[v][s][e]);
    }
  }
}

// Inputs whose rows start at multiples of 16 bytes.  Block: rows [16 kBMs m,
// ...) by tokens [16 kBNs n, ...), as kWM x kWN waves.  Steps of kBK hidden
// columns are copied straight to LDS, kStages - 1 of them ahead; a row is a
// line of eight 16-byte columns, exchanged by the row's number so that the
// matrix operands are read without bank conflicts.  Columns past the end are
// copied from a line of zeros.
template <int kBMs, int kBNs, int kWM, int kWN, int kStages>
struct Shape {
  static constexpr int BM = 16 * kBMs, BN = 16 * kBNs, Threads = 64 * kWM * kWN;
  static constexpr int M = kBMs / kWM, N = kBNs / kWN;  // subtiles of a wave
  static constexpr int WM = kWM, WN = kWN, Stages = kStages;
  // 16-byte copies of a thread and step: tokens', rows'
  static constexpr int CW = BN * 8 / Threads, CX = (BM * 8 + Threads - 1) / Threads;
  static constexpr int XLanes = BM * 8 / CX / (kWM * kWN);  // lanes of a wave in the rows' copies
};

__device__ __forceinline__ void copy_to_lds(const void* from, void* to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)from,
                                   (__attribute__((address_space(3))) uint32_t*)to, 16, 0, 0);
}

// All LDS reads of the wave are done, and all its copies but the last n.
template <int n>
__device__ __forceinline__ void wait_copies() {
  asm volatile("" ::: "memory");
  // vmcnt n, lgkmcnt 0, the third counter free
  __builtin_amdgcn_s_waitcnt((n & 15) | (n >> 4) << 14 | 7 << 4);
}

template <typename T, typename O, typename S>
__global__ void __launch_bounds__(S::Threads) logits_staged(Args a) {
  // (an array a stage: the compiler tells their copies and reads apart)
  __shared__ u32x4 st0[(S::BM + S::BN) * 8], st1[(S::BM + S::BN) * 8];
  __shared__ u32x4 st2[S::Stages > 2 ? (S::BM + S::BN) * 8 : 1];
  __shared__ u32x4 st3[S::Stages > 3 ? (S::BM + S::BN) * 8 : 1];
  __shared__ int32_t ad[S::BM], to[S::BM];
  __shared__ float zsc[S::BM];
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t wm = wave % S::WM, wn = wave / S::WM;
  // Consecutive workgroups go to the XCDs in turn: each XCD takes a run of
  // tiles, the row tiles of a few token tiles together, so that its L2
  // serves the shared operands.
  const uint32_t n = gridDim.x, run = n / 8;
  const uint32_t tile = blockIdx.x < run * 8 ? (blockIdx.x % 8) * run + blockIdx.x / 8 : blockIdx.x;
  const uint32_t m0 = tile % a.row_tiles * S::BM, n0 = tile / a.row_tiles * S::BN;
  const uint32_t rows = min((uint32_t)S::BM, a.rows - m0);
  for (uint32_t i = tid; i < (uint32_t)S::BM; i += S::Threads) {
    const uint32_t m = m0 + min(i, rows - 1);
    to[i] = a.perm[m];
    ad[i] = i < rows ? a.sorted[m] : -1;
    zsc[i] = a.zscale[m];
  }
  __syncthreads();

  // this thread's part of each copy: a row and one of its columns
  const T* wp[S::CW];
  const T* xp[S::CX];
  uint32_t wk[S::CW], xk[S::CX];
#pragma unroll
  for (int i = 0; i < S::CW; ++i) {
    const uint32_t at = i * S::Threads + tid, r = at / 8;
    wk[i] = ((at & 7) ^ (r & 7)) * 8;
    wp[i] = (const T*)a.weight + (int64_t)min(n0 + r, a.vocab - 1) * a.weight_stride;
  }
#pragma unroll
  for (int i = 0; i < S::CX; ++i) {
    const uint32_t at = (i * S::WM * S::WN + wave) * S::XLanes + lane, r = min(at / 8, S::BM - 1u);
    xk[i] = ((at & 7) ^ (r & 7)) * 8;
    xp[i] = (const T*)a.x + (int64_t)to[r] * a.x_stride;
  }
  const auto copy = [&](u32x4* st, uint32_t k0) {
#pragma unroll
    for (int i = 0; i < S::CW; ++i) {
      const uint32_t k = k0 + wk[i];
      copy_to_lds(k < a.hidden ? (const void*)(wp[i] + k) : (const void*)a.zeros,
                  st + i * S::Threads + wave * 64);
    }
#pragma unroll
    for (int i = 0; i < S::CX; ++i) {
      const uint32_t k = k0 + xk[i];
      if (S::XLanes == 64 || lane < (uint32_t)S::XLanes)
        copy_to_lds(k < a.hidden ? (const void*)(xp[i] + k) : (const void*)a.zeros,
                    st + S::BN * 8 + (i * S::WM * S::WN + wave) * S::XLanes);
    }
  };
  f32x4 acc[S::N][S::M] = {};
  const auto multiply = [&](const u32x4* st) {
    const u32x4* ws = st + (wn * S::N * 16 + col) * 8;
    const u32x4* xs = st + S::BN * 8 + (wm * S::M * 16 + col) * 8;
#pragma unroll
    for (int kk = 0; kk < kBK / 32; ++kk) {
      const uint32_t c = (kk * 4 + q) ^ (col & 7);
      u32x4 wf[S::N], xf[S::M];
#pragma unroll
      for (int i = 0; i < S::N; ++i) wf[i] = ws[i * 128 + c];
#pragma unroll
      for (int j = 0; j < S::M; ++j) xf[j] = xs[j * 128 + c];
#pragma unroll
      for (int j = 0; j < S::M; ++j)
#pragma unroll
        for (int i = 0; i < S::N; ++i) acc[i][j] = mfma(wf[i], xf[j], acc[i][j], T{});
    }
  };
  // One barrier a step: past it, every wave's copies of this step are in LDS
  // and every wave has read the step before, whose place the next copy
  // takes.  Copies complete in order, so those of later steps may be left.
  constexpr int kCopies = S::CW + S::CX;
  const uint32_t steps = (a.hidden + kBK - 1) / kBK;
  const auto step = [&](uint32_t i, const u32x4* st, u32x4* next) {
    if (i + S::Stages - 1 <= steps) wait_copies<kCopies * (S::Stages - 2)>();
    else wait_copies<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + S::Stages - 1 < steps) copy(next, (i + S::Stages - 1) * kBK);
    multiply(st);
  };
  copy(st0, 0);
  if (S::Stages > 2 && steps > 1) copy(st1, kBK);
  if (S::Stages > 3 && steps > 2) copy(st2, 2 * kBK);
  for (uint32_t i = 0; i < steps; i += S::Stages) {
    if (S::Stages == 2) {
      step(i, st0, st1);
      if (i + 1 < steps) step(i + 1, st1, st0);
    } else if (S::Stages == 3) {
      step(i, st0, st2);
      if (i + 1 < steps) step(i + 1, st1, st0);
      if (i + 2 < steps) step(i + 2, st2, st1);
    } else {
      step(i, st0, st3);
      if (i + 1 < steps) step(i + 1, st1, st0);
      if (i + 2 < steps) step(i + 2, st2, st1);
      if (i + 3 < steps) step(i + 3, st3, st2);
    }
  }
  add_adapters<T, S::N, S::M>(a, ad, zsc, m0, rows, n0 + wn * S::N * 16, wm * S::M, acc);
  // 16 rows at a time through LDS (a part of it for each wave), so that a
  // row's tokens are stored side by side
  __syncthreads();
  constexpr int kRow = S::N * 16 + 4;  // floats; shifted by four banks a row
  static_assert(kRow * 16 * 4 * S::WM * S::WN <= (S::BM + S::BN) * 128 * 2, "fits two stages");
  constexpr int kHalf = S::WM * S::WN / 2;
  float* const mine = (float*)(wave < (uint32_t)kHalf ? st0 : st1) +
                      (wave < (uint32_t)kHalf ? wave : wave - kHalf) * (kRow * 16);
  constexpr int kE = 16 / (int)sizeof(O), kPer = S::N * 16 / kE;  // elements, pieces of a row
#pragma unroll
  for (int s = 0; s < S::M; ++s) {
#pragma unroll
    for (int i = 0; i < S::N; ++i) *(f32x4*)(mine + col * kRow + i * 16 + q * 4) = acc[i][s];
    asm volatile("" ::: "memory");  // (a wave's LDS accesses are in order)
#pragma unroll
    for (int p = 0; p < 16 * kPer / 64; ++p) {
      const uint32_t at = p * 64 + lane, r = at / kPer, c = at % kPer * kE;
      const uint32_t row = (wm * S::M + s) * 16 + r, tok = n0 + wn * S::N * 16 + c;
      if (row < rows && tok < a.vocab) {
        const bool bad = ad[row] >= 0 && (uint32_t)ad[row] >= a.adapters;
        float y[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) y[e] = bad ? NAN : mine[r * kRow + c + e];
        O* out = (O*)a.out + (int64_t)to[row] * a.out_stride + tok;
        const u32x4 o = from_float<O>(y);
        if (tok + kE <= a.vocab) store_vec(out, o);
        else store_part(out, (int)(a.vocab - tok), o);
      }
    }
    asm volatile("" ::: "memory");
  }
}

struct Plan {
  uint64_t perm, sorted, zscale, zeros, z, bytes;
};

Plan plan(const ft_adapter_logits_args& a) {
  Plan p{};
  Arena ar;
  const uint64_t parts = a.dtype == FT_BF16 ? kParts<__bf16> : kParts<_Float16>;
  p.perm = ar.take(a.rows * 4);
  p.sorted = ar.take(a.rows * 4);
  p.zscale = ar.take(a.rows * 4);
  p.zeros = ar.take(16);
  p.z = ar.take(round_up(a.rows, 16) * parts * round_up(a.rank, 32) * 2);
  p.bytes = ar.used;
  return p;
}

template <typename T, typename O, typename S>
hipError_t launch_staged(Args a, hipStream_t s) {
  a.row_tiles = (a.rows + S::BM - 1) / S::BM;
  const uint32_t tiles = (a.vocab + S::BN - 1) / S::BN;
  hipLaunchKernelGGL((logits_staged<T, O, S>), dim3(tiles * a.row_tiles), dim3(S::Threads), 0, s, a);
  return hipGetLastError();
}

bool whole_vectors(const void* p, int64_t stride) {
  return (uintptr_t)p % 16 == 0 && stride % 8 == 0;
}

template <typename T, typename O>
hipError_t launch(Args a, hipStream_t s) {
  hipLaunchKernelGGL(logits_order, dim3(1), dim3(1024), 0, s, a);
  hipLaunchKernelGGL((logits_shrink<T>), dim3((a.rows + 15) / 16), dim3(256), 0, s, a);
  if (a.hidden % 8 == 0 && whole_vectors(a.x, a.x_stride) &&
      whole_vectors(a.weight, a.weight_stride)) {
    if (a.rows <= 16) return launch_staged<T, O, Shape<1, 8, 1, 4, 4>>(a, s);
    if (a.rows <= 32) return launch_staged<T, O, Shape<2, 8, 1, 4, 3>>(a, s);
    if (a.rows <= 64) return launch_staged<T, O, Shape<4, 8, 1, 4, 3>>(a, s);
    if (a.rows <= 96) return launch_staged<T, O, Shape<6, 16, 1, 8, 3>>(a, s);
    if (a.rows <= 128) return launch_staged<T, O, Shape<8, 16, 1, 8, 3>>(a, s);
    return launch_staged<T, O, Shape<16, 16, 2, 4, 2>>(a, s);
  }
  a.row_tiles = (a.rows + kBM - 1) / kBM;
  const uint32_t tiles = (a.vocab + kBN - 1) / kBN;
  hipLaunchKernelGGL((logits_product<T, O>), dim3(tiles * a.row_tiles), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace

uint64_t adapter_logits_workspace(const ft_adapter_logits_args& a) { return plan(a).bytes; }

hipError_t launch_adapter_logits(const ft_adapter_logits_args& q, uint8_t* ws, hipStream_t s) {
  if (q.rows == 0) return hipSuccess;
  const Plan p = plan(q);
  Args a{};
  a.x = q.x;
  a.weight = q.weight;
  a.down = q.down;
  a.up = q.up;
  a.x_stride = q.x_stride;
  a.weight_stride = q.weight_stride;
  for (int i = 0; i < 2; ++i) {
    a.down_stride[i] = q.down_stride[i];
    a.up_stride[i] = q.up_stride[i];
  }
  a.out_stride = q.out_stride;
  a.rows = (uint32_t)q.rows;
  a.hidden = q.hidden;
  a.vocab = q.vocab;
  a.adapters = q.adapters;
  a.rank = q.rank;
  a.rank32 = (uint32_t)round_up(q.rank, 32);
  a.adapter = q.adapter;
  a.scale = q.scale;
  a.out = q.out;
  a.perm = (int32_t*)(ws + p.perm);
  a.sorted = (int32_t*)(ws + p.sorted);
  a.zscale = (float*)(ws + p.zscale);
  a.z = (uint16_t*)(ws + p.z);
  a.zeros = (uint32_t*)(ws + p.zeros);
  if (q.dtype == FT_BF16)
    return q.out_dtype == FT_F32 ? launch<__bf16, float>(a, s) : launch<__bf16, __bf16>(a, s);
  return q.out_dtype == FT_F32 ? launch<_Float16, float>(a, s)
                               : launch<_Float16, _Float16>(a, s);
}

}  // namespace fto
