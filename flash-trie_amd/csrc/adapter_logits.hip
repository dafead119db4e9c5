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

constexpr int kBM = 64, kBN = 128, kBK = 64, kThreads = 256;

// Block: rows [kBM m, ...) of the order by tokens [kBN n, ...); wave w has
// tokens 32 w ... 32 w + 31 of them, and all rows.
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
  // the adapters of the tile's rows, each for the rows that have it
  for (uint32_t i = 0; i < rows;) {
    const int32_t g = ad[i];
    uint32_t j = i + 1;
    while (j < rows && ad[j] == g) ++j;
    if (g >= 0 && (uint32_t)g < a.adapters) {
      const uint32_t s0 = i / 16, s1 = (j + 15) / 16;
      f32x4 d[2][kBM / 16] = {};
      for (uint32_t k0 = 0; k0 < a.rank32; k0 += 32) {
        u32x4 uf[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint32_t tok = min(n0 + wave * 32 + v * 16 + col, a.vocab - 1);
          uf[v] = load_k((const T*)a.up + (int64_t)g * a.up_stride[0] + (int64_t)tok * a.up_stride[1],
                         k0 + q * 8, a.rank);
        }
#pragma unroll
        for (int s = 0; s < kBM / 16; ++s) {
          if ((uint32_t)s < s0 || (uint32_t)s >= s1) continue;
          const T* z = (const T*)a.z + (uint64_t)(m0 + s * 16 + col) * kParts<T> * a.rank32 + k0 + q * 8;
#pragma unroll
          for (int part = 0; part < kParts<T>; ++part) {
            const u32x4 zf = load_vec(z + part * a.rank32);
#pragma unroll
            for (int v = 0; v < 2; ++v) d[v][s] = mfma(uf[v], zf, d[v][s], T{});
          }
        }
      }
#pragma unroll
      for (int s = 0; s < kBM / 16; ++s) {
        const uint32_t row = s * 16 + col;
        if (row >= i && row < j) {
          const float f = zsc[row];
#pragma unroll
          for (int v = 0; v < 2; ++v) acc[v][s] += d[v][s] * f;
        }
      }
    }
    i = j;
  }
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

struct Plan {
  uint64_t perm, sorted, zscale, z, bytes;
};

Plan plan(const ft_adapter_logits_args& a) {
  Plan p{};
  Arena ar;
  const uint64_t parts = a.dtype == FT_BF16 ? kParts<__bf16> : kParts<_Float16>;
  p.perm = ar.take(a.rows * 4);
  p.sorted = ar.take(a.rows * 4);
  p.zscale = ar.take(a.rows * 4);
  // (whole tiles of rows are read)
  p.z = ar.take(round_up(a.rows, kBM) * parts * round_up(a.rank, 32) * 2);
  p.bytes = ar.used;
  return p;
}

template <typename T, typename O>
hipError_t launch(const ft_adapter_logits_args& q, const Args& a, hipStream_t s) {
  hipLaunchKernelGGL(logits_order, dim3(1), dim3(1024), 0, s, a);
  hipLaunchKernelGGL((logits_shrink<T>), dim3((a.rows + 15) / 16), dim3(256), 0, s, a);
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
  a.row_tiles = (a.rows + kBM - 1) / kBM;
  if (q.dtype == FT_BF16)
    return q.out_dtype == FT_F32 ? launch<__bf16, float>(q, a, s) : launch<__bf16, __bf16>(q, a, s);
  return q.out_dtype == FT_F32 ? launch<_Float16, float>(q, a, s)
                               : launch<_Float16, _Float16>(q, a, s);
}

}  // namespace fto
