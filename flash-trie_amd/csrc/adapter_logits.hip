// adapter_logits.hip -- logits of a shared vocabulary projection, each row
// with its request's low-rank adapter.
//
//   y[t, v] = sum_h x[t, h] w[v, h] + s_g sum_j z[t, j] up[g, v, j],
//   z[t, j] = sum_h x[t, h] down[g, j, h],  g = adapter[t]
//
// Rows are taken in the order of their adapters, so that the 16 rows of a
// matrix tile have few different ones:
//   logits_order    one workgroup: the rows by adapter
//   logits_shrink   16 rows: z, kept as a sum of 16-bit parts (three bf16 or
//                   two f16 of a row scaled to [1, 2)), 22 bits or more
//   logits_product, logits_staged, logits_tile  a tile of rows x tokens: the
//                   product by w, then for each adapter among the tile's rows
//                   the product of z by its up.  Inputs of any alignment; of
//                   whole 16-byte vectors; the same with many rows
//
// Up to 96 rows one read of w bounds it: 16 rows, 2,200,000 x 512 bf16: 481
// us, 5.1 TB/s; 84 rows, 262,144 x 1024, 6 adapters of rank 12 in no order:
// 172 us, 3.5 TB/s, with the adapters' turns (no adapters: 132).  From 97 to
// 250 rows of that size neither memory (125-140 us of bytes) nor the matrix
// cores do: 112 rows take 205 us (no adapters: 149) with one workgroup on a CU,
// whose adapters' turns nothing hides, 144 to 250 rows 241-255 us in tiles of
// 256 rows that are part empty.  Above, the matrix cores do: 4096 rows, 32,768
// x 1024 f16, 16 adapters of rank 64: 378 us, 0.77 PFLOP/s counting the
// adapters' products once.
#include <algorithm>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kCUs = 256;
constexpr int kMaxBins = 510;  // adapters that logits_order sorts by

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
  uint32_t shares;  // of logits_shrink's blocks
  bool whole_up;  // up's rows are whole vectors at multiples of 16 bytes
};

// Eight elements of a row of n from column k on, zero past its end.
template <typename T>
__device__ __forceinline__ u32x4 load_k(const T* row, uint32_t k, uint32_t n) {
  return load_row_vec(row, k, n, (T)0.0f);
}

// Rows of an adapter stay in their order, so that a row's place, and with it
// the order of its sums, is the same in every call.  A wave takes a run of
// rows: counts them by adapter, then places them 64 at a time.
__global__ void __launch_bounds__(1024) logits_order(Args a) {
  // bin 0: none; 1 + g; the last: out of range
  __shared__ uint32_t at[kMaxBins + 2][16];  // of a bin and wave
  __shared__ uint32_t waves[16];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, bins = a.adapters + 2;
  const auto bin = [&](int32_t g) {
    return g < 0 ? 0u : (uint32_t)g < a.adapters ? (uint32_t)g + 1 : bins - 1;
  };
  if (tid < 4) a.zeros[tid] = 0;
  if (a.adapters > (uint32_t)kMaxBins) {  // as they come
    for (uint32_t i = tid; i < a.rows; i += 1024) {
      a.perm[i] = (int32_t)i;
      a.sorted[i] = max(a.adapter[i], -1);
    }
    return;
  }
  const uint32_t run = (a.rows + 1023) / 1024 * 64;
  const uint32_t r0 = min(wave * run, a.rows), r1 = min(r0 + run, a.rows);
  for (uint32_t i = tid; i < bins * 16; i += 1024) (&at[0][0])[i] = 0;
  __syncthreads();
  for (uint32_t i = r0 + lane; i < r1; i += 64) atomicAdd(&at[bin(a.adapter[i])][wave], 1u);
  __syncthreads();
  // exclusive sums over (bin, wave), neighbours a thread
  const uint32_t cells = bins * 16, each = (cells + 1023) / 1024;
  const uint32_t b0 = min(tid * each, cells), b1 = min(b0 + each, cells);
  uint32_t sum = 0, t;
  for (uint32_t i = b0; i < b1; ++i) sum += (&at[0][0])[i];
  uint32_t front = wave_scan(sum, &t);
  if (lane == 0) waves[wave] = t;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) front += waves[w];
  for (uint32_t i = b0; i < b1; ++i) {
    const uint32_t n = (&at[0][0])[i];
    (&at[0][0])[i] = front;
    front += n;
  }
  __syncthreads();
  for (uint32_t i0 = r0; i0 < r1; i0 += 64) {
    const bool in = i0 + lane < r1;
    const int32_t g = in ? a.adapter[i0 + lane] : 0;
    const uint32_t mine = in ? bin(g) : ~0u;
    uint64_t left = __ballot(in);
    while (left) {  // the bins among the 64 rows
      const uint32_t b = (uint32_t)__builtin_amdgcn_readlane(
          (int)mine, (int)__ffsll((unsigned long long)left) - 1);
      const uint64_t same = __ballot(mine == b);
      const uint32_t base = at[b][wave];
      if (mine == b) {
        const uint32_t p = base + (uint32_t)__popcll(same & ((1ull << lane) - 1));
        a.perm[p] = (int32_t)(i0 + lane);
        a.sorted[p] = max(g, -1);
      }
      if (lane == 0) at[b][wave] = base + (uint32_t)__popcll(same);
      left &= ~same;
    }
  }
}

// Rows [16 b, 16 b + 16) of the order by `shares` blocks, which take their
// runs of rows with the same adapter in turn; 64 ranks at a time; the 16
// waves share the hidden columns, a run of steps each with its loads
// together, and add up in LDS.  Bound by latency: one way to memory for each
// run, so there are as many blocks as CUs (16 rows of an adapter each, 32768
// x 1024, rank 8: 66 us with one block, 34 with 16).  At most 16 rows are put
// in order here, as logits_order would (16 rows of 4 adapters in turn, 262144
// x 1024: 126 us, in their own order 144).
constexpr int kShrinkT = 1024;

template <typename T>
__global__ void __launch_bounds__(kShrinkT) logits_shrink(Args a) {
  __shared__ float part[16][64][16 + 1];     // wave, rank, row
  __shared__ float zs[16][FT_MAX_RANK + 1];  // row, rank
  __shared__ uint32_t order[16];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t share = blockIdx.x % a.shares;
  const uint32_t r0 = blockIdx.x / a.shares * 16, n = min(16u, a.rows - r0), col = lane & 15, q = lane >> 4;
  const bool alone = a.rows <= 16;
  for (uint32_t i = tid; i < 16 * a.rank32; i += kShrinkT) zs[i / a.rank32][i % a.rank32] = 0.0f;
  const uint32_t mine = r0 + min(col, n - 1);
  uint32_t at = mine;
  // the adapters of the 16 rows, a row a lane
  int32_t own;
  if (alone) {
    own = max(a.adapter[mine], -1);
    uint32_t rank = 0;  // of this lane's row
    for (uint32_t j = 0; j < n; ++j) {
      const int32_t g = __builtin_amdgcn_readlane(own, (int)j);
      rank += g < own || (g == own && j < mine);
    }
    if (tid < n) order[rank] = tid;
    __syncthreads();
    at = order[mine];
    own = __shfl(own, (int)at, 64);
    if (share == 0 && tid < n) {
      a.perm[tid] = (int32_t)at;
      a.sorted[tid] = own;
    }
    if (share == 0 && tid < 4) a.zeros[tid] = 0;
  } else {
    at = (uint32_t)a.perm[mine];
    own = max(a.sorted[mine], -1);
  }
  const T* x = (const T*)a.x + (int64_t)at * a.x_stride;
  __syncthreads();
  uint32_t run = 0, written = share == 0 ? ~0u << n : 0u;  // rows that this block writes
  for (uint32_t i = 0; i < n; ++run) {
    const int32_t g = __builtin_amdgcn_readlane(own, (int)i);
    // rows from i on with the same adapter
    const uint64_t other = __ballot(own != g) & 0xFFFFu & ~((2u << i) - 1u);
    const uint32_t j = min(n, other ? (uint32_t)__ffsll((unsigned long long)other) - 1u : 16u);
    if (run % a.shares != share) {
      i = j;
      continue;
    }
    written |= (1u << j) - (1u << i);
    if (g >= 0 && (uint32_t)g < a.adapters) {
      const T* down = (const T*)a.down + (int64_t)g * a.down_stride[0];
      const float scale = a.scale[g];
      for (uint32_t k0 = 0; k0 < a.rank; k0 += 64) {
        const uint32_t tiles = min(4u, (a.rank - k0 + 15) / 16);
        const T* d[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
          d[t] = down + (int64_t)min(k0 + t * 16 + col, a.rank - 1) * a.down_stride[1];
        f32x4 acc[4] = {};
#pragma unroll 2
        for (uint32_t h = wave * 32; h < a.hidden; h += 16 * 32) {
          const u32x4 xf = load_k(x, h + q * 8, a.hidden);
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if ((uint32_t)t < tiles) acc[t] = mfma(load_k(d[t], h + q * 8, a.hidden), xf, acc[t], T{});
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if ((uint32_t)t < tiles)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[wave][t * 16 + q * 4 + e][col] = acc[t][e];
        __syncthreads();
        const uint32_t k = tid >> 4, row = tid & 15;
        if (row >= i && row < j && k0 + k < a.rank) {
          float v = 0.0f;
#pragma unroll
          for (int w = 0; w < 16; ++w) v += part[w][k][row];
          zs[row][k0 + k] = scale * v;
        }
        __syncthreads();
      }
    }
    i = j;
  }
  // a wave a row: its power of two, then the parts
  const uint32_t row = wave;
  if (!(written >> row & 1)) return;
  float big = 0.0f;
  for (uint32_t k = lane; k < a.rank; k += 64) big = fmaxf(big, fabsf(zs[row][k]));
  big = wave_max(big);
  int e = 0;
  // f16: its largest to [1, 2); bf16 has the range of z
  if (kParts<T> == 2 && big > 0.0f && big < INFINITY) (void)frexpf(big, &e), e -= 1;
  if (lane == 0 && row < n) a.zscale[r0 + row] = ldexpf(1.0f, e);
  T* out = (T*)a.z + (uint64_t)(r0 + row) * kParts<T> * a.rank32;
  for (uint32_t k = lane; k < a.rank32; k += 64) {
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

// What a workgroup knows of its tile's rows: their places, adapters and z's
// powers of two, and the runs of rows with the same adapter.
template <int kBM>
struct Rows {
  int32_t ad[kBM], to[kBM];
  float zsc[kBM];
  int32_t run_g[kBM];  // runs of rows with an adapter
  uint16_t run_i[kBM], run_j[kBM];
  uint32_t runs;
};

template <int kBM>
__device__ __forceinline__ void read_rows(const Args& a, Rows<kBM>& r, uint32_t m0, uint32_t rows) {
  for (uint32_t i = threadIdx.x; i < (uint32_t)kBM; i += blockDim.x) {
    const uint32_t m = m0 + min(i, rows - 1);
    r.to[i] = a.perm[m];
    r.ad[i] = i < rows ? a.sorted[m] : -1;
    r.zsc[i] = a.zscale[m];
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    constexpr int kWords = (kBM + 63) / 64;
    const uint32_t lane = threadIdx.x;
    uint64_t starts[kWords], own[kWords];  // rows that start a run; with an adapter
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      const uint32_t i = w * 64 + lane;
      const int32_t g = i < rows ? r.ad[i] : -1;
      const bool start = i == rows || (i < rows && (i == 0 || r.ad[i - 1] != g));
      starts[w] = __ballot(start);
      own[w] = __ballot(i < rows && start && g >= 0 && (uint32_t)g < a.adapters);
    }
    uint32_t n = 0;
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
      if (own[w] >> lane & 1) {
        const uint64_t after = lane < 63 ? starts[w] >> (lane + 1) << (lane + 1) : 0;
        uint32_t j = after ? w * 64 + (uint32_t)__ffsll((unsigned long long)after) - 1 : rows;
        if (!after) {
#pragma unroll
          for (int v = kWords - 1; v > w; --v)
            if (starts[v]) j = v * 64 + (uint32_t)__ffsll((unsigned long long)starts[v]) - 1;
        }
        const uint32_t at = n + (uint32_t)__popcll(own[w] & ((1ull << lane) - 1));
        r.run_g[at] = r.ad[w * 64 + lane];
        r.run_i[at] = (uint16_t)(w * 64 + lane);
        r.run_j[at] = (uint16_t)j;
      }
      n += (uint32_t)__popcll(own[w]);
    }
    if (lane == 0) r.runs = n;
  }
  __syncthreads();
}

// 16 bytes a lane, from each lane's address to the wave's place in LDS.
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

// This thread's vectors of the ups of runs b ... b + n - 1, ranks k0 ... k0 +
// 31, those numbered t0 ... t0 + kF - 1 of its share.
template <typename T, int kBM, int kBN, uint32_t kT, uint32_t kF>
__device__ __forceinline__ void load_ups(const Args& a, const Rows<kBM>& r, uint32_t n0, uint32_t tid,
                                         uint32_t b, uint32_t n, uint32_t k0, uint32_t t0,
                                         u32x4 (&piece)[kF]) {
#pragma unroll
  for (uint32_t t = 0; t < kF; ++t) {
    const uint32_t p = (t0 + t) * kT + tid, k = p / (kBN * 4), row = p / 4 % kBN;
    piece[t] = u32x4{};
    if (k < n)
      piece[t] = load_k((const T*)a.up + (int64_t)r.run_g[b + k] * a.up_stride[0] +
                            (int64_t)min(n0 + row, a.vocab - 1) * a.up_stride[1],
                        k0 + (p & 3) * 8, a.rank);
  }
}

// The adapters of the tile's rows: each run's product of z by its adapter's
// up, 32 ranks at a time, is added to the rows of the run (not to the others
// in a 16-row tile: their product may hold a NaN of an adapter that is not
// theirs).  z and the ups of several runs are brought to LDS together, since
// a tile waits for each such turn; `zs` holds kBM * kParts * 4 vectors, each
// of up0, up1, up2 kHeld runs' kBN * 4.  kAhead: the first turn's ups are in
// `ahead`, loaded before the main product.  The workgroup's tokens are n0 ...;
// the wave's are the subtiles vs ... of them, its rows the subtiles s0 ....
template <typename T, int kBM, int kBN, int kN, int kM, uint32_t kT, uint32_t kHeld, uint32_t kBuffers,
          bool kAhead, uint32_t kPieces>
__device__ __forceinline__ void add_adapters(const Args& a, const Rows<kBM>& r, uint32_t m0,
                                             uint32_t rows, uint32_t n0, uint32_t vs, uint32_t s0,
                                             uint32_t tid, u32x4* zs, u32x4* up0, u32x4* up1, u32x4* up2,
                                             const u32x4 (&ahead)[kPieces], f32x4 (&acc)[kN][kM]) {
  static_assert(kHeld >= 1, "a run's up fits");
  const uint32_t lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t runs = (uint32_t)__builtin_amdgcn_readfirstlane((int)r.runs);
  constexpr uint32_t kBatch = kHeld * kBuffers, kFlight = kN * kM >= 32 ? 2 : kPieces;
  const auto buffer = [&](uint32_t k) {
    return (k < kHeld ? up0 : k < 2 * kHeld ? up1 : up2) + k % kHeld * (kBN * 4);
  };
  // (rows of half a line, four columns, exchanged by half the row's number)
  const uint32_t c = q ^ (col >> 1 & 3);
  for (uint32_t k0 = 0; k0 < a.rank32; k0 += 32) {
    for (uint32_t b = 0; b < runs; b += kBatch) {
      const uint32_t n = min(kBatch, runs - b);
      __syncthreads();
      const uint32_t first = tid & ~63u;  // of the wave
      if (b == 0) {  // z, a vector a thread and turn (rows past the tile's last sixteen: not read)
        constexpr uint32_t kVecs = kParts<T> * kBM * 4;
        for (uint32_t p = tid; p < kVecs; p += kT) {
          const uint32_t part = p / (kBM * 4), row = p / 4 % kBM, k = (p & 3) ^ (row >> 1 & 3);
          if (row < (rows + 15) / 16 * 16)
            copy_to_lds((const T*)a.z + ((uint64_t)(m0 + row) * kParts<T> + part) * a.rank32 + k0 + k * 8,
                        zs + (p - tid + first));
        }
      }
      if (!kAhead && a.whole_up) {
        for (uint32_t p = tid; p < n * (kBN * 4); p += kT) {
          const uint32_t k = p / (kBN * 4), row = p / 4 % kBN, at = k0 + ((p & 3) ^ (row >> 1 & 3)) * 8;
          const T* up = (const T*)a.up + (int64_t)r.run_g[b + k] * a.up_stride[0] +
                        (int64_t)min(n0 + row, a.vocab - 1) * a.up_stride[1] + at;
          copy_to_lds(at < a.rank ? (const void*)up : (const void*)a.zeros,
                      buffer(k) + (p - tid + first) % (kBN * 4));
        }
      } else {
        // several loads in flight, as far as there are registers beside the
        // accumulators
        static_assert(kPieces % kFlight == 0 && kPieces * kT == kBatch * kBN * 4, "whole turns");
#pragma unroll
        for (uint32_t t0 = 0; t0 < kPieces; t0 += kFlight) {
          u32x4 piece[kFlight];
          if (kAhead && b == 0 && k0 == 0) {
#pragma unroll
            for (uint32_t t = 0; t < kFlight; ++t) piece[t] = ahead[t0 + t];
          } else {
            load_ups<T, kBM, kBN, kT>(a, r, n0, tid, b, n, k0, t0, piece);
          }
#pragma unroll
          for (uint32_t t = 0; t < kFlight; ++t) {
            const uint32_t p = (t0 + t) * kT + tid, k = p / (kBN * 4), row = p / 4 % kBN;
            if (k < n) buffer(k)[row * 4 + ((p & 3) ^ (row >> 1 & 3))] = piece[t];
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      wait_copies<0>();  // (a barrier alone does not wait for them)
      __syncthreads();
      for (uint32_t k = 0; k < n; ++k) {
        const uint32_t i = (uint32_t)__builtin_amdgcn_readfirstlane((int)r.run_i[b + k]);
        const uint32_t j = (uint32_t)__builtin_amdgcn_readfirstlane((int)r.run_j[b + k]);
        if (j <= s0 * 16 || i >= (s0 + kM) * 16) continue;
        // (four token subtiles at a time: the accumulators leave few registers)
        constexpr int kV = kN < 4 ? kN : 4;
#pragma unroll
        for (int v0 = 0; v0 < kN; v0 += kV) {
          const u32x4* up = buffer(k) + ((vs + v0) * 16 + col) * 4 + c;
          u32x4 uf[kV];
#pragma unroll
          for (int v = 0; v < kV; ++v) uf[v] = up[v * 64];
#pragma unroll
          for (int s = 0; s < kM; ++s) {
            const uint32_t r0 = (s0 + s) * 16, row = r0 + col;
            if (r0 + 16 <= i || r0 >= j) continue;
            const bool whole = r0 >= i && r0 + 16 <= j;
            if (kParts<T> == 3 && whole) {  // bf16: z is not scaled
#pragma unroll
              for (int part = 0; part < kParts<T>; ++part) {
                const u32x4 zf = zs[(part * kBM + row) * 4 + c];
#pragma unroll
                for (int v = 0; v < kV; ++v) acc[v0 + v][s] = mfma(uf[v], zf, acc[v0 + v][s], T{});
              }
              continue;
            }
            f32x4 d[kV] = {};
#pragma unroll
            for (int part = 0; part < kParts<T>; ++part) {
              const u32x4 zf = zs[(part * kBM + row) * 4 + c];
#pragma unroll
              for (int v = 0; v < kV; ++v) d[v] = mfma(uf[v], zf, d[v], T{});
            }
            const float f = r.zsc[row];
            const bool mine = row >= i && row < j;
#pragma unroll
            for (int v = 0; v < kV; ++v)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (!whole) d[v][e] = mine ? d[v][e] : 0.0f;
                acc[v0 + v][s][e] = __builtin_fmaf(d[v][e], f, acc[v0 + v][s][e]);
              }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  }
}

// Tile (row tile, token tile) of a workgroup.  Consecutive workgroups go to
// the XCDs in turn, so each XCD takes a run of tiles; a run goes over four
// row tiles at a time, then over the tokens.  So the 32 workgroups that an
// XCD runs at once share four tiles' rows and eight tiles' tokens in its L2.
__device__ __forceinline__ void tile_of(uint32_t row_tiles, uint32_t* tm, uint32_t* tn) {
  const uint32_t n = gridDim.x, run = n / 8, token_tiles = n / row_tiles;
  const uint32_t t = blockIdx.x < run * 8 ? (blockIdx.x % 8) * run + blockIdx.x / 8 : blockIdx.x;
  constexpr uint32_t kGroup = 4;
  const uint32_t g = t / (kGroup * token_tiles), in = t - g * kGroup * token_tiles;
  const uint32_t width = min(kGroup, row_tiles - g * kGroup);
  *tn = in / width;
  *tm = g * kGroup + in % width;
}

// A wave's LDS to store 16 rows of 16 kN tokens: rows shifted by four banks.
template <int kN>
constexpr int stored_floats() {
  return 16 * (kN * 16 + 4);
}

// The wave's results, 16 rows at a time through its own LDS `mine`, so that
// a row's tokens are stored side by side.
template <typename T, typename O, int kN, int kM, int kBM>
__device__ __forceinline__ void store_lines(const Args& a, const Rows<kBM>& tile, uint32_t rows,
                                           uint32_t v0, uint32_t s0, uint32_t tid,
                                           const f32x4 (&acc)[kN][kM], float* mine) {
  const uint32_t lane = tid & 63, col = lane & 15, q = lane >> 4;
  constexpr int kRow = kN * 16 + 4;
  constexpr int kE = 16 / (int)sizeof(O), kPer = kN * 16 / kE;  // elements, pieces of a row
#pragma unroll
  for (int s = 0; s < kM; ++s) {
#pragma unroll
    for (int i = 0; i < kN; ++i) *(f32x4*)(mine + col * kRow + i * 16 + q * 4) = acc[i][s];
    asm volatile("" ::: "memory");  // (a wave's LDS accesses are in order)
#pragma unroll 1
    for (int p = 0; p < (16 * kPer + 63) / 64; ++p) {
      const uint32_t at = p * 64 + lane, r = at / kPer, c = at % kPer * kE;
      if (16 * kPer < 64 && at >= 16 * kPer) break;
      const uint32_t row = (s0 + s) * 16 + r, tok = v0 + c;
      if (row < rows && tok < a.vocab) {
        const bool bad = tile.ad[row] >= 0 && (uint32_t)tile.ad[row] >= a.adapters;
        float y[kE];
#pragma unroll
        for (int e = 0; e < kE; ++e) y[e] = bad ? NAN : mine[r * kRow + c + e];
        O* out = (O*)a.out + (int64_t)tile.to[row] * a.out_stride + tok;
        const u32x4 o = from_float<O>(y);
        if (tok + kE <= a.vocab) store_vec(out, o);
        else store_part(out, (int)(a.vocab - tok), o);
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Few rows: a lane has four neighbouring tokens of a row, which it stores at
// once.
template <typename T, typename O, int kN, int kM, int kBM>
__device__ __forceinline__ void store_rows(const Args& a, const Rows<kBM>& tile, uint32_t rows,
                                           uint32_t v0, uint32_t s0, const f32x4 (&acc)[kN][kM]) {
  const uint32_t lane = threadIdx.x & 63, col = lane & 15, q = lane >> 4;
  struct __attribute__((packed, aligned(sizeof(O)))) Four {
    O e[4];
  };
#pragma unroll
  for (int s = 0; s < kM; ++s) {
    const uint32_t row = (s0 + s) * 16 + col;
    if (row < rows) {
      O* out = (O*)a.out + (int64_t)tile.to[row] * a.out_stride + v0 + q * 4;
      const bool bad = tile.ad[row] >= 0 && (uint32_t)tile.ad[row] >= a.adapters;
#pragma unroll
      for (int v = 0; v < kN; ++v) {
        Four o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.e[e] = (O)(bad ? NAN : acc[v][s][e]);
        const uint32_t tok = v0 + v * 16 + q * 4;
        if (tok + 4 <= a.vocab) {
          *(Four*)(out + v * 16) = o;
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tok + e < a.vocab) out[v * 16 + e] = o.e[e];
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
}

constexpr int kBK = 64;  // hidden columns of a step: a line of a row

// Any alignment: operands pass registers on their way to LDS, by loads that
// straddle lines, and no step is ahead (4096 x 32768 x 1024, 8 adapters of rank
// 16: 867 us, where logits_tile takes 343).
// Block: rows [64 m, ...) of the order by tokens [128 n,
// ...); wave w has tokens 32 w ... 32 w + 31 of them, and all rows.
constexpr int kBM = 64, kBN = 128, kThreads = 256;
template <typename T, typename O>
__global__ void __launch_bounds__(kThreads) logits_product(Args a) {
  __shared__ u32x4 ws[kBN][kBK / 8];  // columns by 8, exchanged within a row
  __shared__ u32x4 xs[kBM][kBK / 8];
  __shared__ u32x4 zs[kBM * kParts<T> * 4];
  __shared__ Rows<kBM> r;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, col = lane & 15, q = lane >> 4;
  uint32_t tm, tn;
  tile_of(a.row_tiles, &tm, &tn);
  const uint32_t m0 = tm * kBM, n0 = tn * kBN;
  const uint32_t rows = min((uint32_t)kBM, a.rows - m0);
  read_rows(a, r, m0, rows);
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
      xr[i] = load_k((const T*)a.x + (int64_t)r.to[at / 8] * a.x_stride, k0 + at % 8 * 8, a.hidden);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBN * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid, row = at / 8;
      ws[row][(at % 8) ^ (row & 7)] = wr[i];
    }
#pragma unroll
    for (int i = 0; i < kBM * kBK / 8 / kThreads; ++i) {
      const uint32_t at = i * kThreads + tid, row = at / 8;
      xs[row][(at % 8) ^ (row & 7)] = xr[i];
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
  u32x4 none[2 * kBN * 4 / kThreads];
  add_adapters<T, kBM, kBN, 2, kBM / 16, kThreads, 2, 1, false>(
      a, r, m0, rows, n0, wave * 2, 0, tid, zs, &ws[0][0], nullptr, nullptr, none, acc);
  store_rows<T, O, 2, kBM / 16>(a, r, rows, n0 + wave * 32, 0, acc);
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
  static constexpr bool Ahead = M * N < 16;  // registers for ups loaded before the product
};

// The same from a 32-bit offset (a lane's and the wave's) of a buffer.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t whole_buffer(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)0xFFFFFFFFu, 0x00027000);
}
__device__ __forceinline__ void copy_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t lane, uint32_t wave,
                                            void* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16,
                                           (int)lane, (int)wave, 0, 0);
}

template <typename T, typename O, typename S>
__global__ void __launch_bounds__(S::Threads) logits_staged(Args a) {
  // (an array a stage: the compiler tells their copies and reads apart)
  __shared__ u32x4 st0[(S::BM + S::BN) * 8], st1[(S::BM + S::BN) * 8];
  __shared__ u32x4 st2[S::Stages > 2 ? (S::BM + S::BN) * 8 : 1];
  __shared__ u32x4 st3[S::Stages > 3 ? (S::BM + S::BN) * 8 : 1];
  __shared__ Rows<S::BM> r;
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t wm = wave % S::WM, wn = wave / S::WM;
  uint32_t tm, tn;
  tile_of(a.row_tiles, &tm, &tn);
  const uint32_t m0 = tm * S::BM, n0 = tn * S::BN;
  const uint32_t rows = min((uint32_t)S::BM, a.rows - m0);
  read_rows(a, r, m0, rows);

  constexpr uint32_t kUp = (S::BM + S::BN) * 8 / (S::BN * 4);  // runs' ups of a stage
  u32x4 ahead[kUp * (S::Stages - 1) * S::BN * 4 / S::Threads];
  if constexpr (S::Ahead)
    load_ups<T, S::BM, S::BN, S::Threads>(a, r, n0, tid, 0, min(r.runs, kUp * (S::Stages - 1)), 0, 0,
                                          ahead);
  // this thread's part of each copy: a row and one of its columns
  const T* wp[S::CW];
  const T* xp[S::CX];
  uint32_t wk[S::CW], xk[S::CX];
#pragma unroll
  for (int i = 0; i < S::CW; ++i) {
    const uint32_t at = i * S::Threads + tid, row = at / 8;
    wk[i] = ((at ^ row) & 7) * 8;
    wp[i] = (const T*)a.weight + (int64_t)min(n0 + row, a.vocab - 1) * a.weight_stride;
  }
#pragma unroll
  for (int i = 0; i < S::CX; ++i) {
    const uint32_t at = (i * S::WM * S::WN + wave) * S::XLanes + lane;
    const uint32_t row = min(at / 8, S::BM - 1u);
    xk[i] = ((at ^ row) & 7) * 8;
    xp[i] = (const T*)a.x + (int64_t)r.to[row] * a.x_stride;
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
      for (int i = 0; i < S::N; ++i) wf[i] = ws[i * 16 * 8 + c];
#pragma unroll
      for (int j = 0; j < S::M; ++j) xf[j] = xs[j * 16 * 8 + c];
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
  static_assert(S::BM * kParts<T> * 4 <= (S::BM + S::BN) * 8, "z fits a stage");
  add_adapters<T, S::BM, S::BN, S::N, S::M, S::Threads, kUp, S::Stages - 1, S::Ahead>(
      a, r, m0, rows, n0, wn * S::N, wm * S::M, tid, st1, st0, st2, st3, ahead, acc);
  if constexpr (S::M <= 2) {
    store_rows<T, O, S::N, S::M>(a, r, rows, n0 + wn * S::N * 16, wm * S::M, acc);
  } else {
    __syncthreads();
    constexpr uint32_t kHeld = (S::BM + S::BN) * 8 * 16 / (stored_floats<S::N>() * 4);
    static_assert(S::WM * S::WN <= S::Stages * kHeld, "fits the stages");
    store_lines<T, O, S::N, S::M>(a, r, rows, n0 + wn * S::N * 16, wm * S::M, tid, acc,
                                  (float*)(wave < kHeld ? st0 : wave < 2 * kHeld ? st1 : wave < 3 * kHeld ? st2 : st3) +
                                      wave % kHeld * stored_floats<S::N>());
  }
}

// Many rows, where the matrix cores are the bound: tiles of 16 kBMs rows by 16
// kBNs tokens, steps of a line (64 hidden columns) in two LDS stages.  The
// operands of a half step are read from LDS during the matrix instructions
// of the half before, so that past a barrier there is work at once.  4096 x
// 32768 x 1024 bf16, 8 adapters of rank 16: 343 us (as tiles of 256 x 128 of
// logits_staged: 451); without adapters 304, 0.90 PFLOP/s, where the clock
// under load is the bound.
template <int kBMs, int kBNs, int kWM, int kWN>
struct TileShape {
  static constexpr int BM = 16 * kBMs, BN = 16 * kBNs, Threads = 64 * kWM * kWN;
  static constexpr int M = kBMs / kWM, N = kBNs / kWN, WM = kWM, WN = kWN;
  static constexpr int CW = BN * 8 / Threads, CX = BM * 8 / Threads;
};

template <typename T, typename O, typename S>
__global__ void __launch_bounds__(S::Threads) logits_tile(Args a) {
  constexpr int kStage = (S::BM + S::BN) * 8;
  __shared__ u32x4 st0[kStage], st1[kStage];
  __shared__ Rows<S::BM> r;
  const uint32_t tid = threadIdx.x, lane = tid & 63, col = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t wm = wave % S::WM, wn = wave / S::WM;
  uint32_t tm, tn;
  tile_of(a.row_tiles, &tm, &tn);
  // (the last token tile ends with the vocabulary, on some of the tokens of
  // the one before it)
  const uint32_t m0 = tm * S::BM, n0 = min(tn * S::BN, a.vocab - S::BN);
  const uint32_t rows = min((uint32_t)S::BM, a.rows - m0);
  read_rows(a, r, m0, rows);
  // A row is a line of eight columns, exchanged by the row's number.  Offsets
  // from the operands' uniform addresses, which advance by steps.
  const uint32_t kc = ((tid & 7) ^ (tid >> 3 & 7)) * 8;
  const uint32_t woff = (tid / 8 * (uint32_t)a.weight_stride + kc) * 2;
  const uint32_t wnext = S::Threads / 8 * 2 * (uint32_t)a.weight_stride;  // to the next copy's row
  uint32_t xoff[S::CX];
#pragma unroll
  for (int i = 0; i < S::CX; ++i)
    xoff[i] = ((uint32_t)r.to[(i * S::Threads + tid) / 8] * (uint32_t)a.x_stride + kc) * 2;
  const __amdgpu_buffer_rsrc_t wb = whole_buffer((const T*)a.weight + (int64_t)n0 * a.weight_stride);
  const __amdgpu_buffer_rsrc_t xb = whole_buffer(a.x);
  const uint32_t steps = a.hidden / kBK;
  const auto copy = [&](u32x4* st, uint32_t i) {
    const uint32_t k = min(i, steps - 1) * (kBK * 2);  // (past the end: again, unused)
#pragma unroll
    for (int c = 0; c < S::CW; ++c)
      copy_to_lds(wb, woff, k + c * wnext, st + c * S::Threads + wave * 64);
#pragma unroll
    for (int c = 0; c < S::CX; ++c)
      copy_to_lds(xb, xoff[c], k, st + S::BN * 8 + c * S::Threads + wave * 64);
  };
  // byte addresses in a stage, of either half (hidden from the compiler, so
  // that it adds the constants in the instructions)
  uint32_t w0 = ((wn * S::N * 16 + col) * 8 + (q ^ (col & 7))) * 16, w1 = w0 ^ 64;
  uint32_t xa0 = ((wm * S::M * 16 + col) * 8 + (q ^ (col & 7))) * 16, xa1 = xa0 ^ 64;
  asm volatile("" : "+v"(w0), "+v"(w1), "+v"(xa0), "+v"(xa1));
  const auto at = [](const u32x4* st, uint32_t bytes, int more) {
    return *(const u32x4*)((const char*)st + bytes + more);
  };
  f32x4 acc[S::N][S::M] = {};
  constexpr int kCopies = S::CW + S::CX;
  // Half a step: the products of w and x, while w and `ahead` take the next
  // half's operands, at `wat` and `xat` of the stage `next`.  A token operand's
  // register is free when its products are issued; the rows' have two sets.
  u32x4 w[S::N], x0[S::M], x1[S::M];
  const auto half = [&](const u32x4 (&x)[S::M], u32x4 (&ahead)[S::M], const u32x4* next, uint32_t wat, uint32_t xat) {
#pragma unroll
    for (int v = 0; v < S::N; ++v) {
#pragma unroll
      for (int j = 0; j < S::M; ++j) acc[v][j] = mfma(w[v], x[j], acc[v][j], T{});
      w[v] = at(next, wat, v * 2048);
      if (v < S::M) ahead[v] = at(next + S::BN * 8, xat, v * 2048);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = S::N; j < S::M; ++j) ahead[j] = at(next + S::BN * 8, xat, j * 2048);
  };
  // Step i: w and x0 hold its first half's operands.  At the barrier all of
  // the step has been read, and the next is there.
  const auto step = [&](uint32_t i, u32x4* st, const u32x4* next) {
    half(x0, x1, st, w1, xa1);
    wait_copies<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    copy(st, i + 2);
    half(x1, x0, next, w0, xa0);
  };
  const auto begin = [&](u32x4* first, u32x4* second) {
    copy(first, 0);
    copy(second, 1);
    wait_copies<kCopies>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int v = 0; v < S::N; ++v) w[v] = at(first, w0, v * 2048);
#pragma unroll
    for (int j = 0; j < S::M; ++j) x0[j] = at(first + S::BN * 8, xa0, j * 2048);
  };
  uint32_t i = steps & 1;
  if (i) {  // an odd step in front
    begin(st1, st0);
    step(0, st1, st0);
  } else {
    begin(st0, st1);
  }
  for (; i < steps; i += 2) {
    step(i, st0, st1);
    step(i + 1, st1, st0);
  }
  wait_copies<0>();
  // (numbers of the thread anew, so that none of what follows is computed
  // ahead and takes the loop's registers: the accumulators and operands are
  // 192 of 256)
  uint32_t after = threadIdx.x;
  asm volatile("" : "+v"(after));
  const uint32_t wave_after = (uint32_t)__builtin_amdgcn_readfirstlane((int)(after >> 6));
  const uint32_t wm_after = wave_after % S::WM, wn_after = wave_after / S::WM;
  constexpr uint32_t kUp = kStage / (S::BN * 4);  // runs' ups of a stage
  static_assert(S::BM * kParts<T> * 4 <= kStage, "z fits a stage");
  u32x4 none[kUp * S::BN * 4 / S::Threads];
  // (a block of its own: without the branch the accumulators change their
  // registers here by way of memory)
  if (__builtin_amdgcn_readfirstlane((int)r.runs) != 0)
    add_adapters<T, S::BM, S::BN, S::N, S::M, S::Threads, kUp, 1, false>(
        a, r, m0, rows, n0, wn_after * S::N, wm_after * S::M, after, st1, st0, nullptr, nullptr, none, acc);
  __syncthreads();
  constexpr uint32_t kHeld = kStage * 16 / (stored_floats<S::N>() * 4);  // waves' parts of a stage
  static_assert(S::WM * S::WN <= 2 * kHeld, "fits the stages");
  store_lines<T, O, S::N, S::M>(a, r, rows, n0 + wn_after * S::N * 16, wm_after * S::M, after, acc,
                                (float*)(wave_after < kHeld ? st0 : st1) +
                                    wave_after % kHeld * stored_floats<S::N>());
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
hipError_t launch_tile(Args a, hipStream_t s) {
  a.row_tiles = (a.rows + S::BM - 1) / S::BM;
  const uint32_t tiles = (a.vocab + S::BN - 1) / S::BN;
  return start(logits_tile<T, O, S>, tiles * a.row_tiles, S::Threads, s, a);
}

template <typename T, typename O, typename S>
hipError_t launch_staged(Args a, hipStream_t s) {
  a.row_tiles = (a.rows + S::BM - 1) / S::BM;
  const uint32_t tiles = (a.vocab + S::BN - 1) / S::BN;
  return start(logits_staged<T, O, S>, tiles * a.row_tiles, S::Threads, s, a);
}

bool whole_vectors(const void* p, int64_t stride) {
  return (uintptr_t)p % 16 == 0 && stride % 8 == 0;
}

template <typename T, typename O>
hipError_t launch(Args a, hipStream_t s) {
  hipError_t e = a.rows > 16 ? start(logits_order, 1, 1024, s, a) : hipSuccess;
  if (e != hipSuccess) return e;
  const uint32_t blocks = (a.rows + 15) / 16;
  a.shares = std::min(16u, std::max(1u, kCUs / blocks));
  e = start(logits_shrink<T>, blocks * a.shares, kShrinkT, s, a);
  if (e != hipSuccess) return e;
  if (a.hidden % 8 == 0 && whole_vectors(a.x, a.x_stride) &&
      whole_vectors(a.weight, a.weight_stride)) {
    // Up to 96 rows the weights' stream is the bound: two or more workgroups
    // on a CU, some in their adapters' turns while others stream (84 x 262144
    // x 1024, 6 adapters of rank 12: 174 us; with tiles of 256 tokens and
    // three stages, one workgroup on a CU: 196).  Up to 16 rows, tiles of 64
    // tokens where those make one round of them, three a CU (8 x 49152 x 512:
    // 24.9 us to 27.3 with 128 tokens; 8 x 65536 x 512: 38.6 to 34.6).
    if (a.rows <= 16 && a.vocab <= 48 * 1024) return launch_staged<T, O, Shape<1, 4, 1, 4, 4>>(a, s);
    if (a.rows <= 16) return launch_staged<T, O, Shape<1, 8, 1, 4, 2>>(a, s);
    if (a.rows <= 32) return launch_staged<T, O, Shape<2, 8, 1, 8, 2>>(a, s);
    if (a.rows <= 64) return launch_staged<T, O, Shape<4, 8, 1, 8, 2>>(a, s);
    if (a.rows <= 96) return launch_staged<T, O, Shape<6, 8, 1, 8, 2>>(a, s);
    if (a.rows <= 128) return launch_staged<T, O, Shape<8, 16, 1, 8, 3>>(a, s);
    // Up to 128 rows one row tile, so that w is read once (112 x 262144 x
    // 1024: 206 us, by logits_tile 238); above, logits_tile (144 rows: 246,
    // by logits_staged 287) where 32-bit offsets reach a tile's operands.
    // (the end of the last row counts: rows may be less than their own length
    // apart)
    if (a.hidden % 64 == 0 && a.x_stride >= 0 && a.weight_stride >= 0 &&
        (a.rows - 1) * (uint64_t)a.x_stride + a.hidden < 1ull << 31 &&
        a.weight_stride < 1ll << 22 && a.vocab >= 256)
      return launch_tile<T, O, TileShape<16, 16, 2, 4>>(a, s);
    return launch_staged<T, O, Shape<16, 8, 2, 8, 2>>(a, s);
  }
  a.row_tiles = (a.rows + kBM - 1) / kBM;
  const uint32_t tiles = (a.vocab + kBN - 1) / kBN;
  return start(logits_product<T, O>, tiles * a.row_tiles, kThreads, s, a);
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
  a.whole_up = q.rank % 8 == 0 && whole_vectors(q.up, q.up_stride[0]) && q.up_stride[1] % 8 == 0;
  if (q.dtype == FT_BF16)
    return q.out_dtype == FT_F32 ? launch<__bf16, float>(a, s) : launch<__bf16, __bf16>(a, s);
  return q.out_dtype == FT_F32 ? launch<_Float16, float>(a, s)
                               : launch<_Float16, _Float16>(a, s);
}

}  // namespace fto
