// packed_logits.hip -- the vocabulary's table in 4 bits with a scale for each
// group of columns, and logits by it.
//
//   y[t, v] = sum_g s[v, g] sum_{h in g} x[t, h] (c[v, h] - 8)
//
// The layout is the matrix instruction's own operand: of a tile of 16 tokens
// and a chunk of 128 columns a lane's 16 bytes are its four operands of 8
// columns, so a wave streams 1 KB at a time from memory to registers.  Four
// bits become the halves of 32-bit words that hold 1024 + c (the code in the
// low bits of a float16 of that size), less 1032: whole numbers that float16
// holds, no rounding.  x is in float16 too: bfloat16 rows are divided by a
// power of two that brings their largest to [2^14, 2^15), which leaves
// everything down to 2^-32 of it exact.
//
// Bound by the weights' stream for up to 16 rows (2,200,000 x 512, groups of 64,
// float32 logits: 134-164 us, 4.5-5.5 TB/s; adapter_logits reads four times as
// much and takes 481), by the unpacking and the reads of x from LDS for more (84
// rows x 100,003 x 1,024: 34-37 us, of which the bytes take 14), by its one launch
// for a single request (8 rows x 32,768 x 512: 7.0 us on the device).
#include <algorithm>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// 16 x 16 tile by 32: lane l gives 8 of row l % 16 of either operand, from
// column 8 (l / 16) on; it gets rows 4 (l / 16) ... + 3 of column l % 16.

// Eight codes of a word, less 8.  The masks are registers' (unknown to the
// compiler), so that a mask and the bits of 1024 are one instruction: nine a
// word.
struct Masks {
  uint32_t low = 0x000F000Fu, high = 0x00F000F0u, base = 0x64006400u;
  __device__ __forceinline__ Masks() { asm volatile("" : "+v"(low), "+v"(high), "+v"(base)); }
};
__device__ __forceinline__ u32x4 unpack(uint32_t w, const Masks& k) {
  const f16x2 low = {(_Float16)1032.0f, (_Float16)1032.0f};
  const f16x2 sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
  const f16x2 high = {(_Float16)-72.0f, (_Float16)-72.0f};
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t v = w >> (8 * i);
    const f16x2 a = __builtin_bit_cast(f16x2, (v & k.low) | k.base);
    const f16x2 b = __builtin_bit_cast(f16x2, (v & k.high) | k.base);  // 1024 + 16 c
    r[2 * i] = __builtin_bit_cast(uint32_t, a - low);
    r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(b, sixteenth, high));
  }
  return r;
}

// --- pack_weight ------------------------------------------------------------

struct PackArgs {
  const void* weight;
  int64_t stride;
  uint32_t hidden, vocab, chunks;
  void* packed;
  void* scales;
};

// The element of larger magnitude, the first of equals; NaN and infinities
// make `odd`.
struct Largest {
  float value;
  bool odd;
};
__device__ __forceinline__ Largest first_largest(Largest a, Largest b) {
  return Largest{fabsf(b.value) > fabsf(a.value) ? b.value : a.value, a.odd || b.odd};
}

// A wave a tile and chunk.  Bound by the table's one read.
template <typename T, int kPer>
__global__ void __launch_bounds__(256) pack_table(PackArgs a) {
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const uint64_t at = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const uint32_t tiles = (a.vocab + 15) / 16;
  if (at >= (uint64_t)tiles * a.chunks) return;
  const uint32_t tile = (uint32_t)(at / a.chunks), chunk = (uint32_t)(at % a.chunks);
  const uint32_t token = tile * 16 + n;
  const T* row = (const T*)a.weight + (int64_t)min(token, a.vocab - 1) * a.stride;
  float w[4][8];
  Largest big[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    to_float<T>(load_row_vec(row, chunk * 128 + i * 32 + q * 8, a.hidden, (T)0.0f), w[i]);
    big[i] = Largest{0.0f, false};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (token >= a.vocab) w[i][j] = 0.0f;
      big[i] = first_largest(big[i], Largest{w[i][j], !(fabsf(w[i][j]) < INFINITY)});
    }
#pragma unroll
    for (int d = 16; d < 64; d *= 2) {  // the lane with the lower columns first
      const Largest other{__shfl_xor(big[i].value, d, 64), (bool)__shfl_xor((int)big[i].odd, d, 64)};
      big[i] = lane & d ? first_largest(other, big[i]) : first_largest(big[i], other);
    }
  }
  constexpr int kWords = 4 / kPer;
  union {
    u32x4 v;
    uint32_t w[4];
  } out;
  T scale[kPer];
#pragma unroll
  for (int g = 0; g < kPer; ++g) {
    Largest l = big[g * kWords];
#pragma unroll
    for (int i = 1; i < kWords; ++i) l = first_largest(l, big[g * kWords + i]);
    scale[g] = l.odd ? (T)NAN : (T)(l.value * -0.125f);
    const float s = (float)scale[g];
#pragma unroll
    for (int i = g * kWords; i < (g + 1) * kWords; ++i) {
      uint32_t word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float c = s == 0.0f || l.odd ? 0.0f : fminf(fmaxf(rintf(w[i][j] / s), -8.0f), 7.0f);
        word |= (uint32_t)((int)c + 8) << (4 * ((j >> 1) + 4 * (j & 1)));
      }
      out.w[i] = word;
    }
  }
  ((u32x4*)a.packed)[at * 64 + lane] = out.v;
  if (q == 0) {
    T* to = (T*)a.scales + (at * 16 + n) * kPer;
#pragma unroll
    for (int g = 0; g < kPer; ++g) to[g] = scale[g];
  }
}

template <typename T>
hipError_t launch_pack(const PackArgs& a, uint32_t group, hipStream_t s) {
  const uint64_t blocks = ((uint64_t)(a.vocab + 15) / 16 * a.chunks + 3) / 4;
  return group == 32   ? start(pack_table<T, 4>, blocks, 256, s, a)
         : group == 64 ? start(pack_table<T, 2>, blocks, 256, s, a)
                       : start(pack_table<T, 1>, blocks, 256, s, a);
}

// --- packed_logits ----------------------------------------------------------

struct Args {
  const void* x;
  int64_t x_stride, out_stride;
  uint32_t rows, hidden, vocab, chunks, row_tiles;
  const u32x4* packed;
  const void* scales;
  void* out;
  // workspace
  u32x4* xs;      // [row tiles][4 chunks][64]: x as the matrix operand
  float* xscale;  // [rows to whole 16s]: power of two that x was divided by
};

// A wave puts a row's operands to `to`, 64 vectors from step to step and 16
// from quarter to quarter, zero where it is none; returns the power of two
// that it was divided by.
template <typename T>
__device__ __forceinline__ float put_row(const T* row, uint32_t hidden, uint32_t steps, uint32_t lane, bool any,
                                         u32x4* to) {
  int e = 0;
  if (!__is_same(T, _Float16)) {
    float big = 0.0f;
    for (uint32_t k = lane * 8; k < hidden; k += 512) {
      float v[8];
      to_float<T>(load_row_vec(row, k, hidden, (T)0.0f), v);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (fabsf(v[i]) < INFINITY) big = fmaxf(big, fabsf(v[i]));
    }
    big = wave_max(big);
    if (big > 0.0f) (void)frexpf(big, &e), e -= 15;
  }
  for (uint32_t k = lane; k < steps * 4; k += 64) {
    u32x4 v{};
    if (any) v = load_row_vec(row, k * 8, hidden, (T)0.0f);
    if (!__is_same(T, _Float16)) {
      float f[8];
      to_float<T>(v, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = ldexpf(f[i], -e);
      v = from_float<_Float16>(f);
    }
    to[(k >> 2) * 64 + (k & 3) * 16] = v;
  }
  return ldexpf(1.0f, e);
}

// A wave a row.
template <typename T>
__global__ void __launch_bounds__(256) packed_rows(Args a) {
  const uint32_t lane = threadIdx.x & 63, r = blockIdx.x * 4 + (threadIdx.x >> 6), steps = a.chunks * 4;
  if (r >= a.row_tiles * 16) return;
  const T* row = (const T*)a.x + (int64_t)min(r, a.rows - 1) * a.x_stride;
  const float down = put_row<T>(row, a.hidden, steps, lane, r < a.rows,
                                a.xs + (uint64_t)(r >> 4) * steps * 64 + (r & 15));
  if (lane == 0) a.xscale[r] = down;
}

// The scales of a chunk's groups for this lane's token.
template <typename T, int kPer>
struct alignas(2 * kPer) Scales {
  T s[kPer];
};

// Adds chunk c's products to the sums of kM row tiles: a group's product in
// whole numbers, then times its scale.  x(m, i): row tile m's operand of step i.
template <typename T, int kPer, int kM, typename X>
__device__ __forceinline__ void add_chunk(const Masks& masks, u32x4 w, Scales<T, kPer> sc, uint32_t c, uint32_t hidden,
                                          f32x4 (&acc)[kM], X&& x) {
  constexpr int kWords = 4 / kPer;
#pragma unroll
  for (int g = 0; g < kPer; ++g) {
    // (a group past the columns: whatever its scale)
    const float s = c * 128 + g * (128 / kPer) < hidden ? (float)sc.s[g] : 0.0f;
    f32x4 part[kM] = {};
#pragma unroll
    for (int i = g * kWords; i < (g + 1) * kWords; ++i) {
      const u32x4 wf = unpack(w[i], masks);
#pragma unroll
      for (int m = 0; m < kM; ++m) part[m] = mfma(x(m, i), wf, part[m]);
    }
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][e] = __builtin_fmaf(part[m][e], s, acc[m][e]);
  }
}

// Any number of columns: x's operands from memory (they stay in the caches).
// A wave a tile of 16 tokens, kM row tiles at a time.
template <typename T, typename O, int kPer, int kM>
__global__ void __launch_bounds__(256) packed_direct(Args a) {
  const uint32_t lane = threadIdx.x & 63, n = lane & 15, q = lane >> 4;
  const uint32_t tile = blockIdx.x * 4 + (threadIdx.x >> 6), tiles = (a.vocab + 15) / 16;
  if (tile >= tiles) return;
  const uint32_t steps = a.chunks * 4, token = tile * 16 + n;
  const Masks masks;
  for (uint32_t m0 = 0; m0 < a.row_tiles; m0 += kM) {
    f32x4 acc[kM] = {};
    for (uint32_t c = 0; c < a.chunks; ++c) {
      const uint64_t at = (uint64_t)tile * a.chunks + c;
      const u32x4 w = a.packed[at * 64 + lane];
      const Scales<T, kPer> sc = ((const Scales<T, kPer>*)a.scales)[at * 16 + n];
      add_chunk<T, kPer, kM>(masks, w, sc, c, a.hidden, acc, [&](int m, int i) {
        return a.xs[((uint64_t)min(m0 + m, a.row_tiles - 1) * steps + c * 4 + i) * 64 + lane];
      });
    }
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t row = (m0 + m) * 16 + q * 4 + e;
        if (row < a.rows && token < a.vocab)
          ((O*)a.out)[(int64_t)row * a.out_stride + token] = (O)(acc[m][e] * a.xscale[row]);
      }
  }
}

// Up to kHeld vectors of x's operands in LDS, kM row tiles of them: a
// workgroup a CU, whose waves take tiles of 16 tokens in turn, with the loads
// of kAhead chunks in flight.  Past the first barrier the waves run by
// themselves.  More rows than LDS holds go to other workgroups, beside these on
// the same XCD, whose L2 then has the weights.
constexpr uint32_t kHeld = 128 * 1024 / 16, kCUs = 256;
constexpr int kStreamT = 1024, kAhead = 4;

// kOnce: one group of rows, so that the weights need not stay in the caches
// (16 x 2,200,000 x 512: 134 us, else 161; two groups, 84 x 100,003 x 1,024: 40
// us, else 38.5).
template <typename T, typename O, int kPer, int kM, bool kOnce>
__global__ void __launch_bounds__(kStreamT) packed_stream(Args a) {
  __shared__ u32x4 xs[kHeld];
  __shared__ float xscale[kM * 16];
  const uint32_t tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  const uint32_t groups = (a.row_tiles + kM - 1) / kM, workers = gridDim.x / groups;
  // (workgroup b goes to XCD b % 8)
  const uint32_t eight = blockIdx.x / 8, whole = gridDim.x / (8 * groups) * 8 * groups;
  const uint32_t group = blockIdx.x < whole ? eight % groups : (blockIdx.x - whole) % groups;
  const uint32_t worker = blockIdx.x < whole ? eight / groups * 8 + blockIdx.x % 8
                                             : whole / groups + (blockIdx.x - whole) / groups;
  const uint32_t r0 = group * kM * 16, rows = min((uint32_t)kM * 16, a.rows - r0);
  const uint32_t tiles = (a.vocab + 15) / 16, steps = a.chunks * 4;
  const uint32_t first = worker * 16 + wave, stride = workers * 16;

  // the loads run ahead of the products: chunk ac of tile at
  uint32_t at = first, ac = 0;
  u32x4 w[kAhead];
  Scales<T, kPer> sc[kAhead];
  const auto load = [&](int u) {
    const uint64_t place = (uint64_t)min(at, tiles - 1) * a.chunks + ac;
    w[u] = kOnce ? __builtin_nontemporal_load(a.packed + place * 64 + lane) : a.packed[place * 64 + lane];
    sc[u] = ((const Scales<T, kPer>*)a.scales)[place * 16 + n];
    if (++ac == a.chunks) {
      ac = 0;
      at += stride;
    }
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(u);

  for (uint32_t r = wave; r < kM * 16; r += kStreamT / 64) {
    const T* row = (const T*)a.x + (int64_t)(r0 + min(r, rows - 1)) * a.x_stride;
    const float down = put_row<T>(row, a.hidden, steps, lane, r < rows, xs + (r >> 4) * steps * 64 + (r & 15));
    if (lane == 0) xscale[r] = down;
  }
  __syncthreads();

  const Masks masks;
  f32x4 acc[kM] = {};
  uint32_t tile = first, c = 0;
  while (tile < tiles) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (tile >= tiles) break;
      add_chunk<T, kPer, kM>(masks, w[u], sc[u], c, a.hidden, acc,
                             [&](int m, int i) { return xs[(m * steps + c * 4 + i) * 64 + lane]; });
      load(u);
      if (++c < a.chunks) continue;
      const uint32_t token = tile * 16 + n;
#pragma unroll
      for (int m = 0; m < kM; ++m) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t row = m * 16 + q * 4 + e;
          if (row < rows && token < a.vocab)
            ((O*)a.out)[(int64_t)(r0 + row) * a.out_stride + token] = (O)(acc[m][e] * xscale[row]);
        }
        acc[m] = f32x4{};
      }
      c = 0;
      tile += stride;
    }
  }
}

// Row tiles whose operands LDS holds; 0: not even one's.
uint32_t held_tiles(uint32_t chunks) { return std::min<uint32_t>(4, kHeld / (chunks * 256)); }

struct Plan {
  uint64_t xs, xscale, bytes;
};
Plan plan(const ft_packed_logits_args& a) {
  Plan p{};
  if (held_tiles((a.hidden + 127) / 128)) return p;
  Arena ar;
  const uint64_t rows = round_up(a.rows, 16);
  p.xs = ar.take(rows * round_up(a.hidden, 128) * 2);
  p.xscale = ar.take(rows * 4);
  p.bytes = ar.used;
  return p;
}

template <typename T, typename O, int kPer, bool kOnce>
hipError_t launch_stream(const Args& a, uint32_t each, uint64_t blocks, hipStream_t s) {
  return each == 1   ? start(packed_stream<T, O, kPer, 1, kOnce>, blocks, kStreamT, s, a)
         : each == 2 ? start(packed_stream<T, O, kPer, 2, kOnce>, blocks, kStreamT, s, a)
         : each == 3 ? start(packed_stream<T, O, kPer, 3, kOnce>, blocks, kStreamT, s, a)
                     : start(packed_stream<T, O, kPer, 4, kOnce>, blocks, kStreamT, s, a);
}

template <typename T, typename O, int kPer>
hipError_t launch(const Args& a, hipStream_t s) {
  const uint32_t tiles = (a.vocab + 15) / 16;
  if (const uint32_t held = held_tiles(a.chunks)) {
    const uint32_t groups = (a.row_tiles + held - 1) / held, each = (a.row_tiles + groups - 1) / groups;
    const uint32_t used = (a.row_tiles + each - 1) / each;
    const uint64_t blocks = (uint64_t)used * std::max(1u, std::min(kCUs / used, (tiles + 15) / 16));
    return used == 1 ? launch_stream<T, O, kPer, true>(a, each, blocks, s)
                     : launch_stream<T, O, kPer, false>(a, each, blocks, s);
  }
  const hipError_t e = start(packed_rows<T>, (a.row_tiles * 16 + 3) / 4, 256, s, a);
  if (e != hipSuccess) return e;
  return start(packed_direct<T, O, kPer, 4>, (tiles + 3) / 4, 256, s, a);
}
template <typename T, typename O>
hipError_t launch(const Args& a, uint32_t group, hipStream_t s) {
  return group == 32   ? launch<T, O, 4>(a, s)
         : group == 64 ? launch<T, O, 2>(a, s)
                       : launch<T, O, 1>(a, s);
}

}  // namespace

uint64_t pack_weight_workspace(const ft_pack_weight_args&) { return 0; }

hipError_t launch_pack_weight(const ft_pack_weight_args& q, uint8_t*, hipStream_t s) {
  const PackArgs a{q.weight, q.weight_stride, q.hidden, q.vocab, (q.hidden + 127) / 128, q.packed,
                   q.scales};
  return q.dtype == FT_BF16 ? launch_pack<__bf16>(a, q.group, s)
                            : launch_pack<_Float16>(a, q.group, s);
}

uint64_t packed_logits_workspace(const ft_packed_logits_args& a) { return plan(a).bytes; }

hipError_t launch_packed_logits(const ft_packed_logits_args& q, uint8_t* ws, hipStream_t s) {
  if (q.rows == 0) return hipSuccess;
  const Plan p = plan(q);
  Args a{};
  a.x = q.x;
  a.x_stride = q.x_stride;
  a.out_stride = q.out_stride;
  a.rows = (uint32_t)q.rows;
  a.hidden = q.hidden;
  a.vocab = q.vocab;
  a.chunks = (q.hidden + 127) / 128;
  a.row_tiles = (a.rows + 15) / 16;
  a.packed = (const u32x4*)q.packed;
  a.scales = q.scales;
  a.out = q.out;
  a.xs = (u32x4*)(ws + p.xs);
  a.xscale = (float*)(ws + p.xscale);
  if (q.dtype == FT_BF16)
    return q.out_dtype == FT_F32 ? launch<__bf16, float>(a, q.group, s)
                                 : launch<__bf16, __bf16>(a, q.group, s);
  return q.out_dtype == FT_F32 ? launch<_Float16, float>(a, q.group, s)
                               : launch<_Float16, _Float16>(a, q.group, s);
}

}  // namespace fto
