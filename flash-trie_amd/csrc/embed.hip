// embed.hip -- rows of the vocabulary's table for the tokens of keys, and the
// table's gradient.
//
//   y[n] = scale table[tok[n]];   dtable[v] = scale sum over n with tok[n] = v of g[n]
//
// The gradient's tokens are sorted with their positions (stable, by digits of
// up to 9 bits), so that a token's rows are added in the order of its
// positions, in 32 bits: a result depends on no order of workgroups.  A wave
// adds the rows of kRun sorted positions; a token that goes on past them
// leaves parts, which one workgroup joins in order.  The tokens that do not
// occur get their zeros from workgroups beside those that sort.
//
// Bound by memory: 128,000 tokens x 512 bf16 are looked up in 30-38 us (6.2 TB/s
// counting each row once); their gradient in a table of 262,144 x 1,024 takes 163
// us, where a trace of one table again and again has 147: zeros and sorting 100 (537
// MB at 5.4 TB/s; sorting alone would take some 60 in its six launches), sums 41,
// parts 7.
#include <algorithm>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

// --- embed ------------------------------------------------------------------

struct LookupArgs {
  const int32_t* tokens;
  const int32_t* lengths;
  const void* table;
  int64_t table_stride;
  void* out;
  uint32_t count;  // of tokens
  uint32_t steps, hidden, vocab, panels;
  float scale;
};

// A wave kTokens tokens and 64 vectors of their rows.
constexpr int kTokens = 4;
template <typename T>
__global__ void __launch_bounds__(256) embed_rows(LookupArgs a) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t n0 = (blockIdx.x / a.panels * 4 + wave) * kTokens;
  const uint32_t e = (blockIdx.x % a.panels * 64 + lane) * kVec<T>;
  if (n0 >= a.count || e >= a.hidden) return;
  int32_t tok[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    const uint32_t n = min(n0 + i, a.count - 1);
    tok[i] = a.tokens[n];
    if (a.lengths && (int64_t)(n % a.steps) >= (int64_t)a.lengths[n / a.steps]) tok[i] = -1;
  }
  u32x4 v[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    v[i] = u32x4{};
    if (tok[i] >= 0 && (uint32_t)tok[i] < a.vocab)
      v[i] = load_row_vec((const T*)a.table + (int64_t)tok[i] * a.table_stride, e, a.hidden, (T)0.0f);
  }
#pragma unroll
  for (int i = 0; i < kTokens; ++i) {
    if (n0 + i >= a.count) break;
    float f[kVec<T>];
    to_float<T>(v[i], f);
#pragma unroll
    for (int k = 0; k < kVec<T>; ++k) {
      // (a token without a row: 0, also for an infinite scale)
      f[k] = tok[i] < 0 ? 0.0f : (uint32_t)tok[i] < a.vocab ? f[k] * a.scale : NAN;
    }
    T* out = (T*)a.out + (uint64_t)(n0 + i) * a.hidden + e;
    if (e + kVec<T> <= a.hidden) store_vec(out, from_float<T>(f));
    else store_part(out, (int)(a.hidden - e), from_float<T>(f));
  }
}

// --- embed_grad -------------------------------------------------------------

constexpr uint32_t kSortT = 1024, kBins = 512;
constexpr uint32_t kSmall = 2048;      // positions that one workgroup sorts in LDS
constexpr uint32_t kSortBlocks = 64;   // workgroups that sort more

struct GradArgs {
  const int32_t* tokens;
  const int32_t* lengths;
  const void* grad;
  int64_t grad_stride, dtable_stride;
  void* dtable;
  uint32_t count, steps, hidden, vocab, panels, runs;
  float scale;
  int add;
  // sorting
  uint32_t* key[2];
  uint32_t* pos[2];
  uint32_t* hist;  // [blocks][kBins]
  uint32_t from, bits, passes, pass, blocks, each;  // pass: from key[from]; positions of a block
  // zeros: rows of `length` elements, `stride` apart; units of them by the
  // workgroups behind the sorting ones
  uint64_t zero_length;
  int64_t zero_stride;
  uint64_t zero_first, zero_last;  // units of this launch
  uint32_t zero_units;             // of a row
  // sums
  float* parts;  // [2][runs][hidden]
  const uint32_t* sorted_key;
  const uint32_t* sorted_pos;
};

__device__ __forceinline__ uint32_t key_of(const GradArgs& a, uint32_t n) {
  if (a.lengths && (int64_t)(n % a.steps) >= (int64_t)a.lengths[n / a.steps]) return a.vocab;
  const int32_t t = a.tokens[n];
  return t < 0 || (uint32_t)t >= a.vocab ? a.vocab : (uint32_t)t;
}

constexpr uint64_t kZeroUnit = kSortT * 16;  // vectors

template <typename T>
__device__ __forceinline__ void write_zeros(const GradArgs& a, uint32_t block, uint32_t blocks) {
  for (uint64_t u = a.zero_first + block; u < a.zero_last; u += blocks) {
    const uint64_t row = u / a.zero_units, at = (u - row * a.zero_units) * kZeroUnit;
    T* to = (T*)a.dtable + (int64_t)row * a.zero_stride;
    const uint64_t length = a.zero_length;
#pragma unroll 4
    for (uint64_t v = at + threadIdx.x; v < at + kZeroUnit; v += kSortT) {
      const uint64_t e = v * kVec<T>;
      if (e >= length) break;
      if (e + kVec<T> <= length) store_to<true>(to + e, u32x4{});
      else store_part(to + e, (int)(length - e), u32x4{});
    }
  }
}

// Places `n` items of a workgroup by digit, in order: the waves take runs of
// them, count their digits, and place 64 at a time.  base[d]: the first place
// of digit d for this workgroup; a barrier is in front of its reads.
struct Placer {
  uint32_t at[kBins][16];
  uint32_t waves[16];
};

__device__ __forceinline__ uint32_t exclusive_over_block(uint32_t v, uint32_t* waves) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t total, front = wave_scan(v, &total);
  if (lane == 0) waves[wave] = total;
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) front += waves[w];
  __syncthreads();
  return front;
}

template <typename Key, typename Store>
__device__ __forceinline__ void place(Placer& p, uint32_t n, uint32_t shift, uint32_t bits, const uint32_t* base,
                                      Key&& key, Store&& store) {
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, mask = (1u << bits) - 1;
  const uint32_t run = (n + kSortT - 1) / kSortT * 64;
  const uint32_t r0 = min(wave * run, n), r1 = min(r0 + run, n);
  for (uint32_t i = tid; i < (16u << bits); i += kSortT) (&p.at[0][0])[i] = 0;
  __syncthreads();
  for (uint32_t i = r0 + lane; i < r1; i += 64) atomicAdd(&p.at[key(i) >> shift & mask][wave], 1u);
  __syncthreads();
  if (tid <= mask) {
    uint32_t front = base[tid];
    for (int w = 0; w < 16; ++w) {
      const uint32_t c = p.at[tid][w];
      p.at[tid][w] = front;
      front += c;
    }
  }
  __syncthreads();
  for (uint32_t i0 = r0; i0 < r1; i0 += 64) {
    const bool in = i0 + lane < r1;
    const uint32_t k = in ? key(i0 + lane) : 0u, d = k >> shift & mask;
    uint64_t same = __ballot(in);
    for (uint32_t b = 0; b < bits; ++b) {
      const uint64_t one = __ballot(d >> b & 1);
      same &= d >> b & 1 ? one : ~one;
    }
    if (in) {
      const uint32_t first = p.at[d][wave];
      const uint32_t rank = (uint32_t)__popcll(same & ((1ull << lane) - 1));
      store(first + rank, k, i0 + lane);
      if (rank == 0) p.at[d][wave] = first + (uint32_t)__popcll(same);
    }
    asm volatile("" ::: "memory");  // (a wave's LDS accesses are in order)
  }
}

// All passes for few positions, in LDS.
template <typename T>
__global__ void __launch_bounds__(kSortT) embed_sort_few(GradArgs a) {
  __shared__ Placer p;
  __shared__ uint32_t base[kBins], key[2][kSmall];
  __shared__ uint16_t pos[2][kSmall];
  const uint32_t tid = threadIdx.x;
  if (blockIdx.x > 0) {
    write_zeros<T>(a, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  for (uint32_t i = tid; i < a.count; i += kSortT) {
    key[0][i] = key_of(a, i);
    pos[0][i] = (uint16_t)i;
  }
  for (uint32_t pass = 0; pass < a.passes; ++pass) {
    const uint32_t from = pass & 1, shift = pass * a.bits, mask = (1u << a.bits) - 1;
    for (uint32_t i = tid; i < kBins; i += kSortT) base[i] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < a.count; i += kSortT) atomicAdd(&base[key[from][i] >> shift & mask], 1u);
    __syncthreads();
    const uint32_t front = exclusive_over_block(tid < kBins ? base[tid] : 0u, p.waves);
    if (tid < kBins) base[tid] = front;
    __syncthreads();
    place(p, a.count, shift, a.bits, base, [&](uint32_t i) { return key[from][i]; },
          [&](uint32_t to, uint32_t k, uint32_t i) {
            key[from ^ 1][to] = k;
            pos[from ^ 1][to] = pos[from][i];
          });
    __syncthreads();
  }
  const uint32_t last = a.passes & 1;
  for (uint32_t i = tid; i < a.count; i += kSortT) {
    a.key[0][i] = key[last][i];
    a.pos[0][i] = pos[last][i];
  }
}

template <typename T>
__global__ void __launch_bounds__(kSortT) embed_digits(GradArgs a) {
  __shared__ uint32_t bins[kBins];
  const uint32_t tid = threadIdx.x;
  if (blockIdx.x >= a.blocks) {
    write_zeros<T>(a, blockIdx.x - a.blocks, gridDim.x - a.blocks);
    return;
  }
  for (uint32_t i = tid; i < kBins; i += kSortT) bins[i] = 0;
  __syncthreads();
  const uint32_t i0 = min(blockIdx.x * a.each, a.count), i1 = min(i0 + a.each, a.count);
  const uint32_t shift = a.pass * a.bits, mask = (1u << a.bits) - 1;
  for (uint32_t i = i0 + tid; i < i1; i += kSortT)
    atomicAdd(&bins[(a.pass ? a.key[a.from][i] : key_of(a, i)) >> shift & mask], 1u);
  __syncthreads();
  for (uint32_t i = tid; i < kBins; i += kSortT) a.hist[blockIdx.x * kBins + i] = bins[i];
}

template <typename T>
__global__ void __launch_bounds__(kSortT) embed_place(GradArgs a) {
  __shared__ Placer p;
  __shared__ uint32_t base[kBins];
  const uint32_t tid = threadIdx.x;
  if (blockIdx.x >= a.blocks) {
    write_zeros<T>(a, blockIdx.x - a.blocks, gridDim.x - a.blocks);
    return;
  }
  // two threads a digit, half of the workgroups' counts each, all their loads
  // together
  const uint32_t bin = tid % kBins, half = tid / kBins;
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t i = 0; i < kSortBlocks / 2; ++i) {
    const uint32_t b = 2 * i + half, c = b < a.blocks ? a.hist[b * kBins + bin] : 0u;
    before += b < blockIdx.x ? c : 0u;
    all += c;
  }
  if (half) {
    p.at[bin][0] = before;
    p.at[bin][1] = all;
  }
  __syncthreads();
  if (!half) {
    before += p.at[bin][0];
    all += p.at[bin][1];
  }
  const uint32_t front = exclusive_over_block(half ? 0u : all, p.waves);
  if (!half) base[bin] = front + before;
  __syncthreads();
  const uint32_t i0 = min(blockIdx.x * a.each, a.count), i1 = min(i0 + a.each, a.count);
  const uint32_t* key = a.key[a.from] + i0;
  const uint32_t* pos = a.pos[a.from] + i0;
  uint32_t* to_key = a.key[a.from ^ 1];
  uint32_t* to_pos = a.pos[a.from ^ 1];
  const uint32_t shift = a.pass * a.bits;
  if (a.pass == 0)
    place(p, i1 - i0, shift, a.bits, base, [&](uint32_t i) { return key_of(a, i0 + i); },
          [&](uint32_t to, uint32_t k, uint32_t i) {
            to_key[to] = k;
            to_pos[to] = i0 + i;
          });
  else
    place(p, i1 - i0, shift, a.bits, base, [&](uint32_t i) { return key[i]; },
          [&](uint32_t to, uint32_t k, uint32_t i) {
            to_key[to] = k;
            to_pos[to] = pos[i];
          });
}

// Past the caches where positions are many: 19,200 x 1,024 into tables of 50 to 300
// MB take 49 to 78 us so, 53 to 84 through them.
template <typename T, bool kPast>
__device__ __forceinline__ void write_row(const GradArgs& a, uint32_t token, uint32_t e, float (&sum)[kVec<T>]) {
  T* to = (T*)a.dtable + (int64_t)token * a.dtable_stride + e;
  float old[kVec<T>] = {};
  if (a.add) to_float<T>(load_row_vec(to - e, e, a.hidden, (T)0.0f), old);
#pragma unroll
  for (int k = 0; k < kVec<T>; ++k) sum[k] = __builtin_fmaf(sum[k], a.scale, old[k]);
  if (e + kVec<T> <= a.hidden) store_to<kPast>(to, from_float<T>(sum));
  else store_part(to, (int)(a.hidden - e), from_float<T>(sum));
}

template <typename T>
__device__ __forceinline__ float* part_of(const GradArgs& a, uint32_t which, uint32_t run, uint32_t e) {
  const uint32_t width = (a.hidden + kVec<T> - 1) / kVec<T> * kVec<T>;
  return a.parts + ((uint64_t)which * a.runs + run) * width + e;
}
template <typename T>
__device__ __forceinline__ void store_floats(float* to, const float (&v)[kVec<T>]) {
#pragma unroll
  for (int k = 0; k < kVec<T>; k += 4) *(f32x4*)(to + k) = f32x4{v[k], v[k + 1], v[k + 2], v[k + 3]};
}

// Walks over rows pos(0 ... n - 1) of the gradient, up to eight loads ahead
// whatever the runs are: take(i, values) in order.
constexpr uint32_t kBatch = 4;
template <typename T, typename Pos, typename Take>
__device__ __forceinline__ void walk_rows(const GradArgs& a, uint32_t n, uint32_t e, Pos&& pos, Take&& take) {
  u32x4 v[2][kBatch];
  const auto load = [&](u32x4 (&to)[kBatch], uint32_t r) {
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) {
      to[u] = u32x4{};
      if (r + u < n) {
        const uint32_t row = pos(r + u);
        if (e < a.hidden) to[u] = load_row_vec((const T*)a.grad + (int64_t)row * a.grad_stride, e, a.hidden, (T)0.0f);
      }
    }
  };
  const auto add = [&](const u32x4 (&from)[kBatch], uint32_t r) {
#pragma unroll
    for (uint32_t u = 0; u < kBatch; ++u) {
      if (r + u >= n) break;
      float f[kVec<T>];
      to_float<T>(from[u], f);
      take(r + u, f);
    }
  };
  load(v[0], 0);
  for (uint32_t r = 0; r < n; r += 2 * kBatch) {
    load(v[1], r + kBatch);
    add(v[0], r);
    load(v[0], r + 2 * kBatch);
    add(v[1], r + kBatch);
  }
}

// A wave kRun sorted positions by 64 vectors of their rows.
template <typename T, int kRun>
__global__ void __launch_bounds__(256) embed_sums(GradArgs a) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t task = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t run = task / a.panels, e = (task % a.panels * 64 + lane) * kVec<T>;
  if (run >= a.runs) return;
  const uint32_t i0 = run * kRun, n = min((uint32_t)kRun, a.count - i0);
  const uint32_t key = lane < n ? a.sorted_key[i0 + lane] : a.vocab;
  const uint32_t pos = lane < n ? a.sorted_pos[i0 + lane] : 0u;
  const uint32_t prev = i0 ? a.sorted_key[i0 - 1] : ~0u;
  const uint32_t next = i0 + n < a.count ? a.sorted_key[i0 + n] : ~0u;
  // positions with a token (those without are behind them)
  const uint32_t used = (uint32_t)__popcll(__ballot(key < a.vocab));
  const auto key_at = [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)key, (int)i); };
  float sum[kVec<T>] = {};
  bool starts = used && key_at(0) != prev;
  walk_rows<T>(
      a, used, e, [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readlane((int)pos, (int)i); },
      [&](uint32_t i, const float (&f)[kVec<T>]) {
#pragma unroll
        for (int c = 0; c < kVec<T>; ++c) sum[c] += f[c];
        const uint32_t k = key_at(i), after = i + 1 < n ? key_at(i + 1) : next;
        if (after == k && i + 1 < n) return;
        // the token's last here
        if (e < a.hidden) {
          if (starts && after != k) write_row<T, true>(a, k, e, sum);
          else store_floats<T>(part_of<T>(a, starts ? 1 : 0, run, e), sum);
        }
        starts = true;
#pragma unroll
        for (int c = 0; c < kVec<T>; ++c) sum[c] = 0.0f;
      });
}

// Few positions of rows that are whole vectors, in one launch (80 tokens, 32,768 x
// 512 f32: 11.5 us where sort, sums and join take 20; 1,664 tokens, 100,003 x 768
// f16: 28.6, the zeros' 154 MB at 5.4 TB/s): a workgroup a position and 64 vectors
// looks for the others of its token (and is done if there is one before it), its
// waves share a long list of them, and other workgroups write zeros to the rows
// of other tokens.  2,048 positions of one token x 512: 51 us (by a wave each 341).
constexpr int kFewT = 512, kFewWaves = kFewT / 64;
template <typename T, bool kPast>
__global__ void __launch_bounds__(kFewT) embed_few(GradArgs a) {
  __shared__ uint32_t list[kSmall];  // positions; or the bits of the zeros' rows
  __shared__ uint32_t found[kFewWaves], earliest[kFewWaves];
  __shared__ float parts[kFewWaves - 1][64][kVec<T> + 1];
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6));
  // (the two kinds mixed, so that neither waits for the other's end)
  const uint32_t adds = (uint32_t)((uint64_t)blockIdx.x * a.blocks / gridDim.x);  // of those in front
  if ((uint32_t)((uint64_t)(blockIdx.x + 1) * a.blocks / gridDim.x) > adds) {
    const uint32_t p = adds / a.panels, e = (adds % a.panels * 64 + lane) * kVec<T>;
    const uint32_t k = key_of(a, p);
    if (k >= a.vocab) return;
    constexpr uint32_t kMasks = kSmall / 64 / kFewWaves;
    uint64_t same[kMasks];
    uint32_t n = 0, first = ~0u;
#pragma unroll
    for (uint32_t i = 0; i < kMasks; ++i) {
      const uint32_t at = (wave * kMasks + i) * 64 + lane;
      same[i] = __ballot(at < a.count && key_of(a, at) == k);
      if (same[i] && first == ~0u) first = (wave * kMasks + i) * 64 + (uint32_t)__ffsll((unsigned long long)same[i]) - 1;
      n += (uint32_t)__popcll(same[i]);
    }
    if (lane == 0) {
      found[wave] = n;
      earliest[wave] = first;
    }
    __syncthreads();
    uint32_t front = 0, all = 0, least = ~0u;
#pragma unroll
    for (uint32_t w = 0; w < (uint32_t)kFewWaves; ++w) {
      front += w < wave ? found[w] : 0u;
      all += found[w];
      least = min(least, earliest[w]);
    }
    if (least < p) return;
#pragma unroll
    for (uint32_t i = 0; i < kMasks; ++i) {
      if (same[i] >> lane & 1)
        list[front + (uint32_t)__popcll(same[i] & ((1ull << lane) - 1))] = (wave * kMasks + i) * 64 + lane;
      front += (uint32_t)__popcll(same[i]);
    }
    __syncthreads();
    const uint32_t waves = all <= 16 ? 1 : kFewWaves, each = (all + waves - 1) / waves;
    const uint32_t i0 = min(wave * each, all), i1 = wave < waves ? min(i0 + each, all) : i0;
    float sum[kVec<T>] = {};
    walk_rows<T>(
        a, i1 - i0, e, [&](uint32_t i) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)list[i0 + i]); },
        [&](uint32_t, const float (&f)[kVec<T>]) {
#pragma unroll
          for (int c = 0; c < kVec<T>; ++c) sum[c] += f[c];
        });
    if (waves > 1) {
      if (wave > 0)
#pragma unroll
        for (int c = 0; c < kVec<T>; ++c) parts[wave - 1][lane][c] = sum[c];
      __syncthreads();
      if (wave == 0)
        for (uint32_t w = 1; w < waves; ++w)
#pragma unroll
          for (int c = 0; c < kVec<T>; ++c) sum[c] += parts[w - 1][lane][c];
    }
    if (wave == 0 && e < a.hidden) write_row<T, kPast>(a, k, e, sum);
    return;
  }
  // rows r0 ... of the table, which have no gaps
  const uint32_t per = a.hidden / kVec<T>, rows = a.zero_units, r0 = (blockIdx.x - adds) * rows;
  const uint32_t n = min(rows, a.vocab - r0);
  for (uint32_t i = tid; i < (n + 31) / 32; i += kFewT) list[i] = 0;
  __syncthreads();
  for (uint32_t i = tid; i < a.count; i += kFewT) {
    const uint32_t k = key_of(a, i) - r0;
    if (k < n) atomicOr(&list[k / 32], 1u << k % 32);
  }
  __syncthreads();
  T* to = (T*)a.dtable + (uint64_t)r0 * a.hidden;
#pragma unroll 4
  for (uint32_t v = tid; v < n * per; v += kFewT) {
    const uint32_t row = v / per;
    if (!(list[row / 32] >> row % 32 & 1)) store_to<kPast>(to + (uint64_t)v * kVec<T>, u32x4{});
  }
}

// Joins the parts of a token that goes on past the positions of run
// blockIdx / panels, where it starts: that run's second part, then the first
// parts of the runs behind it.  Four waves take a quarter of them each.
template <typename T, int kRun>
__global__ void __launch_bounds__(256) embed_join(GradArgs a) {
  __shared__ float quarter[3][64][kVec<T> + 1];
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const uint32_t run = blockIdx.x / a.panels, e = (blockIdx.x % a.panels * 64 + lane) * kVec<T>;
  const uint32_t i0 = run * kRun, i1 = i0 + kRun;
  if (i1 >= a.count) return;
  const uint32_t k = a.sorted_key[i1 - 1];
  if (k >= a.vocab || a.sorted_key[i1] != k) return;
  if (a.sorted_key[i0] == k && i0 > 0 && a.sorted_key[i0 - 1] == k) return;
  // runs behind it that the token reaches: the first whose next one it does not
  uint32_t more = 1;
  for (;;) {
    const uint64_t i = (uint64_t)(run + more + lane + 1) * kRun;
    const uint64_t stops = __ballot(i >= a.count || a.sorted_key[i] != k);
    if (stops) {
      more += (uint32_t)__ffsll((unsigned long long)stops) - 1;
      break;
    }
    more += 64;
  }
  const uint32_t each = (more + 3) / 4, m0 = min(wave * each, more), m1 = min(m0 + each, more);
  float sum[kVec<T>] = {};
  const bool in = e < a.hidden;
  if (in) {
    if (wave == 0) {
      const float* p = part_of<T>(a, 1, run, e);
#pragma unroll
      for (int c = 0; c < kVec<T>; ++c) sum[c] = p[c];
    }
#pragma unroll 4
    for (uint32_t m = m0; m < m1; ++m) {
      const float* p = part_of<T>(a, 0, run + 1 + m, e);
#pragma unroll
      for (int c = 0; c < kVec<T>; ++c) sum[c] += p[c];
    }
    if (wave > 0)
#pragma unroll
      for (int c = 0; c < kVec<T>; ++c) quarter[wave - 1][lane][c] = sum[c];
  }
  __syncthreads();
  if (wave > 0 || !in) return;
#pragma unroll
  for (int w = 0; w < 3; ++w)
#pragma unroll
    for (int c = 0; c < kVec<T>; ++c) sum[c] += quarter[w][lane][c];
  write_row<T, true>(a, k, e, sum);
}

// Positions of a wave: few where there are few of them.
uint32_t run_of(uint64_t count) { return count < 16384 ? 8 : 32; }

struct GradPlan {
  uint64_t key[2], pos[2], hist, parts, bytes;
};
GradPlan plan(const ft_embed_grad_args& a) {
  GradPlan p{};
  Arena ar;
  const uint64_t n = a.groups * a.steps, vec = a.dtype == FT_F32 ? 4 : 8;
  for (int i = 0; i < 2; ++i) {
    p.key[i] = ar.take(n * 4);
    p.pos[i] = ar.take(n * 4);
  }
  p.hist = ar.take((uint64_t)kSortBlocks * kBins * 4);
  const uint64_t run = run_of(n);
  p.parts = ar.take(2 * ((n + run - 1) / run) * round_up(a.hidden, vec) * 4);
  p.bytes = ar.used;
  return p;
}

template <typename T>
hipError_t launch_grad(GradArgs a, hipStream_t s) {
  constexpr uint32_t kZeroBlocks = 512;
  const uint64_t units = a.add ? 0 : (uint64_t)a.zero_units * (a.zero_length == a.hidden ? a.vocab : 1);
  hipError_t e;
  // (the zeros' rows without gaps, 128 KB or a row a workgroup; a bit for each)
  constexpr uint32_t kZeroVecs = 8192;
  static_assert(kZeroVecs <= kSmall * 32, "bits for a row of a vector each");
  const uint32_t per = a.hidden / kVec<T>;
  if (a.count <= kSmall && a.count > 0 && a.hidden % kVec<T> == 0 && (a.add || a.dtable_stride == (int64_t)a.hidden)) {
    a.blocks = a.count * a.panels;
    a.zero_units = std::max(1u, kZeroVecs / per);
    const uint64_t blocks = a.blocks + (a.add ? 0 : (a.vocab + a.zero_units - 1) / a.zero_units);
    // (past the caches or through them: 80 tokens x 512 into 67 MB 13.1 us and 11.5;
    // 1,664 x 768 into 154 MB, another gradient each call, 28.6 and 37)
    return (uint64_t)a.vocab * a.hidden * sizeof(T) > kPastBytes ? start(embed_few<T, true>, blocks, kFewT, s, a)
                                                                 : start(embed_few<T, false>, blocks, kFewT, s, a);
  }
  if (a.count <= kSmall) {
    a.zero_last = units;
    e = start(embed_sort_few<T>, 1 + std::min<uint64_t>(units, kZeroBlocks), kSortT, s, a);
    if (e != hipSuccess) return e;
    a.sorted_key = a.key[0];
    a.sorted_pos = a.pos[0];
  } else {
    a.blocks = std::min(kSortBlocks, (a.count + kSmall - 1) / kSmall);
    a.each = ((a.count + a.blocks - 1) / a.blocks + kSortT - 1) / kSortT * kSortT;
    // the zeros go beside the sorting, a share in each launch
    uint64_t done = 0;
    const uint32_t launches = 2 * a.passes;
    for (uint32_t l = 0; l < launches; ++l) {
      a.pass = l / 2;
      a.from = a.pass & 1;
      a.zero_first = done;
      a.zero_last = done = units * (l + 1) / launches;
      const uint64_t grid = a.blocks + std::min<uint64_t>(a.zero_last - a.zero_first, kZeroBlocks);
      e = start(l & 1 ? embed_place<T> : embed_digits<T>, grid, kSortT, s, a);
      if (e != hipSuccess) return e;
    }
    a.sorted_key = a.key[a.passes & 1];
    a.sorted_pos = a.pos[a.passes & 1];
  }
  if (a.count == 0) return hipSuccess;
  const uint64_t tasks = (uint64_t)a.runs * a.panels;
  const bool few = run_of(a.count) == 8;
  e = start(few ? embed_sums<T, 8> : embed_sums<T, 32>, (tasks + 3) / 4, 256, s, a);
  if (e != hipSuccess) return e;
  return start(few ? embed_join<T, 8> : embed_join<T, 32>, tasks, 256, s, a);
}

}  // namespace

uint64_t embed_workspace(const ft_embed_args&) { return 0; }

hipError_t launch_embed(const ft_embed_args& q, uint8_t*, hipStream_t s) {
  if (q.groups == 0 || q.steps == 0) return hipSuccess;
  LookupArgs a{};
  a.tokens = q.tokens;
  a.lengths = q.lengths;
  a.table = q.table;
  a.table_stride = q.table_stride;
  a.out = q.out;
  a.count = (uint32_t)(q.groups * q.steps);
  a.steps = (uint32_t)q.steps;
  a.hidden = q.hidden;
  a.vocab = q.vocab;
  a.scale = q.scale;
  a.panels = (q.hidden + 64 * (q.dtype == FT_F32 ? 4 : 8) - 1) / (64 * (q.dtype == FT_F32 ? 4 : 8));
  const uint64_t blocks = (uint64_t)((a.count + 4 * kTokens - 1) / (4 * kTokens)) * a.panels;
  return q.dtype == FT_F32   ? start(embed_rows<float>, blocks, 256, s, a)
         : q.dtype == FT_F16 ? start(embed_rows<_Float16>, blocks, 256, s, a)
                             : start(embed_rows<__bf16>, blocks, 256, s, a);
}

uint64_t embed_grad_workspace(const ft_embed_grad_args& a) { return plan(a).bytes; }

hipError_t launch_embed_grad(const ft_embed_grad_args& q, uint8_t* ws, hipStream_t s) {
  const GradPlan p = plan(q);
  const uint32_t vec = q.dtype == FT_F32 ? 4 : 8;
  GradArgs a{};
  a.tokens = q.tokens;
  a.lengths = q.lengths;
  a.grad = q.grad;
  a.grad_stride = q.grad_stride;
  a.dtable = q.dtable;
  a.dtable_stride = q.dtable_stride;
  a.count = (uint32_t)(q.groups * q.steps);
  a.steps = (uint32_t)q.steps;
  a.hidden = q.hidden;
  a.vocab = q.vocab;
  a.scale = q.scale;
  a.add = q.add != 0;
  a.panels = (q.hidden + 64 * vec - 1) / (64 * vec);
  const uint32_t run = run_of(a.count);
  a.runs = (a.count + run - 1) / run;
  for (int i = 0; i < 2; ++i) {
    a.key[i] = (uint32_t*)(ws + p.key[i]);
    a.pos[i] = (uint32_t*)(ws + p.pos[i]);
  }
  a.hist = (uint32_t*)(ws + p.hist);
  a.parts = (float*)(ws + p.parts);
  uint32_t bits = 1;  // of the keys 0 ... vocab
  while (q.vocab >> bits) ++bits;
  a.passes = (bits + 8) / 9;
  a.bits = (bits + a.passes - 1) / a.passes;
  // a table without gaps is one row
  const bool dense = q.dtable_stride == (int64_t)q.hidden && q.vocab > 1;
  a.zero_length = dense ? (uint64_t)q.vocab * q.hidden : q.hidden;
  a.zero_stride = dense ? 0 : q.dtable_stride;
  a.zero_units = (uint32_t)(((a.zero_length + vec - 1) / vec + kZeroUnit - 1) / kZeroUnit);
  return q.dtype == FT_F32   ? launch_grad<float>(a, s)
         : q.dtype == FT_F16 ? launch_grad<_Float16>(a, s)
                             : launch_grad<__bf16>(a, s);
}

}  // namespace fto
