// propose.hip -- proposal rows from logits: the topk largest of each row in
// ascending token order, with their log-probabilities.
//
// One pass over the logits gives each row's (max, sum of exponentials) and
// the maximum of every group of neighbouring logits.  A key that at least
// topk group maxima reach is a lower bound of the topk-th largest logit, so
// the groups that reach it hold every logit that can be proposed, and only
// they are read again.  Where ties let too many reach it, those above it and
// the first of those at it do, topk in all: each of these holds one logit at
// the bound, so the lowest ids of such logits are among them.
// Selections are by histograms of keys, whose counts depend on no order, and
// rows are written by ordered compaction: ascending, as they are, no sort.
//
// Bound by one read of the logits where the rows are long (128 rows of
// 2,200,000 bf16, 1000 each: 144 us; in a trace 116 the scan at 4.9 TB/s, 32
// the rows' ends), by the latency of a row's end where they are short (8
// rows of 32,768 f32, 32 each: 14 us for 1 MB).
#include <type_traits>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

constexpr int kScanT = 256;     // threads of a scanning workgroup
constexpr int kScanU = 4;       // vectors in flight a thread
constexpr int kFinT = 1024;     // of a finishing one
constexpr int kFinWaves = kFinT / 64;
constexpr uint32_t kMaxGroups = 65536;  // of a row
constexpr uint32_t kRowVecs = 16384;    // of a row that one workgroup scans
constexpr uint32_t kCap = 8192;         // candidates held in LDS

struct ScanPlan {
  uint32_t lanes_log2;   // lanes of a group: G = kVec << lanes_log2
  uint32_t groups;       // of a row
  uint32_t chunks;       // workgroups of a row
  uint32_t chunk_vecs;   // vectors of a workgroup
  uint64_t gmax, part;   // workspace offsets
  uint64_t bytes;
};

// Groups: as long as leaves four of them a proposal (the bound is then
// close: about 1.15 topk logits reach it in random rows), at most 64 logits
// (one or two lines; longer only to stay within kMaxGroups).  Chunks: about
// 4096 workgroups in all, 16 a CU, in whole turns of its loads.
template <typename T>
ScanPlan plan(const ft_propose_args& a) {
  ScanPlan p{};
  const uint32_t vec = (uint32_t)kVec<T>;
  const uint64_t rows = a.batch * a.steps;
  uint32_t lg = 0;
  while ((vec << (lg + 1)) <= 64 && (uint64_t)4 * a.topk * (vec << (lg + 1)) <= a.vocab) ++lg;
  while ((a.vocab + (vec << lg) - 1) / (vec << lg) > kMaxGroups) ++lg;
  p.lanes_log2 = lg;
  const uint32_t G = vec << lg;
  p.groups = (a.vocab + G - 1) / G;
  const uint32_t vecs = (a.vocab + vec - 1) / vec, least = kScanU * kScanT;
  uint64_t want = rows ? (4096 + rows - 1) / rows : 1;
  uint64_t each = (vecs + want - 1) / want;
  if (each < least) each = least;
  p.chunk_vecs = (uint32_t)round_up(each, least);
  p.chunks = (vecs + p.chunk_vecs - 1) / p.chunk_vecs;
  Arena ar;
  p.gmax = ar.take(rows * p.groups * sizeof(T));
  p.part = ar.take(rows * p.chunks * sizeof(MaxSum));
  p.bytes = ar.used;
  return p;
}

struct Args {
  const void* logits;
  uint64_t steps;
  int64_t stride[2];
  uint32_t vocab, topk;
  uint32_t lanes_log2, groups, chunks, chunk_vecs;
  void* gmax;
  MaxSum* part;
  int32_t* ids;
  float* logp;
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Args& a, uint64_t row) {
  const uint64_t b = row / a.steps, t = row - b * a.steps;
  return (const T*)a.logits + (int64_t)b * a.stride[0] + (int64_t)t * a.stride[1];
}

template <typename T>
__device__ __forceinline__ u32x4 load_row(const T* p, uint32_t vec, uint32_t vocab) {
  return load_row_vec(p, vec * kVec<T>, vocab, (T)-INFINITY);
}

// Block (row, chunk): a vector a lane, so that a group's lanes exchange their
// maxima within the wave; four loads in flight a thread keep memory busy at
// eight workgroups a CU.
template <typename T>
__global__ void __launch_bounds__(kScanT) propose_scan(Args a) {
  const uint64_t row = blockIdx.x / a.chunks;
  const uint32_t chunk = blockIdx.x - (uint32_t)(row * a.chunks), tid = threadIdx.x;
  const T* p = row_of<T>(a, row);
  T* gmax = (T*)a.gmax + row * a.groups;
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  const uint32_t v0 = chunk * a.chunk_vecs, v1 = min(v0 + a.chunk_vecs, vecs);
  MaxSum ms{-INFINITY, 0.0f};
  for (uint32_t v = v0; v < v1; v += kScanU * kScanT) {
    u32x4 raw[kScanU];
    load_run<kScanU>(raw, p, v + tid, kScanT, a.vocab, (T)-INFINITY,
                     (v + kScanU * kScanT) * kVec<T> <= a.vocab);
#pragma unroll
    for (int u = 0; u < kScanU; ++u) {
      const uint32_t at = v + u * kScanT + tid;
      float x[kVec<T>];
      to_float<T>(raw[u], x);
      if (at < v1) add_terms(ms, x);
      float g = x[0];
#pragma unroll
      for (int i = 1; i < kVec<T>; ++i) g = fmaxf(g, x[i]);
      for (uint32_t d = 0; d < a.lanes_log2; ++d) g = fmaxf(g, __shfl_xor(g, 1 << d, 64));
      if ((tid & ((1u << a.lanes_log2) - 1)) == 0 && at < v1) gmax[at >> a.lanes_log2] = (T)g;
    }
  }
  ms = wave_merge(ms);
  __shared__ MaxSum waves[kScanT / 64];
  if ((tid & 63) == 0) waves[tid >> 6] = ms;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kScanT / 64; ++w) ms = merge(ms, waves[w]);
    a.part[row * a.chunks + chunk] = ms;
  }
}

// Keys are the type's own order, as unsigned numbers of its size: NaN as
// -infinity, -0 as 0.
template <typename T>
using Half = std::conditional_t<sizeof(T) == 2, T, _Float16>;
template <typename T>
using Key = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

template <typename T>
__device__ __forceinline__ uint32_t key_of(float x) {
  if (sizeof(T) == 4) return order_key(x);
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t b = __builtin_bit_cast(uint16_t, (T)x);
  return b & 0x8000u ? b ^ 0xFFFFu : b | 0x8000u;
}
template <>
__device__ __forceinline__ uint32_t key_of<float>(float x) {
  return order_key(x);
}
template <typename T>
__device__ __forceinline__ float value_of(uint32_t k) {
  return (float)__builtin_bit_cast(T, (uint16_t)(k & 0x8000u ? k & 0x7FFFu : k ^ 0xFFFFu));
}
template <>
__device__ __forceinline__ float value_of<float>(uint32_t k) {
  return key_value(k);
}

// The kernels that end a row are bound by latencies: a workgroup walks once
// through some thousand instructions, with barriers, and every line of them
// comes from L2.  So their loops are short and rolled, over keys in LDS, and
// selections are by histograms of 11 bits.
constexpr uint32_t kKeyBytes = 72u << 10;  // LDS for a row's group keys
constexpr uint32_t kBins = 2 * kFinT;

struct Shared {
  uint32_t hist[kBins];
  uint32_t found[2];
  uint32_t scan[2][kFinWaves];
  uint32_t cells[8][kFinWaves], all_cells;  // sums of a turn and wave
  MaxSum ms[kFinWaves];
  float lse, m;
  uint32_t ckey[kCap], cid[kCap];  // candidates, ascending ids
};

// The cells' first `turns` rows to the sums of all cells in front; the whole
// sum is all_cells.  Between barriers.
__device__ __forceinline__ void scan_cells(Shared& sh, uint32_t turns) {
  __syncthreads();
  if (threadIdx.x < 64) {
    uint32_t front = 0;
    for (uint32_t i = threadIdx.x; i - threadIdx.x < turns * kFinWaves; i += 64) {
      uint32_t* c = &sh.cells[0][0] + i;
      const uint32_t v = i < turns * kFinWaves ? *c : 0u;
      uint32_t total;
      const uint32_t f = wave_scan(v, &total);
      if (i < turns * kFinWaves) *c = front + f;
      front += total;
    }
    if (threadIdx.x == 0) sh.all_cells = front;
  }
  __syncthreads();
}

// The highest bin that `need` keys reach, and how many reach it; the
// histogram is filled (before a barrier) and holds at least as many.
__device__ __forceinline__ uint32_t pick_bin(Shared& sh, uint32_t need, uint32_t* reach) {
  const uint32_t tid = threadIdx.x, wave = tid >> 6, top = kBins - 1 - 2 * tid;
  const uint32_t a = sh.hist[top], own = a + sh.hist[top - 1];
  uint32_t total, front = wave_scan(own, &total);
  if ((tid & 63) == 0) sh.scan[0][wave] = total;
  __syncthreads();
#pragma unroll 4
  for (uint32_t w = 0; w < kFinWaves; ++w) front += w < wave ? sh.scan[0][w] : 0;
  if (front < need && need <= front + own) {
    const bool first = need <= front + a;
    sh.found[0] = first ? top : top - 1;
    sh.found[1] = first ? front + a : front + own;
  }
  __syncthreads();
  *reach = sh.found[1];
  return sh.found[0];
}

// A key that at least `need` of all keys reach, and how many do (n): the
// largest such key, or the first one found that at most `enough` keys reach.
// n keys reach lo, at least `need`; over of them, fewer, reach hi.  key(i),
// i < size, are the keys.
template <typename F>
__device__ __forceinline__ uint32_t largest_reached(Shared& sh, uint32_t need, uint32_t enough,
                                                    uint32_t lo, uint32_t hi, uint32_t over,
                                                    uint32_t size, uint32_t* n, F&& key) {
  const uint32_t tid = threadIdx.x;
  while (hi - lo > 1 && *n > enough) {
    const int bits = 32 - __clz((int)(hi - lo - 1)), shift = bits > 11 ? bits - 11 : 0;
    sh.hist[tid] = sh.hist[tid + kFinT] = 0;
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = tid; i < size; i += kFinT) {
      const uint32_t k = key(i);
      if (k >= lo && k < hi) atomicAdd(&sh.hist[(k - lo) >> shift], 1u);
    }
    __syncthreads();
    uint32_t reach;
    const uint32_t bin = pick_bin(sh, need - over, &reach);
    *n = over + reach;
    over = *n - sh.hist[bin];
    lo += bin << shift;
    hi = min(hi - lo, 1u << shift) + lo;
    __syncthreads();
  }
  return lo;
}

// Sums over the threads in front of (a, b), and all's in *ta, *tb; every
// thread of the block.
__device__ __forceinline__ void block_scan2(Shared& sh, uint32_t& a, uint32_t& b, uint32_t* ta,
                                            uint32_t* tb) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t wave_a, wave_b;
  a = wave_scan(a, &wave_a);
  b = wave_scan(b, &wave_b);
  if (lane == 0) {
    sh.scan[0][wave] = wave_a;
    sh.scan[1][wave] = wave_b;
  }
  __syncthreads();
  uint32_t all_a = 0, all_b = 0;
#pragma unroll 4
  for (uint32_t w = 0; w < kFinWaves; ++w) {
    const uint32_t wa = sh.scan[0][w], wb = sh.scan[1][w];
    all_a += wa;
    all_b += wb;
    a += w < wave ? wa : 0;
    b += w < wave ? wb : 0;
  }
  *ta = all_a;
  *tb = all_b;
  __syncthreads();
}

// How many groups may reach the bound T: it need not be the very K-th
// largest group maximum (that of vectors of eight groups' keys lets through
// an eighth more in random rows), and a turn saved is worth more than that.
__device__ __forceinline__ uint32_t enough_groups(uint32_t K) { return K + K / 4 + 32; }
constexpr uint32_t kListTurns = 5;  // turns of vectors of the keys that LDS holds
constexpr uint32_t kMaxListed = FT_MAX_PROPOSALS + FT_MAX_PROPOSALS / 4 + 32;

// Writes a row's proposals; sh.m and sh.lse are there, gkey(g) is group g's
// key (kLds: keys[g]).
template <typename T, bool kLds, typename G>
__device__ __forceinline__ void finish_row(Shared& sh, uint16_t* list, const Args& a, uint64_t row,
                                           uint32_t groups, uint32_t lg, const Key<T>* keys,
                                           G&& gkey) {
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, K = a.topk;
  const T* p = row_of<T>(a, row);
  // The bound T: first by a histogram of distances from the row's maximum,
  // 2047 steps of 1/64 (differences of logits are of that order, whatever
  // their size), of the groups or, where there are enough of them, of vectors
  // of their keys, whose maxima bound as well; then, where too many groups
  // reach its bin, by the groups' keys.  (A row of -infinity has m = 0, above
  // its keys too.)
  constexpr float kSteps = 64.0f;
  const float m = sh.m, lse = sh.lse;
  const auto bin_of = [&](float x) {  // (x = m may be infinity)
    return kBins - 1 - (x == m ? 0u : (uint32_t)fminf((m - x) * kSteps, (float)(kBins - 1)));
  };
  const uint32_t top = key_of<T>(m) + 1, enough = enough_groups(K);
  constexpr uint32_t kKeys = kLds ? 16 / sizeof(Key<T>) : 1;  // of a vector
  const uint32_t kvecs = (groups + kKeys - 1) / kKeys;
  const auto keys_of = [&](uint32_t v, uint32_t (&k)[kKeys]) {
    if constexpr (kLds) {
      const u32x4 raw = *(const u32x4*)(keys + v * kKeys);
#pragma unroll
      for (uint32_t e = 0; e < kKeys; ++e) {
        const uint32_t w = raw[e * sizeof(Key<T>) / 4];
        k[e] = sizeof(Key<T>) == 4 ? w : e & 1 ? w >> 16 : w & 0xFFFFu;
        if (v * kKeys + e >= groups) k[e] = 0;
      }
    } else {
      k[0] = gkey(v);
    }
  };
  uint32_t bound = 0, reached = groups;
  if (groups > K) {
    const bool by_vector = kKeys > 1 && kvecs >= 2 * K;
    sh.hist[tid] = sh.hist[tid + kFinT] = 0;
    __syncthreads();
    if (by_vector) {
#pragma unroll 1
      for (uint32_t v = tid; v < kvecs; v += kFinT) {
        uint32_t k[kKeys], most = 0;
        keys_of(v, k);
#pragma unroll
        for (uint32_t e = 0; e < kKeys; ++e) most = max(most, k[e]);
        atomicAdd(&sh.hist[bin_of(value_of<T>(most))], 1u);
      }
    } else {
#pragma unroll 2
      for (uint32_t g = tid; g < groups; g += kFinT)
        atomicAdd(&sh.hist[bin_of(value_of<T>(gkey(g)))], 1u);
    }
    __syncthreads();
    const uint32_t bin = pick_bin(sh, K, &reached);
    // the smallest key whose bin is at least b: 64 guesses a round
    uint32_t lo = 0, hi = top - 1;  // too small; large enough
    while (bin > 0 && hi - lo > 1) {
      const uint32_t step = (hi - lo - 1) / 64 + 1;
      const uint32_t k = (uint32_t)min((uint64_t)hi, (uint64_t)lo + (uint64_t)(lane + 1) * step);
      const uint64_t yes = __ballot(bin_of(value_of<T>(k)) >= bin);
      const uint32_t f = (uint32_t)__ffsll((unsigned long long)yes) - 1u;
      hi = (uint32_t)min((uint64_t)hi, (uint64_t)lo + (uint64_t)(f + 1) * step);
      lo += f * step;
    }
    bound = bin > 0 ? hi : 0u;
  }
  // The groups to read again, ascending: those that reach the bound.
  uint32_t most = 0;
  const auto list_turns = [&](uint32_t v0, uint32_t most, bool write) {
    // vectors of keys v0 ... of up to kListTurns turns: counted, or listed
    uint32_t hits[kListTurns];
#pragma unroll
    for (uint32_t t = 0; t < kListTurns; ++t) {
      const uint32_t v = v0 + t * kFinT + tid;
      uint32_t k[kKeys], h = 0;
      if (v < kvecs) {
        keys_of(v, k);
#pragma unroll
        for (uint32_t e = 0; e < kKeys; ++e) h |= (k[e] >= max(bound, 1u) ? 1u : 0u) << e;
      }
      hits[t] = h;
      uint32_t total = wave_add((uint32_t)__popc(h));
      if (lane == 0) sh.cells[t][wave] = total;
    }
    scan_cells(sh, kListTurns);
    const uint32_t n = sh.all_cells;
    if (write && most + n <= kMaxListed) {
#pragma unroll
      for (uint32_t t = 0; t < kListTurns; ++t) {
        uint32_t h = hits[t], none;
        uint32_t at = most + sh.cells[t][wave] + wave_scan((uint32_t)__popc(h), &none);
        while (h) {
          const uint32_t e = (uint32_t)__ffs(h) - 1u;
          h &= h - 1;
          list[at++] = (uint16_t)((v0 + t * kFinT + tid) * kKeys + e);
        }
      }
    }
    __syncthreads();
    return n;
  };
  for (uint32_t v0 = 0; v0 < kvecs; v0 += kListTurns * kFinT) most += list_turns(v0, most, true);
  if (groups > K && most > enough) {
    // Too many: the bound by the keys, as exact as it takes; where ties are
    // too many still, those above it and the first of those at it, up to K.
    reached = most;
    bound = largest_reached(sh, K, enough, bound, top, 0, groups, &reached, gkey);
    const bool cut = reached > enough;
    most = cut ? K : reached;
    const uint32_t run = (groups + kFinT - 1) / kFinT * 64;
    const uint32_t g0 = min(wave * run, groups), g1 = min(g0 + run, groups);
    uint32_t above = 0, tied = 0, sum, ties;
    for (uint32_t g = g0 + lane; g < g1; g += 64) {
      above += gkey(g) > bound;
      tied += gkey(g) == bound;
    }
    block_scan2(sh, above, tied, &sum, &ties);
    ties = most - sum;
    // (lane 0 has the sums over the waves in front)
    above = (uint32_t)__builtin_amdgcn_readfirstlane((int)above);
    tied = (uint32_t)__builtin_amdgcn_readfirstlane((int)tied);
    const uint64_t before = (1ull << lane) - 1;
#pragma unroll 1
    for (uint32_t i = g0; i < g1; i += 64) {
      const uint32_t g = i + lane, k = g < g1 ? gkey(g) : 0u;
      const uint64_t ma = __ballot(g < g1 && k > bound), mt = __ballot(g < g1 && k == bound);
      const uint32_t pa = above + (uint32_t)__popcll(ma & before);
      const uint32_t pt = tied + (uint32_t)__popcll(mt & before);
      if (g < g1 && (k > bound || (k == bound && pt < ties))) list[pa + min(pt, ties)] = (uint16_t)g;
      above += (uint32_t)__popcll(ma);
      tied += (uint32_t)__popcll(mt);
    }
  }
  __syncthreads();
  const uint32_t vecs = most << lg, beyond = (a.vocab + kVec<T> - 1) / kVec<T>;
  const auto place = [&](uint32_t i) {  // where vector i of the listed groups is
    return i < vecs ? ((uint32_t)list[i >> lg] << lg) + (i & ((1u << lg) - 1)) : beyond;
  };

  // The logits there that reach the bound, in order; those past kCap are
  // counted only.  NaN is -infinity here; a bound at or below that lets all
  // through.
  const bool all = bound <= key_of<T>(-INFINITY);
  const float least_value = value_of<T>(bound);
  uint32_t n = 0;
  constexpr uint32_t kRun = 4;    // neighbouring vectors a thread and turn
  constexpr uint32_t kTurns = 3;  // loaded together
  for (uint32_t i0 = 0; i0 < vecs; i0 += kTurns * kRun * kFinT) {
    u32x4 raw[kTurns][kRun];
    uint32_t hits[kTurns];
#pragma unroll
    for (uint32_t t = 0; t < kTurns; ++t)
      if (i0 + t * kRun * kFinT < vecs) {
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u)
          raw[t][u] = load_row(p, place(i0 + (t * kFinT + tid) * kRun + u), a.vocab);
      }
#pragma unroll
    for (uint32_t t = 0; t < kTurns; ++t) {
      hits[t] = 0;
      if (i0 + t * kRun * kFinT < vecs) {
#pragma unroll
        for (uint32_t u = 0; u < kRun; ++u) {
          const uint32_t id = place(i0 + (t * kFinT + tid) * kRun + u) * kVec<T>;
          float x[kVec<T>];
          to_float<T>(raw[t][u], x);
          uint32_t h = 0;
#pragma unroll
          for (int e = 0; e < kVec<T>; ++e) h |= (all || x[e] >= least_value ? 1u : 0u) << e;
          if (id + kVec<T> > a.vocab) h &= id < a.vocab ? (1u << (a.vocab - id)) - 1u : 0u;
          hits[t] |= h << (u * kVec<T>);
        }
      }
      const uint32_t total = wave_add((uint32_t)__popc(hits[t]));
      if (lane == 0) sh.cells[t][wave] = total;
    }
    scan_cells(sh, kTurns);
#pragma unroll
    for (uint32_t t = 0; t < kTurns; ++t) {
      uint32_t none, at = n + sh.cells[t][wave] + wave_scan((uint32_t)__popc(hits[t]), &none);
      while (hits[t]) {
        const uint32_t bit = (uint32_t)__ffs(hits[t]) - 1u, u = bit / kVec<T>, e = bit % kVec<T>;
        hits[t] &= hits[t] - 1;
        if (at < kCap) {
          const u32x4 v = u < 2 ? (u == 0 ? raw[t][0] : raw[t][1]) : u == 2 ? raw[t][2] : raw[t][3];
          const uint32_t w = e * sizeof(T) / 4;
          const uint32_t word = w < 2 ? (w == 0 ? v.x : v.y) : w == 2 ? v.z : v.w;
          float x;
          if (sizeof(T) == 4) x = __uint_as_float(word);
          else x = (float)__builtin_bit_cast(Half<T>, (uint16_t)(word >> (e & 1) * 16));
          sh.ckey[at] = key_of<T>(x);
          sh.cid[at] = place(i0 + (t * kFinT + tid) * kRun + u) * kVec<T> + e;
        }
        ++at;
      }
    }
    n += sh.all_cells;
    __syncthreads();
  }

  const auto put = [&](uint32_t at, uint32_t id, uint32_t key) {
    const float x = value_of<T>(key);
    a.ids[row * K + at] = (int32_t)id;
    a.logp[row * K + at] = x == -INFINITY && lse == lse ? x : (x - m) - lse;
  };
  reached = n;
  if (n <= kCap) {
    const uint32_t least = largest_reached(sh, K, K, bound, top, 0, n, &reached,
                                           [&](uint32_t i) { return sh.ckey[i]; });
    // neighbouring candidates a thread
    const uint32_t each = (n + kFinT - 1) / kFinT, c0 = min(tid * each, n), c1 = min(c0 + each, n);
    uint32_t gt = 0, eq = 0, above, ties;
    for (uint32_t i = c0; i < c1; ++i) {
      const uint32_t k = sh.ckey[i];
      gt += k > least;
      eq += k == least;
    }
    block_scan2(sh, gt, eq, &above, &ties);
    ties = K - above;
    for (uint32_t i = c0; i < c1; ++i) {
      const uint32_t k = sh.ckey[i];
      const bool t = k == least;
      if (k > least || (t && eq < ties)) put(gt + min(eq, ties), sh.cid[i], k);
      gt += k > least;
      eq += t;
    }
    return;
  }
  // More logits reach the bound than are held (rows in order, or of few
  // values): the same on the logits in memory.
  const uint32_t size = vecs * kVec<T>;
  const auto logit = [&](uint32_t i, uint32_t* id) -> uint32_t {  // its key; 0: none
    *id = place(i / kVec<T>) * kVec<T> + i % kVec<T>;
    return *id < a.vocab ? key_of<T>((float)p[*id]) : 0u;
  };
  const uint32_t least = largest_reached(sh, K, K, bound, top, 0, size, &reached, [&](uint32_t i) {
    uint32_t id;
    return logit(i, &id);
  });
  uint32_t ties = K;
  for (int pass = 0; pass < 2; ++pass) {  // counts, then writes
    uint32_t gt = 0, eq = 0;
    for (uint32_t i0 = 0; i0 < size; i0 += kFinT) {
      uint32_t id = 0;
      const uint32_t k = i0 + tid < size ? logit(i0 + tid, &id) : 0u;
      uint32_t g = k > least, q = k != 0 && k == least, all_g, all_q;
      const bool any = g || q;
      block_scan2(sh, g, q, &all_g, &all_q);
      g += gt;
      q += eq;
      if (pass && any && (k > least || q < ties)) put(g + min(q, ties), id, k);
      gt += all_g;
      eq += all_q;
    }
    ties = K - gt;
  }
}

template <typename T>
__device__ __forceinline__ void set_row_sum(Shared& sh, MaxSum ms) {
  ms = wave_merge(ms);
  if ((threadIdx.x & 63) == 0) {
    sh.m = exp_base(ms.m);
    sh.lse = logf(ms.s);
  }
}

// A row's end.  kLds: the groups' keys fit there.
template <typename T, bool kLds>
__global__ void __launch_bounds__(kFinT) propose_finish(Args a) {
  __shared__ Shared sh;
  __shared__ uint16_t list[kMaxListed];
  __shared__ __attribute__((aligned(16))) Key<T> keys[kLds ? kKeyBytes / sizeof(T) : 1];
  const uint64_t row = blockIdx.x;
  const T* gmax = (const T*)a.gmax + row * a.groups;
  if (kLds) {
    const uint32_t vecs = (a.groups + kVec<T> - 1) / kVec<T>;
    for (uint32_t v = threadIdx.x; v < vecs; v += kFinT) {
      const uint32_t g = v * kVec<T>;
      const u32x4 raw = g + kVec<T> <= a.groups ? load_vec(gmax + g)
                                                : load_part(gmax + g, (int)(a.groups - g), (T)0.0f);
      float x[kVec<T>];
      to_float<T>(raw, x);
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e) keys[g + e] = (Key<T>)key_of<T>(x[e]);
    }
  }
  if (threadIdx.x < 64) {
    MaxSum ms{-INFINITY, 0.0f};
    for (uint32_t i = threadIdx.x; i < a.chunks; i += 64)
      ms = merge(ms, a.part[row * a.chunks + i]);
    set_row_sum<T>(sh, ms);
  }
  __syncthreads();
  finish_row<T, kLds>(sh, list, a, row, a.groups, a.lanes_log2, keys, [&](uint32_t g) -> uint32_t {
    return kLds ? (uint32_t)keys[g] : key_of<T>((float)gmax[g]);
  });
}

// A whole row in one workgroup; the groups are its vectors.
template <typename T>
__global__ void __launch_bounds__(kFinT) propose_row(Args a) {
  __shared__ Shared sh;
  __shared__ uint16_t list[kMaxListed];
  __shared__ __attribute__((aligned(16))) Key<T> keys[kRowVecs];
  const uint64_t row = blockIdx.x;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const T* p = row_of<T>(a, row);
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  MaxSum ms{-INFINITY, 0.0f};
  for (uint32_t v = tid; v < vecs; v += kScanU * kFinT) {
    u32x4 raw[kScanU];
    load_run<kScanU>(raw, p, v, kFinT, a.vocab, (T)-INFINITY,
                     (v - tid + kScanU * kFinT) * kVec<T> <= a.vocab);
#pragma unroll
    for (int u = 0; u < kScanU; ++u) {
      float x[kVec<T>];
      to_float<T>(raw[u], x);
      float g = x[0];
#pragma unroll
      for (int e = 1; e < kVec<T>; ++e) g = fmaxf(g, x[e]);
      if (v + u * kFinT < vecs) keys[v + u * kFinT] = (Key<T>)key_of<T>(g);
      add_terms(ms, x);
    }
  }
  ms = wave_merge(ms);
  if (lane == 0) sh.ms[wave] = ms;
  __syncthreads();
  if (wave == 0) {
    ms = lane < kFinWaves ? sh.ms[lane] : MaxSum{-INFINITY, 0.0f};
    set_row_sum<T>(sh, ms);
  }
  __syncthreads();
  finish_row<T, true>(sh, list, a, row, vecs, 0, keys, [&](uint32_t g) -> uint32_t { return keys[g]; });
}

template <typename T>
hipError_t launch(const ft_propose_args& a, uint8_t* ws, hipStream_t s) {
  const ScanPlan p = plan<T>(a);
  Args k{};
  k.logits = a.logits;
  k.steps = a.steps;
  k.stride[0] = a.stride[0];
  k.stride[1] = a.stride[1];
  k.vocab = a.vocab;
  k.topk = a.topk;
  k.lanes_log2 = p.lanes_log2;
  k.groups = p.groups;
  k.chunks = p.chunks;
  k.chunk_vecs = p.chunk_vecs;
  k.gmax = ws + p.gmax;
  k.part = (MaxSum*)(ws + p.part);
  k.ids = a.ids;
  k.logp = a.logp;
  const uint32_t rows = (uint32_t)(a.batch * a.steps);
  // One launch, a row a workgroup, up to 8192 vectors a row (128 rows of
  // 32,768 bf16, 1000 each: 16.6 us, in two launches 18.5; 8 of 32,768 f32:
  // 14.5, 15.5), and up to 16384 where the rows fill the chip (256 of 100,003
  // f16: 22.9, 26.2; but 39 of them: 20.5, 18.8).
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  if (vecs <= (rows >= 256 ? kRowVecs : kRowVecs / 2))
    return start(propose_row<T>, rows, kFinT, s, k);
  const hipError_t e = start(propose_scan<T>, (uint64_t)rows * p.chunks, kScanT, s, k);
  if (e != hipSuccess) return e;
  if (p.groups <= kKeyBytes / sizeof(T)) return start(propose_finish<T, true>, rows, kFinT, s, k);
  return start(propose_finish<T, false>, rows, kFinT, s, k);
}

}  // namespace

uint64_t propose_workspace(const ft_propose_args& a) {
  switch (a.dtype) {
    case FT_F32: return plan<float>(a).bytes;
    case FT_F16: return plan<_Float16>(a).bytes;
    default: return plan<__bf16>(a).bytes;
  }
}

hipError_t launch_propose(const ft_propose_args& a, uint8_t* ws, hipStream_t s) {
  if (a.batch == 0 || a.steps == 0) return hipSuccess;
  switch (a.dtype) {
    case FT_F32: return launch<float>(a, ws, s);
    case FT_F16: return launch<_Float16>(a, ws, s);
    default: return launch<__bf16>(a, ws, s);
  }
}

}  // namespace fto
