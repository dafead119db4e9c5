// propose.hip -- proposal rows from logits: the topk largest of each row in
// ascending token order, with their log-probabilities.
//
// One pass over the logits gives each row's (max, sum of exponentials) and
// the maximum of every group of G neighbouring logits.  The topk-th largest
// group maximum, T, is a lower bound of the topk-th largest logit, and topk
// groups hold every logit that can be proposed: the groups whose maximum is
// above T (fewer than topk; all logits above T lie in them), and of those
// whose maximum is T the first ones up to topk in all (each holds one T, so
// the lowest ids among the logits equal to T are in them).  Only these
// groups are read again: topk * G of the row's logits, whatever the data.
// Selections are by counting: the largest key that at least topk keys reach
// is bisected with ballots over keys in registers, with no atomics and no
// sort, and rows are written by ordered compaction, ascending as they are.
#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

constexpr int kScanT = 256;     // threads of a scanning workgroup
constexpr int kScanU = 4;       // vectors in flight a thread
constexpr int kFinT = 1024;     // of a finishing one
constexpr int kFinWaves = kFinT / 64;
constexpr uint32_t kMaxGroups = 65536;  // of a row: 64 keys a thread
constexpr uint32_t kCap = 8192;         // candidates held in LDS

struct ScanPlan {
  uint32_t lanes_log2;   // lanes of a group: G = kVec << lanes_log2
  uint32_t groups;       // of a row
  uint32_t chunks;       // workgroups of a row
  uint32_t chunk_vecs;   // vectors of a workgroup
  uint64_t gmax, part;   // workspace offsets
  uint64_t bytes;
};

// Groups: as long as leaves four of them a proposal (the bound T is then
// close: about 1.15 topk logits reach it in random rows), at most 64 logits
// (one or two lines; longer only to stay within kMaxGroups).  Chunks: about
// 4096 workgroups in all, in whole turns of its loads.
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
  const uint32_t e = vec * kVec<T>;
  if (e + kVec<T> <= vocab) return load_vec(p + e);
  return load_part(p + (e < vocab ? e : 0u), e < vocab ? (int)(vocab - e) : 0, (T)-INFINITY);
}

// Block (row, chunk).
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
#pragma unroll
    for (int u = 0; u < kScanU; ++u) raw[u] = load_row(p, v + u * kScanT + tid, a.vocab);
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

// Keys are the type's own order: the float's, without the bits that are
// the same for every value of the type.
template <typename T>
constexpr int kShift = sizeof(T) == 4 ? 0 : 13;
template <>
constexpr int kShift<__bf16> = 16;

template <typename T>
__device__ __forceinline__ uint32_t key_of(float x) {
  return order_key(x) >> kShift<T>;
}
template <typename T>
__device__ __forceinline__ float value_of(uint32_t k) {
  // (a negative value's dropped bits are ones)
  k <<= kShift<T>;
  if (!(k & 0x80000000u)) k |= (1u << kShift<T>) - 1u;
  return key_value(k);
}

struct FinShared {
  uint32_t count[2][3][kFinWaves];
  uint32_t scan[2][kFinWaves];
  float lse, m;
};

// The largest key that at least `need` of all keys reach (0 if fewer reach
// any): count(t1, t2, t3, out) adds up how many of this wave's keys reach
// each bound; three bounds a round, so two bits.
template <typename F>
__device__ __forceinline__ uint32_t nth_largest(FinShared& sh, uint32_t need, uint32_t top,
                                                F&& count) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t lo = 0, hi = top;  // reached by enough; not
  for (int round = 0; hi - lo > 1; ++round) {
    const uint32_t d = hi - lo, q = d >> 2;
    const uint32_t t2 = lo + (d >> 1), t1 = q ? lo + q : t2, t3 = q ? t2 + q : t2;
    uint32_t n[3] = {0, 0, 0};
    count(t1, t2, t3, n);
    if (lane == 0)
      for (int i = 0; i < 3; ++i) sh.count[round & 1][i][wave] = n[i];
    __syncthreads();
    uint32_t s[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      s[i] = lane < kFinWaves ? sh.count[round & 1][i][lane] : 0;
#pragma unroll
      for (int k = 1; k < kFinWaves; k <<= 1) s[i] += (uint32_t)__shfl_xor((int)s[i], k, 64);
      s[i] = (uint32_t)__builtin_amdgcn_readfirstlane((int)s[i]);
    }
    if (s[2] >= need) lo = t3;
    else if (s[1] >= need) lo = t2, hi = t3;
    else if (s[0] >= need) lo = t1, hi = t2;
    else hi = t1;
  }
  __syncthreads();
  return lo;
}

// Sums over the threads in front of (a, b); every thread of the block.
__device__ __forceinline__ void block_scan2(FinShared& sh, uint32_t& a, uint32_t& b,
                                            uint32_t* total_a) {
  const uint32_t wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  uint32_t ta, tb;
  a = wave_scan(a, lane, &ta);
  b = wave_scan(b, lane, &tb);
  if (lane == 0) {
    sh.scan[0][wave] = ta;
    sh.scan[1][wave] = tb;
  }
  __syncthreads();
  uint32_t all = 0;
  for (uint32_t w = 0; w < kFinWaves; ++w) {
    const uint32_t wa = sh.scan[0][w], wb = sh.scan[1][w];
    all += wa;
    if (w < wave) {
      a += wa;
      b += wb;
    }
  }
  *total_a = all;
  __syncthreads();
}

// A row's end: kK group keys a thread.
template <typename T, int kK>
__global__ void __launch_bounds__(kFinT) propose_finish(Args a) {
  __shared__ FinShared sh;
  __shared__ uint32_t list[FT_MAX_PROPOSALS];
  __shared__ uint32_t ckey[kCap], cid[kCap];
  const uint64_t row = blockIdx.x;
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, K = a.topk;
  const T* p = row_of<T>(a, row);
  const T* gmax = (const T*)a.gmax + row * a.groups;

  // the groups' keys, kK neighbours a thread
  uint32_t gk[kK];
#pragma unroll
  for (int i = 0; i < kK; ++i) {
    const uint32_t g = tid * kK + i;
    gk[i] = g < a.groups ? key_of<T>((float)gmax[g]) : 0u;
  }
  // the row's sum
  if (wave == 0) {
    MaxSum ms{-INFINITY, 0.0f};
    for (uint32_t i = lane; i < a.chunks; i += 64) ms = merge(ms, a.part[row * a.chunks + i]);
    ms = wave_merge(ms);
    if (lane == 0) {
      sh.m = exp_base(ms.m);
      sh.lse = logf(ms.s);
    }
  }
  __syncthreads();

  const uint32_t top = key_of<T>(INFINITY) + 1;
  uint32_t bound = 0;  // T
  if (a.groups > K)
    bound = nth_largest(sh, K, top, [&](uint32_t t1, uint32_t t2, uint32_t t3, uint32_t (&n)[3]) {
#pragma unroll
      for (int i = 0; i < kK; ++i) {
        n[0] += (uint32_t)__popcll(__ballot(gk[i] >= t1));
        n[1] += (uint32_t)__popcll(__ballot(gk[i] >= t2));
        n[2] += (uint32_t)__popcll(__ballot(gk[i] >= t3));
      }
    });
  // the groups to read again, ascending
  uint32_t above = 0, tied = 0, sel;
#pragma unroll
  for (int i = 0; i < kK; ++i) {
    const uint32_t g = tid * kK + i;
    above += g < a.groups && gk[i] > bound;
    tied += g < a.groups && gk[i] == bound;
  }
  block_scan2(sh, above, tied, &sel);
  {
    const uint32_t ties = K - sel;  // (sel < K, or every group is wanted)
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      const uint32_t g = tid * kK + i;
      if (g >= a.groups) continue;
      const bool t = gk[i] == bound;
      if (gk[i] > bound || (t && tied < ties)) list[above + min(tied, ties)] = g;
      above += gk[i] > bound;
      tied += t;
    }
    sel = min(K, a.groups);
  }
  __syncthreads();

  // the logits of those groups that reach the bound, in order: each wave
  // takes a run of vectors, counts, then writes
  const uint32_t lg = a.lanes_log2, vecs = sel << lg;
  const uint32_t run = (uint32_t)(((uint64_t)vecs + kFinT - 1) / kFinT) * 64;
  const uint32_t r0 = min(wave * run, vecs), r1 = min(r0 + run, vecs);
  auto load = [&](uint32_t i, float (&x)[kVec<T>]) -> uint32_t {  // logits there, their id
    const uint32_t vec = (list[i >> lg] << lg) + (i & ((1u << lg) - 1));
    to_float<T>(load_row(p, vec, a.vocab), x);
    return vec * kVec<T>;
  };
  uint32_t mine = 0, zero = 0, n;
  for (uint32_t i = r0 + lane; i < r1; i += 64) {
    float x[kVec<T>];
    const uint32_t id = load(i, x);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) mine += id + e < a.vocab && key_of<T>(x[e]) >= bound;
  }
  block_scan2(sh, mine, zero, &n);
  const bool held = n <= kCap;
  if (held) {
    // (a thread's logits are not neighbours: the order is by vector, so the
    // wave's offset advances vector row by vector row)
    uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)mine);  // lane 0: the waves in front
    for (uint32_t i0 = r0; i0 < r1; i0 += 64) {
      const uint32_t i = i0 + lane;
      float x[kVec<T>];
      uint32_t id = 0, c = 0, t;
      if (i < r1) {
        id = load(i, x);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e) c += id + e < a.vocab && key_of<T>(x[e]) >= bound;
      }
      uint32_t w = at + wave_scan(c, lane, &t);
      if (c) {
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
          if (id + e < a.vocab && key_of<T>(x[e]) >= bound) {
            ckey[w] = key_of<T>(x[e]);
            cid[w++] = id + e;
          }
      }
      at += t;
    }
  }
  __syncthreads();

  const float m = sh.m, lse = sh.lse;
  const auto put = [&](uint32_t at, uint32_t id, uint32_t key) {
    const float x = value_of<T>(key);
    a.ids[row * K + at] = (int32_t)id;
    a.logp[row * K + at] = x == -INFINITY && lse == lse ? x : (x - m) - lse;
  };
  if (held) {
    // up to 8 neighbouring candidates a thread
    const uint32_t each = (n + kFinT - 1) / kFinT, c0 = min(tid * each, n), c1 = min(c0 + each, n);
    uint32_t k[kCap / kFinT];
#pragma unroll
    for (uint32_t i = 0; i < kCap / kFinT; ++i) k[i] = c0 + i < c1 ? ckey[c0 + i] : 0u;
    const uint32_t least =
        nth_largest(sh, K, top, [&](uint32_t t1, uint32_t t2, uint32_t t3, uint32_t (&cnt)[3]) {
#pragma unroll
          for (uint32_t i = 0; i < kCap / kFinT; ++i) {
            if (i >= each) break;
            cnt[0] += (uint32_t)__popcll(__ballot(k[i] >= t1));
            cnt[1] += (uint32_t)__popcll(__ballot(k[i] >= t2));
            cnt[2] += (uint32_t)__popcll(__ballot(k[i] >= t3));
          }
        });
    uint32_t gt = 0, eq = 0, all;
    for (uint32_t i = 0; c0 + i < c1; ++i) {
      gt += ckey[c0 + i] > least;
      eq += ckey[c0 + i] == least;
    }
    block_scan2(sh, gt, eq, &all);
    const uint32_t ties = K - all;
    for (uint32_t i = c0; i < c1; ++i) {
      const uint32_t key = ckey[i];
      const bool t = key == least;
      if (key > least || (t && eq < ties)) put(gt + min(eq, ties), cid[i], key);
      gt += key > least;
      eq += t;
    }
    return;
  }
  // More than kCap logits reach the bound (rows in order, or of few values):
  // the same on the groups in memory.
  const uint32_t least =
      nth_largest(sh, K, top, [&](uint32_t t1, uint32_t t2, uint32_t t3, uint32_t (&cnt)[3]) {
        for (uint32_t i0 = r0; i0 < r1; i0 += 64) {
          const uint32_t i = i0 + lane;
          float x[kVec<T>];
          uint32_t id = a.vocab;
          if (i < r1) id = load(i, x);
#pragma unroll
          for (int e = 0; e < kVec<T>; ++e) {
            const uint32_t key = i < r1 && id + e < a.vocab ? key_of<T>(x[e]) : 0u;
            cnt[0] += (uint32_t)__popcll(__ballot(key >= t1));
            cnt[1] += (uint32_t)__popcll(__ballot(key >= t2));
            cnt[2] += (uint32_t)__popcll(__ballot(key >= t3));
          }
        }
      });
  uint32_t gt = 0, eq = 0, all;
  for (uint32_t i = r0 + lane; i < r1; i += 64) {
    float x[kVec<T>];
    const uint32_t id = load(i, x);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) {
      const uint32_t key = id + e < a.vocab ? key_of<T>(x[e]) : 0u;
      gt += key > least;
      eq += id + e < a.vocab && key == least;
    }
  }
  block_scan2(sh, gt, eq, &all);
  const uint32_t ties = K - all;
  uint32_t gat = (uint32_t)__builtin_amdgcn_readfirstlane((int)gt);
  uint32_t eat = (uint32_t)__builtin_amdgcn_readfirstlane((int)eq);
  for (uint32_t i0 = r0; i0 < r1; i0 += 64) {
    const uint32_t i = i0 + lane;
    float x[kVec<T>];
    uint32_t id = a.vocab, cg = 0, ce = 0, tg, te;
    if (i < r1) id = load(i, x);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) {
      const bool in = i < r1 && id + e < a.vocab;
      const uint32_t key = in ? key_of<T>(x[e]) : 0u;
      cg += in && key > least;
      ce += in && key == least;
    }
    uint32_t g = gat + wave_scan(cg, lane, &tg), q = eat + wave_scan(ce, lane, &te);
    gat += tg;
    eat += te;
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) {
      if (!(i < r1 && id + e < a.vocab)) continue;
      const uint32_t key = key_of<T>(x[e]);
      const bool t = key == least;
      if (key > least || (t && q < ties)) put(g + min(q, ties), id + e, key);
      g += key > least;
      q += t;
    }
  }
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
  hipLaunchKernelGGL((propose_scan<T>), dim3(rows * p.chunks), dim3(kScanT), 0, s, k);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.groups <= 4 * kFinT)
    hipLaunchKernelGGL((propose_finish<T, 4>), dim3(rows), dim3(kFinT), 0, s, k);
  else if (p.groups <= 16 * kFinT)
    hipLaunchKernelGGL((propose_finish<T, 16>), dim3(rows), dim3(kFinT), 0, s, k);
  else
    hipLaunchKernelGGL((propose_finish<T, 64>), dim3(rows), dim3(kFinT), 0, s, k);
  return hipGetLastError();
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
