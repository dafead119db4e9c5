// key_loss.hip -- the losses on the keys of a search, and their gradient with
// respect to the logits that scored them.
//
// With lp = x[tok] - lse(x) for each token and g = dloss/dlp,
//   dloss/dx[v] = sum over the row's tokens of (tok = v ? g : 0) - p[v] g
//               = (sum of the g's of v) - p[v] G,  p[v] = exp(x[v] - lse),
// so a row needs its lse, G and a short list of (token, summed g); many keys
// share a token at the first positions of a trie.  Results do not depend on
// the order in which threads run: sums are made in a fixed order, or of whole
// numbers.
//
//   key_stats    (row, chunk): (max, sum of exponentials) of the chunk
//   key_scores   16 lanes a key: token scores and the key's margin (preference)
//   key_pairs    64 keys a workgroup: dloss/ds over all pairs, loss's terms
//   key_rows     row: token scores, the loss's terms and g (policy); the list
//                of (token, summed g), and what key_gradient needs of the row
//   key_gradient (row, span): the gradient; block 0 also adds up the loss
//   key_whole    row: all of the policy loss in one workgroup, for rows that
//                fit its registers: the logits are read once
// The gradient is stored as -p G first; then, past a barrier, the list's
// tokens are stored over it.
//
// Bound by the logits: read twice (the second time mostly from the last
// level's cache) and the gradient written, 128 rows x 262,144 bf16 with 1000
// keys a request: 56 us a call; in a trace 17 the statistics at 3.9 TB/s, 12
// the rows' tables and 23 the gradient at 5.9 TB/s; or read once by key_whole,
// 2048 rows x 32,768 bf16: 58 us a call on new inputs, 4.7 TB/s (in a trace,
// with a part of the logits in the last level's cache, 44).  Few rows are bound
// by latency: 8 rows x 32,768 f32, 10 keys: 16 us for 2 MB.
#include <type_traits>

#include "op_device.h"
#include "operators.h"

namespace fto {
namespace {

constexpr int kStatT = 256;
constexpr int kStatU = 4;   // vectors in flight a thread
constexpr int kListT = 1024;

// logits of a workgroup of key_gradient
template <typename T>
constexpr uint32_t span_of() {
  return kStatU * kStatT * kVec<T>;
}

struct RowInfo;
struct Args {
  const void* logits;
  int64_t stride[2];
  void* dlogits;
  int64_t dstride[2];
  uint32_t batch, steps, vocab, keys, rows, chunks, chunk_vecs;
  const int32_t* tokens;
  const int32_t* lengths;
  float* logp;
  float* loss;
  const float* old_logp;
  const float* ref_logp;
  const float* advantage;
  const float* weight;
  float low, high, kl;  // clip bounds, KL coefficient
  uint64_t pairs;
  const int32_t* pair;
  float beta, smoothing;
  // workspace
  MaxSum* part;      // [rows, chunks]
  float* g;          // [rows]: dloss/dlp of the row's token (policy, keys = 1)
  float* margin;     // [batch * keys] (preference)
  float* gkey;       // [batch * keys]: dloss/ds (preference)
  float* terms;      // [nterms]: parts of the loss
  uint32_t nterms;
  RowInfo* info;      // [rows] (keys > 1)
  uint32_t* ltok;    // [rows, keys]
  float* lg;         // [rows, keys]
  uint32_t* from;    // [rows, spans + 1]: the list's entries of each span
  uint32_t spans;
};

// What key_gradient needs of a row: p G = scale exp(x - base).
struct RowInfo {
  float base, scale;
  uint32_t used;
};

// A row of nothing but -infinity has s = 0 and probability nowhere.
__device__ __forceinline__ float row_scale(float total, float s) {
  return s == 0.0f ? total * 0.0f : total / s;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const Args& a, uint32_t row) {
  const uint32_t r = row / a.steps, t = row - r * a.steps;
  return (const T*)a.logits + (int64_t)r * a.stride[0] + (int64_t)t * a.stride[1];
}

__device__ __forceinline__ uint32_t length_of(const Args& a, uint32_t key) {
  const int32_t n = a.lengths[key];
  return n < 0 ? 0u : min((uint32_t)n, a.steps);
}

// Whether row (r, t) scores any token; every thread of the block.
__device__ __forceinline__ bool row_used(const Args& a, uint32_t row) {
  const uint32_t r = row / a.steps, t = row - r * a.steps;
  bool any = false;
  for (uint32_t c = threadIdx.x; c < a.keys; c += blockDim.x)
    any = any || length_of(a, r * a.keys + c) > t;
  return __syncthreads_or(any);
}

// Block (row, chunk).  Rows without a token are not read.
template <typename T>
__global__ void __launch_bounds__(kStatT) key_stats(Args a) {
  const uint32_t row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
  const uint32_t tid = threadIdx.x;
  if (!row_used(a, row)) return;
  const T* p = row_of<T>(a, row);
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  const uint32_t v0 = chunk * a.chunk_vecs, v1 = min(v0 + a.chunk_vecs, vecs);
  MaxSum ms{-INFINITY, 0.0f};
  for (uint32_t v = v0; v < v1; v += kStatU * kStatT) {
    u32x4 raw[kStatU];
    load_run<kStatU>(raw, p, v + tid, kStatT, a.vocab, (T)-INFINITY,
                     (v + kStatU * kStatT) * kVec<T> <= a.vocab);
#pragma unroll
    for (int u = 0; u < kStatU; ++u) {
      float x[kVec<T>];
      to_float<T>(raw[u], x);
      add_terms(ms, x);
    }
  }
  ms = wave_merge(ms);
  __shared__ MaxSum waves[kStatT / 64];
  if ((tid & 63) == 0) waves[tid >> 6] = ms;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kStatT / 64; ++w) ms = merge(ms, waves[w]);
    a.part[(uint64_t)row * a.chunks + chunk] = ms;
  }
}

// The row's (max, sum) from its chunks' parts: by a thread, loads and
// exponentials side by side, or by a wave.
__device__ __forceinline__ MaxSum row_sum(const Args& a, uint32_t row) {
  const MaxSum* part = a.part + (uint64_t)row * a.chunks;
  MaxSum ms{-INFINITY, 0.0f};
#pragma unroll 8
  for (uint32_t i = 0; i < a.chunks; ++i) ms.m = fmaxf(ms.m, part[i].m);
  const float base = exp_base(ms.m);
#pragma unroll 8
  for (uint32_t i = 0; i < a.chunks; ++i) ms.s += part[i].s * exp_term(part[i].m, base);
  return ms;
}
__device__ __forceinline__ MaxSum row_sum_wave(const Args& a, uint32_t row) {
  const MaxSum* part = a.part + (uint64_t)row * a.chunks;
  MaxSum ms{-INFINITY, 0.0f};
  for (uint32_t i = threadIdx.x & 63; i < a.chunks; i += 64) ms = merge(ms, part[i]);
  return wave_merge(ms);
}

// A token's log-probability; NaN for one out of range.
template <typename T>
__device__ __forceinline__ float score(const T* p, int32_t tok, uint32_t vocab, float m, float ls) {
  if ((uint32_t)tok >= vocab) return NAN;
  const float x = (float)p[tok];
  return x == -INFINITY && ls == ls ? x : (x - m) - ls;
}

// The policy loss of one token, and its derivative by lp.
__device__ __forceinline__ float policy_term(const Args& a, uint64_t at, float lp, float adv,
                                             float w, float* g) {
  const float ratio = expf(lp - a.old_logp[at]);
  const float clipped = fminf(fmaxf(ratio, a.low), a.high);
  const float u = ratio * adv, v = clipped * adv;
  const bool moves = !(u > v);  // (NaN too: the loss and gradient show it)
  float each = moves ? -u : -v, d = moves ? -u : 0.0f;
  if (a.kl != 0.0f) {
    const float r = a.ref_logp[at] - lp, e = expm1f(r);
    each += a.kl * (r == INFINITY ? r : e - r);  // (a token whose logit is -infinity)
    d -= a.kl * e;
  }
  *g = w * d;
  return w * each;
}

__device__ __forceinline__ float block_sum(float v, float* waves) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0f;
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) v += waves[w];
  __syncthreads();
  return v;
}

// The block's sums of a and b and its largest c.
__device__ __forceinline__ void block_sums(float& a, float& b, float& c, float (*waves)[3]) {
  a = wave_sum(a);
  b = wave_sum(b);
  c = wave_max(c);
  if ((threadIdx.x & 63) == 0) {
    float* w = waves[threadIdx.x >> 6];
    w[0] = a;
    w[1] = b;
    w[2] = c;
  }
  __syncthreads();
  a = b = c = 0.0f;
  for (uint32_t w = 0; w < blockDim.x / 64; ++w) {
    a += waves[w][0];
    b += waves[w][1];
    c = fmaxf(c, waves[w][2]);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) key_scores(Args a) {
  const uint32_t key = blockIdx.x * 16 + (threadIdx.x >> 4), lane = threadIdx.x & 15;
  if (key >= a.batch * a.keys) return;
  const uint32_t r = key / a.keys, len = length_of(a, key);
  float sum = 0.0f;
  for (uint32_t t = lane; t < a.steps; t += 16) {
    const uint64_t at = (uint64_t)key * a.steps + t;
    float lp = 0.0f;
    if (t < len) {
      const MaxSum ms = row_sum(a, r * a.steps + t);
      lp = score(row_of<T>(a, r * a.steps + t), a.tokens[at], a.vocab, exp_base(ms.m), logf(ms.s));
    }
    a.logp[at] = lp;
    sum += lp;
  }
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d, 64);
  if (lane == 0) a.margin[key] = sum - a.ref_logp[key];
}

// Wave w of a workgroup takes the pairs of its share in their order, one at
// a time for its 64 keys, a key a lane; the waves' sums are added in order.
// So its time goes with keys times pairs: 96 rows x 262,144 bf16, 8000 keys:
// the whole call 57 us with 400 pairs, 84 with 4000, 304 with 32,000.
__global__ void __launch_bounds__(1024) key_pairs(Args a) {
  __shared__ float sums[16][64];
  __shared__ float waves[16];
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t keys = a.batch * a.keys, key = blockIdx.x * 64 + lane;
  const uint64_t each = (a.pairs + 15) / 16;
  const uint64_t p0 = wave * each, p1 = min(p0 + each, a.pairs);
  float g = 0.0f, loss = 0.0f;
  for (uint64_t q = p0; q < p1; q += 64) {
    // a pair a lane: its derivative
    uint32_t ka = ~0u, kb = ~0u;
    float d = 0.0f;
    if (q + lane < p1) {
      ka = (uint32_t)a.pair[2 * (q + lane)];
      kb = (uint32_t)a.pair[2 * (q + lane) + 1];
      const float w = a.weight[q + lane];
      const float h =
          ka < keys && kb < keys ? a.beta * (a.margin[ka] - a.margin[kb]) : NAN;
      // sigmoid(h) and softplus(-h), softplus(h) without overflow
      const float e = expf(-fabsf(h)), tail = log1pf(e);
      const float sig = (h >= 0.0f ? 1.0f : e) / (1.0f + e);
      d = w * a.beta * (sig - (1.0f - a.smoothing));
      const float won = tail + (h < 0.0f ? -h : 0.0f), lost = tail + (h > 0.0f ? h : 0.0f);
      // (one of the two is infinite where h is, and counts only with a share)
      const float kept = 1.0f - a.smoothing;
      loss += w * ((kept > 0.0f ? kept * won : 0.0f) +
                   (a.smoothing > 0.0f ? a.smoothing * lost : 0.0f));
    }
    const uint32_t n = (uint32_t)min((uint64_t)64, p1 - q);
    for (uint32_t i = 0; i < n; ++i) {
      const uint32_t pa = (uint32_t)__builtin_amdgcn_readlane((int)ka, (int)i);
      const uint32_t pb = (uint32_t)__builtin_amdgcn_readlane((int)kb, (int)i);
      const float pd = __uint_as_float(
          (uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(d), (int)i));
      if (pa == key) g += pd;
      if (pb == key) g -= pd;
    }
  }
  sums[wave][lane] = g;
  __syncthreads();
  if (wave == 0) {
    g = 0.0f;
    for (int w = 0; w < 16; ++w) g += sums[w][lane];
    if (key < keys) a.gkey[key] = g;
  }
  if (blockIdx.x == 0) {
    loss = block_sum(loss, waves);
    if (tid == 0) a.terms[0] = loss;
  }
}

// A row's tokens and the sums of their slopes: a hash table.  Sums are whole
// numbers of 2^-kBits of the row's largest slope, so that they do not depend
// on the order of the atomics and are finer than a 32-bit sum's roundings.
// All of a row's slopes may be the largest, of one sign and of one token
// (keys of a prefix, an advantage for all): kP * 1024 times 2^kBits is 2^62.
template <int kP>
struct Table {
  static constexpr uint32_t kSlots = 2 * kListT * kP;
  static constexpr int kBits = kP == 1 ? 52 : 50;
  static_assert((uint64_t)kListT * kP << kBits <= 1ull << 62, "a row's slopes fit a sum");
  static constexpr double kOne = (double)(1ull << kBits);
  uint32_t tok[kSlots];  // ~0: free
  unsigned long long sum[kSlots];
  float waves[kListT / 64][3];
};

// The keys' scores and slopes of row (r, t) and the loss's terms (policy),
// and the table of its tokens, whose sums count *unit each.  *total = G,
// *loss the row's terms.
template <typename T, bool kPolicy, int kP>
__device__ __forceinline__ void row_table(const Args& a, Table<kP>& sh, uint32_t row, float m, float ls,
                                          float* total, float* loss, double* unit) {
  const uint32_t r = row / a.steps, t = row - r * a.steps, tid = threadIdx.x;
  const T* p = row_of<T>(a, row);
  if (a.dlogits)
    for (uint32_t i = tid; i < Table<kP>::kSlots; i += kListT) {
      sh.tok[i] = ~0u;
      sh.sum[i] = 0;
    }
  float sum = 0.0f, terms = 0.0f, most = 0.0f, gs[kP];
  uint32_t toks[kP];
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    const uint32_t c = i * kListT + tid;
    gs[i] = 0.0f;
    toks[i] = ~0u;
    if (c < a.keys) {
      const uint32_t key = r * a.keys + c;
      const uint64_t at = (uint64_t)key * a.steps + t;
      // (read before the length is known: the arrays hold it)
      const int32_t tok = a.tokens[at];
      const bool in = length_of(a, key) > t;
      float lp = 0.0f;
      if (kPolicy) {
        if (in) {
          lp = score(p, tok, a.vocab, m, ls);
          terms += policy_term(a, at, lp, a.advantage[key], a.weight[key], &gs[i]);
        }
        a.logp[at] = lp;
      } else if (in) {
        gs[i] = a.gkey[key];
      }
      if (in && (uint32_t)tok < a.vocab) toks[i] = (uint32_t)tok;
      sum += gs[i];
      most = fmaxf(most, fabsf(gs[i]));
    }
  }
  block_sums(sum, terms, most, sh.waves);
  *total = sum;
  *loss = terms;
  if (!a.dlogits) return;
  // (a slope that is not finite makes the sums NaN)
  const bool finite = fabsf(*total) < INFINITY && most < INFINITY;
  const double scale = most > 0.0f ? Table<kP>::kOne / (double)most : 0.0;
  *unit = finite ? (double)most / Table<kP>::kOne : (double)NAN;
#pragma unroll
  for (int i = 0; i < kP; ++i) {
    if (toks[i] == ~0u) continue;
    uint32_t h = toks[i] * 2654435761u % Table<kP>::kSlots;
    for (;;) {  // (half the slots stay free)
      const uint32_t old = atomicCAS(&sh.tok[h], ~0u, toks[i]);
      if (old == ~0u || old == toks[i]) break;
      h = (h + 1) % Table<kP>::kSlots;
    }
    if (finite) atomicAdd(&sh.sum[h], (unsigned long long)(long long)rint((double)gs[i] * scale));
  }
  __syncthreads();
}

// A row of a request's keys: the table's entries by span.
constexpr uint32_t kMaxSpans = 4096;  // of 2^24 logits

template <typename T, bool kPolicy, int kP>
__global__ void __launch_bounds__(kListT) key_rows(Args a) {
  static_assert((1u << 24) / span_of<T>() <= kMaxSpans, "counters of the spans");
  __shared__ Table<kP> sh;
  __shared__ uint32_t count[kMaxSpans], waves[kListT / 64];
  const uint32_t row = blockIdx.x, tid = threadIdx.x;
  const bool used = row_used(a, row);
  MaxSum ms{0.0f, 1.0f};
  if (used) ms = row_sum_wave(a, row);
  const float base = exp_base(ms.m);
  float total, loss = 0.0f;
  double unit = 0.0;
  for (uint32_t i = tid; i < a.spans; i += kListT) count[i] = 0;
  row_table<T, kPolicy, kP>(a, sh, row, base, logf(ms.s), &total, &loss, &unit);
  if (tid == 0) {
    if (kPolicy) a.terms[row] = loss;
    a.info[row] = RowInfo{base, row_scale(total, ms.s), used};
  }
  if (!a.dlogits) return;
  for (uint32_t i = tid; i < Table<kP>::kSlots; i += kListT)
    if (sh.tok[i] != ~0u) atomicAdd(&count[sh.tok[i] / span_of<T>()], 1u);
  __syncthreads();
  // exclusive sums over the spans, neighbours a thread
  uint32_t* from = a.from + (uint64_t)row * (a.spans + 1);
  const uint32_t each = (a.spans + kListT - 1) / kListT;
  const uint32_t s0 = min(tid * each, a.spans), s1 = min(s0 + each, a.spans);
  uint32_t sum = 0, all;
  for (uint32_t i = s0; i < s1; ++i) sum += count[i];
  uint32_t front = wave_scan(sum, &all);
  if ((tid & 63) == 0) waves[tid >> 6] = all;
  __syncthreads();
#pragma unroll 1
  for (uint32_t w = 0; w < tid >> 6; ++w) front += waves[w];
  for (uint32_t i = s0; i < s1; ++i) {
    const uint32_t n = count[i];
    count[i] = from[i] = front;
    front += n;
  }
  if (tid == kListT - 1) from[a.spans] = front;
  __syncthreads();
  for (uint32_t i = tid; i < Table<kP>::kSlots; i += kListT)
    if (sh.tok[i] != ~0u) {
      const uint32_t at = atomicAdd(&count[sh.tok[i] / span_of<T>()], 1u);
      a.ltok[(uint64_t)row * a.keys + at] = sh.tok[i];
      a.lg[(uint64_t)row * a.keys + at] = (float)((double)(long long)sh.sum[i] * unit);
    }
}

// Policy, one key a request: a row a thread.
template <typename T>
__global__ void __launch_bounds__(256) key_single(Args a) {
  const uint32_t row = blockIdx.x * 256 + threadIdx.x;
  if (row >= a.rows) return;
  const uint32_t r = row / a.steps, t = row - r * a.steps;
  float lp = 0.0f, g = 0.0f, term = 0.0f;
  if (length_of(a, r) > t) {
    const MaxSum ms = row_sum(a, row);
    lp = score(row_of<T>(a, row), a.tokens[row], a.vocab, exp_base(ms.m), logf(ms.s));
    term = policy_term(a, row, lp, a.advantage[r], a.weight[r], &g);
  }
  a.logp[row] = lp;
  a.g[row] = g;
  a.terms[row] = term;
}

__device__ __forceinline__ void add_loss(const Args& a, float* waves) {
  float v = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.nterms; i += blockDim.x) v += a.terms[i];
  v = block_sum(v, waves);
  if (threadIdx.x == 0) *a.loss = v;
}

__global__ void __launch_bounds__(256) key_loss(Args a) {
  __shared__ float waves[4];
  add_loss(a, waves);
}

// A vector of -p G.
template <typename T>
__device__ __forceinline__ void store_plain(T* out, uint32_t vec, uint32_t vocab, const RowInfo& info,
                                            u32x4 raw, bool whole) {
  const uint32_t e = vec * kVec<T>;
  float x[kVec<T>];
  to_float<T>(raw, x);
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) x[i] = info.used ? -info.scale * exp_term(x[i], info.base) : 0.0f;
  const u32x4 o = from_float<T>(x);
  if (whole || e + kVec<T> <= vocab) store_vec(out + e, o);
  else store_part(out + e, (int)(vocab - e), o);
}

// Past this, the block's stores are in memory's order before its later ones.
__device__ __forceinline__ void stores_done() {
  __builtin_amdgcn_s_waitcnt(0);
  __threadfence_block();
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void store_token(const T* p, T* out, uint32_t tok, float g,
                                            const RowInfo& info) {
  out[tok] = (T)(g - info.scale * exp_term((float)p[tok], info.base));
}

// Block (row, span): kStatU vectors a thread, in one go.
template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kStatT) key_gradient(Args a) {
  __shared__ float waves[kStatT / 64];
  const uint32_t row = blockIdx.x / a.spans, span = blockIdx.x - row * a.spans, tid = threadIdx.x;
  const uint32_t r = row / a.steps, t = row - r * a.steps;
  if (blockIdx.x == 0) add_loss(a, waves);
  const T* p = row_of<T>(a, row);
  T* out = (T*)a.dlogits + (int64_t)r * a.dstride[0] + (int64_t)t * a.dstride[1];
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  const uint32_t v0 = span * kStatU * kStatT, e0 = v0 * kVec<T>;
  RowInfo info;
  const uint32_t* ltok = a.ltok + (uint64_t)row * a.keys;
  const float* lg = a.lg + (uint64_t)row * a.keys;
  uint32_t l0 = 0, l1 = 0;
  if (a.keys == 1) {
    info = RowInfo{0.0f, 0.0f, length_of(a, r) > t};
    if (info.used) {
      const MaxSum ms = row_sum_wave(a, row);
      info.base = exp_base(ms.m);
      lg = kPolicy ? a.g + row : a.gkey + r;
      info.scale = row_scale(*lg, ms.s);
      ltok = (const uint32_t*)a.tokens + row;
      const uint32_t tok = *ltok;
      l1 = tok < a.vocab && tok >= e0 && tok - e0 < span_of<T>();
    }
  } else {
    info = a.info[row];
    const uint32_t* from = a.from + (uint64_t)row * (a.spans + 1) + span;
    l0 = from[0];
    l1 = from[1];
  }
  u32x4 raw[kStatU];
  const bool whole = (v0 + kStatU * kStatT) * kVec<T> <= a.vocab;
  if (info.used) load_run<kStatU>(raw, p, v0 + tid, kStatT, a.vocab, (T)-INFINITY, whole);
#pragma unroll
  for (int u = 0; u < kStatU; ++u) {
    const uint32_t vec = v0 + u * kStatT + tid;
    if (whole || vec < vecs) store_plain(out, vec, a.vocab, info, raw[u], whole);
  }
  if (l1 > l0) {
    stores_done();
    for (uint32_t i = l0 + tid; i < l1; i += kStatT) store_token(p, out, ltok[i], lg[i], info);
  }
}

// The policy loss of a row, kU vectors of it a thread of kT.  kMany: several
// keys (kT = kListT).
template <typename T, bool kMany, int kT, int kU>
__global__ void __launch_bounds__(kT) key_whole(Args a) {
  __shared__ std::conditional_t<kMany, Table<1>, int> sh;
  __shared__ MaxSum waves[kT / 64];
  const uint32_t row = blockIdx.x, r = row / a.steps, t = row - r * a.steps, tid = threadIdx.x;
  const T* p = row_of<T>(a, row);
  T* out = (T*)a.dlogits + (int64_t)r * a.dstride[0] + (int64_t)t * a.dstride[1];
  const uint32_t vecs = (a.vocab + kVec<T> - 1) / kVec<T>;
  const bool used = kMany ? row_used(a, row) : length_of(a, r) > t;
  const bool whole = (uint32_t)(kU * kT * kVec<T>) <= a.vocab;
  u32x4 raw[kU];
  MaxSum ms{-INFINITY, 0.0f};
  if (used) {
    load_run<kU>(raw, p, tid, kT, a.vocab, (T)-INFINITY, whole);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float x[kVec<T>];
      repack(raw[u]);
      to_float<T>(raw[u], x);
      add_terms(ms, x);
    }
    ms = wave_merge(ms);
    if ((tid & 63) == 0) waves[tid >> 6] = ms;
    __syncthreads();
    ms = wave_merge(tid % 64 < kT / 64 ? waves[tid % 64] : MaxSum{-INFINITY, 0.0f});
  } else {
    ms = MaxSum{0.0f, 1.0f};
  }
  const float base = exp_base(ms.m), ls = logf(ms.s);
  float total = 0.0f, loss = 0.0f;
  double unit = 0.0;
  int32_t tok = -1;
  if constexpr (kMany) {
    row_table<T, true, 1>(a, sh, row, base, ls, &total, &loss, &unit);
  } else {  // every thread for itself
    float lp = 0.0f;
    if (used) {
      tok = a.tokens[row];
      lp = score(p, tok, a.vocab, base, ls);
      loss = policy_term(a, row, lp, a.advantage[r], a.weight[r], &total);
    }
    if (tid == 0) a.logp[row] = lp;
  }
  if (tid == 0) a.terms[row] = loss;
  if (!a.dlogits) return;
  const RowInfo info{base, row_scale(total, ms.s), used};
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t vec = u * kT + tid;
    repack(raw[u]);
    if (whole || vec < vecs) store_plain(out, vec, a.vocab, info, raw[u], whole);
  }
  if (!used) return;
  stores_done();
  if constexpr (kMany) {
    for (uint32_t i = tid; i < Table<1>::kSlots; i += kT)
      if (sh.tok[i] != ~0u)
        store_token(p, out, sh.tok[i], (float)((double)(long long)sh.sum[i] * unit), info);
  } else if (tid == 0 && (uint32_t)tok < a.vocab) {
    store_token(p, out, (uint32_t)tok, total, info);
  }
}

struct Plan {
  uint32_t vecs, chunks, chunk_vecs, spans;
  uint64_t part, g, margin, gkey, terms, info, ltok, lg, from, bytes;
};

Plan plan(const ft_keys& k, bool policy) {
  Plan p{};
  const uint64_t rows = k.batch * k.steps, keys = k.batch * k.keys;
  const uint32_t vec = k.dtype == FT_F32 ? 4 : 8;
  p.vecs = (k.vocab + vec - 1) / vec;
  // about 4096 workgroups, in whole turns of their loads
  uint64_t each = rows ? (p.vecs * rows + 4095) / 4096 : 1;
  p.chunk_vecs = (uint32_t)round_up(each ? each : 1, kStatU * kStatT);
  p.chunks = (p.vecs + p.chunk_vecs - 1) / p.chunk_vecs;
  Arena ar;
  p.part = ar.take(rows * p.chunks * sizeof(MaxSum));
  p.spans = (p.vecs + kStatU * kStatT - 1) / (kStatU * kStatT);
  if (policy) p.g = ar.take(rows * 4);
  else {
    p.margin = ar.take(keys * 4);
    p.gkey = ar.take(keys * 4);
  }
  p.terms = ar.take((policy ? rows : 1) * 4);
  if (k.keys > 1) {
    p.info = ar.take(rows * sizeof(RowInfo));
    p.from = ar.take(rows * (p.spans + 1) * 4);
    p.ltok = ar.take(rows * k.keys * 4);
    p.lg = ar.take(rows * k.keys * 4);
  }
  p.bytes = ar.used;
  return p;
}

Args base_args(const ft_keys& k, const Plan& p, uint8_t* ws) {
  Args a{};
  a.logits = k.logits;
  a.dlogits = k.dlogits;
  for (int i = 0; i < 2; ++i) {
    a.stride[i] = k.stride[i];
    a.dstride[i] = k.dstride[i];
  }
  a.batch = (uint32_t)k.batch;
  a.steps = (uint32_t)k.steps;
  a.vocab = k.vocab;
  a.keys = k.keys;
  a.rows = (uint32_t)(k.batch * k.steps);
  a.chunks = p.chunks;
  a.chunk_vecs = p.chunk_vecs;
  a.tokens = k.tokens;
  a.lengths = k.lengths;
  a.logp = k.logp;
  a.loss = k.loss;
  a.part = (MaxSum*)(ws + p.part);
  a.g = (float*)(ws + p.g);
  a.margin = (float*)(ws + p.margin);
  a.gkey = (float*)(ws + p.gkey);
  a.terms = (float*)(ws + p.terms);
  a.info = (RowInfo*)(ws + p.info);
  a.from = (uint32_t*)(ws + p.from);
  a.spans = p.spans;
  a.ltok = (uint32_t*)(ws + p.ltok);
  a.lg = (float*)(ws + p.lg);
  return a;
}

template <typename T, bool kPolicy>
hipError_t launch(const Args& a, const Plan& p, hipStream_t s) {
  if (a.rows == 0) return start(key_loss, 1, 256, s, a);
  hipError_t e;
  // Rows that fit a workgroup's registers in one kernel: 512 rows x 32,768
  // bf16, 64 keys a request: 22 us, in parts 31 (1024 threads of four vectors;
  // of eight: 25); 2048 rows of a key each: 51, in parts 69 (512 threads of
  // eight vectors; 1024: 65); 8 rows x 32,768 f32: 15.6, in parts 18.1.
  if (kPolicy && p.vecs <= 8 * kListT && a.keys <= (uint32_t)kListT) {
    if (a.keys > 1 && p.vecs <= 4 * kListT)
      e = start(key_whole<T, true, kListT, 4>, a.rows, kListT, s, a);
    else if (a.keys > 1)
      e = start(key_whole<T, true, kListT, 8>, a.rows, kListT, s, a);
    else if (p.vecs <= 8 * 512)
      e = start(key_whole<T, false, 512, 8>, a.rows, 512, s, a);
    else
      e = start(key_whole<T, false, 1024, 8>, a.rows, 1024, s, a);
    return e == hipSuccess ? start(key_loss, 1, 256, s, a) : e;
  }
  e = start(key_stats<T>, (uint64_t)a.rows * a.chunks, kStatT, s, a);
  if (!kPolicy) {
    const uint32_t keys = a.batch * a.keys;
    if (e == hipSuccess) e = start(key_scores<T>, (keys + 15) / 16, 256, s, a);
    if (e == hipSuccess) e = start(key_pairs, (keys + 63) / 64, 1024, s, a);
  }
  if (e != hipSuccess) return e;
  if (a.keys > (uint32_t)kListT)
    e = start(key_rows<T, kPolicy, 4>, a.rows, kListT, s, a);
  else if (a.keys > 1)
    e = start(key_rows<T, kPolicy, 1>, a.rows, kListT, s, a);
  else if (kPolicy)
    e = start(key_single<T>, (a.rows + 255) / 256, 256, s, a);
  if (e != hipSuccess) return e;
  if (a.dlogits)
    return start(key_gradient<T, kPolicy>, (uint64_t)a.rows * a.spans, kStatT, s, a);
  return start(key_loss, 1, 256, s, a);
}

template <bool kPolicy>
hipError_t launch_typed(int dtype, const Args& a, const Plan& p, hipStream_t s) {
  switch (dtype) {
    case FT_F32: return launch<float, kPolicy>(a, p, s);
    case FT_F16: return launch<_Float16, kPolicy>(a, p, s);
    default: return launch<__bf16, kPolicy>(a, p, s);
  }
}

}  // namespace

uint64_t policy_loss_workspace(const ft_policy_loss_args& q) { return plan(q.k, true).bytes; }

hipError_t launch_policy_loss(const ft_policy_loss_args& q, uint8_t* ws, hipStream_t s) {
  const Plan p = plan(q.k, true);
  Args a = base_args(q.k, p, ws);
  a.old_logp = q.old_logp;
  a.ref_logp = q.ref_logp;
  a.advantage = q.advantage;
  a.weight = q.weight;
  a.low = 1.0f - q.clip_low;
  a.high = 1.0f + q.clip_high;
  a.kl = q.kl_coef;
  a.nterms = a.rows;
  return launch_typed<true>(q.k.dtype, a, p, s);
}

uint64_t preference_loss_workspace(const ft_preference_loss_args& q) {
  return plan(q.k, false).bytes;
}

hipError_t launch_preference_loss(const ft_preference_loss_args& q, uint8_t* ws, hipStream_t s) {
  const Plan p = plan(q.k, false);
  Args a = base_args(q.k, p, ws);
  a.pairs = q.pairs;
  a.pair = q.pair;
  a.ref_logp = q.ref_logp;
  a.weight = q.weight;
  a.beta = q.beta;
  a.smoothing = q.smoothing;
  a.nterms = a.rows ? 1 : 0;
  return launch_typed<false>(q.k.dtype, a, p, s);
}

}  // namespace fto
