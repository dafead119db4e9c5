// op_device.h -- what the model head's kernels share on the device: number
// types, 16-byte loads of rows at any alignment, and sums of exponentials.
#ifndef FTAMD_OP_DEVICE_H_
#define FTAMD_OP_DEVICE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fto {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A row of V elements starts at any element of memory (V may be odd), so
// vectors are loaded and stored with the element's alignment: the hardware
// takes it, and a wave's 1 KB touches one more line.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec16 {
  u32x4 v;
};

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);  // elements of a vector

template <typename T>
__device__ __forceinline__ u32x4 load_vec(const T* p) {
  return ((const Vec16<T>*)p)->v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, u32x4 v) {
  ((Vec16<T>*)p)->v = v;
}

// The first n elements of a vector, the others `fill`; p[0] is there.
template <typename T>
__device__ __forceinline__ u32x4 load_part(const T* p, int n, T fill) {
  union {
    u32x4 v;
    T e[kVec<T>];
  } u;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) {
    const T e = p[max(min(i, n - 1), 0)];
    u.e[i] = i < n ? e : fill;
  }
  return u.v;
}
// Elements e ... of a row of `size`, `fill` past its end: one load also for
// the vector that the row ends in (its last whole vector, shifted), none past
// it.
template <typename T>
__device__ __forceinline__ u32x4 load_row_vec(const T* row, uint32_t e, uint32_t size, T fill) {
  if (e + kVec<T> <= size) return load_vec(row + e);
  union {
    u32x4 v;
    uint64_t q[2];
    T e[kVec<T>];
  } f;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) f.e[i] = fill;
  if (e >= size) return f.v;
  if (size < (uint32_t)kVec<T>) return load_part(row + e, (int)(size - e), fill);
  union {
    u32x4 v;
    uint64_t q[2];
  } u;
  u.v = load_vec(row + size - kVec<T>);
  const uint32_t drop = (e + kVec<T> - size) * (uint32_t)sizeof(T) * 8;  // bits, 1 to 127
  const uint32_t keep = 128 - drop;
  union {
    u32x4 v;
    uint64_t q[2];
  } o;
  o.q[0] = drop < 64 ? u.q[0] >> drop | u.q[1] << (64 - drop) : u.q[1] >> (drop - 64);
  o.q[1] = drop < 64 ? u.q[1] >> drop : 0;
  if (keep < 64) {
    o.q[0] |= f.q[0] << keep;
    o.q[1] = f.q[1];
  } else {
    o.q[1] |= keep == 64 ? f.q[1] : f.q[1] << (keep - 64);
  }
  return o.v;
}

// kU vectors of a row, kStep apart from vector v on; `whole` says that all
// threads' are inside it.
template <int kU, typename T>
__device__ __forceinline__ void load_run(u32x4 (&raw)[kU], const T* row, uint32_t v, uint32_t step,
                                         uint32_t size, T fill, bool whole) {
  if (whole) {
#pragma unroll
    for (int u = 0; u < kU; ++u) raw[u] = load_vec(row + (v + u * step) * kVec<T>);
  } else {
#pragma unroll
    for (int u = 0; u < kU; ++u) raw[u] = load_row_vec(row, (v + u * step) * kVec<T>, size, fill);
  }
}

template <typename T>
__device__ __forceinline__ void store_part(T* p, int n, u32x4 v) {
  union {
    u32x4 v;
    T e[kVec<T>];
  } u;
  u.v = v;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i)
    if (i < n) p[i] = u.e[i];
}

// Hides where a vector came from, so that its elements are unpacked again at
// each use instead of being kept: registers hold the packed row.
__device__ __forceinline__ void repack(u32x4& v) { asm volatile("" : "+v"(v)); }

template <typename T>
__device__ __forceinline__ void to_float(u32x4 v, float (&f)[kVec<T>]) {
  union {
    u32x4 v;
    T e[kVec<T>];
  } u;
  u.v = v;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) f[i] = (float)u.e[i];
}
// rounded to nearest even, once
template <typename T>
__device__ __forceinline__ u32x4 from_float(const float (&f)[kVec<T>]) {
  union {
    u32x4 v;
    T e[kVec<T>];
  } u;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) u.e[i] = (T)f[i];
  return u.v;
}

// --- sums of exponentials ---------------------------------------------------
// A part of a row is summed up as (m, s): its maximum (NaN left out) and
// s = sum of exp(x - m), in 32 bits, relative to 0 where m is -infinity.
// Terms are 2^((x - m) log2 e): the difference first, so that logits of any
// size keep their own precision (a mask of the type's lowest value among
// them).  A NaN, or an infinity (inf - inf), makes s NaN, as the formula
// does.
constexpr float kLog2e = 1.44269504088896340736f;

__device__ __forceinline__ float exp2_raw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float exp_base(float m) { return m == -INFINITY ? 0.0f : m; }
__device__ __forceinline__ float exp_term(float x, float base) {
  return exp2_raw((x - base) * kLog2e);
}

struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b) {
  MaxSum r;
  r.m = fmaxf(a.m, b.m);
  const float base = exp_base(r.m);
  r.s = a.s * exp_term(a.m, base) + b.s * exp_term(b.m, base);
  return r;
}
template <int kN>
__device__ __forceinline__ void add_terms(MaxSum& a, const float (&x)[kN]) {
  float v = x[0];
#pragma unroll
  for (int i = 1; i < kN; ++i) v = fmaxf(v, x[i]);
  if (v > a.m) {
    a.s *= exp_term(a.m, v);
    a.m = v;
  }
  const float base = exp_base(a.m);
#pragma unroll
  for (int i = 0; i < kN; ++i) a.s += exp_term(x[i], base);
}

// --- a wave's sums ----------------------------------------------------------
// By the lanes' own paths (shifts within 16 lanes, then broadcasts of lanes 15
// and 31 to the rows behind): some ten cycles a step, where a shuffle by way of
// LDS takes a hundred.  Lane 63 ends with the whole.
template <int kCtrl, int kRows>
__device__ __forceinline__ uint32_t dpp(uint32_t fill, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)fill, (int)v, kCtrl, kRows, 0xF, false);
}
template <typename F>
__device__ __forceinline__ uint32_t wave_prefix(uint32_t v, uint32_t fill, F&& op) {
  v = op(v, dpp<0x111, 0xF>(fill, v));  // one lane down, then 2, 4, 8
  v = op(v, dpp<0x112, 0xF>(fill, v));
  v = op(v, dpp<0x114, 0xF>(fill, v));
  v = op(v, dpp<0x118, 0xF>(fill, v));
  v = op(v, dpp<0x142, 0xA>(fill, v));  // lane 15 to the second and fourth row
  v = op(v, dpp<0x143, 0xC>(fill, v));  // lane 31 to the last two
  return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

__device__ __forceinline__ float wave_max(float v) {  // NaN left out
  const uint32_t r = wave_prefix(__float_as_uint(v), 0xFF800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  });
  return __uint_as_float(last_lane(r));
}
__device__ __forceinline__ float wave_sum(float v) {
  const uint32_t r = wave_prefix(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  });
  return __uint_as_float(last_lane(r));
}
__device__ __forceinline__ uint32_t wave_add(uint32_t v) {
  return last_lane(wave_prefix(v, 0u, [](uint32_t a, uint32_t b) { return a + b; }));
}
// exclusive sum over the lanes in front
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t* total) {
  const uint32_t s = wave_prefix(v, 0u, [](uint32_t a, uint32_t b) { return a + b; });
  *total = last_lane(s);
  return s - v;
}
__device__ __forceinline__ MaxSum wave_merge(MaxSum a) {
  const float m = wave_max(a.m);
  return MaxSum{m, wave_sum(a.s * exp_term(a.m, exp_base(m)))};
}

// unsigned order of the floats; NaN as -infinity, -0 as 0
__device__ __forceinline__ uint32_t order_key(float x) {
  x = x == x ? x + 0.0f : -INFINITY;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

}  // namespace fto

#endif  // FTAMD_OP_DEVICE_H_
