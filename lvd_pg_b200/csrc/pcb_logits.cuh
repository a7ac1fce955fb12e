// pcb_logits.cuh — categorical distributions given by logits, for pcb_logits.cu (log-probabilities), pcb_logits_grad.cu
// (their gradient) and pcb_evidence.cu (soft evidence made of logits, with its gradient).
//
// With s = x / T, m = max x, c = log2(e) / T and d_j = (x_j - m) c every kernel works on 2^d_j = exp(s_j - max s).  With
// S = sum 2^d, A = sum 2^d d:
//   logp_j = ln2 d_j - ln S          H = ln S - ln2 A / S          p_j = 2^d_j / S
// d is formed in one of two ways.  Near: fma(x, c, -round(m c)) with x raised to a floor first, so that impossible
// categories (-inf) have 2^d = 0 and a finite d: 0 * inf stays out of A, one instruction per two elements; what rounding
// m c leaves off is the same in every d of the row, in S and in A, and cancels.  It has to stay small, since the largest
// power of the row is two to it: at most 2^-5 below |m c| = 2^20, 2^7 and out of range from 2^31 on.  Far, where m c is
// above that (rows that a mask's -1e10 or lowest value fills, temperatures near 0) or the floor would still weigh:
// (x - m) c, clamped at -200.  NaN passes both (max.NaN).  A row without any possible category has S = 0, logp -inf, H = 0
// and gradient 0.
#pragma once
#include "pcb_internal.h"
#include "pcb_tc.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace pcblogits {

using pcbtc::ex2_ftz;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float NO_MASS = -200.0f;   // 2^-200 is zero in fp32 with flushed denormals
constexpr uint32_t MAX_TOP = 32;

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float finite_shift(float m) { return m == -INFINITY ? 0.0f : m; }

// Order of the alternatives: larger values first, NaN before everything, of equal values the lower index.  As one
// number: the value's bits made monotone above the complement of the index; 0 is below every entry.
__device__ __forceinline__ uint32_t order_bits(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t u = __float_as_uint(v + 0.0f);   // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order_key(float v, uint32_t j) { return (uint64_t)order_bits(v) << 32 | (uint32_t)~j; }

// Words of 4 bytes as they lie in memory: one fp32 element or two of 16 bits.
template <typename T> struct Word;
template <> struct Word<float> {
  static constexpr uint32_t NONE = 0xff800000u;   // -inf
  static constexpr float FLOOR = -1e30f;
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
  static __device__ __forceinline__ float top(uint32_t a) { return __uint_as_float(a); }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr uint32_t NONE = 0xff80ff80u;
  static constexpr float FLOOR = -1e30f;
  static __device__ __forceinline__ __nv_bfloat162 of(uint32_t a) { return *reinterpret_cast<const __nv_bfloat162*>(&a); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat162 a) { return *reinterpret_cast<const uint32_t*>(&a); }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return bits(__hmax2(of(a), of(b))); }
  static __device__ __forceinline__ uint32_t raised(uint32_t a) { return bits(__hmax2_nan(of(a), __float2bfloat162_rn(FLOOR))); }
  static __device__ __forceinline__ float2 floats(uint32_t a) { return {__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u)}; }
  static __device__ __forceinline__ float top(uint32_t a) { const float2 f = floats(a); return fmaxf(f.x, f.y); }
  static __device__ __forceinline__ uint32_t equal(uint32_t a, float v) { return __heq2_mask(of(a), __float2bfloat162_rn(v)); }
};
template <> struct Word<__half> {
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static constexpr float FLOOR = -65504.0f;
  static __device__ __forceinline__ __half2 of(uint32_t a) { return *reinterpret_cast<const __half2*>(&a); }
  static __device__ __forceinline__ uint32_t bits(__half2 a) { return *reinterpret_cast<const uint32_t*>(&a); }
  static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) { return bits(__hmax2(of(a), of(b))); }
  static __device__ __forceinline__ uint32_t raised(uint32_t a) { return bits(__hmax2_nan(of(a), __float2half2_rn(FLOOR))); }
  static __device__ __forceinline__ float2 floats(uint32_t a) { return __half22float2(of(a)); }
  static __device__ __forceinline__ float top(uint32_t a) { const float2 f = floats(a); return fmaxf(f.x, f.y); }
  static __device__ __forceinline__ uint32_t equal(uint32_t a, float v) { return __heq2_mask(of(a), __float2half2_rn(v)); }
};
template <typename T> constexpr uint32_t PER_WORD = 4 / sizeof(T);

// Where the powers of a row count from.
struct Shift {
  float m, c, mc;   // mc: m c, rounded: an explicit product, since fused into a difference it is not what powers count from
  bool near;
};
template <typename T>
__device__ __forceinline__ Shift shift_of(float m, float c) {
  return {m, c, __fmul_rn(m, c), fabsf(m * c) < 0x1p20f && (m - Word<T>::FLOOR) * c > 200.0f && c < 1e8f};
}
__device__ __forceinline__ float scaled(const Shift& s, float x) {   // d, clamped; x finite or not
  return max_nan(s.near ? fmaf(x, s.c, -s.mc) : (x - s.m) * s.c, NO_MASS);
}
// what rounding m c has left off
__device__ __forceinline__ float left_off(const Shift& s) { return s.near ? fmaf(s.m, s.c, -s.mc) : 0.0f; }
// Statistics go out, and come back to the gradients, as sums of exp(s_j - max s), free of that.
__device__ __forceinline__ float sum_out(const Shift& s, float S) { return S * ex2_ftz(-left_off(s)); }
__device__ __forceinline__ float sum_in(const Shift& s, float S) { return S * ex2_ftz(left_off(s)); }
// log2 of the factor between powers counted from a and from b
__device__ __forceinline__ float between(const Shift& a, const Shift& b) {
  return max_nan(a.near && b.near ? a.mc - b.mc : fmaf(a.m - b.m, a.c, left_off(b) - left_off(a)), NO_MASS);
}

struct Stat { float m, S, A; };   // maximum, sum of 2^d, sum of 2^d d

// lanes' statistics joined over `width` neighbouring lanes.  Where a side has no possible value, S is 0 (or NaN, which has
// to pass): it is taken as it is.
template <typename T, int width>
__device__ __forceinline__ Stat lanes_join(Stat s, float c) {
  float m = s.m;
#pragma unroll
  for (int o = width / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float d = s.m == -INFINITY || s.m == m ? 0.0f : between(shift_of<T>(s.m, c), shift_of<T>(m, c)), f = ex2_ftz(d);
  s.A = f * (s.A + d * s.S);
  s.S *= f;
#pragma unroll
  for (int o = width / 2; o; o >>= 1) {
    s.S += __shfl_xor_sync(0xffffffffu, s.S, o);
    s.A += __shfl_xor_sync(0xffffffffu, s.A, o);
  }
  s.m = m;
  return s;
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.f32x2 w, x, y, z;\n\t"
      "mov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}

// 16-byte granules
template <typename T> struct Vec { static constexpr uint32_t N = 16 / sizeof(T); };
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// elements e and e + 1 (e even) of words
template <typename T>
__device__ __forceinline__ float2 pair_of(const uint32_t* w, int e) {
  if constexpr (sizeof(T) == 4) return {__uint_as_float(w[e]), __uint_as_float(w[e + 1])};
  else return Word<T>::floats(w[e / 2]);
}
template <typename T>
__device__ __forceinline__ float element_of(const uint32_t* w, int e) {
  const float2 p = pair_of<T>(w, e & ~1);
  return e & 1 ? p.y : p.x;
}
template <typename T, int W>
__device__ __forceinline__ float most_of_words(const uint32_t* w) {   // NaN does not count
  uint32_t m = w[0];
#pragma unroll
  for (int i = 1; i < W; ++i) m = Word<T>::most(m, w[i]);
  return fmaxf(Word<T>::top(m), -INFINITY);
}
// 2^d (and 2^d d) of W words (an even number of elements) added to S (and A)
template <typename T, int W, bool WITH_A = true>
__device__ __forceinline__ void add_words(const uint32_t* w, const Shift& s, float2& S, float2& A) {
  constexpr int E = W * (int)PER_WORD<T>;
  if (s.near) {
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      float2 x;
      if constexpr (sizeof(T) == 4) x = {max_nan(__uint_as_float(w[e]), Word<T>::FLOOR), max_nan(__uint_as_float(w[e + 1]), Word<T>::FLOOR)};
      else x = Word<T>::floats(Word<T>::raised(w[e / 2]));
      const float2 d = fma2(x, {s.c, s.c}, {-s.mc, -s.mc});
      const float2 p = {ex2_ftz(d.x), ex2_ftz(d.y)};
      S = add2(S, p);
      if (WITH_A) A = fma2(p, d, A);
    }
  } else {
    const float m = finite_shift(s.m);
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 x = pair_of<T>(w, e);
      const float2 d = {max_nan((x.x - m) * s.c, NO_MASS), max_nan((x.y - m) * s.c, NO_MASS)};
      const float2 p = {ex2_ftz(d.x), ex2_ftz(d.y)};
      S = add2(S, p);
      if (WITH_A) A = fma2(p, d, A);
    }
  }
}

__device__ __forceinline__ int64_t token_at(const void* tokens, uint32_t bytes, uint64_t r) {
  return bytes == 8 ? static_cast<const int64_t*>(tokens)[r] : static_cast<const int32_t*>(tokens)[r];
}

// A row's log-probabilities: logp = (x - m) / T - ln S, where S counts from the rounded m c: what that is off by goes into
// the logarithm.  No scaling by log2(e), which would take a mask's value out of range.
struct LogScale { float m, invT, ln; };
template <typename T>
__device__ __forceinline__ LogScale log_scale(const Shift& s, float S, float invT) {
  const float ln = S == 0.0f ? 0.0f : logf(S);
  return {finite_shift(s.m), invT, fmaf(-LN2, left_off(s), ln)};
}
__device__ __forceinline__ float logp_of(float x, const LogScale& l) { return fmaf(x - l.m, l.invT, -l.ln); }
__device__ __forceinline__ float ln_of(float S) { return S == 0.0f ? 0.0f : logf(S); }
// The part of a row that a block reads: granules [g0, g1) counted from the 16-byte boundary at or below the row's start.
template <typename T>
struct Part {
  const T* base;        // that boundary
  uint32_t off, end;    // the row's elements are base[off .. end)
  uint32_t g0, g1, shift;
  __device__ __forceinline__ bool whole(uint32_t g) const { return g * Vec<T>::N >= off && (g + 1) * Vec<T>::N <= end; }
  // the granule as it lies in memory, -inf outside of the row
  __device__ __forceinline__ uint4 read(uint32_t g) const {
    if (whole(g)) return load16(base + (size_t)g * Vec<T>::N);
    uint32_t w[4] = {Word<T>::NONE, Word<T>::NONE, Word<T>::NONE, Word<T>::NONE};
#pragma unroll
    for (uint32_t v = 0; v < Vec<T>::N; ++v) {
      const uint32_t j = g * Vec<T>::N + v;
      if (j < off || j >= end) continue;
      if constexpr (sizeof(T) == 4) w[v] = reinterpret_cast<const uint32_t*>(base)[j];
      else w[v / 2] = (w[v / 2] & (v & 1 ? 0xffffu : 0xffff0000u)) | (uint32_t)reinterpret_cast<const uint16_t*>(base)[j] << (16 * (v & 1));
    }
    return {w[0], w[1], w[2], w[3]};
  }
  __device__ __forceinline__ void read(uint32_t g, float* f) const {   // its elements in fp32
    const uint4 q = read(g);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (uint32_t v = 0; v < Vec<T>::N; ++v) f[v] = element_of<T>(w, v);
  }
  __device__ __forceinline__ bool inside(uint32_t g, uint32_t v) const {
    const uint32_t j = g * Vec<T>::N + v;
    return j >= off && j < end;
  }
  __device__ __forceinline__ uint32_t index(uint32_t g, uint32_t v) const { return g * Vec<T>::N + v - off; }
};

// ---- short rows: L = 2^lg lanes of a warp per row, the whole row in registers -------------------------------------------
// E elements per lane, kept as they came; element (i, v) of lane l is (l + i L) N + v in rows that are read as granules,
// l + i L otherwise.  Few lanes per row make few shuffles: one shuffle serves all rows of the warp.
template <typename T> struct Most;   // elements a lane holds at most: 64 bytes
template <> struct Most<float> { static constexpr uint32_t E = 16; };
template <> struct Most<__nv_bfloat16> { static constexpr uint32_t E = 32; };
template <> struct Most<__half> { static constexpr uint32_t E = 32; };

__device__ __forceinline__ float sum_of(float x, float y) { return x + y; }
// the largest value over the 2^lg lanes of a row (NaN does not count), and the smallest index: one instruction where a warp
// holds one row
__device__ __forceinline__ float most_over_lanes(float v, uint32_t lg) {
  if (lg == 5) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  }
#pragma unroll
  for (uint32_t o = 1u << lg >> 1; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint32_t least_over_lanes(uint32_t v, uint32_t lg) {
  if (lg == 5) return __reduce_min_sync(0xffffffffu, v);
#pragma unroll
  for (uint32_t o = 1u << lg >> 1; o; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename V, typename F>
__device__ __forceinline__ V over_lanes(V v, uint32_t lg, F f) {   // f over the 2^lg lanes of a row
#pragma unroll
  for (uint32_t o = 1u << lg >> 1; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Granules lie where memory has them: a row that begins inside one has `off` elements of others' in front, and its ends are
// masked in registers.  (No granule is read that reaches over an end of the tensor, [lo, hi): its elements are.)
struct Bounds { uintptr_t lo, hi; };
enum Form { ELEMENTS, WHOLE, LOOSE };   // read by elements; in granules that rows begin and end on; in granules wherever rows begin
template <typename T, int E, Form FORM>
struct ShortRow {
  static constexpr uint32_t N = FORM != ELEMENTS ? Vec<T>::N : 1;
  static constexpr int W = E / (int)PER_WORD<T>;
  uint32_t w[W];
  uint32_t off;   // of a LOOSE row
  __device__ __forceinline__ uint32_t front() const { return FORM == LOOSE ? off : 0; }

  __device__ __forceinline__ uint32_t index(int e, uint32_t sub, uint32_t lg) const {   // 2^32 - 1 and less for what lies in front
    return (sub + ((uint32_t)(e / N) << lg)) * N + e % N - front();
  }
  __device__ __forceinline__ void load(const T* x, uint32_t sub, uint32_t lg, uint32_t cats, const Bounds& bounds) {
    if constexpr (FORM == WHOLE) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint32_t g = sub + ((uint32_t)i << lg);
        uint4 v = {Word<T>::NONE, Word<T>::NONE, Word<T>::NONE, Word<T>::NONE};
        if (g * N < cats) v = load16(x + g * N);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
    } else if constexpr (FORM == LOOSE) {
      off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
      const T* base = x - off;
      const uint32_t end = off + cats;
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint32_t g = sub + ((uint32_t)i << lg);
        const T* at = base + g * N;
        uint4 v = {Word<T>::NONE, Word<T>::NONE, Word<T>::NONE, Word<T>::NONE};
        if (g * N < end && reinterpret_cast<uintptr_t>(at) >= bounds.lo && reinterpret_cast<uintptr_t>(at + N) <= bounds.hi) v = load16(at);
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint32_t g = sub + ((uint32_t)i << lg);
        if (g * N >= end || (g * N >= off && (g + 1) * N <= end)) continue;
        const T* at = base + g * N;
        const bool held = reinterpret_cast<uintptr_t>(at) >= bounds.lo && reinterpret_cast<uintptr_t>(at + N) <= bounds.hi;
#pragma unroll
        for (uint32_t v = 0; v < N; ++v) {
          const uint32_t j = g * N + v, word = 4 * i + v / PER_WORD<T>;
          const bool mine = j >= off && j < end;
          if constexpr (sizeof(T) == 4) {
            if (!mine) w[word] = Word<T>::NONE;
            else if (!held) w[word] = reinterpret_cast<const uint32_t*>(at)[v];
          } else {
            const uint32_t shift = 16 * (v & 1);
            uint32_t bits = mine ? w[word] >> shift & 0xffffu : Word<T>::NONE & 0xffffu;
            if (mine && !held) bits = reinterpret_cast<const uint16_t*>(at)[v];
            w[word] = (w[word] & (0xffff0000u >> shift)) | bits << shift;
          }
        }
      }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < E; ++e) w[e] = index(e, sub, lg) < cats ? __float_as_uint(x[index(e, sub, lg)]) : Word<T>::NONE;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const uint32_t lo = index(e, sub, lg) < cats ? h[index(e, sub, lg)] : Word<T>::NONE & 0xffffu;
        const uint32_t hi = index(e + 1, sub, lg) < cats ? h[index(e + 1, sub, lg)] : Word<T>::NONE & 0xffffu;
        w[e / 2] = lo | hi << 16;
      }
    }
  }
  // W words of results to the row's places at y, which lies towards 16-byte boundaries as the row does
  __device__ __forceinline__ void store(T* y, const uint32_t* out, uint32_t sub, uint32_t lg, uint32_t cats) const {
    if constexpr (FORM == WHOLE) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint32_t at = (sub + ((uint32_t)i << lg)) * N;
        if (at < cats) *reinterpret_cast<uint4*>(y + at) = {out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]};
      }
    } else if constexpr (FORM == LOOSE) {
      T* base = y - off;
      const uint32_t end = off + cats;
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint32_t g = sub + ((uint32_t)i << lg);
        if (g * N >= off && (g + 1) * N <= end) {
          *reinterpret_cast<uint4*>(base + g * N) = {out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]};
        } else if (g * N < end) {
#pragma unroll
          for (uint32_t v = 0; v < N; ++v) {
            const uint32_t j = g * N + v;
            if (j < off || j >= end) continue;
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(base)[j] = out[4 * i + v];
            else reinterpret_cast<uint16_t*>(base)[j] = (uint16_t)(out[4 * i + v / 2] >> (16 * (v & 1)));
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t j = index(e, sub, lg);
        if (j >= cats) continue;
        if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(y)[j] = out[e];
        else reinterpret_cast<uint16_t*>(y)[j] = (uint16_t)(out[e / 2] >> (16 * (e & 1)));
      }
    }
  }
  // the element at a place of this lane
  __device__ __forceinline__ float pick(uint32_t place) const {
    uint32_t v = w[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v = place / PER_WORD<T> == (uint32_t)i ? w[i] : v;
    if constexpr (sizeof(T) == 4) return __uint_as_float(v);
    else return place & 1 ? Word<T>::floats(v).y : Word<T>::floats(v).x;
  }
  // NaN in its place: counts no more in the lane's maximum and equals nothing
  __device__ __forceinline__ void strike(uint32_t e, bool yes) {
    const uint32_t place = yes ? e / PER_WORD<T> : 0xffffffffu, bits = sizeof(T) == 4 ? 0x7fffffffu : e & 1 ? 0x7fff0000u : 0x7fffu;
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] |= place == (uint32_t)i ? bits : 0u;
  }
  // the first place of the row that holds v, 0xffffffff if none does
  __device__ __forceinline__ uint32_t find(float v, uint32_t sub) const {
    const uint32_t front = sub == 0 ? this->front() : 0;   // places in front of the row
    uint32_t hits = 0;   // fp32: bit e; else bit i for element 2 i, 16 + i for 2 i + 1
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < E; ++e) hits |= __uint_as_float(w[e]) == v ? 1u << e : 0u;
      hits &= 0xffffffffu << front;
      return hits ? __ffs(hits) - 1 : 0xffffffffu;
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) hits |= Word<T>::equal(w[i], v) & (0x10001u << i);
      const uint32_t lo = hits & 0xffffu & 0xffffffffu << ((front + 1) / 2), hi = hits >> 16 & 0xffffffffu << (front / 2);
      return min(lo ? 2 * (uint32_t)__ffs(lo) - 2 : 0xffffffffu, hi ? 2 * (uint32_t)__ffs(hi) - 1 : 0xffffffffu);
    }
  }
};

constexpr uint32_t STAGES = 3, STAGED_THREADS = 128, STAGED_ROWS_MOST = 128;
constexpr uint32_t STAGE_BYTES = 2048 + 32;   // 32 lanes' 64 bytes, and the granules that the rows share with others

struct ShortShape {
  Form form;
  bool staged;             // short rows that lie one behind the other
  uint32_t lg, each;       // log2 of the lanes per row, elements per lane
};
// Few lanes per row; four at least where it is read in granules (64 contiguous bytes per load), sixteen where it is read
// from memory by elements.  With y: results of the rows go there, and have to lie towards 16-byte boundaries as the rows do.
template <typename T>
ShortShape short_shape(uint32_t cats, uint64_t stride, const void* x, const void* y = nullptr) {
  ShortShape s;
  const bool alike = !y || (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(y)) | (stride - cats) * sizeof(T)) & 15) == 0;
  constexpr uint32_t N = Vec<T>::N;
  const bool whole = ((reinterpret_cast<uintptr_t>(x) | stride * sizeof(T) | (uint64_t)cats * sizeof(T)) & 15) == 0;
  const uint32_t units = whole ? cats / N : (cats + 2 * N - 2) / N;   // granules that a row may touch
  // (loose granules from 512 bytes on: us both directions, 800000 rows of 51 fp16 staged 170, loose 228; one way 200000 of 333
  // bf16 188, 168)
  s.form = alike && units <= 32 * Most<T>::E / N && (whole || cats * sizeof(T) >= 512) ? whole ? WHOLE : LOOSE : ELEMENTS;
  s.staged = s.form == ELEMENTS && alike && stride == cats;
  const bool granules = s.form != ELEMENTS;
  const uint32_t parts = granules ? units : cats, most = granules ? Most<T>::E / N : Most<T>::E, wanted = granules ? 4 : s.staged ? 1 : 16;
  s.lg = 0;
  while (s.lg < 5 && (parts > (most << s.lg) || (1u << s.lg) < std::min(parts, wanted))) ++s.lg;
  s.each = ((parts + (1u << s.lg) - 1) >> s.lg) * (granules ? N : 1);
  return s;
}

// rows per stage: whole passes of 32 rows where they fit, else whole rows of lanes
template <typename T>
uint32_t staged_rows(uint32_t cats, uint32_t lg) {
  const uint32_t per_warp = 32u >> lg, fit = std::min(2048 / (cats * (uint32_t)sizeof(T)), STAGED_ROWS_MOST);
  return fit >= 32 ? fit / 32 * 32 : fit > per_warp ? fit / per_warp * per_warp : per_warp;
}
// CALL(LG) for the lanes per row that a kernel instance is made for: known when it is compiled where a lane's registers are
// full (few lanes: shuffles without loops), -1 (its argument says) otherwise.
#define PCB_LANES(full, lg, CALL)  \
  do {                             \
    if ((full) && (lg) == 2) CALL(2);      \
    else if ((full) && (lg) == 3) CALL(3); \
    else if ((full) && (lg) == 4) CALL(4); \
    else if ((full) && (lg) == 5) CALL(5); \
    else CALL(-1);                 \
  } while (0)

// passes per warp: as many as results can be written together, while the launch is a few times what fits on the GPU
inline uint32_t short_passes(uint64_t rows, uint32_t lg, uint32_t sms) {
  const uint32_t per_pass = 256u >> lg;
  uint32_t passes = 1u << lg;
  while (passes > 1 && rows < (uint64_t)per_pass * passes * 12 * sms) passes /= 2;
  return passes;
}
inline int32_t check_logits(const void* x, int32_t dtype, uint32_t cats, float temperature) {
  PCB_REQUIRE(x, "null logits");
  PCB_REQUIRE(dtype == PCB_F32 || dtype == PCB_BF16 || dtype == PCB_F16, "logits are f32, bf16 or f16");
  PCB_REQUIRE(((uintptr_t)x & (dtype == PCB_F32 ? 3 : 1)) == 0, "logits that are not aligned to their own size");
  PCB_REQUIRE(cats >= 1 && cats <= 0x7fffffffu, "the number of categories must be between 1 and 2^31 - 1");
  PCB_REQUIRE(temperature > 0.0f && LOG2E / temperature < INFINITY && 1.0f / temperature > 0.0f, "the temperature must be positive and finite");
  return PCB_OK;
}

}  // namespace pcblogits
