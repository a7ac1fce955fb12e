// pcb_logits.cu — categorical distributions given by logits: log-probabilities of given categories with entropy and
// best alternatives, their gradient, and soft evidence made of logits, with its gradient.
//
// With s = x / T, m = max x, c = log2(e) / T and d_j = (x_j - m) c every kernel works on 2^d_j = exp(s_j - max s).  With
// S = sum 2^d, A = sum 2^d d:
//   logp_j = ln2 d_j - ln S          H = ln S - ln2 A / S          p_j = 2^d_j / S
// d is formed in one of two ways.  Near: fma(x, c, -round(m c)) with x raised to a floor first, so that impossible
// categories (-inf) have 2^d = 0 and a finite d: 0 * inf stays out of A, one instruction per two elements; what rounding
// m c leaves off is the same in every d of the row, in S and in A, and cancels.  Far, where m c could overflow (a row of
// the type's lowest values, as masks leave it) or the floor would still weigh: (x - m) c, clamped at -200.  NaN passes
// both (max.NaN).  A row without any possible category has S = 0, logp -inf, H = 0 and gradient 0.
#include "pcb_internal.h"
#include "pcb_tc.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace {

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
  float m, c, mc;   // mc: m c, rounded
  bool near;
};
template <typename T>
__device__ __forceinline__ Shift shift_of(float m, float c) {
  return {m, c, m * c, fabsf(m) < 1e29f && (m - Word<T>::FLOOR) * c > 200.0f && c < 1e8f};
}
__device__ __forceinline__ float scaled(const Shift& s, float x) {   // d, clamped; x finite or not
  return max_nan(s.near ? fmaf(x, s.c, -s.mc) : (x - s.m) * s.c, NO_MASS);
}
// what rounding m c has left off
__device__ __forceinline__ float left_off(const Shift& s) { return s.near ? fmaf(s.m, s.c, -s.mc) : 0.0f; }
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

struct LogprobArgs {
  const void* x;
  uint64_t rows, stride;
  uint32_t cats, top_k, token_bytes;
  float invT, c;
  const void* tokens;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
};

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
__device__ __forceinline__ float entropy_of(float S, float A, float lnS) { return S == 0.0f ? 0.0f : lnS - LN2 * __fdividef(A, S); }
__device__ __forceinline__ bool is_category(const LogprobArgs& a, int64_t token) { return token >= 0 && token < (int64_t)a.cats; }
__device__ __forceinline__ float token_logp(const LogprobArgs& a, int64_t token, float x, const LogScale& l) {
  return token < 0 ? 0.0f : token >= (int64_t)a.cats ? NAN : logp_of(x, l);
}

// ---- long rows: a block, or the blocks of a cluster, per row -------------------------------------------------------
// One pass over the row.  A thread takes tiles of 128 (fp32) or 64 bytes, keeps a running (max, S, A) that is rescaled
// once per tile whose maximum is new, and notes every tile's maximum in shared memory.
//
// Alternatives without a second pass: the k-th largest of the maxima of 32 groups of threads is a lower bound of the
// k-th largest value (the groups hold different elements), so only tiles whose noted maximum reaches it are read
// again: a few more than k of them.  What reaches the bound is collected and ordered by counting.  More than CAND of
// those (rows of few different values, or large ones side by side in few groups) raise the bound to the k-th of what
// was collected, as long as that helps; what is left then (mostly ties) goes by rounds over what lies above the bound and
// one walk in index order over what equals it.
constexpr uint32_t SLOTS = 16, CAND = 256, PAIRS = 256, MAX_CLUSTER = 8;

template <typename T> struct Tile { static constexpr uint32_t U = sizeof(T) == 4 ? 8 : 4; };   // granules per thread

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

template <uint32_t THREADS>
struct RowShared {
  float slot[SLOTS][THREADS];
  uint64_t cand[CAND];
  uint64_t best[MAX_TOP];   // this block's alternatives, in order
  uint64_t all[THREADS == 256 ? MAX_CLUSTER : 1][MAX_TOP];   // first block of a cluster: every block's
  Stat part[8], joined[MAX_CLUSTER];
  float group[32];
  uint64_t round[THREADS / 32];
  uint32_t pair[PAIRS];   // slot * THREADS + thread
  uint32_t pairs, count, warp_count[THREADS / 32];
};

__device__ __forceinline__ float value_of(uint64_t key) {   // inverse of order_bits, but for NaN
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0xffffffffu ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// f(granule) for the granules of the thread's tiles whose noted maximum passes `pick`
template <uint32_t THREADS, typename T, typename P, typename F>
__device__ __forceinline__ void picked_granules(const Part<T>& p, const RowShared<THREADS>& sh, P pick, F f) {
  constexpr uint32_t U = Tile<T>::U, STEP = THREADS * U;
  const uint32_t tiles = (p.g1 - p.g0 + STEP - 1) / STEP, slots = (tiles + (1u << p.shift) - 1) >> p.shift;
  for (uint32_t s = 0; s < slots; ++s) {
    if (!pick(sh.slot[s][threadIdx.x])) continue;
    const uint32_t t1 = min(tiles, (s + 1) << p.shift);
    for (uint32_t t = s << p.shift; t < t1; ++t)
      for (uint32_t u = 0; u < U; ++u) {
        const uint32_t g = p.g0 + t * STEP + u * THREADS + threadIdx.x;
        if (g < p.g1) f(g);
      }
  }
}

// The block's `top_k` largest, in order, into sh.best (0: there is no further one).  `mine`: the thread's largest value;
// `wild`: the part holds NaN, which no noted maximum shows.
template <uint32_t THREADS, typename T>
__device__ void block_top(const Part<T>& p, RowShared<THREADS>& sh, uint32_t top_k, float mine, bool wild) {
  constexpr uint32_t U = Tile<T>::U, STEP = THREADS * U, WARPS = THREADS / 32;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < MAX_TOP) sh.best[tid] = 0;
  float gm = mine;
#pragma unroll
  for (uint32_t o = WARPS / 2; o; o >>= 1) gm = fmaxf(gm, __shfl_xor_sync(0xffffffffu, gm, o));
  if (lane % WARPS == 0) sh.group[tid / WARPS] = gm;
  if (tid == 0) sh.pairs = sh.count = 0;
  __syncthreads();
  float bound;
  {
    const float v = sh.group[lane];
    uint32_t above = 0;
#pragma unroll
    for (uint32_t j = 0; j < 32; ++j) {
      const float w = sh.group[j];
      above += w > v || (w == v && j < lane);
    }
    bound = __shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, above == top_k - 1)) - 1);
  }
  const uint32_t tiles = (p.g1 - p.g0 + STEP - 1) / STEP, slots = (tiles + (1u << p.shift) - 1) >> p.shift;
  bool again = !wild;
  for (uint32_t tries = 0; again && tries < 8; ++tries) {
    // the slots that reach the bound, then their granules over all threads: one trip to memory
    for (uint32_t s = 0; s < slots; ++s)
      if (sh.slot[s][tid] >= bound) {
        const uint32_t at = atomicAdd(&sh.pairs, 1u);
        if (at < PAIRS) sh.pair[at] = s * THREADS + tid;
      }
    __syncthreads();
    const uint32_t pairs = sh.pairs;
    if (pairs > PAIRS) break;   // ties, mostly: by rounds
    const uint32_t per_pair = U << p.shift;   // granules, a power of two
    for (uint32_t i = tid; i < pairs * per_pair; i += THREADS) {
      const uint32_t pr = sh.pair[i / per_pair], k = i % per_pair;
      const uint32_t g = p.g0 + (((pr / THREADS) << p.shift) + k / U) * STEP + k % U * THREADS + pr % THREADS;
      if (g >= p.g1) continue;
      float f[Vec<T>::N];
      p.read(g, f);
#pragma unroll
      for (uint32_t v = 0; v < Vec<T>::N; ++v)
        if (f[v] >= bound && p.inside(g, v)) {
          const uint32_t at = atomicAdd(&sh.count, 1u);
          if (at < CAND) sh.cand[at] = order_key(f[v], p.index(g, v));
        }
    }
    __syncthreads();
    const uint32_t found = sh.count, n = min(found, CAND);
    for (uint32_t i = tid; i < n; i += THREADS) {
      const uint64_t key = sh.cand[i];
      uint32_t above = 0;
      for (uint32_t j = 0; j < n; ++j) above += sh.cand[j] > key;
      if (above < top_k) sh.best[above] = key;
    }
    __syncthreads();
    if (found <= CAND) return;
    const float better = value_of(sh.best[top_k - 1]);   // of CAND values that reach the bound
    again = better > bound;
    bound = again ? better : bound;
    if (tid == 0) sh.pairs = sh.count = 0;
    __syncthreads();
    if (tid < MAX_TOP) sh.best[tid] = 0;
  }
  // rounds over what lies above the bound (with NaN in the row: over everything)
  uint32_t have = 0;
  uint64_t last = ~0ull;
  __syncthreads();
  while (have < top_k) {
    uint64_t key = 0;
    picked_granules<THREADS>(p, sh, [&](float m) { return wild || m > bound; }, [&](uint32_t g) {
      float f[Vec<T>::N];
      p.read(g, f);
#pragma unroll
      for (uint32_t v = 0; v < Vec<T>::N; ++v)
        if ((wild || f[v] > bound) && p.inside(g, v)) {
          const uint64_t k = order_key(f[v], p.index(g, v));
          if (k < last && k > key) key = k;
        }
    });
#pragma unroll
    for (int o = 16; o; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (lane == 0) sh.round[warp] = key;
    __syncthreads();
    for (uint32_t w = 0; w < WARPS; ++w) key = max(key, sh.round[w]);
    __syncthreads();
    if (key == 0) break;
    if (tid == 0) sh.best[have] = key;
    ++have;
    last = key;
  }
  // what equals the bound, in index order
  for (uint32_t g0 = p.g0; g0 < p.g1 && have < top_k && !wild; g0 += THREADS) {
    const uint32_t g = g0 + tid;
    float f[Vec<T>::N];
    uint32_t hits = 0;
    if (g < p.g1) {
      p.read(g, f);
#pragma unroll
      for (uint32_t v = 0; v < Vec<T>::N; ++v) hits |= (uint32_t)(f[v] == bound && p.inside(g, v)) << v;
    }
    uint32_t before = __popc(hits);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= (uint32_t)o) before += x;
    }
    if (lane == 31) sh.warp_count[warp] = before;
    before -= __popc(hits);
    __syncthreads();
    uint32_t total = 0;
    for (uint32_t w = 0; w < WARPS; ++w) {
      if (w < warp) before += sh.warp_count[w];
      total += sh.warp_count[w];
    }
    for (uint32_t at = have + before; hits && at < top_k; hits &= hits - 1, ++at)
      sh.best[at] = order_key(bound, p.index(g, __ffs(hits) - 1));
    have += total;
    __syncthreads();
  }
  __syncthreads();
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
// the address of `p` in the first block of the cluster, and stores to it
__device__ __forceinline__ uint32_t in_first_block(const void* p) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(pcbtc::smem_u32(p)));
  return r;
}
__device__ __forceinline__ void store_there(uint32_t at, uint64_t v) { asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory"); }
__device__ __forceinline__ void store_there(uint32_t at, float v) { asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }

// `split` blocks (a cluster; 1: no cluster) per row, split = the cluster's size; joined through distributed shared memory,
// so that no call needs a workspace.
template <typename T, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprob_row_kernel(LogprobArgs a, uint32_t split) {
  constexpr uint32_t N = Vec<T>::N, U = Tile<T>::U, STEP = THREADS * U, WARPS = THREADS / 32;
  __shared__ RowShared<THREADS> sh;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = blockIdx.x % split;
  for (uint64_t row = blockIdx.x / split; row < a.rows; row += gridDim.x / split) {
    if (THREADS == 256 && split > 1) cluster_arrive();   // the others run: their shared memory may be written from the wait on
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    // asked for early: the row's token and its logit
    int64_t token = -1;
    float x_token = 0.0f;
    if (tid == 0 && rank == 0 && a.tokens) {
      token = token_at(a.tokens, a.token_bytes, row);
      if (is_category(a, token)) x_token = to_f32(x[token]);
    }
    Part<T> p;
    p.off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    p.base = x - p.off;
    p.end = p.off + a.cats;
    const uint32_t granules = (uint32_t)(((uint64_t)p.end + N - 1) / N), each = (granules + split - 1) / split;
    p.g0 = min(granules, rank * each);
    p.g1 = min(granules, p.g0 + each);
    p.shift = 0;
    while ((((p.g1 - p.g0 + STEP - 1) / STEP) >> p.shift) >= SLOTS) ++p.shift;

    Stat s{-INFINITY, 0.0f, 0.0f};
    Shift from = shift_of<T>(-INFINITY, a.c);
    float2 S2 = {0.0f, 0.0f}, A2 = {0.0f, 0.0f};
    float slot = -INFINITY;
    uint32_t tile = 0;
    for (uint32_t g0 = p.g0; g0 < p.g1; g0 += STEP, ++tile) {
      uint32_t w[U * 4];
      if (g0 * N >= p.off && g0 + STEP <= p.g1 && (g0 + STEP) * N <= p.end) {   // every granule lies in the row
        const T* at = p.base + (size_t)(g0 + tid) * N;
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint4 q = load16(at + (size_t)u * THREADS * N);
          w[4 * u] = q.x; w[4 * u + 1] = q.y; w[4 * u + 2] = q.z; w[4 * u + 3] = q.w;
        }
      } else {
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
          const uint32_t g = g0 + u * THREADS + tid;
          uint4 q = {Word<T>::NONE, Word<T>::NONE, Word<T>::NONE, Word<T>::NONE};
          if (g < p.g1) q = p.read(g);
          w[4 * u] = q.x; w[4 * u + 1] = q.y; w[4 * u + 2] = q.z; w[4 * u + 3] = q.w;
        }
      }
      const float most = most_of_words<T, U * 4>(w);
      if (most > s.m) {
        const Shift to = shift_of<T>(most, a.c);
        if (s.m != -INFINITY) {   // else: the sums are 0, or NaN
          const float d = between(from, to), e = ex2_ftz(d);
          A2 = mul2({e, e}, fma2({d, d}, S2, A2));
          S2 = mul2({e, e}, S2);
        }
        s.m = most;
        from = to;
      }
      add_words<T, U * 4>(w, from, S2, A2);
      slot = fmaxf(slot, most);
      if (a.top_k && ((tile + 1) & ((1u << p.shift) - 1)) == 0) {
        sh.slot[tile >> p.shift][tid] = slot;
        slot = -INFINITY;
      }
    }
    if (a.top_k && (tile & ((1u << p.shift) - 1)) != 0) sh.slot[tile >> p.shift][tid] = slot;
    s.S = S2.x + S2.y;
    s.A = A2.x + A2.y;
    const float mine = s.m;
    s = lanes_join<T, 32>(s, a.c);
    if (lane == 0) sh.part[warp] = s;
    __syncthreads();
    s = lanes_join<T, WARPS>(sh.part[lane % WARPS], a.c);
    if (a.top_k) block_top<THREADS>(p, sh, a.top_k, mine, s.S != s.S);
    if (THREADS == 256 && split > 1) {
      cluster_wait();
      if (tid == 0) {
        const uint32_t at = in_first_block(&sh.joined[rank]);
        store_there(at, s.m);
        store_there(at + 4, s.S);
        store_there(at + 8, s.A);
      }
      if (tid < a.top_k) store_there(in_first_block(&sh.all[THREADS == 256 ? rank : 0][tid]), sh.best[tid]);
      cluster_arrive();
      cluster_wait();
      if (rank == 0) {
        s = lanes_join<T, 8>((lane & 7) < split ? sh.joined[lane & 7] : Stat{-INFINITY, 0.0f, 0.0f}, a.c);
        if (a.top_k) {
          const uint64_t key = tid < split * a.top_k ? sh.all[THREADS == 256 ? tid / a.top_k : 0][tid % a.top_k] : 0;
          uint32_t above = 0;
          for (uint32_t r = 0; r < split; ++r)
            for (uint32_t k = 0; k < a.top_k; ++k) above += sh.all[THREADS == 256 ? r : 0][k] > key;
          if (key && above < a.top_k) sh.best[above] = key;
          __syncthreads();
        }
      }
    }
    if (rank == 0) {
      const LogScale l = log_scale<T>(shift_of<T>(s.m, a.c), s.S, a.invT);
      if (tid == 0) {
        if (a.tokens) a.logp[row] = token_logp(a, token, x_token, l);
        a.entropy[row] = entropy_of(s.S, s.A, ln_of(s.S));
        if (a.stats) reinterpret_cast<float2*>(a.stats)[row] = {s.m, s.S};
      }
      if (tid < a.top_k) {
        const uint64_t key = sh.best[tid];
        a.top_ids[row * a.top_k + tid] = (uint32_t)~key;
        a.top_logp[row * a.top_k + tid] = logp_of(value_of(key), l);
      }
    }
    __syncthreads();
  }
}

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
  for (uint32_t o = 1u << lg >> 1; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint32_t least_over_lanes(uint32_t v, uint32_t lg) {
  if (lg == 5) return __reduce_min_sync(0xffffffffu, v);
  for (uint32_t o = 1u << lg >> 1; o; o >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename V, typename F>
__device__ __forceinline__ V over_lanes(V v, uint32_t lg, F f) {   // f over the 2^lg lanes of a row
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

// What a row leaves for its results.
struct Kept { float m, S, A, best; uint32_t at; };

// A row's statistics, in all lanes that hold it, and its alternatives: a single one goes into `k`, several are written at
// once (`valid`: there is such a row).
template <typename T, int E, Form FORM>
__device__ __forceinline__ Kept short_row(const LogprobArgs& a, ShortRow<T, E, FORM>& r, uint64_t row, bool valid, uint32_t sub, uint32_t lg) {
  using Row = ShortRow<T, E, FORM>;
  Kept k;
  k.m = most_over_lanes(most_of_words<T, Row::W>(r.w), lg);
  const Shift from = shift_of<T>(k.m, a.c);
  float2 S2 = {0.0f, 0.0f}, A2 = {0.0f, 0.0f};
  add_words<T, Row::W>(r.w, from, S2, A2);
  k.S = over_lanes(S2.x + S2.y, lg, sum_of);
  k.A = over_lanes(A2.x + A2.y, lg, sum_of);
  k.best = k.m;
  k.at = 0;
  if (a.top_k == 0) return k;
  LogScale l = {0.0f, 0.0f, 0.0f};
  if (a.top_k > 1) l = log_scale<T>(from, k.S, a.invT);
  const uint32_t width = 1u << lg;
  if (__any_sync(0xffffffffu, k.S != k.S)) {   // NaN or inf somewhere: by keys, which order them too
    uint32_t w[Row::W];   // a copy to be indexed, so that the registers need not be
#pragma unroll
    for (int i = 0; i < Row::W; ++i) w[i] = r.w[i];
    uint64_t last = ~0ull;
    for (uint32_t n = 0; n < a.top_k; ++n) {
      uint64_t key = 0;
#pragma unroll 1
      for (int e = 0; e < E; ++e) {
        const uint32_t j = r.index(e, sub, lg);
        const uint64_t o = j < a.cats ? order_key(element_of<T>(w, e), j) : 0;
        if (o < last && o > key) key = o;
      }
      key = over_lanes(key, lg, [](uint64_t x, uint64_t y) { return x > y ? x : y; });
      k.best = value_of(key);
      k.at = (uint32_t)~key;
      if (a.top_k > 1 && valid && sub == 0) {
        a.top_ids[row * a.top_k + n] = k.at;
        a.top_logp[row * a.top_k + n] = logp_of(k.best, l);
      }
      last = key;
    }
    return k;
  }
  // One alternative a round: the largest value that is left, then the lowest index that holds it.  (Places past the last
  // category hold -inf at indices above every category's: they are never the lowest while a category is left.)  A lane
  // keeps every 2^lg-th and writes it with the others' at the end of as many rounds.
  float best = k.m, kept = 0.0f;
  uint32_t kept_at = 0;
  for (uint32_t n = 0; n < a.top_k; ++n) {
    if (n) best = most_over_lanes(most_of_words<T, Row::W>(r.w), lg);
    const uint32_t own = r.find(best, sub), at = own == 0xffffffffu ? own : r.index(0, sub, lg) + (((own / Row::N) << lg) * Row::N) + own % Row::N;
    const uint32_t first = least_over_lanes(at, lg);
    if (a.top_k == 1) {
      k.at = first;
      break;
    }
    if ((n & (width - 1)) == sub) {
      kept = best;
      kept_at = first;
    }
    if (n + 1 < a.top_k) r.strike(own, at == first);
    if ((n & (width - 1)) == width - 1 || n + 1 == a.top_k) {
      const uint32_t place = (n & ~(width - 1)) + sub;
      if (valid && place <= n) {
        a.top_ids[row * a.top_k + place] = kept_at;
        a.top_logp[row * a.top_k + place] = logp_of(kept, l);
      }
    }
  }
  return k;
}

// The results of up to 32 rows, one per lane.
template <typename T>
__device__ __forceinline__ void short_results(const LogprobArgs& a, const Kept& k, uint64_t row, int64_t token, float x_token) {
  const LogScale l = log_scale<T>(shift_of<T>(k.m, a.c), k.S, a.invT);
  if (a.tokens) a.logp[row] = token_logp(a, token, x_token, l);
  a.entropy[row] = entropy_of(k.S, k.A, ln_of(k.S));
  if (a.stats) reinterpret_cast<float2*>(a.stats)[row] = {k.m, k.S};
  if (a.top_k == 1) {
    a.top_ids[row] = k.at;
    a.top_logp[row] = logp_of(k.best, l);
  }
}

// Rows in memory: in 16-byte granules, or element by element, whatever their distance.  A warp takes `passes` times the rows
// that its lanes hold at once, the next ones on their way while it works on these (granules), and writes the results of all
// of them together: lane (g, j) those of the g-th row of pass j.
template <typename T, int E, Form FORM>
__global__ void __launch_bounds__(256, E >= 16 ? 3 : 4) logprob_short_kernel(LogprobArgs a, uint32_t lg, uint32_t passes) {
  using Row = ShortRow<T, E, FORM>;
  const uint32_t lane = threadIdx.x & 31, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const uint64_t step = (uint64_t)gridDim.x * 8 * per_warp * passes;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.stride + a.cats)};
  for (uint64_t r0 = ((uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * per_warp * passes; r0 < a.rows; r0 += step) {
    const auto row_of = [&](uint32_t pass) { return min(a.rows - 1, r0 + pass * per_warp + group); };
    const auto row_at = [&](uint64_t row) { return static_cast<const T*>(a.x) + row * a.stride; };
    Row next;
    next.load(row_at(row_of(0)), sub, lg, a.cats, bounds);
    const uint64_t mine = r0 + sub * per_warp + group;   // the row whose results this lane writes
    const bool writes = sub < passes && mine < a.rows;
    int64_t token = -1;
    float x_token = 0.0f;
    if (writes && a.tokens) {
      token = token_at(a.tokens, a.token_bytes, mine);
      if (is_category(a, token)) x_token = to_f32(row_at(mine)[token]);
    }
    Kept kept = {0.0f, 0.0f, 0.0f, 0.0f, 0};
    for (uint32_t pass = 0; pass < passes && r0 + pass * per_warp < a.rows; ++pass) {
      Row r = next;
      if (FORM != ELEMENTS && pass + 1 < passes) next.load(row_at(row_of(pass + 1)), sub, lg, a.cats, bounds);
      const Kept k = short_row<T, E, FORM>(a, r, row_of(pass), r0 + pass * per_warp + group < a.rows, sub, lg);
      if (sub == pass) kept = k;
      if (FORM == ELEMENTS && pass + 1 < passes) next.load(row_at(row_of(pass + 1)), sub, lg, a.cats, bounds);
    }
    if (writes) short_results<T>(a, kept, mine, token, x_token);
  }
}

// Rows one behind the other (stride = cats), of any length and alignment: every warp stages the bytes of `rows_staged` of
// them, from the 16-byte boundary below their beginning on, with asynchronous copies, STAGES - 1 of them ahead of its work,
// and its lanes read their elements there.
constexpr uint32_t STAGES = 3, STAGED_THREADS = 128, STAGED_ROWS_MOST = 128;
constexpr uint32_t STAGE_BYTES = 2048 + 32;   // 32 lanes' 64 bytes, and the granules that the rows share with others

template <typename T, int E>
__global__ void __launch_bounds__(STAGED_THREADS, 6) logprob_staged_kernel(LogprobArgs a, uint32_t lg, uint32_t rows_staged) {
  using Row = ShortRow<T, E, ELEMENTS>;
  constexpr uint32_t WARPS = STAGED_THREADS / 32;
  __shared__ __align__(16) uint8_t stages[WARPS][STAGES][STAGE_BYTES];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(a.x), x1 = x0 + a.rows * a.cats * sizeof(T);
  const uint64_t step = (uint64_t)gridDim.x * WARPS * rows_staged;
  const uint64_t first = ((uint64_t)blockIdx.x * WARPS + warp) * rows_staged;
  const auto fetch = [&](uint64_t q0, uint8_t* stage) {   // the rows from q0 on
    if (q0 < a.rows) {
      const uint32_t n = (uint32_t)min((uint64_t)rows_staged, a.rows - q0);
      const uintptr_t lo = x0 + q0 * a.cats * sizeof(T), hi = lo + (uintptr_t)n * a.cats * sizeof(T);
      uint8_t* dst = stage + 16 * lane;
      for (uintptr_t at = (lo & ~(uintptr_t)15) + 16 * lane; at < hi; at += 512, dst += 512) {
        if (at >= x0 && at + 16 <= x1) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(pcbtc::smem_u32(dst)), "l"(at) : "memory");
        } else {   // the granule reaches over an end of the tensor
          for (uint32_t i = 0; i < 16; i += sizeof(T))
            if (at + i >= x0 && at + i < x1) *reinterpret_cast<T*>(dst + i) = *reinterpret_cast<const T*>(at + i);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (uint32_t i = 0; i + 1 < STAGES; ++i) fetch(first + i * step, stages[warp][i]);
  uint32_t buf = 0;
  for (uint64_t q0 = first; q0 < a.rows; q0 += step) {
    fetch(q0 + (STAGES - 1) * step, stages[warp][buf == 0 ? STAGES - 1 : buf - 1]);   // the stage that was read last
    const uint32_t n = (uint32_t)min((uint64_t)rows_staged, a.rows - q0);
    // 32 rows at a time, so that every lane has one to write
    for (uint32_t i0 = 0; i0 < n; i0 += 32) {
      const uint32_t mine = i0 + sub * per_warp + group;
      const int64_t token = a.tokens && mine < n ? token_at(a.tokens, a.token_bytes, q0 + mine) : -1;
      if (i0 == 0) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
      }
      const T* rows = reinterpret_cast<const T*>(stages[warp][buf] + ((x0 + q0 * a.cats * sizeof(T)) & 15));
      Kept kept = {0.0f, 0.0f, 0.0f, 0.0f, 0};
      for (uint32_t pass = 0; pass < (1u << lg) && i0 + pass * per_warp < n; ++pass) {
        const uint32_t i = i0 + pass * per_warp + group;
        Row r;
        r.load(rows + min(i, n - 1) * a.cats, sub, lg, a.cats, Bounds{0, 0});
        const Kept k = short_row<T, E, ELEMENTS>(a, r, q0 + min(i, n - 1), i < n, sub, lg);
        if (sub == pass) kept = k;
      }
      if (mine < n) short_results<T>(a, kept, q0 + mine, token, is_category(a, token) ? to_f32(rows[mine * a.cats + (uint32_t)token]) : 0.0f);
    }
    __syncwarp();   // everybody has read this stage
    buf = buf + 1 == STAGES ? 0 : buf + 1;
  }
}

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

// blocks of `kernel` that fill the GPU, at most `needed`
template <auto kernel, int threads>
uint32_t resident_blocks(uint32_t sms, uint64_t needed) {
  static std::atomic<int> known[64];   // per device
  int dev = 0, per_sm = 1;
  if (cudaGetDevice(&dev) == cudaSuccess && (per_sm = known[dev & 63].load(std::memory_order_relaxed)) < 1) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess || per_sm < 1) per_sm = 1;
    known[dev & 63].store(per_sm, std::memory_order_relaxed);
  }
  const uint64_t all = (uint64_t)per_sm * sms;
  return (uint32_t)(needed < all ? needed : all);
}

// rows per stage: whole passes of 32 rows where they fit, else whole rows of lanes
template <typename T>
uint32_t staged_rows(uint32_t cats, uint32_t lg) {
  const uint32_t per_warp = 32u >> lg, fit = std::min(2048 / (cats * (uint32_t)sizeof(T)), STAGED_ROWS_MOST);
  return fit >= 32 ? fit / 32 * 32 : fit > per_warp ? fit / per_warp * per_warp : per_warp;
}
template <typename T, int E>
void launch_staged(const LogprobArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  const uint32_t rows = staged_rows<T>(a.cats, s.lg), per_block = rows * (STAGED_THREADS / 32);
  const uint32_t grid = resident_blocks<logprob_staged_kernel<T, E>, STAGED_THREADS>(sms, (a.rows + per_block - 1) / per_block);
  logprob_staged_kernel<T, E><<<grid, STAGED_THREADS, 0, st>>>(a, s.lg, rows);
}
// passes per warp: as many as results can be written together, while the launch is a few times what fits on the GPU
uint32_t short_passes(uint64_t rows, uint32_t lg, uint32_t sms) {
  const uint32_t per_pass = 256u >> lg;
  uint32_t passes = 1u << lg;
  while (passes > 1 && rows < (uint64_t)per_pass * passes * 12 * sms) passes /= 2;
  return passes;
}
template <typename T, int E, Form FORM>
void launch_passes(const LogprobArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  const uint32_t per_pass = 256u >> s.lg, passes = short_passes(a.rows, s.lg, sms);
  const uint64_t blocks = (a.rows + per_pass * passes - 1) / (per_pass * passes);
  logprob_short_kernel<T, E, FORM><<<(uint32_t)std::min<uint64_t>(blocks, 0x7fffffff), 256, 0, st>>>(a, s.lg, passes);
}
template <typename T, int E>
void launch_short_as(const LogprobArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  if constexpr (E >= (int)Vec<T>::N) {
    if (s.form == WHOLE) return launch_passes<T, E, WHOLE>(a, s, sms, st);
    if (s.form == LOOSE) return launch_passes<T, E, LOOSE>(a, s, sms, st);
  }
  if (s.staged) return launch_staged<T, E>(a, s, sms, st);
  launch_passes<T, E, ELEMENTS>(a, s, sms, st);
}
template <typename T>
void launch_short(const LogprobArgs& a, uint32_t sms, cudaStream_t st) {
  const ShortShape s = short_shape<T>(a.cats, a.stride, a.x);
  if (s.each <= 4) launch_short_as<T, 4>(a, s, sms, st);
  else if (s.each <= 8) launch_short_as<T, 8>(a, s, sms, st);
  else if (s.each <= 16) launch_short_as<T, 16>(a, s, sms, st);
  else launch_short_as<T, Most<T>::E>(a, s, sms, st);
}

// The blocks that share a long row: as many as keep the launch within two blocks per SM, and each with a granule of the row
// per thread at least.
template <typename T>
uint32_t row_split(uint64_t rows, uint32_t cats, uint32_t sms) {
  uint32_t split = 1;
  while (split < MAX_CLUSTER && rows * split * 2 <= 2 * (uint64_t)sms && cats >= split * 2 * 256 * Vec<T>::N) split *= 2;
  return split;
}

template <typename T>
cudaError_t launch_rows(const LogprobArgs& a, uint32_t sms, cudaStream_t st) {
  if (a.cats <= 32 * Most<T>::E) {
    launch_short<T>(a, sms, st);
    return cudaGetLastError();
  }
  const uint32_t grid = (uint32_t)(a.rows < (1u << 24) ? a.rows : 1u << 24);
  const uint64_t bytes = (uint64_t)a.cats * sizeof(T);
  // Where there are enough rows to fill the GPU: by one warp each if they have few tiles, else by four.  (Eight warps leave the
  // last rows to half-empty SMs: us with eight / four, 2048 rows of 131072 bf16 105.0 / 104.2, 1021 of 50021 31.7 / 25.9, 2000
  // of 32768 fp32 56.0 / 48.3.)
  if (bytes <= 16384 && a.rows >= 16 * (uint64_t)sms) {
    logprob_row_kernel<T, 32><<<grid, 32, 0, st>>>(a, 1);
    return cudaGetLastError();
  }
  if (a.rows >= 4 * (uint64_t)sms) {
    logprob_row_kernel<T, 128><<<grid, 128, 0, st>>>(a, 1);
    return cudaGetLastError();
  }
  const uint32_t split = row_split<T>(a.rows, a.cats, sms);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid * split);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, logprob_row_kernel<T, 256>, a, split);
}

struct LogprobGradArgs {
  const void* x;
  uint64_t rows, stride, g_logp_stride, g_entropy_stride;
  uint32_t cats, top_k, token_bytes;
  float invT, c;
  const void* tokens;
  const int64_t* top_ids;
  const float *stats, *entropy, *g_logp, *g_entropy, *g_top;
  void* dx;
};

// What a row's gradient is made of: dx_j = 2^d_j (alpha + beta d_j) + the parts of the token and the alternatives, with
// alpha = -(gL + sum gK + gH (H - ln S)) / (T S), beta = -gH ln2 / (T S).
struct RowGrad {
  Shift from;
  float S, alpha, beta, gl;
  int64_t token;   // negative: none
};
template <typename T>
__device__ __forceinline__ RowGrad row_grad(const LogprobGradArgs& a, uint64_t row) {
  RowGrad g;
  g.from = shift_of<T>(a.stats[2 * row], a.c);
  g.S = a.stats[2 * row + 1];
  g.token = -1;
  g.gl = 0.0f;
  if (a.g_logp && a.tokens) {
    g.token = token_at(a.tokens, a.token_bytes, row);
    if (g.token >= 0) g.gl = g.token < (int64_t)a.cats ? a.g_logp[row * a.g_logp_stride] : NAN;
  }
  float total = g.gl;
  if (a.g_top)
    for (uint32_t k = 0; k < a.top_k; ++k) total += a.g_top[row * a.top_k + k];
  const float gh = a.g_entropy ? a.g_entropy[row * a.g_entropy_stride] : 0.0f;
  const float scale = a.invT / g.S;
  g.alpha = -(total + (gh != 0.0f ? gh * (a.entropy[row] - logf(g.S)) : 0.0f)) * scale;
  g.beta = -gh * LN2 * scale;
  return g;
}
__device__ __forceinline__ float grad_of(const RowGrad& g, float x) {
  const float d = scaled(g.from, x);
  return ex2_ftz(d) * fmaf(g.beta, d, g.alpha);
}
__device__ __forceinline__ bool no_mass(const RowGrad& g) { return g.S == 0.0f; }
// the whole gradient of an element that the token or an alternative points to
__device__ __forceinline__ float pointed_grad(const LogprobGradArgs& a, const RowGrad& g, uint64_t row, uint32_t j, float x) {
  if (no_mass(g)) return 0.0f;
  float v = grad_of(g, x);
  if (g.token == (int64_t)j) v += g.gl * a.invT;
  if (a.g_top)
    for (uint32_t k = 0; k < a.top_k; ++k)
      if (a.top_ids[row * a.top_k + k] == (int64_t)j) v += a.g_top[row * a.top_k + k] * a.invT;
  return v;
}
// p_j (alpha + beta d) of W words, as words
template <typename T, int W>
__device__ __forceinline__ void grad_words(const uint32_t* w, const RowGrad& g, uint32_t* out) {
  constexpr int E = W * (int)PER_WORD<T>;
  const float alpha = no_mass(g) ? 0.0f : g.alpha, beta = no_mass(g) ? 0.0f : g.beta;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    float2 d;
    if (g.from.near) {
      float2 x;
      if constexpr (sizeof(T) == 4) x = {max_nan(__uint_as_float(w[e]), Word<T>::FLOOR), max_nan(__uint_as_float(w[e + 1]), Word<T>::FLOOR)};
      else x = Word<T>::floats(Word<T>::raised(w[e / 2]));
      d = fma2(x, {g.from.c, g.from.c}, {-g.from.mc, -g.from.mc});
    } else {
      const float2 x = pair_of<T>(w, e);
      const float m = finite_shift(g.from.m);
      d = {max_nan((x.x - m) * g.from.c, NO_MASS), max_nan((x.y - m) * g.from.c, NO_MASS)};
    }
    const float2 v = mul2({ex2_ftz(d.x), ex2_ftz(d.y)}, fma2({beta, beta}, d, {alpha, alpha}));
    if constexpr (sizeof(T) == 4) {
      out[e] = __float_as_uint(v.x);
      out[e + 1] = __float_as_uint(v.y);
    } else if constexpr (std::is_same<T, __half>::value) {
      out[e / 2] = Word<T>::bits(__floats2half2_rn(v.x, v.y));
    } else {
      out[e / 2] = Word<T>::bits(__floats2bfloat162_rn(v.x, v.y));
    }
  }
}

// A block takes GRAD_TILE bytes of a row: 64 per thread.  Granules are those of dx; x is read in them where it lies alike
// towards 16-byte boundaries, by elements otherwise.  The last rows come first: the forward pass read them last, and some of them are still in the L2 cache.
constexpr uint32_t GRAD_THREADS = 256, GRAD_TILE = 64 * GRAD_THREADS;
template <typename T>
__global__ void __launch_bounds__(GRAD_THREADS) logprob_grad_kernel(LogprobGradArgs a, uint32_t chunks) {
  constexpr uint32_t N = Vec<T>::N, STEP = GRAD_TILE / 16;
  const uint32_t tid = threadIdx.x;
  for (uint64_t i = blockIdx.x; i < a.rows * chunks; i += gridDim.x) {
    const uint64_t row = a.rows - 1 - i / chunks;
    const uint32_t chunk = (uint32_t)(i % chunks);
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* dx = static_cast<T*>(a.dx) + row * a.cats;
    Part<T> p;   // of dx
    p.off = (uint32_t)((reinterpret_cast<uintptr_t>(dx) & 15) / sizeof(T));
    p.base = dx - p.off;
    p.end = p.off + a.cats;
    const bool alike = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const uint32_t g0 = chunk * STEP, g1 = min((uint32_t)(((uint64_t)p.end + N - 1) / N), g0 + STEP);
    const T* xs = x - p.off;   // x's element for place j of the granules
    // what the token and the alternatives point to in this chunk, one thread each
    const uint32_t n = a.g_top ? a.top_k + 1 : a.g_logp ? 1 : 0;
    int64_t pointed = -1;
    float x_pointed = 0.0f;
    if (tid < n) {
      pointed = tid > 0 ? a.top_ids[row * a.top_k + tid - 1] : a.g_logp ? token_at(a.tokens, a.token_bytes, row) : -1;
      if (pointed < 0 || pointed >= (int64_t)a.cats || ((uint32_t)pointed + p.off) / N < g0 || ((uint32_t)pointed + p.off) / N >= g1) pointed = -1;
      else x_pointed = to_f32(x[pointed]);
    }
    uint32_t w[4][4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t at = g0 + u * GRAD_THREADS + tid;
      if (at >= g1) continue;
      if (alike && p.whole(at)) {
        const uint4 q = load16(xs + (size_t)at * N);
        w[u][0] = q.x; w[u][1] = q.y; w[u][2] = q.z; w[u][3] = q.w;
      } else {
#pragma unroll
        for (uint32_t v = 0; v < N; v += PER_WORD<T>) {
          uint32_t word = 0;
#pragma unroll
          for (uint32_t h = 0; h < PER_WORD<T>; ++h) {
            const uint32_t j = at * N + v + h;
            if (j < p.off || j >= p.end) continue;
            if constexpr (sizeof(T) == 4) word = reinterpret_cast<const uint32_t*>(xs)[j];
            else word |= (uint32_t)reinterpret_cast<const uint16_t*>(xs)[j] << (16 * h);
          }
          w[u][v / PER_WORD<T>] = word;
        }
      }
    }
    const RowGrad g = row_grad<T>(a, row);
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t at = g0 + u * GRAD_THREADS + tid;
      if (at >= g1) continue;
      uint32_t out[4];
      grad_words<T, 4>(w[u], g, out);
      T* to = const_cast<T*>(p.base) + (size_t)at * N;
      if (p.whole(at)) {
        *reinterpret_cast<uint4*>(to) = {out[0], out[1], out[2], out[3]};
      } else {
#pragma unroll
        for (uint32_t v = 0; v < N; ++v)
          if (at * N + v >= p.off && at * N + v < p.end) {
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(to)[v] = out[v];
            else reinterpret_cast<uint16_t*>(to)[v] = (uint16_t)(out[v / 2] >> (16 * (v & 1)));
          }
      }
    }
    if (n > 0) {
      __syncthreads();   // the block's stores come before these
      if (pointed >= 0) dx[pointed] = from_f32<T>(pointed_grad(a, g, row, (uint32_t)pointed, x_pointed));
    }
  }
}

// Short rows, 2^lg lanes each, as in logprob_short_kernel: a warp takes `passes` times the rows that its lanes hold at
// once, lane (g, j) prepares the g-th row of pass j, and the next rows are on their way while it works on these.
template <typename T, int E, Form FORM>
__global__ void __launch_bounds__(256, E >= 16 ? 3 : 5) logprob_grad_short_kernel(LogprobGradArgs a, uint32_t lg, uint32_t passes) {
  using Row = ShortRow<T, E, FORM>;
  const uint32_t lane = threadIdx.x & 31, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.stride + a.cats)};
  const uint64_t rows_each = (uint64_t)per_warp * passes, all = (a.rows + rows_each - 1) / rows_each, step = (uint64_t)gridDim.x * 8;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += step) {
    const uint64_t r0 = (all - 1 - i) * rows_each;   // the last rows first
    const auto row_of = [&](uint32_t pass) { return min(a.rows - 1, r0 + pass * per_warp + group); };
    const auto row_at = [&](uint64_t row) { return static_cast<const T*>(a.x) + row * a.stride; };
    Row next;
    next.load(row_at(row_of(0)), sub, lg, a.cats, bounds);
    const RowGrad mine = row_grad<T>(a, min(a.rows - 1, r0 + min(sub, passes - 1) * per_warp + group));
    const int32_t my_token = mine.token >= 0 && mine.token < (int64_t)a.cats ? (int32_t)mine.token : -1;
    for (uint32_t pass = 0; pass < passes && r0 + pass * per_warp < a.rows; ++pass) {
      const Row r = next;
      if (pass + 1 < passes) next.load(row_at(row_of(pass + 1)), sub, lg, a.cats, bounds);
      const uint32_t from = (lane & ~((1u << lg) - 1)) + pass;   // the lane that prepared this row
      RowGrad g;
      g.from = shift_of<T>(__shfl_sync(0xffffffffu, mine.from.m, from), a.c);
      g.S = __shfl_sync(0xffffffffu, mine.S, from);
      g.alpha = __shfl_sync(0xffffffffu, mine.alpha, from);
      g.beta = __shfl_sync(0xffffffffu, mine.beta, from);
      g.gl = __shfl_sync(0xffffffffu, mine.gl, from);
      g.token = __shfl_sync(0xffffffffu, my_token, from);
      const uint64_t row = row_of(pass);
      const bool valid = r0 + pass * per_warp + group < a.rows;
      T* dx = static_cast<T*>(a.dx) + row * a.cats;
      uint32_t out[Row::W];
      grad_words<T, Row::W>(r.w, g, out);
      if (valid) r.store(dx, out, sub, lg, a.cats);
      if (a.g_logp) {   // the token's, by the lane that holds it, over what it has just written
        const uint32_t j = (uint32_t)g.token, at = j + r.front(), place = ((at / Row::N) >> lg) * Row::N + at % Row::N;
        const float x = r.pick(place);
        if (valid && (int32_t)g.token >= 0 && ((at / Row::N) & ((1u << lg) - 1)) == sub) dx[j] = from_f32<T>(pointed_grad(a, g, row, j, x));
      }
      if (a.g_top) {
        __syncwarp();   // the lanes' stores come before these
        for (uint32_t k = sub; k < a.top_k; k += 1u << lg) {
          const int64_t j = a.top_ids[row * a.top_k + k];
          if (valid && j >= 0 && j < (int64_t)a.cats) dx[j] = from_f32<T>(pointed_grad(a, g, row, (uint32_t)j, to_f32(row_at(row)[j])));
        }
      }
    }
  }
}

// Short rows one behind the other, of any length, staged as in logprob_staged_kernel: the gradient takes the place of the
// logits in shared memory and leaves in granules, but for those that the stage shares with its neighbours.
template <typename T, int E>
__global__ void __launch_bounds__(STAGED_THREADS, 6) logprob_grad_staged_kernel(LogprobGradArgs a, uint32_t lg, uint32_t rows_staged) {
  using Row = ShortRow<T, E, ELEMENTS>;
  constexpr uint32_t WARPS = STAGED_THREADS / 32;
  __shared__ __align__(16) uint8_t stages[WARPS][STAGE_BYTES];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const uint64_t all = (a.rows + rows_staged - 1) / rows_staged, step = (uint64_t)gridDim.x * WARPS;
  uint8_t* stage = stages[warp];
  for (uint64_t i = (uint64_t)blockIdx.x * WARPS + warp; i < all; i += step) {
    const uint64_t q0 = (all - 1 - i) * rows_staged;   // the last rows first
    const uint32_t n = (uint32_t)min((uint64_t)rows_staged, a.rows - q0);
    const uintptr_t lo = reinterpret_cast<uintptr_t>(a.x) + q0 * a.cats * sizeof(T), hi = lo + (uintptr_t)n * a.cats * sizeof(T);
    const intptr_t to = reinterpret_cast<uintptr_t>(a.dx) - reinterpret_cast<uintptr_t>(a.x);   // a multiple of 16
    for (uint32_t k = 16 * lane; (lo & ~(uintptr_t)15) + k < hi; k += 512) {
      const uintptr_t at = (lo & ~(uintptr_t)15) + k;
      if (at >= lo && at + 16 <= hi) {
        *reinterpret_cast<uint4*>(stage + k) = load16(reinterpret_cast<const void*>(at));
      } else {
        for (uint32_t e = 0; e < 16; e += sizeof(T))
          if (at + e >= lo && at + e < hi) *reinterpret_cast<T*>(stage + k + e) = *reinterpret_cast<const T*>(at + e);
      }
    }
    __syncwarp();
    T* rows = reinterpret_cast<T*>(stage + (lo & 15));
    for (uint32_t i0 = 0; i0 < n; i0 += per_warp) {
      const bool valid = i0 + group < n;
      const uint32_t r = valid ? i0 + group : n - 1;
      const uint64_t row = q0 + r;
      T* x = rows + r * a.cats;
      Row in;
      in.load(x, sub, lg, a.cats, Bounds{0, 0});
      const RowGrad g = row_grad<T>(a, row);
      uint32_t out[Row::W];
      grad_words<T, Row::W>(in.w, g, out);
      // what is pointed to, from the logits, before they are gone
      const uint32_t most = a.g_top ? a.top_k + 1 : a.g_logp ? 1 : 0;
      for (uint32_t k0 = 0; k0 < most || k0 == 0; k0 += 1u << lg) {
        const uint32_t k = k0 + sub;
        int64_t j = -1;
        T value = from_f32<T>(0.0f);
        if (valid && k < most) {
          j = k == 0 ? g.token : a.top_ids[row * a.top_k + k - 1];
          if (j < 0 || j >= (int64_t)a.cats) j = -1;
          else if (k0 == 0) value = from_f32<T>(pointed_grad(a, g, row, (uint32_t)j, to_f32(x[j])));
          else value = from_f32<T>(pointed_grad(a, g, row, (uint32_t)j, to_f32(static_cast<const T*>(a.x)[row * a.cats + (uint32_t)j])));
        }
        __syncwarp();   // everybody has read the row
        if (k0 == 0 && valid) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const uint32_t c = in.index(e, sub, lg);
            if (c >= a.cats) continue;
            if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(x)[c] = out[e];
            else reinterpret_cast<uint16_t*>(x)[c] = (uint16_t)(out[e / 2] >> (16 * (e & 1)));
          }
        }
        __syncwarp();
        if (j >= 0) x[j] = value;
        __syncwarp();
      }
    }
    for (uint32_t k = 16 * lane; (lo & ~(uintptr_t)15) + k < hi; k += 512) {
      const uintptr_t at = (lo & ~(uintptr_t)15) + k;
      if (at >= lo && at + 16 <= hi) {
        *reinterpret_cast<uint4*>(at + to) = *reinterpret_cast<const uint4*>(stage + k);
      } else {
        for (uint32_t e = 0; e < 16; e += sizeof(T))
          if (at + e >= lo && at + e < hi) *reinterpret_cast<T*>(at + e + to) = *reinterpret_cast<const T*>(stage + k + e);
      }
    }
    __syncwarp();
  }
}

template <typename T, int E>
void launch_grad_short_as(const LogprobGradArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  const uint32_t lg = s.lg;
  if (s.staged) {
    const uint32_t rows = staged_rows<T>(a.cats, lg), per_block = rows * (STAGED_THREADS / 32);
    const uint64_t n = (a.rows + per_block - 1) / per_block;
    logprob_grad_staged_kernel<T, E><<<(uint32_t)std::min<uint64_t>(n, 0x7fffffff), STAGED_THREADS, 0, st>>>(a, lg, rows);
    return;
  }
  const uint32_t passes = short_passes(a.rows, lg, sms);
  const uint64_t blocks = (a.rows + (uint64_t)(256u >> lg) * passes - 1) / ((uint64_t)(256u >> lg) * passes);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, 0x7fffffff);
  if constexpr (E >= (int)Vec<T>::N) {
    if (s.form == WHOLE) {
      logprob_grad_short_kernel<T, E, WHOLE><<<grid, 256, 0, st>>>(a, lg, passes);
      return;
    }
    if (s.form == LOOSE) {
      logprob_grad_short_kernel<T, E, LOOSE><<<grid, 256, 0, st>>>(a, lg, passes);
      return;
    }
  }
  logprob_grad_short_kernel<T, E, ELEMENTS><<<grid, 256, 0, st>>>(a, lg, passes);
}
template <typename T>
void launch_grad(const LogprobGradArgs& a, uint32_t sms, cudaStream_t st) {
  if (a.cats <= 32 * Most<T>::E) {
    const ShortShape s = short_shape<T>(a.cats, a.stride, a.x, a.dx);
    if (s.each <= 4) launch_grad_short_as<T, 4>(a, s, sms, st);
    else if (s.each <= 8) launch_grad_short_as<T, 8>(a, s, sms, st);
    else if (s.each <= 16) launch_grad_short_as<T, 16>(a, s, sms, st);
    else launch_grad_short_as<T, Most<T>::E>(a, s, sms, st);
    return;
  }
  const uint32_t chunks = (uint32_t)(((uint64_t)a.cats + 2 * Vec<T>::N) * sizeof(T) / GRAD_TILE + 1);
  logprob_grad_kernel<T><<<(uint32_t)std::min<uint64_t>(a.rows * chunks, 0x7fffffff), GRAD_THREADS, 0, st>>>(a, chunks);
}

struct EvidenceArgs {
  const void* x;
  uint64_t rows, row_stride, var_stride, miss_row_stride, miss_var_stride;
  uint32_t vars, cats;
  float invT, c;
  const uint8_t* miss;
  float *out, *stats_out;
  const float *stats, *g;
  void* dx;
};

// ---- soft evidence -----------------------------------------------------------------------------------------------------
// Logits have the category fastest, evidence the row.  A block takes a tile of 32 rows and up to EV_COLUMNS columns (the
// categories of one variable, or of several short ones that lie one behind the other).  Distributions are worked on where
// they are contiguous: 2^lg lanes hold one, as in logprob_short_kernel.  Evidence and its gradient move by columns of 32
// neighbouring rows, 128 bytes, a warp each; shared memory stands between the two orders.  Columns are 33 floats apart there;
// for fp32 logits, where four neighbouring granules would share a bank, one more per row of a warp after every 32 columns
// (37 x 192 x 500: 16.0 -> 15.0 us; 16-bit logits, two to a bank, lose more by the arithmetic than the conflicts cost:
// 512 x 784 x 256 bf16 119 -> 125).  A distribution of more than `cap` categories passes twice, in chunks: once for its
// sum, once for its values.
constexpr uint32_t EV_THREADS = 256, EV_WARPS = 8, EV_COLUMNS = 256, EV_PITCH = 33;

struct EvidenceTile {
  uint32_t cap;         // columns of a tile
  uint32_t vars;        // variables per tile (1 where a variable has more than cap categories)
  uint32_t row_tiles, var_tiles, lg, each;   // tiles of rows and of variables; lanes per distribution (log2), elements per lane
  Form form;
};

template <typename T>
__host__ __device__ __forceinline__ uint32_t tile_place(uint32_t column, uint32_t lg) {
  return column * EV_PITCH + (sizeof(T) == 4 ? (column >> 5) << (5 - lg) : 0);
}

// a granule's columns from here on are EV_PITCH apart
template <typename T> __device__ __forceinline__ bool tile_run(uint32_t column) { return sizeof(T) == 2 || column % Vec<T>::N == 0; }

// The distributions of a tile: q = row * vars + variable.
struct TileOrder {
  uint32_t nv, magic;
  __device__ __forceinline__ explicit TileOrder(uint32_t nv_) : nv(nv_), magic(0xffffffffu / nv_ + 1) {}
  __device__ __forceinline__ uint32_t row(uint32_t q) const { return nv == 1 ? q : __umulhi(q, magic); }   // q < 2^13, nv <= 2^8
};

// Columns of the tile and rows-fastest memory from `at` on, a warp per column: f(place in the tile, pointer).
template <typename P, typename F>
__device__ __forceinline__ void tile_columns(uint32_t cats, uint32_t nv, uint64_t rows, uint32_t vars, P* at, F f) {
  const uint32_t warp = threadIdx.x >> 5;
  const uint64_t cat_step = rows * vars;
  if (nv == 1) {
    at += cat_step * warp;
    const uint64_t step = cat_step * EV_WARPS;
    uint32_t c = warp;
    for (; c + 3 * EV_WARPS < cats; c += 4 * EV_WARPS) {
#pragma unroll
      for (uint32_t k = 0; k < 4; ++k, at += step) f(c + k * EV_WARPS, at);
    }
    for (; c < cats; c += EV_WARPS, at += step) f(c, at);
  } else {
    uint32_t v = warp / cats, c = warp % cats;
    for (uint32_t column = warp; column < nv * cats; column += EV_WARPS) {
      f(column, at + rows * v + cat_step * c);
      c += EV_WARPS;
      while (c >= cats) { c -= cats; ++v; }
    }
  }
}

// A warp's statistics of a whole row of any length and alignment, in all lanes.
template <typename T>
__device__ float2 stream_row(const T* x, uint32_t cats, float c) {
  const uint32_t lane = threadIdx.x & 31;
  Part<T> p;
  p.off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  p.base = x - p.off;
  p.end = p.off + cats;
  const uint32_t granules = (uint32_t)(((uint64_t)p.end + Vec<T>::N - 1) / Vec<T>::N);
  float m = -INFINITY;
  float2 S2 = {0.0f, 0.0f}, none = {0.0f, 0.0f};
  for (uint32_t g0 = 0; g0 < granules; g0 += 128) {
    uint32_t w[16];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      uint4 q = {Word<T>::NONE, Word<T>::NONE, Word<T>::NONE, Word<T>::NONE};
      if (g0 + 32 * u + lane < granules) q = p.read(g0 + 32 * u + lane);
      w[4 * u] = q.x; w[4 * u + 1] = q.y; w[4 * u + 2] = q.z; w[4 * u + 3] = q.w;
    }
    const float most = most_of_words<T, 16>(w);
    if (most > m) {
      if (m != -INFINITY) {
        const float f = ex2_ftz(between(shift_of<T>(m, c), shift_of<T>(most, c)));
        S2 = mul2(S2, {f, f});
      }
      m = most;
    }
    add_words<T, 16, false>(w, shift_of<T>(m, c), S2, none);
  }
  const Stat s = lanes_join<T, 32>(Stat{m, S2.x + S2.y, 0.0f}, c);
  return {s.m, s.S};
}

template <typename T, int E, Form FORM>
__global__ void __launch_bounds__(EV_THREADS, sizeof(T) == 4 || FORM == ELEMENTS ? 4 : 5) evidence_kernel(EvidenceArgs a, EvidenceTile et) {
  using Row = ShortRow<T, E, FORM>;
  extern __shared__ __align__(16) float tile[];
  __shared__ float2 streamed[32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = et.lg, sub = lane & ((1u << lg) - 1), per_pass = EV_THREADS >> lg;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.row_stride + (a.vars - 1) * a.var_stride + a.cats)};
  const uint64_t b0 = (uint64_t)blockIdx.x * 32;   // neighbouring blocks write neighbouring rows
  for (uint32_t vt = blockIdx.y; vt < et.var_tiles; vt += gridDim.y) {
    const uint32_t v0 = vt * et.vars, nv = min(et.vars, a.vars - v0);
    const uint32_t rows = (uint32_t)min((uint64_t)32, a.rows - b0), width = min(a.cats, et.cap);   // categories of a pass
    const bool one = width == a.cats;
    const TileOrder order(nv);
    const T* x = static_cast<const T*>(a.x) + b0 * a.row_stride + (uint64_t)v0 * a.var_stride;
    if (!one) {
      for (uint32_t r = warp; r < rows; r += EV_WARPS) {
        const float2 s = stream_row<T>(x + r * a.row_stride, a.cats, a.c);
        if (lane == 0) streamed[r] = s;
      }
      __syncthreads();
    }
    for (uint32_t c0 = 0; c0 < a.cats; c0 += width) {
      const uint32_t n = min(width, a.cats - c0);
      for (uint32_t q0 = 0; q0 < rows * nv; q0 += per_pass) {
        const uint32_t q = q0 + (threadIdx.x >> lg), qq = min(q, rows * nv - 1), r = order.row(qq), v = qq - r * nv;
        Row in;
        in.load(x + r * a.row_stride + v * a.var_stride + c0, sub, lg, n, bounds);
        const uint64_t b = b0 + r;
        const bool missing = a.miss && a.miss[b * a.miss_row_stride + (v0 + v) * a.miss_var_stride];
        float m, S;
        if (one) {
          m = most_over_lanes(most_of_words<T, Row::W>(in.w), lg);
          float2 S2 = {0.0f, 0.0f}, none = {0.0f, 0.0f};
          add_words<T, Row::W, false>(in.w, shift_of<T>(m, a.c), S2, none);
          S = over_lanes(S2.x + S2.y, lg, sum_of);
        } else {
          m = streamed[r].x;
          S = streamed[r].y;
        }
        if (a.stats_out && c0 == 0 && sub == 0 && q == qq) reinterpret_cast<float2*>(a.stats_out)[b * a.vars + v0 + v] = {m, S};
        const LogScale l = log_scale<T>(shift_of<T>(m, a.c), S, a.invT);
        const uint32_t column = v * a.cats, mine = q == qq ? n : 0;   // a place is written where it lies below
#pragma unroll
        for (int e = 0; e < E; e += Row::N) {
          const uint32_t first = in.index(e, sub, lg);
          if (first < mine && first + Row::N <= mine && tile_run<T>(column + first)) {
            float* at = tile + tile_place<T>(column + first, lg) + r;
#pragma unroll
            for (uint32_t h = 0; h < Row::N; ++h) at[h * EV_PITCH] = missing ? 0.0f : logp_of(element_of<T>(in.w, e + h), l);
          } else {
#pragma unroll
            for (uint32_t h = 0; h < Row::N; ++h)
              if (first + h < mine) tile[tile_place<T>(column + first + h, lg) + r] = missing ? 0.0f : logp_of(element_of<T>(in.w, e + h), l);
          }
        }
      }
      __syncthreads();
      float* out = a.out + b0 + lane + a.rows * (v0 + (uint64_t)a.vars * c0);
      if (lane < rows) tile_columns(n, nv, a.rows, a.vars, out, [&](uint32_t column, float* at) { *at = tile[tile_place<T>(column, lg) + lane]; });
      __syncthreads();
    }
  }
}

// dx_c = (g_c - p_c sum g) / T
template <typename T, int E, Form FORM>
__global__ void __launch_bounds__(EV_THREADS, FORM == WHOLE ? 4 : 3) evidence_grad_kernel(EvidenceArgs a, EvidenceTile et) {
  using Row = ShortRow<T, E, FORM>;
  extern __shared__ __align__(16) float tile[];
  __shared__ float part[EV_WARPS][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = et.lg, sub = lane & ((1u << lg) - 1), per_pass = EV_THREADS >> lg;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.row_stride + (a.vars - 1) * a.var_stride + a.cats)};
  const uint64_t b0 = (uint64_t)blockIdx.x * 32;
  for (uint32_t vt = blockIdx.y; vt < et.var_tiles; vt += gridDim.y) {
    const uint32_t v0 = vt * et.vars, nv = min(et.vars, a.vars - v0);
    const uint32_t rows = (uint32_t)min((uint64_t)32, a.rows - b0), width = min(a.cats, et.cap);
    const bool one = width == a.cats;
    const TileOrder order(nv);
    const T* x = static_cast<const T*>(a.x) + b0 * a.row_stride + (uint64_t)v0 * a.var_stride;
    T* dx = static_cast<T*>(a.dx) + (b0 * a.vars + v0) * a.cats;
    const float* g = a.g + b0 + lane + a.rows * v0;
    if (!one) {   // the sum of all chunks first
      float sum = 0.0f;
      if (lane < rows) tile_columns(a.cats, 1, a.rows, a.vars, g, [&](uint32_t, const float* at) { sum += *at; });
      part[warp][lane] = sum;
    }
    for (uint32_t c0 = 0; c0 < a.cats; c0 += width) {
      const uint32_t n = min(width, a.cats - c0);
      const float* gc = g + a.rows * ((uint64_t)a.vars * c0);
      if (lane < rows) {
        uint32_t c = warp;
        if (nv == 1) {   // eight loads in flight
          const uint64_t step = a.rows * a.vars * EV_WARPS;
          const float* at = gc + a.rows * a.vars * warp;
          for (; c + 7 * EV_WARPS < n; c += 8 * EV_WARPS) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k, at += step) v[k] = *at;
#pragma unroll
            for (int k = 0; k < 8; ++k) tile[tile_place<T>(c + k * EV_WARPS, lg) + lane] = v[k];
          }
          for (; c < n; c += EV_WARPS, at += step) tile[tile_place<T>(c, lg) + lane] = *at;
        } else {
          tile_columns(n, nv, a.rows, a.vars, gc, [&](uint32_t column, const float* at) { tile[tile_place<T>(column, lg) + lane] = *at; });
        }
      }
      __syncthreads();
      for (uint32_t q0 = 0; q0 < rows * nv; q0 += per_pass) {
        const uint32_t q = q0 + (threadIdx.x >> lg), qq = min(q, rows * nv - 1), r = order.row(qq), v = qq - r * nv;
        Row in;
        in.load(x + r * a.row_stride + v * a.var_stride + c0, sub, lg, n, bounds);
        const uint64_t b = b0 + r;
        const bool missing = a.miss && a.miss[b * a.miss_row_stride + (v0 + v) * a.miss_var_stride];
        const float2 st = reinterpret_cast<const float2*>(a.stats)[b * a.vars + v0 + v];
        const uint32_t column = v * a.cats;
        float ge[E], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e += Row::N) {
          const uint32_t first = in.index(e, sub, lg);
          if (first < n && first + Row::N <= n && tile_run<T>(column + first)) {
            const float* at = tile + tile_place<T>(column + first, lg) + r;
#pragma unroll
            for (uint32_t h = 0; h < Row::N; ++h) ge[e + h] = at[h * EV_PITCH];
          } else {
#pragma unroll
            for (uint32_t h = 0; h < Row::N; ++h) ge[e + h] = first + h < n ? tile[tile_place<T>(column + first + h, lg) + r] : 0.0f;
          }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) sum += ge[e];
        if (one) {
          sum = over_lanes(sum, lg, sum_of);
        } else {
          sum = 0.0f;
          for (uint32_t k = 0; k < EV_WARPS; ++k) sum += part[k][r];
        }
        const Shift from = shift_of<T>(st.x, a.c);
        const float scale = missing || st.y == 0.0f ? 0.0f : a.invT, k = -sum / st.y * a.invT;
        uint32_t out[Row::W];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 xe = pair_of<T>(in.w, e);
          float2 d = fma2(xe, {from.c, from.c}, {-from.mc, -from.mc});
          if (!from.near) d = {scaled(from, xe.x), scaled(from, xe.y)};
          float2 value = fma2({ex2_ftz(d.x), ex2_ftz(d.y)}, {k, k}, mul2({ge[e], ge[e + 1]}, {scale, scale}));
          if (scale == 0.0f) value = {0.0f, 0.0f};
          if constexpr (sizeof(T) == 4) {
            out[e] = __float_as_uint(value.x);
            out[e + 1] = __float_as_uint(value.y);
          } else if constexpr (std::is_same<T, __half>::value) {
            out[e / 2] = Word<T>::bits(__floats2half2_rn(value.x, value.y));
          } else {
            out[e / 2] = Word<T>::bits(__floats2bfloat162_rn(value.x, value.y));
          }
        }
        if (q == qq) in.store(dx + ((uint64_t)r * a.vars + v) * a.cats + c0, out, sub, lg, n);
      }
      __syncthreads();
    }
  }
}

// Variables of at most 32 categories that lie one behind the other: a lane is a row, holds a distribution of at most C
// categories, and needs no shuffles; rows come (and the gradient's go) by elements, 32 neighbouring ones at a time.
template <typename T, int C, bool GRADIENT>
__global__ void __launch_bounds__(EV_THREADS, GRADIENT ? 3 : 4) evidence_thin_kernel(EvidenceArgs a, EvidenceTile et) {
  extern __shared__ __align__(16) float tile[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint64_t step = a.rows * a.vars, b0 = (uint64_t)blockIdx.x * 32, b = b0 + lane;
  for (uint32_t vt = blockIdx.y; vt < et.var_tiles; vt += gridDim.y) {
    const uint32_t v0 = vt * et.vars, nv = min(et.vars, a.vars - v0), columns = nv * a.cats;
    const uint32_t rows = (uint32_t)min((uint64_t)32, a.rows - b0);
    const T* x = static_cast<const T*>(a.x) + b0 * a.row_stride + (uint64_t)v0 * a.var_stride;
    for (uint32_t r = warp; r < rows; r += EV_WARPS) {
      const T* from = x + r * a.row_stride;
      T raw[EV_COLUMNS / 32];
#pragma unroll
      for (uint32_t k = 0; k < EV_COLUMNS / 32; ++k)
        if (32 * k + lane < columns) raw[k] = from[32 * k + lane];
#pragma unroll
      for (uint32_t k = 0; k < EV_COLUMNS / 32; ++k)
        if (32 * k + lane < columns) tile[(32 * k + lane) * EV_PITCH + r] = to_f32(raw[k]);
    }
    __syncthreads();
    for (uint32_t v = warp; v < nv; v += EV_WARPS) {
      if (lane >= rows) continue;
      float* at = tile + v * a.cats * EV_PITCH + lane;
      const bool missing = a.miss && a.miss[b * a.miss_row_stride + (v0 + v) * a.miss_var_stride];
      const uint64_t memory = b + a.rows * (v0 + v);
      float xc[C];
#pragma unroll
      for (int c = 0; c < C; ++c) xc[c] = c < (int)a.cats ? at[c * EV_PITCH] : -INFINITY;
      if constexpr (!GRADIENT) {
        float m = xc[0], S = 0.0f;
#pragma unroll
        for (int c = 1; c < C; ++c) m = fmaxf(m, xc[c]);
        m = fmaxf(m, -INFINITY);
        const Shift from = shift_of<T>(m, a.c);
        if (from.near) {
#pragma unroll
          for (int c = 0; c < C; ++c) S += ex2_ftz(fmaf(xc[c], from.c, -from.mc));
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) S += ex2_ftz(max_nan((xc[c] - finite_shift(m)) * from.c, NO_MASS));
        }
        const LogScale l = log_scale<T>(from, S, a.invT);
        if (a.stats_out) reinterpret_cast<float2*>(a.stats_out)[b * a.vars + v0 + v] = {m, S};
        float* out = a.out + memory;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c < (int)a.cats) out[step * c] = missing ? 0.0f : logp_of(xc[c], l);
      } else {
        const float* g = a.g + memory;
        float gc[C], sum = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) gc[c] = c < (int)a.cats ? g[step * c] : 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) sum += gc[c];
        const float2 st = reinterpret_cast<const float2*>(a.stats)[b * a.vars + v0 + v];
        const Shift from = shift_of<T>(st.x, a.c);
        const bool none = missing || st.y == 0.0f;
        const float k = sum / st.y;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c < (int)a.cats) at[c * EV_PITCH] = none ? 0.0f : (gc[c] - ex2_ftz(scaled(from, xc[c])) * k) * a.invT;
      }
    }
    __syncthreads();
    if constexpr (GRADIENT) {
      T* dx = static_cast<T*>(a.dx) + (b0 * a.vars + v0) * a.cats;
      for (uint32_t r = warp; r < rows; r += EV_WARPS) {
        T* to = dx + (uint64_t)r * a.vars * a.cats;
        for (uint32_t j = lane; j < columns; j += 32) to[j] = from_f32<T>(tile[j * EV_PITCH + r]);
      }
      __syncthreads();
    }
  }
}

// Tiles of up to EV_COLUMNS columns; a variable of up to EV_MOST categories is held whole.
template <typename T> constexpr uint32_t EV_MOST = 32 * Most<T>::E < 768 ? 32 * Most<T>::E : 768;
template <typename T>
EvidenceTile evidence_tile(const EvidenceArgs& a) {
  EvidenceTile t;
  t.vars = a.var_stride == a.cats && a.cats <= EV_COLUMNS / 2 ? std::min(EV_COLUMNS / a.cats, a.vars) : 1;
  t.cap = t.vars > 1 ? t.vars * a.cats : a.cats <= EV_MOST<T> ? a.cats : EV_COLUMNS;
  t.row_tiles = (uint32_t)((a.rows + 31) / 32);
  t.var_tiles = (a.vars - 1) / t.vars + 1;
  constexpr uint32_t N = Vec<T>::N;
  const auto whole_at = [&](uint64_t row, uint64_t var) { return ((row | (a.vars > 1 ? var : 0)) * sizeof(T) & 15) == 0; };
  const bool whole = (reinterpret_cast<uintptr_t>(a.x) & 15) == 0 && whole_at(a.row_stride, a.var_stride) && a.cats % N == 0;
  // dx is contiguous: it has to lie towards 16-byte boundaries as x does
  const bool alike = !a.dx || (((reinterpret_cast<uintptr_t>(a.x) ^ reinterpret_cast<uintptr_t>(a.dx)) & 15) == 0 &&
                               whole_at(a.row_stride - (uint64_t)a.vars * a.cats, a.var_stride - a.cats));
  const uint32_t n = std::min(a.cats, t.cap), units = whole ? n / N : (n + 2 * N - 2) / N;
  t.form = alike && units <= 32 * Most<T>::E / N && (whole || n * sizeof(T) >= 64) ? whole ? WHOLE : LOOSE : ELEMENTS;
  const bool granules = t.form != ELEMENTS;
  // few lanes per distribution; four at least where it is read in granules, eight where it is read by elements
  const uint32_t parts = granules ? units : n, most = granules ? Most<T>::E / N : Most<T>::E, wanted = granules ? 4 : 8;
  t.lg = 0;
  while (t.lg < 5 && (parts > (most << t.lg) || (1u << t.lg) < std::min(parts, wanted))) ++t.lg;
  t.each = ((parts + (1u << t.lg) - 1) >> t.lg) * (granules ? N : 1);
  return t;
}

template <typename T, int E, Form FORM>
cudaError_t launch_evidence_as(const EvidenceArgs& a, const EvidenceTile& t, cudaStream_t st) {
  const dim3 grid(t.row_tiles, std::min(t.var_tiles, 65535u));
  const uint32_t smem = (tile_place<T>(t.cap, t.lg) + 32) * (uint32_t)sizeof(float);
  static PcbPerDeviceOnce once;
  const cudaError_t e = once.run([] {
    const int most = (int)((tile_place<T>(768, 0) + 32) * sizeof(float));
    const cudaError_t f = cudaFuncSetAttribute(evidence_kernel<T, E, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return f != cudaSuccess ? f : cudaFuncSetAttribute(evidence_grad_kernel<T, E, FORM>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  });
  if (e != cudaSuccess) return e;
  if (a.dx) evidence_grad_kernel<T, E, FORM><<<grid, EV_THREADS, smem, st>>>(a, t);
  else evidence_kernel<T, E, FORM><<<grid, EV_THREADS, smem, st>>>(a, t);
  return cudaGetLastError();
}
template <typename T, int E>
cudaError_t launch_evidence_of(const EvidenceArgs& a, const EvidenceTile& t, cudaStream_t st) {
  if constexpr (E >= (int)Vec<T>::N) {
    if (t.form == WHOLE) return launch_evidence_as<T, E, WHOLE>(a, t, st);
    if (t.form == LOOSE) return launch_evidence_as<T, E, LOOSE>(a, t, st);
  }
  return launch_evidence_as<T, E, ELEMENTS>(a, t, st);
}
template <typename T, int C>
cudaError_t launch_thin(const EvidenceArgs& a, const EvidenceTile& t, cudaStream_t st) {
  const dim3 grid(t.row_tiles, std::min(t.var_tiles, 65535u));
  const uint32_t smem = t.cap * EV_PITCH * (uint32_t)sizeof(float);
  if (a.dx) evidence_thin_kernel<T, C, true><<<grid, EV_THREADS, smem, st>>>(a, t);
  else evidence_thin_kernel<T, C, false><<<grid, EV_THREADS, smem, st>>>(a, t);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_evidence(const EvidenceArgs& a, cudaStream_t st) {   // the gradient where dx is given
  const EvidenceTile t = evidence_tile<T>(a);
  if (a.cats <= 32 && (t.vars > 1 || a.vars == 1)) {
    if (a.cats <= 2) return launch_thin<T, 2>(a, t, st);
    if (a.cats <= 4) return launch_thin<T, 4>(a, t, st);
    if (a.cats <= 8) return launch_thin<T, 8>(a, t, st);
    if (a.cats <= 16) return launch_thin<T, 16>(a, t, st);
    return launch_thin<T, 32>(a, t, st);
  }
  if (t.each <= 4) return launch_evidence_of<T, 4>(a, t, st);
  if (t.each <= 8) return launch_evidence_of<T, 8>(a, t, st);
  if (t.each <= 16) return launch_evidence_of<T, 16>(a, t, st);
  return launch_evidence_of<T, Most<T>::E>(a, t, st);
}

int32_t check_logits(const void* x, int32_t dtype, uint32_t cats, float temperature) {
  PCB_REQUIRE(x, "null logits");
  PCB_REQUIRE(dtype == PCB_F32 || dtype == PCB_BF16 || dtype == PCB_F16, "logits are f32, bf16 or f16");
  PCB_REQUIRE(((uintptr_t)x & (dtype == PCB_F32 ? 3 : 1)) == 0, "logits that are not aligned to their own size");
  PCB_REQUIRE(cats >= 1 && cats <= 0x7fffffffu, "the number of categories must be between 1 and 2^31 - 1");
  PCB_REQUIRE(temperature > 0.0f && LOG2E / temperature < INFINITY && 1.0f / temperature > 0.0f, "the temperature must be positive and finite");
  return PCB_OK;
}

}  // namespace

extern "C" int32_t pcb_token_logprobs(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t cats, uint64_t row_stride,
                                      float temperature, const void* tokens_dev, uint32_t token_bytes, uint32_t top_k,
                                      float* logp_out_dev, float* entropy_dev, float* stats_dev, int64_t* top_ids_dev,
                                      float* top_logp_dev, pcb_stream s) {
  if (rows == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(entropy_dev && ((uintptr_t)stats_dev & 7) == 0, "null argument, or statistics that are not 8-byte aligned");
  PCB_REQUIRE(!tokens_dev || (logp_out_dev && (token_bytes == 4 || token_bytes == 8)), "tokens are int32 or int64 and need an output");
  PCB_REQUIRE(top_k <= MAX_TOP && top_k <= cats, "at most 32 alternatives, and no more than there are categories");
  PCB_REQUIRE(top_k == 0 || (top_ids_dev && top_logp_dev), "alternatives need their outputs");
  LogprobArgs a{x_dev, rows, row_stride, cats, top_k, token_bytes, 1.0f / temperature, LOG2E / temperature, tokens_dev,
                logp_out_dev, entropy_dev, stats_dev, top_logp_dev, top_ids_dev};
  const uint32_t sms = pcb_sm_count();
  if (sms == 0) return pcb_fail(PCB_ERR_CUDA, "no CUDA device");
  PCB_CUDA(dtype == PCB_F32 ? launch_rows<float>(a, sms, (cudaStream_t)s) : dtype == PCB_BF16 ? launch_rows<__nv_bfloat16>(a, sms, (cudaStream_t)s)
                                                                                          : launch_rows<__half>(a, sms, (cudaStream_t)s));
  return PCB_OK;
}

extern "C" int32_t pcb_token_logprobs_backward(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t cats, uint64_t row_stride,
                                               float temperature, const void* tokens_dev, uint32_t token_bytes, uint32_t top_k,
                                               const int64_t* top_ids_dev, const float* stats_dev, const float* entropy_dev,
                                               const float* g_logp_dev, uint64_t g_logp_stride, const float* g_entropy_dev,
                                               uint64_t g_entropy_stride, const float* g_top_dev, void* dx_dev, pcb_stream s) {
  if (rows == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(stats_dev && entropy_dev && dx_dev, "null argument");
  PCB_REQUIRE(((uintptr_t)dx_dev & (dtype == PCB_F32 ? 3 : 1)) == 0, "a gradient that is not aligned to its own size");
  PCB_REQUIRE(!g_logp_dev || (tokens_dev && (token_bytes == 4 || token_bytes == 8)), "a gradient of logp needs the tokens, int32 or int64");
  PCB_REQUIRE(top_k <= MAX_TOP && top_k <= cats, "at most 32 alternatives, and no more than there are categories");
  PCB_REQUIRE(!g_top_dev || (top_k > 0 && top_ids_dev), "a gradient of the alternatives needs their indices");
  LogprobGradArgs a{x_dev, rows, row_stride, g_logp_stride, g_entropy_stride, cats, top_k, token_bytes, 1.0f / temperature,
                    LOG2E / temperature, tokens_dev, top_ids_dev, stats_dev, entropy_dev, g_logp_dev, g_entropy_dev, g_top_dev, dx_dev};
  const uint32_t sms = pcb_sm_count();
  if (sms == 0) return pcb_fail(PCB_ERR_CUDA, "no CUDA device");
  if (dtype == PCB_F32) launch_grad<float>(a, sms, (cudaStream_t)s);
  else if (dtype == PCB_BF16) launch_grad<__nv_bfloat16>(a, sms, (cudaStream_t)s);
  else launch_grad<__half>(a, sms, (cudaStream_t)s);
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_soft_evidence(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t vars, uint32_t cats,
                                     uint64_t row_stride, uint64_t var_stride, const uint8_t* miss_dev, uint64_t miss_row_stride,
                                     uint64_t miss_var_stride, float temperature, float* out_dev, float* stats_dev, pcb_stream s) {
  if (rows == 0 || vars == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(out_dev, "null argument");
  EvidenceArgs a{x_dev, rows, row_stride, var_stride, miss_row_stride, miss_var_stride, vars, cats, 1.0f / temperature,
                 LOG2E / temperature, miss_dev, out_dev, stats_dev, nullptr, nullptr, nullptr};
  PCB_REQUIRE(!stats_dev || ((uintptr_t)stats_dev & 7) == 0, "statistics that are not 8-byte aligned");
  PCB_REQUIRE(rows < (1ull << 35), "at most 2^35 rows");
  cudaStream_t st = (cudaStream_t)s;
  PCB_CUDA(dtype == PCB_F32 ? launch_evidence<float>(a, st) : dtype == PCB_BF16 ? launch_evidence<__nv_bfloat16>(a, st) : launch_evidence<__half>(a, st));
  return PCB_OK;
}

extern "C" int32_t pcb_soft_evidence_backward(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t vars, uint32_t cats,
                                              uint64_t row_stride, uint64_t var_stride, const uint8_t* miss_dev,
                                              uint64_t miss_row_stride, uint64_t miss_var_stride, float temperature,
                                              const float* stats_dev, const float* g_dev, void* dx_dev, pcb_stream s) {
  if (rows == 0 || vars == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(stats_dev && g_dev && dx_dev, "null argument");
  PCB_REQUIRE(((uintptr_t)dx_dev & (dtype == PCB_F32 ? 3 : 1)) == 0, "a gradient that is not aligned to its own size");
  EvidenceArgs a{x_dev, rows, row_stride, var_stride, miss_row_stride, miss_var_stride, vars, cats, 1.0f / temperature,
                 LOG2E / temperature, miss_dev, nullptr, nullptr, stats_dev, g_dev, dx_dev};
  PCB_REQUIRE(((uintptr_t)stats_dev & 7) == 0, "statistics that are not 8-byte aligned");
  PCB_REQUIRE(rows < (1ull << 35), "at most 2^35 rows");
  cudaStream_t st = (cudaStream_t)s;
  PCB_CUDA(dtype == PCB_F32 ? launch_evidence<float>(a, st) : dtype == PCB_BF16 ? launch_evidence<__nv_bfloat16>(a, st)
                                                                                    : launch_evidence<__half>(a, st));
  return PCB_OK;
}
