// pcb_logits.cu — categorical distributions given by logits: log-probabilities of given categories with entropy and
// best alternatives, their gradient, and soft evidence made of logits, with its gradient.
//
// With s = x / T, m = max x and c = log2(e) / T every kernel works on d_j = (x_j - m) c, so that exp(s_j - max s) =
// 2^d_j: the difference is taken before the scaling, which keeps a row of the type's lowest values (a mask) finite where
// x c would overflow.  S = sum 2^d, A = sum 2^d d:
//   logp_j = (x_j - m) / T - ln S          H = ln S - ln2 A / S          p_j = 2^d_j / S
// Terms of impossible categories (d = -inf) are clamped at -200, where 2^d is zero in fp32: 0 * inf stays out of A, and
// NaN still passes (max.NaN).  A row without any possible category has S = 0, logp -inf, H = 0 and gradient 0.
#include "pcb_internal.h"
#include "pcb_tc.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

struct Stat { float m, S, A; };   // running maximum, sum of 2^d, sum of 2^d d

__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  // a side without a possible value has S = 0 (or NaN, which has to pass): taken as it is
  const float da = a.m == -INFINITY ? 0.0f : max_nan((a.m - r.m) * c, NO_MASS);
  const float db = b.m == -INFINITY ? 0.0f : max_nan((b.m - r.m) * c, NO_MASS);
  const float fa = ex2_ftz(da), fb = ex2_ftz(db);
  r.S = a.S * fa + b.S * fb;
  r.A = fa * (a.A + da * a.S) + fb * (b.A + db * b.S);
  return r;
}
__device__ __forceinline__ Stat warp_join(Stat s, float c) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    Stat t;
    t.m = __shfl_xor_sync(0xffffffffu, s.m, o);
    t.S = __shfl_xor_sync(0xffffffffu, s.S, o);
    t.A = __shfl_xor_sync(0xffffffffu, s.A, o);
    s = join(s, t, c);
  }
  return s;
}
// one more value into a running statistic
__device__ __forceinline__ void put(Stat& s, float x, float c) {
  if (x > s.m) {
    const float d = max_nan((s.m - x) * c, NO_MASS), f = ex2_ftz(d);   // s.m may be -inf: d = -200, f = 0
    s.A = f * (s.A + d * s.S);
    s.S *= f;
    s.m = x;
  }
  const float d = max_nan((x - finite_shift(s.m)) * c, NO_MASS), e = ex2_ftz(d);
  s.S += e;
  s.A += e * d;
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

// log-probability of the value x in a row of statistics (m, ln S)
__device__ __forceinline__ float logp_of(float x, float m, float lnS, float invT) {
  return m == -INFINITY && !(lnS != lnS) ? -INFINITY : (x - m) * invT - lnS;
}

// the row's results but for the alternatives
template <typename T>
__device__ void write_row(const LogprobArgs& a, uint64_t row, const T* x, Stat s) {
  const float lnS = s.m == -INFINITY && s.S == 0.0f ? 0.0f : logf(s.S);
  if (a.tokens) {
    const int64_t t = token_at(a.tokens, a.token_bytes, row);
    a.logp[row] = t < 0 ? 0.0f : t >= (int64_t)a.cats ? NAN : logp_of(to_f32(x[t]), s.m, lnS, a.invT);
  }
  a.entropy[row] = s.m == -INFINITY && s.S == 0.0f ? 0.0f : lnS - LN2 * s.A / s.S;
  a.stats[2 * row] = s.m;
  a.stats[2 * row + 1] = s.S;
}

// One block per row: the statistics of the threads' values joined, then one pass per alternative.
template <typename T>
__global__ void __launch_bounds__(256) logprob_row_kernel(LogprobArgs a) {
  __shared__ Stat part[8];
  __shared__ uint64_t best[8];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    Stat s{-INFINITY, 0.0f, 0.0f};
    for (uint32_t j = threadIdx.x; j < a.cats; j += blockDim.x) put(s, to_f32(x[j]), a.c);
    s = warp_join(s, a.c);
    if (lane == 0) part[warp] = s;
    __syncthreads();
    s = part[0];
    for (uint32_t w = 1; w < 8; ++w) s = join(s, part[w], a.c);
    if (threadIdx.x == 0) write_row(a, row, x, s);
    const float lnS = s.m == -INFINITY && s.S == 0.0f ? 0.0f : logf(s.S);
    uint64_t last = ~0ull;
    for (uint32_t k = 0; k < a.top_k; ++k) {
      uint64_t key = 0;
      for (uint32_t j = threadIdx.x; j < a.cats; j += blockDim.x) {
        const uint64_t o = order_key(to_f32(x[j]), j);
        if (o < last && o > key) key = o;
      }
      for (int o = 16; o; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
      if (lane == 0) best[warp] = key;
      __syncthreads();
      key = best[0];
      for (uint32_t w = 1; w < 8; ++w) key = max(key, best[w]);
      if (threadIdx.x == 0) {
        const uint32_t j = ~(uint32_t)key;
        a.top_ids[row * a.top_k + k] = j;
        a.top_logp[row * a.top_k + k] = logp_of(to_f32(x[j]), s.m, lnS, a.invT);
      }
      last = key;
      __syncthreads();
    }
    __syncthreads();
  }
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
  float m, S, alpha, beta, gl;
  int64_t token;   // negative: none
};
__device__ __forceinline__ RowGrad row_grad(const LogprobGradArgs& a, uint64_t row) {
  RowGrad g;
  g.m = a.stats[2 * row];
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
__device__ __forceinline__ float grad_of(const RowGrad& g, float x, float c) {
  const float d = max_nan((x - g.m) * c, NO_MASS);
  return ex2_ftz(d) * fmaf(g.beta, d, g.alpha);
}
__device__ __forceinline__ bool no_mass(const RowGrad& g) { return g.S == 0.0f; }
// the whole gradient of an element that the token or an alternative may point to
__device__ __forceinline__ float pointed_grad(const LogprobGradArgs& a, const RowGrad& g, uint64_t row, uint32_t j, float x) {
  if (no_mass(g)) return 0.0f;
  float v = grad_of(g, x, a.c);
  if (g.token == (int64_t)j) v += g.gl * a.invT;
  if (a.g_top)
    for (uint32_t k = 0; k < a.top_k; ++k)
      if (a.top_ids[row * a.top_k + k] == (int64_t)j) v += a.g_top[row * a.top_k + k] * a.invT;
  return v;
}

template <typename T>
__global__ void __launch_bounds__(256) logprob_grad_kernel(LogprobGradArgs a) {
  for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.stride;
    T* dx = static_cast<T*>(a.dx) + row * a.cats;
    const RowGrad g = row_grad(a, row);
    for (uint32_t j = threadIdx.x; j < a.cats; j += blockDim.x) dx[j] = from_f32<T>(pointed_grad(a, g, row, j, to_f32(x[j])));
  }
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

// One warp per (row, variable).
template <typename T>
__global__ void __launch_bounds__(256) evidence_kernel(EvidenceArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t total = a.rows * a.vars;
  for (uint64_t i = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < total; i += (uint64_t)gridDim.x * 8) {
    const uint64_t b = i % a.rows;
    const uint32_t v = (uint32_t)(i / a.rows);
    const T* x = static_cast<const T*>(a.x) + b * a.row_stride + v * a.var_stride;
    float* out = a.out + b + a.rows * v;
    const uint64_t step = a.rows * a.vars;
    const bool missing = a.miss && a.miss[b * a.miss_row_stride + v * a.miss_var_stride];
    Stat s{-INFINITY, 0.0f, 0.0f};
    for (uint32_t j = lane; j < a.cats; j += 32) put(s, to_f32(x[j]), a.c);
    s = warp_join(s, a.c);
    const float lnS = s.m == -INFINITY && s.S == 0.0f ? 0.0f : logf(s.S);
    for (uint32_t j = lane; j < a.cats; j += 32) out[j * step] = missing ? 0.0f : logp_of(to_f32(x[j]), s.m, lnS, a.invT);
    if (a.stats_out && lane == 0) {
      a.stats_out[2 * (b * a.vars + v)] = s.m;
      a.stats_out[2 * (b * a.vars + v) + 1] = s.S;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) evidence_grad_kernel(EvidenceArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t total = a.rows * a.vars;
  for (uint64_t i = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < total; i += (uint64_t)gridDim.x * 8) {
    const uint64_t b = i % a.rows;
    const uint32_t v = (uint32_t)(i / a.rows);
    const T* x = static_cast<const T*>(a.x) + b * a.row_stride + v * a.var_stride;
    const float* g = a.g + b + a.rows * v;
    T* dx = static_cast<T*>(a.dx) + (b * a.vars + v) * a.cats;
    const uint64_t step = a.rows * a.vars;
    const float m = a.stats[2 * (b * a.vars + v)], S = a.stats[2 * (b * a.vars + v) + 1];
    const bool none = (a.miss && a.miss[b * a.miss_row_stride + v * a.miss_var_stride]) || S == 0.0f;
    float sum = 0.0f;
    for (uint32_t j = lane; j < a.cats; j += 32) sum += g[j * step];
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    for (uint32_t j = lane; j < a.cats; j += 32) {
      const float e = ex2_ftz(max_nan((to_f32(x[j]) - m) * a.c, NO_MASS));
      dx[j] = from_f32<T>(none ? 0.0f : (g[j * step] - e * (sum / S)) * a.invT);
    }
  }
}

int32_t check_logits(const void* x, int32_t dtype, uint32_t cats, float temperature) {
  PCB_REQUIRE(x, "null logits");
  PCB_REQUIRE(dtype == PCB_F32 || dtype == PCB_BF16 || dtype == PCB_F16, "logits are f32, bf16 or f16");
  PCB_REQUIRE(cats >= 1 && cats <= 0x7fffffffu, "the number of categories must be between 1 and 2^31 - 1");
  PCB_REQUIRE(temperature > 0.0f && LOG2E / temperature < INFINITY && 1.0f / temperature > 0.0f, "the temperature must be positive and finite");
  return PCB_OK;
}

// kernel<T><<<...>>>(args) for the logits' type
#define PCB_BY_DTYPE(dtype, kernel, grid, block, smem, st, args)                               \
  do {                                                                                         \
    if ((dtype) == PCB_F32) kernel<float><<<grid, block, smem, st>>>(args);                    \
    else if ((dtype) == PCB_BF16) kernel<__nv_bfloat16><<<grid, block, smem, st>>>(args);      \
    else kernel<__half><<<grid, block, smem, st>>>(args);                                      \
  } while (0)

}  // namespace

extern "C" int32_t pcb_token_logprobs(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t cats, uint64_t row_stride,
                                      float temperature, const void* tokens_dev, uint32_t token_bytes, uint32_t top_k,
                                      float* logp_out_dev, float* entropy_dev, float* stats_dev, int64_t* top_ids_dev,
                                      float* top_logp_dev, pcb_stream s) {
  if (rows == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(entropy_dev && stats_dev, "null argument");
  PCB_REQUIRE(!tokens_dev || (logp_out_dev && (token_bytes == 4 || token_bytes == 8)), "tokens are int32 or int64 and need an output");
  PCB_REQUIRE(top_k <= MAX_TOP && top_k <= cats, "at most 32 alternatives, and no more than there are categories");
  PCB_REQUIRE(top_k == 0 || (top_ids_dev && top_logp_dev), "alternatives need their outputs");
  LogprobArgs a{x_dev, rows, row_stride, cats, top_k, token_bytes, 1.0f / temperature, LOG2E / temperature, tokens_dev,
                logp_out_dev, entropy_dev, stats_dev, top_logp_dev, top_ids_dev};
  const uint32_t grid = (uint32_t)(rows < 0x7fffffffull ? rows : 0x7fffffffull);
  PCB_BY_DTYPE(dtype, logprob_row_kernel, grid, 256, 0, (cudaStream_t)s, a);
  PCB_CUDA(cudaGetLastError());
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
  PCB_REQUIRE(!g_logp_dev || (tokens_dev && (token_bytes == 4 || token_bytes == 8)), "a gradient of logp needs the tokens, int32 or int64");
  PCB_REQUIRE(top_k <= MAX_TOP && top_k <= cats, "at most 32 alternatives, and no more than there are categories");
  PCB_REQUIRE(!g_top_dev || (top_k > 0 && top_ids_dev), "a gradient of the alternatives needs their indices");
  LogprobGradArgs a{x_dev, rows, row_stride, g_logp_stride, g_entropy_stride, cats, top_k, token_bytes, 1.0f / temperature,
                    LOG2E / temperature, tokens_dev, top_ids_dev, stats_dev, entropy_dev, g_logp_dev, g_entropy_dev, g_top_dev, dx_dev};
  const uint32_t grid = (uint32_t)(rows < 0x7fffffffull ? rows : 0x7fffffffull);
  PCB_BY_DTYPE(dtype, logprob_grad_kernel, grid, 256, 0, (cudaStream_t)s, a);
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
  const uint64_t blocks = (rows * vars + 7) / 8;
  const uint32_t grid = (uint32_t)(blocks < 0x7fffffffull ? blocks : 0x7fffffffull);
  PCB_BY_DTYPE(dtype, evidence_kernel, grid, 256, 0, (cudaStream_t)s, a);
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_soft_evidence_backward(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t vars, uint32_t cats,
                                              uint64_t row_stride, uint64_t var_stride, const uint8_t* miss_dev,
                                              uint64_t miss_row_stride, uint64_t miss_var_stride, float temperature,
                                              const float* stats_dev, const float* g_dev, void* dx_dev, pcb_stream s) {
  if (rows == 0 || vars == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(stats_dev && g_dev && dx_dev, "null argument");
  EvidenceArgs a{x_dev, rows, row_stride, var_stride, miss_row_stride, miss_var_stride, vars, cats, 1.0f / temperature,
                 LOG2E / temperature, miss_dev, nullptr, nullptr, stats_dev, g_dev, dx_dev};
  const uint64_t blocks = (rows * vars + 7) / 8;
  const uint32_t grid = (uint32_t)(blocks < 0x7fffffffull ? blocks : 0x7fffffffull);
  PCB_BY_DTYPE(dtype, evidence_grad_kernel, grid, 256, 0, (cudaStream_t)s, a);
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}
