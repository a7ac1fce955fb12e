// pcb_logits_grad.cu — the gradient of log-probabilities, entropy and alternatives with respect to the logits.
#include "pcb_logits.cuh"

namespace {

using namespace pcblogits;

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
  g.S = sum_in(g.from, a.stats[2 * row + 1]);
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
  const float d = scaled(g.from, x), power = ex2_ftz(d);
  return fmaf(power * d, g.beta, power * g.alpha);
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
// p_j alpha + p_j d beta of W words, as words
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
    // 2^d d first: it is 0 where 2^d is, while beta d passes the range beside a floor's d of -1e30 and more
    const float2 power = {ex2_ftz(d.x), ex2_ftz(d.y)}, v = fma2(mul2(power, d), {beta, beta}, mul2(power, {alpha, alpha}));
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
// towards 16-byte boundaries, by elements otherwise.  Small blocks: they wait for one another's stores before what is pointed to
// is written (us both directions, 256 / 128 / 64 threads: 1021 rows of 50021 bf16 75.3 / 73.2 / 73.6, 20000 of 2000 130 / 92 / 76).
// The last rows come first: the forward pass read them last, and some of them are still in the L2 cache.  The logits twice and
// the gradient once move at 4.2 TB/s in both directions together (two thirds of a copy; 102 MB of logits).  Bound by
// instructions as much as by memory: 72 % of the issue slots are taken, since every thread prepares its row.
constexpr uint32_t GRAD_THREADS = 64, GRAD_TILE = 64 * GRAD_THREADS;
static_assert(GRAD_THREADS > MAX_TOP, "a thread for the token and for every alternative");
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
// once, lane (g, j) prepares the g-th row of pass j, and the next rows are on their way while it works on these.  235200 rows of
// 200 fp32, both directions 119 us: logits twice and gradient once at 4.8 TB/s, three quarters of a copy.
template <typename T, int E, Form FORM, int LG>
__global__ void __launch_bounds__(256, E >= 16 ? 3 : 5) logprob_grad_short_kernel(LogprobGradArgs a, uint32_t lanes_log2, uint32_t passes) {
  using Row = ShortRow<T, E, FORM>;
  const uint32_t lg = LG >= 0 ? (uint32_t)LG : lanes_log2;
  const uint32_t lane = threadIdx.x & 31, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.stride + a.cats)};
  const uint64_t rows_each = (uint64_t)per_warp * passes, all = (a.rows + rows_each - 1) / rows_each, step = (uint64_t)gridDim.x * 8;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += step) {
    const uint64_t r0 = (all - 1 - i) * rows_each, first = min(a.rows - 1, r0 + group);   // the last rows first
    const uint32_t there = (uint32_t)min((uint64_t)passes, (a.rows - r0 + per_warp - 1) / per_warp);   // passes with rows
    const uint32_t last = (uint32_t)min((uint64_t)passes, (a.rows - 1 - first) / per_warp);            // this lane's last pass with a row
    const T* x = static_cast<const T*>(a.x) + first * a.stride;
    T* dx0 = static_cast<T*>(a.dx) + first * a.cats;
    const auto row_at = [&](uint32_t pass) { return x + (uint64_t)(min(pass, last) * per_warp) * a.stride; };
    Row next;
    next.load(row_at(0), sub, lg, a.cats, bounds);
    const RowGrad mine = row_grad<T>(a, min(a.rows - 1, r0 + min(sub, passes - 1) * per_warp + group));
    const int32_t my_token = mine.token >= 0 && mine.token < (int64_t)a.cats ? (int32_t)mine.token : -1;
    for (uint32_t pass = 0; pass < there; ++pass) {
      const Row r = next;
      if (pass + 1 < there) next.load(row_at(pass + 1), sub, lg, a.cats, bounds);
      const uint32_t from = (lane & ~((1u << lg) - 1)) + pass;   // the lane that prepared this row
      RowGrad g;
      g.from = shift_of<T>(__shfl_sync(0xffffffffu, mine.from.m, from), a.c);
      g.S = __shfl_sync(0xffffffffu, mine.S, from);
      g.alpha = __shfl_sync(0xffffffffu, mine.alpha, from);
      g.beta = __shfl_sync(0xffffffffu, mine.beta, from);
      g.gl = __shfl_sync(0xffffffffu, mine.gl, from);
      g.token = __shfl_sync(0xffffffffu, my_token, from);
      const uint64_t row = first + min(pass, last) * per_warp;
      const bool valid = r0 + group < a.rows && pass <= last;
      T* dx = dx0 + (uint64_t)(min(pass, last) * per_warp) * a.cats;
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
          if (valid && j >= 0 && j < (int64_t)a.cats) dx[j] = from_f32<T>(pointed_grad(a, g, row, (uint32_t)j, to_f32(row_at(pass)[j])));
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
#define PCB_CALL(LG) logprob_grad_short_kernel<T, E, FORM, LG><<<grid, 256, 0, st>>>(a, lg, passes)
  constexpr bool full = E == (int)Most<T>::E;
  if constexpr (E >= (int)Vec<T>::N) {
    if (s.form == WHOLE) {
      constexpr Form FORM = WHOLE;
      if constexpr (full) PCB_LANES(true, lg, PCB_CALL);
      else PCB_CALL(-1);
      return;
    }
    if (s.form == LOOSE) {
      constexpr Form FORM = LOOSE;
      if constexpr (full) PCB_LANES(true, lg, PCB_CALL);
      else PCB_CALL(-1);
      return;
    }
  }
  constexpr Form FORM = ELEMENTS;
  PCB_CALL(-1);
#undef PCB_CALL
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

}  // namespace

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
  PCB_REQUIRE(!g_logp_dev || (uintptr_t)tokens_dev % token_bytes == 0, "tokens that are not aligned to their own size");
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
