// pcb_evidence.cu — soft evidence made of logits, and its gradient.
#include "pcb_logits.cuh"

namespace {

using namespace pcblogits;

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
// 512 x 784 x 256 bf16 119 -> 125).  512 x 784 x 256 bf16 takes 104 us (5.9 TB/s, 92 % of a copy), 37 x 192 x 500 fp32 12.2 us: a
// few tiles per SM, latency; forward and gradient of 500 x 192 x 256 fp16 81 us (4.2 TB/s with the logits read twice): what
// bounds the gradient is the way of g and of dx through shared memory between two barriers.  A distribution of more than `cap` categories passes twice, in chunks: once for its
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

template <typename T, int E, Form FORM, int LG>
__global__ void __launch_bounds__(EV_THREADS, sizeof(T) == 4 || FORM == ELEMENTS ? 4 : 5) evidence_kernel(EvidenceArgs a, EvidenceTile et) {
  using Row = ShortRow<T, E, FORM>;
  extern __shared__ __align__(16) float tile[];
  __shared__ float2 streamed[32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = LG >= 0 ? (uint32_t)LG : et.lg, sub = lane & ((1u << lg) - 1), per_pass = EV_THREADS >> lg;
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
        const Shift from = shift_of<T>(m, a.c);
        if (a.stats_out && c0 == 0 && sub == 0 && q == qq) reinterpret_cast<float2*>(a.stats_out)[b * a.vars + v0 + v] = {m, sum_out(from, S)};
        const LogScale l = log_scale<T>(from, S, a.invT);
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
template <typename T, int E, Form FORM, int LG>
__global__ void __launch_bounds__(EV_THREADS, FORM == WHOLE ? 4 : 3) evidence_grad_kernel(EvidenceArgs a, EvidenceTile et) {
  using Row = ShortRow<T, E, FORM>;
  extern __shared__ __align__(16) float tile[];
  __shared__ float part[EV_WARPS][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = LG >= 0 ? (uint32_t)LG : et.lg, sub = lane & ((1u << lg) - 1), per_pass = EV_THREADS >> lg;
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
        const float scale = missing || st.y == 0.0f ? 0.0f : a.invT, k = -sum / sum_in(from, st.y) * a.invT;
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
// categories, and needs no shuffles; rows come (and the gradient's go) by elements, 32 neighbouring ones at a time.  What lies by
// rows goes through shared memory too, since a load by a lane per row touches 32 lines: statistics always, missing variables
// where there are many (gradient, us by rows / by lanes: 1000 x 784 x 2 16.3 / 20.9, 100 x 784 x 8 10.2 / 9.6, 500 x 192 x 16 12.7 / 12.2).
// The gradient makes the statistics anew, from the powers that it needs anyway, and asks for the g of several short distributions
// at a time (16000 x 784 x 2: 183 us, one at a time 208).  Bound by the 32-byte pieces that rows of few columns come and go in,
// and by latency in small batches: 2.3 TB/s at 16000 x 784 x 2, 2.8 TB/s one way at 5000 x 784 x 4 bf16.
template <typename T, int C, bool GRADIENT>
__global__ void __launch_bounds__(EV_THREADS, C <= 8 ? 5 : GRADIENT ? 3 : 4) evidence_thin_kernel(EvidenceArgs a, EvidenceTile et) {
  constexpr bool BY_ROWS = C <= 4;
  constexpr uint32_t AT_ONCE = GRADIENT && C <= 8 ? 8 / C : 1;   // variables
  extern __shared__ __align__(16) float tile[];
  __shared__ uint32_t missing_bits[EV_COLUMNS / 32][32];   // [variables / 32][row]
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
    if (BY_ROWS && a.miss) {
      const uint8_t* miss = a.miss + b0 * a.miss_row_stride + (v0 + lane) * a.miss_var_stride;
      for (uint32_t k = 0; 32 * k < nv; ++k, miss += 32 * a.miss_var_stride) {
        uint8_t gone[32 / EV_WARPS];
#pragma unroll
        for (uint32_t i = 0; i < 32 / EV_WARPS; ++i) {
          const uint32_t r = warp + i * EV_WARPS;
          gone[i] = r < rows && 32 * k + lane < nv ? miss[r * a.miss_row_stride] : 0;
        }
#pragma unroll
        for (uint32_t i = 0; i < 32 / EV_WARPS; ++i) {
          const uint32_t bits = __ballot_sync(0xffffffffu, gone[i] != 0);
          if (lane == 0) missing_bits[k][warp + i * EV_WARPS] = bits;
        }
      }
    }
    __syncthreads();
    for (uint32_t first = warp; first < nv; first += EV_WARPS * AT_ONCE) {
      if (lane >= rows) continue;
      float gc[GRADIENT ? AT_ONCE : 1][C];
      if constexpr (GRADIENT) {
#pragma unroll
        for (uint32_t u = 0; u < AT_ONCE; ++u) {
          const uint32_t v = first + u * EV_WARPS;
          const float* g = a.g + b + a.rows * (v0 + v);
#pragma unroll
          for (int c = 0; c < C; ++c) gc[u][c] = v < nv && c < (int)a.cats ? g[step * c] : 0.0f;
        }
      }
#pragma unroll
      for (uint32_t u = 0; u < AT_ONCE; ++u) {
        const uint32_t v = first + u * EV_WARPS;
        if (v >= nv) continue;
        float* at = tile + v * a.cats * EV_PITCH + lane;
        bool missing = false;
        if (BY_ROWS) missing = a.miss && missing_bits[v >> 5][lane] >> (v & 31) & 1;
        else missing = a.miss && a.miss[b * a.miss_row_stride + (v0 + v) * a.miss_var_stride];
        float p[C], xc[C];
#pragma unroll
        for (int c = 0; c < C; ++c) xc[c] = c < (int)a.cats ? at[c * EV_PITCH] : -INFINITY;
        float m = xc[0], S = 0.0f;
#pragma unroll
        for (int c = 1; c < C; ++c) m = fmaxf(m, xc[c]);
        m = fmaxf(m, -INFINITY);
        const Shift from = shift_of<T>(m, a.c);
        if (from.near) {
#pragma unroll
          for (int c = 0; c < C; ++c) S += p[c] = ex2_ftz(fmaf(xc[c], from.c, -from.mc));
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c) S += p[c] = ex2_ftz(max_nan((xc[c] - finite_shift(m)) * from.c, NO_MASS));
        }
        if constexpr (!GRADIENT) {
          const LogScale l = log_scale<T>(from, S, a.invT);
          float* out = a.out + b + a.rows * (v0 + v);
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (c < (int)a.cats) out[step * c] = missing ? 0.0f : logp_of(xc[c], l);
          if (a.stats_out) {   // in the places of the first two categories; with one category, behind all
            at[0] = m;
            tile[(a.cats > 1 ? v * a.cats + 1 : columns + v) * EV_PITCH + lane] = sum_out(from, S);
          }
        } else {
          float sum = 0.0f;
#pragma unroll
          for (int c = 0; c < C; ++c) sum += gc[u][c];
          const bool none = missing || S == 0.0f;
          const float k = sum / S;
#pragma unroll
          for (int c = 0; c < C; ++c)
            if (c < (int)a.cats) at[c * EV_PITCH] = none ? 0.0f : (gc[u][c] - p[c] * k) * a.invT;
        }
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
    } else if (a.stats_out) {
      for (uint32_t r = warp; r < rows; r += EV_WARPS) {
        float2* to = reinterpret_cast<float2*>(a.stats_out) + (b0 + r) * a.vars + v0;
        for (uint32_t v = lane; v < nv; v += 32)
          to[v] = {tile[v * a.cats * EV_PITCH + r], tile[(a.cats > 1 ? v * a.cats + 1 : columns + v) * EV_PITCH + r]};
      }
      __syncthreads();
    }
  }
}

// Tiles of up to EV_COLUMNS columns; a variable of up to EV_MOST categories is held whole.
template <typename T> constexpr uint32_t EV_MOST = 32 * Most<T>::E < 768 ? 32 * Most<T>::E : 768;
template <typename T>
EvidenceTile evidence_tile(const EvidenceArgs& a, uint32_t sms) {
  EvidenceTile t;
  t.vars = a.var_stride == a.cats && a.cats <= EV_COLUMNS / 2 ? std::min(EV_COLUMNS / a.cats, a.vars) : 1;
  const uint64_t row_tiles = (a.rows + 31) / 32;
  // smaller tiles where there are few (us with none / 2 / 4 tiles per SM wanted: 1000 x 784 x 2 gradient 28.8 / 20.9 / 25.2,
  // one way 9.7 / 6.6 / 7.6, 100 x 784 x 8 14.6 / 9.7 / 9.7)
  while (t.vars > 8 && row_tiles * ((a.vars - 1) / t.vars + 1) < 2 * (uint64_t)sms) t.vars = (t.vars + 1) / 2;
  t.cap = t.vars > 1 ? t.vars * a.cats : a.cats <= EV_MOST<T> ? a.cats : EV_COLUMNS;
  t.row_tiles = (uint32_t)row_tiles;
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

template <typename T, int E, Form FORM, int LG>
cudaError_t launch_evidence_lanes(const EvidenceArgs& a, const EvidenceTile& t, cudaStream_t st) {
  const dim3 grid(t.row_tiles, std::min(t.var_tiles, 65535u));
  const uint32_t smem = (tile_place<T>(t.cap, t.lg) + 32) * (uint32_t)sizeof(float);
  static PcbPerDeviceOnce once;
  const cudaError_t e = once.run([] {
    const int most = (int)((tile_place<T>(768, 0) + 32) * sizeof(float));
    const cudaError_t f = cudaFuncSetAttribute(evidence_kernel<T, E, FORM, LG>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    return f != cudaSuccess ? f : cudaFuncSetAttribute(evidence_grad_kernel<T, E, FORM, LG>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
  });
  if (e != cudaSuccess) return e;
  if (a.dx) evidence_grad_kernel<T, E, FORM, LG><<<grid, EV_THREADS, smem, st>>>(a, t);
  else evidence_kernel<T, E, FORM, LG><<<grid, EV_THREADS, smem, st>>>(a, t);
  return cudaGetLastError();
}
template <typename T, int E, Form FORM>
cudaError_t launch_evidence_as(const EvidenceArgs& a, const EvidenceTile& t, cudaStream_t st) {
#define PCB_CALL(LG) return launch_evidence_lanes<T, E, FORM, LG>(a, t, st)
  if constexpr (FORM != ELEMENTS && E == (int)Most<T>::E) PCB_LANES(true, t.lg, PCB_CALL);
  else PCB_CALL(-1);
#undef PCB_CALL
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
  const uint32_t smem = (t.cap + (a.cats == 1 && a.stats_out ? t.vars : 0)) * EV_PITCH * (uint32_t)sizeof(float);
  static PcbPerDeviceOnce once;   // distributions of one category need twice the columns
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(evidence_thin_kernel<T, C, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * EV_COLUMNS * EV_PITCH * (int)sizeof(float));
  });
  if (e != cudaSuccess) return e;
  if (a.dx) evidence_thin_kernel<T, C, true><<<grid, EV_THREADS, smem, st>>>(a, t);
  else evidence_thin_kernel<T, C, false><<<grid, EV_THREADS, smem, st>>>(a, t);
  return cudaGetLastError();
}
template <typename T>
cudaError_t launch_evidence(const EvidenceArgs& a, cudaStream_t st) {   // the gradient where dx is given
  const uint32_t sms = pcb_sm_count();
  if (sms == 0) return cudaErrorNoDevice;
  const EvidenceTile t = evidence_tile<T>(a, sms);
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

}  // namespace

extern "C" int32_t pcb_soft_evidence(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t vars, uint32_t cats,
                                     uint64_t row_stride, uint64_t var_stride, const uint8_t* miss_dev, uint64_t miss_row_stride,
                                     uint64_t miss_var_stride, float temperature, float* out_dev, float* stats_dev, pcb_stream s) {
  if (rows == 0 || vars == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(out_dev, "null argument");
  EvidenceArgs a{x_dev, rows, row_stride, var_stride, miss_row_stride, miss_var_stride, vars, cats, 1.0f / temperature,
                 LOG2E / temperature, miss_dev, out_dev, stats_dev, nullptr, nullptr, nullptr};
  PCB_REQUIRE(!stats_dev || ((uintptr_t)stats_dev & 7) == 0, "statistics that are not 8-byte aligned");
  PCB_REQUIRE(rows < (1ull << 35) && vars <= 0x7fffffffu, "at most 2^35 - 1 rows and 2^31 - 1 variables");
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
  PCB_REQUIRE(rows < (1ull << 35) && vars <= 0x7fffffffu, "at most 2^35 - 1 rows and 2^31 - 1 variables");
  cudaStream_t st = (cudaStream_t)s;
  PCB_CUDA(dtype == PCB_F32 ? launch_evidence<float>(a, st) : dtype == PCB_BF16 ? launch_evidence<__nv_bfloat16>(a, st)
                                                                                    : launch_evidence<__half>(a, st));
  return PCB_OK;
}
