// pcb_logits.cu — log-probabilities of given categories, entropy and best alternatives of logits.
#include "pcb_logits.cuh"

namespace {

using namespace pcblogits;

struct LogprobArgs {
  const void* x;
  uint64_t rows, stride;
  uint32_t cats, top_k, token_bytes;
  float invT, c;
  const void* tokens;
  float *logp, *entropy, *stats, *top_logp;
  int64_t* top_ids;
};

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
//
// Bound by memory and by the end of each row, where a block reads what it noted: 2048 rows of 131072 bf16 with 8 alternatives
// 105 us (5.1 TB/s, 79 % of a copy; 96 us without alternatives); a single row of 131072 fp32 with 20 alternatives, on a cluster
// of eight blocks, 9.0 us, all of it latency: 2.6 for the shortest row there is, 4.7 for this one without alternatives, 7.0 with
// one, the rest for ordering twenty.
constexpr uint32_t SLOTS = 16, CAND = 256, PAIRS = 256, MAX_CLUSTER = 8;

template <typename T> struct Tile { static constexpr uint32_t U = sizeof(T) == 4 ? 8 : 4; };   // granules per thread

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
      const Shift from_all = shift_of<T>(s.m, a.c);
      const LogScale l = log_scale<T>(from_all, s.S, a.invT);
      if (tid == 0) {
        if (a.tokens) a.logp[row] = token_logp(a, token, x_token, l);
        a.entropy[row] = entropy_of(s.S, s.A, ln_of(s.S));
        if (a.stats) reinterpret_cast<float2*>(a.stats)[row] = {s.m, sum_out(from_all, s.S)};
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
  const Shift from = shift_of<T>(k.m, a.c);
  const LogScale l = log_scale<T>(from, k.S, a.invT);
  if (a.tokens) a.logp[row] = token_logp(a, token, x_token, l);
  a.entropy[row] = entropy_of(k.S, k.A, ln_of(k.S));
  if (a.stats) reinterpret_cast<float2*>(a.stats)[row] = {k.m, sum_out(from, k.S)};
  if (a.top_k == 1) {
    a.top_ids[row] = k.at;
    a.top_logp[row] = logp_of(k.best, l);
  }
}

// Rows in memory: in 16-byte granules, or element by element, whatever their distance.  A warp takes `passes` times the rows
// that its lanes hold at once, the next ones on their way while it works on these (granules), and writes the results of all
// of them together: lane (g, j) those of the g-th row of pass j.  Bound by instructions (a power, two sums and the maximum per
// element; finding the best alternative and writing results per row): 401408 rows of 256 fp16 with one alternative 53.4 us
// (4.1 TB/s, 63 % of a copy).
template <typename T, int E, Form FORM, int LG>
__global__ void __launch_bounds__(256, E >= 16 ? 3 : 4) logprob_short_kernel(LogprobArgs a, uint32_t lanes_log2, uint32_t passes) {
  using Row = ShortRow<T, E, FORM>;
  const uint32_t lg = LG >= 0 ? (uint32_t)LG : lanes_log2;
  const uint32_t lane = threadIdx.x & 31, per_warp = 32u >> lg, sub = lane & ((1u << lg) - 1), group = lane >> lg;
  const uint64_t step = (uint64_t)gridDim.x * 8 * per_warp * passes;
  const Bounds bounds = {reinterpret_cast<uintptr_t>(a.x), reinterpret_cast<uintptr_t>(static_cast<const T*>(a.x) + (a.rows - 1) * a.stride + a.cats)};
  for (uint64_t r0 = ((uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * per_warp * passes; r0 < a.rows; r0 += step) {
    const uint64_t first = min(a.rows - 1, r0 + group);
    const uint32_t there = (uint32_t)min((uint64_t)passes, (a.rows - r0 + per_warp - 1) / per_warp);   // passes with rows
    const uint32_t last = (uint32_t)min((uint64_t)passes, (a.rows - 1 - first) / per_warp);            // this lane's last pass with a row
    const T* x = static_cast<const T*>(a.x) + first * a.stride;
    const auto row_at = [&](uint32_t pass) { return x + (uint64_t)(min(pass, last) * per_warp) * a.stride; };
    Row next;
    next.load(row_at(0), sub, lg, a.cats, bounds);
    const uint64_t mine = r0 + sub * per_warp + group;   // the row whose results this lane writes
    const bool writes = sub < passes && mine < a.rows;
    int64_t token = -1;
    float x_token = 0.0f;
    if (writes && a.tokens) {
      token = token_at(a.tokens, a.token_bytes, mine);
      if (is_category(a, token)) x_token = to_f32((static_cast<const T*>(a.x) + mine * a.stride)[token]);
    }
    Kept kept = {0.0f, 0.0f, 0.0f, 0.0f, 0};
    for (uint32_t pass = 0; pass < there; ++pass) {
      Row r = next;
      if (FORM != ELEMENTS && pass + 1 < there) next.load(row_at(pass + 1), sub, lg, a.cats, bounds);
      const Kept k = short_row<T, E, FORM>(a, r, first + pass * per_warp, r0 + group < a.rows && pass <= last, sub, lg);
      if (sub == pass) kept = k;
      if (FORM == ELEMENTS && pass + 1 < there) next.load(row_at(pass + 1), sub, lg, a.cats, bounds);
    }
    if (writes) short_results<T>(a, kept, mine, token, x_token);
  }
}

// Rows one behind the other (stride = cats), of any length and alignment: every warp stages the bytes of `rows_staged` of
// them, from the 16-byte boundary below their beginning on, with asynchronous copies, STAGES - 1 of them ahead of its work,
// and its lanes read their elements there.  (Both directions of 800000 rows of 51 fp16: 170 us, by granules from memory 228.)
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

template <typename T, int E>
void launch_staged(const LogprobArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  const uint32_t rows = staged_rows<T>(a.cats, s.lg), per_block = rows * (STAGED_THREADS / 32);
  const uint32_t grid = resident_blocks<logprob_staged_kernel<T, E>, STAGED_THREADS>(sms, (a.rows + per_block - 1) / per_block);
  logprob_staged_kernel<T, E><<<grid, STAGED_THREADS, 0, st>>>(a, s.lg, rows);
}
template <typename T, int E, Form FORM>
void launch_passes(const LogprobArgs& a, const ShortShape& s, uint32_t sms, cudaStream_t st) {
  const uint32_t per_pass = 256u >> s.lg, passes = short_passes(a.rows, s.lg, sms);
  const uint64_t blocks = (a.rows + per_pass * passes - 1) / (per_pass * passes);
  const uint32_t grid = (uint32_t)std::min<uint64_t>(blocks, 0x7fffffff);
#define PCB_CALL(LG) logprob_short_kernel<T, E, FORM, LG><<<grid, 256, 0, st>>>(a, s.lg, passes)
  if constexpr (FORM != ELEMENTS && E == (int)Most<T>::E) PCB_LANES(true, s.lg, PCB_CALL);
  else PCB_CALL(-1);
#undef PCB_CALL
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

}  // namespace

extern "C" int32_t pcb_token_logprobs(const void* x_dev, int32_t dtype, uint64_t rows, uint32_t cats, uint64_t row_stride,
                                      float temperature, const void* tokens_dev, uint32_t token_bytes, uint32_t top_k,
                                      float* logp_out_dev, float* entropy_dev, float* stats_dev, int64_t* top_ids_dev,
                                      float* top_logp_dev, pcb_stream s) {
  if (rows == 0) return PCB_OK;
  if (int32_t rc = check_logits(x_dev, dtype, cats, temperature)) return rc;
  PCB_REQUIRE(entropy_dev && ((uintptr_t)stats_dev & 7) == 0, "null argument, or statistics that are not 8-byte aligned");
  PCB_REQUIRE(!tokens_dev || (logp_out_dev && (token_bytes == 4 || token_bytes == 8)), "tokens are int32 or int64 and need an output");
  PCB_REQUIRE(!tokens_dev || (uintptr_t)tokens_dev % token_bytes == 0, "tokens that are not aligned to their own size");
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
