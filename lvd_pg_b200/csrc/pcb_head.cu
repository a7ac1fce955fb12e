// pcb_head.cu — a categorical head with weights in 4 bits and group scales, for few feature vectors:
//   y[m, n] = sum_k scale[n, k / group] (code[n, k] - 8) x[m, k] + bias[n].
//
// The weights are the A operand of mma.sync m16n8k16: 16 categories x 16 features, codes turned into integers -8..7 in the
// features' own type, where they and their products with x are exact; a group's sum stays in the fp32 accumulator and meets
// its scale there, once: features up to 3.3e35 in magnitude keep it in range (128 of them, times 8).  (fp32 features go in as
// three bf16 terms, which hold all 24 bits.)
//
// Packed order: tiles of 16 categories, in each blocks of 64 features of 512 bytes, a 16-byte word per lane.  Lane 4 g + t
// holds the codes of categories g and g + 8; its 32-bit word w belongs to the k16 step j = w & 1 of the 32 features
// h = w >> 1, where it stands for features 32 h + 8 t + 4 j + (0..3): the order of k inside a product is free, and this one
// makes a lane's share of x eight consecutive features.  Nibble i + 4 e of a word is element e of fragment register i:
// category g + 8 (i & 1), feature + 2 (i >> 1) + e.  Behind the codes: the scales of a tile, [quad of groups][g][4 groups]
// [g, g + 8], so that one 16-byte load brings four groups' scales of a lane's two categories.
#include "pcb_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

namespace {

constexpr uint32_t MAX_FEATURES = 32768;   // three columns of them fit into shared memory

struct HeadShape {
  uint32_t cats, features, group;
  uint32_t tiles, blocks, quads;   // 16 categories, 64 features, 4 groups
  __host__ __device__ uint64_t code_words() const { return (uint64_t)tiles * blocks * 128; }     // of 32 bits
  __host__ __device__ uint64_t scale_words() const { return (uint64_t)tiles * quads * 32; }
};
HeadShape head_shape(uint32_t cats, uint32_t features, uint32_t group) {
  HeadShape h{cats, features, group, 0, 0, 0};
  h.tiles = (uint32_t)(((uint64_t)cats + 15) / 16);
  h.blocks = (uint32_t)(((uint64_t)features + 63) / 64);
  const uint32_t groups = (uint32_t)(((uint64_t)features + group - 1) / group);
  h.quads = (groups + 3) / 4;
  return h;
}
int32_t check_shape(uint32_t cats, uint32_t features, uint32_t group) {
  PCB_REQUIRE(cats >= 1 && cats <= 0x7fffffffu && features >= 1, "a head has at least one category and one feature");
  PCB_REQUIRE(group == 32 || group == 64 || group == 128, "groups hold 32, 64 or 128 features");
  if (features > MAX_FEATURES) return pcb_fail(PCB_ERR_TOO_LARGE, "a head has at most 32768 features");
  return PCB_OK;
}
bool is_dtype(int32_t d) { return d == PCB_F32 || d == PCB_BF16 || d == PCB_F16; }
bool is_scale_dtype(int32_t d) { return d == PCB_BF16 || d == PCB_F16; }

__device__ __forceinline__ float load_as_f32(const void* p, uint64_t i, int32_t dtype) {
  if (dtype == PCB_F32) return static_cast<const float*>(p)[i];
  if (dtype == PCB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ float scale_f32(uint32_t bits16, int32_t dtype) {
  return dtype == PCB_BF16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}

// One warp per (category, group): scale = max |w| / 7, code = round(w / scale) + 8 with the scale as stored.  NaN or an infinite
// weight makes the scale NaN, and with it all weights of the group: no finite weights stand for it.
__global__ void __launch_bounds__(256) head_quantize_kernel(const void* w, int32_t dtype, uint32_t cats, uint32_t features, uint32_t group,
                                                            int32_t scale_dtype, uint8_t* codes, uint16_t* scales) {
  const uint32_t lane = threadIdx.x & 31, groups = (features + group - 1) / group, bytes = (features + 1) / 2;
  const uint64_t total = (uint64_t)cats * groups;
  for (uint64_t i = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < total; i += (uint64_t)gridDim.x * 8) {
    const uint64_t n = i / groups;
    const uint32_t k0 = (uint32_t)(i % groups) * group, k1 = min(features, k0 + group);
    float most = 0.0f;
    bool odd = false;
    for (uint32_t k = k0 + lane; k < k1; k += 32) {
      const float v = fabsf(load_as_f32(w, n * features + k, dtype));
      odd |= !(v < INFINITY);
      most = fmaxf(most, v);
    }
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float want = __any_sync(0xffffffffu, odd) ? NAN : most / 7.0f;
    // To the nearest; a scale that is subnormal in its type, up: half a step is up to half of it there (all of it below the
    // smallest), and the largest weights would be cut off at 7 of a scale that was rounded down, or all be lost.
    uint16_t bits;
    if (scale_dtype == PCB_BF16) bits = __bfloat16_as_ushort(want < 0x1p-126f ? __float2bfloat16_ru(want) : __float2bfloat16_rn(want));
    else bits = __half_as_ushort(want < 0x1p-14f ? __float2half_ru(want) : __float2half_rn(want));
    const float scale = scale_f32(bits, scale_dtype);
    if (lane == 0) scales[i] = bits;
    for (uint32_t k = k0 + 2 * lane; k < k1; k += 64) {
      uint32_t byte = 0x88;
      for (uint32_t e = 0; e < 2 && k + e < k1; ++e) {
        const float q = scale > 0.0f ? rintf(load_as_f32(w, n * features + k + e, dtype) / scale) : 0.0f;
        const uint32_t code = (uint32_t)(int)(fminf(fmaxf(q, -8.0f), 7.0f) + 8.0f);
        byte = e ? (byte & 0x0fu) | code << 4 : (byte & 0xf0u) | code;
      }
      codes[n * bytes + k / 2] = (uint8_t)byte;
    }
  }
}

// where a word's nibble comes from
__device__ __forceinline__ void nibble_place(uint32_t lane, uint32_t w, uint32_t p, uint32_t& row, uint32_t& k) {
  const uint32_t i = p & 3, e = p >> 2;
  row = (lane >> 2) + 8 * (i & 1);
  k = 32 * (w >> 1) + 8 * (lane & 3) + 4 * (w & 1) + 2 * (i >> 1) + e;
}

// A block per tile.  A word's nibbles are two bytes of category g and two of g + 8.
__global__ void __launch_bounds__(256) head_pack_kernel(HeadShape h, const uint8_t* codes, const uint16_t* scales, uint32_t* out) {
  const uint32_t bytes = (h.features + 1) / 2, groups = (h.features + h.group - 1) / h.group;
  for (uint64_t tile = blockIdx.x; tile < h.tiles; tile += gridDim.x) {
    uint32_t* words = out + tile * h.blocks * 128;
    for (uint32_t i = threadIdx.x; i < h.blocks * 128; i += 256) {
      const uint32_t w = i & 3, lane = i >> 2 & 31, k = (i >> 7) * 64 + 32 * (w >> 1) + 8 * (lane & 3) + 4 * (w & 1);
      const uint64_t n = tile * 16 + (lane >> 2);
      uint32_t word = 0;
#pragma unroll
      for (uint32_t half = 0; half < 2; ++half) {
        uint32_t four = 0x8888u;   // features k .. k + 3 of one category; what is not there is 0
        if (n + 8 * half < h.cats && k < h.features) {
          const uint8_t* at = codes + (n + 8 * half) * bytes + k / 2;
          four = at[0];
          if (k + 2 < h.features) four |= (uint32_t)at[1] << 8;
          const uint32_t there = min(4u, h.features - k);
          four = (four & ((1u << (4 * there)) - 1)) | (0x8888u & ~((1u << (4 * there)) - 1));
        }
        // features k, k + 1 to nibbles half, half + 4, features k + 2, k + 3 to half + 2, half + 6
        word |= ((four & 0xfu) | (four & 0xf0u) << 12 | (four & 0xf00u) | (four & 0xf000u) << 12) << (4 * half);
      }
      words[i] = word;
    }
    uint32_t* two = out + h.code_words() + tile * h.quads * 32;   // [quad][g][group of the quad]
    for (uint32_t i = threadIdx.x; i < h.quads * 32; i += 256) {
      const uint64_t n = tile * 16 + (i >> 2 & 7);
      const uint32_t group = (i >> 5) * 4 + (i & 3);
      uint32_t word = 0;
      if (group < groups) {
        if (n < h.cats) word = scales[n * groups + group];
        if (n + 8 < h.cats) word |= (uint32_t)scales[(n + 8) * groups + group] << 16;
      }
      two[i] = word;
    }
  }
}

__global__ void __launch_bounds__(256) head_weight_kernel(HeadShape h, const uint32_t* packed, int32_t scale_dtype, float* weight) {
  const uint64_t nc = h.code_words();
  const uint32_t* scales = packed + nc;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < nc; i += (uint64_t)gridDim.x * blockDim.x) {
    const uint32_t w = i & 3, lane = (i >> 2) & 31, word = packed[i];
    const uint64_t tb = i >> 7, tile = tb / h.blocks, block = tb % h.blocks;
    for (uint32_t p = 0; p < 8; ++p) {
      uint32_t row, k;
      nibble_place(lane, w, p, row, k);
      const uint64_t n = tile * 16 + row, kk = block * 64 + k;
      if (n >= h.cats || kk >= h.features) continue;
      const uint64_t group = kk / h.group;
      const uint32_t two = scales[(tile * h.quads + group / 4) * 32 + (row & 7) * 4 + group % 4];
      weight[n * h.features + kk] = scale_f32(row < 8 ? two & 0xffffu : two >> 16, scale_dtype) * ((int)(word >> (4 * p) & 15u) - 8);
    }
  }
}

// ---- products ---------------------------------------------------------------------------------------------
struct HeadArgs {
  HeadShape h;
  const uint32_t* packed;
  int32_t scale_dtype, y_dtype;
  const void* x;
  uint64_t rows, x_stride;
  const float* bias;
  void* y;
};

// Two 16-bit values of the tensor cores' operand type.  A nibble in the mantissa of BASE is BASE + code 2^offset, exactly;
// one multiply-add takes it to code - 8: the known way from integers to floating point through the mantissa of a power of two,
// which Kim, Henry, Fahim and Awadalla describe for weights of 4 bits ("Who Says Elephants Can't Run: Bringing Large Scale
// MoE Models into Cloud Scale Production", 2022).  bf16 has room for the lowest place only (three shifts per word of eight
// codes), fp16 for two (one shift).
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t base) {   // one instruction
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(base));
  return r;
}
template <typename T> struct Operand;
template <> struct Operand<__nv_bfloat16> {
  static constexpr uint32_t BASE = 0x43004300u;   // 128: the codes' ulp there is 1
  static __device__ __forceinline__ uint32_t minus8(uint32_t v) {   // (128 + code) - 136
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), __floats2bfloat162_rn(136.0f, 136.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t* a) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = minus8(and_or(w >> (4 * i), 0x000f000fu, BASE));
  }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void mma_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {   // from zero
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};
template <> struct Operand<__half> {
  static constexpr uint32_t BASE = 0x64006400u;   // 1024
  static __device__ __forceinline__ __half2 based(uint32_t w, uint32_t mask) {
    const uint32_t v = and_or(w, mask, BASE);
    return *reinterpret_cast<const __half2*>(&v);
  }
  static __device__ __forceinline__ uint32_t bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
  static __device__ __forceinline__ void weights(uint32_t w, uint32_t* a) {
    const __half2 lo = __floats2half2_rn(-1032.0f, -1032.0f), sixteenth = __floats2half2_rn(0.0625f, 0.0625f), hi = __floats2half2_rn(-72.0f, -72.0f);
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const uint32_t v = w >> (4 * i);
      a[i] = bits(__hadd2(based(v, 0x000f000fu), lo));                       // 1024 + code - 1032
      a[i + 1] = bits(__hfma2(based(v, 0x00f000f0u), sixteenth, hi));       // (1024 + 16 code) / 16 - 72
    }
  }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void mma_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {   // from zero
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// x as `terms` values of the operand type whose sum it is
template <typename X> struct Feature { using Op = X; static constexpr int TERMS = 1; };
template <> struct Feature<float> { using Op = __nv_bfloat16; static constexpr int TERMS = 3; };

__device__ __forceinline__ void terms_of(float v, uint16_t* t) {
  if (!(fabsf(v) < INFINITY)) {   // the first term alone carries inf and NaN
    t[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    t[1] = t[2] = 0;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) {   // eight bits at a time, truncated: 24 in three terms, and no overflow
    const uint32_t top = __float_as_uint(v) & 0xffff0000u;
    t[i] = (uint16_t)(top >> 16);
    v -= __uint_as_float(top);
  }
}
__device__ __forceinline__ void terms_of(__nv_bfloat16 v, uint16_t* t) { t[0] = __bfloat16_as_ushort(v); }
__device__ __forceinline__ void terms_of(__half v, uint16_t* t) { t[0] = __half_as_ushort(v); }

__device__ __forceinline__ void store_y(void* y, uint64_t i, float v, int32_t dtype) {
  if (dtype == PCB_F32) static_cast<float*>(y)[i] = v;
  else if (dtype == PCB_BF16) static_cast<__nv_bfloat16*>(y)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(y)[i] = __float2half_rn(v);
}

// Persistent blocks of sixteen warps, in teams of four or eight.  A team takes R tiles of 16 categories a round; its warps
// share the features and add up their parts through shared memory: large teams for heads with few categories, which fill the
// GPU so, smaller ones where there are enough (fewer wait for one another).  The feature vectors stay in shared memory, as
// columns of the B operand (fp32: three columns each, one per term, joined at the end); codes and scales go straight from
// memory to registers, four 16-byte loads per lane ahead of the four that are worked on, across the boundaries of rounds.
//
// Bound by what turns codes into operands, not by the products: one vector at 131072 x 4096 bf16 takes 62.6 us for 285 MB
// (4.5 TB/s, 70 % of what a copy reaches) with the pipe of shifts and masks 60 % busy, three shifts, four masks and four
// subtractions per eight codes.  Wide multiplies in place of shifts (76 -> 88 us then), a step loop unrolled by two (64 -> 65)
// and prefetching the next round into the L2 cache (64 -> 78) did not pay.  fp16 needs one shift: 32000 x 2048, sixteen
// vectors, 15.2 us (2.3 TB/s: launch, feature vectors and the last round weigh there).  More vectors than a pass takes unpack
// the weights again for every 32 of them: 1024 at 32000 x 2048 bf16 0.80 ms, 401408 at 256 x 512 bf16 4.0 ms (fp32 13.6).
constexpr uint32_t HEAD_THREADS = 512, HEAD_WARPS = 16;

template <bool G32>
struct Codes {   // R tiles x 4 / R blocks
  uint4 q[4];
  uint32_t s[4][G32 ? 2 : 1];
};

struct HeadPass {
  uint32_t columns;     // per pass: feature vectors x terms
  uint32_t vectors;     // feature vectors per pass
  uint32_t pitch;       // bytes between columns in shared memory
  uint32_t groups;      // R tiles each
  uint32_t team;        // warps
};

__device__ __forceinline__ uint4 load_codes(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

template <typename X, int R, int NT, bool G32, bool BF16_SCALES>   // G32: a block of 64 features has two groups
__global__ void __launch_bounds__(HEAD_THREADS, 1) head_kernel(HeadArgs a, HeadPass ps) {
  using F = Feature<X>;
  using Op = Operand<typename F::Op>;
  constexpr int D = 4 / R;   // blocks per step
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t team = tid / 32 / ps.team, warp = tid / 32 % ps.team, teams = HEAD_WARPS / ps.team;
  uint8_t* xs = smem;
  float* all_parts = reinterpret_cast<float*>(smem + ps.columns * ps.pitch) + team * 2 * (ps.team * ps.columns * R * 16);   // twice [warp][column][16 R]
  const uint64_t m0 = (uint64_t)blockIdx.y * ps.vectors;
  const uint32_t vectors = (uint32_t)min((uint64_t)ps.vectors, a.rows - m0);
  const uint32_t per_warp = (a.h.blocks + ps.team - 1) / ps.team;
  const uint32_t b0 = min(a.h.blocks, warp * per_warp), b1 = min(a.h.blocks, b0 + per_warp), steps = (per_warp + D - 1) / D, last = b1 > b0 ? b1 - 1 : a.h.blocks - 1;
  const uint4* codes = reinterpret_cast<const uint4*>(a.packed) + lane;
  const uint32_t* scales = a.packed + a.h.code_words() + g * 4;
  const uint32_t per_group = a.h.group == 128 ? 1 : 0;   // blocks share a scale in pairs

  // Tiles behind the last and blocks behind the warp's are read again, but not used.
  const auto fetch = [&](uint32_t group, uint32_t step) {
    Codes<G32> c;
    const uint32_t tile = group * R, most = a.h.tiles - 1 - tile;
    const uint4* q = codes + (uint64_t)tile * a.h.blocks * 32;
    const uint32_t* s = scales + (uint64_t)tile * a.h.quads * 32;
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const uint32_t b = min(b0 + step * D + d, last), first = G32 ? 2 * b : b >> per_group, at = (first & ~3u) * 8 + (first & 3u);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t rr = R == 1 ? 0 : min((uint32_t)r, most);
        c.q[d * R + r] = load_codes(q + (rr * a.h.blocks + b) * 32);
        const uint32_t* to = s + rr * a.h.quads * 32 + at;
        if constexpr (G32) {
          const uint2 two = __ldg(reinterpret_cast<const uint2*>(to));
          c.s[d * R + r][0] = two.x;
          c.s[d * R + r][1] = two.y;
        } else {
          c.s[d * R + r][0] = __ldg(to);
        }
      }
    }
    return c;
  };
  const uint32_t stride = gridDim.x * teams;
  uint32_t group = team * gridDim.x + blockIdx.x;   // the first round spreads over the blocks
  Codes<G32> next = fetch(min(group, ps.groups - 1), 0);

  // the feature vectors: eight features a time, four times that in flight per thread, zeros behind the last
  const uint32_t eights = a.h.blocks * 8, all = ps.vectors * eights, magic = 0xffffffffu / eights + 1;   // all < 2^18, eights <= 2^12: i / eights is exact
  for (uint32_t i0 = tid; i0 < all; i0 += 4 * HEAD_THREADS) {
    __align__(16) X v[4][8];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t i = i0 + u * HEAD_THREADS, m = __umulhi(i, magic), k = (i - m * eights) * 8;
      const X* x = static_cast<const X*>(a.x) + (m0 + m) * a.x_stride + k;
      if (i < all && m < vectors && k + 8 <= a.h.features && (reinterpret_cast<uintptr_t>(x) & 15) == 0) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(X) / 2; ++j) reinterpret_cast<uint4*>(v[u])[j] = __ldg(reinterpret_cast<const uint4*>(x) + j);
      } else {
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) v[u][e] = i < all && m < vectors && k + e < a.h.features ? x[e] : X(0.0f);
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
      const uint32_t i = i0 + u * HEAD_THREADS, m = __umulhi(i, magic), k = (i - m * eights) * 8;
      if (i >= all) continue;
      uint16_t terms[8][3];
#pragma unroll
      for (int e = 0; e < 8; ++e) terms_of(v[u][e], terms[e]);
#pragma unroll
      for (int s = 0; s < F::TERMS; ++s) {
        uint4 w;
        w.x = terms[0][s] | (uint32_t)terms[1][s] << 16;
        w.y = terms[2][s] | (uint32_t)terms[3][s] << 16;
        w.z = terms[4][s] | (uint32_t)terms[5][s] << 16;
        w.w = terms[6][s] | (uint32_t)terms[7][s] << 16;
        *reinterpret_cast<uint4*>(xs + (m * F::TERMS + s) * ps.pitch + k * 2) = w;
      }
    }
  }
  __syncthreads();
  const uint8_t* column[NT];   // columns behind the last: the last again, not stored
#pragma unroll
  for (int n = 0; n < NT; ++n) column[n] = xs + min(n * 8 + g, ps.columns - 1) * ps.pitch + t * 16;

  for (uint32_t turn = 0; group < ps.groups; group += stride, turn ^= 1) {
    float* parts = all_parts + turn * (ps.team * ps.columns * R * 16);
    float sum[R][NT][4];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[r][n][0] = sum[r][n][1] = sum[r][n][2] = sum[r][n][3] = 0.0f;
    for (uint32_t step = 0; step < steps; ++step) {
      const Codes<G32> c = next;
      const bool more = step + 1 < steps;
      if (more || group + stride < ps.groups) next = fetch(more ? group : group + stride, more ? step + 1 : 0);
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const uint32_t b = b0 + step * D + d;
        if (b >= b1) continue;
        uint4 x[2][NT];   // eight features of a column: two k16 steps
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            x[h][n] = *reinterpret_cast<const uint4*>(column[n] + b * 128 + h * 64);
          }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint4 q = c.q[d * R + r];
          const uint32_t words[4] = {q.x, q.y, q.z, q.w};
          float acc[NT][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t frag[4];
              Op::weights(words[2 * h + j], frag);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                if (j == 0 && (h == 0 || G32)) Op::mma_first(acc[n], frag, x[h][n].x, x[h][n].y);
                else Op::mma(acc[n], frag, j ? x[h][n].z : x[h][n].x, j ? x[h][n].w : x[h][n].y);
              }
            }
            if (h == 1 || G32) {
              const uint32_t two = c.s[d * R + r][G32 ? h : 0];
              const float s0 = BF16_SCALES ? __uint_as_float(two << 16) : scale_f32(two & 0xffffu, PCB_F16);
              const float s1 = BF16_SCALES ? __uint_as_float(two & 0xffff0000u) : scale_f32(two >> 16, PCB_F16);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                sum[r][n][0] = fmaf(s0, acc[n][0], sum[r][n][0]);
                sum[r][n][1] = fmaf(s0, acc[n][1], sum[r][n][1]);
                sum[r][n][2] = fmaf(s1, acc[n][2], sum[r][n][2]);
                sum[r][n][3] = fmaf(s1, acc[n][3], sum[r][n][3]);
              }
            }
          }
        }
      }
    }
    // the warps' parts, added up in order
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t column = n * 8 + 2 * t + (i & 1);
          if (column < ps.columns) parts[(warp * ps.columns + column) * (R * 16) + r * 16 + g + 8 * (i >> 1)] = sum[r][n][i];
        }
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(ps.team * 32) : "memory");
    for (uint32_t i = warp * 32 + lane; i < vectors * (R * 16); i += ps.team * 32) {
      const uint32_t m = i / (R * 16), n = i % (R * 16);
      float y = 0.0f;
#pragma unroll
      for (int s = F::TERMS - 1; s >= 0; --s) {   // the smallest term first
        float part = 0.0f;
        for (uint32_t w = 0; w < ps.team; ++w) part += parts[(w * ps.columns + m * F::TERMS + s) * (R * 16) + n];
        y += part;
      }
      const uint64_t cat = (uint64_t)group * (R * 16) + n;
      if (cat < a.h.cats) store_y(a.y, (m0 + m) * a.h.cats + cat, y + (a.bias ? a.bias[cat] : 0.0f), a.y_dtype);
    }
    // the next round's parts go beside these; nobody is two rounds ahead of the slowest reader, for the barrier in between
  }
}

// Shared memory a block may have.  A pass takes up to 32 columns (32 feature vectors of 16 bits, 10 of fp32), or what fits;
// more vectors than that read the weights again.
constexpr uint32_t HEAD_SMEM = 220 * 1024;

template <typename X, int R, int NT, bool G32, bool BF16_SCALES>
cudaError_t launch_head(const HeadArgs& a, HeadPass ps, uint32_t sms, cudaStream_t st) {
  static PcbPerDeviceOnce once;
  const cudaError_t e = once.run([] {
    return cudaFuncSetAttribute(head_kernel<X, R, NT, G32, BF16_SCALES>, cudaFuncAttributeMaxDynamicSharedMemorySize, HEAD_SMEM);
  });
  if (e != cudaSuccess) return e;
  ps.groups = (a.h.tiles + R - 1) / R;
  const uint32_t smem = ps.columns * (ps.pitch + 2 * HEAD_WARPS * R * 16 * (uint32_t)sizeof(float));
  const uint32_t passes = (uint32_t)((a.rows + ps.vectors - 1) / ps.vectors);
  head_kernel<X, R, NT, G32, BF16_SCALES><<<dim3(std::min(ps.groups, sms), passes), HEAD_THREADS, smem, st>>>(a, ps);
  return cudaGetLastError();
}
template <typename X, int R, int NT>
cudaError_t launch_head_group(const HeadArgs& a, const HeadPass& ps, uint32_t sms, cudaStream_t st) {
  const bool bf16 = a.scale_dtype == PCB_BF16;
  if (a.h.group == 32) return bf16 ? launch_head<X, R, NT, true, true>(a, ps, sms, st) : launch_head<X, R, NT, true, false>(a, ps, sms, st);
  return bf16 ? launch_head<X, R, NT, false, true>(a, ps, sms, st) : launch_head<X, R, NT, false, false>(a, ps, sms, st);
}
template <typename X>
cudaError_t launch_head_of(const HeadArgs& a, uint32_t sms, cudaStream_t st) {
  constexpr uint32_t TERMS = Feature<X>::TERMS;
  HeadPass ps;
  ps.pitch = a.h.blocks * 128 + 64;   // 64 modulo 128: eight lanes of a load meet all banks
  uint32_t most = HEAD_SMEM / (ps.pitch + 2 * HEAD_WARPS * 16 * (uint32_t)sizeof(float)) / TERMS;   // vectors that fit with R = 1
  most = std::min(most, 32 / TERMS);
  ps.vectors = (uint32_t)std::min<uint64_t>(a.rows, most);
  ps.columns = ps.vectors * TERMS;
  // Tiles per round (R, as many as the columns' registers allow) and warps per team.  us, R / team:
  //   131072 x 4096, one vector   4/8 63.6   2/4 65.0   1/2 67.7        50000 x 8192, four   4/8 53.2   2/4 51.1   1/2 53.3
  //   32000 x 2048, one           4/8 13.8   2/4 12.5   1/2 13.7        4096 x 4096, one     4/8 10.4   2/4  9.7   1/8  7.1
  //   32000 x 2048 fp16, sixteen  2/4 15.2   2/8 16.7   1/4 15.7   1/8 16.6    50000 x 1024 bf16, nine  2/4 13.9   2/8 15.3   1/4 15.2   1/8 18.5
  const uint32_t nt = (ps.columns + 7) / 8;
  const auto fits = [&](uint32_t r) { return ps.columns * (ps.pitch + 2 * HEAD_WARPS * r * 16 * (uint32_t)sizeof(float)) <= HEAD_SMEM; };
  uint32_t tiles = 1;
  ps.team = 8;
  if (a.h.tiles >= 4 * sms && nt <= 2 && fits(2)) {
    tiles = 2;
    ps.team = 4;
  }
  if (a.h.tiles >= 24 * sms && nt <= 1 && fits(4)) {
    tiles = 4;
    ps.team = 8;
  }
  if (nt <= 1) {
    if (tiles == 4) return launch_head_group<X, 4, 1>(a, ps, sms, st);
    if (tiles == 2) return launch_head_group<X, 2, 1>(a, ps, sms, st);
    return launch_head_group<X, 1, 1>(a, ps, sms, st);
  }
  if (nt <= 2) {
    if (tiles == 2) return launch_head_group<X, 2, 2>(a, ps, sms, st);
    return launch_head_group<X, 1, 2>(a, ps, sms, st);
  }
  return launch_head_group<X, 1, 4>(a, ps, sms, st);
}

}  // namespace

extern "C" int32_t pcb_head_packed_bytes(uint32_t cats, uint32_t features, uint32_t group, uint64_t* bytes_out) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  PCB_REQUIRE(bytes_out, "null argument");
  const HeadShape h = head_shape(cats, features, group);
  *bytes_out = 4 * (h.code_words() + h.scale_words());
  return PCB_OK;
}

static uint32_t blocks_for(uint64_t threads) {
  const uint64_t b = (threads + 255) / 256;
  return (uint32_t)(b < 65536 ? b : 65536);
}

extern "C" int32_t pcb_head_quantize(const void* weight_dev, int32_t dtype, uint32_t cats, uint32_t features, uint32_t group,
                                     int32_t scale_dtype, uint8_t* codes_dev, void* scales_dev, pcb_stream s) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  PCB_REQUIRE(weight_dev && codes_dev && scales_dev, "null argument");
  PCB_REQUIRE(is_dtype(dtype) && is_scale_dtype(scale_dtype), "weights are f32, bf16 or f16, scales bf16 or f16");
  PCB_REQUIRE(((uintptr_t)weight_dev & (dtype == PCB_F32 ? 3 : 1)) == 0 && ((uintptr_t)scales_dev & 1) == 0,
              "weights or scales that are not aligned to their own size");
  const uint64_t groups = ((uint64_t)features + group - 1) / group;
  head_quantize_kernel<<<blocks_for(cats * groups * 32), 256, 0, (cudaStream_t)s>>>(weight_dev, dtype, cats, features, group, scale_dtype,
                                                                                   codes_dev, static_cast<uint16_t*>(scales_dev));
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_head_pack(const uint8_t* codes_dev, const void* scales_dev, uint32_t cats, uint32_t features, uint32_t group,
                                 void* packed_dev, pcb_stream s) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  PCB_REQUIRE(codes_dev && scales_dev && packed_dev && ((uintptr_t)packed_dev & 15) == 0, "null argument, or a packed head that is not 16-byte aligned");
  PCB_REQUIRE(((uintptr_t)scales_dev & 1) == 0, "scales that are not aligned to their own size");
  const HeadShape h = head_shape(cats, features, group);
  head_pack_kernel<<<h.tiles, 256, 0, (cudaStream_t)s>>>(h, codes_dev, static_cast<const uint16_t*>(scales_dev), static_cast<uint32_t*>(packed_dev));
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_head_weight(const void* packed_dev, int32_t scale_dtype, uint32_t cats, uint32_t features, uint32_t group,
                                   float* weight_dev, pcb_stream s) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  PCB_REQUIRE(packed_dev && weight_dev && ((uintptr_t)packed_dev & 15) == 0, "null argument, or a packed head that is not 16-byte aligned");
  PCB_REQUIRE(is_scale_dtype(scale_dtype), "scales are bf16 or f16");
  const HeadShape h = head_shape(cats, features, group);
  head_weight_kernel<<<blocks_for(h.code_words()), 256, 0, (cudaStream_t)s>>>(h, static_cast<const uint32_t*>(packed_dev), scale_dtype, weight_dev);
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_head_logits(const void* packed_dev, int32_t scale_dtype, uint32_t cats, uint32_t features, uint32_t group,
                                   const void* x_dev, int32_t dtype, uint64_t rows, uint64_t x_row_stride, const float* bias_dev,
                                   void* y_dev, int32_t y_dtype, pcb_stream s) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  if (rows == 0) return PCB_OK;
  PCB_REQUIRE(packed_dev && x_dev && y_dev && ((uintptr_t)packed_dev & 15) == 0, "null argument, or a packed head that is not 16-byte aligned");
  PCB_REQUIRE(is_scale_dtype(scale_dtype) && is_dtype(dtype) && is_dtype(y_dtype), "features and logits are f32, bf16 or f16, scales bf16 or f16");
  PCB_REQUIRE(((uintptr_t)x_dev & (dtype == PCB_F32 ? 3 : 1)) == 0 && ((uintptr_t)y_dev & (y_dtype == PCB_F32 ? 3 : 1)) == 0,
              "features or logits that are not aligned to their own size");
  HeadArgs a{head_shape(cats, features, group), static_cast<const uint32_t*>(packed_dev), scale_dtype, y_dtype, x_dev, rows, x_row_stride, bias_dev, y_dev};
  cudaStream_t st = (cudaStream_t)s;
  const uint32_t sms = pcb_sm_count();
  if (sms == 0) return pcb_fail(PCB_ERR_CUDA, "no CUDA device");
  // the vectors of a launch's passes go into its second grid dimension
  constexpr uint64_t AT_ONCE = 65535;
  for (uint64_t done = 0; done < rows; done += AT_ONCE) {
    HeadArgs part = a;
    part.rows = std::min(rows - done, AT_ONCE);
    part.x = static_cast<const uint8_t*>(x_dev) + done * x_row_stride * (dtype == PCB_F32 ? 4 : 2);
    part.y = static_cast<uint8_t*>(y_dev) + done * cats * (y_dtype == PCB_F32 ? 4 : 2);
    PCB_CUDA(dtype == PCB_F32 ? launch_head_of<float>(part, sms, st) : dtype == PCB_BF16 ? launch_head_of<__nv_bfloat16>(part, sms, st)
                                                                                        : launch_head_of<__half>(part, sms, st));
  }
  return PCB_OK;
}
