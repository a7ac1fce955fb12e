// pcb_head.cu — a categorical head with weights in 4 bits and group scales, for few feature vectors:
//   y[m, n] = sum_k scale[n, k / group] (code[n, k] - 8) x[m, k] + bias[n].
//
// The weights are the A operand of mma.sync m16n8k16: 16 categories x 16 features, codes turned into integers -8..7 in the
// features' own type, where they and their products with x are exact; a group's sum stays in the fp32 accumulator and meets
// its scale there, once.  (fp32 features go in as three bf16 terms, which hold all 24 bits.)
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

namespace {

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
  PCB_REQUIRE(cats >= 1 && cats <= 0x7fffffffu && features >= 1 && features <= 0x7fffffffu, "a head has at least one category and one feature");
  PCB_REQUIRE(group == 32 || group == 64 || group == 128, "groups hold 32, 64 or 128 features");
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

// One warp per (category, group): scale = max |w| / 7, code = round(w / scale) + 8 with the scale as stored.
__global__ void __launch_bounds__(256) head_quantize_kernel(const void* w, int32_t dtype, uint32_t cats, uint32_t features, uint32_t group,
                                                            int32_t scale_dtype, uint8_t* codes, uint16_t* scales) {
  const uint32_t lane = threadIdx.x & 31, groups = (features + group - 1) / group, bytes = (features + 1) / 2;
  const uint64_t total = (uint64_t)cats * groups;
  for (uint64_t i = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; i < total; i += (uint64_t)gridDim.x * 8) {
    const uint64_t n = i / groups;
    const uint32_t k0 = (uint32_t)(i % groups) * group, k1 = min(features, k0 + group);
    float most = 0.0f;
    for (uint32_t k = k0 + lane; k < k1; k += 32) most = fmaxf(most, fabsf(load_as_f32(w, n * features + k, dtype)));
    for (int o = 16; o; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
    const float want = most / 7.0f;
    const uint16_t bits = scale_dtype == PCB_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(want)) : __half_as_ushort(__float2half_rn(want));
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

__global__ void __launch_bounds__(256) head_pack_kernel(HeadShape h, const uint8_t* codes, const uint16_t* scales, uint32_t* out) {
  const uint64_t nc = h.code_words(), total = nc + h.scale_words();
  const uint32_t bytes = (h.features + 1) / 2, groups = (h.features + h.group - 1) / h.group;
  for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (uint64_t)gridDim.x * blockDim.x) {
    uint32_t word = 0;
    if (i < nc) {
      const uint32_t w = i & 3, lane = (i >> 2) & 31;
      const uint64_t tb = i >> 7, tile = tb / h.blocks, block = tb % h.blocks;
      for (uint32_t p = 0; p < 8; ++p) {
        uint32_t row, k;
        nibble_place(lane, w, p, row, k);
        const uint64_t n = tile * 16 + row, kk = block * 64 + k;
        uint32_t code = 8;
        if (n < h.cats && kk < h.features) code = (codes[n * bytes + kk / 2] >> (4 * (kk & 1))) & 15u;
        word |= code << (4 * p);
      }
    } else {
      const uint64_t r = i - nc;   // [tile][quad][g][group of the quad]
      const uint32_t j = r & 3, g = (r >> 2) & 7;
      const uint64_t tq = r >> 5, tile = tq / h.quads, group = tq % h.quads * 4 + j;
      for (uint32_t e = 0; e < 2; ++e) {
        const uint64_t n = tile * 16 + g + 8 * e;
        if (n < h.cats && group < groups) word |= (uint32_t)scales[n * groups + group] << (16 * e);
      }
    }
    out[i] = word;
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

template <typename T> struct Operand;   // two 16-bit values of the tensor cores' operand type
template <> struct Operand<__nv_bfloat16> {
  static constexpr uint32_t BASE = 0x43004300u;   // 128: the codes' ulp there is 1
  static __device__ __forceinline__ uint32_t minus8(uint32_t v) {   // (128 + code) - 136, exact
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), __floats2bfloat162_rn(136.0f, 136.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct Operand<__half> {
  static constexpr uint32_t BASE = 0x64006400u;   // 1024
  static __device__ __forceinline__ uint32_t minus8(uint32_t v) {
    const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&v), __floats2half2_rn(1032.0f, 1032.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
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

// One warp per tile of 16 categories and 8 feature vectors.
template <typename X>
__global__ void __launch_bounds__(128) head_kernel(HeadArgs a) {
  using F = Feature<X>;
  using Op = Operand<typename F::Op>;
  const uint32_t lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint64_t tile = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (tile >= a.h.tiles) return;
  const uint4* codes = reinterpret_cast<const uint4*>(a.packed) + tile * a.h.blocks * 32;
  const uint32_t* scales = a.packed + a.h.code_words() + tile * a.h.quads * 32;
  for (uint64_t m0 = (uint64_t)blockIdx.y * 8; m0 < a.rows; m0 += (uint64_t)gridDim.y * 8) {
    const uint64_t m = m0 + g;
    const X* x = static_cast<const X*>(a.x) + (m < a.rows ? m : 0) * a.x_stride;
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t b = 0; b < a.h.blocks; ++b) {
      const uint4 q = codes[(uint64_t)b * 32 + lane];
      const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (uint32_t h = 0; h < 2; ++h) {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const uint32_t k0 = b * 64 + h * 32;
#pragma unroll
        for (uint32_t j = 0; j < 2; ++j) {
          uint16_t v[4][3];
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            const uint32_t k = k0 + 8 * t + 4 * j + e;
            X xv = X(0.0f);
            if (m < a.rows && k < a.h.features) xv = x[k];
            terms_of(xv, v[e]);
          }
          uint32_t frag[4];
          const uint32_t w = words[2 * h + j];
#pragma unroll
          for (int i = 0; i < 4; ++i) frag[i] = Op::minus8((w >> (4 * i) & 0x000f000fu) | Op::BASE);
#pragma unroll
          for (int s = 0; s < F::TERMS; ++s)
            Op::mma(acc, frag, v[0][s] | (uint32_t)v[1][s] << 16, v[2][s] | (uint32_t)v[3][s] << 16);
        }
        const uint32_t group = k0 / a.h.group;
        if (group >= 4 * a.h.quads) continue;   // the padding of the last block
        const uint32_t two = scales[(group / 4) * 32 + g * 4 + group % 4];
        const float s0 = scale_f32(two & 0xffffu, a.scale_dtype), s1 = scale_f32(two >> 16, a.scale_dtype);
        sum[0] = fmaf(s0, acc[0], sum[0]);
        sum[1] = fmaf(s0, acc[1], sum[1]);
        sum[2] = fmaf(s1, acc[2], sum[2]);
        sum[3] = fmaf(s1, acc[3], sum[3]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t n = tile * 16 + g + 8 * (i >> 1), r = m0 + 2 * t + (i & 1);
      if (n < a.h.cats && r < a.rows) store_y(a.y, r * a.h.cats + n, sum[i] + (a.bias ? a.bias[n] : 0.0f), a.y_dtype);
    }
  }
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
  const HeadShape h = head_shape(cats, features, group);
  head_pack_kernel<<<blocks_for(h.code_words() + h.scale_words()), 256, 0, (cudaStream_t)s>>>(h, codes_dev, static_cast<const uint16_t*>(scales_dev),
                                                                                             static_cast<uint32_t*>(packed_dev));
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}

extern "C" int32_t pcb_head_weight(const void* packed_dev, int32_t scale_dtype, uint32_t cats, uint32_t features, uint32_t group,
                                   float* weight_dev, pcb_stream s) {
  if (int32_t rc = check_shape(cats, features, group)) return rc;
  PCB_REQUIRE(packed_dev && weight_dev, "null argument");
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
  HeadArgs a{head_shape(cats, features, group), static_cast<const uint32_t*>(packed_dev), scale_dtype, y_dtype, x_dev, rows, x_row_stride, bias_dev, y_dev};
  const dim3 grid((a.h.tiles + 3) / 4, (uint32_t)((rows + 7) / 8 < 65535 ? (rows + 7) / 8 : 65535));
  cudaStream_t st = (cudaStream_t)s;
  if (dtype == PCB_F32) head_kernel<float><<<grid, 128, 0, st>>>(a);
  else if (dtype == PCB_BF16) head_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(a);
  else head_kernel<__half><<<grid, 128, 0, st>>>(a);
  PCB_CUDA(cudaGetLastError());
  return PCB_OK;
}
