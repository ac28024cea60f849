// Quantisers of activations and weights for the block-scaled GEMMs, as kernels:
//
//   RMS norm with the residual's addition and FP8 output (bb_rmsnorm_fp8_*)
//     h = round_T(x + r),  y = h * rsqrt(mean(h^2) + eps) * w,
//     s[g] = amax |y[g]| / 448 over the 128 columns of group g (1 where that is 0),
//     q = e4m3(y / s), the scales stored [group][row].
//   4-bit microscaled formats (bb_fp4_quant_*)
//     NVFP4: b = e4m3(min(amax_16 / 6 / g, 448)), q = e2m1(x / (b g)), 0 where b g is 0
//     MXFP4: b = 2^(floor(log2 amax_32) - 2) as E8M0, q = e2m1(x / b)
//     with the scales stored as the 512-byte atoms the tensor core reads.
//
// Both read each input once and are bound by DRAM bandwidth at large sizes and
// by launch latency at small ones. All statistics are FP32. The only
// roundings to fewer bits are the ones in the formulas: the stored h (the next
// layer reads it, so the norm is of the stored value), the scales of the 4-bit
// formats and the values themselves.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <new>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace bb {
extern std::atomic<int64_t> g_kernel_launches;

namespace quant {

constexpr float kE4m3Max = 448.f;
constexpr float kE2m1Max = 6.f;

// ---------------------------------------------------------------- element access
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// 8 consecutive elements. kWide: one or two 16-byte accesses (the host
// checked base and row stride, and cols % 8 == 0, so a vector is whole);
// otherwise element by element, elements from `valid` on read as 0 / are not written.
template <typename T>
union alignas(16) Vec8 {
  T e[8];
  uint4 q[sizeof(T) * 8 / 16];
};

template <bool kWide, typename T>
__device__ __forceinline__ Vec8<T> load8(const T* p, int valid) {
  Vec8<T> v;
  if constexpr (kWide) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) v.q[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v.e[i] = i < valid ? p[i] : from_f32<T>(0.f);
  }
  return v;
}
template <bool kWide, typename T>
__device__ __forceinline__ void store8(T* p, const Vec8<T>& v, int valid) {
  if constexpr (kWide) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = v.q[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = v.e[i];
  }
}

// max that keeps a NaN of either side (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two FP32 operations per instruction (sm_100's packed FP32).
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pack2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack2(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// y[i] / s for the N values of a block whose magnitudes are at most `most`,
// correctly rounded: with r = 1 / s correctly rounded, one residual step
// q = q0 + (y - q0 s) r of q0 = y r gives the rounded quotient (Markstein, IBM
// J. Res. Dev. 34, 1990) while nothing leaves the normal numbers; other blocks
// divide. One and a half instructions per value instead of a division's dozen,
// which would bound the quantisers.
template <int N>
__device__ __forceinline__ void divide(float (&y)[N], float s, float most) {
  const float r = __fdiv_rn(1.f, s);
  if (s > 0x1p-60f && s < 0x1p60f && most * r < 0x1p60f) {
    const F2 r2 = pack2(r, r), s2 = pack2(-s, -s);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const F2 v = pack2(y[i], y[i + 1]);
      const F2 q0 = mul2(v, r2);
      unpack2(fma2(fma2(q0, s2, v), r2, q0), y[i], y[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] = __fdiv_rn(y[i], s);
  }
}

// ================================================================ RMS norm -> FP8
struct NormParams {
  int64_t rows;
  int32_t cols, groups;
  int64_t x_ld, res_ld, out_ld, q_ld, s_ld;
  const void* x;
  const void* residual;
  const void* weight;
  void* residual_out;
  uint8_t* q;
  float* scales;
  float eps;
  int32_t weight_f32;
};

constexpr int kNormMaxThreads = 1024;
constexpr int kNormMaxIters = 8;  // 8 vectors of 8 columns per thread: 65536 columns

// One CTA per row; thread t owns the 8-column vectors t, t + blockDim, ...,
// which stay in registers between the sum and the output (x and r are read
// once). The 16 vectors of a scale group sit in 16 neighbouring lanes.
template <typename T, int kIters, bool kWide>
__global__ void __launch_bounds__(kNormMaxThreads) rmsnorm_fp8_kernel(const NormParams p) {
  __shared__ float warp_sum[32];
  grid_wait();
  grid_trigger();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  T* out = p.residual_out ? static_cast<T*>(p.residual_out) + row * p.out_ld : nullptr;
  // All loads of a thread before its first store: a store to residual_out may
  // alias what is still to be loaded as far as the compiler knows.
  Vec8<T> v[kIters], r[kIters];
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int c = (it * blockDim.x + threadIdx.x) * 8;
    if (c < p.cols) {
      v[it] = load8<kWide>(x + c, p.cols - c);
      if (res) r[it] = load8<kWide>(res + c, p.cols - c);
    }
  }
  float h[kIters][8];
  float sum = 0.f;
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int c = (it * blockDim.x + threadIdx.x) * 8;
    if (c < p.cols) {
      if (res) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[it].e[i] = from_f32<T>(to_f32(v[it].e[i]) + to_f32(r[it].e[i]));
      }
      if (out) store8<kWide>(out + c, v[it], p.cols - c);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[it][i] = to_f32(v[it].e[i]);
        sum = __fmaf_rn(h[it][i], h[it][i], sum);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) h[it][i] = 0.f;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if (threadIdx.x % 32 == 0) warp_sum[threadIdx.x / 32] = sum;
  __syncthreads();
  sum = threadIdx.x % 32 < blockDim.x / 32 ? warp_sum[threadIdx.x % 32] : 0.f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  const float rstd = rsqrtf(sum / static_cast<float>(p.cols) + p.eps);
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int vec = it * blockDim.x + threadIdx.x;
    const int c = vec * 8;
    const int valid = p.cols - c;
    float amax = 0.f;
    if (valid > 0) {
      float w[8];
      if (p.weight_f32) {
        const Vec8<float> v = load8<kWide>(static_cast<const float*>(p.weight) + c, valid);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = v.e[i];
      } else {
        const Vec8<T> v = load8<kWide>(static_cast<const T*>(p.weight) + c, valid);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = to_f32(v.e[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[it][i] = i < valid ? h[it][i] * rstd * w[i] : 0.f;
        amax = max_nan(amax, fabsf(h[it][i]));
      }
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
    if (valid > 0) {
      const float s = amax == 0.f ? 1.f : __fdiv_rn(amax, kE4m3Max);
      if (vec % 16 == 0) p.scales[(vec / 16) * p.s_ld + row] = s;
      divide(h[it], s, amax);
      union {
        uint8_t b[8];
        __nv_fp8x2_storage_t h2[4];
        uint2 q;
      } o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o.h2[i] = __nv_cvt_float2_to_fp8x2(make_float2(h[it][2 * i], h[it][2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
      uint8_t* q = p.q + row * p.q_ld + c;
      if constexpr (kWide) {
        *reinterpret_cast<uint2*>(q) = o.q;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < valid) q[i] = o.b[i];
      }
    }
  }
}

// ================================================================ 4-bit formats
struct Fp4Params {
  int64_t rows;
  uint32_t total;          // threads: rows of whole 128-row atoms x 16 columns
  int32_t cols, atoms_k;   // atoms along K
  int64_t x_ld, v_ld;
  const void* x;
  uint8_t* data;           // rows x cols / 2
  uint8_t* atoms;
  void* values;            // dequantised values, may be null
  const float* partial_max;  // NVFP4 with a scale to be found: the row ranges' maxima
  int32_t partials;
  float tensor_scale;      // NVFP4 with a given scale
  float* tensor_scale_out;
};

constexpr int kFp4Threads = 256;
constexpr int kMaxPartials = 1184;  // CTAs of the maximum's kernel

// E2M1 codes of 8 values, element i in nibble i; the sign of a zero is dropped.
__device__ __forceinline__ uint32_t e2m1x8(const float* y) {
  uint32_t w;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(w)
      : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
  // Nibble magnitude + 7 carries into bit 3 exactly where it is not zero.
  const uint32_t mag = w & 0x77777777u;
  return mag | (w & (mag + 0x77777777u) & 0x88888888u);
}

// The values of 8 codes (element i in nibble i), by way of FP16, which holds them exactly.
__device__ __forceinline__ void e2m1x8_values(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// max |e| of 8 elements; a NaN wins. The 16-bit types compare two at a time.
template <typename T>
__device__ __forceinline__ float absmax8(const Vec8<T>& v) {
  if constexpr (sizeof(T) == 4) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_nan(m, fabsf(v.e[i]));
    return m;
  } else {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(v.q);
    uint32_t m = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __half>)
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
      else
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i] & 0x7fff7fffu));
    }
    const T* e = reinterpret_cast<const T*>(&m);
    return max_nan(to_f32(e[0]), to_f32(e[1]));
  }
}

__device__ __forceinline__ float found_scale(const float* partial, int n) {
  // Whole block: the maximum of the partial maxima (bit patterns of
  // non-negative floats order like the floats, a NaN above all).
  __shared__ uint32_t warp_max[kFp4Threads / 32];
  uint32_t m = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) m = max(m, __float_as_uint(partial[i]));
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
  for (int i = 0; i < kFp4Threads / 32; ++i) m = max(m, warp_max[i]);
  const float amax = __uint_as_float(m);
  const float g = __fdiv_rn(amax, kE4m3Max * kE2m1Max);
  return g > 0.f ? g : 1.f;  // no data, data below 2688 times the least FP32 number, or NaN
}

// Maxima of |x| over ranges of the tensor, one per CTA.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kFp4Threads) absmax_kernel(const Fp4Params p, float* partial) {
  __shared__ uint32_t warp_max[kFp4Threads / 32];
  grid_wait();
  grid_trigger();
  const int vecs = (p.cols + 7) / 8;
  uint32_t m = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
    for (int v = threadIdx.x; v < vecs; v += blockDim.x) {
      const Vec8<T> e = load8<kWide>(x + v * 8, p.cols - v * 8);
      m = max(m, __float_as_uint(fabsf(absmax8(e))));  // a NaN's sign must not count
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kFp4Threads / 32; ++i) m = max(m, warp_max[i]);
    partial[blockIdx.x] = __uint_as_float(m);
  }
}

// A thread owns 16 columns of a row: one NVFP4 block, or half an MXFP4 block
// whose maximum it shares with its neighbour lane. Four scales (4 or 8 lanes)
// make the 4 bytes a row has in one atom.
template <typename T, bool kMx, bool kWide>
__global__ void __launch_bounds__(kFp4Threads) fp4_quant_kernel(const Fp4Params p) {
  grid_wait();
  grid_trigger();
  float g = p.tensor_scale;
  if constexpr (!kMx) {
    if (p.partial_max) {
      g = found_scale(p.partial_max, p.partials);
      if (blockIdx.x == 0 && threadIdx.x == 0) *p.tensor_scale_out = g;
    }
  }
  constexpr int kLanes = kMx ? 8 : 4;  // threads of one row's part of an atom
  const uint32_t per_row = static_cast<uint32_t>(p.atoms_k) * kLanes;
  // With a scale found by the launch before, the tensor is read a second time:
  // from its end, which is what L2 still holds of the first reading.
  const uint32_t block = p.partial_max ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const uint32_t idx = block * kFp4Threads + threadIdx.x;
  const bool live = idx < p.total;
  const uint32_t row32 = live ? idx / per_row : 0;
  const int64_t row = row32;
  const int part = live ? static_cast<int>(idx - row32 * per_row) : 0;
  const int c = part * 16;
  const bool has = live && row < p.rows && c < p.cols;  // cols % 32 == 0: all or none
  float v[16];
  float amax = 0.f;
  if (has) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld + c;
    Vec8<T> e[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) e[j] = load8<kWide>(x + 8 * j, 8);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[8 * j + i] = to_f32(e[j].e[i]);
    }
    amax = max_nan(absmax8(e[0]), absmax8(e[1]));
  }
  if constexpr (kMx) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  uint32_t byte = 0;
  if (has) {
    float unit;
    bool zero = false;
    if constexpr (kMx) {
      // Exponent byte of 2^(floor(log2 amax) - 2): amax's own biased exponent
      // less 2 (a subnormal amax and 0 give 0, as does all below 2^-124); an
      // infinite or NaN block has scale NaN.
      const int e = static_cast<int>((__float_as_uint(amax) >> 23) & 0xffu);
      byte = e == 255 ? 255u : static_cast<uint32_t>(max(e - 2, 0));
      zero = byte == 255u;
      // 2^(127 - byte): exact, so y = x / b exactly. byte <= 252 here.
      const float inv = __uint_as_float((254u - min(byte, 253u)) << 23);
      unit = byte == 255u ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : 0x1p-127f;
      const F2 inv2 = pack2(inv, inv);
#pragma unroll
      for (int i = 0; i < 16; i += 2) unpack2(mul2(pack2(v[i], v[i + 1]), inv2), v[i], v[i + 1]);
    } else {
      const float want = __fdiv_rn(__fdiv_rn(amax, kE2m1Max), g);
      byte = __nv_cvt_float_to_fp8(want, __NV_SATFINITE, __NV_E4M3) & 0x7fu;  // a NaN's sign is dropped
      unit = __half2float(__half(__nv_cvt_fp8_to_halfraw(byte, __NV_E4M3)));
      const float d = unit * g;
      zero = !(d > 0.f);  // an empty block, one below the scales' range, or NaN
      divide(v, zero ? 1.f : d, amax);
    }
    const uint2 codes = zero ? make_uint2(0u, 0u) : make_uint2(e2m1x8(v), e2m1x8(v + 8));
    *reinterpret_cast<uint2*>(p.data + row * (p.cols / 2) + c / 2) = codes;
    if (p.values) {
      T* out = static_cast<T*>(p.values) + row * p.v_ld + c;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float q[8];
        e2m1x8_values(j ? codes.y : codes.x, q);
        Vec8<T> o;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          q[i] *= unit;
          if constexpr (!kMx) q[i] *= g;
          o.e[i] = from_f32<T>(q[i]);
        }
        store8<kWide>(out + 8 * j, o, 8);
      }
    }
  }
  // The four scale bytes of this row and atom, gathered in the first lane.
  const int step = kMx ? 2 : 1;
  uint32_t word = byte;
#pragma unroll
  for (int j = 1; j < 4; ++j) word |= __shfl_down_sync(0xffffffffu, byte, j * step) << (8 * j);
  if (live && part % kLanes == 0) {
    const int64_t rb = row / 128;
    const int r = static_cast<int>(row % 128);
    uint8_t* atom = p.atoms + (rb * p.atoms_k + part / kLanes) * 512;
    *reinterpret_cast<uint32_t*>(atom + (r % 32) * 16 + (r / 32) * 4) = word;
  }
}

}  // namespace quant
}  // namespace bb

using namespace bb;
using namespace bb::quant;

struct bb_quant_plan {
  bool norm = false;
  int dtype = 0, fmt = 0, device = 0;
  bool wide = false;
  cudaStream_t stream = nullptr;
  NormParams np{};
  Fp4Params fp{};
  int threads = 0, iters = 0;
  float* partial = nullptr;  // maxima of the NVFP4 tensor scale
  int partials = 0;
  int64_t launches = 0;
};

namespace {

size_t dtype_size(int dtype) { return dtype == BB_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == BB_DTYPE_BF16 || dtype == BB_DTYPE_F32 || dtype == BB_DTYPE_F16; }
bool aligned16(const void* p, int64_t ld, size_t size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (static_cast<size_t>(ld) * size) % 16 == 0;
}

// Every launch may start before the one before it has ended (the kernels wait).
template <typename... Args, typename... Given>
cudaError_t launch(void (*kernel)(Args...), unsigned grid, int threads, cudaStream_t stream, Given... given) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, given...);
}

template <typename T, bool kWide>
cudaError_t launch_norm(const bb_quant_plan& pl) {
  const unsigned grid = static_cast<unsigned>(pl.np.rows);
  switch (pl.iters) {
    case 1: return launch(rmsnorm_fp8_kernel<T, 1, kWide>, grid, pl.threads, pl.stream, pl.np);
    case 2: return launch(rmsnorm_fp8_kernel<T, 2, kWide>, grid, pl.threads, pl.stream, pl.np);
    case 4: return launch(rmsnorm_fp8_kernel<T, 4, kWide>, grid, pl.threads, pl.stream, pl.np);
    default: return launch(rmsnorm_fp8_kernel<T, 8, kWide>, grid, pl.threads, pl.stream, pl.np);
  }
}

template <typename T, bool kWide>
cudaError_t launch_fp4(const bb_quant_plan& pl) {
  const bool mx = pl.fmt == BB_LOWP_MXFP4;
  if (pl.partials) {
    const cudaError_t e = launch(absmax_kernel<T, kWide>, pl.partials, kFp4Threads, pl.stream, pl.fp, pl.partial);
    if (e != cudaSuccess) return e;
  }
  const unsigned grid = (pl.fp.total + kFp4Threads - 1) / kFp4Threads;
  return mx ? launch(fp4_quant_kernel<T, true, kWide>, grid, kFp4Threads, pl.stream, pl.fp)
            : launch(fp4_quant_kernel<T, false, kWide>, grid, kFp4Threads, pl.stream, pl.fp);
}

template <typename T>
cudaError_t launch_typed(const bb_quant_plan& pl) {
  if (pl.norm) return pl.wide ? launch_norm<T, true>(pl) : launch_norm<T, false>(pl);
  return pl.wide ? launch_fp4<T, true>(pl) : launch_fp4<T, false>(pl);
}

}  // namespace

extern "C" {

BB_API int bb_fp4_quant_plan_create(int format, int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t x_ld,
                                    void* data, void* scales, float tensor_scale, float* tensor_scale_out,
                                    void* values, int64_t values_ld, void* stream, bb_quant_plan** plan) {
  try {
    clear_error();
    if (!plan) {
      set_error("bb_fp4_quant_plan_create: plan out-pointer is null");
      return BB_ERR_ARGUMENT;
    }
    *plan = nullptr;
    if (format != BB_LOWP_NVFP4 && format != BB_LOWP_MXFP4) {
      set_error("bb_fp4_quant_plan_create: unknown format %d", format);
      return BB_ERR_ARGUMENT;
    }
    if (!known_dtype(x_dtype)) {
      set_error("bb_fp4_quant_plan_create: unknown dtype %d", x_dtype);
      return BB_ERR_ARGUMENT;
    }
    if (rows < 0 || rows > (int64_t(1) << 30) || cols <= 0 || cols > (int64_t(1) << 24) || cols % 32 != 0) {
      set_error("bb_fp4_quant_plan_create: rows=%lld must lie in [0, 2^30], cols=%lld in [32, 2^24] and be a multiple of 32",
                (long long)rows, (long long)cols);
      return BB_ERR_ARGUMENT;
    }
    if (rows > 0 && (!x || !data || !scales)) {
      set_error("bb_fp4_quant_plan_create: null pointer");
      return BB_ERR_ARGUMENT;
    }
    if ((rows > 1 && x_ld < cols) || (rows > 1 && values && values_ld < cols)) {
      set_error("bb_fp4_quant_plan_create: row stride below cols");
      return BB_ERR_ARGUMENT;
    }
    const bool find = format == BB_LOWP_NVFP4 && tensor_scale_out != nullptr;
    if (format == BB_LOWP_NVFP4 && !find && !(tensor_scale > 0.f && tensor_scale <= 3.402823466e38f)) {
      set_error("bb_fp4_quant_plan_create: tensor_scale must be positive and finite");
      return BB_ERR_ARGUMENT;
    }
    const size_t size = dtype_size(x_dtype);
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(values) % size ||
        reinterpret_cast<uintptr_t>(data) % 16 || reinterpret_cast<uintptr_t>(scales) % 16 ||
        reinterpret_cast<uintptr_t>(tensor_scale_out) % 4) {
      set_error("bb_fp4_quant_plan_create: data and scales must be 16-byte aligned, x and values to their type");
      return BB_ERR_ARGUMENT;
    }
    const int64_t atom_k = format == BB_LOWP_MXFP4 ? 128 : 64;
    const int64_t atoms_k = (cols + atom_k - 1) / atom_k, rows_pad = (rows + 127) / 128 * 128;
    const int64_t total = rows_pad * atoms_k * (format == BB_LOWP_MXFP4 ? 8 : 4);
    if (total > 0xffffffffll - kFp4Threads) {
      set_error("bb_fp4_quant_plan_create: %lld x %lld is more than one launch covers", (long long)rows, (long long)cols);
      return BB_ERR_ARGUMENT;
    }
    DeviceInfo dev;
    int rc = query_device(&dev);
    if (rc != BB_OK) return rc;
    auto* h = new (std::nothrow) bb_quant_plan();
    if (!h) {
      set_error("bb_fp4_quant_plan_create: out of host memory");
      return BB_ERR_INTERNAL;
    }
    h->device = dev.device;
    h->dtype = x_dtype;
    h->fmt = format;
    h->stream = static_cast<cudaStream_t>(stream);
    h->wide = aligned16(x, rows > 1 ? x_ld : 0, size) && (!values || aligned16(values, rows > 1 ? values_ld : 0, size));
    Fp4Params& p = h->fp;
    p.rows = rows;
    p.total = static_cast<uint32_t>(total);
    p.cols = static_cast<int32_t>(cols);
    p.atoms_k = static_cast<int32_t>(atoms_k);
    p.x_ld = x_ld;
    p.v_ld = values_ld;
    p.x = x;
    p.data = static_cast<uint8_t*>(data);
    p.atoms = static_cast<uint8_t*>(scales);
    p.values = values;
    p.tensor_scale = tensor_scale;
    p.tensor_scale_out = tensor_scale_out;
    if (find && rows > 0) {
      const int64_t most = 8ll * dev.sm_count < kMaxPartials ? 8ll * dev.sm_count : kMaxPartials;
      h->partials = static_cast<int>(rows < most ? rows : most);
      rc = check_cuda(cudaMalloc(&h->partial, h->partials * sizeof(float)), "cudaMalloc(maxima)");
      if (rc != BB_OK) {
        delete h;
        return rc;
      }
      p.partial_max = h->partial;
      p.partials = h->partials;
    }
    *plan = h;
    return BB_OK;
  } catch (...) {
    set_error("bb_fp4_quant_plan_create: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_rmsnorm_fp8_plan_create(int64_t rows, int64_t cols, const void* x, int x_dtype, int64_t x_ld,
                                      const void* residual, int64_t residual_ld, void* residual_out,
                                      int64_t residual_out_ld, const void* weight, int weight_dtype, float eps,
                                      void* q, int64_t q_ld, float* scales, int64_t scales_ld, void* stream,
                                      bb_quant_plan** plan) {
  try {
    clear_error();
    if (!plan) {
      set_error("bb_rmsnorm_fp8_plan_create: plan out-pointer is null");
      return BB_ERR_ARGUMENT;
    }
    *plan = nullptr;
    if (!known_dtype(x_dtype) || (weight_dtype != x_dtype && weight_dtype != BB_DTYPE_F32)) {
      set_error("bb_rmsnorm_fp8_plan_create: unknown dtype %d, or a weight of dtype %d beside it", x_dtype, weight_dtype);
      return BB_ERR_ARGUMENT;
    }
    constexpr int64_t kMaxCols = int64_t(8) * kNormMaxThreads * kNormMaxIters;
    if (rows < 0 || rows > (int64_t(1) << 30) || cols <= 0 || cols > kMaxCols) {
      set_error("bb_rmsnorm_fp8_plan_create: rows=%lld must lie in [0, 2^30], cols=%lld in [1, %lld]", (long long)rows,
                (long long)cols, (long long)kMaxCols);
      return BB_ERR_ARGUMENT;
    }
    if (rows > 0 && (!x || !weight || !q || !scales)) {
      set_error("bb_rmsnorm_fp8_plan_create: null pointer");
      return BB_ERR_ARGUMENT;
    }
    if (!(eps >= 0.f)) {
      set_error("bb_rmsnorm_fp8_plan_create: eps must not be negative");
      return BB_ERR_ARGUMENT;
    }
    if (rows > 1 && (x_ld < cols || (residual && residual_ld < cols) || (residual_out && residual_out_ld < cols) ||
                     q_ld < cols || scales_ld < rows)) {
      set_error("bb_rmsnorm_fp8_plan_create: row stride below cols, or scales_ld below rows");
      return BB_ERR_ARGUMENT;
    }
    const size_t size = dtype_size(x_dtype), wsize = dtype_size(weight_dtype);
    if (reinterpret_cast<uintptr_t>(x) % size || reinterpret_cast<uintptr_t>(residual) % size ||
        reinterpret_cast<uintptr_t>(residual_out) % size || reinterpret_cast<uintptr_t>(weight) % wsize ||
        reinterpret_cast<uintptr_t>(scales) % 4) {
      set_error("bb_rmsnorm_fp8_plan_create: a pointer is not aligned to its type");
      return BB_ERR_ARGUMENT;
    }
    DeviceInfo dev;
    int rc = query_device(&dev);
    if (rc != BB_OK) return rc;
    auto* h = new (std::nothrow) bb_quant_plan();
    if (!h) {
      set_error("bb_rmsnorm_fp8_plan_create: out of host memory");
      return BB_ERR_INTERNAL;
    }
    h->norm = true;
    h->device = dev.device;
    h->dtype = x_dtype;
    h->stream = static_cast<cudaStream_t>(stream);
    auto wide = [&](const void* ptr, int64_t ld, size_t sz) { return aligned16(ptr, rows > 1 ? ld : 0, sz); };
    h->wide = cols % 8 == 0 && wide(x, x_ld, size) && (!residual || wide(residual, residual_ld, size)) &&
              (!residual_out || wide(residual_out, residual_out_ld, size)) && wide(weight, 0, wsize) &&
              reinterpret_cast<uintptr_t>(q) % 8 == 0 && (rows <= 1 || q_ld % 8 == 0);
    const int64_t vecs = (cols + 7) / 8;
    h->iters = 1;
    while (vecs > int64_t(256) * h->iters && h->iters < 4) h->iters *= 2;
    if (vecs > int64_t(kNormMaxThreads) * h->iters) h->iters = kNormMaxIters;
    h->threads = static_cast<int>(((vecs + h->iters - 1) / h->iters + 31) / 32 * 32);
    NormParams& p = h->np;
    p.rows = rows;
    p.cols = static_cast<int32_t>(cols);
    p.groups = static_cast<int32_t>((cols + 127) / 128);
    p.x_ld = x_ld;
    p.res_ld = residual_ld;
    p.out_ld = residual_out_ld;
    p.q_ld = q_ld;
    p.s_ld = scales_ld;
    p.x = x;
    p.residual = residual;
    p.weight = weight;
    p.residual_out = residual_out;
    p.q = static_cast<uint8_t*>(q);
    p.scales = scales;
    p.eps = eps;
    p.weight_f32 = weight_dtype == BB_DTYPE_F32;
    *plan = h;
    return BB_OK;
  } catch (...) {
    set_error("bb_rmsnorm_fp8_plan_create: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_quant_execute_n(bb_quant_plan* plan, int iterations) {
  try {
    if (!plan || iterations < 0) {
      set_error("bb_quant_execute_n: null plan or negative iteration count");
      return BB_ERR_ARGUMENT;
    }
    const int64_t rows = plan->norm ? plan->np.rows : plan->fp.rows;
    if (rows == 0) return BB_OK;
    DeviceGuard guard(plan->device);
    BB_CUDA_TRY(guard.status);
    for (int i = 0; i < iterations; ++i) {
      const cudaError_t e = plan->dtype == BB_DTYPE_BF16  ? launch_typed<__nv_bfloat16>(*plan)
                            : plan->dtype == BB_DTYPE_F16 ? launch_typed<__half>(*plan)
                                                          : launch_typed<float>(*plan);
      int rc = check_cuda(e, "launch of a quantiser");
      if (rc != BB_OK) return rc;
      const int n = plan->partials ? 2 : 1;
      plan->launches += n;
      g_kernel_launches.fetch_add(n, std::memory_order_relaxed);
    }
    return BB_OK;
  } catch (...) {
    set_error("bb_quant_execute_n: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_quant_synchronize(bb_quant_plan* plan) {
  if (!plan) {
    set_error("bb_quant_synchronize: null plan");
    return BB_ERR_ARGUMENT;
  }
  return check_cuda(cudaStreamSynchronize(plan->stream), "cudaStreamSynchronize");
}

BB_API int64_t bb_quant_launches(const bb_quant_plan* plan) { return plan ? plan->launches : -1; }

BB_API int bb_quant_destroy(bb_quant_plan* plan) {
  if (!plan) return BB_OK;
  int rc = BB_OK;
  if (plan->partial) rc = check_cuda(cudaFree(plan->partial), "cudaFree(maxima)");
  delete plan;
  return rc;
}

}  // extern "C"
