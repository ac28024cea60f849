// Quantisers of activations and weights for the block-scaled GEMMs, as kernels:
//
//   RMS norm with the residual's addition and FP8 output (bb_rmsnorm_fp8_*)
//     h = round_T(x + r),  y = h * rsqrt(mean(h^2) + eps) * w,
//     s[g] = amax |y[g]| / 448 over the 128 columns of group g (1 where that is 0 in FP32),
//     q = e4m3(y / s), the scales stored [group][row].
//   4-bit microscaled formats (bb_fp4_quant_*)
//     NVFP4: b = e4m3(min(amax_16 / 6 / g, 448)), q = e2m1(x / (b g)), 0 where b g is 0
//     MXFP4: b = 2^(floor(log2 amax_32) - 2) as E8M0, q = e2m1(x / b)
//     with the scales stored as the 512-byte atoms the tensor core reads.
//
// Each input is read once, except where an NVFP4 tensor scale is to be found: x is
// then read a second time, and of a few rows by every CTA. They are bound by DRAM
// bandwidth at large sizes and by launch latency at small ones. All statistics are FP32. The only
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

// A thread's unit of columns: 32 bytes, moved by one 256-bit access.
template <typename T>
constexpr int kVE = 32 / sizeof(T);
template <typename T>
union alignas(32) Vec {
  T e[kVE<T>];
  uint32_t w[8];
};

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> v;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]), "=r"(v.w[7])
               : "l"(p)
               : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]), "r"(v.w[2]),
               "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
               : "memory");
}

// max that keeps a NaN of either side (fmaxf drops it).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// max(|a|, |b|, c), NaN if any is.
__device__ __forceinline__ float max_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
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

constexpr int64_t kNormMaxCols = 65536;

// h = round_T(x + r) for one 32-byte vector. The 16-bit additions round the
// exact sum once, which is what rounding the FP32 sum gives: where that is
// inexact (exponents over 13 apart), the smaller term is far below half a step.
template <typename T>
__device__ __forceinline__ void add_vec(Vec<T>& v, const Vec<T>& r) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) v.e[i] += r.e[i];
    else if constexpr (std::is_same_v<T, __half>) asm("add.rn.f16x2 %0, %0, %1;" : "+r"(v.w[i]) : "r"(r.w[i]));
    else asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(v.w[i]) : "r"(r.w[i]));
  }
}

// Elements 2 i and 2 i + 1 as FP32.
template <typename T>
__device__ __forceinline__ F2 pair_f32(const Vec<T>& v, int i) {
  if constexpr (sizeof(T) == 4) {
    return pack2(v.e[2 * i], v.e[2 * i + 1]);
  } else if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v.w[i]));
    return pack2(f.x, f.y);
  } else {
    return pack2(__uint_as_float(v.w[i] << 16), __uint_as_float(v.w[i] & 0xffff0000u));
  }
}

// One CTA per row; a thread's kIters vectors of 32 bytes stay in registers
// between the sum and the output, so x and r are read once. (Rows that take 1024
// threads have 64 registers each: 16-bit rows above 32768 columns keep up to 24
// words a thread in local memory, FP32 rows above 16384 112 to 134. One CTA per
// SM there: FP32 1024 x 32768 176 us; with 32 registers, for two, 273.) 16384 x 8192 BF16:
// 138 us, 6.8 TB/s of the 940 MB it moves; what it took were 256-bit accesses,
// packed FP32 and 16-bit arithmetic (at twice the instructions the issue slots
// were 76 % busy and it took 168 us) and all loads in flight before the first store.
//
// kWide (rows and bases on 32 bytes, whole vectors): a vector is 32 bytes in a
// row, 8 (FP32: 16) neighbouring lanes make a scale group. Otherwise a warp
// takes the same columns with lane l holding columns l, l + 32, ...: every
// access is a coalesced one of single elements, and 4 elements of each lane
// make a group.
template <typename T, int kIters, bool kWide, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads, kMaxThreads == 1024 ? 1 : 0) rmsnorm_fp8_kernel(const NormParams p) {
  constexpr int VE = kVE<T>;
  __shared__ float warp_sum[32];
  grid_wait();
  grid_trigger();
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
  const T* res = p.residual ? static_cast<const T*>(p.residual) + row * p.res_ld : nullptr;
  T* out = p.residual_out ? static_cast<T*>(p.residual_out) + row * p.out_ld : nullptr;
  const int lane = threadIdx.x % 32;
  // First column of a vector, and the column of its element i.
  auto first = [&](int it) {
    const int unit = it * blockDim.x + threadIdx.x;
    return kWide ? unit * VE : (unit - lane) * VE + lane;
  };
  auto load = [&](const T* from, int c) {
    Vec<T> v;
    if constexpr (kWide) {
      v = load_vec(from + c);
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i) v.e[i] = c + 32 * i < p.cols ? from[c + 32 * i] : from_f32<T>(0.f);
    }
    return v;
  };
  // All loads of a thread before its first store: a store to residual_out may
  // alias what is still to be loaded as far as the compiler knows.
  Vec<T> v[kIters];
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int c = first(it);
    if (c < p.cols) v[it] = load(x, c);
  }
  if (res) {
    Vec<T> r[kIters];
#pragma unroll
    for (int it = 0; it < kIters; ++it) {
      const int c = first(it);
      if (c < p.cols) r[it] = load(res, c);
    }
#pragma unroll
    for (int it = 0; it < kIters; ++it) add_vec(v[it], r[it]);
  }
  F2 sum2 = pack2(0.f, 0.f);
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int c = first(it);
    if (c < p.cols) {
      if (out) {
        if constexpr (kWide) {
          store_vec(out + c, v[it]);
        } else {
#pragma unroll
          for (int i = 0; i < VE; ++i)
            if (c + 32 * i < p.cols) out[c + 32 * i] = v[it].e[i];
        }
      }
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const F2 h = pair_f32(v[it], i);
        sum2 = fma2(h, h, sum2);
      }
    }
  }
  // The CTA's sum, the same in every thread.
  auto block_sum = [&](F2 of_thread) {
    float sum, odd;
    unpack2(of_thread, sum, odd);
    sum += odd;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) warp_sum[threadIdx.x / 32] = sum;
    __syncthreads();
    sum = lane < blockDim.x / 32 ? warp_sum[lane] : 0.f;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    return sum;
  };
  float var = block_sum(sum2) / static_cast<float>(p.cols) + p.eps;
  float rstd = rsqrtf(var);
  // Squares that leave FP32's range, or sink below 2^-100 where eps does not
  // cover them, are taken again of h times a power of two. FP16's stay inside.
  // Small rows keep the factor, since 1 / rms may be no FP32 number. (NaN and
  // infinite rows come here too and stay what they are.)
  if (!std::is_same_v<T, __half> && !(var >= 0x1p-100f && var < __int_as_float(0x7f800000))) {
    const bool small = var < 1.f;
    const float f = small ? 0x1p100f : 0x1p-80f;
    const F2 f2 = pack2(f, f);
    sum2 = pack2(0.f, 0.f);
#pragma unroll
    for (int it = 0; it < kIters; ++it) {
      if (first(it) < p.cols) {
#pragma unroll
        for (int i = 0; i < VE / 2; ++i) {
          const F2 h = mul2(pair_f32(v[it], i), f2);
          sum2 = fma2(h, h, sum2);
          if (small) {
            float lo, hi;
            unpack2(h, lo, hi);
            v[it].e[2 * i] = from_f32<T>(lo);  // exact
            v[it].e[2 * i + 1] = from_f32<T>(hi);
          }
        }
      }
    }
    __syncthreads();  // the first sum has been read
    var = block_sum(sum2) / static_cast<float>(p.cols) + p.eps * f * f;
    rstd = small ? rsqrtf(var) : rsqrtf(var) * f;
  }
  const F2 rstd2 = pack2(rstd, rstd);
#pragma unroll
  for (int it = 0; it < kIters; ++it) {
    const int c = first(it);
    const bool has = c < p.cols;
    float y[VE];
#pragma unroll
    for (int i = 0; i < VE; ++i) y[i] = 0.f;
    if (has) {
      if constexpr (kWide) {
        if (p.weight_f32) {
          const float* w = static_cast<const float*>(p.weight) + c;
#pragma unroll
          for (int j = 0; j < VE / 8; ++j) {
            const Vec<float> f = load_vec(w + 8 * j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = 8 * j + 2 * i;
              unpack2(mul2(mul2(pair_f32(v[it], at / 2), rstd2), pair_f32(f, i)), y[at], y[at + 1]);
            }
          }
        } else {
          const Vec<T> w = load_vec(static_cast<const T*>(p.weight) + c);
#pragma unroll
          for (int i = 0; i < VE / 2; ++i)
            unpack2(mul2(mul2(pair_f32(v[it], i), rstd2), pair_f32(w, i)), y[2 * i], y[2 * i + 1]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          if (c + 32 * i >= p.cols) continue;
          const float w = p.weight_f32 ? static_cast<const float*>(p.weight)[c + 32 * i]
                                       : to_f32(static_cast<const T*>(p.weight)[c + 32 * i]);
          y[i] = to_f32(v[it].e[i]) * rstd * w;
        }
      }
    }
    // Scale groups of this thread's elements: one (wide), or one for every four elements.
    constexpr int kGroups = kWide ? 1 : VE / 4, kPer = VE / kGroups, kLanes = kWide ? 128 / VE : 32;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      float(&yg)[kPer] = *reinterpret_cast<float(*)[kPer]>(y + g * kPer);
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; i += 2) amax = max_abs(yg[i], yg[i + 1], amax);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, d));
      const int cg = kWide ? c : c - lane + 128 * g;  // wide: anywhere in the group; else its first column
      if (cg >= p.cols) continue;
      // 1 where the quotient is 0, which a group below 448 times the least FP32
      // number rounds to as well; a NaN stays.
      const float quotient = __fdiv_rn(amax, kE4m3Max);
      const float s = quotient == 0.f ? 1.f : quotient;
      if (lane % kLanes == 0) p.scales[(cg / 128) * p.s_ld + row] = s;
      // Rounded quotients here too: a product with the rounded reciprocal moves
      // two to four times as many values across a border of the E4M3 grid as
      // y's own roundings do (and saves 3 % at the power cap).
      divide(yg, s, amax);
    }
    if (!has) continue;
    union {
      __nv_fp8x2_storage_t h2[VE / 2];
      uint8_t b[VE];
      uint4 q4;
      uint2 q2;
    } o;
#pragma unroll
    for (int i = 0; i < VE / 2; ++i)
      o.h2[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    uint8_t* q = p.q + row * p.q_ld + c;
    if constexpr (kWide && VE == 16) {
      *reinterpret_cast<uint4*>(q) = o.q4;
    } else if constexpr (kWide) {
      *reinterpret_cast<uint2*>(q) = o.q2;
    } else {
#pragma unroll
      for (int i = 0; i < VE; ++i)
        if (c + 32 * i < p.cols) q[32 * i] = o.b[i];
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
  uint32_t* maxima;        // NVFP4 with a scale found by a launch of its own: the CTAs' maxima, or null
  unsigned* finished;      // CTAs that wrote theirs, 0 between launches
  float tensor_scale;      // NVFP4 with a given scale
  float* tensor_scale_out;
};

constexpr int kFp4Threads = 256;
// Vectors of x per thread up to which a CTA of the quantising launch finds the
// tensor scale by itself, in us against a launch of its own: BF16 1 x 4096 (one
// vector) 1.84 / 4.61, 4 x 4096 2.77 / 4.61, 8 x 4096 3.97 / 4.70, 12 x 4096
// 5.14 / 4.62; FP32 4 x 4096 (8 vectors) 3.56 / 4.96, 6 x 4096 4.47 / 4.89.
constexpr int64_t kFindInside = 8;
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

// max |e| of a vector; a NaN wins. The 16-bit types compare two at a time.
template <typename T>
__device__ __forceinline__ float absmax(const Vec<T>& v) {
  if constexpr (sizeof(T) == 4) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) m = max_abs(v.e[i], v.e[i + 1], m);
    return m;
  } else {
    uint32_t m = v.w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) {
      if constexpr (std::is_same_v<T, __half>)
        asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(m) : "r"(v.w[i] & 0x7fff7fffu));
      else
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v.w[i] & 0x7fff7fffu));
    }
    const T* e = reinterpret_cast<const T*>(&m);
    return max_abs(to_f32(e[0]), to_f32(e[1]), 0.f);
  }
}

// One vector, aligned or element by element.
template <bool kWide, typename T>
__device__ __forceinline__ Vec<T> get(const T* p) {
  if constexpr (kWide) {
    return load_vec(p);
  } else {
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < kVE<T>; ++i) v.e[i] = p[i];
    return v;
  }
}
template <bool kWide, typename T>
__device__ __forceinline__ void put(T* p, const Vec<T>& v) {
  if constexpr (kWide) {
    store_vec(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < kVE<T>; ++i) p[i] = v.e[i];
  }
}

// Maxima of |x| as bit patterns (those of non-negative floats order like the
// floats, a NaN above all): over a thread's part of the rows first, first +
// step, ..., and over a block.
template <typename T, bool kWide>
__device__ __forceinline__ uint32_t rows_max(const Fp4Params& p, int64_t first, int64_t step) {
  const int vecs = p.cols / kVE<T>;  // cols % 32 == 0
  uint32_t m = 0;
  for (int64_t row = first; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_ld;
#pragma unroll 4
    for (int v = threadIdx.x; v < vecs; v += kFp4Threads)
      m = max(m, __float_as_uint(absmax(get<kWide>(x + v * kVE<T>))) & 0x7fffffffu);
  }
  return m;
}
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* warp_max) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = v;
  __syncthreads();
  for (int i = 0; i < kFp4Threads / 32; ++i) v = max(v, warp_max[i]);
  return v;
}
__device__ __forceinline__ float scale_of_max(uint32_t m) {
  const float g = __fdiv_rn(__uint_as_float(m), kE4m3Max * kE2m1Max);
  return g > 0.f ? g : 1.f;  // no data, data below 2688 times the least FP32 number, or NaN
}

// The tensor scale of NVFP4: a maximum per CTA; the CTA that finishes last takes
// the maximum of all and writes the scale, so the quantising launch reads one word.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kFp4Threads) absmax_kernel(const Fp4Params p) {
  __shared__ uint32_t warp_max[kFp4Threads / 32];
  __shared__ bool last;
  grid_wait();
  grid_trigger();
  uint32_t m = block_max(rows_max<T, kWide>(p, blockIdx.x, gridDim.x), warp_max);
  if (threadIdx.x == 0) {
    p.maxima[blockIdx.x] = m;
    __threadfence();
    last = atomicInc(p.finished, gridDim.x - 1) == gridDim.x - 1;  // back to 0 for the next launch
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  m = 0;
  for (unsigned i = threadIdx.x; i < gridDim.x; i += blockDim.x) m = max(m, __ldcg(p.maxima + i));
  m = block_max(m, warp_max);
  if (threadIdx.x == 0) *p.tensor_scale_out = scale_of_max(m);
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
    if (p.maxima) {
      g = *p.tensor_scale_out;
    } else if (p.tensor_scale_out) {  // a small tensor: every CTA reads all of it
      __shared__ uint32_t warp_max[kFp4Threads / 32];
      g = scale_of_max(block_max(rows_max<T, kWide>(p, 0, 1), warp_max));
      if (blockIdx.x == 0 && threadIdx.x == 0) *p.tensor_scale_out = g;
    }
  }
  constexpr int kLanes = kMx ? 8 : 4;  // threads of one row's part of an atom
  const uint32_t per_row = static_cast<uint32_t>(p.atoms_k) * kLanes;
  // With a scale found by the launch before, the tensor is read a second time:
  // from its end, which is what L2 still holds of the first reading.
  const uint32_t block = p.maxima ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
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
    constexpr int VE = kVE<T>;
    Vec<T> e[16 / VE];
#pragma unroll
    for (int j = 0; j < 16 / VE; ++j) e[j] = get<kWide>(x + VE * j);
#pragma unroll
    for (int j = 0; j < 16 / VE; ++j) {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) unpack2(pair_f32(e[j], i), v[VE * j + 2 * i], v[VE * j + 2 * i + 1]);
      amax = max_nan(amax, absmax(e[j]));
    }
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
      constexpr int VE = kVE<T>;
      float q[16];
      e2m1x8_values(codes.x, q);
      e2m1x8_values(codes.y, q + 8);
#pragma unroll
      for (int j = 0; j < 16 / VE; ++j) {
        Vec<T> o;
#pragma unroll
        for (int i = 0; i < VE; ++i) {
          float f = q[VE * j + i] * unit;
          if constexpr (!kMx) f *= g;
          o.e[i] = from_f32<T>(f);
        }
        put<kWide>(out + VE * j, o);
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
  int threads = 0, iters = 0;  // RMS norm: vectors per thread, 0 for the widest rows
  int partials = 0;  // CTAs of the launch that finds the NVFP4 tensor scale
  int64_t launches = 0;
};

namespace {

size_t dtype_size(int dtype) { return dtype == BB_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype == BB_DTYPE_BF16 || dtype == BB_DTYPE_F32 || dtype == BB_DTYPE_F16; }
bool aligned(const void* p, int64_t ld, size_t size, size_t to) {
  return reinterpret_cast<uintptr_t>(p) % to == 0 && (static_cast<size_t>(ld) * size) % to == 0;
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
    case 1: return launch(rmsnorm_fp8_kernel<T, 1, kWide, 512>, grid, pl.threads, pl.stream, pl.np);
    case 2: return launch(rmsnorm_fp8_kernel<T, 2, kWide, 512>, grid, pl.threads, pl.stream, pl.np);
    case 4: return launch(rmsnorm_fp8_kernel<T, 4, kWide, 512>, grid, pl.threads, pl.stream, pl.np);
    default: return launch(rmsnorm_fp8_kernel<T, 64 / kVE<T>, kWide, 1024>, grid, pl.threads, pl.stream, pl.np);
  }
}

template <typename T, bool kWide>
cudaError_t launch_fp4(const bb_quant_plan& pl) {
  const bool mx = pl.fmt == BB_LOWP_MXFP4;
  if (pl.partials) {
    const cudaError_t e = launch(absmax_kernel<T, kWide>, pl.partials, kFp4Threads, pl.stream, pl.fp);
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
    h->wide = aligned(x, rows > 1 ? x_ld : 0, size, 32) && (!values || aligned(values, rows > 1 ? values_ld : 0, size, 32));
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
    // A small tensor's scale is found by every CTA of the quantising launch
    // itself, a larger one's by a launch of its own; also where `values` is
    // written, which may be x: a CTA would overwrite what another still reads.
    const int64_t per_thread = (cols * static_cast<int64_t>(size) / 32 + kFp4Threads - 1) / kFp4Threads;
    if (find && rows > 0 && (values || rows * per_thread > kFindInside)) {
      const int64_t most = 8ll * dev.sm_count < kMaxPartials ? 8ll * dev.sm_count : kMaxPartials;
      h->partials = static_cast<int>(rows < most ? rows : most);
      const size_t bytes = (h->partials + 1) * sizeof(uint32_t);
      rc = device_zeros(reinterpret_cast<void**>(&p.maxima), bytes, "allocation of the maxima");
      if (rc != BB_OK) {
        if (p.maxima) cudaFree(p.maxima);
        delete h;
        return rc;
      }
      p.finished = p.maxima + h->partials;
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
    if (rows < 0 || rows > (int64_t(1) << 30) || cols <= 0 || cols > kNormMaxCols) {
      set_error("bb_rmsnorm_fp8_plan_create: rows=%lld must lie in [0, 2^30], cols=%lld in [1, %lld]", (long long)rows,
                (long long)cols, (long long)kNormMaxCols);
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
    auto wide = [&](const void* ptr, int64_t ld, size_t sz, size_t to) { return aligned(ptr, rows > 1 ? ld : 0, sz, to); };
    const int64_t ve = 32 / size;
    h->wide = cols % ve == 0 && wide(x, x_ld, size, 32) && (!residual || wide(residual, residual_ld, size, 32)) &&
              (!residual_out || wide(residual_out, residual_out_ld, size, 32)) && wide(weight, 0, wsize, 32) &&
              wide(q, q_ld, 1, ve);
    // One vector per thread as far as 512 threads go, then two, four; the
    // widest rows with 1024 threads. More vectors per thread were slower at
    // every size (BF16: 1 x 4096 1.9 / 2.4 / 3.7 us with one / two / four,
    // 16384 x 8192 137.9 / 139.3 / 141.8 us).
    const int64_t vecs = (cols + ve - 1) / ve;
    const int64_t widest = 64 / ve;
    const int64_t per = vecs <= 512 ? 1 : vecs <= 1024 ? 2 : vecs <= 2048 ? 4 : widest;
    h->iters = vecs <= 2048 ? static_cast<int>(per) : 0;
    h->threads = static_cast<int>(((vecs + per - 1) / per + 31) / 32 * 32);
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
  DeviceGuard guard(plan->device);  // the default stream is the current device's
  if (guard.status != cudaSuccess) return check_cuda(guard.status, "cudaSetDevice");
  return check_cuda(cudaStreamSynchronize(plan->stream), "cudaStreamSynchronize");
}

BB_API int64_t bb_quant_launches(const bb_quant_plan* plan) { return plan ? plan->launches : -1; }

BB_API int bb_quant_destroy(bb_quant_plan* plan) {
  if (!plan) return BB_OK;
  int rc = BB_OK;
  if (plan->fp.maxima) rc = check_cuda(cudaFree(plan->fp.maxima), "cudaFree(maxima)");
  delete plan;
  return rc;
}

}  // extern "C"
