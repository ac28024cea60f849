// The product of a quantised linear layer, D (M x N) = dequant(A) * dequant(B)^T,
// for any number of rows (bb_linear_*): NVFP4, MXFP4, and FP8 with activations
// scaled per row and 128 K elements and weights per 128 x 128 block.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <new>

#include "common.cuh"
#include "ptx.cuh"

namespace bb {
extern std::atomic<int64_t> g_kernel_launches;

namespace linear {

struct SimpleParams {
  int32_t m, n, k, atoms_k;
  const uint8_t* a;
  const uint8_t* b;
  const uint8_t* sfa;
  const uint8_t* sfb;
  int64_t sfa_ld, ldd;
  float scale_a, scale_b;
  const float* scale_a_dev;
  const float* scale_b_dev;
  void* d;
  int32_t d_dtype;
};

__device__ __forceinline__ float e2m1(uint32_t code) {
  const uint32_t e = (code >> 1) & 3u, m = code & 1u;
  const float mag = e == 0 ? 0.5f * m : __uint_as_float((126u + e) << 23 | m << 22);
  return (code & 8u) ? -mag : mag;
}
__device__ __forceinline__ float e4m3(uint8_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(b, __NV_E4M3)));
}
__device__ __forceinline__ float e8m0(uint8_t b) {
  return b == 255 ? __uint_as_float(0x7fc00000u) : b ? __uint_as_float(static_cast<uint32_t>(b) << 23) : 0x1p-127f;
}
__device__ __forceinline__ uint8_t atom_byte(const uint8_t* atoms, int row, int atoms_k, int j) {
  const int r = row % 128;
  return atoms[(static_cast<int64_t>(row / 128) * atoms_k + j / 4) * 512 + (r % 32) * 16 + (r / 32) * 4 + j % 4];
}

// 64 x 64 outputs per block of 256 threads, 32 K elements at a time dequantised into shared memory.
template <int kKind>
__global__ void __launch_bounds__(256) simple_linear_kernel(const SimpleParams p) {
  __shared__ float sa[32][65], sb[32][65];
  const int tiles_n = (p.n + 63) / 64;
  const int m0 = blockIdx.x / tiles_n * 64, n0 = blockIdx.x % tiles_n * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  const int kb = (p.k + 127) / 128;
  auto value = [&](bool weights, int row, int k) -> float {
    if (row >= (weights ? p.n : p.m) || k >= p.k) return 0.f;
    const uint8_t* v = weights ? p.b : p.a;
    const uint8_t* s = weights ? p.sfb : p.sfa;
    if constexpr (kKind == BB_LOWP_FP8_GROUP128) {
      const float* f = reinterpret_cast<const float*>(s);
      const float scale = weights ? f[static_cast<int64_t>(row / 128) * kb + k / 128] : f[(k / 128) * p.sfa_ld + row];
      return e4m3(v[static_cast<int64_t>(row) * p.k + k]) * scale;
    } else {
      const uint8_t byte = v[static_cast<int64_t>(row) * (p.k / 2) + k / 2];
      const float q = e2m1(k % 2 ? byte >> 4 : byte & 15u);
      if constexpr (kKind == BB_LOWP_MXFP4) return q * e8m0(atom_byte(s, row, p.atoms_k, k / 32));
      return q * e4m3(atom_byte(s, row, p.atoms_k, k / 16));
    }
  };
  for (int k0 = 0; k0 < p.k; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      sa[i % 32][i / 32] = value(false, m0 + i / 32, k0 + i % 32);
      sb[i % 32][i / 32] = value(true, n0 + i / 32, k0 + i % 32);
    }
    __syncthreads();
    for (int k = 0; k < 32; ++k)
      for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + 16 * i], sb[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  const float g = (p.scale_a_dev ? *p.scale_a_dev : p.scale_a) * (p.scale_b_dev ? *p.scale_b_dev : p.scale_b);
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (m >= p.m || n >= p.n) continue;
      const int64_t at = m * p.ldd + n;
      const float v = acc[i][j] * g;
      if (p.d_dtype == BB_DTYPE_BF16) static_cast<__nv_bfloat16*>(p.d)[at] = __float2bfloat16_rn(v);
      else if (p.d_dtype == BB_DTYPE_F16) static_cast<__half*>(p.d)[at] = __float2half_rn(v);
      else static_cast<float*>(p.d)[at] = v;
    }
}

}  // namespace linear
}  // namespace bb

using namespace bb;
using namespace bb::linear;

struct bb_linear_plan {
  int kind = 0, device = 0;
  cudaStream_t stream = nullptr;
  SimpleParams params{};
  int* status_dev = nullptr;
  int64_t launches = 0;
};

extern "C" {

BB_API int64_t bb_linear_scale_bytes(int kind, int weights, int64_t rows, int64_t k) {
  if (rows < 0 || k <= 0) return -1;
  const int64_t rb = (rows + 127) / 128, kb = (k + 127) / 128;
  if (kind == BB_LOWP_NVFP4) return k % 32 ? -1 : rb * ((k + 63) / 64) * 512;
  if (kind == BB_LOWP_MXFP4) return k % 32 ? -1 : rb * kb * 512;
  if (kind == BB_LOWP_FP8_GROUP128) return k % 16 ? -1 : (weights ? rb : rows) * kb * 4;
  return -1;
}

BB_API int bb_linear_plan_create(int kind, int64_t m, int64_t n, int64_t k, const void* a, const void* b,
                                 const void* sfa, int64_t sfa_ld, const void* sfb, float scale_a,
                                 const float* scale_a_dev, float scale_b, const float* scale_b_dev, void* d,
                                 int d_dtype, int64_t ldd, void* stream, bb_linear_plan** plan, bb_lowp_info* info) {
  try {
    clear_error();
    if (!plan) {
      set_error("bb_linear_plan_create: plan out-pointer is null");
      return BB_ERR_ARGUMENT;
    }
    *plan = nullptr;
    if (kind != BB_LOWP_NVFP4 && kind != BB_LOWP_MXFP4 && kind != BB_LOWP_FP8_GROUP128) {
      set_error("bb_linear_plan_create: unknown kind %d", kind);
      return BB_ERR_ARGUMENT;
    }
    if (d_dtype != BB_DTYPE_BF16 && d_dtype != BB_DTYPE_F16 && d_dtype != BB_DTYPE_F32) {
      set_error("bb_linear_plan_create: unknown dtype %d of D", d_dtype);
      return BB_ERR_ARGUMENT;
    }
    const int64_t most = int64_t(1) << 24;
    if (m < 0 || n <= 0 || k <= 0 || m > most || n > most || k > most) {
      set_error("bb_linear_plan_create: extents out of range (m=%lld n=%lld k=%lld, each up to 2^24)", (long long)m,
                (long long)n, (long long)k);
      return BB_ERR_ARGUMENT;
    }
    const bool fp8 = kind == BB_LOWP_FP8_GROUP128;
    if (k % (fp8 ? 16 : 32) != 0) {
      set_error("bb_linear_plan_create: K=%lld must be a multiple of %d for this kind", (long long)k, fp8 ? 16 : 32);
      return BB_ERR_ARGUMENT;
    }
    if (!b || !sfb || (m > 0 && (!a || !sfa || !d))) {
      set_error("bb_linear_plan_create: null operand pointer");
      return BB_ERR_ARGUMENT;
    }
    if (m > 0 && (ldd < n || (fp8 && sfa_ld < m))) {
      set_error("bb_linear_plan_create: ldd=%lld below N or sfa_ld=%lld below M", (long long)ldd, (long long)sfa_ld);
      return BB_ERR_ARGUMENT;
    }
    auto off = [](const void* ptr, size_t to) { return reinterpret_cast<uintptr_t>(ptr) % to != 0; };
    if (off(a, 16) || off(b, 16) || off(sfa, fp8 ? 4 : 16) || off(sfb, fp8 ? 4 : 16) ||
        off(d, d_dtype == BB_DTYPE_F32 ? 4 : 2) || off(scale_a_dev, 4) || off(scale_b_dev, 4)) {
      set_error("bb_linear_plan_create: operands must be 16-byte aligned (FP8 scales 4), D to its type");
      return BB_ERR_ARGUMENT;
    }
    if (((m + 63) / 64) * ((n + 63) / 64) > 0x7fffffff) {
      set_error("bb_linear_plan_create: M=%lld x N=%lld is more than one launch covers", (long long)m, (long long)n);
      return BB_ERR_ARGUMENT;
    }
    DeviceInfo dev;
    int rc = query_device(&dev);
    if (rc != BB_OK) return rc;
    auto* h = new (std::nothrow) bb_linear_plan();
    if (!h) {
      set_error("bb_linear_plan_create: out of host memory");
      return BB_ERR_INTERNAL;
    }
    h->kind = kind;
    h->device = dev.device;
    h->stream = static_cast<cudaStream_t>(stream);
    SimpleParams& p = h->params;
    p.m = static_cast<int32_t>(m);
    p.n = static_cast<int32_t>(n);
    p.k = static_cast<int32_t>(k);
    p.atoms_k = static_cast<int32_t>(kind == BB_LOWP_NVFP4 ? (k + 63) / 64 : (k + 127) / 128);
    p.a = static_cast<const uint8_t*>(a);
    p.b = static_cast<const uint8_t*>(b);
    p.sfa = static_cast<const uint8_t*>(sfa);
    p.sfb = static_cast<const uint8_t*>(sfb);
    p.sfa_ld = sfa_ld;
    p.ldd = ldd;
    p.scale_a = scale_a;
    p.scale_b = scale_b;
    p.scale_a_dev = scale_a_dev;
    p.scale_b_dev = scale_b_dev;
    p.d = d;
    p.d_dtype = d_dtype;
    if (info) {
      *info = bb_lowp_info{};
      info->kind = kind;
      info->tile_m = 64;
      info->tile_n = 64;
      info->tile_k = 32;
      info->threads_per_cta = 256;
      info->num_tiles = ((m + 63) / 64) * ((n + 63) / 64);
      info->grid_ctas = info->num_tiles;
    }
    *plan = h;
    return BB_OK;
  } catch (...) {
    set_error("bb_linear_plan_create: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_linear_execute_n(bb_linear_plan* plan, int iterations) {
  try {
    if (!plan || iterations < 0) {
      set_error("bb_linear_execute_n: null plan or negative iteration count");
      return BB_ERR_ARGUMENT;
    }
    const SimpleParams& p = plan->params;
    if (p.m == 0) return BB_OK;
    DeviceGuard guard(plan->device);
    BB_CUDA_TRY(guard.status);
    for (int i = 0; i < iterations; ++i) {
      const unsigned grid = static_cast<unsigned>((p.n + 63) / 64) * ((p.m + 63) / 64);
      if (plan->kind == BB_LOWP_NVFP4) simple_linear_kernel<BB_LOWP_NVFP4><<<grid, 256, 0, plan->stream>>>(p);
      else if (plan->kind == BB_LOWP_MXFP4) simple_linear_kernel<BB_LOWP_MXFP4><<<grid, 256, 0, plan->stream>>>(p);
      else simple_linear_kernel<BB_LOWP_FP8_GROUP128><<<grid, 256, 0, plan->stream>>>(p);
      int rc = check_cuda(cudaGetLastError(), "launch simple_linear_kernel");
      if (rc != BB_OK) return rc;
      ++plan->launches;
      g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    }
    return BB_OK;
  } catch (...) {
    set_error("bb_linear_execute_n: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_linear_synchronize(bb_linear_plan* plan) {
  if (!plan) {
    set_error("bb_linear_synchronize: null plan");
    return BB_ERR_ARGUMENT;
  }
  return check_cuda(cudaStreamSynchronize(plan->stream), "cudaStreamSynchronize");
}

BB_API int64_t bb_linear_launches(const bb_linear_plan* plan) { return plan ? plan->launches : -1; }

BB_API int bb_linear_destroy(bb_linear_plan* plan) {
  delete plan;
  return BB_OK;
}

}  // extern "C"
