// Block-scaled low-precision GEMMs for sm_100a (FP8 128 x 128-block, NVFP4):
// plans and C ABI (bb_lowp_*) of the kernel in gemm_lowp.cuh.
#include <cstdlib>
#include <new>

#include "gemm_lowp.cuh"

struct bb_lowp_plan {
  int kind = 0;
  int cg = 1;
  int tile_n = 256;
  int stages = 0;
  int64_t m = 0, n = 0, k = 0;
  cudaStream_t stream = nullptr;
  CUtensorMap tm_a{}, tm_b{}, tm_sfa{}, tm_sfb{}, tm_d{};
  bb::lowp::Params params{};
  int grid = 0;
  int smem_bytes = 0;
  int* status_dev = nullptr;
  int64_t launches = 0;
};

using namespace bb;
using namespace bb::lowp;

namespace {

template <int kKind, int kCG>
cudaLaunchConfig_t launch_config(const bb_lowp_plan& pl, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(pl.grid);
  cfg.blockDim = dim3(Cfg<kKind, kCG>::THREADS);
  cfg.dynamicSmemBytes = Cfg<kKind, kCG>::SMEM_BYTES;
  cfg.stream = pl.stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

template <int kKind, int kCG>
int set_attributes() {
  static bool done = false;  // one attribute call per kernel and process
  if (!done) {
    if constexpr (Cfg<kKind, kCG>::kRegSplit) {
      // setmaxnreg.inc waits until the block's register pool can serve it;
      // refuse to launch a build whose pool is smaller than the split needs.
      cudaFuncAttributes fa{};
      BB_CUDA_TRY(cudaFuncGetAttributes(&fa, bb_lowp_gemm_kernel<kKind, kCG>));
      if (fa.numRegs * Cfg<kKind, kCG>::THREADS < 128 * Cfg<kKind, kCG>::CTRL_REGS + 256 * Cfg<kKind, kCG>::EPI_REGS) {
        set_error("bb_lowp: kernel built with %d registers per thread; its register split needs %d", fa.numRegs,
                  kLaunchRegs);
        return BB_ERR_INTERNAL;
      }
    }
    BB_CUDA_TRY(cudaFuncSetAttribute(bb_lowp_gemm_kernel<kKind, kCG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Cfg<kKind, kCG>::SMEM_BYTES));
    done = true;
  }
  return BB_OK;
}

template <int kKind, int kCG>
int launch_kind(const bb_lowp_plan& pl) {
  int rc = set_attributes<kKind, kCG>();
  if (rc != BB_OK) return rc;
  cudaLaunchAttribute attr[1];
  cudaLaunchConfig_t cfg = launch_config<kKind, kCG>(pl, attr);
  return check_cuda(cudaLaunchKernelEx(&cfg, bb_lowp_gemm_kernel<kKind, kCG>, pl.tm_a, pl.tm_b, pl.tm_sfa, pl.tm_sfb,
                                       pl.tm_d, pl.params),
                    "launch bb_lowp_gemm_kernel");
}

int launch(const bb_lowp_plan& pl) {
  if (pl.kind == kNvfp4) return pl.cg == 2 ? launch_kind<kNvfp4, 2>(pl) : launch_kind<kNvfp4, 1>(pl);
  return pl.cg == 2 ? launch_kind<kFp8Block, 2>(pl) : launch_kind<kFp8Block, 1>(pl);
}

// Clusters of kCG CTAs resident at once (one CTA per SM: the shared-memory
// ring takes the whole SM).
template <int kKind, int kCG>
int max_clusters(const bb_lowp_plan& pl, int sm_count) {
  int clusters = sm_count / kCG;
  if (kCG > 1 && set_attributes<kKind, kCG>() == BB_OK) {
    bb_lowp_plan probe = pl;
    probe.grid = kCG * clusters;
    cudaLaunchAttribute attr[1];
    cudaLaunchConfig_t cfg = launch_config<kKind, kCG>(probe, attr);
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, bb_lowp_gemm_kernel<kKind, kCG>, &cfg) == cudaSuccess && n > 0) {
      clusters = n;
    } else {
      cudaGetLastError();
    }
  }
  return clusters;
}

template <int kKind, int kCG>
void plan_geometry(bb_lowp_plan& h, int sm_count) {
  using C = Cfg<kKind, kCG>;
  h.stages = C::STAGES;
  h.tile_n = C::TILE_N;
  h.smem_bytes = C::SMEM_BYTES;
  Params& p = h.params;
  p.tiles_m = static_cast<int32_t>((h.m + C::TILE_M - 1) / C::TILE_M);
  p.tiles_n = static_cast<int32_t>((h.n + C::TILE_N - 1) / C::TILE_N);
  p.num_tiles = p.tiles_m * p.tiles_n;
  const int64_t a_tile_bytes = static_cast<int64_t>(C::TILE_M) * (kKind == kNvfp4 ? h.k / 2 : h.k);
  const int64_t g = kGroupABytes / (a_tile_bytes > 0 ? a_tile_bytes : 1);
  p.group_m = static_cast<int32_t>(g < 1 ? 1 : (g > p.tiles_m ? p.tiles_m : g));
  const int clusters = max_clusters<kKind, kCG>(h, sm_count);
  p.num_clusters = p.num_tiles < clusters ? p.num_tiles : clusters;
  h.grid = p.num_clusters * kCG;
}

}  // namespace

extern "C" {

BB_API size_t bb_lowp_info_size(void) { return sizeof(bb_lowp_info); }

BB_API int64_t bb_lowp_scale_bytes(int kind, int64_t rows, int64_t k) {
  if (rows <= 0 || k <= 0) return -1;
  const int64_t rb = (rows + 127) / 128;
  if (kind == BB_LOWP_NVFP4) return k % 64 ? -1 : rb * (k / 64) * 512;
  if (kind == BB_LOWP_FP8_BLOCK128) return k % 128 ? -1 : rb * (k / 128) * 4;
  return -1;
}

BB_API int bb_lowp_plan_create(int kind, int64_t m, int64_t n, int64_t k, const void* a, const void* b,
                               const void* sfa, const void* sfb, float global_scale, void* d, void* stream,
                               bb_lowp_plan** plan, bb_lowp_info* info) {
  try {
    clear_error();
    if (!plan) {
      set_error("bb_lowp_plan_create: plan out-pointer is null");
      return BB_ERR_ARGUMENT;
    }
    *plan = nullptr;
    if (kind != BB_LOWP_NVFP4 && kind != BB_LOWP_FP8_BLOCK128) {
      set_error("bb_lowp_plan_create: unknown kind %d", kind);
      return BB_ERR_ARGUMENT;
    }
    if (!a || !b || !sfa || !sfb || !d) {
      set_error("bb_lowp_plan_create: null operand pointer");
      return BB_ERR_ARGUMENT;
    }
    if (m <= 0 || n <= 0 || k <= 0 || m > (int64_t(1) << 30) || n > (int64_t(1) << 30) || k > (int64_t(1) << 30)) {
      set_error("bb_lowp_plan_create: extents out of range (m=%lld n=%lld k=%lld)", (long long)m, (long long)n,
                (long long)k);
      return BB_ERR_ARGUMENT;
    }
    const int k_step = kind == BB_LOWP_NVFP4 ? 256 : 128;
    if (k % k_step != 0) {
      set_error("bb_lowp_plan_create: K=%lld must be a multiple of %d for this kind", (long long)k, k_step);
      return BB_ERR_ARGUMENT;
    }
    if (n % 8 != 0) {
      set_error("bb_lowp_plan_create: N=%lld must be a multiple of 8 (16-byte rows of D)", (long long)n);
      return BB_ERR_ARGUMENT;
    }
    for (const void* ptr : {a, b, sfa, sfb, static_cast<const void*>(d)}) {
      if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0) {
        set_error("bb_lowp_plan_create: every buffer must be 16-byte aligned");
        return BB_ERR_ARGUMENT;
      }
    }
    DeviceInfo dev;
    int rc = query_device(&dev);
    if (rc != BB_OK) return rc;
    if (dev.major != 10) {
      set_error("bb_lowp_plan_create: needs an sm_100 device (found sm_%d%d)", dev.major, dev.minor);
      return BB_ERR_UNSUPPORTED;
    }
    auto* h = new (std::nothrow) bb_lowp_plan();
    if (!h) {
      set_error("bb_lowp_plan_create: out of host memory");
      return BB_ERR_INTERNAL;
    }
    h->kind = kind;
    h->m = m;
    h->n = n;
    h->k = k;
    h->stream = static_cast<cudaStream_t>(stream);
    // CTA pairs (256-row tiles) unless A has a single 128-row block. For
    // FP8 the pair is the only shape that can approach the tensor rate: a
    // single CTA's 128 x 256 tile moves 96 KiB of shared memory per 128-K
    // block (48 KiB of TMA writes, 48 KiB of MMA operand reads) against the
    // pair's 64 KiB, i.e. about 750 against 500 clocks at 128 B/clock for
    // 512 clocks of MMA. The pair's price is its per-block accumulator
    // hand-off across the CTAs (8192^3: pair 2320-2377, single 2200-2250
    // TFLOP/s). BB_LOWP_CTA_GROUP=1|2 forces one.
    h->cg = m > 128 ? 2 : 1;
    if (const char* env = std::getenv("BB_LOWP_CTA_GROUP")) {
      if (env[0] == '1') h->cg = 1;
      if (env[0] == '2') h->cg = 2;
    }
    if (kind == kNvfp4) {
      if (h->cg == 2) plan_geometry<kNvfp4, 2>(*h, dev.sm_count); else plan_geometry<kNvfp4, 1>(*h, dev.sm_count);
    } else {
      if (h->cg == 2) plan_geometry<kFp8Block, 2>(*h, dev.sm_count); else plan_geometry<kFp8Block, 1>(*h, dev.sm_count);
    }
    // Operands are byte arrays: K / 2 bytes per row for E2M1, K for E4M3.
    const uint64_t row_bytes = kind == BB_LOWP_NVFP4 ? k / 2 : k;
    const uint64_t rb_m = (m + 127) / 128, rb_n = (n + 127) / 128;
    {
      const uint64_t dims[2] = {row_bytes, static_cast<uint64_t>(m)};
      const uint64_t strides[1] = {row_bytes};
      const uint32_t box[2] = {ROW_BYTES, BM};
      rc = encode_tiled(&h->tm_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 2, a, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    if (rc == BB_OK) {
      const uint64_t dims[2] = {row_bytes, static_cast<uint64_t>(n)};
      const uint64_t strides[1] = {row_bytes};
      const uint32_t box[2] = {ROW_BYTES, static_cast<uint32_t>(h->tile_n / h->cg)};
      rc = encode_tiled(&h->tm_b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 2, b, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
    }
    if (rc == BB_OK && kind == BB_LOWP_NVFP4) {
      // Scale atoms viewed as rows of 8-byte words, one row per 128-row block
      // (K words: K/64 atoms of 64 words); a stage's box is 256 words (4 atoms).
      const uint64_t strides[1] = {static_cast<uint64_t>(k) * 8};
      const uint64_t dims_a[2] = {static_cast<uint64_t>(k), rb_m};
      const uint32_t box_a[2] = {256, 1};
      rc = encode_tiled(&h->tm_sfa, CU_TENSOR_MAP_DATA_TYPE_UINT64, 8, 2, sfa, dims_a, strides, box_a,
                        CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
      if (rc == BB_OK) {
        const uint64_t dims_b[2] = {static_cast<uint64_t>(k), rb_n};
        const uint32_t box_b[2] = {256, 2};
        rc = encode_tiled(&h->tm_sfb, CU_TENSOR_MAP_DATA_TYPE_UINT64, 8, 2, sfb, dims_b, strides, box_b,
                          CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
      }
    } else {
      h->tm_sfa = h->tm_a;  // unused by the FP8 kernel
      h->tm_sfb = h->tm_b;
    }
    if (rc == BB_OK) {
      // D (M x N BF16, row-major) for the epilogue's TMA stores: boxes of 64
      // columns (128 bytes) x 32 rows, 128-byte swizzle.
      const uint64_t dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)};
      const uint64_t strides[1] = {static_cast<uint64_t>(n) * 2};
      const uint32_t box[2] = {64, 32};
      rc = encode_tiled(&h->tm_d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 2, d, dims, strides, box,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
    }
    if (rc == BB_OK) rc = check_cuda(cudaMalloc(&h->status_dev, sizeof(int)), "cudaMalloc(status)");
    if (rc == BB_OK) rc = check_cuda(cudaMemset(h->status_dev, 0, sizeof(int)), "cudaMemset(status)");
    if (rc != BB_OK) {
      if (h->status_dev) cudaFree(h->status_dev);
      delete h;
      return rc;
    }
    Params& p = h->params;
    p.m = static_cast<int32_t>(m);
    p.n = static_cast<int32_t>(n);
    p.k = static_cast<int32_t>(k);
    p.k_stages = static_cast<int32_t>(k / k_step);
    p.rb_m = static_cast<int32_t>(rb_m);
    p.rb_n = static_cast<int32_t>(rb_n);
    p.sfa = static_cast<const uint8_t*>(sfa);
    p.sfb = static_cast<const uint8_t*>(sfb);
    p.global_scale = global_scale;
    p.d = static_cast<__nv_bfloat16*>(d);
    p.status = h->status_dev;
    if (info) {
      info->kind = kind;
      info->tile_m = 128 * h->cg;
      info->tile_n = h->tile_n;
      info->tile_k = k_step;
      info->stages = h->stages;
      info->grid_ctas = h->grid;
      info->num_tiles = p.num_tiles;
      info->smem_bytes = h->smem_bytes;
      info->tmem_columns = TMEM_COLS;
      info->threads_per_cta = kind == BB_LOWP_NVFP4 ? Cfg<kNvfp4, 1>::THREADS : Cfg<kFp8Block, 1>::THREADS;
      info->cta_group = h->cg;
      for (int i = 0; i < 5; ++i) info->reserved[i] = 0;
    }
    *plan = h;
    return BB_OK;
  } catch (...) {
    set_error("bb_lowp_plan_create: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_lowp_execute_n(bb_lowp_plan* plan, int iterations) {
  try {
    if (!plan) {
      set_error("bb_lowp_execute_n: null plan");
      return BB_ERR_ARGUMENT;
    }
    if (iterations < 0) {
      set_error("bb_lowp_execute: negative iteration count %d", iterations);
      return BB_ERR_ARGUMENT;
    }
    for (int i = 0; i < iterations; ++i) {
      int rc = launch(*plan);
      if (rc != BB_OK) return rc;
      ++plan->launches;
      g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    }
    return BB_OK;
  } catch (...) {
    set_error("bb_lowp_execute_n: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int bb_lowp_synchronize(bb_lowp_plan* plan) {
  try {
    if (!plan) {
      set_error("bb_lowp_synchronize: null plan");
      return BB_ERR_ARGUMENT;
    }
    BB_CUDA_TRY(cudaStreamSynchronize(plan->stream));
    int st = 0;
    BB_CUDA_TRY(cudaMemcpy(&st, plan->status_dev, sizeof(int), cudaMemcpyDeviceToHost));
    if (st != 0) {
      set_error("block-scaled GEMM kernel reported device status 0x%x (%s)", st,
                st == 0x200 ? "launch contract violated" : "a bounded wait timed out");
      return st == 0x200 ? BB_ERR_INTERNAL : BB_ERR_TIMEOUT;
    }
    return BB_OK;
  } catch (...) {
    set_error("bb_lowp_synchronize: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int64_t bb_lowp_launches(const bb_lowp_plan* plan) { return plan ? plan->launches : -1; }

BB_API int bb_lowp_destroy(bb_lowp_plan* plan) {
  if (!plan) return BB_OK;
  int rc = BB_OK;
  if (plan->status_dev) {
    cudaError_t e = cudaFree(plan->status_dev);
    if (e != cudaSuccess) rc = check_cuda(e, "cudaFree(status)");
  }
  delete plan;
  return rc;
}

}  // extern "C"
