// The block-scaled low-precision GEMM kernel for sm_100a:
//   D (M x N, BF16) = dequant(A) (M x K) * dequant(B)^T (N x K), FP32 accumulate.
//
// Operand formats of one persistent warp-specialised kernel:
//
//   NVFP4  A, B: E2M1 packed two per byte (element 2i in the low nibble),
//          K-major; one UE4M3 scale per 16 K elements of each row, stored
//          as 512-byte scale atoms (128 rows x 4 scales; scale j of row r
//          at byte (r % 32) * 16 + (r / 32) * 4 + j), atoms ordered
//          [row block][K / 64]; a per-tensor FP32 scale (product of A's and
//          B's) applied in the epilogue. The scales are applied by the tensor
//          core itself: tcgen05.mma.kind::mxf4nvf4.block_scale.block16 reads
//          them from TMEM, where tcgen05.cp.32x128b.warpx4 places each atom.
//
//   FP8    A, B: E4M3, K-major; one FP32 scale per 128 x 128 block of each
//          operand. FP32 scales cannot be applied by the tensor core, so every
//          128-wide K block is accumulated on its own (tcgen05.mma.kind::f8f6f4
//          into one of two TMEM partial buffers) and promoted by the epilogue
//          warps into FP32 registers: acc += partial * sa[m][kb] * sb[n][kb].
//          The MMA of K block kb+1 overlaps the promotion of kb.
//
//   MXFP4  A, B: E2M1 as for NVFP4; one E8M0 scale per 32 K elements in the
//          same atoms (128 K elements each), applied by
//          tcgen05.mma.kind::mxf4.block_scale.block32; no tensor scale.
//
//   FP8 by group (activations)  A's FP32 scales are per row and 128 K
//          elements, stored [K block][row]: the promotion's scale then differs
//          by lane, and one coalesced load per warp and K block brings it.
//
// The linear-layer instantiations (kLinear) take any N and any K the row
// alignment allows (the tensor maps fill K's tail with zeros; a scale's tail
// is zero too), read the tensor scales from device memory where asked, and
// with kDirect write D of any type and stride from registers.
//
// Tiles: 128 x 256 per CTA, or 256 x 256 per CTA pair (tcgen05.mma
// .cta_group::2; each CTA stages its own 128 A rows and 128 of the B rows,
// loads complete on the leader CTA's barriers, the leader's single thread
// issues the scale copies and MMAs and commits to both CTAs' barriers).
// Roles (320 threads, one CTA per SM):
//   warp 0      producer: TMA loads of A (128 x 128 B) and B (256 or 128 x
//               128 B) per K block, plus (NVFP4) the scale atoms (one 2 KiB
//               box for A's 128-row block, one 4 KiB box for B's 256 rows).
//   warp 1      TMEM allocation (512 columns) and the single MMA thread.
//   warps 2-9   epilogue: warp w reads TMEM lane quarter w % 4 and column
//               half (w - 2) / 4, converts to BF16, stages 32 x 64 boxes
//               with the 128-byte swizzle and writes them with TMA stores.
//
// Every wait is bounded (globaltimer budget); a timeout records a status
// code, drains what is in flight and returns.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "ptx.cuh"

namespace bb {
extern std::atomic<int64_t> g_kernel_launches;

namespace lowp {

enum Kind : int {
  kNvfp4 = BB_LOWP_NVFP4,
  kFp8Block = BB_LOWP_FP8_BLOCK128,
  kMxfp4 = BB_LOWP_MXFP4,
  kFp8Group = BB_LOWP_FP8_GROUP128,
};
constexpr bool is_fp4(int kind) { return kind == kNvfp4 || kind == kMxfp4; }

constexpr int BM = 128;         // accumulator rows per CTA
constexpr int ROW_BYTES = 128;  // K bytes of one stage row (one 128-byte swizzle row)
// Every ring and hand-off wait acquires at CTA scope, also for barriers the
// peer CTA of a pair signals (its TMA completions, its commits, its relaxed
// arrivals): what the waiter then touches is read by the tensor core
// (operands, TMEM), whose ordering comes from the barrier's phase and the
// tcgen05 fences, not from a cluster-scope acquire. A completed-phase wait
// costs about 27 clocks at CTA scope against about 50 at cluster scope.
constexpr bool kCtaScope = false;  // bb_wait_warp's kClusterScope argument
constexpr int SF_ATOM = 512;    // bytes of one scale atom (128 rows x 4 scales)
constexpr int EPI_WARPS = 8;
constexpr int kLaunchRegs = 168;  // registers per thread the kernels are built for
constexpr int TMEM_COLS = 512;
constexpr int BAR_BYTES = 256;
// Grouped raster: group_m tile-rows are swept across all tile-columns. The
// host sizes a group's A rows to about 32 MiB (a quarter of L2), so a wave's
// A block stays resident while B streams.
constexpr int64_t kGroupABytes = 32ll << 20;
constexpr int SMEM_LIMIT = 232448;

// kCG = 1: one CTA computes a 128 x 256 tile. kCG = 2: a CTA pair computes a
// 256 x 256 tile with tcgen05.mma.cta_group::2; each CTA stages its own 128
// rows of A and 128 of the 256 B rows, its own A scale atoms and all 256 rows
// of B scale atoms (each CTA's TMEM needs the scales of every B row).
template <int kKind, int kCG>
struct Cfg {
  // Warp roles: 0 producer, 1 MMA, [EPI_W0, EPI_W0 + 8) epilogue. FP8 runs
  // a whole control warpgroup (warps 0-3, 2-3 idle) so setmaxnreg can move
  // registers from it to the two epilogue warpgroups (its promotion keeps a
  // 128-float accumulator per thread and issues two TMEM loads per wait).
  // Tiles are 256 columns wide. The code also supports 128-wide FP8 tiles
  // (four 128-column TMEM partial buffers, 64 accumulators per epilogue
  // thread): as CTA pairs they measured 1.25 PFLOP/s at 8192^3 against 2.2
  // for 256-wide tiles, the MMA warp's two barrier waits per 128-K block
  // then costing as much as the block's 256 clocks of MMA work. Splitting a
  // 256-wide tile's K block into two N = 128 halves with their own commits
  // and sub-buffers (one per epilogue warpgroup, reused after 768 instead
  // of 512 MMA clocks) measured 1843 single / 1976 pair TFLOP/s against
  // 2165: the added wait and commit per block cost more than the slack.
  static constexpr int TILE_N = 256;
  static constexpr int WARP_COLS = TILE_N / 2;         // epilogue columns per warp
  static constexpr int FP8_BUFS = TMEM_COLS / TILE_N;  // FP8 partial buffers
  static constexpr bool kRegSplit = !is_fp4(kKind) && WARP_COLS == 128;
  static constexpr int EPI_W0 = kRegSplit ? 4 : 2;
  static constexpr int THREADS = 32 * EPI_W0 + 32 * EPI_WARPS;
  // FP8's MMA warp waits once per 128-K block on the promotion hand-off:
  // it spins (no suspend hint) so wake-up latency stays off that chain
  // (8192^3: 2244 against 2165 TFLOP/s). Spinning in every producer and
  // MMA wait of both kinds, and of the BF16 GEMM, measured within 0.5 %.
  static constexpr bool kSpinWaits = !is_fp4(kKind);
  static constexpr int CTRL_REGS = 56;   // warpgroup 0 after setmaxnreg.dec
  static constexpr int EPI_REGS = 224;   // epilogue warpgroups after setmaxnreg.inc
  static_assert(!kRegSplit || 128 * CTRL_REGS + 256 * EPI_REGS <= THREADS * kLaunchRegs,
                "register split exceeds the registers the block is launched with");
  static constexpr int TILE_M = BM * kCG;
  static constexpr int B_ROWS = TILE_N / kCG;                      // B rows staged per CTA
  static constexpr int K_PER_STAGE = is_fp4(kKind) ? 256 : 128;  // elements
  static constexpr int MMA_K = is_fp4(kKind) ? 64 : 32;           // elements per instruction
  static constexpr int MMAS = K_PER_STAGE / MMA_K;                 // 4
  static constexpr int A_BYTES = BM * ROW_BYTES;
  static constexpr int B_BYTES = B_ROWS * ROW_BYTES;
  // Scale atoms of a stage per 128 rows: one per instruction (NVFP4), or one
  // per two, whose halves the instructions pick by their scale id (MXFP4).
  static constexpr int ATOMS = kKind == kNvfp4 ? MMAS : kKind == kMxfp4 ? MMAS / 2 : 0;
  static constexpr int SFA_BYTES = ATOMS * SF_ATOM;      // one row block
  static constexpr int SFB_BYTES = 2 * ATOMS * SF_ATOM;  // two row blocks
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
  // Epilogue staging: per epilogue warp EPI_BOXES boxes of 32 rows x 128
  // bytes (64 BF16 columns), written to D by TMA stores. One box per warp:
  // a second one cost the NVFP4 pair its fifth ring stage (6170 -> 6512
  // TFLOP/s at 8192^3 with one box and five stages).
  static constexpr int EPI_BOXES = 1;
  static constexpr int EPI_BOX_BYTES = 32 * 128;
  static constexpr int EPI_BYTES = EPI_WARPS * EPI_BOXES * EPI_BOX_BYTES;
  static constexpr int STAGES_FIT = (SMEM_LIMIT - 1024 - BAR_BYTES - EPI_BYTES) / STAGE_BYTES;
  // NVFP4 keeps one TMEM scale area (48 columns) per stage next to the
  // 256-column accumulator.
  static constexpr int STAGES_MAX = is_fp4(kKind) ? 5 : 8;
  static constexpr int STAGES = STAGES_FIT < STAGES_MAX ? STAGES_FIT : STAGES_MAX;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + EPI_BYTES + BAR_BYTES;
  static_assert(STAGES >= 3, "ring too shallow");
  static_assert((2 * STAGES + 12) * 8 <= BAR_BYTES, "barrier area");
  static_assert(SMEM_BYTES <= SMEM_LIMIT, "shared memory budget");
  static_assert(MMAS * 32 == ROW_BYTES, "one instruction consumes 32 bytes of each row");
  static_assert(A_BYTES % 1024 == 0 && B_BYTES % 1024 == 0, "swizzle atoms need 1 KiB alignment");
};

// NVFP4 TMEM map: two overlapping accumulators, tile j in buffer j % 2 at
// columns [192 b, 192 b + 256): they share one 64-column subtile, which the
// epilogue drains first, so the next tile's MMAs start while the other 192
// columns of the previous tile are still being read. One 48-column scale
// area at 448 (SFA of instruction g at +4g, SFB at +16 + 8g: two 128-row
// atoms), rewritten every stage: scale copies and MMAs of the issuing thread
// execute in issue order, so a copy never overtakes the MMA that reads the
// previous stage's scales. FP8 TMEM map: partial buffer b at 256 b.
constexpr uint32_t kAccStride = 192;     // NVFP4 accumulator b at column 192 b
constexpr uint32_t kOverlapCols = 64;    // columns shared by the two accumulators
constexpr uint32_t kSfBase = 448;
static_assert(kAccStride + 256 <= kSfBase && kSfBase + 48 <= TMEM_COLS, "NVFP4 TMEM map");
static_assert(kAccStride + kOverlapCols == 256, "accumulators overlap by one 64-column subtile");

struct Params {
  int32_t m, n, k;
  int32_t tiles_m, tiles_n, num_tiles;
  int32_t k_stages;    // K / K_PER_STAGE
  int32_t rb_m, rb_n;  // 128-row blocks of A and B
  int32_t num_clusters;
  int32_t group_m;
  const uint8_t* sfa;  // FP8: FP32 block scales (NVFP4 scales travel by TMA)
  const uint8_t* sfb;
  float global_scale;
  __nv_bfloat16* d;
  int* status;
  // Linear layer only.
  const float* scale_dev[2];  // tensor scales in device memory, or null
  int64_t sfa_ld;             // FP8 by group: rows of one K block's scales
  int64_t ldd;                // row stride of D in elements
  int32_t d_dtype;            // BB_DTYPE_* of a D written directly
};

// Instruction descriptors.
//   kind::f8f6f4 (E4M3 x E4M3 -> F32): [4,6) D fmt 1, [7,10) A fmt 0,
//     [10,13) B fmt 0, [17,23) N >> 3, [24,29) M >> 4.
//   kind::mxf4nvf4 block-scaled: [4,6) B scale id 0, [7,10) A fmt 1 (E2M1),
//     [10,13) B fmt 1, [17,23) N >> 3, [23] scale fmt 0 (UE4M3),
//     [24,29) M >> 4, [29,31) A scale id 0, [31] K size 0 (K = 64).
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
  return (1u << 4) | ((static_cast<uint32_t>(n) >> 3) << 17) | ((static_cast<uint32_t>(m) >> 4) << 24);
}
__host__ __device__ constexpr uint32_t idesc_nvf4(int m, int n) {
  return (1u << 7) | (1u << 10) | ((static_cast<uint32_t>(n) >> 3) << 17) |
         ((static_cast<uint32_t>(m) >> 4) << 24);
}
// kind::mxf4 block-scaled: as above with scale fmt 1 (UE8M0) and the scale
// ids 0 or 2, which pick the 2 of a 32-bit scale word's 4 bytes.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n, uint32_t id) {
  return idesc_nvf4(m, n) | (1u << 23) | (id << 4) | (id << 29);
}
static_assert(idesc_f8(128, 256) == 0x08400010u, "f8f6f4 idesc");
static_assert(idesc_nvf4(128, 256) == 0x08400480u, "mxf4nvf4 idesc");
static_assert(idesc_nvf4(256, 256) == 0x10400480u, "mxf4nvf4 idesc, CTA pair");

template <int kCG>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kCG == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
}
template <int kCG>
__device__ __forceinline__ void mma_nvf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t tsfa,
                                         uint32_t tsfb, uint32_t acc) {
  if constexpr (kCG == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(tsfa), "r"(tsfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.block16 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(
            d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(tsfa), "r"(tsfb)
        : "memory");
  }
}
template <int kCG>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t tsfa,
                                         uint32_t tsfb, uint32_t acc) {
  if constexpr (kCG == 1) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(tsfa), "r"(tsfb)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.block32 [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(tsfa), "r"(tsfb)
        : "memory");
  }
}
// Shared-memory descriptor of one 512-byte scale atom (32 rows x 16 bytes):
// interleaved (no-swizzle) K-major layout, 8-row core matrices of 128
// contiguous bytes stacked every 128 bytes along the rows (SBO).
__device__ __forceinline__ uint64_t sf_atom_desc(uint32_t smem_addr) {
  return make_smem_desc(smem_addr, 128, 128, kLayoutNone);
}
// One scale atom into 4 TMEM columns, replicated into the four 32-lane
// quarters (each quarter of the MMA reads its own lanes). With cta_group::2
// each CTA of the pair copies from its own shared memory into its own TMEM.
template <int kCG>
__device__ __forceinline__ void tmem_cp_desc(uint32_t taddr, uint64_t desc) {
  if constexpr (kCG == 1) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  } else {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  }
}

// Rank-2 tile loads: into this CTA's shared memory, completing on this CTA's
// mbarrier (1 CTA) or on the leader CTA's mbarrier (pair form). The data goes
// to the issuing CTA only.
template <int kCG>
__device__ __forceinline__ void load_2d(uint32_t dst, const void* tmap, uint32_t mbar, int32_t x, int32_t y) {
  if constexpr (kCG == 1) {
    tma_load_2d(dst, tmap, mbar, x, y);
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(tmap), "r"(mbar), "r"(x), "r"(y)
        : "memory");
  }
}

__device__ __forceinline__ void tile_coords(const Params& p, int t, int& m_blk, int& n_blk) {
  const int group_size = p.group_m * p.tiles_n;
  const int g = t / group_size;
  const int first_m = g * p.group_m;
  const int gm = min(p.group_m, p.tiles_m - first_m);
  const int local = t - g * group_size;
  m_blk = first_m + local % gm;
  n_blk = local / gm;
}

// Converts 32 FP32 accumulator values (scaled by s) to 16 packed BF16 pairs.
__device__ __forceinline__ void pack32(const float* v, float s, uint32_t* out) {
#pragma unroll
  for (int j = 0; j < 16; ++j) out[j] = pack_bf16x2(v[2 * j] * s, v[2 * j + 1] * s);
}

// FP32 promotion acc += v * s for 32 values, two lanes per instruction
// (packed fma.rn.f32x2 of sm_100).
__device__ __forceinline__ void promote32(float* acc, const uint32_t (&v)[32], float s) {
  const uint64_t s2 = (static_cast<uint64_t>(__float_as_uint(s)) << 32) | __float_as_uint(s);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    uint64_t a2 = (static_cast<uint64_t>(__float_as_uint(acc[2 * j + 1])) << 32) | __float_as_uint(acc[2 * j]);
    const uint64_t v2 = (static_cast<uint64_t>(v[2 * j + 1]) << 32) | v[2 * j];
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a2) : "l"(v2), "l"(s2));
    acc[2 * j] = __uint_as_float(static_cast<uint32_t>(a2));
    acc[2 * j + 1] = __uint_as_float(static_cast<uint32_t>(a2 >> 32));
  }
}

// 32 rows x 32 columns of D from the registers of a warp (lane = row), v * s:
// through the warp's 4 KiB of shared memory, so that a store instruction writes
// 32 columns of one row, whatever D's type, stride and alignment. Rows and
// columns outside D are left out.
__device__ __forceinline__ void store_direct32(const Params& p, uint32_t box, int row0, int col, const float* v, float s,
                                               int lane) {
  if (row0 >= p.m || col >= p.n) return;  // the whole warp
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 8; ++j)
    st_shared_v4(box + lane * 128 + ((j ^ (lane & 7)) << 4), __float_as_uint(v[4 * j] * s), __float_as_uint(v[4 * j + 1] * s),
                 __float_as_uint(v[4 * j + 2] * s), __float_as_uint(v[4 * j + 3] * s));
  __syncwarp();
  const int rows = min(32, p.m - row0);
  const int64_t at = row0 * p.ldd + col + lane;
  if (col + lane < p.n) {
    auto element = [&](int r) { return ld_shared_f32(box + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4); };
    if (p.d_dtype == BB_DTYPE_F32) {
      float* d = reinterpret_cast<float*>(p.d) + at;
#pragma unroll 8
      for (int r = 0; r < rows; ++r, d += p.ldd) *d = element(r);
    } else if (p.d_dtype == BB_DTYPE_F16) {
      __half* d = reinterpret_cast<__half*>(p.d) + at;
#pragma unroll 8
      for (int r = 0; r < rows; ++r, d += p.ldd) *d = __float2half_rn(element(r));
    } else {
      __nv_bfloat16* d = p.d + at;
#pragma unroll 8
      for (int r = 0; r < rows; ++r, d += p.ldd) *d = __float2bfloat16_rn(element(r));
    }
  }
}

template <int kKind, int kCG, bool kLinear = false, bool kDirect = false>
__global__ void __launch_bounds__(Cfg<kKind, kCG>::THREADS, 1)
    bb_lowp_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                        const __grid_constant__ CUtensorMap tm_sfa, const __grid_constant__ CUtensorMap tm_sfb,
                        const __grid_constant__ CUtensorMap tm_d, const Params p) {
  using C = Cfg<kKind, kCG>;
  constexpr int STAGES = C::STAGES;
  constexpr bool kPair = kCG == 2;
  const uint32_t rank = kPair ? cluster_ctarank() : 0u;
  if (blockDim.x != C::THREADS || (kPair && cluster_nctarank() != 2) || (gridDim.x % kCG) != 0) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kDevBadLaunch);
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem_a + STAGES * C::A_BYTES;
  uint8_t* smem_sfa = smem_b + STAGES * C::B_BYTES;        // NVFP4 only
  uint8_t* smem_sfb = smem_sfa + STAGES * C::SFA_BYTES;    // NVFP4 only
  uint8_t* smem_epi = smem + STAGES * C::STAGE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem_epi + C::EPI_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* acc_full = bars + 2 * STAGES;       // [4]
  uint64_t* acc_empty = bars + 2 * STAGES + 4;  // [4], in the leader CTA: buffer fully drained
  uint64_t* ovl_free = bars + 2 * STAGES + 8;   // [2], in the leader CTA: NVFP4 shared subtile drained
  uint64_t* mma_done = bars + 2 * STAGES + 10;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 11);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const bool leader = rank == 0;

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    prefetch_tmap(&tm_d);
    if constexpr (is_fp4(kKind)) {
      prefetch_tmap(&tm_sfa);
      prefetch_tmap(&tm_sfb);
    }
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(smem_u32(&acc_full[b]), 1);
      mbar_init(smem_u32(&acc_empty[b]), EPI_WARPS * kCG);
    }
    for (int b = 0; b < 2; ++b) mbar_init(smem_u32(&ovl_free[b]), (EPI_WARPS / 2) * kCG);
    mbar_init(smem_u32(mma_done), 1);
    fence_mbarrier_init_cluster();
  }
  if (warp == 1) {
    tmem_alloc<kCG>(smem_u32(tmem_slot), TMEM_COLS);
    tmem_relinquish<kCG>();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const int cluster_idx = blockIdx.x / kCG;
  if constexpr (kLinear) {
    grid_wait();
    grid_trigger();
  }

  if (warp < C::EPI_W0) {
    if constexpr (C::kRegSplit) {
      // Warpgroup 0 (producer, MMA, two idle warps) gives registers to the
      // epilogue warpgroups (setmaxnreg sits inside each role's branch so
      // the register allocator sees one limit per region). The host checks
      // the block's launch register pool covers the split before launching.
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::CTRL_REGS));
    }
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    // The whole warp runs the loop and waits; one elected lane issues.
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0;
    for (int t = cluster_idx; ok && t < p.num_tiles; t += p.num_clusters) {
      int m_blk, n_blk;
      tile_coords(p, t, m_blk, n_blk);
      const int a_row = m_blk * C::TILE_M + static_cast<int>(rank) * BM;
      const int b_row = n_blk * C::TILE_N + static_cast<int>(rank) * C::B_ROWS;
      const int sfa_blk = m_blk * kCG + static_cast<int>(rank);
      for (int ks = 0; ks < p.k_stages; ++ks) {
        if (!bb_wait_warp<kCtaScope>(smem_u32(&empty[stage]), phase ^ 1u, p.status, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t fb_own = smem_u32(&full[stage]);
          const uint32_t fb = kPair ? mapa_shared(fb_own, 0) : fb_own;
          if (leader) mbar_arrive_expect_tx(fb_own, C::STAGE_BYTES * kCG);
          load_2d<kCG>(smem_u32(smem_a + stage * C::A_BYTES), &tm_a, fb, ks * ROW_BYTES, a_row);
          load_2d<kCG>(smem_u32(smem_b + stage * C::B_BYTES), &tm_b, fb, ks * ROW_BYTES, b_row);
          if constexpr (is_fp4(kKind)) {
            // Scale atoms as rows of 8-byte words: one row per 128-row block,
            // atoms of 64 words each; a stage is 4 (NVFP4) or 2 (MXFP4) of them.
            load_2d<kCG>(smem_u32(smem_sfa + stage * C::SFA_BYTES), &tm_sfa, fb, ks * 64 * C::ATOMS, sfa_blk);
            load_2d<kCG>(smem_u32(smem_sfb + stage * C::SFB_BYTES), &tm_sfb, fb, ks * 64 * C::ATOMS, 2 * n_blk);
          }
        }
        __syncwarp();
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (ok) {
      // Tail: wait until the MMA has released every stage, so no commit
      // arrival can still be in flight towards this CTA when it exits.
      for (int i = 0; i < STAGES; ++i) {
        if (!bb_wait_warp<kCtaScope>(smem_u32(&empty[stage]), phase ^ 1u, p.status, kDevTimeoutProducer)) break;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } else if (lane == 0) {
      bounded_sleep_ns(2000000);  // aborted: let copies already issued land
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA)
    // Whole warp runs the loop and waits; one elected lane issues the scale
    // copies, MMAs and commits of each stage (always the same lane: elect.sync
    // picks the lowest active lane of the converged warp).
    if (leader) {
      bool ok = true;
      int stage = 0;
      uint32_t phase = 0;
      uint32_t acc_iter = 0;  // NVFP4: tiles; FP8: K blocks (partial buffers)
      // Stage-0 descriptors; stage s adds s times the stage size (in 16-byte
      // units, the unit of the descriptors' start-address field).
      const uint64_t a_desc0 = sw128_kmajor_desc(smem_u32(smem_a));
      const uint64_t b_desc0 = sw128_kmajor_desc(smem_u32(smem_b));
      const uint64_t sfa_desc0 = sf_atom_desc(smem_u32(smem_sfa));
      const uint64_t sfb_desc0 = sf_atom_desc(smem_u32(smem_sfb));
      const uint32_t sf_cols0 = tmem_base + kSfBase;
      auto commit_both = [&](uint64_t* bar) {
        const uint32_t a = smem_u32(bar);
        umma_commit<kCG>(a);
        if constexpr (kPair) umma_commit<kCG>(mapa_shared(a, 1));
      };
      for (int t = cluster_idx; ok && t < p.num_tiles; t += p.num_clusters) {
        uint32_t acc_col = 0;
        if constexpr (is_fp4(kKind)) {
          // Tile j goes to buffer j % 2: wait until tile j - 2 left it, and
          // until tile j - 1 (the other buffer) drained the shared subtile.
          const uint32_t b = acc_iter & 1u;
          if (!bb_wait_warp<kCtaScope>(smem_u32(&acc_empty[b]), ((acc_iter >> 1) & 1u) ^ 1u, p.status,
                                   kDevTimeoutMma)) {
            ok = false;
            break;
          }
          if (acc_iter > 0 && !bb_wait_warp<kCtaScope>(smem_u32(&ovl_free[b ^ 1u]), ((acc_iter - 1) >> 1) & 1u,
                                                   p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          acc_col = b * kAccStride;
        }
        for (int ks = 0; ks < p.k_stages; ++ks) {
          uint32_t d_tmem = tmem_base + acc_col;
          uint32_t buf = 0;
          // The stage's operands are normally resident long before its
          // partial buffer is free (FP8), so the data wait comes first and
          // only the buffer hand-off stands between the release and the MMAs.
          if (!bb_wait_warp<kCtaScope, !C::kSpinWaits>(smem_u32(&full[stage]), phase, p.status, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          if constexpr (!is_fp4(kKind)) {
            buf = acc_iter % C::FP8_BUFS;
            if (!bb_wait_warp<kCtaScope, !C::kSpinWaits>(smem_u32(&acc_empty[buf]), ((acc_iter / C::FP8_BUFS) & 1u) ^ 1u,
                                                     p.status, kDevTimeoutMma)) {
              ok = false;
              break;
            }
            d_tmem = tmem_base + buf * C::TILE_N;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t a_desc = a_desc0 + static_cast<uint64_t>(stage) * (C::A_BYTES >> 4);
            const uint64_t b_desc = b_desc0 + static_cast<uint64_t>(stage) * (C::B_BYTES >> 4);
            if constexpr (kKind == kNvfp4) {
              const uint32_t sf_cols = sf_cols0;
              const uint64_t sfa_desc = sfa_desc0 + static_cast<uint64_t>(stage) * (C::SFA_BYTES >> 4);
              const uint64_t sfb_desc = sfb_desc0 + static_cast<uint64_t>(stage) * (C::SFB_BYTES >> 4);
              constexpr uint32_t idesc = idesc_nvf4(C::TILE_M, C::TILE_N);
              // Per K step: its three scale copies, then its MMA (copies and
              // MMAs of one thread execute in issue order).
#pragma unroll
              for (int g = 0; g < C::MMAS; ++g) {
                tmem_cp_desc<kCG>(sf_cols + 4 * g, sfa_desc + g * (SF_ATOM >> 4));
                tmem_cp_desc<kCG>(sf_cols + 16 + 8 * g, sfb_desc + g * (SF_ATOM >> 4));
                tmem_cp_desc<kCG>(sf_cols + 20 + 8 * g, sfb_desc + (C::SFB_BYTES / 2 + g * SF_ATOM) / 16);
                mma_nvf4<kCG>(d_tmem, a_desc + 2 * g, b_desc + 2 * g, idesc, sf_cols + 4 * g, sf_cols + 16 + 8 * g,
                              (ks | g) != 0 ? 1u : 0u);
              }
            } else if constexpr (kKind == kMxfp4) {
              const uint64_t sfa_desc = sfa_desc0 + static_cast<uint64_t>(stage) * (C::SFA_BYTES >> 4);
              const uint64_t sfb_desc = sfb_desc0 + static_cast<uint64_t>(stage) * (C::SFB_BYTES >> 4);
#pragma unroll
              for (int g = 0; g < C::MMAS; ++g) {
                const uint32_t tsfa = sf_cols0 + 4 * (g / 2), tsfb = sf_cols0 + 16 + 8 * (g / 2);
                if (g % 2 == 0) {
                  tmem_cp_desc<kCG>(tsfa, sfa_desc + (g / 2) * (SF_ATOM >> 4));
                  tmem_cp_desc<kCG>(tsfb, sfb_desc + (g / 2) * (SF_ATOM >> 4));
                  tmem_cp_desc<kCG>(tsfb + 4, sfb_desc + (C::SFB_BYTES / 2 + (g / 2) * SF_ATOM) / 16);
                }
                mma_mxf4<kCG>(d_tmem, a_desc + 2 * g, b_desc + 2 * g, idesc_mxf4(C::TILE_M, C::TILE_N, 2 * (g % 2)), tsfa,
                              tsfb, (ks | g) != 0 ? 1u : 0u);
              }
            } else {
              constexpr uint32_t idesc = idesc_f8(C::TILE_M, C::TILE_N);
#pragma unroll
              for (int g = 0; g < C::MMAS; ++g)
                mma_f8<kCG>(d_tmem, a_desc + 2 * g, b_desc + 2 * g, idesc, g != 0 ? 1u : 0u);
            }
            // FP8: this commit also tells the epilogue that K block
            // acc_iter's partial is complete (its wait is on the stage's
            // barrier), so no second commit per block is needed.
            commit_both(&empty[stage]);
          }
          __syncwarp();
          if constexpr (!is_fp4(kKind)) ++acc_iter;
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (is_fp4(kKind)) {
          if (elect_one()) commit_both(&acc_full[acc_iter & 1u]);
          __syncwarp();
          ++acc_iter;
        }
      }
      // Drain: every MMA issued so far must finish before TMEM is freed.
      if (elect_one()) umma_commit<kCG>(smem_u32(mma_done));
      __syncwarp();
      bb_wait_warp(smem_u32(mma_done), 0, p.status, kDevTimeoutMma, /*honor_abort=*/false);
    }
  }
  } else {
    if constexpr (C::kRegSplit) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::EPI_REGS));
    // ------------------------------------------------------------ epilogue
    const int q = warp & 3;
    const int half = (warp - C::EPI_W0) / 4;
    const uint32_t lane_off = static_cast<uint32_t>(q * 32) << 16;
    uint32_t acc_iter = 0;
    bool ok = true;
    // One arrival per warp on a barrier of the leader CTA, after this
    // warp's TMEM reads completed.
    auto arrive_leader = [&](uint64_t* bar) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        const uint32_t eb = smem_u32(bar);
        if constexpr (kPair) {
          mbar_arrive_cluster_relaxed(mapa_shared(eb, 0));
        } else {
          mbar_arrive(eb);
        }
      }
    };
    auto release = [&](uint32_t buf) { arrive_leader(&acc_empty[buf]); };
    // D rows row0 .. row0 + 31 (lane = row), columns col0 .. col0 + 127 as two
    // 32 x 64 boxes: each staged with the 128-byte swizzle in this warp's
    // boxes of shared memory and written by one TMA store (clipped at the
    // edges of D; boxes wholly outside D are skipped).
    const uint32_t ebuf = smem_u32(smem_epi + (warp - C::EPI_W0) * C::EPI_BOXES * C::EPI_BOX_BYTES);
    uint32_t box_seq = 0;
    const uint64_t d_policy = l2_policy_evict_first();
    float scale = p.global_scale;
    if constexpr (kLinear) {
      if (p.scale_dev[0]) scale *= *p.scale_dev[0];
      if (p.scale_dev[1]) scale *= *p.scale_dev[1];
    }
    auto store_boxes = [&](int row0, int col0_, const uint32_t(&pk_)[C::WARP_COLS / 2]) {
#pragma unroll
      for (int h = 0; h < C::WARP_COLS / 64; ++h) {
        const uint32_t buf = ebuf + (box_seq % C::EPI_BOXES) * C::EPI_BOX_BYTES;
        ++box_seq;
        if (lane == 0) bulk_wait_group_read<C::EPI_BOXES - 1>();
        __syncwarp();
        const uint32_t row_addr = buf + lane * 128;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          st_shared_v4(row_addr + ((j ^ (lane & 7)) << 4), pk_[32 * h + 4 * j], pk_[32 * h + 4 * j + 1],
                       pk_[32 * h + 4 * j + 2], pk_[32 * h + 4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          // D is written once: evict-first in L2.
          if (row0 < p.m && col0_ + 64 * h < p.n) tma_store_2d_hint(&tm_d, buf, col0_ + 64 * h, row0, d_policy);
          bulk_commit_group();
        }
      }
    };
    for (int t = cluster_idx; ok && t < p.num_tiles; t += p.num_clusters) {
      int m_blk, n_blk;
      tile_coords(p, t, m_blk, n_blk);
      const int row = m_blk * C::TILE_M + static_cast<int>(rank) * BM + q * 32 + lane;
      const int col0 = n_blk * C::TILE_N + half * C::WARP_COLS;
      uint32_t pk[C::WARP_COLS / 2];
      if constexpr (is_fp4(kKind)) {
        const uint32_t b = acc_iter & 1u;
        if (!bb_wait_warp<kCtaScope>(smem_u32(&acc_full[b]), (acc_iter >> 1) & 1u, p.status, kDevTimeoutEpilogue)) break;
        tc_fence_after();
        const uint32_t taddr = tmem_base + lane_off + b * kAccStride + half * C::WARP_COLS;
        // The subtile shared with the other buffer is columns [192, 256) of
        // buffer 0 (this warp's chunks 2, 3 when half == 1) and [0, 64) of
        // buffer 1 (chunks 0, 1 when half == 0); its owners read it first
        // and report it drained before reading the rest.
        const bool owner = (b == 0) ? (half == 1) : (half == 0);
        // Chunk pair c, c + 1 (32 columns each) into pk; compile-time chunk
        // indices keep pk in registers.
        auto drain_pair = [&](auto chunk, bool report) {
          constexpr int c = decltype(chunk)::value;
          uint32_t r0[32], r1[32];
          tmem_ld_32x32b_x32(taddr + 32 * c, r0);
          tmem_ld_32x32b_x32(taddr + 32 * (c + 1), r1);
          tmem_ld_wait();
          if (report) arrive_leader(&ovl_free[b]);
          if constexpr (kDirect) {
            store_direct32(p, ebuf, row - lane, col0 + 32 * c, reinterpret_cast<const float*>(r0), scale, lane);
            store_direct32(p, ebuf, row - lane, col0 + 32 * (c + 1), reinterpret_cast<const float*>(r1), scale, lane);
          } else {
            pack32(reinterpret_cast<const float*>(r0), scale, pk + 16 * c);
            pack32(reinterpret_cast<const float*>(r1), scale, pk + 16 * (c + 1));
          }
        };
        if (b == 0) {
          drain_pair(std::integral_constant<int, 2>{}, owner);
          drain_pair(std::integral_constant<int, 0>{}, false);
        } else {
          drain_pair(std::integral_constant<int, 0>{}, owner);
          drain_pair(std::integral_constant<int, 2>{}, false);
        }
        release(b);
        ++acc_iter;
      } else {
        const float* sa = reinterpret_cast<const float*>(p.sfa);
        const float* sb = reinterpret_cast<const float*>(p.sfb);
        // Ragged edges: rows / columns past M / N are never stored, any valid
        // scale row serves them.
        const int mb = min(m_blk * kCG + static_cast<int>(rank), p.rb_m - 1);
        const int nb = min(col0 / 128, p.rb_n - 1);
        const float* sa_row = sa + static_cast<int64_t>(mb) * p.k_stages;
        // By group: lane = row, so the lane's own scale of every K block, four
        // loads ahead in a queue. The epilogue's time per block is what the
        // kernel is made of (8192^3: 538 us back to back, 480 alone, where the
        // block-scaled form takes 450 and 455), and everything that adds
        // instructions to it was slower: sets of four scales with selects 620,
        // a ring in shared memory 610, the loop unrolled by four 620.
        constexpr bool kGroup = kKind == kFp8Group;
        constexpr int kAhead = 4;
        const float* sa_lane = sa + min(row, p.m - 1);
        // A linear layer's launch may begin while the kernel in front still
        // writes the scales; the non-coherent path is for memory that nobody
        // writes as long as the kernel lives.
        auto load_scale = [](const float* at) {
          if constexpr (!kLinear) return __ldg(at);
          float v;
          asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(at));
          return v;
        };
        float sa_next[kAhead];
        if constexpr (kGroup) {
#pragma unroll
          for (int j = 0; j < kAhead; ++j) {
            sa_next[j] = j < p.k_stages ? load_scale(sa_lane) : 0.f;
            sa_lane += p.sfa_ld;
          }
        }
        const float* sb_row = sb + static_cast<int64_t>(nb) * p.k_stages;
        float acc[C::WARP_COLS];
#pragma unroll
        for (int j = 0; j < C::WARP_COLS; ++j) acc[j] = 0.f;
        // Lane l holds the scale product of K block w + l of the current
        // 32-block window (s_win) and the raw scales of the next window,
        // loaded a whole window ahead: the per-block loop reads its scale
        // with one shuffle and never waits on a global load (a load issued
        // one block ahead still stalled each block for an L2 round trip,
        // right before the wait on the MMA hand-off).
        float ra, rb;
        auto load_raw = [&](int kk) {
          ra = 0.f;
          rb = 0.f;
          if (kk < p.k_stages) {
            ra = kGroup ? 1.f : load_scale(sa_row + kk);
            rb = load_scale(sb_row + kk);
          }
        };
        load_raw(lane);
        float s_win = ra * rb;
        load_raw(32 + lane);
        for (int ks = 0; ks < p.k_stages; ++ks) {
          if ((ks & 31) == 0 && ks > 0) {
            s_win = ra * rb;
            load_raw(ks + 32 + lane);
          }
          float s = __shfl_sync(0xffffffffu, s_win, ks & 31);
          if constexpr (kGroup) {
            s *= sa_next[0];
#pragma unroll
            for (int j = 0; j + 1 < kAhead; ++j) sa_next[j] = sa_next[j + 1];
            if (ks + kAhead < p.k_stages) sa_next[kAhead - 1] = load_scale(sa_lane);
            sa_lane += p.sfa_ld;
          }
          const uint32_t buf = acc_iter % C::FP8_BUFS;
          // K block acc_iter's partial is complete when the MMA's commit
          // releases its operand stage (one stage per K block, stage =
          // acc_iter % STAGES, that barrier's phase acc_iter / STAGES). The
          // parity cannot be overtaken: the MMA can run at most FP8_BUFS
          // blocks ahead of this wait, and STAGES > FP8_BUFS.
          // Spin without the suspend hint: this wait is on the per-K-block
          // MMA -> promotion -> MMA hand-off, where wake-up latency counts.
          static_assert(STAGES > C::FP8_BUFS, "stage barrier reused before the epilogue saw it");
          if (!bb_wait_warp<kCtaScope, false>(smem_u32(&empty[acc_iter % STAGES]), (acc_iter / STAGES) & 1u, p.status,
                                          kDevTimeoutEpilogue)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t taddr = tmem_base + lane_off + buf * C::TILE_N + half * C::WARP_COLS;
          constexpr int kChunks = C::WARP_COLS / 32;
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t r0[32], r1[32];
            tmem_ld_32x32b_x32(taddr + 32 * c, r0);
            tmem_ld_32x32b_x32(taddr + 32 * (c + 1), r1);
            tmem_ld_wait();
            if (c == kChunks - 2) release(buf);
            promote32(acc + 32 * c, r0, s);
            promote32(acc + 32 * (c + 1), r1, s);
          }
          ++acc_iter;
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < C::WARP_COLS / 32; ++c) {
          if constexpr (kDirect) {
            store_direct32(p, ebuf, row - lane, col0 + 32 * c, acc + 32 * c, scale, lane);
          } else {
            pack32(acc + 32 * c, scale, pk + 16 * c);
          }
        }
      }
      if constexpr (!kDirect) store_boxes(row - lane, col0, pk);
    }
    if (lane == 0) bulk_wait_group<0>();  // stores read their staging boxes before exit
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) cluster_sync();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<kCG>(tmem_base, TMEM_COLS);
  }
}

}  // namespace lowp
}  // namespace bb

