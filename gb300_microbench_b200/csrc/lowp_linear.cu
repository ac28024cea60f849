// The product of a quantised linear layer, D (M x N) = dequant(A) * dequant(B)^T,
// for any number of rows (bb_linear_*): NVFP4, MXFP4, and FP8 with activations
// scaled per row and 128 K elements and weights per 128 x 128 block.
//
// Many rows run the 256 x 256 (128 x 256) tile kernel of gemm_lowp.cuh. Few
// rows run the kernel below, whose work is to read the weights once.
#include <new>

#include "gemm_lowp.cuh"

namespace bb {
namespace linear {

using namespace lowp;

constexpr int kMaxSplits = 8;  // the portable cluster size

// ---------------------------------------------------------------- few rows
// D^T = W * X^T: the weights' rows are the tensor core's M = 128 (all of them
// useful), the TN tokens its N (16 upwards), so one token costs the same weight
// stream as sixteen and no arithmetic unit decodes a weight. A CTA streams
// 128 weight rows over one share of K. The `splits` CTAs of a cluster share K;
// each owns some of the weight rows, is sent the other CTAs' FP32 partial sums
// of them over distributed shared memory (asynchronous stores of four tokens
// that signal its barrier), and adds them in rank order: the result does not
// depend on timing. Tiles of 128 tokens leave the sums in shared memory and
// read them instead, each CTA some of the tokens (MXFP4 128 x 4096 x 4096 in 4
// splits 8.4 us read, 9.9 sent; up to 64 tokens sending is faster: NVFP4
// 64 x 8192 x 8192 12.6 against 12.8, and one token 2.4 against 3.2 for the
// smallest launch).
//
// FP8: the K blocks' FP32 scales are applied as in the tile kernel, each
// block accumulated alone in one of BUFS TMEM buffers and promoted by the
// epilogue warps: acc[c] += part[c] * sb[kb] * sa[token c][kb].
//
// FP8 tiles of 128 tokens turn the product round (tokens on M, weights on N):
// a lane then holds one token, so a K block has one scale per lane instead of
// one per column, whose 64 shared-memory broadcasts per warp stood in the way of
// the operand traffic (256 x 8192 x 8192: 37 us before, 28.4 after). 4-bit tiles
// gain nothing by it (MXFP4 256 x 8192 x 8192 15.6 us, 15.4 turned; 200 x 5000 x
// 2880 8.8 and 10.2): their scales are the tensor core's.
//
// What bounds it is the weight stream, and then the ends of the launch: two
// CTAs of up to 113 KiB share an SM (all but the turned tiles), so 96 to 160 KiB
// of weights per SM are in flight (16 KiB for each of FewCfg::STAGES; 160 for FP8
// and MXFP4 with 16 tokens), and CTAs of the next launch start beside the
// last ones of this, set up, and fetch their first weights into L2. (A load
// balanced to the row, by tiles of 97 instead of 128 weight rows and so two
// CTAs on every SM, was slower: FP8 1 x 14336 x 4096 14.3 us against 13.0. It
// leaves no place for the next launch.)
template <int kKind, int kTN>
struct FewCfg {
  static constexpr int TN = kTN;
  static constexpr bool FP4 = is_fp4(kKind);
  static constexpr bool TURNED = !FP4 && TN == 128;  // tokens on M
  static constexpr int CTAS_PER_SM = TURNED ? 1 : 2;  // 64 accumulators a thread want a whole SM's registers
  static constexpr int EPI_W = TN <= 32 ? 4 : 8;  // epilogue warps: lane quarters x column halves
  static constexpr int THREADS = 64 + 32 * EPI_W;
  static constexpr int COLS = TN * 4 / EPI_W;     // accumulator columns per epilogue thread
  static constexpr int CHUNK = COLS == 32 ? 32 : 16;  // columns of one TMEM load
  static constexpr int MMAS = 4;
  static constexpr int ATOMS = kKind == kNvfp4 ? 4 : kKind == kMxfp4 ? 2 : 0;
  static constexpr int W_BYTES = 128 * ROW_BYTES;
  static constexpr int X_BYTES = TN * ROW_BYTES;
  static constexpr int SF_BYTES = ATOMS * SF_ATOM;  // of the weights, and as much of the tokens
  static constexpr int STAGE_BYTES = W_BYTES + X_BYTES + 2 * SF_BYTES;
  // Partial sums. Sent: the CTA's own and the others', [split][owned row][token]
  // (splits * owned rows are 128 and a few; the pitch keeps 16-byte accesses of
  // neighbouring rows on different banks), in a place of their own where that
  // is small, otherwise over the ring, once every CTA's is idle. Read:
  // [token][128 rows] over the ring (turned tiles too, whose lanes are tokens:
  // four words more a token keep their writes on different banks).
  static constexpr bool SEND = TN <= 64;
  static constexpr bool OWN_PLACE = TN <= 32;
  static constexpr int PITCH = SEND ? TN + 4 : TURNED ? 132 : 128;
  static constexpr int SUM_BYTES = (SEND ? 128 + kMaxSplits : TN) * PITCH * 4;
  // FP8: every epilogue warp keeps the scales of SCALE_SLOTS K blocks (its
  // tokens' and, behind them, the weights').
  static constexpr int SCALE_SLOTS = 4;
  static constexpr int SCALES = TURNED ? 32 : COLS;  // token scales of a warp and K block
  static constexpr int SCALE_PITCH = SCALES + 4;
  static constexpr int SCALE_BYTES = FP4 ? 0 : EPI_W * SCALE_SLOTS * SCALE_PITCH * 4;
  static constexpr int TAIL_BYTES = (OWN_PLACE ? SUM_BYTES : 0) + SCALE_BYTES + BAR_BYTES;
  static constexpr int LIMIT = CTAS_PER_SM == 2 ? 115712 : SMEM_LIMIT;
  static constexpr int STAGES_FIT = (LIMIT - 1024 - TAIL_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT < 8 ? STAGES_FIT : 8;
  static constexpr int SMEM_BYTES = 1024 + STAGES * STAGE_BYTES + TAIL_BYTES;
  // FP8: partial buffers. FP4: one accumulator, then the scale columns.
  static constexpr int BUFS = FP4 ? 1 : TN == 32 ? 3 : 4;
  static constexpr int SF_COL = TN;
  static constexpr int SF_COLS = ATOMS * 8;
  static constexpr int COLS_USED = FP4 ? TN + SF_COLS : BUFS * TN;
  static constexpr int TMEM = COLS_USED <= 64 ? 64 : COLS_USED <= 128 ? 128 : COLS_USED <= 256 ? 256 : 512;
  static_assert(COLS_USED <= TMEM && TMEM * CTAS_PER_SM <= 512, "TMEM of the CTAs that share an SM");
  static_assert(STAGES >= 3 && SMEM_BYTES <= LIMIT, "shared memory");
  static_assert(OWN_PLACE || SUM_BYTES <= STAGES * STAGE_BYTES, "partial sums fit the ring");
  static_assert((2 * STAGES + BUFS + 3) * 8 <= BAR_BYTES, "barrier area");
  static_assert(BUFS < STAGES, "a stage's barrier tells the epilogue of its block");
};

// Weights fetched into L2 ahead of the wait (NVFP4 1 x 8192 x 8192: none 9.7 us,
// three stages 8.9, six 9.3; FP8 1 x 14336 x 4096: 13.5, 13.1, 13.3).
constexpr int kPrefetchStages = 3;

struct FewParams {
  int32_t m, n;
  int32_t k_stages, splits, tiles_n;
  int32_t owned;       // weight rows a CTA of the cluster owns: rank r has [r * owned, + owned) of the 128
  const float* sfa;    // FP8: [K block][sfa_ld]
  const float* sfb;    // FP8: [weight row block][K block]
  int64_t sfa_ld, ldd;
  float scale;
  const float* scale_dev[2];
  void* d;
  int32_t d_dtype;
  int* status;
};

__device__ __forceinline__ void store_one(void* d, int dtype, int64_t at, float v) {
  if (dtype == BB_DTYPE_BF16) static_cast<__nv_bfloat16*>(d)[at] = __float2bfloat16_rn(v);
  else if (dtype == BB_DTYPE_F16) static_cast<__half*>(d)[at] = __float2half_rn(v);
  else static_cast<float*>(d)[at] = v;
}

// `count` (none if negative) of four neighbouring columns of D, in one access where it is whole and aligned.
__device__ __forceinline__ void store_four(const FewParams& p, int64_t at, int count, const float (&v)[4]) {
  const int bytes = p.d_dtype == BB_DTYPE_F32 ? 4 : 2;
  uint8_t* d = static_cast<uint8_t*>(p.d) + at * bytes;
  if (count == 4 && reinterpret_cast<uintptr_t>(d) % (4 * bytes) == 0) {
    if (p.d_dtype == BB_DTYPE_F32) {
      *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (p.d_dtype == BB_DTYPE_F16) {
      const __half2 lo = __floats2half2_rn(v[0], v[1]), hi = __floats2half2_rn(v[2], v[3]);
      *reinterpret_cast<uint2*>(d) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    } else {
      *reinterpret_cast<uint2*>(d) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < count) store_one(p.d, p.d_dtype, at + i, v[i]);
}

// `count` of N tokens of one column of D.
template <int N>
__device__ __forceinline__ void store_tokens(const FewParams& p, int token, int count, int n, const float (&v)[N], float s) {
  if (n >= p.n) return;
  const int64_t at = token * p.ldd + n;
  if (p.d_dtype == BB_DTYPE_BF16) {
    __nv_bfloat16* d = static_cast<__nv_bfloat16*>(p.d) + at;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < count) d[c * p.ldd] = __float2bfloat16_rn(v[c] * s);
  } else if (p.d_dtype == BB_DTYPE_F16) {
    __half* d = static_cast<__half*>(p.d) + at;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < count) d[c * p.ldd] = __float2half_rn(v[c] * s);
  } else {
    float* d = static_cast<float*>(p.d) + at;
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (c < count) d[c * p.ldd] = v[c] * s;
  }
}

// 16 or 32 columns of this warp's 32 TMEM lanes.
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32, "16 or 32 columns");
  if constexpr (N == 32) {
    tmem_ld_32x32b_x32(taddr, r);
  } else {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
  }
}

// 4 bytes into shared memory, zero where `valid` is false (nothing is read then).
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

// 16 bytes into a CTA of the cluster (shared::cluster addresses), counted by a
// barrier of that CTA.
__device__ __forceinline__ void st_async_v4f(uint32_t addr, const float* v, uint32_t mbar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(addr),
               "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
               "r"(mbar)
               : "memory");
}

__device__ __forceinline__ float4 ld_cluster_v4f(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(cluster_addr)
               : "memory");
  return v;
}

template <int kKind, int kTN>
__global__ void __launch_bounds__(FewCfg<kKind, kTN>::THREADS, FewCfg<kKind, kTN>::CTAS_PER_SM)
    few_rows_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                    const __grid_constant__ CUtensorMap tm_sfw, const __grid_constant__ CUtensorMap tm_sfx,
                    const FewParams p) {
  using C = FewCfg<kKind, kTN>;
  constexpr int STAGES = C::STAGES;
  if (blockDim.x != C::THREADS || p.splits < 1 || cluster_nctarank() != static_cast<uint32_t>(p.splits) ||
      gridDim.x % p.splits != 0) {
    if (threadIdx.x == 0 && p.status) atomicCAS(p.status, 0, kDevBadLaunch);
    return;
  }
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_w = smem;
  uint8_t* smem_x = smem_w + STAGES * C::W_BYTES;
  uint8_t* smem_sfw = smem_x + STAGES * C::X_BYTES;
  uint8_t* smem_sfx = smem_sfw + STAGES * C::SF_BYTES;
  uint8_t* tail = smem + STAGES * C::STAGE_BYTES;
  float* sums = reinterpret_cast<float*>(C::OWN_PLACE ? tail : smem);
  if constexpr (C::OWN_PLACE) tail += C::SUM_BYTES;
  float* smem_scale = reinterpret_cast<float*>(tail);
  uint64_t* bars = reinterpret_cast<uint64_t*>(tail + C::SCALE_BYTES);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* acc_empty = bars + 2 * STAGES;  // [BUFS], FP8
  uint64_t* done = acc_empty + C::BUFS;     // every MMA of this CTA has finished
  uint64_t* received = done + 1;            // the other CTAs' partial sums are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(received + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = p.splits > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / p.splits;  // output tile: 128 weight rows x TN tokens
  const int m0 = unit / p.tiles_n * C::TN, n_blk = unit % p.tiles_n;
  const int ks0 = static_cast<int>(static_cast<int64_t>(p.k_stages) * rank / p.splits);
  const int ks1 = static_cast<int>(static_cast<int64_t>(p.k_stages) * (rank + 1) / p.splits);
  const int mine = min(p.owned, 128 - rank * p.owned);  // weight rows this CTA owns
  const int quads = (min(C::TN, p.m - m0) + 3) / 4;     // the tile's tokens by fours (those behind M are zeros)

  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
    if constexpr (C::FP4) {
      prefetch_tmap(&tm_sfw);
      prefetch_tmap(&tm_sfx);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int b = 0; b < C::BUFS; ++b) mbar_init(smem_u32(&acc_empty[b]), C::EPI_W);
    mbar_init(smem_u32(done), 1);
    mbar_init(smem_u32(received), 1);
    fence_mbarrier_init_cluster();
    if (C::SEND && p.splits > 1) mbar_arrive_expect_tx(smem_u32(received), (p.splits - 1) * mine * quads * 16);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), C::TMEM);
    tmem_relinquish<1>();
  }
  // The weights may come from the launch before, so ahead of the wait below
  // they are fetched into L2 only, where that launch's writes land as well.
  if (warp == 2 && elect_one()) {
    for (int ks = ks0; ks < ks1 && ks < ks0 + kPrefetchStages; ++ks)
      tma_prefetch_2d(&tm_w, ks * ROW_BYTES, n_blk * 128);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  // `received` is ready for the other CTAs' signals; waited for before sending.
  if (C::OWN_PLACE && p.splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  grid_wait();
  grid_trigger();

  const int q = warp & 3, half = (warp - 2) / 4;
  const int row = q * 32 + lane;    // weight row within the block (epilogue)
  const int col0 = half * C::COLS;  // first token of this thread (epilogue)
  const int n = n_blk * 128 + row;
  const int tokens = min(C::COLS, p.m - m0 - col0);  // of this thread; may be negative
  float scale = p.scale;
  F2 acc[C::FP4 ? 1 : C::COLS / 2];
  const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + col0;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = 0;
    uint32_t phase = 0;
    for (int ks = ks0; ks < ks1; ++ks) {
      if (!bb_wait_warp(smem_u32(&empty[stage]), phase ^ 1u, p.status, kDevTimeoutProducer)) {
        ok = false;
        break;
      }
      if (elect_one()) {
        const uint32_t fb = smem_u32(&full[stage]);
        mbar_arrive_expect_tx(fb, C::STAGE_BYTES);
        tma_load_2d(smem_u32(smem_w + stage * C::W_BYTES), &tm_w, fb, ks * ROW_BYTES, n_blk * 128);
        tma_load_2d(smem_u32(smem_x + stage * C::X_BYTES), &tm_x, fb, ks * ROW_BYTES, m0);
        if constexpr (C::FP4) {
          tma_load_2d(smem_u32(smem_sfw + stage * C::SF_BYTES), &tm_sfw, fb, ks * 64 * C::ATOMS, n_blk);
          tma_load_2d(smem_u32(smem_sfx + stage * C::SF_BYTES), &tm_sfx, fb, ks * 64 * C::ATOMS, m0 / 128);
        }
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    if (ok) {
      // Tail: until the MMAs released every stage, so no commit is on its way to a CTA that left.
      for (int i = 0; i < STAGES; ++i) {
        if (!bb_wait_warp(smem_u32(&empty[stage]), phase ^ 1u, p.status, kDevTimeoutProducer)) break;
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    } else if (lane == 0) {
      bounded_sleep_ns(2000000);  // aborted: let copies already issued land
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    int stage = 0;
    uint32_t phase = 0, it = 0;
    const uint64_t w_desc0 = sw128_kmajor_desc(smem_u32(smem_w)), x_desc0 = sw128_kmajor_desc(smem_u32(smem_x));
    const uint64_t sfw_desc0 = sf_atom_desc(smem_u32(smem_sfw)), sfx_desc0 = sf_atom_desc(smem_u32(smem_sfx));
    for (int ks = ks0; ks < ks1; ++ks, ++it) {
      if (!bb_wait_warp<false, false>(smem_u32(&full[stage]), phase, p.status, kDevTimeoutMma)) break;
      uint32_t d_tmem = tmem;
      if constexpr (!C::FP4) {
        const uint32_t buf = it % C::BUFS;
        if (!bb_wait_warp<false, false>(smem_u32(&acc_empty[buf]), ((it / C::BUFS) & 1u) ^ 1u, p.status,
                                        kDevTimeoutMma))
          break;
        d_tmem += buf * C::TN;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint64_t w_desc = w_desc0 + static_cast<uint64_t>(stage) * (C::W_BYTES >> 4);
        const uint64_t x_desc = x_desc0 + static_cast<uint64_t>(stage) * (C::X_BYTES >> 4);
        if constexpr (C::FP4) {
          const uint64_t sfw = sfw_desc0 + static_cast<uint64_t>(stage) * (C::SF_BYTES >> 4);
          const uint64_t sfx = sfx_desc0 + static_cast<uint64_t>(stage) * (C::SF_BYTES >> 4);
          constexpr int per_atom = C::MMAS / C::ATOMS;  // instructions that share an atom
#pragma unroll
          for (int g = 0; g < C::MMAS; ++g) {
            const int a = g / per_atom;
            const uint32_t t_w = tmem + C::SF_COL + 4 * a;
            const uint32_t t_x = t_w + 4 * C::ATOMS;
            if (g % per_atom == 0) {
              tmem_cp_desc<1>(t_w, sfw + a * (SF_ATOM >> 4));
              tmem_cp_desc<1>(t_x, sfx + a * (SF_ATOM >> 4));
            }
            const uint32_t accumulate = (it | g) != 0 ? 1u : 0u;
            if constexpr (kKind == kNvfp4)
              mma_nvf4<1>(d_tmem, w_desc + 2 * g, x_desc + 2 * g, idesc_nvf4(128, C::TN), t_w, t_x, accumulate);
            else
              mma_mxf4<1>(d_tmem, w_desc + 2 * g, x_desc + 2 * g, idesc_mxf4(128, C::TN, 2 * (g % 2)), t_w, t_x, accumulate);
          }
        } else {
#pragma unroll
          for (int g = 0; g < C::MMAS; ++g)
            mma_f8<1>(d_tmem, (C::TURNED ? x_desc : w_desc) + 2 * g, (C::TURNED ? w_desc : x_desc) + 2 * g,
                      idesc_f8(128, C::TN), g != 0 ? 1u : 0u);
        }
        umma_commit<1>(smem_u32(&empty[stage]));
      }
      __syncwarp();
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Tracks every MMA issued: the accumulator is complete, the ring idle.
    if (elect_one()) umma_commit<1>(smem_u32(done));
    __syncwarp();
    bb_wait_warp(smem_u32(done), 0, p.status, kDevTimeoutMma, /*honor_abort=*/false);
  } else {
    // ------------------------------------------------------------ epilogue
    if (p.scale_dev[0]) scale *= *p.scale_dev[0];
    if (p.scale_dev[1]) scale *= *p.scale_dev[1];
    if constexpr (C::FP4) {
      ok = bb_wait_warp<false, false>(smem_u32(done), 0, p.status, kDevTimeoutEpilogue);
      tc_fence_after();
    } else {
      float* my_scale = smem_scale + (warp - 2) * C::SCALE_SLOTS * C::SCALE_PITCH;
      auto fetch_scales = [&](int ks) {
        if (ks < ks1) {
          const uint32_t dst = smem_u32(my_scale + (ks - ks0) % C::SCALE_SLOTS * C::SCALE_PITCH);
          const int t0 = C::TURNED ? q * 32 : col0;  // first token of the warp
          const int count = min(C::SCALES, p.m - m0 - t0);
          const float* src = p.sfa + ks * p.sfa_ld + m0 + t0;
#pragma unroll
          for (int j = 0; j < (C::SCALES + 31) / 32; ++j) {
            const int c = lane + 32 * j;
            if (c < C::SCALES) cp_async_4(dst + c * 4, c < count ? src + c : p.sfa, c < count);
          }
          if (lane == 31) cp_async_4(dst + C::SCALES * 4, p.sfb + static_cast<int64_t>(n_blk) * p.k_stages + ks, true);
        }
        cp_async_commit();
      };
#pragma unroll
      for (int i = 0; i < C::SCALE_SLOTS - 1; ++i) fetch_scales(ks0 + i);
#pragma unroll
      for (int c = 0; c < C::COLS / 2; ++c) acc[c] = pack2(0.f, 0.f);
      for (int ks = ks0; ks < ks1; ++ks) {
        const uint32_t it = ks - ks0, buf = it % C::BUFS;
        __syncwarp();  // the slot written next was read in the block before
        fetch_scales(ks + C::SCALE_SLOTS - 1);
        cp_async_wait<C::SCALE_SLOTS - 1>();
        __syncwarp();
        const float* sc = my_scale + it % C::SCALE_SLOTS * C::SCALE_PITCH;
        const float s_lane = C::TURNED ? sc[lane] * sc[C::SCALES] : sc[C::SCALES];
        const F2 s2 = pack2(s_lane, s_lane);  // turned: the lane's whole scale; else the weights'
        // The commit that releases the operand stage also says that the K
        // block's partial is complete; the MMA warp runs at most BUFS < STAGES
        // blocks ahead, so the parity cannot be overtaken.
        if (!bb_wait_warp<false, false>(smem_u32(&empty[it % STAGES]), (it / STAGES) & 1u, p.status,
                                        kDevTimeoutEpilogue)) {
          ok = false;
          break;
        }
        tc_fence_after();
#pragma unroll
        for (int c0 = 0; c0 < C::COLS; c0 += C::CHUNK) {
          uint32_t r[C::CHUNK];
          tmem_ld_cols(taddr + buf * C::TN + c0, r);
          tmem_ld_wait();
          if (c0 + C::CHUNK == C::COLS) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&acc_empty[buf]));
          }
#pragma unroll
          for (int c = 0; c < C::CHUNK; c += 4) {
            F2& a0 = acc[(c0 + c) / 2];
            F2& a1 = acc[(c0 + c) / 2 + 1];
            const F2 r0 = pack2(__uint_as_float(r[c]), __uint_as_float(r[c + 1]));
            const F2 r1 = pack2(__uint_as_float(r[c + 2]), __uint_as_float(r[c + 3]));
            if constexpr (C::TURNED) {
              a0 = fma2(r0, s2, a0);
              a1 = fma2(r1, s2, a1);
            } else {
              const float4 s = *reinterpret_cast<const float4*>(sc + c0 + c);
              a0 = fma2(mul2(r0, s2), pack2(s.x, s.y), a0);
              a1 = fma2(mul2(r1, s2), pack2(s.z, s.w), a1);
            }
          }
        }
      }
      cp_async_wait<0>();
      if (C::TURNED || (!C::OWN_PLACE && p.splits > 1))
        ok = bb_wait_warp<false, false>(smem_u32(done), 0, p.status, kDevTimeoutEpilogue) && ok;
    }
  }
  if (p.splits > 1) {
    __syncwarp();
    if constexpr (C::OWN_PLACE) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else if constexpr (C::SEND) {
      cluster_sync();  // every CTA's ring is idle (`done`: every copy has landed and been read)
    }
  }
  if (warp >= 2) {
    // This thread's sums, CHUNK tokens at a time: to D, to the row's owner, or
    // into this CTA's ring.
    const int owner = row / p.owned;
    const uint32_t at = ((rank * p.owned + row - owner * p.owned) * C::PITCH + col0) * 4;
    const uint32_t to = mapa_shared(smem_u32(sums) + at, owner), to_bar = mapa_shared(smem_u32(received), owner);
#pragma unroll
    for (int c0 = 0; c0 < C::COLS; c0 += C::CHUNK) {
      if (!C::TURNED && c0 >= tokens) break;
      float v[C::CHUNK];
      if constexpr (C::FP4) {
        uint32_t r[C::CHUNK];
        tmem_ld_cols(taddr + c0, r);
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < C::CHUNK; ++c) v[c] = __uint_as_float(r[c]);
      } else {
#pragma unroll
        for (int c = 0; c < C::CHUNK; c += 2) unpack2(acc[(c0 + c) / 2], v[c], v[c + 1]);
      }
      if constexpr (C::TURNED) {
#pragma unroll
        for (int c = 0; c < C::CHUNK; c += 4)
          *reinterpret_cast<float4*>(sums + row * C::PITCH + col0 + c0 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
      } else if (p.splits == 1) {
        store_tokens(p, m0 + col0 + c0, min(C::CHUNK, tokens - c0), n, v, scale);
      } else if constexpr (!C::SEND) {
#pragma unroll
        for (int c = 0; c < C::CHUNK; ++c) sums[(col0 + c0 + c) * C::PITCH + row] = v[c];
      } else {
#pragma unroll
        for (int c = 0; c < C::CHUNK; c += 4) {
          if (c0 + c >= tokens) continue;
          if (owner == rank)
            *reinterpret_cast<float4*>(sums + at / 4 + c0 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
          else
            st_async_v4f(to + (c0 + c) * 4, v + c, to_bar);
        }
      }
      __syncwarp();
    }
  }
  if (C::SEND && p.splits > 1) {
    // Arrived: this CTA sends nothing more. Waited for at the end: no CTA leaves while another still sends.
    __syncwarp();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (warp >= 2) {
      asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EPI_W) : "memory");  // the CTA's own sums
      bb_wait_warp<true, false>(smem_u32(received), 0, p.status, kDevTimeoutEpilogue);
      // Element e of the quads x mine sums of four tokens, e = thread, thread + threads, ...
      constexpr int kThreads = 32 * C::EPI_W;
      const int e0 = threadIdx.x - 64;
      int quad = e0 / mine, r0 = e0 - quad * mine;
      const int step = kThreads / mine, step_row = kThreads - step * mine;
      while (quad < quads) {
        const float4* from = reinterpret_cast<const float4*>(sums + r0 * C::PITCH) + quad;
        float4 f[kMaxSplits];
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r)
          if (r < p.splits) f[r] = from[r * p.owned * (C::PITCH / 4)];
        float v[4] = {f[0].x, f[0].y, f[0].z, f[0].w};
#pragma unroll
        for (int r = 1; r < kMaxSplits; ++r) {
          if (r < p.splits) {
            v[0] += f[r].x;
            v[1] += f[r].y;
            v[2] += f[r].z;
            v[3] += f[r].w;
          }
        }
        const int token = m0 + 4 * quad;
        store_tokens(p, token, min(4, p.m - token), n_blk * 128 + rank * p.owned + r0, v, scale);
        quad += step;
        r0 += step_row;
        if (r0 >= mine) {
          r0 -= mine;
          ++quad;
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
  if (!C::SEND && (C::TURNED || p.splits > 1)) {
    __syncwarp();
    if (p.splits > 1) cluster_sync();
    if (warp >= 2) {
      if (p.splits == 1) asm volatile("bar.sync 1, %0;" ::"n"(32 * C::EPI_W) : "memory");
      // Rank r adds the tokens r, r + splits, ... of all ranks' partial sums: a
      // warp per token, a lane four weight rows. Remote loads take most of a
      // microsecond each, so those of all ranks and of two tokens are in flight together.
      constexpr int kBatch = 2;
      const int count = min(C::TN, p.m - m0);
      const uint32_t base = smem_u32(sums) + lane * 16;
      const int n4 = n_blk * 128 + lane * 4;
      if (C::TURNED && p.splits == 1) {  // all in this CTA's own shared memory
#pragma unroll 4
        for (int c = warp - 2; c < count; c += C::EPI_W) {
          const float4 f = *reinterpret_cast<const float4*>(sums + c * C::PITCH + lane * 4);
          const float out[4] = {f.x * scale, f.y * scale, f.z * scale, f.w * scale};
          store_four(p, (m0 + c) * p.ldd + n4, min(4, p.n - n4), out);
        }
      } else
      for (int c = rank + (warp - 2) * p.splits; c < count; c += p.splits * C::EPI_W * kBatch) {
        float4 v[kBatch][kMaxSplits];
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r) {
          if (r >= p.splits) break;
          const uint32_t from = mapa_shared(base + c * C::PITCH * 4, r);
#pragma unroll
          for (int j = 0; j < kBatch; ++j)
            if (c + j * p.splits * C::EPI_W < count) v[j][r] = ld_cluster_v4f(from + j * p.splits * C::EPI_W * C::PITCH * 4);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int token = c + j * p.splits * C::EPI_W;
          if (token >= count) break;
          float4 sum = v[j][0];
#pragma unroll
          for (int r = 1; r < kMaxSplits; ++r) {
            if (r >= p.splits) break;
            sum.x += v[j][r].x;
            sum.y += v[j][r].y;
            sum.z += v[j][r].z;
            sum.w += v[j][r].w;
          }
          const float out[4] = {sum.x * scale, sum.y * scale, sum.z * scale, sum.w * scale};
          store_four(p, (m0 + token) * p.ldd + n4, min(4, p.n - n4), out);
        }
      }
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync();  // no CTA leaves while another reads its partial sums
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc<1>(tmem, C::TMEM);
  }
}

}  // namespace linear
}  // namespace bb

using namespace bb;
using namespace bb::linear;

struct bb_linear_plan {
  int kind = 0, device = 0;
  cudaStream_t stream = nullptr;
  bool few = false;
  int tn = 0;      // few rows: tokens of a tile
  int cg = 1;      // tiles: CTAs of a tile
  bool direct = false;
  CUtensorMap tm_a{}, tm_b{}, tm_sfa{}, tm_sfb{}, tm_d{};
  Params tile{};
  FewParams fp{};
  int grid = 0;
  int* status_dev = nullptr;
  int64_t launches = 0;
};

namespace {

constexpr int kMaxDevices = 64;

// Attributes are per device: one call per kernel and device.
template <typename K>
int allow_smem(K kernel, int bytes, int device, bool (&done)[kMaxDevices]) {
  if (device < kMaxDevices && done[device]) return BB_OK;
  BB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (device < kMaxDevices) done[device] = true;
  return BB_OK;
}

cudaLaunchConfig_t config(int grid, int threads, int smem, int cluster, bool dependent, cudaStream_t stream,
                          cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cfg;
}

template <int kKind, int kTN>
int launch_few(const bb_linear_plan& pl) {
  using C = FewCfg<kKind, kTN>;
  static bool done[kMaxDevices] = {};
  auto kernel = few_rows_kernel<kKind, kTN>;
  int rc = allow_smem(kernel, C::SMEM_BYTES, pl.device, done);
  if (rc != BB_OK) return rc;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(pl.grid, C::THREADS, C::SMEM_BYTES, pl.fp.splits, true, pl.stream, attr);
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, pl.tm_b, pl.tm_a, pl.tm_sfb, pl.tm_sfa, pl.fp),
                    "launch few_rows_kernel");
}

template <int kKind>
int launch_few_kind(const bb_linear_plan& pl) {
  switch (pl.tn) {
    case 16: return launch_few<kKind, 16>(pl);
    case 32: return launch_few<kKind, 32>(pl);
    case 64:
      if constexpr (is_fp4(kKind)) return launch_few<kKind, 64>(pl);
      [[fallthrough]];
    default: return launch_few<kKind, 128>(pl);
  }
}

// Clusters of `splits` CTAs that are resident at once: fewer than the SMs would
// hold of single CTAs, since a cluster's SMs are neighbours (148 SMs hold 74, 45,
// 33, 26, 22, 15 and 15 clusters of 2 to 8 CTAs). The query counts one CTA per SM.
// Asked once per kernel, device and size.
template <int kKind, int kTN>
int resident_clusters(int device, int sm_count, int splits, int* clusters) {
  using C = FewCfg<kKind, kTN>;
  static bool done[kMaxDevices] = {};
  static int known[kMaxDevices][kMaxSplits + 1] = {};
  if (device < kMaxDevices && known[device][splits]) {
    *clusters = known[device][splits];
    return BB_OK;
  }
  auto kernel = few_rows_kernel<kKind, kTN>;
  int rc = allow_smem(kernel, C::SMEM_BYTES, device, done);
  if (rc != BB_OK) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config(sm_count / splits * splits, C::THREADS, C::SMEM_BYTES, splits, false, nullptr, attr);
  BB_CUDA_TRY(cudaOccupancyMaxActiveClusters(clusters, kernel, &cfg));
  *clusters *= C::CTAS_PER_SM;
  if (device < kMaxDevices) known[device][splits] = *clusters;
  return BB_OK;
}

template <int kKind>
int resident_clusters_of(int tn, int device, int sm_count, int splits, int* clusters) {
  switch (tn) {
    case 16: return resident_clusters<kKind, 16>(device, sm_count, splits, clusters);
    case 32: return resident_clusters<kKind, 32>(device, sm_count, splits, clusters);
    case 64:
      if constexpr (is_fp4(kKind)) return resident_clusters<kKind, 64>(device, sm_count, splits, clusters);
      [[fallthrough]];
    default: return resident_clusters<kKind, 128>(device, sm_count, splits, clusters);
  }
}

template <int kKind, int kCG, bool kDirect>
int launch_tile(const bb_linear_plan& pl) {
  using C = Cfg<kKind, kCG>;
  static bool done[kMaxDevices] = {};
  auto kernel = bb_lowp_gemm_kernel<kKind, kCG, true, kDirect>;
  if (pl.device >= kMaxDevices || !done[pl.device]) {
    if constexpr (C::kRegSplit) {
      // setmaxnreg.inc waits until the block's register pool can serve it;
      // refuse to launch a build whose pool is smaller than the split needs.
      cudaFuncAttributes fa{};
      BB_CUDA_TRY(cudaFuncGetAttributes(&fa, kernel));
      if (fa.numRegs * C::THREADS < 128 * C::CTRL_REGS + 256 * C::EPI_REGS) {
        set_error("bb_linear: kernel built with %d registers per thread; its register split needs %d", fa.numRegs,
                  kLaunchRegs);
        return BB_ERR_INTERNAL;
      }
    }
    int rc = allow_smem(kernel, C::SMEM_BYTES, pl.device, done);
    if (rc != BB_OK) return rc;
  }
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(pl.grid, C::THREADS, C::SMEM_BYTES, kCG, true, pl.stream, attr);
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, pl.tm_a, pl.tm_b, pl.tm_sfa, pl.tm_sfb, pl.tm_d, pl.tile),
                    "launch bb_lowp_gemm_kernel");
}

// CTA pairs resident at once (SMs that have no partner in their GPC stay idle).
template <int kKind>
int resident_pairs(const bb_linear_plan& pl, int sm_count, int* pairs) {
  using C = Cfg<kKind, 2>;
  static int known[kMaxDevices] = {};
  if (pl.device < kMaxDevices && known[pl.device]) {
    *pairs = known[pl.device];
    return BB_OK;
  }
  static bool done[kMaxDevices] = {};
  auto kernel = bb_lowp_gemm_kernel<kKind, 2, true, false>;
  int rc = allow_smem(kernel, C::SMEM_BYTES, pl.device, done);
  if (rc != BB_OK) return rc;
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = config(sm_count / 2 * 2, C::THREADS, C::SMEM_BYTES, 2, false, pl.stream, attr);
  int n = 0;
  BB_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
  *pairs = n > 0 && n < sm_count / 2 ? n : sm_count / 2;
  if (pl.device < kMaxDevices) known[pl.device] = *pairs;
  return BB_OK;
}

template <int kKind>
int launch_kind(const bb_linear_plan& pl) {
  if (pl.few) return launch_few_kind<kKind>(pl);
  if (pl.cg == 2) return pl.direct ? launch_tile<kKind, 2, true>(pl) : launch_tile<kKind, 2, false>(pl);
  return pl.direct ? launch_tile<kKind, 1, true>(pl) : launch_tile<kKind, 1, false>(pl);
}

int launch_linear(const bb_linear_plan& pl) {
  if (pl.kind == kNvfp4) return launch_kind<kNvfp4>(pl);
  if (pl.kind == kMxfp4) return launch_kind<kMxfp4>(pl);
  return launch_kind<kFp8Group>(pl);
}

// Which kernel: the one for few rows up to 128 rows, and above as long as its
// 128 x 128 tiles are not more than the SMs. The tile kernel's 256 x 256 pairs
// would leave most SMs idle there (FP8, few against tiles: 256 x 4096 x 4096
// 12.1 us / 19.8, 512 x 1024 x 8192 12.3 / 35.2, 512 x 4096 x 4096 17.3 / 20.5;
// MXFP4 200 x 5000 x 2880 8.7 / 9.7), and is faster beyond (FP8 512 x 6144 x 4096
// 33.0 / 20.3, MXFP4 11.6 / 11.4).
bool use_few(int64_t m, int64_t rb_n, int sm_count) { return m <= 128 || rb_n * ((m + 127) / 128) <= sm_count; }

// K splits of the few-rows kernel. A split shortens a CTA's stream of K blocks and
// costs the exchange of the sums; never more CTAs than are resident at once, since
// a second wave costs half the kernel (NVFP4 1 x 8192 x 8192: 4 splits 8.6 us, 6
// 12.0; FP8 512 x 768 x 1536, 24 tiles at one CTA per SM, of which 22 clusters of 6
// fit: 13.5 us, 7.5 with 5 splits).
//
// FP8: one CTA per SM suffices for a short K; a second one keeps more of a long
// weight stream in flight (1 x 14336 x 4096: 1 split 14.4, 2 splits 12.9) where
// each still has kLongShare blocks. Sums of many tokens are read from at most six CTAs.
constexpr int kLongShare = 8;
int fp8_splits(int tn, int64_t units, int k_stages, const DeviceInfo& dev, int* splits) {
  const int ctas_per_sm = tn == 128 ? 1 : 2, most = tn > 32 ? 6 : kMaxSplits;
  // The largest number of splits up to `limit` whose clusters are all resident.
  auto fitting = [&](int64_t limit, int* s) -> int {
    *s = static_cast<int>(limit < most ? limit : most);
    for (; *s > 1; --*s) {
      int clusters = 0;
      const int rc = resident_clusters_of<kFp8Group>(tn, dev.device, dev.sm_count, *s, &clusters);
      if (rc != BB_OK) return rc;
      if (units <= clusters) return BB_OK;
    }
    *s = 1;
    return BB_OK;
  };
  auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  int one = 1, two = 1;
  int rc = fitting(least(dev.sm_count / units, k_stages / 2), &one);
  if (rc == BB_OK) rc = fitting(least(dev.sm_count * ctas_per_sm / units, k_stages / kLongShare), &two);
  *splits = one > two ? one : two;
  return rc;
}

// 4-bit formats: the splits that are estimated fastest, in us: 0.25 to 0.27 per K
// stage of a CTA, against an exchange whose time depends on the tile's tokens and
// grows with the CTAs, above all where SMs hold two of them. Fitted to 400 shapes
// (K 512 to 12288, N 128 to 5000, M 12 to 1100): 0.9 % longer than the best on
// average (12 % at worst), 6 % less than as many splits as the SMs take. MXFP4 60 x
// 5000 x 1024: 1 split 3.5, 2 splits 5.6; 60 x 1024 x 8192: 1, 4, 8 splits 10.6, 6.8,
// 5.8; 500 x 1024 x 12288: 1, 4, 6 splits 16.4, 9.1, 12.8. Where many tokens' tiles
// leave no choice but one split or shared SMs, a long stream of weights (16 MB and
// more) is faster through shared SMs (200 x 5000 x 12288: 1 split 21.1, 2 16.2, 3
// 15.4; 256 x 8192 x 8192, L2 cold: 24.6, 23.3).
template <int kKind>
int fp4_splits(int tn, int64_t units, int64_t rb_n, int k_stages, const DeviceInfo& dev, int* splits) {
  const bool stream = tn == 128 && 2 * units > dev.sm_count && rb_n * k_stages * 128 * ROW_BYTES >= (16 << 20);
  const float block = tn == 128 ? 0.27f : 0.25f;
  const float exchange = tn == 16 ? 0.6f : tn == 32 ? 0.8f : tn == 64 ? 2.0f : 1.9f;
  const float per_cta = (tn == 16 || tn == 32 ? 0.4f : tn == 64 ? 0.5f : 0.6f) / 100;
  const float shared_sms = tn == 16 ? 0.3f : tn == 32 ? 0.5f : tn == 64 ? 1.3f : stream ? 0.f : 3.0f;
  const int most = tn == 128 ? 6 : kMaxSplits;
  float least = 0.f;
  for (int s = 1; s <= most && s <= k_stages; ++s) {
    float t = static_cast<float>(k_stages) / s * block * (stream && s == 1 ? 1.3f : 1.f);
    if (s > 1) {
      int clusters = 0;
      const int rc = resident_clusters_of<kKind>(tn, dev.device, dev.sm_count, s, &clusters);
      if (rc != BB_OK) return rc;
      if (units > clusters) continue;
      t += exchange + static_cast<float>(units * s) * per_cta;
      if (2 * units > clusters) t += shared_sms;
    } else if (units > dev.sm_count) {
      t += shared_sms;
    }
    if (s == 1 || t < least) {
      least = t;
      *splits = s;
    }
  }
  return BB_OK;
}

// Estimated us of the FP8 few-rows kernel with tiles of tn tokens: the launch and
// its ends, the exchange of split sums, a time per K block of a CTA (half as much
// again where two CTAs share an SM) and the operand traffic from L2. Fitted to 518
// shapes (K 256 to 13584, N 64 to 5000, M 24 to 2048, FP8 weights in L2): what it
// chooses takes 0.6 % longer than the best of the three on average (19 % at worst),
// and 18 % less than tiles of 128 always: N x K = 256 x 4096, M = 200: tiles of
// 128 / 32 / 16 7.7 / 4.8 / 5.0 us; 512 x 640, 128: 6.2 / 4.7 / 3.8; 5000 x 2896, 64:
// 8.2 / 10.2 / 12.4; 4096 x 13584, 128: 18.4 / 37 / 57.
float fp8_few_time(int tn, int64_t m, int64_t units, int k_stages, int splits, int sm_count) {
  const int64_t ctas = units * splits, places = sm_count * (tn == 128 ? 1 : 2);
  const int64_t waves = (ctas + places - 1) / places;
  const float start = (tn == 128 ? 3.0f + 0.02f * (m < 128 ? m : 128) : tn == 32 ? 3.0f : 2.5f) + (splits > 1 ? 0.6f : 0.f);
  const float block = tn == 128 ? 0.30f : (tn == 32 ? 0.27f : 0.25f) * (ctas > sm_count ? 1.5f : 1.f);
  const float mbytes = units * k_stages * (128 + tn) * ROW_BYTES * 1e-6f;
  return start * (1 + 0.5f * (waves - 1)) + waves * (static_cast<float>(k_stages) / splits) * block + mbytes / 30.f;
}

// Estimated us of the tile kernel with tiles of a CTA pair (256 x 256) or of one
// CTA (128 x 256), in waves of the tiles that are resident at once, without what
// both have. A pair reads half of B per CTA and ends later; its tiles leave more
// of the last wave and of the rows below M empty. FP8 is bound by the promotion
// either way (us, pairs / single: 1453 x 2560 x 768 8.2 / 7.2, 526 x 12720 x 2240,
// 3 waves against 2, 31 / 23, 2537 x 12720 x 8192 equal); 4-bit tiles by the
// operands (1100 x 2560 x 768 6.6 / 6.0, 526 x 12720 x 768 9.6 / 8.0, x 2240 15.0 /
// 14.3, 1100 x 5120 x 2240 12.2 / 14.0, x 8192 25.8 / 35.2). Where rows do not begin
// on a 32-byte sector, every box of a row is one sector more, and single CTAs are
// bound by the operands sooner (FP8 1453 x 7680 x 1232 23.5 / 27.7, 7765 x 3200 x 528
// 29.2 / 32.3).
float tile_time(bool fp8, int cg, int64_t waves, int k_stages, bool sectors) {
  const float end = cg == 1 ? 0.f : fp8 ? 0.9f : 0.7f;
  const float stage = fp8 ? (cg == 2 ? 0.5f : 0.505f) : (cg == 2 ? 0.33f : 0.48f);
  return end + static_cast<float>(waves * k_stages) * stage * (cg == 1 && !sectors ? 1.3f : 1.f);
}

template <int kKind>
void few_info(int tn, bb_lowp_info* info) {
  auto set = [&](auto cfg) {
    using C = decltype(cfg);
    info->stages = C::STAGES;
    info->smem_bytes = C::SMEM_BYTES;
    info->tmem_columns = C::TMEM;
    info->threads_per_cta = C::THREADS;
  };
  switch (tn) {
    case 16: set(FewCfg<kKind, 16>{}); break;
    case 32: set(FewCfg<kKind, 32>{}); break;
    case 64:
      if constexpr (is_fp4(kKind)) {
        set(FewCfg<kKind, 64>{});
        break;
      }
      [[fallthrough]];
    default: set(FewCfg<kKind, 128>{}); break;
  }
}

template <int kKind>
void tile_info(int cg, bb_lowp_info* info) {
  info->stages = cg == 2 ? Cfg<kKind, 2>::STAGES : Cfg<kKind, 1>::STAGES;
  info->smem_bytes = cg == 2 ? Cfg<kKind, 2>::SMEM_BYTES : Cfg<kKind, 1>::SMEM_BYTES;
  info->tmem_columns = TMEM_COLS;
  info->threads_per_cta = Cfg<kKind, 1>::THREADS;
}

// The operands' tensor maps: 128-byte K rows of `box_rows` rows, and the scale
// atoms as rows of 8-byte words (one row per 128 operand rows).
int map_rows(CUtensorMap* tm, const void* data, int64_t row_bytes, int64_t rows, int box_rows) {
  const uint64_t dims[2] = {static_cast<uint64_t>(row_bytes), static_cast<uint64_t>(rows)};
  const uint64_t strides[1] = {static_cast<uint64_t>(row_bytes)};
  const uint32_t box[2] = {ROW_BYTES, static_cast<uint32_t>(box_rows)};
  return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 2, data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}
int map_atoms(CUtensorMap* tm, const void* atoms, int64_t atoms_k, int64_t blocks, int stage_atoms, int box_blocks) {
  const uint64_t dims[2] = {static_cast<uint64_t>(atoms_k) * 64, static_cast<uint64_t>(blocks)};
  const uint64_t strides[1] = {static_cast<uint64_t>(atoms_k) * 512};
  const uint32_t box[2] = {static_cast<uint32_t>(stage_atoms) * 64, static_cast<uint32_t>(box_blocks)};
  return encode_tiled(tm, CU_TENSOR_MAP_DATA_TYPE_UINT64, 8, 2, atoms, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE,
                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

}  // namespace

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
    const size_t d_size = d_dtype == BB_DTYPE_F32 ? 4 : 2;
    if (off(a, 16) || off(b, 16) || off(sfa, fp8 ? 4 : 16) || off(sfb, fp8 ? 4 : 16) || off(d, d_size) ||
        off(scale_a_dev, 4) || off(scale_b_dev, 4)) {
      set_error("bb_linear_plan_create: operands must be 16-byte aligned (FP8 scales 4), D to its type");
      return BB_ERR_ARGUMENT;
    }
    if (((m + 127) / 128) * ((n + 127) / 128) > 0x0fffffff) {
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
    const int64_t row_bytes = fp8 ? k : k / 2;
    const int64_t atoms_k = kind == BB_LOWP_NVFP4 ? (k + 63) / 64 : (k + 127) / 128;
    const int stage_atoms = kind == BB_LOWP_NVFP4 ? 4 : 2;
    const int64_t rb_m = (m + 127) / 128, rb_n = (n + 127) / 128;
    const int k_stages = static_cast<int>((row_bytes + ROW_BYTES - 1) / ROW_BYTES);
    h->few = use_few(m, rb_n, dev.sm_count);
    if (h->few) {
      // 4-bit: the narrowest tile that holds the tokens (a tile below 128 tokens
      // cannot start inside a 128-row scale block). FP8: what is estimated
      // fastest, of 64 tokens never (64 x 8192 x 8192: 18.4 us, the turned tiles
      // of 128 17.5; 61 x 5000 x 2896 9.5 and 8.9).
      FewParams& p = h->fp;
      if (!fp8) {
        h->tn = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;
        const int64_t units = rb_n * (rb_m > 1 ? rb_m : 1);
        rc = kind == kNvfp4 ? fp4_splits<kNvfp4>(h->tn, units, rb_n, k_stages, dev, &p.splits)
                            : fp4_splits<kMxfp4>(h->tn, units, rb_n, k_stages, dev, &p.splits);
      } else {
        float least = 0.f;
        for (int tn = 16; tn <= 128 && rc == BB_OK; tn = tn == 16 ? 32 : tn * 4) {
          const int64_t units = rb_n * (m > tn ? (m + tn - 1) / tn : 1);
          int splits = 1;
          rc = fp8_splits(tn, units, k_stages, dev, &splits);
          const float t = fp8_few_time(tn, m, units, k_stages, splits, dev.sm_count);
          if (tn == 16 || t < least) {
            least = t;
            h->tn = tn;
            p.splits = splits;
          }
          if (tn >= m) break;  // a wider tile holds no more
        }
      }
      if (rc != BB_OK) {
        delete h;
        return rc;
      }
      p.m = static_cast<int32_t>(m);
      p.n = static_cast<int32_t>(n);
      p.k_stages = k_stages;
      const int units = static_cast<int>(rb_n * (m > h->tn ? (m + h->tn - 1) / h->tn : 1));
      p.tiles_n = static_cast<int32_t>(rb_n);
      p.owned = (128 + p.splits - 1) / p.splits;
      p.sfa = static_cast<const float*>(sfa);
      p.sfb = static_cast<const float*>(sfb);
      p.sfa_ld = sfa_ld;
      p.ldd = ldd;
      p.scale = (scale_a_dev ? 1.f : scale_a) * (scale_b_dev ? 1.f : scale_b);
      p.scale_dev[0] = scale_a_dev;
      p.scale_dev[1] = scale_b_dev;
      p.d = d;
      p.d_dtype = d_dtype;
      h->grid = units * p.splits;
    } else {
      int pairs = 0;
      rc = kind == kNvfp4   ? resident_pairs<kNvfp4>(*h, dev.sm_count, &pairs)
           : kind == kMxfp4 ? resident_pairs<kMxfp4>(*h, dev.sm_count, &pairs)
                            : resident_pairs<kFp8Group>(*h, dev.sm_count, &pairs);
      if (rc != BB_OK) {
        delete h;
        return rc;
      }
      const int64_t tiles_n = (n + 255) / 256;
      auto time = [&](int cg, int64_t resident) {
        const int64_t tiles = (m + BM * cg - 1) / (BM * cg) * tiles_n;
        return tile_time(fp8, cg, (tiles + resident - 1) / resident, k_stages, row_bytes % 32 == 0);
      };
      h->cg = time(1, dev.sm_count) < time(2, pairs) ? 1 : 2;
      const int clusters = h->cg == 2 ? pairs : dev.sm_count;
      Params& p = h->tile;
      const int tile_m = BM * h->cg;
      p.m = static_cast<int32_t>(m);
      p.n = static_cast<int32_t>(n);
      p.k = static_cast<int32_t>(k);
      p.tiles_m = static_cast<int32_t>((m + tile_m - 1) / tile_m);
      p.tiles_n = static_cast<int32_t>(tiles_n);
      p.num_tiles = p.tiles_m * p.tiles_n;
      p.k_stages = k_stages;
      p.rb_m = static_cast<int32_t>(rb_m);
      p.rb_n = static_cast<int32_t>(rb_n);
      const int64_t g = kGroupABytes / (tile_m * row_bytes);
      p.group_m = static_cast<int32_t>(g < 1 ? 1 : g > p.tiles_m ? p.tiles_m : g);
      p.num_clusters = p.num_tiles < clusters ? p.num_tiles : clusters;
      p.sfa = static_cast<const uint8_t*>(sfa);
      p.sfb = static_cast<const uint8_t*>(sfb);
      p.global_scale = (scale_a_dev ? 1.f : scale_a) * (scale_b_dev ? 1.f : scale_b);
      p.scale_dev[0] = scale_a_dev;
      p.scale_dev[1] = scale_b_dev;
      p.sfa_ld = sfa_ld;
      p.ldd = ldd;
      p.d = static_cast<__nv_bfloat16*>(d);
      p.d_dtype = d_dtype;
      const bool rows16 = reinterpret_cast<uintptr_t>(d) % 16 == 0 && (ldd * d_size) % 16 == 0;
      // TMA stores want 16-byte rows; other types and strides are written from registers.
      h->direct = d_dtype != BB_DTYPE_BF16 || !rows16;
      h->grid = p.num_clusters * h->cg;
    }
    if (m > 0) {
      const int box_a = h->few ? h->tn : BM, box_b = h->few ? 128 : 256 / h->cg;
      rc = map_rows(&h->tm_a, a, row_bytes, m, box_a);
      if (rc == BB_OK) rc = map_rows(&h->tm_b, b, row_bytes, n, box_b);
      if (fp8) {
        h->tm_sfa = h->tm_a;  // unused: FP32 scales do not travel by TMA
        h->tm_sfb = h->tm_b;
      } else {
        if (rc == BB_OK) rc = map_atoms(&h->tm_sfa, sfa, atoms_k, rb_m, stage_atoms, 1);
        if (rc == BB_OK) rc = map_atoms(&h->tm_sfb, sfb, atoms_k, rb_n, stage_atoms, h->few ? 1 : 2);
      }
      h->tm_d = h->tm_a;
      if (rc == BB_OK && !h->few && !h->direct) {
        const uint64_t dims[2] = {static_cast<uint64_t>(n), static_cast<uint64_t>(m)};
        const uint64_t strides[1] = {static_cast<uint64_t>(ldd) * 2};
        const uint32_t box[2] = {64, 32};
        rc = encode_tiled(&h->tm_d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, 2, d, dims, strides, box,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE);
      }
      if (rc == BB_OK) rc = device_zeros(reinterpret_cast<void**>(&h->status_dev), sizeof(int), "allocation of the status word");
      if (rc != BB_OK) {
        if (h->status_dev) cudaFree(h->status_dev);
        delete h;
        return rc;
      }
    }
    h->fp.status = h->tile.status = h->status_dev;
    if (info) {
      *info = bb_lowp_info{};
      info->kind = kind;
      info->tile_m = h->few ? h->tn : BM * h->cg;
      info->tile_n = h->few ? 128 : 256;
      info->tile_k = fp8 ? 128 : 256;
      info->grid_ctas = m > 0 ? h->grid : 0;
      info->cta_group = h->cg;
      if (h->few) {
        info->num_tiles = h->grid / h->fp.splits;
        if (kind == kNvfp4) few_info<kNvfp4>(h->tn, info);
        else if (kind == kMxfp4) few_info<kMxfp4>(h->tn, info);
        else few_info<kFp8Group>(h->tn, info);
      } else {
        info->num_tiles = h->tile.num_tiles;
        if (kind == kNvfp4) tile_info<kNvfp4>(h->cg, info);
        else if (kind == kMxfp4) tile_info<kMxfp4>(h->cg, info);
        else tile_info<kFp8Group>(h->cg, info);
      }
      info->reserved[0] = h->few ? 1 : 0;
      info->reserved[1] = h->few ? h->fp.splits : 1;
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
    if (!plan->status_dev) return BB_OK;  // no rows
    DeviceGuard guard(plan->device);
    BB_CUDA_TRY(guard.status);
    for (int i = 0; i < iterations; ++i) {
      int rc = launch_linear(*plan);
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
  try {
    if (!plan) {
      set_error("bb_linear_synchronize: null plan");
      return BB_ERR_ARGUMENT;
    }
    DeviceGuard guard(plan->device);  // the default stream is the current device's
    BB_CUDA_TRY(guard.status);
    BB_CUDA_TRY(cudaStreamSynchronize(plan->stream));
    if (!plan->status_dev) return BB_OK;
    int st = 0;
    BB_CUDA_TRY(cudaMemcpy(&st, plan->status_dev, sizeof(int), cudaMemcpyDeviceToHost));
    if (st != 0) {
      set_error("linear kernel reported device status 0x%x (%s)", st,
                st == kDevBadLaunch ? "launch contract violated" : "a bounded wait timed out");
      return st == kDevBadLaunch ? BB_ERR_INTERNAL : BB_ERR_TIMEOUT;
    }
    return BB_OK;
  } catch (...) {
    set_error("bb_linear_synchronize: unexpected C++ exception");
    return BB_ERR_INTERNAL;
  }
}

BB_API int64_t bb_linear_launches(const bb_linear_plan* plan) { return plan ? plan->launches : -1; }

BB_API int bb_linear_destroy(bb_linear_plan* plan) {
  if (!plan) return BB_OK;
  int rc = BB_OK;
  if (plan->status_dev) rc = check_cuda(cudaFree(plan->status_dev), "cudaFree(status)");
  delete plan;
  return rc;
}

}  // extern "C"
