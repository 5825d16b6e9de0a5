// Products of microscaled 4-bit operands (formats: fp4.cuh):
//
//   y[m, n] = ta tb sum_blocks sa[m, block] sb[n, block] sum_{k in block} a[m, k] b[n, k]
//
// on the tensor cores' own block-scaled MMA (tcgen05.mma kind::mxf4nvf4 / kind::mxf4 .block_scale): codes straight from
// shared memory, block scales from TMEM, float32 accumulation of all of K. Nothing is unpacked or promoted.
//
// Two kernels: gemm_pair_kernel for many rows of a, gemm_few_kernel for few.
#include <atomic>
#include <cstddef>
#include <type_traits>

#include "fp4.cuh"
#include "fp4.h"
#include "fp4_tiles.h"
#include "w4a4_gemm.h"

namespace wdl {
namespace fp4 {

// Instruction descriptor of a block-scaled MMA of E2M1 operands, both K-major: the scales' type (0 E4M3, 1 E8M0) and
// the byte of each TMEM word where the two scales of a K = 64 step begin (0 or 2; E8M0 only).
__host__ __device__ constexpr uint32_t make_idesc_fp4(uint32_t m, uint32_t n, uint32_t scale_format, uint32_t byte) {
  return (byte << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (scale_format << 23) | ((m >> 4) << 24) | (byte << 29);
}

// Step kk of K = 64 in a stage: D[tmem] (+)= (A . scales A) (B . scales B)^T with M = m, N = n, by one CTA or a pair. The
// scales of the stage begin at ta and tb, a tile (four of E4M3 or of E8M0 a row) in step_a or step_b TMEM columns:
// nvfp4 takes a tile a step, mxfp4 half of one.
template <int kFmt, int kCtas>
__device__ __forceinline__ void mma_fp4(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t m, uint32_t n, int kk,
                                        uint32_t ta, int step_a, uint32_t tb, int step_b, uint32_t accumulate) {
#define WDL_MMA_FP4(GROUP, KIND)                                                                                  \
  asm volatile(                                                                                                   \
      "{\n\t.reg .pred p;\n\t"                                                                                    \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                                 \
      "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(tmem_d),      \
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate)                                     \
      : "memory")
  const int tile = kFmt == kNv ? kk : kk >> 1;
  const uint32_t sa = ta + step_a * tile, sb = tb + step_b * tile;
  const uint32_t idesc = kFmt == kNv ? make_idesc_fp4(m, n, 0, 0) : make_idesc_fp4(m, n, 1, (kk & 1) * 2);
  if constexpr (kFmt == kNv && kCtas == 1) WDL_MMA_FP4("1", "mxf4nvf4.block_scale.scale_vec::4X");
  if constexpr (kFmt == kNv && kCtas == 2) WDL_MMA_FP4("2", "mxf4nvf4.block_scale.scale_vec::4X");
  if constexpr (kFmt == kMx && kCtas == 1) WDL_MMA_FP4("1", "mxf4.block_scale.scale_vec::2X");
  if constexpr (kFmt == kMx && kCtas == 2) WDL_MMA_FP4("2", "mxf4.block_scale.scale_vec::2X");
#undef WDL_MMA_FP4
}

// One tile of scales (512 bytes of shared memory) into four TMEM columns, the same 32 lanes in each quarter; of a pair:
// each CTA's own shared memory at this offset into its own TMEM.
template <int kCtas>
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
  if constexpr (kCtas == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Descriptor of a tile of scales: 32 rows of 16 bytes, not swizzled, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_scales(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 16;
  d |= static_cast<uint64_t>(128u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  return d;
}

// A descriptor from its words: only the lower one, with the address, differs between the tiles of a kind.
__device__ __forceinline__ uint64_t desc64(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}

// 16 consecutive columns of this thread's lane, complete on return.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// ---- epilogue -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ float4 load4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }

// v = alpha v + bias for 32 consecutive columns; bias: 32 floats in shared memory, 16-byte aligned.
__device__ __forceinline__ void scaled32(float* v, float alpha, const float* bias) {
  const uint64_t a = pack2(alpha, alpha);
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(bias + j);
    unpack2(fma2(pack2(v[j], v[j + 1]), a, b.x), v[j], v[j + 1]);
    unpack2(fma2(pack2(v[j + 2], v[j + 3]), a, b.y), v[j + 2], v[j + 3]);
  }
}

// v = residual + gate v with the residual's row in a swizzled 32 x 32 tile of shared memory (stage32's layout); gate: 32
// floats, 16-byte aligned.
__device__ __forceinline__ void gated32(float (&v)[32], const uint8_t* buf, int lane, const float* gate) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const ulonglong2 r = *reinterpret_cast<const ulonglong2*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4));
    const ulonglong2 g = *reinterpret_cast<const ulonglong2*>(gate + 4 * j);
    unpack2(fma2(pack2(v[4 * j], v[4 * j + 1]), g.x, r.x), v[4 * j], v[4 * j + 1]);
    unpack2(fma2(pack2(v[4 * j + 2], v[4 * j + 3]), g.y, r.y), v[4 * j + 2], v[4 * j + 3]);
  }
}

// GELU in its tanh form of two values: x sigmoid(2 y) with y = sqrt(2 / pi) (x + 0.044715 x^3) is x / (1 + 2^a),
// a = -2 y log2 e. The special function unit's 16 results a cycle and SM are 4096 cycles a tile, less than its MMAs
// (K 3072: 6100); one reciprocal for two values, or half of the exponentials as polynomials, cost more instructions than
// they save and measured slower (61 and 65 against 59 us for the feed forward of 1392 x 3072 through 14336).
__device__ __forceinline__ void gelu2(float& x0, float& x1) {
  const uint64_t x = pack2(x0, x1), c1 = pack2(-2.3022082f, -2.3022082f), c2 = pack2(-0.10294324f, -0.10294324f);
  float a0, a1, d0, d1;
  unpack2(mul2(x, fma2(mul2(x, x), c2, c1)), a0, a1);
  unpack2(add2(pack2(ex2(a0), ex2(a1)), pack2(1.f, 1.f)), d0, d1);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d0));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d1));
  unpack2(mul2(x, pack2(d0, d1)), x0, x1);
}

template <int kMode>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  if constexpr (kMode == kEpiBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// 64 columns of the hidden layer as the next product's operand: GELU, the codes in w, the scale bytes returned. t: the
// hidden layer's tensor scale, inv_6t = 1 / (6 t). N % 32 == 0 in this mode, so that no block is cut.
template <int kFmt>
__device__ __forceinline__ uint32_t hidden64(float (&v)[64], uint32_t* w, float t, float inv_6t) {
  constexpr int B = block_columns(kFmt);
  uint32_t bytes = 0;
#pragma unroll
  for (int j = 0; j < 64; j += 2) gelu2(v[j], v[j + 1]);
  float amax[64 / B] = {};
#pragma unroll
  for (int j = 0; j < B; ++j)  // the blocks' maxima side by side
#pragma unroll
    for (int c = 0; c < 64 / B; ++c) amax[c] = max_nan(amax[c], fabsf(v[c * B + j]));
  BlockScale sc[64 / B];
  bool plain = true;
#pragma unroll
  for (int c = 0; c < 64 / B; ++c) {
    sc[c] = block_scale_near<kFmt>(amax[c], t, inv_6t);
    bytes |= sc[c].byte << (8 * c);
    plain = plain && sc[c].finite && sc[c].plain;
  }
  if (plain) {  // one branch for all columns: without it around each block the blocks' chains run side by side
#pragma unroll
    for (int j = 0; j < 64; j += 2) unpack2(mul2(pack2(v[j], v[j + 1]), pack2(sc[j / B].r, sc[j / B].r)), v[j], v[j + 1]);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = e2m1x8(v + 8 * j);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = encode8<kFmt>(v + 8 * j, sc[8 * j / B]);
  }
  return bytes;
}

__device__ __forceinline__ float epilogue_alpha(const Epilogue& ep) {
  return (ep.ta ? __ldg(ep.ta) : 1.f) * (ep.tb ? __ldg(ep.tb) : 1.f);
}

// ---- many rows ----------------------------------------------------------------------------------------------------
// A cluster of two CTAs (the two SMs of a TPC) computes tiles of 256 x 256 with 2-SM MMAs, persistently: pair p takes
// tiles p, p + pairs, ..., rows fastest. Each CTA holds its 128 rows of a, half of the tile's rows of w, its own rows'
// scales and all of w's: a stage of 256 columns of K brings 38 KB to each SM (nvfp4) for 512 cycles of MMA, where one
// CTA alone on 128 x 256 would need 54 KB, more than the 71 to 81 bytes a cycle that TMA brings to an SM here.
//   both CTAs, warps 0, 2  TMA producers of its own share; completions count on the first CTA's full[s]
//   first CTA, warp 1      MMA issuer: the stage's scales into both CTAs' TMEM (tcgen05.cp), then the MMAs; its commits
//                          arrive in both CTAs
//   both CTAs, warps 4-11  epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31 (its rows) and every second group of 32
//                          columns; results go through a swizzled buffer in shared memory to a TMA store
// TMEM has 512 columns and two accumulators of 256 would leave none for the scales: the accumulators overlap by 96
// columns, tile i in columns 0 .. 255 or 160 .. 415, scales in the last 96 (two stages). The epilogue drains the shared
// columns first, then hands the accumulator on: the next tile's MMAs wait for two loads of 32 columns a warp, not for
// the tile's stores.
constexpr int BM = 128, BN = 256, BK = 256;
constexpr int kThreads = 384;
constexpr uint32_t kTmemCols = 512, kAccStep = 160, kScaleCols = 416;

// Tiles of scales a 128-row block has in one stage.
__host__ __device__ constexpr int stage_tiles(int fmt) { return BK / tile_columns(fmt); }

// A TMA store of an epilogue warp: 32 rows x 64 columns of 16-bit values (128 bytes a row) or of codes (32 bytes), or
// 32 columns of float32 (128 bytes); each warp has two buffers of that, or one where two groups of columns share a store.
constexpr int store_columns(int mode) { return mode == kEpiF32 || mode == kEpiResidual ? 32 : 64; }
constexpr int buffer_bytes(int mode) { return mode == kEpiGelu ? 1024 : 4096; }
constexpr int buffers(int mode) { return mode == kEpiBf16 || mode == kEpiF16 ? 1 : 2; }

template <int kFmt, int kMode>
struct __align__(1024) Smem {
  static constexpr int T = stage_tiles(kFmt);
  static constexpr int kStages = store_columns(kMode) == 64 ? 5 : 4;
  uint8_t a[kStages][BM * BK / 2];
  uint8_t b[kStages][BM * BK / 2];
  uint8_t sa[kStages][T * kTileBytes];
  uint8_t sb[kStages][2 * T * kTileBytes];
  uint8_t out[8][buffers(kMode)][buffer_bytes(kMode)];
  float bias[2][BN];  // the tile's, of this tile and the next
  float gate[kMode == kEpiResidual ? 2 : 1][kMode == kEpiResidual ? BN : 4];
  uint64_t full[kStages];   // first CTA: both CTAs' shares of stage s have landed, and the scales' TMEM is free
  uint64_t empty[kStages];  // each CTA: the MMAs of stage s have completed
  uint64_t acc_full;        // each CTA: the tile's accumulator is complete
  uint64_t acc_empty;       // first CTA: both epilogues hold the columns that the next tile writes over
  uint64_t res_full[8][2];  // kEpiResidual: a warp's buffer holds its part of the residual
  uint64_t tmem_ready;      // first CTA: the second has allocated its TMEM
  uint64_t done;
  uint32_t tmem_base;
};

// A tile of shared memory to global memory through a tensor map; part of the thread's current bulk group.
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem_src, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(smem_src)), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// All but the last kPending groups of this thread have read their shared memory.
template <int kPending>
__device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kPending) : "memory");
}

// cluster_sync that orders no writes: every CTA of the cluster gets here before any goes on.
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Arrives on `bar` in both CTAs of the pair when every MMA this thread issued before has completed.
__device__ __forceinline__ void tc_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

// One lane's 32 values as (a half of) its row of a tile in the layout that a swizzled TMA store reads: float32, or the
// `half` of 64 16-bit values.
template <int kMode>
__device__ __forceinline__ void stage32(uint8_t* buf, int lane, int half, const float (&v)[32]) {
  if constexpr (store_columns(kMode) == 32) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pair16<kMode>(v[8 * j + 2 * i], v[8 * j + 2 * i + 1]);
      *reinterpret_cast<uint4*>(buf + lane * 128 + (((4 * half + j) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

// The word of column `lane` (float32) or of columns 2 lane, 2 lane + 1 (16 bits) in row r of such a tile.
__device__ __forceinline__ uint32_t* staged_word(uint8_t* buf, int r, int lane) {
  return reinterpret_cast<uint32_t*>(buf + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
}

// What TMA does for 32 columns of float32 or 64 of 16 bits from column x, 32 rows from row m0, for rows whose address or
// stride is not a multiple of 16 bytes: whole rows by the warp.
__device__ __forceinline__ void load_words(uint8_t* buf, const float* src, int ld, int lane, int m0, int x, int M, int N) {
  float f[32];  // all rows' loads under way at once
#pragma unroll
  for (int r = 0; r < 32; ++r) f[r] = m0 + r < M && x + lane < N ? src[static_cast<int64_t>(m0 + r) * ld + x + lane] : 0.f;
#pragma unroll
  for (int r = 0; r < 32; ++r) *staged_word(buf, r, lane) = __float_as_uint(f[r]);
  __syncwarp();
}
template <int kMode>
__device__ __forceinline__ void store_words(uint8_t* buf, void* dst, int ld, int lane, int m0, int x, int M, int N) {
  const int rows = min(32, M - m0);
  if constexpr (store_columns(kMode) == 32) {
    float* out = static_cast<float*>(dst) + static_cast<int64_t>(m0) * ld + x + lane;
    if (x + lane < N)
      for (int r = 0; r < rows; ++r, out += ld) *out = __uint_as_float(*staged_word(buf, r, lane));
  } else {
    const int n = x + 2 * lane;
    uint16_t* out = static_cast<uint16_t*>(dst) + static_cast<int64_t>(m0) * ld + n;
    const bool words = ((reinterpret_cast<uintptr_t>(dst) & 3) | (ld & 1)) == 0;  // x is even
    for (int r = 0; r < rows; ++r, out += ld) {
      const uint32_t w = *staged_word(buf, r, lane);
      if (words && n + 1 < N) {
        *reinterpret_cast<uint32_t*>(out) = w;
      } else {
        if (n < N) out[0] = static_cast<uint16_t>(w);
        if (n + 1 < N) out[1] = static_cast<uint16_t>(w >> 16);
      }
    }
  }
}

template <int kFmt, int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_sa, const __grid_constant__ CUtensorMap map_sb,
                     const __grid_constant__ CUtensorMap map_out, const __grid_constant__ CUtensorMap map_res,
                     const Epilogue ep, int M, int N, int K, int early_w, uint32_t* err) {
  extern __shared__ uint8_t smem_raw[];
  using S = Smem<kFmt, kMode>;
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int T = S::T, kStages = S::kStages;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int G = (K + BK - 1) / BK, bt = tiles_along(kFmt, K);
  const int m_pairs = (M + 2 * BM - 1) / (2 * BM), n_tiles = (N + BN - 1) / BN;
  const int tiles = m_pairs * n_tiles;
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);

  if (warp == 0 && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], 2);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_arrive(&sm.full[0]);  // the first two steps follow no MMAs
    mbar_arrive(&sm.full[1]);
    mbar_init(&sm.acc_full, 1);
    mbar_init(&sm.acc_empty, 16);
    for (int w = 0; w < 8; ++w) {
      mbar_init(&sm.res_full[w][0], 1);
      mbar_init(&sm.res_full[w][1], 1);
    }
    mbar_init(&sm.tmem_ready, 1);
    mbar_init(&sm.done, 1);
    fence_barrier_init();
    prefetch_tensor_map(&map_a);
    prefetch_tensor_map(&map_b);
    prefetch_tensor_map(&map_sa);
    prefetch_tensor_map(&map_sb);
    if (ep.vector) prefetch_tensor_map(&map_out);
    if (kMode == kEpiResidual && ep.vector) prefetch_tensor_map(&map_res);
  }
  __syncwarp();
  cluster_sync();  // both CTAs' barriers are initialized before any copy, commit or arrival reaches them
  // TMEM while the first copies are under way. The MMA issuer is the warp that allocates in the first CTA, and waits
  // for the second's; the epilogues read the address after a commit of MMAs that came after both.
  if (warp == 1) {
    tmem_alloc_pair(&sm.tmem_base, kTmemCols);
    tmem_relinquish_pair();
    __syncwarp();
    if (rank == 1 && lane == 0) mbar_arrive_cluster_relaxed(peer_smem(smem_u32(&sm.tmem_ready), 0));
  }

  if (warp == 0 || warp == 2) {
    if (lane == 0) {
      // ---------------- TMA producers: one thread for w and its scales, one for a and its (issuing a copy takes about
      // 100 cycles, and a stage has four)
      const bool for_w = warp == 0;
      const int steps = (tiles - pair + pairs - 1) / pairs * G;
      const uint32_t full0 = peer_smem(smem_u32(&sm.full[0]), 0);
      int t = pair, g = 0, s = 0;  // the next step: columns g BK of tile t, in stage s
      Tile tile = tile_of(t, m_pairs, n_tiles);
      auto load = [&] {
        if (for_w) {
          if (rank == 0) mbar_arrive_expect_tx(&sm.full[s], 2 * (BM * BK + 3 * T * kTileBytes));
          tma_load_2d_pair(sm.b[s], &map_b, full0 + 8 * s, g * (BK / 2), tile.n_tile * BN + rank * BM);
          tma_load_2d_pair(sm.sb[s], &map_sb, full0 + 8 * s, g * (T * kTileBytes / 8), tile.n_tile * 2);
        } else {
          const int m_tile = tile.m_pair * 2 + rank;
          tma_load_2d_pair(sm.a[s], &map_a, full0 + 8 * s, g * (BK / 2), m_tile * BM);
          tma_load_2d_pair(sm.sa[s], &map_sa, full0 + 8 * s, g * (T * kTileBytes / 8), m_tile);
        }
        if (++s == kStages) s = 0;
        if (++g == G) g = 0, t += pairs, tile = tile_of(t, m_pairs, n_tiles);
      };
      const int first = min(steps, kStages);
      int issued = 0;
      if (for_w && early_w)
        for (; issued < first; ++issued) load();
      grid_dependency_wait();  // the kernel before this one has finished
      if (for_w) grid_dependents_launch();
      for (; issued < first; ++issued) load();
      for (uint32_t phase = 0; issued < steps; ++issued) {
        const bool last = s == kStages - 1;
        if (!mbar_wait(&sm.empty[s], phase, err, kErrWaitEmpty)) break;
        load();
        phase ^= last;
      }
      if (rank == 0 && for_w)  // no copy of either CTA in flight at exit: all count on these barriers
        for (int j = max(0, issued - kStages); j < issued; ++j)
          mbar_wait(&sm.full[j % kStages], (j / kStages) & 1, err, kErrWaitFull);
    }
  } else if (warp == 1 && rank == 0) {
    // ---------------- MMA issuer. Its own instructions are what the tensor cores must not wait for: a stage is 512 cycles
    // of MMA and some 150 instructions of one warp, whose fetches share a cache with the epilogue's. The warp stays
    // together and elects one thread for a stage (the same loop in one lane alone ran 1.25 times longer), the loop is not
    // unrolled (over the stages: 750 cycles a stage), and a stage has one wait (with a second one 586, with one 507).
    const uint32_t tmem = sm.tmem_base;
    constexpr uint32_t kHiCodes = (1024u >> 4) | (1u << 14) | (2u << 29), kHiScales = (128u >> 4) | (1u << 14);
    bool ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.tmem_ready, 0, err, kErrWaitAccEmpty));
    const int whole = K / BK;  // stages without a partial step
    int s = 0, i = 0;
    uint32_t parity = 0, buffer = tmem + kScaleCols;
    for (int t = pair; t < tiles && ok; t += pairs, ++i) {
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.acc_empty, (i & 1) ^ 1, err, kErrWaitAccEmpty));
      const uint32_t acc = tmem + (i & 1) * kAccStep;
#pragma unroll 1
      for (int g = 0; g < G && ok; ++g) {
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.full[s], parity, err, kErrWaitFull));
        if (!ok) break;
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a0 = (smem_u32(sm.a[0]) >> 4) + (1u << 16) + s * (BM * BK / 2 / 16);
          const uint32_t b0 = a0 + static_cast<uint32_t>(offsetof(S, b) - offsetof(S, a)) / 16;
          const uint32_t sa0 = (smem_u32(sm.sa[0]) >> 4) + ((128u >> 4) << 16) + s * (T * kTileBytes / 16);
          const uint32_t sb0 = (smem_u32(sm.sb[0]) >> 4) + ((128u >> 4) << 16) + s * (2 * T * kTileBytes / 16);
          const uint32_t ta = buffer, tb = buffer + 4 * T;
          auto step = [&](int kk) {
            mma_fp4<kFmt, 2>(acc, desc64(a0 + 2 * kk, kHiCodes), desc64(b0 + 2 * kk, kHiCodes), 2 * BM, BN, kk, ta, 4, tb, 8,
                             g > 0 || kk > 0);
          };
          auto scales = [&](int j) {
            scales_to_tmem<2>(ta + 4 * j, desc64(sa0 + j * (kTileBytes / 16), kHiScales));
            scales_to_tmem<2>(tb + 8 * j, desc64(sb0 + j * (kTileBytes / 16), kHiScales));
            scales_to_tmem<2>(tb + 8 * j + 4, desc64(sb0 + (T + j) * (kTileBytes / 16), kHiScales));
          };
          if (g < whole) {
#pragma unroll
            for (int j = 0; j < T; ++j) scales(j);
#pragma unroll
            for (int kk = 0; kk < BK / 64; ++kk) step(kk);
          } else {
#pragma unroll 1
            for (int j = 0; j < bt - g * T; ++j) scales(j);
#pragma unroll 1
            for (int kk = 0; kk < (K - g * BK + 63) / 64; ++kk) step(kk);
          }
          tc_commit_both(&sm.empty[s]);
          // the step after next writes its scales over this one's: its full barrier waits for this one's MMAs as well
          tc_commit_pair(&sm.full[s + 2 < kStages ? s + 2 : s + 2 - kStages]);
          if (g == G - 1) tc_commit_both(&sm.acc_full);
        }
        __syncwarp();
        buffer ^= (tmem + kScaleCols) ^ (tmem + kScaleCols + 12 * T);
        if (++s == kStages) s = 0, parity ^= 1;
      }
    }
    if (elect_one()) tc_commit_pair(&sm.done);
    __syncwarp();
    mbar_wait(&sm.done, 0, err, kErrWaitAccFull);
  } else if (warp >= 4) {
    // ---------------- epilogue
    const int q = warp & 3, h = (warp - 4) >> 2, w = warp - 4;
    const uint32_t acc_empty0 = peer_smem(smem_u32(&sm.acc_empty), 0);
    grid_dependency_wait();  // nothing read or written here before the kernel before this one has finished
    const float alpha = epilogue_alpha(ep);
    const bool staged = ep.vector;  // TMA can read and write the rows
    const bool whole_rows = N % (store_columns(kMode) == 32 ? 4 : 8) == 0;  // they end on a 16-byte boundary
    const float t_hidden = kMode == kEpiGelu && ep.tout ? __ldg(ep.tout) : 1.f, inv_6t = 1.f / (6.f * t_hidden);
    bool ok = true;
    int i = 0, loads = 0, used = 0;  // buffers filled by loads of the residual, and by results
    for (int t = pair; t < tiles; t += pairs, ++i) {
      const Tile tile = tile_of(t, m_pairs, n_tiles);
      const int m0 = (tile.m_pair * 2 + rank) * BM + q * 32, n_tile = tile.n_tile, m = m0 + lane;
      // this warp's four groups of 32 columns, two neighbours at a time, in the order that frees the shared columns first
      auto column = [&](int j) { return ((i & 1 ? j >> 1 : 1 - (j >> 1)) * 4 + h * 2 + (j & 1)) * 32; };
      auto live = [&](int j) { return m0 < M && n_tile * BN + column(j) < N; };  // the same in all lanes
      int next = 0;  // the next group to load the residual of
      auto load_residual = [&] {
        while (next < 4 && !live(next)) ++next;
        if (next == 4) return;
        if (lane == 0) {
          const int b = loads & 1;
          bulk_wait_read<0>();  // the stores from the buffer have read it
          mbar_arrive_expect_tx(&sm.res_full[w][b], 4096);
          tma_load_2d(sm.out[w][b], &map_res, &sm.res_full[w][b], n_tile * BN + column(next), m0);
        }
        ++loads, ++next;
      };
      if constexpr (kMode == kEpiResidual)
        if (staged && ok) {
          load_residual();
          load_residual();
        }
      // the tile's bias, and its gate where its rows share one, into shared memory behind the main loop. A warp can be
      // one tile ahead of another, not two: two copies.
      const int mine = static_cast<int>(threadIdx.x) - 128, n = n_tile * BN + mine;
      sm.bias[i & 1][mine] = ep.bias && n < N ? __ldg(ep.bias + n) : 0.f;
      bool shared_gate = false;
      if constexpr (kMode == kEpiResidual) {
        const int first_row = min(m0 - q * 32, M - 1), last_row = min(m0 - q * 32 + BM - 1, M - 1);
        shared_gate = !ep.gate || first_row / ep.rows_per_group == last_row / ep.rows_per_group;
        if (shared_gate)
          sm.gate[i & 1][mine] = !ep.gate ? 1.f : n < N ? __ldg(ep.gate + static_cast<int64_t>(first_row / ep.rows_per_group) * ep.ld_gate + n) : 0.f;
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // the epilogue's warps
      // after a wait that ran out a warp does no more than meet the others here
      ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(&sm.acc_full, i & 1, err, kErrWaitAccFull));
      if (!ok) continue;
      tc_fence_after();
      const uint32_t t_row = *static_cast<volatile uint32_t*>(&sm.tmem_base) + (static_cast<uint32_t>(q * 32) << 16) + (i & 1) * kAccStep;
#pragma unroll 1
      for (int half = 0; half < 2 && ok; ++half) {
        uint32_t r[2][32];
        tmem_ld32(t_row + column(2 * half), r[0]);
        tmem_ld32(t_row + column(2 * half + 1), r[1]);
        tmem_ld_wait(r[0]);
        tmem_ld_wait(r[1]);
        if (half == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster_relaxed(acc_empty0);  // it hands over no write: the loads are complete
        }
        if (!live(2 * half)) continue;
        if constexpr (kMode == kEpiGelu) {
          // 64 columns at once; those past N (the second group of the last tile's may be) are zeros and not stored
          const int x = n_tile * BN + column(2 * half);
          const bool second = live(2 * half + 1);
          float v[64];
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(r[0][c]), v[32 + c] = second ? __uint_as_float(r[1][c]) : 0.f;
          scaled32(v, alpha, sm.bias[i & 1] + column(2 * half));
          scaled32(v + 32, alpha, sm.bias[i & 1] + column(2 * half) + 32);
          uint32_t c4[8];
          uint32_t scales = hidden64<kFmt>(v, c4, t_hidden, inv_6t);
          if (!second) scales &= kFmt == kNv ? 0xFFFFu : 0xFFu;
          uint8_t* buf = sm.out[w][used & 1];
          ++used;
          if (lane == 0) bulk_wait_read<1>();  // the last store from this buffer has read it
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<uint4*>(buf + lane * 32 + ((k ^ ((lane >> 2) & 1)) << 4)) =
                make_uint4(c4[4 * k], c4[4 * k + 1], c4[4 * k + 2], c4[4 * k + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&map_out, buf, x / 2, m0);
            bulk_commit();
          }
          // 64 columns of nvfp4 are a whole word of a scale tile's row (its padding, if N ends inside, zeros); of mxfp4 half
          if (m < M) {
            uint8_t* scale = ep.out_scales + scale_offset(m, x / block_columns(kFmt), tiles_along(kFmt, N));
            if constexpr (kFmt == kNv) {
              *reinterpret_cast<uint32_t*>(scale) = scales;
            } else {
              *reinterpret_cast<uint16_t*>(scale) = static_cast<uint16_t>(scales);
              if (x + 64 >= N && (N + 127) / 128 * 128 - x > 64) *reinterpret_cast<uint16_t*>(scale + 2) = 0;
            }
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int j = 2 * half + k, n0 = n_tile * BN + column(j);
            const bool alive = live(j);
            float v[32];
#pragma unroll
            for (int c = 0; c < 32; ++c) v[c] = __uint_as_float(r[k][c]);
            scaled32(v, alpha, sm.bias[i & 1] + column(j));
            uint8_t* buf = sm.out[w][used & (buffers(kMode) - 1)];
            constexpr bool kJoined = store_columns(kMode) == 64;  // both groups leave in one store
            if constexpr (kMode == kEpiResidual) {
              if (!alive || !ok) continue;
              if (staged)
                ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.res_full[w][used & 1], (used >> 1) & 1, err, kErrWaitFull));
              else
                load_words(buf, ep.residual, ep.ld_res, lane, m0, n0, M, N);
              if (!ok) continue;
              if (shared_gate) {
                gated32(v, buf, lane, sm.gate[i & 1] + column(j));
              } else {
                const float* gate = ep.gate + static_cast<int64_t>(min(m, M - 1) / ep.rows_per_group) * ep.ld_gate + n0;
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                  const float r = *reinterpret_cast<const float*>(buf + lane * 128 + (((c >> 2) ^ (lane & 7)) << 4) + (c & 3) * 4);
                  v[c] = fmaf(n0 + c < N ? __ldg(gate + c) : 0.f, v[c], r);
                }
              }
            } else if (!kJoined || k == 0) {
              if (!kJoined && !alive) continue;
              if (lane == 0) bulk_wait_read<buffers(kMode) - 1>();  // the last store from this buffer has read it
              __syncwarp();
            }
            stage32<kMode>(buf, lane, k, v);
            if (kJoined && k == 0) continue;
            ++used;
            const int x = n_tile * BN + column(kJoined ? 2 * half : j);
            fence_proxy_async_smem();
            __syncwarp();
            // TMA cuts a store at N only to 16 bytes (N 31 of 16 bits with rows of 32: it wrote the 32nd)
            if (staged && (x + store_columns(kMode) <= N || whole_rows)) {
              if (lane == 0) {
                tma_store_2d(&map_out, buf, x, m0);
                bulk_commit();
              }
            } else {
              store_words<kMode>(buf, ep.out, ep.ld_out, lane, m0, x, M, N);
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) bulk_commit();  // an empty group: the waits count a group for every use of a buffer
            }
            if constexpr (kMode == kEpiResidual)
              if (staged) load_residual();
          }
        }
      }
    }
    if (lane == 0) bulk_wait_read<0>();  // the buffers outlive their readers; the kernel's end completes the writes
    __syncwarp();
  }

  tc_fence_before();
  __syncwarp();
  cluster_meet();  // neither CTA leaves while the other's MMAs, copies or arrivals may still reach it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(sm.tmem_base, kTmemCols);
  }
}

// ---- few rows epilogue --------------------------------------------------------------------------------------------
// Features n .. n + 3 of row m < M, from a warp that holds 128 neighbouring ones: v after alpha and bias. All lanes call it.
template <int kFmt, int kMode>
__device__ __forceinline__ void finish4(const Epilogue& ep, float4 v, int m, int n, int N, float t, float inv_6t) {
  if constexpr (kMode == kEpiGelu) {
    gelu2(v.x, v.y);
    gelu2(v.z, v.w);
    float amax = n < N ? max_nan(max_nan(fabsf(v.x), fabsf(v.y)), max_nan(fabsf(v.z), fabsf(v.w))) : 0.f;
    constexpr int B = block_columns(kFmt);
#pragma unroll
    for (int o = 1; o < B / 4; o *= 2) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const BlockScale sc = block_scale_near<kFmt>(amax, t, inv_6t);
    float q[8] = {v.x, v.y, v.z, v.w, 0.f, 0.f, 0.f, 0.f};
    uint32_t w;
    if (sc.finite && sc.plain) {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] *= sc.r;
      w = e2m1x8(q);
    } else {
      w = encode8<kFmt>(q, sc);
    }
    // the scales of a tile's row (4 B columns): its first lane collects them; blocks past N have 0
    uint32_t word = n < N ? sc.byte : 0u;
    word |= __shfl_down_sync(0xFFFFFFFFu, word, B / 4) << 8;
    word |= __shfl_down_sync(0xFFFFFFFFu, word, B / 2) << 16;
    if (n >= N) return;
    *reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(ep.out) + static_cast<int64_t>(m) * (N / 2) + n / 2) = static_cast<uint16_t>(w);
    if (n % (4 * B) == 0)
      *reinterpret_cast<uint32_t*>(ep.out_scales + scale_offset(m, n / B, tiles_along(kFmt, N))) = word;
  } else {
    if (n >= N) return;
    const bool whole = ep.vector && n + 4 <= N;
    const int64_t at = static_cast<int64_t>(m) * ep.ld_out + n;
    float f[4] = {v.x, v.y, v.z, v.w};
    if constexpr (kMode == kEpiResidual) {
      const float* res = ep.residual + static_cast<int64_t>(m) * ep.ld_res + n;  // may be out itself: an ordinary load
      const float* gate = ep.gate ? ep.gate + static_cast<int64_t>(m / ep.rows_per_group) * ep.ld_gate + n : nullptr;
      if (whole) {
        const float4 r = *reinterpret_cast<const float4*>(res);
        const float4 g = gate ? __ldg(reinterpret_cast<const float4*>(gate)) : make_float4(1.f, 1.f, 1.f, 1.f);
        f[0] = fmaf(g.x, f[0], r.x), f[1] = fmaf(g.y, f[1], r.y), f[2] = fmaf(g.z, f[2], r.z), f[3] = fmaf(g.w, f[3], r.w);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < N) f[j] = fmaf(gate ? __ldg(gate + j) : 1.f, f[j], res[j]);
      }
    }
    if constexpr (kMode == kEpiF32 || kMode == kEpiResidual) {
      float* out = static_cast<float*>(ep.out) + at;
      if (whole) {
        *reinterpret_cast<float4*>(out) = make_float4(f[0], f[1], f[2], f[3]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < N) out[j] = f[j];
      }
    } else {
      uint16_t* out = static_cast<uint16_t*>(ep.out) + at;
      const uint32_t w[2] = {pair16<kMode>(f[0], f[1]), pair16<kMode>(f[2], f[3])};
      if (whole) {
        *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < N) out[j] = static_cast<uint16_t>(w[j / 2] >> (16 * (j & 1)));
      }
    }
  }
}

// ---- few rows -----------------------------------------------------------------------------------------------------
// With few rows of a the weights' bytes are the floor: N K (1/2 + 1/16 or 1/32), read once. The operands change places:
// 128 rows of w are the MMA's M, 16 to 128 rows of a its N, so that the tensor cores take the stream as it comes (no lane
// unpacks a code) and the accumulator has one TMEM column a row of a. K is split over the CTAs of a cluster; each leaves
// its part [NT][128] in its shared memory, and the rows are shared out: CTA r adds row r, r + S, ... of all parts in the
// ranks' order (the same bits every time) and finishes it. Two CTAs an SM.
//   warp 0      TMA producer (the weights' first stages before it waits for the kernel that writes a)
//   warp 1      TMEM owner and MMA issuer
//   warps 2-5   epilogue: warp w reads TMEM lanes 32 (w % 4) .. + 31
// kRaw, one row: it comes as 16- or 32-bit values, and warps 2-5 quantize the CTA's share of it into the stages themselves:
// one launch instead of two (K 3072, N 18432: 7.2 against 8.5 us with the quantizer's launch; 1024 x 1024: 3.8 against 4.4;
// 14336 x 14336: 22.9 either way). Every CTA of the 128-feature tiles does the same row again, by four warps that hide
// little of a division's latency: with 4 rows it was 10.2 against 8.5 us, with 16 rows 25 against 8.5.
constexpr int kFewThreads = 192;
constexpr uint32_t kFewTmemCols = 256;
constexpr int few_stages(int nt) { return nt == 16 ? 5 : 3; }

// NT: the MMA's N. A CTA takes kRows of them: all, or (64 of 128) the first or the second half of a 128-row block, whose
// scales are one tile: the other half's columns of the accumulator hold nothing and are not read.
template <int kFmt, int NT>
struct __align__(1024) FewSmem {
  static constexpr int kStages = few_stages(NT);
  static constexpr int T = stage_tiles(kFmt);
  uint8_t w[kStages][128 * 128];
  uint8_t x[kStages][NT * 128];
  uint8_t sw[kStages][T * kTileBytes];
  uint8_t sx[kStages][T * kTileBytes];
  float bias[128];
  uint64_t full[kStages];
  uint64_t empty[kStages];
  uint64_t done;
  uint32_t tmem_base;
};

__device__ __forceinline__ float4 load_cluster(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr));
  return v;
}

// Rows rank, rank + splits, ... of all CTAs' parts added in the ranks' order and finished: the fourth of them that warp w
// of four takes, 4 features a lane, as many rows at once as there is room for loads under way. kMax >= splits.
template <int kFmt, int kMode, int kMax>
__device__ __forceinline__ void finish_parts(const Epilogue& ep, const float* part, const float* bias, float alpha, int rows,
                                             int rank, int splits, int w, int lane, int m_base, int n, int N) {
  constexpr int kRows = 8 / kMax;
  const uint32_t base = smem_u32(part) + lane * 16;
  const float t = kMode == kEpiGelu && ep.tout ? __ldg(ep.tout) : 1.f, inv_6t = 1.f / (6.f * t);
  const float4 b = *reinterpret_cast<const float4*>(bias + lane * 4);
  for (int m0 = rank + w * splits; m0 < rows; m0 += 4 * kRows * splits) {
    float4 p[kRows][kMax];
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int r = 0; r < kMax; ++r) {
        const int m = m0 + 4 * i * splits;
        if (r < splits && m < rows) p[i][r] = load_cluster(peer_smem(base + m * 512, r));
      }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int m = m0 + 4 * i * splits;
      if (m >= rows) break;
      float4 v = p[i][0];
#pragma unroll
      for (int r = 1; r < kMax; ++r)
        if (r < splits) v.x += p[i][r].x, v.y += p[i][r].y, v.z += p[i][r].z, v.w += p[i][r].w;
      v.x = fmaf(v.x, alpha, b.x), v.y = fmaf(v.y, alpha, b.y), v.z = fmaf(v.z, alpha, b.z), v.w = fmaf(v.w, alpha, b.w);
      finish4<kFmt, kMode>(ep, v, m_base + m, n, N, t, inv_6t);
    }
  }
}

// 8 columns of a row as they lie in memory: 16 bytes of 16-bit values, 32 of float32.
struct Raw8 {
  uint4 lo, hi;
};
__device__ __forceinline__ Raw8 load_raw8(const RawRow& x, int k) {
  const uint8_t* p = static_cast<const uint8_t*>(x.p) + static_cast<int64_t>(k) * (x.dtype == 2 ? 4 : 2);
  Raw8 r;
  r.lo = __ldg(reinterpret_cast<const uint4*>(p));
  r.hi = x.dtype == 2 ? __ldg(reinterpret_cast<const uint4*>(p) + 1) : r.lo;
  return r;
}
__device__ __forceinline__ void raw8_values(const Raw8& r, int dtype, float (&v)[8]) {
  const uint32_t w[8] = {r.lo.x, r.lo.y, r.lo.z, r.lo.w, r.hi.x, r.hi.y, r.hi.z, r.hi.w};
  if (dtype == 2) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else if (dtype == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}

// One warp's part of quantizing a single row's columns g0 BK .. (g0 + G) BK - 1 (zeros past K) into the ring of stages, in
// the layout that TMA would leave there: warp w of four takes every fourth stage, 8 columns a lane, the next ones on their
// way from memory meanwhile. It arrives on every full[] (four of five arrivals); false after a wait that ran out.
template <int kFmt, typename S>
__device__ __forceinline__ bool quantize_stages(S& sm, const RawRow& x, float t, int g0, int G, int K, int w, int lane,
                                                uint32_t* err) {
  constexpr int B = block_columns(kFmt), kAhead = 2;
  Raw8 ahead[kAhead];
  auto fetch = [&](int i) {
    const int k = (g0 + i) * BK + lane * 8;
    return i < G && k < K ? load_raw8(x, k) : Raw8{};
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) ahead[j] = fetch(w + 4 * j);
  bool ok = true;
  int at = 0;  // the first stage that this warp has not arrived for
  auto free_slot = [&](int i) {  // the MMAs of the stage that was there have completed
    ok = ok && (i < S::kStages ||
                __all_sync(0xFFFFFFFFu, mbar_wait(&sm.empty[i % S::kStages], (i / S::kStages - 1) & 1, err, kErrWaitEmpty)));
  };
  auto arrive = [&](int to) {  // for the stages before `to`: what this warp has to do with them is done
    for (; at < to && ok; ++at) {
      free_slot(at);
      if (ok && lane == 0) mbar_arrive(&sm.full[at % S::kStages]);
    }
  };
  arrive(min(w, G));
  for (int first = w; first < G && ok; first += 4 * kAhead) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int i = first + 4 * j, s = i % S::kStages;
      if (i >= G || !ok) break;
      float v[8], amax = 0.f;
      raw8_values(ahead[j], x.dtype, v);
      ahead[j] = fetch(i + 4 * kAhead);
#pragma unroll
      for (int c = 0; c < 8; ++c) amax = max_nan(amax, fabsf(v[c]));
#pragma unroll
      for (int o = 1; o < B / 8; o *= 2) amax = max_nan(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
      const BlockScale sc = block_scale<kFmt>(amax, t);
      const uint32_t codes = encode8<kFmt>(v, sc);
      free_slot(i);
      if (!ok) break;
      *reinterpret_cast<uint32_t*>(sm.x[s] + lane * 4) = codes;  // row 0 of a swizzled tile
      const int block = lane * 8 / B;
      if (lane * 8 % B == 0)
        sm.sx[s][(block >> 2) * kTileBytes + (block & 3)] = (g0 + i) * BK + lane * 8 < K ? static_cast<uint8_t>(sc.byte) : 0;
      fence_proxy_async_smem();
      __syncwarp();
      arrive(min(G, i + 4));
    }
  }
  return ok;
}

template <int kFmt, int kMode, int NT, int kRows, bool kRaw>
__global__ void __launch_bounds__(kFewThreads, 2)
    gemm_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
                    const uint8_t* __restrict__ w_scales, const uint8_t* __restrict__ x_scales, const RawRow raw,
                    const Epilogue ep, int M, int N, int K, int early_w, uint32_t* err) {
  extern __shared__ uint8_t smem_raw[];
  using S = FewSmem<kFmt, NT>;
  // the same offset in every CTA of the cluster: remote addresses are made from local ones
  S& sm = *reinterpret_cast<S*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr int T = S::T, kStages = S::kStages;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_ctarank()), splits = static_cast<int>(cluster_nctas());
  const int n_tile = blockIdx.x / splits, m0 = blockIdx.y * kRows;
  const int skip = kRows < NT ? m0 % NT : 0;  // rows of the block before this CTA's
  const int all = (K + BK - 1) / BK, bt = tiles_along(kFmt, K);
  const int g0 = all * rank / splits, G = all * (rank + 1) / splits - g0;  // this CTA's stages

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&sm.full[s], kRaw ? 5 : 1);
      mbar_init(&sm.empty[s], 1);
    }
    mbar_init(&sm.done, 1);
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensor_map(&map_w);
    if (!kRaw) prefetch_tensor_map(&map_x);
  }
  if (warp == 1) {
    tmem_alloc(&sm.tmem_base, kFewTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem_base;

  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer
      auto scale_bytes = [&](int i) { return static_cast<uint32_t>(min(T, bt - (g0 + i) * T)) * kTileBytes; };
      auto load_w = [&](int i) {
        const int s = i % kStages, g = g0 + i;
        mbar_arrive_expect_tx(&sm.full[s], 128 * 128 + scale_bytes(i) + (kRaw ? 0 : kRows * 128 + scale_bytes(i)));
        tma_load_2d(sm.w[s], &map_w, &sm.full[s], g * 128, n_tile * 128);
        bulk_load(sm.sw[s], w_scales + (static_cast<int64_t>(n_tile) * bt + g * T) * kTileBytes, scale_bytes(i),
                  &sm.full[s]);
      };
      auto load_x = [&](int i) {
        if constexpr (kRaw) return;
        const int s = i % kStages, g = g0 + i;
        tma_load_2d(sm.x[s] + skip * 128, &map_x, &sm.full[s], g * 128, m0);
        bulk_load(sm.sx[s], x_scales + (static_cast<int64_t>(m0 / 128) * bt + g * T) * kTileBytes, scale_bytes(i),
                  &sm.full[s]);
      };
      const int first = min(G, kStages);
      if (early_w)
        for (int i = 0; i < first; ++i) load_w(i);
      grid_dependency_wait();  // the kernel before this one has finished
      grid_dependents_launch();
      for (int i = 0; i < first; ++i) {
        if (!early_w) load_w(i);
        load_x(i);
      }
      int issued = first;
      for (int i = first; i < G; ++i) {
        if (!mbar_wait(&sm.empty[i % kStages], ((i / kStages) & 1) ^ 1, err, kErrWaitEmpty)) break;
        load_w(i);
        load_x(i);
        issued = i + 1;
      }
      for (int i = max(0, issued - kStages); i < issued; ++i)  // no copy in flight at exit
        mbar_wait(&sm.full[i % kStages], (i / kStages) & 1, err, kErrWaitFull);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------- MMA issuer
    for (int i = 0; i < G; ++i) {
      const int s = i % kStages, g = g0 + i;
      ok = __all_sync(0xFFFFFFFFu, mbar_wait(&sm.full[s], (i / kStages) & 1, err, kErrWaitFull));
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t w0 = smem_u32(sm.w[s]), x0 = smem_u32(sm.x[s]);
        const uint32_t sw0 = smem_u32(sm.sw[s]), sx0 = smem_u32(sm.sx[s]);
        const uint32_t tw = tmem + NT + s * (8 * T), tx = tw + 4 * T;
        const int live = min(T, bt - g * T);
        for (int j = 0; j < live; ++j) {
          scales_to_tmem<1>(tw + 4 * j, smem_desc_scales(sw0 + j * kTileBytes));
          scales_to_tmem<1>(tx + 4 * j, smem_desc_scales(sx0 + j * kTileBytes));
        }
        const int steps = min(BK / 64, (K - g * BK + 63) / 64);
        for (int kk = 0; kk < steps; ++kk)
          mma_fp4<kFmt, 1>(tmem, smem_desc_k128(w0 + kk * 32), smem_desc_k128(x0 + kk * 32), 128, NT, kk, tw, 4, tx, 4,
                           i > 0 || kk > 0);
        tc_commit(&sm.empty[s]);
      }
      __syncwarp();
    }
    if (elect_one()) tc_commit(&sm.done);
    __syncwarp();
    mbar_wait(&sm.done, 0, err, kErrWaitAccFull);
  }

  // ---------------- epilogue: the parts into shared memory (over the stages, all of them read by now)
  float* part = reinterpret_cast<float*>(sm.w[0]);
  const int rows = min(kRows, M - m0);
  float alpha = 1.f;
  if (warp >= 2) {
    grid_dependency_wait();  // nothing read or written here before the kernel before this one has finished
    if constexpr (kRaw) ok = quantize_stages<kFmt>(sm, raw, ep.ta ? __ldg(ep.ta) : 1.f, g0, G, K, warp - 2, lane, err);
    alpha = epilogue_alpha(ep);
    const int t = static_cast<int>(threadIdx.x) - 64, n = n_tile * 128 + t;  // t: a feature of the tile
    sm.bias[t] = ep.bias && n < N ? __ldg(ep.bias + n) : 0.f;
    ok = ok && __all_sync(0xFFFFFFFFu, mbar_wait(&sm.done, 0, err, kErrWaitAccFull));
    tc_fence_after();
    const int q = warp & 3;
    if (ok) {
#pragma unroll 1
      for (int c = 0; c < rows; c += 16) {
        uint32_t r[16];
        tmem_ld16(tmem + (static_cast<uint32_t>(q * 32) << 16) + skip + c, r);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * 128 + q * 32 + lane] = __uint_as_float(r[j]);
      }
    }
  }
  tc_fence_before();
  cluster_sync();
  if (warp >= 2 && ok) {
    auto finish = [&](auto most) {
      finish_parts<kFmt, kMode, decltype(most)::value>(ep, part, sm.bias, alpha, rows, rank, splits, warp - 2, lane,
                                                       m0, n_tile * 128 + lane * 4, N);
    };
    if (splits == 1) finish(std::integral_constant<int, 1>{});
    else if (splits == 2) finish(std::integral_constant<int, 2>{});
    else if (splits <= 4) finish(std::integral_constant<int, 4>{});
    else finish(std::integral_constant<int, 8>{});
  }
  cluster_meet();  // no CTA leaves while another may still read its part
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kFewTmemCols);
  }
}

static bool make_map(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t columns, uint64_t rows,
                     uint64_t row_bytes, uint32_t box_columns, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[2] = {columns, rows};
  const cuuint64_t strides[1] = {row_bytes};
  const cuuint32_t box[2] = {box_columns, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return encode_tiled(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Codes in boxes of 256 columns (128 bytes).
static bool codes_map(CUtensorMap* map, const uint8_t* codes, int K, int rows, uint32_t box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, codes, K / 2, rows, K / 2, 128, box_rows,
                  CU_TENSOR_MAP_SWIZZLE_128B);
}

// Tiles of scales in boxes of one stage x `blocks` 128-row blocks (8-byte elements: a box is at most 256 wide).
static bool scales_map(CUtensorMap* map, const uint8_t* scales, int K, int rows, int fmt, uint32_t blocks) {
  const uint64_t row = static_cast<uint64_t>(tiles_along(fmt, K)) * kTileBytes;
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT64, scales, row / 8, (rows + 127) / 128, row,
                  stage_tiles(fmt) * kTileBytes / 8, blocks, CU_TENSOR_MAP_SWIZZLE_NONE);
}

// The attributes a kernel needs before its first launch on a device, set once per device (by every thread that gets here
// before the first has: the same values).
template <typename Kernel>
static cudaError_t allow_smem(Kernel kernel, int bytes, int dev, std::atomic<bool> (&done)[64]) {
  if (dev >= 0 && dev < 64 && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true, std::memory_order_relaxed);
  return e;
}

// cluster: CTAs a cluster (0: what the kernel declares). The launch may begin while the kernel before it on the stream
// still runs; the kernels wait for that one before they read or write what it could have to do with.
template <typename Kernel, typename... Args>
static cudaError_t launch(Kernel kernel, dim3 grid, int threads, int bytes, int cluster, cudaStream_t s, Args... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = bytes, c.stream = s;
  cudaLaunchAttribute at[2];
  c.attrs = at;
  if (cluster) {
    at[c.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[c.numAttrs].val.clusterDim.x = cluster, at[c.numAttrs].val.clusterDim.y = 1, at[c.numAttrs].val.clusterDim.z = 1;
    ++c.numAttrs;
  }
  at[c.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[c.numAttrs].val.programmaticStreamSerializationAllowed = 1;
  ++c.numAttrs;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

struct Device {
  int id, sms;
};

// The tensor maps of a launch: codes of a and w, and for many rows the scales, the output and the residual.
struct Maps {
  CUtensorMap a, b, sa, sb, out, res;
};

template <int kFmt, int kMode>
static cudaError_t launch_many(const GemmArgs& g, const Maps& m, Device d, cudaStream_t s) {
  static std::atomic<bool> done[64] = {};
  auto kernel = gemm_pair_kernel<kFmt, kMode>;
  using S = Smem<kFmt, kMode>;
  static_assert(sizeof(S) + 1024 <= 232448, "shared memory of the stages");
  static_assert(kScaleCols + 2 * 12 * S::T <= kTmemCols, "TMEM columns of the scales");
  const int bytes = static_cast<int>(sizeof(S)) + 1024;
  const cudaError_t e = allow_smem(kernel, bytes, d.id, done);
  if (e != cudaSuccess) return e;
  const int64_t tiles = static_cast<int64_t>((g.M + 2 * BM - 1) / (2 * BM)) * ((g.N + BN - 1) / BN);
  const unsigned pairs = static_cast<unsigned>(tiles < d.sms / 2 ? tiles : d.sms / 2);
  return launch(kernel, dim3(2 * pairs), kThreads, bytes, 0, s, m.a, m.b, m.sa, m.sb, m.out, m.res, g.ep, g.M, g.N, g.K,
                static_cast<int>(g.early_w), g.err);
}

template <int kFmt, int kMode, int NT, int kRows, bool kRaw>
static cudaError_t launch_few(const GemmArgs& g, const Maps& m, Device d, cudaStream_t s) {
  static std::atomic<bool> done[64] = {};
  auto kernel = gemm_few_kernel<kFmt, kMode, NT, kRows, kRaw>;
  using S = FewSmem<kFmt, NT>;
  static_assert(2 * (sizeof(S) + 2048) <= 228 * 1024, "two CTAs an SM");
  static_assert(NT + S::kStages * 8 * S::T <= static_cast<int>(kFewTmemCols), "TMEM columns");
  static_assert(NT * 512 <= S::kStages * (128 + NT) * 128, "the parts fit over the stages");
  const int bytes = static_cast<int>(sizeof(S)) + 1024;
  const cudaError_t e = allow_smem(kernel, bytes, d.id, done);
  if (e != cudaSuccess) return e;
  const int n_tiles = (g.N + 127) / 128, m_tiles = (g.M + kRows - 1) / kRows, stages = (g.K + BK - 1) / BK;
  // K in as many parts as clusters of that many CTAs can all run at once, and in no more than make the longest part
  // shorter. Clusters that do not all fit cost a second wave: 72 tiles in 4 parts (70 clusters of 4 fit) took 7.4 us,
  // in 2 parts 5.0 (N 9216, K 3072, one row).
  static std::atomic<int> room[64][9] = {};
  const int dev = d.id >= 0 && d.id < 64 ? d.id : 0;
  int splits = 1;
  for (int n = 2; n <= 8 && n <= stages; ++n) {
    int fit = room[dev][n].load(std::memory_order_relaxed);
    if (fit == 0) {
      cudaLaunchConfig_t c = {};
      cudaLaunchAttribute at;
      at.id = cudaLaunchAttributeClusterDimension;
      at.val.clusterDim.x = n, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
      c.gridDim = dim3(n), c.blockDim = dim3(kFewThreads), c.dynamicSmemBytes = bytes, c.attrs = &at, c.numAttrs = 1;
      int clusters = 0;
      if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &c) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();  // the query is advisory
        clusters = d.sms / n;
      }
      // the query counts one CTA an SM here where shared memory, registers and TMEM hold two
      int blocks = 1;
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, kFewThreads, bytes) != cudaSuccess) cudaGetLastError();
      fit = blocks >= 2 ? clusters : 2 * clusters;
      room[dev][n].store(fit, std::memory_order_relaxed);
    }
    if (static_cast<int64_t>(n_tiles) * m_tiles <= fit) splits = n;
  }
  const int share = (stages + splits - 1) / splits;
  splits = (stages + share - 1) / share;
  return launch(kernel, dim3(n_tiles * splits, m_tiles), kFewThreads, bytes, splits, s, m.b, m.a, g.b_scales, g.a_scales, g.raw, g.ep, g.M,
                g.N, g.K, static_cast<int>(g.early_w), g.err);
}

template <int kFmt, int kMode>
static cudaError_t launch_mode(const GemmArgs& g, const Maps& m, int few, Device d, cudaStream_t s) {
  if (few == 16)
    return g.raw.p ? launch_few<kFmt, kMode, 16, 16, true>(g, m, d, s) : launch_few<kFmt, kMode, 16, 16, false>(g, m, d, s);
  if (few == 64)
    return g.M <= 64 ? launch_few<kFmt, kMode, 64, 64, false>(g, m, d, s) : launch_few<kFmt, kMode, 128, 64, false>(g, m, d, s);
  if (few == 128) return launch_few<kFmt, kMode, 128, 128, false>(g, m, d, s);
  return launch_many<kFmt, kMode>(g, m, d, s);
}

template <int kFmt>
static cudaError_t launch_fmt(const GemmArgs& g, const Maps& m, int few, Device d, cudaStream_t s) {
  switch (g.mode) {
    case kEpiBf16: return launch_mode<kFmt, kEpiBf16>(g, m, few, d, s);
    case kEpiF16: return launch_mode<kFmt, kEpiF16>(g, m, few, d, s);
    case kEpiF32: return launch_mode<kFmt, kEpiF32>(g, m, few, d, s);
    case kEpiResidual: return launch_mode<kFmt, kEpiResidual>(g, m, few, d, s);
    default: return launch_mode<kFmt, kEpiGelu>(g, m, few, d, s);
  }
}

static bool make_maps(Maps& m, const GemmArgs& g, int few) {
  if (few) return (g.raw.p || codes_map(&m.a, g.a, g.K, g.M, few)) && codes_map(&m.b, g.b, g.K, g.N, 128);
  bool ok = codes_map(&m.a, g.a, g.K, g.M, BM) && codes_map(&m.b, g.b, g.K, g.N, BM) &&
            scales_map(&m.sa, g.a_scales, g.K, g.M, g.fmt, 1) && scales_map(&m.sb, g.b_scales, g.K, g.N, g.fmt, 2);
  if (!g.ep.vector) return ok;
  if (g.mode == kEpiGelu)  // the next product's codes
    return ok && make_map(&m.out, CU_TENSOR_MAP_DATA_TYPE_UINT8, g.ep.out, g.N / 2, g.M, g.N / 2, 32, 32, CU_TENSOR_MAP_SWIZZLE_32B);
  const bool wide = g.mode == kEpiF32 || g.mode == kEpiResidual;
  const CUtensorMapDataType type = wide ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  ok = ok && make_map(&m.out, type, g.ep.out, g.N, g.M, static_cast<uint64_t>(g.ep.ld_out) * (wide ? 4 : 2), wide ? 32 : 64,
                      32, CU_TENSOR_MAP_SWIZZLE_128B);
  if (g.mode == kEpiResidual)
    ok = ok && make_map(&m.res, type, g.ep.residual, g.N, g.M, static_cast<uint64_t>(g.ep.ld_res) * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  return ok;
}

// Up to 64 rows the few-row kernel is the faster one (N 14336, K 3072: 8.2 against 8.9 us at 64 rows, 9.5 against 8.5 at
// 96). Beyond, 64 rows a CTA where these are few enough for K to be split, two thirds of the SMs (128 rows: 4.4 against 5.5
// us for N 512, K 1024, 7.2 against 7.9 for N 3072, K 3072, 5.7 against 13.2 for N 512, K 8192; 256 rows, 96 CTAs: 7.7
// against 7.9 for N 3072, K 3072). Where K is long, two thirds as many: CTAs of 128 rows read w less often (K 14336, N
// 3072: 10.9 against 12.0 us at 128 rows, 13.7 against 13.0 at 160), and are taken as long as their parts find room beside
// each other (18.1 against the many-row kernel's 21.5 us at 384 rows, 22.2 against 21.5 at 512).
int gemm_rows_per_cta(int M, int N, int K, int sms) {
  const int64_t n128 = (static_cast<int64_t>(N) + 127) / 128, tiles64 = (static_cast<int64_t>(M) + 63) / 64 * n128;
  const int64_t tiles128 = (static_cast<int64_t>(M) + 127) / 128 * n128;
  if (M <= 16) return 16;
  if (M <= 64 || tiles64 * (K > 8192 ? 3 : 2) * 3 <= sms * 4) return 64;
  return K > 15 * BK && tiles128 * 3 <= sms * 9 / 5 ? 128 : 0;
}

int gemm_launch(const GemmArgs& g, cudaStream_t s, const char** why) {
  Device d{0, 148};
  if (cudaGetDevice(&d.id) == cudaSuccess) cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, d.id);
  const int few = gemm_rows_per_cta(g.M, g.N, g.K, d.sms);
  Maps m{};
  if (!make_maps(m, g, few)) {
    *why = "cuTensorMapEncodeTiled rejected an operand (alignment or stride)";
    return 2;
  }
  const cudaError_t e = g.fmt == kNv ? launch_fmt<kNv>(g, m, few, d, s) : launch_fmt<kMx>(g, m, few, d, s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    *why = cudaGetErrorString(e);
    return 3;
  }
  return 0;
}

}  // namespace fp4
}  // namespace wdl
