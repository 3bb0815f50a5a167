// Products of 4-bit activations and a 4-bit filter on the tensor cores:
//   y[row][oc] = sum_k a[row][k] w[oc][k] (+ bias, ReLU)
// tcgen05.mma with block scales: kind::mxf4 (32 values a scale, E8M0) and kind::mxf4nvf4 (16 a scale,
// E4M3), both 64 values of K per instruction, FP32 accumulators in tensor memory.
//
// What bounds it.  Large products: clocks of an SM, 230 to 260 for each MMA of N = 256 that could take 128, at any clock
// rate (205 without loads and copies of scales: operands from shared memory), and 1.1 to 1.6 us from tile to tile.  The
// clock falls as the card reaches 1000 W: 4096x4096x16384 MX takes 131 us at 1.95 GHz (the first 300 calls after a
// pause, 4.2 PFLOP/s) and 151 at 1.55 to 1.6 GHz (6000 calls in a row, 3.65 PFLOP/s), 8192x4096x8192 NV 136 and 157.
// Few rows: 2 us of launch, first loads and cluster meeting, then the filter at 5.2 TB/s (1x4096x4096 MX 3.7 us,
// 16x8192x8192 NV 9.3).  Hundreds of rows: the K steps one after the other, 0.36 us each, and 3 us beside them
// (333x2048x1000 NV 6.0 us).  Layers with few columns: the writing of the output (50176x64x256: 11.1 us, 4.8 TB/s).
//
// Which operand is on the M side (128 lanes of tensor memory) depends on the number of rows.
//   Few rows: the filter, D[oc][row].  16 to 64 rows cost a narrow N instead of an empty M; a lane is a channel,
//   and 32 lanes store 32 neighbouring values of an output row.
//   Many rows: the rows, D[row][oc].  A lane then holds neighbouring values of its row; a warp stages 32 rows x 128
//   bytes, which leave as whole lines through a TMA store (each lane storing its own 32 bytes: 3.5 TB/s against 4.9).
// Roles:
//   * warp 0 (one thread): per K step of 256 TMA loads of the tile's codes (rows of 128 bytes, or 64 or 32 where K ends
//     there, swizzled over as much, zeros past both ends) and bulk copies of the scales, into one ring;
//   * warp 1 (one elected lane): scales from shared into tensor memory (tcgen05.cp), then 4 MMAs;
//   * eight storing warps: accumulator -> scale, bias, ReLU -> output, beside the next tile's MMAs.
// Rows that are not quantised yet (DIRECT): before the storing warps store a tile they turn its rows into codes and
// scales in shared memory, K step by K step, while the filter is on its way.
// Tensor memory: two accumulators (one for 128 columns in half an SM).  With N = 256 two of them and the scales
// exceed 512 columns, so the second one lies over the end of the first; the storing warps empty the shared columns
// first and the next tile starts once those are free.
// Scales lie in slots of tensor memory that are written again only when the MMAs that read them are done.
// Few tiles: the K range is cut over a cluster of up to 8 CTAs, whose sums are copied into the shared memory of the
// CTA that owns a column (one bulk copy per owner, counted on its barrier) and added in slice order: bit-reproducible,
// no workspace.
// Every barrier wait is bounded; on a timeout an error flag is raised, all roles stop, what the CTA has in flight lands,
// tensor memory is freed and the kernel returns; tetris_fp4_filter_check reports it.  A role whose wait gave up neither
// arrives at nor commits to a barrier again: a stage is then never sent for while its last phase is open, and the phases
// that the end of the kernel waits for are those of the loads in flight.
// Tried and dropped: pairs of CTAs on a tile of 256 x 256 (cta_group::2, each stage's arrival passed on to the CTA that
// issues: 173 us for 4096x4096x16384 against 138), scales copied a step ahead of the MMAs (181), warps of their own that
// quantise rows of large layers (50176x64x256 15.5 us against 19.4 in two launches, 12544x256x512 20.1 against 12.5).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "fp4.h"
#include "fp4_block.h"

namespace tetris {
namespace {

constexpr int kM = 128;                  // lanes of a tile
constexpr int kStep = 256;               // K values of a step: 128 bytes of codes (one step of 64 or 32 where K is at most 128 or 64)
constexpr int kStoreWarps = 8, kFirstStore = 2, kThreads = 32 * (kFirstStore + kStoreWarps);
constexpr int kStagesMax = 8, kSlotsMax = 8;
constexpr int kBars = 2 * kStagesMax + 8;
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kSumPitch = kM + 4;        // floats between the columns of a cluster's sums (whole 16 bytes)
constexpr int kBiasBytes = kStoreWarps * 64 * 4;
constexpr int kStageOut = 4096;          // a staging block: 32 rows of 128 bytes on their way to the output
// Scale tiles (512 bytes, 128 rows x 4 blocks) of a K step
__host__ __device__ constexpr int step_tiles(int format) { return format == TETRIS_FP4_NV ? 4 : 2; }

struct ProductParams {
  const uint8_t *scales_m, *scales_n;
  const float *bias;
  void *y;
  int64_t ld;
  int m_extent, n_extent;  // rows and channels, or channels and rows
  int m_blocks, n_blocks;  // 128-row blocks of either side's scales
  int steps, last_mmas;    // K steps; MMAs of the last one
  int row_log;             // log2 of the bytes of a row in a stage
  uint32_t codes_high;     // high word of the codes' descriptors
  int tiles_k;             // scale tiles of a 128-row block
  int nt;                  // N of the MMAs
  int m_tiles, n_tiles, group;  // tiles; M tiles that are walked side by side
  Fp4Div by_per, by_group, by_last;  // tiles of a group of M tiles; its M tiles; those of the last group
  int total_tiles;
  int d, per_log;          // CTAs of a cluster = slices of a tile's K range; log2 of the columns a CTA owns
  int stages, slots;
  int stage_bytes, n_at, sm_at, sn_at;  // a stage: codes of M and N, scales of M and N
  int tmem_cols;
  int accs, acc1, sf, slot_cols; // accumulators; columns of the second one, the scales, of a slot of them
  float scale, scale1;     // 2^(sum of the exponents), as two factors where one would leave FP32
  const void *x;           // activations that are not quantised yet
  int x_type, x_vec, K;
  int64_t x_ld;
  Fp4Pixels px;            // (S > 1: a row is a pixel of a strided layer)
  Fp4Div by_OH, by_OW;
  int lx, unit_log;        // log2 of the lanes of a row, of the units (32 lanes) of a tile's rows in a K step
  float tensor_scale, sixth, sixth_rest;  // as in the quantisation
  int relu;
  int tma_store;           // D[row][oc]: the output takes TMA stores (16-byte aligned rows of whole 16 bytes)
  int staging;             // ... staging blocks of a storing warp: 1 or 2
  int *error_flag;
  unsigned spin_limit;
  int withhold_first_load; // failure-detection test only
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
// Bounded wait.  Gives up when the limit (abort_flag[1]) is hit or when another role already gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint32_t limit = (uint32_t)abort_flag[1];
  for (uint32_t i = 1; i < limit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63) == 63) {
      if (*abort_flag) return false;
      __nanosleep(32);
    }
  }
  *abort_flag = 1;
  return false;
}
// After a give-up: wait (bounded) for an asynchronous operation that was started earlier.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < (1u << 16); ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 63) == 63) __nanosleep(64);
  }
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Descriptors of shared memory, low word; the high words are constants.
// K-major codes in rows of 128, 64 or 32 bytes swizzled over as much, 8-row groups together
__host__ __device__ constexpr uint32_t codes_high(int row_log) { return (8u << row_log >> 4) | (1u << 14) | ((row_log == 7 ? 2u : row_log == 6 ? 4u : 6u) << 29); }
// a scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart
constexpr uint32_t kScalesHigh = 8u | (1u << 14);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr) { return ((saddr >> 4) & 0x3FFFu) | (1u << 16); }
// 512 bytes of scales into 4 columns of all four lane quarters
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t desc) {
  asm volatile("{\n.reg .b64 d;\nmov.b64 d, {%1, %2};\ntcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n}" ::"r"(taddr), "r"(desc), "n"(kScalesHigh) : "memory");
}
template <int FMT>
__device__ __forceinline__ void umma_fp4(uint32_t tmem_d, uint32_t da, uint32_t db, uint32_t high, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
#define TETRIS_FP4_MMA(KIND)                                                                                              \
  asm volatile("{\n.reg .pred p;\n.reg .b64 a, b;\nmov.b64 a, {%1, %7};\nmov.b64 b, {%2, %7};\nsetp.ne.b32 p, %6, 0;\n"  \
               "tcgen05.mma.cta_group::1.kind::" KIND " [%0], a, b, %3, [%4], [%5], p;\n}"                                 \
               ::"r"(tmem_d), "r"(da), "r"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(high) : "memory")
  if (FMT == TETRIS_FP4_NV) TETRIS_FP4_MMA("mxf4nvf4.block_scale.scale_vec::4X");
  else TETRIS_FP4_MMA("mxf4.block_scale.scale_vec::2X");
#undef TETRIS_FP4_MMA
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
                 "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
                 "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
                 "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
               : "r"(taddr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// (whole warps, whatever a role's lanes did before)
__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {  // `addr` of this CTA in CTA `rank` of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// shared memory of this CTA into another one's, counted on a barrier there
__device__ __forceinline__ void push(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "r"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(c0), "r"(c1) : "memory");
}
template <typename T> __device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 to_type(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half to_type(float v) { return __float2half_rn(v); }

// Tile t: M tiles in groups of `group`, within a group all N tiles, within an N tile the group's M tiles: CTAs
// that run side by side share both operands.
__device__ __forceinline__ void decode(const ProductParams &p, int t, int &m0, int &n0) {
  const int g = (int)fp4_quot((uint32_t)t, p.by_per), r = t - g * (int)p.by_per.d;
  const Fp4Div &w = (g + 1) * p.group <= p.m_tiles ? p.by_group : p.by_last;
  const int n = (int)fp4_quot((uint32_t)r, w);
  m0 = (g * p.group + r - n * (int)w.d) * kM;
  n0 = n * p.nt;
}

__device__ __forceinline__ float finish(uint32_t v, float scale, float bias, int relu) {
  float u = fmaf(__uint_as_float(v), scale, bias);  // (the product by a power of two is exact)
  if (relu) asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(u));
  return u;
}

// 8 neighbouring values of a row, zeros behind the last one.
__device__ __forceinline__ void load8(const ProductParams &p, int64_t at, int left, float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = 0.f;
  if (p.x_type == TETRIS_FP32) {
    const float *x = static_cast<const float *>(p.x) + at;
    if (p.x_vec && left >= 8) {
      *reinterpret_cast<float4 *>(v) = reinterpret_cast<const float4 *>(x)[0];
      *reinterpret_cast<float4 *>(v + 4) = reinterpret_cast<const float4 *>(x)[1];
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < left) v[k] = x[k];
    }
    return;
  }
  const uint16_t *x = static_cast<const uint16_t *>(p.x) + at;
  alignas(16) uint16_t h[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (p.x_vec && left >= 8) {
    *reinterpret_cast<uint4 *>(h) = *reinterpret_cast<const uint4 *>(x);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < left) h[k] = x[k];
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = p.x_type == TETRIS_BF16 ? __uint_as_float((uint32_t)h[k] << 16) : __half2float(__ushort_as_half(h[k]));
}

// DIRECT: the rows are quantised here (with the filter on the M side at most 64 at a time, else 128).
template <int FMT, typename T, bool ROWS_M, bool DIRECT>
__global__ void __launch_bounds__(kThreads, 2)
product_kernel(const __grid_constant__ CUtensorMap map_m, const __grid_constant__ CUtensorMap map_n, const __grid_constant__ CUtensorMap map_y,
               const ProductParams p) {
  constexpr int kTiles = step_tiles(FMT);
  extern __shared__ unsigned char smem_raw[];
  unsigned char *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  // behind the ring: staging blocks (D[row][oc]), or, for d > 1, the sums of this CTA's columns [slice][column][kSumPitch]
  unsigned char *staging = ring + (size_t)p.stages * p.stage_bytes;
  float *sums = reinterpret_cast<float *>(staging);
  float *bias_rows = reinterpret_cast<float *>(staging + (p.d > 1 ? p.nt * kSumPitch * 4 : kStoreWarps * kStageOut * p.staging));
  uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(bias_rows) + kBiasBytes);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);  // a wait gave up; polls of a wait; K steps sent for
  // (the warp number as a value that is the same in all lanes for the compiler, too: what the tensor core is told
  // can then be worked out in uniform registers; 4096x4096x16384 147 -> 144 us)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  auto bar_full = [&](int s) { return smem_u32(&bars[s]); };
  auto bar_empty = [&](int s) { return smem_u32(&bars[kStagesMax + s]); };
  auto bar_pfull = [&](int b) { return smem_u32(&bars[2 * kStagesMax + b]); };
  auto bar_pempty = [&](int b) { return smem_u32(&bars[2 * kStagesMax + 2 + b]); };
  auto bar_shared = [&](int b) { return smem_u32(&bars[2 * kStagesMax + 4 + b]); };
  auto bar_drain = [&]() { return smem_u32(&bars[2 * kStagesMax + 6]); };
  auto bar_sums = [&]() { return smem_u32(&bars[2 * kStagesMax + 7]); };

  const int rank = p.d > 1 ? (int)(blockIdx.x & (p.d - 1)) : 0;
  const int tile0 = p.d > 1 ? blockIdx.x / p.d : blockIdx.x, tile_step = p.d > 1 ? gridDim.x / p.d : gridDim.x;
  const int step0 = p.d > 1 ? (int)((int64_t)p.steps * rank / p.d) : 0, step1 = p.d > 1 ? (int)((int64_t)p.steps * (rank + 1) / p.d) : p.steps;
  const int rt = p.nt > 128 ? 2 : 1;       // 128-row blocks of a tile's N scales
  const bool over = p.accs == 2 && p.acc1 < p.nt;  // the accumulators share columns
  const int acc_log = p.accs - 1;          // tile i uses accumulator i & acc_log, for the (i >> acc_log)-th time
  const int ahead = min(step1 - step0, p.stages);
  int loads = 0;
  int m0, n0;

  // Bytes of a step: both code boxes whole (zeros past the ends count), the scale tiles that exist.  The filter
  // does not change while kernels run, the activations may until grid_wait.
  auto scale_tiles = [&](int step) { return min(kTiles, p.tiles_k - step * kTiles); };
  auto load_m = [&](uint32_t at, uint32_t bar, int step) {
    tma_load_2d(at, &map_m, bar, step * 128, m0);
    bulk_load(at + p.sm_at, p.scales_m + ((size_t)(m0 / 128) * p.tiles_k + (size_t)step * kTiles) * 512, scale_tiles(step) * 512, bar);
  };
  auto load_n = [&](uint32_t at, uint32_t bar, int step) {
    const int b0 = n0 / 128, blocks = min(rt, p.n_blocks - b0);
    tma_load_2d(at + p.n_at, &map_n, bar, step * 128, n0);
    for (int b = 0; b < blocks; ++b)
      bulk_load(at + p.sn_at + b * (kTiles * 512), p.scales_n + ((size_t)(b0 + b) * p.tiles_k + (size_t)step * kTiles) * 512, scale_tiles(step) * 512, bar);
  };
  auto load_filter = [&](int s, int step) {
    const uint32_t at = smem_u32(ring + (size_t)s * p.stage_bytes), bar = bar_full(s);
    mbar_expect_tx(bar, DIRECT ? (uint32_t)(((ROWS_M ? p.nt : kM) << p.row_log) + scale_tiles(step) * 512)
                               : (uint32_t)(((kM + p.nt) << p.row_log) + scale_tiles(step) * 512 * (1 + min(rt, p.n_blocks - n0 / 128))));
    if (ROWS_M) load_n(at, bar, step); else load_m(at, bar, step);
  };
  auto load_rows = [&](int s, int step) {
    const uint32_t at = smem_u32(ring + (size_t)s * p.stage_bytes), bar = bar_full(s);
    if (loads++ == 0 && p.withhold_first_load) return;
    if (DIRECT) return;
    if (ROWS_M) load_m(at, bar, step); else load_n(at, bar, step);
  };

  if (tid == 0) {
    for (int s = 0; s < kStagesMax; ++s) { mbar_init(bar_full(s), DIRECT ? 1 + kStoreWarps : 1); mbar_init(bar_empty(s), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(bar_pfull(b), 1); mbar_init(bar_pempty(b), kStoreWarps); mbar_init(bar_shared(b), kStoreWarps); }
    mbar_init(bar_drain(), 1);
    mbar_init(bar_sums(), 1);
    abort_flag[0] = 0;
    abort_flag[1] = (int)(p.spin_limit ? p.spin_limit : kSpinLimit);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    // the filter's part of the empty ring is sent for while the launch before this one drains
    decode(p, tile0, m0, n0);
    for (int i = p.withhold_first_load; i < ahead; ++i) load_filter(i, step0 + i);  // (test: the first step never arrives)
    if (p.d > 1) {
      const int live = min(p.nt, p.n_extent - n0) - (rank << p.per_log);  // columns that this CTA adds up
      mbar_expect_tx(bar_sums(), (uint32_t)(max(0, min(1 << p.per_log, live)) * p.d * kSumPitch * 4));
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (p.d > 1) cluster_arrive();  // (waited for before anything reaches into another CTA)
  const uint32_t tmem = *tmem_slot;
  if (tid == 0) grid_release();  // (this CTA has its tensor memory: nothing it waits for can be held by the next launch)
  grid_wait();

  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < ahead; ++i) load_rows(i, step0 + i);
      int s = ahead == p.stages ? 0 : ahead;
      uint32_t parity = ahead == p.stages ? 0 : 1;  // of the empty barriers
      bool ok = true;
      for (int t = tile0; t < p.total_tiles && ok; t += tile_step) {
        if (t != tile0) decode(p, t, m0, n0);
        for (int step = t == tile0 ? step0 + ahead : step0; step < step1; ++step) {
          if (!(ok = mbar_wait(bar_empty(s), parity, abort_flag))) break;
          load_filter(s, step);
          load_rows(s, step);
          if (++s == p.stages) { s = 0; parity ^= 1; }
        }
      }
      abort_flag[2] = loads;
    }
  } else if (warp == 1) {
    // The loop has no early exits: after a wait that gave up it runs dry, without MMAs and commits (what the elected lane
    // has waited for is what counts).
    constexpr uint32_t kFormats = (1u << 7) | (1u << 10) | (FMT == TETRIS_FP4_NV ? 0u : 1u << 23) | ((uint32_t)(kM >> 4) << 24);
    const uint32_t idesc = kFormats | ((uint32_t)(p.nt >> 3) << 17);
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!mbar_try_wait(bar, parity)) ok = ok && mbar_wait(bar, parity, abort_flag);
      __syncwarp();
    };
    const uint32_t ring0 = desc_low(smem_u32(ring)), stage_step = (uint32_t)p.stage_bytes >> 4;
    int s = 0, slot = 0, free_s = 0, behind = 0;   // behind: steps whose scale slots may still be read
    uint32_t parity = 0, free_parity = 0;
    int i = 0;
    for (int t = tile0; t < p.total_tiles; t += tile_step, ++i) {
      decode(p, t, m0, n0);
      const int b = i & acc_log;
      const uint32_t acc = tmem + (b ? p.acc1 : 0);
      const uint32_t sf_row = DIRECT && !ROWS_M ? 0u : (uint32_t)(n0 & 127) >> 5;   // the tile's first 32-row group within its scale tile: 0 or 2
      if (i > acc_log) wait(bar_pempty(b), ((i >> acc_log) & 1) ^ 1);
      if (over && i >= 1) wait(bar_shared(b ^ 1), ((i - 1) >> 1) & 1);
      for (int step = step0; step < step1; ++step) {
        if (behind == p.slots) {
          wait(bar_empty(free_s), free_parity);
          if (++free_s == p.stages) { free_s = 0; free_parity ^= 1; }
          --behind;
        }
        wait(bar_full(s), parity);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = ring0 + (uint32_t)s * stage_step;   // (addresses in units of 16 bytes)
        const uint32_t sfm = tmem + p.sf + slot * p.slot_cols, sfn = sfm + 4 * kTiles, sfn_row = sfn + sf_row;
        const int n = min(kTiles, p.tiles_k - step * kTiles), mmas = step == p.steps - 1 ? p.last_mmas : 4;
        const uint32_t dsm = at + (p.sm_at >> 4), dsn = at + (p.sn_at >> 4), dn = at + (p.n_at >> 4);
        const uint32_t more = step > step0;
        if (elect_one() && ok) {
#pragma unroll
          for (int k = 0; k < kTiles; ++k) {
            if (k < n) {
              copy_scales(sfm + 4 * k, dsm + 32 * k);
              copy_scales(sfn + 4 * rt * k, dsn + 32 * k);
              if (rt == 2) copy_scales(sfn + 8 * k + 4, dsn + 32 * (kTiles + k));
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < mmas) {
              const int k = FMT == TETRIS_FP4_NV ? j : j >> 1;
              const uint32_t id = FMT == TETRIS_FP4_NV || !(j & 1) ? idesc : idesc | (2u << 4) | (2u << 29);  // (second half of the scale words)
              umma_fp4<FMT>(acc, at + 2 * j, dn + 2 * j, p.codes_high, id, sfm + 4 * k, sfn_row + 4 * rt * k, j == 0 ? more : 1u);
            }
          }
          umma_commit(bar_empty(s));
          if (step == step1 - 1) umma_commit(bar_pfull(b));
        }
        __syncwarp();
        ++behind;
        if (++s == p.stages) { s = 0; parity ^= 1; }
        if (++slot == p.slots) slot = 0;
      }
    }
  }
  // DIRECT: the storing warps quantise the rows r0, ... of a tile, K step by K step.  A unit is the lanes' share of 32 >> lx
  // rows; the warps take the units of a step in turn, several at a time so that their loads and instructions overlap, a
  // lane 8 values.  Every warp enters every step, waits for its stage and arrives once it is done with it: a wait for a
  // barrier's phase by its parity only means something to who has seen the phase before.  (After a wait that gave up it
  // walks on without waiting and arriving: its lanes meet in shuffles.)
  int c_stage = 0, c_steps = 0x7FFFFFFF;   // c_steps: steps that it was done with when a wait gave up
  uint32_t c_parity = 1;
  bool c_ok = true;
  auto convert = [&](int r0) {
    constexpr int kLanes = (FMT == TETRIS_FP4_NV ? 16 : 32) / 8;
    const int extent = ROWS_M ? p.m_extent : p.n_extent, units = 1 << p.unit_log, me = warp - kFirstStore;
    const int lane_col = lane & ((1 << p.lx) - 1), lane_row = lane >> p.lx, blk = lane_col / kLanes;
    auto some = [&](auto many, int step, int u0) {  // units u0, u0 + 8, ... of the step
      constexpr int kAtOnce = decltype(many)::value;
      const int col = step * kStep + lane_col * 8, left = p.K - col;
      const uint32_t keep = left >= 8 ? 0xFFFFFFFFu : left <= 0 ? 0u : (1u << (4 * left)) - 1u;
      float v[kAtOnce][8];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int u = u0 + q * kStoreWarps, row = r0 + (u << (5 - p.lx)) + lane_row;
        int64_t from = row;
        if (p.px.S > 1) {
          const uint32_t y = fp4_quot((uint32_t)row, p.by_OW), ox = (uint32_t)row - y * p.px.OW, n = fp4_quot(y, p.by_OH), oy = y - n * p.px.OH;
          from = ((int64_t)n * p.px.H + (int64_t)oy * p.px.S) * p.px.W + (int64_t)ox * p.px.S;
        }
        load8(p, from * p.x_ld + col, u < units && row < extent ? left : 0, v[q]);
      }
      BlockScale b[kAtOnce];
      bool far = false;
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[q][k]) & 0x7FFFFFFFu);  // (as integers: NaN last)
#pragma unroll
        for (int l = 1; l < kLanes; l *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, l));
        b[q] = block_scale<FMT>(__uint_as_float(top), p.tensor_scale, p.sixth, p.sixth_rest);
        far |= b[q].far;
      }
      if (far) {
#pragma unroll
        for (int q = 0; q < kAtOnce; ++q)
          if (b[q].far) bring_near(v[q], b[q]);
      }
      unsigned char *at = ring + (size_t)c_stage * p.stage_bytes;
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int u = u0 + q * kStoreWarps, row = (u << (5 - p.lx)) + lane_row;
        const uint32_t codes = block_codes<FMT>(v[q], b[q]) & keep;
        if (u < units) {
          const int swizzle = row >> (7 - p.row_log) & ((1 << (p.row_log - 4)) - 1);
          *reinterpret_cast<uint32_t *>(at + (ROWS_M ? 0 : p.n_at) + (row << p.row_log) + (((lane_col >> 2) ^ swizzle) << 4) + (lane_col & 3) * 4) = codes;
          if (lane_col % kLanes == 0) at[(ROWS_M ? p.sm_at : p.sn_at) + (blk >> 2) * 512 + (row & 31) * 16 + (row >> 5) * 4 + (blk & 3)] = b[q].byte;
        }
      }
    };
#pragma unroll 1
    for (int step = step0, turn = me; step < step1; ++step) {
      if (!mbar_try_wait(bar_empty(c_stage), c_parity) && !(c_ok && mbar_wait(bar_empty(c_stage), c_parity, abort_flag))) {
        if (c_ok) c_steps = step - step0;
        c_ok = false;
      }
      __syncwarp();
      if (units <= kStoreWarps) {  // (another warp begins each step)
        if (turn < units) some(std::integral_constant<int, 1>(), step, turn);
        turn = (turn - units) & (kStoreWarps - 1);
      } else if (units == 2 * kStoreWarps) {
        some(std::integral_constant<int, 2>(), step, me);
      } else {
#pragma unroll 1
        for (int u = me; u < units; u += 4 * kStoreWarps) some(std::integral_constant<int, 4>(), step, u);
      }
      // (the writes went through the generic proxy, the tensor core reads through the async proxy)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0 && c_ok) mbar_arrive(bar_full(c_stage));
      if (++c_stage == p.stages) { c_stage = 0; c_parity ^= 1; }
    }
  };
  if (warp < kFirstStore) {
  } else if (p.d == 1) {
    constexpr int kUnit = ROWS_M ? 128 / (int)sizeof(T) : 32;   // columns that a warp takes at a time (D[row][oc]: 128 bytes of a row)
    const int me = warp - kFirstStore, quarter = warp & 3, half = me >> 2;
    const int units = max(1, p.nt / kUnit), shared = over ? (p.nt - p.acc1 + kUnit - 1) / kUnit : 0;
    float *bias_row = bias_rows + me * 64;
    unsigned char *blocks = staging + me * kStageOut * p.staging;
    int nblk = 0;
    int i = 0;
    decode(p, tile0, m0, n0);
    for (int t = tile0; t < p.total_tiles; t += tile_step, ++i) {
      const int b = i & acc_log, mq = m0 + quarter * 32, m = mq + lane, n_first = n0;
      const float lane_bias = !ROWS_M && p.bias && m < p.m_extent ? p.bias[m] : 0.f;
      if (DIRECT) convert(ROWS_M ? m0 : n0);
      bool ok = mbar_try_wait(bar_pfull(b), (i >> acc_log) & 1);
      if (!ok) ok = mbar_wait(bar_pfull(b), (i >> acc_log) & 1, abort_flag);
      if (!__all_sync(0xffffffffu, ok)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (b ? p.acc1 : 0);
      bool told = !over;
#pragma unroll 1
      for (int c = half; c < units; c += 2) {
        const int unit = b ? c : units - 1 - c;  // the shared columns: the first accumulator's last, the second one's first
        if (!told && c >= shared) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_shared(b));
          told = true;
        }
        const int n = n_first + unit * kUnit;
        uint32_t v[32];
        if (ROWS_M) {
          // 32 rows x 128 bytes into a staging block in the 128-byte swizzle (16-byte piece c of row r at c ^ (r & 7):
          // eight lanes touch eight bank groups), from there as whole lines to the output.
          unsigned char *blk = blocks + (p.staging == 2 ? (nblk & 1) * kStageOut : 0);
          ++nblk;
          if (p.tma_store) {  // the block's last store has read it
            if (lane == 0) {
              if (p.staging == 2) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
              else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            }
          }
          if (p.bias) {
            __syncwarp();
#pragma unroll
            for (int k = 0; k < kUnit; k += 32) bias_row[k + lane] = n + k + lane < p.n_extent ? p.bias[n + k + lane] : 0.f;
          }
          __syncwarp();
#pragma unroll
          for (int h = 0; h < kUnit / 32; ++h) {
            tmem_ld32(acc + unit * kUnit + h * 32, v);
            if (p.scale1 != 1.f) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * p.scale1);
            }
            constexpr int kPer = 16 / (int)sizeof(T);  // values of a 16-byte piece
#pragma unroll
            for (int j = 0; j < 32; j += kPer) {
              alignas(16) T out[kPer];
#pragma unroll
              for (int k = 0; k < kPer; k += 4) {
                float4 bb = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p.bias) bb = *reinterpret_cast<const float4 *>(bias_row + h * 32 + j + k);
                out[k] = to_type<T>(finish(v[j + k], p.scale, bb.x, p.relu)); out[k + 1] = to_type<T>(finish(v[j + k + 1], p.scale, bb.y, p.relu));
                out[k + 2] = to_type<T>(finish(v[j + k + 2], p.scale, bb.z, p.relu)); out[k + 3] = to_type<T>(finish(v[j + k + 3], p.scale, bb.w, p.relu));
              }
              const int piece = (h * 32 + j) / kPer;
              *reinterpret_cast<uint4 *>(blk + lane * 128 + ((piece ^ (lane & 7)) << 4)) = *reinterpret_cast<const uint4 *>(out);
            }
          }
          if (p.tma_store) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
              if (mq < p.m_extent && n < p.n_extent) tma_store_2d(&map_y, smem_u32(blk), n, mq);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {
            __syncwarp();
            constexpr int kAside = 4 / (int)sizeof(T);  // values of a lane
            const int left = p.n_extent - n - lane * kAside, rows = min(32, p.m_extent - mq);
            T *y = static_cast<T *>(p.y) + (int64_t)mq * p.ld + n + lane * kAside;
#pragma unroll 4
            for (int r = 0; r < rows; ++r, y += p.ld) {
              const T *from = reinterpret_cast<const T *>(blk + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
#pragma unroll
              for (int k = 0; k < kAside; ++k)
                if (k < left) y[k] = from[k];
            }
          }
        } else {
          tmem_ld32(acc + unit * 32, v);
          if (p.scale1 != 1.f) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * p.scale1);
          }
          const int rows = min(32, p.n_extent - n);
          T *y = static_cast<T *>(p.y) + (int64_t)n * p.ld + m;
          if (m < p.m_extent) {
#pragma unroll
            for (int j = 0; j < 32; ++j, y += p.ld)
              if (j < rows) *y = to_type<T>(finish(v[j], p.scale, lane_bias, p.relu));
          }
        }
      }
      if (t + tile_step < p.total_tiles) decode(p, t + tile_step, m0, n0);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (!told) mbar_arrive(bar_shared(b));
        mbar_arrive(bar_pempty(b));
      }
    }
    if (ROWS_M && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // this warp's stores are complete
  } else {
    // The slices of a tile meet: a CTA owns 2^per_log columns; each sends its sums of a column (128 lanes) to
    // the owner, who adds them up in slice order.  They are laid out in the ring, which is idle, and leave as
    // one copy per owner.
    const int quarter = warp & 3, half = (warp - kFirstStore) >> 2, per = 1 << p.per_log;
    decode(p, tile0, m0, n0);
    const int live = min(p.nt, p.n_extent - n0);
    if (DIRECT) convert(ROWS_M ? m0 : n0);
    bool ok = __all_sync(0xffffffffu, mbar_wait(bar_pfull(0), 0, abort_flag));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    float *out = reinterpret_cast<float *>(ring);
#pragma unroll 1
    for (int c = half * 32; c < live; c += 64) {
      uint32_t v[32];
      tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j < live) out[(c + j) * kSumPitch + quarter * 32 + lane] = __uint_as_float(v[j]);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    cluster_wait();  // (every CTA of the cluster runs)
    asm volatile("bar.sync 1, %0;" ::"r"(32 * kStoreWarps) : "memory");
    if (warp == kFirstStore && lane < p.d && ok && !*abort_flag) {
      const int cols = min(per, live - (lane << p.per_log));
      if (cols > 0)
        push(cluster_addr(smem_u32(sums) + (uint32_t)((rank << p.per_log) * kSumPitch) * 4u, lane), smem_u32(out) + (uint32_t)((lane << p.per_log) * kSumPitch) * 4u,
             (uint32_t)(cols * kSumPitch) * 4u, cluster_addr(bar_sums(), lane));
    }
    __syncwarp();
    ok = __all_sync(0xffffffffu, mbar_wait(bar_sums(), 0, abort_flag)) && ok;
    cluster_arrive();  // (what this CTA is owed has come, or it has given up; all of its own copies have been sent)
    const int own = ok ? min(per, live - (rank << p.per_log)) : 0, own0 = n0 + (rank << p.per_log);
    // A thread takes four lanes of a column.  D[oc][row]: neighbouring threads take neighbouring lanes; D[row][oc]:
    // neighbouring columns.
    const bool whole = !ROWS_M && ((reinterpret_cast<uintptr_t>(p.y) | (uint64_t)(p.ld * sizeof(T))) & (4 * sizeof(T) - 1)) == 0;
    for (int e = tid - 32 * kFirstStore; e < per * (kM / 4); e += 32 * kStoreWarps) {
      const int j = ROWS_M ? e & (per - 1) : e / (kM / 4), l = 4 * (ROWS_M ? e >> p.per_log : e % (kM / 4));
      if (j >= own || m0 + l >= p.m_extent) continue;
      const float *from = sums + j * kSumPitch + l;
      float u[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int s = 0; s < p.d; ++s) {
        const float4 a = *reinterpret_cast<const float4 *>(from + (s << p.per_log) * kSumPitch);
        u[0] += a.x; u[1] += a.y; u[2] += a.z; u[3] += a.w;
      }
      T *y = static_cast<T *>(p.y) + (ROWS_M ? (int64_t)(m0 + l) * p.ld + own0 + j : (int64_t)(own0 + j) * p.ld + m0 + l);
      alignas(16) T out[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int oc = ROWS_M ? own0 + j : m0 + l + k;
        const float bias = p.bias && (ROWS_M || oc < p.m_extent) ? p.bias[oc] : 0.f;
        out[k] = to_type<T>(finish(__float_as_uint(u[k] * p.scale1), p.scale, bias, p.relu));
      }
      if (whole && m0 + l + 4 <= p.m_extent) {
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(y) = *reinterpret_cast<const uint4 *>(out);
        else *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(out);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (m0 + l + k < p.m_extent) y[ROWS_M ? k * p.ld : k] = out[k];
      }
    }
  }
  __syncwarp();
  if (p.d > 1 && warp < kFirstStore) {
    cluster_wait();
    cluster_arrive();
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (*abort_flag) {  // what this CTA has in flight must land before it leaves
    // (stages on their way also wait for the arrivals of quantising warps that stopped before them: at most one each, since
    // a stage is sent for again only after its last phase)
    if (DIRECT && warp >= kFirstStore && lane == 0)
      for (int v = c_steps; v < abort_flag[2]; ++v) mbar_arrive(bar_full(v % p.stages));
    if (tid == 0)
      for (int v = max(loads - p.stages, p.withhold_first_load ? 1 : 0); v < loads; ++v) mbar_drain(bar_full(v % p.stages), (uint32_t)(v / p.stages) & 1u);
    if (warp == 1) {
      if (elect_one()) umma_commit(bar_drain());
      __syncwarp();
      mbar_drain(bar_drain(), 0);
    }
    if (tid == 0) atomicExch(p.error_flag, 1);
    __syncwarp();
  }
  if (p.d > 1) {
    cluster_wait();  // (no CTA leaves while another one may still push into it)
    if (tid == 0 && *abort_flag) mbar_drain(bar_sums(), 0);  // (one that gave up did not wait for what the others sent)
  }
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn get_encode() {
  static const EncodeFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess ? (EncodeFn)p : nullptr;
  }();
  return fn;
}

// A product takes half of an SM (113 KB of shared memory, 256 columns of tensor memory) or all of it.  Two halves
// overlap: one CTA stores while the other one computes, and the next launch is placed and fetches its filter while
// this one ends.  Nothing that holds tensor memory and waits for another CTA may sit beside a CTA that waits for
// tensor memory: two halves always fit, and a half beside anything that takes 116 KB or more never does.
constexpr size_t kSmemMost = 227 * 1024, kSmemHalf = 113 * 1024;   // (1 KB of either goes into the ring's alignment)
constexpr size_t kSmemLeast = 117 * 1024;

// A product quantises its rows itself where a storing warp has at most this many units of it to do.  Up to there it takes
// about as long as a launch of its own before the product (16x1024x1024, 2 units: 4.1 us on the device in one launch,
// 4.3 in two; 22x832x32, 4 units: 4.8 and 4.5; 51x1824x640, 8 units: 7.5 and 5.8; 16x8192x8192, 16 units: 18 and 10.8),
// and the host has one launch less, 2.2 us.  At four units the host is why: a captured graph pays 0.3 us for it.
constexpr int kDirectUnits = 4;

// How the rows of a tile are cut into units of a warp: 2^lx lanes take a row's part of a K step.
struct Units {
  int lx, log;             // log: units of a K step
};
Units units_of(int cols, int64_t tile_rows) {
  Units u = {cols <= 64 ? 3 : cols <= 128 ? 4 : 5, 0};
  while ((int64_t)(32 >> u.lx) << u.log < tile_rows) ++u.log;
  return u;
}

struct Geometry {
  bool rows_m;
  int nt, d;
  bool half;
};

// Bytes of a row's codes in a stage, as a logarithm: a TMA load takes its time for the zeros behind the last column, too
// (200704x32x64: 28 us with 128-byte rows).
int row_log_of(int cols) { return cols <= 64 ? 5 : cols <= 128 ? 6 : 7; }

// The least of an estimate in nanoseconds, whose terms were fitted to 60 shapes (1 to 50000 rows, 64 to 16384
// columns and channels, columns in multiples of 64 and channels in multiples of 16) in every geometry: its choice takes
// 1.5 % longer than the best of those, 15 % at worst.  It has no term for outputs that TMA stores do not take
// (1352x1024 to 255 channels 4.8 us, to 256 4.2).
//   a K step    the longer of its MMAs and its loads: 51 bytes a nanosecond for half an SM alone, 2 x 40 for two
//               halves, 75 for a whole one (16x8192x8192: 12.2 us in 128 halves, 9.5 in 256)
//   a tile      the longer of its steps and the store of the one before it; the last store stands alone
//   a whole SM  hands over to the next tile 500 ns late; two halves hide that
//               (1024x4096x4096: 128 columns 13.1 us in halves and 18.1 whole, 256 columns 12.7)
//   a cluster   its meeting grows with the columns (64x4096x4096: 10.2 us in one slice, 7.6 in four)
//   a launch that leaves no room for the next one's CTAs beside its own takes 600 ns longer
//               (1x4096x4096: 4.1 us in 128 halves, 5.5 in 256)
Geometry estimate(const tetris_fp4_filter *f, int64_t rows) {
  const int steps = (f->in_channel + kStep - 1) / kStep;
  const double sms = f->sm_count, row_bytes = (1 << row_log_of(f->in_channel)) + (f->format == TETRIS_FP4_NV ? 16 : 8);  // of a step
  Geometry best = {false, 16, 1, true};
  double least = 1e300;
  for (int rows_m = 0; rows_m < 2; ++rows_m) {
    const int64_t m = rows_m ? rows : f->out_channel, n = rows_m ? f->out_channel : rows;
    for (int nt = 16; nt <= 256; nt *= 2) {
      // The scales of a tile begin at its first 32-row group's column, and an MMA takes scales from even columns
      // only (an odd one is a misaligned address): tiles below 64 begin at 0.
      if (nt < 64 && n > nt) continue;
      const int64_t tiles = (m + kM - 1) / kM * ((n + nt - 1) / nt);
      const double bytes = (kM + nt) * row_bytes, store = (rows_m ? 5.8 : 9.7) * nt;
      for (int half = nt <= 128; half >= 0; --half) {
        for (int d = 1; d <= 8; d *= 2) {
          if (d > 1 && (d > steps || nt > (half ? 64 : 128) || tiles * d > (half ? 2 : 1) * f->sm_count)) break;
          const double ctas = (double)tiles * d, k = (double)((steps + d - 1) / d);
          double cost;
          if (half && ctas <= sms) {
            cost = k * std::max(bytes / 51., 1.1 * nt);
          } else if (half) {
            const double rounds = ctas <= 4 * sms ? std::max(1., ctas / (2 * sms)) : std::ceil(ctas / (2 * sms) - 0.1);
            cost = rounds * std::max(k * std::max(bytes / 40., 2.5 * nt), 2.5 * store) + 620.;
          } else {
            const double rounds = std::ceil(ctas / sms);
            cost = rounds * std::max(k * std::max(bytes / 75., 1.1 * nt), store) + (rounds - 1) * (nt > 128 ? 500. : 580.) + 36. + (2 * ctas > sms ? 620. : 0.);
          }
          cost += d > 1 ? 100. + 20. * nt : store;
          if (cost < least) { least = cost; best = {rows_m != 0, nt, d, half != 0}; }
        }
      }
    }
  }
  return best;
}

bool is_direct(const tetris_fp4_filter *f, int64_t rows, const Geometry &g) {
  const int64_t tiles = ((g.rows_m ? rows : f->out_channel) + kM - 1) / kM * (((g.rows_m ? f->out_channel : rows) + g.nt - 1) / g.nt);
  if (g.nt > (g.rows_m ? 128 : 64) || tiles * g.d > (g.half ? 2 : 1) * f->sm_count) return false;  // (one tile per CTA)
  const Units u = units_of(f->in_channel, std::min<int64_t>(rows, g.rows_m ? kM : g.nt));
  const int steps = ((f->in_channel + kStep - 1) / kStep + g.d - 1) / g.d;
  return ((int64_t)steps << u.log) <= kDirectUnits * kStoreWarps;
}

// The estimate takes the host 0.3 us, so the filter keeps it for the last few numbers of rows.
Geometry choose(const tetris_fp4_filter *f, int64_t rows) {
  std::atomic<uint64_t> &kept = f->plans[rows & 7];
  const uint64_t k = kept.load(std::memory_order_relaxed);
  if (k >> 24 == (uint64_t)rows) return {(k & 1) != 0, (int)(k >> 8 & 0x1FF), 1 << (k >> 4 & 3), (k & 2) != 0};
  const Geometry g = estimate(f, rows);
  int d_log = 0;
  while (1 << d_log < g.d) ++d_log;
  kept.store((uint64_t)rows << 24 | (uint64_t)g.nt << 8 | (uint64_t)d_log << 4 | (g.half ? 2 : 0) | (g.rows_m ? 1 : 0), std::memory_order_relaxed);
  return g;
}

template <int FMT, typename T, bool ROWS_M, bool DIRECT>
int launch(const CUtensorMap &map_m, const CUtensorMap &map_n, const CUtensorMap &map_y, const ProductParams &p, unsigned grid, size_t smem, cudaStream_t st) {
  static std::atomic<bool> ready[64];  // per device
  int dev = 0;
  TETRIS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev]) {
    TETRIS_CUDA_TRY(cudaFuncSetAttribute(product_kernel<FMT, T, ROWS_M, DIRECT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMost));
    if (dev < 64) ready[dev] = true;
  }
  TETRIS_CUDA_TRY(launch_overlapped(product_kernel<FMT, T, ROWS_M, DIRECT>, dim3(grid), kThreads, smem, st, (unsigned)p.d, map_m, map_n, map_y, p));
  count_launch();
  return TETRIS_OK;
}
template <int FMT, typename T>
int launch(bool rows_m, const CUtensorMap &map_m, const CUtensorMap &map_n, const CUtensorMap &map_y, const ProductParams &p, unsigned grid, size_t smem, cudaStream_t st) {
  if (p.x)
    return rows_m ? launch<FMT, T, true, true>(map_m, map_n, map_y, p, grid, smem, st) : launch<FMT, T, false, true>(map_m, map_n, map_y, p, grid, smem, st);
  return rows_m ? launch<FMT, T, true, false>(map_m, map_n, map_y, p, grid, smem, st) : launch<FMT, T, false, false>(map_m, map_n, map_y, p, grid, smem, st);
}

// A matrix whose rows are `pitch` bytes apart, in boxes of 2^row_log bytes x `box_rows`, swizzled.
int encode(CUtensorMap *map, CUtensorMapDataType type, int type_bytes, const void *matrix, int64_t cols, int64_t pitch, int64_t rows, int box_rows, int row_log = 7) {
  EncodeFn enc = get_encode();
  if (!enc) { set_error("cuTensorMapEncodeTiled is not available from this driver"); return TETRIS_ERR_UNSUPPORTED; }
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {(1u << row_log) / (cuuint32_t)type_bytes, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUtensorMapSwizzle swizzle = row_log == 7 ? CU_TENSOR_MAP_SWIZZLE_128B : row_log == 6 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
  const CUresult r = enc(map, type, 2, const_cast<void *>(matrix), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed with code %d", (int)r); return TETRIS_ERR_CUDA; }
  return TETRIS_OK;
}

}  // namespace

// Geometries and units change behind powers of two and multiples of 16 rows.
int64_t fp4_product_direct_rows(const tetris_fp4_filter *f) {
  int64_t rows = 0;
  for (int64_t next = 1; is_direct(f, next, estimate(f, next)); next += next < 16 ? next : 16) rows = next;
  return rows;
}

int launch_fp4_product(const tetris_fp4_filter *f, const Fp4Rows &a, int64_t rows, int exponent, const float *bias, void *y, int y_type, int64_t ld,
                       int relu, cudaStream_t st) {
  const bool direct = !a.codes;
  const Geometry g = choose(f, rows);
  const bool nv = f->format == TETRIS_FP4_NV;
  const int kt = step_tiles(f->format), rt = g.nt > 128 ? 2 : 1, bytes = y_type == TETRIS_FP32 ? 4 : 2;
  ProductParams p = {};
  p.scales_m = g.rows_m ? a.scales : f->d_scales; p.scales_n = g.rows_m ? f->d_scales : a.scales;
  p.bias = bias;
  p.y = y; p.ld = ld;
  p.m_extent = (int)(g.rows_m ? rows : f->out_channel); p.n_extent = (int)(g.rows_m ? f->out_channel : rows);
  p.m_blocks = (p.m_extent + 127) / 128; p.n_blocks = (p.n_extent + 127) / 128;
  p.steps = (f->in_channel + kStep - 1) / kStep;
  p.last_mmas = (f->in_channel - (p.steps - 1) * kStep + 63) / 64;
  p.tiles_k = fp4_tiles(f->in_channel, f->format);
  p.nt = g.nt; p.d = g.d;
  for (p.per_log = 0; g.nt / g.d >> (p.per_log + 1); ++p.per_log) {}
  p.m_tiles = p.m_blocks;
  p.n_tiles = (p.n_extent + g.nt - 1) / g.nt;
  p.group = std::min(p.m_tiles, 16);
  p.by_per = fp4_div((uint32_t)(p.group * p.n_tiles)); p.by_group = fp4_div((uint32_t)p.group);
  p.by_last = fp4_div((uint32_t)std::max(1, p.m_tiles % p.group));
  const int64_t total = (int64_t)p.m_tiles * p.n_tiles;
  if (total > 0x3FFFFFFF) { set_error("a product of %lld tiles is outside what the kernels cover", (long long)total); return TETRIS_ERR_UNSUPPORTED; }
  p.total_tiles = (int)total;
  p.row_log = row_log_of(f->in_channel);
  p.codes_high = codes_high(p.row_log);
  p.n_at = kM << p.row_log;
  p.sm_at = p.n_at + (g.nt << p.row_log);
  p.sn_at = p.sm_at + kt * 512;
  p.stage_bytes = (p.sn_at + rt * kt * 512 + 1023) / 1024 * 1024;
  p.staging = !g.rows_m ? 0 : rt == 2 || g.half ? 1 : 2;
  const size_t tail = 1024 + (g.d > 1 ? (size_t)g.nt * kSumPitch * 4 : (size_t)kStoreWarps * kStageOut * p.staging) + kBiasBytes + kBars * 8 + 16;
  p.stages = std::min<int>(kStagesMax, (int)(((g.half ? kSmemHalf : kSmemMost) - tail) / p.stage_bytes));
  p.tmem_cols = g.half ? 256 : 512;
  p.slot_cols = 4 * kt * (1 + rt);
  p.accs = g.half && g.nt > 64 ? 1 : 2;
  p.slots = rt == 2 ? 2 : std::min(g.half ? 4 : kSlotsMax, p.stages);  // (at most `stages`: a step's empty barrier is waited for before the stage is used again)
  p.sf = p.tmem_cols - p.slots * p.slot_cols;
  p.acc1 = p.accs == 2 ? std::min(std::max(g.nt, 32), (p.sf - g.nt) / 32 * 32) : 0;
  const int e = exponent + f->exponent, e0 = std::max(-126, std::min(126, e));
  p.scale = ldexpf(1.f, e0); p.scale1 = ldexpf(1.f, e - e0);
  p.K = f->in_channel;
  if (direct) {
    const int x_bytes = a.x_type == TETRIS_FP32 ? 4 : 2;
    p.x = a.x; p.x_type = a.x_type; p.x_ld = a.ld;
    p.x_vec = ((reinterpret_cast<uintptr_t>(a.x) | (uint64_t)(a.ld * x_bytes)) & 15) == 0;
    p.px.S = 1;
    if (a.px) {
      p.px = *a.px;
      p.by_OH = fp4_div((uint32_t)a.px->OH); p.by_OW = fp4_div((uint32_t)a.px->OW);
    }
    const Units u = units_of(p.K, std::min<int64_t>(rows, g.rows_m ? kM : g.nt));
    p.lx = u.lx; p.unit_log = u.log;
    fp4_scale_factors(exponent, &p.tensor_scale, &p.sixth, &p.sixth_rest);
  }
  p.relu = relu;
  // A TMA store leaves out what lies behind a row's end by whole 16 bytes only: a row that ends inside of them would have
  // zeros written behind it, into whatever lies between rows that are apart.  (The distance between rows in a tensor
  // map is below 2^40 bytes.)
  p.tma_store = g.rows_m && g.d == 1 && ((reinterpret_cast<uintptr_t>(y) | (uint64_t)(ld * bytes) | (uint64_t)f->out_channel * bytes) & 15) == 0 &&
                ld * bytes < (1ll << 40);
  p.error_flag = f->d_error;
  p.withhold_first_load = test_injection(&p.spin_limit);
  CUtensorMap map_w, map_a = {}, map_y = {};
  int rc;
  if ((rc = encode(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, f->d_codes, f->pitch, f->pitch, f->out_channel, g.rows_m ? g.nt : kM, p.row_log)) ||
      (!direct && (rc = encode(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.codes, f->pitch, f->pitch, rows, g.rows_m ? kM : g.nt, p.row_log))) ||
      (p.tma_store && (rc = encode(&map_y, y_type == TETRIS_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, bytes, y,
                                   f->out_channel, ld * bytes, rows, 32))))
    return rc;
  const CUtensorMap &map_m = g.rows_m ? map_a : map_w, &map_n = g.rows_m ? map_w : map_a;
  const unsigned grid = (unsigned)(g.d > 1 ? p.total_tiles * g.d : std::min(p.total_tiles, (g.half ? 2 : 1) * f->sm_count));
  const size_t smem = g.half ? kSmemHalf : std::max(kSmemLeast, (size_t)p.stages * p.stage_bytes + tail);
  switch (y_type) {
    case TETRIS_FP32: return nv ? launch<TETRIS_FP4_NV, float>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st) : launch<TETRIS_FP4_MX, float>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st);
    case TETRIS_BF16: return nv ? launch<TETRIS_FP4_NV, __nv_bfloat16>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st) : launch<TETRIS_FP4_MX, __nv_bfloat16>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st);
    default: return nv ? launch<TETRIS_FP4_NV, __half>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st) : launch<TETRIS_FP4_MX, __half>(g.rows_m, map_m, map_n, map_y, p, grid, smem, st);
  }
}

}  // namespace tetris
