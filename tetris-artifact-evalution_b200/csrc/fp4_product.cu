// Products of 4-bit activations and a 4-bit filter on the tensor cores:
//   y[row][oc] = sum_k a[row][k] w[oc][k] (+ bias, ReLU)
// tcgen05.mma with block scales: kind::mxf4 (32 values a scale, E8M0) and kind::mxf4nvf4 (16 a scale,
// E4M3), both 64 values of K per instruction, FP32 accumulators in tensor memory.
//
// D[oc][row]: the M side is 128 output channels (the filter), the N side 16 to 256 rows.  A lane of
// tensor memory then is a channel, so 32 lanes store 32 neighbouring values of an output row: whole lines
// without staging, for any row distance and alignment, and few rows cost a narrow N, not an empty M.
//   * warp 0 (one thread): per K step of 256 TMA loads of 128 filter rows and of the tile's rows (128
//     bytes each, 128-byte swizzle, zeros past both ends) and bulk copies of the scales, into one ring;
//   * warp 1 (one elected lane): scales from shared into tensor memory (tcgen05.cp), then 4 MMAs;
//   * eight storing warps: accumulator -> scale, bias, ReLU -> output, beside the next tile's MMAs.
// Tensor memory: two accumulators.  With 256 rows two of them and the scales exceed 512 columns, so the
// second one lies over the end of the first; the storing warps empty the shared columns first and the next
// tile starts once those are free.
// Scales lie in slots of tensor memory that are written again only when the MMAs that read them are done.
// Few tiles: the K range is cut over a cluster of up to 8 CTAs, whose sums are pushed into the shared
// memory of the CTA that owns a row and added in slice order (bit-reproducible, no workspace).
// Every barrier wait is bounded; on a timeout an error flag is raised, all roles drain, tensor memory is
// freed and the kernel returns; tetris_fp4_filter_check reports it.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "fp4.h"

namespace tetris {
namespace {

constexpr int kChannels = 128;           // channels of a tile
constexpr int kStep = 256;               // K values of a step: 128 bytes of codes
constexpr int kStoreWarps = 8, kFirstStore = 2, kThreads = 32 * (kFirstStore + kStoreWarps);
constexpr int kStagesMax = 8, kSlotsMax = 8;
constexpr int kBars = 2 * kStagesMax + 8;
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kTmemCols = 512;
// Scale tiles (512 bytes, 128 rows x 4 blocks) of a K step
__host__ __device__ constexpr int step_tiles(int format) { return format == TETRIS_FP4_NV ? 4 : 2; }

struct ProductParams {
  const uint8_t *scales_a, *scales_w;
  const float *bias;
  void *y;
  int64_t ld;
  int rows, N;
  int steps, last_mmas;    // K steps; MMAs of the last one
  int tiles_k;             // scale tiles of 128 rows
  int nt;                  // rows of a tile = N of the MMAs
  int row_tiles_128;       // 128-row blocks of the activations' scales
  int oc_tiles, row_tiles, group;  // tiles; channel tiles that are walked side by side
  int total_tiles;
  int d;                   // CTAs of a cluster = slices of a tile's K range
  int stages, slots;
  int stage_bytes, a_at, sw_at, sa_at;  // a stage: filter codes, activation codes, filter scales, activation scales
  int acc1, sf, slot_cols; // columns of the second accumulator, the scales, of a slot of them
  float scale0, scale1;    // 2^(sum of the exponents) as two factors
  int relu;
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
// K-major codes in 128-byte rows with the 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t codes_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// a scale tile: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t scales_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 16) | (8ull << 32) | (1ull << 46);
}
// 512 bytes of scales into 4 columns of all four lane quarters
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void umma_fp4(uint32_t tmem_d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (FMT == TETRIS_FP4_NV)
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  else
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(tmem_d), "l"(da), "l"(db), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
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
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t addr, uint32_t rank) {  // `addr` of this CTA in CTA `rank` of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
template <typename T> __device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 to_type(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half to_type(float v) { return __float2half_rn(v); }

// Tile t: channel tiles in groups of `group`, within a group all row tiles, within a row tile the group's
// channels: CTAs that run side by side share rows and the group's part of the filter.
__device__ __forceinline__ void decode(const ProductParams &p, int t, int &oc0, int &row0) {
  const int per = p.group * p.row_tiles, g = t / per, r = t - g * per;
  const int width = min(p.group, p.oc_tiles - g * p.group);
  row0 = r / width;
  oc0 = (g * p.group + r - row0 * width) * kChannels;
  row0 *= p.nt;
}

template <int FMT, typename T>
__global__ void __launch_bounds__(kThreads, 1)
product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a, const ProductParams p) {
  constexpr int kTiles = step_tiles(FMT);
  extern __shared__ unsigned char smem_raw[];
  unsigned char *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char *tail = ring + (size_t)p.stages * p.stage_bytes;
  uint64_t *bars = reinterpret_cast<uint64_t *>(tail);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar_full = [&](int s) { return smem_u32(&bars[s]); };
  auto bar_empty = [&](int s) { return smem_u32(&bars[kStagesMax + s]); };
  auto bar_pfull = [&](int b) { return smem_u32(&bars[2 * kStagesMax + b]); };
  auto bar_pempty = [&](int b) { return smem_u32(&bars[2 * kStagesMax + 2 + b]); };
  auto bar_shared = [&](int b) { return smem_u32(&bars[2 * kStagesMax + 4 + b]); };
  auto bar_drain = [&]() { return smem_u32(&bars[2 * kStagesMax + 6]); };

  if (tid == 0) {
    for (int s = 0; s < kStagesMax; ++s) { mbar_init(bar_full(s), 1); mbar_init(bar_empty(s), 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(bar_pfull(b), 1); mbar_init(bar_pempty(b), kStoreWarps); mbar_init(bar_shared(b), kStoreWarps); }
    mbar_init(bar_drain(), 1);
    abort_flag[0] = 0;
    abort_flag[1] = (int)(p.spin_limit ? p.spin_limit : kSpinLimit);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  if (tid == 0) grid_release();  // (this CTA has its tensor memory: nothing it waits for can be held by the next launch)
  if (warp != 0) grid_wait();    // (warp 0 sends for the filter first)

  const int rank = p.d > 1 ? (int)(blockIdx.x % p.d) : 0;
  const int tile0 = blockIdx.x / p.d, tile_step = gridDim.x / p.d;
  const int step0 = (int)((int64_t)p.steps * rank / p.d), step1 = (int)((int64_t)p.steps * (rank + 1) / p.d);
  const int rt = p.nt > 128 ? 2 : 1;       // 128-row blocks of a tile's scales
  const bool over = p.acc1 < p.nt;         // the accumulators share columns
  int loads = 0;

  if (warp == 0) {
    if (lane == 0) {
      int oc0, row0;
      // Bytes of a step: both code boxes whole (zeros past the ends count), the scale tiles that exist.
      auto scale_tiles = [&](int step) { return min(kTiles, p.tiles_k - step * kTiles); };
      auto load_w = [&](int s, int step) {
        const uint32_t at = smem_u32(ring + (size_t)s * p.stage_bytes), bar = bar_full(s);
        const int n = scale_tiles(step), blocks = min(rt, p.row_tiles_128 - row0 / 128);
        mbar_expect_tx(bar, (uint32_t)((kChannels + p.nt) * 128 + n * 512 * (1 + blocks)));
        tma_load_2d(at, &map_w, bar, step * 128, oc0);
        bulk_load(at + p.sw_at, p.scales_w + ((size_t)(oc0 / 128) * p.tiles_k + (size_t)step * kTiles) * 512, n * 512, bar);
      };
      auto load_a = [&](int s, int step) {
        const uint32_t at = smem_u32(ring + (size_t)s * p.stage_bytes), bar = bar_full(s);
        const int n = scale_tiles(step), b0 = row0 / 128, blocks = min(rt, p.row_tiles_128 - b0);
        if (loads++ == 0 && p.withhold_first_load) return;  // (test: that step never arrives, its reader gives up)
        tma_load_2d(at + p.a_at, &map_a, bar, step * 128, row0);
        for (int b = 0; b < blocks; ++b)
          bulk_load(at + p.sa_at + b * (kTiles * 512), p.scales_a + ((size_t)(b0 + b) * p.tiles_k + (size_t)step * kTiles) * 512, n * 512, bar);
      };
      int s = 0;
      uint32_t parity = 1;  // of the empty barriers
      bool ok = true;
      for (int t = tile0; t < p.total_tiles && ok; t += tile_step) {
        decode(p, t, oc0, row0);
        int step = step0;
        if (t == tile0) {  // the ring is empty: the filter's part is sent for while the launch before this one drains
          const int ahead = min(step1 - step0, p.stages);
          for (int i = 0; i < ahead; ++i) load_w(i, step0 + i);
          grid_wait();
          for (int i = 0; i < ahead; ++i) load_a(i, step0 + i);
          step += ahead;
          s = ahead;
          if (s == p.stages) { s = 0; parity ^= 1; }
        }
        for (; step < step1; ++step) {
          if (!(ok = mbar_wait(bar_empty(s), parity, abort_flag))) break;
          load_w(s, step);
          load_a(s, step);
          if (++s == p.stages) { s = 0; parity ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    // The loop has no early exits: a wait that gave up raises the abort flag, later waits then return at once.
    constexpr uint32_t kFormats = (1u << 7) | (1u << 10) | (FMT == TETRIS_FP4_NV ? 0u : 1u << 23) | ((uint32_t)(kChannels >> 4) << 24);
    const uint32_t idesc = kFormats | ((uint32_t)(p.nt >> 3) << 17);
    auto wait = [&](uint32_t bar, uint32_t parity) {
      if (!mbar_try_wait(bar, parity)) mbar_wait(bar, parity, abort_flag);
      __syncwarp();
    };
    int s = 0, slot = 0, free_s = 0, behind = 0;   // behind: steps whose scale slots may still be read
    uint32_t parity = 0, free_parity = 0;
    int i = 0;
    for (int t = tile0; t < p.total_tiles; t += tile_step, ++i) {
      int oc0, row0;
      decode(p, t, oc0, row0);
      const int b = i & 1;
      const uint32_t acc = tmem + (b ? p.acc1 : 0);
      const uint32_t sf_row = (uint32_t)(row0 & 127) >> 5;   // the tile's first 32-row group within its scale tile: 0 or 2
      if (i >= 2) wait(bar_pempty(b), ((i >> 1) & 1) ^ 1);
      if (over && i >= 1) wait(bar_shared(b ^ 1), ((i - 1) >> 1) & 1);
      for (int step = step0; step < step1; ++step) {
        if (behind == p.slots) {
          wait(bar_empty(free_s), free_parity);
          if (++free_s == p.stages) { free_s = 0; free_parity ^= 1; }
          --behind;
        }
        wait(bar_full(s), parity);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = smem_u32(ring + (size_t)s * p.stage_bytes);
        const uint32_t sfw = tmem + p.sf + slot * p.slot_cols, sfa = sfw + 4 * kTiles;
        const int n = min(kTiles, p.tiles_k - step * kTiles), mmas = step == p.steps - 1 ? p.last_mmas : 4;
        if (elect_one()) {
          const uint64_t dsw = scales_desc(at + p.sw_at), dsa = scales_desc(at + p.sa_at);
#pragma unroll
          for (int k = 0; k < kTiles; ++k) {
            if (k < n) {
              copy_scales(sfw + 4 * k, dsw + 32 * k);
              copy_scales(sfa + 4 * rt * k, dsa + 32 * k);
              if (rt == 2) copy_scales(sfa + 8 * k + 4, dsa + 32 * (kTiles + k));
            }
          }
          const uint64_t dw = codes_desc(at), da = codes_desc(at + p.a_at);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (j < mmas) {
              const int k = FMT == TETRIS_FP4_NV ? j : j >> 1;
              const uint32_t id = FMT == TETRIS_FP4_NV || !(j & 1) ? idesc : idesc | (2u << 4) | (2u << 29);  // (second half of the scale words)
              umma_fp4<FMT>(acc, dw + 2 * j, da + 2 * j, id, sfw + 4 * k, sfa + 4 * rt * k + sf_row, step > step0 || j > 0);
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
  } else {
    const int quarter = warp & 3, half = (warp - kFirstStore) >> 2;
    const int chunks = (p.nt + 31) / 32, shared = over ? (p.nt - p.acc1) / 32 : 0;
    int i = 0;
    for (int t = tile0; t < p.total_tiles; t += tile_step, ++i) {
      int oc0, row0;
      decode(p, t, oc0, row0);
      const int b = i & 1;
      if (!mbar_try_wait(bar_pfull(b), (i >> 1) & 1)) mbar_wait(bar_pfull(b), (i >> 1) & 1, abort_flag);
      __syncwarp();
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      if (p.d > 1) break;  // a slice of a tile: its sums stay in tensor memory until the cluster meets
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + (b ? p.acc1 : 0);
      const int oc = oc0 + quarter * 32 + lane;
      const float bias = p.bias && oc < p.N ? p.bias[oc] : 0.f;
      bool told = !over;
      for (int c = half; c < chunks; c += 2) {
        const int chunk = b ? c : chunks - 1 - c;  // the shared columns: the first accumulator's last, the second one's first
        if (!told && c >= shared) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_shared(b));
          told = true;
        }
        uint32_t v[32];
        tmem_ld32(acc + chunk * 32, v);
        const int row = row0 + chunk * 32, n = oc < p.N ? p.rows - row : 0;
        T *y = static_cast<T *>(p.y) + (int64_t)row * p.ld + oc;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          float u = __uint_as_float(v[j]) * p.scale0 * p.scale1 + bias;
          if (p.relu && u < 0.f) u = 0.f;  // (a NaN stays)
          if (j < n) y[j * p.ld] = to_type<T>(u);
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (!told) mbar_arrive(bar_shared(b));
        mbar_arrive(bar_pempty(b));
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (*abort_flag) {  // what this CTA has in flight must land before it leaves
    if (tid == 0)
      for (int v = max(loads - p.stages, p.withhold_first_load ? 1 : 0); v < loads; ++v) mbar_drain(bar_full(v % p.stages), (uint32_t)(v / p.stages) & 1u);
    if (warp == 1) {
      if (elect_one()) umma_commit(bar_drain());
      __syncwarp();
      mbar_drain(bar_drain(), 0);
    }
    if (tid == 0) atomicExch(p.error_flag, 1);
  }
  if (p.d > 1) {
    // The slices of a tile meet: a CTA owns `per` rows; each pushes its sums of a row (128 channels) to the
    // owner, once every ring of the cluster is idle, and the owner adds them up in slice order.
    const int per = (p.nt + p.d - 1) / p.d;
    int oc0, row0;
    decode(p, tile0, oc0, row0);
    const int live = min(p.nt, p.rows - row0);
    cluster_sync_all();
    if (warp >= kFirstStore && !*abort_flag) {
      const int quarter = warp & 3, half = (warp - kFirstStore) >> 2;
      const uint32_t mine = smem_u32(ring) + (uint32_t)(quarter * 32 + lane) * 4u;
      for (int c = half * 32; c < live; c += 64) {
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          if (c + j < live) {
            const int owner = (c + j) / per;
            st_cluster(cluster_addr(mine + (uint32_t)((rank * per + c + j - owner * per) * kChannels) * 4u, (uint32_t)owner), __uint_as_float(v[j]));
          }
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // (all sums have arrived; nothing reaches into another CTA after this)
    const float *sums = reinterpret_cast<const float *>(ring);
    const int mine = *abort_flag ? 0 : min(per, live - rank * per);
    for (int e = tid; e < mine * kChannels; e += kThreads) {
      const int j = e / kChannels, c = e % kChannels, oc = oc0 + c;
      if (oc >= p.N) continue;
      float u = 0.f;
      for (int s = 0; s < p.d; ++s) u += sums[(s * per + j) * kChannels + c];
      u = u * p.scale0 * p.scale1 + (p.bias ? p.bias[oc] : 0.f);
      if (p.relu && u < 0.f) u = 0.f;
      static_cast<T *>(p.y)[(int64_t)(row0 + rank * per + j) * p.ld + oc] = to_type<T>(u);
    }
  }
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
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

constexpr size_t kSmemMost = 227 * 1024 - 1024;   // (the ring is aligned to 1024 bytes)
constexpr size_t kSmemLeast = 117 * 1024;         // one CTA per SM, also beside the other kernels that take all of an SM's tensor memory

struct Geometry {
  int nt, d;
};

Geometry choose(const tetris_fp4_filter *f, int64_t rows) {
  const int steps = (f->in_channel + kStep - 1) / kStep, oc_tiles = (f->out_channel + kChannels - 1) / kChannels;
  Geometry best = {16, 1};
  double least = 1e300;
  for (int nt = 16; nt <= 256; nt *= 2) {
    // The scales of a tile begin at its first 32-row group's column, and an MMA takes scales from even columns
    // only (an odd one is a misaligned address): tiles below 64 rows begin at row 0.
    if (nt < 64 && rows > nt) continue;
    const int64_t tiles = (rows + nt - 1) / nt * oc_tiles;
    for (int d = 1; d <= 8; d *= 2) {
      if (d > 1 && (d > steps || nt > 64 || tiles * d > f->sm_count)) continue;
      const double waves = (double)((tiles * d + f->sm_count - 1) / f->sm_count);
      const double step = std::max(2.0 * nt, (kChannels * 144 + nt * 144) / 40.0), store = 300 + 6.0 * nt;
      const double cost = waves * ((double)((steps + d - 1) / d) * step + (d > 1 ? 2000 : 0)) + (waves > 1 ? 0 : store) + 2000;
      if (cost < least) { least = cost; best = {nt, d}; }
    }
  }
  return best;
}

template <int FMT, typename T>
int launch(const CUtensorMap &map_w, const CUtensorMap &map_a, const ProductParams &p, unsigned grid, size_t smem, cudaStream_t st) {
  static bool ready[64] = {};  // per device
  int dev = 0;
  TETRIS_CUDA_TRY(cudaGetDevice(&dev));
  if (dev >= 64 || !ready[dev]) {
    TETRIS_CUDA_TRY(cudaFuncSetAttribute(product_kernel<FMT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSmemMost + 1024)));
    if (dev < 64) ready[dev] = true;
  }
  TETRIS_CUDA_TRY(launch_overlapped(product_kernel<FMT, T>, dim3(grid), kThreads, smem, st, (unsigned)p.d, map_w, map_a, p));
  count_launch();
  return TETRIS_OK;
}

int encode(CUtensorMap *map, const uint8_t *codes, int64_t pitch, int64_t rows, int box_rows) {
  EncodeFn enc = get_encode();
  if (!enc) { set_error("cuTensorMapEncodeTiled is not available from this driver"); return TETRIS_ERR_UNSUPPORTED; }
  const cuuint64_t dims[2] = {(cuuint64_t)pitch, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)pitch};
  const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { set_error("cuTensorMapEncodeTiled failed with code %d", (int)r); return TETRIS_ERR_CUDA; }
  return TETRIS_OK;
}

}  // namespace

int launch_fp4_product(const tetris_fp4_filter *f, const uint8_t *codes, const uint8_t *scales, int64_t rows, int exponent, const float *bias,
                       void *y, int y_type, int64_t ld, int relu, cudaStream_t st) {
  const Geometry g = choose(f, rows);
  const bool nv = f->format == TETRIS_FP4_NV;
  const int kt = step_tiles(f->format), rt = g.nt > 128 ? 2 : 1;
  ProductParams p = {};
  p.scales_a = scales; p.scales_w = f->d_scales; p.bias = bias;
  p.y = y; p.ld = ld;
  p.rows = (int)rows; p.N = f->out_channel;
  p.steps = (f->in_channel + kStep - 1) / kStep;
  p.last_mmas = (f->in_channel - (p.steps - 1) * kStep + 63) / 64;
  p.tiles_k = fp4_tiles(f->in_channel, f->format);
  p.nt = g.nt; p.d = g.d;
  p.row_tiles_128 = (int)((rows + 127) / 128);
  p.oc_tiles = (f->out_channel + kChannels - 1) / kChannels;
  p.row_tiles = (int)((rows + g.nt - 1) / g.nt);
  p.group = std::min(p.oc_tiles, 8);
  const int64_t total = (int64_t)p.oc_tiles * p.row_tiles;
  if (total > 0x3FFFFFFF) { set_error("a product of %lld tiles is outside what the kernels cover", (long long)total); return TETRIS_ERR_UNSUPPORTED; }
  p.total_tiles = (int)total;
  p.a_at = kChannels * 128;
  p.sw_at = p.a_at + std::max(g.nt * 128, 2048);
  p.sa_at = p.sw_at + kt * 512;
  p.stage_bytes = (p.sa_at + rt * kt * 512 + 1023) / 1024 * 1024;
  const size_t tail = kBars * 8 + 16;
  p.stages = std::min<int>(kStagesMax, (int)((kSmemMost - tail) / p.stage_bytes));
  p.slot_cols = 4 * kt * (1 + rt);
  p.slots = rt == 2 ? 2 : std::min(kSlotsMax, p.stages);  // (at most `stages`: a step's empty barrier is waited for before the stage is used again)
  p.sf = kTmemCols - p.slots * p.slot_cols;
  p.acc1 = std::min(std::max(g.nt, 32), (p.sf - g.nt) / 32 * 32);
  const int e = exponent + f->exponent, e0 = std::max(-126, std::min(126, e));
  p.scale0 = ldexpf(1.f, e0); p.scale1 = ldexpf(1.f, e - e0);
  p.relu = relu;
  p.error_flag = f->d_error;
  p.withhold_first_load = test_injection(&p.spin_limit);
  CUtensorMap map_w, map_a;
  int rc;
  if ((rc = encode(&map_w, f->d_codes, f->pitch, f->out_channel, kChannels)) || (rc = encode(&map_a, codes, f->pitch, rows, g.nt))) return rc;
  const unsigned grid = (unsigned)(g.d > 1 ? p.total_tiles * g.d : std::min(p.total_tiles, f->sm_count));
  const size_t smem = std::max(kSmemLeast, (size_t)p.stages * p.stage_bytes + tail + 1024);
  switch (y_type) {
    case TETRIS_FP32: return nv ? launch<TETRIS_FP4_NV, float>(map_w, map_a, p, grid, smem, st) : launch<TETRIS_FP4_MX, float>(map_w, map_a, p, grid, smem, st);
    case TETRIS_BF16: return nv ? launch<TETRIS_FP4_NV, __nv_bfloat16>(map_w, map_a, p, grid, smem, st) : launch<TETRIS_FP4_MX, __nv_bfloat16>(map_w, map_a, p, grid, smem, st);
    default: return nv ? launch<TETRIS_FP4_NV, __half>(map_w, map_a, p, grid, smem, st) : launch<TETRIS_FP4_MX, __half>(map_w, map_a, p, grid, smem, st);
  }
}

}  // namespace tetris
