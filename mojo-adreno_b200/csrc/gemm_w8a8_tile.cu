// The int8 products for many tokens: pairs of CTAs on 256 x 256 tiles (see gemm_w8a8.cu for the operator).
//
//  * Here the tokens are the MMA's A and the weights its B. A pair of CTAs (tcgen05 cta_group::2, M = 256,
//    N = 256, K = 32 per instruction) works on 256 tokens x 256 weight rows: each CTA loads 128 rows of
//    each, its TMEM holds its 128 tokens x 256 int32 sums, and the instruction reads both CTAs' shared memory. Per
//    stage of 128 k a CTA fetches 32 KB for 512 cycles of MMA, where one CTA alone on 128 x 256 would
//    need 48 KB (gate|up 8192x12288x4096: 435 us against the streaming kernel's 570 with constant operands;
//    with random ones power caps the clock and it takes 526-600 us, 2.7-3.1 POP/s).
//  * gate|up: the even CTA loads 128 gate rows, the odd one the matching 128 up rows, so columns j and
//    128 + j of the tile belong together and one thread holds both.
//  * Persistent pairs over the tiles in bands of 8 token tiles (a band's tokens and the weights it walks
//    through stay in L2), accumulators double-buffered (2 x 256 columns of TMEM): eight warps of each
//    CTA scale, convert and store one tile while the next one is multiplied.
//  * The epilogue stages 32 rows x 128 bytes per warp in the swizzled layout and writes it with one TMA
//    store, which clips the last rows and columns. y whose rows are not 16-byte aligned, and add, are
//    written from the staged rows by plain stores, consecutive lanes on consecutive outputs.
#include "common.cuh"

namespace mq {
namespace w8 {

constexpr int kTileM = 256, kTileB = 256;   // tokens and weight rows of a pair's tile
constexpr int kTileStages = 5, kTileStageBytes = 2 * 128 * kBK;
constexpr int kTileEpiWarps = 8, kTileThreads = 64 + 32 * kTileEpiWarps;
constexpr int kStageOutBytes = 4096;        // 32 rows x 128 bytes
constexpr int kTileSmem = kTileStages * kTileStageBytes + kTileEpiWarps * 2 * kStageOutBytes + 1024;
constexpr int kBand = 8, kTileMaxSplits = 4;

struct TileParams {
  const float *xs, *ws, *bias;
  void *y;
  int64_t ldy;
  int y_dtype, add, y_tma;
  int m, n, k;  // n: output columns
  int tiles_m, tiles_n, tiles;
  int splits;  // pairs of a cluster that share a tile's k (1: persistent pairs, each tile's k whole)
};

__device__ __forceinline__ void mbar_arrive_remote(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A load into this CTA's shared memory that completes on a barrier of this or the paired CTA.
__device__ __forceinline__ void tma_load_2d_pair(void *dst, const CUtensorMap *map, uint32_t bar_cluster, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` of both CTAs of the pair once every MMA this thread issued has completed.
__device__ __forceinline__ void umma_commit_pair(uint64_t *bar, uint16_t mask) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   smem_u32(bar)),
               "h"(mask)
               : "memory");
}

struct TileAt {
  int m0, n0;
};
template <int P>
__device__ __forceinline__ TileAt tile_at(const TileParams &p, int t) {
  const int per_band = kBand * p.tiles_n, band = t / per_band, r = t - band * per_band;
  const int height = min(kBand, p.tiles_m - band * kBand);
  return {(band * kBand + r % height) * kTileM, r / height * (kTileB / P)};
}

template <int P>
__global__ void __launch_bounds__(kTileThreads, 1)
    w8a8_tile_kernel(const __grid_constant__ CUtensorMap xmap, const __grid_constant__ CUtensorMap wmap,
                     const __grid_constant__ CUtensorMap ymap, const TileParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *out_stage = ring + kTileStages * kTileStageBytes;
  __shared__ uint64_t full[kTileStages], empty[kTileStages], tfull[2], tempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  constexpr int S = kTileStages;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t crank = cluster_rank(), rank = crank & 1, leader = crank & ~1u;  // rank: within the pair
  const int split = crank / 2, nkb_all = (p.k + kBK - 1) / kBK;
  const int kb0 = nkb_all * split / p.splits, nkb = nkb_all * (split + 1) / p.splits - kb0;
  const int first = blockIdx.x / (2 * p.splits), step = gridDim.x / (2 * p.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);   // the even CTA's: both CTAs' copies complete on it
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2 * kTileEpiWarps);  // the even CTA's: both CTAs' epilogue warps
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  griddep_wait();  // (before TMEM is taken, as in the streaming kernel)
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the pair's barriers exist before anything completes on them
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = tmem_slot;
  bool live = false;  // an epilogue warp of a split tile whose sums are in TMEM

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&xmap);
      prefetch_tmap(&wmap);
    }
    int s = 0, round = 0;
    int64_t issued = 0;
    bool ok = true;
    for (int t = first; ok && t < p.tiles; t += step) {
      const TileAt at = tile_at<P>(p, t);
      const int m0 = at.m0 + 128 * rank, n0 = at.n0 + (P == 1 ? 128 : p.n) * rank;
      for (int kb = 0; kb < nkb; ++kb) {
        if (round > 0 && !__all_sync(0xffffffffu, mbar_wait(&empty[s], (round - 1) & 1))) {
          if (lane == 0) {
            raise_status(kStatusW8TmaWait);
            abort_flag = 1;
          }
          ok = false;
          break;
        }
        if (lane == 0 && rank == 0) mbar_expect_tx(&full[s], 2 * kTileStageBytes);
        __syncwarp();
        if (lane < 2)  // lane 0: the tokens, lane 1: the weights
          tma_load_2d_pair(ring + s * kTileStageBytes + lane * 128 * kBK, lane ? &wmap : &xmap,
                           map_shared(smem_u32(&full[s]), leader), (kb0 + kb) * kBK, lane ? n0 : m0);
        ++issued;
        if (++s == S) s = 0, ++round;
      }
    }
    // Leave no copy in flight: the MMAs that read the last copy into each slot have finished.
    if (lane == 0)
      for (int64_t i = issued > S ? issued - S : 0; i < issued; ++i) mbar_wait(&empty[i % S], (i / S) & 1);
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = umma_idesc_i8(256, 256);
      const uint16_t both = static_cast<uint16_t>(3u << leader);
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int t = first; t < p.tiles; t += step, ++it) {
        const int b = it & 1;
        bool ok = mbar_wait(&tempty[b], ((it >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int kb = 0; ok && kb < nkb; ++kb) {
          if (!mbar_wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + s * kTileStageBytes);
          const uint64_t da = umma_desc_sw128(base), db = umma_desc_sw128(base + 128 * kBK);
#pragma unroll
          for (int j = 0; j < kBK / 32; ++j) umma_i8_pair(tmem + b * 256, da + 2 * j, db + 2 * j, idesc, kb != 0 || j != 0);
          umma_commit_pair(&empty[s], both);
          if (++s == S) s = 0, ph ^= 1;
        }
        umma_commit_pair(&tfull[b], both);
        if (!ok) {
          raise_status(kStatusW8MmaWait);
          abort_flag = 1;
          mbar_wait(&tfull[b], (it >> 1) & 1);  // the MMAs that were issued have finished
          break;
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    uint8_t *mine = out_stage + (warp - 2) * 2 * kStageOutBytes;
    const uint32_t tempty_leader[2] = {map_shared(smem_u32(&tempty[0]), leader), map_shared(smem_u32(&tempty[1]), leader)};
    const bool f32 = p.y_dtype == MQ_F32 || p.add;  // staged as fp32: y is added before the one rounding
    constexpr int width = 128 / P, kChunks = width / 32;  // output columns of this half of the warps
    int it = 0, buf = 0;
    for (int t = first; t < p.tiles; t += step, ++it) {
      const int b = it & 1;
      const TileAt at = tile_at<P>(p, t);
      const int row0 = at.m0 + 128 * rank + 32 * quarter, row = row0 + lane;
      // Scales and biases come while the tile is still being multiplied: fetched at their use they cost the
      // epilogue an L2 latency per 32 columns (2.4 instead of 1 us a tile). Lane l holds column c + l's.
      const float sx = row < p.m ? p.xs[row] : 0.f;
      float sw[kChunks], more[kChunks];  // more: the up scales, or the bias
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int col = at.n0 + half * width + 32 * i + lane;
        sw[i] = col < p.n ? p.ws[col] : 0.f;
        more[i] = col >= p.n ? 0.f : P == 2 ? p.ws[p.n + col] : p.bias ? p.bias[col] : 0.f;
      }
      const bool ok = !abort_flag && mbar_wait(&tfull[b], (it >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok && !abort_flag)) {
        if (lane == 0 && !abort_flag) {
          raise_status(kStatusW8EpiWait);
          abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      if (p.splits > 1) {  // the one tile of this cluster: joined below
        live = true;
        break;
      }
      const uint32_t acc = tmem + b * 256 + lanes + half * width;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        const int c = 32 * i, col0 = at.n0 + half * width + c;
        float v[32];
        tmem_ld32(acc + c, v);
        if (P == 2) {
          float u[32];
          tmem_ld32(acc + 128 + c, u);
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j] = silu_mul(static_cast<float>(__float_as_int(v[j])) * sx * __shfl_sync(0xffffffffu, sw[i], j),
                            static_cast<float>(__float_as_int(u[j])) * sx * __shfl_sync(0xffffffffu, more[i], j));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            v[j] = static_cast<float>(__float_as_int(v[j])) * sx * __shfl_sync(0xffffffffu, sw[i], j);
          if (p.bias) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += __shfl_sync(0xffffffffu, more[i], j);
          }
        }
        if (c + 32 >= width) {  // the last read of this accumulator
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_remote(tempty_leader[b]);
        }
        // fp32: a staged row of 128 bytes is these 32 columns; 16-bit types: two such steps fill it.
        const int part = f32 ? 0 : c / 32 & 1;
        if (part == 0) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");  // this buffer is free again
          __syncwarp();
        }
        uint8_t *dst = mine + buf * kStageOutBytes + lane * 128;
        if (f32) {
#pragma unroll
          for (int u = 0; u < 8; ++u)
            *reinterpret_cast<float4 *>(dst + (u ^ (lane & 7)) * 16) = make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const float lo = v[8 * u + 2 * h], hi = v[8 * u + 2 * h + 1];
              if (p.y_dtype == MQ_F16) {
                w[h] = pack_half2(lo, hi);
              } else {
                const __nv_bfloat162 b2 = __floats2bfloat162_rn(lo, hi);
                w[h] = *reinterpret_cast<const uint32_t *>(&b2);
              }
            }
            *reinterpret_cast<uint4 *>(dst + ((4 * part + u) ^ (lane & 7)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        if (f32 || part == 1) {
          const int x = f32 ? col0 : col0 - 32;
          if (p.y_tma) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (x < p.n && row0 < p.m) tma_store_2d(&ymap, mine + buf * kStageOutBytes, x, row0, false);
              asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
          } else {  // a row at a time, consecutive lanes on consecutive outputs
            __syncwarp();
            by_type(p.y_dtype, [&](auto type) {
              using T = decltype(type);
              const uint8_t *const staged = mine + buf * kStageOutBytes;
              const int cols = p.n - x;
              T *y = static_cast<T *>(p.y) + row0 * p.ldy + x + lane;
              const int rows = min(32, p.m - row0);
              // Eight rows are read before any is written: the compiler may not move the reads across the writes.
#pragma unroll 1
              for (int r0 = 0; r0 < rows; r0 += 8, y += 8 * p.ldy) {
                if (f32) {
                  float o[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    o[i] = *reinterpret_cast<const float *>(staged + (r0 + i) * 128 + ((lane / 4) ^ i) * 16 + lane % 4 * 4);
                  if (p.add) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                      if (r0 + i < rows && lane < cols) o[i] += static_cast<float>(y[i * p.ldy]);
                  }
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    if (r0 + i < rows && lane < cols) y[i * p.ldy] = from_float<T>(o[i]);
                } else {
                  T o[8][2];
#pragma unroll
                  for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                      const int at = 32 * h + lane;
                      o[i][h] = *reinterpret_cast<const T *>(staged + (r0 + i) * 128 + ((at / 8) ^ i) * 16 + at % 8 * 2);
                    }
#pragma unroll
                  for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                      if (r0 + i < rows && 32 * h + lane < cols) y[i * p.ldy + 32 * h] = o[i][h];
                }
              }
            });
          }
          buf ^= 1;
        }
      }
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // shared memory stays until it is read
  }
  if (p.splits > 1) {
    // Join the splits' int32 sums through distributed shared memory: groups of 32 columns are dealt to the
    // cluster's pairs in turn; a pair's even CTA joins its own rows, the odd one its. The parts land in the
    // ring and the staging area, [split][plane][group][4 columns][row] of int4, once the MMAs are done.
    cluster_sync_all();
    constexpr int kGroups = 256 / P / 32;
    const int owned = (kGroups + p.splits - 1) / p.splits, quarter = warp & 3, half = (warp - 2) >> 2;
    if (live) {
      const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t row_at = smem_u32(ring) + (quarter * 32 + lane) * 16;
      for (int g = half; g < kGroups; g += 2) {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          float v[32];
          tmem_ld32(acc + q * 128 + 32 * g, v);
          const uint32_t dst = map_shared(row_at + ((split * P + q) * owned + g / p.splits) * 8 * 128 * 16,
                                          2 * (g % p.splits) + rank);
#pragma unroll
          for (int u = 0; u < 8; ++u)
            st_remote_v4(dst + u * 128 * 16, make_int4(__float_as_int(v[4 * u]), __float_as_int(v[4 * u + 1]),
                                                       __float_as_int(v[4 * u + 2]), __float_as_int(v[4 * u + 3])));
        }
      }
    }
    cluster_sync_all();
    const TileAt at = tile_at<P>(p, first);
    const int row = at.m0 + 128 * rank + quarter * 32 + lane;
    if (live && !abort_flag) {
      const float sx = row < p.m ? p.xs[row] : 0.f;
      for (int o = 0; split + o * p.splits < kGroups; ++o) {  // 16 columns of each group for this warp
        const int col0 = at.n0 + (split + o * p.splits) * 32 + half * 16, col = col0 + lane % 16;
        const float sw = col < p.n ? p.ws[col] : 0.f;
        const float more = col >= p.n ? 0.f : P == 2 ? p.ws[p.n + col] : p.bias ? p.bias[col] : 0.f;
        int a[P][16] = {};
#pragma unroll
        for (int z = 0; z < kTileMaxSplits; ++z)
          if (z < p.splits)
#pragma unroll
            for (int q = 0; q < P; ++q)
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int4 v = *reinterpret_cast<const int4 *>(
                    ring + ((((z * P + q) * owned + o) * 8 + half * 4 + u) * 128 + quarter * 32 + lane) * 16);
                a[q][4 * u] += v.x, a[q][4 * u + 1] += v.y, a[q][4 * u + 2] += v.z, a[q][4 * u + 3] += v.w;
              }
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float wj = __shfl_sync(0xffffffffu, sw, j), mj = __shfl_sync(0xffffffffu, more, j);
          v[j] = static_cast<float>(a[0][j]) * sx * wj;
          v[j] = P == 2 ? silu_mul(v[j], static_cast<float>(a[P - 1][j]) * sx * mj) : v[j] + mj;
        }
        if (row < p.m)
          by_type(p.y_dtype, [&](auto type) {
            using T = decltype(type);
            T *const y = static_cast<T *>(p.y) + row * p.ldy + col0;
            if (p.y_tma && col0 + 16 <= p.n) {  // 16-byte aligned rows
              struct alignas(16) Vec {
                T t[16 / sizeof(T)];
              };
#pragma unroll
              for (int j = 0; j < 16; j += 16 / sizeof(T)) {
                Vec o16;
#pragma unroll
                for (int i = 0; i < 16 / sizeof(T); ++i) o16.t[i] = from_float<T>(v[j + i]);
                *reinterpret_cast<Vec *>(y + j) = o16;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (col0 + j < p.n) y[j] = from_float<T>(p.add ? v[j] + static_cast<float>(y[j]) : v[j]);
            }
          });
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // neither CTA's barriers or operands go away while the other uses them
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

template <int P>
int launch_tile(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, const Params &q, cudaStream_t stream,
                const DeviceInfo &dev, const char *what, int splits) {
  TileParams p{};
  p.xs = q.xs, p.ws = q.ws, p.bias = q.bias, p.y = q.y, p.ldy = q.ldy, p.y_dtype = q.y_dtype, p.add = q.add;
  p.m = q.m, p.n = q.n, p.k = q.k;
  p.tiles_m = (p.m + kTileM - 1) / kTileM;
  p.tiles_n = (p.n + kTileB / P - 1) / (kTileB / P);
  p.tiles = p.tiles_m * p.tiles_n;
  p.splits = splits;
  const int es = p.y_dtype == MQ_F32 ? 4 : 2;
  p.y_tma = !p.add && aligned(p.y, 16) && p.ldy * es % 16 == 0;
  CUtensorMap xmap, wmap, ymap;
  if (int rc = encode_tmap_2d_now(&xmap, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, p.m, ldx, kBK, 128,
                                  CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  if (int rc = encode_tmap_2d_now(&wmap, wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, static_cast<uint64_t>(P) * p.n, ldw, kBK,
                                  128, CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  ymap = xmap;  // not used without y_tma
  if (p.y_tma)
    if (int rc = encode_tmap_2d_now(&ymap, p.y, p.y_dtype == MQ_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                              : p.y_dtype == MQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                    es, p.n, p.m, p.ldy * es, 128 / es, 32, CU_TENSOR_MAP_SWIZZLE_128B, what))
      return rc;
  auto kern = w8a8_tile_kernel<P>;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(kern, kTileSmem, configured, what)) return rc;
  const int grid = 2 * (p.splits > 1 ? p.tiles * p.splits : std::min(p.tiles, dev.sms / 2));
  return launch_overlapped_clusters(kern, dim3(grid), dim3(kTileThreads), 2 * p.splits, kTileSmem, stream, what, xmap, wmap,
                                    ymap, p);
}

}  // namespace w8
}  // namespace mq
