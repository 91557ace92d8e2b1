// int8 matrix products with a scale per token and per output channel (mq_gemm_w8a8, mq_gate_up_w8a8).
//
// y[t][r] = xs[t] * ws[r] * sum_k xq[t][k] * wq[r][k], xq [m][k] and wq [n][k] int8 rows, the sums exact
// in int32 (k <= 131071: 128 * 128 * k < 2^31). The gate|up form multiplies by both halves of a fused
// [2f][k] matrix and writes silu(gate) * up.
//  * The MMA sees the weights as A (128 rows) and the tokens as B (bn of them, a multiple of 16 up to
//    256), so the accumulator in TMEM is [128 weight rows][bn tokens]: a decode batch pads its tokens to
//    16, not to 128, and an epilogue warp writes 32 consecutive outputs of one token at a time.
//  * gate|up: two weight tiles per stage (128 gate rows, the matching 128 up rows) into two accumulators,
//    so one thread holds both values of an output.
//  * Persistent CTAs: warp 0 streams 128-byte k blocks of both operands through a ring of TMA slots that
//    keeps running across tiles, one thread of warp 1 issues tcgen05.mma kind::i8, warps 2-5 move the
//    finished accumulator out while the next tile's (the other half of TMEM) is being computed.
//  * Few tiles: a cluster of up to 8 CTAs shares a tile's k, each with its part of the sums, joined in
//    distributed shared memory in int32: exact, so the result does not depend on the split.
// Decode is bound by the weights' bytes once every SM has a tile, below that by latency; B200: head 128256x2048
// for one token 42-44 us (6.2 TB/s, 0.96 of the copy bandwidth), 2048x2048 4.2 us, gate|up 64x8192x2048
// 11.9 us (64 CTAs: 2.9 TB/s), 431x2048x8192 14.0 us (the join of 224 x 128 parts takes a third of it:
// distributed shared memory moves 32 GB/s per SM, by stores as by bulk copies).
// Many tokens go to pairs of CTAs (gemm_w8a8_tile.cu).
// Every wait on an mbarrier is bounded; on a time-out the kernel records a status code, stops issuing,
// drains its copies, frees its TMEM and returns.
#include <algorithm>

#include "common.cuh"

namespace mq {
namespace w8 {

constexpr int kRows = 128;      // weight rows of a tile (the MMA's M)
constexpr int kBK = 128;        // k per stage: one 128-byte swizzled row
constexpr int kMaxStages = 12;
constexpr int kEpiWarps = 4;    // one per TMEM lane quarter; eight measured slower (4.4 -> 5.8 us for 1x2048x2048)
constexpr int kThreads = 64 + 32 * kEpiWarps;  // warp 0 TMA, warp 1 MMA + TMEM, then the epilogue
constexpr int kWBytes = kRows * kBK;
constexpr int kStaticShared = 4352;  // of w8a8_kernel (barriers, token scales), as ptxas reports it
constexpr int kMaxSplits = 8;
// Clusters of 1 .. 8 CTAs, one CTA per SM, that run at once on a B200 (cudaOccupancyMaxActiveClusters; the
// SMs of a cluster share a GPC): a split whose clusters do not all fit takes twice as long (16 clusters
// of 8: 4.9 -> 8.3 us for 1x2048x2048).
__host__ __device__ constexpr int clusters_at_once(int size) {
  return size == 1 ? 148 : size == 2 ? 74 : size == 3 ? 45 : size == 4 ? 33 : size == 5 ? 26 : size == 6 ? 22 : 15;
}
constexpr int64_t kMaxK = 131071;  // 128 * 128 * k stays below 2^31
// 128-k blocks per stage: the issuing thread's wait and commit cost about 0.17 us together, four 128 x 16 MMAs 0.1 us,
// so a stage has eight MMAs at least (16x2048x8192 on 16 CTAs 21.8 -> 15.5 us), and sixteen where that leaves the
// ring slots small enough, up to 32 tokens (12.9 us; head for one token 43.7 -> 41.8, gate|up 1x8192x2048 10.1 -> 8.9;
// with 64 tokens the fewer slots cost more: gate|up 64x12288x4096 20.8 -> 21.8).
__host__ __device__ constexpr int sub_blocks(int planes, int bn) { return (planes == 1 ? 2 : 1) * (bn <= 32 ? 2 : 1); }

struct Params {
  const float *xs, *ws, *bias;
  void *y;
  int64_t ldy;
  int y_dtype, add;
  int m, n, k;      // n: output columns (f of the gate|up form)
  int bn, tiles_m, tiles;
  int splits;       // CTAs of a cluster that share a tile's k (1: persistent CTAs, each tile's k whole)
  int stages, buf_cols, tmem_cols;  // TMEM columns of one accumulator buffer (all planes), allocated
};

// D[tmem] (+)= A[smem] * B[smem]^T on int8, int32 accumulator; issued by one thread.
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Instruction descriptor of kind::i8: int32 accumulator, signed A and B, both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();  // the barrier is taken by whole warps; of some, one lane comes from a branch of its own
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The address of the same shared variable in the CTA of the given rank of this cluster.
__device__ __forceinline__ uint32_t map_shared(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void st_remote_v4(uint32_t cluster_addr, int4 v) {
  asm volatile("st.shared::cluster.v4.s32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr), "r"(v.x), "r"(v.y), "r"(v.z),
               "r"(v.w)
               : "memory");
}

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// silu(g) * u = g / (1 + e^-g) * u through E = e^-|g|, at most 1: g / (1 + E) where g is positive, g E / (1 + E) where it
// is not, so the divisor stays within 1 .. 2 and its reciprocal is good to an ulp. E = 2^t (1 + c) with t = -|g| log2 e
// rounded and c = -|g| - t ln 2 what the rounding took (ln 2 in two parts): without c the error would grow with |g|, to some
// 80 ulp. As it is the whole stays within 6 * 2^-23 (2^t two, the rest roundings), and E, so the result, is 0 below
// g = -87.3, where silu is above -1.1e-36. gate|up 2048x8192x512 fp16 37.2 us, fp32 37.2, 400x8192x2048 bf16 18.5; with expf
// and a division 41.1, 40.9 and 18.8, with an E that keeps its subnormals 40.1, 40.5 and 19.0; c for fp32 outputs only, in
// two copies of the loops, 35.6, 39.2 and 18.4: not kept for what it takes from fp32.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float a = fmaxf(-fabsf(g), -200.f), t = a * 1.44269504f;  // (of an infinite g, c would be NaN)
  const float c = fmaf(t, 1.904654299e-9f, fmaf(t, -0.693147182f, a));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  e = fmaf(e, c, e);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return g * (g < 0.f ? e : 1.f) * r * u;
}

template <int P, int SUB>  // weight planes of a tile: 1, or 2 (gate and up); 128-k blocks per stage
__global__ void __launch_bounds__(kThreads, 1)
    w8a8_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2];
  __shared__ __align__(16) float token_scale[kEpiWarps][256];  // a copy for each epilogue warp
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int S = p.stages, sub_bytes = P * kWBytes + p.bn * kBK, slot_bytes = SUB * sub_bytes;
  const int nst_all = (p.k + SUB * kBK - 1) / (SUB * kBK);
  const int split = p.splits > 1 ? static_cast<int>(cluster_rank()) : 0;
  const int st0 = nst_all * split / p.splits, nst = nst_all * (split + 1) / p.splits - st0;
  const int first = blockIdx.x / p.splits, step = gridDim.x / p.splits;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 32 * kEpiWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  // TMEM is taken when the kernels before this one have theirs back, and the kernels after it start when it has
  // been taken: a grid that waits for another never holds TMEM that the other still needs.
  griddep_wait();
  if (warp == 1) tmem_alloc(&tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = tmem_slot;
  bool live = false;  // an epilogue warp of a split tile whose sums are in TMEM
  float sw = 0.f, su = 0.f, bias = 0.f;  // of an epilogue thread's weight row

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&wmap);
      prefetch_tmap(&xmap);
    }
    int s = 0, round = 0;
    int64_t issued = 0;
    bool ok = true;
    for (int t = first; ok && t < p.tiles; t += step) {
      const int m0 = t % p.tiles_m * p.bn, n0 = t / p.tiles_m * kRows;
      for (int st = 0; st < nst; ++st) {
        if (round > 0 && !__all_sync(0xffffffffu, mbar_wait(&empty[s], (round - 1) & 1))) {
          if (lane == 0) {
            raise_status(kStatusW8TmaWait);
            abort_flag = 1;
          }
          ok = false;
          break;
        }
        if (lane == 0) mbar_expect_tx(&full[s], slot_bytes);
        __syncwarp();
        if (lane < SUB * (P + 1)) {  // per 128 k: P weight planes, then the tokens; one instruction for all
          const int j = lane / (P + 1), q = lane % (P + 1);
          tma_load_2d(ring + s * slot_bytes + j * sub_bytes + q * kWBytes, q < P ? &wmap : &xmap, &full[s],
                      ((st0 + st) * SUB + j) * kBK, q < P ? n0 + q * p.n : m0);
        }
        ++issued;
        if (++s == S) s = 0, ++round;
      }
    }
    // Leave no copy in flight: the last load issued into each slot has landed before the CTA ends.
    if (lane == 0)
      for (int64_t i = issued > S ? issued - S : 0; i < issued; ++i) mbar_wait(&full[i % S], (i / S) & 1);
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_i8(kRows, p.bn);
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int t = first; t < p.tiles; t += step, ++it) {
        const int b = it & 1;
        bool ok = mbar_wait(&tempty[b], ((it >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int st = 0; ok && st < nst; ++st) {
          if (!mbar_wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + s * slot_bytes);
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            const uint64_t db = umma_desc_sw128(base + u * sub_bytes + P * kWBytes);
#pragma unroll
            for (int q = 0; q < P; ++q) {
              const uint64_t da = umma_desc_sw128(base + u * sub_bytes + q * kWBytes);
              const uint32_t d = tmem + b * p.buf_cols + q * (p.buf_cols / P);
#pragma unroll
              for (int j = 0; j < kBK / 32; ++j) umma_i8(d, da + 2 * j, db + 2 * j, idesc, st != 0 || u != 0 || j != 0);
            }
          }
          umma_commit(&empty[s]);
          if (++s == S) s = 0, ph ^= 1;
        }
        umma_commit(&tfull[b]);
        if (!ok) {
          raise_status(kStatusW8MmaWait);
          abort_flag = 1;
          mbar_wait(&tfull[b], (it >> 1) & 1);  // the MMAs that were issued have finished
          break;
        }
      }
    }
  } else {
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    float *sx = token_scale[warp - 2];
    int it = 0;
    for (int t = first; t < p.tiles; t += step, ++it) {
      const int b = it & 1;
      // The scales are fetched while the tile is still being multiplied.
      const int m0 = t % p.tiles_m * p.bn, toks = min(p.bn, p.m - m0), r = t / p.tiles_m * kRows + row;
      const bool in = r < p.n;
      sw = in ? p.ws[r] : 0.f, su = in && P == 2 ? p.ws[p.n + r] : 0.f;
      bias = in && P == 1 && p.bias ? p.bias[r] : 0.f;
      __syncwarp();
      for (int i = lane; i < toks; i += 32) sx[i] = p.xs[m0 + i];
      __syncwarp();
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
      for (int c0 = 0; c0 < toks; c0 += 32) {
        float v[32], u[32];
        tmem_ld32(tmem + b * p.buf_cols + lanes + c0, v);
        if (P == 2) tmem_ld32(tmem + b * p.buf_cols + p.buf_cols / P + lanes + c0, u);
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
          if (c0 + j >= toks) break;
          const float4 s4 = *reinterpret_cast<const float4 *>(sx + c0 + j);
          const float sj[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float &o = v[j + i];
            o = static_cast<float>(__float_as_int(o)) * sj[i] * sw + bias;
            if (P == 2) o = silu_mul(o, static_cast<float>(__float_as_int(u[j + i])) * sj[i] * su);
          }
        }
        if (in)
          by_type(p.y_dtype, [&](auto type) {
            using T = decltype(type);
            T *const y = static_cast<T *>(p.y) + (m0 + c0) * p.ldy + r;
            if (p.add) {
              const T *from = y;
#pragma unroll
              for (int j = 0; j < 32; ++j, from += p.ldy)
                if (c0 + j < toks) v[j] += static_cast<float>(*from);
            }
            T *to = y;
#pragma unroll
            for (int j = 0; j < 32; ++j, to += p.ldy)
              if (c0 + j < toks) *to = from_float<T>(v[j]);
          });
      }
      tc_fence_before();
      mbar_arrive(&tempty[b]);
    }
  }
  if (p.splits > 1) {
    // Join the splits' int32 sums through distributed shared memory: groups of 4 tokens are dealt to the
    // cluster's CTAs in turn. The parts land in their owner's ring, [split][plane][group][row] of int4,
    // once every CTA's MMAs are done with theirs.
    cluster_sync_all();
    const int m0 = first % p.tiles_m * p.bn, toks = min(p.bn, p.m - m0);
    const int owned = (p.bn / 4 + p.splits - 1) / p.splits;  // groups of one CTA
    const int row = (warp & 3) * 32 + lane;
    if (live) {
      const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t part = smem_u32(ring) + (split * P * owned * kRows + row) * 16;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        int owner = 0, at = 0;
        for (int c0 = 0; c0 < toks; c0 += 32) {
          float v[32];
          tmem_ld32(tmem + q * (p.buf_cols / P) + lanes + c0, v);
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            if (c0 + j < toks) {
              st_remote_v4(map_shared(part + (q * owned + at) * kRows * 16, owner),
                           make_int4(__float_as_int(v[j]), __float_as_int(v[j + 1]), __float_as_int(v[j + 2]),
                                     __float_as_int(v[j + 3])));
              if (++owner == p.splits) owner = 0, ++at;
            }
        }
      }
    }
    cluster_sync_all();
    const int r = first / p.tiles_m * kRows + row;
    if (live && r < p.n && !abort_flag) {
      const int4 *parts = reinterpret_cast<const int4 *>(ring) + row;
      by_type(p.y_dtype, [&](auto type) {
        using T = decltype(type);
        for (int at = 0; 4 * (at * p.splits + split) < toks; ++at) {
          const int tok = 4 * (at * p.splits + split);
          int4 sum[P];
#pragma unroll
          for (int q = 0; q < P; ++q) {
            sum[q] = parts[(q * owned + at) * kRows];
#pragma unroll
            for (int z = 1; z < kMaxSplits; ++z)
              if (z < p.splits) {
                const int4 o = parts[((z * P + q) * owned + at) * kRows];
                sum[q].x += o.x, sum[q].y += o.y, sum[q].z += o.z, sum[q].w += o.w;
              }
          }
          const float4 s4 = *reinterpret_cast<const float4 *>(&token_scale[warp - 2][tok]);
          const float sx[4] = {s4.x, s4.y, s4.z, s4.w};
          const int a[4] = {sum[0].x, sum[0].y, sum[0].z, sum[0].w};
          const int c[4] = {sum[P - 1].x, sum[P - 1].y, sum[P - 1].z, sum[P - 1].w};
          T *const y = static_cast<T *>(p.y) + (m0 + tok) * p.ldy + r;
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            v[i] = static_cast<float>(a[i]) * sx[i] * sw + bias;
            if (P == 2) v[i] = silu_mul(v[i], static_cast<float>(c[i]) * sx[i] * su);
            if (p.add && tok + i < toks) v[i] += static_cast<float>(y[i * p.ldy]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tok + i < toks) y[i * p.ldy] = from_float<T>(v[i]);
        }
      });
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

// The token tiles (of bn, at most 256 / P: two buffers of P accumulators in the 512 columns of TMEM) and
// the tiles of the streaming kernel.
struct Shape {
  int tiles_m, bn, tiles;
};
inline Shape shape_of(int planes, int m, int n) {
  Shape s;
  s.tiles_m = (m + 256 / planes - 1) / (256 / planes);
  s.bn = ((m + s.tiles_m - 1) / s.tiles_m + 15) / 16 * 16;
  s.tiles = s.tiles_m * ((n + kRows - 1) / kRows);
  return s;
}

template <int P, int SUB>
int launch_sub(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, Params p, cudaStream_t stream,
           const DeviceInfo &dev, const char *what, int splits) {
  const Shape sh = shape_of(P, p.m, p.n);
  p.tiles_m = sh.tiles_m, p.bn = sh.bn, p.tiles = sh.tiles, p.splits = splits;
  p.buf_cols = P * std::max(32, p.bn);  // the epilogue reads 32 columns at a time
  const int used = splits > 1 ? p.buf_cols : 2 * p.buf_cols;  // (a split's CTA has one tile: no second buffer)
  p.tmem_cols = 32;
  while (p.tmem_cols < used) p.tmem_cols *= 2;
  // As many slots as shared memory holds, and no more than a CTA fills: the next kernel's CTAs can then
  // come in beside these.
  const int slot = SUB * (P * kWBytes + p.bn * kBK), nst = (p.k + SUB * kBK - 1) / (SUB * kBK);
  const int grid = splits > 1 ? p.tiles * splits : std::min(p.tiles, dev.sms);
  const int64_t fills = splits > 1 ? (nst + splits - 1) / splits : static_cast<int64_t>(nst) * ((p.tiles + grid - 1) / grid);
  p.stages = static_cast<int>(std::min<int64_t>({kMaxStages, fills, static_cast<int64_t>(dev.smem_optin - 1024 - 5120) / slot}));
  const size_t parts = splits > 1 ? static_cast<size_t>(splits) * P * ((p.bn / 4 + splits - 1) / splits) * kRows * 16 : 0;
  // At least the share of an SM's shared memory (228 KB) that the tile takes of its TMEM: CTAs that fit beside one
  // another, of any stream, then never wait for TMEM, which those of two clusters could for good.
  const size_t share = std::min<size_t>(static_cast<size_t>(p.tmem_cols) * (228 * 1024 / 512) - 1024 - kStaticShared,
                                        dev.smem_optin - kStaticShared);
  const size_t smem = std::max(std::max(static_cast<size_t>(p.stages) * slot, parts) + 1024, share);
  CUtensorMap wmap, xmap;
  if (int rc = encode_tmap_2d_now(&wmap, wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, static_cast<uint64_t>(P) * p.n, ldw,
                                  kBK, kRows, CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  if (int rc = encode_tmap_2d_now(&xmap, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, p.m, ldx, kBK, p.bn,
                                  CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  auto kern = w8a8_kernel<P, SUB>;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(kern, smem, configured, what)) return rc;
  return launch_overlapped_clusters(kern, dim3(grid), dim3(kThreads), p.splits, smem, stream, what, wmap, xmap, p);
}

template <int P>
int launch(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, const Params &p, cudaStream_t stream,
           const DeviceInfo &dev, const char *what, int splits) {
  constexpr int kFew = sub_blocks(P, 32), kMany = sub_blocks(P, 256);
  if (shape_of(P, p.m, p.n).bn <= 32) return launch_sub<P, kFew>(xq, ldx, wq, ldw, p, stream, dev, what, splits);
  return launch_sub<P, kMany>(xq, ldx, wq, ldw, p, stream, dev, what, splits);
}

int check(const int8_t *xq, int64_t ldx, const float *xs, const int8_t *wq, int64_t ldw, const float *ws, const void *y,
          int y_dtype, int64_t ldy, int64_t m, int64_t n, int planes, int64_t k, const char *what) {
  MQ_REQUIRE(m >= 0 && n > 0 && k > 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(y_dtype == MQ_F32 || y_dtype == MQ_F16 || y_dtype == MQ_BF16, MQ_EINVAL,
             "%s: the output type must be MQ_F32, MQ_F16 or MQ_BF16", what);
  MQ_REQUIRE(ldx >= k && ldw >= k && ldy >= n, MQ_EINVAL, "%s: a row stride is less than the row", what);
  MQ_REQUIRE(k <= kMaxK, MQ_EUNSUPPORTED, "%s: k is above %lld (the int32 sums)", what, static_cast<long long>(kMaxK));
  MQ_REQUIRE(m < (1LL << 30) && n < (1LL << 30) / planes, MQ_EUNSUPPORTED, "%s: m and n must be below 2^30", what);
  if (m == 0) return MQ_OK;
  MQ_REQUIRE(xq && xs && wq && ws && y, MQ_EINVAL, "%s: null pointer", what);
  MQ_REQUIRE(aligned(xq, 16) && aligned(wq, 16) && ldx % 16 == 0 && ldw % 16 == 0, MQ_EALIGN,
             "%s: xq and wq must be 16-byte aligned, their row strides multiples of 16 bytes", what);
  MQ_REQUIRE(aligned(xs, 4) && aligned(ws, 4) && aligned(y, y_dtype == MQ_F32 ? 4 : 2), MQ_EALIGN,
             "%s: xs, ws and y must be aligned to their elements", what);
  return MQ_OK;
}

}  // namespace w8
}  // namespace mq

#include "gemm_w8a8_tile.cu"

namespace mq {
namespace w8 {

// Which kernel, and how many CTAs (pairs of CTAs) share a tile's k: the least of the times below, in us,
// fitted to measurements on a B200 with weights from HBM. Streaming kernel: 0.2 us per 128 k and wave of tiles up
// to about 150 tokens per tile (the issue of the MMAs; 0.8 of it up to 32), 0.33 at 256 (its operands' way into shared memory),
// for gate|up 0.3 and 0.45 at 128, but at least 0.0215 us per token to write a tile; 2.2 us and 0.015 per token and
// plane outside the loop, 3 and 0.028 with the parts of a split to join. Pairs: 0.285 us per 128 k and wave of 256 x
// 256 tiles, at least 3.5 us to write one (fp32 5), 5.5 where y's rows are not 16-byte aligned (fp32 8.5); 5.2 us
// outside, 9.8 with parts to join and 12 more to write those to such rows. Measured, streaming against pairs:
// 128x4096x4096 8.9 / 13.8, 431x2048x8192 14.5 / 17.0, 512x4096x4096 17.3 / 15.3, 1024x4096x4096 18.8 / 16.5,
// 1609x21624x411 43.8 / 32.5, 459x2110x6087 (unaligned rows) 17.8 / 24.7, gate|up 64x8192x2048 12.0 / 13.1,
// 400x8192x2048 20.5 / 17.7.
struct Plan {
  bool pairs;
  int splits;
};
inline Plan plan_of(int planes, const Params &p) {
  Plan best{false, 1};
  float least = 1e30f;
  auto consider = [&](bool pairs, int splits, float us) {
    if (us < least) least = us, best = Plan{pairs, splits};
  };
  const Shape sh = shape_of(planes, p.m, p.n);
  const float few = sh.bn <= 32 ? 0.8f : 1.f;
  const float block = planes == 1 ? std::max(0.2f * few, 0.33f / 256 * sh.bn) : std::max(0.3f * few, 0.45f / 128 * sh.bn);
  const int sub = sub_blocks(planes, sh.bn), blocks = (p.k + kBK - 1) / kBK, stages = (blocks + sub - 1) / sub;
  consider(false, 1, 2.2f + 0.015f * planes * sh.bn + ((sh.tiles + 147) / 148) * std::max(blocks * block, 0.0215f * sh.bn));
  for (int z = 2; z <= std::min(kMaxSplits, stages); ++z)
    if (sh.tiles <= clusters_at_once(z))
      consider(false, z, 3.f + 0.028f * planes * sh.bn + (stages + z - 1) / z * sub * block);
  const int es = p.y_dtype == MQ_F32 ? 4 : 2;
  const bool rows_aligned = !p.add && aligned(p.y, 16) && p.ldy * es % 16 == 0;
  const float write = rows_aligned ? (es == 2 ? 3.5f : 5.f) : (es == 2 ? 5.5f : 8.5f);
  const int tiles = ((p.m + kTileM - 1) / kTileM) * ((p.n + kTileB / planes - 1) / (kTileB / planes));
  consider(true, 1, 5.2f + ((tiles + 73) / 74 - 1) * std::max(blocks * 0.285f, write) + blocks * 0.285f + write - 3.5f);
  for (int z = 2; z <= std::min(kTileMaxSplits, blocks); ++z)
    if (tiles <= clusters_at_once(2 * z))
      consider(true, z, 9.8f + (blocks + z - 1) / z * 0.285f + (rows_aligned ? 0.f : 12.f));
  return best;
}

template <int P>
int run(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, const Params &p, cudaStream_t stream,
        const char *what) {
  DeviceInfo dev;
  if (int rc = device_info(&dev)) return rc;
  const Plan plan = plan_of(P, p);
  if (plan.pairs) return launch_tile<P>(xq, ldx, wq, ldw, p, stream, dev, what, plan.splits);
  return launch<P>(xq, ldx, wq, ldw, p, stream, dev, what, plan.splits);
}

}  // namespace w8
}  // namespace mq

extern "C" int mq_gemm_w8a8(const int8_t *xq, int64_t ldx, const float *xs, const int8_t *wq, int64_t ldw,
                            const float *ws, const float *bias, void *y, int y_dtype, int64_t ldy, int64_t m, int64_t n,
                            int64_t k, int add, void *stream) {
  const char *what = "mq_gemm_w8a8";
  if (int rc = mq::w8::check(xq, ldx, xs, wq, ldw, ws, y, y_dtype, ldy, m, n, 1, k, what)) return rc;
  MQ_REQUIRE(mq::aligned(bias, 4), MQ_EALIGN, "%s: bias must be 4-byte aligned", what);
  if (m == 0) return MQ_OK;
  mq::w8::Params p{};
  p.xs = xs, p.ws = ws, p.bias = bias, p.y = y, p.ldy = ldy, p.y_dtype = y_dtype, p.add = add != 0;
  p.m = static_cast<int>(m), p.n = static_cast<int>(n), p.k = static_cast<int>(k);
  return mq::w8::run<1>(xq, ldx, wq, ldw, p, static_cast<cudaStream_t>(stream), what);
}

extern "C" int mq_gate_up_w8a8(const int8_t *xq, int64_t ldx, const float *xs, const int8_t *wq, int64_t ldw,
                               const float *ws, void *a, int a_dtype, int64_t lda, int64_t m, int64_t f, int64_t k,
                               void *stream) {
  const char *what = "mq_gate_up_w8a8";
  if (int rc = mq::w8::check(xq, ldx, xs, wq, ldw, ws, a, a_dtype, lda, m, f, 2, k, what)) return rc;
  if (m == 0) return MQ_OK;
  mq::w8::Params p{};
  p.xs = xs, p.ws = ws, p.y = a, p.ldy = lda, p.y_dtype = a_dtype;
  p.m = static_cast<int>(m), p.n = static_cast<int>(f), p.k = static_cast<int>(k);
  return mq::w8::run<2>(xq, ldx, wq, ldw, p, static_cast<cudaStream_t>(stream), what);
}
