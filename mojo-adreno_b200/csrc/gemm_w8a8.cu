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
// Every wait on an mbarrier is bounded; on a time-out the kernel records a status code, stops issuing,
// drains its copies, frees its TMEM and returns.
#include <algorithm>

#include "common.cuh"

namespace mq {
namespace w8 {

constexpr int kRows = 128;      // weight rows of a tile (the MMA's M)
constexpr int kBK = 128;        // k per stage: one 128-byte swizzled row
constexpr int kMaxStages = 12;
constexpr int kThreads = 192;   // warp 0 TMA, warp 1 MMA + TMEM, warps 2-5 epilogue
constexpr int kWBytes = kRows * kBK;
constexpr int64_t kMaxK = 131071;  // 128 * 128 * k stays below 2^31

struct Params {
  const float *xs, *ws, *bias;
  void *y;
  int64_t ldy;
  int y_dtype, add;
  int m, n, k;      // n: output columns (f of the gate|up form)
  int bn, tiles_m, tiles;
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

__device__ __forceinline__ void store_out(void *y, int dtype, int64_t at, float v, int add) {
  if (dtype == MQ_F32) {
    float *p = static_cast<float *>(y) + at;
    *p = add ? *p + v : v;
  } else if (dtype == MQ_F16) {
    __half *p = static_cast<__half *>(y) + at;
    *p = __float2half_rn(add ? __half2float(*p) + v : v);
  } else {
    __nv_bfloat16 *p = static_cast<__nv_bfloat16 *>(y) + at;
    *p = __float2bfloat16_rn(add ? __bfloat162float(*p) + v : v);
  }
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.f + expf(-g)) * u; }

template <int P>  // weight planes of a tile: 1, or 2 (gate and up)
__global__ void __launch_bounds__(kThreads, 1)
    w8a8_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Params p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int S = p.stages, slot_bytes = P * kWBytes + p.bn * kBK;
  const int nkb = (p.k + kBK - 1) / kBK;

  griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 128);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  griddep_wait();

  if (warp == 0) {
    if (lane == 0) {
      prefetch_tmap(&wmap);
      prefetch_tmap(&xmap);
    }
    int s = 0, round = 0;
    int64_t issued = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x) {
      const int m0 = t % p.tiles_m * p.bn, n0 = t / p.tiles_m * kRows;
      bool ok = true;
      for (int kb = 0; kb < nkb; ++kb) {
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
        if (lane <= P) {  // lanes 0 .. P - 1: the weight planes; lane P: the tokens
          const bool w = lane < P;
          tma_load_2d(ring + s * slot_bytes + lane * kWBytes, w ? &wmap : &xmap, &full[s], kb * kBK,
                      w ? n0 + lane * p.n : m0);
        }
        ++issued;
        if (++s == S) s = 0, ++round;
      }
      if (!ok) break;
    }
    // Leave no copy in flight: the last load issued into each slot has landed before the CTA ends.
    if (lane == 0)
      for (int64_t i = issued > S ? issued - S : 0; i < issued; ++i) mbar_wait(&full[i % S], (i / S) & 1);
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = umma_idesc_i8(kRows, p.bn);
      int s = 0, it = 0;
      uint32_t ph = 0;
      for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
        const int b = it & 1;
        bool ok = mbar_wait(&tempty[b], ((it >> 1) & 1) ^ 1);
        tc_fence_after();
        for (int kb = 0; ok && kb < nkb; ++kb) {
          if (!mbar_wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t base = smem_u32(ring + s * slot_bytes);
          const uint64_t db = umma_desc_sw128(base + P * kWBytes);
#pragma unroll
          for (int q = 0; q < P; ++q) {
            const uint64_t da = umma_desc_sw128(base + q * kWBytes);
            const uint32_t d = tmem + b * p.buf_cols + q * (p.buf_cols / P);
#pragma unroll
            for (int j = 0; j < kBK / 32; ++j) umma_i8(d, da + 2 * j, db + 2 * j, idesc, kb != 0 || j != 0);
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
    int it = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++it) {
      const int b = it & 1;
      const bool ok = !abort_flag && mbar_wait(&tfull[b], (it >> 1) & 1);
      if (!__all_sync(0xffffffffu, ok && !abort_flag)) {
        if (lane == 0 && !abort_flag) {
          raise_status(kStatusW8EpiWait);
          abort_flag = 1;
        }
        break;
      }
      tc_fence_after();
      const int m0 = t % p.tiles_m * p.bn, r = t / p.tiles_m * kRows + row;
      const bool live = r < p.n;
      const float sw = live ? p.ws[r] : 0.f, su = live && P == 2 ? p.ws[p.n + r] : 0.f;
      const float bias = live && P == 1 && p.bias ? p.bias[r] : 0.f;
      for (int c0 = 0; c0 < p.bn; c0 += 32) {
        float v[32], u[32];
        tmem_ld32(tmem + b * p.buf_cols + lanes + c0, v);
        if (P == 2) tmem_ld32(tmem + b * p.buf_cols + p.buf_cols / P + lanes + c0, u);
        if (live) {
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            const int tok = m0 + c0 + j;
            if (c0 + j >= p.bn || tok >= p.m) break;
            const float sx = p.xs[tok];
            float out = static_cast<float>(__float_as_int(v[j])) * sx * sw + bias;
            if (P == 2) out = silu_mul(out, static_cast<float>(__float_as_int(u[j])) * sx * su);
            store_out(p.y, p.y_dtype, tok * p.ldy + r, out, p.add);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty[b]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

template <int P>
int launch(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, Params p, cudaStream_t stream,
           const DeviceInfo &dev, const char *what) {
  constexpr int kMaxBn = 256 / P;  // two buffers of P accumulators in the 512 columns of TMEM
  p.tiles_m = (p.m + kMaxBn - 1) / kMaxBn;
  p.bn = ((p.m + p.tiles_m - 1) / p.tiles_m + 15) / 16 * 16;
  p.tiles = p.tiles_m * ((p.n + kRows - 1) / kRows);
  p.buf_cols = P * std::max(32, p.bn);  // the epilogue reads 32 columns at a time
  p.tmem_cols = 64;
  while (p.tmem_cols < 2 * p.buf_cols) p.tmem_cols *= 2;
  const int slot = P * kWBytes + p.bn * kBK;
  p.stages = static_cast<int>(std::min<size_t>(kMaxStages, (dev.smem_optin - 4096) / slot));
  const size_t smem = static_cast<size_t>(p.stages) * slot + 1024;
  CUtensorMap wmap, xmap;
  if (int rc = encode_tmap_2d_now(&wmap, wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, static_cast<uint64_t>(P) * p.n, ldw,
                                  kBK, kRows, CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  if (int rc = encode_tmap_2d_now(&xmap, xq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.k, p.m, ldx, kBK, p.bn,
                                  CU_TENSOR_MAP_SWIZZLE_128B, what))
    return rc;
  auto kern = w8a8_kernel<P>;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(kern, smem, configured, what)) return rc;
  return launch_overlapped(kern, dim3(std::min(p.tiles, dev.sms)), dim3(kThreads), smem, stream, what, wmap, xmap, p);
}

int check(const int8_t *xq, int64_t ldx, const float *xs, const int8_t *wq, int64_t ldw, const float *ws, const void *y,
          int y_dtype, int64_t ldy, int64_t m, int64_t n, int64_t wrows, int64_t k, const char *what) {
  MQ_REQUIRE(m >= 0 && n > 0 && k > 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(y_dtype == MQ_F32 || y_dtype == MQ_F16 || y_dtype == MQ_BF16, MQ_EINVAL,
             "%s: the output type must be MQ_F32, MQ_F16 or MQ_BF16", what);
  MQ_REQUIRE(ldx >= k && ldw >= k && ldy >= n, MQ_EINVAL, "%s: a row stride is less than the row", what);
  MQ_REQUIRE(k <= kMaxK, MQ_EUNSUPPORTED, "%s: k is above %lld (the int32 sums)", what, static_cast<long long>(kMaxK));
  MQ_REQUIRE(m < (1LL << 30) && wrows < (1LL << 30), MQ_EUNSUPPORTED, "%s: m and n must be below 2^30", what);
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

template <int P>
int run(const int8_t *xq, int64_t ldx, const int8_t *wq, int64_t ldw, const Params &p, cudaStream_t stream,
        const char *what) {
  DeviceInfo dev;
  if (int rc = device_info(&dev)) return rc;
  if (p.m > 256) return launch_tile<P>(xq, ldx, wq, ldw, p, stream, dev, what);
  return launch<P>(xq, ldx, wq, ldw, p, stream, dev, what);
}

}  // namespace w8
}  // namespace mq

extern "C" int mq_gemm_w8a8(const int8_t *xq, int64_t ldx, const float *xs, const int8_t *wq, int64_t ldw,
                            const float *ws, const float *bias, void *y, int y_dtype, int64_t ldy, int64_t m, int64_t n,
                            int64_t k, int add, void *stream) {
  const char *what = "mq_gemm_w8a8";
  if (int rc = mq::w8::check(xq, ldx, xs, wq, ldw, ws, y, y_dtype, ldy, m, n, n, k, what)) return rc;
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
  if (int rc = mq::w8::check(xq, ldx, xs, wq, ldw, ws, a, a_dtype, lda, m, f, 2 * f, k, what)) return rc;
  if (m == 0) return MQ_OK;
  mq::w8::Params p{};
  p.xs = xs, p.ws = ws, p.y = a, p.ldy = lda, p.y_dtype = a_dtype;
  p.m = static_cast<int>(m), p.n = static_cast<int>(f), p.k = static_cast<int>(k);
  return mq::w8::run<2>(xq, ldx, wq, ldw, p, static_cast<cudaStream_t>(stream), what);
}
