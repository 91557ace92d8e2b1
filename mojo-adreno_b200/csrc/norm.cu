// The norms around a block, fused with its gate, its residual and the quantisation that follows
// (mq_pre_norm, mq_post_norm, mq_quantize_s8).
//
//   post:  r' = residual + scale * gate * n,  n = y / rms(y) * w  (or y itself without w)
//   pre:   h = v * inv,  v = z * next_w,  inv = 1 / sqrt(mean(z^2) + eps),  z = r' (or the row itself)
//   int8:  inv is positive and cancels from the quantised row: with a = max |v|,
//          q = rint(v * (127 / a)), s = a / 127 * inv. So q does not depend on the order in which the
//          row's squares are summed. A row of zeros gives q = 0, s = 0; a row with a NaN or an
//          infinity gives q = 0, s = NaN (the products of that token are then NaN).
// Memory bound: each row is read once into registers, and its sums and maxima run over `tpr` threads
// (warp shuffles, then shared memory), in one fixed order. Sums and r' are fp32; r' is rounded only where
// it is stored, the norm that follows reads the unrounded value.
#include <algorithm>

#include "common.cuh"

namespace mq {
namespace norm {

constexpr int kMaxThreads = 512;

struct Params {
  const void *y, *w, *residual, *gate, *next_w;
  void *out, *h;
  float *hs;
  int64_t ldy, ldr, ldo, ldh, ldg, rows;
  int64_t rows_per_gate;
  int y_dt, w_dt, r_dt, g_dt, nw_dt, h_dt;  // out has residual's type
  int cols, tpr;
  float scale, eps, next_eps;
};

template <int VEC>
__device__ __forceinline__ void load_vec(const void *p, int dt, int64_t at, float *v) {
  if (VEC == 1) {
    v[0] = dt == MQ_F32   ? static_cast<const float *>(p)[at]
           : dt == MQ_F16 ? __half2float(static_cast<const __half *>(p)[at])
                          : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
  } else if (dt == MQ_F32) {
    const float4 *q = reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 f = q[i];
      v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
    }
  } else {
    const uint4 u = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at);
    const uint32_t r[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (dt == MQ_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {  // a bf16 is the upper half of its fp32
        v[2 * i] = __uint_as_float(r[i] << 16), v[2 * i + 1] = __uint_as_float(r[i] & 0xFFFF0000u);
      }
    }
  }
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, int dt) {
  if (dt == MQ_F16) return pack_half2(lo, hi);
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&b);
}

template <int VEC>
__device__ __forceinline__ void store_vec(void *p, int dt, int64_t at, const float *v) {
  if (VEC == 1) {
    if (dt == MQ_F32)
      static_cast<float *>(p)[at] = v[0];
    else if (dt == MQ_F16)
      static_cast<__half *>(p)[at] = __float2half_rn(v[0]);
    else
      static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v[0]);
  } else if (dt == MQ_F32) {
    float4 *q = reinterpret_cast<float4 *>(static_cast<float *>(p) + at);
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) q[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p) + at) =
        make_uint4(pack2(v[0], v[1], dt), pack2(v[2], v[3], dt), pack2(v[4], v[5], dt), pack2(v[6], v[7], dt));
  }
}

template <int VEC>
__device__ __forceinline__ void store_s8(int8_t *p, const int *q) {
  if (VEC == 1) {
    *p = static_cast<int8_t>(q[0]);
  } else {
    uint32_t r[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r[i] = (q[4 * i] & 255) | (q[4 * i + 1] & 255) << 8 | (q[4 * i + 2] & 255) << 16 |
             static_cast<uint32_t>(q[4 * i + 3]) << 24;
    *reinterpret_cast<uint2 *>(p) = make_uint2(r[0], r[1]);
  }
}

// Sum and largest bit pattern of |v| over the threads of a row (every thread gets both). The
// patterns of non-negative floats are ordered as the values, with infinity and NaN above all.
__device__ __forceinline__ void row_reduce(float &sum, uint32_t &top, int tpr, float *ssum, uint32_t *stop) {
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  top = __reduce_max_sync(0xffffffffu, top);
  if (tpr == 32) return;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = tpr / 32;
  if (lane == 0) ssum[warp] = sum, stop[warp] = top;
  __syncthreads();
  sum = lane < warps ? ssum[lane] : 0.f;
  top = lane < warps ? stop[lane] : 0u;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  top = __reduce_max_sync(0xffffffffu, top);
}

// E vectors of VEC values per thread; a row has p.tpr threads (threadIdx.x), a CTA blockDim.y rows.
// EARLY: the dependents may start before this grid ends (not when it may be writing weights).
template <int VEC, int E, bool POST, bool EARLY>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const Params p) {
  __shared__ float ssum[2][16];
  __shared__ uint32_t stop[2][16];
  if (EARLY) griddep_launch_dependents();
  griddep_wait();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // rows of one warp each where blockDim.y > 1: no barrier is skipped
  float z[E * VEC];
  float sum = 0.f;
  uint32_t top = 0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e * p.tpr + threadIdx.x) * VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) z[e * VEC + i] = 0.f;
    if (c < p.cols) load_vec<VEC>(p.y, p.y_dt, row * p.ldy + c, z + e * VEC);
  }
  if (POST) {
    float inv = 1.f;
    if (p.w) {
#pragma unroll
      for (int e = 0; e < E * VEC; ++e) sum += z[e] * z[e];
      row_reduce(sum, top, p.tpr, ssum[0], stop[0]);
      inv = rsqrtf(sum / p.cols + p.eps);
    }
    inv *= p.scale;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (e * p.tpr + threadIdx.x) * VEC;
      if (c >= p.cols) continue;
      float r[VEC], g[VEC];
      load_vec<VEC>(p.residual, p.r_dt, row * p.ldr + c, r);
      if (p.w) {
        load_vec<VEC>(p.w, p.w_dt, c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= g[i];
      }
      if (p.gate) {
        load_vec<VEC>(p.gate, p.g_dt, row / p.rows_per_gate * p.ldg + c, g);
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[e * VEC + i] = fmaf(z[e * VEC + i], inv, r[i]);
      store_vec<VEC>(p.out, p.r_dt, row * p.ldo + c, z + e * VEC);
    }
    if (!p.h) return;
  }
  sum = 0.f, top = 0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e * p.tpr + threadIdx.x) * VEC;
    if (c >= p.cols) continue;
    float w[VEC];
    if (p.next_w) load_vec<VEC>(p.next_w, p.nw_dt, c, w);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      float &v = z[e * VEC + i];
      sum += v * v;
      if (p.next_w) v *= w[i];
      top = max(top, __float_as_uint(v) & 0x7FFFFFFFu);
    }
  }
  row_reduce(sum, top, p.tpr, ssum[1], stop[1]);
  const float inv = p.next_w ? rsqrtf(sum / p.cols + p.next_eps) : 1.f;
  if (p.h_dt != MQ_S8) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (e * p.tpr + threadIdx.x) * VEC;
      if (c >= p.cols) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= inv;
      store_vec<VEC>(p.h, p.h_dt, row * p.ldh + c, z + e * VEC);
    }
    return;
  }
  // A maximum below 1e-30 is lifted by 2^80 (exact) first, so 127 / a stays finite.
  const float a = __uint_as_float(top), lift = a < 1e-30f ? 0x1p80f : 1.f;
  const bool bad = top >= 0x7F800000u || !(inv < INFINITY);
  const float f = bad || top == 0u ? 0.f : 127.f / (a * lift);
  if (threadIdx.x == 0) p.hs[row] = bad ? NAN : a / 127.f * inv;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e * p.tpr + threadIdx.x) * VEC;
    if (c >= p.cols) continue;
    int q[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) q[i] = bad ? 0 : __float2int_rn(z[e * VEC + i] * lift * f);
    store_s8<VEC>(static_cast<int8_t *>(p.h) + row * p.ldh + c, q);
  }
}

template <int VEC, int E, bool POST, bool EARLY>
int launch_e(const Params &p, int threads, int rows_per_cta, cudaStream_t s, const char *what) {
  const int64_t grid = (p.rows + rows_per_cta - 1) / rows_per_cta;
  MQ_REQUIRE(grid < (1LL << 31), MQ_EUNSUPPORTED, "%s: too many rows", what);
  return launch_overlapped(block_norm_kernel<VEC, E, POST, EARLY>, dim3(static_cast<unsigned>(grid)),
                           dim3(threads, rows_per_cta), 0, s, what, p);
}

constexpr int kMaxCols = 64 * kMaxThreads;

template <bool POST, bool EARLY>
int launch(Params p, bool vec, cudaStream_t s, const char *what) {
  MQ_REQUIRE(p.cols <= kMaxCols, MQ_EUNSUPPORTED, "%s: cols is above %d", what, kMaxCols);
  if (vec) {
    // 8 values per thread (one warp up to 256 columns), 16 to 64 only where a row is too long for that
    p.tpr = std::min(kMaxThreads, (p.cols + 255) / 256 * 32);
    if (p.cols <= 8 * p.tpr) return launch_e<8, 1, POST, EARLY>(p, p.tpr, p.tpr == 32 ? 4 : 1, s, what);
    if (p.cols <= 16 * p.tpr) return launch_e<8, 2, POST, EARLY>(p, p.tpr, 1, s, what);
    if (p.cols <= 32 * p.tpr) return launch_e<8, 4, POST, EARLY>(p, p.tpr, 1, s, what);
    return launch_e<8, 8, POST, EARLY>(p, p.tpr, 1, s, what);
  }
  p.tpr = std::min(kMaxThreads, (p.cols + 127) / 128 * 32);
  if (p.cols <= 4 * p.tpr) return launch_e<1, 4, POST, EARLY>(p, p.tpr, p.tpr == 32 ? 4 : 1, s, what);
  if (p.cols <= 16 * p.tpr) return launch_e<1, 16, POST, EARLY>(p, p.tpr, 1, s, what);
  return launch_e<1, 64, POST, EARLY>(p, p.tpr, 1, s, what);
}

inline int size_of(int dt) { return dt == MQ_F32 ? 4 : dt == MQ_S8 ? 1 : 2; }
inline bool is_float(int dt) { return dt == MQ_F32 || dt == MQ_F16 || dt == MQ_BF16; }

// Whether 8-value vectors of this tensor are aligned in every row (null: not used, no limit).
inline bool vec_ok(const void *p, int dt, int64_t ld, int64_t rows) {
  const int bytes = dt == MQ_S8 ? 8 : 16;
  return !p || (aligned(p, bytes) && (rows <= 1 || ld * size_of(dt) % bytes == 0));
}

}  // namespace norm
}  // namespace mq

namespace {
// The checks every entry point shares; `what` names it in messages.
int norm_check_h(const void *h, int h_dt, int64_t ldh, const float *hs, int64_t rows, int64_t cols, const char *what) {
  MQ_REQUIRE(mq::norm::is_float(h_dt) || h_dt == MQ_S8, MQ_EINVAL,
             "%s: the output type must be MQ_F32, MQ_F16, MQ_BF16 or MQ_S8", what);
  MQ_REQUIRE(ldh >= cols, MQ_EINVAL, "%s: the output's row stride is less than cols", what);
  MQ_REQUIRE(rows == 0 || h_dt != MQ_S8 || hs, MQ_EINVAL, "%s: null scales for an int8 output", what);
  MQ_REQUIRE(mq::aligned(h, mq::norm::size_of(h_dt)) && mq::aligned(hs, 4), MQ_EALIGN,
             "%s: the output must be aligned to its elements", what);
  return MQ_OK;
}

int norm_check_in(const void *x, int dt, int64_t ld, int64_t cols, const char *name, const char *what) {
  MQ_REQUIRE(mq::norm::is_float(dt), MQ_EINVAL, "%s: %s must be MQ_F32, MQ_F16 or MQ_BF16", what, name);
  MQ_REQUIRE(ld >= cols, MQ_EINVAL, "%s: %s's row stride is less than cols", what, name);
  MQ_REQUIRE(mq::aligned(x, mq::norm::size_of(dt)), MQ_EALIGN, "%s: %s must be aligned to its elements", what, name);
  return MQ_OK;
}
}  // namespace

extern "C" int mq_quantize_s8(const void *x, int x_dtype, int64_t ldx, int8_t *q, int64_t ldq, float *s, int64_t rows,
                              int64_t cols, void *stream) {
  const char *what = "mq_quantize_s8";
  MQ_REQUIRE(rows >= 0 && cols > 0 && cols < (1LL << 31), MQ_EINVAL, "%s: bad shape", what);
  if (int rc = norm_check_in(x, x_dtype, ldx, cols, "x", what)) return rc;
  if (int rc = norm_check_h(q, MQ_S8, ldq, s, rows, cols, what)) return rc;
  if (rows == 0) return MQ_OK;
  MQ_REQUIRE(x && q, MQ_EINVAL, "%s: null pointer", what);
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  mq::norm::Params p{};
  p.y = x, p.y_dt = x_dtype, p.ldy = ldx, p.h = q, p.h_dt = MQ_S8, p.ldh = ldq, p.hs = s;
  p.rows = rows, p.cols = static_cast<int>(cols);
  const bool vec = cols % 8 == 0 && mq::norm::vec_ok(x, x_dtype, ldx, rows) && mq::norm::vec_ok(q, MQ_S8, ldq, rows);
  // No early start of the dependents: q may be a weight matrix, which a product may read ahead.
  return mq::norm::launch<false, false>(p, vec, static_cast<cudaStream_t>(stream), what);
}

extern "C" int mq_pre_norm(const void *x, int x_dtype, int64_t ldx, const void *w, int w_dtype, float eps, void *h,
                           int h_dtype, int64_t ldh, float *hs, int64_t rows, int64_t cols, void *stream) {
  const char *what = "mq_pre_norm";
  MQ_REQUIRE(rows >= 0 && cols > 0 && cols < (1LL << 31), MQ_EINVAL, "%s: bad shape", what);
  if (int rc = norm_check_in(x, x_dtype, ldx, cols, "x", what)) return rc;
  if (int rc = norm_check_in(w, w_dtype, cols, cols, "w", what)) return rc;
  if (int rc = norm_check_h(h, h_dtype, ldh, hs, rows, cols, what)) return rc;
  if (rows == 0) return MQ_OK;
  MQ_REQUIRE(x && w && h, MQ_EINVAL, "%s: null pointer", what);
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  mq::norm::Params p{};
  p.y = x, p.y_dt = x_dtype, p.ldy = ldx, p.next_w = w, p.nw_dt = w_dtype, p.next_eps = eps;
  p.h = h, p.h_dt = h_dtype, p.ldh = ldh, p.hs = hs;
  p.rows = rows, p.cols = static_cast<int>(cols);
  using mq::norm::vec_ok;
  const bool vec = cols % 8 == 0 && vec_ok(x, x_dtype, ldx, rows) && vec_ok(w, w_dtype, cols, 1) &&
                   vec_ok(h, h_dtype, ldh, rows);
  return mq::norm::launch<false, true>(p, vec, static_cast<cudaStream_t>(stream), what);
}

extern "C" int mq_post_norm(const void *y, int y_dtype, int64_t ldy, const void *w, int w_dtype, float eps,
                            const void *residual, int r_dtype, int64_t ldr, const void *gate, int gate_dtype,
                            int64_t ldg, int64_t rows_per_gate, float scale, void *out, int64_t ldo, const void *next_w,
                            int next_w_dtype, float next_eps, void *h, int h_dtype, int64_t ldh, float *hs, int64_t rows,
                            int64_t cols, void *stream) {
  const char *what = "mq_post_norm";
  MQ_REQUIRE(rows >= 0 && cols > 0 && cols < (1LL << 31), MQ_EINVAL, "%s: bad shape", what);
  if (int rc = norm_check_in(y, y_dtype, ldy, cols, "y", what)) return rc;
  if (int rc = norm_check_in(residual, r_dtype, ldr, cols, "residual", what)) return rc;
  if (int rc = norm_check_in(out, r_dtype, ldo, cols, "out", what)) return rc;
  if (w)
    if (int rc = norm_check_in(w, w_dtype, cols, cols, "w", what)) return rc;
  if (gate) {
    if (int rc = norm_check_in(gate, gate_dtype, ldg, cols, "gate", what)) return rc;
    MQ_REQUIRE(rows_per_gate > 0, MQ_EINVAL, "%s: rows_per_gate must be positive", what);
  }
  if (h) {
    MQ_REQUIRE(next_w, MQ_EINVAL, "%s: h without next_w", what);
    if (int rc = norm_check_in(next_w, next_w_dtype, cols, cols, "next_w", what)) return rc;
    if (int rc = norm_check_h(h, h_dtype, ldh, hs, rows, cols, what)) return rc;
  }
  if (rows == 0) return MQ_OK;
  MQ_REQUIRE(y && residual && out, MQ_EINVAL, "%s: null pointer", what);
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  mq::norm::Params p{};
  p.y = y, p.y_dt = y_dtype, p.ldy = ldy, p.w = w, p.w_dt = w_dtype, p.eps = eps;
  p.residual = residual, p.r_dt = r_dtype, p.ldr = ldr, p.out = out, p.ldo = ldo, p.scale = scale;
  p.gate = gate, p.g_dt = gate_dtype, p.ldg = ldg, p.rows_per_gate = rows_per_gate;
  p.next_w = next_w, p.nw_dt = next_w_dtype, p.next_eps = next_eps;
  p.h = h, p.h_dt = h_dtype, p.ldh = ldh, p.hs = hs;
  p.rows = rows, p.cols = static_cast<int>(cols);
  using mq::norm::vec_ok;
  const bool vec = cols % 8 == 0 && vec_ok(y, y_dtype, ldy, rows) && vec_ok(residual, r_dtype, ldr, rows) &&
                   vec_ok(out, r_dtype, ldo, rows) && vec_ok(w, w_dtype, cols, 1) &&
                   vec_ok(gate, gate_dtype, ldg, rows) && vec_ok(h ? next_w : nullptr, next_w_dtype, cols, 1) &&
                   vec_ok(h, h_dtype, ldh, rows);
  return mq::norm::launch<true, true>(p, vec, static_cast<cudaStream_t>(stream), what);
}
