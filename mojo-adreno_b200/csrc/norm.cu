// The norms around a block, fused with its gate, its residual and the quantisation that follows
// (mq_pre_norm, mq_post_norm, mq_quantize_s8).
//
//   post:  r' = residual + scale * gate * n,  n = y / rms(y) * w  (or y itself without w)
//   pre:   h = v * inv,  v = z * next_w,  inv = 1 / sqrt(mean(z^2) + eps),  z = r' (or the row itself)
//   int8:  inv is positive and cancels from the quantised row: with a = max |v|,
//          q = rint(v * (127 / a)), s = a / 127 * inv. So q does not depend on the order in which the
//          row's squares are summed. A row of zeros gives q = 0, s = 0; a row with a NaN or an
//          infinity gives q = 0, s = NaN (the products of that token are then NaN).
// Memory bound for many rows, launch latency for a few: each row is read once into registers, and its sums and
// maxima run over `tpr` threads (warp shuffles, then shared memory), in one fixed order. Sums and r' are fp32;
// r' is rounded only where it is stored, the norm that follows reads the unrounded value.
// Three kernels: block_norm_kernel (a row per CTA or warp: few rows, rows below 768 or above 8192 columns),
// row_stream_kernel (many aligned rows) and row_stream1_kernel (many rows without alignment).
// B200: pre_norm 8192x4096 bf16 26.5 us (5.1 TB/s), to int8 28.3; post_norm 12337x4096 bf16 with its gate
// and the next norm 70.8-73 us (5.6 TB/s, 0.87 of the copy bandwidth); one row of 4096: 2.1 and 3.0-3.7 us. Rows below 768
// columns do not stream, and a warp per short row does not fill the memory pipe: 262144x128 bf16 68 us, three floors.
#include <algorithm>
#include <type_traits>

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
  float scale, eps, next_eps, inv_cols;
};

template <typename T, int VEC>
struct alignas(VEC == 1 ? sizeof(T) : 16) Raw {
  T v[VEC];
};
// Values of a vector as fp32 and back: two at a time for the 16-bit types (a bf16 is the upper half of its fp32).
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Raw<T, VEC> &raw, float *v) {
  if constexpr (VEC == 1 || std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = static_cast<float>(raw.v[i]);
  } else {
    const uint4 q = *reinterpret_cast<const uint4 *>(&raw);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
  if constexpr (std::is_same<T, float>::value && VEC == 8) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (VEC == 8) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        w[i] = pack_half2(v[2 * i], v[2 * i + 1]);
      } else {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
      }
    }
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    if constexpr (std::is_same<T, float>::value) *p = v[0];
    if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(v[0]);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) *p = __float2bfloat16_rn(v[0]);
  }
}

// This thread's E vectors of a row: f(e, values) for each, zeros outside the row. All loads are on their way before
// the first is used.
template <typename T, int VEC, int E, typename F>
__device__ __forceinline__ void each_vec_of(const T *row, int cols, int tpr, F f) {
  Raw<T, VEC> raw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e * tpr + threadIdx.x) * VEC;
    raw[e] = Raw<T, VEC>{};
    if (c < cols) raw[e] = *reinterpret_cast<const Raw<T, VEC> *>(row + c);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    float v[VEC];
    unpack<T, VEC>(raw[e], v);
    f(e, v);
  }
}
// The same for a row that starts at element `at` of an array of a type known at run time.
template <int VEC, int E, typename F>
__device__ __forceinline__ void each_vec(const void *base, int dt, int64_t at, int cols, int tpr, F f) {
  by_type(dt, [&](auto type) {
    using T = decltype(type);
    each_vec_of<T, VEC, E>(static_cast<const T *>(base) + at, cols, tpr, f);
  });
}

// rint(v * f) as int8, |v * f| <= 127: the sum with 1.5 * 2^23 has the integer in its low bits, rounded to nearest,
// ties to even. (Conversion instructions run at an eighth of the rate.)
template <int VEC>
__device__ __forceinline__ void store_s8(int8_t *p, const float *v, float f) {
  uint32_t b[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) b[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], f), 12582912.f));
  if constexpr (VEC == 1)
    *p = static_cast<int8_t>(b[0]);
  else
    *reinterpret_cast<uint2 *>(p) =
        make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                   __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// The bits of the largest |v|, a NaN where there is one. The patterns of non-negative floats are ordered as the
// values, with infinity and NaN above all.
template <int N>
__device__ __forceinline__ uint32_t top_of(const float *z) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(z[i])));
  return __float_as_uint(top);
}

struct Scratch {  // of one reduction: a value per warp, the sums 0 where there is no warp (clear_scratch)
  float sum[16];
  uint32_t top[16];
};

// Before the first reduction, behind which there is a barrier.
__device__ __forceinline__ void clear_scratch(Scratch *s, int n, int warps) {
  for (int i = threadIdx.x; i < 16 * n; i += blockDim.x)
    if (i % 16 >= warps) s[i / 16].sum[i % 16] = 0.f;
}

// Sum of the squares and (with_top) largest |v| of a row over its `tpr` threads; every thread gets both, in one
// fixed order. With more than one warp the threads pass one barrier.
template <int N>
__device__ __forceinline__ void row_reduce(const float *z, float &sum, uint32_t &top, bool with_top, int tpr, Scratch &s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (with_top) top = __reduce_max_sync(0xffffffffu, top_of<N>(z));
  if (tpr == 32) return;
  const int warp = threadIdx.x / 32, warps = tpr / 32;
  if (threadIdx.x % 32 == 0) {
    s.sum[warp] = sum;
    if (with_top) s.top[warp] = top;
  }
  __syncthreads();
  sum = 0.f;
  for (int w = 0; w < warps; w += 4) {
    const float4 f = *reinterpret_cast<const float4 *>(&s.sum[w]);
    sum += (f.x + f.y) + (f.z + f.w);
  }
  if (with_top)
    for (int w = 0; w < warps; ++w) top = max(top, s.top[w]);
}

template <int N>
__device__ __forceinline__ float squares(const float *z) {
  float part[4] = {};
#pragma unroll
  for (int i = 0; i < N; ++i) part[i % 4] = fmaf(z[i], z[i], part[i % 4]);
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// h from v = z * next_w (z itself without next_w) and the row's sum of squares and largest |v|.
// TPR: p.tpr where it is known when compiling, else 0.
template <int VEC, int E, int TPR = 0>
__device__ __forceinline__ void write_h(const Params &p, int64_t row, float *z, float sum, uint32_t top) {
  const int tpr = TPR ? TPR : p.tpr;
  const float inv = p.next_w ? rsqrtf(fmaf(sum, p.inv_cols, p.next_eps)) : 1.f;
  if (p.h_dt != MQ_S8) {
    by_type(p.h_dt, [&](auto type) {
      using T = decltype(type);
      T *h = static_cast<T *>(p.h) + row * p.ldh;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (e * tpr + threadIdx.x) * VEC;
        if (c >= p.cols) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= inv;
        store_vec<T, VEC>(h + c, z + e * VEC);
      }
    });
    return;
  }
  const float a = __uint_as_float(top);
  const bool bad = !(a < INFINITY) || !(inv < INFINITY);
  if (threadIdx.x == 0) p.hs[row] = bad ? NAN : a / 127.f * inv;
  float f = a > 0.f ? 127.f / a : 0.f;
  if (bad || a < 1e-30f) {  // (the whole row)
    // A maximum below 1e-30 is lifted by 2^80 (exact) first, so 127 / a stays finite.
    f = bad || a == 0.f ? 0.f : 127.f / (a * 0x1p80f);
#pragma unroll
    for (int i = 0; i < E * VEC; ++i) z[i] = bad ? 0.f : z[i] * 0x1p80f;
  }
  int8_t *h = static_cast<int8_t *>(p.h) + row * p.ldh;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = (e * tpr + threadIdx.x) * VEC;
    if (c < p.cols) store_s8<VEC>(h + c, z + e * VEC, f);
  }
}

// E vectors of VEC values per thread; a row has p.tpr threads (threadIdx.x), a CTA blockDim.y rows.
// EARLY: the dependents may start before this grid ends (not when it may be writing weights).
template <int VEC, int E, bool POST, bool EARLY>
__global__ void __launch_bounds__(kMaxThreads) block_norm_kernel(const Params p) {
  __shared__ __align__(16) Scratch scratch[2];
  if (EARLY) griddep_launch_dependents();
  griddep_wait();
  if (p.tpr > 32) clear_scratch(scratch, 2, p.tpr / 32);  // (read behind the reductions' barriers)
  const int64_t row = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
  if (row >= p.rows) return;  // rows of one warp each where blockDim.y > 1: no barrier is skipped
  const int cols = p.cols, tpr = p.tpr;
  float z[E * VEC];
  uint32_t top = 0u;
  each_vec<VEC, E>(p.y, p.y_dt, row * p.ldy, cols, tpr, [&](int e, const float *v) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) z[e * VEC + i] = v[i];
  });
  if (POST) {
    float r[E * VEC];  // fetched before the reduction, which hides its latency
    each_vec<VEC, E>(p.residual, p.r_dt, row * p.ldr, cols, tpr, [&](int e, const float *v) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) r[e * VEC + i] = v[i];
    });
    float inv = p.scale;
    if (p.w) {
      float sum = squares<E * VEC>(z);
      row_reduce<E * VEC>(z, sum, top, false, tpr, scratch[0]);
      inv *= rsqrtf(fmaf(sum, p.inv_cols, p.eps));
      each_vec<VEC, E>(p.w, p.w_dt, 0, cols, tpr, [&](int e, const float *v) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
      });
    }
    if (p.gate)
      each_vec<VEC, E>(p.gate, p.g_dt, row / p.rows_per_gate * p.ldg, cols, tpr, [&](int e, const float *v) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
      });
    by_type(p.r_dt, [&](auto type) {
      using T = decltype(type);
      T *out = static_cast<T *>(p.out) + row * p.ldo;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (e * tpr + threadIdx.x) * VEC;
        if (c >= cols) continue;
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] = fmaf(z[e * VEC + i], inv, r[e * VEC + i]);
        store_vec<T, VEC>(out + c, z + e * VEC);
      }
    });
    if (!p.h) return;
  }
  float sum = squares<E * VEC>(z);
  if (p.next_w)
    each_vec<VEC, E>(p.next_w, p.nw_dt, 0, cols, tpr, [&](int e, const float *v) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
    });
  row_reduce<E * VEC>(z, sum, top, p.h_dt == MQ_S8, tpr, scratch[1]);
  write_h<VEC, E>(p, row, z, sum, top);
}

// The same for many rows: persistent CTAs of one row at a time, whose next rows (y, residual) are on their
// way into a ring in shared memory while one is worked on, and which fetch the weights once. Against one CTA per
// row, which loads, reduces and stores in turn, with its weights from L2 each time: pre_norm 8192x4096 33.7 -> 26.5
// us, post_norm 12337x4096 114.6 -> 70.8. A thread has 16 values: with 32 there are too few warps for the
// latency of the reductions (28.9 and 91 us). The gate comes by plain loads: in the ring it took the room of
// a third CTA per SM (82 us).
constexpr int kRingMax = 8, kStreamThreads = 512;
struct Ring {
  int stages;                // rows on their way, each of y and, after a block, of the residual
  int row_bytes[2], at[2];   // of the two, and where they are in a stage
  int stage_bytes, w_at, next_w_at, total;  // bytes; the weights lie behind the ring
};

// Where the first wait ran out for the thread that fetches. It then fetches no more, and at the end (code inside the
// row loop cost post_norm 12337x4096 77 -> 79.7 us) the rows that were on their way are waited for: they land before the CTA
// ends.
struct Lost {
  int64_t row;
  int slot;
  uint32_t phase;
};
__device__ __forceinline__ void drain_ring(uint64_t *full, const Ring &g, int64_t rows, const Lost &lost) {
  int slot = lost.slot;
  uint32_t phase = lost.phase;
  int64_t row = lost.row;
  for (int i = 0; i < g.stages && row < rows; ++i, row += gridDim.x) {
    mbar_wait(&full[slot], phase);
    if (++slot == g.stages) slot = 0, phase ^= 1;
  }
}

// TY, TR, TW: the types of y, of the residual, and of w, next_w and the gate (a branch on a type inside would
// have the loads of all three from shared memory speculated, and spilled).
template <typename TY, typename TR, typename TW, int E, bool POST, bool EARLY>
__global__ void __launch_bounds__(kStreamThreads) row_stream_kernel(const Params p, const Ring g) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kRingMax + 1];  // the last one: the weights
  __shared__ __align__(16) Scratch scratch[2][2];
  __shared__ Lost lost;  // by thread 0
  constexpr int VEC = 8;
  if (EARLY) griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1);
    mbar_init(&full[kRingMax], 1);
    fence_mbar_init();
  }
  clear_scratch(&scratch[0][0], 4, p.tpr / 32);
  __syncthreads();
  griddep_wait();
  const int cols = p.cols, tpr = p.tpr;
  const int step = gridDim.x;
  auto fetch = [&](int64_t row, int slot) {  // by thread 0
    uint8_t *at = smem + slot * g.stage_bytes;
    mbar_expect_tx(&full[slot], g.stage_bytes);
    bulk_load(at, static_cast<const uint8_t *>(p.y) + row * p.ldy * sizeof(TY), g.row_bytes[0], &full[slot]);
    if (POST) {
      bulk_load(at + g.at[1], static_cast<const uint8_t *>(p.residual) + row * p.ldr * sizeof(TR), g.row_bytes[1], &full[slot]);
    }
  };
  bool arrived = true;
  if (threadIdx.x == 0) {
    const int w_bytes = POST && p.w ? cols * static_cast<int>(sizeof(TW)) : 0;
    const int nw_bytes = p.next_w ? cols * static_cast<int>(sizeof(TW)) : 0;
    mbar_expect_tx(&full[kRingMax], w_bytes + nw_bytes);
    if (w_bytes) bulk_load(smem + g.w_at, p.w, w_bytes, &full[kRingMax]);
    if (nw_bytes) bulk_load(smem + g.next_w_at, p.next_w, nw_bytes, &full[kRingMax]);
    int64_t row = blockIdx.x;
    for (int i = 0; i < g.stages && row < p.rows; ++i, row += step) fetch(row, i);
  }
  if (!mbar_wait(&full[kRingMax], 0)) {
    raise_status(kStatusNormLoadWait);
    arrived = false;
    if (threadIdx.x == 0) lost = Lost{blockIdx.x, 0, 0};
  }
  int slot = 0, parity = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += step, parity ^= 1) {
    if (arrived && !mbar_wait(&full[slot], phase)) {
      raise_status(kStatusNormLoadWait);  // what there is goes on; the status says that it may be wrong
      arrived = false;
      if (threadIdx.x == 0) lost = Lost{row, slot, phase};
    }
    const uint8_t *at = smem + slot * g.stage_bytes;
    Raw<TW, VEC> gate[E];  // (a row of it serves many rows, or comes from memory while this one is reduced)
    if (POST && p.gate) {
      const TW *from = static_cast<const TW *>(p.gate) + row / p.rows_per_gate * p.ldg;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = (e * tpr + threadIdx.x) * VEC;
        gate[e] = Raw<TW, VEC>{};
        if (c < cols) gate[e] = *reinterpret_cast<const Raw<TW, VEC> *>(from + c);
      }
    }
    float z[E * VEC], sum = 0.f;
    uint32_t top = 0u;
    each_vec_of<TY, VEC, E>(reinterpret_cast<const TY *>(at), cols, tpr, [&](int e, const float *v) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[e * VEC + i] = v[i];
    });
    if (POST) {
      float inv = p.scale;
      if (p.w) {
        sum = squares<E * VEC>(z);
        row_reduce<E * VEC>(z, sum, top, false, tpr, scratch[parity][0]);
        inv *= rsqrtf(fmaf(sum, p.inv_cols, p.eps));
        each_vec_of<TW, VEC, E>(reinterpret_cast<const TW *>(smem + g.w_at), cols, tpr, [&](int e, const float *v) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
        });
      }
      if (p.gate)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float v[VEC];
          unpack<TW, VEC>(gate[e], v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
        }
      TR *out = static_cast<TR *>(p.out) + row * p.ldo;
      each_vec_of<TR, VEC, E>(reinterpret_cast<const TR *>(at + g.at[1]), cols, tpr, [&](int e, const float *v) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) z[e * VEC + i] = fmaf(z[e * VEC + i], inv, v[i]);
        const int c = (e * tpr + threadIdx.x) * VEC;
        if (c < cols) store_vec<TR, VEC>(out + c, z + e * VEC);
      });
    }
    if (!POST || p.h) {
      sum = squares<E * VEC>(z);
      if (EARLY || p.next_w)
        each_vec_of<TW, VEC, E>(reinterpret_cast<const TW *>(smem + g.next_w_at), cols, tpr, [&](int e, const float *v) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) z[e * VEC + i] *= v[i];
        });
      row_reduce<E * VEC>(z, sum, top, p.h_dt == MQ_S8, tpr, scratch[parity][1]);
    }
    if (tpr == 32 || (POST && !p.h)) __syncthreads();  // else row_reduce's barrier: every thread has read the slot
    if (threadIdx.x == 0 && arrived && row + static_cast<int64_t>(g.stages) * step < p.rows)
      fetch(row + static_cast<int64_t>(g.stages) * step, slot);
    if (++slot == g.stages) slot = 0, phase ^= 1;
    if (!POST || p.h) write_h<VEC, E>(p, row, z, sum, top);
  }
  if (threadIdx.x == 0 && !arrived) {
    mbar_wait(&full[kRingMax], 0);  // the weights
    drain_ring(full, g, p.rows, lost);
  }
}

// Rows that are not 16-byte aligned, or not a multiple of 8 long: the 16-byte granules that lie inside a row come
// through the ring, the few elements before and after them by plain loads one row ahead, each by the thread that
// works on it, which puts them into their places. A thread has every tpr-th element, 16 at most; its weights
// stay in registers.
template <typename T>
struct Edge {
  T head, tail;
};
template <typename T>
struct Span {
  static constexpr int kPer = 16 / static_cast<int>(sizeof(T));  // elements of a granule
  int head, end;  // elements before the first granule, first element after the last one
  __device__ __forceinline__ Span(const T *row, int cols) {
    head = static_cast<int>((0 - reinterpret_cast<uintptr_t>(row)) % 16 / sizeof(T));
    end = cols - ((cols - head) & (kPer - 1));
  }
  // This thread's elements outside the granules: element threadIdx.x of the first few, element `last` (its one column
  // among the row's last tpr) of the last few.
  __device__ __forceinline__ Edge<T> edge(const T *row, int last) const {
    Edge<T> e{};
    if (static_cast<int>(threadIdx.x) < head) e.head = row[threadIdx.x];
    if (last >= end) e.tail = row[last];
    return e;
  }
  // Element 0's place in a slot (the granules start at byte 16) with this thread's edge elements put in.
  __device__ __forceinline__ const T *put(uint8_t *at, Edge<T> e, int last) const {
    T *row = reinterpret_cast<T *>(at + 16) - head;
    const bool first = static_cast<int>(threadIdx.x) < head, final = last >= end;
    if (first) row[threadIdx.x] = e.head;
    if (final) row[last] = e.tail;
    if (first || final) fence_proxy_async_smem();  // before a later row's granules come to the same place
    return row;
  }
};

// TPR: the threads of a row, known so that its elements lie at fixed distances: with a distance known at run time
// the addresses took most of the instructions (pre_norm 20000x1001 42 us instead of 23; a row per CTA: 48).
template <typename TY, typename TR, int TPR, bool POST, bool EARLY>
__global__ void __launch_bounds__(TPR) row_stream1_kernel(const Params p, const Ring g) {
  constexpr int E = 16;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t full[kRingMax];
  __shared__ __align__(16) Scratch scratch[2][2];
  __shared__ Lost lost;  // by thread 0
  if (EARLY) griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
  }
  clear_scratch(&scratch[0][0], 4, TPR / 32);
  __syncthreads();
  griddep_wait();
  constexpr int tpr = TPR;
  const int cols = p.cols, step = gridDim.x;
  const int last = cols - 1 - ((cols - 1) % tpr + tpr - static_cast<int>(threadIdx.x)) % tpr;
  const TY *y = static_cast<const TY *>(p.y) + blockIdx.x * p.ldy;  // of this row; `step` rows further on:
  const TR *r = POST ? static_cast<const TR *>(p.residual) + blockIdx.x * p.ldr : nullptr;
  const int64_t y_step = step * p.ldy, r_step = step * p.ldr;
  auto fetch = [&](int64_t row, int slot) {  // by thread 0
    uint8_t *at = smem + slot * g.stage_bytes + 16;
    const TY *yr = static_cast<const TY *>(p.y) + row * p.ldy;
    const Span<TY> ys(yr, cols);
    const uint32_t y_bytes = (ys.end - ys.head) * sizeof(TY);
    if (POST) {
      const TR *rr = static_cast<const TR *>(p.residual) + row * p.ldr;
      const Span<TR> rs(rr, cols);
      const uint32_t r_bytes = (rs.end - rs.head) * sizeof(TR);
      mbar_expect_tx(&full[slot], y_bytes + r_bytes);
      bulk_load(at + g.at[1], rr + rs.head, r_bytes, &full[slot]);
    } else {
      mbar_expect_tx(&full[slot], y_bytes);
    }
    bulk_load(at, yr + ys.head, y_bytes, &full[slot]);
  };
  if (threadIdx.x == 0) {
    int64_t row = blockIdx.x;
    for (int i = 0; i < g.stages && row < p.rows; ++i, row += step) fetch(row, i);
  }
  auto weights = [&](const void *base, int dt, float *w) {
    by_type(dt, [&](auto type) {
      using T = decltype(type);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = e * tpr + threadIdx.x;
        w[e] = c < cols ? static_cast<float>((static_cast<const T *>(base) + threadIdx.x)[e * TPR]) : 0.f;
      }
    });
  };
  float w[E], next_w[E];
  if (POST && p.w) weights(p.w, p.w_dt, w);
  if (EARLY && p.next_w) weights(p.next_w, p.nw_dt, next_w);
  Edge<TY> y_edge{};
  Edge<TR> r_edge{};
  if (blockIdx.x < p.rows) {
    y_edge = Span<TY>(y, cols).edge(y, last);
    if (POST) r_edge = Span<TR>(r, cols).edge(r, last);
  }
  bool arrived = true;
  int slot = 0, parity = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += step, parity ^= 1) {
    float gate[E];
    if (POST && p.gate)
      by_type(p.g_dt, [&](auto type) {
        using T = decltype(type);
        const T *from = static_cast<const T *>(p.gate) + row / p.rows_per_gate * p.ldg + threadIdx.x;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int c = e * tpr + threadIdx.x;
          gate[e] = c < cols ? static_cast<float>(from[e * TPR]) : 0.f;
        }
      });
    const Span<TY> ys(y, cols);
    const Span<TR> rs(r, cols);
    const Edge<TY> y_now = y_edge;
    const Edge<TR> r_now = r_edge;
    y += y_step;
    if (POST) r += r_step;
    if (row + step < p.rows) {
      y_edge = Span<TY>(y, cols).edge(y, last);
      if (POST) r_edge = Span<TR>(r, cols).edge(r, last);
    }
    if (arrived && !mbar_wait(&full[slot], phase)) {
      raise_status(kStatusNormLoadWait);  // what there is goes on; the status says that it may be wrong
      arrived = false;
      if (threadIdx.x == 0) lost = Lost{row, slot, phase};
    }
    uint8_t *at = smem + slot * g.stage_bytes;
    float z[E], sum = 0.f;
    uint32_t top = 0u;
    const TY *from = ys.put(at, y_now, last) + threadIdx.x;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e * tpr + threadIdx.x;
      z[e] = c < cols ? static_cast<float>(from[e * TPR]) : 0.f;
    }
    if (POST) {
      float inv = p.scale;
      if (p.w) {
        sum = squares<E>(z);
        row_reduce<E>(z, sum, top, false, tpr, scratch[parity][0]);
        inv *= rsqrtf(fmaf(sum, p.inv_cols, p.eps));
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] *= w[e];
      }
      if (p.gate)
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] *= gate[e];
      const TR *residual = rs.put(at + g.at[1], r_now, last) + threadIdx.x;
      TR *out = static_cast<TR *>(p.out) + row * p.ldo + threadIdx.x;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int c = e * tpr + threadIdx.x;
        if (c < cols) {
          z[e] = fmaf(z[e], inv, static_cast<float>(residual[e * TPR]));
          store_vec<TR, 1>(out + e * TPR, z + e);
        }
      }
    }
    if (!POST || p.h) {
      sum = squares<E>(z);
      if (EARLY && p.next_w)
#pragma unroll
        for (int e = 0; e < E; ++e) z[e] *= next_w[e];
      row_reduce<E>(z, sum, top, p.h_dt == MQ_S8, tpr, scratch[parity][1]);
    }
    if (tpr == 32 || (POST && !p.h)) __syncthreads();  // else row_reduce's barrier: every thread has read the slot
    if (threadIdx.x == 0 && arrived && row + static_cast<int64_t>(g.stages) * step < p.rows)
      fetch(row + static_cast<int64_t>(g.stages) * step, slot);
    if (++slot == g.stages) slot = 0, phase ^= 1;
    if (!POST || p.h) write_h<1, E, TPR>(p, row, z, sum, top);
  }
  if (threadIdx.x == 0 && !arrived) drain_ring(full, g, p.rows, lost);
}

template <int VEC, int E, bool POST, bool EARLY>
int launch_e(const Params &p, int threads, int rows_per_cta, cudaStream_t s, const char *what) {
  const int64_t grid = (p.rows + rows_per_cta - 1) / rows_per_cta;
  MQ_REQUIRE(grid < (1LL << 31), MQ_EUNSUPPORTED, "%s: too many rows", what);
  return launch_overlapped(block_norm_kernel<VEC, E, POST, EARLY>, dim3(static_cast<unsigned>(grid)),
                           dim3(threads, rows_per_cta), 0, s, what, p);
}

constexpr int kMaxCols = 64 * kMaxThreads;

inline int bytes_of(int dt) { return dt == MQ_F32 ? 4 : 2; }

// The ring for this row size with `per_sm` CTAs on an SM; stages < 2: it does not fit.
template <bool POST>
Ring ring_of(const Params &p, int per_sm) {
  Ring g{};
  const int dts[2] = {p.y_dt, p.r_dt};
  for (int i = 0; i < (POST ? 2 : 1); ++i) {
    g.at[i] = g.stage_bytes;
    g.row_bytes[i] = p.cols * bytes_of(dts[i]);
    g.stage_bytes += g.row_bytes[i];
  }
  const int w = POST && p.w ? p.cols * bytes_of(p.w_dt) : 0, nw = p.next_w ? p.cols * bytes_of(p.nw_dt) : 0;
  g.stages = std::min(kRingMax, (200 * 1024 / per_sm - 1536 - w - nw) / g.stage_bytes);
  g.w_at = g.stages * g.stage_bytes;
  g.next_w_at = g.w_at + w;
  g.total = g.next_w_at + nw;
  return g;
}

// CTAs per SM of the streaming kernel, 0 where it does not apply: 16 values a thread, 1024 threads per SM, fewer
// where the ring would have less than three stages. The residual has y's type or fp32; w, next_w and the gate one
// type, y's or fp32.
template <bool POST>
int plan_ring(Params &p) {
  if (POST && p.r_dt != p.y_dt && p.r_dt != MQ_F32) return 0;
  const int dts[3] = {POST && p.w ? p.w_dt : -1, POST && p.gate ? p.g_dt : -1, p.next_w ? p.nw_dt : -1};
  int one = -1;
  for (int dt : dts) {
    if (dt < 0) continue;
    if ((dt != p.y_dt && dt != MQ_F32) || (one >= 0 && dt != one)) return 0;
    one = dt;
  }
  p.w_dt = p.g_dt = p.nw_dt = one < 0 ? p.y_dt : one;
  p.tpr = (p.cols + 511) / 512 * 32;
  if (p.cols < 768 || p.tpr > kStreamThreads) return 0;
  for (int per_sm = std::min(16, 1024 / p.tpr); per_sm >= 1; --per_sm)
    if (ring_of<POST>(p, per_sm).stages >= (per_sm > 1 ? 3 : 2)) return per_sm;
  return 0;
}

// As many CTAs as run at once: those that had to wait would start their rows when the others are done.
template <typename Kern>
int launch_persistent(Kern kern, int per_sm, const Params &p, const Ring &g, cudaStream_t s, const char *what) {
  int fit = 0;
  const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kern, p.tpr, g.total);
  if (e != cudaSuccess || fit < 1) return fail(MQ_ECUDA, "%s: occupancy: %s", what, cudaGetErrorString(e));
  const int64_t grid = std::min<int64_t>(p.rows, 148 * std::min(per_sm, fit));
  return launch_overlapped(kern, dim3(static_cast<unsigned>(grid)), dim3(p.tpr), g.total, s, what, p, g);
}

template <typename TY, typename TR, typename TW, int E, bool POST, bool EARLY>
int launch_ring_e(const Params &p, int per_sm, cudaStream_t s, const char *what) {
  const Ring g = ring_of<POST>(p, per_sm);
  auto kern = row_stream_kernel<TY, TR, TW, E, POST, EARLY>;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(kern, g.total, configured, what)) return rc;
  return launch_persistent(kern, per_sm, p, g, s, what);
}

template <typename TY, bool POST, bool EARLY>
int launch_ring_y(const Params &p, int per_sm, cudaStream_t s, const char *what) {
  auto wide = [&](auto r, auto w) {
    using TR = decltype(r);
    using TW = decltype(w);
    return launch_ring_e<TY, TR, TW, 2, POST, EARLY>(p, per_sm, s, what);
  };
  auto with_r = [&](auto r) {
    if constexpr (EARLY && !std::is_same<TY, float>::value)  // (the quantiser has no weights)
      if (p.nw_dt != p.y_dt) return wide(r, float());
    return wide(r, TY());
  };
  if constexpr (POST && !std::is_same<TY, float>::value)
    if (p.r_dt != p.y_dt) return with_r(float());
  return with_r(TY());
}

template <bool POST, bool EARLY>
int launch_ring(const Params &p, int per_sm, cudaStream_t s, const char *what) {
  if (p.y_dt == MQ_F32) return launch_ring_y<float, POST, EARLY>(p, per_sm, s, what);
  if (p.y_dt == MQ_F16) return launch_ring_y<__half, POST, EARLY>(p, per_sm, s, what);
  return launch_ring_y<__nv_bfloat16, POST, EARLY>(p, per_sm, s, what);
}

// The ring of the kernel for unaligned rows: the same without the weights.
template <typename TY, typename TR, int TPR, bool POST, bool EARLY>
int launch_ring1_e(const Params &p, const Ring &g, int per_sm, cudaStream_t s, const char *what) {
  auto kern = row_stream1_kernel<TY, TR, TPR, POST, EARLY>;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(kern, g.total, configured, what)) return rc;
  return launch_persistent(kern, per_sm, p, g, s, what);
}

template <typename TY, typename TR, bool POST, bool EARLY>
int launch_ring1_t(const Params &p, const Ring &g, int per_sm, cudaStream_t s, const char *what) {
  if (p.tpr == 64) return launch_ring1_e<TY, TR, 64, POST, EARLY>(p, g, per_sm, s, what);
  if (p.tpr == 128) return launch_ring1_e<TY, TR, 128, POST, EARLY>(p, g, per_sm, s, what);
  if (p.tpr == 256) return launch_ring1_e<TY, TR, 256, POST, EARLY>(p, g, per_sm, s, what);
  return launch_ring1_e<TY, TR, 512, POST, EARLY>(p, g, per_sm, s, what);
}

template <typename TY, bool POST, bool EARLY>
int launch_ring1_y(const Params &p, const Ring &g, int per_sm, cudaStream_t s, const char *what) {
  if constexpr (POST && !std::is_same<TY, float>::value)
    if (p.r_dt == MQ_F32) return launch_ring1_t<TY, float, POST, EARLY>(p, g, per_sm, s, what);
  return launch_ring1_t<TY, TY, POST, EARLY>(p, g, per_sm, s, what);
}

template <bool POST, bool EARLY>
int launch_ring1(Params p, cudaStream_t s, const char *what) {
  p.tpr = 64;
  while (16 * p.tpr < p.cols) p.tpr *= 2;
  const int per_sm = std::min(16, 1024 / p.tpr);
  Ring g{};
  const int dts[2] = {p.y_dt, p.r_dt};
  for (int i = 0; i < (POST ? 2 : 1); ++i) {
    g.at[i] = g.stage_bytes;
    g.stage_bytes += 16 + (p.cols * bytes_of(dts[i]) + 15) / 16 * 16;
  }
  g.stages = std::max(2, std::min(kRingMax, (200 * 1024 / per_sm - 1536) / g.stage_bytes));
  g.total = g.stages * g.stage_bytes;
  if (p.y_dt == MQ_F32) return launch_ring1_y<float, POST, EARLY>(p, g, per_sm, s, what);
  if (p.y_dt == MQ_F16) return launch_ring1_y<__half, POST, EARLY>(p, g, per_sm, s, what);
  return launch_ring1_y<__nv_bfloat16, POST, EARLY>(p, g, per_sm, s, what);
}

template <bool POST, bool EARLY>
int launch(Params p, bool vec, cudaStream_t s, const char *what) {
  MQ_REQUIRE(p.cols <= kMaxCols, MQ_EUNSUPPORTED, "%s: cols is above %d", what, kMaxCols);
  if (vec && p.rows >= 4 * 148)
    if (const int per_sm = plan_ring<POST>(p)) return launch_ring<POST, EARLY>(p, per_sm, s, what);
  if (!vec && p.rows >= 4 * 148 && p.cols >= 256 && p.cols <= 16 * kStreamThreads && (!POST || p.r_dt == p.y_dt || p.r_dt == MQ_F32))
    return launch_ring1<POST, EARLY>(p, s, what);
  // Few rows: a thread of a row for each 8 values, for the least latency. Many: 16, so that what a reduction costs
  // each thread (as much as some 20 values) is spread over more of them. Without alignment 4 and 16 single values.
  const int per = p.rows >= 4 * 148 ? 16 : vec ? 8 : 4;
  p.tpr = std::min(kMaxThreads, (p.cols + 32 * per - 1) / (32 * per) * 32);
  const int rows_per_cta = p.tpr == 32 ? 4 : 1, each = (p.cols + p.tpr - 1) / p.tpr;
  if (vec) {
    if (each <= 8) return launch_e<8, 1, POST, EARLY>(p, p.tpr, rows_per_cta, s, what);
    if (each <= 16) return launch_e<8, 2, POST, EARLY>(p, p.tpr, rows_per_cta, s, what);
    if (each <= 32) return launch_e<8, 4, POST, EARLY>(p, p.tpr, rows_per_cta, s, what);
    return launch_e<8, 8, POST, EARLY>(p, p.tpr, 1, s, what);
  }
  if (each <= 4) return launch_e<1, 4, POST, EARLY>(p, p.tpr, rows_per_cta, s, what);
  if (each <= 16) return launch_e<1, 16, POST, EARLY>(p, p.tpr, rows_per_cta, s, what);
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
  p.rows = rows, p.cols = static_cast<int>(cols), p.inv_cols = 1.f / static_cast<float>(cols);
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
  p.rows = rows, p.cols = static_cast<int>(cols), p.inv_cols = 1.f / static_cast<float>(cols);
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
  if (h) p.next_w = next_w, p.nw_dt = next_w_dtype, p.next_eps = next_eps;  // (unchecked, and not read, without h)
  p.h = h, p.h_dt = h_dtype, p.ldh = ldh, p.hs = hs;
  p.rows = rows, p.cols = static_cast<int>(cols), p.inv_cols = 1.f / static_cast<float>(cols);
  using mq::norm::vec_ok;
  const bool vec = cols % 8 == 0 && vec_ok(y, y_dtype, ldy, rows) && vec_ok(residual, r_dtype, ldr, rows) &&
                   vec_ok(out, r_dtype, ldo, rows) && vec_ok(w, w_dtype, cols, 1) &&
                   vec_ok(gate, gate_dtype, ldg, rows) && vec_ok(p.next_w, next_w_dtype, cols, 1) &&
                   vec_ok(h, h_dtype, ldh, rows);
  return mq::norm::launch<true, true>(p, vec, static_cast<cudaStream_t>(stream), what);
}
