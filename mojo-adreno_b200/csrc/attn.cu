// Attention of new tokens over a paged cache, for sequences with few rows per kv head (mq_paged_attention; many rows:
// attn_tile.cu).
//
//   o[i] = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i.k_j),  j over the positions that row i sees:
//   p - window < j <= p with p the row's own position.
//
// The group's query heads of all of a sequence's new tokens are the rows of one product with a kv head's keys, so a
// key or value is read once for all of them: up to 16 rows here, a decode batch. What bounds it is the stream of keys and values;
// arithmetic goes to the warp-level mma.m16n8k16, which has the rate for it (64 keys x 128 dim x 16 rows: 128 of them, 280 cycles,
// against the 1400 that an SM's share of the bandwidth needs for the 16-bit rows) and takes its operands without a detour through
// TMEM. 64 sequences of 4000 positions on average, 8 kv heads of 128: bf16 163 us (6.5 TB/s, the copy bandwidth), int8 144 us
// (3.8 TB/s: conversions and their latency, a third of the cycles issue). One sequence of 1001: 8.7 us with the joining
// kernel, latency: a traced run had 1.3 for the shares, 0.6 until an item is known and 5.1 for the whole launch.
//
//  * A producer warp walks through the CTA's items and brings blocks of 64 keys and values (int8: 128) through a ring, one tiled
//    copy per page (or part of one) and 128 (int8: 64) bytes of a row, a lane each. Only an item's end joins the consumers.
//  * Four consumer warps share a block's keys. Each keeps its own running maximum, sum and accumulators, in fp32, and they
//    meet once, when an item ends.
//  * All CTAs take equal shares of all blocks (paged.cuh), so lengths need not be known on the host and a long
//    sequence takes as many SMs as it has work for. Parts of cut items are joined by a kernel behind this one, in a fixed
//    order: results do not vary from run to run.
//  * int8: k_j = s_j * integers, v_j = t_j * integers. The integers go to fp16 exactly (a byte next to 0x64 is
//    1024 + it), the rows' q to fp16 after a power of two that its largest |q| fixes (exact but below 2^-24 of that). s_j scales
//    the scores; t_j goes into the exponent: w_j t_j = 2^(score + log2 t_j - m) with m the maximum of that, so the
//    weights that meet the integers are at most 2^8 whatever the scales, and the sum of w is that of (w t) (1 / t).
//  * Weights are rounded to the MMA's 16 bits (scores, maxima, sums and accumulators are fp32). A 16-bit cache's are summed as
//    they were rounded, which takes the error back where one key has most of the weight.
//  * Neither kernel lets the next one start early (64x1 int8: 210 us with both doing so, 146 with either or neither). Why is not
//    traced; early CTAs taking places of a grid that is as many CTAs as run at once would explain it.
//  * The maximum may lag by 2^8 before accumulators are rescaled: weights up to 2^8 are as exact in fp16 and bf16.
//  * Blocks that some row sees only in part: scores are replaced, not added to, so no hidden key's value matters; a
//    value that is no number is taken out of the product and makes the sum, so the result, of the rows that see it NaN.
#include "paged.cuh"

namespace mq {
namespace paged {

constexpr int kFewRows = 16;  // the most rows of an item
constexpr int kFewWarps = 4, kFewThreads = 32 * (kFewWarps + 1);
constexpr int kPadCols = 72;                 // floats between rows of the joining buffer: no bank conflicts

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool BF>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_16816(d, a[0], a[1], a[2], a[3], b0, b1);
}
template <bool BF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&b);
  }
  return pack_half2(lo, hi);
}
// Two bytes of x (biased by 128), which SEL puts beside 0x64 each, as fp16 integers in -128 .. 127.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t x) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0x64646464u), "n"(SEL));
  const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&r), __half2half2(__ushort_as_half(0x6480)));  // 1152
  return *reinterpret_cast<const uint32_t *>(&h);
}
// 0xffff in each half of x that is infinite or no number.
template <bool BF>
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {
  constexpr uint32_t e = BF ? 0x7f807f80u : 0x7c007c00u;
  return __vcmpeq2(x & e, e);
}
// V scales count as at least this: their inverses and the sums of those stay finite.
constexpr float kLeastScale = 1e-30f;

struct AttnParams {
  Seqs seqs;
  Shape shape;
  const void *q;
  int64_t q_token, q_head;  // strides in elements
  int q_dtype;
  const float *k_scale, *v_scale;
  int64_t ks_stride[3], vs_stride[3];
  Output o;
  float scale;  // times log2(e)
  Parts parts;
};

template <typename T>
__device__ __forceinline__ void store4(void *out, int64_t at, float a, float b, float c, float d) {
  struct alignas(4 * sizeof(T)) Four {
    T t[4];
  };
  *reinterpret_cast<Four *>(static_cast<T *>(out) + at) = Four{{T(a), T(b), T(c), T(d)}};
}
__device__ __forceinline__ void store_out4(const Output &o, int64_t token, int64_t head, int col, float a, float b, float c, float d) {
  const int64_t at = token * o.token_stride + head * o.head_stride + col;
  if (o.dtype == MQ_F16)
    store4<__half>(o.out, at, a, b, c, d);
  else
    store4<__nv_bfloat16>(o.out, at, a, b, c, d);
}
// What a row's accumulators are multiplied by: 0 for a row that sees nothing, NaN where its sum is.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }

template <int D, int KIND>
struct Few {
  static constexpr int kBytes = KIND == MQ_S8 ? 1 : 2;
  // Keys of a block: 32 KB of keys and values either way at 128 dim (int8 64x1: 144 us with two CTAs and 128 keys, 148 with three
  // and 64, 186 with two and 64).
  static constexpr int kKeys = KIND == MQ_S8 ? 128 : 64;
  using Units = Grain<kFewRows, kKeys, 2>;
  static constexpr int kBox = KIND == MQ_S8 ? 64 : 128;                 // bytes of a row in a box
  static constexpr int kBoxes = D * kBytes / kBox;
  static constexpr int kTile = kKeys * D * kBytes;                   // of keys, or of values
  static constexpr int kScales = KIND == MQ_S8 ? 3 * kKeys * 4 : 0;  // keys' scales, values': log2 and inverse
  static constexpr int kStageBytes = 2 * kTile + (kScales + 1023) / 1024 * 1024;
  // Two CTAs on an SM where a stage has 32 KB, else three; as many stages, up to four, as fit beside the joining buffer.
  static constexpr int kCtas = D == 128 ? 2 : 3;
  static constexpr int kJoin = kFewWarps * kFewRows * kPadCols * 4;
  static constexpr int kRoom = (227 * 1024 / kCtas - 1024 - kJoin - 2048) / kStageBytes;
  static constexpr int kStages = kRoom > 4 ? 4 : kRoom;
  static constexpr int kSmem = kStages * kStageBytes + kJoin + 1024;
};

template <int D, int KIND>
__global__ void __launch_bounds__(kFewThreads, Few<D, KIND>::kCtas)
    attn_few_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AttnParams p) {
  using F = Few<D, KIND>;
  constexpr bool BF = KIND == MQ_BF16, S8 = KIND == MQ_S8;
  constexpr int kFewKeys = F::kKeys, WK = kFewWarps, KW = kFewKeys / WK;  // the warps share a block's keys
  constexpr int NT = KW / 8, S = F::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *ring = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  float *join = reinterpret_cast<float *>(ring + S * F::kStageBytes);  // [WK][kFewRows][kPadCols]
  __shared__ uint64_t full[S], empty[S], meeting;
  __shared__ ShareScratch<kFewThreads> scratch;
  __shared__ ItemRing items;
  __shared__ float2 row_stats[WK][kFewRows];
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(&full[i], S8 ? 33 : 1);  // the copies' bytes; the lanes whose scales have come
      mbar_init(&empty[i], kFewWarps);
    }
    items.init(kFewWarps);
    mbar_init(&meeting, kFewWarps);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  griddep_wait();
  find_share<kFewThreads, typename F::Units>(p.seqs, p.shape, scratch);
  if (blockIdx.x == 0 && tid == 0) p.parts.counts[0] = scratch.found.total, p.parts.counts[1] = scratch.found.parts;
  if (static_cast<int>(blockIdx.x) >= scratch.found.parts) return;
  Item item;

  if (warp == kFewWarps) {
    if (lane == 0) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
    const int box_rows = min(kFewKeys, 1 << p.seqs.page_log2), per_block = kFewKeys / box_rows;
    const int boxes = per_block * F::kBoxes;  // of keys, and as many of values
    Walk<typename F::Units> walk;
    walk.start(p.shape, scratch.found);
    const Walk<typename F::Units> begin = walk;
    int s = 0, round = 0, k = 0;
    uint32_t issued = 0;
    bool ok = true;
    while (ok) {
      if (!walk.next(p.seqs, p.shape, item)) item.blocks = 0;
      if (!items.put(k++, item)) {
        if (lane == 0) raise_status(kStatusAttnLoadWait), abort_flag = 1;
        break;
      }
      if (item.blocks == 0) break;
      for (int i = 0; i < item.blocks; ++i) {
        const int key0 = (item.block + i) * kFewKeys;
        // Boxes behind the sequence's end are not fetched: their table entries may be anything.
        const int live = max(0, min(per_block, (item.s.length - key0 + box_rows - 1) / box_rows));
        int page = -1;  // lane l knows the page of box l of the block
        if (lane < live) page = page_of(p.seqs, item.b, key0 + lane * box_rows);
        float sk[kFewKeys / 32], sv[kFewKeys / 32];  // scales of keys lane, lane + 32 ..
        if (S8) {
#pragma unroll
          for (int h = 0; h < kFewKeys / 32; ++h) {
            const int key = lane + 32 * h, of = __shfl_sync(0xffffffffu, page, key / box_rows);
            sk[h] = 0.f, sv[h] = 0.f;
            if (of >= 0 && key0 + key < item.s.length) {
              const int row = (key0 + key) & ((1 << p.seqs.page_log2) - 1);
              sk[h] = p.k_scale[of * p.ks_stride[0] + item.head * p.ks_stride[1] + row * p.ks_stride[2]];
              sv[h] = p.v_scale[of * p.vs_stride[0] + item.head * p.vs_stride[1] + row * p.vs_stride[2]];
            }
            // (An infinite key scale would make a score of minus infinity, so no weight, where the product is negative.)
            if (!(sk[h] < INFINITY)) sk[h] = NAN;
            if (sv[h] < kLeastScale) sv[h] = kLeastScale;  // (fmaxf would drop a NaN)
          }
        }
        if (round > 0 && !__all_sync(0xffffffffu, wait_for(&empty[s], (round - 1) & 1))) {
          if (lane == 0) raise_status(kStatusAttnLoadWait), abort_flag = 1;
          ok = false;
          break;
        }
        uint8_t *stage = ring + s * F::kStageBytes;
        if (S8) {
          float *sc = reinterpret_cast<float *>(stage + 2 * F::kTile);
#pragma unroll
          for (int h = 0; h < kFewKeys / 32; ++h)
            sc[lane + 32 * h] = sk[h], sc[kFewKeys + lane + 32 * h] = lg2(sv[h]), sc[2 * kFewKeys + lane + 32 * h] = __frcp_rn(sv[h]);
        }
        if (lane == 0) mbar_expect_tx(&full[s], 2 * live * F::kBoxes * box_rows * F::kBox);
        __syncwarp();
        for (int base = 0; base < 2 * boxes; base += 32) {
          const int l = base + lane, which = l / boxes, box = l % boxes, part = box / per_block, at = box % per_block;
          const int of = __shfl_sync(0xffffffffu, page, at);
          if (l < 2 * boxes && at < live) {
            const int row = (key0 + at * box_rows) & ((1 << p.seqs.page_log2) - 1);
            uint8_t *dst = stage + which * F::kTile + part * kFewKeys * F::kBox + at * box_rows * F::kBox;
            // (a page outside the pool lies outside the map: zeros)
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(which ? &vmap : &kmap)), "r"(smem_u32(&full[s])),
                "r"(part * (F::kBox / F::kBytes)), "r"(row), "r"(item.head), "r"(of < 0 ? p.seqs.pages : of)
                : "memory");
          }
        }
        if (S8) mbar_arrive(&full[s]);
        ++issued;
        if (++s == S) s = 0, ++round;
      }
    }
    if (lane == 0) p.parts.cuts[blockIdx.x] = cut_at(begin, p.shape, scratch.found);
    // Leave no copy in flight.
    if (lane == 0)
      for (uint32_t i = issued > S ? issued - S : 0; i < issued; ++i) wait_for(&full[i % S], (i / S) & 1);
    return;
  }

  const int wk = warp, g = lane / 4, t = lane % 4;
  const int heads = p.shape.group;
  int s = 0;
  uint32_t phase = 0, meetings = 0;
  // All four warps, or false for those that waited in vain.
  auto meet = [&]() -> bool {
    __syncwarp();
    if (lane == 0) mbar_arrive(&meeting);
    const bool met = !abort_flag && wait_for(&meeting, meetings++ & 1);
    if (__all_sync(0xffffffffu, met)) return true;
    if (lane == 0 && !abort_flag) raise_status(kStatusAttnSoftmaxWait), abort_flag = 1;
    return false;
  };
  for (int k = 0;; ++k) {
    const bool told = wait_for(&items.full[k % kItems], (k / kItems) & 1);
    if (!__all_sync(0xffffffffu, told)) {
      if (lane == 0 && !abort_flag) raise_status(kStatusAttnSoftmaxWait), abort_flag = 1;
      break;  // (what the others wait for next does not come either)
    }
    item = items.item[k % kItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(&items.empty[k % kItems]);
    if (item.blocks == 0) break;
    const int rows = item.s.n * heads;
    // A thread's rows are g and g + 8 of its warp's 16; q as the MMA's A, in registers.
    uint32_t qa[D / 16][4];
    float row_scale[2];
    int lo[2], hi[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = g + 8 * r, i = over_group(p.shape, min(row, rows - 1));
      const int pos = item.s.pos0 + i;
      hi[r] = max(pos + 1, 0);
      lo[r] = p.shape.window ? max(0, pos + 1 - p.shape.window) : 0;
      row_scale[r] = p.scale;
      const int64_t at = static_cast<int64_t>(item.s.first + i) * p.q_token + static_cast<int64_t>(item.head * heads + row - i * heads) * p.q_head;
      const bool real = row < rows;
      if constexpr (S8) {
        float v[D / 4];  // d = 64 h + 16 t + 0 .. 15: bytes that a 16-byte load of the keys brings to this thread
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int d = 64 * h + 16 * t + 8 * u;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (real && d < p.o.dim) w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + at + d);
            const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float2 f;
              if (p.q_dtype == MQ_F16)
                f = __half22float2(*reinterpret_cast<const __half2 *>(&ws[e]));
              else
                f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&ws[e]));
              v[16 * h + 8 * u + 2 * e] = f.x, v[16 * h + 8 * u + 2 * e + 1] = f.y;
            }
          }
        float big = 0.f;
#pragma unroll
        for (int e = 0; e < D / 4; ++e) big = fmaxf(big, fabsf(v[e]));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
        // 2^e with 1 <= big / 2^e < 2, from the exponent's bits (an infinite row stays one; a tiny one counts as 2^-100's).
        const uint32_t e = min(max(__float_as_uint(big) >> 23, 27u), 227u);
        const float up = __uint_as_float(e << 23), down = __uint_as_float((254 - e) << 23);
        row_scale[r] *= up;
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            qa[4 * h + i4][r] = pack_half2(v[16 * h + 4 * i4] * down, v[16 * h + 4 * i4 + 1] * down);
            qa[4 * h + i4][r + 2] = pack_half2(v[16 * h + 4 * i4 + 2] * down, v[16 * h + 4 * i4 + 3] * down);
          }
      } else {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int d = 16 * k + 8 * u + 2 * t;
            qa[k][r + 2 * u] = real && d < p.o.dim ? *reinterpret_cast<const uint32_t *>(static_cast<const uint16_t *>(p.q) + at + d) : 0u;
          }
      }
    }
    // Blocks outside [most_lo, least_hi) are seen in part by some row (rows rise with their position).
    const int least_hi = max(item.s.pos0 + 1, 0);
    const int most_lo = p.shape.window ? max(0, item.s.pos0 + item.s.n - p.shape.window) : 0;

    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l: this thread's columns

    for (int b = 0; b < item.blocks; ++b) {
      const bool came = !abort_flag && wait_for(&full[s], phase);
      if (!__all_sync(0xffffffffu, came)) {
        if (lane == 0 && !abort_flag) raise_status(kStatusAttnSoftmaxWait), abort_flag = 1;
        break;
      }
      const uint32_t stage = smem_u32(ring + s * F::kStageBytes);
      const float *scales = reinterpret_cast<const float *>(ring + s * F::kStageBytes + 2 * F::kTile);
      const int key0 = (item.block + b) * kFewKeys + wk * KW;  // of this warp
      const bool edge = key0 + KW > least_hi || key0 < most_lo;
      float c[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[j][e] = 0.f;
      // Scores. int8: word w of a thread's 16 bytes is its k of one step, for keys and q alike.
      if constexpr (S8) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const int key = wk * KW + 8 * j + g;
#pragma unroll
          for (int h = 0; h < D / 64; ++h) {
            uint32_t w[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                         : "r"(stage + h * kFewKeys * 64 + key * 64 + ((t ^ ((key >> 1) & 3)) * 16)));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t x = w[e] ^ 0x80808080u;
              mma16<false>(c[j], qa[4 * h + e], bytes_to_half2<0x4140>(x), bytes_to_half2<0x4342>(x));
            }
          }
        }
      } else {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int j = 0; j < NT / 2; ++j) {
            const int key = wk * KW + 16 * j + (lane & 7) + ((lane >> 4) & 1) * 8, chunk = 2 * k + ((lane >> 3) & 1);
            uint32_t f[4];
            ldsm4(f, stage + (chunk / 8) * kFewKeys * 128 + key * 128 + (((chunk & 7) ^ (key & 7)) * 16));
            mma16<BF>(c[2 * j], qa[k], f[0], f[1]);
            mma16<BF>(c[2 * j + 1], qa[k], f[2], f[3]);
          }
      }
      const uint32_t values = stage + F::kTile;
      // 16 keys (step kk) x 16 columns (16-bit) or 32 (int8) of the values, as the MMA's B of two or four column tiles.
      auto value_at = [&](int kk, int j, uint32_t (&f)[4]) {
        const int key = wk * KW + 16 * kk + (lane & 7) + ((lane >> 3) & 1) * 8, chunk = 2 * j + (lane >> 4);
        if (S8)
          ldsm4t(f, values + (chunk / 4) * kFewKeys * 64 + key * 64 + (((chunk & 3) ^ ((key >> 1) & 3)) * 16));
        else
          ldsm4t(f, values + (chunk / 8) * kFewKeys * 128 + key * 128 + (((chunk & 7) ^ (key & 7)) * 16));
      };
      // Scaled scores, log2: of columns 8 j + 2 t + (e & 1), rows g + 8 (e >> 1).
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        if (S8) {
          const float2 ks = *reinterpret_cast<const float2 *>(scales + wk * KW + 8 * j + 2 * t);
          const float2 lv = *reinterpret_cast<const float2 *>(scales + kFewKeys + wk * KW + 8 * j + 2 * t);
          c[j][0] = fmaf(c[j][0] * row_scale[0], ks.x, lv.x), c[j][1] = fmaf(c[j][1] * row_scale[0], ks.y, lv.y);
          c[j][2] = fmaf(c[j][2] * row_scale[1], ks.x, lv.x), c[j][3] = fmaf(c[j][3] * row_scale[1], ks.y, lv.y);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[j][e] *= p.scale;
        }
      }
      if (edge) {
        if constexpr (!S8) {
#pragma unroll
          for (int kk = 0; kk < KW / 16; ++kk) {
            uint32_t bad[2] = {0, 0};  // keys 2 t, 2 t + 1 and 8 more of this step
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              uint32_t f[4];
              value_at(kk, j, f);
              bad[0] |= not_finite2<BF>(f[0]) | not_finite2<BF>(f[2]);
              bad[1] |= not_finite2<BF>(f[1]) | not_finite2<BF>(f[3]);
            }
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) {
              bad[0] |= __shfl_xor_sync(0xffffffffu, bad[0], x);
              bad[1] |= __shfl_xor_sync(0xffffffffu, bad[1], x);
            }
            if (bad[0] | bad[1])  // (rare: a row that sees one of them ends as NaN)
#pragma unroll
              for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int key = key0 + 16 * kk + 8 * u + 2 * t + (e & 1);
                  if ((bad[u] >> (e & 1 ? 16 : 0) & 1) && key < hi[e >> 1] && key >= lo[e >> 1]) l[e >> 1] = NAN;
                }
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int key = key0 + 8 * j + 2 * t + (e & 1);
            if (key >= hi[e >> 1] || key < lo[e >> 1]) c[j][e] = -INFINITY;
          }
      }
      float ref[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float top = fmaxf(c[0][2 * r], c[0][2 * r + 1]);
#pragma unroll
        for (int j = 1; j < NT; ++j) top = fmaxf(top, fmaxf(c[j][2 * r], c[j][2 * r + 1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const bool grows = top > m[r] + 8.f;  // (-inf + 8 is -inf)
        if (__any_sync(0xffffffffu, grows)) {
          const float next = grows ? top : m[r];
          const float a = m[r] == next ? 1.f : ex2(m[r] - next);
          l[r] *= a;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) o[j][2 * r] *= a, o[j][2 * r + 1] *= a;
          m[r] = next;
        }
        ref[r] = m[r] == -INFINITY ? 0.f : m[r];
      }
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) c[j][e] = ex2(c[j][e] - ref[e >> 1]);
      if (S8) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const float2 iv = *reinterpret_cast<const float2 *>(scales + 2 * kFewKeys + wk * KW + 8 * j + 2 * t);
          if (edge) {  // (a key that the row does not see may have any scale; its weight is 0)
            l[0] += (c[j][0] == 0.f ? 0.f : c[j][0] * iv.x) + (c[j][1] == 0.f ? 0.f : c[j][1] * iv.y);
            l[1] += (c[j][2] == 0.f ? 0.f : c[j][2] * iv.x) + (c[j][3] == 0.f ? 0.f : c[j][3] * iv.y);
          } else {
            l[0] += c[j][0] * iv.x + c[j][1] * iv.y;
            l[1] += c[j][2] * iv.x + c[j][3] * iv.y;
          }
        }
      }
      // Weights become the MMA's A; 16-bit caches sum them as they were rounded, so that the two roundings cancel where
      // one key has most of the weight.
#pragma unroll
      for (int kk = 0; kk < KW / 16; ++kk) {
        const uint32_t a[4] = {pack16<BF>(c[2 * kk][0], c[2 * kk][1]), pack16<BF>(c[2 * kk][2], c[2 * kk][3]),
                               pack16<BF>(c[2 * kk + 1][0], c[2 * kk + 1][1]), pack16<BF>(c[2 * kk + 1][2], c[2 * kk + 1][3])};
        if (!S8) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float2 f;
            if (BF)
              f = make_float2(__uint_as_float(a[e] << 16), __uint_as_float(a[e] & 0xffff0000u));
            else
              f = __half22float2(*reinterpret_cast<const __half2 *>(&a[e]));
            l[e & 1] += f.x + f.y;
          }
        }
        if constexpr (S8) {
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            uint32_t f[4];
            value_at(kk, j, f);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t x0 = f[2 * u] ^ 0x80808080u, x1 = f[2 * u + 1] ^ 0x80808080u;
              mma16<false>(o[4 * j + 2 * u], a, bytes_to_half2<0x4240>(x0), bytes_to_half2<0x4240>(x1));
              mma16<false>(o[4 * j + 2 * u + 1], a, bytes_to_half2<0x4341>(x0), bytes_to_half2<0x4341>(x1));
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            uint32_t f[4];
            value_at(kk, j, f);
            if (edge)
#pragma unroll
              for (int e = 0; e < 4; ++e) f[e] &= ~not_finite2<BF>(f[e]);
            mma16<BF>(o[2 * j], a, f[0], f[1]);
            mma16<BF>(o[2 * j + 1], a, f[2], f[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
      if (++s == S) s = 0, phase ^= 1;
    }

    // The warps that shared the keys join.
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t == 0) row_stats[wk][g + 8 * r] = make_float2(m[r], l[r]);
    }
    if (!meet()) break;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < WK; ++w) top = fmaxf(top, row_stats[w][g + 8 * r].x);
      const float a = m[r] == top ? 1.f : ex2(m[r] - top);
#pragma unroll
      for (int j = 0; j < D / 8; ++j) o[j][2 * r] *= a, o[j][2 * r + 1] *= a;
    }
    const bool goes_on = item.before > 0, whole = !goes_on && item.blocks == item.whole;
    const int64_t part0 = (2 * static_cast<int64_t>(blockIdx.x) + (goes_on ? 0 : 1)) * (kFewRows);
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
      float *mine = join + (wk * kFewRows) * kPadCols;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float *at = mine + (g + 8 * r) * kPadCols;
        if (S8) {  // columns 16 c + 4 t + 0 .. 3 of tiles 2 c (even ones) and 2 c + 1
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const auto &ev = o[8 * h + 2 * c], &od = o[8 * h + 2 * c + 1];
            *reinterpret_cast<float4 *>(at + 16 * c + 4 * t) = make_float4(ev[2 * r], od[2 * r], ev[2 * r + 1], od[2 * r + 1]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float2 *>(at + 8 * c + 2 * t) = make_float2(o[8 * h + c][2 * r], o[8 * h + c][2 * r + 1]);
        }
      }
      if (!meet()) return;
      for (int e = tid; e < kFewRows * 16; e += 32 * kFewWarps) {
        const int row = e / 16, col = e % 16 * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float4 x = *reinterpret_cast<const float4 *>(join + (w * kFewRows + row) * kPadCols + col);
          v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
          top = fmaxf(top, row_stats[w][row].x);
        }
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float2 st = row_stats[w][row];
          sum += st.x == top ? st.y : st.y * ex2(st.x - top);
        }
        if (row < rows) {
          if (whole) {
            const float inv = inverse_sum(sum);
            const int i = over_group(p.shape, row);
            if (64 * h + col < p.o.dim)
              store_out4(p.o, item.s.first + i, item.head * heads + row - i * heads, 64 * h + col, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
          } else {
            *reinterpret_cast<float4 *>(p.parts.sums + (part0 + row) * D + 64 * h + col) = v;
            if (h == 0 && col == 0) p.parts.stats[part0 + row] = make_float2(top, sum);
          }
        }
      }
      if (!meet()) return;
    }
  }
}

// Joins the parts of the items that CTAs of the launch before shared. CTA c (of x) takes the item that c goes on with
// where c is the first to do so; a warp a row. What a row needs is known after one load (the cut), so that the
// parts' statistics and sums come together: with nothing to join the launch took 3 us (profiled, cold).
struct JoinParams {
  Shape shape;
  Output o;
  Parts parts;
  int rows;  // of an item's parts
};
constexpr int kJoinWarps = 8;
template <int D, int TILE_ROWS>
__global__ void __launch_bounds__(32 * kJoinWarps) attn_join_kernel(const JoinParams p) {
  griddep_wait();
  const int c = blockIdx.x, lane = threadIdx.x % 32;
  if (c == 0) return;
  const int64_t total = p.parts.counts[0], ctas = p.parts.counts[1];
  const Cut cut = p.parts.cuts[c];  // (there is one, used or not)
  if (c >= ctas || !cut.goes_on || total * (c - 1) / ctas > cut.first) return;
  const int rows = min(TILE_ROWS, cut.n * p.shape.group - cut.tile * TILE_ROWS);
  // Part 0 is CTA c - 1's, which began the item (its slot 1), the others what CTAs c .. last went on with (slot 0); CTA `last`
  // is the last whose share begins before the item's end.
  const int last = static_cast<int>((cut.end * ctas + total - 1) / total) - 1, n = last - c + 2;
  for (int row = blockIdx.y * kJoinWarps + threadIdx.x / 32; row < rows; row += gridDim.y * kJoinWarps) {
    auto at = [&](int i) { return (2 * static_cast<int64_t>(c - 1 + i) + (i == 0 ? 1 : 0)) * p.rows + row; };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, p.parts.stats[at(i)].x);
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    constexpr int kLanes = D / 4, kTurns = 32 / kLanes;  // lanes of a part, parts at a time
    const int u = lane % kLanes;
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = lane / kLanes; i < n; i += kTurns) {
      const int64_t a = at(i);
      const float2 st = p.parts.stats[a];
      const float4 x = *reinterpret_cast<const float4 *>(p.parts.sums + a * D + u * 4);
      const float w = st.x == top ? 1.f : ex2(st.x - top);
      sum += st.y * w;
      v.x += x.x * w, v.y += x.y * w, v.z += x.z * w, v.w += x.w * w;
    }
    if (kTurns == 2) {
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      v.x += __shfl_xor_sync(0xffffffffu, v.x, 16), v.y += __shfl_xor_sync(0xffffffffu, v.y, 16);
      v.z += __shfl_xor_sync(0xffffffffu, v.z, 16), v.w += __shfl_xor_sync(0xffffffffu, v.w, 16);
    }
    const float inv = inverse_sum(sum);
    const int r = cut.tile * TILE_ROWS + row, i = over_group(p.shape, r);
    if (lane < kLanes && u * 4 < p.o.dim)
      store_out4(p.o, cut.token + i, cut.head * p.shape.group + r - i * p.shape.group, u * 4, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
  }
}

// A map of a pool's rows: (dim, row of the page, head, page), boxes of `box_bytes` of `box_rows` rows.
inline int encode_pages(CUtensorMap *map, void *base, int dtype, const mq_kv_pages *c, const int64_t *stride, int box_bytes,
                        int box_rows, CUtensorMapSwizzle swizzle, const char *what) {
  const int es = element_size(dtype);
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c->dim), static_cast<cuuint64_t>(c->page), static_cast<cuuint64_t>(c->heads),
                              static_cast<cuuint64_t>(c->pages)};
  // (a stride is not used where its dimension has one index, and may then be anything)
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 16 : static_cast<cuuint64_t>(stride[2 - i]) * es;
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(box_bytes / es), static_cast<cuuint32_t>(box_rows), 1, 1};
  return encode_tmap_4d(map, base, dtype == MQ_S8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : dtype == MQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                        dims, strides, box, swizzle, what);
}

template <int D, int KIND>
int launch_few(const mq_kv_pages *c, AttnParams p, int ctas, void *workspace, cudaStream_t stream, const char *what) {
  using F = Few<D, KIND>;
  CUtensorMap kmap, vmap;
  const int box_rows = std::min(F::kKeys, c->page);
  const CUtensorMapSwizzle swizzle = KIND == MQ_S8 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (int rc = encode_pages(&kmap, c->k, KIND, c, c->k_stride, F::kBox, box_rows, swizzle, what)) return rc;
  if (int rc = encode_pages(&vmap, c->v, KIND, c, c->v_stride, F::kBox, box_rows, swizzle, what)) return rc;
  p.parts = parts_at(workspace, ctas, kFewRows);
  static size_t configured[64] = {};
  auto kern = attn_few_kernel<D, KIND>;
  if (int rc = ensure_smem(kern, F::kSmem, configured, what)) return rc;
  if (int rc = launch_overlapped(kern, dim3(ctas), dim3(kFewThreads), F::kSmem, stream, what, kmap, vmap, p)) return rc;
  JoinParams j{p.shape, p.o, p.parts, kFewRows};
  return launch_overlapped(attn_join_kernel<D, kFewRows>, dim3(ctas, kFewRows / kJoinWarps), dim3(32 * kJoinWarps), 0, stream, what, j);
}

}  // namespace paged
}  // namespace mq
