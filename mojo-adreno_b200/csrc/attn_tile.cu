// Attention of new tokens over a paged cache, for sequences with more than 16 rows per kv head: 256 rows of an item on one SM's
// tensor core (see attn.cu for the operator, paged.cuh for items and shares).
//
//  * Two accumulators of 128 rows. A step is 64 keys: S = Q K^T (M = 128 rows, N = 64) lands in one of two TMEM buffers, a
//    thread of the accumulator's softmax warps reads its row from there, writes the weights back over it as 16-bit values, and
//    they are the A operand of O += P V from TMEM, while the next scores are already made in the other buffer. O stays in TMEM, and
//    is rescaled there only when a row's maximum has grown by 2^8 since the last time. The weights have the cache's type (int8: fp16),
//    since an MMA's operands are of one: bf16 ones make an output's error 0.0021 where its own rounding is 0.0016 (8192 tokens).
//  * An item of more than 128 rows has a tile on each accumulator; a narrow one (drafted tokens) has half of every block's
//    keys on each, joined when it ends.
//  * V is used as it lies, [keys][dim], as an MN-major B operand: nothing is transposed.
//  * Warps 0-3 and 4-7: softmax and output of the two accumulators. Warp 8: walks through the items and copies keys and values, a
//    lane per page (or part of one) and 128 bytes of row. Warps 9 and 10: a thread each issues the MMAs of an accumulator. Warps
//    12 to 15: bring q, and stand between the copies and the MMAs: of an int8 cache they make fp16 of every block; of a 16-bit one
//    they take what is no number out of the values of the blocks that some row sees only in part, and say which keys had any.
//  * An int8 cache's scales meet the scores and weights in fp32 (attn.cu), three numbers per key and row from shared memory. In the
//    operands, as fp16(integer * scale / the largest of 32 keys), they would take less (2048 of 30,001 tokens: 1244 us, 1340 here;
//    2048 of 2048: 125, 119 here), but a ratio's rounding is common to all terms of a score, and a scale far above its neighbours'
//    takes their bits. Error beside the bf16 output's own rounding: 0.0012 so, 0.00015 here.
//  * One persistent CTA per SM, all of TMEM, equal shares of the blocks: causal or ragged, no SM waits for another.
//
// 8192 tokens, 32 heads on 8 of 128, bf16: 535-620 us, 0.9-1.03 PFLOP/s (0.53-0.61 of the measured burst, 0.63-0.72 of the
// sustained rate; power caps the clock). A step of both accumulators takes some 2000 cycles where its MMAs take 1280 and its
// exponentials 1024: what is left over is waiting between the two. Short calls are latency: 431 tokens 22 us; a traced
// run had 2.8 for the shares, 3.8 more until the first scores, 3.0 for one to four steps, 2.6 for the output, then the join.
#include "paged.cuh"

namespace mq {
namespace paged {

constexpr int kTileKeys = 128, kTileRows = 256;
constexpr int kTileThreads = 512, kAuxWarps = 4;
using TileGrain = Grain<kTileRows, kTileKeys, 2>;
// Registers of a thread at launch, of a softmax thread (half a row of scores is 64 of them) and of the others.
constexpr int kTileRegs = 128, kSoftmaxRegs = 152, kOtherRegs = 104;
static_assert(256 * kSoftmaxRegs + 256 * kOtherRegs <= kTileThreads * kTileRegs, "more registers than the block was launched with");
constexpr int kStageBytes = 2048;  // per softmax warp: 64 bytes of each of its rows on their way out

template <int D, int KIND>
struct Tile {
  static constexpr bool kS8 = KIND == MQ_S8;
  static constexpr int kBlock = kTileKeys * D * 2;          // of keys or values, as operands
  static constexpr int kSlots = kS8 ? 3 : 4;                // keys and values in turn
  static constexpr int kRaw = kS8 ? kTileKeys * D : 0;      // int8 as it was copied, two of them
  static constexpr int kQ = kTileRows * D * 2;
  // All of shared memory, since it takes all of TMEM: no other CTA that wants TMEM then fits beside it.
  static constexpr int kSmem = 220 * 1024;
  static_assert(kQ + kSlots * kBlock + 2 * kRaw + 8 * kStageBytes + 1024 <= kSmem, "shared memory");
};

// Row-major rows of 128 bytes, 128 of them to a 64-column part: where 16-byte chunk c of row r lies.
__device__ __forceinline__ int swizzled(int r, int c) { return (c >> 3) * 16384 + r * 128 + ((c ^ r) & 7) * 16; }

// The MN-major descriptor of a [keys][dim] block: 64 columns of 128 bytes, 8-key atoms 1024 bytes apart (stride
// offset), the next 64 columns 16 KB on (leading offset).
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFF) | (static_cast<uint64_t>(16384 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}
constexpr uint32_t idesc_16(int m, int n, bool bf, bool b_mn) {
  return umma_idesc_f16(m, n) | (bf ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// 32 columns, without the wait; tmem_loaded() stands between the wait and their use.
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_loaded(float (&v)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 16)
    asm volatile(""
                 : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]),
                   "+f"(v[i + 7]), "+f"(v[i + 8]), "+f"(v[i + 9]), "+f"(v[i + 10]), "+f"(v[i + 11]), "+f"(v[i + 12]),
                   "+f"(v[i + 13]), "+f"(v[i + 14]), "+f"(v[i + 15]));
}

// (x, y) = (x, y) * a + b, and (x, y) = (x, y) + (a, b): two fp32 operations of one instruction.
__device__ __forceinline__ void fma2(float &x, float &y, float ax, float ay, float bx, float by) {
  asm("{\n .reg .b64 p, q, r;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n mov.b64 r, {%4, %5};\n"
      " fma.rn.f32x2 p, p, q, r;\n mov.b64 {%0, %1}, p;\n}"
      : "+f"(x), "+f"(y)
      : "f"(ax), "f"(ay), "f"(bx), "f"(by));
}
__device__ __forceinline__ void add2(float &x, float &y, float ax, float ay) {
  asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n add.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
      : "+f"(x), "+f"(y)
      : "f"(ax), "f"(ay));
}
__device__ __forceinline__ void mul2(float &x, float &y, float ax, float ay) {
  asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n mul.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
      : "+f"(x), "+f"(y)
      : "f"(ax), "f"(ay));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D, int KIND>
__global__ void __launch_bounds__(kTileThreads, 1)
    attn_tile_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AttnParams p) {
  using T = Tile<D, KIND>;
  constexpr bool BF = KIND == MQ_BF16, S8 = T::kS8;
  constexpr int NS = T::kSlots, NF = S8 ? 2 : NS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *q_tile = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t *ring = q_tile + T::kQ, *raw = ring + NS * T::kBlock, *stages = raw + 2 * T::kRaw;
  __shared__ uint64_t full[NF], raw_empty[2], ready[NS], empty[NS], q_full[2], q_empty[2], drained[2], s_full[2][2], p_full[2][2], o_step[2], o_full[2], half_done, half_read, turn[2][4], factors_read[2];
  __shared__ uint32_t bad_keys[NS][4];
  __shared__ __align__(16) float scales[S8 ? 2 : 1][3][S8 ? kTileKeys : 1], row_factor[2][S8 ? kTileRows : 1];
  __shared__ ItemRing items;
  __shared__ float2 half_stats[128];
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 0) {
    for (int i = 0; i < NF; ++i) mbar_init(&full[i], 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&raw_empty[i], kAuxWarps);
      mbar_init(&o_step[i], 1);
      mbar_init(&o_full[i], 1);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[i][b], 1);
        mbar_init(&p_full[i][b], 4);
      }
      mbar_init(&q_full[i], kAuxWarps);
      mbar_init(&q_empty[i], 2);  // of both MMA threads, or twice of the one that used it
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&ready[i], kAuxWarps);
      mbar_init(&empty[i], 2);  // of both MMA threads
    }
    mbar_init(&drained[0], 1);
    mbar_init(&drained[1], 1);
    for (int i = 0; i < 8; ++i) mbar_init(&turn[i / 4][i % 4], 1);
    mbar_init(&half_done, 4);
    mbar_init(&half_read, 4);
    for (int i = 0; i < 2; ++i) mbar_init(&factors_read[i], 8);
    items.init(2 + kAuxWarps + 8);
    fence_mbar_init();
  }
  griddep_wait();  // (before TMEM is taken: the kernels before this one have returned theirs)
  if (warp == 9) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = tmem_slot;
  ShareScratch<kTileThreads> &scratch = *reinterpret_cast<ShareScratch<kTileThreads> *>(ring);  // (nothing has been copied yet)
  find_share<kTileThreads, TileGrain>(p.seqs, p.shape, scratch);
  const Share share = scratch.found;
  fence_proxy_async_smem();  // (copies into the ring come behind what was written there by ordinary stores)
  __syncthreads();           // (the ring is free again)
  if (blockIdx.x == 0 && tid == 0) p.parts.counts[0] = share.total, p.parts.counts[1] = share.parts;
  const bool works = static_cast<int>(blockIdx.x) < share.parts;
  const int group = p.shape.group;
  Item item;
  // A role whose wait gives up leaves; so do then those that wait for it.
  auto wait = [&](uint64_t *bar, uint32_t parity, int code) -> bool {
    if (wait_for(bar, parity)) return true;
    raise_status(code);
    return false;
  };
  auto warp_wait = [&](uint64_t *bar, uint32_t parity, int code) -> bool {
    return __all_sync(0xffffffffu, wait(bar, parity, code));
  };
  // The next item, by a whole warp; false behind the last.
  int k_item = 0;
  auto next_item = [&](int code) -> bool {
    if (!warp_wait(&items.full[k_item % kItems], (k_item / kItems) & 1, code)) return false;
    item = items.item[k_item % kItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(&items.empty[k_item % kItems]);
    ++k_item;
    return item.blocks > 0;
  };
  // Rows of an item's two tiles; whether some row of the item sees a block only in part.
  auto rows_of = [&](const Item &it) { return min(kTileRows, it.s.n * group - it.tile * kTileRows); };
  auto least_hi = [&](const Item &it) { return max(it.s.pos0 + over_group(p.shape, it.tile * kTileRows) + 1, 0); };
  auto most_lo = [&](const Item &it) {
    return p.shape.window ? max(0, it.s.pos0 + over_group(p.shape, it.tile * kTileRows + rows_of(it) - 1) + 1 - p.shape.window) : 0;
  };

  if (!works) {
  } else if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
  if (warp == 8) {
    if (lane == 0) {
      prefetch_tmap(&kmap);
      prefetch_tmap(&vmap);
    }
    constexpr int kBox = S8 ? D : 128, kBoxes = S8 ? 1 : D / 64;  // bytes of a row in a box, boxes of a row
    const int page = 1 << p.seqs.page_log2, box_rows = min(kTileKeys, page), per_block = kTileKeys / box_rows;
    Walk<TileGrain> walk;
    walk.start(p.shape, share);
    const Walk<TileGrain> begin = walk;
    uint32_t issued = 0;
    bool ok = true;
    while (ok) {
      if (!walk.next(p.seqs, p.shape, item)) item.blocks = 0;
      if (!items.put(k_item++, item)) {
        if (lane == 0) raise_status(kStatusAttnLoadWait);
        break;
      }
      if (item.blocks == 0) break;
      for (int i = 0; ok && i < item.blocks; ++i) {
        const int key0 = (item.block + i) * kTileKeys;
        // Boxes behind the sequence's end are not fetched: their table entries may be anything.
        const int live = max(0, min(per_block, (item.s.length - key0 + box_rows - 1) / box_rows));
        int id = p.seqs.pages;  // (outside the map: zeros)
        if (lane < live) {
          const int of = page_of(p.seqs, item.b, key0 + lane * box_rows);
          if (of >= 0) id = of;
        }
        for (int which = 0; which < 2; ++which) {
          const uint32_t slot = issued % NF, round = issued / NF;
          if (round > 0 && !warp_wait(S8 ? &raw_empty[slot] : &empty[slot], (round - 1) & 1, kStatusAttnLoadWait)) {
            ok = false;
            break;
          }
          uint8_t *dst = S8 ? raw + slot * T::kRaw : ring + slot * T::kBlock;
          if (lane == 0) mbar_expect_tx(&full[slot], live * box_rows * kBox * kBoxes);
          __syncwarp();
          const int part = lane / per_block, at = lane % per_block;  // (at most 8 x 2 boxes)
          const int of = __shfl_sync(0xffffffffu, id, at);
          if (part < kBoxes && at < live)
            asm volatile(
                "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                ::"r"(smem_u32(dst + part * 16384 + at * box_rows * kBox)), "l"(reinterpret_cast<uint64_t>(which ? &vmap : &kmap)),
                "r"(smem_u32(&full[slot])), "r"(part * 64), "r"((key0 + at * box_rows) & (page - 1)), "r"(item.head), "r"(of)
                : "memory");
          ++issued;
        }
      }
    }
    if (lane == 0) p.parts.cuts[blockIdx.x] = cut_at(begin, p.shape, share);
    // Leave no copy in flight.
    if (lane == 0)
      for (uint32_t i = issued > NF ? issued - NF : 0; i < issued; ++i) wait_for(&full[i % NF], (i / NF) & 1);
  } else if (warp == 9 || warp == 10) {
    {
      // A thread for each accumulator: what it waits for and what it commits takes as long as its MMAs, so one thread for both
      // left the tensor core idle half of the time.
      constexpr uint32_t qk = idesc_16(128, 64, BF, false), pv = idesc_16(128, D, BF, true);
      const int g = warp - 9;
      // Keys and values take the ring's slots in turn: where the next scores' keys are, and the next product's values.
      struct At {
        int slot;
        uint32_t phase;
        __device__ void next() {
          if ((slot += 2) >= NS) slot -= NS, phase ^= 1;
        }
      } at_k{0, 0}, at_v{1, 0};
      uint32_t p_phase = 0, q_phase[2] = {0, 0};  // p_phase: a bit for each buffer
      bool ok = true;
      // Descriptors' low words; the high ones are constant. 64 columns of a K-major operand are 16 KB apart, its 16-column
      // steps 32 bytes, 64 keys 8 KB; the 16-key steps of the values 2 KB.
      const uint32_t q_low = (smem_u32(q_tile) >> 4) & 0x3FFF, ring_low = (smem_u32(ring) >> 4) & 0x3FFF;
      const uint32_t s_tmem = tmem + g * 128, o_tmem = tmem + 256 + g * D;
      constexpr uint32_t kHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
      auto desc = [](uint32_t low) { return static_cast<uint64_t>(kHigh) << 32 | low; };
      auto await = [&](uint64_t *bar, uint32_t parity) {
        if (ok) ok = wait(bar, parity, kStatusAttnMmaWait);
        return ok;
      };
      while (next_item(kStatusAttnMmaWait)) {
        if (lane == 0) {
          // A step is 64 keys. An item of two tiles: both halves of each block for this one's rows. A narrow one: half g of
          // each block. Scores run two steps ahead of the values, in the two halves of the accumulator in turn.
          const bool narrow = rows_of(item) <= 128;
          const int q = narrow ? 0 : g, steps = narrow ? item.blocks : 2 * item.blocks;
          auto score = [&](int i) {
            const int half = narrow ? g : i & 1;
            if ((narrow || half == 0) && !await(&ready[at_k.slot], at_k.phase)) return;
            const uint32_t a = q_low + q * (T::kQ / 2 >> 4) + (1u << 16);
            const uint32_t b = ring_low + at_k.slot * (T::kBlock >> 4) + half * (8192 >> 4) + (1u << 16);
#pragma unroll
            for (int k = 0; k < D / 16; ++k)
              umma_f16(s_tmem + (i & 1) * 64, desc(a + (k / 4) * 1024 + 2 * (k % 4)), desc(b + (k / 4) * 1024 + 2 * (k % 4)), qk, k != 0);
            umma_commit(&s_full[g][i & 1]);
            if (narrow || half == 1) {
              umma_commit(&empty[at_k.slot]);
              at_k.next();
            }
            if (i == steps - 1) {
              umma_commit(&q_empty[q]);
              if (!narrow) umma_commit(&q_empty[q]);
            }
          };
          await(&q_full[q], q_phase[q]);
          q_phase[0] ^= 1;
          if (!narrow) q_phase[1] ^= 1;
          if (ok) score(0);
          if (ok && steps > 1) score(1);
#pragma unroll 1
          for (int i = 0; ok && i < steps; ++i) {
            const int half = narrow ? g : i & 1, buffer = i & 1;
            if (narrow || half == 0) await(&ready[at_v.slot], at_v.phase);
            if (!await(&p_full[g][buffer], p_phase >> buffer & 1)) break;
            p_phase ^= 1u << buffer;
            tc_fence_after();
            const uint32_t b = ring_low + at_v.slot * (T::kBlock >> 4) + half * (8192 >> 4) + (1024u << 16);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16_ts(o_tmem, s_tmem + buffer * 64 + k * 8, desc(b + k * 128), pv, i != 0 || k != 0);
            umma_commit(&o_step[g]);
            if (i == steps - 1) umma_commit(&o_full[g]);
            if (narrow || half == 1) {
              umma_commit(&empty[at_v.slot]);  // (before the next keys are waited for, which may need this slot)
              at_v.next();
            }
            if (i + 2 < steps) score(i + 2);
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
      }
      if (!ok && lane == 0) {  // what was issued ends before TMEM goes
        umma_commit(&drained[g]);
        wait_for(&drained[g], 0);
      }
    }
    __syncwarp();
  } else if (warp >= 12) {
    const int at = tid - 384;  // 0 .. 127
    uint32_t n = 0;
    int at_item = 0, q_uses[2] = {0, 0};
    bool ok = true;
    while (ok && next_item(kStatusAttnLoadWait)) {
      const int rows = rows_of(item), row0 = item.tile * kTileRows;
      auto q_row = [&](int row) {
        const int r = row0 + row, i = over_group(p.shape, r);
        return static_cast<const uint16_t *>(p.q) + static_cast<int64_t>(item.s.first + i) * p.q_token +
               static_cast<int64_t>(item.head * group + (r - i * group)) * p.q_head;
      };
      const int tiles = rows > 128 ? 2 : 1;
      // The rows' factors take the place of those of the item before last. q_empty does not say that both accumulators' softmax
      // warps are through with them: a narrow item's are read by both, and behind an item of one block and two tiles only the
      // first one's MMA thread has spoken.
      if (S8 && at_item >= 2) ok = warp_wait(&factors_read[at_item & 1], (at_item / 2 - 1) & 1, kStatusAttnLoadWait);
      for (int g = 0; ok && g < tiles; ++g) {
        uint8_t *dst = q_tile + g * (T::kQ / 2);
        if (q_uses[g] > 0) ok = warp_wait(&q_empty[g], (q_uses[g] - 1) & 1, kStatusAttnLoadWait);
        if (!ok) break;
        ++q_uses[g];
        if constexpr (S8) {
          const int r = at, row = g * 128 + r;
          const uint16_t *src = q_row(min(row, rows - 1));
          const bool f16 = p.q_dtype == MQ_F16;
          auto chunk = [&](int c) {
            return row < rows && 8 * c < p.o.dim ? *reinterpret_cast<const uint4 *>(src + 8 * c) : make_uint4(0, 0, 0, 0);
          };
          uint32_t big = 0;  // the largest |q|'s bits, of either half
#pragma unroll 8
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = chunk(c);
            big = __vmaxu2(__vmaxu2(big, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
          }
          const uint16_t top = static_cast<uint16_t>(max(big & 0xffff, big >> 16));
          const float most = f16 ? __half2float(__ushort_as_half(top)) : __uint_as_float(static_cast<uint32_t>(top) << 16);
          const uint32_t e2 = min(max(__float_as_uint(most) >> 23, 27u), 227u);
          const float down = __uint_as_float((254 - e2) << 23);
          row_factor[at_item & 1][row] = __uint_as_float(e2 << 23) * p.scale;
#pragma unroll 4
          for (int c = 0; c < D / 8; ++c) {
            const uint4 w = chunk(c);
            const uint32_t x[4] = {w.x, w.y, w.z, w.w};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = f16 ? __half22float2(*reinterpret_cast<const __half2 *>(&x[e]))
                                   : make_float2(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u));
              o[e] = pack_half2(f.x * down, f.y * down);
            }
            *reinterpret_cast<uint4 *>(dst + swizzled(r, c)) = make_uint4(o[0], o[1], o[2], o[3]);
          }
        } else {
          constexpr int kLanes = D / 8;  // of a row
          const int c = at % kLanes;
#pragma unroll 4
          for (int r = at / kLanes; r < 128; r += 128 / kLanes) {
            const int row = g * 128 + r;
            const bool real = row < rows && 8 * c < p.o.dim;
            const uint16_t *src = q_row(min(row, rows - 1)) + (real ? 8 * c : 0);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + swizzled(r, c))), "l"(src), "r"(real ? 16 : 0)
                         : "memory");
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
        }
      }
      if (!ok) break;
      for (int g = 0; g < tiles; ++g) {
        if (g + 1 < tiles)
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        else
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[g]);
      }
      ++at_item;

      const int part_hi = least_hi(item), part_lo = most_lo(item);
      for (int j = 0; ok && j < item.blocks; ++j) {
        const int key0 = (item.block + j) * kTileKeys;
        const int r = at, key = key0 + r;  // this thread's
        float sk = 0.f, sv = 0.f;
        if (S8 && key < item.s.length) {
          const int of = page_of(p.seqs, item.b, key), row = key & ((1 << p.seqs.page_log2) - 1);
          if (of >= 0) {
            sk = p.k_scale[of * p.ks_stride[0] + item.head * p.ks_stride[1] + row * p.ks_stride[2]];
            sv = p.v_scale[of * p.vs_stride[0] + item.head * p.vs_stride[1] + row * p.vs_stride[2]];
          }
        }
        const bool edge = key0 + kTileKeys > part_hi || key0 < part_lo;
        for (int which = 0; which < 2; ++which, ++n) {
          const int src = static_cast<int>(n % NF), slot = static_cast<int>(n % NS);
          ok = warp_wait(&full[src], (n / NF) & 1, kStatusAttnLoadWait);
          if (ok && S8 && n >= NS) ok = warp_wait(&empty[slot], (n / NS - 1) & 1, kStatusAttnLoadWait);
          if (!ok) break;
          uint8_t *dst = ring + slot * T::kBlock;
          if constexpr (S8) {
            const uint8_t *from = raw + src * T::kRaw;
            if (which == 0) {
              // (the softmax has read block n / 2 - 2's by now: the slot just waited for came behind its weights)
              float (&sc)[3][kTileKeys] = scales[(n >> 1) & 1];
              const float vs = sv < kLeastScale ? kLeastScale : sv;
              sc[0][r] = sk < INFINITY ? sk : NAN, sc[1][r] = lg2(vs), sc[2][r] = __frcp_rn(vs);
            }
            uint4 w[D / 16];
#pragma unroll
            for (int c = 0; c < D / 16; ++c)
              w[c] = *reinterpret_cast<const uint4 *>(from + (D == 128 ? r * 128 + ((c ^ r) & 7) * 16 : r * 64 + ((c ^ (r >> 1)) & 3) * 16));
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              const uint32_t x[4] = {w[c].x ^ 0x80808080u, w[c].y ^ 0x80808080u, w[c].z ^ 0x80808080u, w[c].w ^ 0x80808080u};
              uint32_t o[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) o[2 * e] = bytes_to_half2<0x4140>(x[e]), o[2 * e + 1] = bytes_to_half2<0x4342>(x[e]);
              *reinterpret_cast<uint4 *>(dst + swizzled(r, 2 * c)) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4 *>(dst + swizzled(r, 2 * c + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&raw_empty[src]);
          } else if (which == 1 && edge) {
            bool bad = false;
            const bool gone = key >= item.s.length;  // what lies there was never copied, or is another's
#pragma unroll 4
            for (int c = 0; c < D / 8; ++c) {
              uint4 *v = reinterpret_cast<uint4 *>(dst + swizzled(r, c));
              uint4 x = *v;
              const uint4 m = {not_finite2<BF>(x.x), not_finite2<BF>(x.y), not_finite2<BF>(x.z), not_finite2<BF>(x.w)};
              if (m.x | m.y | m.z | m.w) {
                bad = true;
                x.x &= ~m.x, x.y &= ~m.y, x.z &= ~m.z, x.w &= ~m.w;
                *v = x;
              }
            }
            const uint32_t bits = __ballot_sync(0xffffffffu, bad && !gone);
            if (lane == 0) bad_keys[slot][warp - 12] = bits;
            fence_proxy_async_smem();
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(&ready[slot]);
        }
      }
    }
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int g = warp / 4, r = tid % 128;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + g * 128, o_at = tmem + lanes + 256 + g * D;
    uint8_t *const stage = stages + warp * kStageBytes;
    uint32_t n0 = 0, s_phase = 0, o_steps = 0, half_phase = 0, turn_phase = g ^ 1;  // s_phase: a bit for each buffer; o_steps: products so far
    bool ok = true;
    while (ok && next_item(kStatusAttnSoftmaxWait)) {
      // An item of two tiles: each group has one, half a block a step. A narrow one: each group has half of every block, and
      // group 0 joins the two.
      const int rows = rows_of(item);
      const bool narrow = rows <= 128;
      const int row = (narrow ? 0 : g * 128) + r;
      const int index = item.tile * kTileRows + min(row, rows - 1), i = over_group(p.shape, index);
      const int hi = row < rows ? max(item.s.pos0 + i + 1, 0) : 0;
      const int lo = p.shape.window ? max(0, item.s.pos0 + i + 1 - p.shape.window) : 0;
      const int part_hi = least_hi(item), part_lo = most_lo(item);
      const bool idle = row - lane >= rows;  // no row of this warp is one: its weights may be anything
      float m = -INFINITY, l = 0.f;
      const int steps = narrow ? item.blocks : 2 * item.blocks;
      for (int step = 0; step < steps; ++step) {
        const int buffer = step & 1, half = narrow ? g : buffer;
        const uint32_t n = n0 + 2 * (narrow ? step : step >> 1);
        const int block0 = (item.block + (narrow ? step : step >> 1)) * kTileKeys, key0 = block0 + 64 * half;
        ok = warp_wait(&s_full[g][buffer], s_phase >> buffer & 1, kStatusAttnSoftmaxWait);
        if (!ok) break;
        s_phase ^= 1u << buffer;
        tc_fence_after();
        if (idle) {
          ok = warp_wait(&turn[g][warp & 3], turn_phase, kStatusAttnSoftmaxWait);
          if (!ok) break;
          turn_phase ^= 1;
          if (lane == 0) mbar_arrive(&turn[g ^ 1][warp & 3]), mbar_arrive(&p_full[g][buffer]);
          continue;
        }
        const uint32_t at = s_at + buffer * 64;
        float v[2][32];
        tmem_ld32_async(at, v[0]);
        tmem_ld32_async(at + 32, v[1]);
        tmem_wait_ld();
        tmem_loaded(v[0]);
        tmem_loaded(v[1]);
        const bool edge = block0 + kTileKeys > part_hi || block0 < part_lo;
        // int8: a score's log2, with the values' (attn.cu), from the row's factor and the keys' and values' scales. A 16-bit cache's is
        // p.scale times it, which the maximum and the exponents apply.
        if constexpr (S8) {
          const float factor = row_factor[(k_item - 1) & 1][row];
          const float (&sc)[3][kTileKeys] = scales[(n >> 1) & 1];
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              float4 k4 = *reinterpret_cast<const float4 *>(&sc[0][64 * half + 32 * c + e]);
              const float4 l4 = *reinterpret_cast<const float4 *>(&sc[1][64 * half + 32 * c + e]);
              mul2(k4.x, k4.y, factor, factor);
              mul2(k4.z, k4.w, factor, factor);
              fma2(v[c][e], v[c][e + 1], k4.x, k4.y, l4.x, l4.y);
              fma2(v[c][e + 2], v[c][e + 3], k4.z, k4.w, l4.z, l4.w);
            }
        }
        if (edge) {
          // The columns that this row sees, a bit each: from lo - key0 up to hi - key0.
          uint32_t sees[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int to = min(max(hi - key0 - 32 * c, 0), 32), from = min(max(lo - key0 - 32 * c, 0), 32);
            sees[c] = (to == 32 ? ~0u : (1u << to) - 1) & ~(from == 32 ? ~0u : (1u << from) - 1);
          }
          if constexpr (!S8) {
            const int slot = static_cast<int>((n + 1) % NS);
            ok = warp_wait(&ready[slot], ((n + 1) / NS) & 1, kStatusAttnSoftmaxWait);
            if (!ok) break;
            const uint32_t bad = (bad_keys[slot][2 * half] & sees[0]) | (bad_keys[slot][2 * half + 1] & sees[1]);
            if (bad) l = NAN;  // (a row that sees a value that is no number ends as NaN)
          }
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(sees[c] >> e & 1)) v[c][e] = -INFINITY;
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float *x = &v[c / 2][16 * (c & 1)];
          top[c] = fmaxf(x[0], x[1]);
#pragma unroll
          for (int e = 2; e < 16; e += 2) top[c] = max3(top[c], x[e], x[e + 1]);
        }
        const float most = max3(fmaxf(top[0], top[1]), top[2], top[3]) * (S8 ? 1.f : p.scale);
        const bool grows = most > m + 8.f;
        if (__any_sync(0xffffffffu, grows)) {
          const float next = grows ? most : m;
          const float a = m == next ? 1.f : ex2(m - next);
          l *= a;
          m = next;
          if (step > 0) {
            // Behind the product of the step before. (That of the one before it was done when these scores came, so the parity
            // is this one's.)
            ok = warp_wait(&o_step[g], (o_steps + step - 1) & 1, kStatusAttnSoftmaxWait);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              float o[16];
              tmem_ld16(o_at + c, o);
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * a);
              tmem_st16(o_at + c, w);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : -m;
        // The exponentials of the two warps that share a scheduler take turns, half a step apart: side by side they would also
        // wait for their scores side by side (8192 tokens: 541 us without turns, 548 with whole ones, 536 with halves).
        ok = warp_wait(&turn[g][warp & 3], turn_phase, kStatusAttnSoftmaxWait);
        if (!ok) break;
        turn_phase ^= 1;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t w[16];
          float part[2] = {0.f, 0.f};
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            if (S8)
              add2(v[c][e], v[c][e + 1], ref, ref);
            else
              fma2(v[c][e], v[c][e + 1], p.scale, p.scale, ref, ref);
            const float a = ex2(v[c][e]), b = ex2(v[c][e + 1]);
            w[e / 2] = pack16<BF>(a, b);
            if constexpr (S8) {
              const float2 iv = *reinterpret_cast<const float2 *>(&scales[(n >> 1) & 1][2][64 * half + 32 * c + e]);
              if (edge)  // (a key that the row does not see may have any scale)
                add2(part[0], part[1], a == 0.f ? 0.f : a * iv.x, b == 0.f ? 0.f : b * iv.y);
              else
                part[0] = fmaf(a, iv.x, part[0]), part[1] = fmaf(b, iv.y, part[1]);
            } else if (BF) {  // as they were rounded: the roundings cancel where one key has most of the weight
              add2(part[0], part[1], __uint_as_float(w[e / 2] << 16), __uint_as_float(w[e / 2] & 0xffff0000u));
            } else {
              add2(part[0], part[1], a, b);
            }
          }
          sum[0] += part[0], sum[1] += part[1];
          tmem_st16(at + 16 * c, w);
          if (c == 0 && lane == 0) mbar_arrive(&turn[g ^ 1][warp & 3]);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g][buffer]);
        l += sum[0] + sum[1];
      }
      if (!ok) break;
      n0 += 2 * item.blocks;
      o_steps += steps;
      if (S8) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&factors_read[(k_item - 1) & 1]);
      }
      if (narrow && g == 1) {
        half_stats[r] = make_float2(m, l);
        __syncwarp();
        if (lane == 0) mbar_arrive(&half_done);
        ok = warp_wait(&half_read, half_phase, kStatusAttnSoftmaxWait);  // then this accumulator is free again
        half_phase ^= 1;
        continue;
      }
      const uint32_t done = (k_item - 1) & 1;
      ok = warp_wait(&o_full[g], done, kStatusAttnSoftmaxWait);
      if (ok && narrow) {
        ok = warp_wait(&half_done, half_phase, kStatusAttnSoftmaxWait) && warp_wait(&o_full[1], done, kStatusAttnSoftmaxWait);
        half_phase ^= 1;
      }
      if (!ok) break;
      tc_fence_after();
      float a0 = 1.f, a1 = 0.f;
      if (narrow) {
        const float2 other = half_stats[r];
        const float most = fmaxf(m, other.x);
        a0 = m == most ? 1.f : ex2(m - most), a1 = other.x == most ? 1.f : ex2(other.x - most);
        l = l * a0 + other.y * a1;
        m = most;
      }
      const bool goes_on = item.before > 0, whole = !goes_on && item.blocks == item.whole;
      if (whole) {
        const float inv = inverse_sum(l);
        a0 *= inv, a1 *= inv;
      }
      const int64_t part = (2 * static_cast<int64_t>(blockIdx.x) + (goes_on ? 0 : 1)) * kTileRows + row;
      if (!whole && row < rows) p.parts.stats[part] = make_float2(m, l);
      // 64 bytes of each of the warp's rows at a time: through shared memory, so that eight rows leave with one store
      // instead of each lane's own (six times the cycles).
      const int64_t out_at = static_cast<int64_t>(item.s.first + i) * p.o.token_stride +
                             static_cast<int64_t>(item.head * group + (index - i * group)) * p.o.head_stride;
      char *const base = whole ? static_cast<char *>(p.o.out) : reinterpret_cast<char *>(p.parts.sums);
      const int64_t mine = whole ? 2 * out_at : 4 * part * D;
      const int pieces = whole ? (p.o.dim + 31) / 32 : D / 16, width = whole ? 2 * p.o.dim : 4 * D;
#pragma unroll 1
      for (int c = 0; c < pieces; ++c) {
        uint4 w[4];
        uint32_t *words = reinterpret_cast<uint32_t *>(w);
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // 16 columns a time: 8 words of a 16-bit row, or all 16 of a part's
          if (half == 1 && !whole) break;
          const int col = whole ? 32 * c + 16 * half : 16 * c;
          float o[16];
          tmem_ld16(o_at + col, o);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] *= a0;
          if (narrow) {
            float x[16];
            tmem_ld16(o_at + D + col, x);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] += x[e] * a1;
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              words[8 * half + e] = p.o.dtype == MQ_F16 ? pack16<false>(o[2 * e], o[2 * e + 1]) : pack16<true>(o[2 * e], o[2 * e + 1]);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) words[e] = __float_as_uint(o[e]);
          }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 4; ++u) *reinterpret_cast<uint4 *>(stage + lane * 64 + ((u ^ (lane >> 1)) & 3) * 16) = w[u];
        __syncwarp();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const int from = it * 8 + lane / 4, u = lane % 4;
          const int64_t to = __shfl_sync(0xffffffffu, mine, from) + 64 * c + 16 * u;
          if (row - lane + from < rows && 64 * c + 16 * u < width)
            *reinterpret_cast<uint4 *>(base + to) = *reinterpret_cast<const uint4 *>(stage + from * 64 + ((u ^ (from >> 1)) & 3) * 16);
        }
      }
      tc_fence_before();
      if (narrow) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&half_read);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int D, int KIND>
int launch_tile(const mq_kv_pages *c, AttnParams p, int ctas, void *workspace, cudaStream_t stream, const char *what) {
  using T = Tile<D, KIND>;
  CUtensorMap kmap, vmap;
  const int box_rows = std::min(kTileKeys, c->page), box = T::kS8 ? D : 128;
  const CUtensorMapSwizzle swizzle = box == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (int rc = encode_pages(&kmap, c->k, c->dtype, c, c->k_stride, box, box_rows, swizzle, what)) return rc;
  if (int rc = encode_pages(&vmap, c->v, c->dtype, c, c->v_stride, box, box_rows, swizzle, what)) return rc;
  p.parts = parts_at(workspace, ctas, kTileRows);
  static size_t configured[64] = {};
  auto kern = attn_tile_kernel<D, KIND>;
  if (int rc = ensure_smem(kern, T::kSmem, configured, what)) return rc;
  // The kernel deals its registers out anew, which waits for good where a block has fewer of them.
  static const int regs = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
  }();
  MQ_REQUIRE(regs == kTileRegs, MQ_ECUDA, "%s: the kernel was built with %d registers, not %d", what, regs, kTileRegs);
  if (int rc = launch_overlapped(kern, dim3(ctas), dim3(kTileThreads), T::kSmem, stream, what, kmap, vmap, p)) return rc;
  JoinParams j{p.shape, p.o, p.parts, kTileRows};
  return launch_overlapped(attn_join_kernel<D, kTileRows>, dim3(ctas, kTileRows / kJoinWarps), dim3(32 * kJoinWarps), 0, stream, what, j);
}

// The rows of a kv head above which a sequence goes to the tensor core's tiles.
constexpr int kRowsForTiles = kFewRows;

struct Plan {
  int few_ctas, tile_ctas;  // 0 without that launch
  int d, most_rows;
  size_t bytes;
};
// Which launches a call needs: sequences may have from one to max_new new tokens.
inline int plan_for(Plan *plan, const mq_kv_pages *c, int64_t heads, int64_t batch, int64_t tokens, int64_t max_new, int starts,
                    int sms, const char *what) {
  const int64_t group = heads / c->heads;
  MQ_REQUIRE(tokens * group < (1LL << 31) - 512, MQ_EUNSUPPORTED, "%s: too many rows", what);
  int64_t most = starts ? std::min(tokens, max_new > 0 ? max_new : tokens) : 1;
  plan->most_rows = static_cast<int>(most * group);
  plan->d = c->dim <= 64 ? 64 : 128;
  // One sequence may have all the tokens. And where sequences have some drafted tokens each, a launch for those that may have one
  // or two costs more than they do among the others. Without it and with it, us: 16 sequences of 5 tokens, 8 heads to a kv head,
  // up to 4100 positions: 34.7 and 39.3; 64 of 1 to 8 tokens: 85.5 and 97.7; 64 of which 16 have 13 and the others one, up to 8000:
  // 132 and 138. From int8 the tiles are slower for single tokens (the last: 187 and 145; of 16 sequences 65 and 66), so more than
  // 16 sequences go there only where at most a quarter can have few rows, by their mean and the most that one may have (64 of 5
  // tokens: 122 and 127; but of 1 to 8, which are so many by that: 122 and, as it is, 127).
  const int64_t rows = tokens * group;
  const bool drafts = plan->most_rows > kRowsForTiles && plan->most_rows <= 128 && rows >= 2 * kRowsForTiles * batch;
  const bool singles = c->dtype == MQ_S8 && batch > 16 && 4 * (plan->most_rows * batch - rows) > (plan->most_rows - kRowsForTiles) * batch;
  const bool few = group <= kRowsForTiles && !(batch == 1 && most == tokens && rows > kRowsForTiles) && !(drafts && !singles);
  const bool tile = plan->most_rows > kRowsForTiles || !few;
  plan->few_ctas = !few ? 0 : sms * (plan->d == 128 ? 2 : 3);
  plan->tile_ctas = tile ? sms : 0;
  plan->bytes = 0;
  if (few) plan->bytes = parts_bytes(plan->few_ctas, kFewRows, plan->d);
  if (tile) plan->bytes = std::max(plan->bytes, parts_bytes(sms, kTileRows, plan->d));
  return MQ_OK;
}

template <int D, int KIND>
int launch_attention(const Plan &plan, const mq_kv_pages *c, AttnParams p, void *workspace, cudaStream_t s, const char *what) {
  p.shape.rows_most = plan.most_rows;
  if (plan.few_ctas) {
    p.shape.rows_from = 0, p.shape.rows_to = kRowsForTiles;
    if (int rc = launch_few<D, KIND>(c, p, plan.few_ctas, workspace, s, what)) return rc;
  }
  if (plan.tile_ctas) {
    p.shape.rows_from = plan.few_ctas ? kRowsForTiles : 0, p.shape.rows_to = plan.most_rows;
    return launch_tile<D, KIND>(c, p, plan.tile_ctas, workspace, s, what);
  }
  return MQ_OK;
}

}  // namespace paged
}  // namespace mq

extern "C" size_t mq_paged_attention_workspace_size(const mq_kv_pages *cache, int64_t heads, int64_t batch, int64_t tokens,
                                                    int64_t max_new) {
  using namespace mq::paged;
  if (check_cache(cache, "mq_paged_attention_workspace_size") || heads <= 0 || heads % cache->heads || heads > 65535 || batch <= 0 ||
      tokens <= 0 || tokens >= (1LL << 30))
    return 0;
  mq::DeviceInfo dev;
  if (mq::device_info(&dev)) return 0;
  Plan plan;
  if (plan_for(&plan, cache, heads, batch, tokens, max_new, 1, dev.sms, "mq_paged_attention_workspace_size")) return 0;
  return plan.bytes;
}

extern "C" int mq_paged_attention(const void *q, int q_dtype, int64_t q_token, int64_t q_head, const mq_kv_pages *cache,
                                  const int32_t *table, int64_t ldt, int64_t width, const int32_t *lengths,
                                  const int32_t *starts, int64_t batch, int64_t tokens, int64_t heads, float scale, int64_t window,
                                  int64_t max_new, void *out, int64_t o_token, int64_t o_head, void *workspace,
                                  size_t workspace_bytes, void *stream) {
  using namespace mq::paged;
  const char *what = "mq_paged_attention";
  if (int rc = check_cache(cache, what)) return rc;
  AttnParams p{};
  if (int rc = check_seqs(&p.seqs, cache, table, ldt, width, lengths, starts, batch, tokens, what)) return rc;
  MQ_REQUIRE(heads > 0 && heads % cache->heads == 0, MQ_EINVAL, "%s: the heads must be a multiple of the cache's", what);
  MQ_REQUIRE(heads <= 65535, MQ_EUNSUPPORTED, "%s: too many heads", what);
  MQ_REQUIRE(q_dtype == MQ_F16 || q_dtype == MQ_BF16, MQ_EINVAL, "%s: q must be MQ_F16 or MQ_BF16", what);
  MQ_REQUIRE(cache->dtype == MQ_S8 || cache->dtype == q_dtype, MQ_EINVAL, "%s: q must have the type of a 16-bit cache", what);
  MQ_REQUIRE(scale > 0.f && scale < INFINITY, MQ_EINVAL, "%s: the scale must be positive and finite", what);
  MQ_REQUIRE(window >= 0 && max_new >= 0, MQ_EINVAL, "%s: bad window or number of new tokens", what);
  MQ_REQUIRE(window <= (1 << 30), MQ_EUNSUPPORTED, "%s: the window is above 2^30", what);
  if (batch == 0 || tokens == 0) return MQ_OK;
  if (int rc = check_rows(q, q_dtype, q_token, q_head, "q", what)) return rc;
  if (int rc = check_rows_out(out, q_dtype, tokens, heads, cache->dim, o_token, o_head, "out", what)) return rc;
  // (out may be q: an item's rows are read before any of them is written)
  const Area rows_q = area_of_rows(q, 2, tokens, heads, cache->dim, q_token, q_head);
  const Area rows_out = area_of_rows(out, 2, tokens, heads, cache->dim, o_token, o_head);
  if (!(out == q && (tokens == 1 || o_token == q_token) && (heads == 1 || o_head == q_head)))
    MQ_REQUIRE(!share_bytes(rows_q, rows_out), MQ_EINVAL, "%s: out shares memory with q, and is not q", what);
  Area held[4];
  const int nheld = areas_of(cache, held);
  for (int i = 0; i < nheld; ++i) MQ_REQUIRE(!share_bytes(held[i], rows_out), MQ_EINVAL, "%s: out shares memory with the pages", what);
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  Plan plan;
  if (int rc = plan_for(&plan, cache, heads, batch, tokens, max_new, starts != nullptr, dev.sms, what)) return rc;
  MQ_REQUIRE(workspace && mq::aligned(workspace, 16), MQ_EALIGN, "%s: the workspace must be 16-byte aligned", what);
  MQ_REQUIRE(workspace_bytes >= plan.bytes, MQ_EINVAL, "%s: the workspace is too small", what);
  const Area work = {static_cast<const char *>(workspace), static_cast<__int128>(plan.bytes), {0, 0, 0}, {1, 1, 1}};
  bool meets = share_bytes(rows_q, work) || share_bytes(rows_out, work);
  for (int i = 0; i < nheld; ++i) meets = meets || share_bytes(held[i], work);
  MQ_REQUIRE(!meets, MQ_EINVAL, "%s: the workspace shares memory with q, out or the pages", what);
  set_group(&p.shape, static_cast<int>(heads / cache->heads));
  p.shape.kv_heads = cache->heads, p.shape.window = static_cast<int>(window);
  p.q = q, p.q_token = q_token, p.q_head = q_head, p.q_dtype = q_dtype;
  p.k_scale = cache->k_scale, p.v_scale = cache->v_scale;
  for (int i = 0; i < 3; ++i) p.ks_stride[i] = cache->ks_stride[i], p.vs_stride[i] = cache->vs_stride[i];
  p.o = Output{out, o_token, o_head, q_dtype, cache->dim};
  p.scale = scale * 1.44269504088896340736f;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool wide = plan.d == 128;
  if (cache->dtype == MQ_F16)
    return wide ? launch_attention<128, MQ_F16>(plan, cache, p, workspace, s, what) : launch_attention<64, MQ_F16>(plan, cache, p, workspace, s, what);
  if (cache->dtype == MQ_BF16)
    return wide ? launch_attention<128, MQ_BF16>(plan, cache, p, workspace, s, what) : launch_attention<64, MQ_BF16>(plan, cache, p, workspace, s, what);
  return wide ? launch_attention<128, MQ_S8>(plan, cache, p, workspace, s, what) : launch_attention<64, MQ_S8>(plan, cache, p, workspace, s, what);
}
