// Beam search's selection over beams x vocabulary, and the states that follow their beams
// (mq_beam_select, mq_beam_reorder).
//
// Candidate (beam i, token v) of a request scores c = score[i] + (logit[i][v] - lse[i]) with
// lse = log(sum exp(logit[i])); of a finished beam the eos token scores score[i] and every other token
// -inf; so does every token of a beam whose score is -inf or NaN or whose lse is not finite. The `beams`
// largest are taken in order, the lowest flat index i * vocab + v among equal ones.
//
// beam_scan_kernel reads every logit once: `splits` CTAs per row, each thread keeps a running maximum and
// sum of exponentials, the CTA the best kp = beams + 1 (logit, token) pairs of its part. Within a row the
// score grows with the logit, so no other token can be among the `beams` best -- except where rounding
// gives unequal logits equal scores; the pair beyond the `beams` best shows whether that can matter.
// beam_merge_kernel, one CTA per request, joins the sums, scores the kept pairs and picks the best.
//
// Many rows: 64x8x128256 57 us in fp32 (4.6 TB/s), 57 in fp16 (2.3 TB/s), 58 in bf16; of that the merge is 5. Neither the bytes nor
// the issue slots bound it (14 instructions per logit, 0.54 issued per cycle and scheduler): of the seven warps of a
// scheduler most wait at the barrier of their chunk (a quarter of the stalls, a third in fp16) or for the
// instruction before (a quarter). One request (1x4x151669): 13.6 us in a graph, latency: some 5 for a chunk, 5.5 for the merge, the
// launches. The states' reordering moves 6.5 TB/s (64x8 states of 2 x 8 x 1001 x 64 fp16, five beams of eight
// moving: 161 us, the copy bandwidth).
#include <algorithm>
#include <cmath>
#include <memory>
#include <new>

#include "common.cuh"

namespace mq {
namespace beam {

constexpr int kThreads = 256;
constexpr int kMaxBeams = 32;
constexpr int kMaxLists = 256;  // (beam, split) lists of a request: one per thread of the merge
constexpr int kVecs = 4;        // 16-byte vectors per thread and chunk
constexpr int kScan = 128, kScanCtas = 7;  // threads of a scan CTA, CTAs per SM
constexpr int kChunkBytes = kScan * kVecs * 16;
constexpr int kFresh = 1280;    // pairs that may wait to be merged into the list: at least (kMaxBeams + 1) * 32
constexpr int kStages = 2;      // chunks on their way into shared memory: 16 KB for each of the CTAs of an SM
// So many CTAs fit in an SM's shared memory: their static and dynamic part, and 1 KB that the system takes.
static_assert(kScanCtas * (1024 + kStages * kChunkBytes + (2 * (kMaxBeams + 1) + kFresh + kScan) * 8 + 128) <= 228 * 1024,
              "the scan plans with more CTAs than run at once");
constexpr float kNegInf = -INFINITY, kLowest = -3.402823466e38f, kLog2e = 1.44269504088896340736f;

// (Counted in fp32 chunks for every type, so that the workspace's size does not depend on it.)
// As many CTAs as run at once (a few more start a second wave: 32x4x151669 fp32 8 splits 28.1 us, 9 36.2; 16x4x50257 16 splits
// 15.6 us, 18 18.5); at most one list per thread of the merge.
__host__ __device__ constexpr int splits_for(int64_t rows, int beams, int64_t vocab) {
  const int64_t chunks = (vocab * 4 + kChunkBytes - 1) / kChunkBytes;
  int64_t s = 148 * kScanCtas / rows;
  if (s > kMaxLists / beams) s = kMaxLists / beams;
  if (s > chunks) s = chunks;
  return s < 1 ? 1 : static_cast<int>(s);
}

// What the CTAs leave for the merge: the largest logit and the sum relative to it each (NaN where a logit is NaN
// or +infinity), then kp keys each, best first, 0 = none.
struct Parts {
  float2 *sums;    // [rows * splits]
  uint64_t *keys;  // [rows * splits][kp]
};
inline size_t parts_bytes(int64_t lists, int kp) { return static_cast<size_t>(lists) * (sizeof(float2) + 8 * kp); }
inline Parts parts_at(void *workspace, int64_t lists) {
  float2 *sums = static_cast<float2 *>(workspace);
  return {sums, reinterpret_cast<uint64_t *>(sums + lists)};
}

// Order-preserving bits of a float; -0 counts as +0.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
// Larger is better: the value, then the lower index.
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
  return static_cast<uint64_t>(order_of(v)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - static_cast<uint32_t>(key); }
__device__ __forceinline__ float value_of_key(uint64_t key) { return value_of(static_cast<uint32_t>(key >> 32)); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A sum s stands for s * 2^(unit(m)) with m the largest logit it has seen. unit(m) is the rounded fp32 product m log2 e, so
// that a term is one FMA, 2^(v log2 e - unit(m)), and the unit's rounding error does not enter the result, being in the
// term and in the unit. It is in the term as a factor, though, of 2^128 and more where m is some 1e10 (a row masked with -1e10):
// above 1e6, where it is 2^(1/16) at most, terms are 2^((v - m) log2 e) and s stands for s * e^m.
__device__ __forceinline__ bool moderate(float m) { return fabsf(m) < 1e6f; }
__device__ __forceinline__ float unit_of(float m) { return __fmul_rn(m, kLog2e); }  // (never part of an FMA)
// What takes a sum from m to another m that is not smaller; 1 where they are equal.
__device__ __forceinline__ float rescale(float from, float to) {
  float e = __fsub_rn(unit_of(from), unit_of(to));
  if (__builtin_expect(!moderate(fmaxf(fabsf(from), fabsf(to))), 0))
    e = moderate(from) ? fmaf(-to, kLog2e, unit_of(from)) : moderate(to) ? fmaf(from, kLog2e, -unit_of(to)) : (from - to) * kLog2e;
  return exp2_fast(e);
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) { return v; }
template <>
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

struct ScanParams {
  const void *logits;
  const float *scores;
  const uint8_t *finished;
  Parts parts;
  int64_t ld;
  int beams, vocab, splits;
};

__device__ __forceinline__ bool live_beam(const float *scores, const uint8_t *finished, int64_t row) {
  return scores[row] > kNegInf && !(finished && finished[row]);
}

template <typename T>
__global__ void __launch_bounds__(kScan, kScanCtas) beam_scan_kernel(const ScanParams p) {
  constexpr int V = 16 / sizeof(T), U = kVecs, kElems = V * U;  // elements of a vector; vectors, elements per chunk
  constexpr int kChunk = kScan * kElems;
  extern __shared__ __align__(16) uint8_t slots[];   // kStages chunks
  __shared__ uint64_t full[kStages];
  __shared__ uint64_t list[2][kMaxBeams + 1];
  __shared__ uint64_t fresh[kFresh];
  __shared__ uint64_t best_of[kScan];
  __shared__ uint64_t raised;
  __shared__ int nfresh;
  __shared__ float red[2][kScan / 32];
  const int tid = threadIdx.x, kp = p.beams + 1;
  griddep_launch_dependents();
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_mbar_init();
    nfresh = 0;
  }
  __syncthreads();
  griddep_wait();
  const int64_t row = blockIdx.x / p.splits;
  const int split = blockIdx.x % p.splits;
  if (!live_beam(p.scores, p.finished, row)) return;
  const T *x = static_cast<const T *>(p.logits) + row * p.ld;
  // The row's 16-byte aligned vectors come in chunks; the elements before the first and after the last
  // (at most V - 1 each) are one more step of the first split's CTA.
  const int head = min(p.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int nvec = (p.vocab - head) / V, body_end = head + nvec * V, edges = head + p.vocab - body_end;
  const int chunks = (nvec + kScan * U - 1) / (kScan * U);
  const int c_begin = static_cast<int>(static_cast<int64_t>(chunks) * split / p.splits);
  const int c_end = static_cast<int>(static_cast<int64_t>(chunks) * (split + 1) / p.splits);
  const int c_last = c_end + (split == 0 && edges > 0);
  auto fetch = [&](int c) {  // by thread 0
    const int slot = (c - c_begin) % kStages;
    const uint32_t bytes = min(nvec - c * kScan * U, kScan * U) * 16;
    mbar_expect_tx(&full[slot], bytes);
    bulk_load(slots + slot * kChunkBytes, x + head + static_cast<int64_t>(c) * kChunk, bytes, &full[slot]);
  };
  if (tid == 0)
    for (int c = c_begin; c < min(c_end, c_begin + kStages); ++c) fetch(c);

  float m = kLowest, s = 0.f;  // the largest logit, the sum of exponentials relative to it
  int cur = 0, have = 0;
  int bound = 0;     // at least as many pairs as wait in `fresh`; the same in every thread
  uint64_t bar = 0;  // a pair is offered only above this key
  float bar_value = kNegInf;
  // Merges `fresh` into the list by counting, for each pair, the better ones. Called by the whole CTA, after
  // a barrier behind the last append; the next append comes behind a barrier too.
  auto merge = [&]() {
    const int n = have + nfresh, old = have;
    for (int i = tid; i < n; i += kScan) {
      const uint64_t key = i < old ? list[cur][i] : fresh[i - old];
      int rank = 0;
      for (int j = 0; j < old; ++j) rank += list[cur][j] > key;
      for (int j = 0; j < n - old; ++j) rank += fresh[j] > key;
      if (rank < kp) list[cur ^ 1][rank] = key;
    }
    __syncthreads();
    if (tid == 0) nfresh = 0;
    cur ^= 1;
    have = min(n, kp);
    if (have == kp) bar = list[cur][kp - 1], bar_value = value_of_key(bar);
  };
  bool arrived = true;  // false once a wait ran out: the rest counts as -inf
  for (int c = c_begin; c < c_last; ++c) {
    const bool edge = c == c_end;
    const int edge_col = tid < head ? tid : body_end + tid - head;
    const int slot = (c - c_begin) % kStages;
    float v[kElems];
    if (!edge && arrived && !mbar_wait(&full[slot], (c - c_begin) / kStages & 1)) {
      raise_status(kStatusBeamLoadWait);
      arrived = false;
      if (tid == 0)  // fetches no more; what is on its way lands before the CTA ends
        for (int d = c; d < min(c_end, c + kStages); ++d) mbar_wait(&full[(d - c_begin) % kStages], (d - c_begin) / kStages & 1);
    }
    const uint8_t *mine_at = slots + slot * kChunkBytes + tid * 16;
    auto take = [&](int u) {
      const uint4 q = *reinterpret_cast<const uint4 *>(mine_at + u * kScan * 16);
      const T *e = reinterpret_cast<const T *>(&q);
#pragma unroll
      for (int i = 0; i < V; ++i) v[u * V + i] = to_float(e[i]);
    };
    if (!edge && arrived && (c + 1) * kScan * U <= nvec) {  // a whole chunk
#pragma unroll
      for (int u = 0; u < U; ++u) take(u);
    } else {
#pragma unroll
      for (int i = 0; i < kElems; ++i) v[i] = kNegInf;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (!edge && arrived && (c * U + u) * kScan + tid < nvec) take(u);
    }
    if (edge && tid < edges) v[0] = to_float(x[edge_col]);
    float big = v[0];
#pragma unroll
    for (int i = 1; i < kElems; ++i) big = fmaxf(big, v[i]);
    if (big > m) {
      s *= rescale(m, big);
      m = big;
    }
    // A NaN or +infinity (m infinite: inf - inf) makes s NaN.
    if (moderate(m)) {
      const float unit = unit_of(m);
#pragma unroll
      for (int i = 0; i < kElems; ++i) s += exp2_fast(fmaf(v[i], kLog2e, -unit));
    } else {
#pragma unroll
      for (int i = 0; i < kElems; ++i) s += exp2_fast((v[i] - m) * kLog2e);
    }
    // The best pairs. A logit below the bar's is never offered, and after a few chunks hardly any thread has one
    // that is not: the keys are formed only there.
    auto key_at = [&](int i) -> uint64_t {
      if (edge) return i == 0 && tid < edges ? key_of(v[0], edge_col) : 0;
      const int g = (c * U + i / V) * kScan + tid;
      return g < nvec ? key_of(v[i], head + g * V + i % V) : 0;
    };
    const int offers = __syncthreads_count(big >= bar_value);
    if (tid == 0 && arrived && c + kStages < c_end) fetch(c + kStages);  // every thread has read this slot
    if (offers == 0) continue;
    bound += offers * kElems;
    uint64_t limit = bar;
    const bool full = bound > kFresh;
    if (full) {  // no room for all that might be offered: merge what waits, which raises the bar
      if (bound > offers * kElems) {
        merge();
        __syncthreads();
      }
      limit = bar;
      uint64_t mine = 0;
      if (big >= bar_value)
#pragma unroll
        for (int i = 0; i < kElems; ++i) mine = max(mine, key_at(i));
      if (__syncthreads_count(mine > bar) * kElems > kFresh) {
        // Still none (the first chunk, rising logits): kp threads' largest pairs are enough, no pair below the
        // smallest of those kp can be kept. Of the first 64 threads, which is quick and does for logits in no
        // order; else of all, so that at most kp * kElems pairs come in, whatever the order.
        best_of[tid] = mine > bar ? mine : 0;
        if (tid == 0) raised = bar;
        __syncthreads();
        for (int n = 64; n <= kScan; n *= kScan / 64) {
          if (tid < n && mine > bar) {
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += best_of[j] > mine;
            if (rank == kp - 1) raised = mine - 1;
          }
          __syncthreads();
          limit = raised;
          if (__syncthreads_count(mine > limit) * kElems <= kFresh) break;
        }
      }
    }
    const float limit_value = limit ? value_of_key(limit) : kNegInf;
    if (big >= limit_value) {
#pragma unroll
      for (int i = 0; i < kElems; ++i)
        if (v[i] >= limit_value) {
          const uint64_t key = key_at(i);
          if (key > limit) fresh[atomicAdd(&nfresh, 1)] = key;
        }
    }
    // Chunks 0, 1, 2, 4, 8 ..: with a bar at most half as old as the row, each chunk offers about kp pairs.
    const int done = c - c_begin;
    if (full || (done & (done - 1)) == 0) {
      __syncthreads();
      merge();
      __syncthreads();
      bound = 0;
    }
  }
  __syncthreads();
  merge();

  // Join the threads' sums, in one fixed order.
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (tid % 32 == 0) red[0][tid / 32] = top;
  __syncthreads();
  top = red[0][0];
  for (int w = 1; w < kScan / 32; ++w) top = fmaxf(top, red[0][w]);
  s *= rescale(m, top);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (tid % 32 == 0) red[1][tid / 32] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.f;
    for (int w = 0; w < kScan / 32; ++w) s += red[1][w];
    p.parts.sums[blockIdx.x] = make_float2(top, s);
  }
  uint64_t *keys = p.parts.keys + static_cast<int64_t>(blockIdx.x) * kp;
  if (tid < kp) keys[tid] = tid < have ? list[cur][tid] : 0;
}

template <typename T>
int scan_launch(const ScanParams &p, dim3 grid, cudaStream_t s, const char *what) {
  const size_t smem = kStages * kChunkBytes;
  static size_t configured[64] = {};
  if (int rc = ensure_smem(beam_scan_kernel<T>, smem, configured, what)) return rc;
  return launch_overlapped(beam_scan_kernel<T>, grid, dim3(kScan), smem, s, what, p);
}

struct MergeParams {
  const void *logits;
  const float *scores;
  const uint8_t *finished;
  Parts parts;
  float *next_scores;
  int32_t *tokens, *parents;
  uint8_t *next_finished;
  int64_t ld;
  int dtype, beams, vocab, splits, eos;
};

enum : int { kLive = 0, kFinished = 1, kDead = 2 };

__device__ __forceinline__ float read_logit(const MergeParams &p, int64_t row, int v) {
  const int64_t at = row * p.ld + v;
  if (p.dtype == MQ_F32) return static_cast<const float *>(p.logits)[at];
  if (p.dtype == MQ_F16) return __half2float(static_cast<const __half *>(p.logits)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p.logits)[at]);
}

// The next value of the logits' type below v (finite, or -inf): its bit pattern one step down.
__device__ __forceinline__ float next_below(float v, int dtype) {
  if (!(v > kNegInf)) return kNegInf;
  if (dtype == MQ_F32) {
    const uint32_t b = __float_as_uint(v);
    return __uint_as_float(v > 0.f ? b - 1 : v < 0.f ? b + 1 : 0x80000001u);
  }
  const uint16_t b = dtype == MQ_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
  const uint16_t d = v > 0.f ? b - 1 : v < 0.f ? b + 1 : 0x8001;
  return dtype == MQ_F16 ? __half2float(__ushort_as_half(d)) : __bfloat162float(__ushort_as_bfloat16(d));
}

__device__ __forceinline__ float score_of(float score, float logit, float lse) {
  const float c = score + (logit - lse);
  return c == c ? c : kNegInf;
}

// One warp takes the best head of the sorted lists `count` times: a lane has lists lane, lane + 32 .. (N of them).
template <int N>
__device__ __forceinline__ void take_best(const uint64_t *cand, int lists, int kp, int count, int lane, uint64_t *chosen) {
  uint64_t head[N], best = 0;
  int at[N];  // where each list's head is
#pragma unroll
  for (int n = 0; n < N; ++n) {
    at[n] = (lane + 32 * n) * kp;
    head[n] = lane + 32 * n < lists ? cand[at[n]] : 0;
    best = max(best, head[n]);
  }
  for (int k = 0; k < count; ++k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(best >> 32));
    const bool in = static_cast<uint32_t>(best >> 32) == hi;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, in ? static_cast<uint32_t>(best) : 0u);
    if (in && static_cast<uint32_t>(best) == lo) {  // keys are unique: one lane, one of its lists
      chosen[k] = best;
      int list = 0, next_at = 0;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (head[n] == best) list = n, next_at = at[n] + 1;
      const uint64_t next = next_at < (lane + 32 * list + 1) * kp ? cand[next_at] : 0;
      best = 0;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (n == list) head[n] = next, at[n] = next_at;
        best = max(best, head[n]);
      }
    }
  }
}

// One CTA per request. Dynamic shared memory: kp keys per (beam, split) list.
__global__ void __launch_bounds__(kThreads) beam_merge_kernel(const MergeParams p) {
  extern __shared__ uint64_t cand[];
  __shared__ float2 sums[kMaxLists];
  __shared__ float lse[kMaxBeams], score[kMaxBeams];
  __shared__ int kind[kMaxBeams];
  __shared__ uint64_t chosen[kMaxBeams];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, kp = p.beams + 1, lists = p.beams * p.splits;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.beams;
  const uint64_t *keys = p.parts.keys + row0 * p.splits * kp;

  // Everything is fetched at once; the lists of beams that are not live hold nothing and are replaced below.
  for (int e = tid; e < lists * kp; e += kThreads) cand[e] = keys[e];
  if (tid < lists) sums[tid] = p.parts.sums[row0 * p.splits + tid];
  if (tid < p.beams) {
    const float sc = p.scores[row0 + tid];
    score[tid] = sc == sc ? sc : kNegInf;
    kind[tid] = p.finished && p.finished[row0 + tid] ? kFinished : sc > kNegInf ? kLive : kDead;
  }
  __syncthreads();
  for (int i = warp; i < p.beams; i += kThreads / 32) {
    if (kind[i] != kLive) continue;
    float top = kLowest, total = 0.f;
    for (int j = lane; j < p.splits; j += 32) top = fmaxf(top, sums[i * p.splits + j].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    for (int j = lane; j < p.splits; j += 32) total += sums[i * p.splits + j].y * rescale(sums[i * p.splits + j].x, top);
#pragma unroll
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) {
      if (total != total) raise_status(kStatusBeamNonFinite);
      total = static_cast<float>(moderate(top) ? (unit_of(top) + log2(static_cast<double>(total))) / static_cast<double>(kLog2e)
                                               : top + log(static_cast<double>(total)));
      lse[i] = total;
      if (!(fabsf(total) < INFINITY)) kind[i] = kDead;
    }
  }
  __syncthreads();
  uint64_t last = 0;  // the logit key that ends list `tid` if it is full
  int equal = 0;      // pairs of that logit at the list's end
  if (tid < lists && kind[tid / p.splits] == kLive) {
    last = cand[tid * kp + kp - 1];
    do ++equal;
    while (equal < kp && cand[tid * kp + kp - 1 - equal] >> 32 == last >> 32);
  }
  __syncthreads();
  // e / kp and l / splits by multiplication: exact for e < kMaxLists * kp, l < kMaxLists.
  const uint32_t per_kp = ((1u << 22) + kp - 1) / kp, per_split = ((1u << 16) + p.splits - 1) / p.splits;
  for (int e = tid; e < lists * kp; e += kThreads) {  // (logit, token) -> (score, flat index)
    const int l = e * per_kp >> 22, j = e - l * kp, i = l * per_split >> 16;
    const uint32_t flat0 = static_cast<uint32_t>(i) * p.vocab;
    uint64_t key = 0;
    if (kind[i] == kLive) {
      key = cand[e];
      if (key) key = key_of(score_of(score[i], value_of_key(key), lse[i]), flat0 + index_of(key));
    } else if (l == i * p.splits && j < p.vocab) {
      // eos first if it scores, then the others from token 0 on, all -inf
      const int at = kind[i] == kFinished ? p.eos : p.vocab;
      key = j == 0 && at < p.vocab ? key_of(score[i], flat0 + at)
                                   : key_of(kNegInf, flat0 + (at == p.vocab ? j : j - 1 < at ? j - 1 : j));
    }
    cand[e] = key;
  }
  __syncthreads();
  bool inverted = false;
  for (int e = tid; e < lists * kp - 1; e += kThreads) {
    const int l = e * per_kp >> 22;
    inverted |= e - l * kp < kp - 1 && cand[e] < cand[e + 1];
  }
  // The lists are in order of their logits; where rounding made scores equal, the index decides.
  if (__syncthreads_or(inverted) && tid < lists) {
    uint64_t *own = cand + tid * kp;
    for (int j = 1; j < kp; ++j) {
      const uint64_t key = own[j];
      int at = j;
      for (; at > 0 && own[at - 1] < key; --at) own[at] = own[at - 1];
      if (at < j) own[at] = key;
    }
  }
  __syncthreads();
  if (warp == 0) {
    if (lists <= 32)
      take_best<1>(cand, lists, kp, p.beams, lane, chosen);
    else
      take_best<kMaxLists / 32>(cand, lists, kp, p.beams, lane, chosen);
  }
  __syncthreads();

  // Unequal logits with equal scores: a token that was not kept could tie with the last chosen one and have a lower
  // index where a full list's last pair ties with it, and so does the next lower logit, or a pair of the list with
  // a larger logit (the token may have the last pair's logit, and an index above that pair's but below the other's).
  const uint32_t edge = static_cast<uint32_t>(chosen[p.beams - 1] >> 32);
  bool open = false;
  if (last) {
    const int i = tid / p.splits;
    const float l = value_of_key(last);
    open = order_of(score_of(score[i], l, lse[i])) == edge &&
           ((equal < kp && static_cast<uint32_t>(cand[tid * kp + kp - 1 - equal] >> 32) == edge) ||
            order_of(score_of(score[i], next_below(l, p.dtype), lse[i])) == edge);
  }
  if (__syncthreads_or(open)) {
    // Take the ties from the logits themselves, in the order of their flat index.
    __shared__ int warp_count[kThreads / 32];
    int k = 0;
    while (static_cast<uint32_t>(chosen[k] >> 32) != edge) ++k;  // the ones above the ties stay
    __syncthreads();
    for (int i = 0; i < p.beams && k < p.beams; ++i) {
      for (int v0 = 0; v0 < p.vocab && k < p.beams; v0 += kThreads) {
        const int v = v0 + tid;
        bool tie = false;
        if (v < p.vocab) {
          float c = kNegInf;
          if (kind[i] == kLive)
            c = score_of(score[i], read_logit(p, row0 + i, v), lse[i]);
          else if (kind[i] == kFinished && v == p.eos)
            c = score[i];
          tie = order_of(c) == edge;
        }
        const unsigned vote = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) warp_count[warp] = __popc(vote);
        __syncthreads();
        int at = k, all = 0;
        for (int w = 0; w < kThreads / 32; ++w) {
          if (w < warp) at += warp_count[w];
          all += warp_count[w];
        }
        at += __popc(vote & ((1u << lane) - 1));
        if (tie && at < p.beams) chosen[at] = static_cast<uint64_t>(edge) << 32 | (0xFFFFFFFFu - (static_cast<uint32_t>(i) * p.vocab + v));
        k = min(p.beams, k + all);
        __syncthreads();
      }
    }
  }
  if (tid < p.beams) {
    const uint32_t flat = index_of(chosen[tid]);
    const int parent = static_cast<int>(flat / static_cast<uint32_t>(p.vocab)), token = static_cast<int>(flat % static_cast<uint32_t>(p.vocab));
    p.next_scores[row0 + tid] = value_of_key(chosen[tid]);
    p.parents[row0 + tid] = parent;
    p.tokens[row0 + tid] = token;
    if (p.next_finished) p.next_finished[row0 + tid] = kind[parent] == kFinished || token == p.eos;
  }
}

// ---- states ---------------------------------------------------------------------------------------

constexpr int kMaxStates = 64;  // tensors of one launch
struct ReorderParams {
  void *states[kMaxStates];
  const int32_t *parents;
  int64_t row_stride;               // bytes from one beam's state to the next
  int64_t outer_stride[3];          // bytes; outer dimensions, the last one fastest
  uint32_t outer1, outer2;          // sizes of the last two outer dimensions
  uint32_t vecs;                    // vectors of the contiguous inner part
  int64_t items;                    // vectors of one beam's state
  int beams;
};

// One dimension of a state's layout: bytes from one index to the next, indices.
struct Dim {
  int64_t stride, size;
};

// Whether two states of one layout, `delta` bytes apart, share a byte: some difference of their positions,
// sum_d i_d stride_d with |i_d| < size_d, lies within inner_bytes of delta. `dims` goes from the largest
// stride down, each at least the extent (extents[d + 1]) of what follows it, so that only the two multiples of a
// stride around what is left of delta can lead there.
inline bool share_bytes(const Dim *dims, const int64_t *extents, int n, int64_t delta) {
  if (n == 0) return delta > -extents[0] && delta < extents[0];
  const int64_t stride = dims[0].stride, top = dims[0].size - 1, rest = extents[1];
  int64_t i = delta < 0 || delta >= stride ? delta / stride : 0;  // rounded towards 0
  if (delta < i * stride) --i;
  for (int k = 0; k < 2; ++k, ++i) {
    const int64_t left = delta - i * stride;
    if (i >= -top && i <= top && left > -rest && left < rest && share_bytes(dims + 1, extents + 1, n - 1, left)) return true;
  }
  return false;
}

// state[b][i] <- state[b][parent[i]] in place: a thread owns one vector position of a request, loads
// what the moving beams need and then stores it, so no other thread touches what it reads or writes.
template <typename V, int B>
__global__ void __launch_bounds__(256) beam_reorder_kernel(const __grid_constant__ ReorderParams p) {
  griddep_wait();
  const int32_t *par = p.parents + static_cast<int64_t>(blockIdx.y) * p.beams;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (item >= p.items) return;
  const int64_t o = item / p.vecs;
  const uint32_t c = static_cast<uint32_t>(item - o * p.vecs);
  const int64_t o12 = static_cast<int64_t>(p.outer1) * p.outer2;
  const int64_t o0 = o / o12;
  const uint32_t rest = static_cast<uint32_t>(o - o0 * o12);
  uint8_t *base = static_cast<uint8_t *>(p.states[blockIdx.z]) + static_cast<int64_t>(blockIdx.y) * p.beams * p.row_stride +
                  o0 * p.outer_stride[0] + rest / p.outer2 * p.outer_stride[1] + rest % p.outer2 * p.outer_stride[2] +
                  static_cast<int64_t>(c) * sizeof(V);
  V v[B];
  uint32_t moves = 0;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    if (i < p.beams) {
      const int from = par[i];
      if (from < 0 || from >= p.beams) {
        if (item == 0 && blockIdx.z == 0) raise_status(kStatusBeamBadParent);
      } else if (from != i) {
        v[i] = *reinterpret_cast<const V *>(base + from * p.row_stride);
        moves |= 1u << i;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < B; ++i)
    if (moves >> i & 1) *reinterpret_cast<V *>(base + i * p.row_stride) = v[i];
}

template <typename V>
int reorder_launch(const ReorderParams &p, int batch, int nstates, cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((p.items + 255) / 256), batch, nstates);
  const char *what = "mq_beam_reorder";
  if (p.beams <= 4) return launch_overlapped(beam_reorder_kernel<V, 4>, grid, dim3(256), 0, s, what, p);
  if (p.beams <= 8) return launch_overlapped(beam_reorder_kernel<V, 8>, grid, dim3(256), 0, s, what, p);
  if (p.beams <= 16) return launch_overlapped(beam_reorder_kernel<V, 16>, grid, dim3(256), 0, s, what, p);
  return launch_overlapped(beam_reorder_kernel<V, 32>, grid, dim3(256), 0, s, what, p);
}

}  // namespace beam
}  // namespace mq

// The sizes that mq_beam_select takes, beams being in range (by division: no product of them overflows).
static bool beam_sizes_fit(int64_t batch, int beams, int64_t vocab) {
  return vocab <= ((1LL << 31) - mq::beam::kChunkBytes - 1) / beams && batch <= ((1LL << 22) - 1) / beams;
}

extern "C" size_t mq_beam_workspace_size(int64_t batch, int beams, int64_t vocab) {
  if (batch <= 0 || beams <= 0 || beams > mq::beam::kMaxBeams || vocab <= 0 || !beam_sizes_fit(batch, beams, vocab)) return 0;
  const int64_t rows = batch * beams;
  return mq::beam::parts_bytes(rows * mq::beam::splits_for(rows, beams, vocab), beams + 1);
}

extern "C" int mq_beam_select(const void *logits, int dtype, int64_t ld, const float *scores, const uint8_t *finished,
                              int eos, float *next_scores, int32_t *tokens, int32_t *parents, uint8_t *next_finished,
                              int64_t batch, int beams, int64_t vocab, void *workspace, size_t workspace_bytes,
                              void *stream) {
  using namespace mq::beam;
  const char *what = "mq_beam_select";
  MQ_REQUIRE(batch >= 0 && beams > 0 && vocab > 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(beams <= kMaxBeams, MQ_EUNSUPPORTED, "%s: beams is above %d", what, kMaxBeams);
  MQ_REQUIRE(beam_sizes_fit(batch, beams, vocab), MQ_EUNSUPPORTED, "%s: beams * vocab or batch * beams is too large", what);
  MQ_REQUIRE(dtype == MQ_F32 || dtype == MQ_F16 || dtype == MQ_BF16, MQ_EINVAL,
             "%s: the logits' type must be MQ_F32, MQ_F16 or MQ_BF16", what);
  MQ_REQUIRE(ld >= vocab, MQ_EINVAL, "%s: the logits' row stride is less than vocab", what);
  MQ_REQUIRE(eos >= -1 && eos < vocab && !(finished && eos < 0), MQ_EINVAL,
             "%s: eos must be a token (-1 only without finished)", what);
  if (batch == 0) return MQ_OK;
  MQ_REQUIRE(logits && scores && next_scores && tokens && parents && workspace, MQ_EINVAL, "%s: null pointer", what);
  MQ_REQUIRE(mq::aligned(logits, dtype == MQ_F32 ? 4 : 2) && mq::aligned(scores, 4) && mq::aligned(next_scores, 4) &&
                 mq::aligned(tokens, 4) && mq::aligned(parents, 4) && mq::aligned(workspace, 16),
             MQ_EALIGN, "%s: the workspace must be 16-byte aligned, the others aligned to their elements", what);
  MQ_REQUIRE(workspace_bytes >= mq_beam_workspace_size(batch, beams, vocab), MQ_EINVAL, "%s: the workspace is too small",
             what);
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t rows = batch * beams;
  const int splits = splits_for(rows, beams, vocab);
  const Parts parts = parts_at(workspace, rows * splits);
  ScanParams sp{logits, scores, finished, parts, ld, beams, static_cast<int>(vocab), splits};
  const dim3 grid(static_cast<unsigned>(rows * splits));
  int rc;
  if (dtype == MQ_F32)
    rc = scan_launch<float>(sp, grid, s, what);
  else if (dtype == MQ_F16)
    rc = scan_launch<__half>(sp, grid, s, what);
  else
    rc = scan_launch<__nv_bfloat16>(sp, grid, s, what);
  if (rc) return rc;
  MergeParams mp{logits, scores, finished, parts, next_scores, tokens, parents, next_finished, ld, dtype, beams,
                 static_cast<int>(vocab), splits, eos};
  const size_t smem = static_cast<size_t>(beams) * splits * (beams + 1) * 8;
  static size_t configured[64] = {};
  if (int rc2 = mq::ensure_smem(beam_merge_kernel, smem, configured, what)) return rc2;
  return mq::launch_overlapped(beam_merge_kernel, dim3(static_cast<unsigned>(batch)), dim3(kThreads), smem, s, what, mp);
}

namespace mq {
namespace beam {

// The checks of mq_beam_reorder, and its launches' parameters but for the states: p.items stays 0 where there is nothing
// to move. width: bytes of a vector.
int reorder_plan(void *const *states, int nstates, const int32_t *parents, int64_t batch, int beams, int64_t row_stride,
                 const int64_t *outer, const int64_t *outer_stride, int64_t inner_bytes, ReorderParams &p, int &width) {
  const char *what = "mq_beam_reorder";
  MQ_REQUIRE(nstates >= 0 && batch >= 0 && beams > 0 && inner_bytes >= 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(beams <= kMaxBeams && batch <= 65535, MQ_EUNSUPPORTED, "%s: beams is above %d or batch above 65535", what,
             kMaxBeams);
  if (nstates == 0 || batch == 0 || inner_bytes == 0) return MQ_OK;
  MQ_REQUIRE(inner_bytes < (1LL << 60), MQ_EUNSUPPORTED, "%s: a state is too large", what);
  MQ_REQUIRE(states && parents && outer && outer_stride, MQ_EINVAL, "%s: null pointer", what);
  // Every (row, outer index) must have bytes of its own: sorted by stride, each dimension has to step
  // over all that the faster ones cover.
  int64_t count = 1;
  int align = 16;
  auto divides = [&](int64_t v) { while (align > 1 && v % align) align /= 2; };
  Dim dims[4] = {{outer_stride[0], outer[0]}, {outer_stride[1], outer[1]}, {outer_stride[2], outer[2]},
                 {row_stride, batch * beams}};
  std::sort(dims, dims + 4, [](const Dim &a, const Dim &b) { return a.stride < b.stride; });
  int64_t extent = inner_bytes, extents[5] = {0, 0, 0, 0, inner_bytes};  // of the last n dimensions of `steps`
  Dim steps[4];  // those with more than one index, from the largest stride down
  int first_step = 4;
  for (const Dim &d : dims) {
    MQ_REQUIRE(d.size >= 0 && d.size < (1LL << 31), MQ_EINVAL, "%s: bad outer dimension", what);
    if (d.size == 0) return MQ_OK;
    if (d.size == 1) continue;
    MQ_REQUIRE(d.stride >= extent, MQ_EINVAL, "%s: states overlap (a stride is less than what it steps over)", what);
    MQ_REQUIRE(d.stride < (1LL << 60) / d.size, MQ_EUNSUPPORTED, "%s: a state is too large", what);
    divides(d.stride);
    extent += d.stride * (d.size - 1);
    steps[--first_step] = d, extents[first_step] = extent;
  }
  for (int d = 0; d < 3; ++d) count *= outer[d];
  MQ_REQUIRE(outer[1] * outer[2] < (1LL << 31), MQ_EUNSUPPORTED, "%s: the outer dimensions are too large", what);
  divides(inner_bytes);
  for (int i = 0; i < nstates; ++i) {
    MQ_REQUIRE(states[i], MQ_EINVAL, "%s: null state", what);
    divides(static_cast<int64_t>(reinterpret_cast<uintptr_t>(states[i]) % 16));
  }
  if (nstates > 1) {  // two states of one launch that share memory would race
    std::unique_ptr<uintptr_t[]> at(new (std::nothrow) uintptr_t[nstates]);
    MQ_REQUIRE(at, MQ_EINVAL, "%s: no memory to compare %d states", what, nstates);
    for (int i = 0; i < nstates; ++i) at[i] = reinterpret_cast<uintptr_t>(states[i]);
    std::sort(at.get(), at.get() + nstates);
    for (int i = 0; i < nstates; ++i)
      for (int j = i + 1; j < nstates && at[j] - at[i] < static_cast<uintptr_t>(extent); ++j)
        MQ_REQUIRE(!share_bytes(steps + first_step, extents + first_step, 4 - first_step, static_cast<int64_t>(at[j] - at[i])),
                   MQ_EINVAL, "%s: states overlap one another", what);
  }
  p.parents = parents, p.row_stride = row_stride, p.beams = beams;
  for (int d = 0; d < 3; ++d) p.outer_stride[d] = outer_stride[d];
  p.outer1 = static_cast<uint32_t>(outer[1]), p.outer2 = static_cast<uint32_t>(outer[2]);
  width = align == 16 ? 16 : align >= 4 ? 4 : align;
  MQ_REQUIRE(inner_bytes / width < (1LL << 31), MQ_EUNSUPPORTED, "%s: the inner part is too large", what);
  p.vecs = static_cast<uint32_t>(inner_bytes / width);
  p.items = count * p.vecs;
  MQ_REQUIRE(p.items < (1LL << 31) * 256 - 256, MQ_EUNSUPPORTED, "%s: a state is too large", what);
  return MQ_OK;
}

}  // namespace beam
}  // namespace mq

extern "C" int mq_beam_reorder_check(void *const *states, int nstates, const int32_t *parents, int64_t batch, int beams,
                                     int64_t row_stride, const int64_t *outer, const int64_t *outer_stride,
                                     int64_t inner_bytes) {
  mq::beam::ReorderParams p{};
  int width = 0;
  return mq::beam::reorder_plan(states, nstates, parents, batch, beams, row_stride, outer, outer_stride, inner_bytes, p, width);
}

extern "C" int mq_beam_reorder(void *const *states, int nstates, const int32_t *parents, int64_t batch, int beams,
                               int64_t row_stride, const int64_t *outer, const int64_t *outer_stride, int64_t inner_bytes,
                               void *stream) {
  using namespace mq::beam;
  ReorderParams p{};
  int width = 0;
  if (int rc = reorder_plan(states, nstates, parents, batch, beams, row_stride, outer, outer_stride, inner_bytes, p, width))
    return rc;
  if (p.items == 0) return MQ_OK;
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  for (int first = 0; first < nstates; first += kMaxStates) {
    const int n = std::min(kMaxStates, nstates - first);
    for (int i = 0; i < n; ++i) p.states[i] = states[first + i];
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int rc;
    if (width == 16)
      rc = reorder_launch<uint4>(p, static_cast<int>(batch), n, s);
    else if (width == 4)
      rc = reorder_launch<uint32_t>(p, static_cast<int>(batch), n, s);
    else if (width == 2)
      rc = reorder_launch<uint16_t>(p, static_cast<int>(batch), n, s);
    else
      rc = reorder_launch<uint8_t>(p, static_cast<int>(batch), n, s);
    if (rc) return rc;
  }
  return MQ_OK;
}
