// Drafted tokens against the target's distribution (mq_verify_drafts): beam.cu's and mq_head_argmax's place where a
// drafter proposes several tokens at once.
//
// p_i = softmax(target row i / T), q_i = softmax(draft row i / T) (without draft logits: all on the drafted token). Drafted
// token d_i is kept while u_i q_i(d_i) < p_i(d_i). At the first that is not, i = n, one token is drawn from max(p_n - q_n, 0), where
// all are kept from p_n: the first v whose running sum exceeds u times the whole, u the number behind the drafts' (one that was
// looked at for a token that it rejected is no longer uniform). At T = 0 p is all on the largest logit, the
// lowest index among equal ones.
//
// verify_scan_kernel reads every logit once: `splits` CTAs per row keep a maximum and a sum of exponentials, in fp32:
// a comparison of u q with p is off by some 1e-7, so it decides otherwise once in 10^7 times. It is bound by the bandwidth
// (64 requests of 128256 fp32 and 4 drafts, 21 of them greedy, so 252 MB: 47 us, 5.4 TB/s, 0.82 of a copy's).
//
// verify_draw_kernel, a cluster per request, decides, and goes through the chosen row again for the draw. There fp32 does not do:
// the running sum passes some 10^5 borders between tokens, and a relative error of 1e-8 in it would move the drawn token
// to its neighbour once in a thousand draws. So the sums and the exponentials in them are fp64: 2^y with
// y = n / 32 + r, |r| <= 1/64, is 2^(n / 32) from a table of 32 times a Taylor polynomial of degree 5 (2e-15), nine
// fp64 instructions. Each warp has a stretch of the row of its own; the CTA whose stretch holds the drawn token looks for it.
// It goes through the row twice where q is taken off (first for the two sums): 60 us for the 43 of those 64 requests that sample, bound by the latency of the fetches and of the cluster's three exchanges. A greedy request needs neither (4 drafts of
// 151669: 6 us in all, 27 where it samples).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace mq {
namespace verify {

constexpr int kScan = 256, kVecs = 4;        // threads of a scan CTA, 16-byte vectors per thread and step
// The drawing CTAs of a request and their threads: many for the latency of a few requests with a long row, fewer where that lets all
// CTAs run at once (four of 256 on an SM). Sixteen CTAs against eight, requests of 4 drafts that all sample, scan and draw, us:
//   fp32  151669: 1: 25.4 (28.5), 4: 34.8 (37.4), 12: 49.6 (54.6), but 18: 69.8 (62.9), 37: 120 (100); 100352: 1: 21.5 (24.4),
//         12: 39.8 (44.0); but 48000: 4: 26.3 (23.2), 32000: 1: 18.4 (17.3), 4: 25.1 (20.1), 12: 27.8 (23.8); 80000: about equal.
//   bf16  151669: 1: 26.0 (29.5), 6: 34.1 (38.1), but 8: 44.9 (42.2), 12: 46.6 (43.0); 100352: 6: 29.8 (33.4), but 12: 39.7 (37.4).
constexpr int kClusterFew = 16, kCluster = 8;
constexpr int kDrawFew = 512, kDrawMany = 256, kManyRequests = 148 * 2 / kCluster;
constexpr int kFewRequests = 12, kFewRequests16 = 6;  // of fp32, of 16-bit logits
constexpr int64_t kLongRow = 100000;
constexpr int kMaxDrafts = 32, kMaxSplits = 64;
constexpr float kLeastTemperature = 1e-5f;   // below: 0
// Less than this of p - q is nothing: equal distributions leave the roundings of their terms, 1e-14 in all (of two rows with the
// same bits 1e-17: one product is rounded before the other is taken off it, in one operation).
constexpr double kNothingLeft = 1e-13;
constexpr double kLog2e = 1.4426950408889634074, kLn2 = 0.69314718055994530942;

// CTAs of a scan that run at once: eight on each of 148 SMs.
constexpr int kScanCtas = 148 * 8;
// As many CTAs as run at once, a step of each at least. rows * splits is at most the larger of rows and kScanCtas.
__host__ __device__ constexpr int splits_for(int64_t rows, int64_t vocab) {
  const int64_t steps = (vocab * 4 + kScan * kVecs * 16 - 1) / (kScan * kVecs * 16);
  int64_t s = kScanCtas / rows;
  if (s > kMaxSplits) s = kMaxSplits;
  if (s > steps) s = steps;
  return s < 1 ? 1 : static_cast<int>(s);
}

struct Params {
  const void *target, *draft;  // draft may be null
  int64_t ld_target, ld_draft;
  const int32_t *drafted, *counts;  // counts may be null
  const float *uniform, *temperature;  // temperature may be null: 1
  float2 *parts;  // [batch][2 drafts + 1][splits]: the largest logit, and the sum relative to it (T = 0: its index's bits)
  int32_t *tokens, *accepted;
  float *logprobs;
  int batch, drafts, vocab, splits, dtype;
};

__device__ __forceinline__ int rows_per_request(const Params &p) { return p.draft ? 2 * p.drafts + 1 : p.drafts + 1; }
__device__ __forceinline__ float temperature_of(const Params &p, int b) {
  const float t = p.temperature ? p.temperature[b] : 1.f;
  return t >= kLeastTemperature ? fminf(t, 1e30f) : 0.f;  // (an infinite one would make -infinity / T no number)
}
__device__ __forceinline__ int count_of(const Params &p, int b) {
  const int n = p.counts ? p.counts[b] : p.drafts;
  if (n < 0 || n > p.drafts) raise_status(kStatusVerifyBadToken);
  return min(max(n, 0), p.drafts);
}
// Row i of a request: target rows 0 .. drafts, then the draft's.
__device__ __forceinline__ const char *row_at(const Params &p, int b, int i) {
  const int es = p.dtype == MQ_F32 ? 4 : 2;
  if (i <= p.drafts) return static_cast<const char *>(p.target) + (static_cast<int64_t>(b) * (p.drafts + 1) + i) * p.ld_target * es;
  return static_cast<const char *>(p.draft) + (static_cast<int64_t>(b) * p.drafts + i - p.drafts - 1) * p.ld_draft * es;
}

template <typename T>
__global__ void __launch_bounds__(kScan) verify_scan_kernel(const Params p) {
  constexpr int V = 16 / sizeof(T), kElems = V * kVecs;
  __shared__ float red[kScan / 32];
  __shared__ float sums[kScan / 32];
  __shared__ int index_red[kScan / 32];
  griddep_launch_dependents();
  griddep_wait();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, per = rows_per_request(p);
  const int split = blockIdx.x % p.splits, i = blockIdx.x / p.splits % per, b = blockIdx.x / p.splits / per;
  const float hot = temperature_of(p, b);
  const int n = count_of(p, b);
  if (i <= p.drafts ? i > n : i - p.drafts - 1 >= n || hot == 0.f) return;  // nobody asks for that row
  const T *x = reinterpret_cast<const T *>(row_at(p, b, i));
  // The row's 16-byte aligned vectors, dealt to the splits; the elements before and behind them (at most V - 1 each) are
  // split 0's.
  const int head = min(p.vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
  const int nvec = (p.vocab - head) / V, body_end = head + nvec * V, edges = head + p.vocab - body_end;
  const int v0 = static_cast<int>(static_cast<int64_t>(nvec) * split / p.splits);
  const int v1 = static_cast<int>(static_cast<int64_t>(nvec) * (split + 1) / p.splits);
  const float k = static_cast<float>(kLog2e / (hot > 0.f ? static_cast<double>(hot) : 1.0));
  float m = -INFINITY, s = 0.f;
  int at = p.vocab;  // T = 0: the first place of m
  auto take = [&](const float (&v)[kElems], const int (&first)[kVecs]) {
    float big = v[0];
#pragma unroll
    for (int e = 1; e < kElems; ++e) big = fmaxf(big, v[e]);
    if (hot > 0.f) {
      if (big > m) s *= exp2f((m - big) * k), m = big;
      const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int e = 0; e < kElems; ++e) {
        float y;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"((v[e] - ref) * k));
        s += y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < kElems; ++e) s += v[e] < INFINITY ? 0.f : NAN;
      if (big > m) {
        m = big;
#pragma unroll
        for (int e = kElems - 1; e >= 0; --e)
          if (v[e] == big) at = first[e / V] + e % V;
      }
    }
  };
  const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
#pragma unroll 1
  for (int base = v0; base < v1; base += kScan * kVecs) {
    float v[kElems];
    int first[kVecs];
    uint4 q[kVecs];
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const int g = base + u * kScan + tid;
      first[u] = head + g * V;
      if (g < v1) q[u] = ldg_stream_v4(body + g);
    }
#pragma unroll
    for (int u = 0; u < kVecs; ++u) {
      const bool in = base + u * kScan + tid < v1;
      const T *e = reinterpret_cast<const T *>(&q[u]);
#pragma unroll
      for (int j = 0; j < V; ++j) v[u * V + j] = in ? static_cast<float>(e[j]) : -INFINITY;
    }
    take(v, first);
  }
  if (split == 0 && tid < edges) {
    float v[kElems];
    int first[kVecs] = {};
#pragma unroll
    for (int e = 0; e < kElems; ++e) v[e] = -INFINITY;
    first[0] = tid < head ? tid : body_end + tid - head;
    v[0] = static_cast<float>(x[first[0]]);
    if (hot == 0.f && v[0] == m && first[0] < at) at = first[0];  // (an edge before the body)
    take(v, first);
  }
  // Join the threads', in one fixed order.
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
  top = red[0];
  for (int w = 1; w < kScan / 32; ++w) top = fmaxf(top, red[w]);
  if (hot > 0.f) s = m == -INFINITY ? s : s * exp2f((m - top) * k);  // (an empty thread's sum is 0, or NaN)
  int where = m == top ? at : p.vocab;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    where = min(where, __shfl_xor_sync(0xffffffffu, where, o));
  }
  if (lane == 0) sums[warp] = s, index_red[warp] = where;
  __syncthreads();
  if (tid == 0) {
    s = 0.f;
    where = p.vocab;
    for (int w = 0; w < kScan / 32; ++w) s += sums[w], where = min(where, index_red[w]);
    if (hot == 0.f) s = s == s ? __int_as_float(where) : __int_as_float(-1);
    p.parts[blockIdx.x] = make_float2(top, s);
  }
}

template <typename T>
__device__ __forceinline__ float read(const char *row, int v) {
  return static_cast<float>(reinterpret_cast<const T *>(row)[v]);
}

// 2^((x - top) k / 32) in fp64, relative error below 1e-14 (k: 32 log2(e) / T). The sum with 1.5 * 2^52 rounds to an integer.
struct Exp {
  double k, magic;
  float least;
  const double *table;  // 2^(i / 32)
  __device__ __forceinline__ void start(float top, float hot, const double *t) {
    k = 32.0 * kLog2e / hot;
    // (Logits so large that the next one below is 2^-10000 of the largest: only that one counts.)
    if (!(fabs(top * k) < 1e15)) k = 0;
    magic = 6755399441055744.0 - rint(top * k);
    least = fmaxf(top - 600.f * hot, -3.402823466e38f);  // below: 0 (2^-865 of the largest)
    table = t;
  }
  __device__ __forceinline__ double operator()(float x) const {
    const double y = fmaxf(x, least), t = fma(y, k, magic), n = t - magic, r = fma(y, k, -n);
    constexpr double a = kLn2 / 32;
    double e = fma(r, a * a * a * a * a / 120, a * a * a * a / 24);
    e = fma(e, r, a * a * a / 6);
    e = fma(e, r, a * a / 2);
    e = fma(e, r, a);
    e = fma(e, r, 1.0);
    const int low = __double2loint(t);
    const double z = table[low & 31];
    e *= __hiloint2double(__double2hiint(z) + ((low >> 5) << 20), __double2loint(z));
    return x >= least ? e : 0.0;  // (no branch: several are computed side by side)
  }
};

__device__ __forceinline__ uint32_t rank_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void sync_cluster() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T, int kDraw, int kCluster>
__global__ void __launch_bounds__(kDraw, 1024 / kDraw) verify_draw_kernel(const Params p) {
  constexpr int kWarps = kDraw / 32, stretch = kCluster * kWarps, kPer = stretch / 32;  // stretches of a row; of a lane
  __shared__ double table[32];
  __shared__ float top[2 * kMaxDrafts + 1], total[2 * kMaxDrafts + 1];  // of the request's rows; T = 0: total holds the index
  __shared__ int kept_s, bad_s, last_s;
  __shared__ double warp_sums[3][kWarps];    // p, q; then the weights
  __shared__ double all_sums[3][kCluster][kWarps];
  griddep_launch_dependents();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, rank = rank_in_cluster(), b = blockIdx.x / kCluster;
  if (tid < 32) table[tid] = exp2(tid / 32.0);
  griddep_wait();
  const int per = rows_per_request(p), n = count_of(p, b);
  const float hot = temperature_of(p, b);
  for (int i = warp; i < per; i += kWarps) {
    if (i <= p.drafts ? i > n : i - p.drafts - 1 >= n || hot == 0.f) continue;
    const float2 *parts = p.parts + (static_cast<int64_t>(b) * per + i) * p.splits;
    float m = -INFINITY;
    for (int j = lane; j < p.splits; j += 32) m = fmaxf(m, parts[j].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (hot > 0.f) {
      double s = 0;
      for (int j = lane; j < p.splits; j += 32) {
        const float2 q = parts[j];
        s += q.x == -INFINITY ? static_cast<double>(q.y) : q.y * exp2((static_cast<double>(q.x) - m) * kLog2e / hot);
      }
      s = warp_sum(s);
      if (lane == 0) top[i] = m, total[i] = static_cast<float>(s);
    } else {
      int where = p.vocab;
      bool bad = false;
      for (int j = lane; j < p.splits; j += 32) {
        const int at = __float_as_int(parts[j].y);
        bad |= at < 0;
        if (parts[j].x == m && at >= 0) where = min(where, at);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) where = min(where, __shfl_xor_sync(0xffffffffu, where, o));
      bad = __any_sync(0xffffffffu, bad) || !(m > -INFINITY);
      if (lane == 0) top[i] = m, total[i] = __int_as_float(bad ? -1 : where);
    }
  }
  __syncthreads();
  auto good = [&](int i) { return hot > 0.f ? total[i] > 0.f && total[i] < INFINITY && fabsf(top[i]) < INFINITY : __float_as_int(total[i]) >= 0; };
  if (warp == 0) {  // lane i: drafted token i
    const int64_t at = static_cast<int64_t>(b) * (p.drafts + 1) + lane;
    bool keep = false;
    int status = 0;
    float logprob = 0.f;
    if (lane <= n && !good(lane)) {
      status = kStatusVerifyBadRow;
    } else if (lane < n) {
      const int d = p.drafted[static_cast<int64_t>(b) * p.drafts + lane], j = p.drafts + 1 + lane;
      if (d < 0 || d >= p.vocab) {
        status = kStatusVerifyBadToken;
      } else if (hot == 0.f) {
        keep = d == __float_as_int(total[lane]);
      } else if (p.draft && !good(j)) {
        status = kStatusVerifyBadRow;
      } else {
        const double z = (static_cast<double>(read<T>(row_at(p, b, lane), d)) - top[lane]) / hot;
        const double pd = exp(z) / total[lane];
        const double qd = p.draft ? exp((static_cast<double>(read<T>(row_at(p, b, j), d)) - top[j]) / hot) / total[j] : 1.0;
        keep = p.uniform[at] * qd < pd;
        logprob = static_cast<float>(z - log(static_cast<double>(total[lane])));
      }
    }
    const unsigned not_kept = ~__ballot_sync(0xffffffffu, keep);  // (at most 32 drafts: lane 31 may be a kept one)
    const int first = not_kept ? __ffs(not_kept) - 1 : 32;
    if (lane < first && rank == 0) p.logprobs[at] = logprob;
    if (lane == first && status) raise_status(status);
    if (lane == 0) {
      kept_s = first, bad_s = !good(first);
      if (first == 32 && bad_s) raise_status(kStatusVerifyBadRow);
    }
  }
  __syncthreads();
  const int kept = kept_s, bad = bad_s;
  const int64_t out0 = static_cast<int64_t>(b) * (p.drafts + 1);
  if (rank == 0) {
    if (tid == 0) p.accepted[b] = kept;
    for (int i = tid; i <= p.drafts; i += kDraw) {
      if (i < kept)
        p.tokens[out0 + i] = p.drafted[static_cast<int64_t>(b) * p.drafts + i];
      else if (i > kept || bad || hot == 0.f) {
        p.tokens[out0 + i] = i == kept && !bad ? __float_as_int(total[kept]) : -1;
        p.logprobs[out0 + i] = 0.f;
      }
    }
  }
  if (bad || hot == 0.f) return;  // (the whole cluster)

  // The draw. This warp's stretch of the row:
  const int mine = rank * kWarps + warp;
  const int v0 = static_cast<int>(static_cast<int64_t>(p.vocab) * mine / stretch);
  const int v1 = static_cast<int>(static_cast<int64_t>(p.vocab) * (mine + 1) / stretch);
  const char *pr = row_at(p, b, kept);
  const int d = kept < n ? p.drafted[static_cast<int64_t>(b) * p.drafts + kept] : -1;
  const bool two = p.draft && kept < n && d >= 0 && d < p.vocab && good(p.drafts + 1 + kept);
  const char *qr = two ? row_at(p, b, p.drafts + 1 + kept) : nullptr;
  // Without draft logits the drafted token has all of q, so nothing of it is left.
  const int without = !p.draft ? d : -1;
  Exp ep, eq;
  ep.start(top[kept], hot, table);
  eq.start(two ? top[p.drafts + 1 + kept] : 0.f, hot, table);

  // Sums over the cluster of what every warp has; all_sums keeps each warp's, in the row's order.
  auto gather = [&](int which, double v) {
    v = warp_sum(v);
    if (lane == 0) warp_sums[which][warp] = v;
    sync_cluster();
    for (int e = tid; e < stretch; e += kDraw) {
      uint32_t from;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(smem_u32(&warp_sums[which][e % kWarps])), "r"(e / kWarps));
      double x;
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(x) : "r"(from) : "memory");
      all_sums[which][e / kWarps][e % kWarps] = x;
    }
    __syncthreads();
    const double *all = &all_sums[which][0][0];
    double sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += all[lane + 32 * e];
    return warp_sum(sum);
  };
  // f(token, its logit in p, in q) of this warp's stretch, a lane every 32nd: kAhead of them are fetched before any is used.
  constexpr int kAhead = 8;
  auto sweep = [&](auto both, auto f) {
    constexpr bool kBoth = decltype(both)::value;
#pragma unroll 1
    for (int base = v0 + lane; base < v1; base += 32 * kAhead) {
      float x[kAhead], y[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int v = base + 32 * u;
        x[u] = v < v1 ? read<T>(pr, v) : -INFINITY;
        y[u] = kBoth && v < v1 ? read<T>(qr, v) : -INFINITY;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) f(base + 32 * u, x[u], y[u]);
    }
  };
  double ip = 1, iq = 0;
  bool rest = two;
  if (two) {
    double sp = 0, sq = 0;
    sweep(std::true_type(), [&](int, float x, float y) { sp += ep(x), sq += eq(y); });
    ip = 1 / gather(0, sp);
    iq = 1 / gather(1, sq);
  }
  double whole = 0;
  for (int round = 0; round < 2; ++round) {
    double w = 0;
    if (rest)
      sweep(std::true_type(), [&](int, float x, float y) {
        const double left = fma(eq(y), -iq, ep(x) * ip);
        w += left > 0 ? left : 0.0;
      });
    else
      sweep(std::false_type(), [&](int v, float x, float) { w += v == without ? 0.0 : ep(x); });
    if (round) sync_cluster();  // (everybody has read the first round's sums)
    whole = gather(2, w);
    if (whole > kNothingLeft || !rest) break;
    rest = false;  // p and q are one, so the draw is from p
  }
  const double goal = p.uniform[out0 + p.drafts] * whole;
  // The first stretch whose running sum passes the goal, else the last that has any weight.
  double before = 0;  // of lane's first stretch; then of the one that was found
  int found = -1;
  {
    const double *all = &all_sums[2][0][0] + kPer * lane;
    double incl = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) incl += all[e];
    const double own = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    double run = incl - own;
    int over = -1, last = -1;
    double over_at = 0, last_at = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      if (all[e] > 0) {
        last = kPer * lane + e, last_at = run;
        if (over < 0 && run + all[e] > goal) over = last, over_at = run;
      }
      run += all[e];
    }
    const unsigned overs = __ballot_sync(0xffffffffu, over >= 0), lasts = __ballot_sync(0xffffffffu, last >= 0);
    const int from = overs ? __ffs(overs) - 1 : lasts ? 31 - __clz(lasts) : 0;
    found = __shfl_sync(0xffffffffu, overs ? over : last, from);
    before = __shfl_sync(0xffffffffu, overs ? over_at : last_at, from);
  }
  sync_cluster();  // (nobody reads another's sums from here on: who is done may leave)
  if (found < 0) {  // no token has weight: the only one was drafted and is not kept
    if (rank == 0 && tid == 0) p.tokens[out0 + kept] = -1, p.logprobs[out0 + kept] = 0.f;
    return;
  }
  if (found / kWarps != static_cast<int>(rank)) return;
  // The CTA whose stretch it is looks for the token: each warp takes a part, and has its weights in registers when it is known
  // which part the goal lies in. (One warp alone took 50 us, 32 tokens after 32.)
  const int f0 = static_cast<int>(static_cast<int64_t>(p.vocab) * found / stretch);
  const int f1 = static_cast<int>(static_cast<int64_t>(p.vocab) * (found + 1) / stretch);
  double run = before;
  if (tid == 0) last_s = -1;  // the last token with any weight so far
  for (int first = f0; first < f1; first += 32 * kAhead * kWarps) {  // (once, up to vocabularies of 131072)
    const int part = (min(f1 - first, 32 * kAhead * kWarps) + kWarps - 1) / kWarps, g0 = first + warp * part, g1 = min(g0 + part, f1);
    float x[kAhead], y[kAhead];
    double w[kAhead], own = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = g0 + 32 * u + lane;
      x[u] = v < g1 ? read<T>(pr, v) : -INFINITY;
      y[u] = rest && v < g1 ? read<T>(qr, v) : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int v = g0 + 32 * u + lane;
      const double e = v >= g1 || v == without ? 0.0 : ep(x[u]);
      const double left = rest && v < g1 ? fma(eq(y[u]), -iq, e * ip) : e;
      w[u] = left > 0 ? left : 0.0;
      own += w[u];
    }
    own = warp_sum(own);
    __syncthreads();
    if (lane == 0) warp_sums[0][warp] = own;
#pragma unroll
    for (int u = kAhead - 1; u >= 0; --u) {
      const unsigned any = __ballot_sync(0xffffffffu, w[u] > 0);
      if (any) {
        if (lane == 0) atomicMax(&last_s, g0 + 32 * u + 31 - __clz(any));
        break;
      }
    }
    __syncthreads();
    double ahead = run, at_part = 0;
    int holds = -1;  // the warp whose part holds the goal
    for (int v = 0; v < kWarps; ++v) {
      const double s = warp_sums[0][v];
      if (s > 0 && holds < 0 && ahead + s > goal) holds = v, at_part = ahead;
      ahead += s;
    }
    const bool ends = first + 32 * kAhead * kWarps >= f1;
    // (Rounding may leave the goal beyond the last weight, of the stretch or of the part.)
    if (warp == (holds >= 0 ? holds : 0) && (holds >= 0 || ends)) {
      double sum = at_part;
      int token = holds < 0 ? last_s : -1, last = -1;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        double incl = w[u];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double up = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += up;
        }
        const unsigned over = __ballot_sync(0xffffffffu, w[u] > 0 && sum + incl > goal), any = __ballot_sync(0xffffffffu, w[u] > 0);
        if (token < 0 && over) token = g0 + 32 * u + __ffs(over) - 1;
        if (any) last = g0 + 32 * u + 31 - __clz(any);
        sum += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (token < 0) token = last;
      if (lane == 0) {
        p.tokens[out0 + kept] = token;
        const double z = (static_cast<double>(read<T>(pr, token)) - top[kept]) / hot;
        p.logprobs[out0 + kept] = static_cast<float>(z - log(static_cast<double>(total[kept])));
      }
    }
    if (holds >= 0) return;
    run = ahead;
  }
}

template <typename T>
int scan(const Params &p, int64_t ctas, cudaStream_t s, const char *what) {
  return launch_overlapped(verify_scan_kernel<T>, dim3(static_cast<unsigned>(ctas)), dim3(kScan), 0, s, what, p);
}

// Whether this device runs clusters of kClusterFew, which are more than every device of the architecture has to take: asked
// once per kernel and device. Two threads that ask at once get the same answer.
template <typename T>
bool wide_clusters_run() {
  static std::atomic<int> known[64];  // 0 not asked, 1 yes, 2 no
  auto *kern = verify_draw_kernel<T, kDrawFew, kClusterFew>;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return false;
  int yes = known[device].load(std::memory_order_acquire);
  if (yes == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kClusterFew);
    cfg.blockDim = dim3(kDrawFew);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kClusterFew;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    const bool ok = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) == cudaSuccess && clusters > 0;
    if (!ok) cudaGetLastError();  // (the answer is no, not an error of this call)
    yes = ok ? 1 : 2;
    known[device].store(yes, std::memory_order_release);
  }
  return yes == 1;
}

template <typename T>
int draw(const Params &p, cudaStream_t s, const char *what) {
  auto go = [&](auto kern, int threads, int cluster) {
    return launch_overlapped_clusters(kern, dim3(static_cast<unsigned>(p.batch * cluster)), dim3(threads), cluster, 0, s, what, p);
  };
  if (p.batch > kManyRequests) return go(verify_draw_kernel<T, kDrawMany, kCluster>, kDrawMany, kCluster);
  if (p.batch <= (sizeof(T) == 4 ? kFewRequests : kFewRequests16) && p.vocab >= kLongRow && wide_clusters_run<T>()) return go(verify_draw_kernel<T, kDrawFew, kClusterFew>, kDrawFew, kClusterFew);
  return go(verify_draw_kernel<T, kDrawFew, kCluster>, kDrawFew, kCluster);
}

inline bool sizes_fit(int64_t batch, int64_t drafts, int64_t vocab) {
  return batch >= 0 && batch <= (1LL << 20) && drafts >= 0 && drafts <= kMaxDrafts && vocab > 0 && vocab <= (1LL << 30);
}

}  // namespace verify
}  // namespace mq

extern "C" size_t mq_verify_workspace_size(int64_t batch, int64_t drafts, int64_t vocab) {
  using namespace mq::verify;
  if (batch <= 0 || !sizes_fit(batch, drafts, vocab)) return 0;
  // What rows * splits can be, not what it is: that falls and rises with the rows, and a larger call's workspace serves a smaller one.
  return sizeof(float2) * std::max<int64_t>(batch * (2 * drafts + 1), kScanCtas);
}

extern "C" int mq_verify_drafts(const void *target, int64_t ld_target, const void *draft, int64_t ld_draft, int dtype,
                                const int32_t *drafted, const int32_t *counts, const float *uniform, const float *temperature,
                                int32_t *tokens, int32_t *accepted, float *logprobs, int64_t batch, int64_t drafts, int64_t vocab,
                                void *workspace, size_t workspace_bytes, void *stream) {
  using namespace mq::verify;
  const char *what = "mq_verify_drafts";
  MQ_REQUIRE(batch >= 0 && drafts >= 0 && vocab > 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(sizes_fit(batch, drafts, vocab), MQ_EUNSUPPORTED, "%s: batch is above 2^20, drafts above %d or vocab above 2^30", what,
             kMaxDrafts);
  MQ_REQUIRE(dtype == MQ_F32 || dtype == MQ_F16 || dtype == MQ_BF16, MQ_EINVAL, "%s: the logits' type must be MQ_F32, MQ_F16 or MQ_BF16",
             what);
  MQ_REQUIRE(ld_target >= vocab && (!draft || ld_draft >= vocab), MQ_EINVAL, "%s: the logits' row stride is less than vocab", what);
  if (batch == 0) return MQ_OK;
  MQ_REQUIRE(target && uniform && tokens && accepted && logprobs && workspace && (drafted || drafts == 0), MQ_EINVAL, "%s: null pointer",
             what);
  const int es = dtype == MQ_F32 ? 4 : 2;
  MQ_REQUIRE(mq::aligned(target, es) && mq::aligned(draft, es) && mq::aligned(drafted, 4) && mq::aligned(counts, 4) &&
                 mq::aligned(uniform, 4) && mq::aligned(temperature, 4) && mq::aligned(tokens, 4) && mq::aligned(accepted, 4) &&
                 mq::aligned(logprobs, 4) && mq::aligned(workspace, 16),
             MQ_EALIGN, "%s: the workspace must be 16-byte aligned, the others aligned to their elements", what);
  MQ_REQUIRE(workspace_bytes >= mq_verify_workspace_size(batch, drafts, vocab), MQ_EINVAL, "%s: the workspace is too small", what);
  if (drafts == 0) draft = nullptr;
  const int64_t rows = batch * (draft ? 2 * drafts + 1 : drafts + 1), given = 4 * batch * (drafts + 1);
  {
    // Some CTAs of a request write while others still read.
    struct Range {
      const void *at;
      __int128 bytes;
    };
    const Range written[] = {{tokens, given}, {accepted, 4 * batch}, {logprobs, given}, {workspace, static_cast<int64_t>(mq_verify_workspace_size(batch, drafts, vocab))}};
    const Range read[] = {{target, (static_cast<__int128>(batch * (drafts + 1) - 1) * ld_target + vocab) * es},
                          {draft, (static_cast<__int128>(batch * drafts - 1) * ld_draft + vocab) * es},
                          {drafted, 4 * batch * drafts}, {counts, 4 * batch}, {uniform, given}, {temperature, 4 * batch}};
    auto meet = [](const Range &a, const Range &b) {
      return a.at && b.at && a.bytes > 0 && b.bytes > 0 &&
             (a.at <= b.at ? static_cast<const char *>(b.at) - static_cast<const char *>(a.at) < a.bytes
                           : static_cast<const char *>(a.at) - static_cast<const char *>(b.at) < b.bytes);
    };
    for (int i = 0; i < 4; ++i) {
      for (const Range &r : read) MQ_REQUIRE(!meet(written[i], r), MQ_EINVAL, "%s: an output or the workspace shares memory with an input", what);
      for (int j = 0; j < i; ++j) MQ_REQUIRE(!meet(written[i], written[j]), MQ_EINVAL, "%s: outputs or the workspace share memory", what);
    }
  }
  mq::DeviceInfo dev;
  if (int rc = mq::device_info(&dev)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Params p{target, draft, ld_target, ld_draft, drafted, counts, uniform, temperature, static_cast<float2 *>(workspace), tokens, accepted,
           logprobs, static_cast<int>(batch), static_cast<int>(drafts), static_cast<int>(vocab), splits_for(rows, vocab), dtype};
  int rc;
  if (dtype == MQ_F32)
    rc = scan<float>(p, rows * p.splits, s, what);
  else if (dtype == MQ_F16)
    rc = scan<__half>(p, rows * p.splits, s, what);
  else
    rc = scan<__nv_bfloat16>(p, rows * p.splits, s, what);
  if (rc) return rc;
  if (dtype == MQ_F32) return draw<float>(p, s, what);
  if (dtype == MQ_F16) return draw<__half>(p, s, what);
  return draw<__nv_bfloat16>(p, s, what);
}
