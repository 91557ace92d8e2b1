// A paged cache's rows: the new tokens' keys and values into their pages (mq_kv_store), and what the pages hold back into
// rows (mq_kv_load).
//
// A row is the keys (or values) of one token and head. Rows go in rounded once to a 16-bit cache's type; an int8
// cache takes a = max |x| of the row, q = rint(x * (127 / a)) and the scale a / 127 (mq_quantize_s8's
// arithmetic, bit for bit). Rows come back as q * scale in fp32, rounded once.
//
// Both are a copy: what bounds them is the bandwidth, or for a few tokens the launch and the chain of loads that finds a
// token's page. A CTA looks up the places of its tokens (up to 64) at once; then each of its threads has one piece of 8 values of
// a token's rows, 8 or 16 lanes to a row, and takes it from token to token, four on their way (two: 75 and 183 us, eight: 79 and
// 200). 53,223 tokens of 2 x 8 x 128 bf16 into pages: 74 us (5.9 TB/s), into int8 pages 115 (2.9); 137,835 of int8 back as bf16: 168 us (5.1 TB/s: the
// conversions); one token: 2 us.
#include <type_traits>

#include "paged.cuh"

namespace mq {
namespace paged {

constexpr int kCopyThreads = 256, kMostTokens = 64, kAhead = 4;

struct CopyParams {
  Seqs seqs;
  void *pages[2];  // keys, values
  float *scales[2];
  int64_t stride[2][3], scale_stride[2][3];
  void *rows[2];
  int64_t token_stride[2], head_stride[2];
  int heads, dim, tokens_per_cta;
};

// Eight values of a row, as they come.
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T *p) {
    if constexpr (sizeof(T) == 1) {
      const uint2 a = *reinterpret_cast<const uint2 *>(p);
      w[0] = a.x, w[1] = a.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 a = reinterpret_cast<const uint4 *>(p)[i / 4];
        w[i] = a.x, w[i + 1] = a.y, w[i + 2] = a.z, w[i + 3] = a.w;
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 1) {
      // A biased byte beside 0x4b0000 is 2^23 + it.
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t b = w[i / 4] ^ 0x80808080u;
        v[i] = __uint_as_float(__byte_perm(b, 0x4b000000u, 0x7650 + i % 4)) - 8388736.f;
      }
    } else {
      const T *t = reinterpret_cast<const T *>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(t[i]);
    }
  }
};
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8]) {
  struct alignas(16) Vec {
    T t[16 / sizeof(T)];
  };
#pragma unroll
  for (int u = 0; u < static_cast<int>(sizeof(T) / 2); ++u) {
    Vec x;
#pragma unroll
    for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) x.t[i] = T(v[u * (16 / sizeof(T)) + i]);
    reinterpret_cast<Vec *>(p)[u] = x;
  }
}

// STORE: rows of type X into pages of type C; else the other way.
template <bool STORE, typename C, typename X, int LANES>
__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(const __grid_constant__ CopyParams p) {
  __shared__ int page[kMostTokens];         // -1: nothing to do; -2: reads as zeros
  __shared__ int64_t at[kMostTokens][4];    // where the token's rows begin in the pages of keys and values, and the scales'
  griddep_launch_dependents();
  griddep_wait();
  const int token0 = blockIdx.x * p.tokens_per_cta, tokens = min(p.tokens_per_cta, p.seqs.tokens - token0);
  if (static_cast<int>(threadIdx.x) < tokens) {
    const int token = token0 + threadIdx.x;
    int b = token;
    page[threadIdx.x] = -1;
    if (p.seqs.starts) {
      // The last sequence that starts at the token or before it (empty ones end there too, and come before).
      int lo = 0, hi = p.seqs.batch;  // starts[lo] <= token < starts[hi], if the starts rise
      const int end = p.seqs.starts[hi];
      if (end > p.seqs.tokens) raise_status(kStatusKvBadStarts);
      if (p.seqs.starts[0] <= token && token < end) {
        while (hi - lo > 1) {
          const int mid = (lo + hi) / 2;
          if (p.seqs.starts[mid] <= token)
            lo = mid;
          else
            hi = mid;
        }
        b = lo;
      } else {
        b = -1;  // before the first sequence or behind the last
      }
    }
    if (b >= 0) {
      const Seq s = sequence<false>(p.seqs, b);
      const int i = token - s.first, position = s.pos0 + i;
      if (i < 0 || i >= s.n) {  // starts that do not rise
      } else if (position >= 0 && position < s.length) {
        const int id = page_of(p.seqs, b, position);
        page[threadIdx.x] = id >= 0 ? id : STORE ? -1 : -2;
        const int row = position & ((1 << p.seqs.page_log2) - 1);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          at[threadIdx.x][w] = id * p.stride[w][0] + row * p.stride[w][2];
          at[threadIdx.x][2 + w] = id * p.scale_stride[w][0] + row * p.scale_stride[w][2];
        }
      } else if (!STORE) {
        page[threadIdx.x] = -2;
      }
    }
  }
  __syncthreads();
  // A thread has one piece of a token's rows, the same for each of its tokens, so that a token costs it one addition per
  // address; kAhead of them are fetched before the first is written.
  const int pieces = 2 * p.heads * LANES, side = pieces < kCopyThreads ? kCopyThreads / pieces : 1;  // side: tokens side by side
  const int mine = side > 1 ? threadIdx.x / pieces : 0, lane = threadIdx.x % LANES;
  if (mine >= side) return;
  const bool in = lane * 8 < p.dim;
  for (int piece = side > 1 ? threadIdx.x - mine * pieces : threadIdx.x; piece < pieces; piece += kCopyThreads) {
    const int r = piece / LANES, which = r >= p.heads, head = r - which * p.heads;
    const int64_t xs = p.token_stride[which];
    X *const x = static_cast<X *>(p.rows[which]) + token0 * xs + head * p.head_stride[which] + lane * 8;
    C *const c = static_cast<C *>(p.pages[which]) + head * p.stride[which][1] + lane * 8;
    float *const s = sizeof(C) == 1 ? p.scales[which] + head * p.scale_stride[which][1] : nullptr;
    for (int base = mine; base < tokens; base += side * kAhead) {
      Eight<typename std::conditional<STORE, X, C>::type> raw[kAhead];
      float scale[kAhead];
      int id[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = base + u * side;
        id[u] = i < tokens ? page[i] : -1;
        if (STORE ? id[u] == -1 : id[u] < 0) continue;
        if constexpr (STORE) {
          if (in) raw[u].load(x + i * xs);
        } else {
          if (in) raw[u].load(c + at[i][which]);
          if (sizeof(C) == 1) scale[u] = s[at[i][2 + which]];
        }
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (id[u] == -1) continue;  // (a row's lanes go together)
        const int i = base + u * side;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 0.f;
        if (in && (STORE || id[u] >= 0)) raw[u].get(v);
        if constexpr (!STORE) {
          if (sizeof(C) == 1 && id[u] >= 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= scale[u];
          }
          if (in) store8(x + i * xs, v);
        } else if constexpr (sizeof(C) == 1) {
          float a = 0.f;
          bool bad = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e])), bad |= !(fabsf(v[e]) < INFINITY);
          const unsigned lanes = ((1u << LANES) - 1) << (threadIdx.x % 32 / LANES * LANES);
#pragma unroll
          for (int o = LANES / 2; o; o >>= 1) a = fmaxf(a, __shfl_xor_sync(lanes, a, o));
          bad = __ballot_sync(lanes, bad) != 0;
          if (lane == 0) s[at[i][2 + which]] = bad ? NAN : a / 127.f;
          // A maximum below 1e-30 is lifted by 2^80 (exact) first, so 127 / a stays finite.
          const float lift = a < 1e-30f ? 0x1p80f : 1.f;
          const float f = bad || a == 0.f ? 0.f : 127.f / (a * lift);
          uint32_t w[2] = {0, 0};
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int n = bad ? 0 : __float2int_rn((v[e] * lift) * f);
            w[e / 4] |= (static_cast<uint32_t>(n) & 0xff) << (8 * (e % 4));
          }
          if (in) *reinterpret_cast<uint2 *>(c + at[i][which]) = make_uint2(w[0], w[1]);
        } else {
          if (in) store8(c + at[i][which], v);
        }
      }
    }
  }
}

template <bool STORE, typename C, typename X>
int launch_copy(CopyParams &p, int sms, cudaStream_t s, const char *what) {
  const int lanes = p.dim <= 64 ? 8 : 16;
  // A token's place takes a chain of loads, so a CTA looks up many at once, as long as there are CTAs for every SM: four or so
  // of 16-byte pieces a thread for few tokens.
  const int64_t threads = 2LL * p.heads * lanes;  // of a token
  const int64_t least = std::max<int64_t>(1, 4 * kCopyThreads / threads), fill = p.seqs.tokens / (16LL * sms);
  p.tokens_per_cta = static_cast<int>(std::min<int64_t>(kMostTokens, std::max(least, fill)));
  const dim3 grid((p.seqs.tokens + p.tokens_per_cta - 1) / p.tokens_per_cta);
  if (lanes == 8) return launch_overlapped(kv_copy_kernel<STORE, C, X, 8>, grid, dim3(kCopyThreads), 0, s, what, p);
  return launch_overlapped(kv_copy_kernel<STORE, C, X, 16>, grid, dim3(kCopyThreads), 0, s, what, p);
}
template <bool STORE, typename C>
int copy_by_rows(CopyParams &p, int dtype, int sms, cudaStream_t s, const char *what) {
  if (dtype == MQ_F32) return launch_copy<STORE, C, float>(p, sms, s, what);
  if (dtype == MQ_F16) return launch_copy<STORE, C, __half>(p, sms, s, what);
  return launch_copy<STORE, C, __nv_bfloat16>(p, sms, s, what);
}

// Whether a cache's keys, values and scales share a byte with one another.
inline bool cache_overlaps(const mq_kv_pages *c) {
  Area a[4];
  const int n = areas_of(c, a);
  for (int i = 0; i < n; ++i)
    for (int j = 0; j < i; ++j)
      if (share_bytes(a[i], a[j])) return true;
  return false;
}

template <bool STORE>
int kv_copy(void *k, int64_t k_token, int64_t k_head, void *v, int64_t v_token, int64_t v_head, int dtype, const mq_kv_pages *c,
            const int32_t *table, int64_t ldt, int64_t width, const int32_t *lengths, const int32_t *starts, int64_t batch,
            int64_t tokens, void *stream, const char *what) {
  if (int rc = check_cache(c, what)) return rc;
  CopyParams p{};
  if (int rc = check_seqs(&p.seqs, c, table, ldt, width, lengths, starts, batch, tokens, what)) return rc;
  MQ_REQUIRE(dtype == MQ_F32 || dtype == MQ_F16 || dtype == MQ_BF16, MQ_EINVAL, "%s: rows must be MQ_F32, MQ_F16 or MQ_BF16", what);
  if (batch == 0 || tokens == 0) return MQ_OK;
  MQ_REQUIRE(tokens * c->heads < (1LL << 31), MQ_EUNSUPPORTED, "%s: too many rows", what);
  if (STORE) {
    if (int rc = check_rows(k, dtype, k_token, k_head, "k", what)) return rc;
    if (int rc = check_rows(v, dtype, v_token, v_head, "v", what)) return rc;
    MQ_REQUIRE(!cache_overlaps(c), MQ_EINVAL, "%s: keys and values, or their scales, share memory", what);
  } else {
    if (int rc = check_rows_out(k, dtype, tokens, c->heads, c->dim, k_token, k_head, "k", what)) return rc;
    if (int rc = check_rows_out(v, dtype, tokens, c->heads, c->dim, v_token, v_head, "v", what)) return rc;
    const int64_t es = element_size(dtype);
    const Area rows_k = area_of_rows(k, es, tokens, c->heads, c->dim, k_token, k_head), rows_v = area_of_rows(v, es, tokens, c->heads, c->dim, v_token, v_head);
    MQ_REQUIRE(!share_bytes(rows_k, rows_v), MQ_EINVAL, "%s: k and v share memory", what);
    Area held[4];
    for (int i = areas_of(c, held) - 1; i >= 0; --i)
      MQ_REQUIRE(!share_bytes(rows_k, held[i]) && !share_bytes(rows_v, held[i]), MQ_EINVAL, "%s: k or v shares memory with the pages", what);
  }
  mq::DeviceInfo dev;
  if (int rc = device_info(&dev)) return rc;
  p.pages[0] = c->k, p.pages[1] = c->v, p.scales[0] = c->k_scale, p.scales[1] = c->v_scale;
  for (int i = 0; i < 3; ++i) {
    p.stride[0][i] = c->k_stride[i], p.stride[1][i] = c->v_stride[i];
    p.scale_stride[0][i] = c->ks_stride[i], p.scale_stride[1][i] = c->vs_stride[i];
  }
  p.rows[0] = k, p.rows[1] = v;
  p.token_stride[0] = k_token, p.token_stride[1] = v_token, p.head_stride[0] = k_head, p.head_stride[1] = v_head;
  p.heads = c->heads, p.dim = c->dim;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (c->dtype == MQ_S8) return copy_by_rows<STORE, int8_t>(p, dtype, dev.sms, s, what);
  if (c->dtype == MQ_F16) return copy_by_rows<STORE, __half>(p, dtype, dev.sms, s, what);
  return copy_by_rows<STORE, __nv_bfloat16>(p, dtype, dev.sms, s, what);
}

}  // namespace paged
}  // namespace mq

extern "C" int mq_kv_store(const void *k, int64_t k_token, int64_t k_head, const void *v, int64_t v_token, int64_t v_head,
                           int dtype, const mq_kv_pages *cache, const int32_t *table, int64_t ldt, int64_t width,
                           const int32_t *lengths, const int32_t *starts, int64_t batch, int64_t tokens, void *stream) {
  return mq::paged::kv_copy<true>(const_cast<void *>(k), k_token, k_head, const_cast<void *>(v), v_token, v_head, dtype, cache,
                                  table, ldt, width, lengths, starts, batch, tokens, stream, "mq_kv_store");
}

extern "C" int mq_kv_load(const mq_kv_pages *cache, const int32_t *table, int64_t ldt, int64_t width, const int32_t *lengths,
                          const int32_t *starts, int64_t batch, int64_t tokens, void *k, int64_t k_token, int64_t k_head, void *v,
                          int64_t v_token, int64_t v_head, int dtype, void *stream) {
  return mq::paged::kv_copy<false>(k, k_token, k_head, v, v_token, v_head, dtype, cache, table, ldt, width, lengths, starts,
                                   batch, tokens, stream, "mq_kv_load");
}
