// What the operators on a paged cache share: the host's checks of a cache and its tensor maps, and the device's view of
// sequences, their pages and the split of a launch's work.
//
// Sequence b has rows starts[b] .. starts[b + 1] of the tokens (row b where starts is NULL) and lengths[b] positions in
// the cache, its new tokens' among them: row r is position lengths[b] - (starts[b + 1] - r), whether or not all of these rows
// are there. Position p lies in page table[b][p / page], row p % page.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace mq {
namespace paged {

constexpr int kMaxDim = 128, kMinPage = 16, kMaxPage = 256;

struct Seqs {
  const int32_t *table, *lengths, *starts;
  int64_t ldt;
  int batch, tokens, width, page_log2;
  int pages;  // of the pool
};

struct Seq {
  int first, n;  // its rows
  int length;    // positions in the cache
  int pos0;      // position of its first row; negative where it has more rows than positions
};

// Rows that are not there (before the first, behind the last: reported) are left out, the others keep their positions. Starts that
// fall make an empty sequence. Lengths that pass the table are reported and cut; the copies' rows keep their positions, beyond
// the table for some, which are then left out. The attention's (ATTEND) count from the cut length, and an end that can be none,
// with more rows than the table has positions and none of those that are there at one of them, counts as the rows' end.
template <bool ATTEND>
__device__ __forceinline__ Seq sequence(const Seqs &s, int b) {
  Seq q;
  const int length = s.lengths[b], most = s.width << s.page_log2;
  q.length = min(max(length, 0), most);
  if (q.length != length) raise_status(kStatusKvBadLength);
  const int last = ATTEND ? q.length : max(length, 0);
  q.first = b, q.n = 1, q.pos0 = last - 1;
  if (s.starts) {
    q.first = min(max(s.starts[b], 0), s.tokens);
    int end = max(s.starts[b + 1], q.first);
    q.n = min(end, s.tokens) - q.first;
    if (end > s.tokens) {
      if (ATTEND && q.n > 0 && end - q.first > most && end - s.tokens >= q.length)
        end = s.tokens;
      else
        raise_status(kStatusKvBadStarts);
    }
    // (The bound keeps what is added to and taken from it in range; it is below 0 as far as there are rows.)
    q.pos0 = max(last - (end - q.first), -(1 << 30));
  }
  return q;
}

// The page that holds a position of sequence b: -1 (reported) where the table names none of the pool's.
__device__ __forceinline__ int page_of(const Seqs &s, int b, int position) {
  const int id = s.table[b * s.ldt + (position >> s.page_log2)];
  if (static_cast<unsigned>(id) < static_cast<unsigned>(s.pages)) return id;
  raise_status(kStatusKvBadPage);
  return -1;
}

// mbar_wait in fewer instructions: a role waits in many places, and code that is not in the instruction cache yet costs
// a short call more than the waiting.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer();
  do {
    if (mbar_try_wait(bar, parity)) return true;
  } while (globaltimer() - t0 < kWaitTimeoutNs);
  return false;
}

// ---- host: checks -----------------------------------------------------------------------------------

inline int element_size(int dtype) { return dtype == MQ_F32 ? 4 : dtype == MQ_S8 ? 1 : 2; }
inline int log2_of(int v) { return 31 - __builtin_clz(static_cast<unsigned>(v)); }

// Every (page, head, position) row needs bytes of its own: by rising stride, each dimension steps over all that the
// ones before cover. `row`: elements of a row.
inline bool rows_apart(const int64_t *stride, int64_t pages, int64_t heads, int64_t page, int64_t row) {
  int64_t size[3] = {pages, heads, page};
  int order[3] = {0, 1, 2};
  std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
  int64_t extent = row;
  for (int d : order) {
    if (size[d] == 1) continue;
    if (stride[d] < extent || stride[d] >= (1LL << 40) / size[d]) return false;
    extent += stride[d] * (size[d] - 1);
  }
  return true;
}

inline int check_cache(const mq_kv_pages *c, const char *what) {
  MQ_REQUIRE(c && c->k && c->v, MQ_EINVAL, "%s: null pointer", what);
  MQ_REQUIRE(c->dtype == MQ_F16 || c->dtype == MQ_BF16 || c->dtype == MQ_S8, MQ_EINVAL,
             "%s: the cache's type must be MQ_F16, MQ_BF16 or MQ_S8", what);
  MQ_REQUIRE(c->pages > 0 && c->pages < (1LL << 31) && c->heads > 0 && c->heads <= 65535, MQ_EINVAL, "%s: bad number of pages or heads",
             what);
  MQ_REQUIRE(c->page >= kMinPage && c->page <= kMaxPage && (c->page & (c->page - 1)) == 0, MQ_EUNSUPPORTED,
             "%s: a page must hold 16, 32, 64, 128 or 256 positions", what);
  MQ_REQUIRE(c->dim >= 16 && c->dim <= kMaxDim && c->dim % 16 == 0, MQ_EUNSUPPORTED,
             "%s: dim must be a multiple of 16 up to %d", what, kMaxDim);
  const int es = element_size(c->dtype);
  for (int i = 0; i < 3; ++i)
    MQ_REQUIRE(c->k_stride[i] * es % 16 == 0 && c->v_stride[i] * es % 16 == 0, MQ_EALIGN,
               "%s: every row of the cache must start 16-byte aligned", what);
  MQ_REQUIRE(aligned(c->k, 16) && aligned(c->v, 16), MQ_EALIGN, "%s: every row of the cache must start 16-byte aligned", what);
  MQ_REQUIRE(rows_apart(c->k_stride, c->pages, c->heads, c->page, c->dim) &&
                 rows_apart(c->v_stride, c->pages, c->heads, c->page, c->dim),
             MQ_EINVAL, "%s: rows of the cache overlap", what);
  if (c->dtype == MQ_S8) {
    MQ_REQUIRE(c->k_scale && c->v_scale, MQ_EINVAL, "%s: an int8 cache needs its scales", what);
    MQ_REQUIRE(aligned(c->k_scale, 4) && aligned(c->v_scale, 4), MQ_EALIGN, "%s: scales must be 4-byte aligned", what);
    MQ_REQUIRE(rows_apart(c->ks_stride, c->pages, c->heads, c->page, 1) && rows_apart(c->vs_stride, c->pages, c->heads, c->page, 1),
               MQ_EINVAL, "%s: scales of the cache overlap", what);
  }
  return MQ_OK;
}

inline int check_seqs(Seqs *s, const mq_kv_pages *c, const int32_t *table, int64_t ldt, int64_t width, const int32_t *lengths,
                      const int32_t *starts, int64_t batch, int64_t tokens, const char *what) {
  MQ_REQUIRE(batch >= 0 && tokens >= 0 && width >= 0, MQ_EINVAL, "%s: bad shape", what);
  MQ_REQUIRE(batch < (1LL << 22) && tokens < (1LL << 30), MQ_EUNSUPPORTED, "%s: too many sequences or tokens", what);
  MQ_REQUIRE(width <= ((1LL << 31) - 1024) / c->page, MQ_EUNSUPPORTED, "%s: the table's rows name too many positions", what);
  MQ_REQUIRE(starts || tokens == batch, MQ_EINVAL, "%s: without starts every sequence has one row", what);
  if (batch > 0 && tokens > 0) {
    MQ_REQUIRE(lengths && (table || width == 0), MQ_EINVAL, "%s: null pointer", what);
    MQ_REQUIRE(aligned(table, 4) && aligned(lengths, 4) && aligned(starts, 4), MQ_EALIGN, "%s: the table, lengths and starts must be 4-byte aligned",
               what);
    MQ_REQUIRE(ldt >= width || batch == 1, MQ_EINVAL, "%s: the table's row stride is less than its width", what);
  }
  *s = Seqs{table, lengths, starts, ldt, static_cast<int>(batch), static_cast<int>(tokens), static_cast<int>(width),
            log2_of(c->page), static_cast<int>(c->pages)};
  return MQ_OK;
}

// Rows [tokens][heads][dim] of a strided tensor (strides in elements), each 16-byte aligned.
inline int check_rows(const void *p, int dtype, int64_t token_stride, int64_t head_stride, const char *name, const char *what) {
  MQ_REQUIRE(p, MQ_EINVAL, "%s: null pointer", what);
  const int es = element_size(dtype);
  MQ_REQUIRE(aligned(p, 16) && token_stride * es % 16 == 0 && head_stride * es % 16 == 0, MQ_EALIGN,
             "%s: every row of %s must start 16-byte aligned", what, name);
  MQ_REQUIRE(token_stride >= 0 && head_stride >= 0, MQ_EINVAL, "%s: %s has a negative stride", what, name);
  return MQ_OK;
}
// The same of rows that are written: none may share bytes with another.
inline int check_rows_out(const void *p, int dtype, int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride,
                          int64_t head_stride, const char *name, const char *what) {
  if (int rc = check_rows(p, dtype, token_stride, head_stride, name, what)) return rc;
  const int64_t stride[3] = {token_stride, head_stride, 0};
  MQ_REQUIRE(rows_apart(stride, tokens, heads, 1, dim), MQ_EINVAL, "%s: rows of %s overlap", what, name);
  return MQ_OK;
}

// ---- host: what shares memory ------------------------------------------------------------------------

// Rows of `row` bytes, [size[0]][size[1]][size[2]] of them, strides in bytes (0 or more).
struct Area {
  const char *base;
  __int128 row, stride[3];
  int64_t size[3];
  __int128 extent() const {
    __int128 e = row;
    for (int i = 0; i < 3; ++i) e += stride[i] * (size[i] - 1);
    return e;
  }
  // The same bytes, dimensions by falling stride and as few as will do: the others have size 1 and stride 0.
  Area plain() const {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] > stride[b]; });
    Area a{base, row, {0, 0, 0}, {1, 1, 1}};
    int n = 0;
    for (int d : order) {
      if (size[d] == 1 || stride[d] == 0) continue;
      if (n > 0 && a.stride[n - 1] == stride[d] * size[d])  // one dimension of both
        a.stride[n - 1] = stride[d], a.size[n - 1] *= size[d];
      else
        a.stride[n] = stride[d], a.size[n++] = size[d];
    }
    if (n > 0 && a.stride[n - 1] == row) a.row = row * a.size[n - 1], a.stride[n - 1] = 0, a.size[n - 1] = 1;
    return a;
  }
  // Whether a row, of a plain area whose rows lie apart, has a byte in [at, at + bytes) behind the base. Rows rise in the
  // order of their dimensions, so the last row that starts before the end is the only one to look at.
  bool has(__int128 at, __int128 bytes) const {
    __int128 rest = at + bytes - 1;
    if (rest < 0) return false;
    for (int i = 0; i < 3; ++i)
      if (stride[i] > 0) rest -= stride[i] * std::min<__int128>(size[i] - 1, rest / stride[i]);
    return rest - (bytes - 1) < row;
  }
};
// The dimensions of two areas by falling stride, with the size that each has there (1: not one of its own).
struct Both {
  int n;
  __int128 stride[6], rest[7];  // rest[d]: the larger extent of what lies within dimension d - 1
  int64_t a[6], b[6];
};
// Whether a row of a and one of b, `delta` bytes behind it so far, share a byte. A stride is at least the extent of what follows, so
// only the two multiples of it around what is left can bring them together.
inline bool rows_meet(const Both &p, __int128 row_a, __int128 row_b, int d, __int128 delta) {
  if (d == p.n) return delta < row_a && -delta < row_b;
  __int128 i = delta / p.stride[d];
  if (i * p.stride[d] > delta) --i;
  for (int k = 0; k < 2; ++k, ++i) {
    const __int128 left = delta - i * p.stride[d];
    if (i < p.a[d] && -i < p.b[d] && left < p.rest[d + 1] && -left < p.rest[d + 1] && rows_meet(p, row_a, row_b, d + 1, left)) return true;
  }
  return false;
}
// Whether two areas share a byte. The rows of `apart` lie apart (rows_apart); those of the other need not. Two that lie between one
// another in strides that do not go together are compared row by row, as far as kMostCompared: beyond, they count as apart.
constexpr int64_t kMostCompared = 4096;
inline bool share_bytes(const Area &any, const Area &apart) {
  const __int128 delta = static_cast<__int128>(reinterpret_cast<intptr_t>(apart.base)) - reinterpret_cast<intptr_t>(any.base);
  if (delta >= any.extent() || -delta >= apart.extent()) return false;  // (nearly always)
  const Area a = any.plain(), b = apart.plain();
  Both p{};
  for (int i = 0, j = 0; (i < 3 && a.stride[i] > 0) || (j < 3 && b.stride[j] > 0); ++p.n) {
    const __int128 x = i < 3 ? a.stride[i] : 0, y = j < 3 ? b.stride[j] : 0;
    p.stride[p.n] = std::max(x, y);
    p.a[p.n] = x == p.stride[p.n] ? a.size[i++] : 1;
    p.b[p.n] = y == p.stride[p.n] ? b.size[j++] : 1;
  }
  bool regular = true;
  p.rest[p.n] = std::max(a.row, b.row);
  for (int d = p.n - 1; d >= 0; --d) {
    regular = regular && p.stride[d] >= p.rest[d + 1];
    p.rest[d] = p.rest[d + 1] + p.stride[d] * (std::max(p.a[d], p.b[d]) - 1);
  }
  if (regular) return rows_meet(p, a.row, b.row, 0, delta);
  int64_t left = kMostCompared;
  for (int64_t x = 0; x < a.size[0] && left > 0; ++x)
    for (int64_t y = 0; y < a.size[1] && left > 0; ++y)
      for (int64_t z = 0; z < a.size[2] && left > 0; ++z, --left)
        if (b.has(x * a.stride[0] + y * a.stride[1] + z * a.stride[2] - delta, a.row)) return true;
  return false;
}

inline Area area_of_pages(const mq_kv_pages *c, const void *base, const int64_t *stride, int64_t es, int64_t row) {
  const __int128 bytes = es;
  return {static_cast<const char *>(base), row * es, {stride[0] * bytes, stride[1] * bytes, stride[2] * bytes}, {c->pages, c->heads, c->page}};
}
// A cache's keys, values and, int8, their scales: how many areas.
inline int areas_of(const mq_kv_pages *c, Area (&a)[4]) {
  const int64_t es = element_size(c->dtype);
  a[0] = area_of_pages(c, c->k, c->k_stride, es, c->dim), a[1] = area_of_pages(c, c->v, c->v_stride, es, c->dim);
  if (c->dtype != MQ_S8) return 2;
  a[2] = area_of_pages(c, c->k_scale, c->ks_stride, 4, 1), a[3] = area_of_pages(c, c->v_scale, c->vs_stride, 4, 1);
  return 4;
}
inline Area area_of_rows(const void *base, int64_t es, int64_t tokens, int64_t heads, int64_t dim, int64_t token_stride, int64_t head_stride) {
  const __int128 bytes = es;
  return {static_cast<const char *>(base), dim * es, {token_stride * bytes, head_stride * bytes, 0}, {tokens, heads, 1}};
}

// ---- attention: items, units and shares --------------------------------------------------------------

// The rows of one kv head of a sequence are its tokens' `group` query heads, token by token: row r is head r % group of
// token r / group. An item is ROWS of them and the blocks of KEYS positions that any of them sees. Its units are its blocks
// and EXTRA more before them, for what an item costs beside its blocks. Units are numbered by sequence, kv head, row tile and
// block, and the launch's CTAs take equal shares of them, whatever the sequences' lengths: an item may be cut between CTAs, which
// then leave its parts to be joined.
struct Shape {
  int group, kv_heads, window;
  int rows_from, rows_to;  // the sequences of this launch: those with rows_from < rows <= rows_to
  int rows_most;           // a sequence with more was not announced: reported, and left out by every launch
  uint32_t by_group, by_group_shift;
};
// x / group for 0 <= x < 2^31: with k = 31 + ceil(log2(group)), ceil(2^k / group) x >> k is exact.
inline void set_group(Shape *a, int group) {
  int log = 0;
  while ((1 << log) < group) ++log;
  a->group = group, a->by_group_shift = 31 + log;
  a->by_group = static_cast<uint32_t>(((1ull << a->by_group_shift) + group - 1) / group);
}
__device__ __forceinline__ int over_group(const Shape &a, int x) {
  return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(x)) * a.by_group >> a.by_group_shift);
}

template <int R, int K, int E>
struct Grain {
  static constexpr int ROWS = R, KEYS = K, EXTRA = E;
};
struct Range {
  int lo, blocks;  // the first block, how many (one, with nothing in it, where no row sees a key)
};
template <typename G>
__device__ __forceinline__ Range tile_range(const Seq &s, const Shape &a, int t) {
  const int rows = s.n * a.group;
  const int i0 = over_group(a, t * G::ROWS), i1 = over_group(a, min(rows, (t + 1) * G::ROWS) - 1);
  const int hi = min(max(s.pos0 + i1 + 1, 0), s.length), lo = a.window ? max(0, s.pos0 + i0 + 1 - a.window) : 0;
  const int b0 = min(lo, max(hi - 1, 0)) / G::KEYS;
  return {b0, max(1, (hi + G::KEYS - 1) / G::KEYS - b0)};
}
__device__ __forceinline__ bool takes_part(const Seq &s, const Shape &a) {
  const int64_t rows = static_cast<int64_t>(s.n) * a.group;
  return rows > a.rows_from && rows <= a.rows_to;
}
template <typename G>
__device__ __forceinline__ int tiles_of(const Seq &s, const Shape &a) {
  return (s.n * a.group + G::ROWS - 1) / G::ROWS;
}

struct Share {
  int64_t total, begin, end;  // units of the launch, and of this CTA
  int parts;                  // CTAs with a share
  int b, head, tile, rest;    // where it begins: `rest` units into that item
  Seq s;                      // sequence b
};
// total * i / parts, without a 64-bit division where none is needed (they are a subroutine of a hundred instructions).
__device__ __forceinline__ int64_t portion(int64_t total, int i, int parts) {
  if (total < (1 << 21) && i <= 1023) return static_cast<uint32_t>(total) * static_cast<uint32_t>(i) / static_cast<uint32_t>(parts);
  return total * i / parts;
}
template <int THREADS>
struct ShareScratch {
  int64_t costs[THREADS];  // units of THREADS sequences
  int64_t sums[THREADS / 32];
  Share found;
};

// This CTA's share, in sm.found; called by all THREADS threads. parts <= blockIdx.x: none.
template <int THREADS, typename G>
__device__ __forceinline__ void find_share(const Seqs &s, const Shape &a, ShareScratch<THREADS> &sm) {
  constexpr int kWarps = THREADS / 32;
  constexpr bool kOneTile = G::ROWS <= 64;  // a sequence has one tile at most
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  int64_t total = 0;
  Seq own{};  // the last sequence this thread (with one tile each) or its warp looked at
  // Twice through the sequences, THREADS at a time: for the total, and for the one in which the share begins. Once where
  // one step takes all.
  for (int pass = s.batch <= THREADS ? 1 : 0; pass < 2; ++pass) {
    int64_t before = 0;
    for (int base = 0; base < s.batch; base += THREADS) {
      int64_t cost = 0;
      if (kOneTile) {
        if (base + tid < s.batch) {
          const Seq q = own = sequence<true>(s, base + tid);
          if (static_cast<int64_t>(q.n) * a.group > a.rows_most) raise_status(kStatusAttnTooManyRows);
          if (takes_part(q, a)) cost = static_cast<int64_t>(G::EXTRA + tile_range<G>(q, a, 0).blocks) * a.kv_heads;
        }
      } else {  // a warp for a sequence, its lanes for the tiles
        for (int b = warp; b < min(THREADS, s.batch - base); b += kWarps) {
          const Seq q = sequence<true>(s, base + b);
          int64_t units = 0;
          if (static_cast<int64_t>(q.n) * a.group > a.rows_most) raise_status(kStatusAttnTooManyRows);
          if (takes_part(q, a))
            for (int t = lane, tiles = tiles_of<G>(q, a); t < tiles; t += 32) units += G::EXTRA + tile_range<G>(q, a, t).blocks;
#pragma unroll
          for (int o = 16; o; o >>= 1) units += __shfl_xor_sync(0xffffffffu, units, o);
          if (lane == 0) sm.costs[b] = units * a.kv_heads;
        }
        __syncthreads();
        if (base + tid < s.batch) cost = sm.costs[tid];
      }
      int64_t incl = cost;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      if (lane == 31) sm.sums[warp] = incl;
      __syncthreads();
      int64_t start = before + incl - cost;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int64_t sum = sm.sums[w];
        if (w < warp) start += sum;
        before += sum;
      }
      if (s.batch <= THREADS) total = before;
      if (pass == 1) {
        const int parts = static_cast<int>(total < gridDim.x ? total : gridDim.x);
        if (base == 0 && tid == 0) sm.found.total = total, sm.found.parts = parts;
        if (static_cast<int>(blockIdx.x) < parts) {
          const int64_t begin = portion(total, blockIdx.x, parts);
          // The warp with the sequence in which the share begins finds the tile.
          const unsigned here = __ballot_sync(0xffffffffu, start <= begin && begin < start + cost);
          if (here) {
            const int from = __ffs(here) - 1, b = base + warp * 32 + from;
            const int64_t all = __shfl_sync(0xffffffffu, cost, from);
            int64_t rest = begin - __shfl_sync(0xffffffffu, start, from), per_head;
            int head;
            if (all < (1LL << 31)) {
              per_head = static_cast<uint32_t>(all) / static_cast<uint32_t>(a.kv_heads);
              head = static_cast<uint32_t>(rest) / static_cast<uint32_t>(per_head);
            } else {
              per_head = all / a.kv_heads;
              head = static_cast<int>(rest / per_head);
            }
            rest -= head * per_head;
            Seq q = own;
            q.first = __shfl_sync(0xffffffffu, q.first, from), q.n = __shfl_sync(0xffffffffu, q.n, from);
            q.length = __shfl_sync(0xffffffffu, q.length, from), q.pos0 = __shfl_sync(0xffffffffu, q.pos0, from);
            int tile = 0;
            if (!kOneTile) {
              q = sequence<true>(s, b);
              for (const int tiles = tiles_of<G>(q, a);; tile += 32) {
                const int t = tile + lane;
                const int64_t units = t < tiles ? G::EXTRA + tile_range<G>(q, a, t).blocks : 0;
                int64_t sum = units;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                  const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
                  if (lane >= o) sum += up;
                }
                const unsigned in = __ballot_sync(0xffffffffu, rest < sum);
                if (in) {  // (the units of all tiles are more than `rest`, so some lane's is)
                  const int l = __ffs(in) - 1;
                  rest -= __shfl_sync(0xffffffffu, sum - units, l);
                  tile += l;
                  break;
                }
                rest -= __shfl_sync(0xffffffffu, sum, 31);
              }
            }
            if (lane == 0) {
              sm.found.begin = begin, sm.found.end = portion(total, blockIdx.x + 1, parts);
              sm.found.s = q;
              sm.found.b = b, sm.found.head = head, sm.found.tile = tile, sm.found.rest = static_cast<int>(rest);
            }
          }
        }
      }
      __syncthreads();
    }
    total = before;
  }
}

struct Item {
  Seq s;
  int b, head, tile;
  int block, blocks;  // of this CTA
  int before, whole;  // blocks of the item before them, blocks of the item
};

// Walks through a share's items: the warp that brings keys and values does, and tells the others.
template <typename G>
struct Walk {
  Seq s;
  int b, head, tile, tiles, rest;
  int64_t left;
  __device__ __forceinline__ void start(const Shape &a, const Share &share) {
    b = share.b, head = share.head, tile = share.tile, rest = share.rest, left = share.end - share.begin;
    s = share.s;
    tiles = tiles_of<G>(s, a);
  }
  __device__ __forceinline__ bool next(const Seqs &q, const Shape &a, Item &item) {
    if (left <= 0) return false;
    if (tile == tiles) {
      tile = 0;
      if (++head == a.kv_heads) {
        head = 0;
        do s = sequence<true>(q, ++b);
        while (!takes_part(s, a));  // (units are left, so such a sequence follows)
        tiles = tiles_of<G>(s, a);
      }
    }
    const Range r = tile_range<G>(s, a, tile);
    const int take = static_cast<int>(left < G::EXTRA + r.blocks - rest ? left : G::EXTRA + r.blocks - rest);
    item.s = s, item.b = b, item.head = head, item.tile = tile;
    item.before = max(rest - G::EXTRA, 0), item.whole = r.blocks, item.block = r.lo + item.before;
    item.blocks = rest + take - G::EXTRA - item.before;
    left -= take;
    rest = 0;
    ++tile;
    return item.blocks > 0;  // (a share may end before the first block of its last item)
  }
};

// Where it does: the next item is in item[k % kItems] when its `full` barrier says so; an item without blocks ends it.
constexpr int kItems = 4;
struct ItemRing {
  Item item[kItems];
  uint64_t full[kItems], empty[kItems];
  __device__ __forceinline__ void init(int readers) {
    for (int i = 0; i < kItems; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], readers);
  }
  // By a whole warp.
  __device__ __forceinline__ bool put(int k, const Item &it) {
    if (k >= kItems && !__all_sync(0xffffffffu, wait_for(&empty[k % kItems], (k / kItems - 1) & 1))) return false;
    if (threadIdx.x % 32 == 0) {
      item[k % kItems] = it;
      mbar_arrive(&full[k % kItems]);
    }
    __syncwarp();
    return true;
  }
};

// A CTA leaves at most two parts of items that others share: one that it goes on with (slot 0) and one that it
// begins and does not end (slot 1). `cut` says which item the CTA goes on with.
struct Cut {
  int32_t token, n;  // the sequence's first row, its rows
  int32_t head, tile, goes_on, unused[3];
  int64_t first, end;  // the units of the item's blocks
};
// Of a walk that has just started.
template <typename G>
__device__ __forceinline__ Cut cut_at(const Walk<G> &w, const Shape &a, const Share &share) {
  const int64_t first = share.begin - share.rest + G::EXTRA;
  return {w.s.first, w.s.n, w.head, w.tile, share.rest > G::EXTRA, {}, first, first + tile_range<G>(w.s, a, w.tile).blocks};
}
struct Parts {
  int64_t *counts;  // units, CTAs with a share
  Cut *cuts;        // [ctas]
  float2 *stats;    // [ctas][2][rows]: the maximum that the part's sums are relative to (log2), the sum of weights
  float *sums;      // [ctas][2][rows][D]
};
inline size_t parts_bytes(int ctas, int rows, int d) {
  static_assert(sizeof(Cut) % 16 == 0, "the sums are read 16 bytes at a time");
  return 256 + static_cast<size_t>(ctas) * (sizeof(Cut) + 2ull * rows * (sizeof(float2) + 4ull * d));
}
inline Parts parts_at(void *workspace, int ctas, int rows) {
  char *p = static_cast<char *>(workspace);
  Parts parts;
  parts.counts = reinterpret_cast<int64_t *>(p);
  parts.cuts = reinterpret_cast<Cut *>(p + 256);
  parts.stats = reinterpret_cast<float2 *>(parts.cuts + ctas);
  parts.sums = reinterpret_cast<float *>(parts.stats + 2ull * ctas * rows);
  return parts;
}

struct Output {
  void *out;
  int64_t token_stride, head_stride;
  int dtype, dim;
};

}  // namespace paged
}  // namespace mq
