// Attention of a batch of sequences over a paged key/value cache, with the
// positions that all sequences share read once for all of them.
#include <math.h>

#include "common.cuh"
#include "paged.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace ipuc {

ipuc_status check_paged(const char *who, const ipuc_paged_cache *cache, const ipuc_paged_batch *batch) {
  const std::string w = who;
  IPUC_CHECK_ARG(cache && batch, w + ": null cache or batch");
  IPUC_CHECK_ARG(cache->heads >= 1 && cache->heads < (1 << 16) && cache->head_dim >= 1 && cache->page_size >= 1 &&
                     cache->pages >= 1 && cache->pages < (1ll << 31),
                 w + ": cache extent out of range");
  IPUC_CHECK_ARG(cache->row_stride >= cache->head_dim && cache->head_stride >= cache->head_dim &&
                     cache->page_stride >= cache->head_dim && cache->row_stride < (1ll << 40) &&
                     cache->head_stride < (1ll << 40) && cache->page_stride < (1ll << 40),
                 w + ": cache stride out of range");
  IPUC_CHECK_ARG(batch->sequences >= 0 && batch->rows >= 0 && batch->rows < (1ll << 31) && batch->max_pages >= 0,
                 w + ": batch extent out of range");
  IPUC_CHECK_ARG((int64_t)batch->max_pages * cache->page_size < (1ll << 31) - 256, w + ": max_pages * page_size too large");
  IPUC_CHECK_ARG(batch->table_stride >= batch->max_pages, w + ": table stride shorter than max_pages");
  IPUC_CHECK_ARG(batch->row_offsets || batch->rows == batch->sequences,
                 w + ": without row offsets there is one row per sequence");
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  IPUC_CHECK_ARG(cache->keys && cache->values && cache->keys != cache->values, w + ": null pointer");
  IPUC_CHECK_ARG(batch->lengths && (batch->page_table || batch->max_pages == 0), w + ": null pointer");
  IPUC_CHECK_ALIGN(aligned(batch->lengths, 4) && aligned(batch->page_table, 4) && aligned(batch->row_offsets, 4),
                   w + ": int32 arrays must be 4-byte aligned");
  return IPUC_OK;
}

PagedView paged_view(const ipuc_paged_cache *c, const ipuc_paged_batch *b) {
  PagedView v;
  v.page_table = b->page_table;
  v.lengths = b->lengths;
  v.row_offsets = b->row_offsets;
  v.table_stride = b->table_stride;
  v.page_stride = c->page_stride;
  v.head_stride = c->head_stride;
  v.row_stride = c->row_stride;
  v.sequences = b->sequences;
  v.max_pages = b->max_pages;
  v.page_size = c->page_size;
  v.pages = (int32_t)c->pages;
  return v;
}

namespace {

using namespace sm100;

// Exponentials are taken relative to a running maximum that lags the true one
// by at most 2^8 (kLazy) and scaled up by 2^4 (kShift), which keeps weights
// within f16 (at most 2^12) and those down to 2^-18 of the largest normal.
// Both factors cancel in O / l as long as every partial result has them.
constexpr float kLazy = 8.0f, kShift = 4.0f;
constexpr float kLog2e = 1.4426950408889634f;

// What loading a unit's queries and storing its result costs, in key tiles: it
// takes 5 to 6 us of a CTA of the tile kernel against 2.15 for a key tile, and
// 2 to 3 us of a worker of the stream kernel against 1.2.  With 0, 1, 2, 3 and 4:
// a batch of 128 behind 32768 shared positions 189, 172, 159, 152 and 153 us,
// pieces of 8 prompts behind 4096 181, 146, 134, 122 and 122 us.
constexpr int kUnitCost = 3;
__device__ __forceinline__ int32_t unit_cost(int32_t tiles) { return tiles > 0 ? tiles + kUnitCost : 0; }

// A place on a line: offset `x` in a unit of `n` key tiles, `left` to the
// piece's end.  Tile i of the unit lies at x = kUnitCost + i.
struct LinePlace {
  int32_t x, n;
  int64_t left;
  __device__ __forceinline__ int32_t first() const { return max(0, x - kUnitCost); }
  __device__ __forceinline__ int32_t end_x() const { return (int32_t)min((int64_t)unit_cost(n), x + left); }
  // key tiles of this unit in this piece
  __device__ __forceinline__ int32_t here() const { return max(0, end_x() - kUnitCost) - first(); }
  // goes to the end of the unit or piece; true if the piece goes on in the next unit
  __device__ __forceinline__ bool pass() {
    const int32_t to = end_x();
    left -= to - x;
    x = to == unit_cost(n) ? 0 : to;
    return left > 0;
  }
};

struct PagedAttnParams {
  uint16_t *out;
  const uint16_t *q;
  PagedView paged;
  const int32_t *prefix_pages;
  int64_t q_stride, rows;
  int32_t q_heads, heads, group, head_dim, prefix;
  int32_t chunk;          // keys per TMA box: gcd(page_size, 64)
  int32_t pitch, stages;  // stream kernel: bytes of a key in shared memory, ring stages
  float scale_log2;       // softmax scale * log2(e)
  // Each kernel lays its units (rows that read the same keys of one head) on a
  // line, a unit's length being its key tiles and kUnitCost more for its start
  // and end, and cuts the line into equal pieces, one per CTA or worker.  A unit
  // that a piece ends in has several partial results: unnormalised O (f32,
  // head_dim wide) and (running maximum in log2 units, sum of weights) per row,
  // in slot (unit + piece).
  float *stream_o, *tile_o;
  float2 *stream_ml, *tile_ml;
  int32_t stream_rows, tile_slot_rows;  // rows of a slot
  // Written by CTA 0 of either kernel for the join: the length per head of the
  // own parts before row unit u, at (its) units + 1 the line's, then the number
  // of pieces; and the row units before sequence b.
  int64_t *stream_sums, *unit_sums;
  int32_t *stream_base, *unit_base;
  int32_t sms;                     // CTAs of each kernel
  int32_t stream, tile_own;        // which of the two take own parts (both: see few_rows)
  int32_t join_rows;               // rows of a block of the join: 1, 8 or kJoinRows
  int32_t stream_prefix;  // the stream kernel takes the prefix too, for so many groups of 16 rows; or 0
  uint64_t over_group;    // 2^36 / group, rounded up
  int32_t stream_units, tile_units;  // of own parts at most, for sorted row offsets
  int32_t prefix_units;   // tile kernel: row units of the prefix
  int32_t tile_rows;      // tile kernel: batch rows per 128-row MMA tile, 128 / group
  uint32_t *err;
};

// Bounded wait.  Its slow path is one function for all call sites: code that a
// kernel has not run yet comes from HBM, at a microsecond or more a stretch, so
// the kernels here are kept small.
__device__ __noinline__ bool wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort, uint64_t limit_ns) {
  return mbar_wait_bounded(bar, parity, abort, limit_ns);
}
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort,
                                     uint64_t limit_ns = 4000000000ull) {
  return mbar_try_wait(bar, parity) || wait_slow(bar, parity, abort, limit_ns);
}

// Two f32 to packed f16 in one conversion.
__device__ __forceinline__ uint32_t to_h2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Bits [from, to) of a word, for any from and to.
__device__ __forceinline__ uint32_t bits_between(int32_t from, int32_t to) {
  const uint32_t below_to = to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u;
  const uint32_t below_from = from >= 32 ? 0xffffffffu : from <= 0 ? 0u : (1u << from) - 1u;
  return below_to & ~below_from;
}

// Named barrier over `count` threads that says whether `pred` holds for any of them.
__device__ __forceinline__ bool barrier_any(uint32_t id, uint32_t count, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %3, 0;\n bar.red.or.pred q, %1, %2, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(r)
      : "r"(id), "r"(count), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

// What the f16 pair `h` of two f32 leaves of them.
__device__ __forceinline__ uint32_t rest_h2(float lo, float hi, uint32_t h) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
  return to_h2(lo - f.x, hi - f.y);
}

// (Maximum in log2 units, sum) of a partial result.  A maximum drops NaN scores,
// the sum keeps them: with scores of NaN alone the maximum is that of no keys.
__device__ __forceinline__ float2 partial_ml(float m, float l, float c) {
  return make_float2(l != l ? l : m == -INFINITY ? m : m * c, l);
}

// Length of sequence b as far as its table row can hold it.
__device__ __forceinline__ int32_t checked_length(const PagedAttnParams &p, int32_t b, bool report) {
  const int32_t n = p.paged.lengths[b], cap = p.paged.max_pages * p.paged.page_size;
  if (n > cap && report && n > p.prefix) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_LENGTH);
  return n < 0 ? 0 : min(n, max(cap, p.prefix));
}

// The call's first row of sequence b.
__device__ __forceinline__ int32_t first_row(const PagedAttnParams &p, int32_t b) {
  return p.paged.row_offsets ? max(0, min(p.paged.row_offsets[b], (int32_t)p.rows)) : b;
}

// x / group for 0 <= x < 2^28 and group <= 16: the product stays below 2^64 (over_group
// is at most 2^36), and group * over_group exceeds 2^36 by less than group, x times
// which stays below 2^36.  Callers count query heads of a sequence of few rows or of
// a call whose prefix the stream kernel takes, below 2^15.
__device__ __forceinline__ int32_t over_group(const PagedAttnParams &p, int32_t x) {
  return (int32_t)((uint64_t)(uint32_t)x * p.over_group >> 36);
}

// The call's rows of a sequence: [begin, end), the first at position pos0, and
// its length.
struct SequenceRows {
  int32_t begin, end, length;
  int64_t pos0;
  __device__ __forceinline__ SequenceRows(const PagedAttnParams &p, int32_t b, bool report) {
    begin = first_row(p, b);
    end = first_row(p, b + 1);
    length = checked_length(p, b, report);
    pos0 = (int64_t)p.paged.lengths[b] - (end - begin);
    if (report && p.paged.row_offsets &&
        (p.paged.row_offsets[b] != begin || p.paged.row_offsets[b + 1] != end || end < begin))
      record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_OFFSET);
  }
  // End of the keys that the rows up to row `last` of the sequence attend to.
  __device__ __forceinline__ int32_t keys_to(int64_t last) const {
    return (int32_t)max((int64_t)0, min((int64_t)length, pos0 + last + 1));
  }
};

// Who takes a sequence's own part.  The stream kernel reads the keys once per 16
// rows, counted in query heads of a key head, the tile kernel once per 256, and
// pays for all of them.  Two units of 16 are where they meet: 32 sequences of 1
// to 4 rows x 4 heads over 500 to 4000 keys take 72 us with the first and 84 us
// with the second; 16 sequences of 1 to 8 rows x 8 heads 83 us with the second,
// 90 us with those of 5 to 8 rows there and the others here, 116 us with the
// first alone.
constexpr int kFewRows = 32;
__device__ __forceinline__ bool few_rows(const PagedAttnParams &p, const SequenceRows &r) {
  return p.stream && (!p.tile_own || (int64_t)(r.end - r.begin) * p.group <= kFewRows);
}

// Lines of units: sums over sequences carry the number of row units in front,
// above 2^40, and the length in front of them per head.
constexpr int64_t kLength = (1ll << 40) - 1;

// A thread's contiguous share of [0, n) in a block of kThreads.
template <int kThreads>
struct Share {
  int32_t lo, hi;
  __device__ __forceinline__ explicit Share(int32_t n) {
    const int32_t size = (n + kThreads - 1) / kThreads;
    lo = min(n, (int32_t)threadIdx.x * size);
    hi = min(n, lo + size);
  }
};

// The page id of the chunk of keys at position `pos`, if the chunk has a key of
// [lo, hi); checked_page makes a page coordinate of it, out of range (the TMA
// then fills zeros) where the chunk has none or the id is not a page.  Two
// steps, so that the load is in flight while the caller waits for a stage.
__device__ __forceinline__ int32_t page_id(const PagedAttnParams &p, const int32_t *ids, int32_t pos, int32_t lo,
                                           int32_t hi) {
  return pos < hi && pos + p.chunk > lo ? ids[pos / p.paged.page_size] : -1;
}
__device__ __forceinline__ int32_t checked_page(const PagedAttnParams &p, int32_t id, int32_t pos, int32_t lo,
                                                int32_t hi) {
  if (id >= 0 && id < p.paged.pages) return id;
  if (pos < hi && pos + p.chunk > lo) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PAGE);
  return p.paged.pages;
}

// ---- few rows: the sequences' own parts ----------------------------------------
//
// O = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m) with s = q k scale log2(e), in one
// pass with a running maximum m: when m grows, O and the sum so far are scaled.
//
// At most 16 query heads per key head: the group of a row (or rows) is one
// m16n8k16 tile, so a key costs 16 x 128 multiply-adds whatever the group, and K
// and V are streamed once: HBM-bound.  64 rows over 2000 to 4000 keys of 8 heads
// of 128 (790 MB) take 145 us, 5.5 TB/s.  (tcgen05's tile has 128 rows, an eighth
// of it filled: see few_rows for the two side by side.)  The key tiles
// (64 keys, at absolute multiples of 64) of all units (16 rows of a sequence,
// head) form one line that is cut into equal pieces, one per worker, so ragged
// lengths leave no CTA idle.  When the call has so few rows that the tile
// kernel's start would cost more, the shared prefix is on the line too, in front,
// as a unit per head and group of 16 rows (the later groups' reads of it come
// from L2).
// A CTA is two workers with a piece each: a producer warp fills a ring of
// tiles by TMA, box by box of gcd(page_size, 64) keys, and hands out units with
// their queries; four warps take 16 keys of every tile each, with a running
// maximum, sum and O of their own, and meet once per unit.
// Two layouts of K and V in shared memory.  Heads of 64 and 128 lie in halves
// of 64 elements with the 128-byte swizzle.  Others would waste up to half of
// that (72 elements: 9 KB of keys in 16, 0.52 of HBM): their rows are single
// boxes, unswizzled, `pitch` bytes apart, an odd multiple of 16 where the
// boxes' 128-byte alignment allows it, so that ldmatrix's eight rows meet no
// bank twice (heads of 72: 170 -> 113 us; heads of 128 lose by it, the rows
// start inside 128-byte lines: 58 -> 66 us).  The ring has as many stages as fit.
template <int N>
struct Number {
  static constexpr int value = N;
};
constexpr int kStreamKeys = 64, kStreamWorkers = 2, kStreamThreads = kStreamWorkers * 160;
constexpr int kStreamStages = 8;  // at most
constexpr int kMergeBytes = 4 * 16 * 20 * 4, kStreamRingBytes = 98304;
constexpr int kQueryLd = 136, kQueryBytes = 16 * kQueryLd * 2;  // a unit's 16 query rows, an odd multiple of 16 bytes apart

struct StreamShape {
  int32_t pitch, stages, bytes;  // bytes: dynamic shared memory
};
constexpr bool stream_swizzled(int padded_dim) { return padded_dim % 64 == 0; }
constexpr StreamShape stream_shape(int32_t padded_dim, int32_t chunk) {
  StreamShape r = {};
  const int32_t align = 128 / (chunk < 8 ? chunk : 8);
  r.pitch = stream_swizzled(padded_dim) ? padded_dim * 2 : (padded_dim * 2 + 16 + align - 1) / align * align;
  const int32_t stage = 2 * kStreamKeys * r.pitch;
  r.stages = kStreamRingBytes / stage < kStreamStages ? kStreamRingBytes / stage : kStreamStages;
  r.bytes = kStreamWorkers * (r.stages * stage + kMergeBytes + 2 * kQueryBytes) + 1024;
  return r;
}
// The most that a kernel takes with any page size: its limit, which all host threads
// share, is the same in every call.
constexpr int32_t stream_bytes(int32_t padded_dim) {
  int32_t most = 0;
  for (int32_t chunk = 1; chunk <= kStreamKeys; chunk *= 2)
    if (stream_shape(padded_dim, chunk).bytes > most) most = stream_shape(padded_dim, chunk).bytes;
  return most;
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes to shared memory, of which `bytes` are read and the rest zeros.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// This thread's arrival on the barrier, once its cp.async so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A worker's place on the line: unit (b, rows16, h): 16 rows of sequence b (of
// the call for the prefix, b = -1), counted in query heads of key head h, from
// row 16 rows16 on; keys [lo, hi).
struct StreamWalk {
  LinePlace at;
  int32_t b, rows16, h, lo, hi;
  int32_t unit, behind;     // own part: row units before this one; those of the sequence behind it
  int32_t begin, rows;      // first batch row of the sequence; rows of the unit
  int32_t pos0;             // own part: position of the sequence's first row
  int32_t prefix_end;       // of the prefix's keys that any sequence reaches

  __device__ __forceinline__ static int32_t units(const PagedAttnParams &p, const SequenceRows &r) {
    return few_rows(p, r) ? max(0, ((r.end - r.begin) * p.group + 15) / 16) : 0;
  }
  // Key tiles of row unit `j`.
  __device__ __forceinline__ static int32_t tiles(const PagedAttnParams &p, const SequenceRows &r, int32_t j) {
    const int32_t to = r.keys_to(over_group(p, min((r.end - r.begin) * p.group, 16 * j + 16) - 1));
    return to > p.prefix ? (to + kStreamKeys - 1) / kStreamKeys - p.prefix / kStreamKeys : 0;
  }
  __device__ __forceinline__ void prefix(const PagedAttnParams &p, int32_t j) {
    b = -1;
    rows16 = j;
    unit = -1;
    begin = 0;
    rows = min(16, (int32_t)p.rows * p.group - 16 * j);
    pos0 = 0;
    lo = 0;
    hi = prefix_end;
    at.n = (p.prefix + kStreamKeys - 1) / kStreamKeys;
  }
  __device__ __forceinline__ void own(const PagedAttnParams &p, const SequenceRows &r, int32_t j) {
    const int32_t all_rows = (r.end - r.begin) * p.group;
    rows16 = j;
    behind = units(p, r) - j - 1;
    begin = r.begin;
    rows = min(16, all_rows - 16 * j);
    pos0 = (int32_t)max(r.pos0, (int64_t)INT32_MIN);
    lo = p.prefix;
    hi = r.keys_to(over_group(p, 16 * j + rows - 1));
    at.n = tiles(p, r, j);
  }
  __device__ __noinline__ void next(const PagedAttnParams &p) {
    if (!at.pass()) return;
    if (b < 0) {  // units are in the order (head, rows)
      if (rows16 + 1 < p.stream_prefix) {
        prefix(p, rows16 + 1);
        return;
      }
      if (++h < p.heads) {
        prefix(p, 0);
        return;
      }
      behind = 0;
    } else if (++h < p.heads) {
      return;
    }
    h = 0;
    do {  // the next row unit with keys
      ++unit;
      if (behind) {
        own(p, SequenceRows(p, b, false), rows16 + 1);
        continue;
      }
      int32_t n = 0;
#pragma unroll 1
      while (!n) {
        if (++b >= p.paged.sequences) {
          at.left = 0;
          return;
        }
        const SequenceRows r(p, b, false);
        n = units(p, r);
        if (n) own(p, r, 0);
      }
    } while (at.n == 0);
  }
};

constexpr int kTileRows = 128, kTileKeys = 128;
constexpr int kTileBytes = 128 * 128 * 2, kTileHalf = kTileBytes / 2;
constexpr int kTileThreads = 576, kTileSmem = 6 * kTileBytes + 1024;

// A CTA's place on the tile kernel's line: unit (row unit, head h); `seq` < 0:
// the prefix, whose row units cover all rows.
struct TileWalk {
  LinePlace at;
  int32_t seq, j, h;         // row unit j of its sequence (or of the prefix)
  int32_t unit;              // own part: row units before it
  int32_t rows, lo, hi;      // batch rows; keys [lo, hi)
  int64_t row0, pos0;        // first batch row and (own part) its position
  int32_t prefix_end;        // as in StreamWalk

  // Key tiles of row unit j of a sequence.
  __device__ __forceinline__ static int32_t tiles(const PagedAttnParams &p, const SequenceRows &r, int32_t j) {
    const int32_t to = r.keys_to(min((int64_t)(r.end - r.begin), (int64_t)(j + 1) * 2 * p.tile_rows) - 1);
    return to > p.prefix ? (to + kTileKeys - 1) / kTileKeys - p.prefix / kTileKeys : 0;
  }
  __device__ __noinline__ void own(const PagedAttnParams &p, int32_t b, int32_t row_unit) {
    const SequenceRows r(p, b, false);
    const int32_t per_unit = 2 * p.tile_rows;
    seq = b;
    j = row_unit;
    row0 = r.begin + (int64_t)j * per_unit;
    rows = (int32_t)max((int64_t)0, min((int64_t)per_unit, r.end - row0));
    pos0 = r.pos0 + (row0 - r.begin);
    lo = p.prefix;
    hi = r.keys_to(row0 - r.begin + rows - 1);
    at.n = tiles(p, r, j);
  }
  __device__ __forceinline__ void prefix(const PagedAttnParams &p, int32_t row_unit) {
    const int32_t per_unit = 2 * p.tile_rows;
    seq = -1;
    j = row_unit;
    row0 = (int64_t)j * per_unit;
    rows = (int32_t)min((int64_t)per_unit, p.rows - row0);
    pos0 = 0;
    lo = 0;
    hi = prefix_end;
    at.n = (p.prefix + kTileKeys - 1) / kTileKeys;
  }
  __device__ __forceinline__ static int32_t units(const PagedAttnParams &p, const SequenceRows &r) {
    const int32_t per_unit = 2 * p.tile_rows;
    return few_rows(p, r) ? 0 : max(0, (r.end - r.begin + per_unit - 1) / per_unit);
  }
  __device__ __forceinline__ int64_t slot_unit(const PagedAttnParams &p) const {
    return seq < 0 ? (int64_t)h * p.prefix_units + j : (int64_t)(p.prefix_units + unit) * p.heads + h;
  }
  __device__ __noinline__ void next(const PagedAttnParams &p) {
    if (!at.pass()) return;
    if (seq < 0) {  // units are in the order (head, row unit)
      if (++j < p.prefix_units) {
        prefix(p, j);
        return;
      }
      if (++h < p.heads) {
        prefix(p, 0);
        return;
      }
      unit = -1;
      j = 0;
      h = 0;
    } else if (++h < p.heads) {
      return;
    } else {
      h = 0;
      ++j;
    }
    // the next row unit with keys
    ++unit;
    if (seq < 0) seq = 0;
#pragma unroll 1
    for (;; ++unit) {
#pragma unroll 1
      while (j >= units(p, SequenceRows(p, seq, false))) {
        if (++seq >= p.paged.sequences) {
          at.left = 0;
          return;
        }
        j = 0;
      }
      own(p, seq, j);
      if (at.n > 0) return;
      ++j;
    }
  }
};

// SMs that stream while the others work on row tiles, of two lines (key tiles):
// so many that both end together, by what was measured with both kernels
// running: a start of 8 us and 0.6 us a key tile and SM (heads of 128) against
// 13 us and 2.15 us a key tile (a row tile alone: 1.5).  More than
// kStreamSaturated saturate HBM.
constexpr int kStreamSaturated = 112;
__device__ __forceinline__ int32_t stream_sms(const PagedAttnParams &p, int64_t stream_line, int64_t tile_line) {
  if (stream_line == 0) return 0;
  if (tile_line == 0) return p.sms;
  const float stream = (float)stream_line * (0.25f + 0.35f / 128 * p.head_dim);
  const float tile = (float)tile_line * (p.rows > p.tile_rows ? 2.15f : 1.5f);
  int32_t lo = 1, hi = min(kStreamSaturated, p.sms - 1);
#pragma unroll 1
  while (lo < hi) {
    const int32_t x = (lo + hi) >> 1;
    if (8.0f + __fdividef(stream, (float)x) > 13.0f + __fdividef(tile, (float)(p.sms - x))) lo = x + 1;
    else hi = x;
  }
  return lo;
}

// Row units and length of a sequence's own part (see kLength) in the kernel that takes it.
template <typename Walk>
__device__ __forceinline__ int64_t own_part(const PagedAttnParams &p, const SequenceRows &r) {
  const int32_t n = Walk::units(p, r);
  int64_t sum = (int64_t)n << 40;
#pragma unroll 1
  for (int32_t j = 0; j < n; ++j) sum += unit_cost(Walk::tiles(p, r, j));
  return sum;
}

// Both kernels' lines, in key tiles: a CTA of either needs both to know how many
// SMs each has.  Summed by the whole block.
template <int kThreads>
struct Lines {
  int64_t stream_ahead, stream, tile_ahead, tile;  // the prefix's part, which is in front; the whole
  int64_t stream_before, tile_before;              // sums of own_part() in front of this thread's share
  int32_t sms_to_stream;
  // End of the prefix's keys: the longest sequence's length, where all are shorter
  // than the prefix.  Slots behind it may hold anything.
  int32_t prefix_end;
  __device__ __forceinline__ Lines(const PagedAttnParams &p, int64_t (&scratch)[kThreads / 32][2],
                                   int32_t (&longest)[kThreads / 32], bool report) {
    const Share<kThreads> share(p.paged.sequences);
    int64_t mine[2] = {0, 0};
    int32_t length = 0;
#pragma unroll 1
    for (int32_t b = share.lo; b < share.hi; ++b) {
      const SequenceRows r(p, b, report);
      length = max(length, r.length);
      if (few_rows(p, r)) mine[0] += own_part<StreamWalk>(p, r);
      else mine[1] += own_part<TileWalk>(p, r);
    }
    int64_t sum[2] = {mine[0], mine[1]};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum[0], d), y = __shfl_up_sync(0xffffffffu, sum[1], d);
      if (lane >= d) {
        sum[0] += x;
        sum[1] += y;
      }
    }
    length = __reduce_max_sync(0xffffffffu, length);
    if (lane == 31) {
      scratch[warp][0] = sum[0];
      scratch[warp][1] = sum[1];
      longest[warp] = length;
    }
    __syncthreads();
    stream_before = sum[0] - mine[0];
    tile_before = sum[1] - mine[1];
    stream = tile = 0;
    length = 0;
#pragma unroll 1
    for (int w = 0; w < kThreads / 32; ++w) {
      length = max(length, longest[w]);
      if (w < warp) {
        stream_before += scratch[w][0];
        tile_before += scratch[w][1];
      }
      stream += scratch[w][0];
      tile += scratch[w][1];
    }
    stream_ahead = (int64_t)unit_cost((p.prefix + kStreamKeys - 1) / kStreamKeys) * p.stream_prefix * p.heads;
    tile_ahead = (int64_t)unit_cost((p.prefix + kTileKeys - 1) / kTileKeys) * p.prefix_units * p.heads;
    stream = stream_ahead + (stream & kLength) * p.heads;
    tile = tile_ahead + (tile & kLength) * p.heads;
    sms_to_stream = stream_sms(p, stream, tile);
    prefix_end = min(p.prefix, length);
  }
};

// One unit's share of a worker's piece, as the producer hands it to the others.
struct StreamTask {
  int64_t slot;              // of the partial result
  int32_t n, key0, lo, hi;   // key tiles from position key0 on, keys [lo, hi); n = 0: the piece is done
  int32_t rows, whole;       // rows of the unit; the result is final
  int32_t prefix, begin;     // the prefix, or a sequence whose rows start at batch row `begin`
  int32_t row0, pos0, h;     // the unit's first row, in heads of the group from `begin` on; the position at `begin`
};

template <int DP>
__global__ void __launch_bounds__(kStreamThreads, 1)
    paged_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ PagedAttnParams p) {
  constexpr int KS = DP / 16, NT = DP / 8, HALVES = stream_swizzled(DP) ? DP / 64 : 1, HALF_BYTES = kStreamKeys * 128;
  const int tile_bytes = kStreamKeys * p.pitch, ring_bytes = p.stages * 2 * tile_bytes;  // K or V of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t all_full[kStreamWorkers][kStreamStages], all_empty[kStreamWorkers][kStreamStages];
  __shared__ uint64_t all_unit_full[kStreamWorkers][2], all_unit_empty[kStreamWorkers][2];  // queries and task
  __shared__ StreamTask all_tasks[kStreamWorkers][2];
  __shared__ int64_t scratch[kStreamThreads / 32][2];
  __shared__ int32_t longest[kStreamThreads / 32];
  __shared__ int32_t first_unit[kStreamWorkers][5];
  __shared__ float all_m[kStreamWorkers][4][16], all_l[kStreamWorkers][4][16];
  __shared__ int aborted;
  volatile int *abort_flag = &aborted;

  const int worker = threadIdx.x / 160, warp = (threadIdx.x >> 5) % 5, lane = threadIdx.x & 31;
  uint64_t *full = all_full[worker], *empty = all_empty[worker];
  uint64_t *unit_full = all_unit_full[worker], *unit_empty = all_unit_empty[worker];
  StreamTask *tasks = all_tasks[worker];
  float(&warp_m)[4][16] = all_m[worker], (&warp_l)[4][16] = all_l[worker];
  float *merge = reinterpret_cast<float *>(smem + kStreamWorkers * ring_bytes + worker * kMergeBytes);
  uint8_t *queries = smem + kStreamWorkers * (ring_bytes + kMergeBytes) + worker * 2 * kQueryBytes;
  smem += worker * ring_bytes;
  if (threadIdx.x == 0) {
#pragma unroll 1
    for (int w = 0; w < kStreamWorkers; ++w) {
#pragma unroll 1
      for (int i = 0; i < p.stages; ++i) {
        mbar_init(&all_full[w][i], 1);
        mbar_init(&all_empty[w][i], 4);
      }
#pragma unroll 1
      for (int i = 0; i < 2; ++i) {
        mbar_init(&all_unit_full[w][i], 33);  // the task, and the queries from each lane
        mbar_init(&all_unit_empty[w][i], 4);
      }
    }
    aborted = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // (sums of unsorted row offsets may run over and find no first unit)
  if (threadIdx.x >= 32 && threadIdx.x < 32 + kStreamWorkers * 5) (&first_unit[0][0])[threadIdx.x - 32] = 0;
  // Sums first, then this worker's piece [W c / C, W (c + 1) / C) of the line's W.
  const Lines<kStreamThreads> lines(p, scratch, longest, blockIdx.x == 0 && !p.tile_own);
  const int64_t line = lines.stream, ahead = lines.stream_ahead, sms = lines.sms_to_stream;
  int64_t before = lines.stream_before;
  // (No piece is empty, and there is at most one for two places of the line, of which
  // a unit's start and end count kUnitCost, so one may hold no key tile.  More pieces
  // cost more in the join: 16.0 against 15.5 us for 4 rows of 32 heads behind 512.)
  const int64_t pieces = min(kStreamWorkers * sms, (line + 1) / 2);
  // Worker w of CTA c has piece w * sms + c: few pieces spread over many SMs.
  auto piece_of = [&](int w) { return w * sms + (int64_t)blockIdx.x; };
  auto start_of = [&](int w) { return line * piece_of(w) / pieces; };
  const bool idle = (int64_t)blockIdx.x >= min(sms, pieces);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.stream_sums[p.stream_units + 1] = line;
    p.stream_sums[p.stream_units + 2] = pieces;
  }
  if (!idle || blockIdx.x == 0) {
    const int64_t start0 = idle ? -1 : start_of(0), start1 = idle ? -1 : start_of(1);
    static_assert(kStreamWorkers == 2, "two starts");
    const Share<kStreamThreads> mine(p.paged.sequences);
#pragma unroll 1
    for (int32_t b = mine.lo; b < mine.hi; ++b) {
      const SequenceRows r(p, b, false);
      const int32_t n = StreamWalk::units(p, r), base = (int32_t)(before >> 40);
      int64_t cost = before & kLength;
      if (blockIdx.x == 0) p.stream_base[b] = base;
#pragma unroll 1
      for (int32_t j = 0; j < n; ++j) {
        const int32_t here = unit_cost(StreamWalk::tiles(p, r, j));
#pragma unroll 1
        for (int w = 0; w < kStreamWorkers; ++w) {
          const int64_t at = (w ? start1 : start0) - ahead - cost * p.heads;
          if (at >= 0 && at < (int64_t)here * p.heads) {
            first_unit[w][0] = b;
            first_unit[w][1] = j;
            first_unit[w][2] = (int32_t)(at / here);
            first_unit[w][3] = (int32_t)(at % here);
            first_unit[w][4] = base + j;
          }
        }
        // (stream_units holds for sorted row offsets; sums of others may even be negative)
        if (blockIdx.x == 0 && (uint32_t)(base + j) < (uint32_t)p.stream_units) {
          p.stream_sums[base + j] = cost;
          p.stream_sums[base + j + 1] = cost + here;
        }
        cost += here;
      }
      before = ((before >> 40) + n) << 40 | cost;
    }
  }
  if (idle) {
    if (blockIdx.x == 0) griddep_wait();  // (see the end)
    return;
  }
  __syncthreads();  // (the barriers' initialisation too)
  const int64_t cta = piece_of(worker), start = start_of(worker);
  if (cta >= pieces) return;  // (a second worker)
  StreamWalk w;
  w.prefix_end = lines.prefix_end;
  if (start < ahead) {
    w.prefix(p, 0);
    const int32_t unit = (int32_t)(start / unit_cost(w.at.n));
    w.h = unit / p.stream_prefix;
    w.prefix(p, unit % p.stream_prefix);
    w.at.x = (int32_t)(start % unit_cost(w.at.n));
  } else {
    w.b = first_unit[worker][0];
    w.own(p, SequenceRows(p, w.b, false), first_unit[worker][1]);
    w.h = first_unit[worker][2];
    w.at.x = first_unit[worker][3];
    w.unit = first_unit[worker][4];
  }
  w.at.left = line * (cta + 1) / pieces - start;

  if (warp == 4) {
    // Producer: lane l issues boxes l, l + 32, ... of a tile: (K or V, half,
    // chunk).  The first one's page id is loaded a tile ahead.
    const int chunks = kStreamKeys / p.chunk, boxes = 2 * HALVES * chunks;
    const int chunk_bytes = p.chunk * (stream_swizzled(DP) ? 128 : p.pitch);
    const int my_chunk = lane % chunks;
    bool ok = true;
    int st = 0, filled = 0;
    uint32_t phase = 0;  // of the stage's barriers
    uint32_t unit = 0;
    // Hands out the next task and its query rows; zeros behind them and behind head_dim.
    auto publish = [&](int32_t n) {
      const uint32_t buffer = unit & 1;
      if (!wait(&unit_empty[buffer], ((unit >> 1) & 1) ^ 1, abort_flag)) return false;
      ++unit;
      if (n) {
#pragma unroll 1
        for (int x = lane; x < 16 * (DP / 8); x += 32) {
          const int r = x / (DP / 8), col = x % (DP / 8) * 8, row = 16 * w.rows16 + r, token = over_group(p, row);
          const bool there = r < w.rows && col < p.head_dim;
          const uint16_t *src = p.q + (int64_t)(w.begin + token) * p.q_stride +
                                (w.h * p.group + row - token * p.group) * p.head_dim + col;
          cp_async_16(smem_u32(queries) + buffer * kQueryBytes + (r * kQueryLd + col) * 2, there ? src : p.q, there ? 16 : 0);
        }
      }
      if (lane == 0) {
        StreamTask &task = tasks[buffer];
        const int64_t at = w.b < 0 ? w.h * p.stream_prefix + w.rows16 : (int64_t)(p.stream_prefix + w.unit) * p.heads + w.h;
        task.slot = (at + cta) * p.stream_rows;
        task.n = n;
        task.key0 = (w.lo / kStreamKeys + w.at.first()) * kStreamKeys;
        task.lo = w.lo;
        task.hi = w.hi;
        // (for unsorted row offsets nothing is written past the last unit)
        task.rows = w.b < 0 || (uint32_t)w.unit < (uint32_t)p.stream_units ? w.rows : 0;
        task.whole = p.prefix == 0 && n == w.at.n;
        task.prefix = w.b < 0;
        task.row0 = 16 * w.rows16;
        task.begin = w.begin;
        task.pos0 = w.pos0;
        task.h = w.h;
        mbar_arrive(&unit_full[buffer]);
      }
      cp_async_arrive(&unit_full[buffer]);
      return true;
    };
#pragma unroll 1
    for (; w.at.left > 0 && ok; w.next(p)) {
      const int32_t count_here = w.at.here();
      if (count_here == 0) continue;  // the piece ends in front of the unit's first tile
      if (!publish(count_here)) {
        ok = false;
        break;
      }
      const int32_t *ids = w.b < 0 ? p.prefix_pages : p.paged.page_table + w.b * p.paged.table_stride;
      int32_t key0 = (w.lo / kStreamKeys + w.at.first()) * kStreamKeys;
      int32_t id = lane < boxes ? page_id(p, ids, key0 + my_chunk * p.chunk, w.lo, w.hi) : -1;
#pragma unroll 1
      for (int32_t k = 0; k < count_here; ++k, key0 += kStreamKeys) {
        const int32_t id_next = k + 1 < count_here && lane < boxes
                                    ? page_id(p, ids, key0 + kStreamKeys + my_chunk * p.chunk, w.lo, w.hi)
                                    : -1;
        if (!wait(&empty[st], phase ^ 1, abort_flag)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * tile_bytes);
        __syncwarp();
        uint8_t *base = smem + st * 2 * tile_bytes;
#pragma unroll 1
        for (int x = lane; x < boxes; x += 32) {
          const int chunk = x % chunks, half = x / chunks % HALVES, v = x / (chunks * HALVES);
          const int32_t pos = key0 + chunk * p.chunk;
          if (x >= 32) id = page_id(p, ids, pos, w.lo, w.hi);
          tma_load_4d(base + v * tile_bytes + half * HALF_BYTES + chunk * chunk_bytes, v ? &tm_v : &tm_k, &full[st],
                      half * 64, pos % p.paged.page_size, w.h, checked_page(p, id, pos, w.lo, w.hi));
        }
        id = id_next;
        if (filled < p.stages) ++filled;
        if (++st == p.stages) {
          st = 0;
          phase ^= 1;
        }
      }
    }
    if (ok) ok = publish(0);
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PRODUCER);
      *abort_flag = 1;
      // nothing leaves while copies into its shared memory are in flight: the
      // stages from st on were last filled in the other phase
#pragma unroll 1
      for (int x = 0; x < filled; ++x) wait(&full[x], x < st ? phase : phase ^ 1, nullptr, 1000000000ull);
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    return;
  }

  // Consumers.  Fragments: rows lane / 4 and lane / 4 + 8 of the unit.
  const int r0 = lane >> 2, r1 = r0 + 8, cq = (lane & 3) * 2;
  // ldmatrix addresses: lane -> row lane % 8 of matrix lane / 8.  K matrices:
  // (keys 0-7, 8-15) x (two 16-byte column chunks); V: keys fastest.
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t k_row = warp * 16 + (mi >> 1) * 8 + mr, v_row = warp * 16 + (mi & 1) * 8 + mr;
  // Q: (rows 0-7, 8-15) x (two 16-byte column chunks).
  const uint32_t q_at = smem_u32(queries) + (((mi & 1) * 8 + mr) * kQueryLd + (mi >> 1) * 8) * 2;
  const uint32_t sbase = smem_u32(smem), pitch = p.pitch;
  // 16-byte column `col` of key `row` of a K or V tile
  auto place = [&](uint32_t row, uint32_t col) {
    return stream_swizzled(DP) ? (col >> 3) * HALF_BYTES + row * 128 + (((col & 7) ^ (row & 7)) << 4) : row * pitch + col * 16;
  };
  const float c = p.scale_log2;
  bool ok = true;
  int st = 0;
  uint32_t phase = 0;
#pragma unroll 1
  for (uint32_t unit = 0;; ++unit) {
    // (the four warps go on or stop together: they meet at barriers below)
    const bool late = !wait(&unit_full[unit & 1], (unit >> 1) & 1, abort_flag);
    if (barrier_any(1 + worker, 128, late || !ok)) {
      ok = false;
      break;
    }
    const StreamTask &task = tasks[unit & 1];
    const int32_t count_here = task.n, lo = task.lo, hi = task.hi, first_key = task.key0 + warp * 16;
    const int32_t rows_here = task.rows;
    const bool whole = task.whole, prefix = task.prefix, few = rows_here <= 8;
    const int64_t slot0 = task.slot;
    const int32_t row0 = task.row0, begin = task.begin, pos0 = task.pos0, head = task.h * p.group;
    uint32_t q[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) ldmatrix_x4(q_at + (unit & 1) * kQueryBytes + k * 32, q[k]);
    __syncwarp();
    if (lane == 0) mbar_arrive(&unit_empty[unit & 1]);
    if (count_here == 0) break;
    // Keys a row attends to end at its position, at the unit's end at the latest.
    auto row_end = [&](int r) {
      if (r >= rows_here) return hi;
      const int32_t place = over_group(p, row0 + r);
      int64_t position = (int64_t)pos0 + place;
      if (prefix) {
        PagedRow at;
        position = paged_row(p.paged, place, at) ? at.position : -1;
      }
      return (int32_t)max((int64_t)0, min((int64_t)hi, position + 1));
    };
    const int32_t end0 = row_end(r0), end1 = row_end(r1);
    const int32_t end = __reduce_min_sync(0xffffffffu, min(end0, end1));
    float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll 1
    for (int32_t k = 0; k < count_here; ++k) {
      // (a wait that ran out is not left early: the barriers below need every warp)
      if (ok && !wait(&full[st], phase, abort_flag)) ok = false;
      const uint32_t ks = sbase + st * 2 * tile_bytes, vs = ks + tile_bytes;
      const int32_t key0 = first_key + k * kStreamKeys;
      float s[2][4] = {}, s2[2][4] = {};  // even and odd steps: two chains
#pragma unroll
      for (int d = 0; d < KS; ++d) {
        uint32_t b[4];
        ldmatrix_x4(ks + place(k_row, d * 2 + (mi & 1)), b);
        mma_16816(d & 1 ? s2[0] : s[0], q[d], b[0], b[1]);
        mma_16816(d & 1 ? s2[1] : s[1], q[d], b[2], b[3]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[0][j] += s2[0][j];
        s[1][j] += s2[1][j];
      }
      if (key0 < lo || key0 + 16 > end) {
        // The unit's first or last tile: scores of keys that are not its own
        // are dropped, and the warp's V rows of such keys, which may hold
        // anything, are zeroed (0 * NaN is NaN).
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t key = key0 + x * 8 + cq + (j & 1);
            if (key < lo || key >= (j & 2 ? end1 : end0)) s[x][j] = -INFINITY;
          }
#pragma unroll 1
        for (int x = lane; x < 16 * NT; x += 32) {
          const int row = x / NT;
          if (key0 + row < lo || key0 + row >= hi) {
            const uint32_t at = vs + place(warp * 16 + row, x % NT);
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
          }
        }
        fence_proxy_async_smem();  // before the stage's next TMA write
        __syncwarp();
      }
      float x0 = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
      float x1 = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1));
      x0 = fmaxf(m0, fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2)));
      x1 = fmaxf(m1, fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2)));
      if (few) x1 = x0;
      if (__any_sync(0xffffffffu, (x0 - m0) * c > kLazy || (x1 - m1) * c > kLazy)) {
        // (m = -inf: the factor is 0, as are l and O)
        const float a0 = x0 == -INFINITY ? 1.0f : ex2_approx((m0 - x0) * c);
        const float a1 = x1 == -INFINITY ? 1.0f : ex2_approx((m1 - x1) * c);
        m0 = x0;
        m1 = x1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          o[i][0] *= a0;
          o[i][1] *= a0;
          o[i][2] *= a1;
          o[i][3] *= a1;
        }
      }
      // (m = -inf: every score so far is -inf and gives 0)
      const float n0 = m0 == -INFINITY ? 0.0f : kShift - m0 * c, n1 = m1 == -INFINITY ? 0.0f : kShift - m1 * c;
      // A weight goes into the product in two f16 parts, hi + lo, so that its
      // rounding (2^-11) does not add to the result's: in units of at most 8
      // rows the lo parts take the fragments' idle rows 8 to 15, in larger ones
      // a second product.  HBM bounds the kernel either way.  An infinite value
      // meets a part that is 0 or negative and gives NaN.
      uint32_t a[4], a_lo[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float p0 = ex2_approx(fmaf(s[x][0], c, n0)), p1 = ex2_approx(fmaf(s[x][1], c, n0));
        l0 += p0 + p1;
        a[2 * x] = to_h2(p0, p1);
        a_lo[2 * x] = rest_h2(p0, p1, a[2 * x]);
        a[2 * x + 1] = a_lo[2 * x];
        a_lo[2 * x + 1] = 0;
        if (!few) {
          const float p2 = ex2_approx(fmaf(s[x][2], c, n1)), p3 = ex2_approx(fmaf(s[x][3], c, n1));
          l1 += p2 + p3;
          a[2 * x + 1] = to_h2(p2, p3);
          a_lo[2 * x + 1] = rest_h2(p2, p3, a[2 * x + 1]);
        }
      }
#pragma unroll
      for (int d = 0; d < NT; d += 2) {
        uint32_t b[4];
        ldmatrix_x4_trans(vs + place(v_row, d + (mi >> 1)), b);
        mma_16816(o[d], a, b[0], b[1]);
        mma_16816(o[d + 1], a, b[2], b[3]);
        if (!few) {
          mma_16816(o[d], a_lo, b[0], b[1]);
          mma_16816(o[d + 1], a_lo, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == p.stages) {
        st = 0;
        phase ^= 1;
      }
    }
    // The four warps' results meet: the weights of their maxima, then O in as
    // many rounds as shared memory needs for the unit's rows.
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if ((lane & 3) == 0) {
      warp_m[warp][r0] = m0;
      warp_m[warp][r1] = m1;
      warp_l[warp][r0] = l0;
      warp_l[warp][r1] = l1;
    }
    named_barrier_sync(1 + worker, 128);
    auto weight = [&](float m, int row) {
      const float t = fmaxf(fmaxf(warp_m[0][row], warp_m[1][row]), fmaxf(warp_m[2][row], warp_m[3][row]));
      return m == -INFINITY ? 0.0f : ex2_approx((m - t) * c);
    };
    const float a0 = weight(m0, r0), a1 = weight(m1, r1);
    if (few) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        o[i][0] += o[i][2];
        o[i][1] += o[i][3];
      }
    }
    auto meet = [&](auto per_round) {
      constexpr int NI = decltype(per_round)::value, ROWS = 32 / NI, LD = NI * 8 + 4;  // n8 tiles a round; rows
      const int orow = (warp * 32 + lane) / (NI * 2), ocol = (lane % (NI * 2)) * 4;   // this thread's share of the sums
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int x = 0; x < 4; ++x) top = fmaxf(top, warp_m[x][orow & 15]);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (warp_l[x][orow & 15] != 0.0f) sum += warp_l[x][orow & 15] * ex2_approx((warp_m[x][orow & 15] - top) * c);
      const int64_t slot = slot0 + orow;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      if (!whole && orow < rows_here && ocol == 0) p.stream_ml[slot] = partial_ml(top, sum, c);
#pragma unroll
      for (int round = 0; round < (NT + NI - 1) / NI; ++round) {
        if (round) named_barrier_sync(1 + worker, 128);
        float *mine = merge + warp * ROWS * LD;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (round * NI + i >= NT) continue;
          const float(&v)[4] = o[round * NI + i];
          if (r0 < ROWS) *reinterpret_cast<float2 *>(mine + r0 * LD + i * 8 + cq) = make_float2(v[0] * a0, v[1] * a0);
          if (ROWS == 16) *reinterpret_cast<float2 *>(mine + r1 * LD + i * 8 + cq) = make_float2(v[2] * a1, v[3] * a1);
        }
        named_barrier_sync(1 + worker, 128);
        const int col = round * NI * 8 + ocol;
        if (orow < rows_here && col < p.head_dim) {
          float4 r = *reinterpret_cast<const float4 *>(merge + orow * LD + ocol);
#pragma unroll
          for (int x = 1; x < 4; ++x) {
            const float4 y = *reinterpret_cast<const float4 *>(merge + (x * ROWS + orow) * LD + ocol);
            r.x += y.x;
            r.y += y.y;
            r.z += y.z;
            r.w += y.w;
          }
          if (whole) {
            uint2 h;
            h.x = sum == 0.0f ? 0u : to_h2(r.x * inv, r.y * inv);  // (no keys: 0 * V, where V may be anything)
            h.y = sum == 0.0f ? 0u : to_h2(r.z * inv, r.w * inv);
            const int32_t place = over_group(p, row0 + orow), in_group = row0 + orow - place * p.group;
            *reinterpret_cast<uint2 *>(p.out + ((int64_t)(begin + place) * p.q_heads + head + in_group) * p.head_dim + col) = h;
          } else {
            *reinterpret_cast<float4 *>(p.stream_o + slot * p.head_dim + col) = r;
          }
        }
      }
    };
    if (rows_here <= 4) meet(Number<8>());
    else if (rows_here <= 8) meet(Number<4>());
    else meet(Number<2>());
  }
  if (!ok) {
    if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_EPILOGUE);
    *abort_flag = 1;
  }
  // What follows waits for this grid, so it ends after the tile kernel, beside
  // which it runs.
  if (blockIdx.x == 0) griddep_wait();
}

// ---- many rows: tiles of 128 on the tensor cores --------------------------------

// The same sums as above, bound by the softmax and the tensor core together: a
// key tile takes 2.15 us of an SM, 4 x 256 x 128 x 128 operations, which is 1.15
// PFLOP/s on all SMs; 128 rows of 32 heads behind 32768 shared positions take 84
// us, 820 TFLOP/s with start and end (K and V, read once by each row unit, come
// to 3.2 TB/s).
// Rows that read the same keys (all rows of the call for the shared prefix;
// one sequence's rows for its own part) are packed group by group into
// 128-row MMA tiles, tile_rows = 128 / group batch rows to a tile, two tiles
// to a unit.  As above, the 128-key tiles of all (row unit, head) units form a
// line, the prefix's first, and each of the CTAs, one per SM, has an equal
// piece of it:
//   warp 0      loads: Q of a unit, K and V tiles through two-stage rings, box
//               by box of gcd(page_size, 64) keys
//   warp 1      S_t = Q_t K^T into TMEM, O_t += P_t V with P_t read from TMEM
//               (it overwrites S_t as packed f16)
//   warps 2-17  softmax: two warps per lane quarter of a tile, 64 keys each
// so the tensor core works on one tile while the other's softmax runs, and a
// unit's Q and first K tile load while the last unit's results are stored.
// A unit whose rows fill one row tile only has it twice, for even and for odd
// key tiles (`dual`), and joins both at its end: each row's two O lie in the same
// TMEM lane.
// One unit's share of a CTA's piece, as the load warp hands it to the others:
// only that warp walks the line, which costs the softmax warps no registers.
struct TileTask {
  int64_t row0, pos0, slot;
  int32_t rows, lo, hi, h, first, n;  // key tiles [first, first + n); n = 0: the piece is done
  int32_t dual;                       // one row tile, for even and odd key tiles
  int32_t prefix, direct, store;
  // V rows outside [lo, hi) of a chunk that has both kinds may hold anything
  // and are zeroed in shared memory (0 * NaN is NaN); whole chunks outside are
  // zero-filled by the TMA.  Chunks with lo and hi inside: in the first key tile,
  // and in the one with this index in the task (-1: none; the unit's last, or an
  // earlier one of the prefix where no sequence reaches its end).
  int32_t fix_first, fix_at;
};

// The MMA warp runs as a whole and one elected lane issues: in code that only
// one lane reaches, the compiler moves every descriptor from a thread's to a
// uniform register before each MMA, which took 95 cycles an MMA (64 is what the
// tensor core needs) and bound the kernel.  Loop bounds and flags go through
// uniform() and all() so that it knows them to be the same in all lanes.
__device__ __forceinline__ int32_t uniform(int32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
__device__ __forceinline__ bool all(bool x) { return __all_sync(0xffffffffu, x); }
template <bool kAccumulate>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "n"(kAccumulate ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
  asm volatile(
      "{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
      " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// S = Q K^T of one row tile, K steps of 16 head dims.
template <int K>
__device__ __forceinline__ void issue_scores(uint32_t d, uint64_t q_desc, uint64_t k_desc) {
  constexpr uint32_t idesc = make_idesc(128, kTileKeys, 0, false, false);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const uint64_t step = (uint64_t)(((k >> 2) * kTileHalf + (k & 3) * 32) >> 4);
    if (k) mma_ss<true>(d, q_desc + step, k_desc + step, idesc);
    else mma_ss<false>(d, q_desc + step, k_desc + step, idesc);
  }
}

__global__ void __launch_bounds__(kTileThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *s_q = smem, *s_k = smem + 2 * kTileBytes, *s_v = smem + 4 * kTileBytes;
  __shared__ uint64_t q_full, q_empty, k_full[2], v_full[2], k_empty[2], v_empty[2], v_fixed[2];  // per ring stage
  __shared__ uint64_t s_full[2], p_ready[2], o_final[2], o_empty[2];                             // per row tile
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted;
  __shared__ float x_max[2][2][kTileRows], x_sum[2][2][kTileRows];
  __shared__ int64_t scratch[kTileThreads / 32][2];
  __shared__ int32_t longest[kTileThreads / 32];
  __shared__ int32_t found[5];
  __shared__ uint64_t task_full[2], task_empty[2];
  __shared__ TileTask tasks[2];
  volatile int *abort_flag = &aborted;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&q_empty, 1);
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_fixed[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 8);
      mbar_init(&o_final[i], 1);
      mbar_init(&o_empty[i], 16);
      mbar_init(&task_full[i], 1);
      mbar_init(&task_empty[i], 17);  // the MMA thread and 16 softmax warps
    }
    aborted = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (threadIdx.x >= 32 && threadIdx.x < 37) found[threadIdx.x - 32] = 0;  // (as first_unit above)
  // This CTA's piece of the line's W, [W c / C, W (c + 1) / C).
  const int64_t cta = blockIdx.x;
  const Lines<kTileThreads> lines(p, scratch, longest, cta == 0);
  const int64_t line = lines.tile, ahead = lines.tile_ahead, ctas = min((int64_t)(p.sms - lines.sms_to_stream), line);
  int64_t before = lines.tile_before;
  const bool idle = cta >= ctas;  // no piece is empty
  const int64_t start = idle ? -1 : line * cta / ctas;
  griddep_launch_dependents();
  if (p.tile_own && (!idle || cta == 0)) {
    const Share<kTileThreads> mine(p.paged.sequences);
#pragma unroll 1
    for (int32_t b = mine.lo; b < mine.hi; ++b) {
      const SequenceRows r(p, b, false);
      const int32_t u = TileWalk::units(p, r), base = (int32_t)(before >> 40);
      int64_t cost = before & kLength;
      if (cta == 0) p.unit_base[b] = base;
#pragma unroll 1
      for (int32_t j = 0; j < u; ++j) {
        const int32_t n = unit_cost(TileWalk::tiles(p, r, j));
        const int64_t at = start - ahead - cost * p.heads;
        if (at >= 0 && at < (int64_t)n * p.heads) {
          found[0] = b;
          found[1] = j;
          found[2] = (int32_t)(at / n);
          found[3] = (int32_t)(at % n);
          found[4] = base + j;
        }
        if (cta == 0 && (uint32_t)(base + j) < (uint32_t)p.tile_units) {
          p.unit_sums[base + j] = cost;
          p.unit_sums[base + j + 1] = cost + n;
        }
        cost += n;
      }
      before = ((before >> 40) + u) << 40 | cost;
    }
  }
  if (cta == 0 && threadIdx.x == 0) {
    p.unit_sums[p.tile_units + 1] = line;
    p.unit_sums[p.tile_units + 2] = ctas;
  }
  if (idle) return;
  __syncthreads();
  TileWalk walk;
  walk.unit = -1;
  walk.prefix_end = lines.prefix_end;
  if (start < ahead) {
    walk.prefix(p, 0);
    const int64_t u = start / unit_cost(walk.at.n);
    walk.h = (int32_t)(u / p.prefix_units);
    walk.prefix(p, (int32_t)(u % p.prefix_units));
    walk.at.x = (int32_t)(start % unit_cost(walk.at.n));
  } else {
    walk.own(p, found[0], found[1]);
    walk.h = found[2];
    walk.at.x = found[3];
    walk.unit = found[4];
  }
  walk.at.left = line * (cta + 1) / ctas - start;
  const int halves = p.head_dim > 64 ? 2 : 1, k_steps = (p.head_dim + 15) / 16;

  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(tmem_slot);  // S_t at column t * 128, O_t at 256 + t * 128
  if (warp == 0) {
    // Lane l issues boxes l, l + 32, ... of a tile: (half, chunk).  Where the
    // first one comes from is known before the stage is free: the softmax
    // warps leave this one little of its scheduler, and every instruction
    // between a free stage and its load lengthens the chain.
    const int chunks = kTileKeys / p.chunk, boxes = halves * chunks;
    const int my_chunk = lane % chunks, my_half = lane / chunks;
    const int my_offset = my_half * kTileHalf + my_chunk * p.chunk * 128;
    bool ok = true;
    uint32_t unit = 0, k_issued = 0, v_issued = 0, q_issued = 0;
    // Tasks are written two ahead of the last reader at most; after the last comes one with n = 0.
    auto publish = [&](const TileTask &task, uint32_t index) {
      const bool free = wait(&task_empty[index & 1], ((index >> 1) & 1) ^ 1, abort_flag);
      if (free && lane == 0) {
        tasks[index & 1] = task;
        mbar_arrive(&task_full[index & 1]);
      }
      return free;
    };
#pragma unroll 1
    for (; walk.at.left > 0 && ok; walk.next(p)) {
      if (walk.at.here() == 0) continue;  // the piece ends in front of the unit's first tile
      TileTask task;
      task.row0 = walk.row0;
      task.pos0 = walk.pos0;
      task.slot = walk.slot_unit(p) + cta;
      task.rows = walk.rows;
      task.lo = walk.lo;
      task.hi = walk.hi;
      task.h = walk.h;
      task.n = walk.at.here();
      task.first = walk.lo / kTileKeys + walk.at.first();
      task.dual = walk.rows <= p.tile_rows;
      task.prefix = walk.seq < 0;
      task.direct = p.prefix == 0 && task.n == walk.at.n;
      // (for unsorted row offsets nothing is written past the last unit)
      task.store = walk.seq < 0 || (uint32_t)walk.unit < (uint32_t)p.tile_units;
      task.fix_first = task.first * kTileKeys < walk.lo && walk.lo % p.chunk != 0;
      task.fix_at = walk.hi % p.chunk != 0 ? walk.hi / kTileKeys - task.first : -1;
      if (!publish(task, unit)) {
        ok = false;
        break;
      }
      const int32_t *ids = walk.seq < 0 ? p.prefix_pages : p.paged.page_table + walk.seq * p.paged.table_stride;
      // K runs a tile ahead of V: its stages are free earlier.
      int32_t id = -1, slot = 0, page = 0;  // of the next K tile
      int32_t v_slot = 0, v_page = 0;       // of the next V tile
      auto look = [&](int32_t key0) {
        const int32_t pos = key0 + my_chunk * p.chunk;
        id = lane < boxes ? page_id(p, ids, pos, walk.lo, walk.hi) : -1;
        slot = pos % p.paged.page_size;
      };
      auto load = [&](uint8_t *base, const CUtensorMap *map, uint64_t *bar, int32_t key0, int32_t from_slot, int32_t from_page) {
        if (lane == 0) mbar_arrive_expect_tx(bar, halves * kTileHalf);
        __syncwarp();
        if (lane < boxes) tma_load_4d(base + my_offset, map, bar, my_half * 64, from_slot, walk.h, from_page);
#pragma unroll 1
        for (int i = lane + 32; i < boxes; i += 32) {
          const int chunk = i % chunks, half = i / chunks;
          const int32_t pos = key0 + chunk * p.chunk;
          tma_load_4d(base + half * kTileHalf + chunk * p.chunk * 128, map, bar, half * 64, pos % p.paged.page_size,
                      walk.h, checked_page(p, page_id(p, ids, pos, walk.lo, walk.hi), pos, walk.lo, walk.hi));
        }
      };
      look(task.first * kTileKeys);
#pragma unroll 1
      for (int32_t j = 0; j <= task.n && ok; ++j) {
        if (j < task.n) {
          const int st = k_issued & 1;
          const int32_t key0 = (task.first + j) * kTileKeys;
          page = lane < boxes ? checked_page(p, id, key0 + my_chunk * p.chunk, walk.lo, walk.hi) : 0;
          ok = wait(&k_empty[st], ((k_issued >> 1) & 1) ^ 1, abort_flag);
          if (!ok) break;
          load(s_k + st * kTileBytes, &tm_k, &k_full[st], key0, slot, page);
          ++k_issued;
          if (j == 0) {
            // Q's buffer: the previous unit's S products are done
            ok = wait(&q_empty, (unit & 1) ^ 1, abort_flag);
            if (!ok) break;
            if (lane == 0) {
              const int tiles = task.dual ? 1 : 2;
              mbar_arrive_expect_tx(&q_full, tiles * halves * p.tile_rows * p.group * 128);
#pragma unroll 1
              for (int t = 0; t < tiles; ++t)
#pragma unroll 1
                for (int half = 0; half < halves; ++half)
                  tma_load_4d(s_q + t * kTileBytes + half * kTileHalf, &tm_q, &q_full, half * 64, 0, walk.h,
                              (int32_t)walk.row0 + t * p.tile_rows);
            }
            ++q_issued;
          }
        }
        if (j > 0) {
          const int st = v_issued & 1;
          const int32_t key0 = (task.first + j - 1) * kTileKeys;
          ok = wait(&v_empty[st], ((v_issued >> 1) & 1) ^ 1, abort_flag);
          if (!ok) break;
          load(s_v + st * kTileBytes, &tm_v, &v_full[st], key0, v_slot, v_page);
          ++v_issued;
          if ((task.fix_first && j == 1) || j - 1 == task.fix_at) {
            ok = wait(&v_full[st], ((v_issued - 1) >> 1) & 1, abort_flag);
            if (!ok) break;
#pragma unroll 1
            for (int i = lane; i < kTileKeys * halves * 8; i += 32) {
              const int row = i / (halves * 8), half = (i >> 3) % halves;
              if (key0 + row < walk.lo || key0 + row >= walk.hi)
                *reinterpret_cast<uint4 *>(s_v + st * kTileBytes + half * kTileHalf + row * 128 + (i & 7) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_fixed[st]);
          }
        }
        v_slot = slot;
        v_page = page;
        if (j + 1 < task.n) look((task.first + j + 1) * kTileKeys);
      }
      ++unit;
    }
    if (ok) {
      TileTask done = {};
      ok = publish(done, unit);
    }
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PRODUCER);
      *abort_flag = 1;
      // nothing leaves while copies into its shared memory are in flight
      if (q_issued) wait(&q_full, (q_issued - 1) & 1, nullptr, 1000000000ull);
#pragma unroll 1
      for (uint32_t i = k_issued > 2 ? k_issued - 2 : 0; i < k_issued; ++i)
        wait(&k_full[i & 1], (i >> 1) & 1, nullptr, 1000000000ull);
#pragma unroll 1
      for (uint32_t i = v_issued > 2 ? v_issued - 2 : 0; i < v_issued; ++i)
        wait(&v_full[i & 1], (i >> 1) & 1, nullptr, 1000000000ull);
    }
  } else if (warp == 1) {
    const uint32_t idesc_o = make_idesc(128, k_steps * 16, 0, false, true);  // V: head dims contiguous
    const uint64_t q_desc = make_smem_desc(smem_u32(s_q), 16, 1024, kSwizzle128B);
    const uint64_t k_desc = make_smem_desc(smem_u32(s_k), 16, 1024, kSwizzle128B);
    const uint64_t v_desc = make_smem_desc(smem_u32(s_v), kTileHalf, 1024, kSwizzle128B);
    auto issue_s = [&](int t, int q_tile, int st) {
      const uint32_t d = tmem + t * 128;
      const uint64_t qd = q_desc + (uint64_t)(q_tile * (kTileBytes >> 4)), kd = k_desc + (uint64_t)(st * (kTileBytes >> 4));
      if (k_steps > 4) issue_scores<8>(d, qd, kd);  // (columns from head_dim on are zero)
      else issue_scores<4>(d, qd, kd);
      commit(&s_full[t]);
    };
    // Per key tile j and row tile t that takes it: PV_t(j) as soon as P_t(j) is
    // there, then t's next S product behind it.  A stage of K is released
    // behind its last S product, one of V behind its last PV product.  A
    // unit's first S products queue behind the last unit's last PV products,
    // so its S tiles (which held the last P) are free by then.
    bool ok = true;
    uint32_t unit = 0, g = 0;  // units begun, key tiles of the units before
    uint32_t p_count[2] = {0, 0}, fixes[2] = {0, 0};
    auto there = [&](uint64_t *bar, uint32_t parity) { return all(wait(bar, parity & 1, abort_flag)); };
    auto k_there = [&](uint32_t i) { return there(&k_full[i & 1], i >> 1); };
#pragma unroll 1
    for (;; ++unit) {
      ok = there(&task_full[unit & 1], unit >> 1);
      if (!ok) break;
      const TileTask &task = tasks[unit & 1];
      const int32_t n = uniform(task.n), flags = uniform(task.fix_first | task.dual << 1), fix_at = uniform(task.fix_at);
      const bool fix_first = flags & 1, dual = flags & 2;
      if (lane == 0) mbar_arrive(&task_empty[unit & 1]);
      __syncwarp();
      if (n == 0) break;
      const int32_t step = dual ? 2 : 1;  // key tiles from a row tile's one to its next
      ok = k_there(g) && there(&q_full, unit);
      if (!ok) break;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        if (dual && t == 1) {
          if (n == 1) break;
          ok = k_there(g + 1);
          if (!ok) break;
        }
        const int st = dual ? (g + t) & 1 : g & 1;
        issue_s(t, dual ? 0 : t, st);
        if (dual || t == 1) commit(&k_empty[st]);
      }
      if (!ok) break;
      if (n <= step) commit(&q_empty);
#pragma unroll 1
      for (int32_t j = 0; j < n && ok; ++j) {
        const uint32_t i = g + j;
        const int st = i & 1;
        const bool more = j + step < n;
        const uint64_t vd = v_desc + (uint64_t)(st * (kTileBytes >> 4));
        if ((fix_first && j == 0) || j == fix_at) ok = there(&v_fixed[st], fixes[st]++);
        else ok = there(&v_full[st], i >> 1);
#pragma unroll 1
        for (int x = dual ? 1 : 0; x < 2 && ok; ++x) {
          const int t = dual ? j & 1 : x;
          ok = there(&p_ready[t], p_count[t]++);
          // the last unit's O_t has been read out before this one's first PV_t
          if (ok && j < step && unit) ok = there(&o_empty[t], unit - 1);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            mma_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vd + (uint64_t)((k * 2048) >> 4), idesc_o,
                   j >= step || k > 0 ? 1u : 0u);
          if (x == 1) commit(&v_empty[st]);
          if (!more) {
            commit(&o_final[t]);
            continue;
          }
          const int next = (i + step) & 1;
          if (dual || t == 0) {
            ok = k_there(i + step);
            if (!ok) break;
          }
          issue_s(t, dual ? 0 : t, next);
          if (x == 1) commit(&k_empty[next]);
        }
        if (ok && j + step == n - 1) commit(&q_empty);
      }
      if (!ok) break;
      g += n;
    }
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_MMA);
      *abort_flag = 1;
    }
  } else {
    const int sw = warp - 2, t = sw >> 3, half = (sw >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t bar_id = 1 + t * 4 + quarter;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_off + t * 128, o_col = tmem + lane_off + 256 + t * 128 + half * 64;
    const float c = p.scale_log2;
    const bool in_tile = row < p.tile_rows * p.group;
    bool ok = true;
    uint32_t g = 0, units[2] = {0, 0};  // key tiles of this row tile so far; units that have had PV_0 and PV_1
#pragma unroll 1
    for (uint32_t index = 0;; ++index) {
      // (the four warps of a lane quarter go on or stop together: they meet at barriers below)
      const bool late = ok && !wait(&task_full[index & 1], (index >> 1) & 1, abort_flag);
      if (barrier_any(9 + quarter, 128, late || !ok)) {
        ok = false;
        break;
      }
      const TileTask &task = tasks[index & 1];
      if (task.n == 0) break;
      // This row tile's key tiles: all, or every second from t on.
      const bool dual = task.dual, both = !dual || task.n > 1;
      const int32_t n = dual ? (task.n - t + 1) >> 1 : task.n, step = dual ? 2 : 1;
      const int32_t row_tile = dual ? 0 : t, local = row_tile * p.tile_rows + row / p.group;  // batch row within the unit
      // This row's keys: [lo, limit).
      const bool row_ok = in_tile && local < task.rows && task.store;
      const int64_t token = task.row0 + local;
      const int32_t lo = task.lo, first = task.first + (dual ? t : 0);
      const bool direct = task.direct;
      const int64_t head = token * p.q_heads + task.h * p.group + row % p.group;
      const int32_t slot_row = row_tile * p.tile_rows * p.group + row;
      const int64_t slot = task.slot;
      int32_t limit = 0;
      if (row_ok) {
        PagedRow r;
        int64_t position = task.pos0 + local;
        if (task.prefix) position = paged_row(p.paged, token, r) ? r.position : -1;
        limit = (int32_t)max((int64_t)0, min((int64_t)task.hi, position + 1));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&task_empty[index & 1]);
      float m = -INFINITY, l = 0.0f;
#pragma unroll 1
      for (int32_t j = 0; j < n; ++j, ++g) {
        // (a wait that ran out is not left early: the barriers below need every warp)
        if (ok && !wait(&s_full[t], g & 1, abort_flag)) ok = false;
        tc_fence_after();
        const int32_t key0 = (first + j * step) * kTileKeys + half * 64;
        uint32_t a[32], b[32];
        tmem_ld_32x32b_x32(s_col + half * 64, a);
        tmem_ld_32x32b_x32(s_col + half * 64 + 32, b);
        tmem_wait_ld(a);
        tmem_regs_fence(b);
        const int from = lo - key0, to = limit - key0;
        if (__any_sync(0xffffffffu, from > 0 || to < 64)) {
          const uint32_t keep0 = bits_between(from, to), keep1 = bits_between(from - 32, to - 32);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (!(keep0 >> i & 1u)) a[i] = __float_as_uint(-INFINITY);
            if (!(keep1 >> i & 1u)) b[i] = __float_as_uint(-INFINITY);
          }
        }
        float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          mx = max3_nan(mx, __uint_as_float(a[i]), __uint_as_float(a[i + 1]));
          mx1 = max3_nan(mx1, __uint_as_float(a[i + 2]), __uint_as_float(a[i + 3]));
          mx = max3_nan(mx, __uint_as_float(b[i]), __uint_as_float(b[i + 1]));
          mx1 = max3_nan(mx1, __uint_as_float(b[i + 2]), __uint_as_float(b[i + 3]));
        }
        mx = max_nan(mx, mx1);
        x_max[t][half][row] = mx;
        named_barrier_sync(bar_id, 64);
        // A score of NaN or +inf makes the row NaN.  The maximum carries that (+inf up
        // to the unit's end): the polynomial below, which takes one pair in three, does not.
        const float m_new = max3_nan(m, mx, x_max[t][half ^ 1][row]);
        bool rescale = false;
        float alpha = 1.0f;
        if (j == 0) {
          m = m_new;
        } else if ((m_new - m) * c > kLazy || isnan(m_new)) {
          alpha = ex2_approx((m - m_new) * c);  // 0 where m = -inf: so are O and l
          rescale = true;
          m = m_new;
          l *= alpha;
        }
        // (m = -inf: every score so far is -inf and gives 0)
        const float mc = m == -INFINITY ? 0.0f : kShift - m * c;
        const uint64_t c2 = f2_pack(c, c), nmc2 = f2_pack(mc, mc);
        uint64_t sum2 = f2_pack(0.0f, 0.0f);
        uint32_t packed[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float x0 = __uint_as_float(i < 16 ? a[2 * i] : b[2 * i - 32]);
          const float x1 = __uint_as_float(i < 16 ? a[2 * i + 1] : b[2 * i - 31]);
          const uint64_t tt = f2_fma(f2_pack(x0, x1), c2, nmc2);
          // (one pair in three on the FMA pipe: the exponential unit alone would bound the kernel)
          uint64_t pp;
          float p0, p1;
          if (i % 3 == 2) {
            pp = exp2_poly2(tt);
            f2_unpack(pp, p0, p1);
          } else {
            float t0, t1;
            f2_unpack(tt, t0, t1);
            p0 = ex2_approx(t0);
            p1 = ex2_approx(t1);
            pp = f2_pack(p0, p1);
          }
          sum2 = f2_add(sum2, pp);
          // The weight's f16 rounding, 2^-11 of it at most, is the largest error here:
          // results are 2.9e-4 (2-norm, relative) off 64 bits, where their own store
          // alone makes 2.1e-4.  A second f16 part as in the stream kernel brings
          // 2.1e-4 and half as many MMAs more: 64 rows behind 8192 shared positions
          // take 61 us for 54, 128 behind 32768 192 for 155, pieces of prompts 151 for
          // 125.  One part, as in the flash attention kernel.
          packed[i] = to_h2(p0, p1);
        }
        tmem_st_32x32b_x32(s_col + half * 32, packed);
        float s0, s1;
        f2_unpack(sum2, s0, s1);
        l += s0 + s1;
        if (__any_sync(0xffffffffu, rescale)) {
          // O_t is stable: PV_t(j-1) was issued before S_t(j), which has been seen complete.
#pragma unroll
          for (int ch = 0; ch < 2; ++ch) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(o_col + ch * 32, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x32(o_col + ch * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[t]);
      }
      if (m == INFINITY) l = NAN;
      x_sum[t][half][row] = l;
      named_barrier_sync(bar_id, 64);
      l += x_sum[t][half ^ 1][row];
      if (ok && (t == 0 || dual) && !wait(&o_final[0], units[0] & 1, abort_flag)) ok = false;
      if (ok && both && (t == 1 || dual) && !wait(&o_final[1], units[1] & 1, abort_flag)) ok = false;
      ++units[0];
      if (both) ++units[1];
      tc_fence_after();
      // A thread stores 64 columns of its row's O, or (dual) 32 of the sum of its
      // two O: columns half * 64 + t * 32 on.
      float own = 1.0f, other = 0.0f;  // (dual) weights of O_t and of the other
      if (dual) {
        if (half == 0) {
          x_max[t][0][row] = m;
          x_max[t][1][row] = l;
        }
        named_barrier_sync(9 + quarter, 128);
        const float m2 = x_max[t ^ 1][0][row], l2 = x_max[t ^ 1][1][row], top = max_nan(m, m2);
        own = m == -INFINITY ? 0.0f : ex2_approx((m - top) * c);
        other = m2 == -INFINITY ? 0.0f : ex2_approx((m2 - top) * c);
        l = l * own + l2 * other;
        m = top;
        named_barrier_sync(9 + quarter, 128);  // read before the next unit's maxima are written
      }
      if (row_ok && !direct && half == 0 && (!dual || t == 0))
        p.tile_ml[slot * p.tile_slot_rows + slot_row] = partial_ml(m, l, c);
      const float inv = 1.0f / l;
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        const int32_t at = dual ? t * 32 : ch * 32;  // column in this thread's half
        uint32_t r[32];
        if (!dual || ch == 0) {
          tmem_ld_32x32b_x32(o_col + at, r);
          tmem_wait_ld(r);
        }
        if (dual && ch == 0) {
          // (O_1 is not there after a single key tile; its weight is 0)
          uint32_t r2[32];
          tmem_ld_32x32b_x32(o_col + at + (t ? -128 : 128), r2);
          tmem_wait_ld(r2);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            r[i] = __float_as_uint((own != 0.0f ? __uint_as_float(r[i]) * own : 0.0f) +
                                   (other != 0.0f ? __uint_as_float(r2[i]) * other : 0.0f));
        }
        if (ch == (dual ? 0 : 1)) {
          // read out: the next unit's first PV products may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&o_empty[t]);
            mbar_arrive(&o_empty[dual ? t ^ 1 : t]);
          }
        }
        const int col0 = half * 64 + at;
        if (!row_ok || (dual && ch == 1)) continue;
        if (direct) {
          // (a row without keys: O is 0 * V, which a non-finite V of another row's keys makes NaN.
          // Its sum is not 0: the polynomial makes 2^-125 of a masked score.)
          uint16_t *o = p.out + head * p.head_dim + col0;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (col0 + i >= p.head_dim) break;
            uint4 v;
            v.x = to_h2(__uint_as_float(r[i]) * inv, __uint_as_float(r[i + 1]) * inv);
            v.y = to_h2(__uint_as_float(r[i + 2]) * inv, __uint_as_float(r[i + 3]) * inv);
            v.z = to_h2(__uint_as_float(r[i + 4]) * inv, __uint_as_float(r[i + 5]) * inv);
            v.w = to_h2(__uint_as_float(r[i + 6]) * inv, __uint_as_float(r[i + 7]) * inv);
            *reinterpret_cast<uint4 *>(o + i) = m == -INFINITY ? make_uint4(0u, 0u, 0u, 0u) : v;
          }
        } else {
          // [slot][dim / 4][row][4]: a lane holds a row, so a warp's 16-byte stores are
          // neighbours (row by row they cost 15 us a unit on all SMs, half-filled sectors)
          float *o = p.tile_o + ((slot * (p.head_dim >> 2) + (col0 >> 2)) * p.tile_slot_rows + slot_row) * 4;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (col0 + i >= p.head_dim) break;
            *reinterpret_cast<float4 *>(o + (int64_t)i * p.tile_slot_rows) =
                make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]), __uint_as_float(r[i + 2]),
                            __uint_as_float(r[i + 3]));
          }
        }
      }
    }
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_EPILOGUE);
      *abort_flag = 1;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---- the partial results' sum -----------------------------------------------------

// A block joins join_rows neighbouring rows of one key head (batch row, head of the
// group): eight at a time, a thread four dims of one of them, so that 16-byte reads
// are neighbours row by row (tile slots) or dim by dim (stream slots); 32 in calls
// with more rows than fill the GPU eight times, where finding the pieces counts; one
// in calls of few rows (kSplit).  A row's partials are
// the pieces of its prefix unit and those of its own unit, both runs of slots.
// Bound by latency, two lookups and two rounds of loads: 64 rows of 32 heads take
// 7 us.  Weights are 2^(m_i - m), sums and O stay in f32 up to the one rounding.
struct Pieces {
  const float2 *ml;  // of the first one's row; a piece is `rows` rows further
  const float *o;    // its dim 0; four dims further on `dims`, a piece rows * head_dim
  int32_t count, rows, dims;  // count < 0: padding
};
// Pieces of unit `unit`, at [first, first + cost) of a line of length `line`:
// piece c of C is [line c / C, line (c + 1) / C), so place t is in c = ((t + 1) C
// - 1) / line, and the unit's tiles are its places from kUnitCost on.
__device__ __forceinline__ Pieces pieces_of(const PagedAttnParams &p, bool stream, int64_t first, int64_t cost, int64_t unit,
                                            int32_t row) {
  Pieces r = {p.stream ? p.stream_ml : p.tile_ml, p.stream ? p.stream_o : p.tile_o, 0, 0, 0};
  if (cost <= 0) return r;
  const int64_t *sums = stream ? p.stream_sums + p.stream_units : p.unit_sums + p.tile_units, line = sums[1], c = sums[2];
  const int64_t last = first + cost;
  first += kUnitCost;
  int32_t c0, c1;
  if (line * c < (1ll << 31)) {  // (32-bit divisions: a quarter of the time)
    c0 = (int32_t)(((uint32_t)(first + 1) * (uint32_t)c - 1) / (uint32_t)line);
    c1 = (int32_t)(((uint32_t)last * (uint32_t)c - 1) / (uint32_t)line);
  } else {
    c0 = (int32_t)(((first + 1) * c - 1) / line);
    c1 = (int32_t)((last * c - 1) / line);
  }
  // (in bounds whatever the sums of unsorted row offsets are)
  c0 = max(0, min(c0, (int32_t)c - 1));
  c1 = max(c0, min(c1, (int32_t)c - 1));
  r.count = c1 - c0 + 1;
  const int64_t slot = unit + c0;
  if (stream) {
    r.rows = p.stream_rows;
    r.dims = 4;
    r.ml = p.stream_ml + slot * r.rows + row;
    r.o = p.stream_o + (slot * r.rows + row) * p.head_dim;
  } else {
    r.rows = p.tile_slot_rows;
    r.dims = r.rows * 4;
    r.ml = p.tile_ml + slot * r.rows + row;
    r.o = p.tile_o + (slot * (p.head_dim >> 2) * r.rows + row) * 4;
  }
  return r;
}

// kSplit: a block joins one row, eight neighbouring threads sharing its partials:
// for calls whose rows would leave most of the GPU idle and have many.  A call in
// all, without and with it: a row of 32 heads over 8000 keys (37 partials) 25.1
// and 20.3 us, 4 rows of 32 heads behind 512 15.5 and 14.3, 11 rows in 4
// sequences over 500 to 4000 29.3 and 27.1, but 16 rows over 100 to 900 (3
// partials) 21.5 and 21.9.
constexpr int kJoinRows = 32;
template <bool kSplit>
__global__ void __launch_bounds__(256, 4) paged_combine_kernel(const __grid_constant__ PagedAttnParams p) {
  constexpr int32_t step = kSplit ? 8 : 1;
  const int32_t dim = (threadIdx.x >> 3) * 4, kv = blockIdx.y;
  const int32_t stream_cost = p.stream_prefix ? unit_cost((p.prefix + kStreamKeys - 1) / kStreamKeys) : 0;
  __shared__ Pieces shared_pieces[2][kJoinRows];  // own, prefix
  // One thread per row and kind finds the pieces.
  if (threadIdx.x < 2 * kJoinRows && (int32_t)(threadIdx.x % kJoinRows) < p.join_rows) {
    const bool prefix = threadIdx.x >= kJoinRows;
    const uint32_t index = blockIdx.x * p.join_rows + threadIdx.x % kJoinRows, row = index / (uint32_t)p.group;
    const int32_t in_group = (int32_t)(index - row * (uint32_t)p.group);
    Pieces r = {nullptr, nullptr, -1, 0, 0};
    PagedRow where;
    if (row < p.rows && paged_row(p.paged, row, where)) {
      r.count = 0;
      const int32_t tile_cost = unit_cost((p.prefix + kTileKeys - 1) / kTileKeys), per_unit = 2 * p.tile_rows;
      if (prefix && stream_cost) {
        const int32_t unit = kv * p.stream_prefix + (int32_t)index / 16;
        r = pieces_of(p, true, (int64_t)unit * stream_cost, stream_cost, unit, (int32_t)index % 16);
      } else if (prefix && p.prefix_units) {
        const int32_t unit = kv * p.prefix_units + (int32_t)row / per_unit;
        r = pieces_of(p, false, (int64_t)unit * tile_cost, tile_cost, unit, (int32_t)row % per_unit * p.group + in_group);
      } else if (!prefix) {
        const SequenceRows rows(p, where.sequence, false);
        const int32_t place = (int32_t)row - rows.begin, flat = place * p.group + in_group;
        if (few_rows(p, rows)) {
          const int32_t unit = p.stream_base[where.sequence] + flat / 16;
          if ((uint32_t)unit < (uint32_t)p.stream_units) {
            const int64_t before = p.stream_sums[unit], n = p.stream_sums[unit + 1] - before;
            r = pieces_of(p, true, ((int64_t)stream_cost * p.stream_prefix + before) * p.heads + kv * n, n,
                          (int64_t)(p.stream_prefix + unit) * p.heads + kv, flat % 16);
          }
        } else {
          const int32_t unit = p.unit_base[where.sequence] + place / per_unit;
          if ((uint32_t)unit < (uint32_t)p.tile_units) {
            const int64_t before = p.unit_sums[unit], n = p.unit_sums[unit + 1] - before;
            r = pieces_of(p, false, ((int64_t)p.prefix_units * tile_cost + before) * p.heads + kv * n, n,
                          (int64_t)(p.prefix_units + unit) * p.heads + kv, place % per_unit * p.group + in_group);
          }
        }
      }
    }
    shared_pieces[prefix][threadIdx.x % kJoinRows] = r;
  }
  __syncthreads();
  if (!kSplit && dim >= p.head_dim) return;
#pragma unroll 1
  for (int32_t sub = kSplit ? 0 : threadIdx.x & 7; sub < p.join_rows; sub += 8) {
    const Pieces own = shared_pieces[0][sub], pre = shared_pieces[1][sub];
    if (own.count < 0) continue;  // padding
    if (p.prefix == 0 && own.count == 1) continue;  // the whole unit was one CTA's, which wrote the result
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f, top = -INFINITY;
    // Four partials' loads are issued before the first is used, with no branch between them.
    const int64_t pre_step = (int64_t)pre.rows * p.head_dim, own_step = (int64_t)own.rows * p.head_dim;
    const float *pre_part = pre.o + (dim >> 2) * pre.dims, *own_part = own.o + (dim >> 2) * own.dims - pre.count * own_step;
    const float2 *own_ml = own.ml - (int64_t)pre.count * own.rows;
    const int32_t count = dim < p.head_dim ? pre.count + own.count : 0;
#pragma unroll 1
    for (int32_t first = kSplit ? threadIdx.x & 7 : 0; first < count; first += 4 * step) {
      float2 s[4];
      float4 v[4];
      float t = top;
#pragma unroll
      for (int32_t x = 0; x < 4; ++x) {
        s[x] = make_float2(-INFINITY, 0.0f);
        v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int32_t i = first + x * step;
        if (i < count) {
          const bool shared = i < pre.count;
          s[x] = shared ? pre.ml[(int64_t)i * pre.rows] : own_ml[(int64_t)i * own.rows];
          v[x] = *reinterpret_cast<const float4 *>(shared ? pre_part + i * pre_step : own_part + i * own_step);
        }
      }
#pragma unroll
      for (int32_t x = 0; x < 4; ++x) t = max_nan(t, s[x].x);
      if (t == -INFINITY) continue;  // no keys
      const float a = ex2_approx(top - t);
      top = t;
      l *= a;
      o.x *= a;
      o.y *= a;
      o.z *= a;
      o.w *= a;
#pragma unroll
      for (int32_t x = 0; x < 4; ++x) {
        if (s[x].x == -INFINITY) continue;  // (its O was not written)
        const float w = ex2_approx(s[x].x - t);
        l = fmaf(s[x].y, w, l);
        o.x = fmaf(v[x].x, w, o.x);
        o.y = fmaf(v[x].y, w, o.y);
        o.z = fmaf(v[x].z, w, o.z);
        o.w = fmaf(v[x].w, w, o.w);
      }
    }
    if (kSplit) {
#pragma unroll
      for (int m = 1; m < 8; m <<= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, m), t = max_nan(top, other);
        const float a = top == -INFINITY ? 0.0f : ex2_approx(top - t), b = other == -INFINITY ? 0.0f : ex2_approx(other - t);
        auto join = [&](float x) { return fmaf(x, a, __shfl_xor_sync(0xffffffffu, x, m) * b); };
        top = t;
        l = join(l);
        o = make_float4(join(o.x), join(o.y), join(o.z), join(o.w));
      }
      if ((threadIdx.x & 7) || dim >= p.head_dim) continue;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint2 v;
    v.x = to_h2(o.x * inv, o.y * inv);
    v.y = to_h2(o.z * inv, o.w * inv);
    const uint32_t index = blockIdx.x * p.join_rows + sub, row = index / (uint32_t)p.group;
    const int32_t in_group = (int32_t)(index - row * (uint32_t)p.group);
    *reinterpret_cast<uint2 *>(p.out + ((int64_t)row * p.q_heads + kv * p.group + in_group) * p.head_dim + dim) = v;
  }
}

// ---- host ---------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// How a call is cut up, from sizes the host knows, and its workspace.
struct PagedPlan {
  bool stream, tile_own;       // which kernels take own parts
  int32_t stream_prefix;       // the stream kernel takes the prefix, for so many groups of 16 rows
  bool tile;                   // the tile kernel runs
  int32_t sms, stream_rows, tile_rows, tile_slot_rows;
  int64_t prefix_units, stream_units, tile_units;
  uint64_t stream_o, stream_ml, stream_sums, stream_base, tile_o, tile_ml, unit_sums, unit_base, bytes;
};

PagedPlan paged_plan(int64_t rows, int64_t sequences, int64_t q_heads, int64_t heads, int64_t head_dim,
                     int64_t prefix_rows, bool ragged) {
  PagedPlan plan = {};
  const int64_t group = q_heads / heads;
  plan.sms = sm_count();
  // Sequences of few rows go to the stream kernel, the others to the tile kernel
  // (few_rows): 63 single rows next to a prompt of 512 over 600 to 3000 keys take
  // 108 us so and 188 us on the tile kernel alone.  No sequence can have many
  // where the call has few; and where they fill a unit of the tile kernel on
  // average, it takes all of them, which saves a launch.
  plan.stream = group <= 16 && (!ragged || rows * group <= 2 * kTileRows * sequences);
  plan.tile_own = !plan.stream || (ragged && rows * group > kFewRows);
  // The stream kernel takes the prefix too where its extra time, 0.6 us a key
  // tile and SM, is below the tile kernel's start: 23 rows of 16 heads behind
  // 729 positions take 20 against 25 us, 4 rows of 32 heads on 8 behind 512 15
  // against 22 us.
  const int64_t groups = ceil_div(rows * group, 16);
  if (plan.stream && prefix_rows > 0 && groups * heads * ceil_div(prefix_rows, kStreamKeys) * 0.6 < plan.sms * 8.0)
    plan.stream_prefix = (int32_t)groups;
  if (plan.stream && prefix_rows > 0 && groups == 1) plan.stream_prefix = 1;
  plan.tile_rows = (int32_t)(kTileRows / group);
  plan.tile_slot_rows = (int32_t)(2 * plan.tile_rows * group);
  plan.stream_rows = (int32_t)(plan.stream_prefix || ragged ? 16 : group);
  const int64_t per_unit = 2 * plan.tile_rows;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~uint64_t(255);
    return here;
  };
  if (plan.stream) {
    plan.stream_units = ragged ? rows * group / 16 + sequences : sequences;
    const int64_t slots =
        ((plan.stream_units + plan.stream_prefix) * heads + kStreamWorkers * plan.sms) * plan.stream_rows;
    plan.stream_o = take(slots * head_dim * 4);
    plan.stream_ml = take(slots * 8);
    plan.stream_sums = take((plan.stream_units + 3) * 8);
    plan.stream_base = take(sequences * 4);
  }
  if (prefix_rows > 0 && !plan.stream_prefix) plan.prefix_units = ceil_div(rows, per_unit);
  if (plan.tile_own) {
    const int64_t several = plan.stream ? rows * group / (kFewRows + 1) : rows;  // sequences with that many rows
    plan.tile_units = rows / per_unit + (sequences < several ? sequences : several);
  }
  if (plan.prefix_units || plan.tile_own) {
    plan.tile = true;
    const int64_t slots = ((plan.prefix_units + plan.tile_units) * heads + plan.sms) * plan.tile_slot_rows;
    plan.tile_o = take(slots * head_dim * 4);
    plan.tile_ml = take(slots * 8);
    plan.unit_sums = take((plan.tile_units + 3) * 8);
    plan.unit_base = take(sequences * 4);
  }
  plan.bytes = at > 256 ? at : 256;
  return plan;
}

int32_t gcd(int32_t a, int32_t b) {
  while (b) {
    const int32_t t = a % b;
    a = b;
    b = t;
  }
  return a;
}

// 4-D tile map (head_dim, d1, d2, d3) with box {b0, b1, 1, b3}, zero fill, 128-byte swizzle for b0 = 64.
ipuc_status make_map_paged(CUtensorMap *map, const void *base, int64_t head_dim, int64_t d1, int64_t d2, int64_t d3,
                           int64_t s1, int64_t s2, int64_t s3, int32_t b0, int32_t b1, int32_t b3) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(IPUC_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)d1, (cuuint64_t)d2, (cuuint64_t)d3};
  const cuuint64_t strides[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s3 * 2};
  const cuuint32_t box[4] = {(cuuint32_t)b0, (cuuint32_t)b1, 1, (cuuint32_t)b3};
  const CUresult r = encode_tiled(fn, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box,
                                  b0 == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE);
  if (r != CUDA_SUCCESS)
    return fail(IPUC_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
  return IPUC_OK;
}

}  // namespace
}  // namespace ipuc

using namespace ipuc;


extern "C" uint64_t ipuc_paged_attention_workspace_bytes(int64_t rows, int64_t sequences, int64_t q_heads,
                                                         int64_t heads, int64_t head_dim, int64_t prefix_rows,
                                                         int32_t ragged) {
  if (rows < 0 || sequences < 0 || heads < 1 || q_heads < heads || q_heads > 128 * heads || head_dim < 1 || prefix_rows < 0)
    return 0;  // the call refuses these
  return paged_plan(rows, sequences, q_heads, heads, head_dim, prefix_rows, ragged != 0).bytes;
}

extern "C" ipuc_status ipuc_paged_attention_f16(void *out, const void *q, int64_t q_stride, int64_t q_heads,
                                                const ipuc_paged_cache *cache, const ipuc_paged_batch *batch,
                                                int64_t prefix_rows, const int32_t *prefix_pages, float scale,
                                                void *workspace, uint64_t workspace_bytes, ipuc_stream stream) {
  ipuc_status st = check_paged("paged_attention", cache, batch);
  if (st != IPUC_OK) return st;
  const int64_t d = cache->head_dim;
  IPUC_CHECK_ARG(d % 8 == 0, "paged_attention: head_dim must be a multiple of 8");
  if (d > 128) return fail(IPUC_ERR_UNSUPPORTED, "paged_attention: head_dim above 128 is not supported");
  IPUC_CHECK_ARG(q_heads >= 1 && q_heads < (1 << 16) && q_heads % cache->heads == 0,
                 "paged_attention: query heads must be a multiple of the cache's heads");
  if (q_heads / cache->heads > 128)
    return fail(IPUC_ERR_UNSUPPORTED, "paged_attention: more than 128 query heads per key head are not supported");
  IPUC_CHECK_ARG(prefix_rows >= 0 && prefix_rows < (1ll << 31) - 256, "paged_attention: prefix_rows out of range");
  IPUC_CHECK_ARG(prefix_rows == 0 || prefix_pages, "paged_attention: null prefix_pages");
  IPUC_CHECK_ARG(isfinite(scale) && (scale <= 0.0f || isfinite(scale * kLog2e)), "paged_attention: scale must be finite");
  IPUC_CHECK_ARG(q_stride >= q_heads * d, "paged_attention: token stride shorter than q_heads * head_dim");
  IPUC_CHECK_ALIGN(q_stride % 8 == 0 && cache->page_stride % 8 == 0 && cache->head_stride % 8 == 0 &&
                       cache->row_stride % 8 == 0,
                   "paged_attention: strides must be multiples of 8 elements");
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  IPUC_CHECK_ARG(out && q, "paged_attention: null pointer");
  IPUC_CHECK_ALIGN(aligned(out, 16) && aligned(q, 16) && aligned(cache->keys, 16) && aligned(cache->values, 16),
                   "paged_attention: pointers must be 16-byte aligned");
  IPUC_CHECK_ALIGN(aligned(prefix_pages, 4), "paged_attention: int32 arrays must be 4-byte aligned");
  const uintptr_t out_at = reinterpret_cast<uintptr_t>(out), q_at = reinterpret_cast<uintptr_t>(q);
  IPUC_CHECK_ARG(batch->rows < (1ll << 31) / q_heads && q_stride < (1ll << 40), "paged_attention: extent too large");
  IPUC_CHECK_ARG(out_at >= q_at + (uint64_t)((batch->rows - 1) * q_stride + q_heads * d) * 2 ||
                     q_at >= out_at + (uint64_t)(batch->rows * q_heads * d) * 2,
                 "paged_attention: out overlaps q");
  const PagedPlan plan = paged_plan(batch->rows, batch->sequences, q_heads, cache->heads, d, prefix_rows,
                                    batch->row_offsets != nullptr);
  IPUC_CHECK_ARG(workspace && workspace_bytes >= plan.bytes,
                 "paged_attention: workspace smaller than ipuc_paged_attention_workspace_bytes");
  IPUC_CHECK_ALIGN(aligned(workspace, 256), "paged_attention: workspace must be 256-byte aligned");
  PagedAttnParams p = {};
  uint8_t *ws = static_cast<uint8_t *>(workspace);
  p.out = static_cast<uint16_t *>(out);
  p.q = static_cast<const uint16_t *>(q);
  p.paged = paged_view(cache, batch);
  p.prefix_pages = prefix_pages;
  p.q_stride = q_stride;
  p.rows = batch->rows;
  p.q_heads = (int32_t)q_heads;
  p.heads = cache->heads;
  p.group = (int32_t)(q_heads / cache->heads);
  p.head_dim = (int32_t)d;
  p.prefix = (int32_t)prefix_rows;
  p.chunk = gcd(cache->page_size, kStreamKeys);
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)d)) * kLog2e;
  p.stream_o = reinterpret_cast<float *>(ws + plan.stream_o);
  p.stream_ml = reinterpret_cast<float2 *>(ws + plan.stream_ml);
  p.stream_sums = reinterpret_cast<int64_t *>(ws + plan.stream_sums);
  p.stream_base = reinterpret_cast<int32_t *>(ws + plan.stream_base);
  p.stream_rows = plan.stream_rows;
  p.stream = plan.stream;
  p.sms = plan.sms;
  p.stream_prefix = plan.stream_prefix;
  p.tile_o = reinterpret_cast<float *>(ws + plan.tile_o);
  p.tile_ml = reinterpret_cast<float2 *>(ws + plan.tile_ml);
  p.unit_sums = reinterpret_cast<int64_t *>(ws + plan.unit_sums);
  p.unit_base = reinterpret_cast<int32_t *>(ws + plan.unit_base);
  p.tile_slot_rows = plan.tile_slot_rows;
  p.tile_own = plan.tile_own;
  p.prefix_units = (int32_t)plan.prefix_units;
  p.stream_units = (int32_t)plan.stream_units;
  p.tile_units = (int32_t)plan.tile_units;
  p.over_group = ((1ull << 36) + (uint64_t)p.group - 1) / (uint64_t)p.group;
  p.tile_rows = plan.tile_rows;
  p.err = device_error_word();
  const int64_t tasks = p.rows * q_heads;
  // (sums over units are held in 23 bits, their key tiles in 40)
  const int64_t units = plan.prefix_units + plan.tile_units + plan.stream_prefix + plan.stream_units;
  const int64_t keys = (int64_t)batch->max_pages * cache->page_size;
  IPUC_CHECK_ARG(tasks < (1ll << 31) - 256 && units < (1ll << 23) &&
                     units * p.heads < (1ll << 40) / ((keys > prefix_rows ? keys : prefix_rows) / kStreamKeys + 4),
                 "paged_attention: extent too large");
  CUtensorMap tm_q, tm_k, tm_v;
  auto cache_map = [&](CUtensorMap *map, const void *base, int32_t box) {
    return make_map_paged(map, base, d, cache->page_size, cache->heads, cache->pages, cache->row_stride,
                          cache->head_stride, cache->page_stride, box, p.chunk, 1);
  };
  // The stream kernel runs beside the tile kernel, whose start takes longer, on
  // the SMs that leaves it (programmatic dependent launch).  The join is an
  // ordinary launch: an early one gained nothing (15.9 against 16.0 us for few
  // rows, 31 against 29 for few rows of ragged batches).
  auto launch = [&](auto kernel, dim3 grid, int threads, int bytes, int most, bool beside, auto... args) -> ipuc_status {
    if (most) IPUC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = beside ? 1 : 0;
    IPUC_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return check_launch("paged_attention");
  };
  if (plan.tile) {
    st = make_map_paged(&tm_q, q, d, p.group, cache->heads, p.rows, d, p.group * d, q_stride, 64, p.group, p.tile_rows);
    if (st == IPUC_OK) st = cache_map(&tm_k, cache->keys, 64);
    if (st == IPUC_OK) st = cache_map(&tm_v, cache->values, 64);
    if (st == IPUC_OK) st = launch(paged_tile_kernel, p.sms, kTileThreads, kTileSmem, kTileSmem, false, tm_q, tm_k, tm_v, p);
    if (st != IPUC_OK) return st;
  }
  if (plan.stream) {
    const int32_t padded = d <= 64 ? 64 : d <= 80 ? 80 : d <= 96 ? 96 : 128;
    const StreamShape shape = stream_shape(padded, p.chunk);
    p.pitch = shape.pitch;
    p.stages = shape.stages;
    const int32_t box = stream_swizzled(padded) ? 64 : shape.pitch / 2;
    if (!plan.tile || box != 64) {  // (else they are there)
      st = cache_map(&tm_k, cache->keys, box);
      if (st == IPUC_OK) st = cache_map(&tm_v, cache->values, box);
      if (st != IPUC_OK) return st;
    }
    auto stream_kernel = [&](auto kernel, int most) {
      return launch(kernel, p.sms, kStreamThreads, shape.bytes, most, plan.tile, tm_k, tm_v, p);
    };
    st = padded == 64   ? stream_kernel(paged_stream_kernel<64>, stream_bytes(64))
         : padded == 80 ? stream_kernel(paged_stream_kernel<80>, stream_bytes(80))
         : padded == 96 ? stream_kernel(paged_stream_kernel<96>, stream_bytes(96))
                        : stream_kernel(paged_stream_kernel<128>, stream_bytes(128));
    if (st != IPUC_OK) return st;
  }
  // Few rows: many small blocks; more than fill the GPU: fewer, which find their pieces at once.
  const int64_t heads_rows = p.rows * q_heads, resident = 4 * (int64_t)p.sms;
  const bool split = heads_rows <= 3 * p.sms;
  p.join_rows = split ? 1 : heads_rows >= 8 * resident ? kJoinRows : 8;
  const dim3 grid((unsigned)ceil_div(p.rows * p.group, p.join_rows), (unsigned)p.heads);
  return split ? launch(paged_combine_kernel<true>, grid, 256, 0, 0, false, p)
               : launch(paged_combine_kernel<false>, grid, 256, 0, 0, false, p);
}
