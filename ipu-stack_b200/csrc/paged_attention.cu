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

struct PagedAttnParams {
  uint16_t *out;
  const uint16_t *q;
  PagedView paged;
  const int32_t *prefix_pages;
  int64_t q_stride, rows;
  int32_t q_heads, heads, group, head_dim, prefix;
  int32_t chunk;          // keys per TMA box: gcd(page_size, 64)
  float scale_log2;       // softmax scale * log2(e)
  // Partial results: unnormalised O (f32, head_dim wide) and (running maximum
  // in log2 units, sum of weights) per row and query head.
  float *own_o, *prefix_o;
  float2 *own_ml, *prefix_ml;
  int64_t *tile_sums;     // single rows: own key tiles of the sequences before b, [sequences + 1]
  int32_t stream_ctas;    // single rows: CTAs of the own-part kernel; 0: the tile kernel took it
  int32_t own_splits, prefix_splits;
  int32_t row_units;      // tile kernel: units of 2 * tile_rows rows per head
  int32_t tile_rows;      // tile kernel: batch rows per 128-row MMA tile, 128 / group
  int32_t direct;         // the tile kernel's result is final
  uint32_t *err;
};

// Length of sequence b as far as its table row can hold it.
__device__ __forceinline__ int32_t checked_length(const PagedAttnParams &p, int32_t b, bool report) {
  const int32_t n = p.paged.lengths[b], cap = p.paged.max_pages * p.paged.page_size;
  if (n > cap && report && n > p.prefix) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_LENGTH);
  return n < 0 ? 0 : min(n, max(cap, p.prefix));
}

// Exclusive sums of count(b) over the block's threads' contiguous shares of
// [0, n): returns the total; store(b, sum before b) is called for every b.
template <int kThreads, typename Count, typename Store>
__device__ __forceinline__ int64_t block_sums(int32_t n, int64_t *scratch, Count count, Store store) {
  const int32_t share = (n + kThreads - 1) / kThreads;
  const int32_t lo = min(n, (int32_t)threadIdx.x * share), hi = min(n, lo + share);
  int64_t mine = 0;
  for (int32_t b = lo; b < hi; ++b) mine += count(b);
  int64_t sum = mine;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += x;
  }
  if (lane == 31) scratch[warp] = sum;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += scratch[w];
    total += scratch[w];
  }
  before += sum - mine;
  for (int32_t b = lo; b < hi; ++b) {
    store(b, before);
    before += count(b);
  }
  return total;
}

// Page coordinate of the chunk of keys at position `pos`: out of range (the
// TMA then fills zeros) where the chunk has no key of [lo, hi) or its page id
// is not one.
__device__ __forceinline__ int32_t page_of(const PagedAttnParams &p, const int32_t *ids, int32_t pos, int32_t lo,
                                           int32_t hi) {
  if (pos >= hi || pos + p.chunk <= lo) return p.paged.pages;
  const int32_t id = ids[pos / p.paged.page_size];
  if (id < 0 || id >= p.paged.pages) {
    record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PAGE);
    return p.paged.pages;
  }
  return id;
}

// ---- single rows: the sequences' own parts ------------------------------------

// One row per sequence and at most 16 query heads per key head: the group is
// one m16n8k16 tile, so a key costs 16 x 128 multiply-adds whatever the group,
// and K and V are streamed once: HBM-bound.  The key tiles (64 keys, at
// absolute multiples of 64) of all (sequence, head) units form one line that
// is cut into equal pieces, one per CTA, so ragged lengths leave no CTA idle.
// A producer warp fills a ring of tiles by TMA, box by box of gcd(page_size,
// 64) keys; four warps take 16 keys of every tile each, with a running
// maximum, sum and O of their own, and meet once per unit.
constexpr int kStreamKeys = 64, kStreamStages = 3, kStreamThreads = 160, kMergeLd = 36;

template <int DP>
constexpr int stream_smem_bytes() {
  return kStreamStages * 2 * kStreamKeys * DP * 2 + 4 * 16 * kMergeLd * 4 + 1024;
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
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A CTA's place on the line of key tiles: unit (b, h), tile i of its n.
struct StreamWalk {
  int32_t b, h, i, n, len;
  int64_t left;

  __device__ __forceinline__ static int32_t tiles(const PagedAttnParams &p, int32_t len) {
    return len > p.prefix ? (len + kStreamKeys - 1) / kStreamKeys - p.prefix / kStreamKeys : 0;
  }
  __device__ __forceinline__ void step(const PagedAttnParams &p, int32_t count) {
    left -= count;
    i += count;
    if (i < n || left <= 0) return;
    i = 0;
    if (++h < p.heads) return;
    h = 0;
    do {
      if (++b >= p.paged.sequences) {
        left = 0;
        return;
      }
      len = checked_length(p, b, false);
      n = tiles(p, len);
    } while (n == 0);
  }
};

template <int DP>
__global__ void __launch_bounds__(kStreamThreads, 2)
    paged_stream_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                        const __grid_constant__ PagedAttnParams p) {
  constexpr int HALVES = DP / 64, KS = DP / 16, NT = DP / 8;
  constexpr int HALF_BYTES = kStreamKeys * 128, TILE_BYTES = HALVES * HALF_BYTES;  // K or V of a tile
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float *merge = reinterpret_cast<float *>(smem + kStreamStages * 2 * TILE_BYTES);  // [4][16][kMergeLd]
  __shared__ uint64_t full[kStreamStages], empty[kStreamStages];
  __shared__ int64_t scratch[kStreamThreads / 32], first_left[2];
  __shared__ int32_t first_unit[4];
  __shared__ float warp_m[4][16], warp_l[4][16];
  __shared__ int aborted;
  volatile int *abort_flag = &aborted;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStreamStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    aborted = 0;
    first_left[1] = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  const int64_t cta = blockIdx.x;
  auto count = [&](int32_t b) { return StreamWalk::tiles(p, checked_length(p, b, cta == 0)); };
  // Sums first, then this CTA's piece [W c / C, W (c + 1) / C) of the line of W tiles.
  int64_t starts[2] = {0, 0};
  const int64_t total = block_sums<kStreamThreads>(p.paged.sequences, scratch, count, [&](int32_t b, int64_t sum) {
    if (cta == 0) p.tile_sums[b] = sum;
  });
  if (cta == 0 && threadIdx.x == 0) p.tile_sums[p.paged.sequences] = total;
  griddep_launch_dependents();
  const int64_t line = total * p.heads, ctas = min((int64_t)gridDim.x, line);  // no piece is empty
  if (cta >= ctas) return;
  starts[0] = line * cta / ctas;
  starts[1] = line * (cta + 1) / ctas;
  __syncthreads();  // scratch is read before it is written again
  block_sums<kStreamThreads>(p.paged.sequences, scratch, count, [&](int32_t b, int64_t sum) {
    const int32_t n = count(b);
    const int64_t at = starts[0] - sum * p.heads;
    if (at >= 0 && at < (int64_t)n * p.heads) {
      first_unit[0] = b;
      first_unit[1] = (int32_t)(at / n);
      first_unit[2] = (int32_t)(at % n);
      first_unit[3] = n;
    }
  });
  __syncthreads();
  StreamWalk w;
  w.b = first_unit[0];
  w.h = first_unit[1];
  w.i = first_unit[2];
  w.n = first_unit[3];
  w.len = checked_length(p, w.b, false);
  w.left = starts[1] - starts[0];
  const int32_t tile0 = p.prefix / kStreamKeys;  // first key tile of every unit

  if (warp == 4) {
    // Producer: lane l issues boxes l, l + 32, ... of a tile: (K or V, half, chunk).
    const int chunks = kStreamKeys / p.chunk, boxes = 2 * HALVES * chunks;
    bool ok = true;
    uint32_t t = 0;
    for (; w.left > 0 && ok; ++t, w.step(p, 1)) {
      const int st = t % kStreamStages;
      const int32_t key0 = (tile0 + w.i) * kStreamKeys;
      const int32_t *ids = p.paged.page_table + w.b * p.paged.table_stride;
      // this lane's first box's page is looked up before the stage is free
      int32_t page = lane < boxes ? page_of(p, ids, key0 + (lane % chunks) * p.chunk, p.prefix, w.len) : 0;
      if (!mbar_wait_bounded(&empty[st], ((t / kStreamStages) & 1) ^ 1, abort_flag)) {
        ok = false;
        break;
      }
      if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * TILE_BYTES);
      __syncwarp();
      uint8_t *base = smem + st * 2 * TILE_BYTES;
      for (int x = lane; x < boxes; x += 32) {
        const int chunk = x % chunks, half = (x / chunks) % HALVES, v = x / (chunks * HALVES);
        const int32_t pos = key0 + chunk * p.chunk;
        if (x >= 32) page = page_of(p, ids, pos, p.prefix, w.len);
        tma_load_4d(base + v * TILE_BYTES + half * HALF_BYTES + chunk * p.chunk * 128, v ? &tm_v : &tm_k, &full[st],
                    half * 64, pos % p.paged.page_size, w.h, page);
      }
    }
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PRODUCER);
      *abort_flag = 1;
      // nothing leaves while copies into its shared memory are in flight
      for (uint32_t x = t > kStreamStages ? t - kStreamStages : 0; x < t; ++x)
        mbar_wait_bounded(&full[x % kStreamStages], (x / kStreamStages) & 1, nullptr, 1000000000ull);
    }
    return;
  }

  // Consumers.  A fragments: rows lane / 4 and lane / 4 + 8 of the group.
  const int r0 = lane >> 2, r1 = r0 + 8, cq = (lane & 3) * 2;
  auto load_q = [&](const StreamWalk &u, uint32_t (&a)[KS][4]) {
    const uint16_t *base = p.q + u.b * p.q_stride + (int64_t)u.h * p.group * p.head_dim;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = j & 1 ? r1 : r0, col = k * 16 + cq + (j & 2 ? 8 : 0);
        a[k][j] = row < p.group && col < p.head_dim
                      ? *reinterpret_cast<const uint32_t *>(base + row * p.head_dim + col)
                      : 0u;
      }
  };
  uint32_t q[KS][4];
  load_q(w, q);
  // ldmatrix addresses: lane -> row lane % 8 of matrix lane / 8.  K matrices:
  // (keys 0-7, 8-15) x (two 16-byte column chunks); V: keys fastest.
  const int mi = lane >> 3, mr = lane & 7;
  const uint32_t k_row = warp * 16 + (mi >> 1) * 8 + mr, v_row = warp * 16 + (mi & 1) * 8 + mr;
  const uint32_t sbase = smem_u32(smem);
  const float c = p.scale_log2;
  bool ok = true;
  uint32_t t = 0;
  while (w.left > 0) {
    const int32_t count_here = (int32_t)min((int64_t)(w.n - w.i), w.left);
    float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    for (int32_t k = 0; k < count_here; ++k, ++t) {
      const int st = t % kStreamStages;
      // (a wait that ran out is not left early: the barriers below need every warp)
      if (ok && !mbar_wait_bounded(&full[st], (t / kStreamStages) & 1, abort_flag)) ok = false;
      const uint32_t ks = sbase + st * 2 * TILE_BYTES, vs = ks + TILE_BYTES;
      const int32_t key0 = (tile0 + w.i + k) * kStreamKeys + warp * 16;
      float s[2][4] = {}, s2[2][4] = {};  // even and odd steps: two chains
#pragma unroll
      for (int d = 0; d < KS; ++d) {
        uint32_t b[4];
        const uint32_t chunk = (d * 2 + (mi & 1)) & 7;
        ldmatrix_x4(ks + (d >> 2) * HALF_BYTES + k_row * 128 + ((chunk ^ (k_row & 7)) << 4), b);
        mma_16816(d & 1 ? s2[0] : s[0], q[d], b[0], b[1]);
        mma_16816(d & 1 ? s2[1] : s[1], q[d], b[2], b[3]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[0][j] += s2[0][j];
        s[1][j] += s2[1][j];
      }
      if (key0 < p.prefix || key0 + 16 > w.len) {
        // The unit's first or last tile: scores of keys that are not its own
        // are dropped, and the warp's V rows of such keys, which may hold
        // anything, are zeroed (0 * NaN is NaN).
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int32_t key = key0 + x * 8 + cq + (j & 1);
            if (key < p.prefix || key >= w.len) s[x][j] = -INFINITY;
          }
        for (int x = lane; x < 16 * HALVES * 8; x += 32) {
          const int row = x / (HALVES * 8), half = (x >> 3) % HALVES;
          if (key0 + row < p.prefix || key0 + row >= w.len) {
            const uint32_t at = vs + half * HALF_BYTES + (warp * 16 + row) * 128 + (x & 7) * 16;
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
      uint32_t a[4];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const float p0 = ex2_approx(fmaf(s[x][0], c, n0)), p1 = ex2_approx(fmaf(s[x][1], c, n0));
        const float p2 = ex2_approx(fmaf(s[x][2], c, n1)), p3 = ex2_approx(fmaf(s[x][3], c, n1));
        l0 += p0 + p1;
        l1 += p2 + p3;
        a[2 * x] = pack_h2(p0, p1);
        a[2 * x + 1] = pack_h2(p2, p3);
      }
#pragma unroll
      for (int d = 0; d < NT; d += 2) {
        uint32_t b[4];
        const uint32_t chunk = (d + (mi >> 1)) & 7;
        ldmatrix_x4_trans(vs + (d >> 3) * HALF_BYTES + v_row * 128 + ((chunk ^ (v_row & 7)) << 4), b);
        mma_16816(o[d], a, b[0], b[1]);
        mma_16816(o[d + 1], a, b[2], b[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }
    // The next unit's queries load while this one's results meet.
    StreamWalk next = w;
    next.step(p, count_here);
    uint32_t qn[KS][4];
    if (next.left > 0) load_q(next, qn);
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
    named_barrier_sync(1, 128);
    const float t0 = fmaxf(fmaxf(warp_m[0][r0], warp_m[1][r0]), fmaxf(warp_m[2][r0], warp_m[3][r0]));
    const float t1 = fmaxf(fmaxf(warp_m[0][r1], warp_m[1][r1]), fmaxf(warp_m[2][r1], warp_m[3][r1]));
    const float a0 = m0 == -INFINITY ? 0.0f : ex2_approx((m0 - t0) * c);
    const float a1 = m1 == -INFINITY ? 0.0f : ex2_approx((m1 - t1) * c);
    const int orow = threadIdx.x >> 3, ocol = (threadIdx.x & 7) * 4;  // this thread's share of the sums
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) top = fmaxf(top, warp_m[x][orow]);
#pragma unroll
    for (int x = 0; x < 4; ++x)
      if (warp_m[x][orow] != -INFINITY) sum += warp_l[x][orow] * ex2_approx((warp_m[x][orow] - top) * c);
    const bool whole = p.prefix == 0 && count_here == w.n;
    const int64_t slot = ((int64_t)w.b * p.heads + w.h + cta) * p.group + orow;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (!whole && orow < p.group && ocol == 0) p.own_ml[slot] = make_float2(top == -INFINITY ? top : top * c, sum);
#pragma unroll
    for (int round = 0; round < DP / 32; ++round) {
      float *mine = merge + warp * 16 * kMergeLd;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float(&v)[4] = o[round * 4 + i];
        *reinterpret_cast<float2 *>(mine + r0 * kMergeLd + i * 8 + cq) = make_float2(v[0] * a0, v[1] * a0);
        *reinterpret_cast<float2 *>(mine + r1 * kMergeLd + i * 8 + cq) = make_float2(v[2] * a1, v[3] * a1);
      }
      named_barrier_sync(1, 128);
      const int col = round * 32 + ocol;
      if (orow < p.group && col < p.head_dim) {
        float4 r = *reinterpret_cast<const float4 *>(merge + orow * kMergeLd + ocol);
#pragma unroll
        for (int x = 1; x < 4; ++x) {
          const float4 y = *reinterpret_cast<const float4 *>(merge + (x * 16 + orow) * kMergeLd + ocol);
          r.x += y.x;
          r.y += y.y;
          r.z += y.z;
          r.w += y.w;
        }
        if (whole) {
          uint2 h;
          h.x = pack_h2(r.x * inv, r.y * inv);
          h.y = pack_h2(r.z * inv, r.w * inv);
          const int64_t head = (int64_t)w.b * p.q_heads + w.h * p.group + orow;
          *reinterpret_cast<uint2 *>(p.out + head * p.head_dim + col) = h;
        } else {
          *reinterpret_cast<float4 *>(p.own_o + slot * p.head_dim + col) = r;
        }
      }
      named_barrier_sync(1, 128);
    }
    w = next;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) q[k][j] = qn[k][j];
  }
  if (!ok) {
    if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_EPILOGUE);
    *abort_flag = 1;
  }
}

// ---- many rows: tiles of 128 on the tensor cores --------------------------------

// Rows that read the same keys (all rows of the call for the shared prefix;
// one sequence's rows for its own part) are packed group by group into
// 128-row MMA tiles, tile_rows = 128 / group batch rows to a tile.  One CTA
// owns two tiles of one key head and a range of 128-key tiles:
//   warp 0      loads: Q once, then K and V tiles through two-stage rings, box
//               by box of gcd(page_size, 64) keys
//   warp 1      S_t = Q_t K^T into TMEM, O_t += P_t V with P_t read from TMEM
//               (it overwrites S_t as packed f16)
//   warps 2-17  softmax: two warps per lane quarter of a tile, 64 keys each
// so the tensor core works on one tile while the other's softmax runs.
constexpr int kTileRows = 128, kTileKeys = 128;
constexpr int kTileBytes = 128 * 128 * 2, kTileHalf = kTileBytes / 2;
constexpr int kTileThreads = 576, kTileSmem = 6 * kTileBytes + 1024;

template <bool kPrefix>
__global__ void __launch_bounds__(kTileThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ PagedAttnParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *s_q = smem, *s_k = smem + 2 * kTileBytes, *s_v = smem + 4 * kTileBytes;
  __shared__ uint64_t q_full, k_full[2], v_full[2], k_empty[2], v_empty[2], s_full[2], p_ready[2], v_fixed[2], o_final;
  __shared__ uint32_t tmem_slot;
  __shared__ int aborted;
  __shared__ float x_max[2][2][kTileRows], x_sum[2][2][kTileRows];
  __shared__ int64_t scratch[kTileThreads / 32];
  __shared__ int32_t found[2];
  volatile int *abort_flag = &aborted;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // The unit: `rows` batch rows from row0 on (of sequence `seq` at position
  // pos0, or of all sequences), key head h, share `split` of the key tiles of
  // positions [lo, hi).
  int32_t x = blockIdx.x;
  const int32_t unit = x % p.row_units;
  x /= p.row_units;
  const int32_t h = x % p.heads, split = x / p.heads, splits = kPrefix ? p.prefix_splits : p.own_splits;
  const int32_t per_unit = 2 * p.tile_rows;
  int64_t row0 = (int64_t)unit * per_unit, pos0 = 0;
  int32_t rows = 0, lo = 0, hi = 0, seq = 0;
  if (kPrefix) {
    rows = (int32_t)min((int64_t)per_unit, p.rows - row0);
    hi = p.prefix;
  } else {
    // Sequence b has ceil(rows / per_unit) units.
    auto first_row = [&](int32_t b) {
      return p.paged.row_offsets ? max(0, min(p.paged.row_offsets[b], (int32_t)p.rows)) : b;
    };
    auto count = [&](int32_t b) { return max(0, (first_row(b + 1) - first_row(b) + per_unit - 1) / per_unit); };
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    block_sums<kTileThreads>(p.paged.sequences, scratch, count, [&](int32_t b, int64_t sum) {
      if (unit >= sum && unit < sum + count(b)) {
        found[0] = b;
        found[1] = (int32_t)(unit - sum);
      }
    });
    __syncthreads();
    seq = found[0];
    if (seq < 0) return;  // the grid is an upper bound
    const int32_t begin = first_row(seq), end = first_row(seq + 1);
    row0 = begin + (int64_t)found[1] * per_unit;
    rows = (int32_t)min((int64_t)per_unit, end - row0);
    const int32_t len = checked_length(p, seq, true);
    pos0 = (int64_t)p.paged.lengths[seq] - (end - begin) + (row0 - begin);
    lo = p.prefix;
    hi = (int32_t)max((int64_t)0, min((int64_t)len, pos0 + rows));
  }
  const int32_t first = lo / kTileKeys, count = hi > lo ? (hi + kTileKeys - 1) / kTileKeys - first : 0;
  const int32_t j_begin = first + (int32_t)((int64_t)count * split / splits);
  const int32_t n_tiles = first + (int32_t)((int64_t)count * (split + 1) / splits) - j_begin;
  float *part_o = kPrefix ? p.prefix_o : p.own_o;
  float2 *part_ml = kPrefix ? p.prefix_ml : p.own_ml;
  if (n_tiles == 0) {
    // No keys: empty partials (O is not read where the maximum is -inf), or zero rows.
    for (int32_t i = threadIdx.x; i < rows * p.group; i += kTileThreads) {
      const int64_t head = (row0 + i / p.group) * p.q_heads + h * p.group + i % p.group;
      if (!p.direct) {
        part_ml[split * p.rows * p.q_heads + head] = make_float2(-INFINITY, 0.0f);
      } else {
        for (int d = 0; d < p.head_dim; d += 8)
          *reinterpret_cast<uint4 *>(p.out + head * p.head_dim + d) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }
  const int tiles = rows > p.tile_rows ? 2 : 1;  // row tiles in use
  const int halves = p.head_dim > 64 ? 2 : 1, k_steps = (p.head_dim + 15) / 16;

  if (threadIdx.x == 0) {
    mbar_init(&q_full, 1);
    mbar_init(&o_final, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 8);
      mbar_init(&v_fixed[i], 1);
    }
    aborted = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;  // S_t at column t * 128, O_t at 256 + t * 128
  // V rows outside [lo, hi) of a chunk that has both kinds may hold anything and
  // are zeroed in shared memory (0 * NaN is NaN): in the first tile (0) and in
  // the last one (1).  Whole chunks outside are zero-filled by the TMA.
  const bool fix_first = j_begin * kTileKeys < lo && lo % p.chunk != 0;
  const bool fix_last = (j_begin + n_tiles) * kTileKeys > hi && hi % p.chunk != 0;

  if (warp == 0) {
    const int chunks = kTileKeys / p.chunk, boxes = halves * chunks;
    const int32_t *ids = kPrefix ? p.prefix_pages : p.paged.page_table + seq * p.paged.table_stride;
    bool ok = true;
    int k_issued = 0, v_issued = 0;
    if (lane == 0) {
      mbar_arrive_expect_tx(&q_full, tiles * halves * p.tile_rows * p.group * 128);
      for (int t = 0; t < tiles; ++t)
        for (int half = 0; half < halves; ++half)
          tma_load_4d(s_q + t * kTileBytes + half * kTileHalf, &tm_q, &q_full, half * 64, 0, h,
                      (int32_t)row0 + t * p.tile_rows);
    }
    auto load = [&](uint8_t *base, const CUtensorMap *map, uint64_t *bar, int32_t key0) {
      if (lane == 0) mbar_arrive_expect_tx(bar, halves * kTileHalf);
      __syncwarp();
      for (int i = lane; i < boxes; i += 32) {
        const int chunk = i % chunks, half = i / chunks;
        const int32_t pos = key0 + chunk * p.chunk;
        tma_load_4d(base + half * kTileHalf + chunk * p.chunk * 128, map, bar, half * 64, pos % p.paged.page_size, h,
                    page_of(p, ids, pos, lo, hi));
      }
    };
    for (int j = 0; j < n_tiles && ok; ++j) {
      const int st = j & 1;
      const int32_t key0 = (j_begin + j) * kTileKeys;
      if (!mbar_wait_bounded(&k_empty[st], ((j >> 1) & 1) ^ 1, abort_flag)) {
        ok = false;
        break;
      }
      load(s_k + st * kTileBytes, &tm_k, &k_full[st], key0);
      ++k_issued;
      if (!mbar_wait_bounded(&v_empty[st], ((j >> 1) & 1) ^ 1, abort_flag)) {
        ok = false;
        break;
      }
      load(s_v + st * kTileBytes, &tm_v, &v_full[st], key0);
      ++v_issued;
      const bool is_last = j == n_tiles - 1;
      if ((fix_first && j == 0) || (fix_last && is_last)) {
        if (!mbar_wait_bounded(&v_full[st], (j >> 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        for (int i = lane; i < kTileKeys * halves * 8; i += 32) {
          const int row = i / (halves * 8), half = (i >> 3) % halves;
          if (key0 + row < lo || key0 + row >= hi)
            *reinterpret_cast<uint4 *>(s_v + st * kTileBytes + half * kTileHalf + row * 128 + (i & 7) * 16) =
                make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_fixed[fix_first && j == 0 ? 0 : 1]);
      }
    }
    if (!ok) {
      if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_PRODUCER);
      *abort_flag = 1;
    }
    // Nothing leaves while copies into its shared memory are in flight (at once
    // unless a wait ran out above: the MMA warp has waited for all of them).
    mbar_wait_bounded(&q_full, 0, nullptr, 1000000000ull);
    for (int i = max(0, k_issued - 2); i < k_issued; ++i)
      mbar_wait_bounded(&k_full[i & 1], (i >> 1) & 1, nullptr, 1000000000ull);
    for (int i = max(0, v_issued - 2); i < v_issued; ++i)
      mbar_wait_bounded(&v_full[i & 1], (i >> 1) & 1, nullptr, 1000000000ull);
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc_s = make_idesc(128, kTileKeys, 0, false, false);
      const uint32_t idesc_o = make_idesc(128, k_steps * 16, 0, false, true);  // V: head dims contiguous
      const uint64_t q_desc = make_smem_desc(smem_u32(s_q), 16, 1024, kSwizzle128B);
      const uint64_t k_desc = make_smem_desc(smem_u32(s_k), 16, 1024, kSwizzle128B);
      const uint64_t v_desc = make_smem_desc(smem_u32(s_v), kTileHalf, 1024, kSwizzle128B);
      auto issue_s = [&](int t, int st) {
        const uint64_t qd = q_desc + (uint64_t)(t * (kTileBytes >> 4)), kd = k_desc + (uint64_t)(st * (kTileBytes >> 4));
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (k < k_steps) {
            const uint64_t step = (uint64_t)(((k >> 2) * kTileHalf + (k & 3) * 32) >> 4);
            mma_f16_ss(tmem + t * 128, qd + step, kd + step, idesc_s, k > 0 ? 1u : 0u);
          }
        }
        mma_commit(&s_full[t]);
      };
      // Per key tile j: PV_t(j) as soon as P_t(j) is there, then S_t(j + 1) behind it.
      bool ok = mbar_wait_bounded(&q_full, 0, abort_flag) && mbar_wait_bounded(&k_full[0], 0, abort_flag);
      for (int t = 0; t < tiles && ok; ++t) issue_s(t, 0);
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int st = j & 1;
        const bool more = j + 1 < n_tiles, fix = (fix_first && j == 0) || (fix_last && !more);
        const uint64_t vd = v_desc + (uint64_t)(st * (kTileBytes >> 4));
        ok = fix ? mbar_wait_bounded(&v_fixed[fix_first && j == 0 ? 0 : 1], 0, abort_flag)
                 : mbar_wait_bounded(&v_full[st], (j >> 1) & 1, abort_flag);
        for (int t = 0; t < tiles && ok; ++t) {
          if (!mbar_wait_bounded(&p_ready[t], j & 1, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + k * 8, vd + (uint64_t)((k * 2048) >> 4), idesc_o,
                       j > 0 || k > 0 ? 1u : 0u);
          if (t == 0) {
            // K's stage was last read by the S products that P_t(j) came from
            mma_commit(&k_empty[st]);
            if (more && !mbar_wait_bounded(&k_full[st ^ 1], ((j + 1) >> 1) & 1, abort_flag)) {
              ok = false;
              break;
            }
          }
          if (t == tiles - 1) mma_commit(&v_empty[st]);
          if (more) issue_s(t, st ^ 1);
        }
      }
      if (ok) {
        mma_commit(&o_final);
      } else {
        record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_MMA);
        *abort_flag = 1;
      }
    }
  } else {
    const int sw = warp - 2, t = sw >> 3, half = (sw >> 2) & 1, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t bar_id = 1 + t * 4 + quarter;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_off + t * 128, o_col = tmem + lane_off + 256 + t * 128 + half * 64;
    const float c = p.scale_log2;
    if (t < tiles) {
      // This row's keys: [lo, limit).
      const int32_t local = t * p.tile_rows + row / p.group;  // batch row within the unit
      const bool row_ok = row < p.tile_rows * p.group && local < rows;
      const int64_t token = row0 + local;
      int64_t limit = 0;
      if (row_ok) {
        if (kPrefix) {
          PagedRow r;
          limit = paged_row(p.paged, token, r) ? min((int64_t)hi, r.position + 1) : 0;
        } else {
          limit = min((int64_t)hi, pos0 + local + 1);
        }
      }
      bool ok = true;
      float m = -INFINITY, l = 0.0f;
      for (int j = 0; j < n_tiles; ++j) {
        // (a wait that ran out is not left early: the barriers below need every warp)
        if (ok && !mbar_wait_bounded(&s_full[t], j & 1, abort_flag)) ok = false;
        tc_fence_after();
        const int32_t key0 = (j_begin + j) * kTileKeys + half * 64;
        uint32_t a[32], b[32];
        tmem_ld_32x32b_x32(s_col + half * 64, a);
        tmem_ld_32x32b_x32(s_col + half * 64 + 32, b);
        tmem_wait_ld(a);
        tmem_regs_fence(b);
        const int from = max(0, lo - key0), to = (int)max((int64_t)0, min((int64_t)64, limit - key0));
        if (__any_sync(0xffffffffu, from > 0 || to < 64)) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            if (i < from || i >= to) a[i] = __float_as_uint(-INFINITY);
            if (i + 32 < from || i + 32 >= to) b[i] = __float_as_uint(-INFINITY);
          }
        }
        float mx = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          mx = max3(mx, __uint_as_float(a[i]), __uint_as_float(a[i + 1]));
          mx1 = max3(mx1, __uint_as_float(a[i + 2]), __uint_as_float(a[i + 3]));
          mx = max3(mx, __uint_as_float(b[i]), __uint_as_float(b[i + 1]));
          mx1 = max3(mx1, __uint_as_float(b[i + 2]), __uint_as_float(b[i + 3]));
        }
        mx = fmaxf(mx, mx1);
        x_max[t][half][row] = mx;
        named_barrier_sync(bar_id, 64);
        const float m_new = fmaxf(m, fmaxf(mx, x_max[t][half ^ 1][row]));
        bool rescale = false;
        float alpha = 1.0f;
        if (j == 0) {
          m = m_new;
        } else if ((m_new - m) * c > kLazy) {
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
          float t0, t1;
          f2_unpack(tt, t0, t1);
          const float p0 = ex2_approx(t0), p1 = ex2_approx(t1);
          sum2 = f2_add(sum2, f2_pack(p0, p1));
          packed[i] = pack_h2(p0, p1);
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
      x_sum[t][half][row] = l;
      named_barrier_sync(bar_id, 64);
      l += x_sum[t][half ^ 1][row];
      if (ok && !mbar_wait_bounded(&o_final, 0, abort_flag)) ok = false;
      tc_fence_after();
      const int64_t head = token * p.q_heads + h * p.group + row % p.group;
      const int64_t slot = split * p.rows * p.q_heads + head;
      if (row_ok && !p.direct && half == 0) part_ml[slot] = make_float2(m == -INFINITY ? m : m * c, l);
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int ch = 0; ch < 2; ++ch) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(o_col + ch * 32, r);
        tmem_wait_ld(r);
        const int col0 = half * 64 + ch * 32;
        if (!row_ok) continue;
        if (p.direct) {
          // (a row without keys: O is 0 * V, which a non-finite V of another row's keys makes NaN)
          uint16_t *o = p.out + head * p.head_dim + col0;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            if (col0 + i >= p.head_dim) break;
            uint4 v;
            v.x = pack_h2(__uint_as_float(r[i]) * inv, __uint_as_float(r[i + 1]) * inv);
            v.y = pack_h2(__uint_as_float(r[i + 2]) * inv, __uint_as_float(r[i + 3]) * inv);
            v.z = pack_h2(__uint_as_float(r[i + 4]) * inv, __uint_as_float(r[i + 5]) * inv);
            v.w = pack_h2(__uint_as_float(r[i + 6]) * inv, __uint_as_float(r[i + 7]) * inv);
            *reinterpret_cast<uint4 *>(o + i) = l == 0.0f ? make_uint4(0u, 0u, 0u, 0u) : v;
          }
        } else {
          float *o = part_o + slot * p.head_dim + col0;
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            if (col0 + i >= p.head_dim) break;
            *reinterpret_cast<float4 *>(o + i) = make_float4(__uint_as_float(r[i]), __uint_as_float(r[i + 1]),
                                                             __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
          }
        }
      }
      if (!ok) {
        if (lane == 0) record_device_error(p.err, ERR_KERNEL_PAGED_ATTENTION | ERR_SITE_EPILOGUE);
        *abort_flag = 1;
      }
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

// One warp per row and query head, four dims per lane: the partials' weights
// 2^(m - max m), then the weighted sum of their O over the weighted sum of l.
__global__ void __launch_bounds__(256) paged_combine_kernel(const __grid_constant__ PagedAttnParams p) {
  const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int64_t row = unit / p.q_heads;
  const int32_t head = (int32_t)(unit - row * p.q_heads);
  if (row >= p.rows) return;
  if (p.paged.row_offsets && row >= p.paged.row_offsets[p.paged.sequences]) return;  // padding
  if (p.paged.row_offsets && row < p.paged.row_offsets[0]) return;
  // Own partials: slots own0 + i * own_step.
  int64_t own0 = row * p.q_heads + head, own_step = p.rows * p.q_heads;
  int32_t own_n = p.own_splits;
  if (p.stream_ctas) {
    const int64_t before = p.tile_sums[row], n = p.tile_sums[row + 1] - before;
    const int64_t line = p.tile_sums[p.paged.sequences] * p.heads, ctas = min((int64_t)p.stream_ctas, line);
    const int32_t kv = head / p.group;
    own_n = 0;
    if (n > 0) {
      // CTA c has tiles [line c / C, line (c + 1) / C): tile t is c = ((t + 1) C - 1) / line's
      const int64_t t0 = before * p.heads + kv * n;
      const int64_t c0 = ((t0 + 1) * ctas - 1) / line, c1 = ((t0 + n) * ctas - 1) / line;
      if (c0 == c1 && p.prefix == 0) return;  // written by that CTA
      own_n = (int32_t)(c1 - c0 + 1);
      own0 = (row * p.heads + kv + c0) * p.group + head % p.group;
      own_step = p.group;
    }
  }
  const int64_t pre0 = row * p.q_heads + head, pre_step = p.rows * p.q_heads;
  float top = -INFINITY;
  for (int32_t i = lane; i < p.prefix_splits; i += 32) top = fmaxf(top, p.prefix_ml[pre0 + i * pre_step].x);
  for (int32_t i = lane; i < own_n; i += 32) top = fmaxf(top, p.own_ml[own0 + i * own_step].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float l = 0.0f;
  const bool mine = lane * 4 < p.head_dim;
  auto add = [&](const float *part, const float2 *ml, int64_t slot) {
    const float2 s = ml[slot];
    if (s.x == -INFINITY) return;
    const float w = ex2_approx(s.x - top);
    l += w * s.y;
    if (mine) {
      const float4 x = *reinterpret_cast<const float4 *>(part + slot * p.head_dim + lane * 4);
      o.x += w * x.x;
      o.y += w * x.y;
      o.z += w * x.z;
      o.w += w * x.w;
    }
  };
#pragma unroll 4
  for (int32_t i = 0; i < p.prefix_splits; ++i) add(p.prefix_o, p.prefix_ml, pre0 + i * pre_step);
#pragma unroll 2
  for (int32_t i = 0; i < own_n; ++i) add(p.own_o, p.own_ml, own0 + i * own_step);
  if (!mine) return;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint2 v;
  v.x = pack_h2(o.x * inv, o.y * inv);
  v.y = pack_h2(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2 *>(p.out + (row * p.q_heads + head) * p.head_dim + lane * 4) = v;
}

// ---- host ---------------------------------------------------------------------------

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Key tiles split over `splits` CTAs per unit: the smallest time of whole waves,
// counting a CTA's start and result as two tiles.
int32_t splits_for(int64_t units, int64_t key_tiles) {
  const int64_t sms = sm_count();
  int64_t best = 1, cost = -1;
  for (int64_t s = 1; s <= key_tiles && s <= 64 && (s == 1 || units * s <= 4 * sms); ++s) {
    const int64_t c = ceil_div(units * s, sms) * (ceil_div(key_tiles, s) + 2);
    if (cost < 0 || c < cost) {
      best = s;
      cost = c;
    }
  }
  return (int32_t)best;
}

// How a call is cut up, from sizes the host knows, and its workspace.
struct PagedPlan {
  bool stream;             // single rows, group <= 16: paged_stream_kernel
  bool own_direct;         // one partial per row: the tile kernel writes the result
  int32_t stream_ctas, own_splits, prefix_splits, tile_rows;
  int64_t own_units, prefix_units;
  uint64_t own_o, own_ml, prefix_o, prefix_ml, tile_sums, bytes;
};

PagedPlan paged_plan(int64_t rows, int64_t sequences, int64_t q_heads, int64_t heads, int64_t head_dim,
                     int64_t prefix_rows, bool ragged) {
  PagedPlan plan = {};
  const int64_t group = q_heads / heads;
  plan.stream = !ragged && group <= 16;
  plan.tile_rows = (int32_t)(kTileRows / group);
  const int64_t per_unit = 2 * plan.tile_rows;
  uint64_t at = 0;
  auto take = [&](uint64_t bytes) {
    const uint64_t here = at;
    at += (bytes + 255) & ~uint64_t(255);
    return here;
  };
  int64_t own_slots;
  if (plan.stream) {
    plan.stream_ctas = 2 * sm_count();
    plan.own_splits = 0;
    own_slots = (sequences * heads + plan.stream_ctas) * group;
    plan.tile_sums = take((sequences + 1) * 8);
  } else {
    plan.own_units = ragged ? rows / per_unit + sequences : sequences;
    if (plan.own_units > rows) plan.own_units = rows;
    // how many keys there are is not known here: as many CTAs as there are SMs
    const int64_t want = sm_count() / (plan.own_units * heads > 0 ? plan.own_units * heads : 1);
    plan.own_splits = (int32_t)(want < 1 ? 1 : want > 32 ? 32 : want);
    plan.own_direct = plan.own_splits == 1 && prefix_rows == 0;
    own_slots = plan.own_direct ? 0 : plan.own_splits * rows * q_heads;
  }
  plan.own_o = take(own_slots * head_dim * 4);
  plan.own_ml = take(own_slots * 8);
  if (prefix_rows > 0) {
    plan.prefix_units = ceil_div(rows, per_unit);
    plan.prefix_splits = splits_for(plan.prefix_units * heads, ceil_div(prefix_rows, kTileKeys));
    const int64_t slots = plan.prefix_splits * rows * q_heads;
    plan.prefix_o = take(slots * head_dim * 4);
    plan.prefix_ml = take(slots * 8);
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

// 4-D tile map (head_dim, d1, d2, d3) with box {64, b1, 1, b3}, 128-byte swizzle, zero fill.
ipuc_status make_map_paged(CUtensorMap *map, const void *base, int64_t head_dim, int64_t d1, int64_t d2, int64_t d3,
                           int64_t s1, int64_t s2, int64_t s3, int32_t b1, int32_t b3) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (!fn) return fail(IPUC_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[4] = {(cuuint64_t)head_dim, (cuuint64_t)d1, (cuuint64_t)d2, (cuuint64_t)d3};
  const cuuint64_t strides[3] = {(cuuint64_t)s1 * 2, (cuuint64_t)s2 * 2, (cuuint64_t)s3 * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)b1, 1, (cuuint32_t)b3}, ones[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(base), dims, strides, box, ones,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(IPUC_ERR_CUDA, "paged_attention: cuTensorMapEncodeTiled failed");
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
  IPUC_CHECK_ARG(q_stride >= q_heads * d, "paged_attention: token stride shorter than q_heads * head_dim");
  IPUC_CHECK_ALIGN(q_stride % 8 == 0 && cache->page_stride % 8 == 0 && cache->head_stride % 8 == 0 &&
                       cache->row_stride % 8 == 0,
                   "paged_attention: strides must be multiples of 8 elements");
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  IPUC_CHECK_ARG(out && q, "paged_attention: null pointer");
  IPUC_CHECK_ALIGN(aligned(out, 16) && aligned(q, 16) && aligned(cache->keys, 16) && aligned(cache->values, 16),
                   "paged_attention: pointers must be 16-byte aligned");
  IPUC_CHECK_ALIGN(aligned(prefix_pages, 4), "paged_attention: int32 arrays must be 4-byte aligned");
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
  p.scale_log2 = (scale > 0.0f ? scale : 1.0f / sqrtf((float)d)) * 1.4426950408889634f;
  p.own_o = reinterpret_cast<float *>(ws + plan.own_o);
  p.own_ml = reinterpret_cast<float2 *>(ws + plan.own_ml);
  p.prefix_o = reinterpret_cast<float *>(ws + plan.prefix_o);
  p.prefix_ml = reinterpret_cast<float2 *>(ws + plan.prefix_ml);
  p.tile_sums = reinterpret_cast<int64_t *>(ws + plan.tile_sums);
  p.stream_ctas = plan.stream_ctas;
  p.own_splits = plan.own_splits;
  p.prefix_splits = plan.prefix_splits;
  p.tile_rows = plan.tile_rows;
  p.err = device_error_word();
  const int64_t own_grid = plan.own_units * p.heads * plan.own_splits;
  const int64_t prefix_grid = plan.prefix_units * p.heads * plan.prefix_splits, heads_all = p.rows * q_heads;
  IPUC_CHECK_ARG(own_grid < (1ll << 31) && prefix_grid < (1ll << 31) && heads_all < (1ll << 31),
                 "paged_attention: extent too large");
  CUtensorMap tm_q, tm_k, tm_v;
  st = make_map_paged(&tm_k, cache->keys, d, cache->page_size, cache->heads, cache->pages, cache->row_stride,
                      cache->head_stride, cache->page_stride, p.chunk, 1);
  if (st != IPUC_OK) return st;
  st = make_map_paged(&tm_v, cache->values, d, cache->page_size, cache->heads, cache->pages, cache->row_stride,
                      cache->head_stride, cache->page_stride, p.chunk, 1);
  if (st != IPUC_OK) return st;
  if (!plan.stream || prefix_rows > 0) {
    st = make_map_paged(&tm_q, q, d, p.group, cache->heads, p.rows, d, p.group * d, q_stride, p.group, p.tile_rows);
    if (st != IPUC_OK) return st;
  }
  if (plan.stream) {
    auto launch = [&](auto kernel, int bytes) -> ipuc_status {
      IPUC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      kernel<<<plan.stream_ctas, kStreamThreads, bytes, stream>>>(tm_k, tm_v, p);
      return check_launch("paged_stream_kernel");
    };
    st = d > 64 ? launch(paged_stream_kernel<128>, stream_smem_bytes<128>())
                : launch(paged_stream_kernel<64>, stream_smem_bytes<64>());
    if (st != IPUC_OK) return st;
  }
  auto tiles = [&](auto kernel, int64_t grid, int32_t units, bool direct) -> ipuc_status {
    IPUC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTileSmem));
    p.row_units = units;
    p.direct = direct;
    kernel<<<(unsigned)grid, kTileThreads, kTileSmem, stream>>>(tm_q, tm_k, tm_v, p);
    return check_launch("paged_tile_kernel");
  };
  if (!plan.stream) {
    st = tiles(paged_tile_kernel<false>, own_grid, (int32_t)plan.own_units, plan.own_direct);
    if (st != IPUC_OK || plan.own_direct) return st;
  }
  if (prefix_rows > 0) {
    st = tiles(paged_tile_kernel<true>, prefix_grid, (int32_t)plan.prefix_units, false);
    if (st != IPUC_OK) return st;
  }
  paged_combine_kernel<<<(unsigned)((heads_all + 7) / 8), 256, 0, stream>>>(p);
  return check_launch("paged_combine_kernel");
}
