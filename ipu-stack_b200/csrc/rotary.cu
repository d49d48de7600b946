// Rotary positions and what is fused with them: the table of cosines and
// sines, the rotation of a projection's heads, the per-head norm of queries
// and keys with the rotation in the same pass, and the append of keys and
// values to a paged cache with the rotation applied on the way.
//
// Pair i of a head's first `rotary_dim` elements turns by the angle
// theta(p, i) = p * f_i at position p: (a, b) -> (a c - b s, b c + a s).  The
// pairs are (x_i, x_{i+R/2}) (half) or (x_2i, x_2i+1) (interleaved); elements
// from rotary_dim on pass unturned.  All arithmetic is f32 with one rounding
// to f16 at the store.
#include <math.h>

#include "common.cuh"
#include "paged.cuh"

namespace ipuc {
namespace {

// ---- the table ----------------------------------------------------------------

constexpr int kMaxPairs = 128;

struct TableParams {
  float *table;
  int64_t positions;
  int32_t pairs;
  float magnitude, magnitude_rest;  // in two parts: 1.1 alone is off by 2^-25 of it in f32
  uint64_t turns[kMaxPairs];  // f_i / 2pi, turns per position, in units of 2^-64
};

// Angles of far positions need more than 32 bits (131072 * f leaves 7 bits of
// a fraction in f32).  An angle is a fraction of a turn in 64-bit fixed point, so
// position times frequency drops the whole turns by itself; the nearest whole
// quarter is its rounded top two bits, and what is left, t in [-1/2, 1/2) of a
// quarter, comes in steps of 2^-32 and goes to f32, which rounds it by 2^-26 at
// most.  Sine and cosine of pi/2 t
// are their Taylor polynomials to t^9 and t^10 (the next terms are below 2e-9);
// pi/2 in two parts keeps the sine to half a step and the rounding of t.  The
// whole quarters swap and negate the two.  A thread writes V neighbouring pairs.
// Bound by the stores: 131072 x 128 takes 13.4 us (5.0 TB/s), torch's fill of it
// 17.9, a bare loop of 16-byte stores 12.6.  Products and the remainder in f64
// with CUDA's sincospif took 17.7: bound by the instructions.
__device__ __forceinline__ void sincos_quarter(float t, float &s, float &c) {
  constexpr double h = 1.57079632679489661923;  // pi / 2
  constexpr float h0 = (float)h, h1 = (float)(h - (double)h0);
  constexpr float s3 = (float)(-h * h * h / 6), s5 = (float)(h * h * h * h * h / 120);
  constexpr float s7 = (float)(-h * h * h * h * h * h * h / 5040);
  constexpr float s9 = (float)(h * h * h * h * h * h * h * h * h / 362880);
  constexpr float c2 = (float)(-h * h / 2), c4 = (float)(h * h * h * h / 24);
  constexpr float c6 = (float)(-h * h * h * h * h * h / 720), c8 = (float)(h * h * h * h * h * h * h * h / 40320);
  constexpr float c10 = (float)(-h * h * h * h * h * h * h * h * h * h / 3628800);
  const float t2 = t * t;
  const float p = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, s9, s7), s5), s3), h1);
  s = fmaf(t, h0, t * p);
  c = fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, fmaf(t2, c10, c8), c6), c4), c2), 1.0f);
}

template <int V>
__global__ void __launch_bounds__(256) rotary_table_kernel(const __grid_constant__ TableParams p) {
  const int groups = p.pairs / V, rows = 256 / groups;  // positions per block and step
  const int i = (threadIdx.x % groups) * V;
  if ((int)threadIdx.x >= rows * groups) return;
  uint64_t f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = p.turns[i + j];
  for (int64_t pos = (int64_t)blockIdx.x * rows + threadIdx.x / groups; pos < p.positions;
       pos += (int64_t)gridDim.x * rows) {
    float cs[V], sn[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const uint64_t angle = (uint64_t)pos * f[j];
      float s, c;
      sincos_quarter((float)(int32_t)(uint32_t)(angle >> 30) * 0x1p-32f, s, c);
      const uint32_t q = ((uint32_t)(angle >> 61) + 1) >> 1;  // (the carry out of two bits is a whole turn)
      // cosine, sine of the quarters: (c, s), (-s, c), (-c, -s), (s, -c)
      const float a = __uint_as_float(__float_as_uint(q & 1 ? s : c) ^ ((q + 1) & 2) << 30);
      const float b = __uint_as_float(__float_as_uint(q & 1 ? c : s) ^ (q & 2) << 30);
      cs[j] = fmaf(a, p.magnitude, a * p.magnitude_rest);
      sn[j] = fmaf(b, p.magnitude, b * p.magnitude_rest);
    }
    float *row = p.table + pos * 2 * p.pairs + i;
    if constexpr (V == 4) {
      *reinterpret_cast<float4 *>(row) = make_float4(cs[0], cs[1], cs[2], cs[3]);
      *reinterpret_cast<float4 *>(row + p.pairs) = make_float4(sn[0], sn[1], sn[2], sn[3]);
    } else {
      row[0] = cs[0];
      row[p.pairs] = sn[0];
    }
  }
}

// ---- heads: rotate, norm, append -------------------------------------------------

// One of the (at most two) tensors of a call: [tokens][heads][head_dim].
struct Segment {
  const void *in;
  uint16_t *out;          // dense output, or a paged cache's base
  const uint16_t *weight; // norm: [head_dim] or null (ones)
  int64_t in_stride, out_stride;  // elements from token to token (paged: unused)
  int32_t heads;
  int32_t rotate;
};

struct HeadsParams {
  Segment seg[2];
  const float *table;       // [table_rows][rotary_dim]: cosines, then sines; null: no rotation
  const int32_t *positions; // null: the token's index (paged: its position in the cache)
  PagedView paged;
  int64_t table_rows;
  int64_t tokens;
  int32_t head_dim, rotary_dim;
  int32_t interleaved;
  int32_t lane_shift;  // log2 of the lanes that share a head
  int32_t heads;       // of both tensors
  float inv_dim;       // 1 / head_dim
  float eps;
  uint32_t *err;
};

template <typename T, int V>
struct alignas(V * sizeof(T) < 16 ? V * sizeof(T) : 16) Vec {
  T v[V];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return h2f(x); }

template <int V>
__device__ __forceinline__ Vec<uint16_t, V> to_f16(const float *y) {
  Vec<uint16_t, V> o;
  if constexpr (V == 1) {
    o.v[0] = f2h(y[0]);
  } else {
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const __half2 h = __floats2half2_rn(y[j], y[j + 1]);
      o.v[j] = __half_as_ushort(__low2half(h));
      o.v[j + 1] = __half_as_ushort(__high2half(h));
    }
  }
  return o;
}

// Rows are read and written once: streaming hints on both sides keep them from
// pushing the table out of L2 (8192 x 32 x 128: 31.8 -> 27.5 us).
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
  if constexpr (sizeof(T) * V % 16 == 0) {
    Vec<T, V> o;
    uint4 *q = reinterpret_cast<uint4 *>(&o);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * V / 16); ++i) q[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    return o;
  } else {
    return *reinterpret_cast<const Vec<T, V> *>(p);
  }
}
template <int V>
__device__ __forceinline__ void store(uint16_t *p, const Vec<uint16_t, V> &v) {
  if constexpr (V == 8) __stcs(reinterpret_cast<uint4 *>(p), *reinterpret_cast<const uint4 *>(&v));
  else *reinterpret_cast<Vec<uint16_t, V> *>(p) = v;
}

// An item is two vectors of V elements that one lane holds: the two sides of V
// pairs, or 2V neighbouring elements.  A head's head_dim / 2V items are spread
// over 2^lane_shift neighbouring lanes (a group), IPL to a lane, so the norm's
// sum is a shuffle tree.
//
// HBM-bound: x is read and written once, and the rows' loads are issued before
// the chain position -> table row, which they do not depend on.  8192 x 32 x 128
// takes 24.9 us (5.6 TB/s; torch's copy of the same bytes 22.4), the norm of
// 8191 x 40 x 128 in f32 with the rotation 42.5 (6.0 TB/s).  One head per group:
// two or four heads that share the lookups and the table row measured the same
// and slower on 32 tokens (2.6 and 3.4 against 2.2 us); resident blocks that
// loop with the next group's loads in flight 35.8 us; fewer registers for more
// resident warps (42 of 47) 31 us; 8-byte loads 30.8 us.  Small blocks, which
// end and begin one by one: 25.6 and 45.9 us with 256 threads, 43.2 with 64.
// In a cache a group takes a key head and its value head: the chain there is
// longer (row -> sequence -> length -> page), and 8000 x 8 x 128 of each, 16
// sequences, take 14.8 us (4.7 TB/s) for 18.1 with a group for each.
constexpr int kHeadsThreads = 128;
template <int V, typename TIN, bool kNorm, bool kPaged>
__global__ void __launch_bounds__(kHeadsThreads) heads_kernel(const __grid_constant__ HeadsParams p) {
  constexpr int IPL = V >= 4 ? 1 : V == 2 ? 2 : 4;  // head_dim <= 256
  const uint32_t lanes = 1u << p.lane_shift;
  const uint32_t lane = threadIdx.x & (lanes - 1);
  const uint32_t group = blockIdx.x * ((uint32_t)kHeadsThreads >> p.lane_shift) + (threadIdx.x >> p.lane_shift);
  const uint32_t token = group / (uint32_t)p.heads, head = group - token * (uint32_t)p.heads;
  const bool inside = token < p.tokens;
  const int items = p.head_dim / (2 * V), turned = p.rotary_dim / (2 * V);
  // Dense: heads of the first tensor, then of the second.  Cache: a key head and
  // its value head, which share the lookups.
  constexpr int S = kPaged ? 2 : 1;
  const bool second = !kPaged && head >= (uint32_t)p.seg[0].heads;
  const int at = second ? (int)head - p.seg[0].heads : (int)head;
  int e0[IPL], e1[IPL];
#pragma unroll
  for (int k = 0; k < IPL; ++k) {
    const int item = (int)(lane + k * lanes);
    const bool split = item < turned && !p.interleaved;
    e0[k] = split ? item * V : 2 * V * item;
    e1[k] = split ? p.rotary_dim / 2 + item * V : e0[k] + V;
  }
  Vec<TIN, V> x[S][IPL][2];
#pragma unroll
  for (int t = 0; t < S; ++t) {
    const Segment &g = p.seg[kPaged ? t : second ? 1 : 0];
    const TIN *in = static_cast<const TIN *>(g.in) + token * g.in_stride + at * p.head_dim;
#pragma unroll
    for (int k = 0; k < IPL; ++k) {
      if (inside && (int)(lane + k * lanes) < items) {
        x[t][k][0] = load<TIN, V>(in + e0[k]);
        x[t][k][1] = load<TIN, V>(in + e1[k]);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[t][k][0].v[j] = x[t][k][1].v[j] = TIN(0);
      }
    }
  }
  // The token's position (-1: nothing is written) and, in a cache, its slot.
  int32_t position = 0;
  int64_t page_at = 0;
  if (!inside) {
    position = -1;
  } else if constexpr (kPaged) {
    PagedRow r;
    if (!paged_row(p.paged, token, r) || r.position < 0) {
      position = -1;
    } else if (r.position >= (int64_t)p.paged.max_pages * p.paged.page_size) {
      position = -1;
      record_device_error(p.err, ERR_KERNEL_HEADS | ERR_SITE_LENGTH);
    } else {
      position = (int32_t)r.position;
      const int32_t page = position / p.paged.page_size;
      const int32_t id = p.paged.page_table[r.sequence * p.paged.table_stride + page];
      page_at = id * p.paged.page_stride + (int64_t)(position - page * p.paged.page_size) * p.paged.row_stride;
      if (id < 0 || id >= p.paged.pages) {
        position = -1;
        record_device_error(p.err, ERR_KERNEL_HEADS | ERR_SITE_PAGE);
      }
    }
  } else {
    position = p.positions ? p.positions[token] : (int32_t)token;
  }
  if (p.table && position >= p.table_rows) {
    position = -1;
    record_device_error(p.err, ERR_KERNEL_HEADS | ERR_SITE_POSITION);
  }
  Vec<float, V> cs[IPL], sn[IPL];
#pragma unroll
  for (int k = 0; k < IPL; ++k) {
    const int item = (int)(lane + k * lanes);
    if (p.table && item < turned && position >= 0) {
      const float *row = p.table + (int64_t)position * p.rotary_dim + item * V;
      cs[k] = *reinterpret_cast<const Vec<float, V> *>(row);
      sn[k] = *reinterpret_cast<const Vec<float, V> *>(row + p.rotary_dim / 2);
    }
  }
  float rstd = 1.0f;
  if constexpr (kNorm) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < IPL; ++k)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = to_f32(x[0][k][0].v[j]), b = to_f32(x[0][k][1].v[j]);
        sum = fmaf(a, a, fmaf(b, b, sum));
      }
    for (uint32_t m = lanes >> 1; m; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    rstd = rsqrtf(sum * p.inv_dim + p.eps);
  }
  if (position < 0) return;
#pragma unroll
  for (int t = 0; t < S; ++t) {
    const Segment &g = p.seg[kPaged ? t : second ? 1 : 0];
    uint16_t *out = g.out + (kPaged ? page_at + at * p.paged.head_stride : token * g.out_stride + at * p.head_dim);
#pragma unroll
    for (int k = 0; k < IPL; ++k) {
      const int item = (int)(lane + k * lanes);
      if (item >= items) continue;
      float y[2 * V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y[j] = to_f32(x[t][k][0].v[j]);
        y[V + j] = to_f32(x[t][k][1].v[j]);
      }
      if constexpr (kNorm) {
        if (g.weight) {
          const Vec<uint16_t, V> w0 = *reinterpret_cast<const Vec<uint16_t, V> *>(g.weight + e0[k]);
          const Vec<uint16_t, V> w1 = *reinterpret_cast<const Vec<uint16_t, V> *>(g.weight + e1[k]);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            y[j] *= rstd * h2f(w0.v[j]);
            y[V + j] *= rstd * h2f(w1.v[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 2 * V; ++j) y[j] *= rstd;
        }
      }
      if (p.table && g.rotate && item < turned) {
        // (two loops: indices known at compile time keep y in registers)
        if (p.interleaved) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = y[2 * j], b = y[2 * j + 1];
            y[2 * j] = a * cs[k].v[j] - b * sn[k].v[j];
            y[2 * j + 1] = b * cs[k].v[j] + a * sn[k].v[j];
          }
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = y[j], b = y[V + j];
            y[j] = a * cs[k].v[j] - b * sn[k].v[j];
            y[V + j] = b * cs[k].v[j] + a * sn[k].v[j];
          }
        }
      }
      store(out + e0[k], to_f16<V>(y));
      store(out + e1[k], to_f16<V>(y + V));
    }
  }
}

// Largest vector width that every address of the call allows: 2V divides the
// turned part and the head, and pointers and strides are multiples of V.
int vector_width(const HeadsParams &p, size_t in_bytes, bool paged) {
  for (int v = 8; v > 1; v /= 2) {
    bool ok = p.head_dim % (2 * v) == 0 && p.rotary_dim % (2 * v) == 0;
    for (const Segment &g : p.seg) {
      if (!g.heads) continue;
      const uintptr_t in_align = v * in_bytes < 16 ? v * in_bytes : 16;
      ok = ok && aligned(g.in, in_align) && aligned(g.out, v * 2) && g.in_stride % v == 0;
      if (g.weight) ok = ok && aligned(g.weight, v * 2);
      if (!paged) ok = ok && g.out_stride % v == 0;
    }
    if (paged)
      ok = ok && p.paged.page_stride % v == 0 && p.paged.head_stride % v == 0 && p.paged.row_stride % v == 0;
    if (p.table) ok = ok && aligned(p.table, 16);
    if (ok) return v;
  }
  return 1;
}

template <typename TIN, bool kNorm, bool kPaged>
ipuc_status launch_heads(HeadsParams &p, cudaStream_t stream) {
  const int v = vector_width(p, sizeof(TIN), kPaged);
  const int items = p.head_dim / (2 * v);
  p.lane_shift = 0;
  while ((1 << p.lane_shift) < items && p.lane_shift < 5) ++p.lane_shift;
  p.heads = p.seg[0].heads + (kPaged ? 0 : p.seg[1].heads);
  p.inv_dim = 1.0f / (float)p.head_dim;
  const int64_t groups = p.tokens * p.heads, per_block = kHeadsThreads >> p.lane_shift;
  IPUC_CHECK_ARG(groups < (1ll << 31), "heads: extent too large");
  const unsigned grid = (unsigned)((groups + per_block - 1) / per_block);
  switch (v) {
    case 8: heads_kernel<8, TIN, kNorm, kPaged><<<grid, kHeadsThreads, 0, stream>>>(p); break;
    case 4: heads_kernel<4, TIN, kNorm, kPaged><<<grid, kHeadsThreads, 0, stream>>>(p); break;
    case 2: heads_kernel<2, TIN, kNorm, kPaged><<<grid, kHeadsThreads, 0, stream>>>(p); break;
    default: heads_kernel<1, TIN, kNorm, kPaged><<<grid, kHeadsThreads, 0, stream>>>(p); break;
  }
  return check_launch("heads_kernel");
}

ipuc_status check_rotary(const char *who, const ipuc_rotary *r, int64_t head_dim, HeadsParams &p) {
  p.table = nullptr;
  p.table_rows = 0;
  p.rotary_dim = 0;
  p.interleaved = 0;
  if (!r || r->rotary_dim == 0) return IPUC_OK;
  const std::string w = who;
  IPUC_CHECK_ARG(r->rotary_dim > 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= head_dim,
                 w + ": rotary_dim must be even and within the head");
  IPUC_CHECK_ARG(r->layout == IPUC_ROTARY_HALF || r->layout == IPUC_ROTARY_INTERLEAVED, w + ": bad rotary layout");
  IPUC_CHECK_ARG(r->table != nullptr && r->positions > 0, w + ": rotary table missing");
  IPUC_CHECK_ALIGN(aligned(r->table, 4), w + ": rotary table must be 4-byte aligned");
  p.table = r->table;
  p.table_rows = r->positions;
  p.rotary_dim = r->rotary_dim;
  p.interleaved = r->layout == IPUC_ROTARY_INTERLEAVED;
  return IPUC_OK;
}

// One dense tensor [tokens][heads][head_dim] of a call; rows may lie further
// apart than heads * head_dim (a projection's slice).
ipuc_status check_segment(const char *who, Segment &g, void *out, int64_t out_stride, const void *in,
                          int64_t in_stride, ipuc_precision precision, int64_t heads, int64_t head_dim, bool dense) {
  const std::string w = who;
  IPUC_CHECK_ARG(out && in, w + ": null pointer");
  IPUC_CHECK_ALIGN(aligned(in, precision == IPUC_F32 ? 4 : 2) && aligned(out, 2),
                   w + ": pointers must be element-aligned");
  IPUC_CHECK_ARG(in_stride >= heads * head_dim && (!dense || out_stride >= heads * head_dim),
                 w + ": token stride shorter than heads * head_dim");
  IPUC_CHECK_ARG(in != out || (precision == IPUC_F16 && in_stride == out_stride),
                 w + ": in place needs f16 input and equal strides");
  g.in = in;
  g.out = static_cast<uint16_t *>(out);
  g.in_stride = in_stride;
  g.out_stride = out_stride;
  g.heads = (int32_t)heads;
  g.rotate = 1;
  g.weight = nullptr;
  return IPUC_OK;
}

ipuc_status check_heads(const char *who, int64_t tokens, int64_t heads, int64_t head_dim, ipuc_precision precision) {
  const std::string w = who;
  IPUC_CHECK_ARG(precision == IPUC_F16 || precision == IPUC_F32, w + ": bad input precision");
  IPUC_CHECK_ARG(tokens >= 0 && heads >= 0 && tokens < (1ll << 31) && heads < (1ll << 16),
                 w + ": extent out of range");
  IPUC_CHECK_ARG(head_dim > 0 && head_dim % 2 == 0, w + ": head_dim must be even and positive");
  if (head_dim > 256) return fail(IPUC_ERR_UNSUPPORTED, w + ": head_dim above 256 is not supported");
  return IPUC_OK;
}

}  // namespace
}  // namespace ipuc

using namespace ipuc;

extern "C" ipuc_status ipuc_rotary_table(float *table, int64_t positions, int64_t rotary_dim,
                                         const ipuc_rotary_scaling *scaling, ipuc_stream stream) {
  IPUC_CHECK_ARG(scaling != nullptr, "rotary_table: null scaling");
  IPUC_CHECK_ARG(positions >= 0 && positions < (1ll << 31), "rotary_table: positions out of range");
  IPUC_CHECK_ARG(rotary_dim > 0 && rotary_dim % 2 == 0, "rotary_table: rotary_dim must be even and positive");
  if (rotary_dim > 2 * kMaxPairs) return fail(IPUC_ERR_UNSUPPORTED, "rotary_table: rotary_dim above 256 is not supported");
  const ipuc_rotary_scaling &c = *scaling;
  IPUC_CHECK_ARG(c.kind >= IPUC_ROTARY_SCALE_NONE && c.kind <= IPUC_ROTARY_SCALE_BANDS, "rotary_table: bad scaling kind");
  IPUC_CHECK_ARG(isfinite(c.base) && c.base > 1.0, "rotary_table: base must be above 1");
  IPUC_CHECK_ARG(isfinite(c.magnitude) && c.magnitude > 0.0, "rotary_table: magnitude must be positive");
  if (c.kind != IPUC_ROTARY_SCALE_NONE)
    IPUC_CHECK_ARG(isfinite(c.factor) && c.factor >= 1.0, "rotary_table: factor must be at least 1");
  if (c.kind == IPUC_ROTARY_SCALE_BASE)
    IPUC_CHECK_ARG(rotary_dim > 2, "rotary_table: base scaling needs rotary_dim above 2");
  if (c.kind == IPUC_ROTARY_SCALE_BANDS)
    IPUC_CHECK_ARG(isfinite(c.low) && isfinite(c.high) && c.low < c.high && isfinite(c.original) && c.original > 0.0,
                   "rotary_table: bands need low < high and a positive original length");
  if (positions == 0) return IPUC_OK;
  IPUC_CHECK_ARG(table != nullptr, "rotary_table: null pointer");
  IPUC_CHECK_ALIGN(aligned(table, 4), "rotary_table: table must be 4-byte aligned");
  TableParams p;
  p.table = table;
  p.positions = positions;
  p.pairs = (int32_t)(rotary_dim / 2);
  p.magnitude = (float)c.magnitude;
  p.magnitude_rest = (float)(c.magnitude - (double)p.magnitude);
  const double pi = 3.14159265358979323846, r = (double)rotary_dim;
  const double base = c.kind == IPUC_ROTARY_SCALE_BASE ? c.base * pow(c.factor, r / (r - 2.0)) : c.base;
  for (int i = 0; i < p.pairs; ++i) {
    double f = pow(base, -2.0 * i / r);
    if (c.kind == IPUC_ROTARY_SCALE_LINEAR) f /= c.factor;
    if (c.kind == IPUC_ROTARY_SCALE_BANDS) {
      const double turns = c.original * f / (2.0 * pi);
      const double keep = fmin(1.0, fmax(0.0, (turns - c.low) / (c.high - c.low)));
      f *= keep + (1.0 - keep) / c.factor;
    }
    p.turns[i] = (uint64_t)(f / (2.0 * pi) * 0x1p64);  // (f is at most 1)
  }
  const bool wide = p.pairs % 4 == 0 && aligned(table, 16);
  const int64_t rows = 256 / (wide ? p.pairs / 4 : p.pairs), want = (positions + rows - 1) / rows, cap = (int64_t)sm_count() * 8;
  const unsigned grid = (unsigned)(want < cap ? want : cap);
  if (wide) rotary_table_kernel<4><<<grid, 256, 0, stream>>>(p);
  else rotary_table_kernel<1><<<grid, 256, 0, stream>>>(p);
  return check_launch("rotary_table_kernel");
}

extern "C" ipuc_status ipuc_rotary_f16(void *out, int64_t out_stride, const void *in, int64_t in_stride,
                                       ipuc_precision in_precision, int64_t tokens, int64_t heads, int64_t head_dim,
                                       const ipuc_rotary *rotary, const int32_t *positions, ipuc_stream stream) {
  ipuc_status st = check_heads("rotary", tokens, heads, head_dim, in_precision);
  if (st != IPUC_OK) return st;
  HeadsParams p = {};
  if ((st = check_rotary("rotary", rotary, head_dim, p)) != IPUC_OK) return st;
  IPUC_CHECK_ARG(p.table != nullptr, "rotary: rotary table missing");
  if (tokens == 0 || heads == 0) return IPUC_OK;
  st = check_segment("rotary", p.seg[0], out, out_stride, in, in_stride, in_precision, heads, head_dim, true);
  if (st != IPUC_OK) return st;
  p.positions = positions;
  p.tokens = tokens;
  p.head_dim = (int32_t)head_dim;
  p.err = device_error_word();
  return in_precision == IPUC_F16 ? launch_heads<uint16_t, false, false>(p, stream)
                                  : launch_heads<float, false, false>(p, stream);
}

extern "C" ipuc_status ipuc_qk_norm_rotary_f16(void *q_out, int64_t q_out_stride, void *k_out, int64_t k_out_stride,
                                               const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                                               ipuc_precision in_precision, const void *q_weight,
                                               const void *k_weight, float eps, int64_t tokens, int64_t q_heads,
                                               int64_t k_heads, int64_t head_dim, const ipuc_rotary *rotary,
                                               const int32_t *positions, ipuc_stream stream) {
  ipuc_status st = check_heads("qk_norm_rotary", tokens, q_heads, head_dim, in_precision);
  if (st == IPUC_OK) st = check_heads("qk_norm_rotary", tokens, k_heads, head_dim, in_precision);
  if (st != IPUC_OK) return st;
  IPUC_CHECK_ARG(isfinite(eps) && eps >= 0.0f, "qk_norm_rotary: eps must be finite and not negative");
  HeadsParams p = {};
  if ((st = check_rotary("qk_norm_rotary", rotary, head_dim, p)) != IPUC_OK) return st;
  if (tokens == 0 || q_heads + k_heads == 0) return IPUC_OK;
  if (q_heads) {
    st = check_segment("qk_norm_rotary", p.seg[0], q_out, q_out_stride, q, q_stride, in_precision, q_heads, head_dim, true);
    if (st != IPUC_OK) return st;
  }
  if (k_heads) {
    st = check_segment("qk_norm_rotary", p.seg[1], k_out, k_out_stride, k, k_stride, in_precision, k_heads, head_dim, true);
    if (st != IPUC_OK) return st;
  }
  IPUC_CHECK_ALIGN(aligned(q_weight, 2) && aligned(k_weight, 2), "qk_norm_rotary: pointers must be element-aligned");
  p.seg[0].weight = static_cast<const uint16_t *>(q_weight);
  p.seg[1].weight = static_cast<const uint16_t *>(k_weight);
  p.positions = positions;
  p.tokens = tokens;
  p.head_dim = (int32_t)head_dim;
  p.eps = eps;
  p.err = device_error_word();
  return in_precision == IPUC_F16 ? launch_heads<uint16_t, true, false>(p, stream)
                                  : launch_heads<float, true, false>(p, stream);
}

extern "C" ipuc_status ipuc_paged_append_f16(const ipuc_paged_cache *cache, const ipuc_paged_batch *batch,
                                             const void *k, int64_t k_stride, const void *v, int64_t v_stride,
                                             ipuc_precision in_precision, const ipuc_rotary *rotary,
                                             ipuc_stream stream) {
  ipuc_status st = check_paged("paged_append", cache, batch);
  if (st != IPUC_OK) return st;
  st = check_heads("paged_append", batch->rows, cache->heads, cache->head_dim, in_precision);
  if (st != IPUC_OK) return st;
  HeadsParams p = {};
  if ((st = check_rotary("paged_append", rotary, cache->head_dim, p)) != IPUC_OK) return st;
  if (batch->rows == 0 || batch->sequences == 0) return IPUC_OK;
  st = check_segment("paged_append", p.seg[0], cache->keys, 0, k, k_stride, in_precision, cache->heads,
                     cache->head_dim, false);
  if (st == IPUC_OK)
    st = check_segment("paged_append", p.seg[1], cache->values, 0, v, v_stride, in_precision, cache->heads,
                       cache->head_dim, false);
  if (st != IPUC_OK) return st;
  p.seg[1].rotate = 0;
  p.paged = paged_view(cache, batch);
  p.tokens = batch->rows;
  p.head_dim = cache->head_dim;
  p.err = device_error_word();
  return in_precision == IPUC_F16 ? launch_heads<uint16_t, false, true>(p, stream)
                                  : launch_heads<float, false, true>(p, stream);
}
