// paged_attention.hip — attention of a step's new rows over their requests' pages of a key-value cache, split over the
// cache's length and joined.
//
// Row i of the n rows of request b stands at position p = len[b] - n + i and sees the keys j <= p, with a window those
// with j > p - window or j < sinks:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q k_j).
// One pass over the keys keeps, per query, a reference m close to the largest score so far, l = sum w_j e^-m and the sum
// of w_j e^-m v_j; parts of the keys join by rescaling each to the largest m.
#include "device_common.h"
#include "kernels.h"

#include <algorithm>

namespace mh {
namespace {

constexpr int kTileKeys = 32;  // keys a wave takes at once
constexpr int kWaves = 4;
// Scores (in octaves) may pass the reference by so much before the sums are rescaled: weights up to 2^8.
constexpr float kSlack = 8.0f;

typedef short s8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));
typedef int v2i __attribute__((ext_vector_type(2)));

// What a request's rows see, in tiles of kTileKeys keys: those of the sinks, then those from the window's first key on.
struct Span {
  int first_pos, last_pos;  // of the rows of one query tile
  int sink_tiles, low_tile, tiles;
  __device__ int tile(int i) const { return i < sink_tiles ? i : i - sink_tiles + low_tile; }
};
__device__ __forceinline__ Span span_of(int first_pos, int last_pos, int window, int sinks) {
  Span s;
  s.first_pos = first_pos;
  s.last_pos = last_pos;
  const int low = window > 0 ? max(0, first_pos - window + 1) : 0;
  s.low_tile = low / kTileKeys;
  s.sink_tiles = min((min(sinks, low) + kTileKeys - 1) / kTileKeys, s.low_tile);
  s.tiles = last_pos < 0 ? 0 : s.sink_tiles + last_pos / kTileKeys + 1 - s.low_tile;
  return s;
}

// A request's rows, checked: n = 0 if there are none or they cannot be taken.
struct Request {
  int row0, n, len;
};
__device__ __forceinline__ Request request_of(const PagedAttnArgs& g, int b, bool report) {
  const int row0 = g.cu[b], end = g.cu[b + 1], len = g.length[b];
  const int64_t n = (int64_t)end - row0;
  const bool ok = row0 >= 0 && n >= 0 && end <= g.rows && n <= g.max_rows && len >= 0 && len <= g.max_keys &&
                  len <= (int64_t)g.max_blocks << g.page_shift;
  if (!ok && report && g.err) *g.err = 1;
  return {row0, ok ? (int)n : 0, len};
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// fp32 as the sum of three bf16 parts, each a truncation of what the ones before leave: exact but for parts below
// fp32's normal numbers.  Pairs of values as the packed words of the matrix operands.
__device__ __forceinline__ void split3(float a, float b, int& hi, int& mid, int& lo) {
  const uint32_t ah = __float_as_uint(a) & 0xFFFF0000u, bh = __float_as_uint(b) & 0xFFFF0000u;
  const float ar = a - __uint_as_float(ah), br = b - __uint_as_float(bh);
  const uint32_t am = __float_as_uint(ar) & 0xFFFF0000u, bm = __float_as_uint(br) & 0xFFFF0000u;
  const float al = ar - __uint_as_float(am), bl = br - __uint_as_float(bm);
  hi = (int)__builtin_amdgcn_perm(bh, ah, 0x07060302u);
  mid = (int)__builtin_amdgcn_perm(bm, am, 0x07060302u);
  lo = (int)__builtin_amdgcn_perm(__float_as_uint(bl), __float_as_uint(al), 0x07060302u);
}

__device__ __forceinline__ f4v mfma32(v4i a, v4i b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8v, a), __builtin_bit_cast(b8v, b), c, 0, 0, 0);
}
__device__ __forceinline__ f4v mfma16(v2i a, v2i b, f4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4v, a), __builtin_bit_cast(s4v, b), c, 0, 0, 0);
}

// The operands of one tile, in the order of the matrix instructions' lanes.  A wave's lane is (m, g) = (lane % 16,
// lane / 16).  S^T = K Q^T comes in two products of 16 keys, row 4a + i of product t being key 8a + 4t + i of the
// tile: then lane (m, g) holds the weights of query m for keys 8g .. 8g + 7, which is what O^T = V^T W^T wants of its
// right operand, and its left operand is eight neighbouring keys of one dimension, 16 bytes of the value cache.
template <int D, bool CB16>
struct Tile;

template <int D>
struct Tile<D, true> {
  static constexpr int KS = D / 32, DT = D / 16;
  static constexpr bool HALF = D % 32 != 0;  // 16 dimensions more
  v4i k[2][KS];
  v2i kh[2];
  v4i v[DT];
  __device__ __forceinline__ void load_k(const char* kc, int64_t at, int g) {  // at: element of the row's first dimension
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* p = kc + 2 * (at + t * 4 * D);
#pragma unroll
      for (int s = 0; s < KS; ++s) k[t][s] = *(const v4i*)(p + 64 * s + 16 * g);
      if constexpr (HALF) kh[t] = *(const v2i*)(p + 64 * KS + 8 * g);
    }
  }
  __device__ __forceinline__ void load_v(const char* vc, int64_t at, int page_shift) {  // at: element of (dimension m, key 8g)
#pragma unroll
    for (int d = 0; d < DT; ++d) v[d] = *(const v4i*)(vc + 2 * (at + ((int64_t)(16 * d) << page_shift)));
  }
  // Keys of this lane's eight that `keep` does not name count as zero.
  __device__ __forceinline__ void keep_v(uint32_t keep) {
    v4i mask;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      mask[i] = ((keep >> (2 * i)) & 1 ? 0x0000FFFF : 0) | ((keep >> (2 * i + 1)) & 1 ? (int)0xFFFF0000 : 0);
#pragma unroll
    for (int d = 0; d < DT; ++d) v[d] &= mask;
  }
};

template <int D>
struct Tile<D, false> {
  static constexpr int DT = D / 16;
  f4v k[2][DT];
  f4v v[2][DT];
  __device__ __forceinline__ void load_k(const char* kc, int64_t at, int g) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < DT; ++c) k[t][c] = *(const f4v*)(kc + 4 * (at + t * 4 * D + 16 * c + 4 * g));
  }
  __device__ __forceinline__ void load_v(const char* vc, int64_t at, int page_shift) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int t = 0; t < 2; ++t) v[t][d] = *(const f4v*)(vc + 4 * (at + ((int64_t)(16 * d) << page_shift) + 4 * t));
  }
  __device__ __forceinline__ void keep_v(uint32_t keep) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int d = 0; d < DT; ++d) v[t][d][i] = (keep >> (4 * t + i)) & 1 ? v[t][d][i] : 0.0f;
  }
};

// Queries of one 16-column tile, scale not applied.
template <int D, bool CB16, int QP>
struct Query;

template <int D, int QP>
struct Query<D, true, QP> {
  static constexpr int KS = D / 32;
  static constexpr bool HALF = D % 32 != 0;
  v4i q[QP][KS];
  v2i qh[QP];
  __device__ __forceinline__ void load(const void* base, int64_t at, bool there, int, int g) {
    if constexpr (QP == 1) {
      const uint16_t* p = (const uint16_t*)base + at;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[0][s] = there ? *(const v4i*)(p + 32 * s + 8 * g) : v4i{0, 0, 0, 0};
      if constexpr (HALF) qh[0] = there ? *(const v2i*)(p + 32 * KS + 4 * g) : v2i{0, 0};
    } else {
      const float* p = (const float*)base + at;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const f4v z = {0, 0, 0, 0};
        const f4v a = there ? *(const f4v*)(p + 32 * s + 8 * g) : z, b = there ? *(const f4v*)(p + 32 * s + 8 * g + 4) : z;
        int w[3][4];
        split3(a[0], a[1], w[0][0], w[1][0], w[2][0]);
        split3(a[2], a[3], w[0][1], w[1][1], w[2][1]);
        split3(b[0], b[1], w[0][2], w[1][2], w[2][2]);
        split3(b[2], b[3], w[0][3], w[1][3], w[2][3]);
#pragma unroll
        for (int j = 0; j < 3; ++j) q[j][s] = v4i{w[j][0], w[j][1], w[j][2], w[j][3]};
      }
      if constexpr (HALF) {
        const f4v a = there ? *(const f4v*)(p + 32 * KS + 4 * g) : f4v{0, 0, 0, 0};
        int w[3][2];
        split3(a[0], a[1], w[0][0], w[1][0], w[2][0]);
        split3(a[2], a[3], w[0][1], w[1][1], w[2][1]);
#pragma unroll
        for (int j = 0; j < 3; ++j) qh[j] = v2i{w[j][0], w[j][1]};
      }
    }
  }
  __device__ __forceinline__ f4v scores(const Tile<D, true>& x, int t) const {
    f4v c = {0, 0, 0, 0};
#pragma unroll
    for (int j = QP - 1; j >= 0; --j) {  // the small parts first
#pragma unroll
      for (int s = 0; s < KS; ++s) c = mfma32(x.k[t][s], q[j][s], c);
      if constexpr (HALF) c = mfma16(x.kh[t], qh[j], c);
    }
    return c;
  }
};

template <int D, int QP>
struct Query<D, false, QP> {
  static constexpr int DT = D / 16;
  f4v q[DT];
  __device__ __forceinline__ void load(const void* base, int64_t at, bool there, int bf16, int g) {
#pragma unroll
    for (int c = 0; c < DT; ++c) {
      q[c] = f4v{0, 0, 0, 0};
      if (!there) continue;
      if (bf16) {
        const uint16_t* p = (const uint16_t*)base + at + 16 * c + 4 * g;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[c][e] = bf16_to_f32(p[e]);
      } else {
        q[c] = *(const f4v*)((const float*)base + at + 16 * c + 4 * g);
      }
    }
  }
  __device__ __forceinline__ f4v scores(const Tile<D, false>& x, int t) const {
    f4v s = {0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[t][c][e], q[c][e], s, 0, 0, 0);
    return s;
  }
};

// O^T += V^T W^T; w: the lane's eight weights.
template <int D>
__device__ __forceinline__ void add_values(f4v (&o)[D / 16], const Tile<D, true>& x, const float (&w)[8]) {
  v4i p[3];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    int hi, mid, lo;
    split3(w[2 * i], w[2 * i + 1], hi, mid, lo);
    p[0][i] = hi;
    p[1][i] = mid;
    p[2][i] = lo;
  }
#pragma unroll
  for (int d = 0; d < D / 16; ++d) {
    o[d] = mfma32(x.v[d], p[2], o[d]);
    o[d] = mfma32(x.v[d], p[1], o[d]);
    o[d] = mfma32(x.v[d], p[0], o[d]);
  }
}
template <int D>
__device__ __forceinline__ void add_values(f4v (&o)[D / 16], const Tile<D, false>& x, const float (&w)[8]) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[t][d][i], w[4 * t + i], o[d], 0, 0, 0);
}

// One workgroup: a request, a key head, 16 NT (row, query head) pairs and one chunk of the tiles that they see; its
// waves take turns at the tiles and join at the end.
template <int D, bool CB16, int QP, int NT>
__global__ __launch_bounds__(kWaves * 64) void k_paged_attention(PagedAttnArgs g) {
  constexpr int DT = D / 16;
  __shared__ __attribute__((aligned(16))) float lds_o[kWaves][DT * 64 * 4];
  __shared__ float lds_m[kWaves][NT][16], lds_l[kWaves][NT][16];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int m = lane & 15, grp = lane >> 4;
  int id = blockIdx.x;
  const int chunk = id % g.chunks;
  id /= g.chunks;
  const int head = id % g.kv_heads;
  id /= g.kv_heads;
  const int qt = id % g.qtiles, b = id / g.qtiles;
  const Request rq = request_of(g, b, chunk == 0 && head == 0 && qt == 0 && threadIdx.x == 0);
  const int cols = rq.n * g.group, col0 = qt * 16 * NT;
  if (col0 >= cols) return;
  const int pos0 = rq.len - rq.n;
  const Span span = span_of(pos0 + col0 / g.group, pos0 + (min(cols, col0 + 16 * NT) - 1) / g.group, g.window, g.sinks);
  const int t0 = chunk * g.chunk_tiles, t1 = min(span.tiles, t0 + g.chunk_tiles);
  if (t0 >= t1 && chunk > 0) return;

  Query<D, CB16, QP> q[NT];
  int pos[NT];      // of the lane's column
  f4v o[NT][DT];
  float ref[NT], sum[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = col0 + 16 * n + m, i = min(col, cols - 1) / g.group, hq = head * g.group + min(col, cols - 1) % g.group;
    q[n].load(g.q, (int64_t)(rq.row0 + i) * g.ldq + hq * D, col < cols, g.q_bf16, grp);
    pos[n] = pos0 + i;
    ref[n] = -INFINITY;
    sum[n] = 0.0f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[n][d] = f4v{0, 0, 0, 0};
  }

  const int ps = 1 << g.page_shift;
  const int32_t* table = g.table + (int64_t)b * g.max_blocks;
  // Page of key group a (8 keys) of a tile; keys past the request's last give the last one's.
  auto page_at = [&](int tile, int a) -> int {
    return table[min(tile * kTileKeys + 8 * a, rq.len - 1) >> g.page_shift];
  };
  auto in_range = [&](int page) { return (uint32_t)page < (uint32_t)g.num_pages; };
  auto block = [&](int page) -> int64_t { return ((int64_t)(in_range(page) ? page : 0) * g.kv_heads + head) * D << g.page_shift; };

  Tile<D, CB16> x;
  int it = t0 + wave;
  int page_k = 0, page_v = 0, next_k = 0, next_v = 0;
  auto load_k = [&](int tile, int page) {
    const int key = tile * kTileKeys + 8 * (m >> 2) + (m & 3);
    x.load_k((const char*)g.k, block(page) + (int64_t)(key & (ps - 1)) * D, grp);
  };
  if (it < t1) {
    const int tile = span.tile(it);
    page_k = page_at(tile, m >> 2);
    page_v = page_at(tile, grp);
    load_k(tile, page_k);
    if (it + kWaves < t1) {
      next_k = page_at(span.tile(it + kWaves), m >> 2);
      next_v = page_at(span.tile(it + kWaves), grp);
    }
  }
#pragma unroll 1
  for (; it < t1; it += kWaves) {
    const int tile = span.tile(it), key0 = tile * kTileKeys;
    const int kg = key0 + 8 * grp;  // this lane's first key
    x.load_v((const char*)g.v, block(page_v) + ((int64_t)m << g.page_shift) + (kg & (ps - 1)), g.page_shift);
    f4v s[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[n][t] = q[n].scores(x, t);
    const int page = page_v;
    if (it + kWaves < t1) {
      load_k(span.tile(it + kWaves), next_k);
      page_v = next_v;
      if (it + 2 * kWaves < t1) {
        next_k = page_at(span.tile(it + 2 * kWaves), m >> 2);
        next_v = page_at(span.tile(it + 2 * kWaves), grp);
      }
    }
    // Tiles that not every row sees whole: keys out of sight leave the sums alone, whatever they hold.
    const bool whole = key0 + kTileKeys - 1 <= span.first_pos &&
                       (g.window <= 0 || key0 > span.last_pos - g.window || key0 + kTileKeys <= g.sinks);
    const bool bad = !in_range(page);
    if (!whole || __any(bad)) {
      uint32_t some = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int key = kg + i;
        const bool any = key <= span.last_pos && (g.window <= 0 || key > span.first_pos - g.window || key < g.sinks);
        some |= any ? 1u << i : 0u;
      }
      if (bad && some && g.err) *g.err = 1;
      if (bad) some = 0;
      x.keep_v(some);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int key = kg + i;
          const bool see = (some >> i & 1) && key <= pos[n] && (g.window <= 0 || key > pos[n] - g.window || key < g.sinks);
          s[n][i >> 2][i & 3] = see ? s[n][i >> 2][i & 3] : -INFINITY;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                        fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3]))) * g.scale_log2e;
      if (__any(top > ref[n] + kSlack)) {
        top = fmaxf(top, xor_lane_f<16>(top));
        top = fmaxf(top, xor_lane_f<32>(top));
        const float to = fmaxf(ref[n], top);
        const float by = to > -INFINITY ? exp2_fast(ref[n] - to) : 1.0f;
        ref[n] = to;
        sum[n] *= by;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] *= by;
      }
      const float base = ref[n] > -INFINITY ? -ref[n] : 0.0f;
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = exp2_fast(__builtin_fmaf(s[n][i >> 2][i & 3], g.scale_log2e, base));
      sum[n] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      add_values<D>(o[n], x, w);
    }
  }

  // ---- the waves' parts, then the row's or the chunk's ----
  const bool alone = span.tiles <= g.chunk_tiles;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sum[n] += xor_lane_f<16>(sum[n]);
    sum[n] += xor_lane_f<32>(sum[n]);
    if (lane < 16) {
      lds_m[wave][n][m] = ref[n];
      lds_l[wave][n][m] = sum[n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top = lds_m[0][n][m];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lds_m[w][n][m]);
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float r = lds_m[w][n][m];
      total += r > -INFINITY ? lds_l[w][n][m] * exp2_fast(r - top) : lds_l[w][n][m];
    }
    const float by = ref[n] > -INFINITY ? exp2_fast(ref[n] - top) : 1.0f;
    if (n) __syncthreads();
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f4v*)&lds_o[wave][(d * 64 + lane) * 4] = o[n][d] * by;
    __syncthreads();
    const int col = col0 + 16 * n + m;
    const int i = col / g.group, hq = head * g.group + col % g.group;
    const int64_t row = rq.row0 + i;
    // A row that sees no key gives zeros; one whose weights are all zero what the formula gives, 0 / 0.
    const bool sees = pos0 + i >= 0;
    for (int d = wave; d < DT; d += kWaves) {
      f4v v = *(const f4v*)&lds_o[0][(d * 64 + lane) * 4];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) v += *(const f4v*)&lds_o[w][(d * 64 + lane) * 4];
      if (col >= cols) continue;
      if (alone) {
        v = sees ? v / total : f4v{0, 0, 0, 0};
        *(f4v*)(g.out + row * g.ldo + hq * D + 16 * d + 4 * grp) = v;
      } else {
        const int64_t at = (row * g.heads + hq) * g.chunks + chunk;
        *(f4v*)(g.part_o + at * D + 16 * d + 4 * grp) = v;
        if (d == 0 && grp == 0) *(float2*)(g.part_ml + 2 * at) = make_float2(top, total);
      }
    }
  }
}

// Joins the chunks of one (row, query head): a wave each.
template <int D>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttnArgs g, int nt16) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int per = g.max_rows * g.heads;
  const int b = (int)(item / per), i = (int)(item % per) / g.heads, hq = (int)(item % g.heads);
  if (b >= g.requests) return;
  const Request rq = request_of(g, b, false);
  if (i >= rq.n) return;
  const int cols = rq.n * g.group, qt = (i * g.group + hq % g.group) / nt16, col0 = qt * nt16, pos0 = rq.len - rq.n;
  const Span span = span_of(pos0 + col0 / g.group, pos0 + (min(cols, col0 + nt16) - 1) / g.group, g.window, g.sinks);
  if (span.tiles <= g.chunk_tiles) return;  // written already
  const int chunks = (span.tiles + g.chunk_tiles - 1) / g.chunk_tiles;
  const int64_t row = rq.row0 + i, at = (row * g.heads + hq) * g.chunks;
  const float2* ml = (const float2*)g.part_ml + at;
  float top = -INFINITY;
  for (int c = lane; c < chunks; c += 64) top = fmaxf(top, ml[c].x);
  top = wave_max(top);
  const float base = top > -INFINITY ? top : 0.0f;
  constexpr int PER = (D + 63) / 64;
  float total = 0.0f, v[PER] = {};
#pragma unroll 4
  for (int c = 0; c < chunks; ++c) {
    const float2 e = ml[c];
    const float by = e.x > -INFINITY ? exp2_fast(e.x - base) : 1.0f;
    total += e.y * by;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j * 64 + lane < D) v[j] += g.part_o[(at + c) * D + j * 64 + lane] * by;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (j * 64 + lane < D) g.out[row * g.ldo + hq * D + j * 64 + lane] = pos0 + i >= 0 ? v[j] / total : 0.0f;
}

// How a call is split: by sizes that the host knows.
struct Plan {
  int nt, qtiles, chunks, chunk_tiles;
};
Plan plan_of(const PagedAttnArgs& g) {
  Plan p;
  const int cols = g.max_rows * g.group;
  p.nt = cols > 16 ? 2 : 1;
  p.qtiles = (cols + 16 * p.nt - 1) / (16 * p.nt);
  int64_t keys = g.max_keys;
  if (g.window > 0) keys = std::min<int64_t>(keys, (int64_t)g.window + g.max_rows + g.sinks + 2 * kTileKeys);
  const int64_t tiles = (keys + kTileKeys - 1) / kTileKeys;
  const int64_t groups = (int64_t)std::max(1, g.requests) * g.kv_heads * p.qtiles;
  const int64_t want = std::max<int64_t>(1, 2048 / groups);  // workgroups: eight a compute unit
  p.chunk_tiles = (int)std::max<int64_t>(2 * kWaves, (tiles + want - 1) / want);
  p.chunks = (int)std::max<int64_t>(1, (tiles + p.chunk_tiles - 1) / p.chunk_tiles);
  return p;
}

template <int D, bool CB16, int QP, int NT>
hipError_t launch(const PagedAttnArgs& g, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL((k_paged_attention<D, CB16, QP, NT>), dim3((unsigned)blocks), dim3(kWaves * 64), 0, s, g);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || g.chunks == 1) return e;
  const int64_t items = (int64_t)g.requests * g.max_rows * g.heads;
  hipLaunchKernelGGL((k_paged_join<D>), dim3((unsigned)((items + 3) / 4)), dim3(256), 0, s, g, 16 * NT);
  return hipGetLastError();
}
template <int D>
hipError_t launch_d(const PagedAttnArgs& g, int nt, int64_t blocks, hipStream_t s) {
  if (!g.cache_bf16) return nt == 1 ? launch<D, false, 1, 1>(g, blocks, s) : launch<D, false, 1, 2>(g, blocks, s);
  if (g.q_bf16) return nt == 1 ? launch<D, true, 1, 1>(g, blocks, s) : launch<D, true, 1, 2>(g, blocks, s);
  return nt == 1 ? launch<D, true, 3, 1>(g, blocks, s) : launch<D, true, 3, 2>(g, blocks, s);
}

}  // namespace

bool paged_attention_launchable(const PagedAttnArgs& g) {
  const Plan p = plan_of(g);
  return (int64_t)g.requests * g.kv_heads * p.qtiles * p.chunks <= 0x7FFFFF &&  // 2^31 threads
         (int64_t)g.requests * g.max_rows * g.heads <= 0x1FFFFFF;
}

size_t paged_attention_bytes(const PagedAttnArgs& g) {
  const Plan p = plan_of(g);
  return p.chunks == 1 ? 0 : (size_t)g.rows * g.heads * p.chunks * (g.head_dim + 2) * sizeof(float);
}

hipError_t launch_paged_attention(const PagedAttnArgs& args, void* workspace, hipStream_t s) {
  PagedAttnArgs g = args;
  if (g.requests == 0 || g.rows == 0) return hipSuccess;
  const Plan p = plan_of(g);
  g.qtiles = p.qtiles;
  g.chunks = p.chunks;
  g.chunk_tiles = p.chunk_tiles;
  g.part_o = (float*)workspace;
  g.part_ml = g.part_o + (size_t)g.rows * g.heads * p.chunks * g.head_dim;
  const int64_t blocks = (int64_t)g.requests * g.kv_heads * p.qtiles * p.chunks;
  if (!paged_attention_launchable(g)) return hipErrorInvalidValue;
  if (g.head_dim == 48) return launch_d<48>(g, p.nt, blocks, s);
  if (g.head_dim == 64) return launch_d<64>(g, p.nt, blocks, s);
  if (g.head_dim == 128) return launch_d<128>(g, p.nt, blocks, s);
  return hipErrorInvalidValue;
}

}  // namespace mh
