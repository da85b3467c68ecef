// paged_attention.hip — attention of a step's new rows over their requests' pages of a key-value cache, split over the
// cache's length and joined.
//
// Row i of the n rows of request b stands at position p = len[b] - n + i and sees the keys j <= p, with a window those
// with j > p - window or j < sinks:
//   out = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q k_j).
// One pass over the keys keeps, per query, a reference m close to the largest score so far, l = sum w_j e^-m and the sum
// of w_j e^-m v_j; parts of the keys join by rescaling each to the largest m.  m is -inf only where no key has been seen: a
// seen one, whatever its score, makes it kSeen at least (scores of -inf alone give 0 / 0, no key at all gives 0).
#include "device_common.h"
#include "kernels.h"
#include "mass.h"

#include <algorithm>

namespace mh {
namespace {

constexpr int kTileKeys = 32;  // keys a wave takes at once
constexpr int kWaves = 4;
// Least tiles of a share (us, 4 | 8 | 16 | 32: 1 request of 4000 keys of 8 heads of 64 13.5 | 14.2 | 15.3 | 17.7, 8 of up to 4000
// of 8 heads of 128 with 6 rows of 4 heads each 28.0 | 31.3 | 26.9 | 34.6; calls whose shares are longer all the same).
constexpr int kMinTiles = 2 * kWaves;
// What splitting sequences costs (another beginning and end in every workgroup, a second launch, 7 to 10 us), as tiles
// that one workgroup works on meanwhile: 0.11 us for 8 KB of keys and values.  us, unsplit | split, 8 key heads of 64, bf16:
// 1 request of 1024 keys 9.5 | 12.1, of 2048 13.6 | 12.4, of 4000 22.5 | 13.2; 64 ragged ones of up to 1024 17.7 | 21.5, of up
// to 2048 29.6 | 33.2; 24 of up to 16000 121 | 85; with 6 rows of 4 heads of 128 each, up to 8192 keys, 289 | 211.
constexpr int kSplitCost = 64;
// Workgroups that read as fast as the whole chip does (32, 64 and 128 within 1 % of each other from 1 to 300 requests, but for
// 128 of up to 3000 keys of one head of 64: 24.1, 24.1 and 22.3 us).
constexpr int kRate = 64;
template <int D, bool CB16, int NT>
constexpr int split_cost() {
  return kSplitCost * 8 / (D / 8 * (CB16 ? 1 : 2)) / NT;
}
// Scores (in octaves) may pass the reference by so much before the sums are rescaled: weights up to 2^8.
constexpr float kSlack = 8.0f;
constexpr float kSeen = -0x1.fffffep127f;  // the lowest finite value

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
// An operand of half a product: four values a lane, the other four zero.  The instruction for 16 summed values is not
// taken: right behind one of 32 on the same sums it adds to what they were before, and the compiler puts no wait
// between the two (six in turns: all 256 sums wrong; with a wait for loads between them, none).  Sums that one kind of
// instruction alone adds to are passed on in order.
__device__ __forceinline__ v4i half(v2i a) { return v4i{a[0], a[1], 0, 0}; }

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
  v4i kh[2];
  v4i v[DT];
  __device__ __forceinline__ void load_k(const char* kc, int64_t at, int g) {  // at: element of the row's first dimension
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char* p = kc + 2 * (at + t * 4 * D);
#pragma unroll
      for (int s = 0; s < KS; ++s) k[t][s] = *(const v4i*)(p + 64 * s + 16 * g);
      if constexpr (HALF) kh[t] = half(*(const v2i*)(p + 64 * KS + 8 * g));
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
  v4i qh[QP];
  __device__ __forceinline__ void load(const void* base, int64_t at, bool there, int, int g) {
    if constexpr (QP == 1) {
      const uint16_t* p = (const uint16_t*)base + at;
#pragma unroll
      for (int s = 0; s < KS; ++s) q[0][s] = there ? *(const v4i*)(p + 32 * s + 8 * g) : v4i{0, 0, 0, 0};
      if constexpr (HALF) qh[0] = half(there ? *(const v2i*)(p + 32 * KS + 4 * g) : v2i{0, 0});
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
        int x[3], y[3];
        split3(a[0], a[1], x[0], x[1], x[2]);
        split3(a[2], a[3], y[0], y[1], y[2]);
#pragma unroll
        for (int j = 0; j < 3; ++j) qh[j] = v4i{x[j], y[j], 0, 0};
      }
    }
  }
  __device__ __forceinline__ f4v scores(const Tile<D, true>& x, int t) const {
    f4v c = {0, 0, 0, 0};
#pragma unroll
    for (int j = QP - 1; j >= 0; --j) {  // the small parts first
#pragma unroll
      for (int s = 0; s < KS; ++s) c = mfma32(x.k[t][s], q[j][s], c);
      if constexpr (HALF) c = mfma32(x.kh[t], qh[j], c);
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

// Registers a thread of an instance needs, as waves a SIMD: workgroups a compute unit, one wave of each on a SIMD.
template <int D, bool CB16, int QP, int NT>
constexpr int waves_a_simd() {
  if (D == 128) return NT == 1 ? (CB16 && QP == 1 ? 3 : 2) : (CB16 && QP == 1 ? 2 : 1);
  if (D == 64 && (!CB16 || QP == 3)) return NT == 1 ? (CB16 ? 4 : 3) : 2;
  return NT == 1 ? 4 : 3;
}

// A sequence is what one query tile and key head of a request see.  Work is counted in its tiles and kBegin more for its
// beginning and end, in the order request, query tile, head.
// us with 2 | 4 | 8 | 16: 61 ragged requests of up to 4001 keys 93.5 | 89.3 | 89.2 | 92.7, 64 of up to 8192 with 6 rows 213 | 211 |
// 211 | 218, 24 of up to 16000 86.5 | 86.1 | 85.2 | 85.5.
constexpr int kBegin = 8;
template <int NT>
__device__ __forceinline__ int64_t request_tiles(const PagedAttnArgs& g, const Request& r, int& longest) {
  const int cols = r.n * g.group, pos0 = r.len - r.n;
  int64_t all = 0;
  for (int col0 = 0; col0 < cols; col0 += 16 * NT) {
    const int n = kBegin + span_of(pos0 + col0 / g.group, pos0 + (min(cols, col0 + 16 * NT) - 1) / g.group, g.window, g.sinks).tiles;
    longest = max(longest, n);
    all += n;
  }
  return all * g.kv_heads;
}

template <class T>
__device__ __forceinline__ T uniform(T v) {
  static_assert(sizeof(T) == 4, "one register");
  return __builtin_bit_cast(T, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)v));
}

// Where a workgroup's share of all tiles begins: request b, `into` tiles into it, `quota` tiles to take; quota 0: every
// sequence is one workgroup's.
struct Share {
  int b;
  int64_t into, quota;
};
constexpr int kThreads = kWaves * 64;
struct ShareLds {
  int64_t sum[kPlanMaxRequests / kThreads + 1], wave[kWaves], into;
  int b, longest[kWaves];
};
template <int NT>
__device__ __forceinline__ Share share_of(const PagedAttnArgs& g, int worker, int cost, ShareLds& L) {
  const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6);
  const int steps = (g.requests + kThreads - 1) / kThreads;
  int64_t mine = 0, upto = 0, total = 0;
  int longest = 0;
  auto step = [&](int i) {  // this thread's request's tiles, and their running sum within the step
    const int b = i * kThreads + t;
    mine = b < g.requests ? request_tiles<NT>(g, request_of(g, b, worker == 0), longest) : 0;
    upto = (int64_t)wave_scan_mass((uint64_t)mine);
    if (lane == 63) L.wave[wave] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      upto += w < wave ? L.wave[w] : 0;
      all += L.wave[w];
    }
    return all;
  };
  if (t == 0) L.b = g.requests;
  for (int i = 0; i < steps; ++i) {
    const int64_t all = step(i);
    if (steps > 1) {
      if (t == 0) L.sum[i] = all;
      __syncthreads();
    }
    total += all;
  }
  longest = (int)wave_max((float)longest);  // at most 2^22: exact
  if (lane == 0) L.longest[wave] = longest;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) longest = max(longest, L.longest[w]);
  longest = uniform(longest);
  total = uniform64(total);
  // Unsplit, the longest sequence ends last, and by so much later as it is longer than what the others do on average.
  const int64_t at_rate = total / kRate, even = total / min((int64_t)g.workers, (int64_t)g.requests * g.qtiles * g.kv_heads);
  if (max((int64_t)longest, at_rate) + max(longest - even, (int64_t)0) <= at_rate + cost) return {0, 0, 0};
  const int64_t quota = max((total + g.workers - 1) / g.workers, (int64_t)kMinTiles + kBegin);
  int64_t at = (int64_t)worker * quota;
  int i = 0;
  if (steps > 1) {
    for (; i < steps - 1 && at >= L.sum[i]; ++i) at -= L.sum[i];
    step(i);
  }
  if (worker < g.workers && mine && upto - mine <= at && at < upto) {
    L.b = i * kThreads + t;
    L.into = at - (upto - mine);
  }
  __syncthreads();
  return {uniform(L.b), uniform64(L.into), quota};
}

// One column's keys one after the other, a wave's lanes (m, g): the column of query m, dimensions d % 4 == g of the score
// and 16 d + 4 g .. 4 g + 3 of the sums, which are kept in `o` (LDS).  One key after the other, each a trip to memory: one NaN among
// the values that a call's rows see takes 131000 keys from 103 us to 2.6 ms, 2000 keys of 8 heads of 64 from 15 us to 1.0 ms.
template <int D, bool CB16>
struct Slow {
  const PagedAttnArgs& g;
  const Span& span;
  const int32_t* table;
  f4v* o;
  int head, lane;
  float ref, sum;
  __device__ __forceinline__ float value(const void* p, int64_t i) const {
    return CB16 ? bf16_to_f32(((const uint16_t*)p)[i]) : ((const float*)p)[i];
  }
  __device__ __forceinline__ float query_at(int64_t i) const {
    return g.q_bf16 ? bf16_to_f32(((const uint16_t*)g.q)[i]) : ((const float*)g.q)[i];
  }
  __device__ bool finite(int64_t query) const {
    float z = 0.0f;
#pragma unroll 4
    for (int d = lane >> 4; d < D; d += 4) z = __builtin_fmaf(query_at(query + d), 0.0f, z);
    z += xor_lane_f<16>(z);
    z += xor_lane_f<32>(z);
    return z == 0.0f;
  }
  __device__ void sum_keys(int64_t query, int pos, int first, int last) {
    const int grp = lane >> 4, place_mask = (1 << g.page_shift) - 1;
    ref = -INFINITY;
    sum = 0.0f;
#pragma unroll 1
    for (int d = 0; d < D / 16; ++d) o[d * 64 + lane] = f4v{0, 0, 0, 0};
#pragma unroll 1
    for (int it = first; it < last; it += kWaves) {
#pragma unroll 1
      for (int i = 0; i < kTileKeys; ++i) {
        const int key = span.tile(it) * kTileKeys + i;
        if (key > span.last_pos) break;
        const int page = table[key >> g.page_shift], place = key & place_mask;
        const bool there = (uint32_t)page < (uint32_t)g.num_pages;
        const int64_t block = ((int64_t)(there ? page : 0) * g.kv_heads + head) * D << g.page_shift;
        float score = 0.0f;
#pragma unroll 4
        for (int d = grp; d < D; d += 4)
          score = __builtin_fmaf(query_at(query + d), value(g.k, block + (int64_t)place * D + d), score);
        score += xor_lane_f<16>(score);
        score += xor_lane_f<32>(score);
        score *= g.scale_log2e;
        if (!there || key > pos || (g.window > 0 && key <= pos - g.window && key >= g.sinks)) continue;
        const float to = fmaxf(fmaxf(score, kSeen), ref), by = exp2_fast(ref - to), w = exp2_fast(score - to);
        ref = to;
        sum = sum * by + w;
#pragma unroll 2
        for (int d = 0; d < D / 16; ++d) {
          f4v v = o[d * 64 + lane] * by;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = __builtin_fmaf(w, value(g.v, block + ((int64_t)(16 * d + 4 * grp + e) << g.page_shift) + place), v[e]);
          o[d * 64 + lane] = v;
        }
      }
    }
  }
};

// A workgroup of four waves takes tiles of one sequence, in turns, and joins the waves' sums at its end.  With few keys
// (g.whole), and where no sequence is long beside the rest, a sequence is one workgroup's.  Otherwise as many
// workgroups as run at once take the same number of tiles each, one sequence after another, whatever their lengths; what
// is not a whole sequence goes to the workspace: part 0 of a workgroup is the end or middle of a sequence, part 1 the
// beginning of one.
// Each key and value is read once for the heads and rows of a tile, one operation a byte (bf16) and column: memory bounds
// it.  One request of 131000 keys of 8 heads of 128: 537 MB in 97 us, 5.5 TB/s, and 5 us for the join; one of a few hundred
// keys 8.5 us from call to call, the launch and a chain of loads.
template <int D, bool CB16, int QP, int NT>
__global__ __launch_bounds__(kThreads, (waves_a_simd<D, CB16, QP, NT>())) void k_paged_attention(PagedAttnArgs g) {
  constexpr int DT = D / 16;
  __shared__ __attribute__((aligned(16))) float lds_o[kWaves][DT * 64 * 4];
  __shared__ float lds_m[kWaves][NT][16], lds_l[kWaves][NT][16];
  __shared__ ShareLds share;
  __shared__ int lds_odd[kWaves];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int m = lane & 15, grp = lane >> 4;
  int b, qt = 0, head = 0;
  int64_t quota = 0, left = 0;  // of work to take: in all, still
  int u0 = 0;                   // of the sequence's work, where this part begins
  if (!g.whole) {
    const Share s = share_of<NT>(g, blockIdx.x, split_cost<D, CB16, NT>(), share);
    b = s.b;
    quota = left = s.quota;
    if (b >= g.requests) return;
  }
  if (quota == 0) {
    int id = blockIdx.x;
    head = id % g.kv_heads;
    id /= g.kv_heads;
    qt = id % g.qtiles;
    b = id / g.qtiles;
    if (b >= g.requests) return;
    left = 0x7FFFFFFF;
  } else {
    const Share s = {b, uniform64(share.into), quota};
    // The query tile and head that the share begins in.
    const Request rq = request_of(g, b, false);
    const int cols = rq.n * g.group, pos0 = rq.len - rq.n;
    int64_t into = s.into;
    for (;; ++qt) {
      const int col0 = qt * 16 * NT;
      const int tiles = kBegin + span_of(pos0 + col0 / g.group, pos0 + (min(cols, col0 + 16 * NT) - 1) / g.group, g.window, g.sinks).tiles;
      if (into < (int64_t)tiles * g.kv_heads || col0 + 16 * NT >= cols) {
        head = (int)(into / tiles);
        u0 = (int)(into % tiles);
        break;
      }
      into -= (int64_t)tiles * g.kv_heads;
    }
  }
  const int ps = 1 << g.page_shift;
  auto in_range = [&](int page) { return (uint32_t)page < (uint32_t)g.num_pages; };

  for (;;) {
    const Request rq = request_of(g, b, g.whole && head == 0 && qt == 0 && threadIdx.x == 0);
    const int cols = uniform(rq.n * g.group), col0 = qt * 16 * NT;
    if (col0 >= cols) {  // no (more) rows
      if (quota == 0 || ++b >= g.requests) return;
      qt = head = u0 = 0;
      continue;
    }
    const int pos0 = rq.len - rq.n;
    const Span span = span_of(pos0 + col0 / g.group, pos0 + (min(cols, col0 + 16 * NT) - 1) / g.group, g.window, g.sinks);
    const int all = kBegin + span.tiles, u1 = (int)min((int64_t)all, u0 + left);
    const int t0 = max(0, u0 - kBegin), last = max(0, u1 - kBegin);  // of its tiles
    const bool alone = u0 == 0 && u1 == all;
    if (!g.whole && u0 == 0 && threadIdx.x == 0)  // its rest is the next workgroups'
      g.begun[((int64_t)b * g.qtiles + qt) * g.kv_heads + head] =
          make_int2(blockIdx.x, alone ? 1 : (int)((quota - left + all + quota - 1) / quota));
    left -= u1 - u0;

    Query<D, CB16, QP> q[NT];
    int pos[NT];  // of the lane's column
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

    const int32_t* table = g.table + (int64_t)b * g.max_blocks;
    // Page of key group a (8 keys) of a tile; keys past the request's last give the last one's.
    auto page_at = [&](int tile, int a) -> int {
      return table[min(tile * kTileKeys + 8 * a, rq.len - 1) >> g.page_shift];
    };
    auto block = [&](int page) -> int64_t { return ((int64_t)(in_range(page) ? page : 0) * g.kv_heads + head) * D << g.page_shift; };

    Tile<D, CB16> x;
    int it = t0 + wave;
    bool saw = false;  // a tile that every row sees whole
    int page_k = 0, page_v = 0, next_k = 0, next_v = 0;
    auto load_k = [&](int tile, int page) {
      const int key = tile * kTileKeys + 8 * (m >> 2) + (m & 3);
      x.load_k((const char*)g.k, block(page) + (int64_t)(key & (ps - 1)) * D, grp);
    };
    if (it < last) {
      const int tile = span.tile(it);
      page_k = page_at(tile, m >> 2);
      page_v = page_at(tile, grp);
      load_k(tile, page_k);
      const int next = span.tile(min(it + kWaves, last - 1));
      next_k = page_at(next, m >> 2);
      next_v = page_at(next, grp);
    }
#pragma unroll 1
    for (; it < last; it += kWaves) {
      const int tile = span.tile(it), key0 = tile * kTileKeys;
      const int kg = key0 + 8 * grp;  // this lane's first key
      x.load_v((const char*)g.v, block(page_v) + ((int64_t)m << g.page_shift) + (kg & (ps - 1)), g.page_shift);
      f4v s[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[n][t] = q[n].scores(x, t);
      const int page = page_v;
      // The next tile's keys, and the pages of the one after (at the end some tile once more: behind a branch the
      // values' wait would have to cover these loads too).
      load_k(span.tile(min(it + kWaves, last - 1)), next_k);
      page_v = next_v;
      const int after = span.tile(min(it + 2 * kWaves, last - 1));
      next_k = page_at(after, m >> 2);
      next_v = page_at(after, grp);
      // Tiles that not every row sees whole: keys out of sight leave the sums alone, whatever they hold.
      const bool whole = key0 + kTileKeys - 1 <= span.first_pos &&
                         (g.window <= 0 || key0 > span.last_pos - g.window || key0 + kTileKeys <= g.sinks);
      const bool bad = !in_range(page);
      if (!whole || __any(bad)) {
        // Which of the lane's eight keys are seen by rows from position `low` to `high`.
        auto first_of = [](int n) { return (1u << min(max(n, 0), 8)) - 1; };
        auto seen = [&](int low, int high) {
          const uint32_t out = g.window > 0 ? first_of(low - g.window + 1 - kg) & ~first_of(g.sinks - kg) : 0u;
          return first_of(high + 1 - kg) & ~out;
        };
        uint32_t some = seen(span.first_pos, span.last_pos);
        if (bad && some && g.err) *g.err = 1;
        if (bad) some = 0;
        x.keep_v(some);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const uint32_t see = some & seen(pos[n], pos[n]);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[n][i >> 2][i & 3] = see >> i & 1 ? s[n][i >> 2][i & 3] : -INFINITY;
          if (see) ref[n] = fmaxf(ref[n], kSeen);  // as long as it is kSeen the column's lanes may differ: all sums are 0
        }
      } else {
        saw = true;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                          fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3]))) * g.scale_log2e;
        if (__any(top > ref[n] + kSlack)) {
          top = fmaxf(top, xor_lane_f<16>(top));
          top = fmaxf(top, xor_lane_f<32>(top));
          const float to = top > ref[n] + kSlack ? top : ref[n];  // each column by its own scores, whatever the others'
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

    // ---- the waves' parts, then the rows' or the share's ----
    // The lane, unknown to the compiler: it would keep what follows from it in registers all along.
    int l = lane;
    asm volatile("" : "+v"(l));
    const int lm = l & 15, lg = l >> 4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      ref[n] = fmaxf(ref[n], saw ? kSeen : -INFINITY);
      ref[n] = fmaxf(ref[n], xor_lane_f<16>(ref[n]));
      ref[n] = fmaxf(ref[n], xor_lane_f<32>(ref[n]));
      sum[n] += xor_lane_f<16>(sum[n]);
      sum[n] += xor_lane_f<32>(sum[n]);
      if (l < 16) {
        lds_m[wave][n][lm] = ref[n];
        lds_l[wave][n][lm] = sum[n];
      }
    }
    // Infinities and NaN: a weight of zero times one that a row does not see, or a part of a product, makes a NaN of what is
    // none.  Columns with any, but for those whose query is the cause, are formed again, key by key in the formula's own
    // terms, as slow as that is.
    float zero[NT], any_zero = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      zero[n] = sum[n] * 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) zero[n] = __builtin_fmaf(o[n][d][i], 0.0f, zero[n]);
      any_zero += zero[n];
    }
    const bool odd = __any(any_zero != 0.0f);
    if (l == 0) lds_odd[wave] = odd;
    __syncthreads();
    if (lds_odd[0] | lds_odd[1] | lds_odd[2] | lds_odd[3]) {
      if (odd) {
        Slow<D, CB16> slow = {g, span, table, (f4v*)lds_o[wave], head, l};
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {
          float z = zero[0];
#pragma unroll
          for (int k = 1; k < NT; ++k) z = k == n ? zero[k] : z;
          z += xor_lane_f<16>(z);
          z += xor_lane_f<32>(z);
          const int col = min(col0 + 16 * n + lm, cols - 1);
          const int64_t query = (int64_t)(rq.row0 + col / g.group) * g.ldq + (head * g.group + col % g.group) * D;
          const bool again = z != 0.0f && slow.finite(query);
          if (!__any(again)) continue;
          slow.sum_keys(query, pos0 + col / g.group, t0 + wave, last);
          if (again && l < 16) {
            lds_m[wave][n][l] = slow.ref;
            lds_l[wave][n][l] = slow.sum;
          }
#pragma unroll
          for (int k = 0; k < NT; ++k) {
            if (k != n || !again) continue;
            ref[k] = slow.ref;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[k][d] = slow.o[d * 64 + l];
          }
        }
      }
      __syncthreads();
    }
    const int64_t part = (int64_t)blockIdx.x * 2 + (u0 > 0 ? 0 : 1);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float top = lds_m[0][n][lm];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, lds_m[w][n][lm]);
      float total = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float r = lds_m[w][n][lm];
        total += r > -INFINITY ? lds_l[w][n][lm] * exp2_fast(r - top) : lds_l[w][n][lm];
      }
      const float by = ref[n] > -INFINITY ? exp2_fast(ref[n] - top) : 1.0f;
      if (n) __syncthreads();
#pragma unroll
      for (int d = 0; d < DT; ++d) *(f4v*)&lds_o[wave][(d * 64 + l) * 4] = o[n][d] * by;
      __syncthreads();
      const int col = col0 + 16 * n + lm;
      const int i = col / g.group, hq = head * g.group + col % g.group;
      for (int d = wave; d < DT; d += kWaves) {
        f4v v = *(const f4v*)&lds_o[0][(d * 64 + l) * 4];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) v += *(const f4v*)&lds_o[w][(d * 64 + l) * 4];
        if (col >= cols) continue;
        if (alone) {
          v = top > -INFINITY ? v / total : f4v{0, 0, 0, 0};
          *(f4v*)(g.out + (int64_t)(rq.row0 + i) * g.ldo + hq * D + 16 * d + 4 * lg) = v;
        } else {
          const int64_t at = part * (16 * NT) + 16 * n + lm;
          *(f4v*)(g.part_o + at * D + 16 * d + 4 * lg) = v;
          if (d == 0 && lg == 0) *(float2*)(g.part_ml + 2 * at) = make_float2(top, total);
        }
      }
    }
    if (quota == 0 || left <= 0) return;
    u0 = 0;
    if (++head == g.kv_heads) {
      head = 0;
      ++qt;
    }
  }
}

// Joins the parts of a sequence's columns, 1 << lg_cols columns a workgroup: the largest reference first, then the parts'
// sums, four dimensions a lane, as many parts at once as fit, and the parts shared among a column's waves.
template <int D, int NT>
__global__ __launch_bounds__(kThreads) void k_paged_join(PagedAttnArgs g, int lg_cols) {
  constexpr int QUADS = D / 4, AT_ONCE = 64 / QUADS;  // D = 48: 5 parts, and four lanes idle
  __shared__ f4v lds_o[kWaves][QUADS];
  __shared__ float lds_l[kWaves];
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6);
  const int groups = 16 * NT >> lg_cols, seq = blockIdx.x / groups, split = wave >> lg_cols, splits = kWaves >> lg_cols;
  const int base_col = blockIdx.x % groups << lg_cols, col_in = base_col + (wave & ((1 << lg_cols) - 1));
  const int head = seq % g.kv_heads, qt = seq / g.kv_heads % g.qtiles, b = seq / g.kv_heads / g.qtiles;
  const Request rq = request_of(g, b, false);
  const int cols = uniform(rq.n * g.group) - qt * 16 * NT;
  if (base_col >= cols) return;
  const int2 begun = g.begun[seq];
  const int first = uniform(begun.x), parts = uniform(begun.y);
  if (parts < 2) return;
  if (first < 0 || parts > g.workers - first) return;  // not of this call: something else wrote to the workspace
  auto place = [&](int p) -> int64_t { return ((int64_t)(first + p) * 2 + (p == 0 ? 1 : 0)) * (16 * NT) + col_in; };
  const float2* ml = (const float2*)g.part_ml;
  const int quad = lane % QUADS, row = lane / QUADS;
  f4v v = {0, 0, 0, 0};
  float sum = 0.0f, top = -INFINITY;
  if (col_in < cols) {
    for (int p = lane; p < parts; p += 64) top = fmaxf(top, ml[place(p)].x);
    top = wave_max(top);
    const float base = top > -INFINITY ? top : 0.0f;
    if (row < AT_ONCE) {
#pragma unroll 8
      for (int p = split * AT_ONCE + row; p < parts; p += splits * AT_ONCE) {
        const int64_t at = place(p);
        const float2 e = ml[at];
        const f4v x = *(const f4v*)(g.part_o + at * D + 4 * quad);
        const float by = e.x > -INFINITY ? exp2_fast(e.x - base) : 1.0f;
        sum += e.y * by;
        v += x * by;
      }
    }
    const f4v own = v;
    const float own_sum = sum;
#pragma unroll
    for (int r = 1; r < AT_ONCE; ++r) {  // into the first lanes
      const int from = (lane + r * QUADS) & 63;
      sum += __shfl(own_sum, from);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += __shfl(own[i], from);
    }
  }
  if (splits > 1) {
    if (lane < QUADS) lds_o[wave][lane] = v;
    if (lane == 0) lds_l[wave] = sum;
    __syncthreads();
    if (split > 0) return;
    for (int w = 1; w < splits; ++w) {
      v += lds_o[wave + (w << lg_cols)][quad];
      sum += lds_l[wave + (w << lg_cols)];
    }
  }
  if (col_in < cols && lane < QUADS) {
    const int col = qt * 16 * NT + col_in, i = col / g.group, hq = head * g.group + col % g.group;
    *(f4v*)(g.out + (int64_t)(rq.row0 + i) * g.ldo + hq * D + 4 * quad) =
        top > -INFINITY ? v / sum : f4v{0, 0, 0, 0};
  }
}

constexpr int kComputeUnits = 256;
template <int D>
int instance_waves(const PagedAttnArgs& g, int nt) {
  if (!g.cache_bf16) return nt == 1 ? waves_a_simd<D, false, 1, 1>() : waves_a_simd<D, false, 1, 2>();
  if (g.q_bf16) return nt == 1 ? waves_a_simd<D, true, 1, 1>() : waves_a_simd<D, true, 1, 2>();
  return nt == 1 ? waves_a_simd<D, true, 3, 1>() : waves_a_simd<D, true, 3, 2>();
}

// How a call is laid out, by sizes that the host knows.
struct Plan {
  int nt, qtiles, whole, workers;
};
Plan plan_of(const PagedAttnArgs& g) {
  Plan p;
  const int cols = g.max_rows * g.group;
  p.nt = cols > 16 ? 2 : 1;
  p.qtiles = (cols + 16 * p.nt - 1) / (16 * p.nt);
  int64_t keys = g.max_keys;
  if (g.window > 0) keys = std::min<int64_t>(keys, (int64_t)g.window + g.max_rows + g.sinks + 2 * kTileKeys);
  const int64_t sequences = (int64_t)g.requests * p.qtiles * g.kv_heads;
  const int waves = g.head_dim == 48    ? instance_waves<48>(g, p.nt)
                    : g.head_dim == 64 ? instance_waves<64>(g, p.nt)
                                       : instance_waves<128>(g, p.nt);
  const int64_t tiles_most = (keys + kTileKeys - 1) / kTileKeys, work = sequences * (tiles_most + kBegin);
  const int cost = kSplitCost * 8 / (g.head_dim / 8 * (g.cache_bf16 ? 1 : 2)) / p.nt;
  // Few sequences are cut into as few parts as fill the chip's memory (us, one request of 131000 keys with two | three
  // workgroups a compute unit 101.6 | 106.3), many by as many workgroups as run at once (61 requests of up to 4001 keys,
  // two | four: 91.1 | 89.7).
  const int64_t at_once = (int64_t)kComputeUnits * (sequences < kComputeUnits ? std::min(waves, 2) : waves);
  p.workers = (int)std::max<int64_t>(1, std::min(at_once, (work + kMinTiles + kBegin - 1) / (kMinTiles + kBegin)));
  // No second launch where a sequence is not worth splitting at its longest, or there are many.
  p.whole = tiles_most <= cost || sequences >= 4 * kComputeUnits * waves;
  return p;
}

template <int D, bool CB16, int QP, int NT>
hipError_t launch(const PagedAttnArgs& g, hipStream_t s) {
  // At most 2^21 workgroups: 8192 requests of 256 sequences (64 rows of 128 heads, 32 columns each).
  const int64_t sequences = (int64_t)g.requests * g.qtiles * g.kv_heads;
  hipLaunchKernelGGL((k_paged_attention<D, CB16, QP, NT>), dim3((unsigned)(g.whole ? sequences : std::max<int64_t>(sequences, g.workers))),
                     dim3(kThreads), 0, s, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || g.whole) return e;
  const int lg_cols = sequences < kComputeUnits ? 0 : 2;
  hipLaunchKernelGGL((k_paged_join<D, NT>), dim3((unsigned)(sequences * (16 * NT >> lg_cols))), dim3(kThreads), 0, s, g, lg_cols);
  return hipGetLastError();
}
template <int D>
hipError_t launch_d(const PagedAttnArgs& g, int nt, hipStream_t s) {
  if (!g.cache_bf16) return nt == 1 ? launch<D, false, 1, 1>(g, s) : launch<D, false, 1, 2>(g, s);
  if (g.q_bf16) return nt == 1 ? launch<D, true, 1, 1>(g, s) : launch<D, true, 1, 2>(g, s);
  return nt == 1 ? launch<D, true, 3, 1>(g, s) : launch<D, true, 3, 2>(g, s);
}

}  // namespace

size_t paged_attention_bytes(const PagedAttnArgs& g) {
  const Plan p = plan_of(g);
  const size_t sequences = (size_t)g.requests * p.qtiles * g.kv_heads;
  return p.whole ? 0 : (size_t)p.workers * 2 * 16 * p.nt * (g.head_dim + 2) * sizeof(float) + sequences * sizeof(int2);
}

hipError_t launch_paged_attention(const PagedAttnArgs& args, void* workspace, size_t workspace_bytes, hipStream_t s) {
  PagedAttnArgs g = args;
  if (g.requests == 0 || g.rows == 0) return hipSuccess;
  const size_t bytes = paged_attention_bytes(g);
  if (bytes && (!workspace || workspace_bytes < bytes)) return hipErrorInvalidValue;
  const Plan p = plan_of(g);
  g.qtiles = p.qtiles;
  g.whole = p.whole;
  g.workers = p.workers;
  g.part_o = (float*)workspace;
  g.part_ml = g.part_o + (size_t)p.workers * 2 * 16 * p.nt * g.head_dim;
  g.begun = (int2*)(g.part_ml + (size_t)p.workers * 2 * 16 * p.nt * 2);
  if (g.head_dim == 48) return launch_d<48>(g, p.nt, s);
  if (g.head_dim == 64) return launch_d<64>(g, p.nt, s);
  if (g.head_dim == 128) return launch_d<128>(g, p.nt, s);
  return hipErrorInvalidValue;
}

}  // namespace mh
