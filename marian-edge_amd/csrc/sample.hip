// sample.hip — one drawn id per row of logits: temperature, top-k, top-p, min-p
// and a given uniform number.
//
// A row's ids are ordered by logit, descending, equal logits by ascending id.
// With p ~ exp((l - max) / T): top-k keeps the first k ids of that order, top-p
// the shortest prefix of those with at least top_p of their mass, min-p those
// with p >= min_p max(p).  Each keeps a prefix, so together they keep a prefix,
// and the row's kept set is "at or before one (logit, id) pair": that pair is
// what the kernel looks for.  The drawn id is the first in ascending id order
// whose running kept mass exceeds u times the kept mass.
//
// Mass is an integer, 2^44 exp((l - max) / T) rounded to nearest: sums of up to
// 2^19 of them are exact in 64 bits, so they do not depend on the order in which
// lanes and atomics add them, and a row's result is the same whatever the launch
// shape.  The exponential is 2^y by a polynomial in 64 bits: a drawn number
// close to a border of the running mass needs more than fp32's 24 bits (32000
// borders at 2^-24 each would misplace one row in several hundred).
#include "device_common.h"
#include "kernels.h"

#include <algorithm>

namespace mh {
namespace {

constexpr uint32_t kNothing = 0x007FFFFFu;  // argmax_order of -inf (and of NaN): ids that cannot be drawn
constexpr int kBins = 1024;
constexpr int kBinsPerOctave = 16;     // of p, in the histogram over log2 p
constexpr int kMassBits = 44;          // mass of the row's maximum
constexpr float kMinOctave = -45.5f;   // below, the mass rounds to 0
constexpr int kLastBin = 46 * kBinsPerOctave;  // ids past it have no mass
constexpr int kList = 256;             // ids compared pairwise to find a border

// 2^f, |f| <= 1/2: the degree-10 interpolant at Chebyshev nodes (relative error 4e-16).
__device__ __forceinline__ double exp2_poly(double f) {
  double p = 0x1.e6063f7217bc6p-28;
  p = __builtin_fma(p, f, 0x1.b675bca4eeebbp-24);
  p = __builtin_fma(p, f, 0x1.62bfd47773353p-20);
  p = __builtin_fma(p, f, 0x1.ffcb54062e698p-17);
  p = __builtin_fma(p, f, 0x1.430913096fd9fp-13);
  p = __builtin_fma(p, f, 0x1.5d87fe9d7a584p-10);
  p = __builtin_fma(p, f, 0x1.3b2ab6fba1ddap-7);
  p = __builtin_fma(p, f, 0x1.c6b08d703ce49p-5);
  p = __builtin_fma(p, f, 0x1.ebfbdff82c598p-3);
  p = __builtin_fma(p, f, 0x1.62e42fefa3a19p-1);
  return __builtin_fma(p, f, 1.0);
}

// round(2^44 2^y), 0 below kMinOctave and for NaN.
__device__ __forceinline__ uint64_t mass_of(double y) {
  if (!(y >= (double)kMinOctave)) return 0;
  const double k = rint(y);
  const double m = ldexp(exp2_poly(y - k), (int)k + kMassBits);        // at most 2^44
  const double r = m + 0x1p52;                                         // rounds to an integer
  return (uint64_t)__double_as_longlong(r) & 0x000FFFFFFFFFFFFFull;
}

__device__ __forceinline__ float key_logit(uint32_t k) {  // inverse of argmax_order
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}

// DPP move that leaves 0 in the lanes it does not write.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp0_u64(uint64_t v) {
  return ((uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | dpp0<CTRL, ROWS>((uint32_t)v);
}
// Inclusive prefix sums over the wave.
__device__ __forceinline__ uint64_t wave_scan(uint64_t v) {
  v += dpp0_u64<0x111, 0xF>(v);  // row_shr:1
  v += dpp0_u64<0x112, 0xF>(v);  // row_shr:2
  v += dpp0_u64<0x114, 0xF>(v);  // row_shr:4
  v += dpp0_u64<0x118, 0xF>(v);  // row_shr:8
  v += dpp0_u64<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp0_u64<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v += dpp0<0x111, 0xF>(v);
  v += dpp0<0x112, 0xF>(v);
  v += dpp0<0x114, 0xF>(v);
  v += dpp0<0x118, 0xF>(v);
  v += dpp0<0x142, 0xA>(v);
  v += dpp0<0x143, 0xC>(v);
  return v;
}

__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

template <class V>
__device__ __forceinline__ void lds_add(V* p, V v) {
  __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// Ids in descending order of this pair: logit, then ascending id.
__device__ __forceinline__ uint64_t pair_of(uint32_t key, uint32_t id) {
  return ((uint64_t)key << 32) | (0xFFFFFFFFu - id);
}

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));

template <int T, int IDS>
struct SampleLds {
  static constexpr int NW = T / 64;
  uint32_t key[IDS ? IDS : 4];  // order keys, each written and read by one thread
  uint32_t cnt[kBins];
  uint64_t mass[kBins];
  uint32_t zcnt[kBins];   // the finer histogram of a crowded bin
  uint64_t zmass[kBins];  // its masses; then the kept mass of groups of consecutive ids
  uint64_t pair[kList], weight[kList];
  uint64_t wave[NW];
  uint32_t wcnt[NW];
  uint64_t wmass[NW];
  int found;
  uint32_t listed, lo, hi;
  uint64_t border, upto;
};

// Inclusive prefix sums of kBins counts and masses in place; the histogram is
// complete (a barrier before), the prefixes are on return.
template <int T, class Lds>
__device__ __forceinline__ void scan_bins(Lds& L, uint32_t* cnt, uint64_t* mass) {
  constexpr int B = kBins / T, NW = T / 64;
  const int t = threadIdx.x, w = t >> 6;
  uint32_t c[B];
  uint64_t m[B];
#pragma unroll
  for (int i = 0; i < B; ++i) {
    c[i] = cnt[t * B + i] + (i ? c[i - 1] : 0u);
    m[i] = mass[t * B + i] + (i ? m[i - 1] : 0ull);
  }
  uint32_t cs = wave_scan(c[B - 1]);
  uint64_t ms = wave_scan(m[B - 1]);
  if ((t & 63) == 63) {
    L.wcnt[w] = cs;
    L.wmass[w] = ms;
  }
  wg_lds_barrier();
  cs -= c[B - 1];
  ms -= m[B - 1];
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    cs += i < w ? L.wcnt[i] : 0u;
    ms += i < w ? L.wmass[i] : 0ull;
  }
#pragma unroll
  for (int i = 0; i < B; ++i) {
    cnt[t * B + i] = cs + c[i];
    mass[t * B + i] = ms + m[i];
  }
  wg_lds_barrier();
}

// The first of the kBins whose prefix reaches need (of the counts, or of the masses); -1: none.
template <int T, class Lds, class V>
__device__ __forceinline__ int find_bin(Lds& L, const V* prefix, V need) {
  constexpr int B = kBins / T;
  const int t = threadIdx.x;
  wg_lds_barrier();  // every thread has read the previous result
  if (t == 0) {
    L.found = -1;
    L.listed = 0;
    L.lo = 0xFFFFFFFFu;
    L.hi = 0;
  }
  wg_lds_barrier();
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const int b = t * B + i;
    const V before = b ? prefix[b - 1] : (V)0;
    if (before < need && need <= prefix[b]) L.found = b;
  }
  wg_lds_barrier();
  return __builtin_amdgcn_readfirstlane(L.found);
}

// One workgroup of T threads per row.  Thread t holds ids 4(jT + t) + c, so that
// a wave's 256 values of one j are consecutive ids: the final draw sums those,
// finds the group that the number falls into, and one wave scans its 256.  A row
// of up to IDS ids is read from memory once and kept in LDS as order keys, each
// thread its own (in registers the loops over them must be unrolled, which spills
// and outgrows the instruction cache); IDS = 0: each pass reads memory again.
//
// The border of top-k or top-p: a histogram over log2 p (counts, and masses
// where top-p needs them), its prefix sums, the bin where the count or mass is
// reached, then every id of that bin against every other.  A bin of more than
// kList ids (many equal logits) is cut again by (logit, id) pairs, kBins ways a
// time, until few are left.
template <int T, int IDS, bool BF16>
__global__ __launch_bounds__(T) void k_sample(SampleArgs g) {
  constexpr int NW = T / 64;
  // Groups of 256 ids whose kept mass is one of kBins sums.
  constexpr int GROUP = ((IDS ? IDS : kSampleMaxIds) / 256 + kBins - 1) / kBins;
  __shared__ __attribute__((aligned(16))) SampleLds<T, IDS> L;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row = blockIdx.x;

  // ---- the row and its settings (uniform) ----
  uint32_t o0 = 0;
  int n = g.V;
  const void* base;
  if (g.off) {
    o0 = g.off[row];
    const int64_t len = (int64_t)g.off[row + 1] - (int64_t)o0;
    if ((len < 0 || len > g.V) && t == 0 && g.err) *g.err = 1;
    n = (int)min(max(len, (int64_t)0), (int64_t)g.V);
  }
  {
    const int64_t first = g.off ? (int64_t)o0 : row * g.ld;
    base = BF16 ? (const void*)((const uint16_t*)g.logits + first) : (const void*)((const float*)g.logits + first);
  }
  const float temp = g.temperature ? g.temperature[row] : 1.0f;
  const int top_k = g.top_k ? g.top_k[row] : 0;
  const float top_p = g.top_p ? g.top_p[row] : 1.0f;
  const float min_p = g.min_p ? g.min_p[row] : 0.0f;
  const float u = g.u[row];
  const bool valid = temp >= 0.0f && top_p >= 0.0f && min_p >= 0.0f && min_p <= 1.0f && u >= 0.0f && u < 1.0f;
  auto finish = [&](int id, float logprob) {  // one thread
    g.token[row] = id < 0 ? -1 : g.off ? (int32_t)g.cand[(int64_t)o0 + id] : id;
    if (g.logprob) g.logprob[row] = logprob;
  };
  if (!valid && t == 0 && g.err) *g.err = 1;
  if (n == 0) {
    if (t == 0) finish(-1, -INFINITY);
    return;
  }

  // ---- the row's values at ids 4 slot + c (its last ones once more past it) ----
  auto load4 = [&](int slot) -> f4v {
    f4v v;
    if (n >= 4) {
      const int at = min(4 * slot, n - 4);
      if constexpr (BF16) {
        const h4u h = *(const h4u*)((const uint16_t*)base + at);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = bf16_to_f32(h[c]);
      } else {
        const f4u f = *(const f4u*)((const float*)base + at);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = f[c];
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int at = min(c, n - 1);
        v[c] = BF16 ? bf16_to_f32(((const uint16_t*)base)[at]) : ((const float*)base)[at];
      }
    }
    return v;
  };
  // Their order keys, 0 past the row.
  auto order4 = [&](int slot, f4v v, uint32_t (&k)[4]) {
    const int sh = n >= 4 ? max(0, 4 * slot - (n - 4)) : 0;
    const float v1 = v[1], v2 = v[2], v3 = v[3];
    v[0] = sh == 0 ? v[0] : sh == 1 ? v1 : sh == 2 ? v2 : v3;
    v[1] = sh == 0 ? v1 : sh == 1 ? v2 : v3;
    v[2] = sh == 0 ? v2 : v3;
#pragma unroll
    for (int c = 0; c < 4; ++c) k[c] = 4 * slot + c < n ? argmax_order(v[c]) : 0u;
  };
  const int nj = (n + 4 * T - 1) / (4 * T);
  // f(j, first id, keys of four ids) for every slot of this thread, from memory
  // with BATCH loads in flight.
  auto each_read = [&](auto&& f) {
    constexpr int BATCH = 8;
    for (int j0 = 0; j0 < nj; j0 += BATCH) {
      f4v v[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) v[b] = load4((j0 + b) * T + t);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (j0 + b >= nj) break;
        uint32_t k[4];
        order4((j0 + b) * T + t, v[b], k);
        f(j0 + b, 4 * ((j0 + b) * T + t), k);
      }
    }
  };
  auto each = [&](auto&& f) {
    if constexpr (IDS > 0) {
#pragma unroll 1
      for (int j = 0; j < nj; ++j) {
        const uint4 q = *(const uint4*)(L.key + 4 * (j * T + t));
        uint32_t k[4] = {q.x, q.y, q.z, q.w};
        f(j, 4 * (j * T + t), k);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < nj; ++j) {
        uint32_t k[4];
        order4(j * T + t, load4(j * T + t), k);
        f(j, 4 * (j * T + t), k);
      }
    }
  };

  // ---- the maximum, lowest id first ----
  {
    uint32_t bk = 0, bi = 0;
    each_read([&](int, int i, uint32_t (&k)[4]) {
      if constexpr (IDS > 0) *(uint4*)(L.key + i) = uint4{k[0], k[1], k[2], k[3]};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        bi = k[c] > bk ? (uint32_t)(i + c) : bi;
        bk = max(bk, k[c]);
      }
    });
    const uint64_t best = wave_max_u64(pair_of(bk, bi));
    if (lane == 0) L.wave[wave] = best;
  }
  wg_lds_barrier();
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) best = umax64(best, L.wave[i]);
  const uint32_t kmax = (uint32_t)(best >> 32);
  const int imax = (int)(0xFFFFFFFFu - (uint32_t)best);
  if (kmax <= kNothing) {  // only -inf and NaN
    if (t == 0) finish(0, -INFINITY);
    return;
  }
  if (!valid || temp == 0.0f || top_k == 1 || top_p == 0.0f) {
    if (t == 0) finish(imax, 0.0f);
    return;
  }
  const float lmax = key_logit(kmax);
  const double per_logit = 1.4426950408889634 / (double)temp;  // octaves of p
  const float bins_per_logit = (float)(per_logit * kBinsPerOctave);
  // log2 of p over the maximum's
  auto octave = [&](uint32_t key) -> double {
    return key == kmax ? 0.0 : ((double)key_logit(key) - (double)lmax) * per_logit;
  };
  // Monotone in the logit: fp32 subtraction and product are.
  auto bin_of = [&](uint32_t key) -> int {
    const float d = (lmax - key_logit(key)) * bins_per_logit;
    return key == kmax ? 0 : (int)fminf(d, (float)(kBins - 1));
  };

  // ---- the border of top-k and top-p ----
  uint64_t border = 0;  // kept: pairs at or above
  const bool by_k = top_k > 0 && top_k < n, by_p = top_p < 1.0f;
  if (by_k || by_p) {
    for (int b = t; b < kBins; b += T) {
      L.cnt[b] = 0;
      L.mass[b] = 0;
    }
    wg_lds_barrier();
    each([&](int, int, uint32_t (&k)[4]) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int b = bin_of(k[c]);
        if (k[c] > kNothing && b <= kLastBin) {
          lds_add(&L.cnt[b], 1u);
          if (by_p) lds_add(&L.mass[b], mass_of(octave(k[c])));
        }
      }
    });
    wg_lds_barrier();
    scan_bins<T>(L, L.cnt, L.mass);
    uint64_t total = L.mass[kBins - 1];

    // The pair at which the count (or mass) `need` is reached within bin b, and the mass up to it.
    auto refine = [&](int b, bool count, uint64_t need) {
      uint32_t cb = b ? L.cnt[b - 1] : 0u;
      uint64_t mb = b ? L.mass[b - 1] : 0ull;
      uint32_t in_bin = L.cnt[b] - cb;
      uint64_t lo = 0, hi = ~0ull;  // pairs looked at
      if (in_bin > kList) {
        each([&](int, int, uint32_t (&k)[4]) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (k[c] > kNothing && bin_of(k[c]) == b) {
              __hip_atomic_fetch_min(&L.lo, k[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
              __hip_atomic_fetch_max(&L.hi, k[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            }
        });
        wg_lds_barrier();
        lo = pair_of(L.lo, (uint32_t)(n - 1));
        hi = pair_of(L.hi, 0);
        while (in_bin > kList) {  // kBins parts of [lo, hi] at a time: a part of one pair at the end
          const uint64_t span = hi - lo;
          const int shift = max(0, 64 - 10 - __builtin_clzll(span | 1));
          for (int z = t; z < kBins; z += T) {
            L.zcnt[z] = 0;
            L.zmass[z] = 0;
          }
          wg_lds_barrier();
          each([&](int, int i, uint32_t (&k)[4]) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint64_t p = pair_of(k[c], (uint32_t)(i + c));
              if (p >= lo && p <= hi) {
                const int z = (int)((hi - p) >> shift);
                lds_add(&L.zcnt[z], 1u);
                if (by_p) lds_add(&L.zmass[z], mass_of(octave(k[c])));
              }
            }
          });
          wg_lds_barrier();
          scan_bins<T>(L, L.zcnt, L.zmass);
          const int z = count ? find_bin<T>(L, L.zcnt, (uint32_t)need - cb) : find_bin<T>(L, L.zmass, need - mb);
          in_bin = L.zcnt[z] - (z ? L.zcnt[z - 1] : 0u);
          cb += z ? L.zcnt[z - 1] : 0u;
          mb += z ? L.zmass[z - 1] : 0ull;
          hi -= (uint64_t)z << shift;
          lo = umax64(lo, hi - ((1ull << shift) - 1));
          wg_lds_barrier();  // the prefixes are read before the next histogram clears them
        }
      }
      // Every remaining pair and its mass, then each against all.
      each([&](int, int i, uint32_t (&k)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint64_t p = pair_of(k[c], (uint32_t)(i + c));
          if (k[c] > kNothing && p >= lo && p <= hi && bin_of(k[c]) == b) {
            const uint32_t at =
                __hip_atomic_fetch_add(&L.listed, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
            if (at < (uint32_t)kList) L.pair[at] = p;
          }
        }
      });
      wg_lds_barrier();
      const bool mine_in = t < (int)in_bin;
      const uint64_t mine = L.pair[mine_in ? t : 0], w = mine_in && by_p ? mass_of(octave((uint32_t)(mine >> 32))) : 0ull;
      if (mine_in) L.weight[t] = w;
      wg_lds_barrier();
      if (mine_in) {
        for (uint32_t i = 0; i < in_bin; ++i) {
          const bool before = L.pair[i] > mine;
          cb += before ? 1u : 0u;
          mb += before ? L.weight[i] : 0ull;
        }
        if (count ? cb + 1 == (uint32_t)need : mb < need && need <= mb + w) {
          L.border = mine;
          L.upto = mb + w;
        }
      }
      wg_lds_barrier();
      border = L.border;
      return L.upto;
    };

    if (by_k) {
      const int b = find_bin<T>(L, L.cnt, (uint32_t)top_k);
      if (b >= 0) total = refine(b, true, (uint64_t)top_k);  // else fewer than k ids have mass
    }
    if (by_p) {
      // The least mass that is at least top_p total: exact, top_p as a multiple of 2^-64.
      const uint64_t pf = (uint64_t)ldexp((double)top_p, 64);
      uint64_t need = __umul64hi(total, pf);
      need += total * pf != 0 ? 1 : 0;
      need = need ? need : 1;
      const int b = find_bin<T>(L, L.mass, need);
      if (b >= 0) refine(b, false, need);
    }
  }

  // ---- the draw: kept mass of every 256 consecutive ids, then one id ----
  const double min_octave = min_p > 0.0f ? log2((double)min_p) : -INFINITY;
  auto kept_mass = [&](uint32_t key, int id) -> uint64_t {
    if (key <= kNothing || pair_of(key, (uint32_t)id) < border) return 0;
    const double y = octave(key);
    return y >= min_octave ? mass_of(y) : 0ull;
  };
  wg_lds_barrier();
  for (int b = t; b < kBins; b += T) {
    L.cnt[b] = 0;
    L.zmass[b] = 0;
  }
  wg_lds_barrier();
  each([&](int j, int i, uint32_t (&k)[4]) {
    uint64_t m = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) m += kept_mass(k[c], i + c);
    if (__any(m != 0)) {
      const uint64_t s = wave_scan(m);
      if (lane == 63) lds_add(&L.zmass[(j * NW + wave) / GROUP], s);
    }
  });
  wg_lds_barrier();
  scan_bins<T>(L, L.cnt, L.zmass);
  const uint64_t total = L.zmass[kBins - 1];
  // first running mass > floor(u total), u as a multiple of 2^-32
  const uint64_t need = __umul64hi(total, (uint64_t)(uint32_t)(u * 0x1p32f) << 32) + 1;
  const int seg = find_bin<T>(L, L.zmass, need);
  if (wave == 0) {
    uint64_t before = seg ? L.zmass[seg - 1] : 0ull;
    for (int part = 0; part < GROUP; ++part) {  // 256 ids at a time
      const int slot = (seg * GROUP + part) * 64 + lane;
      uint32_t k[4];
      order4(slot, load4(slot), k);
      uint64_t m[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) m[c] = kept_mass(k[c], 4 * slot + c);
      const uint64_t own = m[0] + m[1] + m[2] + m[3], upto = wave_scan(own);
      uint64_t run = before + upto - own;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (run < need && need <= run + m[c])
          finish(4 * slot + c, (float)(octave(k[c]) * 0.6931471805599453 - log(ldexp((double)total, -kMassBits))));
        run += m[c];
      }
      before = lane_u64(run, 63);
    }
  }
}

template <int T, int IDS>
hipError_t launch(const SampleArgs& g, hipStream_t s) {
  auto kern = g.bf16 ? k_sample<T, IDS, true> : k_sample<T, IDS, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)g.rows), dim3(T), 0, s, g);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const SampleArgs& g, hipStream_t s) {
  if (!g.logits || !g.u || !g.token || g.V <= 0 || g.V > kSampleMaxIds || g.rows < 0 || (g.off && !g.cand))
    return hipErrorInvalidValue;
  if (g.rows == 0) return hipSuccess;
  if (g.V <= 4096) return launch<256, 4096>(g, s);
  if (g.V <= 32768) return launch<1024, 32768>(g, s);
  return launch<1024, 0>(g, s);
}

}  // namespace mh
