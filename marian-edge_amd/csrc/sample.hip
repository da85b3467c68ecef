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

constexpr uint32_t kNothing = 0x007FFFFFu;     // argmax_order of -inf: ids that cannot be drawn
constexpr int kBins = 2048;
constexpr int kBinsPerOctave = 32;             // of p, in the histograms over log2 p
constexpr int kLastBin = 46 * kBinsPerOctave;  // ids past it have no mass
constexpr int kMassBits = 44;                  // mass of the row's maximum
constexpr int kList = 256;                     // ids compared pairwise

// 2^(j/32)
__device__ const double kExp2[32] = {
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0,
    0x1.172b83c7d517bp+0, 0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0,
    0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0, 0x1.3dea64c123422p+0, 0x1.44e086061892dp+0,
    0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0, 0x1.6247eb03a5585p+0,
    0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0,
    0x1.ae89f995ad3adp+0, 0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0,
    0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0, 0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0,
};

// log2 of p over the maximum's (at least -60; NaN counts as that) in steps of
// 1/32, and what is left, |rest| <= 1/64.  Adding 1.5 * 2^47 rounds to a step and
// leaves their number in the low word: conversion and rounding instructions take
// four times an addition's time.  steps is monotone in the logit, so -steps is the
// histogram's bin.
struct Octave {
  int steps;
  double rest;
};
__device__ __forceinline__ Octave octave_steps(double y) {
  y = fmax(y, -60.0);
  const double t = y + 0x1.8p47;
  return {(int)(uint32_t)__double_as_longlong(t), y - (t - 0x1.8p47)};
}
// round(2^44 2^y): a table of 2^(j/32), a polynomial of degree 4 (interpolated at
// Chebyshev nodes, relative error 8e-14), the power of two added to the exponent,
// and an addition of 2^52, which leaves the integer in the low 52 bits.  The
// table's entries fill every LDS bank once: no lane waits for another.
__device__ __forceinline__ uint64_t mass_of_steps(Octave o, const double* exp2) {
  double p = 0x1.3b2b1bee88b09p-7;
  p = __builtin_fma(p, o.rest, 0x1.c6b167e571135p-5);
  p = __builtin_fma(p, o.rest, 0x1.ebfbdff8131c3p-3);
  p = __builtin_fma(p, o.rest, 0x1.62e42fef6d01ap-1);
  p = __builtin_fma(p, o.rest, 0x1.0000000000000p+0) * exp2[o.steps & 31];
  const int e = (o.steps >> 5) + kMassBits;  // -16 to 44
  p = __hiloint2double(__double2hiint(p) + e * (1 << 20), __double2loint(p));
  return (uint64_t)__double_as_longlong(p + 0x1p52) & 0x000FFFFFFFFFFFFFull;
}

// DPP move that leaves 0 in the lanes it does not write.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp0(uint64_t v) {
  return ((uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32) | dpp0<CTRL, ROWS>((uint32_t)v);
}
// Inclusive prefix sums over the wave.
template <class V>
__device__ __forceinline__ V wave_scan(V v) {
  v += dpp0<0x111, 0xF>(v);  // row_shr:1
  v += dpp0<0x112, 0xF>(v);  // row_shr:2
  v += dpp0<0x114, 0xF>(v);  // row_shr:4
  v += dpp0<0x118, 0xF>(v);  // row_shr:8
  v += dpp0<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
  v += dpp0<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
  return v;
}
// wave_scan of masses in 12 additions, the lanes moved by the additions themselves
// (the compiler moves them first: 36 instructions).  A lane's result is read by the
// next step two instructions later, as the hardware asks.
__device__ __forceinline__ uint64_t wave_scan_mass(uint64_t v) {
  uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
#define STEP(CTRL)                                                                     \
  "s_nop 1\n\tv_add_co_u32_dpp %0, vcc, %0, %0 " CTRL                                  \
  " bank_mask:0xf bound_ctrl:0\n\ts_nop 1\n\tv_addc_co_u32_dpp %1, vcc, %1, %1, vcc " \
  CTRL " bank_mask:0xf bound_ctrl:0\n\t"
  asm(STEP("row_shr:1 row_mask:0xf") STEP("row_shr:2 row_mask:0xf") STEP("row_shr:4 row_mask:0xf")
          STEP("row_shr:8 row_mask:0xf") STEP("row_bcast:15 row_mask:0xa") STEP("row_bcast:31 row_mask:0xc")
              "s_nop 1"
      : "+v"(lo), "+v"(hi)
      :
      : "vcc");
#undef STEP
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

template <class V>
__device__ __forceinline__ V lds_add(V* p, V v) {
  return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}

// Ids in descending order of this pair: logit, then ascending id.
__device__ __forceinline__ uint64_t pair_of(float v, uint32_t id) {
  return ((uint64_t)argmax_order(v) << 32) | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ float order_logit(uint32_t k) {  // inverse of argmax_order
  return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ float pair_logit(uint64_t p) { return order_logit((uint32_t)(p >> 32)); }
__device__ __forceinline__ int pair_id(uint64_t p) { return (int)(0xFFFFFFFFu - (uint32_t)p); }

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));

template <int T, int IDS>
struct SampleLds {
  static constexpr int NW = T / 64, SEGS = (IDS ? IDS : kSampleMaxIds) / 256;
  float val[IDS ? IDS : 4];  // the row, each value written and read by one thread
  union {
    uint64_t mass[kBins];
    uint32_t cnt[kBins];
  };
  double exp2[32];
  uint64_t seg[SEGS];  // kept mass of every 256 consecutive ids
  uint64_t pair[kList], weight[kList], before[kList];
  uint64_t wsum[NW];
  float wmax[NW];
  int found, best;
  uint32_t listed;
  uint64_t lo, hi, found_before, border;
};

// The first of h's kBins at which the running sum reaches need(sum of all), and
// the running sum before it; bin -1: none.  Called with h complete (a barrier
// before); on return h may be written again.
struct Found {
  int bin;
  uint64_t before, total;
};
template <int T, class Lds, class V, class Need>
__device__ __forceinline__ Found locate(Lds& L, const V* h, Need&& need_of) {
  constexpr int B = kBins / T, NW = T / 64;
  const int t = threadIdx.x, w = t >> 6;
  V c[B];
#pragma unroll
  for (int i = 0; i < B; ++i) c[i] = h[t * B + i] + (i ? c[i - 1] : (V)0);
  uint64_t s = wave_scan(c[B - 1]);
  if ((t & 63) == 63) L.wsum[w] = s;
  if (t == 0) {
    L.found = -1;
    L.listed = 0;
    L.lo = ~0ull;
    L.hi = 0;
  }
  wg_lds_barrier();
  s -= c[B - 1];
  uint64_t total = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    const uint64_t v = L.wsum[i];
    total += v;
    s += i < w ? v : 0ull;
  }
  const uint64_t need = need_of(total);
#pragma unroll
  for (int i = 0; i < B; ++i) {
    const uint64_t before = s + (i ? c[i - 1] : (V)0);
    if (before < need && need <= s + c[i]) {
      L.found = t * B + i;
      L.found_before = before;
    }
  }
  wg_lds_barrier();
  return {__builtin_amdgcn_readfirstlane(L.found), L.found_before, total};
}

// Sum over the workgroup; two barriers.
template <int T, class Lds>
__device__ __forceinline__ uint64_t block_sum(Lds& L, uint64_t v) {
  v = wave_scan(v);
  wg_lds_barrier();  // earlier sums are read
  if ((threadIdx.x & 63) == 63) L.wsum[threadIdx.x >> 6] = v;
  wg_lds_barrier();
  uint64_t s = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) s += L.wsum[i];
  return s;
}

// One workgroup of T threads per row.  Thread t holds ids 4(jT + t) + c, so that
// a wave's 256 values of one j are consecutive ids: the final draw sums those,
// finds the group that the number falls into, and one wave scans its 256.  A row
// of up to IDS ids is read from memory once and kept in LDS, each thread its own
// values; IDS = 0: each pass reads memory again.  One compute unit works on a row,
// so instructions per id and pass are what bounds it, and the passes are rolled
// loops: unrolled (values and masses in registers) they outgrow the instruction
// cache and took longer.
//
// Few ids to draw from (at most kList ids in the row, or a top-k of which at most
// kList ids can be part): all of them in a list, compared pairwise.  The k-th
// largest of the threads' maxima is a lower bound of the k-th largest id, so a
// histogram of T values finds the ids that the list needs.
//
// Otherwise the border of top-k, then of top-p among what is left: a histogram over
// log2 p (of counts, or of masses), the bin where the count or mass is reached, then
// every id of that bin against every other.  A bin of more than kList ids (many
// equal logits) is cut again by (logit, id) pairs, kBins ways a time, until few
// are left.
template <int T, int IDS, bool BF16>
__global__ __launch_bounds__(T) void k_sample(SampleArgs g) {
  constexpr int NW = T / 64, NJ = IDS / (4 * T);  // slots of four ids per thread
  static_assert(NJ * 4 * T == IDS && T >= kList && kBins % T == 0, "whole slots");
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

  // ---- the row's values at ids 4 slot + c: -inf for NaN and past the row ----
  bool only_inf = false;  // the maximum is infinite: those ids alone, as if of logit 0
  auto load4 = [&](int slot) -> f4v {  // as stored; the row's last values once more past it
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
  auto clean4 = [&](int slot, f4v v) -> f4v {
    if (__any(4 * slot + 4 > n)) {  // the row's end is inside or before this slot
      const int sh = n >= 4 ? max(0, 4 * slot - (n - 4)) : 0;
      const float v1 = v[1], v2 = v[2], v3 = v[3];
      v[0] = sh == 0 ? v[0] : sh == 1 ? v1 : sh == 2 ? v2 : v3;
      v[1] = sh == 0 ? v1 : sh == 1 ? v2 : v3;
      v[2] = sh == 0 ? v2 : v3;
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = 4 * slot + c < n ? v[c] : -INFINITY;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = fmaxf(v[c], -INFINITY);
    if (only_inf) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = v[c] == INFINITY ? 0.0f : -INFINITY;
    }
    return v;
  };
  const int nj = (n + 4 * T - 1) / (4 * T);
  // f(j, first id, four values) for every slot of this thread, from memory with
  // BATCH loads in flight.
  auto each_read = [&](auto&& f) {
    constexpr int BATCH = IDS ? NJ : 4;
    for (int j0 = 0; j0 < nj; j0 += BATCH) {
      f4v v[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) v[b] = load4((j0 + b) * T + t);
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (j0 + b >= nj) break;
        f(j0 + b, 4 * ((j0 + b) * T + t), clean4((j0 + b) * T + t, v[b]));
      }
    }
  };
  auto each = [&](auto&& f) {
    if constexpr (IDS > 0) {
#pragma unroll 1
      for (int j = 0; j < nj; ++j) f(j, 4 * (j * T + t), *(const f4v*)(L.val + 4 * (j * T + t)));
    } else {
      each_read(f);
    }
  };

  // ---- the maximum ----
  float tmax = -INFINITY;  // this thread's
  each_read([&](int, int i, f4v v) {
    if constexpr (IDS > 0) *(f4v*)(L.val + i) = v;
    tmax = fmaxf(fmaxf(fmaxf(tmax, v[0]), fmaxf(v[1], v[2])), v[3]);
  });
  {
    const float m = wave_max(tmax);
    if (lane == 0) L.wmax[wave] = m;
  }
  if (t == 0) L.best = 0x7FFFFFFF;
  if (t < 32) L.exp2[t] = kExp2[t];
  for (int b = t; b < kBins; b += T) L.mass[b] = 0;
  wg_lds_barrier();
  float lmax = L.wmax[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) lmax = fmaxf(lmax, L.wmax[i]);
  if (lmax == -INFINITY) {  // only -inf and NaN
    if (t == 0) finish(0, -INFINITY);
    return;
  }
  if (!valid || temp == 0.0f || top_k == 1 || top_p == 0.0f) {  // the maximum's lowest id
    int best = 0x7FFFFFFF;
    if (tmax == lmax)
      each([&](int, int i, f4v v) {
#pragma unroll
        for (int c = 3; c >= 0; --c) best = v[c] == lmax ? min(best, i + c) : best;
      });
    if (best != 0x7FFFFFFF)
      __hip_atomic_fetch_min(&L.best, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    wg_lds_barrier();
    if (t == 0) finish(L.best, 0.0f);
    return;
  }
  if (lmax == INFINITY) {
    only_inf = true;
    tmax = tmax == INFINITY ? 0.0f : -INFINITY;
    lmax = 0.0f;
    if constexpr (IDS > 0)
      each_read([&](int, int i, f4v v) { *(f4v*)(L.val + i) = v; });
  }
  const double per_logit = 1.4426950408889634 / (double)temp;  // octaves of p
  auto octave = [&](float v) -> double { return ((double)v - (double)lmax) * per_logit; };
  auto mass_of = [&](float v) -> uint64_t { return mass_of_steps(octave_steps(octave(v)), L.exp2); };
  auto bin_of = [&](float v) -> int { return -octave_steps(octave(v)).steps; };
  // Values of bins [first, last] lie within [least_of(last), most_of(first)]: a
  // cheap test before the exact one (a tenth of a bin and rounding errors to spare).
  const float logits_per_bin = 1.0f / (float)(per_logit * kBinsPerOctave), slack = fabsf(lmax) * 0x1p-21f;
  auto least_of = [&](int b) -> float { return lmax - ((float)b + 0.6f) * logits_per_bin - slack; };
  auto most_of = [&](int b) -> float { return lmax - ((float)b - 0.6f) * logits_per_bin + slack; };
  // The least mass that is at least top_p of the whole: exact, top_p as a multiple of 2^-64.
  auto need_p = [&](uint64_t total) -> uint64_t {
    const uint64_t part = (uint64_t)ldexp((double)top_p, 64);
    const uint64_t need = __umul64hi(total, part) + (total * part != 0 ? 1 : 0);
    return need ? need : 1ull;
  };
  // First running mass > floor(u total), u as a multiple of 2^-32.
  auto need_u = [&](uint64_t total) -> uint64_t {
    return __umul64hi(total, (uint64_t)(uint32_t)(u * 0x1p32f) << 32) + 1;
  };
  auto share = [&](float v, uint64_t total) -> float {
    return (float)(octave(v) * 0.6931471805599453 - log(ldexp((double)total, -kMassBits)));
  };
  const bool by_k = top_k > 0 && top_k < n, by_p = top_p < 1.0f;
  // The least logit that min-p keeps, by its order key: steps of 1, 2, 4 ... from
  // where rounding apart it should be, then halves of what the last one jumped over.
  float least_v = -INFINITY;
  if (min_p > 0.0f) {
    const double least = log2((double)min_p);
    auto in = [&](int64_t k) { return octave(order_logit((uint32_t)k)) >= least; };
    int64_t lo = kNothing, hi = argmax_order(lmax);  // out, in
    const int64_t k = min(max((int64_t)argmax_order((float)((double)lmax + least / per_logit)), lo + 1), hi);
    int64_t step = 1;
    if (in(k)) {
      hi = k;
      for (; hi - lo > step && in(hi - step); step *= 2) hi -= step;
      lo = max(lo, hi - step);
    } else {
      lo = k;
      for (; hi - lo > step && !in(lo + step); step *= 2) lo += step;
      hi = min(hi, lo + step);
    }
    while (hi - lo > 1) {
      const int64_t mid = (lo + hi) / 2;
      (in(mid) ? hi : lo) = mid;
    }
    least_v = order_logit((uint32_t)hi);
  }

  // Adds ids of bins [first, last] with pairs in [lo, hi] to the list, as long as it has room.
  auto gather = [&](int first, int last, uint64_t lo, uint64_t hi, bool range, auto&& also) {
    const float least = least_of(last), most = first ? most_of(first) : INFINITY;
    each([&](int, int i, f4v v) {
      bool in[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) in[c] = (v[c] >= least) & (v[c] <= most);
      if (!__any((in[0] | in[1]) | (in[2] | in[3]))) return;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (!in[c]) continue;
        const int b = bin_of(v[c]);
        if (b < first || b > last || !also(v[c], i + c)) continue;
        const uint64_t p = pair_of(v[c], (uint32_t)(i + c));
        if (p < lo || p > hi) continue;
        const uint32_t at = lds_add(&L.listed, 1u);
        if (at < (uint32_t)kList) L.pair[at] = p;
        if (range) {
          __hip_atomic_fetch_min(&L.lo, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          __hip_atomic_fetch_max(&L.hi, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
    });
    wg_lds_barrier();
  };
  // For the list's entry of this thread's place (t % kList): the sum of weight over
  // the entries that come before it, in L.before.  T / kList groups of threads share
  // the entries.  The weights are complete but for a barrier, and the sums on return.
  auto sum_before = [&](uint32_t listed, auto&& comes_before) {
    if (t < kList) L.before[t] = 0;
    wg_lds_barrier();
    const uint32_t at = t % kList;
    if (at < listed) {
      uint64_t s = 0;
#pragma unroll 4
      for (uint32_t i = t / kList; i < listed; i += T / kList) s += comes_before(L.pair[i]) ? L.weight[i] : 0ull;
      if (s) lds_add(&L.before[at], s);
    }
    wg_lds_barrier();
  };

  // ---- few ids: a list of them ----
  bool few = n <= kList;
  if (few || (by_k && top_k <= kList * 3 / 4)) {
    int last = kLastBin;
    if (few) {
      if (t == 0) L.listed = 0;
      wg_lds_barrier();
    } else {
      const int b = bin_of(tmax);
      if (b <= kLastBin) lds_add(&L.cnt[b], 1u);
      wg_lds_barrier();
      const Found f = locate<T>(L, L.cnt, [&](uint64_t) { return (uint64_t)top_k; });
      for (int z = t; z < kBins; z += T) L.mass[z] = 0;
      few = f.bin >= 0;
      last = f.bin;
    }
    if (few) {
      gather(0, last, 0, ~0ull, false, [](float, int) { return true; });
      few = L.listed <= (uint32_t)kList;
    }
    if (few) {
      const uint32_t listed = L.listed, at = t % kList;
      const uint64_t mine = L.pair[min(at, listed - 1)];
      const bool own = t < (int)listed;  // one thread per entry
      const float v = pair_logit(mine);
      const uint64_t m = own ? mass_of(v) : 0ull;
      bool keep = own;
      if (by_k) {
        if (own) L.weight[t] = 1;
        sum_before(listed, [&](uint64_t p) { return p > mine; });
        keep = own && L.before[at] < (uint64_t)top_k;
        wg_lds_barrier();
      }
      if (by_p) {
        if (own) L.weight[t] = keep ? m : 0ull;
        const uint64_t need = need_p(block_sum<T>(L, keep ? m : 0ull));
        sum_before(listed, [&](uint64_t p) { return p > mine; });
        keep = keep && L.before[at] < need;
        wg_lds_barrier();
      }
      keep = keep && v >= least_v;
      if (own) L.weight[t] = keep ? m : 0ull;
      const uint64_t total = block_sum<T>(L, keep ? m : 0ull), need = need_u(total);
      sum_before(listed, [&](uint64_t p) { return (uint32_t)p > (uint32_t)mine; });  // lower ids
      if (keep && L.before[at] < need && need <= L.before[at] + m) finish(pair_id(mine), share(v, total));
      return;
    }
    wg_lds_barrier();
  }

  // ---- the borders: ids kept are those at or before (border_v, border_id) ----
  float border_v = -INFINITY;
  int border_id = 0x7FFFFFFF;
  auto kept = [&](float v, int id) -> bool { return (v > border_v) | ((v == border_v) & (id <= border_id)); };
  // f(j, octaves and masses of the kept ids), for every slot; slots without any are left out
  auto each_mass = [&](auto&& f) {
    const bool all = border_v == -INFINITY;
    each([&](int j, int i, f4v v) {
      if (!all) {
        bool tie = false;
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          tie |= v[c] == border_v;
          v[c] = v[c] >= border_v ? v[c] : -INFINITY;
          top = fmaxf(top, v[c]);
        }
        if (!__any(top > -INFINITY)) return;
        if (__any(tie)) {
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = v[c] == border_v && i + c > border_id ? -INFINITY : v[c];
        }
      }
      Octave o[4];
      uint64_t m[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        o[c] = octave_steps(octave(v[c]));
        m[c] = mass_of_steps(o[c], L.exp2);
      }
      f(j, o, m);
    });
  };

  // top-k, then top-p: one piece of code for both.
#pragma unroll 1
  for (int stage = by_k ? 0 : 1; stage < (by_p ? 2 : 1); ++stage) {
    const bool count = stage == 0;
    auto need_of = [&](uint64_t total) { return count ? (uint64_t)top_k : need_p(total); };
    Found f;
    if (count) {
      each([&](int, int, f4v v) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int b = bin_of(v[c]);
          if (b <= kLastBin) lds_add(&L.cnt[b], 1u);
        }
      });
      wg_lds_barrier();
      f = locate<T>(L, L.cnt, need_of);
    } else {
      each_mass([&](int, const Octave (&o)[4], const uint64_t (&m)[4]) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (m[c]) lds_add(&L.mass[-o[c].steps], m[c]);
      });
      wg_lds_barrier();
      f = locate<T>(L, L.mass, need_of);
    }
    for (int b = t; b < kBins; b += T) L.mass[b] = 0;  // for the next histogram
    if (f.bin < 0) {  // fewer ids with mass than the count asks for
      wg_lds_barrier();
      continue;
    }
    uint64_t need = need_of(f.total) - f.before;  // within the bin
    auto weigh = [&](float v) -> uint64_t { return count ? 1ull : mass_of(v); };
    gather(f.bin, f.bin, 0, ~0ull, true, kept);
    if (L.listed > (uint32_t)kList) {
      uint64_t lo = L.lo, hi = L.hi;
      do {  // kBins parts of [lo, hi] at a time: a part of one pair at the end
        const uint64_t span = hi - lo;
        const int shift = max(0, 64 - 11 - __builtin_clzll(span | 1));
        each([&](int, int i, f4v v) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint64_t p = pair_of(v[c], (uint32_t)(i + c));
            if (p >= lo && p <= hi) lds_add(&L.mass[(hi - p) >> shift], weigh(v[c]));
          }
        });
        wg_lds_barrier();
        const Found z = locate<T>(L, L.mass, [&](uint64_t) { return need; });
        need -= z.before;
        hi -= (uint64_t)z.bin << shift;
        lo = umax64(lo, hi - ((1ull << shift) - 1));
        for (int b = t; b < kBins; b += T) L.mass[b] = 0;
        gather(f.bin, f.bin, lo, hi, false, kept);
      } while (L.listed > (uint32_t)kList);
    }
    const uint32_t listed = L.listed, at = t % kList;
    const uint64_t mine = L.pair[min(at, listed - 1)];
    uint64_t w = 0;
    if (t < (int)listed) {
      w = weigh(pair_logit(mine));
      L.weight[t] = w;
    }
    sum_before(listed, [&](uint64_t p) { return p > mine; });
    if (t < (int)listed && L.before[at] < need && need <= L.before[at] + w) L.border = mine;
    wg_lds_barrier();
    border_v = pair_logit(L.border);
    border_id = pair_id(L.border);
  }

  // ---- the draw: kept mass of every 256 consecutive ids, then one id ----
  if (least_v > border_v) {
    border_v = least_v;
    border_id = 0x7FFFFFFF;
  }
  for (int b = t; b < (IDS ? nj * NW : kBins); b += T) L.seg[b] = 0;
  wg_lds_barrier();
  each_mass([&](int j, const Octave (&)[4], const uint64_t (&m)[4]) {
    const uint64_t s = wave_scan_mass((m[0] + m[1]) + (m[2] + m[3]));
    if (lane == 63) L.seg[j * NW + wave] = s;
  });
  wg_lds_barrier();
  int seg = -1;
  uint64_t before = 0, total;
  if constexpr (IDS > 0) {  // each wave finds the group by itself
    constexpr int PER = (SampleLds<T, IDS>::SEGS + 63) / 64;
    const int segs = nj * NW;
    uint64_t c[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int s = lane * PER + k;
      c[k] = (s < segs ? L.seg[s] : 0ull) + (k ? c[k - 1] : 0ull);
    }
    const uint64_t upto = wave_scan(c[PER - 1]);
    total = lane_u64(upto, 63);
    const uint64_t need = need_u(total);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const uint64_t b = upto - c[PER - 1] + (k ? c[k - 1] : 0ull);
      const uint64_t who = __ballot(b < need && need <= upto - c[PER - 1] + c[k]);
      if (who) {
        seg = __builtin_ctzll(who) * PER + k;
        before = lane_u64(b, __builtin_ctzll(who));
      }
    }
  } else {
    const Found f = locate<T>(L, L.seg, need_u);
    seg = f.bin;
    before = f.before;
    total = f.total;
  }
  if (wave == seg % NW) {  // the wave that holds the group
    const int slot = seg * 64 + lane;
    f4v v;
    if constexpr (IDS > 0)
      v = *(const f4v*)(L.val + 4 * slot);
    else
      v = clean4(slot, load4(slot));
    uint64_t m[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      v[c] = kept(v[c], 4 * slot + c) ? v[c] : -INFINITY;
      m[c] = mass_of(v[c]);
    }
    const uint64_t own = m[0] + m[1] + m[2] + m[3], need = need_u(total);
    uint64_t run = before + wave_scan(own) - own;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (run < need && need <= run + m[c]) finish(4 * slot + c, share(v[c], total));
      run += m[c];
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
