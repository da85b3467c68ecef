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
// Mass is an integer, at most 2 from 2^44 exp((l - max) / T) and 2^44 for the maximum:
// sums of up to 2^19 of them are exact in 64 bits, so they do not depend on the order in
// which lanes and atomics add them, and a row's result is the same whatever the launch
// shape.  The exponential is 2^y by a polynomial in 64 bits: a drawn number
// close to a border of the running mass needs more than fp32's 24 bits (32000
// borders at 2^-24 each would misplace one row in several hundred).
#include "device_common.h"
#include "kernels.h"
#include "ref_expf.h"

#include <algorithm>

namespace mh {
namespace {

constexpr uint32_t kNothing = 0x007FFFFFu;     // argmax_order of -inf: ids that cannot be drawn
constexpr int kBins = 2048;
constexpr int kBinsPerOctave = 32;             // of p, in the histograms over log2 p
constexpr int kLastBin = 46 * kBinsPerOctave;  // ids past it have no mass
constexpr int kMassBits = 44;                  // mass of the row's maximum
constexpr int kList = 256;                     // ids put in order at once

// The bits of 2^(j/32) less j * 2^47: with kMassBits << 52 and n * 2^47 added (n % 32 = j)
// those of 2^(kMassBits + n/32).
__constant__ uint64_t kSampleExp2Tab[32] = {MH_EXP2_TABLE_32};

// Of a logit d below the maximum (a double): log2 of p over the maximum's, at
// least -60, in steps of 1/32, and what is left, |rest| <= 1/64.  Adding 1.5 * 2^47
// rounds to a step and leaves their number in the low word: conversion and rounding
// instructions take four times an addition's time.  steps is monotone in the logit, so
// -steps is the histogram's bin.
struct Octaves {
  double per_logit, least;  // steps' scale (not 0, so that -inf stays below the rest); the d of -60
};
struct Octave {
  int steps;
  double rest;
};
__device__ __forceinline__ Octave octave_steps(double d, const Octaves& o) {
  d = fmax(d, o.least);
  const double t = __builtin_fma(d, o.per_logit, 0x1.8p47);
  return {(int)(uint32_t)__double_as_longlong(t), __builtin_fma(d, o.per_logit, -(t - 0x1.8p47))};
}
// 2^44 2^y as an integer, + kMassBias, by a table (P. T. P. Tang's method, ACM TOMS 15,
// 1989): 2^(j/32), to whose exponent the whole octaves are added, times a polynomial of
// degree 4 (interpolated at Chebyshev nodes, relative error 8e-14, which is 1.4 of 2^44),
// and 2^52 added to the product, which rounds it and leaves the integer in the low 52
// bits.  The table's entries fill every LDS bank once: no lane waits for another.
constexpr uint64_t kMassBias = 0x4330000000000000ull;  // of 2^52
__device__ __forceinline__ uint64_t biased_mass(Octave o, const uint64_t* exp2) {
  const uint64_t e = exp2[o.steps & 31];
  double p = __builtin_fma(0x1.3b2b1bee88b09p-7, o.rest, 0x1.c6b167e571135p-5);
  p = __builtin_fma(p, o.rest, 0x1.ebfbdff8131c3p-3);
  p = __builtin_fma(p, o.rest, 0x1.62e42fef6d01ap-1);
  p = __builtin_fma(p, o.rest, 0x1.0000000000000p+0);
  const double scale = __hiloint2double((int)((uint32_t)(e >> 32) + ((uint32_t)o.steps << 15)), (int)(uint32_t)e);
  return (uint64_t)__double_as_longlong(__builtin_fma(p, scale, 0x1p52));
}
__device__ __forceinline__ uint64_t mass_of_steps(Octave o, const uint64_t* exp2) {
  return biased_mass(o, exp2) & 0x000FFFFFFFFFFFFFull;
}

// Inclusive prefix sums over the wave, in 12 additions that move the lanes
// themselves (the compiler moves them first: 36 instructions).  The hardware asks for
// two instructions between a lane's result and the next step's read of it.
__device__ __forceinline__ uint64_t wave_scan_mass(uint64_t v) {
  uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
#define STEP(CTRL)                                                                           \
  "v_add_co_u32_dpp %0, vcc, %0, %0 " CTRL " bank_mask:0xf bound_ctrl:0\n\t"                 \
  "v_addc_co_u32_dpp %1, vcc, %1, %1, vcc " CTRL " bank_mask:0xf bound_ctrl:0\n\ts_nop 0\n\t"
  asm("s_nop 1\n\t" STEP("row_shr:1 row_mask:0xf") STEP("row_shr:2 row_mask:0xf") STEP("row_shr:4 row_mask:0xf")
          STEP("row_shr:8 row_mask:0xf") STEP("row_bcast:15 row_mask:0xa") STEP("row_bcast:31 row_mask:0xc")
              "s_nop 0"
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
  // Ids of a top-k that a list is too short for: one per thread where a thread holds many.
  static constexpr int PART = T == 1024 ? T : 0;
  static constexpr int NW = T / 64, SEGS = (IDS ? IDS : kSampleMaxIds) / 256;
  float val[IDS ? IDS : 4];  // the row, each value written and read by one thread
  uint64_t hist[kBins];      // masses or counts
  uint64_t exp2[32];
  uint64_t seg[SEGS];  // kept mass of every 256 consecutive ids
  __attribute__((aligned(16))) uint64_t entry[kList];   // the list's pairs
  __attribute__((aligned(16))) uint64_t sorted[kList];  // in order
  uint32_t ahead[kList];                                // of an entry: how many come before it; zero between uses
  uint64_t part[PART ? PART : 1];  // pairs
  uint32_t kept[kList / 64];
  uint64_t wsum[NW];
  float wmax[NW];
  int found, best;
  uint32_t listed;
  uint64_t lo, hi, found_before;
  uint32_t border;
};

// The first of the kBins of L.hist at which the running sum reaches need(sum of
// all), and the running sum before it; bin -1: none.  Called with the histogram
// complete but for a barrier; it is zero again on return, but for a barrier.
struct Found {
  int bin;
  uint64_t before, total;
};
template <int T, class Lds, class Need>
__device__ __forceinline__ Found locate(Lds& L, Need&& need_of) {
  constexpr int B = kBins / T, NW = T / 64;
  const int t = threadIdx.x, w = t >> 6;
  wg_lds_barrier();
  uint64_t c[B];
#pragma unroll
  for (int i = 0; i < B; ++i) {
    c[i] = L.hist[t * B + i] + (i ? c[i - 1] : 0ull);
    L.hist[t * B + i] = 0;
  }
  uint64_t s = wave_scan_mass(c[B - 1]);
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
    const uint64_t before = s + (i ? c[i - 1] : 0ull);
    if (before < need && need <= s + c[i]) {
      L.found = t * B + i;
      L.found_before = before;
    }
  }
  wg_lds_barrier();
  return {__builtin_amdgcn_readfirstlane(L.found), L.found_before, total};
}

// One workgroup of T threads per row.  Thread t holds ids 4(jT + t) + c, so that
// a wave's 256 values of one j (a slot) are consecutive ids: the final draw sums
// those, finds the group that the number falls into, and one wave scans its 256.
// A row of up to IDS ids is read from memory once and kept in LDS, each thread its
// own values; IDS = 0: each pass reads memory again.  One compute unit works on a
// row, so instructions per id and pass are what bounds it, and, as every
// instruction is fetched once per row, the size of the code: the passes are rolled
// loops and the stages below share one piece of code (unrolled, with values
// and masses in registers, they took half as long again).  32000 fp32 ids, one row, a
// nucleus: 20 us, of which the maximum 2, the histogram of masses 7, the bin's ids 3, the
// draw's masses 6.5; the row itself would be read in 0.03 us by the whole chip.
//
// Few ids to draw from (at most kList ids in the row, or a top-k of which at most
// kList ids can be part): all of them in a list, put in order by counting the entries
// ahead of each; every setting is then a prefix sum over the threads (a pass of
// comparisons per setting took four times as long: 453 lists of up to 215 ids,
// mixed settings, 44 us then and 12 now).  The k-th largest of the threads'
// maxima is a lower bound of the k-th largest id, so a histogram of T values finds
// the ids that the list needs.
//
// Otherwise the border of top-k, then of top-p among what is left: a histogram over
// log2 p (of counts, or of masses), the bin where the count or mass is reached, then
// that bin's ids in order.  A bin of more than kList ids (many equal logits) is cut
// again by (logit, id) pairs, kBins ways a time, until few are left.  The ids of a top-k
// of up to PART go on by themselves, one a thread, in what follows (us: 64 rows of 32000
// ids, mixed settings, 32.6 without and 27.8 so, 7 of 108601 69 and 50; a nucleus' ids,
// whose number is not known before, cost more to gather than that saves: 24.0 and 27.8).
enum Stage { LIST_ALL, LIST_TOP, BORDER_K, BORDER_P, DRAW, DRAWN };

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

  // ---- the row's values: -inf for NaN and past the row ----
  // Of this wave's slots, `full` lie inside the row and `slots` begin there.
  const int w0 = 256 * wave;
  const int full = n >= w0 + 256 ? (n - w0 - 256) / (4 * T) + 1 : 0, slots = n > w0 ? (n - w0 - 1) / (4 * T) + 1 : 0;
  bool only_inf = false;  // the maximum is infinite: those ids alone, as if of logit 0
  auto value = [&](int id) -> float { return BF16 ? bf16_to_f32(((const uint16_t*)base)[id]) : ((const float*)base)[id]; };
  auto load4 = [&](int j) -> f4v {  // a slot inside the row
    f4v v;
    if constexpr (BF16) {
      const h4u h = *(const h4u*)((const uint16_t*)base + 4 * (j * T + t));
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = bf16_to_f32(h[c]);
    } else {
      const f4u f = *(const f4u*)((const float*)base + 4 * (j * T + t));
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = f[c];
    }
    return v;
  };
  auto last4 = [&](int j) -> f4v {  // the slot that the row ends in
    f4v v;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int id = 4 * (j * T + t) + c;
      v[c] = value(min(id, n - 1));
      v[c] = id < n ? v[c] : -INFINITY;
    }
    return v;
  };
  auto clean = [&](f4v v) -> f4v {
#pragma unroll
    for (int c = 0; c < 4; ++c) v[c] = fmaxf(v[c], -INFINITY);
    if (only_inf) {
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = v[c] == INFINITY ? 0.0f : -INFINITY;
    }
    return v;
  };
  constexpr int PART = SampleLds<T, IDS>::PART;
  bool parted = false;  // the kept ids are the top_k of L.part alone
  auto part4 = [&]() -> f4v {  // this thread's id there, by itself in a slot
    return f4v{t < top_k ? pair_logit(L.part[t]) : -INFINITY, -INFINITY, -INFINITY, -INFINITY};
  };
  // f(j, first id, four values) for this thread's slots, from memory, the next
  // BATCH slots requested before BATCH are worked on (from memory: 256 rows of 100003
  // bf16 ids 113 us with one, 110 with two, 112 with four, which are more code).
  auto each_read = [&](auto&& f) {
    constexpr int BATCH = IDS ? NJ : 2;
    if (full > 0 && !parted) {
      f4v v[BATCH], next[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) v[b] = load4(min(b, full - 1));
      for (int j0 = 0; j0 < full; j0 += BATCH) {
        if constexpr (IDS == 0) {
#pragma unroll
          for (int b = 0; b < BATCH; ++b) next[b] = load4(min(j0 + BATCH + b, full - 1));
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b)
          if (j0 + b < full) f(j0 + b, 4 * ((j0 + b) * T + t), clean(v[b]));
        if constexpr (IDS == 0) {
#pragma unroll
          for (int b = 0; b < BATCH; ++b) v[b] = next[b];
        }
      }
    }
    if (parted || slots > full) {  // one copy of f
      int i = 4 * (full * T + t);
      f4v v;
      if (parted) {
        i = pair_id(L.part[min(t, top_k - 1)]);
        v = part4();
      } else {
        v = clean(last4(full));
      }
      f(full, i, v);
    }
  };
  auto each = [&](auto&& f) {
    if constexpr (IDS > 0) {
      const int last = parted ? 1 : slots;
#pragma unroll 1
      for (int j = 0; j < last; ++j) {
        int i = 4 * (j * T + t);
        f4v v = *(const f4v*)(L.val + i);
        if (PART > 0 && parted) {
          i = pair_id(L.part[min(t, top_k - 1)]);
          v = part4();
        }
        f(j, i, v);
      }
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
  if (t == 0) {
    L.best = 0x7FFFFFFF;
    L.listed = 0;
  }
  if (t < 32) L.exp2[t] = kSampleExp2Tab[t] + ((uint64_t)kMassBits << 52);
  if (t < kList) L.ahead[t] = 0;
  for (int b = t; b < kBins; b += T) L.hist[b] = 0;
  for (int s = t; s < SampleLds<T, IDS>::SEGS; s += T) L.seg[s] = 0;
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
    if (__any(tmax == lmax))
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
  const Octaves scale = {fmax(per_logit, 0x1p-900), -60.0 / fmax(per_logit, 0x1p-900)};
  auto steps_of = [&](float v) -> Octave { return octave_steps((double)v - (double)lmax, scale); };
  auto mass_of = [&](float v) -> uint64_t { return mass_of_steps(steps_of(v), L.exp2); };
  auto bin_of = [&](float v) -> int { return -steps_of(v).steps; };
  // Values of bins [first, last] lie within [least_of(last), most_of(first)]: a
  // cheap test before the exact one (a tenth of a bin, rounding errors and, for bins less
  // than 2^-126 wide, all of them to spare).
  const float logits_per_bin = 1.0f / (float)(per_logit * kBinsPerOctave), slack = fabsf(lmax) * 0x1p-21f + 0x1p-114f;
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

  // Ids kept are those at or before (border_v, border_id).
  float border_v = -INFINITY;
  int border_id = 0x7FFFFFFF;
  // f(j, first id, octaves and masses with kMassBias of the kept ids), for every slot; slots without any are left out
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
        o[c] = steps_of(v[c]);
        m[c] = biased_mass(o[c], L.exp2);
      }
      f(j, i, o, m);
    });
  };

  // How many of list's first `count` entries come before entry t (larger & mask), for
  // t < count: 64, 128 or 256 threads take one entry each, and as many groups of
  // them as there are share the comparisons.
  auto count_ahead = [&](const uint64_t* list, uint32_t count, uint64_t mask) -> uint32_t {
    const int lg = count <= 64 ? 6 : count <= 128 ? 7 : 8;
    static_assert(kList == 256, "groups of up to 256 threads");
    const uint32_t at = t & ((1 << lg) - 1), group = wave >> (lg - 6), groups = T >> lg;
    if (at < count) {
      const uint64_t mine = list[at] & mask;
      uint32_t ahead = 0;
#pragma unroll 4
      for (uint32_t i = 2 * group; i + 1 < count; i += 2 * groups) {
        const ulonglong2 e = *(const ulonglong2*)(list + i);
        ahead += (e.x & mask) > mine ? 1u : 0u;
        ahead += (e.y & mask) > mine ? 1u : 0u;
      }
      if ((count & 1) && group == 0) ahead += (list[count - 1] & mask) > mine ? 1u : 0u;
      if (ahead) lds_add(&L.ahead[at], ahead);
    }
    wg_lds_barrier();
    const uint32_t all = L.ahead[t & (kList - 1)];
    wg_lds_barrier();
    if (t < kList) L.ahead[t] = 0;
    return all;
  };
  // The sum of w over the threads before this one, of the first kList.
  auto scan_threads = [&](uint64_t w, uint64_t& total) -> uint64_t {
    uint64_t s = wave_scan_mass(w);
    if (lane == 63) L.wsum[wave] = s;
    wg_lds_barrier();
    s -= w;
    total = 0;
#pragma unroll
    for (int i = 0; i < kList / 64; ++i) {
      const uint64_t v = L.wsum[i];
      total += v;
      s += i < wave ? v : 0ull;
    }
    return s;
  };

  int drawn = -1;  // in the thread that holds it: the id, its logit, the kept mass
  float drawn_v = 0.0f;
  uint64_t drawn_of = 0;
  // A top-k that leaves the list a quarter of room for ids that share its last bin: where they
  // are too many the list was in vain (us, 64 rows, top-k 192 | 200 | 230, list to 128 | 192 |
  // 256: of 32000 ids 18.8 18.7 19.1 | 18.1 18.8 19.1 | 18.1 18.5 26.2, of 100003 39.8 39.5 39.6 |
  // 27.6 39.3 39.6 | 27.7 28.1 51.4; of 4000, with few maxima a thread, 11.0 | 16.6 | 16.6 at 192).
  int stage = n <= kList ? LIST_ALL : !by_k ? (by_p ? BORDER_P : DRAW) : top_k <= kList * 3 / 4 ? LIST_TOP : BORDER_K;
#pragma unroll 1
  while (stage < DRAW) {
    // ---- the list: all ids at their own places, or those of the stage's bins (of a
    // part of one when it is crowded) ----
    uint32_t listed = n;
    uint64_t need = 0;
    if (stage == LIST_ALL) {
      each([&](int, int i, f4v v) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (i + c < n) L.entry[i + c] = pair_of(v[c], (uint32_t)(i + c));
      });
      wg_lds_barrier();
    } else {
      int first = 0, last = 0, shift = -1;  // shift: of a part's number
      uint64_t lo = 0, hi = ~0ull;          // pairs looked at
#pragma unroll 1
      for (;;) {
        if (shift >= 0) {
          each([&](int, int i, f4v v) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const uint64_t p = pair_of(v[c], (uint32_t)(i + c));
              if (p >= lo && p <= hi) lds_add(&L.hist[(hi - p) >> shift], stage == BORDER_P ? mass_of(v[c]) : (uint64_t)1);
            }
          });
        } else if (stage == LIST_TOP) {
          const int b = bin_of(tmax);
          if (b <= kLastBin) lds_add(&L.hist[b], (uint64_t)1);
        } else if (stage == BORDER_K) {
          each([&](int, int, f4v v) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int b = bin_of(v[c]);
              if (b <= kLastBin) lds_add(&L.hist[b], (uint64_t)1);
            }
          });
        } else {
          each_mass([&](int, int, const Octave (&o)[4], const uint64_t (&m)[4]) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (m[c] != kMassBias) lds_add(&L.hist[-o[c].steps], m[c] & ~kMassBias);
          });
        }
        const Found f = locate<T>(L, [&](uint64_t total) {
          return shift >= 0 ? need : stage == BORDER_P ? need_p(total) : (uint64_t)top_k;
        });
        if (shift >= 0) {
          hi -= (uint64_t)f.bin << shift;
          lo = umax64(lo, hi - ((1ull << shift) - 1));
        } else {
          need = stage == BORDER_P ? need_p(f.total) : (uint64_t)top_k;
          last = f.bin;
          first = stage == LIST_TOP ? 0 : f.bin;
        }
        need -= f.before;
        if (last >= 0) {
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
              const uint64_t p = pair_of(v[c], (uint32_t)(i + c));
              if (b < first || b > last || p < lo || p > hi || p < pair_of(border_v, (uint32_t)border_id)) continue;
              const uint32_t at = lds_add(&L.listed, 1u);
              if (at < (uint32_t)kList) L.entry[at] = p;
              if (shift < 0 && stage >= BORDER_K) {  // the range of all, should they be too many
                __hip_atomic_fetch_min(&L.lo, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                __hip_atomic_fetch_max(&L.hi, p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
              }
            }
          });
        }
        wg_lds_barrier();
        if (last < 0 || L.listed <= (uint32_t)kList || stage == LIST_TOP) break;
        if (shift < 0) {
          lo = L.lo;
          hi = L.hi;
        }
        shift = max(0, 64 - 11 - __builtin_clzll((hi - lo) | 1));  // kBins parts of [lo, hi]
      }
      listed = L.listed;
      if (last < 0 || listed > (uint32_t)kList) {  // too few ids with mass for top_k, too many for the list
        stage = stage == LIST_TOP ? BORDER_K : by_p ? BORDER_P : DRAW;
        continue;
      }
    }

    // ---- in order: thread t's entry goes where as many come before it ----
    const uint32_t own_rank = count_ahead(L.entry, listed, ~0ull);
    if (t < (int)listed) L.sorted[own_rank] = L.entry[t];
    wg_lds_barrier();
    if (stage == BORDER_K) {
      border_v = pair_logit(L.sorted[need - 1]);
      border_id = pair_id(L.sorted[need - 1]);
      stage = by_p ? BORDER_P : DRAW;
      if (t == 0) L.listed = 0;
      wg_lds_barrier();  // before the next list
      if (PART > 0 && top_k <= PART) {
        each([&](int, int i, f4v v) {
          if (!__any((v[0] >= border_v) | (v[1] >= border_v) | (v[2] >= border_v) | (v[3] >= border_v))) return;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (v[c] > border_v || (v[c] == border_v && i + c <= border_id)) {  // top_k of them
              const uint32_t at = lds_add(&L.listed, 1u);
              if (at < (uint32_t)PART) L.part[at] = pair_of(v[c], (uint32_t)(i + c));
            }
        });
        wg_lds_barrier();
        parted = true;
      }
      continue;
    }
    const uint32_t upto = stage == LIST_ALL || stage == LIST_TOP ? (by_k ? min(listed, (uint32_t)top_k) : listed) : listed;
    uint64_t pair = L.sorted[min((uint32_t)t, listed - 1)], total;
    uint64_t m = (uint32_t)t < upto ? mass_of(pair_logit(pair)) : 0ull;
    uint64_t before = scan_threads(m, total);
    if (stage == BORDER_P) {
      if (before < need && need <= before + m) L.border = t;
      wg_lds_barrier();
      border_v = pair_logit(L.sorted[L.border]);
      border_id = pair_id(L.sorted[L.border]);
      stage = DRAW;
      continue;
    }
    const bool keep = (uint32_t)t < upto && (!by_p || before < need_p(total)) && pair_logit(pair) >= least_v;
    const uint32_t mine = (uint32_t)__builtin_popcountll(__ballot(keep));
    if (lane == 0 && wave < kList / 64) L.kept[wave] = mine;
    wg_lds_barrier();
    uint32_t kept = 0;  // the first so many
#pragma unroll
    for (int i = 0; i < kList / 64; ++i) kept += L.kept[i];
    // The draw, in ascending ids: the places of a list of all, else sorted once more.
    if (stage == LIST_ALL) {
      pair = L.entry[min((uint32_t)t, listed - 1)];
      m = (uint32_t)t < listed && own_rank < kept ? mass_of(pair_logit(pair)) : 0ull;
    } else {
      const uint32_t id_rank = count_ahead(L.sorted, kept, 0xFFFFFFFFull);
      if ((uint32_t)t < kept) L.entry[id_rank] = pair;
      wg_lds_barrier();
      pair = L.entry[min((uint32_t)t, kept - 1)];
      m = (uint32_t)t < kept ? mass_of(pair_logit(pair)) : 0ull;
    }
    before = scan_threads(m, total);
    const uint64_t number = need_u(total);
    if (before < number && number <= before + m) {
      drawn = pair_id(pair);
      drawn_v = pair_logit(pair);
      drawn_of = total;
    }
    stage = DRAWN;
  }

  // ---- the draw: kept mass of every 256 consecutive ids, then one id ----
  if (stage == DRAW) {
    if (least_v > border_v) {
      border_v = least_v;
      border_id = 0x7FFFFFFF;
    }
    each_mass([&](int j, int i, const Octave (&)[4], const uint64_t (&m)[4]) {
      if (parted) {
        if (m[0] != kMassBias) lds_add(&L.seg[i >> 8], m[0] - kMassBias);
        return;
      }
      const uint64_t s = wave_scan_mass((m[0] + m[1]) + (m[2] + m[3]));
      if (lane == 63) L.seg[j * NW + wave] = s - 256 * kMassBias;
    });
    wg_lds_barrier();
    // Each wave finds the group by itself, 64 PER sums at a time.
    constexpr int PER = IDS ? (SampleLds<T, IDS>::SEGS + 63) / 64 : 8;
    const int segs = (n + 255) / 256;
    uint64_t total = 0, before = 0, need = 0;
    int seg = -1;
#pragma unroll 1
    for (int find = 0; find < 2; ++find) {
      uint64_t run = 0;
#pragma unroll 1
      for (int s0 = 0; s0 < segs && seg < 0; s0 += 64 * PER) {
        uint64_t c[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int s = s0 + lane * PER + k;
          c[k] = (s < segs ? L.seg[s] : 0ull) + (k ? c[k - 1] : 0ull);
        }
        const uint64_t upto = run + wave_scan_mass(c[PER - 1]);
        if (find) {
#pragma unroll
          for (int k = 0; k < PER; ++k) {
            const uint64_t b = upto - c[PER - 1] + (k ? c[k - 1] : 0ull);
            const uint64_t who = __ballot(b < need && need <= upto - c[PER - 1] + c[k]);
            if (who) {
              seg = s0 + __builtin_ctzll(who) * PER + k;
              before = lane_u64(b, __builtin_ctzll(who));
            }
          }
        }
        run = lane_u64(upto, 63);
      }
      if (!find) {
        total = run;
        need = need_u(total);
      }
    }
    if (wave == seg % NW) {  // the wave that holds the group
      const int j = seg / NW, i = 4 * (j * T + t);
      f4v v;
      if constexpr (IDS > 0)
        v = *(const f4v*)(L.val + i);
      else
        v = clean(j < full ? load4(j) : last4(j));
      uint64_t m[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const bool in = (v[c] > border_v) | ((v[c] == border_v) & (i + c <= border_id));
        m[c] = in ? mass_of(v[c]) : 0ull;
      }
      const uint64_t own = (m[0] + m[1]) + (m[2] + m[3]);
      uint64_t run = before + wave_scan_mass(own) - own;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (run < need && need <= run + m[c]) {
          drawn = i + c;
          drawn_v = v[c];
        }
        run += m[c];
      }
      drawn_of = total;
    }
  }
  if (drawn >= 0)
    finish(drawn, (float)(octave(drawn_v) * 0.6931471805599453 - log(ldexp((double)drawn_of, -kMassBits))));
}

template <int T, int IDS>
hipError_t launch(const SampleArgs& g, hipStream_t s) {
  auto kern = g.bf16 ? k_sample<T, IDS, true> : k_sample<T, IDS, false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)g.rows), dim3(T), 0, s, g);
  return hipGetLastError();
}

}  // namespace

// The row in LDS while it fits, four rows a CU up to 4096 ids.  us a call, 256 threads | 1024 |
// 1024 that read memory for each pass, a nucleus: 1 row of 4096 ids 11.5 | 12.1 | 13.8, 64 of 1000
// 8.9 | 10.8 | 12.3, 64 of 4096 13.3 | 13.2 | 15.0, 512 of 4096 15.2 | 24.7 | 28.8 (of 200, all in the
// list, 1 row 10.3 | 7.8 | 8.8, 512 rows 11.3 | 15.6 | 18.9); in LDS | from memory: 64 rows of 5000 ids
// 13.7 | 15.6, 512 of 5000 25.8 | 30.0, 1 of 32768 24.5 | 27.6, 512 of 32768 61.8 | 71.0.
hipError_t launch_sample(const SampleArgs& g, hipStream_t s) {
  if (!g.logits || !g.u || !g.token || g.V <= 0 || g.V > kSampleMaxIds || g.rows < 0 || (g.off && !g.cand))
    return hipErrorInvalidValue;
  if (g.rows == 0) return hipSuccess;
  if (g.V <= 4096) return launch<256, 4096>(g, s);
  if (g.V <= 32768) return launch<1024, 32768>(g, s);
  return launch<1024, 0>(g, s);
}

}  // namespace mh
