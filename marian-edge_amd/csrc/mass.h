// mass.h — probabilities of logits as integers, exact to add up, shared by the kernels that draw ids.
//
// An id's mass is an integer, at most 2 from 2^44 exp((l - max) / T), and 2^44 for the row's maximum: sums of up to 2^19
// of them are exact in 64 bits in any order.
#pragma once

#include "device_common.h"
#include "kernels.h"
#include "ref_expf.h"

namespace mh {
namespace {

constexpr int kMassBits = 44;  // mass of the row's maximum

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

__device__ __forceinline__ Octaves octaves_of(float temperature) {
  const double per_logit = fmax(1.4426950408889634 / (double)temperature, 0x1p-900);
  return {per_logit, -60.0 / per_logit};
}

// The mass of an id with logit v among what a row's settings keep.
__device__ __forceinline__ double kept_mass(const RowKept& k, const Octaves& scale, float v, int id, const uint64_t* exp2) {
  if (k.flags & kKeptOne) return id == k.border_id ? 1.0 : 0.0;
  if (k.flags & kKeptInf) v = v == INFINITY ? 0.0f : -INFINITY;
  if (!(v > k.border_v || (v == k.border_v && id <= k.border_id))) return 0.0;
  return (double)mass_of_steps(octave_steps((double)v - (double)k.max, scale), exp2);
}

}  // namespace
}  // namespace mh
