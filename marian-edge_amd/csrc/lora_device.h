// lora_device.h — device helpers of the low-rank adapters (lora.hip, tile.hip).
#pragma once

#include "device_common.h"
#include "kernels.h"

namespace mh {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));  // an MFMA operand: eight consecutive k

// A row's slot and rank; rank 0: no adapter.  A slot past the table or a rank
// past max_rank sets *err and counts as none.
struct RowAdapter {
  int slot, rank;
};
__device__ __forceinline__ RowAdapter row_adapter(const LoraArgs& g, int slot, int* err) {
  const bool in = slot >= 0 && slot < g.slots;
  const int s = in ? slot : 0, r = g.rank[s];
  const bool ok = in && r >= 0 && r <= g.max_rank;
  if (!ok && slot >= 0 && err) *err = 1;
  return {s, ok ? r : 0};
}

// Keeps a NaN, so that a broken adapter does not come out as clean zeros.
__device__ __forceinline__ float lora_relu(float y) { return y <= 0.0f ? 0.0f : y; }

// A value's three bf16 parts, by truncation: the top 8 bits of the value, of what
// is left, and of what is left then.  Both differences are exact and the last
// part holds all that remains, so their sum is the value (down to 2^-126; an
// infinite value leaves NaN in the second part).
__device__ __forceinline__ void split3_parts(float v, uint32_t (&p)[3]) {
  p[0] = __float_as_uint(v) & 0xFFFF0000u;
  const float r = v - __uint_as_float(p[0]);
  p[1] = __float_as_uint(r) & 0xFFFF0000u;
  p[2] = __float_as_uint(r - __uint_as_float(p[1]));
}
// Of two values, packed (a in the low half).
__device__ __forceinline__ void split3_pair(float a, float b, uint32_t (&p)[3]) {
  uint32_t pa[3], pb[3];
  split3_parts(a, pa);
  split3_parts(b, pb);
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = __builtin_amdgcn_perm(pb[i], pa[i], 0x07060302);  // the upper halves
}
__device__ __forceinline__ void split3(f4v lo, f4v hi, bf8 (&p)[3]) {
  union {
    uint32_t u[4];
    bf8 v;
  } o[3];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t q[3];
    split3_pair(c < 2 ? lo[2 * c] : hi[2 * c - 4], c < 2 ? lo[2 * c + 1] : hi[2 * c - 3], q);
#pragma unroll
    for (int i = 0; i < 3; ++i) o[i].u[c] = q[i];
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) p[i] = o[i].v;
}

// t of many rows in matrix-core operand order: of 32-row block `block`, part `part`
// (0 to 2) and 16-rank step `step`, lane l's eight values (row l % 32, ranks 8 (l /
// 32) ...) lie at this index, so a wave's operand is 1 KB in a row.  ldt: ranks
// stored per row.
__device__ __forceinline__ int64_t lora_t_index(int64_t block, int part, int step, int lane, int ldt) {
  return (((block * 3 + part) * (ldt >> 4) + step) * 64 + lane) * 8;
}

// The first n (0 to 8) values of w, zeros behind them.
__device__ __forceinline__ bf8 first_values(bf8 w, int n) {
  union {
    bf8 v;
    uint32_t u[4];
  } o;
  o.v = w;
#pragma unroll
  for (int c = 0; c < 4; ++c) o.u[c] &= n >= 2 * c + 2 ? 0xFFFFFFFFu : n == 2 * c + 1 ? 0xFFFFu : 0u;
  return o.v;
}

}  // namespace mh
