// lora.hip — the low-rank adapters of many requests beside a shared Q8 layer.
//
//   y_m = W x_m (Q8) + b + c_s B_s (A_s x_m),  s = slot of row m (negative: no adapter)
//
// A_s is [rank_s, K], B_s [N, rank_s] (bf16, stored max_rank apart), x fp32.
// The products of bf16 weights with fp32 activations are summed in fp32.
#include "device_common.h"
#include "kernels.h"

#include <algorithm>

namespace mh {
namespace {

// The row's slot and rank, or rank 0: no adapter.  A slot past the table or a
// rank past max_rank sets *err and counts as none.
struct RowAdapter {
  int slot, rank;
};
__device__ __forceinline__ RowAdapter row_adapter(const LoraArgs& g, int64_t m) {
  const int s = g.slot_of_row[m];
  if (s < 0) return {0, 0};
  if (s >= g.slots) {
    if (g.err) *g.err = 1;
    return {0, 0};
  }
  const int r = g.rank[s];
  if (r < 0 || r > g.max_rank) {
    if (g.err) *g.err = 1;
    return {0, 0};
  }
  return {s, r};
}

// t[m, r] = c_s (A_s[r] . x_m): one workgroup per row, a wave per r.
__global__ __launch_bounds__(256) void k_lora_down(LoraArgs g) {
  const int64_t m = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const RowAdapter a = row_adapter(g, m);
  const float* x = g.x + m * g.K;
  for (int r = wave; r < a.rank; r += 4) {
    const uint16_t* w = g.a + ((int64_t)a.slot * g.max_rank + r) * g.K;
    float s = 0.0f;
    for (int k = lane; k < g.K; k += 64) s = __builtin_fmaf(x[k], bf16_to_f32(w[k]), s);
    s = tree_combine_wave(s);
    if (lane == 0) g.t[m * g.max_rank + r] = s * g.scale[a.slot];
  }
}

// out[m, n] = relu?(out[m, n] + B_s[n] . t[m])
__global__ __launch_bounds__(256) void k_lora_up(LoraArgs g) {
  const int64_t m = blockIdx.y;
  const int n = blockIdx.x * 256 + threadIdx.x;
  if (n >= g.N) return;
  const RowAdapter a = row_adapter(g, m);
  const uint16_t* w = g.b + ((int64_t)a.slot * g.N + n) * g.max_rank;
  float d = 0.0f;
  for (int r = 0; r < a.rank; ++r) d = __builtin_fmaf(g.t[m * g.max_rank + r], bf16_to_f32(w[r]), d);
  float y = g.out[m * g.N + n] + d;
  if (g.relu) y = y > 0.0f ? y : 0.0f;
  g.out[m * g.N + n] = y;
}

}  // namespace

size_t lora_scratch_bytes(int64_t M, int max_rank) { return (size_t)M * max_rank * sizeof(float); }

hipError_t launch_lora_down(const LoraArgs& g, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  hipLaunchKernelGGL(k_lora_down, dim3((unsigned)g.M), dim3(256), 0, s, g);
  return hipGetLastError();
}

hipError_t launch_lora_linear(const GemmArgs& base, const LoraArgs& g, hipStream_t s) {
  Epilogue e;
  e.out = g.out;
  e.ldo = g.N;
  hipError_t rc = launch_gemm_store(base, e, s);
  for (int64_t m0 = 0; rc == hipSuccess && m0 < g.M; m0 += 65535) {
    LoraArgs p = g;
    p.t += m0 * g.max_rank;
    p.slot_of_row += m0;
    p.out += m0 * g.N;
    hipLaunchKernelGGL(k_lora_up, dim3((g.N + 255) / 256, (unsigned)std::min<int64_t>(g.M - m0, 65535)), dim3(256), 0, s, p);
    rc = hipGetLastError();
  }
  return rc;
}

}  // namespace mh
