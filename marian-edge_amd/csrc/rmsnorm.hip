// rmsnorm.hip — residual addition, root-mean-square norm and int8 rows in one pass.
//
//   s = x + r                         (fp32, one rounding; r optional)
//   y = s / sqrt(mean(s^2) + eps) * scale
//   a = 127 / max|y| (1 for a zero row),  q = clamp(rne(y * a), -127, 127)
//
// The mean and each y are computed in 64 bits and rounded once to fp32, so a
// value does not depend on how the row is spread over lanes: the int8 codes,
// which lie next to rounding borders, come out the same for every launch
// shape, and a and q are what marian_hip_quantize_rows makes of the stored y.
// 64-bit products run at the rate of 32-bit ones here and the kernel waits for
// memory, so they cost nothing.
#include "device_common.h"
#include "kernels.h"

#include <algorithm>

namespace mh {
namespace {

// Sum over the wave in a fixed order; every lane returns it.
__device__ __forceinline__ double wave_sum_f64(double v) {
  auto step = [&](auto mov) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    v += __longlong_as_double((long long)mov(b));
  };
  step([](uint64_t b) { return dpp_mov_u64<0xB1>(b); });
  step([](uint64_t b) { return dpp_mov_u64<0x4E>(b); });
  step([](uint64_t b) { return dpp_mov_u64<0x124>(b); });
  step([](uint64_t b) { return dpp_mov_u64<0x128>(b); });
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  double part[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 16 * i);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 16 * i);
    part[i] = __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
  }
  return (part[0] + part[1]) + (part[2] + part[3]);
}

// T threads hold a row: VEC: float4 number j of thread t at columns 4(jT + t);
// otherwise (a width, stride or address that is no multiple of four values)
// value i of thread t at column iT + t.  Loads past the row are clamped to its
// last values and zeroed, so that all of a row's loads are in flight at once.
// One wave per row up to 1024 columns (four rows a workgroup, no barrier), a
// workgroup of 256 or 1024 threads above.
template <int T, int NV, bool BF16, bool VEC>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rms_norm(RmsArgs g) {
  touch_kernargs<sizeof(RmsArgs)>();
  constexpr int ROWS = T < 256 ? 256 / T : 1, NW = T / 64;
  __shared__ double sSum[2][NW];
  __shared__ uint32_t sMax[2][NW];
  const int t = threadIdx.x % T, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int dim = g.dim;

  auto load = [&](const void* p, int64_t at) -> f4v {  // four values from element `at`
    if constexpr (BF16) {
      const ushort4 h = *(const ushort4*)((const uint16_t*)p + at);
      return f4v{bf16_to_f32(h.x), bf16_to_f32(h.y), bf16_to_f32(h.z), bf16_to_f32(h.w)};
    } else {
      return *(const f4v*)((const float*)p + at);
    }
  };
  auto load1 = [&](const void* p, int64_t at) -> float {
    if constexpr (BF16)
      return bf16_to_f32(((const uint16_t*)p)[at]);
    else
      return ((const float*)p)[at];
  };

  f4v gv[NV];
  auto load_scale = [&]() {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (VEC) {
        gv[j] = *(const f4v*)(g.scale + min(4 * (j * T + t), dim - 4));
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) gv[j][c] = g.scale[min((4 * j + c) * T + t, dim - 1)];
      }
    }
  };
  // Few values per thread: with the row, for latency; many: once the row's
  // squares are summed, for registers.
  constexpr bool kEarly = NV <= 2;
  if constexpr (kEarly) load_scale();

  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + (T < 256 ? wave : 0); row < g.rows;
       row += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    f4v s[NV], rv[NV];
    const int64_t x0 = row * g.ldx, r0 = row * g.ldr, o0 = row * dim;
    if constexpr (VEC) {
#pragma unroll
      for (int j = 0; j < NV; ++j) s[j] = load(g.x, x0 + min(4 * (j * T + t), dim - 4));
      if (g.r) {
#pragma unroll
        for (int j = 0; j < NV; ++j) rv[j] = load(g.r, r0 + min(4 * (j * T + t), dim - 4));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[j][c] = s[j][c] + rv[j][c];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = 4 * (j * T + t) < dim ? s[j][c] : 0.0f;
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = load1(g.x, x0 + min((4 * j + c) * T + t, dim - 1));
      if (g.r) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) rv[j][c] = load1(g.r, r0 + min((4 * j + c) * T + t, dim - 1));
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[j][c] = s[j][c] + rv[j][c];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = (4 * j + c) * T + t < dim ? s[j][c] : 0.0f;
    }

    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) ss = __builtin_fma((double)s[j][c], (double)s[j][c], ss);
    if constexpr (!kEarly) load_scale();
    ss = wave_sum_f64(ss);
    if constexpr (NW > 1) {
      if ((t & 63) == 0) sSum[turn][wave] = ss;
      wg_lds_barrier();
      ss = 0.0;
#pragma unroll
      for (int w = 0; w < NW; ++w) ss += sSum[turn][w];
    }
    const double inv = 1.0 / sqrt(ss / (double)dim + (double)g.eps);

    f4v y[NV];
    uint32_t mx = 0;  // bits of max|y|: ordered like the values, NaN above infinity
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        y[j][c] = (float)((double)s[j][c] * inv * (double)gv[j][c]);
        const bool in = VEC ? 4 * (j * T + t) < dim : (4 * j + c) * T + t < dim;
        mx = max(mx, in ? __float_as_uint(y[j][c]) & 0x7fffffffu : 0u);
      }
    if (g.q || g.err) {
      mx = row16_max(mx);
      mx = max(max((uint32_t)__builtin_amdgcn_readlane((int)mx, 0), (uint32_t)__builtin_amdgcn_readlane((int)mx, 16)),
               max((uint32_t)__builtin_amdgcn_readlane((int)mx, 32), (uint32_t)__builtin_amdgcn_readlane((int)mx, 48)));
      if constexpr (NW > 1) {
        if ((t & 63) == 0) sMax[turn][wave] = mx;
        wg_lds_barrier();
#pragma unroll
        for (int w = 0; w < NW; ++w) mx = max(mx, sMax[turn][w]);
      }
      if (g.err && t == 0 && mx >= 0x7f800000u) *g.err = 1;
    }
    const float a = row_multiplier(__uint_as_float(mx));
    if (g.a && t == 0) g.a[row] = a;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (VEC) {
        const int c = 4 * (j * T + t);
        if (c < dim) {
          if (g.sum) *(f4v*)(g.sum + o0 + c) = s[j];
          if (g.out) *(f4v*)(g.out + o0 + c) = y[j];
          if (g.q) *(uint32_t*)(g.q + o0 + c) = quantize_pack4(y[j][0], y[j][1], y[j][2], y[j][3], a);
        }
      } else {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int col = (4 * j + c) * T + t;
          if (col < dim) {
            if (g.sum) g.sum[o0 + col] = s[j][c];
            if (g.out) g.out[o0 + col] = y[j][c];
            if (g.q) g.q[o0 + col] = (int8_t)quantize_one(y[j][c], a);
          }
        }
      }
    }
  }
}

template <int T, int NV, bool VEC>
hipError_t launch_rms(const RmsArgs& g, hipStream_t s) {
  constexpr int ROWS = T < 256 ? 256 / T : 1;
  const int64_t wgs = (g.rows + ROWS - 1) / ROWS;
  auto kern = g.bf16 ? k_rms_norm<T, NV, true, VEC> : k_rms_norm<T, NV, false, VEC>;
  hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, 1 << 20)), dim3(T < 256 ? 256 : T), 0, s, g);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_rms_norm(const RmsArgs& g, hipStream_t s) {
  if (!g.x || !g.scale || g.dim <= 0 || g.dim > kRmsMaxDim || g.rows < 0) return hipErrorInvalidValue;
  if (g.rows == 0) return hipSuccess;
  const uintptr_t in = (uintptr_t)g.x | (uintptr_t)g.r, out = (uintptr_t)g.sum | (uintptr_t)g.out | (uintptr_t)g.scale;
  const bool vec = g.dim % 4 == 0 && g.ldx % 4 == 0 && (!g.r || g.ldr % 4 == 0) && in % (g.bf16 ? 8 : 16) == 0 &&
                   out % 16 == 0 && (uintptr_t)g.q % 4 == 0;
  if (vec) {
    if (g.dim <= 256) return launch_rms<64, 1, true>(g, s);
    if (g.dim <= 512) return launch_rms<64, 2, true>(g, s);
    if (g.dim <= 1024) return launch_rms<64, 4, true>(g, s);
    if (g.dim <= 2048) return launch_rms<256, 2, true>(g, s);
    if (g.dim <= 3 * 1024) return launch_rms<256, 3, true>(g, s);
    if (g.dim <= 4096) return launch_rms<256, 4, true>(g, s);
    if (g.dim <= 5 * 1024) return launch_rms<256, 5, true>(g, s);
    if (g.dim <= 6 * 1024) return launch_rms<256, 6, true>(g, s);
    if (g.dim <= 8192) return launch_rms<256, 8, true>(g, s);
    return launch_rms<1024, 4, true>(g, s);
  }
  if (g.dim <= 512) return launch_rms<64, 2, false>(g, s);
  if (g.dim <= 2048) return launch_rms<256, 2, false>(g, s);
  if (g.dim <= 8192) return launch_rms<1024, 2, false>(g, s);
  return launch_rms<1024, 4, false>(g, s);
}

}  // namespace mh
