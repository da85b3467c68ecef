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
// memory, so they cost nothing: 65536 rows of 512, bf16 in, sum, out and q stored,
// 67 us, 5.5 TB/s (a copy of that size: 5.1); one row of 512: 2.0 us, the launch.
#include "device_common.h"
#include "kernels.h"

#include <algorithm>
#include <type_traits>

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

// Four values at any address of theirs.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32u __attribute__((aligned(1)));

// T threads hold a row, four neighbouring values at a time: quad number j of
// thread t begins at column 4(jT + t).  A quad that ends past the row (TAIL: a width
// that is no multiple of four) holds its last four values instead, of which the sum
// takes those that the quad before does not have; both compute and store the same
// values for the others.  Quads past the row load the last four too, so that all of a
// row's loads are in flight at once.  T = 64: a wave per row, four rows a workgroup and
// no barrier.
template <int T, int NV, bool BF16, bool TAIL>
__global__ __launch_bounds__(T < 256 ? 256 : T) void k_rms_norm(RmsArgs g) {
  touch_kernargs<sizeof(RmsArgs)>();
  constexpr int ROWS = T < 256 ? 256 / T : 1, NW = T / 64;
  __shared__ double sSum[2][NW];
  __shared__ uint32_t sMax[2][NW];
  const int t = threadIdx.x % T, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int dim = g.dim;

  const bool tiny = TAIL && T == 64 && NV == 1 && dim < 4;  // less than a quad, in thread 0
  auto quad = [&](int j) { return 4 * (j * T + t); };
  auto load_f32 = [&](const float* p, int j) -> f4v {
    if (tiny) return f4v{p[0], p[min(1, dim - 1)], p[dim - 1], 0.0f};
    return *(const f4u*)(p + min(quad(j), dim - 4));
  };
  using Quad = std::conditional_t<BF16, h4u, f4v>;
  auto load = [&](const void* row, int64_t first, int j) -> Quad {
    if constexpr (BF16) {
      const uint16_t* p = (const uint16_t*)row + first;
      if (tiny) return h4u{p[0], p[min(1, dim - 1)], p[dim - 1], 0};
      return *(const h4u*)(p + min(quad(j), dim - 4));
    } else {
      return load_f32((const float*)row + first, j);
    }
  };
  auto f32 = [](Quad v, int c) -> float {
    if constexpr (BF16)
      return bf16_to_f32(v[c]);
    else
      return v[c];
  };
  // Whether value c of quad j is one of the row's and no other quad's.
  auto counts = [&](int j, int c) {
    if constexpr (TAIL) return tiny ? t == 0 && c < dim : quad(j) < dim && min(quad(j), dim - 4) + c >= quad(j);
    return quad(j) < dim;
  };

  f4v gv[NV];
  auto load_scale = [&]() {
#pragma unroll
    for (int j = 0; j < NV; ++j) gv[j] = load_f32(g.scale, j);
  };
  // Few values per thread: with the row, for latency; many: once the row's
  // squares are summed, for registers.
  constexpr bool kEarly = NV <= 2;
  if constexpr (kEarly) load_scale();

  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * ROWS + (T < 256 ? wave : 0); row < g.rows;
       row += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    f4v s[NV];
    Quad xv[NV], rv[NV];
    const int64_t o0 = row * dim;
#pragma unroll
    for (int j = 0; j < NV; ++j) xv[j] = load(g.x, row * g.ldx, j);
    if (g.r) {
#pragma unroll
      for (int j = 0; j < NV; ++j) rv[j] = load(g.r, row * g.ldr, j);
      __builtin_amdgcn_sched_barrier(0);  // all loads first
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = f32(xv[j], c) + f32(rv[j], c);
    } else {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[j][c] = f32(xv[j], c);
    }
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const double v = counts(j, c) ? s[j][c] : 0.0f;
        ss = __builtin_fma(v, v, ss);
      }
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
        mx = max(mx, !tiny || c < dim ? __float_as_uint(y[j][c]) & 0x7fffffffu : 0u);
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
      if (quad(j) >= dim) continue;
      const uint32_t q = quantize_pack4(y[j][0], y[j][1], y[j][2], y[j][3], a);
      if (tiny) {
        for (int i = 0; i < dim; ++i) {
          if (g.sum) g.sum[o0 + i] = i == 0 ? s[j][0] : i == 1 ? s[j][1] : s[j][2];
          if (g.out) g.out[o0 + i] = i == 0 ? y[j][0] : i == 1 ? y[j][1] : y[j][2];
          if (g.q) g.q[o0 + i] = (int8_t)(q >> 8 * i);
        }
        continue;
      }
      const int64_t at = o0 + min(quad(j), dim - 4);
      if (g.sum) *(f4u*)(g.sum + at) = s[j];
      if (g.out) *(f4u*)(g.out + at) = y[j];
      if (g.q) *(u32u*)(g.q + at) = q;
    }
  }
}

template <int T, int NV>
hipError_t launch_rms(const RmsArgs& g, hipStream_t s) {
  constexpr int ROWS = T < 256 ? 256 / T : 1;
  const int64_t wgs = (g.rows + ROWS - 1) / ROWS;
  auto kern = g.dim % 4 ? (g.bf16 ? k_rms_norm<T, NV, true, true> : k_rms_norm<T, NV, false, true>)
                        : (g.bf16 ? k_rms_norm<T, NV, true, false> : k_rms_norm<T, NV, false, false>);
  hipLaunchKernelGGL(kern, dim3((unsigned)std::min<int64_t>(wgs, 1 << 20)), dim3(T < 256 ? 256 : T), 0, s, g);
  return hipGetLastError();
}

}  // namespace

// The fewest threads that hold the row in registers: more threads wait for each
// other, and quads past the row cost what others do.  us for 2^25 bf16 | fp32 values
// (sum, out, q stored): 512 columns, one wave 67 | 76, 256 threads 124 | 107; 1001: one
// wave 69 | 88, 256 threads 99 | 88; 2047: 256 threads, 2 quads 84 | 81, 512 threads 94 | 87;
// 5000: 256 threads, 6 quads 74 | 81, 8 quads 74 | 80, 512 threads, 4 quads 86 | 83; 8192:
// 256 threads 69 | 81, 512 threads 75 | 82; 12001: 512 threads, 6 quads 85 | 86, 8 quads
// 89 | 89; 16384: 512 threads 76 | 86, 1024 threads 76 | 86.
hipError_t launch_rms_norm(const RmsArgs& g, hipStream_t s) {
  if (!g.x || !g.scale || g.dim <= 0 || g.dim > kRmsMaxDim || g.rows < 0) return hipErrorInvalidValue;
  if (g.rows == 0) return hipSuccess;
  if (g.dim <= 256) return launch_rms<64, 1>(g, s);
  if (g.dim <= 512) return launch_rms<64, 2>(g, s);
  if (g.dim <= 1024) return launch_rms<64, 4>(g, s);
  if (g.dim <= 2048) return launch_rms<256, 2>(g, s);
  if (g.dim <= 4096) return launch_rms<256, 4>(g, s);
  if (g.dim <= 6144) return launch_rms<256, 6>(g, s);
  if (g.dim <= 8192) return launch_rms<256, 8>(g, s);
  if (g.dim <= 12288) return launch_rms<512, 6>(g, s);
  return launch_rms<512, 8>(g, s);
}

}  // namespace mh
