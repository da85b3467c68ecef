// lora.hip — the low-rank adapters of many requests beside a shared Q8 layer.
//
//   y_m = W x_m (Q8) + b + c_s B_s (A_s x_m),  s = slot of row m (negative: no adapter)
//
// A_s is [rank_s, K], B_s [N, rank_s] (bf16, stored max_rank apart), x fp32.
// Two launches: t = c_s A_s x_m (and the rows' quantization when the caller has
// none), then the int8 product with B_s t added in its epilogue.  Fusing both
// would repeat A_s x_m in every column workgroup; a third launch for the addition
// would read and write the output once more.
//
// Few rows (a decode step): neighbouring rows belong to different requests, so
// each row multiplies with its own A_s and B_s on the vector units and reads them
// once; those reads are what is left to do.  Many rows (prompts): a 16- or 32-row
// tile mostly holds one request's rows, so A_s and B_s are matrix-core operands,
// once per distinct slot of the tile; a row keeps the result of its own slot, by
// selection and not by a product with zero, so that an infinite weight reaches no
// other request's rows.  fp32 operands go to the bf16 matrix cores as three parts of
// 8 bits each, which hold all 24 bits of a value: products are exact and sums fp32.
#include "device_common.h"
#include "kernels.h"
#include "lora_device.h"

#include <algorithm>

namespace mh {
namespace {

// ---------------------------------------------------------------------------
// Few rows, first product: one workgroup of four waves per row.  Each wave holds
// the row (lane l: values 8l + 512 j ...) and takes every fourth r.  KJ: row
// pieces in registers (K up to 512 KJ); 0: read again for each r.
// ---------------------------------------------------------------------------
constexpr int kDownBatch = 4;  // r's whose weights are in flight together

template <int KJ>
__global__ __launch_bounds__(256) void k_lora_down_rows(LoraArgs g) {
  touch_kernargs<sizeof(LoraArgs)>();
  const int64_t m = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int K = g.K;
  const float* x = g.x + m * K;
  float* t = (float*)g.t + m * g.max_rank;
  f4v v[KJ ? KJ : 1][2];
  auto load_x = [&](int j, f4v (&p)[2]) {  // zeros past K
    const int k = 512 * j + 8 * lane;
    const f4v* at = (const f4v*)(x + min(k, K - 8));
    p[0] = at[0];
    p[1] = at[1];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      p[0][c] = k < K ? p[0][c] : 0.0f;
      p[1][c] = k < K ? p[1][c] : 0.0f;
    }
  };
  const int pieces = (K + 511) >> 9;
  if constexpr (KJ > 0) {
#pragma unroll
    for (int j = 0; j < KJ; ++j) load_x(j, v[j]);
  }
  const RowAdapter a = row_adapter(g, g.slot_of_row[m], g.err);
  const float gain = g.scale[a.slot];

  if (g.xq) {  // wave 0: the row's codes, as the row quantization makes them
    if (wave == 0) {
      float mx = 0.0f;
      bool bad = false;
      auto scan = [&](const f4v (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            mx = fmaxf(mx, fabsf(p[h][c]));
            bad |= !(fabsf(p[h][c]) < INFINITY);
          }
      };
      auto store = [&](int j, const f4v (&p)[2], float am) {
        const int k = 512 * j + 8 * lane;
        if (k < K) {
          uint2 q;
          q.x = quantize_pack4(p[0][0], p[0][1], p[0][2], p[0][3], am);
          q.y = quantize_pack4(p[1][0], p[1][1], p[1][2], p[1][3], am);
          *(uint2*)(g.xq + m * K + k) = q;
        }
      };
      if constexpr (KJ > 0) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) scan(v[j]);
      } else {
        for (int j = 0; j < pieces; ++j) {
          f4v p[2];
          load_x(j, p);
          scan(p);
        }
      }
      const float am = row_multiplier(wave_max(mx));
      if (lane == 0) g.xa[m] = am;
      if (__any(bad) && lane == 0 && g.err) *g.err = 1;
      if constexpr (KJ > 0) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) store(j, v[j], am);
      } else {
        for (int j = 0; j < pieces; ++j) {
          f4v p[2];
          load_x(j, p);
          store(j, p, am);
        }
      }
    }
  }

  for (int r = a.rank + tid; r < g.max_rank; r += 256) t[r] = 0.0f;
  const uint16_t* wa = g.a + (int64_t)a.slot * g.max_rank * K;
  for (int r0 = wave; r0 < a.rank; r0 += 4 * kDownBatch) {
    float s[kDownBatch];
#pragma unroll
    for (int b = 0; b < kDownBatch; ++b) s[b] = 0.0f;
    auto piece = [&](int j, const f4v (&p)[2]) {
      const int k = min(512 * j + 8 * lane, K - 8);
      uint4 w[kDownBatch];
#pragma unroll
      for (int b = 0; b < kDownBatch; ++b) w[b] = *(const uint4*)(wa + (int64_t)min(r0 + 4 * b, a.rank - 1) * K + k);
#pragma unroll
      for (int b = 0; b < kDownBatch; ++b) {
        const uint32_t d[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[b] = __builtin_fmaf(p[c >> 1][2 * (c & 1)], __uint_as_float(d[c] << 16), s[b]);
          s[b] = __builtin_fmaf(p[c >> 1][2 * (c & 1) + 1], __uint_as_float(d[c] & 0xFFFF0000u), s[b]);
        }
      }
    };
    if constexpr (KJ > 0) {
#pragma unroll
      for (int j = 0; j < KJ; ++j) piece(j, v[j]);
    } else {
      for (int j = 0; j < pieces; ++j) {
        f4v p[2];
        load_x(j, p);
        piece(j, p);
      }
    }
#pragma unroll
    for (int b = 0; b < kDownBatch; ++b) {
      const float sum = tree_combine_wave(s[b]);
      if (lane == 0 && r0 + 4 * b < a.rank) t[r0 + 4 * b] = sum * gain;
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows, the layer: 16 rows and 16 CT columns per workgroup, its NW waves
// split K (wave w: k-steps w, w + NW, ...), their exact i32 partials meet in LDS,
// and each thread finishes whole outputs: dequantization, then the row's t
// against its slot's 16-byte pieces of B, the first 16 ranks requested before the
// products start.
// ---------------------------------------------------------------------------
constexpr int kUpRows = 16;

template <int NW, int CT, int KSW>
__global__ __launch_bounds__(NW * 64) void k_lora_rows(GemmArgs g, LoraArgs l) {
  touch_kernargs<sizeof(GemmArgs) + sizeof(LoraArgs)>();
  constexpr int NT = NW * 64, COLS = 16 * CT, LDC = COLS + 1;
  constexpr int PER = kUpRows * COLS / NT;  // outputs per thread
  static_assert(PER >= 1 && PER * NT == kUpRows * COLS, "whole outputs");
  __shared__ int32_t sP[NW][kUpRows * LDC];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * COLS, m0 = blockIdx.y * kUpRows;
  const int ksteps = g.K >> 6, kq = (lane >> 4) * 16;
  const int8_t* ar = g.A + (int64_t)min(m0 + (lane & 15), g.M - 1) * g.lda + kq;
  const int8_t* br[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) br[c] = g.W + (int64_t)min(n0 + 16 * c + (lane & 15), g.N - 1) * g.K + kq;

  v4i af[KSW], bf[KSW][CT];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < KSW; ++i) {
      const int s = min(s0 + wave + NW * i, ksteps - 1);
      af[i] = *(const v4i*)(ar + s * 64);
#pragma unroll
      for (int c = 0; c < CT; ++c) bf[i][c] = *(const v4i*)(br[c] + s * 64);
    }
  };
  load(0);

  // This thread's outputs: column n, rows tid / COLS + k (NT / COLS).
  const int n = min(n0 + tid % COLS, g.N - 1);
  const float wm = g.wmult[n], bias = g.bias[n];
  float am[PER];
  RowAdapter ad[PER];
  int64_t row[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    row[k] = min(m0 + tid / COLS + k * (NT / COLS), g.M - 1);
    am[k] = g.a[row[k]];
    ad[k] = row_adapter(l, l.slot_of_row[row[k]], nullptr);
  }
  // Pieces of 8 ranks: B's 16 bytes and t's 32, rank8 below max_rank.
  struct Piece {
    uint4 w;
    f4v t0, t1;
  };
  auto piece = [&](int k, int r8) {
    Piece p;
    p.w = *(const uint4*)(l.b + ((int64_t)ad[k].slot * g.N + n) * l.max_rank + r8);
    const f4v* t = (const f4v*)((const float*)l.t + row[k] * l.max_rank + r8);
    p.t0 = t[0];
    p.t1 = t[1];
    return p;
  };
  Piece first[PER][2];
#pragma unroll
  for (int k = 0; k < PER; ++k)
#pragma unroll
    for (int h = 0; h < 2; ++h) first[k][h] = piece(k, min(8 * h, l.max_rank - 8));

  v4i acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
  for (int s0 = 0; s0 < ksteps; s0 += NW * KSW) {
    if (s0) load(s0);
#pragma unroll
    for (int i = 0; i < KSW; ++i) {
      const v4i a = keep_or_zero(af[i], s0 + wave + NW * i < ksteps);
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, bf[i][c], acc[c], 0, 0, 0);
    }
  }
  // Lane l holds rows 4 (l / 16) + r of column l % 16 of each 16x16 tile.
#pragma unroll
  for (int c = 0; c < CT; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r) sP[wave][((lane >> 4) * 4 + r) * LDC + 16 * c + (lane & 15)] = acc[c][r];
  wg_lds_barrier();

#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int at = (tid / COLS + k * (NT / COLS)) * LDC + tid % COLS;
    int32_t iv = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) iv += sP[w][at];
    float y = dequant(iv, am[k], wm, bias);
    float d = 0.0f;
    auto add = [&](const Piece& p, int r8) {  // ranks past the slot's: weights of any value, not used
      const uint32_t w[4] = {p.w.x, p.w.y, p.w.z, p.w.w};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float b = __uint_as_float(c & 1 ? w[c >> 1] & 0xFFFF0000u : w[c >> 1] << 16);
        const float e = __builtin_fmaf(c < 4 ? p.t0[c & 3] : p.t1[c & 3], b, d);
        d = r8 + c < ad[k].rank ? e : d;
      }
    };
    add(first[k][0], 0);
    add(first[k][1], 8);
    for (int r8 = 16; r8 < l.max_rank && __any(r8 < ad[k].rank); r8 += 8) add(piece(k, r8), r8);
    y += d;
    if (l.relu) y = y > 0.0f ? y : 0.0f;
    if (m0 + tid / COLS + k * (NT / COLS) < g.M && n0 + tid % COLS < g.N) l.out[row[k] * g.N + n] = y;
  }
}

// ---------------------------------------------------------------------------
// Many rows, first product: 16 rows per workgroup, its eight waves split K in
// chunks of 32, RT tiles of 16 ranks.  v_mfma_f32_16x16x32_bf16: lane l holds k
// 8 (l / 16) .. + 8 of x's row l % 16 and of A's row l % 16, and of the result
// column (rank) l % 16, rows 4 (l / 16) + r.  A wave reads and splits its x once, 512
// columns of the row at a time, and multiplies it with each slot of the tile.
// ---------------------------------------------------------------------------
constexpr int kDownRows = 16;
constexpr int kDownWaves = 8;
constexpr int kDownChunks = 2;  // chunks of a wave held at once

template <int RT>
__global__ __launch_bounds__(kDownWaves * 64) void k_lora_down_tile(LoraArgs g) {
  touch_kernargs<sizeof(LoraArgs)>();
  constexpr int LDS_LD = 16 * RT + 1;
  __shared__ float sT[kDownWaves][kDownRows * LDS_LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t m0 = (int64_t)blockIdx.x * kDownRows;
  const int K = g.K, kq = 8 * (lane >> 4), chunks = K >> 5;
  const int64_t row = m0 + (lane & 15) < g.M ? m0 + (lane & 15) : g.M - 1;
  const float* x = g.x + row * K + kq;
  f4v x0[kDownChunks], x1[kDownChunks];
  auto load_x = [&](int c0) {  // past K: the last chunk again
#pragma unroll
    for (int u = 0; u < kDownChunks; ++u) {
      const int c = min(c0 + kDownWaves * u, chunks - 1);
      x0[u] = *(const f4v*)(x + 32 * c);
      x1[u] = *(const f4v*)(x + 32 * c + 4);
    }
  };
  load_x(wave);
  const RowAdapter ad = row_adapter(g, m0 + (lane & 15) < g.M ? g.slot_of_row[row] : -1, g.err);
  const uint32_t with = (uint32_t)__ballot(ad.rank > 0) & 0xFFFFu;  // rows with an adapter
  f4v sum[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) sum[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  for (int c0 = wave; with && c0 < chunks; c0 += kDownWaves * kDownChunks) {
    bf8 p[kDownChunks][3];
    for (uint32_t todo = with; todo;) {  // the tile's slots, one after another
      const int lead = __builtin_ctz(todo);
      const int slot = __builtin_amdgcn_readlane(ad.slot, lead), rank = __builtin_amdgcn_readlane(ad.rank, lead);
      const uint32_t mine = (uint32_t)__ballot(ad.slot == slot && ad.rank > 0) & 0xFFFFu;
      const uint16_t* a = g.a + (int64_t)slot * g.max_rank * K + kq;
      f4v acc[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) acc[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
      // At most eight weight operands in flight.
      constexpr int AT = RT > 8 / kDownChunks ? 8 / kDownChunks : RT;
#pragma unroll
      for (int t0 = 0; t0 < RT; t0 += AT) {
        bf8 w[kDownChunks][AT];
#pragma unroll
        for (int u = 0; u < kDownChunks; ++u)
#pragma unroll
          for (int t = 0; t < AT; ++t)
            w[u][t] = *(const bf8*)(a + (int64_t)min(16 * (t0 + t) + (lane & 15), rank - 1) * K +
                                    32 * min(c0 + kDownWaves * u, chunks - 1));
        if (t0 == 0 && todo == with) {
#pragma unroll
          for (int u = 0; u < kDownChunks; ++u) split3(x0[u], x1[u], p[u]);
          if (c0 + kDownWaves * kDownChunks < chunks) load_x(c0 + kDownWaves * kDownChunks);
        }
#pragma unroll
        for (int u = 0; u < kDownChunks; ++u)
          if (c0 + kDownWaves * u < chunks)  // uniform
#pragma unroll
            for (int t = 0; t < AT; ++t)
#pragma unroll
              for (int i = 2; i >= 0; --i)
                acc[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p[u][i], w[u][t], acc[t0 + t], 0, 0, 0);
      }
      const float gain = g.scale[slot];
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (((mine >> (4 * (lane >> 4) + r)) & 1) && 16 * t + (lane & 15) < rank)
            sum[t][r] += acc[t][r] * gain;
      todo &= ~mine;
    }
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) sT[wave][(4 * (lane >> 4) + r) * LDS_LD + 16 * t + (lane & 15)] = sum[t][r];
  wg_lds_barrier();
  // Eight ranks of a row per thread: the waves' sums, split, one 16-byte store a part.
  const int ldt = lora_ldt(g.max_rank);
  for (int i = tid; i < kDownRows * 2 * RT; i += kDownWaves * 64) {
    const int r = i % kDownRows, c = i / kDownRows * 8;
    if (c >= ldt) break;
    f4v v[2];
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      const float* s = &sT[0][r * LDS_LD + c + h];
      constexpr int W = kDownRows * LDS_LD;
      float d = 0.0f;
#pragma unroll
      for (int w = 0; w < kDownWaves; ++w) d += s[w * W];
      v[h >> 2][h & 3] = d;
    }
    bf8 p[3];
    split3(v[0], v[1], p);
    const int64_t m = m0 + r;
#pragma unroll
    for (int k = 0; k < 3; ++k)
      *(bf8*)((uint16_t*)g.t + lora_t_index(m >> 5, k, c >> 4, (int)(m & 31) + 32 * ((c >> 3) & 1), ldt)) = p[k];
  }
}

}  // namespace

bool lora_few_rows(int64_t M) { return M <= 320; }

size_t lora_scratch_bytes(int64_t M, int max_rank) {
  return lora_few_rows(M) ? (size_t)M * max_rank * 4 : (size_t)(M + 31) / 32 * 32 * 3 * lora_ldt(max_rank) * 2;
}

hipError_t launch_lora_down(const LoraArgs& g, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  if (lora_few_rows(g.M)) {
    auto kern = g.K <= 512 ? k_lora_down_rows<1> : g.K <= 1024 ? k_lora_down_rows<2>
                : g.K <= 2048                    ? k_lora_down_rows<4>
                                                 : k_lora_down_rows<0>;
    hipLaunchKernelGGL(kern, dim3((unsigned)g.M), dim3(256), 0, s, g);
    return hipGetLastError();
  }
  if (g.xq) {
    const hipError_t rc = launch_quantize_rows(g.x, g.K, (int)g.M, nullptr, g.K, g.xq, g.K, g.xa, g.err, s);
    if (rc != hipSuccess) return rc;
  }
  auto kern = g.max_rank <= 16   ? k_lora_down_tile<1>
              : g.max_rank <= 32 ? k_lora_down_tile<2>
              : g.max_rank <= 64 ? k_lora_down_tile<4>
                                 : k_lora_down_tile<8>;
  hipLaunchKernelGGL(kern, dim3((unsigned)((g.M + kDownRows - 1) / kDownRows)),
                     dim3(kDownWaves * 64), 0, s, g);
  return hipGetLastError();
}

template <int NW, int KSW>
static hipError_t launch_rows(const GemmArgs& g, const LoraArgs& l, hipStream_t s) {
  const int rows = (g.M + kUpRows - 1) / kUpRows;
  if (g.N >= 1024)
    hipLaunchKernelGGL((k_lora_rows<NW, 2, KSW>), dim3((g.N + 31) / 32, rows), dim3(NW * 64), 0, s, g, l);
  else
    hipLaunchKernelGGL((k_lora_rows<4, 1, KSW * NW / 4>), dim3((g.N + 15) / 16, rows), dim3(256), 0, s, g, l);
  return hipGetLastError();
}

hipError_t launch_lora_linear(const GemmArgs& g, const LoraArgs& l, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  if (!lora_few_rows(g.M)) return launch_gemm_tile_lora(g, l, s);
  return g.K <= 512 ? launch_rows<4, 2>(g, l, s) : launch_rows<8, 4>(g, l, s);
}

}  // namespace mh
