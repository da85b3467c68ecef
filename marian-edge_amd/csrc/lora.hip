// lora.hip — the low-rank adapters of many requests beside a shared Q8 layer.
//
//   y_m = W x_m (Q8) + b + c_s B_s (A_s x_m),  s = slot of row m (negative: no adapter)
//
// A_s is [rank_s, K], B_s [N, rank_s] (bf16, stored max_rank apart), x fp32.
// Two launches: t = c_s A_s x_m (and the rows' quantization when the caller has
// none), then the int8 product with B_s t added in its epilogue.  Fusing both
// repeats A_s x_m in every column workgroup, which pays for the fewest rows only
// (one launch, k_lora_one); a third launch for the addition would read and write the
// output once more.
//
// Few rows (a decode step): neighbouring rows belong to different requests, so
// each row multiplies with its own A_s and B_s on the vector units and reads them
// once; those reads are what is left to do.  Many rows (prompts): a 16- or 32-row
// tile mostly holds one request's rows, so A_s and B_s are matrix-core operands,
// once per distinct slot of the tile; a row keeps the result of its own slot, by
// selection and not by a product with zero, so that an infinite weight reaches no
// other request's rows.  fp32 operands go to the bf16 matrix cores as three parts of
// 8 bits each, which hold all 24 bits of a value: products are exact and sums fp32.
// A zero part times an infinite weight is NaN where the value times it is infinite:
// sums that are not finite are formed again from the values (cold code; finding them
// costs an addition an output, 8000 rows, K 2048, N 512, rank 64: 68.3 us, 67.8 without).
#include "device_common.h"
#include "kernels.h"
#include "lora_device.h"

#include <algorithm>

namespace mh {
namespace {

// ---------------------------------------------------------------------------
// Few rows, first product: one workgroup of NW waves per row.  Each wave holds
// the row (lane l: values 8l + 512 j ...) and takes four ranks at a time; NW is
// as many waves as ranks / 4 keep busy, so that a row's weights are requested at
// once (200 rows, K 1536, rank 64: 9.6 us with 4 waves, 6.4 with 16).  KJ: row pieces in
// registers (K up to 512 KJ); 0: read again for each batch.
// ---------------------------------------------------------------------------
constexpr int kDownBatch = 4;  // ranks whose weights are in flight together

template <int KJ, int NW>
__global__ __launch_bounds__(NW * 64) void k_lora_down_rows(LoraArgs g) {
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

  for (int r = a.rank + tid; r < g.max_rank; r += NW * 64) t[r] = 0.0f;
  const uint16_t* wa = g.a + (int64_t)a.slot * g.max_rank * K;
  for (int r0 = wave; r0 < a.rank; r0 += NW * kDownBatch) {
    float s[kDownBatch];
#pragma unroll
    for (int b = 0; b < kDownBatch; ++b) s[b] = 0.0f;
    auto piece = [&](int j, const f4v (&p)[2]) {
      const int k = min(512 * j + 8 * lane, K - 8);
      uint4 w[kDownBatch];
#pragma unroll
      for (int b = 0; b < kDownBatch; ++b) w[b] = *(const uint4*)(wa + (int64_t)min(r0 + NW * b, a.rank - 1) * K + k);
#pragma unroll
      for (int b = 0; b < kDownBatch; ++b) {
        const uint32_t d[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
        float e = s[b];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          e = __builtin_fmaf(p[c >> 1][2 * (c & 1)], __uint_as_float(d[c] << 16), e);
          e = __builtin_fmaf(p[c >> 1][2 * (c & 1) + 1], __uint_as_float(d[c] & 0xFFFF0000u), e);
        }
        s[b] = 512 * j + 8 * lane < K ? e : s[b];  // past K: weights of another column
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
      if (lane == 0 && r0 + NW * b < a.rank) t[r0 + NW * b] = sum * gain;
    }
  }
}

// ---------------------------------------------------------------------------
// Few rows, the layer: 16 rows and 16 CT columns per workgroup, its four waves
// split K (wave w: k-steps w, w + 4, ..., two held at a time) and their exact i32
// partials meet in LDS.  The rows' second products go two neighbouring lanes to an
// output, 8 ranks (16 bytes of B) each a time; the first ones are requested before the
// layer's products start, and the sums meet the dequantized outputs in LDS.  Each
// row reads its own B, from the L2: 300 rows, N 2048, rank 64, 79 MB, bound it (us a
// call, K 512: 19.0; four lanes an output 19.5, eight, with whole rows of B a wave
// but 64 registers of it a thread, 25.2; rank 16: 11.4, 14.0, 23.4).  Few rows or
// ranks: the two launches.
// ---------------------------------------------------------------------------
constexpr int kUpRows = 16;

template <int CT>
__global__ __launch_bounds__(256) void k_lora_rows(GemmArgs g, LoraArgs l) {
  touch_kernargs<sizeof(GemmArgs) + sizeof(LoraArgs)>();
  constexpr int NW = 4, KSW = 2, PL = 2;  // waves, k-steps held, lanes per output
  constexpr int NT = NW * 64, COLS = 16 * CT, LDC = COLS + 1;
  constexpr int PER = kUpRows * COLS / NT;  // outputs per thread
  constexpr int ITEMS = PER * PL;           // pieces of 8 ranks per thread
  static_assert(PER >= 1 && PER * NT == kUpRows * COLS, "whole outputs");
  __shared__ int32_t sP[NW][kUpRows * LDC];
  __shared__ float sD[kUpRows * LDC];
  __shared__ __attribute__((aligned(16))) float sT[kUpRows * (kLoraMaxRank + 4)];
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

  // Piece i: of output tid / PL + i NT / PL, row-major; ranks from 8 (tid % PL).
  const int R = l.max_rank, r8 = 8 * (tid % PL), ldt = R + 4;
  RowAdapter ad[ITEMS];
  uint4 w[ITEMS];
  const uint16_t* b[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int o = tid / PL + i * (NT / PL), row = min(m0 + o / COLS, g.M - 1), n = min(n0 + o % COLS, g.N - 1);
    ad[i] = row_adapter(l, l.slot_of_row[row], nullptr);
    b[i] = l.b + ((int64_t)ad[i].slot * g.N + n) * R;
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) w[i] = *(const uint4*)(b[i] + min(r8, R - 8));
  // t's rows into LDS, 4 floats between them.
  for (int i = tid; i < kUpRows * R / 4; i += NT) {
    const int row = i / (R / 4), r = i % (R / 4) * 4;
    *(f4v*)(sT + row * ldt + r) = *(const f4v*)((const float*)l.t + (int64_t)min(m0 + row, g.M - 1) * R + r);
  }
  // This thread's outputs: column n, rows tid / COLS + k (NT / COLS).
  const int n = min(n0 + tid % COLS, g.N - 1);
  const float wm = g.wmult[n], bias = g.bias[n];
  float am[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) am[k] = g.a[min(m0 + tid / COLS + k * (NT / COLS), g.M - 1)];

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
  for (int i = 0; i < ITEMS; ++i) {
    const int o = tid / PL + i * (NT / PL), row = o / COLS;
    float d = 0.0f;
    auto add = [&](uint4 v, int r) {  // ranks past the slot's: weights of any value, not used
      const f4v t0 = *(const f4v*)(sT + row * ldt + r), t1 = *(const f4v*)(sT + row * ldt + r + 4);
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float wv = __uint_as_float(c & 1 ? u[c >> 1] & 0xFFFF0000u : u[c >> 1] << 16);
        const float e = __builtin_fmaf(c < 4 ? t0[c & 3] : t1[c & 3], wv, d);
        d = r + c < ad[i].rank ? e : d;
      }
    };
    add(w[i], min(r8, R - 8));
    if (r8 >= R) d = 0.0f;  // R 8: one piece
    for (int r = r8 + 8 * PL; r < R; r += 8 * PL) add(*(const uint4*)(b[i] + r), r);
    d += __int_as_float(dpp_mov<0xB1>(__float_as_int(d)));  // the output's other lane
    if (tid % PL == 0) sD[row * LDC + o % COLS] = d;
  }
  wg_lds_barrier();

#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int row = tid / COLS + k * (NT / COLS), at = row * LDC + tid % COLS;
    int32_t iv = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) iv += sP[i][at];
    float y = dequant(iv, am[k], wm, bias) + sD[at];
    if (l.relu) y = lora_relu(y);
    if (m0 + row < g.M && n0 + tid % COLS < g.N) l.out[(int64_t)(m0 + row) * g.N + n] = y;
  }
}

// ---------------------------------------------------------------------------
// The fewest rows: both products, and the quantization when the caller has no
// codes, in one launch of 16 CT columns a workgroup (one row, K 512, N 2048, rank 8:
// 5.2 us, a chain of round trips: x, slot, rank, A, B).  Each workgroup repeats its
// rows' first products, which costs less than a second launch and the gap before
// it while they are few (lora_one_launch).  The waves share (row, four ranks)
// items of the first product.
// ---------------------------------------------------------------------------
constexpr int kOneRows = 8;    // of the matrix cores' 16
constexpr int kOneRanks = 64;  // rows times max_rank
constexpr int kOneMaxK = 2048;

template <int NW, int CT, int KSW>
__global__ __launch_bounds__(NW * 64) void k_lora_one(GemmArgs g, LoraArgs l) {
  touch_kernargs<sizeof(GemmArgs) + sizeof(LoraArgs)>();
  constexpr int NT = NW * 64, COLS = 16 * CT, LDC = COLS + 1;
  constexpr int MAXK = NW * KSW * 64;
  static_assert(kOneRows * COLS <= NT, "an output per thread at most");
  __shared__ int32_t sP[NW][kOneRows * LDC];
  __shared__ __attribute__((aligned(16))) float sT[kOneRanks];  // row m's from m max_rank
  __shared__ __attribute__((aligned(16))) int8_t sX[kOneRows * (MAXK + 16)];  // codes made here
  __shared__ float sM[kOneRows];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int M = g.M, K = g.K, n0 = blockIdx.x * COLS, ksteps = K >> 6, kq = (lane >> 4) * 16;
  const int8_t* br[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) br[c] = g.W + (int64_t)min(n0 + 16 * c + (lane & 15), g.N - 1) * K + kq;
  v4i bf[KSW][CT];
#pragma unroll
  for (int i = 0; i < KSW; ++i)
#pragma unroll
    for (int c = 0; c < CT; ++c) bf[i][c] = *(const v4i*)(br[c] + min(wave + NW * i, ksteps - 1) * 64);
  const int n = min(n0 + tid % COLS, g.N - 1);
  const float wm = g.wmult[n], bias = g.bias[n];

  // ---- the rows' codes ----
  const int ldx = K + 16;  // of sX: consecutive rows start in other banks
  if (!g.A) {
    for (int m = wave; m < M; m += NW) {
      const float* x = l.x + (int64_t)m * K;
      f4v v[MAXK / 256];
      float mx = 0.0f;
      bool bad = false;
#pragma unroll
      for (int j = 0; j < MAXK / 256; ++j)
        if (256 * j < K) v[j] = *(const f4v*)(x + min(256 * j + 4 * lane, K - 4));
#pragma unroll
      for (int j = 0; j < MAXK / 256; ++j)
        if (256 * j < K)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            mx = fmaxf(mx, fabsf(v[j][c]));
            bad |= !(fabsf(v[j][c]) < INFINITY);
          }
      const float a = row_multiplier(wave_max(mx));
      if (lane == 0) sM[m] = a;
      if (__any(bad) && lane == 0 && l.err) *l.err = 1;
#pragma unroll
      for (int j = 0; j < MAXK / 256; ++j)
        if (256 * j + 4 * lane < K)
          *(uint32_t*)(sX + m * ldx + 256 * j + 4 * lane) = quantize_pack4(v[j][0], v[j][1], v[j][2], v[j][3], a);
    }
  }

  // ---- the first product: items of a row and four ranks ----
  const int quads = (l.max_rank + 3) >> 2;
  for (int i = wave; i < M * quads; i += NW) {
    const int m = i / quads, r0 = i % quads * 4;
    const RowAdapter a = row_adapter(l, l.slot_of_row[m], l.err);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r0 < a.rank) {
      const float* x = l.x + (int64_t)m * K;
      const uint16_t* w = l.a + (int64_t)a.slot * l.max_rank * K;
#pragma unroll 2
      for (int k0 = 0; k0 < K; k0 += 512) {
        const int k = min(k0 + 8 * lane, K - 8);
        const bool in = k0 + 8 * lane < K;
        const f4v x0 = *(const f4v*)(x + k), x1 = *(const f4v*)(x + k + 4);
        uint4 wr[4];
#pragma unroll
        for (int b = 0; b < 4; ++b) wr[b] = *(const uint4*)(w + (int64_t)min(r0 + b, a.rank - 1) * K + k);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t d[4] = {wr[b].x, wr[b].y, wr[b].z, wr[b].w};
          float e = s[b];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const f4v& xv = c < 2 ? x0 : x1;
            e = __builtin_fmaf(xv[2 * (c & 1)], __uint_as_float(d[c] << 16), e);
            e = __builtin_fmaf(xv[2 * (c & 1) + 1], __uint_as_float(d[c] & 0xFFFF0000u), e);
          }
          s[b] = in ? e : s[b];
        }
      }
    }
    const float gain = l.scale[a.slot];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const float sum = tree_combine_wave(s[b]);
      if (lane == 0 && r0 + b < l.max_rank) sT[m * l.max_rank + r0 + b] = r0 + b < a.rank ? sum * gain : 0.0f;
    }
  }
  wg_lds_barrier();

  // ---- the layer ----
  v4i acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = v4i{0, 0, 0, 0};
  const int m = min(lane & 15, M - 1);
#pragma unroll
  for (int i = 0; i < KSW; ++i) {
    const int s = min(wave + NW * i, ksteps - 1);
    const v4i v = g.A ? *(const v4i*)(g.A + (int64_t)m * g.lda + kq + s * 64) : *(const v4i*)(sX + m * ldx + kq + s * 64);
    const v4i a = keep_or_zero(v, wave + NW * i < ksteps);
#pragma unroll
    for (int c = 0; c < CT; ++c) acc[c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, bf[i][c], acc[c], 0, 0, 0);
  }
  if (lane < 16 * kOneRows / 4) {  // 16 lanes hold four rows
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
      for (int r = 0; r < 4; ++r) sP[wave][((lane >> 4) * 4 + r) * LDC + 16 * c + (lane & 15)] = acc[c][r];
  }
  wg_lds_barrier();
  const int row = tid / COLS, at = row * LDC + tid % COLS;
  if (row >= M || n0 + tid % COLS >= g.N) return;
  int32_t iv = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) iv += sP[w][at];
  float y = dequant(iv, g.A ? g.a[row] : sM[row], wm, bias);
  const RowAdapter a = row_adapter(l, l.slot_of_row[row], nullptr);
  const uint16_t* b = l.b + ((int64_t)a.slot * g.N + n) * l.max_rank;
  const float* t = sT + row * l.max_rank;
  float d = 0.0f;
  for (int r8 = 0; r8 < a.rank; r8 += 8) {
    const uint4 w = *(const uint4*)(b + r8);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float e = __builtin_fmaf(t[r8 + c], __uint_as_float(c & 1 ? u[c >> 1] & 0xFFFF0000u : u[c >> 1] << 16), d);
      d = r8 + c < a.rank ? e : d;
    }
  }
  y += d;
  if (l.relu) y = lora_relu(y);
  l.out[(int64_t)row * g.N + n] = y;
}

// ---------------------------------------------------------------------------
// Many rows, first product: 16 rows per workgroup, its NW waves split K in
// chunks of 32, RT tiles of 16 ranks.  v_mfma_f32_16x16x32_bf16: lane l holds k
// 8 (l / 16) .. + 8 of x's row l % 16 and of A's row l % 16, and of the result
// column (rank) l % 16, rows 4 (l / 16) + r.  A wave reads and splits its x once, 512
// columns of the row at a time, and multiplies it with each slot of the tile; its two
// chunks are neighbours, whole cache lines of A.  blockIdx.y: RT tiles of ranks each;
// the first of them quantizes the rows when the caller has no codes, a row per wave,
// whose second read of x is the cache's (a call of 1459 rows, K 384, N 384, rank 40,
// 15.8 us, 17.7 with a launch of its own for the codes).
//
// A workgroup is a chain of round trips (slot, rank, weights, the waves' sums) that two
// workgroups a CU hide in part: 16384 x 512, rank 32: 16 us, 2.3 TB/s; a call of 4200
// rows, K 2048, N 512, rank 24: 37.6 us, 41.1 with four waves a workgroup.
// ---------------------------------------------------------------------------
constexpr int kDownRows = 16;
constexpr int kDownChunks = 2;  // chunks of a wave held at once

// One wave: row m's codes and multiplier, as the row quantization makes them.
__device__ __forceinline__ void quantize_row(const LoraArgs& g, int64_t m, int lane) {
  constexpr int COLS = 1024;  // at a time; a longer row is read again for its codes
  const int K = g.K;
  const float* x = g.x + m * K;
  f4v v[COLS / 256];
  auto load = [&](int k0) {
#pragma unroll
    for (int j = 0; j < COLS / 256; ++j) v[j] = *(const f4v*)(x + min(k0 + 256 * j + 4 * lane, K - 4));
  };
  float mx = 0.0f;
  bool bad = false;
  for (int k0 = 0; k0 < K; k0 += COLS) {
    load(k0);
#pragma unroll
    for (int j = 0; j < COLS / 256; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        mx = fmaxf(mx, fabsf(v[j][c]));
        bad |= !(fabsf(v[j][c]) < INFINITY);
      }
  }
  const float a = row_multiplier(wave_max(mx));
  if (lane == 0) g.xa[m] = a;
  if (__any(bad) && lane == 0 && g.err) *g.err = 1;
  for (int k0 = 0; k0 < K; k0 += COLS) {
    if (K > COLS) load(k0);
#pragma unroll
    for (int j = 0; j < COLS / 256; ++j) {
      const int k = k0 + 256 * j + 4 * lane;
      if (k < K) *(uint32_t*)(g.xq + m * K + k) = quantize_pack4(v[j][0], v[j][1], v[j][2], v[j][3], a);
    }
  }
}

// One thread: row m's product with rank r of its adapter, in fp32.
__device__ __forceinline__ float down_product(const LoraArgs& g, int64_t m, int r) {
  const RowAdapter a = row_adapter(g, g.slot_of_row[m], nullptr);
  const float* x = g.x + m * g.K;
  const uint16_t* w = g.a + ((int64_t)a.slot * g.max_rank + r) * g.K;
  float s = 0.0f;
  for (int k = 0; k < g.K; ++k) s = __builtin_fmaf(x[k], bf16_to_f32(w[k]), s);
  return s * g.scale[a.slot];
}

template <int RT, int NW>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(4))) void k_lora_down_tile(LoraArgs g) {
  touch_kernargs<sizeof(LoraArgs)>();
  constexpr int LDS_LD = 16 * RT + 1;
  __shared__ float sT[NW][kDownRows * LDS_LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t m0 = (int64_t)blockIdx.x * kDownRows;
  const int K = g.K, kq = 8 * (lane >> 4), chunks = K >> 5, r0 = blockIdx.y * (16 * RT);
  const int64_t row = m0 + (lane & 15) < g.M ? m0 + (lane & 15) : g.M - 1;
  const float* x = g.x + row * K + kq;
  f4v x0[kDownChunks], x1[kDownChunks];
  auto load_x = [&](int c0) {  // past K: the last chunk again
#pragma unroll
    for (int u = 0; u < kDownChunks; ++u) {
      const int c = min(c0 + u, chunks - 1);
      x0[u] = *(const f4v*)(x + 32 * c);
      x1[u] = *(const f4v*)(x + 32 * c + 4);
    }
  };
  load_x(kDownChunks * wave);
  const RowAdapter ad = row_adapter(g, m0 + (lane & 15) < g.M ? g.slot_of_row[row] : -1, g.err);
  const uint32_t with = (uint32_t)__ballot(ad.rank > 0) & 0xFFFFu;  // rows with an adapter
  if (g.xq && blockIdx.y == 0)
    for (int r = wave; r < kDownRows && m0 + r < g.M; r += NW) quantize_row(g, m0 + r, lane);
  f4v sum[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) sum[t] = f4v{0.0f, 0.0f, 0.0f, 0.0f};
  for (int c0 = kDownChunks * wave; with && c0 < chunks; c0 += NW * kDownChunks) {
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
            w[u][t] = *(const bf8*)(a + (int64_t)min(r0 + 16 * (t0 + t) + (lane & 15), rank - 1) * K +
                                    32 * min(c0 + u, chunks - 1));
        if (t0 == 0 && todo == with) {
#pragma unroll
          for (int u = 0; u < kDownChunks; ++u) split3(x0[u], x1[u], p[u]);
          if (c0 + NW * kDownChunks < chunks) load_x(c0 + NW * kDownChunks);
        }
#pragma unroll
        for (int u = 0; u < kDownChunks; ++u)
          if (c0 + u < chunks)  // uniform
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
          if (((mine >> (4 * (lane >> 4) + r)) & 1) && r0 + 16 * t + (lane & 15) < rank)
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
  for (int i = tid; i < kDownRows * 2 * RT; i += NW * 64) {
    const int r = i % kDownRows, c = i / kDownRows * 8;
    if (r0 + c >= ldt) break;
    auto sum = [&](int h) {
      const float* s = &sT[0][r * LDS_LD + c + h];
      constexpr int W = kDownRows * LDS_LD;
      float d = 0.0f;
#pragma unroll
      for (int w = 0; w < NW; ++w) d += s[w * W];
      return d;
    };
    f4v v[2];
#pragma unroll
    for (int h = 0; h < 8; ++h) v[h >> 2][h & 3] = sum(h);
    bf8 p[3];
    split3(v[0], v[1], p);
    const int64_t m = m0 + r;
    auto at = [&](int part) {
      return (uint16_t*)g.t + lora_t_index(m >> 5, part, (r0 + c) >> 4, (int)(m & 31) + 32 * ((c >> 3) & 1), ldt);
    };
#pragma unroll
    for (int k = 0; k < 3; ++k) *(bf8*)at(k) = p[k];
    float all = 0.0f;
#pragma unroll
    for (int h = 0; h < 8; ++h) all += v[h >> 2][h & 3];
    if (!(fabsf(all) < INFINITY)) {  // an infinite weight times a zero part of x made NaN: from x itself
#pragma unroll 1
      for (int h = 0; h < 8; ++h) {
        if (fabsf(sum(h)) < INFINITY) continue;
        const float d = down_product(g, m, r0 + c + h);
        uint32_t q[3] = {__float_as_uint(d), 0, 0};  // an infinity or NaN is its first part alone
        if (fabsf(d) < INFINITY) split3_parts(d, q);
        for (int k = 0; k < 3; ++k) at(k)[h] = (uint16_t)(q[k] >> 16);
      }
    }
  }
}

}  // namespace

// A row's own A and B cost M rank (K + N) values from the L2; tiles cost a chain per
// distinct slot of their rows.  us a call, rows | tiles, of rows in runs and of rows in
// turn: K 2048, N 512, rank 64: 160 rows 15 | 21 and 16 | 61, 320 24 | 22 and 26 | 59, 1000
// 49 | 25 and 53 | 61; K 512, N 2048, rank 16: 320 12 | 11 and 12 | 21, 500 14 | 11 and 14 | 23,
// 1000 22 | 12 and 22 | 24; K 512, N 512, rank 16: 1000 11 | 11 and 11 | 22.  Which they are
// the host cannot see.  Past 320 rows the second bound keeps rows in runs near the tiles' time;
// rows in turn of high rank pay for it, 59 us instead of 26 at
// 321 of rank 64 and K 2048, up to about 1000, where both take as long.
static bool lora_few_rows(const LoraArgs& g) {
  return g.M <= 320 || (g.M <= 1024 && g.M * g.max_rank * (g.K + g.N) <= 1 << 25);
}

// t of few rows (4 bytes a value) takes less.
size_t lora_scratch_bytes(int64_t M, int max_rank) { return (size_t)(M + 31) / 32 * 32 * 3 * lora_ldt(max_rank) * 2; }

template <int NW>
static hipError_t launch_down_rows_k(const LoraArgs& g, hipStream_t s) {
  auto kern = g.K <= 512    ? k_lora_down_rows<1, NW>
              : g.K <= 1024 ? k_lora_down_rows<2, NW>
              : g.K <= 1536 ? k_lora_down_rows<3, NW>
              : g.K <= 2048 ? k_lora_down_rows<4, NW>
                            : k_lora_down_rows<0, NW>;
  hipLaunchKernelGGL(kern, dim3((unsigned)g.M), dim3(NW * 64), 0, s, g);
  return hipGetLastError();
}
static hipError_t launch_down_rows(const LoraArgs& g, hipStream_t s) {
  return g.max_rank <= 16   ? launch_down_rows_k<4>(g, s)
         : g.max_rank <= 32 ? launch_down_rows_k<8>(g, s)
                            : launch_down_rows_k<16>(g, s);
}

// While 16-row tiles do not fill the chip, a workgroup per 16 ranks too, and as many
// waves as a long row has work for: each (512 or 1024 columns, slot) is a round trip
// to memory (500 rows, K 2048, rank 64, us: 26.5 with eight waves and all ranks, 15.6
// with a workgroup per 16 ranks; 1459 rows, rank 16, eight waves | 16: K 512 11.5 | 12.7,
// K 2048 25.9 | 21.8).  More tiles: two or four steps of 16 ranks a workgroup, which read
// x fewer times (K 512, rank 64, one | two | four: 1459 rows 15.6 | 16.0 | 18.4, 5000 27.1 |
// 24.2 | 23.9, 9000 42.7 | 38.2 | 35.0).
static hipError_t launch_down_tile(const LoraArgs& g, hipStream_t s) {
  const int64_t tiles = (g.M + kDownRows - 1) / kDownRows;
  const int steps = lora_ldt(g.max_rank) / 16;
  const int rt = steps == 1 || tiles < 256 ? 1 : steps == 2 || tiles < 512 ? 2 : 4;
  const bool wide = rt == 1 && g.K > 1024 && tiles < 1 << 22;  // a launch is less than 2^32 threads
  auto kern = wide      ? k_lora_down_tile<1, 16>
              : rt == 1 ? k_lora_down_tile<1, 8>
              : rt == 2 ? k_lora_down_tile<2, 8>
                        : k_lora_down_tile<4, 8>;
  hipLaunchKernelGGL(kern, dim3((unsigned)tiles, (steps + rt - 1) / rt), dim3(wide ? 1024 : 512), 0, s, g);
  return hipGetLastError();
}

hipError_t launch_lora_down(const LoraArgs& g, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  return lora_few_rows(g) ? launch_down_rows(g, s) : launch_down_tile(g, s);
}

// Every workgroup repeats the M rank first products, four at a time on four or
// eight waves: few of them, and few columns.  us a call, one launch | two (K 512, N 2048): 1 row of rank 8 8.0 |
// 11.1, 4 of 16 8.5 | 11.4, 2 of 64 14.3 | 11.7, 8 of 16 13.8 | 11.2; K 2048, N 512: 2
// rows of 16 8.1 | 11.3, 4 of 16 11.9 | 11.2, 1 of 64 12.3 | 11.9.
bool lora_one_launch(int64_t M, int64_t K, int max_rank) {
  static_assert(kOneRows == kOneRanks / 8, "max_rank is 8 at least");
  return M * max_rank <= kOneRanks && K <= kOneMaxK && M * max_rank * K <= 65536;
}

hipError_t launch_lora_one(const GemmArgs& g, const LoraArgs& l, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  if (!lora_one_launch(g.M, g.K, l.max_rank)) return hipErrorInvalidValue;
  const dim3 wide((g.N + 31) / 32), narrow((g.N + 15) / 16);
  if (g.K <= 512)
    hipLaunchKernelGGL(g.N >= 1024 ? (k_lora_one<4, 2, 2>) : (k_lora_one<4, 1, 2>), g.N >= 1024 ? wide : narrow, dim3(256), 0, s, g, l);
  else
    hipLaunchKernelGGL(g.N >= 1024 ? (k_lora_one<8, 2, 4>) : (k_lora_one<4, 1, 8>), g.N >= 1024 ? wide : narrow,
                       dim3(g.N >= 1024 ? 512 : 256), 0, s, g, l);
  return hipGetLastError();
}

// 32 columns a workgroup, 16 where they are few (us a call, 300 rows, rank 16, 16 | 32
// columns: K 512, N 384 10.5 | 10.6; K 2048, N 2048 25.0 | 20.8).
hipError_t launch_lora_linear(const GemmArgs& g, const LoraArgs& l, hipStream_t s) {
  if (g.M <= 0) return hipSuccess;
  if (!lora_few_rows(l)) return launch_gemm_tile_lora(g, l, s);
  const int rows = (g.M + kUpRows - 1) / kUpRows;
  if (g.N >= 1024)
    hipLaunchKernelGGL(k_lora_rows<2>, dim3((g.N + 31) / 32, rows), dim3(256), 0, s, g, l);
  else
    hipLaunchKernelGGL(k_lora_rows<1>, dim3((g.N + 15) / 16, rows), dim3(256), 0, s, g, l);
  return hipGetLastError();
}

}  // namespace mh
