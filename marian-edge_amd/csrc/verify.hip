// verify.hip — drafted ids against the target's distribution, from given numbers.
//
// With p the distribution that a target row's settings leave and q the one its draft was drawn from, a draft t is
// accepted with probability min(1, p(t) / q(t)): while u q(t) < p(t).  At the first draft that is not, an id is drawn from
// max(p - q, 0), so that every id comes out with probability p whatever q is; after all drafts one from p of the last row.
// Without draft logits q is 1 at the drafted id (a draft that was looked up, not drawn).
//
// What the settings keep of each row (a prefix in the order of logits) and its mass come from the pass that also draws
// single ids; this kernel, a workgroup per request, looks at the drafts' shares, then goes over one row, or a row and
// its draft row, twice: sums of every 256 ids, then the group that the number falls into.  Weights are multiples of
// 2^-51, so their sums are exact and the drawn id does not depend on the launch.
#include "device_common.h"
#include "kernels.h"
#include "mass.h"

namespace mh {
namespace {

constexpr int kThreads = 1024;
constexpr int kVerifyWaves = kThreads / 64;
constexpr int kSegs = kSampleMaxIds / 256;

// One row's distribution.
template <bool BF16>
struct Row {
  const void* base;
  RowKept k;
  double share;  // of a unit of mass
  Octaves scale;
  __device__ void set(const void* logits, int64_t first, const RowKept& kept, float temperature) {
    base = BF16 ? (const void*)((const uint16_t*)logits + first) : (const void*)((const float*)logits + first);
    k = kept;
    share = k.total ? 1.0 / (double)k.total : 0.0;
    const double per_logit = fmax(1.4426950408889634 / (double)temperature, 0x1p-900);
    scale = {per_logit, -60.0 / per_logit};
    if (k.flags & kKeptInf) k.max = 0.0f;
  }
  __device__ __forceinline__ float value(int id) const {
    const float v = BF16 ? bf16_to_f32(((const uint16_t*)base)[id]) : ((const float*)base)[id];
    return v;
  }
  // p of an id whose logit is v.
  __device__ __forceinline__ double p(float v, int id, const uint64_t* exp2) const {
    if (k.flags & kKeptOne) return id == k.border_id ? 1.0 : 0.0;
    if (k.flags & kKeptInf) v = v == INFINITY ? 0.0f : -INFINITY;
    if (!(v > k.border_v || (v == k.border_v && id <= k.border_id))) return 0.0;
    return (double)mass_of_steps(octave_steps((double)v - (double)k.max, scale), exp2) * share;
  }
};

template <bool BF16>
__global__ __launch_bounds__(kThreads) void k_verify(VerifyArgs g) {
  __shared__ uint64_t exp2[32];
  __shared__ uint64_t seg[kSegs];
  __shared__ int stop;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int b = blockIdx.x;
  const int row0 = g.cu[b], end = g.cu[b + 1];
  const bool ok = row0 >= 0 && end >= row0 && end <= g.rows && end - row0 <= g.max_rows;
  if (!ok || end == row0) {
    if (t == 0) {
      if (!ok && g.err) *g.err = 1;
      g.accepted[b] = 0;
    }
    return;
  }
  const int drafts = end - row0 - 1;
  const float temperature = g.temperature ? g.temperature[b] : 1.0f;
  if (t < 32) exp2[t] = kSampleExp2Tab[t] + ((uint64_t)kMassBits << 52);
  if (t == 0) stop = drafts;
  __syncthreads();

  // ---- the drafts, a thread each ----
  auto source = [&](int r) { return g.draft_row ? g.draft_row[r] : r; };
  for (int i = t; i < drafts; i += kThreads) {
    const int r = row0 + i, id = g.drafts[r];
    const float u = g.u[r];
    bool in = (uint32_t)id < (uint32_t)g.V && u >= 0.0f && u < 1.0f, accept = false;
    if (g.draft_logits) in = in && (uint32_t)source(r) < (uint32_t)g.draft_rows;
    if (!in && g.err) *g.err = 1;
    if (in) {
      Row<BF16> target;
      target.set(g.logits, r * g.ld, g.kept[r], temperature);
      double q = 1.0;
      if (g.draft_logits) {
        Row<BF16> draft;
        draft.set(g.draft_logits, source(r) * g.ld_draft, g.kept[g.rows + r], temperature);
        q = draft.p(draft.value(id), id, exp2);
      }
      accept = (double)u * q < target.p(target.value(id), id, exp2);
    }
    if (!accept) atomicMin(&stop, i);
  }
  __syncthreads();
  const int accepted = stop, r = row0 + accepted;
  Row<BF16> target, draft;
  target.set(g.logits, r * g.ld, g.kept[r], temperature);
  draft = target;
  int without = -1;    // an id whose q is 1
  bool less = false;   // q from `draft`
  if (accepted < drafts) {
    if (!g.draft_logits) {
      without = g.drafts[r];
    } else if ((uint32_t)source(r) < (uint32_t)g.draft_rows) {
      draft.set(g.draft_logits, source(r) * g.ld_draft, g.kept[g.rows + r], temperature);
      less = true;
    }
  }
  float u = g.u_draw[b];
  if (!(u >= 0.0f && u < 1.0f)) {
    if (t == 0 && g.err) *g.err = 1;
    u = 0.0f;
  }
  // The weight of an id, a multiple of 2^-51.
  auto weight = [&](int id) -> uint64_t {
    double w = target.p(target.value(id), id, exp2);
    if (less) w -= draft.p(draft.value(id), id, exp2);
    w = id == without ? 0.0 : fmax(w, 0.0);
    return (uint64_t)__double_as_longlong(__builtin_fma(w, 0.5, 1.0)) & 0x000FFFFFFFFFFFFFull;
  };
  const int segs = (g.V + 255) / 256;
  int drawn = target.k.total ? -1 : 0;
  uint64_t total = 0;
#pragma unroll 1
  while (drawn < 0) {
    for (int s = wave; s < segs; s += kVerifyWaves) {
      uint64_t w = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int id = 256 * s + 4 * lane + c;
        if (id < g.V) w += weight(id);
      }
      w = wave_scan_mass(w);
      if (lane == 63) seg[s] = w;
    }
    __syncthreads();
    // Every wave adds the groups up, then finds the one that the number falls into.
    total = 0;
    for (int s0 = 0; s0 < segs; s0 += 64) total += lane_u64(wave_scan_mass(s0 + lane < segs ? seg[s0 + lane] : 0ull), 63);
    if (total) break;
    // p is nowhere over q (they are equal but for rounding): from p.
    __syncthreads();
    less = false;
    without = -1;
  }
  if (drawn < 0 && wave == 0) {
    const uint64_t need = __umul64hi(total, (uint64_t)(uint32_t)(u * 0x1p32f) << 32) + 1;
    uint64_t run = 0;
    int group = -1;
    for (int s0 = 0; s0 < segs && group < 0; s0 += 64) {
      const uint64_t own = s0 + lane < segs ? seg[s0 + lane] : 0ull, upto = run + wave_scan_mass(own);
      const uint64_t who = __ballot(upto - own < need && need <= upto);
      if (who) {
        group = s0 + __builtin_ctzll(who);
        run = lane_u64(upto - own, __builtin_ctzll(who));
      } else {
        run = lane_u64(upto, 63);
      }
    }
    uint64_t w[4], own = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int id = 256 * group + 4 * lane + c;
      w[c] = id < g.V ? weight(id) : 0ull;
      own += w[c];
    }
    run += wave_scan_mass(own) - own;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (run < need && need <= run + w[c]) g.token[r] = 256 * group + 4 * lane + c;
      run += w[c];
    }
  }
  if (drawn == 0 && t == 0) g.token[r] = 0;  // a row of -inf and NaN alone
  for (int i = t; i <= drafts; i += kThreads)
    if (i != accepted) g.token[row0 + i] = i < accepted ? g.drafts[row0 + i] : -1;
  if (t == 0) g.accepted[b] = accepted;
}

}  // namespace

hipError_t launch_verify(const VerifyArgs& g, hipStream_t s) {
  if (g.requests == 0) return hipSuccess;
  const hipError_t e = launch_kept(g, s);
  if (e != hipSuccess) return e;
  auto kern = g.bf16 ? k_verify<true> : k_verify<false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)g.requests), dim3(kThreads), 0, s, g);
  return hipGetLastError();
}

}  // namespace mh
