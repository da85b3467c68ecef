// verify.hip — drafted ids against the target's distribution, from given numbers.
//
// With p the distribution that a target row's settings leave and q the one its draft was drawn from, a draft t is
// accepted with probability min(1, p(t) / q(t)): while u q(t) < p(t).  At the first draft that is not, an id is drawn from
// max(p - q, 0), so that every id comes out with probability p whatever q is; after all drafts one from p of the last row.
// Without draft logits q is 1 at the drafted id (a draft that was looked up, not drawn).
//
// What the settings keep of each row (a prefix in the order of logits), its mass and the draft's share come from the pass
// that also draws single ids (sample.hip, a workgroup per row).  Here a request's ids are cut among workgroups: each finds
// the first draft that is not accepted for itself and sums the weights of every 256 of its ids; the last one to
// end finds the group that the number falls into, and its id.  Weights are multiples of 2^-51, so their sums are exact and
// the drawn id does not depend on the launch.
#include "device_common.h"
#include "kernels.h"
#include "mass.h"

#include <algorithm>

namespace mh {
namespace {

constexpr int kThreads = 256;
constexpr int kVerifyWaves = kThreads / 64;

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h4u __attribute__((ext_vector_type(4), aligned(2)));

// What workgroups tell each other goes past the caches, in both directions; then all that a release has to do is to wait for
// the stores (a fence for the device writes the cache back: 64 requests in 16 slices took 98 us with it, 15 without).
template <class T>
__device__ __forceinline__ T shared_load(const T* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ void shared_store(T* p, T v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void wait_stores() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Four ids' logits from `id` on; past the row's end the last one's.
template <bool BF16>
__device__ __forceinline__ f4v load4(const void* base, int id, int V) {
  f4v v;
  if (id + 3 < V) {
    if constexpr (BF16) {
      const h4u h = *(const h4u*)((const uint16_t*)base + id);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = bf16_to_f32(h[c]);
    } else {
      const f4u f = *(const f4u*)((const float*)base + id);
#pragma unroll
      for (int c = 0; c < 4; ++c) v[c] = f[c];
    }
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int i = min(id + c, V - 1);
      v[c] = BF16 ? bf16_to_f32(((const uint16_t*)base)[i]) : ((const float*)base)[i];
    }
  }
  return v;
}

template <bool BF16>
__global__ __launch_bounds__(kThreads) void k_verify(VerifyArgs g, int slices) {
  __shared__ uint64_t exp2[32];
  __shared__ int stop, ended;
  __shared__ uint64_t sums[kVerifyWaves];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int b = blockIdx.x / slices, slice = blockIdx.x % slices;
  const int row0 = g.cu[b], end = g.cu[b + 1];
  const float temperature = g.temperature ? g.temperature[b] : 1.0f;
  float u = g.u_draw[b];
  const bool ok = row0 >= 0 && end >= row0 && end <= g.rows && end - row0 <= g.max_rows;
  if (!ok || end == row0) {
    if (t == 0 && slice == 0) {
      if (!ok && g.err) *g.err = 1;
      g.accepted[b] = 0;
    }
    return;
  }
  const int drafts = end - row0 - 1;
  if (t < 32) exp2[t] = kSampleExp2Tab[t] + ((uint64_t)kMassBits << 52);
  if (t == 0) stop = drafts;
  __syncthreads();

  // ---- the drafts, a thread each ----
  auto source = [&](int r) { return g.draft_row ? g.draft_row[r] : r; };
  for (int i = t; i < drafts; i += kThreads) {
    const int r = row0 + i, id = g.drafts[r];
    const float number = g.u[r];
    const double p = g.kept[r].draft_share;
    double q = 1.0;
    bool in = (uint32_t)id < (uint32_t)g.V && number >= 0.0f && number < 1.0f;
    if (g.draft_logits) {
      const int at = source(r);
      q = g.kept[g.rows + r].draft_share;
      in = in && (uint32_t)at < (uint32_t)g.draft_rows;
    }
    if (!in && slice == 0 && g.err) *g.err = 1;
    if (!(in && (double)number * q < p)) atomicMin(&stop, i);
  }
  __syncthreads();
  const int accepted = __builtin_amdgcn_readfirstlane(stop), r = row0 + accepted;
  if (slice == 0) {
    for (int i = t; i <= drafts; i += kThreads)
      if (i != accepted) g.token[row0 + i] = i < accepted ? g.drafts[row0 + i] : -1;
    if (t == 0) {
      g.accepted[b] = accepted;
      if (!(u >= 0.0f && u < 1.0f) && g.err) *g.err = 1;
    }
  }

  // ---- the weights of the row that an id is drawn from ----
  const size_t value = BF16 ? 2 : 4;
  const void* row = (const char*)g.logits + (size_t)r * g.ld * value;
  const RowKept target = g.kept[r];
  const void* other = row;
  RowKept draft = target;
  int without = -1;   // an id whose q is 1
  bool less = false;  // q from `draft`
  if (accepted < drafts) {
    if (!g.draft_logits) {
      without = g.drafts[r];
    } else {
      const int at = source(r);
      if ((uint32_t)at < (uint32_t)g.draft_rows) {
        other = (const char*)g.draft_logits + (size_t)at * g.ld_draft * value;
        draft = g.kept[g.rows + r];
        less = draft.total != 0;
      }
    }
  }
  if (!target.total) {  // a row of -inf and NaN alone
    if (slice == 0 && t == 0) g.token[r] = 0;
    return;
  }
  u = u >= 0.0f && u < 1.0f ? u : 0.0f;
  const Octaves scale = octaves_of(temperature);
  const double of_target = 1.0 / (double)target.total, of_draft = less ? 1.0 / (double)draft.total : 0.0;
  // Weights of four ids, multiples of 2^-51.
  auto weights = [&](f4v v, f4v d, int id, uint64_t (&w)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      double x = kept_mass(target, scale, v[c], id + c, exp2) * of_target;
      if (less) x -= kept_mass(draft, scale, d[c], id + c, exp2) * of_draft;
      x = id + c == without || id + c >= g.V ? 0.0 : fmax(x, 0.0);
      w[c] = (uint64_t)__double_as_longlong(__builtin_fma(x, 0.5, 1.0)) & 0x000FFFFFFFFFFFFFull;
    }
  };
  const int segs = (g.V + 255) / 256, per = (segs + slices - 1) / slices;
  uint64_t* seg = g.seg + (int64_t)b * segs;
  auto sum_groups = [&](int from, int to) {  // of 256 ids, a wave each
    f4v v = load4<BF16>(row, min(256 * (from + wave) + 4 * lane, g.V - 1), g.V), d = v;
    if (less) d = load4<BF16>(other, min(256 * (from + wave) + 4 * lane, g.V - 1), g.V);
#pragma unroll 1
    for (int s = from + wave; s < to; s += kVerifyWaves) {
      const int id = 256 * s + 4 * lane, next = min(id + 256 * kVerifyWaves, g.V - 1);
      const f4v nv = load4<BF16>(row, next, g.V);
      f4v nd = nv;
      if (less) nd = load4<BF16>(other, next, g.V);
      uint64_t all = 0;
      // Groups of which nothing is kept are left out (a row's one id, or its infinities, are not told by the border).
      if (target.flags || __any(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])) >= target.border_v)) {
        uint64_t w[4];
        weights(v, d, id, w);
        all = wave_scan_mass((w[0] + w[1]) + (w[2] + w[3]));
      }
      if (lane == 63) shared_store(&seg[s], all);
      v = nv;
      d = nd;
    }
  };
  sum_groups(slice * per, min(segs, slice * per + per));
  wait_stores();
  __syncthreads();
  if (slices > 1) {
    if (t == 0) ended = __hip_atomic_fetch_add(&g.done[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (ended != slices - 1) return;
  }

  // ---- the last workgroup: the group, and its id ----
  uint64_t total;
#pragma unroll 1
  for (bool again = false;; again = true) {
    uint64_t mine = 0;
    for (int s = t; s < segs; s += kThreads) mine += shared_load(&seg[s]);
    mine = wave_scan_mass(mine);
    if (lane == 63) sums[wave] = mine;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < kVerifyWaves; ++w) total += sums[w];
    if (total || again) break;
    // p is nowhere over q (they are equal but for rounding): from p, whose sum is not 0.
    less = false;
    without = -1;
    __syncthreads();
    sum_groups(0, segs);
    wait_stores();
    __syncthreads();
  }
  if (wave > 0) return;
  const uint64_t need = __umul64hi(total, (uint64_t)(uint32_t)(u * 0x1p32f) << 32) + 1;
  uint64_t run = 0;
  int group = 0;
  for (int s0 = 0; s0 < segs; s0 += 64) {
    const uint64_t own = s0 + lane < segs ? shared_load(&seg[s0 + lane]) : 0ull, upto = run + wave_scan_mass(own);
    const uint64_t who = __ballot(upto - own < need && need <= upto);
    if (who) {
      group = s0 + __builtin_ctzll(who);
      run = lane_u64(upto - own, __builtin_ctzll(who));
      break;
    }
    run = lane_u64(upto, 63);
  }
  const int id = 256 * group + 4 * lane;
  const f4v v = load4<BF16>(row, min(id, g.V - 1), g.V);
  f4v d = v;
  if (less) d = load4<BF16>(other, min(id, g.V - 1), g.V);
  uint64_t w[4];
  weights(v, d, id, w);
  const uint64_t own = (w[0] + w[1]) + (w[2] + w[3]);
  run += wave_scan_mass(own) - own;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (run < need && need <= run + w[c]) g.token[r] = id + c;
    run += w[c];
  }
}

// Workspace: the records, the sums of every 256 ids of each request, and how many workgroups of a request have ended.
struct VerifyWorkspace {
  size_t seg, done, bytes;
};
VerifyWorkspace workspace_of(int64_t rows, int64_t requests, int64_t V, bool drafted) {
  VerifyWorkspace w;
  w.seg = (size_t)rows * (drafted ? 2 : 1) * sizeof(RowKept);
  w.done = w.seg + (size_t)requests * ((V + 255) / 256) * 8;
  w.bytes = w.done + (size_t)requests * 4;
  return w;
}

}  // namespace

size_t verify_bytes(int64_t rows, int64_t requests, int64_t V, bool drafted) {
  return rows && requests ? workspace_of(rows, requests, V, drafted).bytes : 0;
}

hipError_t launch_verify(const VerifyArgs& args, void* workspace, size_t workspace_bytes, hipStream_t s) {
  VerifyArgs g = args;
  if (g.requests == 0) return hipSuccess;
  const VerifyWorkspace w = workspace_of(g.rows, g.requests, g.V, g.draft_logits != nullptr);
  if (g.rows && (!workspace || workspace_bytes < w.bytes)) return hipErrorInvalidValue;
  g.kept = (RowKept*)workspace;
  g.seg = (uint64_t*)((char*)workspace + w.seg);
  g.done = (int32_t*)((char*)workspace + w.done);
  const hipError_t e = launch_kept(g, s);
  if (e != hipSuccess) return e;
  // Four workgroups a compute unit (us, 64 requests of 32000 ids | 100 of 100003, slices for 256, 512, 1024, 2048 workgroups:
  // 75.6 68.6 67.6 73.9 | 201 170 162 163, of which the rows' records 51 | 136).
  const int segs = (g.V + 255) / 256;
  const int slices = std::max(1, std::min(1024 / g.requests, (segs + kVerifyWaves - 1) / kVerifyWaves));
  auto kern = g.bf16 ? k_verify<true> : k_verify<false>;
  hipLaunchKernelGGL(kern, dim3((unsigned)(g.requests * slices)), dim3(kThreads), 0, s, g, slices);
  return hipGetLastError();
}

}  // namespace mh
