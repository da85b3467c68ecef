// paged.hip — a step's bookkeeping of a paged key-value cache, and its keys and values into their slots.
//
// The key cache is [pages, kv_heads, page_size, head_dim], the value cache [pages, kv_heads, head_dim, page_size]: a
// page's keys of one head are one block each, and both products of the attention (over the dimensions, then over the
// keys) read neighbouring values of their summed index.  Slot s is place s % page_size of page s / page_size.
#include "device_common.h"
#include "kernels.h"

#include <type_traits>

namespace mh {
namespace {

template <int N>
using Int = std::integral_constant<int, N>;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

// Inclusive prefix sum over the wave: within rows of 16 lanes, then across them.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const auto moved = [](uint32_t x, auto ctrl, auto rows) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xF, true);
  };
  Int<0xF> all;
  v += moved(v, Int<0x111>{}, all);  // row_shr:1
  v += moved(v, Int<0x112>{}, all);
  v += moved(v, Int<0x114>{}, all);
  v += moved(v, Int<0x118>{}, all);
  v += moved(v, Int<0x142>{}, Int<0xA>{});  // row_bcast:15 into rows 1 and 3
  v += moved(v, Int<0x143>{}, Int<0xC>{});  // row_bcast:31 into rows 2 and 3
  return v;
}

// A slot from its page and position; -1, and *err, if there is no such page.
__device__ __forceinline__ int slot_of(const PagedPlanArgs& g, int page, int position) {
  if ((uint32_t)page < (uint32_t)g.num_pages)
    return (int)(((uint32_t)page << g.page_shift) + (position & ((1 << g.page_shift) - 1)));
  if (g.err) *g.err = 1;
  return -1;
}
__device__ __forceinline__ void put_row(const PagedPlanArgs& g, uint32_t r, int slot, int request, int position) {
  if (g.slot_of_row) g.slot_of_row[r] = slot;
  if (g.request_of_row) g.request_of_row[r] = request;
  if (g.position_of_row) g.position_of_row[r] = position;
}

// One workgroup plans the step: prefix sums over the requests of pages that come back, pages and rows that are asked
// for; the first request that does not fit ends the ones that are served; then pages change hands, and, for few rows
// (ROWS), the rows' maps.  A thread has up to eight requests; one that brings a page or a few rows is its thread's, one
// with many is its wave's.  What bounds it is one compute unit's latency: counts, two barriers, pages, rows, each a trip
// to memory (64 requests of one row: 4.2 us; 1000 with chunks of prompts and 30 ended ones of 250 pages each: 10.2 us, 16.2 with a
// search by every page for its request).
constexpr int kFewRows = 8;  // of a request: on two pages at most
template <bool ROWS>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PagedPlanArgs g) {
  __shared__ uint32_t wave_sum[3][kPlanWaves], given, rows_of_served;
  __shared__ int cut;
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int n = g.requests, page = 1 << g.page_shift;
  const int64_t width = (int64_t)g.max_blocks << g.page_shift;
  const int count_in = *g.free_count;
  if (t == 0) cut = n;

  // Each thread's requests t, t + 1024, ...
  constexpr int PER = kPlanMaxRequests / kPlanThreads;
  int len[PER], held[PER], add[PER];  // add < 0: ended
  uint32_t need[PER], first_back[PER], first_need[PER], first_row[PER];
  uint32_t run[3] = {0, 0, 0};
  bool unfit = false;
  int first_unfit = n;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    const int b = j * kPlanThreads + t;
    uint32_t v[3] = {0, 0, 0};  // pages back, pages needed, rows
    need[j] = 0;
    len[j] = held[j] = add[j] = 0;
    if (b < n) {
      len[j] = g.lengths[b];
      held[j] = g.pages_held[b];
      add[j] = g.new_tokens[b];
      const bool held_ok = held[j] >= 0 && held[j] <= g.max_blocks;
      if (add[j] < 0) {  // an ended request never keeps others from being served
        held[j] = held_ok ? held[j] : 0;
        v[0] = (uint32_t)held[j];
        if (!held_ok && g.err) *g.err = 1;
      } else {
        const bool ok = held_ok && len[j] >= 0 && len[j] <= (int64_t)held[j] << g.page_shift;
        if (!ok && g.err) *g.err = 1;
        if (ok && (int64_t)len[j] + add[j] <= width && add[j] <= g.row_cap) {
          const int want = (int)(((int64_t)len[j] + add[j] + page - 1) >> g.page_shift);
          need[j] = (uint32_t)max(want - held[j], 0);
          v[1] = need[j];
          v[2] = (uint32_t)add[j];
        } else {
          unfit = true;
          first_unfit = min(first_unfit, b);
        }
      }
    }
    uint32_t s[3];
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      s[q] = wave_scan(v[q]);
      if (lane == 63) wave_sum[q][wave] = s[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      uint32_t before = run[q], all = 0;
#pragma unroll
      for (int w = 0; w < kPlanWaves; ++w) {
        before += w < wave ? wave_sum[q][w] : 0u;
        all += wave_sum[q][w];
      }
      s[q] += before - v[q];  // exclusive
      run[q] += all;
    }
    first_back[j] = s[0];
    first_need[j] = s[1];
    first_row[j] = s[2];
    if ((j + 1) * kPlanThreads < n) __syncthreads();  // the sums are used again
  }
  // Pages on the stack once the ended requests' are back (run[0] of them).
  const bool count_ok = count_in >= 0 && count_in <= g.num_pages;
  const uint32_t count = count_ok ? (uint32_t)count_in : 0u, there = min(count + run[0], (uint32_t)g.num_pages);
  if (t == 0 && g.err && (!count_ok || count + run[0] > (uint32_t)g.num_pages)) *g.err = 1;  // a page came back twice
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    const int b = j * kPlanThreads + t;
    if (b < n && add[j] >= 0 && (first_need[j] + need[j] > there || first_row[j] + (uint32_t)add[j] > (uint32_t)g.row_cap)) {
      unfit = true;
      first_unfit = min(first_unfit, b);
    }
  }
  if (unfit) atomicMin(&cut, first_unfit);
  if (t == 0) {
    given = run[1];
    rows_of_served = run[2];
  }

  // ---- pages come back: a wave per ended request ----
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    for (uint64_t m = __ballot(add[j] < 0 && held[j] > 0); m; m &= m - 1) {
      const int at = __builtin_ctzll(m), b = j * kPlanThreads + wave * 64 + at;
      const int pages = __builtin_amdgcn_readlane(held[j], at);
      const uint32_t first = count + (uint32_t)__builtin_amdgcn_readlane((int)first_back[j], at);
      const int32_t* from = g.table + (int64_t)b * g.max_blocks;
      for (int i = lane; i < pages; i += 256) {
        int p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) p[u] = from[min(i + 64 * u, pages - 1)];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (i + 64 * u < pages && first + i + 64 * u < (uint32_t)g.num_pages) g.free_pages[first + i + 64 * u] = p[u];
      }
    }
  }
  __syncthreads();  // the cut and the stack are whole
  const int served = cut;
#pragma unroll
  for (int j = 0; j < PER; ++j)
    if (j * kPlanThreads + t == served && served < n) {
      given = first_need[j];
      rows_of_served = first_row[j];
    }

  // ---- and are given out from the top: one by its request's thread, more by its wave ----
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    const int b = j * kPlanThreads + t;
    if (b >= served || add[j] < 0) need[j] = 0;
    if (need[j] == 1) {
      const int p = g.free_pages[there - 1 - first_need[j]];
      if ((uint32_t)p >= (uint32_t)g.num_pages && g.err) *g.err = 1;
      g.table[(int64_t)b * g.max_blocks + held[j]] = p;
    }
    for (uint64_t m = __ballot(need[j] > 1); m;) {
      int p[4], at[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // four requests' pages on their way at once
        at[u] = m ? __builtin_ctzll(m) : -1;
        if (at[u] < 0) continue;
        m &= m - 1;
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)first_need[j], at[u]);
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)need[j], at[u]);
        p[u] = g.free_pages[there - 1 - first - min((uint32_t)lane, all - 1)];
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (at[u] < 0) continue;
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)first_need[j], at[u]);
        const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)need[j], at[u]);
        int32_t* to = g.table + (int64_t)(j * kPlanThreads + wave * 64 + at[u]) * g.max_blocks +
                      __builtin_amdgcn_readlane(held[j], at[u]);
        for (uint32_t i = lane; i < all; i += 64) {
          if (i >= 64) p[u] = g.free_pages[there - 1 - first - i];
          if ((uint32_t)p[u] >= (uint32_t)g.num_pages && g.err) *g.err = 1;
          to[i] = p[u];
        }
      }
    }
  }
  __syncthreads();  // the tables are whole
  const uint32_t rows = rows_of_served;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    const int b = j * kPlanThreads + t;
    const bool ended = add[j] < 0, go = b < served && !ended;
    if (b < n) {
      g.lengths_out[b] = ended ? 0 : len[j] + (go ? add[j] : 0);
      g.pages_held_out[b] = ended ? 0 : held[j] + (int)need[j];
      g.cu_rows[b] = (int)(b < served ? first_row[j] : rows);
    }
    if constexpr (ROWS) {
      const int mine = go ? add[j] : 0;
      const int32_t* from = g.table + (int64_t)b * g.max_blocks;
      if (mine > 0 && mine <= kFewRows) {
        const int p0 = len[j] >> g.page_shift, p1 = (len[j] + mine - 1) >> g.page_shift;
        const int page0 = from[p0], page1 = from[p1];
        for (int i = 0; i < mine; ++i) {
          const int position = len[j] + i;
          put_row(g, first_row[j] + i, slot_of(g, position >> g.page_shift == p0 ? page0 : page1, position), b, position);
        }
      }
      for (uint64_t m = __ballot(mine > kFewRows); m; m &= m - 1) {
        const int at = __builtin_ctzll(m), request = j * kPlanThreads + wave * 64 + at;
        const int all = __builtin_amdgcn_readlane(add[j], at), begin = __builtin_amdgcn_readlane(len[j], at);
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)first_row[j], at);
        const int32_t* pages = g.table + (int64_t)request * g.max_blocks;
        for (int i = lane; i < all; i += 256) {
          int p[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) p[u] = pages[(begin + min(i + 64 * u, all - 1)) >> g.page_shift];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int k = i + 64 * u, position = begin + k;
            if (k < all) put_row(g, first + k, slot_of(g, p[u], position), request, position);
          }
        }
      }
    }
  }
  if constexpr (ROWS)
    for (uint32_t r = rows + t; r < (uint32_t)g.row_cap; r += kPlanThreads) put_row(g, r, -1, -1, -1);
  if (t == 0) {
    g.cu_rows[n] = (int)rows;
    *g.free_count_out = (int)(there - given);
    *g.served = served;
  }
}

// The maps of many rows, a thread each: the request is the last whose first row is not past it.
__global__ __launch_bounds__(256) void k_paged_rows(PagedPlanArgs g) {
  const int r = blockIdx.x * 256 + threadIdx.x;
  if (r >= g.row_cap) return;
  if (r >= g.cu_rows[g.requests]) {
    put_row(g, r, -1, -1, -1);
    return;
  }
  int lo = 0, hi = g.requests;  // cu_rows[lo] <= r < cu_rows[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (g.cu_rows[mid] <= r ? lo : hi) = mid;
  }
  const int position = g.lengths_out[lo] - (g.cu_rows[lo + 1] - r);
  put_row(g, r, slot_of(g, g.table[(int64_t)lo * g.max_blocks + (position >> g.page_shift)], position), lo, position);
}

__device__ __forceinline__ uint16_t to_bf16(float f) {  // to nearest even; a NaN stays one
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
// N values at any value-aligned address, as fp32.
template <int N, bool IN16>
__device__ __forceinline__ void load_values(const void* p, int64_t i, float (&v)[N]) {
  typedef float fv __attribute__((ext_vector_type(N), aligned(4)));
  typedef uint16_t hv __attribute__((ext_vector_type(N), aligned(2)));
  if constexpr (IN16) {
    const hv h = *(const hv*)((const uint16_t*)p + i);
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = bf16_to_f32(h[c]);
  } else {
    const fv f = *(const fv*)((const float*)p + i);
#pragma unroll
    for (int c = 0; c < N; ++c) v[c] = f[c];
  }
}
// Eight neighbouring values of a cache, 16-byte aligned.
template <bool CB16>
__device__ __forceinline__ void store8(void* cache, int64_t i, const float (&v)[8]) {
  if constexpr (CB16) {
    v4i w;
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = (int)(to_bf16(v[2 * c]) | (uint32_t)to_bf16(v[2 * c + 1]) << 16);
    *(v4i*)((uint16_t*)cache + i) = w;
  } else {
    *(f4v*)((float*)cache + i) = f4v{v[0], v[1], v[2], v[3]};
    *(f4v*)((float*)cache + i + 4) = f4v{v[4], v[5], v[6], v[7]};
  }
}
template <bool CB16>
__device__ __forceinline__ void store1(void* cache, int64_t i, float v) {
  if constexpr (CB16) ((uint16_t*)cache)[i] = to_bf16(v);
  else ((float*)cache)[i] = v;
}

// A workgroup of four waves takes 16 rows of one head.  Keys go as they come, eight dimensions a thread.  Values turn: where
// eight rows have the eight slots of an aligned group, each thread takes two dimensions of all eight and stores
// eight neighbouring places at once (16384 rows of 8 heads of 128: 63 us by single values, 29 so); rows of
// no such group (a decode step's) store single values.  Which rows make a group follows from the slots of the eight rows
// before and after alone, so neighbouring workgroups agree.
constexpr int kAppendRows = 16;
template <int D, bool IN16, bool CB16>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendArgs g) {
  constexpr int PAIRS = D / 2, AT_ONCE = 64 / PAIRS;  // rows or groups a wave takes at once (D = 48: 16 lanes idle)
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int64_t row0 = (int64_t)(blockIdx.x / g.kv_heads) * kAppendRows;
  const int head = blockIdx.x % g.kv_heads, mask = (1 << g.page_shift) - 1;

  // Lane 8 + i: the slot of row row0 + i; the eight rows before and after in the lanes around.
  int slot = -1;
  {
    const int64_t r = row0 - 8 + lane;
    if (lane < 32 && r >= 0 && r < g.rows) slot = g.slot_of_row[r];
    if (slot >= 0 && slot >> g.page_shift >= g.num_pages) {
      if (g.err && head == 0) *g.err = 1;
      slot = -1;
    }
  }
  const bool mine = lane >= 8 && lane < 8 + kAppendRows && slot >= 0;
  const int after = __shfl_down(slot, 1);  // by every lane: what one gives that is masked off is not defined
  const uint32_t next = (uint32_t)__ballot(slot >= 0 && lane < 31 && after == slot + 1);
  const int first = lane - (slot & 7);  // lane of the group's first row
  const bool grouped = first >= 0 && lane < 32 && (next >> (first & 31) & 0x7F) == 0x7F;
  uint32_t groups = (uint32_t)__ballot(mine && grouped && first == lane);
  uint32_t singles = (uint32_t)__ballot(mine && !grouped);
  auto block = [&](int s) -> int64_t { return ((int64_t)(s >> g.page_shift) * g.kv_heads + head) * D << g.page_shift; };

  // ---- keys ----
  {
    const int row = t / (D / 8), d = t % (D / 8) * 8;
    const int s = __shfl(slot, 8 + min(row, kAppendRows - 1));
    if (row < kAppendRows && s >= 0) {
      float v[8];
      load_values<8, IN16>(g.k, (row0 + row) * g.ldk + head * D + d, v);
      store8<CB16>(g.k_cache, block(s) + (int64_t)(s & mask) * D + d, v);
    }
  }

  // ---- values ----
  const int sub = lane / PAIRS, d = lane % PAIRS * 2;
  const auto nth = [](uint32_t m, int n) {  // the n-th set bit, or -1
    for (; n > 0 && m; --n) m &= m - 1;
    return m ? __builtin_ctz(m) : -1;
  };
  const int n_groups = __builtin_popcount(groups), n_singles = __builtin_popcount(singles);
  for (int j = wave * AT_ONCE; j < n_groups; j += 4 * AT_ONCE) {
    const int at = sub < AT_ONCE ? nth(groups, j + sub) : -1;
    const int s = __shfl(slot, max(at, 0));
    if (at < 0) continue;
    float v[8][2], w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) load_values<2, IN16>(g.v, (row0 + at - 8 + i) * g.ldv + head * D + d, v[i]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = v[i][c];
      store8<CB16>(g.v_cache, block(s) + ((int64_t)(d + c) << g.page_shift) + (s & mask), w);
    }
  }
  for (int j = wave * AT_ONCE; j < n_singles; j += 4 * AT_ONCE) {
    const int at = sub < AT_ONCE ? nth(singles, j + sub) : -1;
    const int s = __shfl(slot, max(at, 0));
    if (at < 0) continue;
    float v[2];
    load_values<2, IN16>(g.v, (row0 + at - 8) * g.ldv + head * D + d, v);
#pragma unroll
    for (int c = 0; c < 2; ++c) store1<CB16>(g.v_cache, block(s) + ((int64_t)(d + c) << g.page_shift) + (s & mask), v[c]);
  }
}

// Few rows: a wave per row and head, which has read its values by the time it knows their slot.
template <int D, bool IN16, bool CB16>
__global__ __launch_bounds__(64) void k_paged_append_few(PagedAppendArgs g) {
  const int64_t row = blockIdx.x / g.kv_heads;
  const int head = blockIdx.x % g.kv_heads, lane = threadIdx.x, mask = (1 << g.page_shift) - 1;
  const int slot = g.slot_of_row[row];
  const int d = 2 * lane < D ? 2 * lane : 0;
  float k[2], v[2];
  load_values<2, IN16>(g.k, row * g.ldk + head * D + d, k);
  load_values<2, IN16>(g.v, row * g.ldv + head * D + d, v);
  if (slot < 0 || 2 * lane >= D) return;
  if (slot >> g.page_shift >= g.num_pages) {
    if (g.err && head == 0) *g.err = 1;
    return;
  }
  const int64_t block = ((int64_t)(slot >> g.page_shift) * g.kv_heads + head) * D << g.page_shift;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    store1<CB16>(g.k_cache, block + (int64_t)(slot & mask) * D + d + c, k[c]);
    store1<CB16>(g.v_cache, block + ((int64_t)(d + c) << g.page_shift) + (slot & mask), v[c]);
  }
}

template <int D>
void append_launch(const PagedAppendArgs& g, hipStream_t s) {
  // us of the GPU's time, a wave per row and head | 16 rows a workgroup: 61 rows of 8 heads of 64 2.8 | 4.4; from 8192 rows and
  // heads on the second is as fast or faster (a call from the host: 512 prompt rows 8.1 | 8.2, 2048 of 128 wide 13.1 | 8.0).
  if (g.rows * g.kv_heads <= 4096) {
    auto kern = g.in_bf16 ? (g.cache_bf16 ? k_paged_append_few<D, true, true> : k_paged_append_few<D, true, false>)
                          : (g.cache_bf16 ? k_paged_append_few<D, false, true> : k_paged_append_few<D, false, false>);
    hipLaunchKernelGGL(kern, dim3((unsigned)(g.rows * g.kv_heads)), dim3(64), 0, s, g);
    return;
  }
  const dim3 grid((unsigned)((g.rows + kAppendRows - 1) / kAppendRows * g.kv_heads));  // at most 2^21
  auto kern = g.in_bf16 ? (g.cache_bf16 ? k_paged_append<D, true, true> : k_paged_append<D, true, false>)
                        : (g.cache_bf16 ? k_paged_append<D, false, true> : k_paged_append<D, false, false>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, s, g);
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& g, hipStream_t s) {
  // One workgroup writes some rows a thread in less time than a second launch takes (us, one launch | two: 64 requests of a row
  // in maps of 4096 5.0 | 8.0, 1000 with 2462 rows 6.4 | 8.5, with 4395 8.0 | 8.7, with 8515 25.9 | 8.7); prompts' chunks take longer
  // than that, a wave each (20 with 2322 rows 18.7 | 10.6, 60 with 5805 45 | 19), but the host knows row_cap, not the chunks.
  if (g.row_cap <= 4 * kPlanThreads) {
    hipLaunchKernelGGL(k_paged_plan<true>, dim3(1), dim3(kPlanThreads), 0, s, g);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(k_paged_plan<false>, dim3(1), dim3(kPlanThreads), 0, s, g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k_paged_rows, dim3((unsigned)((g.row_cap + 255) / 256)), dim3(256), 0, s, g);
  return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs& g, hipStream_t s) {
  if (g.rows == 0) return hipSuccess;
  if (g.head_dim == 48) append_launch<48>(g, s);
  else if (g.head_dim == 64) append_launch<64>(g, s);
  else if (g.head_dim == 128) append_launch<128>(g, s);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace mh
