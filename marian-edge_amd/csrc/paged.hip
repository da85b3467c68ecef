// paged.hip — a step's bookkeeping of a paged key-value cache, and its keys and values into their slots.
//
// The key cache is [pages, kv_heads, page_size, head_dim], the value cache [pages, kv_heads, head_dim, page_size]: a
// page's keys of one head are one block each, and both products of the attention (over the dimensions, then over the
// keys) read neighbouring values of their summed index.  Slot s is place s % page_size of page s / page_size.
#include "device_common.h"
#include "kernels.h"

#include <algorithm>

namespace mh {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;

// Inclusive prefix sum over the wave.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t u = (uint32_t)__shfl_up((int)v, d);
    v += lane >= d ? u : 0u;
  }
  return v;
}

// The last index i < n with first[i] <= k, for first[0] <= k.
__device__ __forceinline__ int last_upto(const uint32_t* first, int n, uint32_t k) {
  int lo = 0, hi = n;  // first[lo] <= k, first[hi] > k (or past the end)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    (first[mid] <= k ? lo : hi) = mid;
  }
  return lo;
}

// Row r's maps: the request by its place in cu, position and slot.
__device__ __forceinline__ void fill_row(const PagedPlanArgs& g, const uint32_t* cu, uint32_t r, uint32_t rows) {
  int slot = -1, request = -1, position = -1;
  if (r < rows) {
    request = last_upto(cu, g.requests, r);
    position = g.lengths_out[request] - (int)(cu[request + 1] - r);
    const int page = g.table[(int64_t)request * g.max_blocks + (position >> g.page_shift)];
    if ((uint32_t)page < (uint32_t)g.num_pages)
      slot = (int)(((uint32_t)page << g.page_shift) + (position & ((1 << g.page_shift) - 1)));
    else if (g.err)
      *g.err = 1;
  }
  if (g.slot_of_row) g.slot_of_row[r] = slot;
  if (g.request_of_row) g.request_of_row[r] = request;
  if (g.position_of_row) g.position_of_row[r] = position;
}

// One workgroup plans the step: prefix sums over the requests of pages that come back, pages and rows that are asked
// for; the first request that does not fit ends the ones that are served; then pages change hands, and, for few rows
// (ROWS), the rows' maps.
template <bool ROWS>
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PagedPlanArgs g) {
  __shared__ uint32_t first_back[kPlanMaxRequests], first_need[kPlanMaxRequests], first_row[kPlanMaxRequests + 1];
  __shared__ uint32_t wave_sum[3][kPlanWaves];
  __shared__ int cut;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int n = g.requests, page = 1 << g.page_shift;
  const int64_t width = (int64_t)g.max_blocks << g.page_shift;
  if (t == 0) cut = n;
  const int count_in = *g.free_count;
  const bool count_ok = count_in >= 0 && count_in <= g.num_pages;
  if (!count_ok && t == 0 && g.err) *g.err = 1;
  const uint32_t count = count_ok ? (uint32_t)count_in : 0u;

  // Each thread's requests t, t + 1024, ...
  constexpr int PER = kPlanMaxRequests / kPlanThreads;
  int len[PER], held[PER], add[PER];  // add < 0: ended
  uint32_t need[PER];
  uint32_t run[3] = {0, 0, 0};
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    if (j * kPlanThreads >= n) break;
    const int b = j * kPlanThreads + t;
    uint32_t v[3] = {0, 0, 0};  // pages back, pages needed, rows
    need[j] = 0;
    if (b < n) {
      len[j] = g.lengths[b];
      held[j] = g.pages_held[b];
      add[j] = g.new_tokens[b];
      const bool held_ok = held[j] >= 0 && held[j] <= g.max_blocks;
      bool fits = held_ok;
      if (add[j] < 0) {
        v[0] = held_ok ? (uint32_t)held[j] : 0u;
        fits = true;  // an ended request never keeps others from being served
        if (!held_ok && g.err) *g.err = 1;
      } else {
        const bool ok = held_ok && len[j] >= 0 && len[j] <= (int64_t)held[j] << g.page_shift;
        if (!ok && g.err) *g.err = 1;
        fits = ok && (int64_t)len[j] + add[j] <= width && add[j] <= g.row_cap;
        if (fits) {
          const int want = (int)(((int64_t)len[j] + add[j] + page - 1) >> g.page_shift);
          need[j] = (uint32_t)max(want - held[j], 0);
          v[1] = need[j];
          v[2] = (uint32_t)add[j];
        }
      }
      if (!fits) atomicMin(&cut, b);
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
    if (b < n) {
      first_back[b] = s[0];
      first_need[b] = s[1];
      first_row[b] = s[2];
    }
    __syncthreads();
  }
  // Pages on the stack once the ended requests' are back (run[0] of them).
  uint32_t there = count + run[0];
  if (there > (uint32_t)g.num_pages) {  // a page given back twice
    if (t == 0 && g.err) *g.err = 1;
    there = (uint32_t)g.num_pages;
  }
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = j * kPlanThreads + t;
    if (b < n && add[j] >= 0 && (first_need[b] + need[j] > there || first_row[b] + (uint32_t)add[j] > (uint32_t)g.row_cap))
      atomicMin(&cut, b);
  }
  __syncthreads();
  const int served = cut;
  const uint32_t pages = served < n ? first_need[served] : run[1], rows = served < n ? first_row[served] : run[2];

  // ---- pages come back ----
  for (uint32_t k = t; k < run[0]; k += kPlanThreads) {
    const int b = last_upto(first_back, n, k);
    if (count + k < (uint32_t)g.num_pages) g.free_pages[count + k] = g.table[(int64_t)b * g.max_blocks + (k - first_back[b])];
  }
  __syncthreads();  // the stack is whole, and every held count is read (below in registers)
  // ---- and are given out from the top ----
  for (uint32_t k = t; k < pages; k += kPlanThreads) {
    const int b = last_upto(first_need, served, k);
    const int p = g.free_pages[there - 1 - k];
    if ((uint32_t)p >= (uint32_t)g.num_pages && g.err) *g.err = 1;
    g.table[(int64_t)b * g.max_blocks + g.pages_held[b] + (k - first_need[b])] = p;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int b = j * kPlanThreads + t;
    if (b >= n) break;
    const bool ended = add[j] < 0, go = !ended && b < served;
    g.lengths_out[b] = ended ? 0 : len[j] + (go ? add[j] : 0);
    g.pages_held_out[b] = ended ? 0 : held[j] + (go ? (int)need[j] : 0);
    const uint32_t r = b < served ? first_row[b] : rows;
    first_row[b] = r;
    g.cu_rows[b] = (int)r;
  }
  if (t == 0) {
    first_row[n] = rows;
    g.cu_rows[n] = (int)rows;
    *g.free_count_out = (int)(there - pages);
    *g.served = served;
  }
  if constexpr (ROWS) {
    __syncthreads();
    for (uint32_t r = t; r < (uint32_t)g.row_cap; r += kPlanThreads) fill_row(g, first_row, r, rows);
  }
}

// The rows' maps of many rows, a thread each.
__global__ __launch_bounds__(256) void k_paged_rows(PagedPlanArgs g) {
  const uint32_t r = blockIdx.x * 256 + threadIdx.x;
  if (r < (uint32_t)g.row_cap) fill_row(g, (const uint32_t*)g.cu_rows, r, (uint32_t)g.cu_rows[g.requests]);
}

__device__ __forceinline__ uint16_t to_bf16(float f) {  // to nearest even; a NaN stays one
  const uint32_t u = __float_as_uint(f);
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (uint16_t)((u >> 16) | 0x40u);
  return (uint16_t)((u + 0x7FFFu + ((u >> 16) & 1u)) >> 16);
}
template <bool IN16, bool CB16>
__device__ __forceinline__ auto convert(const void* p, int64_t i) {
  if constexpr (CB16) {
    if constexpr (IN16) return ((const uint16_t*)p)[i];
    else return to_bf16(((const float*)p)[i]);
  } else {
    if constexpr (IN16) return bf16_to_f32(((const uint16_t*)p)[i]);
    else return ((const float*)p)[i];
  }
}

// A workgroup per row and head.
template <bool IN16, bool CB16>
__global__ __launch_bounds__(64) void k_paged_append(PagedAppendArgs g) {
  using T = decltype(convert<IN16, CB16>(nullptr, 0));
  const int64_t row = blockIdx.x / g.kv_heads;
  const int head = blockIdx.x % g.kv_heads, d_n = g.head_dim;
  const int slot = g.slot_of_row[row];
  if (slot < 0) return;
  const int page = slot >> g.page_shift, place = slot & ((1 << g.page_shift) - 1);
  if (page >= g.num_pages) {
    if (threadIdx.x == 0 && g.err) *g.err = 1;
    return;
  }
  const int64_t block = ((int64_t)page * g.kv_heads + head) * d_n << g.page_shift;
  for (int d = threadIdx.x; d < d_n; d += 64) {
    ((T*)g.k_cache)[block + (int64_t)place * d_n + d] = convert<IN16, CB16>(g.k, row * g.ldk + head * d_n + d);
    ((T*)g.v_cache)[block + ((int64_t)d << g.page_shift) + place] = convert<IN16, CB16>(g.v, row * g.ldv + head * d_n + d);
  }
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs& g, hipStream_t s) {
  // One workgroup writes some rows a thread in less time than a second launch takes.
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
  const dim3 grid((unsigned)(g.rows * g.kv_heads));
  if (g.in_bf16) {
    if (g.cache_bf16) hipLaunchKernelGGL((k_paged_append<true, true>), grid, dim3(64), 0, s, g);
    else hipLaunchKernelGGL((k_paged_append<true, false>), grid, dim3(64), 0, s, g);
  } else {
    if (g.cache_bf16) hipLaunchKernelGGL((k_paged_append<false, true>), grid, dim3(64), 0, s, g);
    else hipLaunchKernelGGL((k_paged_append<false, false>), grid, dim3(64), 0, s, g);
  }
  return hipGetLastError();
}

}  // namespace mh
