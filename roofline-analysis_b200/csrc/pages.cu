// pages.cu — block tables and slot maps from request lengths, and the return
// of finished requests' pages: the integer work between a scheduler and the
// append / decode calls, without a trip to the host.
//
// Math (P = page size, L = length, n = new tokens of a request):
//   have = ceil(L / P), need = ceil((L + n) / P) - have
//   token_start = exclusive sum of n, page_start = exclusive sum of need
//   new page k of the step = free_pages[free_count - 1 - k]
//   slot of token i of a request = page((L + i) / P) * P + (L + i) % P
//
// Bound by latency: a decode step moves a few KB, so the whole step is one
// launch.  Every block computes the sums of all requests itself (a few KB
// from L2, the sums stay in shared memory) and then does its share of the
// slots and table entries, finding each one's request by bisection; no block
// waits for another.  The lengths and the free count may be updated in
// place: then the block that is last to finish reading (an arrival counter in
// the workspace header, zero between calls) writes them.  A thread takes 4
// slots at a time, so that their table reads are in flight together.
//
// A negative page never enters the pool: the blocks of a release copy the pages
// above the top of the stack, where nothing counts yet, and tell the last one
// whether they met a negative entry; it moves the top, or leaves everything.
// (The wait for the last block: 512 requests, a tenth finished, 6.5 -> 7.1 us.)
#include "b2d_decode.h"
#include "common.cuh"
#include "host_common.h"

namespace b2d {

constexpr int kPageThreads = 512;
constexpr int kMaxRequests = 16384;

struct PagesParams {
  const int32_t* lens;
  const int32_t* new_tokens;    // append; null: one each
  const uint8_t* finished;      // release
  int32_t* table;
  int64_t table_stride;
  int32_t* free_pages;
  const int32_t* free_count;
  int64_t* slots;
  int32_t* starts;
  int32_t* lens_out;
  int32_t* count_out;
  int* status;
  int* arrivals;
  int B, max_pages, P, max_tokens, capacity;
  int in_place;                 // append: an output is an input, written by the last block
};

__device__ __forceinline__ int64_t pages_of(int64_t tokens, int P) { return (tokens + P - 1) / P; }

__device__ __forceinline__ int length_of(const PagesParams& p, int b) {
  const int n = p.lens[b];
  return n < 0 ? 0 : n;
}

__device__ __forceinline__ int new_of(const PagesParams& p, int b) {
  if (p.new_tokens == nullptr) return 1;
  const int n = p.new_tokens[b];
  return n < 0 ? 0 : n;
}

// Exclusive block-wide sum of two 64-bit values per thread, and their totals.
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t& ta, int64_t& tb) {
  __shared__ int64_t wa[32], wb[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int64_t x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, x, o), v = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += u;
      y += v;
    }
  }
  if (lane == 31) {
    wa[warp] = x;
    wb[warp] = y;
  }
  __syncthreads();
  if (warp == 0) {
    int64_t s = lane < nw ? wa[lane] : 0, t = lane < nw ? wb[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, s, o), v = __shfl_up_sync(0xffffffffu, t, o);
      if (lane >= o) {
        s += u;
        t += v;
      }
    }
    wa[lane] = s;
    wb[lane] = t;
  }
  __syncthreads();
  a = x - a + (warp > 0 ? wa[warp - 1] : 0);
  b = y - b + (warp > 0 ? wb[warp - 1] : 0);
  ta = wa[nw - 1];
  tb = wb[nw - 1];
}

// Last b with start[b] <= i (requests that got nothing come before it).
__device__ __forceinline__ int request_of(const int32_t* start, int B, int i) {
  int lo = 0, hi = B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// True in the block that arrives last: every other block has read its inputs.
// `bad`: whether a thread of this block, on return of any block, has set it (the
// blocks that have are counted above the arrivals; there are at most 65535).
__device__ __forceinline__ bool last_block(int* arrivals, bool& bad) {
  __shared__ int seen;
  bad = __syncthreads_or(bad);
  if (gridDim.x == 1) return true;
  if (threadIdx.x == 0) {
    seen = atomic_add_acq_rel_gpu(arrivals, bad ? 0x10001 : 1);
    if ((seen & 0xffff) == (int)gridDim.x - 1) *arrivals = 0;
  }
  __syncthreads();
  bad = bad || (seen >> 16) != 0;
  return (seen & 0xffff) == (int)gridDim.x - 1;
}

__global__ void __launch_bounds__(kPageThreads) plan_append_kernel(const PagesParams p) {
  extern __shared__ int32_t sm[];
  int32_t* tok_start = sm;             // [B]
  int32_t* page_start = sm + p.B;      // [B]
  int32_t* lens = sm + 2 * p.B;        // [B]
  const int tid = threadIdx.x;
  const int count_in = *p.free_count;
  const int per = (p.B + kPageThreads - 1) / kPageThreads;
  const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  int64_t toks = 0, pages = 0;
  bool fits = true;
  for (int b = b0; b < b1; ++b) {
    const int64_t L = length_of(p, b), n = new_of(p, b);
    const int64_t end = pages_of(L + n, p.P), need = end - pages_of(L, p.P);
    lens[b] = (int)L;
    tok_start[b] = (int)n;             // counts, for now
    page_start[b] = need > INT32_MAX ? INT32_MAX : (int)need;
    toks += n;
    pages += need;
    fits = fits && (n == 0 || end <= p.max_pages);
  }
  int64_t total_toks, total_pages;
  block_scan2(toks, pages, total_toks, total_pages);
  const int count = max(0, min(count_in, p.capacity));
  fits = __syncthreads_and(fits && total_toks <= p.max_tokens && total_pages <= count);
  for (int b = b0; b < b1; ++b) {   // sums that are used only when the totals fit 32 bits
    const int n = tok_start[b], need = page_start[b];
    tok_start[b] = (int)toks;
    page_start[b] = (int)pages;
    toks += n;
    pages += need;
  }
  __syncthreads();
  const int first = blockIdx.x * kPageThreads + tid, step = gridDim.x * kPageThreads;
  for (int b = first; b <= p.B; b += step)
    p.starts[b] = !fits ? 0 : (b == p.B ? (int)total_toks : tok_start[b]);
  const int nt = fits ? (int)total_toks : 0, np = fits ? (int)total_pages : 0;
  constexpr int U = 4;
  for (int t0 = first; t0 < p.max_tokens; t0 += U * step) {
    int page[U], off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * step;
      page[u] = -1;
      off[u] = 0;
      if (t < nt) {
        const int b = request_of(tok_start, p.B, t);
        const int L = lens[b], have = (int)pages_of(L, p.P);
        const int pos = L + (t - tok_start[b]), pi = pos / p.P;
        page[u] = pi < have ? p.table[b * p.table_stride + pi]
                            : p.free_pages[count - 1 - (page_start[b] + pi - have)];
        off[u] = pos - pi * p.P;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = t0 + u * step;
      if (t < p.max_tokens) p.slots[t] = page[u] < 0 ? -1 : (int64_t)page[u] * p.P + off[u];
    }
  }
  for (int k = first; k < np; k += step) {
    const int b = request_of(page_start, p.B, k);
    const int have = (int)pages_of(lens[b], p.P), page = p.free_pages[count - 1 - k];
    if (page < 0) record_status(p.status, kStatusBounds);
    p.table[b * p.table_stride + have + (k - page_start[b])] = page;
  }
  bool unused = false;
  if (p.in_place ? !last_block(p.arrivals, unused) : blockIdx.x != 0) return;
  for (int b = tid; b < p.B; b += kPageThreads) p.lens_out[b] = fits ? lens[b] + new_of(p, b) : p.lens[b];
  if (tid == 0) {
    *p.count_out = fits ? count - np : count_in;
    if (!fits) record_status(p.status, kStatusCapacity);
  }
}

__global__ void __launch_bounds__(kPageThreads) release_pages_kernel(const PagesParams p) {
  extern __shared__ int32_t sm[];
  int32_t* page_start = sm;   // [B]
  const int tid = threadIdx.x;
  const int count_in = *p.free_count;
  const int per = (p.B + kPageThreads - 1) / kPageThreads;
  const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
  bool in_table = true;   // no finished request is longer than its row
  auto given = [&](int b) -> int64_t {
    if (p.finished[b] == 0) return 0;
    const int64_t n = pages_of(length_of(p, b), p.P);
    in_table = in_table && n <= p.max_pages;
    return n;
  };
  int64_t pages = 0, unused = 0, total, unused_total;
  for (int b = b0; b < b1; ++b) pages += given(b);
  block_scan2(pages, unused, total, unused_total);
  const int count = max(0, min(count_in, p.capacity));
  bool fits = __syncthreads_and(in_table && total <= p.capacity - count);
  for (int b = b0; b < b1; ++b) {   // used only when the total fits 32 bits
    page_start[b] = (int)pages;
    pages += given(b);
  }
  __syncthreads();
  const int np = fits ? (int)total : 0;
  bool negative = false;
  for (int k = blockIdx.x * kPageThreads + tid; k < np; k += gridDim.x * kPageThreads) {
    const int b = request_of(page_start, p.B, k);
    const int page = p.table[b * p.table_stride + (k - page_start[b])];
    negative = negative || page < 0;
    p.free_pages[count + k] = page;
  }
  if (!last_block(p.arrivals, negative)) return;
  if (tid == 0 && !(fits && !negative)) record_status(p.status, fits ? kStatusBounds : kStatusCapacity);
  fits = fits && !negative;
  for (int b = tid; b < p.B; b += kPageThreads) {
    const int L = p.lens[b];
    p.lens_out[b] = fits && p.finished[b] ? 0 : L;
  }
  if (tid == 0) *p.count_out = fits ? count + np : count_in;
}

// Blocks for `work` entries: one per 2048, at most one per SM.
static int page_blocks(int64_t work, int sms) {
  const int64_t n = (work + 2047) / 2048;
  return (int)(n < 1 ? 1 : (n > sms ? sms : n));
}

static int check_header(const void* ws, size_t bytes) {
  if (!ws || bytes < kWsHeaderBytes) return B2D_ERR_WORKSPACE;
  return ((uintptr_t)ws & 255) ? B2D_ERR_ALIGNMENT : B2D_OK;
}

// Whether lens_out or count_out overlaps an array that the blocks read.
static bool updates_inputs(const PagesParams& p) {
  auto overlap = [](const void* out, const void* in, size_t n) {
    return in && (uintptr_t)out + n > (uintptr_t)in && (uintptr_t)in + n > (uintptr_t)out;
  };
  const size_t rows = (size_t)p.B * 4;
  return overlap(p.lens_out, p.lens, rows) || overlap(p.lens_out, p.new_tokens, rows) ||
         overlap(p.count_out, p.free_count, 4);
}

}  // namespace b2d

using namespace b2d;

extern "C" int b2d_plan_append(const b2d_plan_append_args* a, void* stream) {
  if (!a || a->num_requests < 0 || a->max_pages_per_seq <= 0 || a->page_size <= 0 ||
      a->max_tokens < 0 || a->free_capacity < 0)
    return B2D_ERR_INVALID_ARG;
  if (a->num_requests > kMaxRequests || a->max_tokens > (1 << 30) ||
      (int64_t)a->max_pages_per_seq * a->page_size > (int64_t)INT32_MAX)
    return B2D_ERR_TOO_LARGE;
  if ((a->num_requests > 0 && (!a->cache_seqlens || !a->block_table || !a->seqlens_out)) ||
      !a->free_count || !a->free_count_out || !a->query_starts ||
      (a->max_tokens > 0 && !a->slot_mapping) || (a->free_capacity > 0 && !a->free_pages))
    return B2D_ERR_INVALID_ARG;
  if (int rc = check_header(a->workspace, a->workspace_bytes)) return rc;
  PagesParams p{};
  p.lens = a->cache_seqlens;
  p.new_tokens = a->new_tokens;
  p.table = a->block_table;
  p.table_stride = a->block_table_stride;
  p.free_pages = const_cast<int32_t*>(a->free_pages);
  p.free_count = a->free_count;
  p.slots = a->slot_mapping;
  p.starts = a->query_starts;
  p.lens_out = a->seqlens_out;
  p.count_out = a->free_count_out;
  p.status = static_cast<int*>(a->workspace);
  p.arrivals = reinterpret_cast<int*>(static_cast<uint8_t*>(a->workspace) + kStatusBytes);
  p.B = a->num_requests;
  p.max_pages = a->max_pages_per_seq;
  p.P = a->page_size;
  p.max_tokens = a->max_tokens;
  p.capacity = a->free_capacity;
  p.in_place = updates_inputs(p);
  int sms = 0;
  if (device_sm_count(&sms)) return B2D_ERR_CUDA;
  const size_t smem = (size_t)p.B * 12;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(plan_append_kernel), smem)) return B2D_ERR_CUDA;
  plan_append_kernel<<<page_blocks(p.max_tokens, sms), kPageThreads, smem,
                       static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? B2D_OK : B2D_ERR_CUDA;
}

extern "C" int b2d_release_pages(const b2d_release_args* a, void* stream) {
  if (!a || a->num_requests < 0 || a->max_pages_per_seq <= 0 || a->page_size <= 0 ||
      a->free_capacity < 0)
    return B2D_ERR_INVALID_ARG;
  if (a->num_requests > kMaxRequests ||
      (int64_t)a->max_pages_per_seq * a->page_size > (int64_t)INT32_MAX)
    return B2D_ERR_TOO_LARGE;
  if ((a->num_requests > 0 && (!a->cache_seqlens || !a->block_table || !a->finished ||
                               !a->seqlens_out)) ||
      !a->free_count || !a->free_count_out || (a->free_capacity > 0 && !a->free_pages))
    return B2D_ERR_INVALID_ARG;
  if (int rc = check_header(a->workspace, a->workspace_bytes)) return rc;
  PagesParams p{};
  p.lens = a->cache_seqlens;
  p.finished = a->finished;
  p.table = const_cast<int32_t*>(a->block_table);
  p.table_stride = a->block_table_stride;
  p.free_pages = a->free_pages;
  p.free_count = a->free_count;
  p.lens_out = a->seqlens_out;
  p.count_out = a->free_count_out;
  p.status = static_cast<int*>(a->workspace);
  p.arrivals = reinterpret_cast<int*>(static_cast<uint8_t*>(a->workspace) + kStatusBytes);
  p.B = a->num_requests;
  p.max_pages = a->max_pages_per_seq;
  p.P = a->page_size;
  p.capacity = a->free_capacity;
  int sms = 0;
  if (device_sm_count(&sms)) return B2D_ERR_CUDA;
  const size_t smem = (size_t)p.B * 4;
  if (ensure_dynamic_smem(reinterpret_cast<const void*>(release_pages_kernel), smem)) return B2D_ERR_CUDA;
  // At most min(all requests' table columns, free capacity) pages come back.
  const int64_t most = (int64_t)p.B * p.max_pages;
  release_pages_kernel<<<page_blocks(most < p.capacity ? most : p.capacity, sms), kPageThreads, smem,
                         static_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? B2D_OK : B2D_ERR_CUDA;
}
