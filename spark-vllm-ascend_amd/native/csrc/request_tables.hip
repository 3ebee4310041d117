// Block tables, slots, positions and offsets of a step, from request lengths on
// the device, and the return of pages to the free list (gfx950).
//
// Request r has context[r] tokens in the cache, num_pages[r] pages in its
// block-table row, and gets query[r] more tokens.  It needs
//   need[r] = max(0, min(ceil((context + query) / block_size), max_blocks) - num_pages)
// pages, taken in request order from the end of the free list: the page of its
// block num_pages[r] + j is free[count - 1 - (sum of need before r) - j], -1
// where that is below the list.  A prefix sum over the requests gives every
// output from the inputs alone, so pages and tokens are dealt to the threads
// evenly, whatever the lengths: thread k finds the request of page (token) k by
// bisection of the sums.  Bound by launch and dependent-load latency: a few
// kilobytes in and 16 bytes a token out.
#include <limits.h>

#include <algorithm>

#include "smx_common.h"
#include "smx_launch.h"

namespace smx {
namespace {

struct TablesArgs {
  const int32_t* query;
  const int32_t* context;
  const int32_t* num_pages;
  const int32_t* free_pages;
  const int32_t* free_count;
  int32_t* table;
  int32_t* num_pages_out;
  int32_t* free_count_out;
  int32_t* query_start;
  int32_t* seq_lens;
  int64_t* positions;
  int64_t* slots;
  int num_reqs, max_tokens, max_blocks, num_free, bs_log2, with_tokens;
  int parts;  // workgroups of the launch (the step runner passes no implicit arguments)
};

// Inclusive prefix sums of two values over a workgroup of NT threads; *ta and *tb
// the totals.
template <int NT>
__device__ __forceinline__ void scan2(int64_t& a, int& b, int64_t* ta, int* tb, int64_t* wa,
                                      int* wb) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // (a < 2^31 in two parts, whose sums fit 32 bits)
  const int lo = wave_scan_i32((int)(a & 0xffffff)), hi = wave_scan_i32((int)(a >> 24));
  a = ((int64_t)hi << 24) + lo;
  b = wave_scan_i32(b);
  __syncthreads();  // the last round's totals have been read
  if (lane == 63) {
    wa[wave] = a;
    wb[wave] = b;
  }
  __syncthreads();
  int64_t sa = 0;
  int sb = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) {
      a += sa;
      b += sb;
    }
    sa += wa[w];
    sb += wb[w];
  }
  *ta = sa;
  *tb = sb;
}

// The last i in [0, n) with first[i] <= k (first[0] <= k, non-decreasing).
__device__ __forceinline__ int last_le(const int32_t* first, int n, int k) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= k)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// One workgroup takes the requests NT at a time.  with_tokens: positions and slots
// too (all requests then fit one round), by more workgroups where there are many
// tokens: each makes the sums again, from inputs that nothing overwrites meanwhile,
// and deals out its share of the pages and tokens; the first alone writes the rest.  24000 tokens of 256 requests: one
// such launch 4.0 us, the sums and then request_tokens_kernel 6.0 (in a graph; 6.1 and
// 9.5 with the host's calls).
template <int NT>
__global__ __launch_bounds__(NT) void request_tables_kernel(TablesArgs A) {
  __shared__ int64_t wa[NT / 64];
  __shared__ int wb[NT / 64];
  __shared__ int32_t start_s[NT], first_s[NT], pages_s[NT], ctx_s[NT];
  const int tid = threadIdx.x;
  const int count = min(max(A.free_count[0], 0), A.num_free);
  const int bs = 1 << A.bs_log2;
  const bool writes = blockIdx.x == 0;
  int64_t tokens = 0;  // of the requests before this round
  int taken = 0;       // pages likewise
  for (int r0 = 0; r0 < A.num_reqs; r0 += NT) {
    const int r = r0 + tid, here = min(NT, A.num_reqs - r0);
    const bool real = r < A.num_reqs;
    const int n = real ? max(A.query[r], 0) : 0;
    const int ctx = real ? max(A.context[r], 0) : 0;
    const int pages = real ? min(max(A.num_pages[r], 0), A.max_blocks) : 0;
    const int64_t len = (int64_t)ctx + n;
    const int want = (int)min((len + bs - 1) >> A.bs_log2, (int64_t)A.max_blocks);
    const int need = real ? max(want - pages, 0) : 0;
    int64_t a = n, tn;
    int b = need, tp;
    scan2<NT>(a, b, &tn, &tp, wa, wb);
    const int start = (int)min(tokens + a - n, (int64_t)INT_MAX);
    const int first = taken + b - need;
    if (real && writes) {
      if (r == 0) st_agent(A.query_start, 0);
      st_agent(A.query_start + r + 1, (int32_t)min(tokens + a, (int64_t)INT_MAX));
      st_agent(A.seq_lens + r, (int32_t)min(len, (int64_t)INT_MAX));
      st_agent(A.num_pages_out + r, pages + min(need, max(count - first, 0)));
    }
    start_s[tid] = start;
    first_s[tid] = first;
    pages_s[tid] = pages;
    ctx_s[tid] = ctx;
    __syncthreads();
    const int64_t step = (int64_t)A.parts * NT;
    for (int64_t k0 = (int64_t)blockIdx.x * NT + tid; k0 < tp; k0 += step) {
      const int k = (int)k0;
      const int i = last_le(first_s, here, taken + k);
      const int at = count - 1 - (taken + k);
      st_agent(A.table + (int64_t)(r0 + i) * A.max_blocks + pages_s[i] + (taken + k - first_s[i]),
               at >= 0 ? A.free_pages[at] : -1);
    }
    if (A.with_tokens) {
      for (int64_t j0 = (int64_t)blockIdx.x * NT + tid; j0 < A.max_tokens; j0 += step) {
        const int j = (int)j0;
        int64_t pos = 0, slot = -1;
        if (j < tn) {
          const int i = last_le(start_s, here, j);
          pos = (int64_t)ctx_s[i] + (j - start_s[i]);
          const int64_t blk = pos >> A.bs_log2;
          if (blk < A.max_blocks) {
            // a page from before this step is in the table, a new one in the free list
            int page = -1;
            if (blk < pages_s[i]) {
              page = A.table[(int64_t)(r0 + i) * A.max_blocks + blk];
            } else {
              const int at = count - 1 - (first_s[i] + (int)blk - pages_s[i]);
              if (at >= 0) page = A.free_pages[at];
            }
            if (page >= 0) slot = ((int64_t)page << A.bs_log2) + (pos & (bs - 1));
          }
        }
        st_agent(reinterpret_cast<uint64_t*>(A.positions) + j, (uint64_t)pos);
        st_agent(reinterpret_cast<uint64_t*>(A.slots) + j, (uint64_t)slot);
      }
    }
    __syncthreads();  // start_s .. ctx_s are read out
    tokens += tn;
    taken += tp;
  }
  if (tid == 0 && writes) st_agent(A.free_count_out, max(count - taken, 0));
  stores_done();
}

// Positions and slots of the tokens, a thread a token, from the tables that
// request_tables_kernel left.  With up to LOCAL requests their offsets are read
// into LDS at once, so that the bisection's steps are LDS reads and not a chain
// of loads (24000 tokens of 256 requests: 3.9 us, 2.9 so).
constexpr int LOCAL = 1024;

template <bool IN_LDS>
__global__ __launch_bounds__(256) void request_tokens_kernel(
    const int32_t* query_start, const int32_t* context, const int32_t* table, int64_t* positions,
    int64_t* slots, int num_reqs, int max_tokens, int max_blocks, int bs_log2) {
  __shared__ int32_t start_s[IN_LDS ? LOCAL + 1 : 1];
  const int32_t* start = query_start;
  if constexpr (IN_LDS) {
    for (int r = threadIdx.x; r <= num_reqs; r += 256) start_s[r] = query_start[r];
    __syncthreads();
    start = start_s;
  }
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j < max_tokens) {
    int64_t pos = 0, slot = -1;
    if (j < start[num_reqs]) {
      const int i = last_le(start, num_reqs, j);
      pos = (int64_t)max(context[i], 0) + (j - start[i]);
      const int64_t blk = pos >> bs_log2;
      if (blk < max_blocks) {
        const int page = table[(int64_t)i * max_blocks + blk];
        if (page >= 0) slot = ((int64_t)page << bs_log2) + (pos & ((1 << bs_log2) - 1));
      }
    }
    st_agent(reinterpret_cast<uint64_t*>(positions) + j, (uint64_t)pos);
    st_agent(reinterpret_cast<uint64_t*>(slots) + j, (uint64_t)slot);
  }
  stores_done();
}

// Bound by the chain of a page's reads (bisection in LDS, its entry), NT pages at a
// time: 8192 pages of 256 requests 9.7 us.
//
// Gives back the pages beyond the first keep[r] tokens of every request, in request
// and block order: they are appended to the free list, their table entries become -1.
template <int NT>
__global__ __launch_bounds__(NT) void release_pages_kernel(const int32_t* keep, int32_t* num_pages,
                                                           int32_t* free_pages,
                                                           int32_t* free_count, int32_t* table,
                                                           int num_reqs, int max_blocks,
                                                           int num_free, int bs_log2) {
  __shared__ int64_t wa[NT / 64];
  __shared__ int wb[NT / 64];
  __shared__ int32_t first_s[NT], kept_s[NT];
  const int tid = threadIdx.x;
  const int count = min(max(free_count[0], 0), num_free);
  int given = 0;
  for (int r0 = 0; r0 < num_reqs; r0 += NT) {
    const int r = r0 + tid, here = min(NT, num_reqs - r0);
    const bool real = r < num_reqs;
    const int pages = real ? min(max(num_pages[r], 0), max_blocks) : 0;
    const int64_t len = real ? max(keep[r], 0) : 0;
    const int kept = (int)min((len + (1 << bs_log2) - 1) >> bs_log2, (int64_t)pages);
    int64_t a = 0, ta;
    int b = pages - kept, tb;
    scan2<NT>(a, b, &ta, &tb, wa, wb);
    first_s[tid] = given + b - (pages - kept);
    kept_s[tid] = kept;
    if (real) st_agent(num_pages + r, kept);
    __syncthreads();
    for (int k = tid; k < tb; k += NT) {
      const int i = last_le(first_s, here, given + k);
      int32_t* const e = table + (int64_t)(r0 + i) * max_blocks + kept_s[i] + (given + k - first_s[i]);
      const int page = *e;
      const int64_t at = (int64_t)count + given + k;
      if (at < num_free) st_agent(free_pages + at, page);
      st_agent(e, -1);
    }
    __syncthreads();
    given += tb;
  }
  if (tid == 0) st_agent(free_count, (int32_t)min((int64_t)count + given, (int64_t)num_free));
  stores_done();
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

#define SMX_TABLES_CHECKS()                                                                      \
  SMX_REQUIRE(num_reqs >= 1 && num_reqs <= 65535, "num_reqs must be in [1, 65535]");             \
  SMX_REQUIRE(max_blocks >= 1 && (int64_t)num_reqs * max_blocks <= INT_MAX - 4096,               \
              "num_reqs * max_blocks must be at most 2^31 - 4097");                              \
  SMX_REQUIRE(num_free >= 1, "the free list must have room for a page");                         \
  SMX_REQUIRE(block_size >= 1 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,     \
              "block_size must be a power of two in [1, 4096]")

extern "C" int smx_request_tables(void* stream, const int32_t* query_lens,
                                  const int32_t* context_lens, const int32_t* num_pages,
                                  const int32_t* free_pages, const int32_t* free_count,
                                  int32_t* block_table, int32_t* num_pages_out,
                                  int32_t* free_count_out, int32_t* query_start_loc,
                                  int32_t* seq_lens, int64_t* positions, int64_t* slot_mapping,
                                  int32_t num_reqs, int32_t max_tokens, int32_t max_blocks,
                                  int32_t num_free, int32_t block_size) {
  SMX_REQUIRE(query_lens && context_lens && num_pages && free_pages && free_count &&
                  block_table && num_pages_out && free_count_out && query_start_loc && seq_lens &&
                  positions && slot_mapping,
              "null pointer argument");
  SMX_REQUIRE(((uintptr_t)query_lens | (uintptr_t)context_lens | (uintptr_t)num_pages |
               (uintptr_t)free_pages | (uintptr_t)free_count | (uintptr_t)block_table |
               (uintptr_t)num_pages_out | (uintptr_t)free_count_out |
               (uintptr_t)query_start_loc | (uintptr_t)seq_lens) % 4 == 0 &&
                  ((uintptr_t)positions | (uintptr_t)slot_mapping) % 8 == 0,
              "int32 arrays must be 4-byte aligned, int64 arrays 8-byte");
  SMX_TABLES_CHECKS();
  SMX_REQUIRE(seq_lens != context_lens && seq_lens != query_lens,
              "seq_lens must not be context_lens or query_lens");
  SMX_REQUIRE(max_tokens >= 1, "max_tokens must be >= 1");
  smx::TablesArgs a{query_lens, context_lens, num_pages, free_pages, free_count, block_table,
                    num_pages_out, free_count_out, query_start_loc, seq_lens, positions,
                    slot_mapping, num_reqs, max_tokens, max_blocks, num_free, 0, 0, 1};
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  // One workgroup deals a few thousand tokens out in about a launch's time.  Several
  // must not see its outputs in their inputs.
  auto apart = [](const int32_t* in, const int32_t* out, int64_t n) {
    const uintptr_t a = (uintptr_t)in, b = (uintptr_t)out, bytes = 4 * (uintptr_t)n;
    return b + bytes <= a || a + bytes <= b;
  };
  const bool several = num_reqs <= 1024 && apart(num_pages, num_pages_out, num_reqs) &&
                       apart(free_count, free_count_out, 1);
  a.with_tokens = num_reqs <= 1024 && (max_tokens <= 4096 || several);
  // (tokens and pages by 256 threads a workgroup if those are all or there are more)
  const bool pages = max_tokens / block_size > 256;
  const int nt = num_reqs <= 256 && (max_tokens <= 256 || several || !(a.with_tokens || pages))
                     ? 256 : 1024;
  if (several) a.parts = (int)std::min<int64_t>(((int64_t)max_tokens + nt - 1) / nt, 2048);
  if (nt == 256)
    SMX_LAUNCH((smx::request_tables_kernel<256>), dim3((unsigned)a.parts), dim3(256), 0,
               (hipStream_t)stream, a);
  else
    SMX_LAUNCH((smx::request_tables_kernel<1024>), dim3((unsigned)a.parts), dim3(1024), 0,
               (hipStream_t)stream, a);
  if (!a.with_tokens) {
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    const dim3 grid((unsigned)(((int64_t)max_tokens + 255) / 256));
    if (num_reqs <= smx::LOCAL)
      SMX_LAUNCH((smx::request_tokens_kernel<true>), grid, dim3(256), 0, (hipStream_t)stream,
                 query_start_loc, context_lens, block_table, positions, slot_mapping, num_reqs,
                 max_tokens, max_blocks, a.bs_log2);
    else
      SMX_LAUNCH((smx::request_tokens_kernel<false>), grid, dim3(256), 0, (hipStream_t)stream,
                 query_start_loc, context_lens, block_table, positions, slot_mapping, num_reqs,
                 max_tokens, max_blocks, a.bs_log2);
  }
  return (int)hipGetLastError();
}

extern "C" int smx_release_pages(void* stream, const int32_t* keep_lens, int32_t* num_pages,
                                 int32_t* free_pages, int32_t* free_count, int32_t* block_table,
                                 int32_t num_reqs, int32_t max_blocks, int32_t num_free,
                                 int32_t block_size) {
  SMX_REQUIRE(keep_lens && num_pages && free_pages && free_count && block_table,
              "null pointer argument");
  SMX_REQUIRE(((uintptr_t)keep_lens | (uintptr_t)num_pages | (uintptr_t)free_pages |
               (uintptr_t)free_count | (uintptr_t)block_table) % 4 == 0,
              "int32 arrays must be 4-byte aligned");
  SMX_TABLES_CHECKS();
  int bs_log2 = 0;
  while ((1 << bs_log2) < block_size) ++bs_log2;
  // (us by 256 threads / by 1024, half of the table's pages given back: 16 rows of 8
  // entries 2.6 / 2.9, 16 of 64 3.3 / 3.1, 64 of 32 4.7 / 3.1, 256 of 64 29.3 / 9.7)
  if (num_reqs <= 256 && num_reqs * max_blocks <= 512)
    SMX_LAUNCH((smx::release_pages_kernel<256>), dim3(1), dim3(256), 0, (hipStream_t)stream,
               keep_lens, num_pages, free_pages, free_count, block_table, num_reqs, max_blocks,
               num_free, bs_log2);
  else
    SMX_LAUNCH((smx::release_pages_kernel<1024>), dim3(1), dim3(1024), 0, (hipStream_t)stream,
               keep_lens, num_pages, free_pages, free_count, block_table, num_reqs, max_blocks,
               num_free, bs_log2);
  return (int)hipGetLastError();
}
