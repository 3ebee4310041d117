// Pages of the cache that several rows of the block tables share (gfx950): block tables of
// the rows that a step goes on with (beams of a search, samples of a prompt), pages moved
// to the front of the pool, and the copies of pages that both ask for.
//
// Who holds a page is read off the tables: a page is in use where a row lists it among its
// num_pages first, and free again once no row does.  No counts are kept, so that there
// are none to go wrong.  A workgroup collects the pages in bit sets in LDS (32768 pages
// a 4 KB set); nothing of a call is left for the next.
//
// One workgroup has all of what the tables say (the others copy): bound by its chains of
// loads and LDS operations.  us: 512 rows of up to 34 pages 12.9, 4 rows 5.3 (a wave a row 57);
// the moves of 256 rows of up to 17 pages in a pool of 2198 14.5, of 16 rows 5.6 (with a
// search for every moved entry 57).  Copies go at memory's rate: 433 MB read and written in 74
// us (5.9 TB/s, some of it from the caches), 1 GB in 195.
#include <limits.h>

#include <algorithm>

#include "smx_common.h"
#include "smx_launch.h"

namespace smx {
namespace {

constexpr int NT = 1024;
constexpr int MAX_PAGES = 1 << 18;

// A row's first `kept` pages go to its children; the tail, a last page that is not full,
// to the first of them alone.
struct ForkArgs {
  const int32_t* parents;
  const int32_t* lens;
  const int32_t* num_pages;
  const int32_t* free_pages;
  const int32_t* free_count;
  const int32_t* table;
  int32_t* table_out;
  int32_t* num_pages_out;
  int32_t* lens_out;
  int32_t* free_pages_out;
  int32_t* free_count_out;
  int32_t* copies;  // [rows, 2]
  int rows, max_blocks, num_blocks, num_free, bs_log2;
};

__device__ __forceinline__ void set_bit(uint32_t* set, int i) {
  atomicOr(set + (i >> 5), 1u << (i & 31));
}
__device__ __forceinline__ bool get_bit(const uint32_t* set, int i) {
  return set[i >> 5] >> (i & 31) & 1;
}

// Inclusive prefix sums over a workgroup; *total the sum.
__device__ __forceinline__ int scan(int v, int* total, int* waves) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = wave_scan_i32(v);
  __syncthreads();  // the last call's sums have been read
  if (lane == 63) waves[wave] = v;
  __syncthreads();
  int sum = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w == wave) v += sum;
    sum += waves[w];
  }
  *total = sum;
  return v;
}

// Calls f(row, aux of the row, place, entry) for the first `pages` entries of each row: 16
// lanes a row, a wave eight rows at a time with eight loads a lane on their way (rows of
// some tens of pages are the common ones), the rows' sizes by one load for 64 of them.
template <typename Pages, typename Aux, typename F>
__device__ __forceinline__ void each_entry(const int32_t* table, int rows, int max_blocks,
                                           Pages pages_of, Aux aux_of, F f) {
  constexpr int WAVES = NT / 64, HELD = 4, SIDE = 2, LANES = 16, AT_ONCE = 64 / LANES;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int base = wave; base < rows; base += NT) {
    const int own = base + WAVES * lane;
    const int pages = own < rows ? pages_of(own) : 0, aux = own < rows ? aux_of(own) : 0;
    const int n = min(64, (rows - base + WAVES - 1) / WAVES);
    for (int l = lane / LANES; l - lane / LANES < n; l += AT_ONCE * SIDE) {
      int count[SIDE], extra[SIDE];
#pragma unroll
      for (int h = 0; h < SIDE; ++h) {  // (a lane past the rows has no pages)
        count[h] = __shfl(pages, l + AT_ONCE * h);
        extra[h] = __shfl(aux, l + AT_ONCE * h);
      }
      int b0 = lane % LANES;
      while (__builtin_amdgcn_ballot_w64(b0 < max(count[0], count[1]))) {
        int v[SIDE][HELD];
#pragma unroll
        for (int h = 0; h < SIDE; ++h)
#pragma unroll
          for (int k = 0; k < HELD; ++k)
            if (b0 + LANES * k < count[h])
              v[h][k] = table[(int64_t)(base + WAVES * (l + AT_ONCE * h)) * max_blocks + b0 +
                              LANES * k];
#pragma unroll
        for (int h = 0; h < SIDE; ++h)
#pragma unroll
          for (int k = 0; k < HELD; ++k)
            if (b0 + LANES * k < count[h])
              f(base + WAVES * (l + AT_ONCE * h), extra[h], b0 + LANES * k, v[h][k]);
        b0 += LANES * HELD;
      }
    }
  }
}

// A row's pages, tokens and pages kept.
__device__ __forceinline__ void row_sizes(const ForkArgs& A, int r, int& pages, int& len,
                                          int& kept) {
  pages = min(max(A.num_pages[r], 0), A.max_blocks);
  len = (int)min((int64_t)max(A.lens[r], 0), (int64_t)pages << A.bs_log2);
  kept = (int)(((int64_t)len + (1 << A.bs_log2) - 1) >> A.bs_log2);
}

// Workgroup 0 does all but the tables' whole columns, which the others copy: 16 rows each,
// a wave a row.
template <int PAGES, int ROWS>
__global__ __launch_bounds__(NT) void fork_pages_kernel(ForkArgs A) {
  __shared__ uint32_t listed[PAGES / 32];  // by an old row, other than as a page that stays
  __shared__ uint32_t live[PAGES / 32];    // whole in a row with children; then all that stay
  __shared__ uint32_t twice[PAGES / 32];   // listed twice among the kept pages of such rows
  __shared__ int first_s[ROWS];            // a row's first child, INT_MAX: none
  __shared__ int waves[NT / 64];
  const int tid = threadIdx.x;
  const int bs = 1 << A.bs_log2;
  if (blockIdx.x > 0) {
    const int j = (blockIdx.x - 1) * (NT / 64) + (tid >> 6), lane = tid & 63;
    if (j < A.rows) {
      const int r = A.parents[j];
      const bool ok = r >= 0 && r < A.rows;
      int pages, len, kept = 0, tail = -1;
      if (ok) {
        row_sizes(A, r, pages, len, kept);
        if (len & (bs - 1)) tail = kept - 1;  // workgroup 0 writes it
      }
      const int32_t* const src = A.table + (int64_t)(ok ? r : 0) * A.max_blocks;
      int32_t* const dst = A.table_out + (int64_t)j * A.max_blocks;
      for (int b = lane; b < A.max_blocks; b += 64)
        if (b != tail) st_agent(dst + b, b < kept ? src[b] : -1);
    }
    stores_done();
    return;
  }
  // What the threads' old rows end with, and their new rows: asked for before all else.
  constexpr int OWN = ROWS / NT;
  const int words = (A.num_blocks + 31) / 32;
  const int count = min(max(A.free_count[0], 0), A.num_free);
  int parent[OWN], kept[OWN], len[OWN], page[OWN], tail[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int j = tid + i * NT;
    parent[i] = page[i] = tail[i] = -1;
    kept[i] = len[i] = 0;
    if (j < A.rows) {
      int pages, n, k;
      row_sizes(A, j, pages, n, k);
      if (n & (bs - 1)) tail[i] = A.table[(int64_t)j * A.max_blocks + k - 1];
      const int r = A.parents[j];
      if (r >= 0 && r < A.rows) {
        parent[i] = r;
        row_sizes(A, r, pages, len[i], kept[i]);
        if (len[i] & (bs - 1)) page[i] = A.table[(int64_t)r * A.max_blocks + kept[i] - 1];
      }
    }
  }
  for (int i = tid; i < words; i += NT) listed[i] = live[i] = twice[i] = 0;
  for (int i = tid; i < A.rows; i += NT) first_s[i] = INT_MAX;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i)
    if (parent[i] >= 0) atomicMin(first_s + parent[i], tid + i * NT);
  __syncthreads();
  const auto pages_of = [&](int r) { return min(max(A.num_pages[r], 0), A.max_blocks); };
  const auto whole_of = [&](int r) {
    int pages, n, k;
    row_sizes(A, r, pages, n, k);
    return first_s[r] == INT_MAX ? 0 : n >> A.bs_log2;
  };
  each_entry(A.table, A.rows, A.max_blocks, pages_of, whole_of,
             [&](int, int whole, int b, int p) {
               if ((unsigned)p >= (unsigned)A.num_blocks) return;
               if (b >= whole) {
                 set_bit(listed, p);
                 return;
               }
               const uint32_t bit = 1u << (p & 31);
               if (atomicOr(live + (p >> 5), bit) & bit) set_bit(twice, p);
             });
  __syncthreads();
  // ---- tails: which of their pages are whole ones elsewhere, then which are listed twice
  // (each new row takes a copy of such a page, so that it stays only as a whole one)
  bool only[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    const int r = tid + i * NT;
    if ((unsigned)tail[i] >= (unsigned)A.num_blocks || first_s[r] == INT_MAX) tail[i] = -1;
    only[i] = tail[i] >= 0 && !get_bit(live, tail[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i)
    if (tail[i] >= 0) {
      const uint32_t bit = 1u << (tail[i] & 31);
      if (atomicOr(live + (tail[i] >> 5), bit) & bit) set_bit(twice, tail[i]);
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OWN; ++i)
    if (only[i] && get_bit(twice, tail[i]))
      atomicAnd(live + (tail[i] >> 5), ~(1u << (tail[i] & 31)));
  // ---- copies, in the order of the new rows, from the end of the free list
  int taken = 0;
#pragma unroll
  for (int i = 0; i < OWN; ++i) {
    if (i * NT >= A.rows) break;
    const int j = tid + i * NT;
    const bool ends = len[i] & (bs - 1);
    const bool copy = ends && (unsigned)page[i] < (unsigned)A.num_blocks &&
                      (first_s[parent[i]] != j || get_bit(twice, page[i]));
    int all;
    const int at = count - taken - scan(copy, &all, waves);
    if (j < A.rows) {
      int src = -1, dst = -1;
      if (copy) {
        // (an entry of the free list outside the pool is no page)
        dst = at >= 0 ? A.free_pages[at] : -1;
        if ((unsigned)dst >= (unsigned)A.num_blocks) dst = -1;
        if (dst >= 0) src = page[i];
      }
      if (ends)
        st_agent(A.table_out + (int64_t)j * A.max_blocks + kept[i] - 1, copy ? dst : page[i]);
      if (copy && dst < 0) {  // no room: the row ends with its whole pages
        --kept[i];
        len[i] = kept[i] << A.bs_log2;
      }
      st_agent(A.num_pages_out + j, kept[i]);
      st_agent(A.lens_out + j, len[i]);
      st_agent(A.copies + 2 * j, src);
      st_agent(A.copies + 2 * j + 1, dst);
    }
    taken += all;
  }
  __syncthreads();
  // ---- pages that no new row lists: free again
  const int left = max(count - taken, 0);
  for (int i = tid; i < left; i += NT)
    if (A.free_pages_out != A.free_pages) st_agent(A.free_pages_out + i, A.free_pages[i]);
  int given = 0;
  for (int w0 = 0; w0 < words; w0 += NT) {
    const int w = w0 + tid;
    uint32_t bits = w < words ? listed[w] & ~live[w] : 0;
    int all;
    int at = left + given + scan(__popc(bits), &all, waves) - __popc(bits);
    while (bits) {
      if (at < A.num_free) st_agent(A.free_pages_out + at, w * 32 + __ffs(bits) - 1);
      bits &= bits - 1;
      ++at;
    }
    given += all;
  }
  const int now = min(left + given, A.num_free);
  for (int i = now + tid; i < A.num_free; i += NT) st_agent(A.free_pages_out + i, -1);
  if (tid == 0) st_agent(A.free_count_out, now);
  stores_done();
}

struct CompactArgs {
  const int32_t* num_pages;
  const int32_t* table;
  int32_t* table_out;
  int32_t* free_pages;  // [num_blocks]
  int32_t* free_count;
  int32_t* moves;  // [num_blocks / 2, 2]
  int rows, max_blocks, num_blocks;
};

// With U pages in use, those from U on move to the unused ones below it, in order: the
// k-th such page to the k-th such place.  Both ranks come from the sums of the set's words;
// the tables' new entries are read off the list of moves.
__global__ __launch_bounds__(NT) void compact_pages_kernel(CompactArgs A) {
  __shared__ uint32_t used[MAX_PAGES / 32];
  __shared__ int32_t before[MAX_PAGES / 32];  // pages in use before a word's
  __shared__ int waves[NT / 64];
  const int tid = threadIdx.x;
  const int words = (A.num_blocks + 31) / 32;
  for (int i = tid; i < words; i += NT) used[i] = 0;
  __syncthreads();
  const auto pages_of = [&](int r) { return min(max(A.num_pages[r], 0), A.max_blocks); };
  each_entry(A.table, A.rows, A.max_blocks, pages_of, [](int) { return 0; },
             [&](int, int, int, int p) {
               if ((unsigned)p < (unsigned)A.num_blocks) set_bit(used, p);
             });
  __syncthreads();
  int total = 0;
  for (int w0 = 0; w0 < words; w0 += NT) {
    const int w = w0 + tid;
    const int c = w < words ? __popc(used[w]) : 0;
    int all;
    const int upto = scan(c, &all, waves);
    if (w < words) before[w] = total + upto - c;
    total += all;
  }
  __syncthreads();
  auto rank_of = [&](int p) {  // pages in use below p
    return before[p >> 5] + __popc(used[p >> 5] & ((1u << (p & 31)) - 1));
  };
  const int kept = total > 0 ? rank_of(total - 1) + get_bit(used, total - 1) : 0;  // below `total`
  // Moves: a thread a word, its pages in use from `total` on and its unused ones below it.
  const int moved = total - kept;
  for (int w = tid; w < words; w += NT) {
    const int rest = total - 32 * w;  // the word's pages below `total`
    const uint32_t low = rest >= 32 ? ~0u : rest <= 0 ? 0u : (1u << rest) - 1;
    int k = before[w] + __popc(used[w] & low) - kept;
    for (uint32_t bits = used[w] & ~low; bits; bits &= bits - 1)
      st_agent(A.moves + 2 * k++, 32 * w + __ffs(bits) - 1);
    k = 32 * w - before[w];
    for (uint32_t bits = ~used[w] & low; bits; bits &= bits - 1)
      st_agent(A.moves + 2 * k++ + 1, 32 * w + __ffs(bits) - 1);
  }
  for (int i = 2 * moved + tid; i < 2 * (A.num_blocks / 2); i += NT) st_agent(A.moves + i, -1);
  stores_done();
  __syncthreads();
  each_entry(A.table, A.rows, A.max_blocks, [&](int) { return A.max_blocks; }, pages_of,
             [&](int r, int pages, int b, int p) {
               if (b >= pages || (unsigned)p >= (unsigned)A.num_blocks)
                 p = -1;
               else if (p >= total)
                 p = __hip_atomic_load(A.moves + 2 * (rank_of(p) - kept) + 1, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
               st_agent(A.table_out + (int64_t)r * A.max_blocks + b, p);
             });
  for (int i = tid; i < A.num_blocks; i += NT)
    st_agent(A.free_pages + i, i < A.num_blocks - total ? A.num_blocks - 1 - i : -1);
  if (tid == 0) st_agent(A.free_count, A.num_blocks - total);
  stores_done();
}

// One plane of a cache: its pages are `bytes` each, one after another from `base`.
struct PagePlane {
  uint64_t base;
  int64_t bytes;
};

// Copies page src to page dst in every plane for each pair (src, dst); a pair with an
// entry outside the pool is skipped.  Bound by memory.  Grid: pieces, planes, pairs.
constexpr int PIECE = 16384;  // bytes a workgroup copies

__global__ __launch_bounds__(256) void copy_pages_kernel(const PagePlane* __restrict__ planes,
                                                         const int32_t* __restrict__ pairs,
                                                         int num_blocks) {
  const int src = pairs[2 * blockIdx.z], dst = pairs[2 * blockIdx.z + 1];
  if ((unsigned)src >= (unsigned)num_blocks || (unsigned)dst >= (unsigned)num_blocks ||
      src == dst)
    return;
  const PagePlane pl = planes[blockIdx.y];
  const uint8_t* const from = (const uint8_t*)pl.base + src * pl.bytes;
  uint8_t* const to = (uint8_t*)pl.base + dst * pl.bytes;
  u32x4 v[4];
  const int64_t at = (int64_t)blockIdx.x * PIECE + threadIdx.x * 16;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < pl.bytes) v[i] = *reinterpret_cast<const u32x4*>(from + at + i * 4096);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 4096 < pl.bytes) st_agent_b128(to + at + i * 4096, v[i]);
  stores_done();
}

}  // namespace
}  // namespace smx

#include "smx_abi_util.h"

#define SMX_PAGES_CHECKS()                                                                       \
  SMX_REQUIRE(num_rows >= 1 && num_rows <= 8192, "num_rows must be in [1, 8192]");               \
  SMX_REQUIRE(max_blocks >= 1 && (int64_t)num_rows * max_blocks <= INT_MAX - 4096,               \
              "num_rows * max_blocks must be at most 2^31 - 4097");                              \
  SMX_REQUIRE(num_blocks >= 1 && num_blocks <= smx::MAX_PAGES,                                   \
              "num_blocks must be in [1, 262144]")

namespace {
// Whether [a, a + bytes) and [b, b + bytes) are apart.
bool apart(const void* a, const void* b, int64_t bytes) {
  return (uintptr_t)a + bytes <= (uintptr_t)b || (uintptr_t)b + bytes <= (uintptr_t)a;
}
}  // namespace

extern "C" int smx_fork_pages(void* stream, const int32_t* parents, const int32_t* lens,
                              const int32_t* num_pages, const int32_t* free_pages,
                              const int32_t* free_count, const int32_t* block_table,
                              int32_t* block_table_out, int32_t* num_pages_out, int32_t* lens_out,
                              int32_t* free_pages_out, int32_t* free_count_out, int32_t* copies,
                              int32_t num_rows, int32_t max_blocks, int32_t num_blocks,
                              int32_t num_free, int32_t block_size) {
  SMX_REQUIRE(parents && lens && num_pages && free_pages && free_count && block_table &&
                  block_table_out && num_pages_out && lens_out && free_pages_out &&
                  free_count_out && copies,
              "null pointer argument");
  SMX_REQUIRE(((uintptr_t)parents | (uintptr_t)lens | (uintptr_t)num_pages |
               (uintptr_t)free_pages | (uintptr_t)free_count | (uintptr_t)block_table |
               (uintptr_t)block_table_out | (uintptr_t)num_pages_out | (uintptr_t)lens_out |
               (uintptr_t)free_pages_out | (uintptr_t)free_count_out | (uintptr_t)copies) % 4 == 0,
              "int32 arrays must be 4-byte aligned");
  SMX_PAGES_CHECKS();
  SMX_REQUIRE(num_free >= 1, "the free list must have room for a page");
  SMX_REQUIRE(block_size >= 1 && block_size <= 4096 && (block_size & (block_size - 1)) == 0,
              "block_size must be a power of two in [1, 4096]");
  // (a new row reads another old one's: the workgroups run side by side)
  const int64_t row_bytes = 4 * (int64_t)num_rows, table_bytes = row_bytes * max_blocks;
  SMX_REQUIRE(apart(block_table, block_table_out, table_bytes),
              "block_table_out must be apart from block_table");
  for (const int32_t* in : {parents, lens, num_pages})
    for (const int32_t* out : {num_pages_out, lens_out})
      SMX_REQUIRE(apart(in, out, row_bytes),
                  "num_pages_out and lens_out must be apart from parents, lens and num_pages");
  SMX_REQUIRE(free_pages == free_pages_out || apart(free_pages, free_pages_out, 4 * (int64_t)num_free),
              "free_pages_out must be free_pages or apart from it");
  smx::ForkArgs a{parents, lens, num_pages, free_pages, free_count, block_table, block_table_out,
                  num_pages_out, lens_out, free_pages_out, free_count_out, copies, num_rows,
                  max_blocks, num_blocks, num_free, 0};
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  const dim3 grid(1 + (num_rows + smx::NT / 64 - 1) / (smx::NT / 64));
  // (less to clear: 4 rows 5.3 us, with the large sets 6.8; 512 rows 20.7 and 22.4)
  const auto kernel = num_blocks <= 32768 && num_rows <= 2048
      ? smx::fork_pages_kernel<32768, 2048> : smx::fork_pages_kernel<smx::MAX_PAGES, 8192>;
  SMX_LAUNCH(kernel, grid, dim3(smx::NT), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

extern "C" int smx_compact_pages(void* stream, const int32_t* num_pages,
                                 const int32_t* block_table, int32_t* block_table_out,
                                 int32_t* free_pages, int32_t* free_count, int32_t* moves,
                                 int32_t num_rows, int32_t max_blocks, int32_t num_blocks) {
  SMX_REQUIRE(num_pages && block_table && block_table_out && free_pages && free_count && moves,
              "null pointer argument");
  SMX_REQUIRE(((uintptr_t)num_pages | (uintptr_t)block_table | (uintptr_t)block_table_out |
               (uintptr_t)free_pages | (uintptr_t)free_count | (uintptr_t)moves) % 4 == 0,
              "int32 arrays must be 4-byte aligned");
  SMX_PAGES_CHECKS();
  SMX_REQUIRE(block_table == block_table_out ||
                  apart(block_table, block_table_out, 4 * (int64_t)num_rows * max_blocks),
              "block_table_out must be block_table or apart from it");
  const smx::CompactArgs a{num_pages, block_table, block_table_out, free_pages, free_count, moves,
                           num_rows, max_blocks, num_blocks};
  SMX_LAUNCH(smx::compact_pages_kernel, dim3(1), dim3(smx::NT), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}

extern "C" int smx_copy_pages(void* stream, const int64_t* planes, int32_t num_planes,
                              int64_t max_page_bytes, const int32_t* pairs, int32_t num_pairs,
                              int32_t num_blocks) {
  SMX_REQUIRE(planes && pairs, "null pointer argument");
  SMX_REQUIRE((uintptr_t)planes % 8 == 0 && (uintptr_t)pairs % 4 == 0,
              "planes must be 8-byte aligned, pairs 4-byte");
  SMX_REQUIRE(num_planes >= 1 && num_planes <= 65535, "num_planes must be in [1, 65535]");
  SMX_REQUIRE(num_pairs >= 1 && num_pairs <= smx::MAX_PAGES, "num_pairs must be in [1, 262144]");
  SMX_REQUIRE(num_blocks >= 1, "num_blocks must be >= 1");
  SMX_REQUIRE(max_page_bytes >= 16 && max_page_bytes <= (1ll << 31), "max_page_bytes out of range");
  const unsigned pieces = (unsigned)((max_page_bytes + smx::PIECE - 1) / smx::PIECE);
  for (int32_t at = 0; at < num_pairs; at += 65535) {
    const dim3 grid(pieces, num_planes, std::min(num_pairs - at, 65535));
    SMX_LAUNCH(smx::copy_pages_kernel, grid, dim3(256), 0, (hipStream_t)stream,
               reinterpret_cast<const smx::PagePlane*>(planes), pairs + 2 * at, num_blocks);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
  }
  return 0;
}
