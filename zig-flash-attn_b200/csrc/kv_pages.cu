// Pages of a key-value cache, for sm_100a: writing new tokens into them, copying them, and the bookkeeping of which
// sequence holds which page (reserve, fork, free, compact). The operators have no counterpart in the reference.
//
// The bookkeeping works on two integer tensors: the block table (sequences, max_pages), whose entry outside
// [0, num_pages) holds no page, and the reference counts (num_pages), where a count <= 0 marks a free page. The kernels
// read them and write new ones; nothing is changed in place. Every choice among free pages takes the lowest page first,
// and requests are served in the order (sequence, entry), so the results do not depend on the schedule.
#include <cooperative_groups.h>

#include "common.h"
#include "fwd_common.cuh"
#include "ptx.cuh"

namespace b200fa {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------------------------- data: append and copy
struct CacheView {
  uint8_t* k;
  uint8_t* v;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;  // strides in bytes
  int num_pages, page_size;
  FastDiv chunks, row_chunks;  // 16-byte pieces of a row of a head, and of all heads
};

struct AppendParams {
  CacheView cache;
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_seq, k_row, k_head, v_seq, v_row, v_head;  // strides in bytes
  const int32_t* cu_seqlens;                           // null: `rows` tokens of every sequence
  const int32_t* lengths;
  const int32_t* table;
  int64_t table_seq, rows;
  int batch, capacity;
};

// One warp per token: finds its sequence (binary search in the prefix sums of a packed batch), its page and its row, then
// copies the heads' pieces, four of each tensor in flight. HBM-bound from a few thousand tokens on: 31 k tokens of 8 x 128
// (129 MB moved) in 23 us; below that the chain length -> table -> page of dependent loads is what it takes, 4 us.
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  const int64_t token = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  int b;
  int64_t row, index;  // row of the token tensors, index within its sequence
  if (p.cu_seqlens) {
    if (token >= p.rows || token < p.cu_seqlens[0] || token >= p.cu_seqlens[p.batch]) return;
    int low = 0, high = p.batch;  // cu[low] <= token < cu[high]
    while (high - low > 1) {
      const int middle = (low + high) >> 1;
      if (p.cu_seqlens[middle] <= token) low = middle; else high = middle;
    }
    b = low;
    row = token;
    index = token - p.cu_seqlens[b];
  } else {
    if (token >= p.rows * p.batch) return;
    b = (int)token / (int)p.rows;  // both below 2^31
    row = index = token - (int64_t)b * p.rows;
  }
  const int64_t position = p.lengths[b] + index;
  if (position < 0 || position >= p.capacity) return;
  const int entry = (int)position / p.cache.page_size, slot = (int)position - entry * p.cache.page_size;
  const int page = p.table[b * p.table_seq + entry];
  if (page < 0 || page >= p.cache.num_pages) return;
  const int64_t seq = p.cu_seqlens ? 0 : b;
  const uint8_t* k_from = p.k + seq * p.k_seq + row * p.k_row;
  const uint8_t* v_from = p.v + seq * p.v_seq + row * p.v_row;
  uint8_t* k_to = p.cache.k + page * p.cache.k_page + slot * p.cache.k_row;
  uint8_t* v_to = p.cache.v + page * p.cache.v_page + slot * p.cache.v_row;
  const int pieces = (int)p.cache.row_chunks.divisor;
  for (int base = lane; base < pieces; base += 128) {
    uint4 k[4], v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * u, head = p.cache.chunks.div(i), at = 16 * (i - head * (int)p.cache.chunks.divisor);
      if (i < pieces) {
        k[u] = *reinterpret_cast<const uint4*>(k_from + head * p.k_head + at);
        v[u] = *reinterpret_cast<const uint4*>(v_from + head * p.v_head + at);
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * u, head = p.cache.chunks.div(i), at = 16 * (i - head * (int)p.cache.chunks.divisor);
      if (i < pieces) {
        *reinterpret_cast<uint4*>(k_to + head * p.cache.k_head + at) = k[u];
        *reinterpret_cast<uint4*>(v_to + head * p.cache.v_head + at) = v[u];
      }
    }
  }
}

// Page copies: one block per (pair, 16 KiB of a page, cache), so that a few pairs of large pages keep every SM busy as well
// as thousands of small ones do; a thread has four 16-byte pieces in flight. Pairs with an entry outside [0, num_pages) are
// skipped. HBM-bound: 3932 pairs of 32 KiB pages, 515 MB moved, in 83 us (6.2 TB/s); 64 pairs of 128 KiB pages in 6 us, with one
// block per pair 36 us.
constexpr int kCopyPieces = 1024;
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CacheView c, const int32_t* source,
                                                         const int32_t* target) {
  const int from = source[blockIdx.x], to = target[blockIdx.x];
  if (from < 0 || to < 0 || from >= c.num_pages || to >= c.num_pages || from == to) return;
  const bool is_v = blockIdx.z;
  const int64_t row_stride = is_v ? c.v_row : c.k_row, head_stride = is_v ? c.v_head : c.k_head;
  const uint8_t* read = is_v ? c.v + from * c.v_page : c.k + from * c.k_page;
  uint8_t* write = is_v ? c.v + to * c.v_page : c.k + to * c.k_page;
  const int pieces = c.page_size * (int)c.row_chunks.divisor, first = blockIdx.y * kCopyPieces + threadIdx.x;
  uint4 data[kCopyPieces / 256];
  int64_t at[kCopyPieces / 256];
#pragma unroll
  for (int u = 0; u < kCopyPieces / 256; ++u) {
    const int i = first + 256 * u;
    const int row = c.row_chunks.div(i), rest = i - row * (int)c.row_chunks.divisor;
    const int head = c.chunks.div(rest), chunk = rest - head * (int)c.chunks.divisor;
    at[u] = row * row_stride + head * head_stride + 16 * chunk;
    if (i < pieces) data[u] = *reinterpret_cast<const uint4*>(read + at[u]);
  }
#pragma unroll
  for (int u = 0; u < kCopyPieces / 256; ++u)
    if (first + 256 * u < pieces) *reinterpret_cast<uint4*>(write + at[u]) = data[u];
}

// ---------------------------------------------------------------------------------------------- bookkeeping
// One cluster works on a call: its blocks take contiguous ranges of the pages and of the sequences and exchange their
// counts through each other's shared memory.
constexpr int kTeamBlocks = 8, kTeamThreads = 1024;

struct PagesParams {
  const int32_t* table;    // (sequences, max_pages), row stride table_seq
  const int32_t* refs;     // (num_pages)
  const int32_t* lengths;  // (sequences)
  const int32_t* extra;    // reserve: new tokens; fork: parents; free: first entries
  const int32_t* extra2;   // free: last entries
  int32_t* table_out;      // (rows, max_pages) contiguous
  int32_t* refs_out;
  int32_t* lengths_out;    // fork: lengths of the children
  int32_t* source;
  int32_t* target;
  int32_t* scratch;        // num_pages
  int64_t table_seq;
  int sequences, rows, max_pages, num_pages, page_size, pairs;
};

// Sum of one value per thread over the block, for all threads.
__device__ __forceinline__ int block_sum(int value, int* warp_sums) {
  const int total = __reduce_add_sync(0xffffffffu, value);
  __syncthreads();  // the sums of an earlier call have been read
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = total;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, warp_sums[threadIdx.x & 31]);
}

// Exclusive prefix sum of one value per thread over the block; *total = the block's sum.
__device__ __forceinline__ int block_scan(int value, int* warp_sums, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inclusive = value;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, inclusive, d);
    if (lane >= d) inclusive += other;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = inclusive;
  __syncthreads();
  int sums = warp_sums[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sums, d);
    if (lane >= d) sums += other;
  }
  *total = __shfl_sync(0xffffffffu, sums, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, sums, (warp - 1) & 31) : 0;
  return before + inclusive - value;
}

// Sum of one value per block over the cluster; *before = over the blocks in front of this one. `slot` is this block's
// own place for the exchange: a place is written once per launch.
__device__ __forceinline__ int team_scan(cg::cluster_group team, int value, int* slot, int* before) {
  if (threadIdx.x == 0) *slot = value;
  team.sync();
  int total = 0;
  *before = 0;
  for (int r = 0; r < kTeamBlocks; ++r) {
    const int other = *team.map_shared_rank(slot, r);
    if (r < (int)team.block_rank()) *before += other;
    total += other;
  }
  return total;
}

// visit(row, entry, load(row, entry)) for all entries of the rows [begin, end), a warp per row, four loads of a lane in flight
// (sixteen measured the same).
template <typename Load, typename Visit>
__device__ __forceinline__ void for_rows(int begin, int end, int columns, Load load, Visit visit) {
  const int lane = threadIdx.x & 31;
  for (int row = begin + (threadIdx.x >> 5); row < end; row += kTeamThreads / 32) {
    for (int base = lane; base < columns; base += 128) {
      int value[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) value[u] = base + 32 * u < columns ? load(row, base + 32 * u) : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (base + 32 * u < columns) visit(row, base + 32 * u, value[u]);
    }
  }
}

struct Range {
  int begin, end;
};
__device__ __forceinline__ Range team_range(cg::cluster_group team, int count) {
  const int each = (count + kTeamBlocks - 1) / kTeamBlocks, begin = imin((int)team.block_rank() * each, count);
  return {begin, imin(begin + each, count)};
}

// Walks a range of pages in order: visit(page, count, is, before) with the page's reference count, whether test(count) holds,
// and for how many pages in front of it test holds, `before` the range included. (Eight pages per thread and round: the
// same or slower.)
template <typename Test, typename Visit>
__device__ __forceinline__ void rank_pages(const PagesParams& p, Range pages, int before, int* warp_sums, Test test, Visit visit) {
  for (int base = pages.begin; base < pages.end; base += kTeamThreads) {
    const int page = base + threadIdx.x;
    const int count = page < pages.end ? p.refs[page] : 0;
    const bool is = page < pages.end && test(count);
    int total;
    const int rank = before + block_scan(is, warp_sums, &total);
    if (page < pages.end) visit(page, count, is, rank);
    before += total;
  }
}

// scratch[r] = r-th free page and refs_out[page] = 1 for r < wanted; the other counts are copied.
__device__ __forceinline__ void list_free_pages(const PagesParams& p, Range pages, int free_before, int wanted, int* warp_sums) {
  rank_pages(p, pages, free_before, warp_sums, [](int count) { return count <= 0; },
             [&](int page, int count, bool is_free, int rank) {
               const bool taken = is_free && rank < wanted;
               if (taken) p.scratch[rank] = page;
               p.refs_out[page] = taken ? 1 : count;
             });
}

__device__ __forceinline__ int count_free(const PagesParams& p, Range pages, int* warp_sums) {
  int mine = 0;
  for (int page = pages.begin + threadIdx.x; page < pages.end; page += kTeamThreads) mine += p.refs[page] <= 0;
  return block_sum(mine, warp_sums);
}

// Entries of sequence b that lack a page for the tokens to come: [first, last).
__device__ __forceinline__ Range missing_entries(const PagesParams& p, int b) {
  const int64_t length = imax(p.lengths[b], 0), need = length + imax(p.extra[b], 0);
  const int64_t first = (length + p.page_size - 1) / p.page_size, last = (need + p.page_size - 1) / p.page_size;
  return {(int)(first < p.max_pages ? first : p.max_pages), (int)(last < p.max_pages ? last : p.max_pages)};
}

__device__ __forceinline__ bool holds_page(const PagesParams& p, int entry) { return entry >= 0 && entry < p.num_pages; }

__global__ void __cluster_dims__(kTeamBlocks) __launch_bounds__(kTeamThreads)
reserve_pages_kernel(const __grid_constant__ PagesParams p) {
  __shared__ int warp_sums[32], exchange[2];
  const cg::cluster_group team = cg::this_cluster();
  const Range seqs = team_range(team, p.sequences), pages = team_range(team, p.num_pages);
  int mine = 0;
  for (int b = seqs.begin + threadIdx.x; b < seqs.end; b += kTeamThreads) {
    const Range e = missing_entries(p, b);
    for (int i = e.begin; i < e.end; ++i) mine += !holds_page(p, p.table[b * p.table_seq + i]);
  }
  const int requests_here = block_sum(mine, warp_sums);
  const int free_here = count_free(p, pages, warp_sums);
  int requests_before, free_before;
  const int requests = team_scan(team, requests_here, &exchange[0], &requests_before);
  const int free_pages = team_scan(team, free_here, &exchange[1], &free_before);
  list_free_pages(p, pages, free_before, requests, warp_sums);
  for_rows(seqs.begin, seqs.end, p.max_pages, [&](int b, int entry) { return p.table[b * p.table_seq + entry]; },
           [&](int b, int entry, int page) { p.table_out[(int64_t)b * p.max_pages + entry] = holds_page(p, page) ? page : -1; });
  team.sync();  // the list of free pages and the copies of the rows are complete
  int rank = requests_before;
  for (int base = seqs.begin; base < seqs.end; base += kTeamThreads) {
    const int b = base + threadIdx.x;
    Range e{0, 0};
    int count = 0;
    if (b < seqs.end) {
      e = missing_entries(p, b);
      for (int i = e.begin; i < e.end; ++i) count += !holds_page(p, p.table[b * p.table_seq + i]);
    }
    int total;
    int at = rank + block_scan(count, warp_sums, &total);
    for (int i = e.begin; i < e.end; ++i) {
      if (holds_page(p, p.table[b * p.table_seq + i])) continue;
      if (at < free_pages) p.table_out[(int64_t)b * p.max_pages + i] = p.scratch[at];
      ++at;
    }
    rank += total;
  }
}

// Length of child i (0 when its parent is no sequence) and the page that it needs a copy of (-1: none).
__device__ __forceinline__ int child_length(const PagesParams& p, int i, int* copied) {
  const int parent = p.extra[i];
  *copied = -1;
  if (parent < 0 || parent >= p.sequences) return 0;
  const int64_t capacity = (int64_t)p.max_pages * p.page_size;
  int length = imax(p.lengths[parent], 0);
  if (length > capacity) length = (int)capacity;
  if (length % p.page_size) {
    const int page = p.table[parent * p.table_seq + length / p.page_size];
    if (holds_page(p, page)) *copied = page;
  }
  return length;
}

__global__ void __cluster_dims__(kTeamBlocks) __launch_bounds__(kTeamThreads)
fork_pages_kernel(const __grid_constant__ PagesParams p) {
  __shared__ int warp_sums[32], exchange[2];
  const cg::cluster_group team = cg::this_cluster();
  const Range children = team_range(team, p.rows), pages = team_range(team, p.num_pages);
  int mine = 0, copied;
  for (int i = children.begin + threadIdx.x; i < children.end; i += kTeamThreads) {
    child_length(p, i, &copied);
    mine += copied >= 0;
  }
  const int requests_here = block_sum(mine, warp_sums);
  const int free_here = count_free(p, pages, warp_sums);
  int requests_before, free_before;
  const int requests = team_scan(team, requests_here, &exchange[0], &requests_before);
  const int free_pages = team_scan(team, free_here, &exchange[1], &free_before);
  list_free_pages(p, pages, free_before, requests, warp_sums);
  team.sync();  // the list of free pages and the copy of the counts are complete
  int rank = requests_before;
  for (int base = children.begin; base < children.end; base += kTeamThreads) {
    const int i = base + threadIdx.x;
    copied = -1;
    int length = 0;
    if (i < children.end) length = child_length(p, i, &copied);
    int total;
    const int at = rank + block_scan(copied >= 0, warp_sums, &total);
    if (i < children.end) {
      const int page = copied >= 0 && at < free_pages ? p.scratch[at] : -1;
      p.lengths_out[i] = length;
      p.source[i] = page >= 0 ? copied : -1;
      p.target[i] = page;
    }
    rank += total;
  }
  __syncthreads();  // the targets of this block's children
  for_rows(
      children.begin, children.end, p.max_pages,
      [&](int child, int entry) {
        const int full = p.lengths_out[child] / p.page_size;
        return entry < full ? p.table[p.extra[child] * p.table_seq + entry] : entry == full ? p.target[child] : -1;
      },
      [&](int child, int entry, int page) {
        if (!holds_page(p, page)) page = -1;
        else if (entry < p.lengths_out[child] / p.page_size) atomicAdd(&p.refs_out[page], 1);
        p.table_out[(int64_t)child * p.max_pages + entry] = page;
      });
}

// refs_out holds a copy of the counts. No order between the rows is needed, so this one runs on the whole GPU, a warp per
// row: 512 rows of 502 entries, 95 k of them freed, with the copy in 7 us, as one cluster 15 us (8 SMs are slow at the
// reductions).
__global__ void __launch_bounds__(256) free_pages_kernel(const __grid_constant__ PagesParams p) {
  const int lane = threadIdx.x & 31, b = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (b >= p.sequences) return;
  const int first = p.extra[b], last = p.extra2[b];
  const int32_t* row = p.table + b * p.table_seq;
  int32_t* row_out = p.table_out + (int64_t)b * p.max_pages;
#pragma unroll 4
  for (int entry = lane; entry < p.max_pages; entry += 32) {
    int page = row[entry];
    if (!holds_page(p, page)) {
      page = -1;
    } else if (entry >= first && entry < last) {
      atomicSub(&p.refs_out[page], 1);
      page = -1;
    }
    row_out[entry] = page;
  }
}

__global__ void __cluster_dims__(kTeamBlocks) __launch_bounds__(kTeamThreads)
compact_pages_kernel(const __grid_constant__ PagesParams p) {
  __shared__ int warp_sums[32], exchange[2];
  const cg::cluster_group team = cg::this_cluster();
  const Range seqs = team_range(team, p.sequences), pages = team_range(team, p.num_pages);
  int live_before, kept_before;
  const int live = team_scan(team, pages.end - pages.begin - count_free(p, pages, warp_sums), &exchange[0], &live_before);
  int mine = 0;  // live pages that stay: those in front of `live`
  for (int page = pages.begin + threadIdx.x; page < imin(pages.end, live); page += kTeamThreads) mine += p.refs[page] > 0;
  const int kept = team_scan(team, block_sum(mine, warp_sums), &exchange[1], &kept_before);
  const int moves = live - kept;
  rank_pages(p, pages, live_before, warp_sums, [](int count) { return count > 0; },
             [&](int page, int count, bool is_live, int rank) {
               if (is_live && page >= live) p.source[rank - kept] = page;
               if (!is_live && page < live) p.target[page - rank] = page;
               p.refs_out[page] = page < live ? count : 0;
             });
  team.sync();
  for (int i = (int)team.block_rank() * kTeamThreads + threadIdx.x; i < p.pairs; i += kTeamBlocks * kTeamThreads) {
    if (i < moves) {
      const int from = p.source[i], to = p.target[i];
      p.scratch[from] = to;
      p.refs_out[to] = p.refs[from];
    } else {
      p.source[i] = -1;
      p.target[i] = -1;
    }
  }
  team.sync();
  for_rows(seqs.begin, seqs.end, p.max_pages,
           [&](int b, int entry) {
             const int page = p.table[b * p.table_seq + entry];
             if (!holds_page(p, page) || p.refs[page] <= 0) return -1;
             return page >= live ? p.scratch[page] : page;
           },
           [&](int b, int entry, int page) { p.table_out[(int64_t)b * p.max_pages + entry] = page; });
}

// ---------------------------------------------------------------------------------------------- host side
static int cache_view(const b200fa_kv_cache& c, CacheView* view) {
  B200FA_REQUIRE(c.num_pages >= 0 && c.page_size > 0 && c.heads_kv > 0, "a cache needs a positive page size and head count");
  B200FA_REQUIRE(c.head_dim > 0 && c.head_dim % 8 == 0 && c.head_dim <= 1024,
                 "head_dim must be a multiple of 8 of at most 1024, got %d", c.head_dim);
  B200FA_REQUIRE((int64_t)c.page_size * c.heads_kv * (c.head_dim / 8) < 0x7fffffffll, "a page has more than 2^31 pieces of 16 bytes");
  for (int i = 0; i < 3; ++i)
    B200FA_REQUIRE(c.k_stride[i] % 8 == 0 && c.v_stride[i] % 8 == 0, "tensor strides must be multiples of 8 elements");
  B200FA_REQUIRE(c.num_pages == 0 || (c.k_cache && c.v_cache), "null tensor pointer");
  B200FA_REQUIRE(reinterpret_cast<uintptr_t>(c.k_cache) % 16 == 0 && reinterpret_cast<uintptr_t>(c.v_cache) % 16 == 0,
                 "tensor pointers must be 16-byte aligned");
  view->k = static_cast<uint8_t*>(c.k_cache);
  view->v = static_cast<uint8_t*>(c.v_cache);
  view->k_page = 2 * c.k_stride[0], view->k_row = 2 * c.k_stride[1], view->k_head = 2 * c.k_stride[2];
  view->v_page = 2 * c.v_stride[0], view->v_row = 2 * c.v_stride[1], view->v_head = 2 * c.v_stride[2];
  view->num_pages = c.num_pages, view->page_size = c.page_size;
  view->chunks = FastDiv::make((uint32_t)c.head_dim / 8), view->row_chunks = FastDiv::make((uint32_t)(c.heads_kv * (c.head_dim / 8)));
  return B200FA_OK;
}

static int pages_params(const b200fa_pages_args* a, PagesParams* p) {
  B200FA_REQUIRE(a != nullptr, "null arguments");
  B200FA_REQUIRE(a->sequences >= 0 && a->rows >= 0 && a->max_pages >= 0 && a->num_pages >= 0, "negative sizes");
  B200FA_REQUIRE(a->page_size > 0, "page_size must be positive");
  B200FA_REQUIRE((int64_t)a->max_pages * a->page_size < 0x7fffff00ll, "the block table covers more than 2^31 - 256 keys");
  B200FA_REQUIRE(a->num_pages < 0x7fff0000, "too many pages");
  B200FA_REQUIRE(a->num_pages == 0 || (a->page_refs && a->page_refs_out), "null tensor pointer");
  B200FA_REQUIRE((int64_t)a->sequences * a->max_pages == 0 || a->block_table, "null tensor pointer");
  B200FA_REQUIRE((int64_t)a->rows * a->max_pages == 0 || a->block_table_out, "null tensor pointer");
  p->table = a->block_table, p->refs = a->page_refs, p->lengths = a->cache_seqlens;
  p->table_out = a->block_table_out, p->refs_out = a->page_refs_out, p->lengths_out = nullptr;
  p->extra = p->extra2 = nullptr;
  p->source = a->source_pages, p->target = a->target_pages;
  p->scratch = static_cast<int32_t*>(a->workspace);
  p->table_seq = a->table_stride;
  p->sequences = a->sequences, p->rows = a->rows, p->max_pages = a->max_pages, p->num_pages = a->num_pages;
  p->page_size = a->page_size, p->pairs = 0;
  return B200FA_OK;
}

static int needs_scratch(const b200fa_pages_args* a) {
  B200FA_REQUIRE(a->workspace_bytes >= b200fa_pages_workspace_bytes(a->num_pages) && (a->num_pages == 0 || a->workspace),
                 "page workspace is too small: need %zu bytes", b200fa_pages_workspace_bytes(a->num_pages));
  B200FA_REQUIRE(reinterpret_cast<uintptr_t>(a->workspace) % 4 == 0, "page workspace must be 4-byte aligned");
  return B200FA_OK;
}

}  // namespace b200fa

using namespace b200fa;

extern "C" {

int b200fa_append_kv(const b200fa_append_args* a, void* stream) {
  B200FA_REQUIRE(a != nullptr, "null arguments");
  AppendParams p;
  int status = cache_view(a->cache, &p.cache);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(a->batch >= 0 && a->rows >= 0 && a->max_pages >= 0, "negative sizes");
  B200FA_REQUIRE((int64_t)a->max_pages * a->cache.page_size < 0x7fffff00ll, "the block table covers more than 2^31 - 256 keys");
  for (int i = 0; i < 3; ++i)
    B200FA_REQUIRE(a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0, "tensor strides must be multiples of 8 elements");
  const int64_t tokens = a->cu_seqlens ? a->rows : a->rows * a->batch;
  if (tokens == 0 || a->batch == 0 || a->max_pages == 0 || a->cache.num_pages == 0) return B200FA_OK;
  B200FA_REQUIRE(a->k && a->v && a->cache_seqlens && a->block_table, "null tensor pointer");
  B200FA_REQUIRE(reinterpret_cast<uintptr_t>(a->k) % 16 == 0 && reinterpret_cast<uintptr_t>(a->v) % 16 == 0,
                 "tensor pointers must be 16-byte aligned");
  B200FA_REQUIRE(tokens < 0x7fffffffll, "too many tokens for one call");
  p.k = static_cast<const uint8_t*>(a->k), p.v = static_cast<const uint8_t*>(a->v);
  p.k_seq = 2 * a->k_stride[0], p.k_row = 2 * a->k_stride[1], p.k_head = 2 * a->k_stride[2];
  p.v_seq = 2 * a->v_stride[0], p.v_row = 2 * a->v_stride[1], p.v_head = 2 * a->v_stride[2];
  p.cu_seqlens = a->cu_seqlens, p.lengths = a->cache_seqlens, p.table = a->block_table;
  p.table_seq = a->table_stride, p.rows = a->rows, p.batch = a->batch, p.capacity = a->max_pages * a->cache.page_size;
  append_kernel<<<(unsigned)((tokens + 7) / 8), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

int b200fa_copy_pages(const b200fa_kv_cache* cache, const int32_t* source_pages, const int32_t* target_pages, int32_t count,
                      void* stream) {
  B200FA_REQUIRE(cache != nullptr, "null arguments");
  CacheView view;
  const int status = cache_view(*cache, &view);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(count >= 0, "negative sizes");
  if (count == 0 || cache->num_pages == 0) return B200FA_OK;
  B200FA_REQUIRE(source_pages && target_pages, "null tensor pointer");
  const int64_t pieces = (int64_t)cache->page_size * cache->heads_kv * (cache->head_dim / 8);
  const int64_t parts = (pieces + kCopyPieces - 1) / kCopyPieces;
  B200FA_REQUIRE(parts < 65536, "a page is larger than 1 GiB");
  copy_pages_kernel<<<dim3((unsigned)count, (unsigned)parts, 2), 256, 0, static_cast<cudaStream_t>(stream)>>>(view, source_pages, target_pages);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

size_t b200fa_pages_workspace_bytes(int32_t num_pages) { return num_pages > 0 ? (size_t)num_pages * 4 : 0; }

int b200fa_reserve_pages(const b200fa_pages_args* a, const int32_t* new_tokens, void* stream) {
  PagesParams p;
  int status = pages_params(a, &p);
  if (status == B200FA_OK) status = needs_scratch(a);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(a->rows == a->sequences, "block_table_out must have the rows of block_table");
  B200FA_REQUIRE(a->sequences == 0 || (a->cache_seqlens && new_tokens), "null tensor pointer");
  p.extra = new_tokens;
  reserve_pages_kernel<<<kTeamBlocks, kTeamThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

int b200fa_fork_pages(const b200fa_pages_args* a, const int32_t* parents, int32_t* child_seqlens, void* stream) {
  PagesParams p;
  int status = pages_params(a, &p);
  if (status == B200FA_OK) status = needs_scratch(a);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(a->rows == 0 || (parents && child_seqlens && a->source_pages && a->target_pages), "null tensor pointer");
  B200FA_REQUIRE(a->sequences == 0 || a->cache_seqlens, "null tensor pointer");
  p.extra = parents;
  p.lengths_out = child_seqlens;
  fork_pages_kernel<<<kTeamBlocks, kTeamThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

int b200fa_free_pages(const b200fa_pages_args* a, const int32_t* first_entry, const int32_t* last_entry, void* stream) {
  PagesParams p;
  const int status = pages_params(a, &p);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(a->rows == a->sequences, "block_table_out must have the rows of block_table");
  B200FA_REQUIRE(a->sequences == 0 || (first_entry && last_entry), "null tensor pointer");
  p.extra = first_entry;
  p.extra2 = last_entry;
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (a->num_pages > 0)
    B200FA_CUDA_CHECK(cudaMemcpyAsync(a->page_refs_out, a->page_refs, (size_t)a->num_pages * 4, cudaMemcpyDeviceToDevice, s));
  if (a->sequences == 0 || a->max_pages == 0) return B200FA_OK;
  free_pages_kernel<<<(unsigned)((a->sequences + 7) / 8), 256, 0, s>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

int b200fa_compact_pages(const b200fa_pages_args* a, void* stream) {
  PagesParams p;
  int status = pages_params(a, &p);
  if (status == B200FA_OK) status = needs_scratch(a);
  if (status != B200FA_OK) return status;
  B200FA_REQUIRE(a->rows == a->sequences, "block_table_out must have the rows of block_table");
  p.pairs = a->num_pages / 2;
  B200FA_REQUIRE(p.pairs == 0 || (a->source_pages && a->target_pages), "null tensor pointer");
  compact_pages_kernel<<<kTeamBlocks, kTeamThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

}  // extern "C"
