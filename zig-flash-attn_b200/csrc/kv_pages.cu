// Pages of a key-value cache, for sm_100a: writing new tokens into them, copying them, and the bookkeeping of which
// sequence holds which page (reserve, fork, free, compact). The operators have no counterpart in the reference.
//
// The bookkeeping works on two integer tensors: the block table (sequences, max_pages), whose entry outside
// [0, num_pages) holds no page, and the reference counts (num_pages), where a count <= 0 marks a free page. The kernels
// read them and write new ones; nothing is changed in place. Every choice among free pages takes the lowest page first,
// and requests are served in the order (sequence, entry), so the results do not depend on the schedule.
#include <cooperative_groups.h>

#include "common.h"
#include "ptx.cuh"

namespace b200fa {

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------------------------- data: append and copy
struct CacheView {
  uint8_t* k;
  uint8_t* v;
  int64_t k_page, k_row, k_head, v_page, v_row, v_head;  // strides in bytes
  int num_pages, page_size, heads, chunks;               // chunks = 16-byte pieces of a row
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

// One warp per token: finds its sequence (binary search in the prefix sums of a packed batch), its page and its row.
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
    b = (int)(token / p.rows);
    row = index = token - b * p.rows;
  }
  const int64_t position = p.lengths[b] + index;
  if (position < 0 || position >= p.capacity) return;
  const int page = p.table[b * p.table_seq + position / p.cache.page_size];
  if (page < 0 || page >= p.cache.num_pages) return;
  const int64_t slot = position % p.cache.page_size;
  const int64_t seq = p.cu_seqlens ? 0 : b;
  for (int i = lane; i < p.cache.heads * p.cache.chunks; i += 32) {
    const int head = i / p.cache.chunks, chunk = i - head * p.cache.chunks;
    *reinterpret_cast<uint4*>(p.cache.k + page * p.cache.k_page + slot * p.cache.k_row + head * p.cache.k_head + 16 * chunk) =
        *reinterpret_cast<const uint4*>(p.k + seq * p.k_seq + row * p.k_row + head * p.k_head + 16 * chunk);
    *reinterpret_cast<uint4*>(p.cache.v + page * p.cache.v_page + slot * p.cache.v_row + head * p.cache.v_head + 16 * chunk) =
        *reinterpret_cast<const uint4*>(p.v + seq * p.v_seq + row * p.v_row + head * p.v_head + 16 * chunk);
  }
}

// One block per pair of pages; pairs with an entry outside [0, num_pages) are skipped.
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CacheView c, const int32_t* source,
                                                         const int32_t* target) {
  const int from = source[blockIdx.x], to = target[blockIdx.x];
  if (from < 0 || to < 0 || from >= c.num_pages || to >= c.num_pages || from == to) return;
  for (int i = threadIdx.x; i < c.page_size * c.heads * c.chunks; i += 256) {
    const int row = i / (c.heads * c.chunks), rest = i - row * (c.heads * c.chunks);
    const int head = rest / c.chunks, chunk = rest - head * c.chunks;
    const int64_t k_at = row * c.k_row + head * c.k_head + 16 * chunk, v_at = row * c.v_row + head * c.v_head + 16 * chunk;
    *reinterpret_cast<uint4*>(c.k + to * c.k_page + k_at) = *reinterpret_cast<const uint4*>(c.k + from * c.k_page + k_at);
    *reinterpret_cast<uint4*>(c.v + to * c.v_page + v_at) = *reinterpret_cast<const uint4*>(c.v + from * c.v_page + v_at);
  }
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

struct Range {
  int begin, end;
};
__device__ __forceinline__ Range team_range(cg::cluster_group team, int count) {
  const int each = (count + kTeamBlocks - 1) / kTeamBlocks, begin = imin((int)team.block_rank() * each, count);
  return {begin, imin(begin + each, count)};
}

// scratch[r] = r-th free page for r < wanted, refs_out[page] = 1 for these (where mark is set) and refs otherwise.
__device__ __forceinline__ void list_free_pages(const PagesParams& p, Range pages, int free_before, int wanted,
                                                int* warp_sums, bool mark) {
  int rank = free_before;
  for (int base = pages.begin; base < pages.end; base += kTeamThreads) {
    const int page = base + threadIdx.x;
    const int count = page < pages.end ? p.refs[page] : 1;
    const bool is_free = count <= 0;
    int total;
    const int at = rank + block_scan(is_free, warp_sums, &total);
    if (page < pages.end) {
      const bool taken = is_free && at < wanted;
      if (taken) p.scratch[at] = page;
      p.refs_out[page] = taken && mark ? 1 : count;
    }
    rank += total;
  }
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
  list_free_pages(p, pages, free_before, requests, warp_sums, true);
  for (int64_t i = (int64_t)seqs.begin * p.max_pages + threadIdx.x; i < (int64_t)seqs.end * p.max_pages; i += kTeamThreads) {
    const int b = (int)(i / p.max_pages), entry = (int)(i - (int64_t)b * p.max_pages);
    const int page = p.table[b * p.table_seq + entry];
    p.table_out[i] = holds_page(p, page) ? page : -1;
  }
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
  list_free_pages(p, pages, free_before, requests, warp_sums, true);
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
  for (int64_t i = (int64_t)children.begin * p.max_pages + threadIdx.x; i < (int64_t)children.end * p.max_pages;
       i += kTeamThreads) {
    const int child = (int)(i / p.max_pages), entry = (int)(i - (int64_t)child * p.max_pages);
    const int full = p.lengths_out[child] / p.page_size;
    int page = -1;
    if (entry < full) {
      page = p.table[p.extra[child] * p.table_seq + entry];
      if (holds_page(p, page)) atomicAdd(&p.refs_out[page], 1); else page = -1;
    } else if (entry == full) {
      page = p.target[child];
    }
    p.table_out[i] = page;
  }
}

__global__ void __cluster_dims__(kTeamBlocks) __launch_bounds__(kTeamThreads)
free_pages_kernel(const __grid_constant__ PagesParams p) {
  const cg::cluster_group team = cg::this_cluster();
  const Range seqs = team_range(team, p.sequences), pages = team_range(team, p.num_pages);
  for (int page = pages.begin + threadIdx.x; page < pages.end; page += kTeamThreads) p.refs_out[page] = p.refs[page];
  team.sync();
  for (int64_t i = (int64_t)seqs.begin * p.max_pages + threadIdx.x; i < (int64_t)seqs.end * p.max_pages; i += kTeamThreads) {
    const int b = (int)(i / p.max_pages), entry = (int)(i - (int64_t)b * p.max_pages);
    int page = p.table[b * p.table_seq + entry];
    if (!holds_page(p, page)) {
      page = -1;
    } else if (entry >= p.extra[b] && entry < p.extra2[b]) {
      atomicSub(&p.refs_out[page], 1);
      page = -1;
    }
    p.table_out[i] = page;
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
  int rank = live_before;
  for (int base = pages.begin; base < pages.end; base += kTeamThreads) {
    const int page = base + threadIdx.x;
    const bool is_live = page < pages.end && p.refs[page] > 0;
    int total;
    const int at = rank + block_scan(is_live, warp_sums, &total);
    if (page < pages.end) {
      if (is_live && page >= live) p.source[at - kept] = page;
      if (!is_live && page < live) p.target[page - at] = page;
      p.refs_out[page] = page < live ? p.refs[page] : 0;
    }
    rank += total;
  }
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
  for (int64_t i = (int64_t)seqs.begin * p.max_pages + threadIdx.x; i < (int64_t)seqs.end * p.max_pages; i += kTeamThreads) {
    const int b = (int)(i / p.max_pages), entry = (int)(i - (int64_t)b * p.max_pages);
    int page = p.table[b * p.table_seq + entry];
    if (!holds_page(p, page) || p.refs[page] <= 0) page = -1;
    else if (page >= live) page = p.scratch[page];
    p.table_out[i] = page;
  }
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
  view->num_pages = c.num_pages, view->page_size = c.page_size, view->heads = c.heads_kv, view->chunks = c.head_dim / 8;
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
  copy_pages_kernel<<<(unsigned)count, 256, 0, static_cast<cudaStream_t>(stream)>>>(view, source_pages, target_pages);
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
  free_pages_kernel<<<kTeamBlocks, kTeamThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
