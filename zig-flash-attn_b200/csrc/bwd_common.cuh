// Shared pieces of the backward kernels: the parameter block, small shared-memory helpers and the launcher of the
// head_dim 256 main kernel (defined in bwd_d256.cu, called from bwd.cu).
#pragma once

#include "common.h"
#include "ptx.cuh"

namespace b200fa {

constexpr float kLog2e = 1.4426950408889634f;
// The reference's rule (zig/fragments.zig:23-30): a key with a probability above 3/4 is the pivot of its row.
constexpr float kPivotProbability = 0.75f;
// Row sums of BF16 dS are multiples of 2^-133; scaled by 2^7 every nonzero sum is a normal FP32 number, which the
// reductions (red.add.f32 flushes subnormal numbers) keep (reference zig/BackwardParams.zig:52-58).
constexpr float kPivotSumScale = 128.f;
// The pivot terms of dK are summed in FP32 by atomic adds, scaled by 2^40 for the same reason: a term as small as
// 2^-166 stays normal, sums up to 2^87 stay finite.
constexpr float kDkFixScale = 1099511627776.f;

// Sinks make the first key blocks of a sequence heavy: every query row sees them, while the others are seen by a window of
// rows. Their work is therefore dealt out in shares of `rows` query rows, one CTA each (rows = 0: it is not), which start
// first and leave FP32 parts of dK and dV, added up in order by the postprocess launch. Sequences of a packed batch with at
// most `rows` query rows have one share, which writes dK and dV itself; with at most `least`, where a sink's key block weighs
// no more than the others, none (their blocks stay in the main list). A longer one that starts at query row q0 has the slots
// from 2 q0 / rows (rounded down) on: with x = its rows / `rows` > 1 it has ceil(x) <= floor(2 x) shares, so no two shares have
// the same slot. There are at most 2 rows_total / rows slots and rows_total / rows + rows_total / least shares, however many
// sequences there are. (1024 documents of 128 tokens, 32/8 heads of 128, 4 sinks, forward and backward: 3.44 ms, 3.40 without
// sinks; with a part and a slot for every document 4.21 ms and 1 GB more.)
struct SinkShares {
  int rows;             // query rows per share, a multiple of 128
  int least;            // packed: sequences of at most so many query rows have no shares; at most `rows`
  int blocks;           // key blocks per sequence that hold sinks, at most
  int ctas;             // leading CTAs (grid.x) that hold shares: fixed length over all head slots, packed per head slot
  int per_sequence;     // fixed length: shares (and slots) per sequence
  bool joins_entries;   // packed: the parts are joined by a walk over the list instead of over the sequences
  const int2* list;     // packed: (sequence, share) entries
  float* part;          // (slots, heads_kv, blocks, dV and dK, 128, compiled width)
};

struct BwdParams {
  Problem prob;
  float scale, scale_log2;
  const float* lse_log2;  // (heads_q, rows) : -lse * log2(e)
  const float* dpsum;     // (heads_q, rows) : -sum_d O * dO
  int64_t rows;           // rows of the statistics / dQ accumulator per head (batch * seqlen_q or total_q)
  // Pivot rows (at most one key of a query row holds more than 3/4 of its probability): the main kernel leaves the dS
  // of that key out, records the key in `pivot_key` (tensor row of K, -1 = none) and adds the BF16 dS of the other keys,
  // times kPivotSumScale, into `pivot_sum`; the postprocess kernel takes the dS of the pivot as minus that sum. Both are
  // (heads_q, rows). Null: pivot gradients are off (b200fa_set_pivot_ds).
  float* pivot_sum;
  int* pivot_key;
  int head_dim;           // columns of the tensors (<= the compiled D; TMA zero-fills the columns in between)
  int dkv_wide;           // 1: dK and dV rows may be written with 32-byte stores (alignment of bases and strides)
  __nv_bfloat16* dk;
  __nv_bfloat16* dv;
  int64_t dk_batch_stride, dk_row_stride, dk_head_stride;
  int64_t dv_batch_stride, dv_row_stride, dv_head_stride;
  const int2* work_list;  // packed problems: (key sequence, key block) per blockIdx.x
  int n_blocks, head_slots, section;  // fixed length: decoding of the linear CTA index, see bwd_cta_of
  SinkShares sinks;                   // kSink instances
  int* status;
  long long* trace;  // optional cycle counters, null = off
};

__device__ __forceinline__ void cp_async_4(uint32_t smem_dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_arrive_noinc(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

// Fixed-length problems launch a one-dimensional grid. CTAs start in index order, so the order decides both the tail of
// the launch and what runs together: a section of `section` (batch entry, head slot) pairs is walked key block by key
// block, first (under a causal mask: heaviest) key blocks first, then the next section. The CTAs that run together
// then read the Q, dO and dQ-accumulator rows of a few heads only, which stay in L2, and the light CTAs of a section
// fill the tail of its heavy ones.
struct BwdCta {
  int seq, n_block, head_slot;
};
__device__ __forceinline__ BwdCta bwd_cta_of(const BwdParams& p, int linear) {
  const int groups = p.prob.batch * p.head_slots;
  const int per_section = p.section * p.n_blocks;
  const int s = linear / per_section, r = linear - s * per_section;
  const int n = imin(p.section, groups - s * p.section);
  BwdCta c;
  c.n_block = r / n;
  const int g = s * p.section + (r - c.n_block * n);
  c.seq = g / p.head_slots;
  c.head_slot = g - c.seq * p.head_slots;
  return c;
}

// What a CTA of a main kernel works on: a key block of a sequence (seq >= batch: nothing), and with kSink, share >= 0, only a
// share of its query rows (SinkShares).
struct BwdItem {
  int seq, n_block, head_slot, share;
};
// Whether a sequence of a packed batch has more than one share, so that these leave parts.
__device__ __forceinline__ bool has_parts(const BwdParams& p, int seq) {
  return p.prob.cu_q[seq + 1] - p.prob.cu_q[seq] > p.sinks.rows;
}
template <bool kSink>
__device__ __forceinline__ BwdItem bwd_item_of(const BwdParams& p, int head_slots) {
  BwdItem item{p.prob.batch, 0, 0, -1};
  if (kSink && blockIdx.x < p.sinks.ctas) {
    const int entry = blockIdx.x / p.sinks.blocks;
    item.n_block = blockIdx.x - entry * p.sinks.blocks;
    if (p.sinks.list) {
      const int2 e = p.sinks.list[entry];
      item.seq = e.x;
      item.share = e.x < p.prob.batch && has_parts(p, e.x) ? e.y : -1;
      item.head_slot = blockIdx.y;
    } else {
      const int pair = entry / p.sinks.per_sequence;
      item.share = entry - pair * p.sinks.per_sequence;
      item.seq = pair / head_slots;
      item.head_slot = pair - item.seq * head_slots;
    }
    return item;
  }
  const int linear = kSink ? blockIdx.x - p.sinks.ctas : blockIdx.x;
  if (p.work_list) {
    const int2 e = p.work_list[linear];
    item.seq = e.x;
    item.n_block = e.y;
    item.head_slot = blockIdx.y;
    if (kSink && p.sinks.rows && item.n_block * kBlockN < p.prob.sink && item.seq < p.prob.batch &&
        p.prob.cu_q[item.seq + 1] - p.prob.cu_q[item.seq] > p.sinks.least)
      item.seq = p.prob.batch;  // the shares' part
  } else {
    const BwdCta cta = bwd_cta_of(p, linear);
    item.seq = cta.seq;
    item.n_block = cta.n_block;
    item.head_slot = cta.head_slot;
    if (kSink && p.sinks.rows) item.n_block += p.sinks.blocks;  // the launch leaves the blocks of the shares out
  }
  return item;
}

// First slot of a sequence's shares.
__device__ __forceinline__ int64_t sink_slot(const BwdParams& p, const SeqInfo& s, int seq) {
  return p.prob.cu_q ? 2 * (int64_t)s.q0 / p.sinks.rows : (int64_t)seq * p.sinks.per_sequence;
}

// Where a share leaves row `row` of its FP32 sums: dV (which = 0) or dK (1), `width` columns.
__device__ __forceinline__ float* sink_part_row(const BwdParams& p, const SeqInfo& s, int seq, int share, int kv_head, int n_block,
                                                int which, int row, int width) {
  const int64_t slot = sink_slot(p, s, seq) + share;
  return p.sinks.part + ((((slot * p.prob.heads_kv + kv_head) * p.sinks.blocks + n_block) * 2 + which) * kBlockN + row) * width;
}

// Main kernel for head_dim in (128, 256]: grid.y = 2 * heads_kv (kv head, half of the head dimension).
int launch_bwd_main_d256(const b200fa_bwd_args& a, const BwdParams& p, dim3 grid, float* dq_accum, int64_t stat_rows,
                         cudaStream_t stream);

}  // namespace b200fa
