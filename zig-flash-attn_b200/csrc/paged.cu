// Attention of one new token per sequence over a paged key-value cache, for sm_100a.
//
//   out[b, h] = sum_j p_j V[j],  p_j = exp(scale q[b, h] . K[j] - lse[b, h])  over the keys j that the token sees
//
// (b200fa_paged_decode; the visible keys are those of PagedRange in paged_index.h.) The operator has no counterpart in
// the reference.
//
// What bounds it: every visible row of K and V is read once, 4 D bytes for 4 D flops per query head of the group, so HBM
// does. The matrix work is a few percent of what even warp-level MMAs can do, and a tcgen05 pipeline would only add
// hand-overs between its roles; what matters is bytes in flight and short chains. So a warp is a pipeline of its own, with
// no barrier between warps until the end:
//   - Keys on the M side: S^T = K Q^T and O^T = V^T P^T (mma.sync m16n8k16), 16 keys a step, the query heads of the group
//     on the N side, where 8 (NT = 1), 16 or 32 of them cost no padding on the streamed operand.
//   - A dot product does not care about the order of its terms, and neither does the order of the output columns matter
//     until they are stored. Both are permuted so that what one thread needs of K and of V for its fragments is whole
//     16-byte pieces: no transposition and no ldmatrix.
//   - Each warp has a ring of its own in shared memory, filled by TMA boxes of 64 columns and 16 or 8 keys (pages whose
//     size is a multiple of 8), its lane 0 issuing. Other page sizes are copied row by row with cp.async, every thread
//     into places that it alone reads back; that stops at 4.1 to 4.8 TB/s, whatever
//     is computed next to it.
//   - The maximum of a column moves only when a score exceeds it by more than 8 (in log2 units), so a step costs one vote
//     instead of a reduction over the lanes. Sums are kept per lane and added up at the end.
// The grid is one wave of blocks, and the steps of all (key head, sequence) pairs, laid end to end, are cut into as many
// equal ranges: every SM is busy until the end however uneven the lengths are. (Shares per sequence, dealt out as whole
// blocks, left the SMs idle a quarter of the time: 235 us instead of 173 us for 64 sequences of 100 to 8192 tokens.) A
// block derives its range from the lengths. Pairs that lie within one range are finished in place; of a pair that is cut,
// every range leaves a part, and a second kernel joins them.
#include "common.h"
#include "fwd_common.cuh"
#include "paged_index.h"
#include "ptx.cuh"

namespace b200fa {

struct PagedParams {
  int batch, heads_q, heads_kv, group, head_dim, num_pages, capacity, window_left, sink;
  FastDiv page_size, chunks;  // chunks of 8 * NT query heads per key head
  int columns, ranges;        // chunks of all key heads; ranges = blocks
  float scale_log2;
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const int32_t* table;
  const int32_t* lengths;
  __nv_bfloat16* out;
  float* lse;
  // Parts of cut pairs, two slots per range: 2 r + 1 for the pair that begins in range r, 2 r for one that began before.
  float* o_part;    // (slots, 8 * NT, head_dim): sum of p V relative to the part's maximum
  float2* ml_part;  // (slots, 8 * NT): maximum (log2 units) and sum of p
  int4* cut;        // (ranges): of the pair that the range begins inside of (sequence, chunk, first range, last range)
  int box_rows;     // keys per TMA box: 16 or 8
  int* status;      // device status word of the library (bounded waits)
  int64_t q_seq, q_head, k_page, k_row, k_head, v_page, v_row, v_head, out_seq, out_head, table_seq;
};

// ---------------------------------------------------------------------------------------------- small wrappers
__device__ __forceinline__ void cp_async_16(uint32_t smem, const void* global, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(global), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// c += a b: a 16 x 16 (row), b 16 x 8 (column), BF16 in, FP32 sums
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Four columns of an output row from their sums, and the row's log-sum-exp. `total` is 0 where no key is seen; a NaN among the
// scores, or an infinite one, makes it NaN, and the row with it.
__device__ __forceinline__ void store_output(const PagedParams& p, int b, int head, int d, float4 sum, float top, float total) {
  const float inv = total == 0.f ? 0.f : 1.f / total;
  *reinterpret_cast<uint2*>(p.out + b * p.out_seq + head * p.out_head + d) =
      make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
  if (d == 0) p.lse[(int64_t)b * p.heads_q + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
}

// ---------------------------------------------------------------------------------------------- dealing out the steps
constexpr int kMinSteps = 6;  // a range has so many steps at least: one per warp at head_dim up to 128

// A sequence without visible keys still has one (empty) step, in which its zeros are written.
__device__ __forceinline__ int steps_of(const PagedParams& p, int b) {
  return imax(1, paged_range(p.lengths[b], p.capacity, p.window_left, p.sink).steps);
}

// Block-wide exclusive prefix sum; adds the block's sum to *total.
template <int kThreads>
__device__ __forceinline__ int64_t prefix_sum(int mine, int64_t* total, int64_t* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inclusive = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t other = __shfl_up_sync(0xffffffffu, inclusive, d);
    if (lane >= d) inclusive += other;
  }
  __syncthreads();  // the sums of an earlier call have been read
  if (lane == 31) warp_sums[warp] = inclusive;
  __syncthreads();
  int64_t before = *total;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    *total += warp_sums[w];
  }
  return before + inclusive - mine;
}

// Quotient of non-negative numbers; the 64-bit division is a subroutine of some hundred instructions.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

// `work` steps in `ranges` ranges whose sizes differ by one at most, the longer ones first.
struct Deal {
  int64_t work, base;
  int ranges, longer;
  __device__ __forceinline__ Deal(int64_t steps, int blocks) : work(steps) {
    const int64_t wanted = quotient(steps + kMinSteps - 1, kMinSteps);
    ranges = wanted < blocks ? (int)wanted : blocks;
    base = quotient(steps, ranges);
    longer = (int)(steps - base * ranges);
  }
  __device__ __forceinline__ int64_t start(int r) const { return base * r + imin(r, longer); }
  __device__ __forceinline__ int owner(int64_t at) const {
    const int64_t front = (base + 1) * longer;
    return (int)(at < front ? quotient(at, base + 1) : longer + quotient(at - front, base));
  }
};

// ---------------------------------------------------------------------------------------------- the ranges
template <int D, int NT>
struct PagedConfig {
  // Twelve warps per SM, each with two steps in its ring, read 6.4 TB/s on 64 sequences of 100 to 8192 tokens (head_dim
  // 128); eight warps with three steps 6.2, four with six 5.4: what counts is how many warps refill at the same time.
  // 32 query heads of head_dim 128 leave registers for eight warps; from head_dim 256 on the ring sets the number.
  static constexpr int kWarps = D <= 128 ? (D == 128 && NT == 4 ? 4 : 6) : 3;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStepBytes = 2 * kPagedStep * D * 2;         // K and V of a step
  static constexpr int kStages = D == 64 ? 4 : D == 128 && NT == 4 ? 3 : 2;
  static constexpr int kRingBytes = kWarps * kStages * kStepBytes;  // 96 KiB (head_dim 512: 192 KiB)
  static constexpr int kColumns = 8 * NT;
  static constexpr int kMergeBytes = kWarps * kColumns * (D * 4 + 8);  // over the ring, at the end of a pair
  static constexpr int kSmemBytes = (kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes) + 1024;  // alignment slack
  static constexpr int kBlocksPerSm = D <= 256 ? 2 : 1;
};

// kTma: page_size is a multiple of 8 and the ring is filled by TMA; otherwise each lane copies its own pieces.
template <int D, int NT, bool kTma>
__global__ void __launch_bounds__(PagedConfig<D, NT>::kThreads, PagedConfig<D, NT>::kBlocksPerSm)
paged_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ PagedParams p) {
  using Cfg = PagedConfig<D, NT>;
  constexpr int kStages = Cfg::kStages, kThreads = Cfg::kThreads, kPanelBytes = kPagedStep * 128;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t barriers[Cfg::kWarps][kStages];
  __shared__ int64_t warp_sums[Cfg::kWarps], found_first;
  __shared__ int found, abort_word;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);  // swizzled boxes: 1024-byte pattern
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const WaitCtx wctx{&abort_word, p.status, nullptr};
  if (kTma && threadIdx.x == 32) {
    tma_prefetch_descriptor(&map_k);
    tma_prefetch_descriptor(&map_v);
  }
  if (threadIdx.x == 0) {
    abort_word = 0;
    for (int i = 0; i < Cfg::kWarps * kStages; ++i) mbar_init(smem_u32(&barriers[0][0]) + 8 * i, 1);
    fence_barrier_init();
  }

  // ---- this block's range: steps [position, last) of the pairs in the order (chunk, sequence, step), or, where the table is
  // too short for pairs to be cut, pairs [position, last)
  const bool whole_pairs = p.cut == nullptr;
  int64_t position, last, pair_start;
  int chunk, b;
  Deal deal(1, 1);
  if (whole_pairs) {
    const int64_t pairs = (int64_t)p.columns * p.batch;
    position = quotient(pairs * blockIdx.x, gridDim.x);
    last = quotient(pairs * (blockIdx.x + 1), gridDim.x);
    pair_start = position;
    chunk = (int)quotient(position, p.batch);
    b = (int)(position - (int64_t)chunk * p.batch);
    __syncthreads();  // the barriers are initialised
  } else {
    int64_t round = 0, before = 0;  // steps of all sequences; of those in front of this thread's
    int mine = 0;
    for (int base = 0; base < p.batch; base += kThreads) {
      const int seq = base + threadIdx.x;
      mine = seq < p.batch ? steps_of(p, seq) : 0;
      before = prefix_sum<kThreads>(mine, &round, warp_sums);
    }
    deal = Deal(round * p.columns, p.ranges);
    if (blockIdx.x >= deal.ranges) {
      if (threadIdx.x == 0) p.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    position = deal.start(blockIdx.x);
    last = deal.start(blockIdx.x + 1);
    chunk = (int)quotient(position, round);
    const int64_t offset = position - chunk * round;
    if (p.batch <= kThreads) {
      if (before <= offset && offset < before + mine) found = threadIdx.x, found_first = before;
    } else {
      int64_t total = 0;
      for (int base = 0; base < p.batch && total <= offset; base += kThreads) {
        const int seq = base + threadIdx.x;
        mine = seq < p.batch ? steps_of(p, seq) : 0;
        before = prefix_sum<kThreads>(mine, &total, warp_sums);
        if (before <= offset && offset < before + mine) found = seq, found_first = before;
      }
    }
    __syncthreads();
    b = found;
    pair_start = chunk * round + found_first;
  }

  const uint32_t ring = smem_u32(smem) + warp * kStages * Cfg::kStepBytes, bars = smem_u32(&barriers[warp][0]);
  // Where this lane finds its pieces in the ring slot of a step. TMA: panels of 16 keys x 64 columns, 128 bytes a key, the
  // 16-byte pieces of key r in the order of the 128-byte swizzle (piece ^ (r & 7)); keys 8 to 15 are 1024 bytes behind keys
  // 0 to 7. Otherwise: the lane's own pieces one after the other, 512 bytes apart.
  const uint32_t k_place = kTma ? g * 128 + ((t ^ g) << 4) : lane * 16;
  const uint32_t v_place0 = kTma ? 2 * t * 128 + ((g ^ (2 * t)) << 4) : lane * 16;
  const uint32_t v_place1 = (2 * t + 1) * 128 + ((g ^ (2 * t + 1)) << 4);
  uint32_t parity = 0;  // bit s: parity of the next completion of the barrier of stage s

  for (bool first_pair = true; position < last; first_pair = false) {
    const int kv_head = p.chunks.div(chunk), column0 = (chunk - kv_head * (int)p.chunks.divisor) * Cfg::kColumns;
    const PagedRange range = paged_range(p.lengths[b], p.capacity, p.window_left, p.sink);
    const int pair_steps = imax(1, range.steps);
    const int begin = (int)(position - pair_start);
    const int end = whole_pairs || last - pair_start >= pair_steps ? pair_steps : (int)(last - pair_start);
    const bool whole = begin == 0 && end == pair_steps;
    if (first_pair && !whole_pairs && threadIdx.x == 0)
      p.cut[blockIdx.x] = begin == 0 ? make_int4(-1, 0, 0, 0)
                                     : make_int4(b, chunk, deal.owner(pair_start), deal.owner(pair_start + pair_steps - 1));
    const int32_t* table = p.table + b * p.table_seq;

    // The table entry of this lane's key (lane & 15) of step v; -1: none.
    auto look_up = [&](int v) -> int {
      if (v >= end) return -1;
      const int key = range.step_of(v) * kPagedStep + (lane & 15);
      return key < range.len ? table[p.page_size.div(key)] : -1;
    };
    // Starts the copies of step v; returns the set of its keys that the token sees.
    auto issue = [&](int v, int stage, int page) -> uint32_t {
      const int step = range.step_of(v), key = step * kPagedStep + (lane & 15);
      const bool ok = v < end && page >= 0 && page < p.num_pages && range.sees(key);
      const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
      const uint32_t at = ring + stage * Cfg::kStepBytes;
      if constexpr (kTma) {
        if (mask != 0) {
          const uint32_t bar = bars + 8 * stage;
          if (lane == 0) mbar_expect_tx(bar, Cfg::kStepBytes);
          __syncwarp();
          if (lane < kPagedStep && (lane & (p.box_rows - 1)) == 0) {
            const int row = key - p.page_size.div(key) * (int)p.page_size.divisor;
            const int from = page >= 0 && page < p.num_pages ? page : p.num_pages;  // out of range: the box is zeros
#pragma unroll 1
            for (int c = 0; c < D / 64; ++c) {
              tma_load_4d(at + c * kPanelBytes + lane * 128, &map_k, bar, 64 * c, kv_head, row, from);
              tma_load_4d(at + (D / 64 + c) * kPanelBytes + lane * 128, &map_v, bar, 64 * c, kv_head, row, from);
            }
          }
        }
      } else {
        if (mask != 0) {
          // 16-byte pieces 8 t of the K rows g and g + 8, pieces 8 g of the V rows 2 t, 2 t + 1, 2 t + 8 and 2 t + 9. Rows
          // that are not seen and columns at and above head_dim become zeros without being read.
          const int row = key - p.page_size.div(key) * (int)p.page_size.divisor;
          const int64_t k_own = ok ? page * p.k_page + row * p.k_row : 0, v_own = ok ? page * p.v_page + row * p.v_row : 0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const __nv_bfloat16* from = p.k + kv_head * p.k_head + 8 * t + __shfl_sync(0xffffffffu, k_own, g + 8 * i);
            const bool seen = (mask >> (g + 8 * i)) & 1u;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              const bool inside = seen && 32 * c + 8 * t < p.head_dim;
              cp_async_16(at + k_place + (i * (D / 32) + c) * 512, inside ? from + 32 * c : p.k, inside);
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int of = 2 * t + (i & 1) + 8 * (i >> 1);
            const __nv_bfloat16* from = p.v + kv_head * p.v_head + 8 * g + __shfl_sync(0xffffffffu, v_own, of);
            const bool seen = (mask >> of) & 1u;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              const bool inside = seen && 64 * c + 8 * g < p.head_dim;
              cp_async_16(at + v_place0 + (D / 16 + i * (D / 64) + c) * 512, inside ? from + 64 * c : p.v, inside);
            }
          }
        }
        cp_async_commit();
      }
      return mask;
    };

    // The first copies are on their way before the queries are read.
    uint32_t masks[kStages];
    int v_next = begin + warp, page_next = look_up(v_next);
#pragma unroll
    for (int i = 0; i < kStages; ++i) {
      const int page = page_next;
      page_next = look_up(v_next + Cfg::kWarps);
      masks[i] = issue(v_next, i, page);
      v_next += Cfg::kWarps;
    }
    uint4 q[NT][D / 32];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int column = column0 + 8 * n + g;
      const __nv_bfloat16* row = p.q + b * p.q_seq + (kv_head * p.group + column) * p.q_head + 8 * t;
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        q[n][c] = column < p.group && 32 * c + 8 * t < p.head_dim ? *reinterpret_cast<const uint4*>(row + 32 * c) : make_uint4(0, 0, 0, 0);
    }
    // Of columns 8 n + 2 t + j: m the reference maximum (the same in the eight lanes of a column), l this lane's sum of p.
    float m[NT][2], l[NT][2], o[NT][D / 64][4][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 64; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][c][j][0] = o[n][c][j][1] = o[n][c][j][2] = o[n][c][j][3] = 0.f;
    }

    int stage = 0;
    for (int v = begin + warp; v < end; v += Cfg::kWarps) {
      const uint32_t mask = masks[0], at = ring + stage * Cfg::kStepBytes;
      if constexpr (!kTma) cp_async_wait<kStages - 1>();
      if (mask != 0) {  // uniform over the warp; 0: a step whose page is missing
        if constexpr (kTma) {
          if (!mbar_wait_warp(bars + 8 * stage, (parity >> stage) & 1u, wctx, kWaitKvFull)) break;
          parity ^= 1u << stage;
          if (mask != 0xffffu) {
            // Rows that are not seen may hold anything; their probabilities are 0, but 0 x NaN is not.
            for (int i = lane; i < kPagedStep * (D / 8); i += 32) {
              const int row = i & 15, piece = i >> 4;
              if (!((mask >> row) & 1u)) st_shared_zero16(at + (D / 64 + (piece >> 3)) * kPanelBytes + row * 128 + (piece & 7) * 16);
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
        }
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          // pieces 32 c + 8 t of keys g and g + 8
          const uint32_t from = kTma ? at + (c >> 1) * kPanelBytes + (k_place ^ ((c & 1) << 6)) : at + k_place + c * 512;
          const uint4 low = ld_shared_u4(from), high = ld_shared_u4(from + (kTma ? 1024 : D / 32 * 512));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_16816(s[n], low.x, high.x, low.y, high.y, q[n][c].x, q[n][c].y);
            mma_16816(s[n], low.z, high.z, low.w, high.w, q[n][c].z, q[n][c].w);
          }
        }
        // Scores in log2 units; keys that are not seen get -inf whatever stands in their rows.
        const bool seen_low = (mask >> g) & 1u, seen_high = (mask >> (g + 8)) & 1u;
        bool grows = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            s[n][j] = seen_low ? s[n][j] * p.scale_log2 : -INFINITY;
            s[n][2 + j] = seen_high ? s[n][2 + j] * p.scale_log2 : -INFINITY;
            grows |= fmaxf(s[n][j], s[n][2 + j]) > m[n][j] + 8.f;
          }
        if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float top = fmaxf(s[n][j], s[n][2 + j]);
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              top = fmaxf(top, m[n][j]);
              const float alpha = top == -INFINITY ? 1.f : ex2_approx(m[n][j] - top);
              m[n][j] = top;
              l[n][j] *= alpha;
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  o[n][c][i][j] *= alpha;
                  o[n][c][i][2 + j] *= alpha;
                }
            }
        }
        uint32_t prob[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0], m1 = m[n][1] == -INFINITY ? 0.f : m[n][1];
          const float p00 = ex2_approx(s[n][0] - m0), p01 = ex2_approx(s[n][1] - m1);
          const float p10 = ex2_approx(s[n][2] - m0), p11 = ex2_approx(s[n][3] - m1);
          l[n][0] += p00 + p10;
          l[n][1] += p01 + p11;
          // Rounded to BF16 for the product, because the tensor core multiplies it with the BF16 V; the sum keeps 32 bits. The
          // output is then 2.3e-3 from 64 bits (norm) instead of the 1.7e-3 of its own rounding, as in the other forward kernels.
          prob[n][0] = transpose_8x8(pack_bf16x2(p00, p01));
          prob[n][1] = transpose_8x8(pack_bf16x2(p10, p11));
        }
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint4 row[4];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9; columns 64 c + 8 g to + 7
#pragma unroll
          for (int i = 0; i < 4; ++i)
            row[i] = ld_shared_u4(kTma ? at + (D / 64 + c) * kPanelBytes + ((i & 1) ? v_place1 : v_place0) + (i >> 1) * 1024
                                       : at + v_place0 + (D / 16 + i * (D / 64) + c) * 512);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w0 = word(row[0], j), w1 = word(row[1], j), w2 = word(row[2], j), w3 = word(row[3], j);
            const uint32_t a0 = __byte_perm(w0, w1, 0x5410), a1 = __byte_perm(w0, w1, 0x7632);
            const uint32_t a2 = __byte_perm(w2, w3, 0x5410), a3 = __byte_perm(w2, w3, 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816(o[n][c][j], a0, a1, a2, a3, prob[n][0], prob[n][1]);
          }
        }
      }
      // The slot is free again: the copies of the step kStages further on go there.
      __syncwarp();
      const int page = page_next;
      page_next = look_up(v_next + Cfg::kWarps);
#pragma unroll
      for (int i = 0; i + 1 < kStages; ++i) masks[i] = masks[i + 1];
      masks[kStages - 1] = issue(v_next, stage, page);
      v_next += Cfg::kWarps;
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }

    // ---- the warps' parts go over the ring (nobody reads copies any more) and are joined
    if constexpr (!kTma) cp_async_wait<0>();
    __syncthreads();
    if (kTma && *wctx.abort_flag) {  // a wait ran out: give copies in flight time to land before the block goes
      for (int i = 0; i < 50; ++i) __nanosleep(20000);
      return;
    }
    float* parts = reinterpret_cast<float*>(smem);  // (warp, column, D), then (warp, column) pairs of m and l
    float2* part_ml = reinterpret_cast<float2*>(parts + Cfg::kWarps * Cfg::kColumns * D);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float sum = l[n][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int column = warp * Cfg::kColumns + 8 * n + 2 * t + j;
        if (g == 0) part_ml[column] = make_float2(m[n][j], sum);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<float2*>(parts + column * D + 64 * c + 8 * g + 2 * i) = make_float2(o[n][c][i][j], o[n][c][i][2 + j]);
      }
    __syncthreads();
    const int columns = imin(Cfg::kColumns, p.group - column0);
    constexpr int kQuads = D / 4;
    for (int i = threadIdx.x; i < columns * kQuads; i += kThreads) {
      const int column = i / kQuads, d = 4 * (i - column * kQuads);
      if (d >= p.head_dim) continue;
      float top = -INFINITY, total = 0.f;
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w) top = fmaxf(top, part_ml[w * Cfg::kColumns + column].x);
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < Cfg::kWarps; ++w) {
        const float2 ml = part_ml[w * Cfg::kColumns + column];
        const float weight = top == -INFINITY ? 0.f : ex2_approx(ml.x - top);
        const float4 part = *reinterpret_cast<const float4*>(parts + (w * Cfg::kColumns + column) * D + d);
        total += weight * ml.y;
        sum.x += weight * part.x, sum.y += weight * part.y, sum.z += weight * part.z, sum.w += weight * part.w;
      }
      if (whole) {
        store_output(p, b, kv_head * p.group + column0 + column, d, sum, top, total);
      } else {
        const int64_t slot = (2 * (int64_t)blockIdx.x + (begin == 0)) * Cfg::kColumns + column;
        *reinterpret_cast<float4*>(p.o_part + slot * p.head_dim + d) = sum;
        if (d == 0) p.ml_part[slot] = make_float2(top, total);
      }
    }
    if constexpr (kTma) fence_proxy_async_smem();
    __syncthreads();  // the ring is free for the copies of the next pair
    position = pair_start = whole_pairs ? position + 1 : pair_start + end;
    if (++b == p.batch) {
      b = 0;
      ++chunk;
    }
  }
}

// Joins the parts of the pairs that were cut: out = sum w o / sum w l, w = exp2(m - max m). One block per (range, query head
// of a chunk); the one of the pair's second range does the work. Its threads form groups of one thread per four columns,
// group i takes the parts i, i + groups, ... in this order, and the groups are joined in order at the end, so the result
// does not depend on the schedule. The blocks start under the last ranges and wait for them. `columns` = 8 * NT.
constexpr int kJoinThreads = 256;
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedParams p, int columns) {
  __shared__ float4 group_o[kJoinThreads];
  __shared__ float2 group_ml[kJoinThreads];
  const int quads = p.head_dim / 4, groups = kJoinThreads / quads;
  const int group = threadIdx.x / quads, quad = threadIdx.x - group * quads, column = blockIdx.y, range = blockIdx.x + 1;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 cut = p.cut[range];  // sequence, chunk, first range, last range
  if (cut.x < 0 || cut.z != range - 1) return;
  const int kv_head = p.chunks.div(cut.y), column0 = (cut.y - kv_head * (int)p.chunks.divisor) * columns;
  if (column0 + column >= p.group) return;
  const int parts = cut.w - cut.z + 1;
  auto slot_of = [&](int i) { return (2 * (int64_t)(cut.z + i) + (i == 0)) * columns + column; };
  float top = -INFINITY, total = 0.f;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  if (group < groups) {
#pragma unroll 4
    for (int i = group; i < parts; i += groups) {
      const float2 own = p.ml_part[slot_of(i)];
      const float4 o = reinterpret_cast<const float4*>(p.o_part + slot_of(i) * p.head_dim)[quad];
      const float higher = fmaxf(top, own.x);
      const float keep = higher == -INFINITY ? 0.f : ex2_approx(top - higher), take = higher == -INFINITY ? 0.f : ex2_approx(own.x - higher);
      top = higher;
      total = total * keep + own.y * take;
      sum.x = sum.x * keep + o.x * take, sum.y = sum.y * keep + o.y * take;
      sum.z = sum.z * keep + o.z * take, sum.w = sum.w * keep + o.w * take;
    }
  }
  group_o[threadIdx.x] = sum;
  group_ml[threadIdx.x] = make_float2(top, total);
  __syncthreads();
  if (threadIdx.x >= quads) return;
  top = -INFINITY;
  for (int i = 0; i < groups; ++i) top = fmaxf(top, group_ml[i * quads].x);
  total = 0.f;
  sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; i < groups; ++i) {
    const float2 own = group_ml[i * quads];
    const float4 o = group_o[i * quads + quad];
    const float weight = top == -INFINITY ? 0.f : ex2_approx(own.x - top);
    total += weight * own.y;
    sum.x += weight * o.x, sum.y += weight * o.y, sum.z += weight * o.z, sum.w += weight * o.w;
  }
  store_output(p, cut.x, kv_head * p.group + column0 + column, 4 * quad, sum, top, total);
}

// ---------------------------------------------------------------------------------------------- host side
constexpr int kPagedSms = 148;  // the plan is a function of the shapes alone, like that of the split forward pass

// Query heads per block, in groups of 8: as many as the accumulators leave registers for, so that K and V are read once.
static int paged_tiles(int head_dim, int group) {
  const int wanted = group <= 8 ? 1 : group <= 16 ? 2 : 4;
  const int limit = head_dim <= 128 ? 4 : head_dim <= 256 ? 2 : 1;
  return wanted < limit ? wanted : limit;
}

struct PagedShape {
  int tiles, chunks, ranges;
  size_t o_bytes, ml_bytes, cut_bytes;
  size_t total() const { return o_bytes + ml_bytes + cut_bytes; }
};
// Pairs of at most so many steps are not cut: up to there the plan and the join kernel take longer than the steps of one
// block. A pair more than the block slots takes a whole round of its own, so longer pairs stay whole only in one round of 100
// pairs or more, and up to head_dim 128 also in several whose last one leaves a quarter of all slots empty at most. Times in
// us whole / cut, pages of 16 in a cache larger than L2, all sequences at the limit or of random lengths up to it:
//   head_dim 128, 8 key heads x 4: 8 pairs of 512 keys 8.9 / 8.8, of 768 10.9 / 6.8; 128 pairs of 1280 keys 17.1 / 18.0 and
//   15.8 / 18.6, of 1536 19.0 / 19.4 and 18.0 / 17.1; 240 of 1536 23.8 / 27.3 and 21.8 / 22.5; 304 of 1024 32.0 / 25.4 and
//   18.2 / 23.7, of 512 20.3 / 19.1 and 15.7 / 19.6; 448 of 1280 39.1 / 38.6 and 35.3 / 32.4; 592 of 1280 40.0 / 41.7 and
//   37.0 / 35.8. head_dim 64: 128 of 1280 13.3 / 14.9 and 11.9 / 14.9.
//   head_dim 256, 4 x 4: 8 pairs of 256 keys 10.6 / 10.8, of 384 12.9 / 8.2; 128 of 512 17.3 / 17.9 and 17.2 / 18.2, of 768
//   23.0 / 20.4 and 23.1 / 19.4; 304 of 512 38.2 / 27.9 and 29.9 / 28.2, of 256 23.1 / 19.5 and 23.0 / 22.8.
//   head_dim 512, 2 x 4: 16 of 256 18.0 / 16.4 and 14.4 / 21.9; 128 of 512 30.1 / 33.7 and 30.7 / 34.8.
static int uncut_steps(int head_dim, int64_t pairs, int slots) {
  const int64_t rounds = (pairs + slots - 1) / slots;
  const bool one_round = pairs >= 100 && pairs <= slots;
  if (head_dim > 128) return one_round ? 32 : 16;
  if (one_round) return 3 * pairs >= 2 * slots ? 96 : 80;
  return rounds > 1 && 4 * pairs >= 3 * rounds * slots ? 80 : 32;
}
static PagedShape paged_shape(const b200fa_paged_args& a) {
  PagedShape s;
  const int group = a.heads_q / a.heads_kv;
  s.tiles = paged_tiles(a.head_dim, group);
  s.chunks = (group + 8 * s.tiles - 1) / (8 * s.tiles);
  const int64_t most_steps = ((int64_t)a.max_pages * a.page_size + kPagedStep - 1) / kPagedStep;
  const int slots = (a.head_dim <= 256 ? 2 : 1) * kPagedSms;  // blocks that run at the same time
  const int64_t most_work = most_steps * a.batch * a.heads_kv * s.chunks, wanted = (most_work + kMinSteps - 1) / kMinSteps;
  s.ranges = wanted < slots ? (int)wanted : slots;
  s.o_bytes = s.ml_bytes = s.cut_bytes = 0;
  const int64_t pairs = (int64_t)a.batch * a.heads_kv * s.chunks;
  // steps of a pair, at most: a window bounds them whatever the table holds
  int64_t pair_steps = most_steps;
  if (a.window_left >= 0) {
    const int64_t seen = ((int64_t)a.window_left + kPagedStep) / kPagedStep + 1 + ((int64_t)a.sink_size + kPagedStep - 1) / kPagedStep;
    pair_steps = seen < most_steps ? seen : most_steps;
  }
  if (pair_steps <= uncut_steps(a.head_dim, pairs, slots)) {
    s.ranges = pairs < slots ? (int)pairs : slots;
    return s;
  }
  const size_t part_rows = 2 * (size_t)s.ranges * 8 * s.tiles;
  s.o_bytes = part_rows * a.head_dim * 4;
  s.ml_bytes = part_rows * 8;
  s.cut_bytes = (size_t)s.ranges * 16;
  return s;
}

template <int D, int NT, bool kTma>
static int launch_paged(const CUtensorMap (&maps)[2], const PagedParams& p, cudaStream_t stream) {
  using Cfg = PagedConfig<D, NT>;
  static bool set[64] = {false};
  const int status = set_dynamic_smem_once(reinterpret_cast<const void*>(&paged_decode_kernel<D, NT, kTma>), Cfg::kSmemBytes, set);
  if (status != B200FA_OK) return status;
  paged_decode_kernel<D, NT, kTma><<<p.ranges, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(maps[0], maps[1], p);
  return B200FA_OK;
}

template <int D, int NT>
static int launch_paged(const CUtensorMap (&maps)[2], const PagedParams& p, cudaStream_t stream) {
  return p.box_rows ? launch_paged<D, NT, true>(maps, p, stream) : launch_paged<D, NT, false>(maps, p, stream);
}

template <int D>
static int launch_paged(int tiles, const CUtensorMap (&maps)[2], const PagedParams& p, cudaStream_t stream) {
  if (tiles == 1) return launch_paged<D, 1>(maps, p, stream);
  if constexpr (D <= 256) {
    if (tiles == 2) return launch_paged<D, 2>(maps, p, stream);
  }
  if constexpr (D <= 128) {
    if (tiles == 4) return launch_paged<D, 4>(maps, p, stream);
  }
  set_error("no paged attention kernel for %d query tiles at head_dim %d", tiles, D);
  return B200FA_ERR_UNSUPPORTED;
}

}  // namespace b200fa

using namespace b200fa;

extern "C" {

static int validate_paged(const b200fa_paged_args* a) {
  B200FA_REQUIRE(a != nullptr, "null arguments");
  B200FA_REQUIRE(a->batch >= 0 && a->num_pages >= 0 && a->max_pages >= 0, "negative sizes");
  B200FA_REQUIRE(a->page_size > 0, "page_size must be positive");
  B200FA_REQUIRE((int64_t)a->max_pages * a->page_size < 0x7fffff00ll, "the block table covers more than 2^31 - 256 keys");
  B200FA_REQUIRE(a->heads_q > 0 && a->heads_kv > 0 && a->heads_q % a->heads_kv == 0,
                 "the query head count must be a positive multiple of the key head count");
  B200FA_REQUIRE(b200fa_supports_head_dim(a->head_dim, 0), "head_dim %d is not supported by paged attention", a->head_dim);
  B200FA_REQUIRE(a->window_left >= -1, "window bounds must each be -1 or non-negative");
  B200FA_REQUIRE(a->sink_size >= 0, "sink_size must not be negative");
  B200FA_REQUIRE(a->q_stride[0] % 8 == 0 && a->q_stride[1] % 8 == 0 && a->out_stride[0] % 8 == 0 && a->out_stride[1] % 8 == 0,
                 "tensor strides must be multiples of 8 elements");
  for (int i = 0; i < 3; ++i)
    B200FA_REQUIRE(a->k_stride[i] % 8 == 0 && a->v_stride[i] % 8 == 0, "tensor strides must be multiples of 8 elements");
  if (a->batch == 0) return B200FA_OK;
  B200FA_REQUIRE(a->q && a->out && a->softmax_lse && a->cache_seqlens, "null tensor pointer");
  B200FA_REQUIRE(a->max_pages == 0 || a->block_table, "null tensor pointer");
  B200FA_REQUIRE(a->num_pages == 0 || (a->k_cache && a->v_cache), "null tensor pointer");
  const void* aligned16[] = {a->q, a->k_cache, a->v_cache, a->out};
  for (const void* pointer : aligned16)
    B200FA_REQUIRE(reinterpret_cast<uintptr_t>(pointer) % 16 == 0, "tensor pointers must be 16-byte aligned");
  return B200FA_OK;
}

size_t b200fa_paged_decode_workspace_bytes(const b200fa_paged_args* a) {
  if (a->batch <= 0 || a->heads_kv <= 0 || a->heads_q < a->heads_kv || a->page_size <= 0 || a->max_pages < 0) return 0;
  return paged_shape(*a).total();
}

int b200fa_paged_decode(const b200fa_paged_args* a, void* stream) {
  int status = validate_paged(a);
  if (status != B200FA_OK || a->batch == 0) return status;
  const PagedShape shape = paged_shape(*a);
  B200FA_REQUIRE(shape.total() == 0 || (a->workspace && a->workspace_bytes >= shape.total()), "paged attention workspace is too small: need %zu bytes",
                 shape.total());
  B200FA_REQUIRE(reinterpret_cast<uintptr_t>(a->workspace) % 16 == 0, "paged attention workspace must be 16-byte aligned");
  PagedParams p;
  p.batch = a->batch, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.group = a->heads_q / a->heads_kv;
  p.head_dim = a->head_dim, p.num_pages = a->num_pages, p.capacity = a->max_pages * a->page_size;
  p.window_left = a->window_left, p.sink = a->sink_size;
  p.page_size = FastDiv::make((uint32_t)a->page_size), p.chunks = FastDiv::make((uint32_t)shape.chunks);
  p.columns = a->heads_kv * shape.chunks, p.ranges = shape.ranges;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.k = static_cast<const __nv_bfloat16*>(a->k_cache);
  p.v = static_cast<const __nv_bfloat16*>(a->v_cache), p.out = static_cast<__nv_bfloat16*>(a->out);
  p.table = a->block_table, p.lengths = a->cache_seqlens, p.lse = a->softmax_lse;
  uint8_t* workspace = static_cast<uint8_t*>(a->workspace);
  p.o_part = reinterpret_cast<float*>(workspace);
  p.ml_part = reinterpret_cast<float2*>(workspace + shape.o_bytes);
  p.cut = shape.total() ? reinterpret_cast<int4*>(workspace + shape.o_bytes + shape.ml_bytes) : nullptr;
  p.q_seq = a->q_stride[0], p.q_head = a->q_stride[1], p.out_seq = a->out_stride[0], p.out_head = a->out_stride[1];
  p.k_page = a->k_stride[0], p.k_row = a->k_stride[1], p.k_head = a->k_stride[2];
  p.v_page = a->v_stride[0], p.v_row = a->v_stride[1], p.v_head = a->v_stride[2];
  p.table_seq = a->table_stride;
  p.status = device_status_word();
  if (!p.status) return B200FA_ERR_CUDA;
  // Boxes must not reach over the end of a page: 16 or 8 keys where the page size is a multiple of that.
  CUtensorMap maps[2] = {};
  p.box_rows = a->num_pages == 0 ? 0 : a->page_size % 16 == 0 ? 16 : a->page_size % 8 == 0 ? 8 : 0;
  if (p.box_rows) {
    for (int i = 0; i < 2; ++i) {
      const int64_t* stride = i ? a->v_stride : a->k_stride;
      status = encode_tensor_map(&maps[i], i ? a->v_cache : a->k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a->head_dim,
                                 a->heads_kv, a->page_size, a->num_pages, stride[2], stride[1], stride[0], 64, p.box_rows);
      if (status != B200FA_OK) return status;
    }
  }
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  status = a->head_dim <= 64    ? launch_paged<64>(shape.tiles, maps, p, s)
           : a->head_dim <= 128 ? launch_paged<128>(shape.tiles, maps, p, s)
           : a->head_dim <= 256 ? launch_paged<256>(shape.tiles, maps, p, s)
                                : launch_paged<512>(shape.tiles, maps, p, s);
  if (status != B200FA_OK) return status;
  B200FA_CUDA_CHECK(cudaGetLastError());
  if (p.cut && shape.ranges > 1) {
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    const int columns = 8 * shape.tiles;
    config.gridDim = dim3((unsigned)shape.ranges - 1, (unsigned)(p.group < columns ? p.group : columns));
    config.blockDim = dim3(kJoinThreads);
    config.stream = s;
    config.attrs = &attribute;
    config.numAttrs = 1;
    B200FA_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_join_kernel, p, columns));
  }
  return B200FA_OK;
}

// Host twin of the key selection: the keys that the token of a sequence of `length` keys sees, in the order the kernel
// walks them; returns their number (at most max_keys are written).
int b200fa_paged_keys_host(int32_t length, int32_t capacity, int32_t window_left, int32_t sink_size, int32_t* keys,
                           int32_t max_keys) {
  const PagedRange r = paged_range(length, capacity, window_left, sink_size);
  int n = 0;
  for (int v = 0; v < r.steps; ++v)
    for (int key = r.step_of(v) * kPagedStep; key < (r.step_of(v) + 1) * kPagedStep; ++key)
      if (r.sees(key)) {
        if (n < max_keys) keys[n] = key;
        ++n;
      }
  return n;
}

}  // extern "C"
