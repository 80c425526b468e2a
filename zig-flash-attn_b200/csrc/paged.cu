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
//     16-byte pieces: a thread copies its own pieces with cp.async into its own places of a ring in shared memory and
//     reads them back itself. No transposition, no ldmatrix, no bank conflicts, no synchronisation.
//   - The maximum of a column moves only when a score exceeds it by more than 8 (in log2 units), so a step costs one vote
//     instead of a reduction over the lanes. Sums are kept per lane and added up at the end.
// The steps of all sequences are dealt out in shares of equal size, so that long and short sequences keep every SM busy;
// each block works out from the lengths which share it has. A sequence with one share is finished in place, the shares of
// the others are joined by a second kernel.
#include "common.h"
#include "fwd_common.cuh"
#include "paged_index.h"
#include "ptx.cuh"

namespace b200fa {

struct PagedParams {
  int batch, heads_q, heads_kv, group, head_dim, num_pages, capacity, window_left, sink;
  FastDiv page_size, chunks;  // chunks of 8 * NT query heads per key head
  int min_steps, target;      // shares: at least so many steps, about so many per (key head, chunk)
  float scale_log2;
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const int32_t* table;
  const int32_t* lengths;
  __nv_bfloat16* out;
  float* lse;
  float* o_part;    // (slots, heads_q, head_dim): sum of p V relative to the share's maximum
  float2* ml_part;  // (slots, heads_q): maximum (log2 units) and sum of p
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

// ---------------------------------------------------------------------------------------------- dealing out the steps
// All blocks (of both kernels) derive the same plan from the lengths: with T steps in all, a share has
// max(min_steps, ceil(T / target)) steps, so there are at most target + batch shares.
struct PagedPlan {
  int64_t share_steps;
  __device__ __forceinline__ int shares(int steps) const {
    return imax(1, (int)((steps + share_steps - 1) / share_steps));
  }
};

__device__ __forceinline__ PagedRange range_of(const PagedParams& p, int b) {
  return paged_range(p.lengths[b], p.capacity, p.window_left, p.sink);
}

template <int kThreads>
__device__ __forceinline__ PagedPlan make_plan(const PagedParams& p, int64_t* warp_sums) {
  int64_t mine = 0;
  for (int b = threadIdx.x; b < p.batch; b += kThreads) mine += range_of(p, b).steps;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = mine;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) total += warp_sums[w];
  const int64_t even = (total + p.target - 1) / p.target;
  return {even > p.min_steps ? even : p.min_steps};
}

// Calls visit(b, first slot, shares) in the threads that own a sequence b, sequences in order, until `done` says so for
// the whole block: first slot = shares of the sequences in front of b.
template <int kThreads, typename Visit, typename Done>
__device__ __forceinline__ void walk_plan(const PagedParams& p, const PagedPlan& plan, int* warp_sums, Visit visit, Done done) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + threadIdx.x;
    const int mine = b < p.batch ? plan.shares(range_of(p, b).steps) : 0;
    int inclusive = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inclusive, d);
      if (lane >= d) inclusive += other;
    }
    if (lane == 31) warp_sums[warp] = inclusive;
    __syncthreads();
    int total = 0, front = before;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) front += warp_sums[w];
      total += warp_sums[w];
    }
    if (b < p.batch) visit(b, front + inclusive - mine, mine);
    before += total;
    __syncthreads();  // what visit() wrote is visible; the sums may be overwritten
    if (done(base + kThreads)) return;
  }
}

// ---------------------------------------------------------------------------------------------- the shares
template <int D, int NT>
struct PagedConfig {
  static constexpr int kWarps = D <= 128 ? 4 : 2;
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kStepBytes = 2 * kPagedStep * D * 2;             // K and V of a step
  static constexpr int kStages = D == 64 ? 6 : 3;                       // steps of a warp in flight
  static constexpr int kRingBytes = kWarps * kStages * kStepBytes;      // 96 KiB: two blocks per SM (head_dim 512: one)
  static constexpr int kColumns = 8 * NT;
  static constexpr int kMergeBytes = kWarps * kColumns * (D * 4 + 8);   // over the ring, at the end
  static constexpr int kSmemBytes = kRingBytes > kMergeBytes ? kRingBytes : kMergeBytes;
};

// kAligned: page_size is a multiple of 16, so the keys of a step lie in one page; otherwise each lane looks up a key.
template <int D, int NT, bool kAligned>
__global__ void __launch_bounds__(PagedConfig<D, NT>::kThreads) paged_decode_kernel(const __grid_constant__ PagedParams p) {
  using Cfg = PagedConfig<D, NT>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int64_t plan_sums[Cfg::kWarps];
  __shared__ int scan_sums[Cfg::kWarps], found[3];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int slot = blockIdx.x, kv_head = p.chunks.div(blockIdx.y);
  const int column0 = (blockIdx.y - kv_head * p.chunks.divisor) * Cfg::kColumns;

  if (threadIdx.x == 0) found[0] = -1;
  const PagedPlan plan = make_plan<Cfg::kThreads>(p, plan_sums);
  walk_plan<Cfg::kThreads>(
      p, plan, scan_sums,
      [&](int b, int first, int shares) {
        if (slot >= first && slot < first + shares) {
          found[0] = b;
          found[1] = slot - first;
          found[2] = shares;
        }
      },
      [&](int) { return found[0] >= 0; });
  const int b = found[0];
  if (b < 0) return;
  const int share = found[1], shares = found[2];
  const PagedRange range = range_of(p, b);
  const int begin = (int)((int64_t)range.steps * share / shares), end = (int)((int64_t)range.steps * (share + 1) / shares);
  const int32_t* table = p.table + b * p.table_seq;
  const __nv_bfloat16* k_head = p.k + kv_head * p.k_head;
  const __nv_bfloat16* v_head = p.v + kv_head * p.v_head;
  const uint32_t ring = smem_u32(smem) + warp * kStages * Cfg::kStepBytes + lane * 16;

  // The table entry that the step with number v needs (of this lane's key when the pages are not aligned); -1: none.
  auto look_up = [&](int v) -> int {
    if (v >= end) return -1;
    const int key = range.step_of(v) * kPagedStep + (kAligned ? 0 : lane & 15);
    return key < range.len ? table[p.page_size.div(key)] : -1;
  };
  // Starts the copies of step v; returns the set of its keys that the token sees.
  auto issue = [&](int v, int stage, int page) -> uint32_t {
    const int step = range.step_of(v), key = step * kPagedStep + (lane & 15);
    const bool ok = v < end && page >= 0 && page < p.num_pages && range.sees(key);
    const uint32_t mask = __ballot_sync(0xffffffffu, ok) & 0xffffu;
    if (mask != 0) {
      const uint32_t at = ring + stage * Cfg::kStepBytes;
      int64_t k_own, v_own = 0;  // aligned: of the step's first row, else of this lane's key
      {
        const int first = kAligned ? step * kPagedStep : key;
        const int row = first - p.page_size.div(first) * (int)p.page_size.divisor;
        const bool have = kAligned || ok;
        k_own = have ? page * p.k_page + row * p.k_row : 0;
        v_own = have ? page * p.v_page + row * p.v_row : 0;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key_of = g + 8 * i;
        const __nv_bfloat16* row = k_head + 8 * t + (kAligned ? k_own + key_of * p.k_row : __shfl_sync(0xffffffffu, k_own, key_of));
        const bool seen = (mask >> key_of) & 1u;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const bool inside = seen && 32 * c + 8 * t < p.head_dim;
          cp_async_16(at + (i * (D / 32) + c) * 512, inside ? row + 32 * c : k_head, inside);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key_of = 2 * t + (i & 1) + 8 * (i >> 1);
        const __nv_bfloat16* row = v_head + 8 * g + (kAligned ? v_own + key_of * p.v_row : __shfl_sync(0xffffffffu, v_own, key_of));
        const bool seen = (mask >> key_of) & 1u;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const bool inside = seen && 64 * c + 8 * g < p.head_dim;
          cp_async_16(at + (D / 16 + i * (D / 64) + c) * 512, inside ? row + 64 * c : v_head, inside);
        }
      }
    }
    cp_async_commit();
    return mask;
  };

  // The first copies are on their way before the queries are read.
  uint32_t masks[kStages];
  int v_next = begin + warp, page_next = look_up(v_next);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
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
    cp_async_wait<kStages - 2>();
    {
      const int page = page_next;
      page_next = look_up(v_next + Cfg::kWarps);
      masks[kStages - 1] = issue(v_next, stage == 0 ? kStages - 1 : stage - 1, page);
      v_next += Cfg::kWarps;
    }
    const uint32_t mask = masks[0];
#pragma unroll
    for (int i = 0; i + 1 < kStages; ++i) masks[i] = masks[i + 1];
    const uint32_t at = ring + stage * Cfg::kStepBytes;
    stage = stage + 1 == kStages ? 0 : stage + 1;
    if (mask == 0) continue;  // uniform over the warp: a step whose page is missing

    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const uint4 low = ld_shared_u4(at + c * 512), high = ld_shared_u4(at + (D / 32 + c) * 512);  // keys g and g + 8
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
      prob[n][0] = transpose_8x8(pack_bf16x2(p00, p01));  // rounded to BF16 for the product, not for the sum
      prob[n][1] = transpose_8x8(pack_bf16x2(p10, p11));
    }
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      uint4 row[4];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9; columns 64 c + 8 g to + 7
#pragma unroll
      for (int i = 0; i < 4; ++i) row[i] = ld_shared_u4(at + (D / 16 + i * (D / 64) + c) * 512);
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

  // ---- the warps' parts go over the ring (nobody reads copies any more) and are joined
  cp_async_wait<0>();
  __syncthreads();
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
  for (int i = threadIdx.x; i < columns * kQuads; i += Cfg::kThreads) {
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
    const int head = kv_head * p.group + column0 + column;
    if (shares == 1) {
      const float inv = total > 0.f ? 1.f / total : 0.f;
      *reinterpret_cast<uint2*>(p.out + b * p.out_seq + head * p.out_head + d) =
          make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
      if (d == 0) p.lse[(int64_t)b * p.heads_q + head] = total > 0.f ? (top + log2f(total)) * 0.69314718055994531f : -INFINITY;
    } else {
      const int64_t at = (int64_t)slot * p.heads_q + head;
      *reinterpret_cast<float4*>(p.o_part + at * p.head_dim + d) = sum;
      if (d == 0) p.ml_part[at] = make_float2(top, total);
    }
  }
}

// Joins the shares of a sequence that has more than one: out = sum w o / sum w l, w = exp2(m - max m), in the order of the
// shares. One block per (sequence, key head); it starts while the last shares are still being computed and waits for them
// behind its own walk over the lengths.
constexpr int kJoinThreads = 128;
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedParams p) {
  __shared__ int64_t plan_sums[kJoinThreads / 32];
  __shared__ int scan_sums[kJoinThreads / 32], found[2];
  const int b = blockIdx.x;
  const PagedPlan plan = make_plan<kJoinThreads>(p, plan_sums);
  walk_plan<kJoinThreads>(
      p, plan, scan_sums,
      [&](int seq, int first, int shares) {
        if (seq == b) {
          found[0] = first;
          found[1] = shares;
        }
      },
      [&](int walked) { return walked > b; });
  const int first = found[0], shares = found[1];
  if (shares == 1) return;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int quads = p.head_dim / 4;
  for (int i = threadIdx.x; i < p.group * quads; i += kJoinThreads) {
    const int column = i / quads, d = 4 * (i - column * quads), head = blockIdx.y * p.group + column;
    const float2* ml = p.ml_part + (int64_t)first * p.heads_q + head;
    const float* part = p.o_part + ((int64_t)first * p.heads_q + head) * p.head_dim + d;
    float top = -INFINITY, total = 0.f;
    for (int s = 0; s < shares; ++s) top = fmaxf(top, ml[(int64_t)s * p.heads_q].x);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    if (top != -INFINITY) {
#pragma unroll 4
      for (int s = 0; s < shares; ++s) {
        const float2 own = ml[(int64_t)s * p.heads_q];
        const float4 o = *reinterpret_cast<const float4*>(part + (int64_t)s * p.heads_q * p.head_dim);
        const float weight = ex2_approx(own.x - top);
        total += weight * own.y;
        sum.x += weight * o.x, sum.y += weight * o.y, sum.z += weight * o.z, sum.w += weight * o.w;
      }
    }
    const float inv = total > 0.f ? 1.f / total : 0.f;
    *reinterpret_cast<uint2*>(p.out + b * p.out_seq + head * p.out_head + d) =
        make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
    if (d == 0) p.lse[(int64_t)b * p.heads_q + head] = total > 0.f ? (top + log2f(total)) * 0.69314718055994531f : -INFINITY;
  }
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
  int tiles, chunks, min_steps, target;
  int64_t slots;  // shares of all sequences, at most
};
static PagedShape paged_shape(const b200fa_paged_args& a) {
  PagedShape s;
  const int group = a.heads_q / a.heads_kv;
  s.tiles = paged_tiles(a.head_dim, group);
  s.chunks = (group + 8 * s.tiles - 1) / (8 * s.tiles);
  const int64_t columns = (int64_t)a.heads_kv * s.chunks;
  s.min_steps = 8;
  s.target = (int)imax(1, (int)((4 * kPagedSms + columns - 1) / columns));
  const int64_t most_steps = ((int64_t)a.max_pages * a.page_size + kPagedStep - 1) / kPagedStep + 1;
  const int64_t each = (most_steps + s.min_steps - 1) / s.min_steps;  // shares of one sequence, at most
  s.slots = each <= 1 ? a.batch : (each * a.batch < (int64_t)s.target + a.batch ? each * a.batch : (int64_t)s.target + a.batch);
  return s;
}

template <int D, int NT, bool kAligned>
static int launch_paged(const PagedParams& p, dim3 grid, cudaStream_t stream) {
  using Cfg = PagedConfig<D, NT>;
  static bool set[64] = {false};
  const int status = set_dynamic_smem_once(reinterpret_cast<const void*>(&paged_decode_kernel<D, NT, kAligned>), Cfg::kSmemBytes, set);
  if (status != B200FA_OK) return status;
  paged_decode_kernel<D, NT, kAligned><<<grid, Cfg::kThreads, Cfg::kSmemBytes, stream>>>(p);
  return B200FA_OK;
}

template <int D, int NT>
static int launch_paged(const PagedParams& p, dim3 grid, cudaStream_t stream) {
  return p.page_size.divisor % kPagedStep == 0 ? launch_paged<D, NT, true>(p, grid, stream)
                                               : launch_paged<D, NT, false>(p, grid, stream);
}

template <int D>
static int launch_paged(int tiles, const PagedParams& p, dim3 grid, cudaStream_t stream) {
  if (tiles == 1) return launch_paged<D, 1>(p, grid, stream);
  if constexpr (D <= 256) {
    if (tiles == 2) return launch_paged<D, 2>(p, grid, stream);
  }
  if constexpr (D <= 128) {
    if (tiles == 4) return launch_paged<D, 4>(p, grid, stream);
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
  if (a->batch <= 0 || a->heads_kv <= 0 || a->heads_q <= 0) return 0;
  const PagedShape s = paged_shape(*a);
  return s.slots <= a->batch ? 0 : (size_t)s.slots * a->heads_q * (a->head_dim * 4 + 8);
}

int b200fa_paged_decode(const b200fa_paged_args* a, void* stream) {
  int status = validate_paged(a);
  if (status != B200FA_OK || a->batch == 0) return status;
  const PagedShape shape = paged_shape(*a);
  const size_t needed = b200fa_paged_decode_workspace_bytes(a);
  B200FA_REQUIRE(a->workspace_bytes >= needed && (needed == 0 || a->workspace), "paged attention workspace is too small: need %zu bytes", needed);
  B200FA_REQUIRE(reinterpret_cast<uintptr_t>(a->workspace) % 16 == 0, "paged attention workspace must be 16-byte aligned");
  const int64_t columns = (int64_t)a->heads_kv * shape.chunks;
  B200FA_REQUIRE(columns < 65536 && a->heads_kv < 65536, "too many heads for one call");
  PagedParams p;
  p.batch = a->batch, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.group = a->heads_q / a->heads_kv;
  p.head_dim = a->head_dim, p.num_pages = a->num_pages, p.capacity = a->max_pages * a->page_size;
  p.window_left = a->window_left, p.sink = a->sink_size;
  p.page_size = FastDiv::make((uint32_t)a->page_size), p.chunks = FastDiv::make((uint32_t)shape.chunks);
  p.min_steps = shape.min_steps, p.target = shape.target;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.k = static_cast<const __nv_bfloat16*>(a->k_cache);
  p.v = static_cast<const __nv_bfloat16*>(a->v_cache), p.out = static_cast<__nv_bfloat16*>(a->out);
  p.table = a->block_table, p.lengths = a->cache_seqlens, p.lse = a->softmax_lse;
  p.o_part = static_cast<float*>(a->workspace);
  p.ml_part = reinterpret_cast<float2*>(p.o_part + (size_t)shape.slots * a->heads_q * a->head_dim);
  p.q_seq = a->q_stride[0], p.q_head = a->q_stride[1], p.out_seq = a->out_stride[0], p.out_head = a->out_stride[1];
  p.k_page = a->k_stride[0], p.k_row = a->k_stride[1], p.k_head = a->k_stride[2];
  p.v_page = a->v_stride[0], p.v_row = a->v_stride[1], p.v_head = a->v_stride[2];
  p.table_seq = a->table_stride;
  const dim3 grid((unsigned)shape.slots, (unsigned)columns);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  status = a->head_dim <= 64    ? launch_paged<64>(shape.tiles, p, grid, s)
           : a->head_dim <= 128 ? launch_paged<128>(shape.tiles, p, grid, s)
           : a->head_dim <= 256 ? launch_paged<256>(shape.tiles, p, grid, s)
                                : launch_paged<512>(shape.tiles, p, grid, s);
  if (status != B200FA_OK) return status;
  B200FA_CUDA_CHECK(cudaGetLastError());
  if (needed > 0) {
    cudaLaunchAttribute attribute;
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)a->batch, (unsigned)a->heads_kv);
    config.blockDim = dim3(kJoinThreads);
    config.stream = s;
    config.attrs = &attribute;
    config.numAttrs = 1;
    B200FA_CUDA_CHECK(cudaLaunchKernelEx(&config, paged_join_kernel, p));
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
