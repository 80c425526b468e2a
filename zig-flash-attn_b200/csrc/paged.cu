// Attention of one new token per sequence over a paged key-value cache, for sm_100a.
//
//   out[b, h] = sum_j p_j V[j],  p_j = exp(scale q[b, h] . K[j] - lse[b, h])  over the keys j that the token sees
//
// (b200fa_paged_decode; the visible keys are those of PagedRange in paged_index.h.) The operator has no counterpart in
// the reference. One block per (sequence, query head): every warp takes every fourth key, keeps a running maximum and sum
// of its own, and the four are joined at the end.
#include "common.h"
#include "paged_index.h"
#include "ptx.cuh"

namespace b200fa {

struct PagedParams {
  int batch, heads_q, heads_kv, head_dim, num_pages, page_size, capacity, window_left, sink;
  float scale_log2;
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  const int32_t* table;
  const int32_t* lengths;
  __nv_bfloat16* out;
  float* lse;
  int64_t q_seq, q_head, k_page, k_row, k_head, v_page, v_row, v_head, out_seq, out_head, table_seq, lse_seq;
};

__global__ void __launch_bounds__(128) paged_decode_kernel(const __grid_constant__ PagedParams p) {
  constexpr int kPerLane = 16;  // columns per lane at head_dim 512
  __shared__ float part[4][512 + 2];
  const int b = blockIdx.x, head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_head = head / (p.heads_q / p.heads_kv);
  const PagedRange range = paged_range(p.lengths[b], p.capacity, p.window_left, p.sink);
  const int32_t* table = p.table + b * p.table_seq;
  float q[kPerLane], o[kPerLane], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + 32 * i;
    q[i] = d < p.head_dim ? __bfloat162float(p.q[b * p.q_seq + head * p.q_head + d]) * p.scale_log2 : 0.f;
    o[i] = 0.f;
  }
  for (int v = warp; v < range.steps * kPagedStep; v += 4) {
    const int key = range.step_of(v / kPagedStep) * kPagedStep + v % kPagedStep;
    if (!range.sees(key)) continue;
    const int page = table[key / p.page_size];
    if (page < 0 || page >= p.num_pages) continue;
    const __nv_bfloat16* k_row = p.k + page * p.k_page + (key % p.page_size) * p.k_row + kv_head * p.k_head;
    const __nv_bfloat16* v_row = p.v + page * p.v_page + (key % p.page_size) * p.v_row + kv_head * p.v_head;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < p.head_dim) s += q[i] * __bfloat162float(k_row[lane + 32 * i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float m_new = fmaxf(m, s), alpha = ex2_approx(m - m_new), e = ex2_approx(s - m_new);
    m = m_new;
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (lane + 32 * i < p.head_dim) o[i] = o[i] * alpha + e * __bfloat162float(v_row[lane + 32 * i]);
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) part[warp][lane + 32 * i] = o[i];
  if (lane == 0) {
    part[warp][512] = m;
    part[warp][513] = l;
  }
  __syncthreads();
  float top = -INFINITY, total = 0.f, w[4];
  for (int i = 0; i < 4; ++i) top = fmaxf(top, part[i][512]);
  for (int i = 0; i < 4; ++i) {
    w[i] = top == -INFINITY ? 0.f : ex2_approx(part[i][512] - top);
    total += w[i] * part[i][513];
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  for (int d = threadIdx.x; d < p.head_dim; d += 128) {
    float sum = 0.f;
    for (int i = 0; i < 4; ++i) sum += w[i] * part[i][d];
    p.out[b * p.out_seq + head * p.out_head + d] = __float2bfloat16(sum * inv);
  }
  if (threadIdx.x == 0) p.lse[b * p.lse_seq + head] = total > 0.f ? (top + log2f(total)) * 0.69314718055994531f : -INFINITY;
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

size_t b200fa_paged_decode_workspace_bytes(const b200fa_paged_args*) { return 0; }

int b200fa_paged_decode(const b200fa_paged_args* a, void* stream) {
  const int status = validate_paged(a);
  if (status != B200FA_OK || a->batch == 0) return status;
  PagedParams p;
  p.batch = a->batch, p.heads_q = a->heads_q, p.heads_kv = a->heads_kv, p.head_dim = a->head_dim;
  p.num_pages = a->num_pages, p.page_size = a->page_size, p.capacity = a->max_pages * a->page_size;
  p.window_left = a->window_left, p.sink = a->sink_size;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.q = static_cast<const __nv_bfloat16*>(a->q), p.k = static_cast<const __nv_bfloat16*>(a->k_cache);
  p.v = static_cast<const __nv_bfloat16*>(a->v_cache), p.out = static_cast<__nv_bfloat16*>(a->out);
  p.table = a->block_table, p.lengths = a->cache_seqlens, p.lse = a->softmax_lse;
  p.q_seq = a->q_stride[0], p.q_head = a->q_stride[1], p.out_seq = a->out_stride[0], p.out_head = a->out_stride[1];
  p.k_page = a->k_stride[0], p.k_row = a->k_stride[1], p.k_head = a->k_stride[2];
  p.v_page = a->v_stride[0], p.v_row = a->v_stride[1], p.v_head = a->v_stride[2];
  p.table_seq = a->table_stride, p.lse_seq = a->heads_q;
  paged_decode_kernel<<<dim3((unsigned)a->batch, (unsigned)a->heads_q), 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
  B200FA_CUDA_CHECK(cudaGetLastError());
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
