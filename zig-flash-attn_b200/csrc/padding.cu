// Rows of packed tensors that belong to no sequence: those in front of cu_seqlens[0] and those at or behind
// cu_seqlens[batch]. The attention kernels never write them; the *_all_rows entries define them: zeros, and a log-sum-exp of
// -inf. A layer in front of the attention sums its weight gradient over all rows, so what stands in the gradients of padding
// rows must be zero and not what the memory held before.
//
// One launch for all results of a pass. How many rows there are is known on the device only, so the grid is that of the
// largest case up to four blocks per SM, and blocks without rows end after two loads.
#include "common.h"

namespace b200fa {

constexpr int kPaddingThreads = 256, kPaddingBlocks = 4 * 148;

// Contiguous tensors of `rows` rows of 16-byte `pieces`; lse: (heads, rows[0]).
struct Padding {
  int count, batch, heads;
  uint4* out[3];
  const int32_t* cu[3];
  int64_t rows[3], pieces[3];
  float* lse;
};

__global__ void __launch_bounds__(kPaddingThreads) clear_padding_kernel(const __grid_constant__ Padding a) {
  const bool is_lse = (int)blockIdx.y == a.count;
  const int which = is_lse ? 0 : blockIdx.y;
  const int64_t rows = a.rows[which], head = a.cu[which][0], tail = a.cu[which][a.batch];
  const int64_t first = head < 0 ? 0 : head < rows ? head : rows;  // rows [0, first) and [last, rows)
  const int64_t last = tail < first ? first : tail < rows ? tail : rows;
  const int64_t count = first + (rows - last), step = (int64_t)gridDim.x * kPaddingThreads;
  if (count == 0) return;
  const int64_t begin = (int64_t)blockIdx.x * kPaddingThreads + threadIdx.x;
  if (is_lse) {
    for (int64_t i = begin; i < a.heads * count; i += step) {
      const int64_t h = i / count, r = i - h * count;
      a.lse[h * rows + (r < first ? r : last + (r - first))] = -INFINITY;
    }
  } else {
    const int64_t pieces = a.pieces[which], front = first * pieces;
    for (int64_t i = begin; i < count * pieces; i += step)
      a.out[which][i < front ? i : last * pieces + (i - front)] = make_uint4(0, 0, 0, 0);
  }
}

static int launch_clear_padding(const Padding& a, cudaStream_t stream) {
  int64_t most = 0;
  for (int i = 0; i < a.count; ++i) most = most < a.rows[i] * a.pieces[i] ? a.rows[i] * a.pieces[i] : most;
  if (most == 0) return B200FA_OK;
  const int64_t blocks = (most + kPaddingThreads - 1) / kPaddingThreads;
  const dim3 grid((unsigned)(blocks < kPaddingBlocks ? blocks : kPaddingBlocks), (unsigned)(a.count + (a.lse ? 1 : 0)));
  clear_padding_kernel<<<grid, kPaddingThreads, 0, stream>>>(a);
  B200FA_CUDA_CHECK(cudaGetLastError());
  return B200FA_OK;
}

// Adds a result of the pass; its rows must lie one behind the other.
static int add(Padding* a, void* out, const int64_t* stride, const int32_t* cu, int64_t rows, int heads, int head_dim) {
  // a tensor without rows may have any strides
  B200FA_REQUIRE(rows == 0 || (stride[2] == head_dim && stride[1] == (int64_t)heads * head_dim), "results of all rows must be contiguous");
  B200FA_REQUIRE((out || rows == 0) && head_dim % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
                 "results of all rows need a 16-byte aligned pointer and rows of whole 16-byte pieces");
  const int i = a->count++;
  a->out[i] = static_cast<uint4*>(out), a->cu[i] = cu, a->rows[i] = rows, a->pieces[i] = (int64_t)heads * head_dim / 8;
  return B200FA_OK;
}

}  // namespace b200fa

using namespace b200fa;

extern "C" {

int b200fa_sink_fwd_all_rows(const b200fa_fwd_args* args, int32_t sink_size, void* stream) {
  Padding a{};
  const bool packed = args && args->problem.cu_seqlens_q;
  if (packed) {
    const b200fa_problem& p = args->problem;
    const int status = add(&a, args->out, args->out_stride, p.cu_seqlens_q, p.seqlen_q, p.heads_q, p.head_dim);
    if (status != B200FA_OK) return status;
    B200FA_REQUIRE(p.seqlen_q == 0 || args->lse_stride[1] == p.seqlen_q, "results of all rows must be contiguous");
    B200FA_REQUIRE(p.seqlen_q == 0 || args->softmax_lse, "null tensor pointer");
    a.batch = p.batch, a.heads = p.heads_q, a.lse = args->softmax_lse;
  }
  const int status = b200fa_sink_fwd(args, sink_size, stream);
  return status == B200FA_OK && packed ? launch_clear_padding(a, static_cast<cudaStream_t>(stream)) : status;
}

int b200fa_sink_bwd_all_rows(const b200fa_bwd_args* args, int32_t sink_size, void* stream) {
  Padding a{};
  const bool packed = args && args->problem.cu_seqlens_q;
  if (packed) {
    const b200fa_problem& p = args->problem;
    int status = add(&a, args->dq, args->dq_stride, p.cu_seqlens_q, p.seqlen_q, p.heads_q, p.head_dim);
    if (status == B200FA_OK) status = add(&a, args->dk, args->dk_stride, p.cu_seqlens_k, p.seqlen_k, p.heads_kv, p.head_dim);
    if (status == B200FA_OK) status = add(&a, args->dv, args->dv_stride, p.cu_seqlens_k, p.seqlen_k, p.heads_kv, p.head_dim);
    if (status != B200FA_OK) return status;
    a.batch = p.batch;
  }
  const int status = b200fa_sink_bwd(args, sink_size, stream);
  return status == B200FA_OK && packed ? launch_clear_padding(a, static_cast<cudaStream_t>(stream)) : status;
}

}  // extern "C"
