// Rows of a block-scaled 8-bit KV cache as 16-bit values: code * scale, rounded once.  What a prompt's attention behind a cached
// prefix reads (the prefill kernel's operands are 16-bit tiles that TMA brings from memory).  HBM-bound: one byte in, two out.
//
// A thread takes eight codes (8 bytes in, 16 out, both coalesced) of kBatch rows, all loads before the first store.
#include "attn_internal.h"
#include "b8.cuh"
#include "ptx.cuh"

namespace minfer_attn {

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8;

__device__ __noinline__ void report_bad_page(int32_t* status, int b, int slot, int page) {
  if (status != nullptr && atomicCAS(status, 0, kStatusBadPage) == 0) {
    status[1] = b;
    status[2] = slot;
    status[3] = page;
  }
}

template <int D, bool BF16, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_b8_kernel(const KvReadArgs a) {
  constexpr int kLanes = D / 8;                  // threads per row
  constexpr int kRows = kThreads / kLanes;       // rows per step
  grid_launch_dependents();
  grid_dependency_wait();
  const unsigned per = static_cast<unsigned>((a.max_len + kRows * kBatch - 1) / (kRows * kBatch));  // thread blocks per sequence and head
  const unsigned pair = blockIdx.x / per;        // sequence and head
  const int first = static_cast<int>(blockIdx.x - pair * per) * (kRows * kBatch);
  const int b = static_cast<int>(pair / static_cast<unsigned>(a.n_kv_heads)), h = static_cast<int>(pair - static_cast<unsigned>(b) * static_cast<unsigned>(a.n_kv_heads));
  const int len = min(a.lens[b], a.max_len);
  const int t = static_cast<int>(threadIdx.x) % kLanes;
  const int row0 = first + static_cast<int>(threadIdx.x) / kLanes;
  if (first >= len) return;
  const bool is_v = blockIdx.y != 0;
  const uint8_t* cache = reinterpret_cast<const uint8_t*>(is_v ? a.v_cache : a.k_cache) + static_cast<int64_t>(h) * a.cache_stride[1] + 8 * t;
  const float* scales = (is_v ? a.v_scale : a.k_scale) + static_cast<int64_t>(h) * a.scale_stride[1];
  uint8_t* out = reinterpret_cast<uint8_t*>(is_v ? a.v_out : a.k_out) + 2 * (static_cast<int64_t>(b) * a.out_stride[0] + static_cast<int64_t>(h) * a.out_stride[1] + 8 * t);
  uint2 c[kBatch];
  float s[kBatch];
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int row = row0 + u * kRows;
    c[u] = make_uint2(0, 0);
    s[u] = 0.f;
    if (row < len) {
      int outer = b, r = row;
      if (a.block_table != nullptr) {
        const int slot = row / a.page_size;
        outer = a.block_table[static_cast<size_t>(b) * a.table_stride + slot];
        if (static_cast<unsigned>(outer) >= static_cast<unsigned>(a.n_pages)) {
          if (t == 0) report_bad_page(a.status, b, slot, outer);
          outer = 0;
        }
        r = row - slot * a.page_size;
      }
      c[u] = *reinterpret_cast<const uint2*>(cache + static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(r) * a.cache_stride[2]);
      s[u] = scales[static_cast<int64_t>(outer) * a.scale_stride[0] + (r >> a.log_block)];
    }
  }
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const int row = row0 + u * kRows;
    if (row < len) {
      float x[8];
      b8_values8<kFmt>(c[u], x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= s[u];
      *reinterpret_cast<uint4*>(out + 2 * static_cast<int64_t>(row) * a.out_stride[2]) =
          make_uint4(pack2<BF16>(x[0], x[1]), pack2<BF16>(x[2], x[3]), pack2<BF16>(x[4], x[5]), pack2<BF16>(x[6], x[7]));
    }
  }
}

template <int D, bool BF16, int kFmt>
cudaError_t launch_one(const KvReadArgs& a, cudaStream_t stream) {
  constexpr int rows = kThreads / (D / 8) * kBatch;
  const int64_t blocks = (static_cast<int64_t>(a.max_len) + rows - 1) / rows * a.batch * a.n_kv_heads;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  LaunchAttrs at(stream);
  at.cfg.gridDim = dim3(static_cast<unsigned>(blocks), 2);
  at.cfg.blockDim = dim3(kThreads);
  return cudaLaunchKernelEx(&at.cfg, kv_read_b8_kernel<D, BF16, kFmt>, a);
}

template <int D, bool BF16>
cudaError_t launch_fmt(const KvReadArgs& a, bool int8, cudaStream_t stream) {
  return int8 ? launch_one<D, BF16, kInt8>(a, stream) : launch_one<D, BF16, kE4M3>(a, stream);
}

}  // namespace

cudaError_t launch_kv_read_b8(const KvReadArgs& a, int head_dim, bool bf16, bool int8, cudaStream_t stream) {
  if (head_dim == 128) return bf16 ? launch_fmt<128, true>(a, int8, stream) : launch_fmt<128, false>(a, int8, stream);
  return bf16 ? launch_fmt<64, true>(a, int8, stream) : launch_fmt<64, false>(a, int8, stream);
}

}  // namespace minfer_attn
