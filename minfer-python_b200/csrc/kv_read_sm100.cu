// Rows of a block-scaled 8-bit KV cache as 16-bit values: code * scale in fp32, then rounded to the
// type (exact before that for e4m3 under powers of two; an int8 product has up to 31 bits).  What a prompt's attention behind a cached
// prefix reads (the prefill kernel's operands are 16-bit tiles that TMA brings from memory).  HBM-bound: one byte in, two out.
// 16000 rows of 8 heads, D=128, int8, pages of 256 tokens: 18.3 us from cold caches, 5.4 TB/s, 0.84 of what a copy reaches.
//
// A warp takes 16 consecutive rows, which lie in one page and in one block of tokens: one look-up for all of them.  A lane takes eight
// codes (8 bytes in, 16 out, both coalesced) of kBatch rows, all loads before the first store.
#include "attn_internal.h"
#include "b8.cuh"
#include "ptx.cuh"

namespace minfer_attn {

namespace {

// Small blocks, so that a finished warp's place is free at once (us with 256 / 128 / 64 threads, 16000 rows of 8 heads, D=128: int8 in pages of 256 tokens
// 19.8 / 19.2 / 18.3, in one piece 18.9 / 18.4 / 17.6, e4m3 17.4 / 17.5 / 17.6; 8 x 512 rows, D=64 3.8 / 3.6 / 3.7)
constexpr int kThreads = 64;
constexpr int kRows = kThreads / 32 * 16;  // per thread block

__device__ __noinline__ void report_bad_page(int32_t* status, int b, int slot, int page) {
  if (status != nullptr && atomicCAS(status, 0, kStatusBadPage) == 0) {
    status[1] = b;
    status[2] = slot;
    status[3] = page;
  }
}

template <int D, bool BF16, int kFmt>
__global__ void __launch_bounds__(kThreads) kv_read_b8_kernel(const KvReadArgs a) {
  constexpr int kLanes = D / 8;             // lanes per row
  constexpr int kSide = 32 / kLanes;        // rows that a warp instruction covers
  constexpr int kBatch = 16 / kSide;
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = static_cast<int>(threadIdx.x) & 31;
  const unsigned per = static_cast<unsigned>((a.max_len + kRows - 1) / kRows);  // thread blocks per sequence and head
  const unsigned pair = blockIdx.x / per;   // sequence and head
  const int row0 = static_cast<int>(blockIdx.x - pair * per) * kRows + static_cast<int>(threadIdx.x) / 32 * 16;  // of this warp
  const int b = static_cast<int>(pair / static_cast<unsigned>(a.n_kv_heads)), h = static_cast<int>(pair - static_cast<unsigned>(b) * static_cast<unsigned>(a.n_kv_heads));
  const int live = max(0, min(a.lens[b], a.max_len)) - row0;  // rows of the 16 that there are (a length near -2^31 less row0 would wrap to a huge one)
  if (live <= 0) return;
  const bool is_v = blockIdx.y != 0;
  int outer = b, r = row0;
  if (a.block_table != nullptr) {
    const int slot = row0 / a.page_size;
    outer = a.block_table[static_cast<size_t>(b) * a.table_stride + slot];
    if (static_cast<unsigned>(outer) >= static_cast<unsigned>(a.n_pages)) {
      if (lane == 0) report_bad_page(a.status, b, slot, outer);
      outer = 0;
    }
    r = row0 - slot * a.page_size;
  }
  const float s = (is_v ? a.v_scale : a.k_scale)[static_cast<int64_t>(outer) * a.scale_stride[0] + static_cast<int64_t>(h) * a.scale_stride[1] + (r >> a.log_block)];
  const int first = lane / kLanes, t = lane % kLanes;
  const uint8_t* src = reinterpret_cast<const uint8_t*>(is_v ? a.v_cache : a.k_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] +
                       static_cast<int64_t>(h) * a.cache_stride[1] + static_cast<int64_t>(r + first) * a.cache_stride[2] + 8 * t;
  uint8_t* dst = reinterpret_cast<uint8_t*>(is_v ? a.v_out : a.k_out) +
                 2 * (static_cast<int64_t>(b) * a.out_stride[0] + static_cast<int64_t>(h) * a.out_stride[1] + static_cast<int64_t>(row0 + first) * a.out_stride[2] + 8 * t);
  const int64_t src_step = kSide * a.cache_stride[2], dst_step = 2 * kSide * a.out_stride[2];
  uint2 c[kBatch];
#pragma unroll
  for (int u = 0; u < kBatch; ++u)
    if (u * kSide + first < live) c[u] = *reinterpret_cast<const uint2*>(src + u * src_step);
  const float2 s2 = make_float2(s, s);
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    if (u * kSide + first < live) {
      float x[8];
      b8_values8<kFmt>(c[u], x);
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = __fmul2_rn(make_float2(x[2 * i], x[2 * i + 1]), s2);
        w[i] = pack2<BF16>(y.x, y.y);
      }
      *reinterpret_cast<uint4*>(dst + u * dst_step) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

template <int D, bool BF16, int kFmt>
cudaError_t launch_one(const KvReadArgs& a, cudaStream_t stream) {
  const int64_t blocks = (static_cast<int64_t>(a.max_len) + kRows - 1) / kRows * a.batch * a.n_kv_heads;
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
