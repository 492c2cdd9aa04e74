// What the decode kernels share: the order in which blocks take the sequences, and how the warps' and blocks' partial
// outputs become one (decode_sm100.cu describes the scheme).
#pragma once

#include "attn_internal.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace minfer_attn {

namespace {

constexpr int kWarps = 4;
constexpr int kMaxParts = 16;    // blocks per cluster (above 8: the non-portable size, which sm_100 has)
constexpr int kMaxRanked = 256;  // sequences a block ranks by length
constexpr int kTileKeys = 16;

// kept out of line: the error path must not cost the streaming loop registers
__device__ __noinline__ void report_bad_page(int32_t* status, int b, int slot, int page) {
  if (status != nullptr && atomicCAS(status, 0, kStatusBadPage) == 0) {
    status[1] = b;
    status[2] = slot;
    status[3] = page;
  }
}

// A block whose wait for the cluster's partial outputs ran out.  It reports that, and stays until nothing can be stored into
// its shared memory any more: the barrier waits for the threads of the cluster that have not ended, so it passes when
// every other block has sent and ended, or has given up (after sending) as well; what is then on its way completes the mbarrier.
__device__ __noinline__ void give_up(uint64_t* arrived, int32_t* status, int part) {
  if (status != nullptr && atomicCAS(status, 0, kStatusWaitTimeout) == 0) {
    status[1] = part;
    status[2] = static_cast<int32_t>(blockIdx.z);
    status[3] = 50;
  }
  cluster_sync_unaligned();
  volatile int own_flag = 0;
  mbar_wait<true>(arrived, 0, &own_flag);
}

// The sequence that is i-th when the batch is ordered by descending length (ties by index); every block finds its own.
// Blocks start in grid order, so the long sequences start first and the last wave holds the short ones.  Four lengths
// per shared-memory read, the reads of one sequence dealt out over the lanes a small batch leaves free.  Returns the
// sequence and its length.  The lengths are clamped to [0, max_len] before they are ranked: only then is every one of them
// above the padding (-1), `mine + 1` exact, and every rank taken once.
__device__ __forceinline__ int2 sequence_by_length(const int32_t* lens, int batch, int max_len, int i, int* scratch, int tid) {
  const int n4 = (batch + 3) / 4;
  for (int t = tid; t < 4 * n4; t += kWarps * 32) scratch[t] = t < batch ? max(0, min(lens[t], max_len)) : -1;
  int lanes = 1;  // per sequence
  while (lanes < 16 && 2 * lanes * batch <= kWarps * 32) lanes *= 2;
  __syncthreads();
  for (int t0 = 0; t0 < batch; t0 += kWarps * 32 / lanes) {
    const int t = t0 + tid / lanes;
    const int mine = t < batch ? scratch[t] : 0;
    int rank = 0;
    for (int u = tid % lanes; u < n4; u += lanes) {
      const int4 x = reinterpret_cast<const int4*>(scratch)[u];
      // lengths before `t` count when equal, those behind it do not
      rank += (x.x >= mine + (4 * u >= t ? 1 : 0)) + (x.y >= mine + (4 * u + 1 >= t ? 1 : 0)) +
              (x.z >= mine + (4 * u + 2 >= t ? 1 : 0)) + (x.w >= mine + (4 * u + 3 >= t ? 1 : 0));
    }
    for (int d = lanes >> 1; d > 0; d >>= 1) rank += __shfl_xor_sync(0xFFFFFFFFu, rank, d);
    if (t < batch && rank == i && tid % lanes == 0) *reinterpret_cast<int2*>(&scratch[kMaxRanked]) = make_int2(t, mine);
  }
  __syncthreads();
  return *reinterpret_cast<const int2*>(&scratch[kMaxRanked]);
}

// Rows that end as zeros: no key; and, unless the kernel hands NaN on, a sum that is NaN.
template <bool kKeepNan>
__device__ __forceinline__ bool no_result(float l) {
  if constexpr (kKeepNan) return l == 0.f;
  return !(l > 0.f);
}

// Merges the warps of the block - each has left its unnormalised output in its part of the ring, D + 4 floats per head,
// and its (max, sum) pairs behind the rings - and the blocks of the cluster, and writes the result.  L: the kernel's shared memory.
template <int D, bool BF16, int NT, class L, bool kKeepNan>
__device__ __forceinline__ void merge_partials(const DecodeArgs& a, uint8_t* smem, uint64_t* arrived, volatile int* abort_flag, int b, int kvh, int part,
                                               int n_parts, bool clustered, int tid) {
  const int group = a.group;
  constexpr int kRow = D + 4;  // floats per head
  float2* wml = reinterpret_cast<float2*>(smem + L::kRingBytes);                       // [kWarps][8 NT] (max, sum) per warp
  float* pbuf = reinterpret_cast<float*>(smem + L::kRingBytes + L::kWmlBytes);         // [n_parts][group][dims]
  float2* pml = reinterpret_cast<float2*>(smem + L::kRingBytes + L::kWmlBytes + L::kPartBytes);  // [n_parts][group]
  static_assert(D / 4 >= kMaxParts, "a head's four-dimension pieces cover the blocks of a cluster");
  constexpr int kLogD = D == 128 ? 7 : 6;
  __syncthreads();
  // Block r of the cluster finishes dimensions [r, r + 1) * D / n_parts of every head (n_parts is a power of two of at
  // most D / 4).  All index arithmetic below is shifts: this is a chain of latencies, and a division by a runtime value is
  // a tenth of it.
  const bool exchange = clustered && n_parts > 1;
  const int log_dims = kLogD - (exchange ? __ffs(n_parts) - 1 : 0);  // dimensions per block
  const int dims = 1 << log_dims;
  if (exchange) cluster_wait();  // every block of the cluster has started and initialised its barrier
  for (int e4 = tid; e4 < group * (D / 4); e4 += kWarps * 32) {
    const int g = e4 / (D / 4), j = e4 % (D / 4), d = j * 4;
    float2 ml[kWarps];
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      ml[w] = wml[w * 8 * NT + g];
      M = fmaxf(M, ml[w].x);
    }
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float sc = (ml[w].x == -INFINITY) ? 0.f : ex2_approx(ml[w].x - M);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + w * L::kWarpBytes) + g * kRow + d);
      o.x += sc * x.x;
      o.y += sc * x.y;
      o.z += sc * x.z;
      o.w += sc * x.w;
      l += sc * ml[w].y;
    }
    const int h = kvh * group + g;
    if (exchange) {
      // the block that finishes these four dimensions gets them, and (from one lane each) every block the (max, sum)
      const uint32_t bar_addr = smem_u32(arrived);
      const int rank = d >> log_dims;
      st_async_v4(cluster_map(smem_u32(&pbuf[(((part * group + g) << log_dims) + d) - (rank << log_dims)]), rank), o, cluster_map(bar_addr, rank));
      if (j < n_parts) st_async_v2(cluster_map(smem_u32(&pml[part * group + g]), j), M, l, cluster_map(bar_addr, j));
    } else if (clustered) {
      const float inv = 1.f / l;
      if (no_result<kKeepNan>(l)) o = make_float4(0.f, 0.f, 0.f, 0.f);
      else o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      uint8_t* op = reinterpret_cast<uint8_t*>(a.out) +
                    2 * (static_cast<size_t>(b) * a.out_stride[0] + static_cast<size_t>(h) * a.out_stride[1] + d);
      *reinterpret_cast<uint2*>(op) = make_uint2(pack2<BF16>(o.x, o.y), pack2<BF16>(o.z, o.w));
    } else {
      const size_t pidx = (static_cast<size_t>(b) * a.n_heads + h) * n_parts + part;
      *reinterpret_cast<float4*>(a.part_o + pidx * D + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(a.part_ml + pidx * 2) = make_float2(M, l);
    }
  }
  if (!exchange) return;
  // ---- merge the cluster's blocks: each finishes its dimensions once every block's values have arrived (a block that
  // has sent its own and received the others' has nothing more to do with them) ----
  // (their stores are released at the scope of the cluster: the wait acquires there)
  if (!mbar_wait<true>(arrived, 0, abort_flag)) {
    give_up(arrived, a.status, part);
    return;
  }
  for (int t = 2 * tid; t < (group << log_dims); t += 2 * kWarps * 32) {
    const int g = t >> log_dims, d = (part << log_dims) + (t & (dims - 1));
    float2 ml[kMaxParts], x[kMaxParts];
    float M = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int p = 0; p < kMaxParts; ++p) {
      const int q = p < n_parts ? p : 0;
      ml[p] = pml[q * group + g];
      x[p] = *reinterpret_cast<const float2*>(&pbuf[((q * group) << log_dims) + t]);
      if (p >= n_parts) {  // counts for nothing, whatever part 0 holds
        ml[p] = make_float2(-INFINITY, 0.f);
        x[p] = make_float2(0.f, 0.f);
      }
      M = fmaxf(M, ml[p].x);
    }
#pragma unroll
    for (int p = 0; p < kMaxParts; ++p) {
      const float sc = (ml[p].x == -INFINITY) ? 0.f : ex2_approx(ml[p].x - M);
      o0 += sc * x[p].x;
      o1 += sc * x[p].y;
      l += sc * ml[p].y;
    }
    const float inv = 1.f / l;
    o0 = no_result<kKeepNan>(l) ? 0.f : o0 * inv;
    o1 = no_result<kKeepNan>(l) ? 0.f : o1 * inv;
    uint8_t* op = reinterpret_cast<uint8_t*>(a.out) + 2 * (static_cast<size_t>(b) * a.out_stride[0] +
                                                           static_cast<size_t>(kvh * group + g) * a.out_stride[1] + d);
    *reinterpret_cast<uint32_t*>(op) = pack2<BF16>(o0, o1);
  }
}

// The merge is a latency problem (a few hundred bytes per thread, every load a trip to L2 or HBM), so the loads are
// issued eight at a time: the (max, sum) pairs of eight splits, then the eight partial outputs they weight.
template <int D, bool BF16>
__global__ void __launch_bounds__(D) decode_combine_kernel(const DecodeArgs a) {
  const int h = blockIdx.x;
  const int b = blockIdx.y;
  const int d = threadIdx.x;
  grid_launch_dependents();
  grid_dependency_wait();
  const int len = min(a.lens[b], a.max_len);
  const int ns = (len + a.chunk - 1) / a.chunk;
  const size_t p0 = (static_cast<size_t>(b) * a.n_heads + h) * a.n_split;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + p0;
  const float* po = a.part_o + p0 * D + d;
  constexpr int kBatch = 8;
  float M = -INFINITY;
  for (int s0 = 0; s0 < ns; s0 += kBatch) {
    float m[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) m[j] = (s0 + j < ns) ? ml[s0 + j].x : -INFINITY;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) M = fmaxf(M, m[j]);
  }
  float o = 0.f, l = 0.f;
  for (int s0 = 0; s0 < ns; s0 += kBatch) {
    float2 w[kBatch];
    float x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const bool live = s0 + j < ns;
      w[j] = live ? ml[s0 + j] : make_float2(-INFINITY, 0.f);
      x[j] = live ? po[static_cast<size_t>(s0 + j) * D] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float sc = (w[j].x == -INFINITY) ? 0.f : ex2_approx(w[j].x - M);
      l += sc * w[j].y;
      o += sc * x[j];
    }
  }
  const float r = (l > 0.f) ? o / l : 0.f;
  uint8_t* op = reinterpret_cast<uint8_t*>(a.out) +
                2 * (static_cast<size_t>(b) * a.out_stride[0] + static_cast<size_t>(h) * a.out_stride[1] + d);
  if constexpr (BF16) *reinterpret_cast<__nv_bfloat16*>(op) = __float2bfloat16_rn(r);
  else *reinterpret_cast<__half*>(op) = __float2half_rn(r);
}

}  // namespace

}  // namespace minfer_attn
