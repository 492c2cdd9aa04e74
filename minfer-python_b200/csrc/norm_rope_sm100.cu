// RMS norms of the query and key heads, rotary position embedding and the KV-cache append in one pass over q, k and v: the step
// before attention for models that norm their heads, and for caches held in 8 bits.  HBM-bound and elementwise but for two
// reductions: a row's sum of squares, and the largest magnitude in a block of an 8-bit cache.
//
//   y     = x * rsqrt(mean(x^2) + eps) * weight          over a head's head_dim values, fp32 (left out without weights)
//   angle = position * freq_base ^ (-2 i / rotary_dim)   i-th pair; interleaved (y[2i], y[2i+1]) or two halves (y[i], y[i + rotary_dim/2])
//   rotated in fp32, rounded once to what is stored
//
// The pair layouts are those of the reference's il_rope / neox_rope
// (src/minfer/kernels/torch_ext/csrc/cuda/il_rope/kernel.cuh:9-39, neox_rope/kernel.cuh:9-38).  The angle is not: an fp32
// product position * frequency is off by 2^-24 of itself, 4e-3 at position 65536, so the frequency is kept in turns as a
// 64-bit fraction (freq / 2 pi mod 1, computed on the host in extended precision), the position multiplies it modulo 2^64 - whole
// turns fall away exactly - and sincospif takes the top 32 bits.  That is also cheaper than sincosf of a large argument.
//
// A row (one head of one token) belongs to TPR = 4, 8 or 16 lanes with two 16-byte chunks each; in the two-halves form they are a chunk and
// its partner, so a rotated pair never leaves its thread.
#include "../../include/minfer_attn.h"
#include "attn_internal.h"
#include "b8.cuh"
#include "ptx.cuh"

#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace minfer_attn {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxAngles = 1024;  // (token, pair) angles a block of rows keeps in shared memory
constexpr int kStages = 4;        // rows of a thread on their way through shared memory (no registers held while they fly)
constexpr int kStageVecs = 2 * kThreads;  // 16-byte pieces of a stage: two chunks per thread
constexpr size_t kRowsSmem = 2 * kMaxAngles * sizeof(float) + kStages * kStageVecs * 16;

template <bool BF16>
__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = t.x;
      f[2 * i + 1] = t.y;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ uint4 pack8(const float* f) {
  return make_uint4(pack2<BF16>(f[0], f[1]), pack2<BF16>(f[2], f[3]), pack2<BF16>(f[4], f[5]), pack2<BF16>(f[6], f[7]));
}

// the two chunks of a lane, and which pairs they hold
template <bool kNeox>
struct Chunks {
  int c0, c1;     // 16-byte chunks of the row
  int i0, i1;     // first pair of chunk c0, and of its second four angles
  bool live;      // head_dim / 16 need not be a power of two: lanes beyond it have no chunk
  bool rot0, rot1;
  __device__ __forceinline__ Chunks(int t, int head_dim, int rotary_dim) {
    const int lanes = head_dim / 16;
    live = t < lanes;
    if (!live) t = 0;
    if constexpr (kNeox) {
      const int half = rotary_dim / 16;
      rot0 = rot1 = t < half;
      c0 = rot0 ? t : 2 * t;
      c1 = rot0 ? t + half : 2 * t + 1;
      i0 = 8 * t;
      i1 = 8 * t + 4;
    } else {
      c0 = t;
      c1 = t + lanes;
      rot0 = c0 < rotary_dim / 8;
      rot1 = c1 < rotary_dim / 8;
      i0 = 4 * c0;
      i1 = 4 * c1;
    }
  }
};

// cos and sin of pair i at a position
__device__ __forceinline__ float2 angle_of(const NormRopeArgs& a, int pos, int i) {
  const uint64_t turns = static_cast<uint64_t>(static_cast<int64_t>(pos)) * a.turns[i];
  float s, c;
  sincospif(static_cast<float>(static_cast<int32_t>(turns >> 32)) * 4.656612873077392578125e-10f, &s, &c);  // 2^-31: half turns
  return make_float2(c, s);
}

// 16 weights of a lane's chunks, fp32; `w` points to a head's row of them
__device__ __forceinline__ void load_weights(const void* w, int kind, int c0, int c1, float* f) {
  if (kind == 2) {  // fp32
    const float4* p = reinterpret_cast<const float4*>(w);
    const float4 x[4] = {p[2 * c0], p[2 * c0 + 1], p[2 * c1], p[2 * c1 + 1]};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[4 * i] = x[i].x;
      f[4 * i + 1] = x[i].y;
      f[4 * i + 2] = x[i].z;
      f[4 * i + 3] = x[i].w;
    }
    return;
  }
  const uint4* p = reinterpret_cast<const uint4*>(w);
  const uint4 x = p[c0], y = p[c1];
  if (kind == 1) {
    unpack8<true>(x, f);
    unpack8<true>(y, f + 8);
  } else {
    unpack8<false>(x, f);
    unpack8<false>(y, f + 8);
  }
}

// 1 / rms of a row, over its TPR lanes (called by whole warps)
template <int TPR>
__device__ __forceinline__ float inverse_rms(const float* x, bool live, float inv_dim, float eps) {
  float ss = 0.f, s2 = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    ss = fmaf(x[i], x[i], ss);
    s2 = fmaf(x[i + 1], x[i + 1], s2);
  }
  ss = live ? ss + s2 : 0.f;
#pragma unroll
  for (int d = TPR / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
  return rsqrtf(fmaf(ss, inv_dim, eps));
}

// x[e0], x[e1] of pair p (p = 0 .. 7): two halves (p, 8 + p), interleaved (2 p, 2 p + 1); pairs 0-3 and 4-7 of the latter lie in chunks 0 and 1
template <bool kNeox>
__device__ __forceinline__ constexpr int pair_lo(int p) { return kNeox ? p : 2 * p; }
template <bool kNeox>
__device__ __forceinline__ constexpr int pair_hi(int p) { return kNeox ? 8 + p : 2 * p + 1; }

// the lane's eight angles out of a token's rows of cosines and sines
template <bool kNeox>
__device__ __forceinline__ void load_angles(const float* cosines, const float* sines, const Chunks<kNeox>& ch, float* cs, float* sn) {
  if (ch.rot0) {
    *reinterpret_cast<float4*>(cs) = *reinterpret_cast<const float4*>(cosines + ch.i0);
    *reinterpret_cast<float4*>(sn) = *reinterpret_cast<const float4*>(sines + ch.i0);
  }
  if (ch.rot1) {
    *reinterpret_cast<float4*>(cs + 4) = *reinterpret_cast<const float4*>(cosines + ch.i1);
    *reinterpret_cast<float4*>(sn + 4) = *reinterpret_cast<const float4*>(sines + ch.i1);
  }
}

__device__ __noinline__ void report(int32_t* status, int code, int x, int y, int z) {
  if (status != nullptr && atomicCAS(status, 0, code) == 0) {
    status[1] = x;
    status[2] = y;
    status[3] = z;
  }
}

// Where position `pos` of sequence b lives: the outer index of the caches (sequence or page) and the row inside it.  False, and a
// report where `tell`, if the position lies outside the cache or the table's entry outside the pools: such a row is never written.
__device__ __forceinline__ bool locate(const NormRopeArgs& a, int b, int pos, bool tell, int& outer, int& row) {
  outer = b;
  row = pos;
  if (pos < 0 || pos >= a.max_len) {
    if (tell) report(a.status, kStatusBadPosition, b, pos, a.max_len);
    return false;
  }
  if (a.block_table != nullptr) {
    const int slot = pos / a.page_size;
    const int page = a.block_table[static_cast<size_t>(b) * a.table_stride + slot];
    if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.n_pages)) {
      if (tell) report(a.status, kStatusBadPage, b, slot, page);
      return false;
    }
    outer = page;
    row = pos - slot * a.page_size;
  }
  return true;
}

// ---- rows one by one: q, and k / v in place or into a 16-bit cache; with an 8-bit cache (kFmt) k and v of a call of one token per
// sequence, whose row alone decides about its block ----
//
// A block takes 2^log_tb tokens; each token's rows are dealt out over the row groups it gets (and over `slices` blocks).  A thread keeps
// its token's angles, multiplied into the weights, in registers for all its rows (32 values; formed anew where the next row has other
// weights), and its next rows on their way through shared memory.
template <int TPR, bool BF16, bool kNeox, int kFmt>
__device__ __forceinline__ void rows_role(const NormRopeArgs& a, unsigned bx, unsigned slice, unsigned slices, int n_k, int n_v, float* smem) {
  constexpr int kGroups = kThreads / TPR;
  float* s_cos = smem;
  float* s_sin = smem + kMaxAngles;
  uint4* s_rows = reinterpret_cast<uint4*>(smem + 2 * kMaxAngles);
  const int tid = static_cast<int>(threadIdx.x);
  const int t = tid % TPR, rg = tid / TPR;
  const int log_gpt = (31 - __clz(kGroups)) - a.log_tb;  // row groups per token, log2
  const unsigned n_tokens = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.seq);
  const unsigned token0 = bx << a.log_tb;
  const int tb = rg >> log_gpt;
  const bool token_ok = token0 + tb < n_tokens;
  const unsigned token = token_ok ? token0 + tb : n_tokens - 1;
  const int b = static_cast<int>(token / static_cast<unsigned>(a.seq));
  const int l = static_cast<int>(token - static_cast<unsigned>(b) * static_cast<unsigned>(a.seq));
  const Chunks<kNeox> ch(t, a.head_dim, a.rotary_dim);
  const int n_q = a.q != nullptr ? a.n_heads : 0;
  const int n_rows = n_q + n_k + n_v;
  uint8_t* q_base = reinterpret_cast<uint8_t*>(a.q) + 2 * (static_cast<int64_t>(b) * a.q_stride[0] + static_cast<int64_t>(l) * a.q_stride[1]);
  const int64_t kv_off = 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + static_cast<int64_t>(l) * a.kv_stride[1]);
  const int step = static_cast<int>(slices) << log_gpt;
  const int first = (static_cast<int>(slice) << log_gpt) + (rg & ((1 << log_gpt) - 1));
  // kind 0: q, 1: k, 2: v
  auto row_at = [&](int r, int& kind, int& h) -> uint8_t* {
    if (r < n_q) {
      kind = 0;
      h = r;
      return q_base + 2 * static_cast<int64_t>(h) * a.q_stride[2];
    }
    kind = r < n_q + n_k ? 1 : 2;
    h = r - n_q - (kind == 2 ? n_k : 0);
    return const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(kind == 1 ? a.k : a.v)) + kv_off + 2 * static_cast<int64_t>(h) * a.kv_stride[2];
  };
  // (all row groups of a block make the same number of steps, so that warps stay whole)
  const int n_steps = n_rows > static_cast<int>(slice << log_gpt) ? (n_rows - static_cast<int>(slice << log_gpt) + step - 1) / step : 0;
  auto issue = [&](int it) {
    const int r = first + it * step;
    if (token_ok && ch.live && r < n_rows) {
      int kind, h;
      const uint8_t* src = row_at(r, kind, h);
      uint4* dst = s_rows + (it % kStages) * kStageVecs + tid;
      cp_async_16(dst, src + 16 * ch.c0, true);
      cp_async_16(dst + kThreads, src + 16 * ch.c1, true);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int it = 0; it < kStages - 1; ++it) issue(it);  // on their way before the position is known

  const int pos = (a.start != nullptr ? a.start[b] : a.start_pos) + l;
  // the block's angles, dealt out over its threads
  const int pairs = a.rotary_dim / 2;
  for (int u = tid; u < (pairs << a.log_tb); u += kThreads) {
    const int ut = u / pairs, i = u - ut * pairs;
    const unsigned utok = min(token0 + ut, n_tokens - 1);
    const int ub = static_cast<int>(utok / static_cast<unsigned>(a.seq));
    const int up = (a.start != nullptr ? a.start[ub] : a.start_pos) + static_cast<int>(utok - static_cast<unsigned>(ub) * static_cast<unsigned>(a.seq));
    const float2 cs = angle_of(a, up, i);
    s_cos[u] = cs.x;
    s_sin[u] = cs.y;
  }
  int outer = 0, crow = 0;
  bool cache_ok = false;
  if (a.k_cache != nullptr && n_k + n_v > 0 && token_ok && first + (n_steps - 1) * step >= n_q)  // (a thread with query rows alone needs no place)
    cache_ok = locate(a, b, pos, t == 0, outer, crow);
  __syncthreads();

  // y_lo = lo * m[0] - hi * m[1], y_hi = lo * m[2] + hi * m[3]
  float m[4][8];
  const uint8_t* w_now = nullptr;
  bool have = false;
  const int w_bytes = a.w_kind == 2 ? 4 : 2;
  for (int it = 0; it < n_steps; ++it) {
    cp_async_wait<kStages - 2>();
    const int r = first + it * step;
    const bool row_ok = token_ok && r < n_rows;
    int kind = 2, h = 0;
    uint8_t* src = nullptr;
    if (row_ok) src = row_at(r, kind, h);
    uint4 raw0 = make_uint4(0, 0, 0, 0), raw1 = raw0;
    if (row_ok && ch.live) {
      raw0 = s_rows[(it % kStages) * kStageVecs + tid];
      raw1 = s_rows[(it % kStages) * kStageVecs + tid + kThreads];
    }
    issue(it + kStages - 1);
    float x[16];
    unpack8<BF16>(raw0, x);
    unpack8<BF16>(raw1, x + 8);
    if (kind != 2) {
      const uint8_t* wp = nullptr;
      if (a.q_weight != nullptr)
        wp = kind == 0 ? reinterpret_cast<const uint8_t*>(a.q_weight) + static_cast<int64_t>(h) * a.w_stride[0] * w_bytes
                       : reinterpret_cast<const uint8_t*>(a.k_weight) + static_cast<int64_t>(h) * a.w_stride[1] * w_bytes;
      if (!have || wp != w_now) {
        float w[16], cs[8], sn[8];
        if (wp != nullptr) {
          load_weights(wp, a.w_kind, ch.c0, ch.c1, w);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = 1.f;
        }
        load_angles<kNeox>(s_cos + tb * pairs, s_sin + tb * pairs, ch, cs, sn);
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const bool rot = (kNeox || p < 4) ? ch.rot0 : ch.rot1;
          const float c = rot ? cs[p] : 1.f, sv = rot ? sn[p] : 0.f;
          m[0][p] = w[pair_lo<kNeox>(p)] * c;
          m[1][p] = w[pair_hi<kNeox>(p)] * sv;
          m[2][p] = w[pair_lo<kNeox>(p)] * sv;
          m[3][p] = w[pair_hi<kNeox>(p)] * c;
        }
        w_now = wp;
        have = true;
      }
    }
    if (a.q_weight != nullptr && __any_sync(0xFFFFFFFFu, kind != 2)) {
      const float scale = inverse_rms<TPR>(x, ch.live, a.inv_dim, a.eps);
      if (kind != 2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= scale;
      }
    }
    if (kind != 2) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        constexpr bool two_chunks = !kNeox;
        const float lo = x[pair_lo<kNeox>(p)], hi = x[pair_hi<kNeox>(p)];
        if ((two_chunks && p >= 4) ? ch.rot1 : ch.rot0) {
          x[pair_lo<kNeox>(p)] = fmaf(lo, m[0][p], -(hi * m[1][p]));
          x[pair_hi<kNeox>(p)] = fmaf(lo, m[2][p], hi * m[3][p]);
        } else {  // (not 0 * hi: an infinite value stays in its place)
          x[pair_lo<kNeox>(p)] = lo * m[0][p];
          x[pair_hi<kNeox>(p)] = hi * m[3][p];
        }
      }
    }
    if constexpr (kFmt == 0) {
      if (!row_ok || !ch.live) continue;
      uint8_t* dst = src;
      if (kind != 0 && a.k_cache != nullptr) {
        if (!cache_ok) continue;
        dst = reinterpret_cast<uint8_t*>(kind == 1 ? a.k_cache : a.v_cache) +
              2 * (static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(h) * a.cache_stride[1] + static_cast<int64_t>(crow) * a.cache_stride[2]);
      }
      if (kind != 2) {
        raw0 = pack8<BF16>(x);
        raw1 = pack8<BF16>(x + 8);
      }
      *reinterpret_cast<uint4*>(dst + 16 * ch.c0) = raw0;
      *reinterpret_cast<uint4*>(dst + 16 * ch.c1) = raw1;
    } else {
      if (row_ok && kind == 0 && ch.live) {
        *reinterpret_cast<uint4*>(src + 16 * ch.c0) = pack8<BF16>(x);
        *reinterpret_cast<uint4*>(src + 16 * ch.c1) = pack8<BF16>(x + 8);
      }
      const bool cached = row_ok && kind != 0 && cache_ok;
      if (!__any_sync(0xFFFFFFFFu, cached)) continue;
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));
#pragma unroll
      for (int d = TPR / 2; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
      const int begun = crow & ((1 << a.log_block) - 1);  // rows of the block that are there
      uint8_t* blk_rows = nullptr;
      float s0 = 0.f, s1 = 0.f;
      if (cached) {
        float* sc = (kind == 1 ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + static_cast<int64_t>(h) * a.scale_stride[1] + (crow >> a.log_block);
        blk_rows = reinterpret_cast<uint8_t*>(kind == 1 ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] +
                   static_cast<int64_t>(h) * a.cache_stride[1] + static_cast<int64_t>(crow - begun) * a.cache_stride[2];
        s0 = begun != 0 ? *sc : 0.f;
        const float need = b8_scale<kFmt>(amax);
        s1 = s0 >= need ? s0 : need;
        const float r1 = b8_inverse(s1);
        uint8_t* dst = blk_rows + static_cast<int64_t>(begun) * a.cache_stride[2];
        *reinterpret_cast<uint2*>(dst + 8 * ch.c0) = b8_code8<kFmt>(x, s1, r1);
        *reinterpret_cast<uint2*>(dst + 8 * ch.c1) = b8_code8<kFmt>(x + 8, s1, r1);
        if (t == 0 && (begun == 0 || s1 != s0)) *sc = s1;  // (a block that begins here held anything)
      }
      // A scale that grew: the rows before are coded again, by the whole warp
      unsigned grown = __ballot_sync(0xFFFFFFFFu, cached && begun != 0 && s1 != s0 && t == 0);
      while (grown != 0) {
        const int from = __ffs(grown) - 1;
        grown &= grown - 1;
        const uint64_t p = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(blk_rows), from);
        const float o0 = __shfl_sync(0xFFFFFFFFu, s0, from), o1 = __shfl_sync(0xFFFFFFFFu, s1, from);
        const int n = __shfl_sync(0xFFFFFFFFu, begun, from);
        recode_rows<kFmt>(reinterpret_cast<uint8_t*>(p), a.cache_stride[2], n, a.head_dim / 16, o0, o1, tid & 31, 32);
      }
    }
  }
}

template <int TPR, bool BF16, bool kNeox, int kFmt>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_rows_kernel(const NormRopeArgs a) {
  __shared__ __align__(16) float s_all[kRowsSmem / 4];
  grid_launch_dependents();
  grid_dependency_wait();
  rows_role<TPR, BF16, kNeox, kFmt>(a, blockIdx.x, blockIdx.y, gridDim.y, a.k != nullptr ? a.n_kv_heads : 0, a.v != nullptr ? a.n_kv_heads : 0, s_all);
}

// ---- blocks of an 8-bit cache: k and v of calls with several tokens per sequence ----
//
// A unit is one block of tokens of one sequence, for a slice of the kv heads, of k or of v.  A head's rows of one block fill 2^log_block * TPR
// lanes: four, two or one head at a time, or two or four rows per thread.  The raw rows wait in shared memory (each thread's own
// pieces: no barrier, and a piece is fetched for the next head as soon as its last reading is done), the angles of the unit's
// tokens as well; the rows are normed and rotated twice, once for the block's largest magnitude and once for the codes, which
// costs less than the registers or the shared memory that fp32 rows would take.
template <int TPR, bool BF16, bool kNeox, int kFmt>
__device__ __forceinline__ void block_role(const NormRopeArgs& a, unsigned unit, bool is_k, unsigned slice, unsigned slices, float* smem, float* s_max) {
  const int tid = static_cast<int>(threadIdx.x);
  const int t = tid % TPR, rg = tid / TPR;
  const int blk = 1 << a.log_block;
  const int pairs = a.rotary_dim / 2;
  float* s_cos = smem;
  float* s_sin = smem + (pairs << a.log_block);
  float* s_norm = smem + (2 * pairs << a.log_block);             // 1 / rms of the rows of the heads at hand
  const int rows = max(1, (blk * TPR) / kThreads);               // per thread
  const int side = max(1, kThreads / (blk * TPR));               // heads side by side
  uint4* s_raw = reinterpret_cast<uint4*>(s_norm + blk * side);  // [rows][2][kThreads]
  const int b = static_cast<int>(unit / static_cast<unsigned>(a.n_touch)), j = static_cast<int>(unit - static_cast<unsigned>(b) * static_cast<unsigned>(a.n_touch));
  const Chunks<kNeox> ch(t, a.head_dim, a.rotary_dim);
  const int64_t start = a.start != nullptr ? a.start[b] : a.start_pos;
  // the j-th block of those that the valid positions of this call touch
  const int64_t p0 = start > 0 ? start : 0, p1 = min(start + a.seq, static_cast<int64_t>(a.max_len));  // positions [p0, p1)
  if (tid == 0 && j == 0 && slice == 0 && is_k && (start < 0 || start + a.seq > a.max_len))
    report(a.status, kStatusBadPosition, b, static_cast<int>(start < 0 ? start : max(start, static_cast<int64_t>(a.max_len))), a.max_len);
  const int64_t base64 = (p0 >> a.log_block << a.log_block) + static_cast<int64_t>(j) * blk;
  if (base64 >= p1) return;
  const int base = static_cast<int>(base64);
  const int lo = static_cast<int>(max(p0 - base, static_cast<int64_t>(0))), hi = static_cast<int>(min(p1 - base, static_cast<int64_t>(blk)));  // new rows of the block
  int outer, row0;
  if (!locate(a, b, base + lo, tid == 0 && is_k && slice == 0, outer, row0)) return;  // (a block lies in one page)
  row0 -= lo;

  const int sub = rg >> a.log_block;                                 // which of the heads side by side
  const int row_a = rg & (blk - 1);                                  // this lane's rows of the block: row_a, row_a + row_step, ...
  const int row_step = kThreads / TPR;
  const int n_groups = (a.n_kv_heads + side - 1) / side;
  const int g0 = static_cast<int>(static_cast<unsigned>(n_groups) * slice / slices), g1 = static_cast<int>(static_cast<unsigned>(n_groups) * (slice + 1) / slices);
  const uint8_t* src_base = reinterpret_cast<const uint8_t*>(is_k ? a.k : a.v) + 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + (base + row_a - start) * a.kv_stride[1]);
  uint8_t* cache = reinterpret_cast<uint8_t*>(is_k ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(row0) * a.cache_stride[2];
  float* scales = (is_k ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + (row0 >> a.log_block);

  auto fetch = [&](int g, int r) {
    const int h = g * side + sub, row = row_a + r * row_step;
    if (g < g1 && h < a.n_kv_heads && ch.live && row >= lo && row < hi) {
      const uint8_t* p = src_base + 2 * (static_cast<int64_t>(h) * a.kv_stride[2] + static_cast<int64_t>(r) * row_step * a.kv_stride[1]);
      cp_async_16(s_raw + (2 * r) * kThreads + tid, p + 16 * ch.c0, true);
      cp_async_16(s_raw + (2 * r + 1) * kThreads + tid, p + 16 * ch.c1, true);
    }
  };
  for (int r = 0; r < rows; ++r) fetch(g0, r);
  cp_async_commit();
  if (is_k) {
    for (int u = tid + lo * pairs; u < hi * pairs; u += kThreads) {
      const int ut = u / pairs, i = u - ut * pairs;
      const float2 cs = angle_of(a, base + ut, i);
      s_cos[u] = cs.x;
      s_sin[u] = cs.y;
    }
    __syncthreads();
  }
  const bool norm = is_k && a.k_weight != nullptr;
  float w[16];
  const uint8_t* w_now = nullptr;
  const int w_bytes = a.w_kind == 2 ? 4 : 2;
  // a row's values as they are to be coded; the first time with the row's 1 / rms found and kept
  auto row_values = [&](int r, bool again, float (&x)[16]) {
    const int row = row_a + r * row_step;
    const bool mine = row >= lo && row < hi;
    uint4 raw0 = make_uint4(0, 0, 0, 0), raw1 = raw0;
    if (mine && ch.live) {
      raw0 = s_raw[(2 * r) * kThreads + tid];
      raw1 = s_raw[(2 * r + 1) * kThreads + tid];
    }
    unpack8<BF16>(raw0, x);
    unpack8<BF16>(raw1, x + 8);
    if (!is_k) return;
    if (norm) {
      float* kept = s_norm + sub * blk + row;
      float f;
      if (again) {
        f = *kept;
      } else {
        f = inverse_rms<TPR>(x, ch.live, a.inv_dim, a.eps);
        if (t == 0) *kept = f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] *= f * w[i];
    }
    if (mine) {
      float cs[8], sn[8];
      load_angles<kNeox>(s_cos + row * pairs, s_sin + row * pairs, ch, cs, sn);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if ((!kNeox && p >= 4) ? ch.rot1 : ch.rot0) {
          const float u = x[pair_lo<kNeox>(p)], v = x[pair_hi<kNeox>(p)];
          x[pair_lo<kNeox>(p)] = fmaf(u, cs[p], -(v * sn[p]));
          x[pair_hi<kNeox>(p)] = fmaf(u, sn[p], v * cs[p]);
        }
      }
    }
  };
  for (int g = g0; g < g1; ++g) {
    const int h = g * side + sub;
    const bool head_ok = h < a.n_kv_heads;
    if (norm) {
      const uint8_t* wp = reinterpret_cast<const uint8_t*>(a.k_weight) + static_cast<int64_t>(head_ok ? h : 0) * a.w_stride[1] * w_bytes;
      if (wp != w_now) load_weights(wp, a.w_kind, ch.c0, ch.c1, w);
      w_now = wp;
    }
    const float s0 = (head_ok && lo != 0) ? scales[static_cast<int64_t>(h) * a.scale_stride[1]] : 0.f;
    cp_async_wait<0>();
    float amax = 0.f;
    for (int r = 0; r < rows; ++r) {
      float x[16];
      row_values(r, false, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[i]));  // (rows that are not new: zeros)
    }
    // over the lanes that hold this head's rows: a warp's lanes, then the group's warps
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
    float* part = s_max + (g & 1) * (kThreads / 32);  // two sets: one barrier per head
    if ((tid & 31) == 0) part[tid >> 5] = amax;
    __syncthreads();
    {
      const int group_warps = min(kThreads, blk * TPR) / 32;
      const int w0 = (tid >> 5) / group_warps * group_warps;
      for (int i = 0; i < group_warps; ++i) amax = fmaxf(amax, part[w0 + i]);
    }
    const float need = b8_scale<kFmt>(amax);
    const float s1 = s0 >= need ? s0 : need;
    const float r1 = b8_inverse(s1);
    uint8_t* dst = cache + static_cast<int64_t>(h) * a.cache_stride[1];
    for (int r = 0; r < rows; ++r) {
      const int row = row_a + r * row_step;
      float x[16];
      row_values(r, true, x);
      fetch(g + 1, r);
      if (!head_ok || !ch.live) continue;
      uint8_t* d = dst + static_cast<int64_t>(row) * a.cache_stride[2];
      if (row >= lo && row < hi) {
        *reinterpret_cast<uint2*>(d + 8 * ch.c0) = b8_code8<kFmt>(x, s1, r1);
        *reinterpret_cast<uint2*>(d + 8 * ch.c1) = b8_code8<kFmt>(x + 8, s1, r1);
      } else if (row < lo && s1 != s0) {  // rows that were there, under a scale that grew
        uint2* d0 = reinterpret_cast<uint2*>(d + 8 * ch.c0);
        uint2* d1 = reinterpret_cast<uint2*>(d + 8 * ch.c1);
        const uint2 y0 = *d0, y1 = *d1;
        *d0 = b8_recode8<kFmt>(y0, s0, s1, r1);
        *d1 = b8_recode8<kFmt>(y1, s0, s1, r1);
      }
    }
    cp_async_commit();
    // one lane of the head's group
    if (head_ok && t == 0 && row_a == 0 && (lo == 0 || s1 != s0)) scales[static_cast<int64_t>(h) * a.scale_stride[1]] = s1;
  }
}

// Blocks [0, kv_blocks): units of k, then of v; behind them the query rows.
template <int TPR, bool BF16, bool kNeox, int kFmt>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_blocks_kernel(const NormRopeArgs a) {
  extern __shared__ __align__(16) float s_dyn[];
  __shared__ float s_max[2 * kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const unsigned per = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.n_touch) * static_cast<unsigned>(a.slices);  // blocks of k, and of v
  if (blockIdx.x < 2 * per) {
    const bool is_k = blockIdx.x < per;
    const unsigned i = is_k ? blockIdx.x : blockIdx.x - per;
    block_role<TPR, BF16, kNeox, kFmt>(a, i / static_cast<unsigned>(a.slices), is_k, i % static_cast<unsigned>(a.slices), static_cast<unsigned>(a.slices), s_dyn, s_max);
  } else {
    rows_role<TPR, BF16, kNeox, 0>(a, blockIdx.x - 2 * per, 0, 1, 0, 0, s_dyn);
  }
}

// frequencies in turns: base ^ (-2 i / rotary_dim) / (2 pi), modulo 1 (positions are whole numbers), as fractions of 2^64
void fill_turns(NormRopeArgs& a, double freq_base) {
  thread_local double cached_base = 0.0;
  thread_local int cached_rot = -1;
  thread_local uint64_t table[128];
  if (cached_base != freq_base || cached_rot != a.rotary_dim) {
    const long double two_pi = 6.283185307179586476925286766559005768L;
    for (int i = 0; i < 128; ++i) {
      if (i >= a.rotary_dim / 2) {
        table[i] = 0;
        continue;
      }
      long double f = std::pow(static_cast<long double>(freq_base), -2.0L * i / a.rotary_dim) / two_pi;
      f -= std::floor(f);
      const long double x = std::ldexp(f, 64);
      table[i] = x >= 18446744073709551615.0L ? 0 : static_cast<uint64_t>(x);
    }
    cached_base = freq_base;
    cached_rot = a.rotary_dim;
  }
  for (int i = 0; i < 128; ++i) a.turns[i] = table[i];
}

template <int TPR, bool BF16, bool kNeox, int kFmt>
cudaError_t launch_rows(const NormRopeArgs& a, unsigned blocks, unsigned slices, cudaStream_t stream) {
  LaunchAttrs at(stream);
  at.cfg.gridDim = dim3(blocks, slices);
  at.cfg.blockDim = dim3(kThreads);
  return cudaLaunchKernelEx(&at.cfg, norm_rope_rows_kernel<TPR, BF16, kNeox, kFmt>, a);
}

template <int TPR, bool BF16, bool kNeox, int kFmt>
cudaError_t launch_blocks(const NormRopeArgs& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  auto* kernel = norm_rope_blocks_kernel<TPR, BF16, kNeox, kFmt>;
  if (smem > 48 * 1024) {
    // (idempotent, and some hundred nanoseconds beside a call of many tokens)
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  LaunchAttrs at(stream);
  at.cfg.gridDim = dim3(blocks);
  at.cfg.blockDim = dim3(kThreads);
  at.cfg.dynamicSmemBytes = smem;
  return cudaLaunchKernelEx(&at.cfg, kernel, a);
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeArgs& a_in, bool bf16, bool neox, int cache_format, double freq_base, cudaStream_t stream) {
  NormRopeArgs a = a_in;
  fill_turns(a, freq_base);
  a.inv_dim = 1.0f / static_cast<float>(a.head_dim);
  const int tpr = a.head_dim <= 64 ? 4 : a.head_dim <= 128 ? 8 : 16;
  const int groups = kThreads / tpr;
  const long long tokens = static_cast<long long>(a.batch) * a.seq;
  const int fmt = cache_format == MINFER_ATTN_KV_E4M3 ? kE4M3 : cache_format == MINFER_ATTN_KV_INT8 ? kInt8 : 0;
  const bool by_block = fmt != 0 && a.seq > 1;
  const int n_kv = by_block ? 0 : (a.k != nullptr ? a.n_kv_heads : 0) + (a.v != nullptr ? a.n_kv_heads : 0);
  const int n_rows = (a.q != nullptr ? a.n_heads : 0) + n_kv;
  // Tokens per block: more share the block's set-up, fewer fill the GPU.
  a.log_tb = 0;
  const int max_tb = a.rotary_dim > 0 ? kMaxAngles / (a.rotary_dim / 2) : groups;
  while ((4 << a.log_tb) <= groups && (2 << a.log_tb) <= max_tb && (tokens >> (a.log_tb + 1)) >= 4 * 148) ++a.log_tb;
  const long long blocks_x = (tokens + (1 << a.log_tb) - 1) >> a.log_tb;
#define MINFER_NR_STYLE(fn, TPR, F, ...) \
  (bf16 ? (neox ? fn<TPR, true, true, F>(__VA_ARGS__) : fn<TPR, true, false, F>(__VA_ARGS__)) \
        : (neox ? fn<TPR, false, true, F>(__VA_ARGS__) : fn<TPR, false, false, F>(__VA_ARGS__)))
  if (!by_block) {
    // few tokens: a token's rows over several blocks, one row per group
    long long slices = 1;
    if (a.log_tb == 0) {
      slices = (n_rows + groups - 1) / groups;
      if (slices * blocks_x > 8 * 148) slices = (8 * 148 + blocks_x - 1) / blocks_x;
      if (slices < 1) slices = 1;
    }
    const unsigned bx = static_cast<unsigned>(blocks_x), sl = static_cast<unsigned>(slices);
    if (fmt == 0) {
      if (tpr == 4) return MINFER_NR_STYLE(launch_rows, 4, 0, a, bx, sl, stream);
      if (tpr == 8) return MINFER_NR_STYLE(launch_rows, 8, 0, a, bx, sl, stream);
      return MINFER_NR_STYLE(launch_rows, 16, 0, a, bx, sl, stream);
    }
    if (fmt == kE4M3) return tpr == 4 ? MINFER_NR_STYLE(launch_rows, 4, kE4M3, a, bx, sl, stream) : MINFER_NR_STYLE(launch_rows, 8, kE4M3, a, bx, sl, stream);
    return tpr == 4 ? MINFER_NR_STYLE(launch_rows, 4, kInt8, a, bx, sl, stream) : MINFER_NR_STYLE(launch_rows, 8, kInt8, a, bx, sl, stream);
  }
  const int blk = 1 << a.log_block;
  a.n_touch = (a.seq + blk - 2) / blk + 1;
  const long long units = static_cast<long long>(a.batch) * a.n_touch;
  const int side = (tpr << a.log_block) < kThreads ? kThreads / (tpr << a.log_block) : 1;  // heads side by side
  const int head_groups = (a.n_kv_heads + side - 1) / side;
  // heads of a unit over several blocks while the GPU is not full
  long long slices = (4 * 148 + units - 1) / units;
  if (slices > head_groups) slices = head_groups;
  if (slices < 1) slices = 1;
  a.slices = static_cast<int>(slices);
  const long long blocks = 2 * units * slices + (a.q != nullptr ? blocks_x : 0);
  if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  // angles, 1 / rms, raw rows
  size_t smem = static_cast<size_t>(a.rotary_dim / 2) * blk * 8 + static_cast<size_t>(blk) * side * 4 +
                static_cast<size_t>((tpr << a.log_block) > kThreads ? tpr << a.log_block : kThreads) * 32;
  if (a.q != nullptr && smem < kRowsSmem) smem = kRowsSmem;
  const unsigned nb = static_cast<unsigned>(blocks);
  if (fmt == kE4M3) return tpr == 4 ? MINFER_NR_STYLE(launch_blocks, 4, kE4M3, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks, 8, kE4M3, a, nb, smem, stream);
  return tpr == 4 ? MINFER_NR_STYLE(launch_blocks, 4, kInt8, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks, 8, kInt8, a, nb, smem, stream);
#undef MINFER_NR_STYLE
}

}  // namespace minfer_attn
