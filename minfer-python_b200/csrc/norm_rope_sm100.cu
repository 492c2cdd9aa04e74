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
constexpr int kMaxAngles = 1024;  // (token, pair) angles a block keeps in shared memory

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

// y = x / rms(x) * weight over the TPR lanes of a row (called by whole warps)
template <int TPR>
__device__ __forceinline__ void norm_row(float* x, const float* w, bool live, float inv_dim, float eps) {
  float ss = 0.f;
  if (live) {
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = fmaf(x[i], x[i], ss);
  }
#pragma unroll
  for (int d = TPR / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
  const float r = rsqrtf(fmaf(ss, inv_dim, eps));
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] *= r * w[i];
}

template <bool kNeox>
__device__ __forceinline__ void rotate_row(float* x, const Chunks<kNeox>& ch, const float* cs, const float* sn) {
  if constexpr (kNeox) {
    if (ch.rot0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float u = x[i], v = x[8 + i];
        x[i] = u * cs[i] - v * sn[i];
        x[8 + i] = u * sn[i] + v * cs[i];
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h ? ch.rot1 : ch.rot0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u = x[8 * h + 2 * i], v = x[8 * h + 2 * i + 1];
          x[8 * h + 2 * i] = u * cs[4 * h + i] - v * sn[4 * h + i];
          x[8 * h + 2 * i + 1] = u * sn[4 * h + i] + v * cs[4 * h + i];
        }
      }
    }
  }
}

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
// A block takes 2^log_tb tokens; each token's rows are dealt out over the row groups it gets (and over `slices` blocks).
template <int TPR, bool BF16, bool kNeox, int kFmt>
__device__ __forceinline__ void rows_role(const NormRopeArgs& a, unsigned bx, unsigned slice, unsigned slices, int n_k, int n_v,
                                          float* s_cos, float* s_sin) {
  constexpr int kGroups = kThreads / TPR;
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
  const uint8_t* q_base = reinterpret_cast<const uint8_t*>(a.q) + 2 * (static_cast<int64_t>(b) * a.q_stride[0] + static_cast<int64_t>(l) * a.q_stride[1]);
  const int64_t kv_off = 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + static_cast<int64_t>(l) * a.kv_stride[1]);
  const int step = static_cast<int>(slices) << log_gpt;
  const int first = (static_cast<int>(slice) << log_gpt) + (rg & ((1 << log_gpt) - 1));
  auto row_at = [&](int r, int& kind, int& h) -> const uint8_t* {
    if (r < n_q) {
      kind = 0;
      h = r;
      return q_base + 2 * static_cast<int64_t>(h) * a.q_stride[2];
    }
    kind = r < n_q + n_k ? 1 : 2;
    h = r - n_q - (kind == 2 ? n_k : 0);
    return reinterpret_cast<const uint8_t*>(kind == 1 ? a.k : a.v) + kv_off + 2 * static_cast<int64_t>(h) * a.kv_stride[2];
  };
  // (all row groups of a block make the same number of steps, so that warps stay whole)
  const int n_steps = n_rows > static_cast<int>(slice << log_gpt) ? (n_rows - static_cast<int>(slice << log_gpt) + step - 1) / step : 0;
  uint4 raw0 = make_uint4(0, 0, 0, 0), raw1 = raw0;
  int kind = 0, h = 0;
  const uint8_t* src = nullptr;
  auto fetch = [&](int r) {
    src = nullptr;
    if (token_ok && r < n_rows) {
      src = row_at(r, kind, h);
      if (ch.live) {
        raw0 = *reinterpret_cast<const uint4*>(src + 16 * ch.c0);
        raw1 = *reinterpret_cast<const uint4*>(src + 16 * ch.c1);
      }
    }
  };
  fetch(first);  // on its way before the position is known

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
  float cs[8], sn[8];
  load_angles<kNeox>(s_cos + tb * pairs, s_sin + tb * pairs, ch, cs, sn);

  float w[16];
  const uint8_t* w_now = nullptr;
  const int w_bytes = a.w_kind == 2 ? 4 : 2;
  for (int it = 0; it < n_steps; ++it) {
    const int kd = kind, hh = h;
    const uint8_t* sp = src;
    float x[16];
    unpack8<BF16>(raw0, x);
    unpack8<BF16>(raw1, x + 8);
    const uint4 v0 = raw0, v1 = raw1;
    if (it + 1 < n_steps) fetch(first + (it + 1) * step);
    if (a.q_weight != nullptr) {
      if (sp != nullptr && kd != 2) {
        const uint8_t* wp = kd == 0 ? reinterpret_cast<const uint8_t*>(a.q_weight) + static_cast<int64_t>(hh) * a.w_stride[0] * w_bytes
                                    : reinterpret_cast<const uint8_t*>(a.k_weight) + static_cast<int64_t>(hh) * a.w_stride[1] * w_bytes;
        if (wp != w_now) load_weights(wp, a.w_kind, ch.c0, ch.c1, w);
        w_now = wp;
      }
      // (rows of v and idle groups take part in the shuffles of their warp)
      float y[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) y[i] = x[i];
      norm_row<TPR>(y, w, ch.live, a.inv_dim, a.eps);
      if (kd != 2) {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = y[i];
      }
    }
    if (kd != 2) rotate_row<kNeox>(x, ch, cs, sn);
    if constexpr (kFmt == 0) {
      if (sp == nullptr || !ch.live) continue;
      uint8_t* dst = const_cast<uint8_t*>(sp);
      if (kd != 0 && a.k_cache != nullptr) {
        if (!cache_ok) continue;
        dst = reinterpret_cast<uint8_t*>(kd == 1 ? a.k_cache : a.v_cache) +
              2 * (static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(hh) * a.cache_stride[1] + static_cast<int64_t>(crow) * a.cache_stride[2]);
      }
      *reinterpret_cast<uint4*>(dst + 16 * ch.c0) = kd == 2 ? v0 : pack8<BF16>(x);
      *reinterpret_cast<uint4*>(dst + 16 * ch.c1) = kd == 2 ? v1 : pack8<BF16>(x + 8);
    } else {
      if (sp != nullptr && kd == 0 && ch.live) {
        *reinterpret_cast<uint4*>(const_cast<uint8_t*>(sp) + 16 * ch.c0) = pack8<BF16>(x);
        *reinterpret_cast<uint4*>(const_cast<uint8_t*>(sp) + 16 * ch.c1) = pack8<BF16>(x + 8);
      }
      const bool cached = sp != nullptr && kd != 0 && cache_ok;
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
        float* sc = (kd == 1 ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + static_cast<int64_t>(hh) * a.scale_stride[1] + (crow >> a.log_block);
        blk_rows = reinterpret_cast<uint8_t*>(kd == 1 ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] +
                   static_cast<int64_t>(hh) * a.cache_stride[1] + static_cast<int64_t>(crow - begun) * a.cache_stride[2];
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
__global__ void __launch_bounds__(kThreads, TPR == 16 ? 2 : 3) norm_rope_rows_kernel(const NormRopeArgs a) {
  __shared__ __align__(16) float s_cos[kMaxAngles];
  __shared__ __align__(16) float s_sin[kMaxAngles];
  grid_launch_dependents();
  grid_dependency_wait();
  rows_role<TPR, BF16, kNeox, kFmt>(a, blockIdx.x, blockIdx.y, gridDim.y, a.k != nullptr ? a.n_kv_heads : 0,
                                    a.v != nullptr ? a.n_kv_heads : 0, s_cos, s_sin);
}

// ---- blocks of an 8-bit cache: k and v of calls with several tokens per sequence ----
//
// A unit is one block of tokens of one sequence, for a slice of the kv heads, of k or of v: its rows are loaded, normed and rotated
// into registers (fp32), the block's largest magnitude is agreed on, and the codes leave.  A head's rows of one block fill 2^log_block * TPR
// lanes: four, two or one head at a time (kRows = 1), or two or four rows per thread.  The angles of a unit's tokens lie in
// shared memory and serve all its heads.
template <int TPR, bool BF16, bool kNeox, int kFmt, int kRows>
__device__ __forceinline__ void block_role(const NormRopeArgs& a, unsigned unit, bool is_k, unsigned slice, unsigned slices, float* s_cos, float* s_sin,
                                           float* s_max) {
  const int tid = static_cast<int>(threadIdx.x);
  const int t = tid % TPR, rg = tid / TPR;
  const int blk = 1 << a.log_block;
  const int b = static_cast<int>(unit / static_cast<unsigned>(a.n_touch)), j = static_cast<int>(unit - static_cast<unsigned>(b) * static_cast<unsigned>(a.n_touch));
  const Chunks<kNeox> ch(t, a.head_dim, a.rotary_dim);
  const int64_t start = a.start != nullptr ? a.start[b] : a.start_pos;
  // the j-th block of those that the valid positions of this call touch
  const int64_t p0 = start > 0 ? start : 0, p1 = min(start + a.seq, static_cast<int64_t>(a.max_len));  // positions [p0, p1)
  if (tid == 0 && j == 0 && slice == 0 && is_k && (start < 0 || start + a.seq > a.max_len))
    report(a.status, kStatusBadPosition, b, static_cast<int>(start < 0 ? start : start + a.seq - 1 > 0x7FFFFFFF ? 0x7FFFFFFF : max(start, static_cast<int64_t>(a.max_len))), a.max_len);
  const int64_t base64 = (p0 >> a.log_block << a.log_block) + static_cast<int64_t>(j) * blk;
  if (base64 >= p1) return;
  const int base = static_cast<int>(base64);
  const int lo = static_cast<int>(max(p0 - base, static_cast<int64_t>(0))), hi = static_cast<int>(min(p1 - base, static_cast<int64_t>(blk)));  // new rows of the block
  int outer, row0;
  if (!locate(a, b, base + lo, tid == 0 && is_k && slice == 0, outer, row0)) return;  // (a block lies in one page)
  row0 -= lo;

  const int per_row_heads = kRows > 1 ? 1 : kThreads / (blk * TPR);  // heads side by side
  const int sub = kRows > 1 ? 0 : rg >> a.log_block;                 // which of them
  const int row_a = kRows > 1 ? rg * kRows : rg & (blk - 1);         // this lane's first row of the block
  // heads of the slice
  const int n_groups = (a.n_kv_heads + per_row_heads - 1) / per_row_heads;
  const int g0 = static_cast<int>(static_cast<unsigned>(n_groups) * slice / slices), g1 = static_cast<int>(static_cast<unsigned>(n_groups) * (slice + 1) / slices);
  const uint8_t* src_base = reinterpret_cast<const uint8_t*>(is_k ? a.k : a.v) + 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + (base + row_a - start) * a.kv_stride[1]);
  uint8_t* cache = reinterpret_cast<uint8_t*>(is_k ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(row0) * a.cache_stride[2];
  float* scales = (is_k ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + (row0 >> a.log_block);

  uint4 raw[kRows][2];
  float s_old = 0.f;
  auto fetch = [&](int g) {
    const int h = g * per_row_heads + sub;
    if (h < a.n_kv_heads) {
      const uint8_t* p = src_base + 2 * static_cast<int64_t>(h) * a.kv_stride[2];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        raw[r][0] = raw[r][1] = make_uint4(0, 0, 0, 0);
        if (ch.live && row_a + r >= lo && row_a + r < hi) {
          const uint8_t* q = p + 2 * static_cast<int64_t>(r) * a.kv_stride[1];
          raw[r][0] = *reinterpret_cast<const uint4*>(q + 16 * ch.c0);
          raw[r][1] = *reinterpret_cast<const uint4*>(q + 16 * ch.c1);
        }
      }
      s_old = lo != 0 ? scales[static_cast<int64_t>(h) * a.scale_stride[1]] : 0.f;
    }
  };
  if (g0 < g1) fetch(g0);
  const int pairs = a.rotary_dim / 2;
  if (is_k) {
    for (int u = tid + lo * pairs; u < hi * pairs; u += kThreads) {
      const int ut = u / pairs, i = u - ut * pairs;
      const float2 cs = angle_of(a, base + ut, i);
      s_cos[u] = cs.x;
      s_sin[u] = cs.y;
    }
    __syncthreads();
  }
  float w[16];
  const uint8_t* w_now = nullptr;
  const int w_bytes = a.w_kind == 2 ? 4 : 2;
  for (int g = g0; g < g1; ++g) {
    const int h = g * per_row_heads + sub;
    const bool head_ok = h < a.n_kv_heads;
    float x[kRows][16];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      unpack8<BF16>(raw[r][0], x[r]);
      unpack8<BF16>(raw[r][1], x[r] + 8);
    }
    const float s0 = s_old;
    if (g + 1 < g1) fetch(g + 1);
    float amax = 0.f;
    if (is_k && a.k_weight != nullptr) {
      const uint8_t* wp = reinterpret_cast<const uint8_t*>(a.k_weight) + static_cast<int64_t>(head_ok ? h : 0) * a.w_stride[1] * w_bytes;
      if (wp != w_now) load_weights(wp, a.w_kind, ch.c0, ch.c1, w);
      w_now = wp;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (is_k) {
        if (a.k_weight != nullptr) norm_row<TPR>(x[r], w, ch.live, a.inv_dim, a.eps);
        if (row_a + r >= lo && row_a + r < hi) {
          float cs[8], sn[8];
          load_angles<kNeox>(s_cos + (row_a + r) * pairs, s_sin + (row_a + r) * pairs, ch, cs, sn);
          rotate_row<kNeox>(x[r], ch, cs, sn);
        }
      }
      if (row_a + r >= lo && row_a + r < hi) {
#pragma unroll
        for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(x[r][i]));
      }
    }
    // over the lanes that hold this head's rows: a warp's lanes, then the group's warps
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
    const int group_warps = kRows > 1 ? kThreads / 32 : (blk * TPR) / 32;
    float* mine = s_max + (g & 1) * (kThreads / 32);  // two sets: one barrier per head
    if ((tid & 31) == 0) mine[tid >> 5] = amax;
    __syncthreads();
    {
      const int w0 = (tid >> 5) / group_warps * group_warps;
      for (int i = 0; i < group_warps; ++i) amax = fmaxf(amax, mine[w0 + i]);
    }
    if (!head_ok || !ch.live) continue;
    const float need = b8_scale<kFmt>(amax);
    const float s1 = s0 >= need ? s0 : need;
    const float r1 = b8_inverse(s1);
    uint8_t* dst = cache + static_cast<int64_t>(h) * a.cache_stride[1];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int row = row_a + r;
      uint8_t* d = dst + static_cast<int64_t>(row) * a.cache_stride[2];
      if (row >= lo && row < hi) {
        *reinterpret_cast<uint2*>(d + 8 * ch.c0) = b8_code8<kFmt>(x[r], s1, r1);
        *reinterpret_cast<uint2*>(d + 8 * ch.c1) = b8_code8<kFmt>(x[r] + 8, s1, r1);
      } else if (row < lo && s1 != s0) {  // rows that were there, under a scale that grew
        uint2* d0 = reinterpret_cast<uint2*>(d + 8 * ch.c0);
        uint2* d1 = reinterpret_cast<uint2*>(d + 8 * ch.c1);
        const uint2 y0 = *d0, y1 = *d1;
        *d0 = b8_recode8<kFmt>(y0, s0, s1, r1);
        *d1 = b8_recode8<kFmt>(y1, s0, s1, r1);
      }
    }
    // one lane of the head's group
    if (t == 0 && (kRows > 1 ? rg == 0 : (rg & (blk - 1)) == 0) && (lo == 0 || s1 != s0)) scales[static_cast<int64_t>(h) * a.scale_stride[1]] = s1;
  }
}

// Blocks [0, kv_blocks): units of k, then of v; behind them the query rows.
template <int TPR, bool BF16, bool kNeox, int kFmt, int kRows>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_blocks_kernel(const NormRopeArgs a) {
  extern __shared__ __align__(16) float s_angles[];
  __shared__ float s_max[2 * kThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const unsigned units = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.n_touch);
  const unsigned kv_blocks = 2u * units * static_cast<unsigned>(a.slices);
  if (blockIdx.x < kv_blocks) {
    const unsigned per = units * static_cast<unsigned>(a.slices);
    const bool is_k = blockIdx.x < per;
    const unsigned i = is_k ? blockIdx.x : blockIdx.x - per;
    float* s_sin = s_angles + (a.rotary_dim / 2 << a.log_block);
    block_role<TPR, BF16, kNeox, kFmt, kRows>(a, i / static_cast<unsigned>(a.slices), is_k, i % static_cast<unsigned>(a.slices), static_cast<unsigned>(a.slices),
                                              s_angles, s_sin, s_max);
  } else {
    rows_role<TPR, BF16, kNeox, 0>(a, blockIdx.x - kv_blocks, 0, 1, 0, 0, s_angles, s_angles + kMaxAngles);
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

template <int TPR, bool BF16, bool kNeox, int kFmt, int kRows>
cudaError_t launch_blocks(const NormRopeArgs& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  auto* kernel = norm_rope_blocks_kernel<TPR, BF16, kNeox, kFmt, kRows>;
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

template <int TPR, bool BF16, bool kNeox, int kFmt>
cudaError_t launch_blocks_rows(const NormRopeArgs& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  const int lanes = TPR << a.log_block;
  if (lanes <= kThreads) return launch_blocks<TPR, BF16, kNeox, kFmt, 1>(a, blocks, smem, stream);
  if (lanes == 2 * kThreads) return launch_blocks<TPR, BF16, kNeox, kFmt, 2>(a, blocks, smem, stream);
  if constexpr (TPR == 8) return launch_blocks<TPR, BF16, kNeox, kFmt, 4>(a, blocks, smem, stream);
  return cudaErrorInvalidValue;
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
  size_t smem = static_cast<size_t>(a.rotary_dim / 2) * blk * 8;
  if (smem < 2 * kMaxAngles * sizeof(float)) smem = 2 * kMaxAngles * sizeof(float);
  const unsigned nb = static_cast<unsigned>(blocks);
  if (fmt == kE4M3) return tpr == 4 ? MINFER_NR_STYLE(launch_blocks_rows, 4, kE4M3, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks_rows, 8, kE4M3, a, nb, smem, stream);
  return tpr == 4 ? MINFER_NR_STYLE(launch_blocks_rows, 4, kInt8, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks_rows, 8, kInt8, a, nb, smem, stream);
#undef MINFER_NR_STYLE
}

}  // namespace minfer_attn
