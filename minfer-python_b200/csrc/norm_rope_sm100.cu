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
//
// Measured (32 / 8 heads, D=128, 4 x 4096 tokens, back to back): 16-bit cache 64.4 us, 6.3 TB/s, 0.97 of what a copy reaches; 8-bit cache (e4m3,
// blocks of 128) 71.8 us, 5.1 TB/s, with norms 83 us, bound by issue slots (56 % busy) and latency at 16 warps per SM; single tokens of 64 sequences 3.1 and
// 3.2-3.4 us, launch and latency.
#include "../../include/minfer_attn.h"
#include "attn_internal.h"
#include "b8.cuh"
#include "ptx.cuh"

#include <cmath>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace minfer_attn {

namespace {

constexpr int kRowThreads = 128;    // a block that works on rows
constexpr int kThreads = 256;       // a block that works on blocks of a cache (and, behind those, on rows)
constexpr int kMaxPairs = 128;      // rotated pairs of a head
// Rows per thread in a step of rows_role - two give two independent chains; the rows of an 8-bit cache need the registers for their codes -
// and steps on their way through shared memory (no registers held while they fly).
constexpr int rows_per_step(int fmt) { return fmt == 0 ? 2 : 1; }
constexpr int ring_stages(int rows) { return rows == 1 ? 4 : 3; }
constexpr int rows_smem(int threads, int rows) { return ring_stages(rows) * 2 * rows * threads * static_cast<int>(sizeof(uint4)); }

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

// cos and sin of pair i at a position.  The table is read from shared memory: in the kernel's arguments, lanes that want
// different entries would be served one after another.  The nearest quarter turn is split off in integers, so that what is rounded to fp32 is an
// eighth of a turn at most: a whole half turn would be rounded by up to pi 2^-25, several times what cos and sin themselves are.
__device__ __forceinline__ float2 angle_of(const uint64_t* s_turns, int pos, int i) {
  const uint64_t turns = static_cast<uint64_t>(static_cast<int64_t>(pos)) * s_turns[i];
  const uint32_t hi = static_cast<uint32_t>(turns >> 32);
  const uint32_t quarters = (hi + 0x20000000u) >> 30;
  float s, c;
  sincospif(static_cast<float>(static_cast<int32_t>(hi - (quarters << 30))) * 4.656612873077392578125e-10f, &s, &c);  // 2^-31: half turns
  const float x = (quarters & 1u) ? s : c, y = (quarters & 1u) ? c : s;
  return make_float2(((quarters + 1u) & 2u) ? -x : x, (quarters & 2u) ? -y : y);
}

template <int kT>
__device__ __forceinline__ void copy_turns(const NormRopeArgs& a, uint64_t* s_turns) {
  for (int u = static_cast<int>(threadIdx.x); u < kMaxPairs; u += kT) s_turns[u] = a.turns[u];
  __syncthreads();
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

// A lane's 16 values of a row as eight pairs (lo, hi): two halves (x[p], x[8 + p]), interleaved (x[2 p], x[2 p + 1]) with pairs 0-3 in
// chunk c0 and 4-7 in chunk c1; two pairs to a register pair, so that the arithmetic goes two values at a time.
struct Pairs {
  float2 lo[4], hi[4];
};

template <bool kNeox>
__device__ __forceinline__ Pairs as_pairs(const float* x) {
  Pairs r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.lo[i] = kNeox ? make_float2(x[2 * i], x[2 * i + 1]) : make_float2(x[4 * i], x[4 * i + 2]);
    r.hi[i] = kNeox ? make_float2(x[8 + 2 * i], x[9 + 2 * i]) : make_float2(x[4 * i + 1], x[4 * i + 3]);
  }
  return r;
}
template <bool kNeox>
__device__ __forceinline__ void as_values(const Pairs& r, float* x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[kNeox ? 2 * i : 4 * i] = r.lo[i].x;
    x[kNeox ? 2 * i + 1 : 4 * i + 2] = r.lo[i].y;
    x[kNeox ? 8 + 2 * i : 4 * i + 1] = r.hi[i].x;
    x[kNeox ? 9 + 2 * i : 4 * i + 3] = r.hi[i].y;
  }
}

// 1 / rms of a row, over its TPR lanes (called by whole warps; lanes without a chunk hold zeros)
template <int TPR>
__device__ __forceinline__ float inverse_rms(const Pairs& x, float inv_dim, float eps) {
  float2 s = __fmul2_rn(x.lo[0], x.lo[0]), u = __fmul2_rn(x.hi[0], x.hi[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    s = __ffma2_rn(x.lo[i], x.lo[i], s);
    u = __ffma2_rn(x.hi[i], x.hi[i], u);
  }
  s = __fadd2_rn(s, u);
  float ss = s.x + s.y;
#pragma unroll
  for (int d = TPR / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
  return rsqrtf(fmaf(ss, inv_dim, eps));
}

__device__ __forceinline__ void scale_pairs(Pairs& x, float f) {
  const float2 f2 = make_float2(f, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.lo[i] = __fmul2_rn(x.lo[i], f2);
    x.hi[i] = __fmul2_rn(x.hi[i], f2);
  }
}

// A lane's angles; pairs that are not rotated are left out by apply_angles, not turned by 0 (an infinite value stays in its place).
struct Angles {
  float2 c[4], s[4];  // cos, sin
};

// t - x * y: two scalar fmas, which negate for nothing.  Negated sines in registers and one packed fma instead made most of these kernels spill (norms, 4 x 4096 tokens,
// bfloat16, two halves: 16-bit cache 72.9 us, now 64.6).
__device__ __forceinline__ float2 minus_product(const float2& x, const float2& y, const float2& t) {
  return make_float2(fmaf(-x.x, y.x, t.x), fmaf(-x.y, y.y, t.y));
}

template <bool kNeox>
__device__ __forceinline__ void apply_angles(Pairs& x, const Angles& g, const Chunks<kNeox>& ch) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if ((!kNeox && i >= 2) ? ch.rot1 : ch.rot0) {
      const float2 lo = x.lo[i], hi = x.hi[i];
      x.lo[i] = minus_product(hi, g.s[i], __fmul2_rn(lo, g.c[i]));
      x.hi[i] = __ffma2_rn(lo, g.s[i], __fmul2_rn(hi, g.c[i]));
    }
  }
}

template <bool kNeox>
__device__ __forceinline__ Pairs weight_pairs(const void* w, int w_kind, const Chunks<kNeox>& ch) {
  float f[16];
  load_weights(w, w_kind, ch.c0, ch.c1, f);
  return as_pairs<kNeox>(f);
}

// x * f * weight
__device__ __forceinline__ void apply_weights(Pairs& x, const Pairs& w, float f) {
  scale_pairs(x, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x.lo[i] = __fmul2_rn(x.lo[i], w.lo[i]);
    x.hi[i] = __fmul2_rn(x.hi[i], w.hi[i]);
  }
}

// the lane's eight angles out of a token's rows of cosines and sines
template <bool kNeox>
__device__ __forceinline__ void load_angles(const float* cosines, const float* sines, const Chunks<kNeox>& ch, Angles& g) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h ? ch.rot1 : ch.rot0) {
      const float4 c = *reinterpret_cast<const float4*>(cosines + (h ? ch.i1 : ch.i0)), s = *reinterpret_cast<const float4*>(sines + (h ? ch.i1 : ch.i0));
      g.c[2 * h] = make_float2(c.x, c.y);
      g.c[2 * h + 1] = make_float2(c.z, c.w);
      g.s[2 * h] = make_float2(s.x, s.y);
      g.s[2 * h + 1] = make_float2(s.z, s.w);
    }
  }
}

// The same computed by a warp whose row groups all work for one token: each group takes its share of a lane's eight angles.
template <int TPR, bool kNeox>
__device__ __forceinline__ void warp_angles(const uint64_t* s_turns, int pos, const Chunks<kNeox>& ch, int t, int group, Angles& g) {
  constexpr int kShare = 8 / (32 / TPR);  // angles per group: 1, 2 or 4
  float2 mine[kShare];
#pragma unroll
  for (int u = 0; u < kShare; ++u) {
    const int p = group * kShare + u;
    const int i = p < 4 ? ch.i0 + p : ch.i1 + p - 4;
    mine[u] = angle_of(s_turns, pos, min(i, kMaxPairs - 1));  // (lanes and pairs beyond rotary_dim: some angle that nobody uses)
  }
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int from = (p / kShare) * TPR + t;
    const float c = __shfl_sync(0xFFFFFFFFu, mine[p % kShare].x, from), s = __shfl_sync(0xFFFFFFFFu, mine[p % kShare].y, from);
    if (p & 1) {
      g.c[p / 2].y = c;
      g.s[p / 2].y = s;
    } else {
      g.c[p / 2].x = c;
      g.s[p / 2].x = s;
    }
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
// A warp takes a token (or, with few tokens, one of `slices` shares of its rows): nothing is shared between warps, no barrier.  Its
// 32 / TPR row groups walk the query heads, the k heads and the v heads side by side, kR rows each per step (two independent chains
// of reduction and arithmetic).  A thread brings its own pieces of the next steps into shared memory with asynchronous copies.  The
// token's angles stay in registers for all rows, the weights too unless every head has its own.  kOnlyQ: beside the blocks of an 8-bit cache, where
// these rows are all there are and knowing so saves the registers that the kernel would spill.
struct Cursor {  // of one row group: its rows of a step
  int s, row, n;
  int kind;            // 0 q, 1 k, 2 v
  int64_t off, step;   // bytes from the kind's base: of the first row, from row to row
};

template <int TPR, bool BF16, bool kNeox, int kFmt, int kT, int kR, bool kOnlyQ>
__device__ __forceinline__ void rows_role(const NormRopeArgs& a, unsigned item, unsigned slices, int n_k, int n_v, const uint64_t* s_turns, uint4* s_rows) {
  constexpr int kSide = 32 / TPR;  // row groups of a warp
  constexpr int kSt = ring_stages(kR);
  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 31;
  const int t = lane % TPR, group = lane / TPR;
  const unsigned token = item / slices, slice = item - token * slices;
  if (token >= static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.seq)) return;
  const int b = static_cast<int>(token / static_cast<unsigned>(a.seq));
  const int l = static_cast<int>(token - static_cast<unsigned>(b) * static_cast<unsigned>(a.seq));
  const Chunks<kNeox> ch(t, a.head_dim, a.rotary_dim);
  const int n_q = a.q != nullptr ? a.n_heads : 0;
  // steps of kR kSide rows: q's, k's, v's; this warp's are [s0, s1)
  const int q_steps = (n_q + kR * kSide - 1) / (kR * kSide), k_steps = (n_k + kR * kSide - 1) / (kR * kSide), v_steps = (n_v + kR * kSide - 1) / (kR * kSide);
  const int steps = q_steps + k_steps + v_steps;
  const int s0 = static_cast<int>(static_cast<unsigned>(steps) * slice / slices), s1 = static_cast<int>(static_cast<unsigned>(steps) * (slice + 1) / slices);
  uint8_t* q_base = reinterpret_cast<uint8_t*>(a.q) + 2 * (static_cast<int64_t>(b) * a.q_stride[0] + static_cast<int64_t>(l) * a.q_stride[1]);
  const int64_t kv_off = 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + static_cast<int64_t>(l) * a.kv_stride[1]);
  uint8_t* k_base = const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(a.k)) + kv_off;
  const uint8_t* v_base = reinterpret_cast<const uint8_t*>(a.v) + kv_off;

  auto enter = [&](Cursor& c) {  // the kind that step c.s belongs to
    c.kind = kOnlyQ || c.s < q_steps ? 0 : c.s < q_steps + k_steps ? 1 : 2;
    c.row = (c.s - (c.kind == 0 ? 0 : c.kind == 1 ? q_steps : q_steps + k_steps)) * kR * kSide + group;
    c.n = c.kind == 0 ? n_q : c.kind == 1 ? n_k : n_v;
    const int64_t stride = 2 * (c.kind == 0 ? a.q_stride[2] : a.kv_stride[2]);
    c.off = c.row * stride;
    c.step = stride * kSide;
  };
  auto advance = [&](Cursor& c) {
    ++c.s;
    c.row += kR * kSide;
    c.off += kR * c.step;
    if (!kOnlyQ && (c.s == q_steps || c.s == q_steps + k_steps)) enter(c);
  };
  Cursor in;  // the step to be fetched next
  in.s = s0;
  enter(in);
  auto issue = [&](int stage) {
    if (in.s < s1) {
      const uint8_t* src = (in.kind == 0 ? q_base : in.kind == 1 ? k_base : v_base) + in.off;
      uint4* dst = s_rows + stage * (2 * kR) * kT + tid;
#pragma unroll
      for (int u = 0; u < kR; ++u) {
        if (ch.live && in.row + u * kSide < in.n) {
          cp_async_16(dst + (2 * u) * kT, src + u * in.step + 16 * ch.c0, true);
          cp_async_16(dst + (2 * u + 1) * kT, src + u * in.step + 16 * ch.c1, true);
        }
      }
      advance(in);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSt - 1; ++i) issue(i);  // on their way before the position is known

  const int pos = static_cast<int>(static_cast<unsigned>(a.start != nullptr ? a.start[b] : a.start_pos) + static_cast<unsigned>(l));
  int outer = 0, crow = 0;
  bool cache_ok = false;
  if (a.k_cache != nullptr && s1 > q_steps) cache_ok = locate(a, b, pos, lane == 0, outer, crow);
  Angles angles = {};
  if (s0 < q_steps + k_steps && a.rotary_dim > 0) warp_angles<TPR, kNeox>(s_turns, pos, ch, t, group, angles);
  Pairs weights = {};
  int weights_of = -1;  // kind
  const int w_bytes = a.w_kind == 2 ? 4 : 2;

  Cursor at;
  at.s = s0;
  enter(at);
  int stage = 0;
  for (; at.s < s1; advance(at)) {
    cp_async_wait<kSt - 2>();
    uint4* sp = s_rows + stage * (2 * kR) * kT + tid;
    const bool both = kR == 2 && at.row - group + kSide < at.n;  // rows for the second half of the step
    uint4 raw[kR][2];
#pragma unroll
    for (int u = 0; u < kR; ++u) {
      const bool there = ch.live && at.row + u * kSide < at.n;
      raw[u][0] = there ? sp[(2 * u) * kT] : make_uint4(0, 0, 0, 0);
      raw[u][1] = there ? sp[(2 * u + 1) * kT] : make_uint4(0, 0, 0, 0);
    }
    issue(stage == 0 ? kSt - 1 : stage - 1);
    stage = stage == kSt - 1 ? 0 : stage + 1;
    const int kind = at.kind;
    float x[kR][16];
    auto turn = [&](auto rows) {  // norm, weights and rotation of one row or two
      constexpr int kRows = decltype(rows)::value;
      const int64_t w_stride = (kind == 0 ? a.w_stride[0] : a.w_stride[1]) * w_bytes;
      const uint8_t* w = reinterpret_cast<const uint8_t*>(kind == 0 ? a.q_weight : a.k_weight);
      Pairs y[kRows];
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        unpack8<BF16>(raw[u][0], x[u]);
        unpack8<BF16>(raw[u][1], x[u] + 8);
        y[u] = as_pairs<kNeox>(x[u]);
      }
      if (w != nullptr) {
        if (w_stride == 0 && weights_of != kind) {
          weights = weight_pairs<kNeox>(w, a.w_kind, ch);
          weights_of = kind;
        }
        float f[kRows];
#pragma unroll
        for (int u = 0; u < kRows; ++u) f[u] = inverse_rms<TPR>(y[u], a.inv_dim, a.eps);
#pragma unroll
        for (int u = 0; u < kRows; ++u) {
          if (w_stride != 0) weights = weight_pairs<kNeox>(w + min(at.row + u * kSide, at.n - 1) * w_stride, a.w_kind, ch);
          apply_weights(y[u], weights, f[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < kRows; ++u) {
        apply_angles<kNeox>(y[u], angles, ch);
        as_values<kNeox>(y[u], x[u]);
        if (kFmt == 0 || kind == 0) {
          raw[u][0] = pack8<BF16>(x[u]);
          raw[u][1] = pack8<BF16>(x[u] + 8);
        }
      }
    };
    if (kind != 2) {
      if (both) turn(std::integral_constant<int, kR>{});
      else turn(std::integral_constant<int, 1>{});
    }
    if (kFmt == 0 || kind == 0) {
      uint8_t* dst;
      int64_t dst_step;
      if (kind == 0 || a.k_cache == nullptr) {
        dst = (kind == 0 ? q_base : k_base) + at.off;
        dst_step = at.step;
      } else {
        if (!cache_ok) continue;
        dst = reinterpret_cast<uint8_t*>(kind == 1 ? a.k_cache : a.v_cache) +
              2 * (static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(at.row) * a.cache_stride[1] + static_cast<int64_t>(crow) * a.cache_stride[2]);
        dst_step = 2 * kSide * a.cache_stride[1];
      }
#pragma unroll
      for (int u = 0; u < kR; ++u) {
        if (!ch.live || at.row + u * kSide >= at.n) continue;
        *reinterpret_cast<uint4*>(dst + u * dst_step + 16 * ch.c0) = raw[u][0];
        *reinterpret_cast<uint4*>(dst + u * dst_step + 16 * ch.c1) = raw[u][1];
      }
    } else if constexpr (kFmt != 0) {
      if (!cache_ok) continue;
      static_assert(kR == 1, "an 8-bit cache takes its rows one by one");
      const int begun = crow & ((1 << a.log_block) - 1);  // rows of the block that are there
#pragma unroll
      for (int u = 0; u < kR; ++u) {
        const int h = at.row + u * kSide;
        const bool row_ok = h < at.n;
        float* sc = (kind == 1 ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + static_cast<int64_t>(h) * a.scale_stride[1] + (crow >> a.log_block);
        const float o0 = row_ok && begun != 0 ? *sc : 0.f;  // the block's scale before and after
        if (kind == 2) {
          unpack8<BF16>(raw[u][0], x[u]);
          unpack8<BF16>(raw[u][1], x[u] + 8);
        }
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmax3(amax, fabsf(x[u][2 * i]), fabsf(x[u][2 * i + 1]));
#pragma unroll
        for (int d = TPR / 2; d > 0; d >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, d));
        const float need = b8_scale<kFmt>(amax);
        const float o1 = o0 >= need ? o0 : need;
        uint8_t* blk_rows = reinterpret_cast<uint8_t*>(kind == 1 ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] +
                            static_cast<int64_t>(h) * a.cache_stride[1] + static_cast<int64_t>(crow - begun) * a.cache_stride[2];
        if (row_ok) {
          const float r1 = b8_inverse(o1);
          uint8_t* dst = blk_rows + static_cast<int64_t>(begun) * a.cache_stride[2];
          *reinterpret_cast<uint2*>(dst + 8 * ch.c0) = b8_code8<kFmt>(x[u], o1, r1);
          *reinterpret_cast<uint2*>(dst + 8 * ch.c1) = b8_code8<kFmt>(x[u] + 8, o1, r1);
          if (b8_wants_quotient<kFmt>(o1)) {  // (the thread's pieces of this step have been read: the values pass through their place)
            float4* f = reinterpret_cast<float4*>(sp);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              f[0] = make_float4(x[u][8 * i], x[u][8 * i + 1], x[u][8 * i + 2], x[u][8 * i + 3]);
              f[kT] = make_float4(x[u][8 * i + 4], x[u][8 * i + 5], x[u][8 * i + 6], x[u][8 * i + 7]);
              e4m3_code_at(dst + 8 * (i ? ch.c1 : ch.c0), f, kT, o1);
            }
          }
        }
        __syncwarp();  // every lane of the row has read the scale
        if (row_ok && t == 0 && (begun == 0 || o1 != o0)) *sc = o1;  // (a block that begins here held anything)
        // A scale that grew: the rows before are coded again, by the whole warp
        unsigned grown = __ballot_sync(0xFFFFFFFFu, row_ok && begun != 0 && o1 != o0 && t == 0);
        while (grown != 0) {
          const int from = __ffs(grown) - 1;
          grown &= grown - 1;
          const uint64_t p = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(blk_rows), from);
          recode_rows<kFmt>(reinterpret_cast<uint8_t*>(p), a.cache_stride[2], begun, a.head_dim / 16, __shfl_sync(0xFFFFFFFFu, o0, from),
                            __shfl_sync(0xFFFFFFFFu, o1, from), lane, 32);
        }
      }
    }
  }
}

template <int TPR, bool BF16, bool kNeox, int kFmt>
__global__ void __launch_bounds__(kRowThreads, 4) norm_rope_rows_kernel(const NormRopeArgs a) {
  constexpr int kR = rows_per_step(kFmt);
  __shared__ __align__(16) uint4 s_rows[rows_smem(kRowThreads, kR) / sizeof(uint4)];
  __shared__ uint64_t s_turns[kMaxPairs];
  grid_launch_dependents();
  copy_turns<kRowThreads>(a, s_turns);
  grid_dependency_wait();
  rows_role<TPR, BF16, kNeox, kFmt, kRowThreads, kR, false>(a, blockIdx.x * (kRowThreads / 32) + threadIdx.x / 32, static_cast<unsigned>(a.slices),
                                                 a.k != nullptr ? a.n_kv_heads : 0, a.v != nullptr ? a.n_kv_heads : 0, s_turns, s_rows);
}

// ---- blocks of an 8-bit cache: k and v of calls with several tokens per sequence ----
//
// A unit is one block of tokens of one sequence, for a slice of the kv heads, of k or of v.  A head's rows of one block fill 2^log_block * TPR
// lanes: four, two or one head at a time, or two or four rows per thread.  The raw rows come through shared memory, each thread's own
// pieces (no barrier; the next head's are fetched as soon as these have been read); k's normed and rotated rows wait there in
// fp32 until the block's largest magnitude is agreed on.  A thread computes the angles of its first row once for all heads of the
// unit and turns those on to each of its other rows, by the angle between the two: one product, whatever the row (from row to row
// its roundings would add up, and more values fall on the wrong side of a border between two codes).
constexpr int kMaxRows = 4;                          // of a thread
constexpr int kTurnFloats = (kMaxRows - 1) * 2 * kMaxPairs;  // cos and sin of the angles to rows 1, 2, 3
constexpr int blocks_smem(int lanes) {  // lanes that the rows of the heads side by side fill (kThreads at least)
  return kTurnFloats * 4 + lanes * (32 + 64);
}

// largest magnitude of a row's raw values (NaN is passed over)
template <bool BF16>
__device__ __forceinline__ float raw_amax(const uint4& p, const uint4& q) {
  const uint32_t w[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
  if constexpr (BF16) {
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
    return fmaxf(__low2float(m), __high2float(m));
  } else {
    __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
    return fmaxf(__low2float(m), __high2float(m));
  }
}

// What a thread's rows of a block that was begun may want besides, in one call out of the way of the registers: rows that were there (`old`, a bit each)
// are coded again under a scale that grew, s0 -> s1; new ones are coded by the quotient where s1 is no power of two.  k's values still wait in shared
// memory, v's are read again.
template <bool BF16, int kFmt, bool kIsK>
__device__ __noinline__ void rows_of_begun_block(uint8_t* dst, int64_t dst_step, const float4* val, const uint8_t* src, int64_t src_step, int c0, int c1, unsigned fresh,
                                                 unsigned old, float s0, float s1) {
  const float r1 = b8_inverse(s1);
#pragma unroll 1
  for (int i = 0; i < 2 * kMaxRows; ++i) {  // both chunks of every row
    const int r = i >> 1, c = (i & 1) ? c1 : c0;
    uint2* d = reinterpret_cast<uint2*>(dst + r * dst_step + 8 * c);
    if ((old >> r) & 1u) {
      *d = b8_recode8<kFmt>(*d, s0, s1, r1);
    } else if (b8_wants_quotient<kFmt>(s1) && ((fresh >> r) & 1u)) {
      float x[8];
      if constexpr (kIsK) {
        *reinterpret_cast<float4*>(x) = val[2 * i * kThreads];
        *reinterpret_cast<float4*>(x + 4) = val[(2 * i + 1) * kThreads];
      } else {
        unpack8<BF16>(*reinterpret_cast<const uint4*>(src + r * src_step + 16 * c), x);
      }
      *d = e4m3_code8(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), s1);
    }
  }
}

template <int TPR, bool BF16, bool kNeox, int kFmt, bool kIsK, int kRows>
__device__ __forceinline__ void block_role(const NormRopeArgs& a, unsigned unit, unsigned slice, unsigned slices, const uint64_t* s_turns, float* smem, float* s_max) {
  const int tid = static_cast<int>(threadIdx.x);
  const int t = tid % TPR, rg = tid / TPR;
  const int blk = 1 << a.log_block;
  const int pairs = a.rotary_dim / 2;
  const int side = max(1, kThreads / (blk * TPR));               // heads side by side
  float* s_turn = smem;                                          // [kMaxRows - 1][2][kMaxPairs]
  uint4* s_raw = reinterpret_cast<uint4*>(smem + kTurnFloats) + tid;                    // [kRows][2] pieces, kThreads apart
  float4* s_val = reinterpret_cast<float4*>(smem + kTurnFloats) + kRows * 2 * kThreads + tid;  // [kRows][4]: k as it is to be coded
  const int b = static_cast<int>(unit / static_cast<unsigned>(a.n_touch)), j = static_cast<int>(unit - static_cast<unsigned>(b) * static_cast<unsigned>(a.n_touch));
  const Chunks<kNeox> ch(t, a.head_dim, a.rotary_dim);
  const int64_t start = a.start != nullptr ? a.start[b] : a.start_pos;
  // the j-th block of those that the valid positions of this call touch
  const int64_t p0 = start > 0 ? start : 0, p1 = min(start + a.seq, static_cast<int64_t>(a.max_len));  // positions [p0, p1)
  if (kIsK && tid == 0 && j == 0 && slice == 0 && (start < 0 || start + a.seq > a.max_len))
    report(a.status, kStatusBadPosition, b, static_cast<int>(start < 0 ? start : max(start, static_cast<int64_t>(a.max_len))), a.max_len);
  const int64_t base64 = (p0 >> a.log_block << a.log_block) + static_cast<int64_t>(j) * blk;
  if (base64 >= p1) return;
  const int base = static_cast<int>(base64);
  const int lo = static_cast<int>(max(p0 - base, static_cast<int64_t>(0))), hi = static_cast<int>(min(p1 - base, static_cast<int64_t>(blk)));  // new rows of the block
  int outer, row0;
  if (!locate(a, b, base + lo, kIsK && tid == 0 && slice == 0, outer, row0)) return;  // (a block lies in one page)
  row0 -= lo;

  const int sub = rg >> a.log_block;                                 // which of the heads side by side
  const int row_a = rg & (blk - 1);                                  // this lane's rows of the block: row_a, row_a + row_step, ...
  const int row_step = kThreads / TPR;
  const int n_groups = (a.n_kv_heads + side - 1) / side;
  const int g0 = static_cast<int>(static_cast<unsigned>(n_groups) * slice / slices), g1 = static_cast<int>(static_cast<unsigned>(n_groups) * (slice + 1) / slices);
  const int64_t src_step = 2 * row_step * a.kv_stride[1], dst_step = row_step * a.cache_stride[2];
  const uint8_t* src = reinterpret_cast<const uint8_t*>(kIsK ? a.k : a.v) + 2 * (static_cast<int64_t>(b) * a.kv_stride[0] + (base + row_a - start) * a.kv_stride[1]);
  uint8_t* cache = reinterpret_cast<uint8_t*>(kIsK ? a.k_cache : a.v_cache) + static_cast<int64_t>(outer) * a.cache_stride[0] + static_cast<int64_t>(row0 + row_a) * a.cache_stride[2];
  float* scales = (kIsK ? a.k_scale : a.v_scale) + static_cast<int64_t>(outer) * a.scale_stride[0] + (row0 >> a.log_block);

  auto is_new = [&](int r) { return row_a + r * row_step >= lo && row_a + r * row_step < hi; };
  auto fetch = [&](int g, int r) {
    const int h = g * side + sub;
    if (g < g1 && h < a.n_kv_heads && ch.live && is_new(r)) {
      const uint8_t* p = src + 2 * static_cast<int64_t>(h) * a.kv_stride[2] + r * src_step;
      cp_async_16(s_raw + (2 * r) * kThreads, p + 16 * ch.c0, true);
      cp_async_16(s_raw + (2 * r + 1) * kThreads, p + 16 * ch.c1, true);
    }
  };
#pragma unroll
  for (int r = 0; r < kRows; ++r) fetch(g0, r);
  cp_async_commit();
  Angles first = {};
  if (kIsK && pairs > 0) {
    if (kRows > 1) {
      for (int u = tid; u < (kRows - 1) * kMaxPairs; u += kThreads) {
        const int r = u / kMaxPairs, i = u % kMaxPairs;
        if (i >= pairs) continue;
        const float2 cs = angle_of(s_turns, (r + 1) * row_step, i);
        s_turn[2 * r * kMaxPairs + i] = cs.x;
        s_turn[(2 * r + 1) * kMaxPairs + i] = cs.y;
      }
      __syncthreads();
    }
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      if (p < 4 ? ch.rot0 : ch.rot1) {
        const float2 cs = angle_of(s_turns, base + row_a, p < 4 ? ch.i0 + p : ch.i1 + p - 4);
        (p & 1 ? first.c[p / 2].y : first.c[p / 2].x) = cs.x;
        (p & 1 ? first.s[p / 2].y : first.s[p / 2].x) = cs.y;
      }
    }
  }
  Pairs weights = {};
  const uint8_t* w_now = nullptr;
  const int w_bytes = a.w_kind == 2 ? 4 : 2;
  for (int g = g0; g < g1; ++g) {
    const int h = g * side + sub;
    const bool head_ok = h < a.n_kv_heads;
    if (kIsK && a.k_weight != nullptr) {
      const uint8_t* wp = reinterpret_cast<const uint8_t*>(a.k_weight) + static_cast<int64_t>(head_ok ? h : 0) * a.w_stride[1] * w_bytes;
      if (wp != w_now) weights = weight_pairs<kNeox>(wp, a.w_kind, ch);
      w_now = wp;
    }
    const float s0 = (head_ok && lo != 0) ? scales[static_cast<int64_t>(h) * a.scale_stride[1]] : 0.f;
    cp_async_wait<0>();
    float amax = 0.f;
    Angles angles = first;
#pragma unroll 2
    for (int r = 0; r < kRows; ++r) {
      uint4 raw0 = make_uint4(0, 0, 0, 0), raw1 = raw0;  // (rows that are not new: zeros)
      if (is_new(r) && ch.live) {
        raw0 = s_raw[(2 * r) * kThreads];
        raw1 = s_raw[(2 * r + 1) * kThreads];
      }
      if constexpr (!kIsK) {
        amax = fmaxf(amax, raw_amax<BF16>(raw0, raw1));
      } else {
        fetch(g + 1, r);
        if (r > 0) {  // the angles of the thread's r-th row
          Angles d = {};
          load_angles<kNeox>(s_turn + 2 * (r - 1) * kMaxPairs, s_turn + (2 * r - 1) * kMaxPairs, ch, d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = first.c[i];
            angles.c[i] = minus_product(first.s[i], d.s[i], __fmul2_rn(c, d.c[i]));
            angles.s[i] = __ffma2_rn(first.s[i], d.c[i], __fmul2_rn(c, d.s[i]));
          }
        }
        float x[16];
        unpack8<BF16>(raw0, x);
        unpack8<BF16>(raw1, x + 8);
        Pairs y = as_pairs<kNeox>(x);
        if (a.k_weight != nullptr) apply_weights(y, weights, inverse_rms<TPR>(y, a.inv_dim, a.eps));
        apply_angles<kNeox>(y, angles, ch);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          amax = fmax3(amax, fabsf(y.lo[i].x), fabsf(y.lo[i].y));
          amax = fmax3(amax, fabsf(y.hi[i].x), fabsf(y.hi[i].y));
        }
        as_values<kNeox>(y, x);
#pragma unroll
        for (int i = 0; i < 4; ++i) s_val[(4 * r + i) * kThreads] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
      }
    }
    if (kIsK) cp_async_commit();
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
#pragma unroll 2
    for (int r = 0; r < kRows; ++r) {
      uint2* d0 = reinterpret_cast<uint2*>(dst + r * dst_step + 8 * ch.c0);
      uint2* d1 = reinterpret_cast<uint2*>(dst + r * dst_step + 8 * ch.c1);
      if (head_ok && ch.live && is_new(r)) {
        float x[16];
        if constexpr (kIsK) {
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(x + 4 * i) = s_val[(4 * r + i) * kThreads];
        } else {
          unpack8<BF16>(s_raw[(2 * r) * kThreads], x);
          unpack8<BF16>(s_raw[(2 * r + 1) * kThreads], x + 8);
          fetch(g + 1, r);
        }
        *d0 = b8_code8<kFmt>(x, s1, r1);
        *d1 = b8_code8<kFmt>(x + 8, s1, r1);
      }
    }
    if (!kIsK) cp_async_commit();
    if (lo != 0 && (s1 != s0 || b8_wants_quotient<kFmt>(s1)) && head_ok && ch.live) {
      unsigned fresh = 0, old = 0;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (is_new(r)) fresh |= 1u << r;
        else if (row_a + r * row_step < lo && s1 != s0) old |= 1u << r;
      }
      rows_of_begun_block<BF16, kFmt, kIsK>(dst, dst_step, s_val, src + 2 * static_cast<int64_t>(h) * a.kv_stride[2], src_step, ch.c0, ch.c1, fresh, old, s0, s1);
    }
    // one lane of the head's group
    if (head_ok && t == 0 && row_a == 0 && (lo == 0 || s1 != s0)) scales[static_cast<int64_t>(h) * a.scale_stride[1]] = s1;
  }
}

// Units of k and of v, which take more arithmetic than bandwidth, spread evenly among the blocks that rewrite q, which take more bandwidth.
template <int TPR, bool BF16, bool kNeox, int kFmt, int kRows>
__global__ void __launch_bounds__(kThreads, 2) norm_rope_blocks_kernel(const NormRopeArgs a) {
  extern __shared__ __align__(16) float s_dyn[];
  __shared__ float s_max[2 * kThreads / 32];
  __shared__ uint64_t s_turns[kMaxPairs];
  grid_launch_dependents();
  copy_turns<kThreads>(a, s_turns);
  grid_dependency_wait();
  const unsigned per = static_cast<unsigned>(a.batch) * static_cast<unsigned>(a.n_touch) * static_cast<unsigned>(a.kv_slices);  // blocks of k, and of v
  const unsigned before = static_cast<unsigned>(static_cast<uint64_t>(blockIdx.x) * (2 * per) / gridDim.x);   // units before this block
  if (static_cast<unsigned>(static_cast<uint64_t>(blockIdx.x + 1) * (2 * per) / gridDim.x) != before) {
    const unsigned slices = static_cast<unsigned>(a.kv_slices), i = before >> 1;
    if (before & 1) block_role<TPR, BF16, kNeox, kFmt, false, kRows>(a, i / slices, i % slices, slices, s_turns, s_dyn, s_max);
    else block_role<TPR, BF16, kNeox, kFmt, true, kRows>(a, i / slices, i % slices, slices, s_turns, s_dyn, s_max);
  } else {
    rows_role<TPR, BF16, kNeox, 0, kThreads, 2, true>(a, (blockIdx.x - before) * (kThreads / 32) + threadIdx.x / 32, static_cast<unsigned>(a.slices), 0, 0,
                                             s_turns, reinterpret_cast<uint4*>(s_dyn));
  }
}

// Frequencies in turns: base ^ (-2 i / rotary_dim) / (2 pi), modulo 1 (positions are whole numbers), as fractions of 2^64.  A thread keeps those of its last base:
// calls that change it (or rotary_dim) take 17 us more of host time each (64 pairs; 20.1 us per call instead of 3.0), which a captured graph does not.
void fill_turns(NormRopeArgs& a, double freq_base) {
  thread_local double cached_base = 0.0;
  thread_local int cached_rot = -1;
  thread_local uint64_t table[kMaxPairs];
  if (cached_base != freq_base || cached_rot != a.rotary_dim) {
    const long double two_pi = 6.283185307179586476925286766559005768L;
    for (int i = 0; i < kMaxPairs; ++i) {
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
  for (int i = 0; i < kMaxPairs; ++i) a.turns[i] = table[i];
}

template <int TPR, bool BF16, bool kNeox, int kFmt>
cudaError_t launch_rows(const NormRopeArgs& a, unsigned blocks, cudaStream_t stream) {
  LaunchAttrs at(stream);
  at.cfg.gridDim = dim3(blocks);
  at.cfg.blockDim = dim3(kRowThreads);
  return cudaLaunchKernelEx(&at.cfg, norm_rope_rows_kernel<TPR, BF16, kNeox, kFmt>, a);
}

template <int TPR, bool BF16, bool kNeox, int kFmt, int kRows>
cudaError_t launch_blocks_rows(const NormRopeArgs& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  auto* kernel = norm_rope_blocks_kernel<TPR, BF16, kNeox, kFmt, kRows>;
  if (smem > 46 * 1024) {  // (48 KB with the static part)
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
cudaError_t launch_blocks(const NormRopeArgs& a, unsigned blocks, size_t smem, cudaStream_t stream) {
  const int lanes = TPR << a.log_block;
  if (lanes <= kThreads) return launch_blocks_rows<TPR, BF16, kNeox, kFmt, 1>(a, blocks, smem, stream);
  if (lanes == 2 * kThreads) return launch_blocks_rows<TPR, BF16, kNeox, kFmt, 2>(a, blocks, smem, stream);
  if constexpr (TPR == 8) return launch_blocks_rows<TPR, BF16, kNeox, kFmt, 4>(a, blocks, smem, stream);
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeArgs& a_in, bool bf16, bool neox, int cache_format, double freq_base, cudaStream_t stream) {
  NormRopeArgs a = a_in;
  fill_turns(a, freq_base);
  a.inv_dim = 1.0f / static_cast<float>(a.head_dim);
  const int tpr = a.head_dim <= 64 ? 4 : a.head_dim <= 128 ? 8 : 16;
  const int side = 32 / tpr;  // row groups of a warp
  const long long tokens = static_cast<long long>(a.batch) * a.seq;
  const int fmt = cache_format == MINFER_ATTN_KV_E4M3 ? kE4M3 : cache_format == MINFER_ATTN_KV_INT8 ? kInt8 : 0;
  const bool by_block = fmt != 0 && a.seq > 1;
  const int kv_rows = by_block ? 0 : a.n_kv_heads;
  const int step_rows = (by_block ? 2 : rows_per_step(fmt)) * side;
  const int steps = (a.q != nullptr ? (a.n_heads + step_rows - 1) / step_rows : 0) + (a.k != nullptr ? (kv_rows + step_rows - 1) / step_rows : 0) +
                    (a.v != nullptr ? (kv_rows + step_rows - 1) / step_rows : 0);
  // A warp takes a token; while that leaves the GPU's warps (16 per SM) without work, a token's rows are dealt out over several.
  long long slices = (16 * 148 + tokens - 1) / tokens;
  if (slices > steps) slices = steps;
  if (slices < 1) slices = 1;
  a.slices = static_cast<int>(slices);
  const int row_warps = (by_block ? kThreads : kRowThreads) / 32;
  const long long row_blocks = (tokens * slices + row_warps - 1) / row_warps;
#define MINFER_NR_STYLE(fn, TPR, F, ...) \
  (bf16 ? (neox ? fn<TPR, true, true, F>(__VA_ARGS__) : fn<TPR, true, false, F>(__VA_ARGS__)) \
        : (neox ? fn<TPR, false, true, F>(__VA_ARGS__) : fn<TPR, false, false, F>(__VA_ARGS__)))
  if (!by_block) {
    const unsigned nb = static_cast<unsigned>(row_blocks);
    if (fmt == 0) {
      if (tpr == 4) return MINFER_NR_STYLE(launch_rows, 4, 0, a, nb, stream);
      if (tpr == 8) return MINFER_NR_STYLE(launch_rows, 8, 0, a, nb, stream);
      return MINFER_NR_STYLE(launch_rows, 16, 0, a, nb, stream);
    }
    if (fmt == kE4M3) return tpr == 4 ? MINFER_NR_STYLE(launch_rows, 4, kE4M3, a, nb, stream) : MINFER_NR_STYLE(launch_rows, 8, kE4M3, a, nb, stream);
    return tpr == 4 ? MINFER_NR_STYLE(launch_rows, 4, kInt8, a, nb, stream) : MINFER_NR_STYLE(launch_rows, 8, kInt8, a, nb, stream);
  }
  const int blk = 1 << a.log_block;
  a.n_touch = static_cast<int>((static_cast<int64_t>(a.seq) + blk - 2) / blk + 1);  // (a call may name nearly 2^31 tokens, of an expanded k and v)
  const long long units = static_cast<long long>(a.batch) * a.n_touch;
  const int abreast = (tpr << a.log_block) < kThreads ? kThreads / (tpr << a.log_block) : 1;  // heads side by side
  const int head_groups = (a.n_kv_heads + abreast - 1) / abreast;
  // A unit's heads over several blocks while all units together are fewer than two per SM; fewer blocks share the angles better (us with this /
  // twice as many: 8 x 512 tokens, D=64, blocks of 16: 16.1 / 18.4; 4 x 4096, D=128, blocks of 128: 71.7 / 69.9).
  long long kv_slices = 2 * 148 / units;
  if (kv_slices > head_groups) kv_slices = head_groups;
  if (kv_slices < 1) kv_slices = 1;
  a.kv_slices = static_cast<int>(kv_slices);
  const long long blocks = 2 * units * kv_slices + (a.q != nullptr ? row_blocks : 0);
  if (blocks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  size_t smem = blocks_smem((tpr << a.log_block) > kThreads ? tpr << a.log_block : kThreads);
  if (a.q != nullptr && smem < static_cast<size_t>(rows_smem(kThreads, 2))) smem = rows_smem(kThreads, 2);
  const unsigned nb = static_cast<unsigned>(blocks);
  if (fmt == kE4M3) return tpr == 4 ? MINFER_NR_STYLE(launch_blocks, 4, kE4M3, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks, 8, kE4M3, a, nb, smem, stream);
  return tpr == 4 ? MINFER_NR_STYLE(launch_blocks, 4, kInt8, a, nb, smem, stream) : MINFER_NR_STYLE(launch_blocks, 8, kInt8, a, nb, smem, stream);
#undef MINFER_NR_STYLE
}

}  // namespace minfer_attn
