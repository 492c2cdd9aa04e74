// Values of a block-scaled 8-bit KV cache: e4m3 or int8 codes, one fp32 scale for each block of tokens and head.
//
//   e4m3  scale = the smallest power of two under which the block's largest magnitude is at most 448.  A floating code loses nothing to
//         a coarse scale but the last factor of two of its range, and in exchange x / scale is exact, and rows coded
//         again under a larger scale keep their values (unless they fall below the smallest normal code, 2^-6).
//   int8  scale = fp32(largest magnitude / 127): a fixed step, where a power of two would cost up to a bit.
//   code  = the one nearest to x / scale, ties to even.  Infinite values saturate; NaN stays NaN in e4m3 and becomes 0 in int8.
// Rows are coded again from code * scale in fp32.
// A block of zeros has scale 0 and codes 0; no other scale is below 2^-126.
#pragma once

#include <cuda_fp16.h>
#include <stdint.h>

namespace minfer_attn {

constexpr int kE4M3 = 1;
constexpr int kInt8 = 2;

// the scale that a block with this largest magnitude needs
template <int kFmt>
__device__ __forceinline__ float b8_scale(float amax) {
  amax = fminf(amax, 3.402823466e38f);  // an infinite value counts as the largest finite one
  if constexpr (kFmt == kE4M3) {
    // 448 = 1.75 * 2^8: the sum carries into the exponent when the significand is above 1.75
    const int e = static_cast<int>((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 8;
    return amax > 0.f ? __uint_as_float(static_cast<uint32_t>(max(e, 1)) << 23) : 0.f;
  } else {
    return amax > 0.f ? fmaxf(__fdiv_rn(amax, 127.f), 1.17549435e-38f) : 0.f;  // (normal, so that its inverse is finite)
  }
}

// 1 / scale (exact for a power of two), 0 for a block of zeros
__device__ __forceinline__ float b8_inverse(float s) { return s > 0.f ? __frcp_rn(s) : 0.f; }

// The int8 code nearest to x / s (the exact quotient, ties to even), for values that lie near a border between two codes or are not
// finite.  q is the rounded quotient: it cannot pass a border, only fall on one, and then the remainder's sign decides.
__device__ __forceinline__ uint32_t int8_code(float x, float s) {
  const float q = s > 0.f ? __fdiv_rn(x, s) : 0.f;
  float n = rintf(q);
  if (fabsf(q - n) == 0.5f) {
    const float rem = fmaf(-q, s, x);
    if (rem != 0.f) n = rem > 0.f ? ceilf(q) : floorf(q);
  }
  n = q == q ? fminf(fmaxf(n, -127.f), 127.f) : 0.f;
  return static_cast<uint32_t>(static_cast<int>(n)) & 0xFFu;
}
static __device__ __noinline__ uint2 int8_code8(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7, float s) {
  return make_uint2(int8_code(x0, s) | (int8_code(x1, s) << 8) | (int8_code(x2, s) << 16) | (int8_code(x3, s) << 24),
                    int8_code(x4, s) | (int8_code(x5, s) << 8) | (int8_code(x6, s) << 16) | (int8_code(x7, s) << 24));
}

// larger of two magnitudes, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// two fp32 -> two e4m3 in the low 16 bits (lo in the low byte), saturating
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// two e4m3 (low 16 bits) -> two fp16, exact
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t pair) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(pair)));
  return r;
}

// two int8 of a word whose bytes were XORed with 0x80 -> two fp16, exact: the byte dropped into the mantissa of 1024.0 reads
// 1024 + 128 + q.  kSel picks the bytes of the low and high value.
template <uint32_t kSel>
__device__ __forceinline__ uint32_t int8_to_half2(uint32_t src) {
  const uint32_t x = __byte_perm(src, 0x64646464u, kSel);
  const uint32_t bias = 0x64806480u;  // 1152.0 twice
  const __half2 q = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&q);
}

// Whether a product with 1 / scale may miss the nearest e4m3 code: it is exact for powers of two, but a block that another program began may
// have any scale (largest / 448, say), and keeps it until it has to grow.
template <int kFmt>
__device__ __forceinline__ bool b8_wants_quotient(float s) { return kFmt == kE4M3 && (__float_as_uint(s) & 0x7FFFFFu) != 0; }

// x / s rounded to fp32, but to the odd one of its two neighbours where it is not exact: on the same side of every border between two codes as the
// exact quotient, as a border has few bits.  The nearest fp32 cannot pass a border, only fall on one; the remainder's sign says which side is right.
__device__ __forceinline__ float odd_quotient(float x, float s) {
  if (s < 8.67361737988403547e-19f) {  // 2^-60: the remainder's last bit may lie below the smallest fp32
    x *= 18446744073709551616.f;       // 2^64; finite values are no larger than 448 s
    s *= 18446744073709551616.f;
  }
  const float q = __fdiv_rn(x, s);
  const uint32_t bits = __float_as_uint(q);
  if (!(fabsf(q) >= 2.44140625e-4f && fabsf(q) < 512.f) || (bits & 1u) != 0) return q;  // (2^-12: no borders below that)
  const float rem = fmaf(-q, s, x);
  return rem == 0.f ? q : __uint_as_float(bits + ((rem < 0.f) == (q < 0.f) ? 1u : 0xFFFFFFFFu));
}

// The e4m3 codes nearest to eight values, by the quotient
__device__ __forceinline__ uint2 e4m3_code8(const float4& a, const float4& b, float s) {
  return make_uint2(e4m3_pair(odd_quotient(a.x, s), odd_quotient(a.y, s)) | (e4m3_pair(odd_quotient(a.z, s), odd_quotient(a.w, s)) << 16),
                    e4m3_pair(odd_quotient(b.x, s), odd_quotient(b.y, s)) | (e4m3_pair(odd_quotient(b.z, s), odd_quotient(b.w, s)) << 16));
}
// The same of values in x[0] and x[step]: in memory, out of the way of the kernel's registers
static __device__ __noinline__ void e4m3_code_at(uint8_t* codes, const float4* x, int step, float s) {
  *reinterpret_cast<uint2*>(codes) = e4m3_code8(x[0], x[step], s);
}

// eight values -> eight codes; r = 1 / s.  e4m3: for scales that are powers of two (b8_wants_quotient).
// Values of magnitude 127.5 s and above do not occur with int8: the scale follows the largest.
template <int kFmt>
__device__ __forceinline__ uint2 b8_code8(const float* x, float s, float r) {
  uint32_t w[2];
  const float2 r2 = make_float2(r, r);
  float off = 0.f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* y = x + 4 * i;
    const float2 u = __fmul2_rn(make_float2(y[0], y[1]), r2), v = __fmul2_rn(make_float2(y[2], y[3]), r2);
    if constexpr (kFmt == kE4M3) {
      w[i] = e4m3_pair(u.x, u.y) | (e4m3_pair(v.x, v.y) << 16);
    } else {
      // adding 1.5 * 2^23 rounds to a whole number, which the low byte of the sum holds in two's complement
      const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f), minus = make_float2(-1.f, -1.f);
      const float2 ku = __fadd2_rn(u, magic), kv = __fadd2_rn(v, magic);
      const float2 du = __ffma2_rn(__fadd2_rn(ku, back), minus, u), dv = __ffma2_rn(__fadd2_rn(kv, back), minus, v);
      off = max_nan(max_nan(max_nan(off, fabsf(du.x)), max_nan(fabsf(du.y), fabsf(dv.x))), fabsf(dv.y));
      w[i] = __byte_perm(__byte_perm(__float_as_uint(ku.x), __float_as_uint(ku.y), 0x0040), __byte_perm(__float_as_uint(kv.x), __float_as_uint(kv.y), 0x0040), 0x5410);
    }
  }
  if constexpr (kFmt == kInt8) {
    // the product with 1 / s is off by at most 127 * 1.5 * 2^-23 = 2.3e-5: nearer to a border, or not finite, the quotient decides
    if (!(off < 0.49994f)) return int8_code8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7], s);
  }
  return make_uint2(w[0], w[1]);
}

// eight codes -> fp32, unscaled
template <int kFmt>
__device__ __forceinline__ void b8_values8(uint2 c, float* x) {
  const uint32_t w[2] = {c.x, c.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t h[2];
    if constexpr (kFmt == kE4M3) {
      h[0] = e4m3_to_half2(w[i]);
      h[1] = e4m3_to_half2(w[i] >> 16);
    } else {
      const uint32_t u = w[i] ^ 0x80808080u;
      h[0] = int8_to_half2<0x4140>(u);
      h[1] = int8_to_half2<0x4342>(u);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      x[4 * i + 2 * j] = f.x;
      x[4 * i + 2 * j + 1] = f.y;
    }
  }
}

// eight codes under scale s0 -> the codes of the same values under s1
template <int kFmt>
__device__ __forceinline__ uint2 b8_recode8(uint2 c, float s0, float s1, float r1) {
  float x[8];
  b8_values8<kFmt>(c, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] *= s0;
    if constexpr (kFmt == kInt8) x[i] = fmaxf(x[i], -127.f * s1);  // (another program's code -128 may pass the largest magnitude of s1)
  }
  return b8_code8<kFmt>(x, s1, r1);
}

// rows [0, n) of a block (row_chunks 16-byte chunks each), coded again by `lanes` threads
template <int kFmt>
__device__ __noinline__ void recode_rows(uint8_t* rows, int64_t row_stride, int n, int row_chunks, float s0, float s1, int lane, int lanes) {
  const float r1 = b8_inverse(s1);
  constexpr int kBatch = 4;  // loads in flight
  for (int i0 = lane; i0 < n * row_chunks; i0 += kBatch * lanes) {
    uint4 c[kBatch];
    uint4* p[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = i0 + u * lanes;
      p[u] = i < n * row_chunks ? reinterpret_cast<uint4*>(rows + static_cast<int64_t>(i / row_chunks) * row_stride) + i % row_chunks : nullptr;
      c[u] = p[u] != nullptr ? *p[u] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      if (p[u] == nullptr) continue;
      const uint2 lo = b8_recode8<kFmt>(make_uint2(c[u].x, c[u].y), s0, s1, r1);
      const uint2 hi = b8_recode8<kFmt>(make_uint2(c[u].z, c[u].w), s0, s1, r1);
      *p[u] = make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
  }
}

}  // namespace minfer_attn
