// Split-KV decode attention over a cache held in 8 bits (e4m3 or int8 codes) with one fp32 scale for each block of tokens and
// head, HBM-bound: 2 head_dim + 8 / block bytes per cached key.
//
//   t_j = (q . k_j) ks_j / sqrt(head_dim)      out = sum_j exp(t_j) vs_j v_j / sum_j exp(t_j)
//
// k_j, v_j: codes; ks_j, vs_j: the scales of key j's block.  The scheme is decode_kernel's (decode_sm100.cu): a block streams a
// part of the keys of one (sequence, kv head) for all its query heads, each warp with a ring of 16-key tiles of its own;
// products transposed (keys, then dimensions, as the 16 rows of an m16n8k16 tile); partial outputs merged through the
// shared memory of a cluster, or through a workspace (decode_common.cuh).  What differs:
//
// A tile lies inside one block of tokens, so its two scales are uniform and neither costs a multiplication per value: ks goes
// into the factor that the scores take anyway, vs into the weights.  Codes of both kinds are exact in fp16, so all products are
// fp16 MMAs on unscaled codes; bfloat16 queries are brought into fp16's range by a power of two per head, under which the largest lies in 2^14 .. 2^15: exact down
// to about 2^-31 of it, and below that off by at most half of fp16's last step, 2^-25, which is 2^-39 of the largest.
//
// Weights: w_j = 2^(t_j - m) vs_j is what is rounded to fp16.  m follows max_j(t_j + ceil(log2 vs_j)) - 14, not max t_j, so that
// whatever the scales are the largest weight lies in (2^13, 2^14]: fp16 has full precision down to 2^-14, so weights keep theirs down to
// 2^-28 of the largest, and a long tail of equal small weights is not rounded in one direction.  The row sum takes 2^(t_j - m)
// in fp32, before the scale and before the rounding.  log2 vs_j counts as -90 or more: 2^104 times the number of keys fits
// fp32, and a block of zeros (scale 0) has weights of 0.  References of different blocks are then up to 90 + log2 of the largest scale apart, which fp32
// holds to 126: from scales of v above 2^36 on (values of 3e13) the share that blocks of zeros have in the sum may be lost.
//
// Shared memory: rows of 128 bytes with the 16-byte chunks XORed by the row, pairs of rows of 64 bytes likewise by their line, so that a lane's
// 16-byte reads - K: chunks 2 tq and 2 tq + 1 of key g0; V: chunk g0 of keys 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9 - meet no bank twice.
// A lane takes consecutive dimensions: for K that permutes the summands of an MMA, for V the rows of the output.
//
// Measured (32 / 8 heads, D=128, back to back in a graph): 64 sequences of 512-8192 keys, e4m3, 92.7 us, 6.2 TB/s, 0.96 of what a copy reaches (102 us, 0.87, as a
// call among other work).  24 ragged sequences of up to 10001, 48 / 8 heads, in one piece / pages of 64 / of 256 keys: e4m3 49.6 / 54.2 / 53.8 us, int8 53.3 / 60.6 /
// 60.4, 0.67 of a copy: a block's look-ups per tile (a division, three products) are 14 % more instructions at the same issue rate (55 % of cycles, ALU 48 %).
#include "b8.cuh"
#include "decode_common.cuh"

#include <atomic>

namespace minfer_attn {

namespace {

constexpr int kShallow = 4;  // stages of a ring where three blocks share an SM
constexpr int kDeep = 6;     // and where no more than two do
constexpr float kWeightLog = 14.f;   // log2 of the largest weight, as stored
constexpr int kLeastScaleLog = -90;  // a scale's log2, as far as the reference m follows it

template <int D, int NT, int kSt>
struct LayoutB8 {
  static constexpr int kStages = kSt;
  static constexpr int kTileBytes = kTileKeys * D;
  static constexpr int kStageBytes = 2 * kTileBytes + 16;  // K, V, the tile's scales (two floats)
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kRingBytes = kWarps * kWarpBytes;
  static constexpr int kWmlBytes = kWarps * 8 * NT * 8;
  static constexpr int kPartBytes = 8 * NT * D * 4;
  static constexpr int kMlBytes = kMaxParts * 8 * NT * 8;
  static constexpr int kBytes = kRingBytes + kWmlBytes + kPartBytes + kMlBytes + 16;  // + the arrival barrier, an abort flag
  static_assert(kWarpBytes >= 8 * NT * (D + 4) * 4, "the per-warp ring also holds the warp's partial output");
  static_assert(kRingBytes >= (kMaxRanked + 2) * 4, "the ranking by length borrows the ring");
};

// byte offset of a 16-byte chunk of a row inside a tile
template <int D>
__device__ __forceinline__ uint32_t chunk_at(int row, int chunk) {
  if constexpr (D == 128) return row * 128 + ((chunk ^ (row & 7)) << 4);
  const int line = row >> 1;
  return line * 128 + (((((row & 1) << 2) | chunk) ^ ((line & 3) << 1)) << 4);
}

__device__ __forceinline__ void cp_async_4(void* smem_dst, const void* gsrc) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem_dst)), "l"(gsrc) : "memory");
}

// four codes of a word -> two pairs of fp16: the A fragments of keys (K), or of one key pair's two dimensions (V, kHigh picks them)
template <bool I8>
__device__ __forceinline__ void word_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (I8) {
    const uint32_t u = w ^ 0x80808080u;
    lo = int8_to_half2<0x4140>(u);
    hi = int8_to_half2<0x4342>(u);
  } else {
    lo = e4m3_to_half2(w);
    hi = e4m3_to_half2(w >> 16);
  }
}

// What a warp keeps of one (sequence, kv head): the queries, and the running output, reference and sum.
template <int D, int NT>
struct WarpState {
  uint32_t qf[NT][D / 16][2];  // Q^T fragments (B operand), fp16
  float qs[NT][2];             // per column (heads 2 tq, 2 tq + 1): softmax scale * log2(e) * the power of two taken out of the queries
  float oacc[NT][D / 16][4];   // O^T
  float m_ref[NT][2], l_run[NT][2];  // reference maximum (log2 domain), this lane's share of the row sum
};

// Queries of kv head kvh of sequence b; step (u, i) of the first product holds dimensions 16 (2 tq + u) + 4 i + {0 .. 3} of lane tq
// (head_dim 64: 16 tq + 4 i).  The running values start anew.
template <int D, bool BF16, int NT>
__device__ __forceinline__ void start_pair(const DecodeB8Args& a, int b, int kvh, int lane, WarpState<D, NT>& w) {
  const int g0 = lane >> 2, tq = lane & 3;
  constexpr int kU = D / 64;
  const uint8_t* qb = reinterpret_cast<const uint8_t*>(a.q) + 2 * static_cast<int64_t>(b) * a.q_stride[0];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int g = g0 + 8 * n;
    const bool live = g < a.group;
    const uint8_t* qp = qb + 2 * static_cast<int64_t>(kvh * a.group + (live ? g : 0)) * a.q_stride[1];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(qp + 32 * (kU * tq + u) + 16 * h);
        w.qf[n][4 * u + 2 * h][0] = live ? x.x : 0u;
        w.qf[n][4 * u + 2 * h][1] = live ? x.y : 0u;
        w.qf[n][4 * u + 2 * h + 1][0] = live ? x.z : 0u;
        w.qf[n][4 * u + 2 * h + 1][1] = live ? x.w : 0u;
      }
    }
    float back = 1.f;  // of head g
    if constexpr (BF16) {
      uint32_t top = 0;  // largest magnitude, as bits
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) top = max(top, max(w.qf[n][s][e] & 0x7FFFu, (w.qf[n][s][e] >> 16) & 0x7FFFu));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      // the largest becomes 2^14 .. 2^15; exponents kept so that neither factor leaves fp32's range
      const int e = max(-113, min(110, 127 + 14 - static_cast<int>(top >> 7)));  // (-113: the largest finite exponent)
      const float f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      back = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2)
          w.qf[n][s][e2] = pack2<false>(__uint_as_float(w.qf[n][s][e2] << 16) * f, __uint_as_float(w.qf[n][s][e2] & 0xFFFF0000u) * f);
    }
    w.qs[n][0] = a.scale_log2 * __shfl_sync(0xFFFFFFFFu, back, 8 * tq);
    w.qs[n][1] = a.scale_log2 * __shfl_sync(0xFFFFFFFFu, back, 8 * tq + 4);
#pragma unroll
    for (int m = 0; m < D / 16; ++m) w.oacc[n][m][0] = w.oacc[n][m][1] = w.oacc[n][m][2] = w.oacc[n][m][3] = 0.f;
    w.m_ref[n][0] = w.m_ref[n][1] = -INFINITY;
    w.l_run[n][0] = w.l_run[n][1] = 0.f;
  }
}

// One tile of 16 keys that lies in a stage of the ring; the first `live` of them count.
template <int D, bool I8, int NT>
__device__ __forceinline__ void process_tile(const uint8_t* tk, int live, int lane, WarpState<D, NT>& w) {
  constexpr int kTileBytes = kTileKeys * D;
  constexpr int kU = D / 64;
  const int g0 = lane >> 2, tq = lane & 3;
  const uint8_t* tv = tk + kTileBytes;
  const float2 scales = *reinterpret_cast<const float2*>(tk + 2 * kTileBytes);
  // ---- S^T[16 keys x 8 heads] = K Q^T (two accumulators: half the chain of dependent MMAs) ----
  float s[NT][4], s2[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint4 x = *reinterpret_cast<const uint4*>(tk + chunk_at<D>(g0, kU * tq + u));
    const uint4 y = *reinterpret_cast<const uint4*>(tk + chunk_at<D>(g0 + 8, kU * tq + u));
    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t kf[4];
      word_to_half<I8>(xw[j], kf[0], kf[2]);
      word_to_half<I8>(yw[j], kf[1], kf[3]);
#pragma unroll
      for (int n = 0; n < NT; ++n) mma_16816<false>((j & 1) ? s2[n] : s[n], kf, w.qf[n][4 * u + j][0], w.qf[n][4 * u + j][1]);
    }
  }
  // ---- online softmax: x = t - m; 2^x times the scale has to stay within 2^14; a tile in which it does needs no reduction over
  // the lanes ----
  const bool dead0 = g0 >= live, dead1 = g0 + 8 >= live;
  const float room = kWeightLog - static_cast<float>(max(static_cast<int>((__float_as_uint(scales.y) + 0x7FFFFFu) >> 23) - 127, kLeastScaleLog));
  float x[NT][4];
  bool move = false;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const float f0 = w.qs[n][0] * scales.x, f1 = w.qs[n][1] * scales.x;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      s[n][e] = (s[n][e] + s2[n][e]) * ((e & 1) ? f1 : f0);
      if (e < 2 ? dead0 : dead1) s[n][e] = -INFINITY;
      x[n][e] = s[n][e] - w.m_ref[n][e & 1];  // +inf before the first tile (-inf - -inf: NaN, which moves nothing)
    }
    move |= fmaxf(fmaxf(x[n][0], x[n][1]), fmaxf(x[n][2], x[n][3])) > room;
  }
  if (__any_sync(0xFFFFFFFFu, move)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float alpha[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = fmaxf(s[n][h], s[n][2 + h]);
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 16));
        const float m_new = fmaxf(w.m_ref[n][h], mx - room);
        alpha[h] = ex2_approx(w.m_ref[n][h] - m_new);
        w.m_ref[n][h] = m_new;
        w.l_run[n][h] *= alpha[h];
      }
#pragma unroll
      for (int m = 0; m < D / 16; ++m) {
        w.oacc[n][m][0] *= alpha[0];
        w.oacc[n][m][1] *= alpha[1];
        w.oacc[n][m][2] *= alpha[0];
        w.oacc[n][m][3] *= alpha[1];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) x[n][e] = s[n][e] - w.m_ref[n][e & 1];
    }
  }
  uint32_t pb[NT][2];  // P^T fragments (B operand): keys 2 tq, 2 tq + 1 (+ 8) of head g0
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[n][e] = ex2_approx(x[n][e]);
    w.l_run[n][0] += x[n][0] + x[n][2];
    w.l_run[n][1] += x[n][1] + x[n][3];
    pb[n][0] = movmatrix_trans(pack2<false>(x[n][0] * scales.y, x[n][1] * scales.y));
    pb[n][1] = movmatrix_trans(pack2<false>(x[n][2] * scales.y, x[n][3] * scales.y));
  }

  // ---- O^T[D x 8 heads] += V^T P^T: lane (g0, tq) reads D / 8 dimensions of its four keys and interleaves the keys pairwise; rows g0 and
  // g0 + 8 of 16-row tile m are dimensions (D / 8) g0 + 2 m and + 1 ----
  constexpr int kVWords = D / 32;
  uint32_t vw[4][kVWords];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 2 * tq + (r & 1) + 8 * (r >> 1);
    if constexpr (D == 128) {
      const uint4 y = *reinterpret_cast<const uint4*>(tv + chunk_at<D>(row, g0));
      vw[r][0] = y.x;
      vw[r][1] = y.y;
      vw[r][2] = y.z;
      vw[r][3] = y.w;
    } else {
      const uint2 y = *reinterpret_cast<const uint2*>(tv + chunk_at<D>(row, g0 >> 1) + 8 * (g0 & 1));
      vw[r][0] = y.x;
      vw[r][1] = y.y;
    }
  }
#pragma unroll
  for (int m = 0; m < D / 16; ++m) {
    const int j = m >> 1;
    uint32_t vf[4];
    word_to_half<I8>(__byte_perm(vw[0][j], vw[1][j], (m & 1) ? 0x7362 : 0x5140), vf[0], vf[1]);
    word_to_half<I8>(__byte_perm(vw[2][j], vw[3][j], (m & 1) ? 0x7362 : 0x5140), vf[2], vf[3]);
#pragma unroll
    for (int n = 0; n < NT; ++n) mma_16816<false>(w.oacc[n][m], vf, pb[n][0], pb[n][1]);
  }
}

// Sums the lanes' shares of the row sums; every lane of a column then holds its sum.
template <int D, int NT>
__device__ __forceinline__ void finish_pair(WarpState<D, NT>& w) {
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w.l_run[n][h] += __shfl_xor_sync(0xFFFFFFFFu, w.l_run[n][h], 4);
      w.l_run[n][h] += __shfl_xor_sync(0xFFFFFFFFu, w.l_run[n][h], 8);
      w.l_run[n][h] += __shfl_xor_sync(0xFFFFFFFFu, w.l_run[n][h], 16);
    }
}

// head g = 8 n + 2 tq + h of the pair: this lane's D / 8 dimensions, from (D / 8) g0 on, to `row` (a row of D floats)
template <int D, int NT>
__device__ __forceinline__ void store_partial(const WarpState<D, NT>& w, int n, int h, float* row, int g0) {
#pragma unroll
  for (int m = 0; m < D / 16; m += 2)
    *reinterpret_cast<float4*>(row + (D / 8) * g0 + 2 * m) = make_float4(w.oacc[n][m][h], w.oacc[n][m][2 + h], w.oacc[n][m + 1][h], w.oacc[n][m + 1][2 + h]);
}

// Asynchronous copies of one tile into a stage: `k`, `v` point to this lane's chunk of its first row, `live` rows from that row on exist.
template <int D>
__device__ __forceinline__ void copy_tile(uint8_t* stage, const uint8_t* k, const uint8_t* v, int64_t load_step, int live, int l_row, int l_chunk,
                                          const void* safe_k, const void* safe_v) {
  constexpr int kRowsPerLoad = 32 / (D / 16);  // rows that one instruction of a warp brings
#pragma unroll
  for (int t = 0; t < kTileKeys / kRowsPerLoad; ++t) {
    const bool pred = t * kRowsPerLoad < live;  // rows beyond the sequence are not read and count as zeros
    const uint32_t at = chunk_at<D>(t * kRowsPerLoad + l_row, l_chunk);
    cp_async_16(stage + at, pred ? k : safe_k, pred);
    cp_async_16(stage + kTileKeys * D + at, pred ? v : safe_v, pred);
    k += load_step;
    v += load_step;
  }
}

template <int D, bool BF16, bool I8, bool Paged, int NT, int kSt>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 && kSt == kShallow ? 3 : 2) decode_b8_kernel(const DecodeB8Args a) {
  using L = LayoutB8<D, NT, kSt>;
  constexpr int kTileBytes = L::kTileBytes;
  constexpr int kWarpBytes = L::kWarpBytes;
  constexpr int kChunksPerRow = D / 16;
  constexpr int kRowsPerLoad = 32 / kChunksPerRow;           // rows that one instruction of a warp brings

  extern __shared__ __align__(128) uint8_t smem[];

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int kvh = blockIdx.y;
  const bool clustered = a.part_o == nullptr;
  const int part = blockIdx.x;
  const int n_parts = gridDim.x;

  uint64_t* arrived = reinterpret_cast<uint64_t*>(smem + L::kBytes - 16);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(arrived + 1);
  grid_launch_dependents();
  if (clustered && n_parts > 1) {
    if (tid == 0) {
      *abort_flag = 0;
      mbar_init(arrived, 1);
      mbar_fence_init();
      mbar_arrive_expect_tx(arrived, static_cast<uint32_t>(a.group * (D * 4 + n_parts * 8)));
    }
    __syncwarp();
    cluster_arrive();
  }
  grid_dependency_wait();

  int b = blockIdx.z, len;
  if (a.by_length) {
    const int2 x = sequence_by_length(a.lens, a.batch, a.max_len, b, reinterpret_cast<int*>(smem), tid);
    b = x.x;
    len = x.y;
  } else {
    len = max(0, min(a.lens[b], a.max_len));
  }
  // the keys of this block: an even share of the sequence's tiles
  // (quotient and remainder: the product of the tiles and a block's number passes 32 bits from 231 million keys on)
  const unsigned nt_seq = (static_cast<unsigned>(len) + kTileKeys - 1) / kTileKeys;
  const unsigned share = nt_seq / static_cast<unsigned>(n_parts), more = nt_seq - share * static_cast<unsigned>(n_parts);  // `more` blocks take one more
  const unsigned t0 = share * static_cast<unsigned>(part) + min(static_cast<unsigned>(part), more);
  const int c0 = static_cast<int>(min(static_cast<unsigned>(len), t0 * kTileKeys));
  const int c1 = static_cast<int>(min(static_cast<unsigned>(len), (t0 + share + (static_cast<unsigned>(part) < more ? 1u : 0u)) * kTileKeys));
  const int nt = (c1 - c0) / kTileKeys + ((c1 - c0) % kTileKeys != 0 ? 1 : 0);
  const int nt_w = (nt > warp) ? (nt - warp + kWarps - 1) / kWarps : 0;

  uint8_t* wsm = smem + warp * kWarpBytes;
  const int l_row = lane / kChunksPerRow, l_chunk = lane % kChunksPerRow;

  // This lane's first row and chunk of the tile to be fetched next, and the scale that it fetches (lane 0 of k's block, lane 1 of v's).  A contiguous
  // cache moves on by a fixed step; pages are looked up tile by tile (a tile lies in one).
  const int64_t lane_off = static_cast<int64_t>(kvh) * a.kv_stride[1] + static_cast<int64_t>(l_row) * a.kv_stride[2] + l_chunk * 16;
  const int64_t load_step = kRowsPerLoad * a.kv_stride[2];
  const float* scale_base = (lane == 0 ? a.k_scale : a.v_scale) + static_cast<int64_t>(kvh) * a.scale_stride[1];
  const int key_w = c0 + warp * kTileKeys;  // first key of this warp
  int64_t off = lane_off;
  if constexpr (!Paged) {
    off += static_cast<int64_t>(b) * a.kv_stride[0] + static_cast<int64_t>(key_w) * a.kv_stride[2];
    scale_base += static_cast<int64_t>(b) * a.scale_stride[0];
  }
  auto issue_tile = [&](int i) {  // i-th tile of this warp -> stage i % kSt; called for i = 0, 1, 2, ...
    if (i < nt_w) {
      const int key0 = key_w + i * (kWarps * kTileKeys);
      int64_t soff;
      if constexpr (Paged) {
        const int slot = key0 / a.page_size;
        int page = a.block_table[static_cast<size_t>(b) * a.table_stride + slot];
        if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.n_pages)) {
          if (lane == 0) report_bad_page(a.status, b, slot, page);
          page = 0;
        }
        const int row = key0 - slot * a.page_size;
        off = lane_off + static_cast<int64_t>(page) * a.kv_stride[0] + static_cast<int64_t>(row) * a.kv_stride[2];
        soff = static_cast<int64_t>(page) * a.scale_stride[0] + (row >> a.log_block);
      } else {
        soff = key0 >> a.log_block;
      }
      uint8_t* dst_k = wsm + (i % kSt) * L::kStageBytes;
      copy_tile<D>(dst_k, reinterpret_cast<const uint8_t*>(a.k) + off, reinterpret_cast<const uint8_t*>(a.v) + off, load_step, c1 - key0 - l_row, l_row, l_chunk, a.k, a.v);
      if (lane < 2) cp_async_4(dst_k + 2 * kTileBytes + 4 * lane, scale_base + soff);
      if constexpr (!Paged) off += (kWarps * kTileKeys) * a.kv_stride[2];
    }
    cp_async_commit();
  };

  if (a.by_length) __syncthreads();  // the ranking's scratch is the ring's memory
#pragma unroll
  for (int s = 0; s < kSt - 1; ++s) issue_tile(s);

  WarpState<D, NT> w;
  start_pair<D, BF16, NT>(a, b, kvh, lane, w);
  for (int i = 0; i < nt_w; ++i) {
    cp_async_wait<kSt - 2>();
    __syncwarp();
    issue_tile(i + kSt - 1);
    process_tile<D, I8, NT>(wsm + (i % kSt) * L::kStageBytes, c1 - key_w - i * (kWarps * kTileKeys), lane, w);
  }
  cp_async_wait<0>();
  finish_pair<D, NT>(w);
  __syncthreads();

  // ---- this warp's partial output into its part of the ring ----
  float* mo = reinterpret_cast<float*>(wsm);
  float2* wml = reinterpret_cast<float2*>(smem + L::kRingBytes);
  const int g0 = lane >> 2, tq = lane & 3;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int g = 8 * n + 2 * tq + h;
      if (g < a.group) {
        store_partial<D, NT>(w, n, h, mo + g * (D + 4), g0);
        if (g0 == 0) wml[warp * 8 * NT + g] = make_float2(w.m_ref[n][h], w.l_run[n][h]);
      }
    }
  merge_partials<D, BF16, NT, L, true>(a, smem, arrived, abort_flag, b, kvh, part, n_parts, clustered, tid);
}

// Grid (n_heads, batch), where the blocks of a pair are too many for a cluster: adds up the n_split partial outputs of one head.  A problem of
// latencies: the maximum, then the weights over all threads, then the outputs over all warps, four loads in flight.
constexpr int kMergeWarps = 8;
constexpr int kMaxSplit = 2 * 148;

template <int D, bool BF16>
__global__ void __launch_bounds__(32 * kMergeWarps) decode_b8_merge_kernel(const DecodeB8Args a) {
  constexpr int kLanes = D / 4, kSide = 32 / kLanes;  // lanes per partial output, outputs side by side in a warp
  __shared__ float s_w[kMaxSplit];
  __shared__ __align__(16) float4 s_o[kMergeWarps * kSide][kLanes];
  __shared__ float s_f[2][kMergeWarps];
  const int h = blockIdx.x, b = blockIdx.y;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const size_t p0 = (static_cast<size_t>(b) * a.n_heads + h) * a.n_split;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + p0;
  grid_launch_dependents();
  grid_dependency_wait();
  float M = -INFINITY;
  for (int i = tid; i < a.n_split; i += 32 * kMergeWarps) M = fmaxf(M, ml[i].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, d));
  if (lane == 0) s_f[0][warp] = M;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kMergeWarps; ++v) M = fmaxf(M, s_f[0][v]);
  float l = 0.f;
  for (int i = tid; i < a.n_split; i += 32 * kMergeWarps) {
    const float2 x = ml[i];
    const float f = x.x == -INFINITY ? 0.f : ex2_approx(x.x - M);
    s_w[i] = f;
    l += f * x.y;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, d);
  if (lane == 0) s_f[1][warp] = l;
  __syncthreads();
  l = 0.f;
#pragma unroll
  for (int v = 0; v < kMergeWarps; ++v) l += s_f[1][v];
  const int sub = lane / kLanes, t = lane % kLanes;
  const float4* po = reinterpret_cast<const float4*>(a.part_o) + p0 * kLanes + t;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp * kSide + sub; i < a.n_split; i += kMergeWarps * kSide) {
    const float4 x = po[static_cast<size_t>(i) * kLanes];
    const float f = s_w[i];
    o.x += f * x.x;
    o.y += f * x.y;
    o.z += f * x.z;
    o.w += f * x.w;
  }
  s_o[warp * kSide + sub][t] = o;
  __syncthreads();
  if (tid < kLanes) {
    o = s_o[0][tid];
#pragma unroll
    for (int v = 1; v < kMergeWarps * kSide; ++v) {
      const float4 x = s_o[v][tid];
      o.x += x.x;
      o.y += x.y;
      o.z += x.z;
      o.w += x.w;
    }
    const float inv = 1.f / l;
    uint8_t* op = reinterpret_cast<uint8_t*>(a.out) + 2 * (static_cast<int64_t>(b) * a.out_stride[0] + static_cast<int64_t>(h) * a.out_stride[1]);
    uint2 r = make_uint2(0u, 0u);
    if (!no_result<true>(l)) r = make_uint2(pack2<BF16>(o.x * inv, o.y * inv), pack2<BF16>(o.z * inv, o.w * inv));
    *reinterpret_cast<uint2*>(op + 8 * tid) = r;
  }
}

// set-once function attributes per device; the attribute calls themselves are idempotent
template <class F>
cudaError_t once_per_device(std::atomic<bool> (&done)[64], F&& set) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !done[dev].load(std::memory_order_acquire)) {
    e = set();
    if (e != cudaSuccess) return e;
    if (dev < 64) done[dev].store(true, std::memory_order_release);
  }
  return cudaSuccess;
}

template <int D, bool BF16, bool I8, bool Paged, int NT, int kSt>
cudaError_t launch_ring(const DecodeB8Args& a, cudaStream_t stream) {
  auto* kernel = decode_b8_kernel<D, BF16, I8, Paged, NT, kSt>;
  constexpr int smem = LayoutB8<D, NT, kSt>::kBytes;
  static std::atomic<bool> done[64] = {};
  cudaError_t e = once_per_device(done, [&] {
    const cudaError_t x = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    return x != cudaSuccess ? x : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  if (e != cudaSuccess) return e;
  const bool clustered = a.part_o == nullptr;
  LaunchAttrs at(stream);
  at.cfg.gridDim = dim3(a.n_split, a.n_kv_heads, a.batch);
  at.cfg.blockDim = dim3(kWarps * 32);
  at.cfg.dynamicSmemBytes = smem;
  if (clustered && a.n_split > 1) at.cluster(a.n_split);
  e = cudaLaunchKernelEx(&at.cfg, kernel, a);
  if (e != cudaSuccess || clustered) return e;
  LaunchAttrs ac(stream);
  ac.cfg.gridDim = dim3(a.n_heads, a.batch);
  ac.cfg.blockDim = dim3(32 * kMergeWarps);
  return cudaLaunchKernelEx(&ac.cfg, decode_b8_merge_kernel<D, BF16>, a);
}

template <int D, bool BF16, bool I8, bool Paged, int NT>
cudaError_t launch_heads(const DecodeB8Args& a, cudaStream_t stream) {
  return a.deep ? launch_ring<D, BF16, I8, Paged, NT, kDeep>(a, stream) : launch_ring<D, BF16, I8, Paged, NT, kShallow>(a, stream);
}

template <int D, bool BF16, bool I8>
cudaError_t launch_one(const DecodeB8Args& a, cudaStream_t stream) {
  if (a.group <= 8)
    return a.block_table != nullptr ? launch_heads<D, BF16, I8, true, 1>(a, stream) : launch_heads<D, BF16, I8, false, 1>(a, stream);
  return a.block_table != nullptr ? launch_heads<D, BF16, I8, true, 2>(a, stream) : launch_heads<D, BF16, I8, false, 2>(a, stream);
}

}  // namespace

cudaError_t launch_decode_b8(const DecodeB8Args& a, int head_dim, bool bf16, bool int8, cudaStream_t stream) {
  if (int8) {
    if (head_dim == 128) return bf16 ? launch_one<128, true, true>(a, stream) : launch_one<128, false, true>(a, stream);
    return bf16 ? launch_one<64, true, true>(a, stream) : launch_one<64, false, true>(a, stream);
  }
  if (head_dim == 128) return bf16 ? launch_one<128, true, false>(a, stream) : launch_one<128, false, false>(a, stream);
  return bf16 ? launch_one<64, true, false>(a, stream) : launch_one<64, false, false>(a, stream);
}

}  // namespace minfer_attn
