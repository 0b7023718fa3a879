// Paged decode attention over the 8-bit KV cache (format: mv_fp8.h), for
// gfx950: one query token per sequence, o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q k_j - m).
//
// Bound: HBM (14 flop per byte at 7 query heads per kv head), and on small
// batches the chain of memory round trips. The plan (fp8_decode_plan_kernel) gives
// one work group per (sequence, kv head, piece of its tokens).
//
// The codes go from memory to registers to the matrix cores, without shared
// memory, because both operand layouts can be loaded directly. A tile is 16
// tokens x D codes, one contiguous run of D * 16 bytes (a block holds at least
// 16 tokens, so a tile has one K and one V scale):
//   S^T = K Q^T (16x16x32 MFMAs, rows = tokens, columns = query heads): the K
//     operand's lane (g, t) wants 8 consecutive k (dims) of one token. The
//     order of the dims is free as long as Q has the same, so the lane takes 16
//     bytes of its token's row: two operands' worth.
//   O^T += V^T P^T (16x16x32, two tiles at once): the V operand's lane (g, t)
//     wants the values of 8 tokens at one dim. The lane loads 4 bytes (8 at D =
//     128) of the tokens g, 4 + g, 8 + g, 12 + g of each tile at dims 4t.. (8t..);
//     byte c of each, collected with v_perm, is the operand of MFMA c. Which
//     token and dim a row stands for is free: row r = 4 g + e of S^T is token
//     4 e + g of the tile, so the scores, packed to 16 bits, are the P operand
//     as they stand; and lane (g, t) ends up with head t's dims g D/4 .. + D/4.
// The scaled conversions make 16-bit operands of the codes, exactly.
// Softmax: one pass; a head's reference m moves (and O and l are rescaled)
// only where a lane's sum of p = exp2(s - m) would pass 4096.
// Measured (us a call, codes from HBM): 1 x 701 tokens at 14 / 2 x 64 5.3, 64 x
// 128-2048 9.3, 16 x 8k-32k 18.7 (4.3 TB/s), 128 x 512-4096 at 28 / 4 x 128 52.2 (6.0
// TB/s; 62.7 with pointer loads and accumulators in AGPRs, which were copied for
// every pair of tiles: two waves per SIMD are asked for, so that they stay in
// VGPRs). 8 or 16 waves a group and 3 or 4 pairs of tiles in flight gained nothing:
// a CU streams 40 KB per us either way.
#include <algorithm>
#include <climits>

#include "mv_coherent.h"
#include "mv_fp8.h"
#include "mv_tile.h"

namespace mv {
namespace {

constexpr int kDwPairs = 2;  // pairs of tiles in flight per wave
constexpr int kRsrcWord3 = 0x00020000;  // raw buffer, 32-bit data
constexpr int kStream = 2;              // non-temporal: every code is read once
constexpr int kDwWaves = 4;
constexpr float kDwFastMax = 4096.f;
constexpr float kDwStart = -3e38f;  // the reference before a head's first token

struct Fp8DecodeArgs {
  const int32_t* work;       // per work group: (seq, kv head, piece, pieces, token begin, end, 0, 0)
  const int32_t* block_ids;  // [work group][ids_per_item]: the piece's pool blocks first
  const char* q;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* scales;
  int64_t q_st, q_sh;  // bytes
  int32_t ids_per_item, num_kv_heads, n_rep, bs_log2;
  float scale_log2;  // scale * log2(e)
  int32_t num_q_heads, max_parts;
  uint32_t num_blocks;
  int32_t* counters;  // [num_seqs * num_kv_heads], zero at rest
  char* out;
  int64_t o_st, o_sh;  // bytes
  float* ws_o;         // [num_seqs, Hq, max_parts, D]: a piece's normalised rows
  float* ws_ml;        // [num_seqs, Hq, max_parts, 2]: (max, sum)
};

template <int DTYPE>
__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DTYPE == MV_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The codes of one tile as loaded: K, KL loads of 16 bytes; V, 4 tokens of D/16 bytes.
template <int D>
struct TileCodes {
  static constexpr int KL = D / 64, VW = D / 64;
  u32x4 k[KL];
  uint32_t v[4][VW];
};

template <int DTYPE, int D>
__global__ __launch_bounds__(kDwWaves * 64) __attribute__((amdgpu_waves_per_eu(2))) void fp8_decode_kernel(Fp8DecodeArgs a) {
  constexpr int W = kDwWaves, P = kDwPairs;
  constexpr int KS = D / 32;  // MFMA steps of K Q^T
  constexpr int C = D / 16;   // MFMAs of V^T P^T
  constexpr int VW = D / 64;
  constexpr int kORow = D + 4;
  constexpr int E = D / (4 * W);  // dims per thread of the merges: 4 W threads a head
  __shared__ __attribute__((aligned(16))) float s_o[W][16][kORow];
  __shared__ float s_m[W][16], s_l[W][16];
  __shared__ int s_last;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int t = lane & 15, g = lane >> 4;
  const int64_t item = blockIdx.x;

  // ---- the work item, and the block of this lane's tile: lane l of wave w
  // holds what tile w + 4 (j0 + l) of the piece needs, for 64 of the wave's
  // tiles at a time. With blocks of 16 tokens the first ids do not depend on
  // the work item, and travel with it.
  const int32_t* ids = a.block_ids + item * a.ids_per_item;
  const bool one = a.bs_log2 == 4;
  int id = 0;
  if (one) id = ids[min(wave + W * lane, a.ids_per_item - 1)];
  const int4 w0 = reinterpret_cast<const int4*>(a.work + 8 * item)[0];
  const int4 w1 = reinterpret_cast<const int4*>(a.work + 8 * item)[1];
  if (w0.x < 0) return;  // an unused slot of a launch of fixed size
  const int b = w0.x, h = w0.y, part = w0.z, n_parts = w0.w;
  const int tok_begin = w1.x, tok_end = w1.y;
  const int first_blk = tok_begin >> a.bs_log2;
  const int tiles = (tok_end - tok_begin + kTile - 1) / kTile;
  const int mine = (tiles - wave + W - 1) / W;  // this wave's tiles
  auto id_of = [&](int j) {  // (lanes past the wave's tiles take its last one's)
    const int tok = tok_begin + (wave + W * min(j, mine - 1)) * kTile;
    return ids[min((tok >> a.bs_log2) - first_blk, a.ids_per_item - 1)];
  };
  if (!one && mine > 0) id = id_of(lane);

  // ---- Q: lane (g, t) holds head t's dims in the order of the K operands
  // (columns past the group's heads repeat its last one and are not stored)
  u32x4 q[KS];
  {
    const char* row = a.q + b * a.q_st + (h * a.n_rep + min(t, a.n_rep - 1)) * a.q_sh;
#pragma unroll
    for (int s = 0; s < KS; ++s) q[s] = *reinterpret_cast<const u32x4*>(row + 2 * (64 * (s >> 1) + 16 * g + 8 * (s & 1)));
  }

  float m = kDwStart, l = 0.f;  // head t's reference; the lane's share of its sum
  f32x4 o[C];                   // o[c][i]: head t, dim (D / 16) (4 g + i) + c
#pragma unroll
  for (int c = 0; c < C; ++c) o[c] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint32_t k_lane = (4 * (t & 3) + (t >> 2)) * D + 16 * g;
  const uint32_t v_lane = g * D + (D / 16) * t;

  for (int j0 = 0; j0 < mine; j0 += 64) {
    const int nw = min(64, mine - j0);
    // an id outside the pool is never an address: its tiles read block 0 and
    // are masked
    const bool have = static_cast<uint32_t>(id) < a.num_blocks;
    // (lanes past the wave's tiles count as held: what they read is no id)
    const uint64_t have_mask = __builtin_amdgcn_ballot_w64(have || lane >= nw);
    const int64_t bh = static_cast<int64_t>(have ? id : 0) * a.num_kv_heads + h;
    const float2 s2 = reinterpret_cast<const float2*>(a.scales)[bh];
    // this lane's tile's place in the pools, in bytes
    const int my_tok = tok_begin + (wave + W * (j0 + lane)) * kTile;
    const uint64_t at = static_cast<uint64_t>((bh << a.bs_log2) + (my_tok & ((1 << a.bs_log2) - 1))) * D;
    const uint32_t at_lo = static_cast<uint32_t>(at), at_hi = static_cast<uint32_t>(at >> 32);
    if (j0 + 64 < mine) id = id_of(j0 + 64 + lane);

    // (a buffer descriptor per tile: a tile past the window's last has no bytes,
    // its loads return zeros without a memory access)
    auto load_tile = [&](int jw, TileCodes<D>& x) __attribute__((always_inline)) {
      const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(at_lo, jw & 63))) |
                          static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(at_hi, jw & 63))) << 32;
      const int bytes = jw < nw ? kTile * D : 0;
      const auto k = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.k_cache) + at, 0, bytes, kRsrcWord3);
      const auto v = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(a.v_cache) + at, 0, bytes, kRsrcWord3);
#pragma unroll
      for (int i = 0; i < TileCodes<D>::KL; ++i)
        x.k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(k, k_lane + 64 * i, 0, kStream));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (VW == 1) {
          x.v[e][0] = __builtin_amdgcn_raw_buffer_load_b32(v, v_lane + 4 * e * D, 0, kStream);
        } else {
          const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(v, v_lane + 4 * e * D, 0, kStream));
          x.v[e][0] = w[0];
          x.v[e][1] = w[1];
        }
      }
    };
    auto scores = [&](const TileCodes<D>& x, float ks) __attribute__((always_inline)) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < TileCodes<D>::KL; ++i) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x2 lo = fp8_unpack4<DTYPE>(x.k[i][2 * u], ks), hi = fp8_unpack4<DTYPE>(x.k[i][2 * u + 1], ks);
          s = mfma16<DTYPE>(u32x4{lo[0], lo[1], hi[0], hi[1]}, q[2 * i + u], s);
        }
      }
      return s;
    };
    // The V operand halves of a tile: out[c] = dim c's values of tokens 0 .. 3
    auto v_operands = [&](const TileCodes<D>& x, float vs, u32x2 (&out)[C]) __attribute__((always_inline)) {
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t a0 = __builtin_amdgcn_perm(x.v[1][w], x.v[0][w], 0x05010400);  // tokens 0, 1 of dims 0, 1
        const uint32_t a1 = __builtin_amdgcn_perm(x.v[1][w], x.v[0][w], 0x07030602);  // of dims 2, 3
        const uint32_t b0 = __builtin_amdgcn_perm(x.v[3][w], x.v[2][w], 0x05010400);
        const uint32_t b1 = __builtin_amdgcn_perm(x.v[3][w], x.v[2][w], 0x07030602);
        out[4 * w] = u32x2{fp8_unpack2<DTYPE, false>(a0, vs), fp8_unpack2<DTYPE, false>(b0, vs)};
        out[4 * w + 1] = u32x2{fp8_unpack2<DTYPE, true>(a0, vs), fp8_unpack2<DTYPE, true>(b0, vs)};
        out[4 * w + 2] = u32x2{fp8_unpack2<DTYPE, false>(a1, vs), fp8_unpack2<DTYPE, false>(b1, vs)};
        out[4 * w + 3] = u32x2{fp8_unpack2<DTYPE, true>(a1, vs), fp8_unpack2<DTYPE, true>(b1, vs)};
      }
    };
    // Tiles jw and jw + 1 of the window.
    auto pair = [&](int jw, TileCodes<D>& xa, TileCodes<D>& xb) __attribute__((always_inline)) {
      // (jw is even: tile jw + 1 is in the window; past the wave's last one it
      // lies past the piece's end)
      const int jb = jw + 1;
      const int tok_a = tok_begin + (wave + W * (j0 + jw)) * kTile;
      const int tok_b = tok_a + W * kTile;
      const float ka = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.x), jw));
      const float kb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.x), jb));
      const float va = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.y), jw));
      const float vb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.y), jb));
      f32x4 sa = scores(xa, ka), sb = scores(xb, kb);
      if (tok_b + kTile > tok_end || have_mask != ~uint64_t(0)) {
        const int end_a = (have_mask >> jw) & 1 ? tok_end : 0;
        const int end_b = (have_mask >> jb) & 1 ? tok_end : 0;
        // tokens that are not attended: score -inf, and V 0 (0 * NaN is NaN)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in_a = tok_a + 4 * e + g < end_a, in_b = tok_b + 4 * e + g < end_b;
          sa[e] = in_a ? sa[e] : kNegInf;
          sb[e] = in_b ? sb[e] : kNegInf;
#pragma unroll
          for (int w = 0; w < VW; ++w) {
            xa.v[e][w] = in_a ? xa.v[e][w] : 0;
            xb.v[e][w] = in_b ? xb.v[e][w] : 0;
          }
        }
      }
      auto ex = [&](float x) __attribute__((always_inline)) {
        return __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2, -m));
      };
      s16x4 pa, pb;
      float sum;
      auto weights = [&]() __attribute__((always_inline)) {
        float s0 = 0.f, s1 = 0.f;
        pa = pack_p<DTYPE>(ex(sa[0]), ex(sa[1]), ex(sa[2]), ex(sa[3]), s0);
        pb = pack_p<DTYPE>(ex(sb[0]), ex(sb[1]), ex(sb[2]), ex(sb[3]), s1);
        sum = s0 + s1;
      };
      weights();
      if (__builtin_amdgcn_ballot_w64(!(sum <= kDwFastMax)) != 0) {
        float mc = kNegInf;
#pragma unroll
        for (int e = 0; e < 4; ++e) mc = fmaxf(mc, fmaxf(sa[e], sb[e]));
        const float mn = fmaxf(m, rows_max(mc) * a.scale_log2);
        const float alpha = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[c][i] *= alpha;
        weights();
      }
      l += sum;
      u32x2 oa[C], ob[C];
      v_operands(xa, va, oa);
      v_operands(xb, vb, ob);
      const uint2 qa = __builtin_bit_cast(uint2, pa), qb = __builtin_bit_cast(uint2, pb);
      const u32x4 p = {qa.x, qa.y, qb.x, qb.y};
#pragma unroll
      for (int c = 0; c < C; ++c) o[c] = mfma16<DTYPE>(u32x4{oa[c][0], oa[c][1], ob[c][0], ob[c][1]}, p, o[c]);
    };

    // P pairs of tiles in flight: a pair's registers are loaded again as soon as it
    // is computed.
    TileCodes<D> x[2 * P];
#pragma unroll
    for (int i = 0; i < 2 * P; ++i) load_tile(i, x[i]);
    int jw = 0;
    for (; jw + 2 * P < nw; jw += 2 * P) {
#pragma unroll
      for (int i = 0; i < 2 * P; i += 2) {
        pair(jw + i, x[i], x[i + 1]);
        load_tile(jw + 2 * P + i, x[i]);
        load_tile(jw + 2 * P + i + 1, x[i + 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2 * P; i += 2)
      if (jw + i < nw) pair(jw + i, x[i], x[i + 1]);
  }

  // ---- merge the waves: thread (r, c) takes dims c E .. of head r
  l = rows_sum(l);
  if (!(l > 0.f)) m = kNegInf;  // saw no token (or NaN: kept in l)
  if (g == 0) {
    s_m[wave][t] = m;
    s_l[wave][t] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int x = 0; x < C; x += 4)
      *reinterpret_cast<float4*>(&s_o[wave][t][C * (4 * g + i) + x]) =
          make_float4(o[x][i], o[x + 1][i], o[x + 2][i], o[x + 3][i]);
  __syncthreads();
  const int r = threadIdx.x / (4 * W), c = threadIdx.x % (4 * W);
  const bool has_row = r < a.n_rep;
  float mx = kNegInf, sum = 0.f;
  float v[E];
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) mx = fmaxf(mx, s_m[w][r]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const float mw = s_m[w][r];
    const float f = mw == kNegInf ? (s_l[w][r] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mw - mx);
    sum += s_l[w][r] * f;
#pragma unroll
    for (int x = 0; x < E; x += 2) {
      const float2 y = *reinterpret_cast<const float2*>(&s_o[w][r][E * c + x]);
      v[x] += y.x * f;
      v[x + 1] += y.y * f;
    }
  }
  const float inv = 1.f / sum;
#pragma unroll
  for (int i = 0; i < E; ++i) v[i] *= inv;
  char* const dst = a.out + b * a.o_st + (h * a.n_rep + (has_row ? r : 0)) * a.o_sh + 2 * E * c;
  auto store_row = [&](const float (&y)[E]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < E; x += 2)
      *reinterpret_cast<uint32_t*>(dst + 2 * x) =
          static_cast<uint32_t>(from_f32<DTYPE>(y[x])) | static_cast<uint32_t>(from_f32<DTYPE>(y[x + 1])) << 16;
  };
  if (n_parts == 1) {
    if (has_row) store_row(v);
    return;
  }

  // ---- merge the pieces: every piece leaves its normalised row and (max,
  // sum) with device-coherent stores; the group that counts last folds them in
  // piece order, so the result does not depend on which one that is
  const int64_t slot0 = (static_cast<int64_t>(b) * a.num_q_heads + h * a.n_rep + (has_row ? r : 0)) * a.max_parts;
  if (has_row) {
    uint64_t* po = reinterpret_cast<uint64_t*>(a.ws_o + (slot0 + part) * D + E * c);
#pragma unroll
    for (int x = 0; x < E; x += 2) store_coherent_u64(po + x / 2, pack_f32x2(v[x], v[x + 1]));
    if (c == 0) store_coherent_u64(reinterpret_cast<uint64_t*>(a.ws_ml) + slot0 + part, pack_f32x2(mx, sum));
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(kWaitVmcnt0);  // every store of this wave is acknowledged
  __syncthreads();
  if (threadIdx.x == 0) {
    const int prev = __hip_atomic_fetch_add(&a.counters[b * a.num_kv_heads + h], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s_last = prev == n_parts - 1;
  }
  __syncthreads();
  if (!s_last) return;
  if (has_row) {
    float m_all = kNegInf, l_all = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = 0.f;
    // rounds of 16 pieces, every load of a round in flight before the first use
    constexpr int R = 16;
    for (int p0 = 0; p0 < n_parts; p0 += R) {
      uint64_t ml[R], ov[R][E / 2];
#pragma unroll
      for (int p = 0; p < R; ++p) {
        const int64_t slot = slot0 + min(p0 + p, n_parts - 1);
        ml[p] = load_coherent_u64(reinterpret_cast<const uint64_t*>(a.ws_ml) + slot);
        const uint64_t* src = reinterpret_cast<const uint64_t*>(a.ws_o + slot * D + E * c);
#pragma unroll
        for (int x = 0; x < E / 2; ++x) ov[p][x] = load_coherent_u64(src + x);
      }
      float m_new = m_all;
#pragma unroll
      for (int p = 0; p < R; ++p) m_new = fmaxf(m_new, unpack_lo(ml[p]));
      const float keep = m_all == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m_all - m_new);
      l_all *= keep;
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] *= keep;
#pragma unroll
      for (int p = 0; p < R; ++p) {
        const float w = p0 + p < n_parts ? unpack_hi(ml[p]) * __builtin_amdgcn_exp2f(unpack_lo(ml[p]) - m_new) : 0.f;
        l_all += w;
#pragma unroll
        for (int x = 0; x < E / 2; ++x) {
          v[2 * x] += w * unpack_lo(ov[p][x]);
          v[2 * x + 1] += w * unpack_hi(ov[p][x]);
        }
      }
      m_all = m_new;
    }
    const float inv_all = 1.f / l_all;
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] *= inv_all;
    store_row(v);
  }
  if (threadIdx.x == 0)  // ready for the next call
    __hip_atomic_store(&a.counters[b * a.num_kv_heads + h], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// ---------------------------------------------------------------- plan --
//
// Cuts each sequence's tokens into pieces of at most L tiles, one work group per
// (sequence, kv head, piece), and deals the groups to the CUs. Joining pieces
// costs a launch 2.4 us or more (three round trips to device-coherent memory), in
// which one group streams 100 KB, so L is chosen by an estimate of the launch's
// time; with C CUs, G groups and p pieces of a sequence in the mean, in us:
//   all     = all bytes / the rate at which a full launch reads (6.3 TB/s)
//   cu      = bytes of the busiest CU / the rate of one group (40 KB per us; 34 at
//             head_dim 128, whose K rows are read in half lines)
//   time(L) = (all^4 + cu^4)^(1/4) + (if any is cut: 2.4 + 0.18 (p - 1) G / C)
//             + 0.4 (groups per CU - 1)
// The busiest CU has the largest piece if there are at most C groups, that or
// the mean plus a few percent for up to 3 C (all of them resident, dealt by
// size), and what is left of the last rounds beyond. Fitted to 50 batches;
// measured (us a call): 64 x 1024 tokens at 14 / 2 x 64 uncut 7.4, in 2 pieces
// 8.5, in 4 9.2; 16 x 8k-32k one group per CU 19.8, two 21.6; 128 x 512-4096 at
// 28 / 4 x 128 uncut, two groups per CU 52, cut for three 63.5; 256 x
// lognormal(300) 11.3 cut for three, 25.8 uncut.
//
// One work group makes the plan. It is bound by its chain of barriers and
// reductions, so totals are taken in registers (lane permutes), a group finds its
// piece by bisection and its rank by counting sizes: 10-12 us for up to 128
// sequences and 512 groups, 20 for 1000 sequences (23-48 with atomics for the
// totals and every pair of groups compared), plus 4 for the id lists.
constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanDealt = 1024;    // groups of a launch that is dealt, at most
constexpr int kPlanSeqs = 4096;     // sequences whose lengths are kept in LDS
constexpr int kPlanMaxParts = 128;  // pieces of a sequence
constexpr int kPlanMinTiles = 4;    // tiles of a piece: one for each wave
constexpr float kHbmBytesPerUs = 6.3e6f;
constexpr float kMergeUs = 2.4f, kMergePartUs = 0.18f, kExtraGroupUs = 0.4f;

// ids per work group: the blocks a piece may touch, to a multiple of 4
__host__ __device__ inline int ids_stride(int64_t partition_tokens, int bs_log2) {
  return static_cast<int>((((partition_tokens + (1 << bs_log2) - 1) >> bs_log2) + 1 + 3) & ~int64_t(3));
}

struct Fp8DecodePlanArgs {
  const void* kv_len;
  const void* block_table;
  int64_t bt_stride, num_blocks;
  int32_t num_seqs, max_blocks, bs_log2, num_kv_heads, cu_count, fixed;
  int32_t kv_i64, bt_i64;
  float cu_bytes_per_us, tile_bytes;
  int32_t* work;
  int64_t max_groups;  // of any plan of this batch
  int64_t work_cap;    // entries of `work`
  int32_t* block_ids;
  int32_t* counters;
  int32_t* status;
};

__device__ __forceinline__ int64_t int_at(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// A reduction over the wave's lanes (all get it), and over groups of 16 lanes.
template <int CTRL>
__device__ __forceinline__ int dpp_lane(int x) {
  return __builtin_amdgcn_mov_dpp(x, CTRL, 0xf, 0xf, true);
}
template <class Op>
__device__ __forceinline__ int row_reduce(int x, Op op) {
  x = op(x, dpp_lane<0xb1>(x));     // lane ^ 1
  x = op(x, dpp_lane<0x4e>(x));     // lane ^ 2
  x = op(x, dpp_lane<0x141>(x));    // 7 - lane of 8
  return op(x, dpp_lane<0x140>(x)); // 15 - lane of 16
}
template <class Op>
__device__ __forceinline__ int wave_reduce(int x, Op op) {
  x = row_reduce(x, op);
  const auto r = __builtin_amdgcn_permlane16_swap(static_cast<uint32_t>(x), static_cast<uint32_t>(x), false, false);
  x = op(static_cast<int>(r[0]), static_cast<int>(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(static_cast<uint32_t>(x), static_cast<uint32_t>(x), false, false);
  return op(static_cast<int>(s[0]), static_cast<int>(s[1]));
}
struct Sum {
  __device__ int operator()(int a, int b) const { return a + b; }
};
struct Max {
  __device__ int operator()(int a, int b) const { return max(a, b); }
};
// The sum of the lanes up to and with this one.
__device__ __forceinline__ int wave_scan(int x, int lane) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const int y = __shfl_up(x, s);
    if (lane >= s) x += y;
  }
  return x;
}

// A sequence's tokens that are planned: 0 where its length is below 1 or past
// its table row (reported).
__device__ __forceinline__ int planned_tokens(const Fp8DecodePlanArgs& a, int64_t kv) {
  return kv < 1 || kv > (static_cast<int64_t>(a.max_blocks) << a.bs_log2) ? 0 : static_cast<int>(kv);
}
__device__ __forceinline__ int tiles_of(int tokens) { return (tokens + kTile - 1) / kTile; }

__global__ __launch_bounds__(kPlanThreads) void fp8_decode_plan_kernel(Fp8DecodePlanArgs a) {
  __shared__ int s_tokens[kPlanSeqs];       // of the first sequences
  __shared__ int s_red[6][kPlanWaves];      // totals of the waves
  __shared__ int4 s_try[kPlanWaves];        // a tried L, its groups / H, pieces, longest piece
  __shared__ float s_cost[kPlanWaves];
  __shared__ int s_first[kPlanThreads];     // a sequence's first piece; places by size
  __shared__ int4 s_item[2 * kPlanDealt];   // the groups to deal, as in the work list
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int H = a.num_kv_heads, C = a.cu_count;
  auto tokens = [&](int b) {
    return b < kPlanSeqs ? s_tokens[b] : planned_tokens(a, int_at(a.kv_len, a.kv_i64, b));
  };
  auto tiles = [&](int b) { return static_cast<uint32_t>(tiles_of(tokens(b))); };
  // ---- lengths: checks, all tiles, the most tiles of a sequence
  int red[6] = {0, 0, 0, 0, 0, -INT_MAX};  // tiles, most, sequences, too short, too long, -shortest
  for (int b = tid; b < a.num_seqs; b += kPlanThreads) {
    const int64_t kv = int_at(a.kv_len, a.kv_i64, b);
    const int n = planned_tokens(a, kv), t = tiles_of(n);
    if (b < kPlanSeqs) s_tokens[b] = n;
    red[0] += t;
    red[1] = max(red[1], t);
    red[2] += t > 0;
    red[3] += kv < 1;
    red[4] += kv > (static_cast<int64_t>(a.max_blocks) << a.bs_log2);
    red[5] = max(red[5], -static_cast<int>(kv < -INT_MAX ? -INT_MAX : kv > INT_MAX ? INT_MAX : kv));
  }
  for (int i = tid; i < a.num_seqs * H; i += kPlanThreads) a.counters[i] = 0;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const int v = k == 1 || k == 5 ? wave_reduce(red[k], Max()) : wave_reduce(red[k], Sum());
    if (lane == 0) s_red[k][wave] = v;
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const int v = s_red[k][lane & (kPlanWaves - 1)];
    red[k] = k == 1 || k == 5 ? row_reduce(v, Max()) : row_reduce(v, Sum());
  }
  __syncthreads();
  const int total = red[0], most = red[1];
  // ---- the piece bound L: every wave tries one, 16 over the whole range, then
  // 16 around the best
  int best = 1, groups = 0, parts = 1, longest = 1;
  if (most > 0) {
    const int least = min(most, max(kPlanMinTiles, (most + kPlanMaxParts - 1) / kPlanMaxParts));
    int hi = most, lo = least;
    for (int round = 0; round < 2; ++round) {
      int L;
      if (round == 0)
        L = static_cast<int>(most * __builtin_amdgcn_exp2f(__builtin_amdgcn_logf(static_cast<float>(least) / most) *
                                                            wave / (kPlanWaves - 1)) + 0.5f);
      else
        L = hi - static_cast<int>(static_cast<uint32_t>(hi - lo) * wave / (kPlanWaves - 1));
      L = min(max(L, least), most);
      int n = 0, np_most = 1, piece = 1;
      for (int b = lane; b < a.num_seqs; b += 64) {
        const uint32_t t = tiles(b);
        const uint32_t np = (t + L - 1) / static_cast<uint32_t>(L);
        n += np;
        np_most = max(np_most, static_cast<int>(np));
        if (np > 0) piece = max(piece, static_cast<int>((t + np - 1) / np));
      }
      n = wave_reduce(n, Sum());
      np_most = wave_reduce(np_most, Max());
      piece = wave_reduce(piece, Max());
      const float G = static_cast<float>(n) * H, mean = static_cast<float>(total) * H / C;
      float busiest = piece;
      if (G > 3.f * C) busiest = mean * 1.1f + piece;
      else if (G > C) busiest = fmaxf(busiest, mean * 1.05f);
      const float all = static_cast<float>(total) * H * a.tile_bytes / kHbmBytesPerUs;
      const float cu = busiest * a.tile_bytes / a.cu_bytes_per_us;
      float cost = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(all * all * all * all + cu * cu * cu * cu)) +
                   (np_most > 1 ? kMergeUs + kMergePartUs * (static_cast<float>(n) / red[2] - 1.f) * G / C : 0.f) +
                   kExtraGroupUs * fminf(ceilf(G / C) - 1.f, 3.f);
      if (static_cast<int64_t>(n) * H > a.max_groups) cost = 3e38f;
      if (lane == 0) {
        s_cost[wave] = cost;
        s_try[wave] = make_int4(L, n, np_most, piece);
      }
      __syncthreads();
      int at = 0;
      float least_cost = s_cost[0];
#pragma unroll
      for (int w = 1; w < kPlanWaves; ++w) {
        const float c = s_cost[w];
        at = c < least_cost ? w : at;  // (ties: the larger L)
        least_cost = fminf(c, least_cost);
      }
      const int4 x = s_try[at];
      best = x.x;
      groups = x.y * H;
      parts = x.z;
      longest = x.w;
      hi = s_try[max(at - 1, 0)].x;
      lo = s_try[min(at + 1, kPlanWaves - 1)].x;
      __syncthreads();
    }
  }
  // ---- the groups, in sequence order, 1024 sequences at a time; up to 3 C of
  // them (and what LDS holds) are dealt: by size, largest first, in snake order
  // over the CUs, on which group i and group i + C run
  const bool dealt = groups <= min(3 * C, kPlanDealt);
  int4* const work = reinterpret_cast<int4*>(a.work);
  for (int b0 = 0, base = 0; b0 < a.num_seqs; b0 += kPlanThreads) {
    const int nb = min(kPlanThreads, a.num_seqs - b0);
    const uint32_t mine = tid < nb ? tiles(b0 + tid) : 0;
    const int np = static_cast<int>((mine + best - 1) / static_cast<uint32_t>(best));
    const int incl = wave_scan(np, lane);  // pieces up to and with this sequence
    if (lane == 63) s_red[0][wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
      const int x = s_red[0][w];
      before += w < wave ? x : 0;
      all += x;
    }
    s_first[tid] = before + incl - np;
    __syncthreads();
    for (int i = tid; i < all * H; i += kPlanThreads) {
      const int p = static_cast<int>(static_cast<uint32_t>(i) / static_cast<uint32_t>(H)), h = i - p * H;
      int at = 0;  // the last sequence whose first piece is p or before
#pragma unroll
      for (int s = kPlanThreads / 2; s >= 1; s >>= 1)
        if (at + s < nb && s_first[at + s] <= p) at += s;
      const int b = b0 + at, j = p - s_first[at];
      const int len = tokens(b);
      const uint32_t t = tiles_of(len), m = (t + best - 1) / static_cast<uint32_t>(best);
      const int q = static_cast<int>(t / m), r = static_cast<int>(t - q * m);
      const int start = j * q + min(j, r), size = q + (j < r);
      const int4 e0 = make_int4(b, h, j, static_cast<int>(m));
      const int4 e1 = make_int4(start * kTile, min(len, (start + size) * kTile), 0, 0);
      // (never past the lists, whatever becomes of the lengths meanwhile)
      const int64_t slot = static_cast<int64_t>(base) * H + i;
      if (slot >= (dealt ? kPlanDealt : a.work_cap)) break;
      int4* const e = dealt ? s_item : work;
      e[2 * slot] = e0;
      e[2 * slot + 1] = e1;
    }
    base += all;
    __syncthreads();
  }
  if (dealt) {
    // ranks by counting: a place for every size of up to 1023 tiles (larger ones
    // share them); which of two equal groups comes first is of no consequence
    const float step = longest < kPlanThreads ? 1.f : static_cast<float>(kPlanThreads - 1) / longest;
    s_first[tid] = 0;
    __syncthreads();
    int4 e0, e1;
    int place = 0, in_place = 0;
    if (tid < groups) {
      e0 = s_item[2 * tid];
      e1 = s_item[2 * tid + 1];
      const int size = (e1.y - e1.x + kTile - 1) / kTile;
      place = kPlanThreads - 1 - min(kPlanThreads - 1, static_cast<int>(size * step));
      in_place = atomicAdd(&s_first[place], 1);
    }
    __syncthreads();
    const int n = s_first[tid], incl = wave_scan(n, lane);
    if (lane == 63) s_red[0][wave] = incl;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) before += w < wave ? s_red[0][w] : 0;
    s_first[tid] = before + incl - n;
    __syncthreads();
    if (tid < groups) {
      const int rank = s_first[place] + in_place;
      const int round = static_cast<int>(static_cast<uint32_t>(rank) / static_cast<uint32_t>(C)), pos = rank - round * C;
      const int in_round = min(C, groups - round * C);
      const int slot = round * C + ((round & 1) ? in_round - 1 - pos : pos);
      work[2 * slot] = e0;
      work[2 * slot + 1] = e1;
    }
  }
  if (a.fixed)
    for (int64_t i = groups + tid; i < a.work_cap; i += kPlanThreads)
      reinterpret_cast<int4*>(a.work)[2 * i] = make_int4(-1, 0, 0, 0);
  if (tid == 0) {
    a.status[MV_PLAN_NUM_ITEMS] = groups;
    a.status[MV_PLAN_BAD_KV_LEN] = red[3];
    a.status[MV_PLAN_INSUFFICIENT] = red[4];
    a.status[MV_PLAN_BAD_BLOCK] = 0;
    a.status[MV_PLAN_MAX_PARTS] = parts;
    a.status[MV_PLAN_MIN_KV_LEN] = a.num_seqs ? -red[5] : INT_MAX;
    a.status[MV_PLAN_PARTITION_TOKENS] = longest * kTile;
    a.status[MV_PLAN_IDS_PER_ITEM] =
        ids_stride(a.fixed ? static_cast<int64_t>(a.max_blocks) << a.bs_log2 : static_cast<int64_t>(longest) * kTile, a.bs_log2);
  }
}

// The pool blocks of every group's piece, a wave per group; an entry that is
// not a pool block becomes -1 (its tokens are masked) and is counted once, by kv
// head 0's piece that holds its first token.
__global__ __launch_bounds__(256) void fp8_decode_ids_kernel(Fp8DecodePlanArgs a) {
  const int64_t slot = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (slot >= a.status[MV_PLAN_NUM_ITEMS]) return;
  const int4 e0 = reinterpret_cast<const int4*>(a.work)[2 * slot], e1 = reinterpret_cast<const int4*>(a.work)[2 * slot + 1];
  const int first = e1.x >> a.bs_log2, n = ((e1.y - 1) >> a.bs_log2) - first + 1;
  int32_t* ids = a.block_ids + slot * a.status[MV_PLAN_IDS_PER_ITEM];
  int bad = 0;
  for (int i = lane; i < n; i += 64) {
    const int64_t blk = int_at(a.block_table, a.bt_i64, e0.x * a.bt_stride + first + i);
    const bool ok = blk >= 0 && blk < a.num_blocks;
    ids[i] = ok ? static_cast<int32_t>(blk) : -1;
    bad += !ok && e0.y == 0 && ((first + i) << a.bs_log2) >= e1.x;
  }
  bad = wave_reduce(bad, Sum());
  if (bad && lane == 0) atomicAdd(&a.status[MV_PLAN_BAD_BLOCK], bad);
}

size_t ws_rows_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t head_dim, int32_t max_parts) {
  const size_t n = static_cast<size_t>(num_seqs) * num_q_heads * max_parts * head_dim * 4;
  return (n + 255) / 256 * 256;
}

}  // namespace
}  // namespace mv

extern "C" int mv_fp8_decode_plan_bounds(int32_t num_seqs, int32_t max_blocks, int32_t block_size,
                                         int32_t num_kv_heads, int32_t cu_count, int32_t fixed, int64_t* out) {
  using namespace mv;
  if (!out) return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan_bounds: null out");
  if (num_seqs < 0 || max_blocks < 0 || num_kv_heads <= 0 || cu_count <= 0)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan_bounds: bad sizes");
  if (!is_pow2(block_size) || block_size < 16 || block_size > 256)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_decode_plan_bounds: block_size %d (a power of two from 16 to 256)", block_size);
  const int64_t units = static_cast<int64_t>(num_seqs) * num_kv_heads;
  const int64_t tokens = static_cast<int64_t>(max_blocks) * block_size;
  const int64_t tiles = (tokens + kTile - 1) / kTile;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(kPlanMaxParts, (tiles + kPlanMinTiles - 1) / kPlanMinTiles));
  const int64_t groups = std::min(units * parts, units + 3 * static_cast<int64_t>(cu_count));
  if (tokens > INT_MAX / 2 || groups > INT_MAX / 8 || static_cast<int64_t>(num_seqs) * tiles > INT_MAX)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan_bounds: batch too large");
  // ids: a launch of fixed size strides its lists by the whole table row; else
  // by pieces of L tiles, at most units + all tiles / L of them:
  // (units + units max_blocks bs / (16 L)) (16 L / bs + 8) with 16 L <= max_blocks bs
  const int64_t ids = fixed ? groups * ids_stride(tokens, ilog2_exact(block_size))
                            : 2 * units * max_blocks + 8 * (units + groups);
  out[0] = groups;
  out[1] = tokens;
  out[2] = parts;
  out[3] = ids;
  return MV_OK;
}

extern "C" int mv_fp8_decode_plan(const void* kv_len, int32_t kv_len_is_i64, const void* block_table,
                                  int32_t bt_is_i64, int64_t bt_stride, int32_t num_seqs, int32_t max_blocks,
                                  int32_t block_size, int64_t num_blocks, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t cu_count, int32_t fixed, int32_t* work_items, int64_t work_capacity,
                                  int32_t* block_ids, int64_t block_ids_capacity, int32_t* counters, int32_t* status,
                                  void* stream) {
  using namespace mv;
  int64_t need[4];
  const int rc = mv_fp8_decode_plan_bounds(num_seqs, max_blocks, block_size, num_kv_heads, cu_count, fixed, need);
  if (rc != MV_OK) return rc;
  if (head_dim != 64 && head_dim != 128)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_decode_plan: head_dim %d not supported (64, 128)", head_dim);
  if (!status || (num_seqs > 0 && (!kv_len || !counters || !work_items || !block_ids || (max_blocks > 0 && !block_table))))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan: null pointer");
  if (num_blocks <= 0 || num_blocks > INT_MAX || work_capacity < need[0] || block_ids_capacity < need[3])
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan: %lld blocks, capacities %lld and %lld (need %lld and %lld)",
                static_cast<long long>(num_blocks), static_cast<long long>(work_capacity),
                static_cast<long long>(block_ids_capacity), static_cast<long long>(need[0]),
                static_cast<long long>(need[3]));
  if (reinterpret_cast<uintptr_t>(work_items) % 16)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_decode_plan: work list not 16-byte aligned");
  Fp8DecodePlanArgs a;
  a.kv_len = kv_len;
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.num_blocks = num_blocks;
  a.num_seqs = num_seqs;
  a.max_blocks = max_blocks;
  a.bs_log2 = ilog2_exact(block_size);
  a.num_kv_heads = num_kv_heads;
  a.cu_count = cu_count;
  a.fixed = fixed;
  a.kv_i64 = kv_len_is_i64 != 0;
  a.bt_i64 = bt_is_i64 != 0;
  a.cu_bytes_per_us = head_dim == 64 ? 40e3f : 34e3f;
  a.tile_bytes = 2.f * kTile * head_dim;
  a.work = work_items;
  a.max_groups = need[0];
  a.work_cap = work_capacity;
  a.block_ids = block_ids;
  a.counters = counters;
  a.status = status;
  hipStream_t s = static_cast<hipStream_t>(stream);
  fp8_decode_plan_kernel<<<1, kPlanThreads, 0, s>>>(a);
  if (need[0] > 0) fp8_decode_ids_kernel<<<static_cast<unsigned>((need[0] + 3) / 4), 256, 0, s>>>(a);
  return check_launch("mv_fp8_decode_plan");
}

extern "C" size_t mv_fp8_paged_decode_workspace_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t head_dim,
                                                      int32_t max_partitions) {
  if (max_partitions <= 1 || num_seqs <= 0 || num_q_heads <= 0 || head_dim <= 0) return 0;
  return mv::ws_rows_bytes(num_seqs, num_q_heads, head_dim, max_partitions) +
         static_cast<size_t>(num_seqs) * num_q_heads * max_partitions * 8;
}

extern "C" int mv_fp8_paged_decode(const void* query, int64_t q_stride_tok, int64_t q_stride_head,
                                   const void* key_cache, const void* value_cache, const float* kv_scales,
                                   const int32_t* work_items, const int32_t* block_ids, int64_t block_ids_capacity,
                                   int32_t num_work_groups, int32_t partition_tokens, int32_t max_partitions,
                                   int32_t* counters, void* out, int64_t out_stride_tok, int64_t out_stride_head,
                                   float scale, int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads,
                                   int32_t head_dim, int32_t block_size, int64_t num_blocks, int32_t dtype,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mv;
  if (dtype != MV_DTYPE_F16 && dtype != MV_DTYPE_BF16)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_paged_decode: dtype %d (fp16 or bf16 rows)", dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_paged_decode: head_dim %d not supported (64, 128)", head_dim);
  if (!is_pow2(block_size) || block_size < 16 || block_size > 256)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_paged_decode: block_size %d (a power of two from 16 to 256)", block_size);
  if (num_seqs < 0 || num_work_groups < 0 || num_kv_heads <= 0 || num_q_heads <= 0 || num_blocks <= 0 ||
      num_q_heads % num_kv_heads || partition_tokens < 0 || max_partitions < 0)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: bad sizes");
  const int n_rep = num_q_heads / num_kv_heads;
  if (n_rep > 16)
    return fail(MV_ERR_UNSUPPORTED, "mv_fp8_paged_decode: %d query heads per kv head (max 16)", n_rep);
  if (num_work_groups == 0 || num_seqs == 0) return MV_OK;
  if (!query || !key_cache || !value_cache || !kv_scales || !work_items || !block_ids || !out)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: null pointer");
  const int bs_log2 = ilog2_exact(block_size);
  const int per_item = ids_stride(partition_tokens, bs_log2);
  if (static_cast<int64_t>(num_work_groups) * per_item > block_ids_capacity)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: %d work groups x %d block ids exceed capacity %lld",
                num_work_groups, per_item, static_cast<long long>(block_ids_capacity));
  if (num_work_groups > static_cast<int64_t>(max_partitions) * num_seqs * num_kv_heads)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: work list larger than the plan allows");
  const uintptr_t ptrs = reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(key_cache) |
                         reinterpret_cast<uintptr_t>(value_cache) | reinterpret_cast<uintptr_t>(work_items) |
                         reinterpret_cast<uintptr_t>(out);
  if (ptrs % 16 || ((q_stride_tok | q_stride_head | out_stride_tok | out_stride_head) * 2) % 16 ||
      reinterpret_cast<uintptr_t>(kv_scales) % 8)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: rows, caches or the work list not 16-byte aligned");
  Fp8DecodeArgs a;
  a.work = work_items;
  a.block_ids = block_ids;
  a.q = static_cast<const char*>(query);
  a.k_cache = static_cast<const uint8_t*>(key_cache);
  a.v_cache = static_cast<const uint8_t*>(value_cache);
  a.scales = kv_scales;
  a.q_st = 2 * q_stride_tok;
  a.q_sh = 2 * q_stride_head;
  a.ids_per_item = per_item;
  a.num_kv_heads = num_kv_heads;
  a.n_rep = n_rep;
  a.bs_log2 = bs_log2;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.num_q_heads = num_q_heads;
  a.max_parts = max_partitions;
  a.num_blocks = static_cast<uint32_t>(std::min<int64_t>(num_blocks, INT_MAX));
  a.counters = counters;
  a.out = static_cast<char*>(out);
  a.o_st = 2 * out_stride_tok;
  a.o_sh = 2 * out_stride_head;
  a.ws_o = nullptr;
  a.ws_ml = nullptr;
  if (max_partitions > 1) {
    const size_t need = mv_fp8_paged_decode_workspace_bytes(num_seqs, num_q_heads, head_dim, max_partitions);
    if (!workspace || workspace_bytes < need)
      return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: workspace %zu bytes, need %zu", workspace_bytes, need);
    if (reinterpret_cast<uintptr_t>(workspace) % 256 || !counters)
      return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_paged_decode: workspace not 256-byte aligned or null counters");
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                       ws_rows_bytes(num_seqs, num_q_heads, head_dim, max_partitions));
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  const unsigned grid = static_cast<unsigned>(num_work_groups);
  if (dtype == MV_DTYPE_F16) {
    if (head_dim == 64) fp8_decode_kernel<MV_DTYPE_F16, 64><<<grid, kDwWaves * 64, 0, s>>>(a);
    else fp8_decode_kernel<MV_DTYPE_F16, 128><<<grid, kDwWaves * 64, 0, s>>>(a);
  } else {
    if (head_dim == 64) fp8_decode_kernel<MV_DTYPE_BF16, 64><<<grid, kDwWaves * 64, 0, s>>>(a);
    else fp8_decode_kernel<MV_DTYPE_BF16, 128><<<grid, kDwWaves * 64, 0, s>>>(a);
  }
  return check_launch("mv_fp8_paged_decode");
}
