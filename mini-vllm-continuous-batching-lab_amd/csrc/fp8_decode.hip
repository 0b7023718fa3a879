// Paged decode attention over the 8-bit KV cache (format: mv_fp8.h), for
// gfx950: one query token per sequence, o = sum_j p_j v_j / sum_j p_j with
// p_j = exp(scale q k_j - m).
//
// Bound: HBM (14 flop per byte at 7 query heads per kv head), and on small
// batches the chain of memory round trips. The work list is the decode plan's
// (mv_decode_plan): one work group per (sequence, kv head, piece of its tokens).
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
#include <algorithm>
#include <climits>

#include "mv_coherent.h"
#include "mv_fp8.h"
#include "mv_tile.h"

namespace mv {
namespace {

constexpr int kDwWaves = 4;
constexpr int kDwThreads = kDwWaves * 64;
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
__global__ __launch_bounds__(kDwThreads) void fp8_decode_kernel(Fp8DecodeArgs a) {
  constexpr int KS = D / 32;  // MFMA steps of K Q^T
  constexpr int C = D / 16;   // MFMAs of V^T P^T
  constexpr int VW = D / 64;
  constexpr int kORow = D + 4;
  __shared__ __attribute__((aligned(16))) float s_o[kDwWaves][16][kORow];
  __shared__ float s_m[kDwWaves][16], s_l[kDwWaves][16];
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
  if (one) id = ids[min(wave + kDwWaves * lane, a.ids_per_item - 1)];
  const int4 w0 = reinterpret_cast<const int4*>(a.work + 8 * item)[0];
  const int4 w1 = reinterpret_cast<const int4*>(a.work + 8 * item)[1];
  if (w0.x < 0) return;  // an unused slot of a launch of fixed size
  const int b = w0.x, h = w0.y, part = w0.z, n_parts = w0.w;
  const int tok_begin = w1.x, tok_end = w1.y;
  const int first_blk = tok_begin >> a.bs_log2;
  const int tiles = (tok_end - tok_begin + kTile - 1) / kTile;
  const int mine = (tiles - wave + kDwWaves - 1) / kDwWaves;  // this wave's tiles
  auto id_of = [&](int j) {  // (lanes past the wave's tiles take its last one's)
    const int tok = tok_begin + (wave + kDwWaves * min(j, mine - 1)) * kTile;
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
    const int cur = have ? id : 0;
    const uint64_t have_mask = __builtin_amdgcn_ballot_w64(have);
    const float2 s2 = reinterpret_cast<const float2*>(a.scales)[static_cast<int64_t>(cur) * a.num_kv_heads + h];
    if (j0 + 64 < mine) id = id_of(j0 + 64 + lane);

    auto load_tile = [&](int jw, TileCodes<D>& x) __attribute__((always_inline)) {
      const int j = min(jw, nw - 1);
      const int64_t blk = __builtin_amdgcn_readlane(cur, j);
      const int tok = tok_begin + (wave + kDwWaves * (j0 + j)) * kTile;
      const int64_t at = (((blk * a.num_kv_heads + h) << a.bs_log2) + (tok & ((1 << a.bs_log2) - 1))) * D;
      const uint8_t* k = a.k_cache + at;
      const uint8_t* v = a.v_cache + at;
#pragma unroll
      for (int i = 0; i < TileCodes<D>::KL; ++i)
        x.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k + k_lane + 64 * i));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (VW == 1) {
          x.v[e][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(v + v_lane + 4 * e * D));
        } else {
          const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(v + v_lane + 4 * e * D));
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
      const int jb = min(jw + 1, 63);
      const int tok_a = tok_begin + (wave + kDwWaves * (j0 + jw)) * kTile;
      const int tok_b = tok_a + kDwWaves * kTile;
      const int end_a = (have_mask >> jw) & 1 ? tok_end : 0;
      const int end_b = jw + 1 < nw && ((have_mask >> jb) & 1) ? tok_end : 0;
      const float ka = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.x), jw));
      const float kb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.x), jb));
      const float va = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.y), jw));
      const float vb = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(s2.y), jb));
      f32x4 sa = scores(xa, ka), sb = scores(xb, kb);
      if (tok_a + kTile > end_a || tok_b + kTile > end_b) {
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

    // Two pairs of tiles in flight: a pair is loaded while the one before it
    // is computed. (Loads past the window's last tile repeat it.)
    TileCodes<D> x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) load_tile(i, x[i]);
    int jw = 0;
    for (; jw + 4 < nw; jw += 4) {
      pair(jw, x[0], x[1]);
      load_tile(jw + 4, x[0]);
      load_tile(jw + 5, x[1]);
      pair(jw + 2, x[2], x[3]);
      load_tile(jw + 6, x[2]);
      load_tile(jw + 7, x[3]);
    }
    pair(jw, x[0], x[1]);
    if (jw + 2 < nw) pair(jw + 2, x[2], x[3]);
  }

  // ---- merge the waves: thread (r, c) takes dims c D/16 .. of head r
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
  const int r = threadIdx.x >> 4, c = threadIdx.x & 15;
  const bool has_row = r < a.n_rep;
  float mx = kNegInf, sum = 0.f;
  float v[C];
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = 0.f;
#pragma unroll
  for (int w = 0; w < kDwWaves; ++w) mx = fmaxf(mx, s_m[w][r]);
#pragma unroll
  for (int w = 0; w < kDwWaves; ++w) {
    const float mw = s_m[w][r];
    const float f = mw == kNegInf ? (s_l[w][r] == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(mw - mx);
    sum += s_l[w][r] * f;
#pragma unroll
    for (int x = 0; x < C; x += 4) {
      const float4 y = *reinterpret_cast<const float4*>(&s_o[w][r][C * c + x]);
      v[x] += y.x * f;
      v[x + 1] += y.y * f;
      v[x + 2] += y.z * f;
      v[x + 3] += y.w * f;
    }
  }
  const float inv = 1.f / sum;
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] *= inv;
  char* const dst = a.out + b * a.o_st + (h * a.n_rep + (has_row ? r : 0)) * a.o_sh + 2 * C * c;
  auto store_row = [&](const float (&y)[C]) __attribute__((always_inline)) {
#pragma unroll
    for (int x = 0; x < C; x += 4) {
      uint32_t w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = static_cast<uint32_t>(from_f32<DTYPE>(y[x + 2 * i])) | static_cast<uint32_t>(from_f32<DTYPE>(y[x + 2 * i + 1])) << 16;
      *reinterpret_cast<uint2*>(dst + 2 * x) = make_uint2(w[0], w[1]);
    }
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
    uint64_t* po = reinterpret_cast<uint64_t*>(a.ws_o + (slot0 + part) * D + C * c);
#pragma unroll
    for (int x = 0; x < C; x += 2) store_coherent_u64(po + x / 2, pack_f32x2(v[x], v[x + 1]));
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
    for (int i = 0; i < C; ++i) v[i] = 0.f;
    // rounds of 8 pieces, every load of a round in flight before the first use
    constexpr int R = 512 / D;
    for (int p0 = 0; p0 < n_parts; p0 += R) {
      uint64_t ml[R], ov[R][C / 2];
#pragma unroll
      for (int p = 0; p < R; ++p) {
        const int64_t slot = slot0 + min(p0 + p, n_parts - 1);
        ml[p] = load_coherent_u64(reinterpret_cast<const uint64_t*>(a.ws_ml) + slot);
        const uint64_t* src = reinterpret_cast<const uint64_t*>(a.ws_o + slot * D + C * c);
#pragma unroll
        for (int x = 0; x < C / 2; ++x) ov[p][x] = load_coherent_u64(src + x);
      }
      float m_new = m_all;
#pragma unroll
      for (int p = 0; p < R; ++p) m_new = fmaxf(m_new, unpack_lo(ml[p]));
      const float keep = m_all == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m_all - m_new);
      l_all *= keep;
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] *= keep;
#pragma unroll
      for (int p = 0; p < R; ++p) {
        const float w = p0 + p < n_parts ? unpack_hi(ml[p]) * __builtin_amdgcn_exp2f(unpack_lo(ml[p]) - m_new) : 0.f;
        l_all += w;
#pragma unroll
        for (int x = 0; x < C / 2; ++x) {
          v[2 * x] += w * unpack_lo(ov[p][x]);
          v[2 * x + 1] += w * unpack_hi(ov[p][x]);
        }
      }
      m_all = m_new;
    }
    const float inv_all = 1.f / l_all;
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] *= inv_all;
    store_row(v);
  }
  if (threadIdx.x == 0)  // ready for the next call
    __hip_atomic_store(&a.counters[b * a.num_kv_heads + h], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

size_t ws_rows_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t head_dim, int32_t max_parts) {
  const size_t n = static_cast<size_t>(num_seqs) * num_q_heads * max_parts * head_dim * 4;
  return (n + 255) / 256 * 256;
}

// ids per work group, as mv_decode_plan lays the lists out
int ids_stride(int partition_tokens, int bs_log2) {
  return (((partition_tokens + (1 << bs_log2) - 1) >> bs_log2) + 1 + 3) & ~3;
}

}  // namespace
}  // namespace mv

extern "C" int mv_fp8_decode_groups_per_cu(int32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? 3 : 0;
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
    if (head_dim == 64) fp8_decode_kernel<MV_DTYPE_F16, 64><<<grid, kDwThreads, 0, s>>>(a);
    else fp8_decode_kernel<MV_DTYPE_F16, 128><<<grid, kDwThreads, 0, s>>>(a);
  } else {
    if (head_dim == 64) fp8_decode_kernel<MV_DTYPE_BF16, 64><<<grid, kDwThreads, 0, s>>>(a);
    else fp8_decode_kernel<MV_DTYPE_BF16, 128><<<grid, kDwThreads, 0, s>>>(a);
  }
  return check_launch("mv_fp8_paged_decode");
}
