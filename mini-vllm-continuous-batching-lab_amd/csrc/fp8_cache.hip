// Append to the 8-bit KV cache, with the rotary embedding on the way, and the
// gather that reads it back (format: mv_fp8.h).
//
// A block's scale covers every row in the block, so an append is not a scatter
// of rows: all new rows of one (block, kv head) are taken together. The plan,
// made once per step and used by all layers, groups the step's tokens by
// block (fp8_write_plan_kernel); the write then gives each (touched block, kv
// head, K or V) to a group of threads:
//   a     = max |x| over the call's finite rows in the block
//   need  = the smallest 2^e >= a / 448, e >= -110
//   old   = 0 if the call writes place 0 of the block, else its scale
//   scale = max(old, need)
//   code  = rne(clamp(x) / scale) of a new row (NaN where x is not finite),
//           rne(code * old / scale) of the others where 0 < old < scale.
// A row at place 0 starts the block anew, so a sequence's codes do not depend
// on who held the block before. No atomics: every output has one writer and
// the maximum does not depend on an order.
#include <algorithm>
#include <climits>

#include "mv_fp8.h"
#include "mv_rope.h"

namespace mv {
namespace {

// ------------------------------------------------------------- the plan --
//
// items[i]: a touched block; table[i * block_size + o]: the token whose slot
// is place o of it, or -1. Built by inserting every token's block into a hash
// table (open addressing, at least twice as many entries as tokens) whose
// first inserter takes the next item. The order of the items depends on the
// atomics; nothing that is computed from them does. Up to 2048 tokens one work
// group does it in LDS in one launch; beyond, four launches over the tokens.
constexpr int kFp8PlanThreads = 1024;
constexpr int kFp8PlanSmall = 2048;  // tokens one work group plans in LDS

struct Fp8PlanArgs {
  const int64_t* slots;
  const int64_t* positions;  // null: not checked
  int64_t num_tokens, total_slots, max_positions;
  int32_t* items;
  int32_t* table;
  int32_t* status;  // out of range, repeated, positions out of range, items
  int32_t* keys;    // hash table (grid form): blocks, then items
  uint32_t mask;
  int32_t bs_log2;
};

__device__ __forceinline__ uint32_t hash_block(uint32_t b) {
  b ^= b >> 16;
  b *= 0x7feb352du;
  return b ^ (b >> 15);
}

// The entry of `block` in the table, claiming an empty one; *claimed says so.
__device__ __forceinline__ uint32_t insert_block(int32_t* keys, uint32_t mask, int32_t block, bool* claimed) {
  uint32_t h = hash_block(static_cast<uint32_t>(block)) & mask;
  *claimed = false;
  while (true) {  // (ends: the table has more entries than tokens)
    const int32_t seen = atomicCAS(&keys[h], -1, block);
    if (seen == -1) *claimed = true;
    if (seen == -1 || seen == block) return h;
    h = (h + 1) & mask;
  }
}

__global__ __launch_bounds__(kFp8PlanThreads) void fp8_write_plan_kernel(Fp8PlanArgs a) {
  __shared__ int32_t s_keys[2 * kFp8PlanSmall], s_item[2 * kFp8PlanSmall];
  __shared__ int32_t s_count[4];
  constexpr int kPer = kFp8PlanSmall / kFp8PlanThreads;
  const int tid = threadIdx.x;
  const int n = static_cast<int>(a.num_tokens);
  for (uint32_t i = tid; i <= a.mask; i += kFp8PlanThreads) s_keys[i] = -1;
  if (tid < 4) s_count[tid] = 0;
  __syncthreads();
  uint32_t at[kPer];
  int32_t off[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int t = i * kFp8PlanThreads + tid;
    off[i] = -1;
    at[i] = 0;
    if (t >= n) continue;
    if (a.positions) {
      const int64_t p = a.positions[t];
      if (p < 0 || p >= a.max_positions) atomicAdd(&s_count[2], 1);
    }
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.total_slots) {
      if (slot != -1) atomicAdd(&s_count[0], 1);
      continue;
    }
    const int32_t block = static_cast<int32_t>(slot >> a.bs_log2);
    off[i] = static_cast<int32_t>(slot & ((1 << a.bs_log2) - 1));
    bool claimed;
    at[i] = insert_block(s_keys, a.mask, block, &claimed);
    if (claimed) {
      const int32_t item = atomicAdd(&s_count[3], 1);
      s_item[at[i]] = item;
      a.items[item] = block;
    }
  }
  __syncthreads();
  const int64_t cells = static_cast<int64_t>(s_count[3]) << a.bs_log2;
  for (int64_t i = tid; i < cells; i += kFp8PlanThreads) a.table[i] = -1;
  // the cells' stores have reached the cache where the atomics below work
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (off[i] < 0) continue;
    const int64_t cell = (static_cast<int64_t>(s_item[at[i]]) << a.bs_log2) + off[i];
    if (atomicMax(&a.table[cell], i * kFp8PlanThreads + tid) >= 0) atomicAdd(&s_count[1], 1);
  }
  __syncthreads();
  if (tid < 4) a.status[tid] = s_count[tid];
}

// The same in four launches, for any number of tokens.
__global__ __launch_bounds__(256) void fp8_plan_clear_kernel(Fp8PlanArgs a) {
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i0 < 4) a.status[i0] = 0;
  for (int64_t i = i0; i <= a.mask; i += static_cast<int64_t>(gridDim.x) * 256) a.keys[i] = -1;
}
__global__ __launch_bounds__(256) void fp8_plan_insert_kernel(Fp8PlanArgs a) {
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < a.num_tokens;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    if (a.positions) {
      const int64_t p = a.positions[t];
      if (p < 0 || p >= a.max_positions) atomicAdd(&a.status[2], 1);
    }
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.total_slots) {
      if (slot != -1) atomicAdd(&a.status[0], 1);
      continue;
    }
    const int32_t block = static_cast<int32_t>(slot >> a.bs_log2);
    bool claimed;
    const uint32_t h = insert_block(a.keys, a.mask, block, &claimed);
    if (claimed) {
      const int32_t item = atomicAdd(&a.status[3], 1);
      a.keys[static_cast<int64_t>(a.mask) + 1 + h] = item;
      a.items[item] = block;
    }
  }
}
__global__ __launch_bounds__(256) void fp8_plan_fill_kernel(Fp8PlanArgs a) {
  const int64_t cells = static_cast<int64_t>(a.status[3]) << a.bs_log2;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < cells;
       i += static_cast<int64_t>(gridDim.x) * 256)
    a.table[i] = -1;
}
__global__ __launch_bounds__(256) void fp8_plan_place_kernel(Fp8PlanArgs a) {
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < a.num_tokens;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.total_slots) continue;
    const int32_t block = static_cast<int32_t>(slot >> a.bs_log2);
    uint32_t h = hash_block(static_cast<uint32_t>(block)) & a.mask;
    int32_t seen;  // (ends: the table has empty entries; the block was inserted)
    while ((seen = a.keys[h]) != block && seen != -1) h = (h + 1) & a.mask;
    if (seen == -1) continue;
    const int64_t cell = (static_cast<int64_t>(a.keys[static_cast<int64_t>(a.mask) + 1 + h]) << a.bs_log2) +
                         (slot & ((1 << a.bs_log2) - 1));
    if (atomicMax(&a.table[cell], static_cast<int32_t>(t)) >= 0) atomicAdd(&a.status[1], 1);
  }
}

uint32_t plan_entries(int64_t num_tokens) {
  uint32_t n = 64;
  while (n < 2 * num_tokens) n <<= 1;
  return n;
}

// ------------------------------------------------------------ the write --

struct Fp8WriteArgs {
  const char* q;  // rotated into q_out (null: no query)
  char* q_out;
  const char* k;
  char* k_out;  // the rotated key as well (null: not wanted)
  const char* v;
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* scales;
  const int32_t* items;
  const int32_t* table;
  const int32_t* status;  // status[3]: the number of items
  const int64_t* positions;
  const char* cos;  // null: nothing is rotated
  const char* sin;
  int64_t q_st, q_sh, qo_st, qo_sh, k_st, k_sh, ko_st, ko_sh, v_st, v_sh;  // bytes
  int64_t table_stride;  // bytes per cos / sin row
  int64_t max_positions, num_blocks;
  int32_t num_tokens, max_items, num_q_heads, num_kv_heads, bs_log2;
  int32_t write_groups;  // work groups of the cache write; those after it rotate rows
};

// n / d, n >= 0, d > 0: the 64-bit division (100 instructions) only where n needs
// it (a prompt's append 37.0 -> 36.0 us; the gather waits for its stores anyway).
__device__ __forceinline__ int64_t quotient(int64_t n, int d) {
  if ((n >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

template <int DTYPE>
__device__ __forceinline__ int64_t clamped_position(const Fp8WriteArgs& a, int64_t t) {
  const int64_t p = a.positions[t];
  return p < 0 ? 0 : (p >= a.max_positions ? a.max_positions - 1 : p);  // reported by the plan
}

// One chunk pair (dims c .. c + 7 and the same of the other half) rotated.
template <int DTYPE>
__device__ __forceinline__ void rotate_pair(const uint4 x1, const uint4 x2, const char* cr, const char* sr,
                                            int o1, int o2, uint4& y1, uint4& y2) {
  const uint4 c1 = *reinterpret_cast<const uint4*>(cr + o1), c2 = *reinterpret_cast<const uint4*>(cr + o2);
  const uint4 s1 = *reinterpret_cast<const uint4*>(sr + o1), s2 = *reinterpret_cast<const uint4*>(sr + o2);
  y1 = rotate_chunk<DTYPE>(x1, x2, c1, s1, true);
  y2 = rotate_chunk<DTYPE>(x2, x1, c2, s2, false);
}

// The query rows (and with k_out the key rows), rotated: a thread owns 8 pairs
// (d, d + D/2) of two heads of a token, which share the tables' values. (9 k
// tokens at 28 / 4 x 128, outputs not in a cache: 38.5 us with one head a thread,
// 36.8 with two, no better with four. Non-temporal stores take another 2 off, and
// give it back in the attention that reads the rows next.)
constexpr int kRotHeads = 2;

template <int DTYPE, int D>
__device__ __forceinline__ void rotate_rows(const Fp8WriteArgs& a, int group, int groups) {
  constexpr int kPer = D / 16;
  const int heads = a.num_q_heads + (a.k_out ? a.num_kv_heads : 0);
  const int sets = (heads + kRotHeads - 1) / kRotHeads;
  const int64_t total = static_cast<int64_t>(a.num_tokens) * sets * kPer;
  for (int64_t i = static_cast<int64_t>(group) * 256 + threadIdx.x; i < total; i += static_cast<int64_t>(groups) * 256) {
    const int c = static_cast<int>(i & (kPer - 1));
    const int64_t ts = i / kPer;
    const int64_t t = quotient(ts, sets);
    const int h0 = static_cast<int>(ts - t * sets) * kRotHeads;
    const int64_t row = clamped_position<DTYPE>(a, t) * a.table_stride;
    const int o1 = c * 16, o2 = o1 + D;
    const uint4 c1 = *reinterpret_cast<const uint4*>(a.cos + row + o1), c2 = *reinterpret_cast<const uint4*>(a.cos + row + o2);
    const uint4 s1 = *reinterpret_cast<const uint4*>(a.sin + row + o1), s2 = *reinterpret_cast<const uint4*>(a.sin + row + o2);
    uint4 x1[kRotHeads], x2[kRotHeads];
    char* y[kRotHeads];
#pragma unroll
    for (int k = 0; k < kRotHeads; ++k) {
      const int hh = min(h0 + k, heads - 1);
      const bool is_q = hh < a.num_q_heads;
      const int h = is_q ? hh : hh - a.num_q_heads;
      const char* x = is_q ? a.q + t * a.q_st + h * a.q_sh : a.k + t * a.k_st + h * a.k_sh;
      y[k] = is_q ? a.q_out + t * a.qo_st + h * a.qo_sh : a.k_out + t * a.ko_st + h * a.ko_sh;
      x1[k] = *reinterpret_cast<const uint4*>(x + o1);
      x2[k] = *reinterpret_cast<const uint4*>(x + o2);
    }
#pragma unroll
    for (int k = 0; k < kRotHeads; ++k) {
      if (h0 + k >= heads) break;
      *reinterpret_cast<uint4*>(y[k] + o1) = rotate_chunk<DTYPE>(x1[k], x2[k], c1, s1, true);
      *reinterpret_cast<uint4*>(y[k] + o2) = rotate_chunk<DTYPE>(x2[k], x1[k], c2, s2, false);
    }
  }
}

// 16 values of one row as they go into the cache: 8 dims from each half of
// the row of K (the rotary pairs), 16 dims in a row of V.
struct Row16 {
  uint4 lo, hi;
};

template <int DTYPE>
__device__ __forceinline__ float elem16(const Row16& r, int i) {
  const uint32_t w = (&(i < 8 ? r.lo : r.hi).x)[(i & 7) >> 1];
  return to_f32<DTYPE>(static_cast<uint16_t>(i & 1 ? w >> 16 : w));
}

__device__ __forceinline__ bool finite_bits(uint32_t abs_bits) { return abs_bits < 0x7f800000u; }

// max over the wave (all lanes get it)
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t x) {
  const uint32_t y = static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), CTRL, 0xf, 0xf, true));
  return x > y ? x : y;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t x) {
  x = dpp_umax<0xb1>(x);   // lane ^ 1
  x = dpp_umax<0x4e>(x);   // lane ^ 2
  x = dpp_umax<0x141>(x);  // 7 - lane of 8
  x = dpp_umax<0x140>(x);  // 15 - lane of 16
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = r[0] > r[1] ? r[0] : r[1];
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return s[0] > s[1] ? s[0] : s[1];
}

// A unit is one (touched block, kv head, K or V): block_size x D values, a
// thread holds 16 of one row. Units of up to 256 threads share a work group
// of 256 (FIT): one pass, the rows kept in registers between the maximum and
// the codes; larger ones go over the rows twice, the second time from the
// caches. A decode step's append is bound by the launch and four rounds of
// dependent loads (plan words; row, position and scale; cos and sin; codes
// that shrink): 3.0 us for one row at 14 / 2 x 64 with the query's rotation,
// 4.2 for 64 (3.25 and 4.45 with the plan's words in two rounds and the wave's
// maximum through LDS). A prompt's is bound by its bytes: 36.0 us for 166 MB (9 k
// tokens at 28 / 4 x 128, rotation and returned key), 4.6 TB/s, nine tenths of a
// large copy's rate; 30 where the outputs' memory is still in a cache.
template <int DTYPE, int D, bool FIT>
__device__ __forceinline__ void write_units(const Fp8WriteArgs& a) {
  constexpr int kPer = D / 16;  // threads per row
  __shared__ uint32_t s_max[4];
  const int unit_threads = kPer << a.bs_log2;  // a power of two, >= 64
  const int width = FIT ? unit_threads : 256;
  const int per_group = 256 / width;
  const int lt = threadIdx.x & (width - 1);
  const int sub = threadIdx.x / width;
  const int wave = threadIdx.x >> 6;
  const int64_t bound = static_cast<int64_t>(a.max_items) * a.num_kv_heads * 2;
  const float limit = fp8_limit<DTYPE>();
  // (every thread of the work group goes through the same number of rounds:
  // the barriers below)
  for (int64_t u0 = static_cast<int64_t>(blockIdx.x) * per_group; u0 < bound;
       u0 += static_cast<int64_t>(a.write_groups) * per_group) {
    const int64_t u = u0 + sub;
    const bool live = u < bound;
    const int j = static_cast<int>(u & 1);  // 0: K, 1: V
    const int64_t ih = live ? u >> 1 : 0;
    const int64_t item = quotient(ih, a.num_kv_heads);
    const int h = static_cast<int>(ih - item * a.num_kv_heads);
    // the plan's words in one round of loads, the number of items among them:
    // what lies behind the last item is read and not used
    const int32_t* tab = a.table + (item << a.bs_log2);
    const int64_t block = a.items[item];
    const int first = tab[0];
    int tok = FIT ? tab[lt / kPer] : 0;
    const int items = a.status[3];
    asm volatile("" : "+v"(tok) : "v"(first), "v"(static_cast<int>(block)), "s"(items));
    if (u0 >= static_cast<int64_t>(items) * a.num_kv_heads * 2) break;
    const bool ok = live && item < items && block >= 0 && block < a.num_blocks;
    const int64_t tile = (block * a.num_kv_heads + h) << a.bs_log2;
    float* const scale_at = a.scales + (block * a.num_kv_heads + h) * 2 + j;
    uint8_t* const cache = j ? a.v_cache : a.k_cache;
    const bool anew = first >= 0;
    const float old = ok && !anew ? *scale_at : 0.f;

    // the rows of this thread: row (it * width + lt) / kPer, piece lt % kPer
    auto token_of = [&](int i) { return tab[i / kPer]; };
    auto load_row = [&](int tok, int i) {
      Row16 x;
      const int c = i & (kPer - 1);
      if (j) {
        const char* src = a.v + tok * a.v_st + h * a.v_sh + c * 32;
        x.lo = *reinterpret_cast<const uint4*>(src);
        x.hi = *reinterpret_cast<const uint4*>(src + 16);
      } else {
        const char* src = a.k + tok * a.k_st + h * a.k_sh + c * 16;
        x.lo = *reinterpret_cast<const uint4*>(src);
        x.hi = *reinterpret_cast<const uint4*>(src + D);
        if (a.cos) {
          const int64_t row = clamped_position<DTYPE>(a, tok) * a.table_stride;
          uint4 y1, y2;
          rotate_pair<DTYPE>(x.lo, x.hi, a.cos + row, a.sin + row, c * 16, c * 16 + D, y1, y2);
          x.lo = y1;
          x.hi = y2;
        }
      }
      return x;
    };
    auto row_max = [&](const Row16& x) {
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t b = __float_as_uint(fminf(__builtin_fabsf(elem16<DTYPE>(x, e)), limit));
        const bool fin = finite_bits(__float_as_uint(elem16<DTYPE>(x, e)) & 0x7fffffffu);
        m = fin && b > m ? b : m;
      }
      return m;
    };

    Row16 x;
    uint32_t amax = 0;
    if constexpr (FIT) {
      if (!ok || tok >= a.num_tokens) tok = -1;
      if (tok >= 0) {
        x = load_row(tok, lt);
        amax = row_max(x);
      }
    } else {
      for (int i = lt; i < unit_threads; i += width) {
        const int tk = ok ? token_of(i) : -1;
        if (tk >= 0 && tk < a.num_tokens) {
          const uint32_t m = row_max(load_row(tk, i));
          amax = m > amax ? m : amax;
        }
      }
    }
    amax = wave_umax(amax);
    if (width > 64) {
      __syncthreads();  // (the round before is done with s_max)
      if ((threadIdx.x & 63) == 0) s_max[wave] = amax;
      __syncthreads();
      const int w0 = sub * (width >> 6);
      for (int w = 0; w < (width >> 6); ++w) amax = max(amax, s_max[w0 + w]);
    }
    const float need = exp2i(fp8_scale_exp(amax));
    const float scale = fmaxf(old, need);
    const float inv = exp2i(-static_cast<int>((__float_as_uint(scale) >> 23) & 0xff) + 127);
    const bool grow = old > 0.f && old < scale;
    const float ratio = old * inv;

    auto put = [&](const Row16& r, int tk, int i) {
      const int c = i & (kPer - 1);
      uint8_t* dst = cache + (tile + i / kPer) * D;
      if (tk >= 0) {
        float y[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float f = elem16<DTYPE>(r, e);
          const bool fin = finite_bits(__float_as_uint(f) & 0x7fffffffu);
          y[e] = fin ? fminf(fmaxf(f, -limit), limit) * inv : __uint_as_float(0x7fc00000u);
        }
        uint2 lo = make_uint2(fp8_pack(y[0], y[1], y[2], y[3]), fp8_pack(y[4], y[5], y[6], y[7]));
        uint2 hi = make_uint2(fp8_pack(y[8], y[9], y[10], y[11]), fp8_pack(y[12], y[13], y[14], y[15]));
        if (j) {
          *reinterpret_cast<uint4*>(dst + c * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          *reinterpret_cast<uint2*>(dst + c * 8) = lo;
          *reinterpret_cast<uint2*>(dst + c * 8 + D / 2) = hi;
        }
      } else if (grow) {
        uint4* p = reinterpret_cast<uint4*>(dst + c * 16);
        const uint4 w = *p;
        auto shrink = [&](uint32_t codes) {
          const auto f0 = __builtin_amdgcn_cvt_pk_f32_fp8(codes, false);
          const auto f1 = __builtin_amdgcn_cvt_pk_f32_fp8(codes, true);
          return fp8_pack(f0[0] * ratio, f0[1] * ratio, f1[0] * ratio, f1[1] * ratio);
        };
        *p = make_uint4(shrink(w.x), shrink(w.y), shrink(w.z), shrink(w.w));
      }
    };
    if (ok) {
      if constexpr (FIT) {
        put(x, tok, lt);
      } else {
        for (int i = lt; i < unit_threads; i += width) {
          int tk = token_of(i);
          if (tk >= a.num_tokens) tk = -1;
          Row16 r;
          if (tk >= 0) r = load_row(tk, i);
          put(r, tk, i);
        }
      }
      if (lt == 0) *scale_at = scale;
    }
  }
}

template <int DTYPE, int D, bool FIT>
__global__ __launch_bounds__(256) void fp8_kv_write_kernel(Fp8WriteArgs a) {
  if (static_cast<int>(blockIdx.x) < a.write_groups) write_units<DTYPE, D, FIT>(a);
  else rotate_rows<DTYPE, D>(a, blockIdx.x - a.write_groups, gridDim.x - a.write_groups);
}

// ----------------------------------------------------------- the gather --

// slots[t] of every prefix token (sequence by sequence), for the gather:
// bad[0] counts the tokens whose table entry is not a pool block (their slot
// is -1).
template <typename BT>
__global__ __launch_bounds__(256) void fp8_prefix_slots_kernel(const BT* bt, int64_t bt_stride, int32_t bt_rows,
                                                               int32_t max_blocks, const int64_t* seq_rows,
                                                               const int64_t* cu, int32_t num_seqs, int64_t total,
                                                               int32_t bs_log2, int64_t num_blocks, int64_t* slots,
                                                               int32_t* bad) {
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
       t += static_cast<int64_t>(gridDim.x) * 256) {
    int lo = 0, hi = num_seqs - 1;  // the last sequence that starts at t or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cu[mid] <= t) lo = mid;
      else hi = mid - 1;
    }
    const int64_t pos = t - cu[lo], row = seq_rows[lo], entry = pos >> bs_log2;
    int64_t blk = -1;
    if (row >= 0 && row < bt_rows && entry < max_blocks) blk = static_cast<int64_t>(bt[row * bt_stride + entry]);
    const bool ok = blk >= 0 && blk < num_blocks;
    if (!ok) atomicAdd(bad, 1);
    slots[t] = ok ? (blk << bs_log2) + (pos & ((1 << bs_log2) - 1)) : -1;
  }
}
__global__ void fp8_zero_word_kernel(int32_t* p) {
  if (threadIdx.x == 0) *p = 0;
}

struct Fp8GatherArgs {
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* scales;
  const int64_t* slots;
  char* out_k;
  char* out_v;
  int64_t total, total_slots;
  int32_t num_kv_heads, bs_log2;
};

// out[t, h, :] = codes * scale; 16 codes a thread, rows outside the pool 0. Bound:
// its writes, twice the bytes read; 61152 tokens of 4 x 128 41 us (188 MB, 4.6 TB/s,
// nine tenths of a large copy's rate; 30-36 where the outputs' memory is still in
// a cache), 301 tokens of 2 x 64 2.2 (a launch). 8 codes a thread 57, K and V in
// one thread 40.7. Non-temporal stores: 37.5, but a copy of the rows right after
// then takes 5 us more.
template <int DTYPE, int D>
__global__ __launch_bounds__(256) void fp8_gather_kernel(Fp8GatherArgs a) {
  constexpr int kPer = D / 16;
  const int64_t per_tensor = a.total * a.num_kv_heads * kPer;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < 2 * per_tensor;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int j = i >= per_tensor;
    const int64_t r = j ? i - per_tensor : i;
    const int c = static_cast<int>(r & (kPer - 1));
    const int64_t row = r / kPer;
    const int64_t t = row / a.num_kv_heads;
    const int h = static_cast<int>(row - t * a.num_kv_heads);
    const int64_t slot = a.slots[t];
    u32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
    if (slot >= 0 && slot < a.total_slots) {
      const int64_t bh = (slot >> a.bs_log2) * a.num_kv_heads + h;
      const float scale = a.scales[2 * bh + j];
      const int64_t src = (bh << a.bs_log2) + (slot & ((1 << a.bs_log2) - 1));
      const uint4 w = *reinterpret_cast<const uint4*>((j ? a.v_cache : a.k_cache) + src * D + c * 16);
      if (scale > 0.f) {
        const u32x2 p0 = fp8_unpack4<DTYPE>(w.x, scale), p1 = fp8_unpack4<DTYPE>(w.y, scale);
        const u32x2 p2 = fp8_unpack4<DTYPE>(w.z, scale), p3 = fp8_unpack4<DTYPE>(w.w, scale);
        lo = u32x4{p0[0], p0[1], p1[0], p1[1]};
        hi = u32x4{p2[0], p2[1], p3[0], p3[1]};
      }
    }
    char* dst = (j ? a.out_v : a.out_k) + (row * D + c * 16) * 2;
    *reinterpret_cast<u32x4*>(dst) = lo;
    *reinterpret_cast<u32x4*>(dst + 16) = hi;
  }
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }

// What every entry point of the 8-bit cache checks of its pool.
int check_pool(const char* who, int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int64_t num_blocks,
               int32_t dtype) {
  if (dtype != MV_DTYPE_F16 && dtype != MV_DTYPE_BF16)
    return fail(MV_ERR_UNSUPPORTED, "%s: dtype %d (fp16 or bf16 rows)", who, dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(MV_ERR_UNSUPPORTED, "%s: head_dim %d not supported (64, 128)", who, head_dim);
  if (!is_pow2(block_size) || block_size < 16 || block_size > 256)
    return fail(MV_ERR_UNSUPPORTED, "%s: block_size %d (a power of two from 16 to 256)", who, block_size);
  if (num_kv_heads <= 0 || num_blocks <= 0 || num_blocks > INT_MAX)
    return fail(MV_ERR_INVALID_ARGUMENT, "%s: bad sizes", who);
  return MV_OK;
}

template <int DTYPE, int D>
void launch_write(const Fp8WriteArgs& a, int groups, hipStream_t s) {
  if (((D / 16) << a.bs_log2) <= 256) fp8_kv_write_kernel<DTYPE, D, true><<<groups, 256, 0, s>>>(a);
  else fp8_kv_write_kernel<DTYPE, D, false><<<groups, 256, 0, s>>>(a);
}

}  // namespace
}  // namespace mv

extern "C" size_t mv_fp8_write_plan_workspace_bytes(int64_t num_tokens) {
  if (num_tokens <= mv::kFp8PlanSmall || num_tokens > INT_MAX / 4) return 0;
  return static_cast<size_t>(mv::plan_entries(num_tokens)) * 8;
}

extern "C" int mv_fp8_write_plan(const int64_t* slot_mapping, int64_t num_tokens, int32_t block_size,
                                 int64_t num_blocks, const int64_t* positions, int64_t max_positions,
                                 int32_t* items, int32_t* table, int32_t* status, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  using namespace mv;
  const int rc = check_pool("mv_fp8_write_plan", 1, 64, block_size, num_blocks, MV_DTYPE_BF16);
  if (rc != MV_OK) return rc;
  if (num_tokens < 0 || num_tokens > INT_MAX / 4)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_write_plan: %lld tokens", static_cast<long long>(num_tokens));
  if (!status || (num_tokens > 0 && (!slot_mapping || !items || !table)))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_write_plan: null pointer");
  const size_t need = mv_fp8_write_plan_workspace_bytes(num_tokens);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_write_plan: workspace %zu bytes, need %zu", workspace_bytes, need);
  Fp8PlanArgs a;
  a.slots = slot_mapping;
  a.positions = positions;
  a.num_tokens = num_tokens;
  a.total_slots = num_blocks * block_size;
  a.max_positions = max_positions;
  a.items = items;
  a.table = table;
  a.status = status;
  a.keys = static_cast<int32_t*>(workspace);
  a.mask = plan_entries(num_tokens) - 1;
  a.bs_log2 = ilog2_exact(block_size);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (!need) {
    fp8_write_plan_kernel<<<1, kFp8PlanThreads, 0, s>>>(a);
  } else {
    const int groups = static_cast<int>(std::min<int64_t>((num_tokens + 255) / 256, 2048));
    fp8_plan_clear_kernel<<<groups, 256, 0, s>>>(a);
    fp8_plan_insert_kernel<<<groups, 256, 0, s>>>(a);
    fp8_plan_fill_kernel<<<groups, 256, 0, s>>>(a);
    fp8_plan_place_kernel<<<groups, 256, 0, s>>>(a);
  }
  return check_launch("mv_fp8_write_plan");
}

extern "C" int mv_fp8_kv_cache_write(
    const void* query, int64_t q_stride_tok, int64_t q_stride_head, void* query_out, int64_t qo_stride_tok,
    int64_t qo_stride_head, const void* key, int64_t k_stride_tok, int64_t k_stride_head, void* key_out,
    int64_t ko_stride_tok, int64_t ko_stride_head, const void* value, int64_t v_stride_tok, int64_t v_stride_head,
    void* key_cache, void* value_cache, float* kv_scales, const int32_t* items, const int32_t* table,
    const int32_t* plan_status, int32_t max_items, const int64_t* positions, const void* cos_table,
    const void* sin_table, int64_t table_stride, int64_t max_positions, int64_t num_tokens, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int64_t num_blocks, int32_t dtype, void* stream) {
  using namespace mv;
  const int rc = check_pool("mv_fp8_kv_cache_write", num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != MV_OK) return rc;
  const bool rope = cos_table != nullptr;
  if (num_tokens < 0 || num_tokens > INT_MAX / 4 || num_q_heads < 0 || max_items < 0 || (rope && max_positions <= 0))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_kv_cache_write: bad sizes");
  if (num_tokens == 0) return MV_OK;
  if (!key || !value || !key_cache || !value_cache || !kv_scales || !items || !table || !plan_status)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_kv_cache_write: null pointer");
  if (rope ? (!sin_table || !positions || (num_q_heads > 0 && (!query || !query_out)))
           : (num_q_heads > 0 || key_out != nullptr))
    return fail(MV_ERR_INVALID_ARGUMENT,
                "mv_fp8_kv_cache_write: rotation needs positions, both tables and the query's rows; without it "
                "there is no query and no key_out");
  // (the rows' groups and the cache's read the key at the same time)
  if (key_out && (key_out == key || key_out == value))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_kv_cache_write: key_out must not be the key's or the value's rows");
  const void* ptrs[] = {query, query_out, key, key_out, value, key_cache, value_cache, cos_table, sin_table};
  for (const void* p : ptrs)
    if (p && off16(p))
      return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_kv_cache_write: pointers must be 16-byte aligned");
  const int64_t strides[] = {q_stride_tok, q_stride_head, qo_stride_tok, qo_stride_head, k_stride_tok, k_stride_head,
                             ko_stride_tok, ko_stride_head, v_stride_tok, v_stride_head, table_stride};
  for (int64_t st : strides)
    if ((st * 2) % 16)
      return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_kv_cache_write: strides must be multiples of 16 bytes");
  Fp8WriteArgs a;
  a.q = static_cast<const char*>(query);
  a.q_out = static_cast<char*>(query_out);
  a.k = static_cast<const char*>(key);
  a.k_out = static_cast<char*>(key_out);
  a.v = static_cast<const char*>(value);
  a.k_cache = static_cast<uint8_t*>(key_cache);
  a.v_cache = static_cast<uint8_t*>(value_cache);
  a.scales = kv_scales;
  a.items = items;
  a.table = table;
  a.status = plan_status;
  a.positions = positions;
  a.cos = static_cast<const char*>(cos_table);
  a.sin = static_cast<const char*>(sin_table);
  a.q_st = 2 * q_stride_tok;
  a.q_sh = 2 * q_stride_head;
  a.qo_st = 2 * qo_stride_tok;
  a.qo_sh = 2 * qo_stride_head;
  a.k_st = 2 * k_stride_tok;
  a.k_sh = 2 * k_stride_head;
  a.ko_st = 2 * ko_stride_tok;
  a.ko_sh = 2 * ko_stride_head;
  a.v_st = 2 * v_stride_tok;
  a.v_sh = 2 * v_stride_head;
  a.table_stride = 2 * table_stride;
  a.max_positions = max_positions;
  a.num_blocks = num_blocks;
  a.num_tokens = static_cast<int32_t>(num_tokens);
  a.max_items = static_cast<int32_t>(std::min<int64_t>(max_items, num_tokens));
  a.num_q_heads = num_q_heads;
  a.num_kv_heads = num_kv_heads;
  a.bs_log2 = ilog2_exact(block_size);
  const int unit_threads = std::min(256, block_size * head_dim / 16);
  const int64_t write = (static_cast<int64_t>(a.max_items) * num_kv_heads * 2 * unit_threads + 255) / 256;
  a.write_groups = static_cast<int>(std::min<int64_t>(write, 8192));
  const int64_t heads = num_q_heads + (key_out ? num_kv_heads : 0);
  const int64_t rot = rope ? num_tokens * ((heads + kRotHeads - 1) / kRotHeads) * (head_dim / 16) : 0;
  const int groups = a.write_groups + static_cast<int>(std::min<int64_t>((rot + 255) / 256, 8192));
  if (groups == 0) return MV_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MV_DTYPE_F16) {
    if (head_dim == 64) launch_write<MV_DTYPE_F16, 64>(a, groups, s);
    else launch_write<MV_DTYPE_F16, 128>(a, groups, s);
  } else {
    if (head_dim == 64) launch_write<MV_DTYPE_BF16, 64>(a, groups, s);
    else launch_write<MV_DTYPE_BF16, 128>(a, groups, s);
  }
  return check_launch("mv_fp8_kv_cache_write");
}

extern "C" int mv_fp8_prefix_slots(const void* block_table, int32_t bt_is_i64, int64_t bt_stride, int32_t bt_rows,
                                   int32_t max_blocks, const int64_t* seq_rows, const int64_t* cu_tokens,
                                   int32_t num_seqs, int64_t total_tokens, int32_t block_size, int64_t num_blocks,
                                   int64_t* slots, int32_t* bad, void* stream) {
  using namespace mv;
  const int rc = check_pool("mv_fp8_prefix_slots", 1, 64, block_size, num_blocks, MV_DTYPE_BF16);
  if (rc != MV_OK) return rc;
  if (num_seqs < 0 || total_tokens < 0 || bt_rows < 0 || max_blocks < 0 || (num_seqs == 0 && total_tokens > 0))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_prefix_slots: bad sizes");
  if (!bad || (total_tokens > 0 && (!seq_rows || !cu_tokens || !slots || (bt_rows > 0 && max_blocks > 0 && !block_table))))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_prefix_slots: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  fp8_zero_word_kernel<<<1, 64, 0, s>>>(bad);
  if (total_tokens > 0) {
    const int groups = static_cast<int>(std::min<int64_t>((total_tokens + 255) / 256, 4096));
    const int bl = ilog2_exact(block_size);
    if (bt_is_i64)
      fp8_prefix_slots_kernel<int64_t><<<groups, 256, 0, s>>>(static_cast<const int64_t*>(block_table), bt_stride,
                                                              bt_rows, max_blocks, seq_rows, cu_tokens, num_seqs,
                                                              total_tokens, bl, num_blocks, slots, bad);
    else
      fp8_prefix_slots_kernel<int32_t><<<groups, 256, 0, s>>>(static_cast<const int32_t*>(block_table), bt_stride,
                                                              bt_rows, max_blocks, seq_rows, cu_tokens, num_seqs,
                                                              total_tokens, bl, num_blocks, slots, bad);
  }
  return check_launch("mv_fp8_prefix_slots");
}

extern "C" int mv_fp8_gather_kv(const void* key_cache, const void* value_cache, const float* kv_scales,
                                const int64_t* slots, int64_t total_tokens, void* out_key, void* out_value,
                                int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int64_t num_blocks,
                                int32_t dtype, void* stream) {
  using namespace mv;
  const int rc = check_pool("mv_fp8_gather_kv", num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != MV_OK) return rc;
  if (total_tokens < 0) return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_gather_kv: bad sizes");
  if (total_tokens == 0) return MV_OK;
  if (!key_cache || !value_cache || !kv_scales || !slots || !out_key || !out_value)
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_gather_kv: null pointer");
  if (off16(key_cache) || off16(value_cache) || off16(out_key) || off16(out_value))
    return fail(MV_ERR_INVALID_ARGUMENT, "mv_fp8_gather_kv: buffers not 16-byte aligned");
  Fp8GatherArgs a;
  a.k_cache = static_cast<const uint8_t*>(key_cache);
  a.v_cache = static_cast<const uint8_t*>(value_cache);
  a.scales = kv_scales;
  a.slots = slots;
  a.out_k = static_cast<char*>(out_key);
  a.out_v = static_cast<char*>(out_value);
  a.total = total_tokens;
  a.total_slots = num_blocks * block_size;
  a.num_kv_heads = num_kv_heads;
  a.bs_log2 = ilog2_exact(block_size);
  const int64_t work = 2 * total_tokens * num_kv_heads * (head_dim / 16);
  const int groups = static_cast<int>(std::min<int64_t>((work + 255) / 256, 65536));
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MV_DTYPE_F16) {
    if (head_dim == 64) fp8_gather_kernel<MV_DTYPE_F16, 64><<<groups, 256, 0, s>>>(a);
    else fp8_gather_kernel<MV_DTYPE_F16, 128><<<groups, 256, 0, s>>>(a);
  } else {
    if (head_dim == 64) fp8_gather_kernel<MV_DTYPE_BF16, 64><<<groups, 256, 0, s>>>(a);
    else fp8_gather_kernel<MV_DTYPE_BF16, 128><<<groups, 256, 0, s>>>(a);
  }
  return check_launch("mv_fp8_gather_kv");
}
