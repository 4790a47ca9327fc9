// Attention over the paged 4-bit cache (format and arguments: include/tilemix_hip.h).
//
// A workgroup takes one (sequence, KV head), up to 16 RT of its query rows -- a row is a (query token,
// query head of the group) pair -- and one split of the keys.  Its four waves take the split's
// 64-key tiles in turn and join their running maxima, sums and outputs in LDS at the end; with
// several splits the parts go to the workspace and kv4_join_kernel adds them up.
//
// The mathematics of a tile, in fp32 but for the operands of the matrix instructions:
//   S^T = K Q^T          keys x rows, K's values fp16(n s + m) exactly as the cache defines them
//   p = exp2(S^T c - M)  c = sm_scale log2(e), M the row's running maximum less 7
//   O^T += V^T P^T       channels x rows
// p is rounded to fp16 for the second product (p <= 2^15, see kKv4Slack and kWeightUp; relative error 2^-11,
// as small as the output's own rounding), and the row sum adds the same rounded weights.
#include "kv4_common.h"

#include <algorithm>

namespace tmx {

namespace {

constexpr int kTile = 64;  // keys
constexpr int kWaves = 4;
constexpr int kChunkRT = 2, kChunkRows = kWaves * 16 * kChunkRT;  // query rows of a wave (in 16s), of a workgroup
// The running maximum is raised when a row exceeds it by this much (in powers of two): most
// tiles then leave the outputs unscaled.
constexpr float kKv4Slack = 8.0f;
// Weights are held 2^7 times too large, at most 2^15: then only those below 2^-32 of the largest vanish in fp16,
// and 131072 of them weigh less than its last place (from 2^-25 on 0.4% of a sum could be lost behind one
// large score).  Sums and outputs carry the same factor, which their quotient drops.
constexpr float kWeightUp = 7.0f;
constexpr float kNoKey = -1e30f;  // running maximum of a row without keys

struct Kv4Args {
  const void* q;
  void* out;
  const uint32_t* kc;
  const uint32_t* kp;
  const uint32_t* vc;
  const uint32_t* vp;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  float* part;     // [item][split][row][channel] sums, unnormalised
  float2* part_ml; // [item][split][row] maximum, sum
  int64_t sq_t, sq_h, so_t, so_h, s_table, tokens;
  float scale;
  int pages, hq, hk, group, d, columns, max_q, max_k, causal, bf, q_vec, o_vec;
  int row_blocks, splits, split_tiles;
  FastDiv by_page, by_group, by_splits;
};

// One (sequence, KV head, block of query rows): its rows and keys.
struct Kv4Item {
  int b, h, rb;
  int64_t start;  // first query token
  int nq, rows;   // queries, rows of all its blocks
  int len;        // keys
  int limit0;     // keys that query 0 sees (may be <= 0)
  int kmax;       // keys that the block's last row sees
};

__device__ __forceinline__ Kv4Item kv4_item(const Kv4Args& a, int b, int h, int rb, int block_rows) {
  Kv4Item it;
  it.b = b;
  it.h = h;
  it.rb = rb;
  int64_t start = (int64_t)b * a.max_q;
  int nq = a.max_q;
  if (a.cu != nullptr) {
    start = a.cu[b];
    nq = a.cu[b + 1] - (int)start;
  }
  if (start < 0 || start > a.tokens) nq = 0;
  nq = (int)min((int64_t)min(nq, a.max_q), a.tokens - start);
  it.start = start;
  it.nq = max(nq, 0);
  it.rows = it.nq * a.group;
  const int64_t room = min((int64_t)a.columns * a.by_page.d, (int64_t)a.max_k);
  it.len = (int)min((int64_t)max(a.lens[b], 0), room);
  it.limit0 = a.causal ? it.len - it.nq + 1 : it.len;
  const int last = min(it.rows, (rb + 1) * block_rows) - 1;
  it.kmax = a.causal ? it.limit0 + fast_div(max(last, 0), a.by_group) : it.len;
  return it;
}

__device__ __forceinline__ float lanes16_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const float2 h = swap_halves(x);
  return fmaxf(h.x, h.y);
}
__device__ __forceinline__ uint32_t lanes16_or(uint32_t x) {
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = r[0] | r[1];
  auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return s[0] | s[1];
}

// ---- lane layouts ---------------------------------------------------------------
// Lane l = 16 g + i of a wave.  Matrix operands of 16x16x32: A holds row i, B column i, both the
// k-slots 8 g .. 8 g + 7; the result holds column i and rows 4 g .. 4 g + 3.  A tile is four blocks
// t = 0 .. 3 of 16 keys; a block lies in one page, so that its rows have one scalar base.
//  * QK: A = K, row i = key 16 t + i.  The slots of step s are the channels of word NG g + s of a row
//    (word: eight channels), in the pairs of kv4_codes: a lane reads NG consecutive words of a
//    key, whose group is theirs alone (NG = 3: one of two).  Result: keys 16 t + 4 g + e of query row i.
//  * PV: A = V^T through ds_read_b64_tr_b4, which transposes a 16 x 16 block of codes in each 16 lanes:
//    lane i gets channel i of the 16 rows that the lanes point at, in their order.  Lane i of
//    group g points at key 16 (i / 4) + 4 g + i % 4: code 4 t + e of the result is the key that the lane
//    holds as result e of block t, so P stays in registers.  Word w of it are blocks 2 w
//    and 2 w + 1, in the pairs (0, 4), (1, 5) .. of kv4_codes: e of the one with e of the other.
template <int NG>
struct Kv4Tile {
  static constexpr int kNP = NG == 3 ? 2 : 1;  // groups that a lane's words of a K row can lie in
  uint32_t k[4][NG], kp[4][kNP], vp[4];
};

// LDS of one wave: two tiles of V codes, then the scales and minima [NG][64] of a tile in the pairs' order.
// A block of V is [chunk of 16 bytes][key] as the copies write it (lane l: byte 16 l); the blocks
// lie 64 bytes more than 1 KB apart, which leaves the transposed reads two lanes to a bank, their least
// while they read one half of each chunk.
constexpr int kBlockLds = 1024 + 64;
template <int NG>
constexpr int kWaveLds = 2 * 4 * kBlockLds + NG * 64 * 4;

template <int NG, int RT>
constexpr int kv4_lds_bytes() {
  const int tiles = kWaves * kWaveLds<NG>, join = kWaves * 2 * NG * 64 * 16;  // one row tile at a time
  return (tiles > join ? tiles : join) + kWaves * RT * 16 * 8;
}

template <int N>
__device__ __forceinline__ void load_words(uint32_t (&to)[N], const uint32_t* from) {
  if constexpr (N == 4) {
    const u32x4 x = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = x[i];
  } else if constexpr (N == 2) {
    const uint2 x = *reinterpret_cast<const uint2*>(from);
    to[0] = x.x;
    to[1] = x.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i] = from[i];
  }
}

// 16 bytes a lane from base + offset to LDS: lane l writes lds + 16 l.  As async_load16_asm
// (attn_common.h), from a scalar address; the same five wait states.
__device__ __forceinline__ void copy16(const uint32_t* base, uint32_t offset, uint32_t lds) {
  asm volatile(
      "s_nop 4\n\t"
      "global_load_lds_dwordx4 %0, %1"
      :
      : "v"(offset), "s"(base), "{m0}"(lds)
      : "memory");
}

// A table entry for a key, within the table's columns whatever the key (the loads of the sequence's bounds, which
// say what the entry is worth, are on their way at the same time).
__device__ __forceinline__ int table_entry(const Kv4Args& a, const int32_t* table, int key) {
  return a.columns > 0 ? table[min(fast_div(key, a.by_page), a.columns - 1)] : -1;
}
// The row of the pool of a block's first key: -1 where there is no page, or the block is at or behind `end`.
__device__ __forceinline__ int block_row(const Kv4Args& a, int id, int h, int key, int end) {
  const int column = fast_div(key, a.by_page);
  return key < end && id >= 0 && id < a.pages ? (id * a.hk + h) * a.by_page.d + (key - column * a.by_page.d) : -1;
}

// The keys of one wave: tiles first + wave, + kWaves, ..  Tile n of them has its blocks' rows in the
// lanes 4 (n % 16) .. + 3 of `rows`, from one load of the block table for every 16 tiles, made 16 tiles ahead.
struct Kv4Walk {
  const int32_t* table;
  int key0, end;  // first key of the wave; no block at or behind `end`
  int rows, ids;

  __device__ __forceinline__ int key(int n) const {
    const int lane = threadIdx.x & 63;
    return key0 + (n + (lane >> 2)) * (kWaves * kTile) + 16 * (lane & 3);
  }
  __device__ __forceinline__ void fetch(const Kv4Args& a, int n) { ids = table_entry(a, table, key(n)); }
  __device__ __forceinline__ void use(const Kv4Args& a, int h, int n) { rows = block_row(a, ids, h, key(n), end); }
};

// Starts the loads of tile n (V codes into LDS); there: which of its blocks have a page.  A block without
// one reads rows of page 0 (there is one): no branch around the loads; they count for nothing, whatever
// they hold.
template <int NG>
__device__ __forceinline__ uint32_t load_tile(Kv4Tile<NG>& x, const Kv4Args& a, const Kv4Walk& walk, int n,
                                              uint32_t lds_v) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4, gc = g < NG ? g : NG - 1;
  const uint32_t words_at = i * (4 * NG) + NG * g, chunk_at = 16 * (i * NG + gc), group_at = i * NG + gc;
  uint32_t there = 0;
  const uint32_t* base[4];
  int64_t row[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int r = __builtin_amdgcn_readlane(walk.rows, 4 * (n & 15) + t);
    there |= r >= 0 ? 1u << t : 0u;
    row[t] = r >= 0 ? r : 0;
    base[t] = a.kc + row[t] * (4 * NG);
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) copy16(a.vc + row[t] * (4 * NG), chunk_at, lds_v + t * kBlockLds);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    load_words(x.k[t], base[t] + words_at);
#pragma unroll
    for (int j = 0; j < Kv4Tile<NG>::kNP; ++j) {
      const uint32_t group = NG == 4 ? g : j == 0 ? NG * g / 4 : (NG * g + NG - 1) / 4;
      x.kp[t][j] = (a.kp + row[t] * NG)[i * NG + group];
    }
    x.vp[t] = (a.vp + row[t] * NG)[group_at];
  }
  return there;
}

// Elements c .. c + n - 1 (n <= 8) of a query row, zeros behind them.
__device__ __forceinline__ u32x4 load_query(const uint16_t* row, int c, int n, bool vec) {
  u32x4 w;
  if (vec && n == 8) {
    w = *reinterpret_cast<const u32x4*>(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = row[2 * e < n ? c + 2 * e : 0], hi = row[2 * e + 1 < n ? c + 2 * e + 1 : 0];
      w[e] = (2 * e < n ? lo : 0u) | (2 * e + 1 < n ? hi << 16 : 0u);
    }
  }
  return w;
}

// Rounds four channels to the output's type and writes those below d.
__device__ __forceinline__ void store_out(void* out, int64_t at, const f32x4& r, int left, bool vec, bool bf) {
  uint16_t* const to = static_cast<uint16_t*>(out) + at;
  const uint2 v = bf ? __builtin_bit_cast(uint2, __builtin_convertvector(r, bf16x4))
                     : __builtin_bit_cast(uint2, __builtin_convertvector(r, f16x4));
  if (vec && left >= 4) {
    *reinterpret_cast<uint2*>(to) = v;
  } else {
    if (left > 0) to[0] = (uint16_t)v.x;
    if (left > 1) to[1] = (uint16_t)(v.x >> 16);
    if (left > 2) to[2] = (uint16_t)v.y;
    if (left > 3) to[3] = (uint16_t)(v.y >> 16);
  }
}

// The queries of rows row0 + 16 rt + i, channels 8 (NG g + s) .. + 7, as they lie in memory.  A row that is not
// there reads the block's first one and becomes zeros.
template <int NG, int RT>
__device__ __forceinline__ void load_queries(const Kv4Args& a, const Kv4Item& it, int row0, u32x4 (&raw)[RT][NG]) {
  const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const bool there = row0 + 16 * rt + i < it.rows;
    const int row = there ? row0 + 16 * rt + i : row0, token = fast_div(row, a.by_group), head = row - token * a.group;
    const uint16_t* const from =
        static_cast<const uint16_t*>(a.q) + (it.start + token) * a.sq_t + (it.h * a.group + head) * a.sq_h;
#pragma unroll
    for (int s = 0; s < NG; ++s) {
      const int c = 8 * (NG * g + s);
      raw[rt][s] = load_query(from, c, there ? min(8, a.d - c) : 0, a.q_vec);
    }
  }
}

// The same as B operand of QK, the factor of their products and the keys that the rows see.
template <int NG, int RT>
__device__ __forceinline__ void use_queries(const Kv4Args& a, const Kv4Item& it, int row0, const u32x4 (&raw)[RT][NG],
                                            f16x8 (&qf)[RT][NG], float (&scale)[RT], int (&limit)[RT]) {
  const int i = threadIdx.x & 15;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    limit[rt] = a.causal ? it.limit0 + fast_div(row0 + 16 * rt + i, a.by_group) : it.len;
    // A negative scale is the queries' sign; none is a product that leaves the maximum at zero.
    scale[rt] = fmaxf(fabsf(a.scale), 1e-37f);
    f32x8 x[NG];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < NG; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t pair = raw[rt][s][e];  // (a bit cast of a vector's element would take the first one)
        const f16x2 h = __builtin_bit_cast(f16x2, pair);
        x[s][2 * e] = a.bf ? __uint_as_float(pair << 16) : (float)h[0];
        x[s][2 * e + 1] = a.bf ? __uint_as_float(pair & 0xffff0000u) : (float)h[1];
        top = fmaxf(top, fmaxf(fabsf(x[s][2 * e]), fabsf(x[s][2 * e + 1])));
      }
    // bf16 queries are held as fp16 times a power of two of their row: exact but for elements below
    // 2^-14 of the row's largest, which lose no more than 2^-25 of that one.
    if (a.bf) {
      const int e = __builtin_amdgcn_frexp_expf(lanes16_max(top));
      scale[rt] = ldexpf(scale[rt], e);
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) x[s][j] = ldexpf(x[s][j], -e);
    }
#pragma unroll
    for (int s = 0; s < NG; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        qf[rt][s][2 * j] = (f16)(a.scale < 0.0f ? -x[s][j] : x[s][j]);
        qf[rt][s][2 * j + 1] = (f16)(a.scale < 0.0f ? -x[s][j + 4] : x[s][j + 4]);
      }
  }
}

// The running softmax of a row tile, in two steps.  acc: products of the lane's keys mine + 16 t + e.  First the
// maximum (keys of blocks not in `there` and at or behind the row's limit are masked, if the tile has any).
__device__ __forceinline__ void mask_tile(f32x4 (&acc)[4], int limit, uint32_t there, int mine) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!((there >> t) & 1) || mine + 16 * t + e >= limit) acc[t][e] = -__builtin_inff();
}
__device__ __forceinline__ float tile_max(const f32x4 (&acc)[4], float scale) {
  float hi = -__builtin_inff();
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) hi = fmaxf(hi, acc[t][e]);
  return lanes16_max(hi) * scale;
}
// Raises the running maximum where a row needs it.
template <int CT>
__device__ __forceinline__ void raise_max(float hi, float& top, f32x4& sum, f32x4 (&o)[CT]) {
  if (__any(hi > top + kKv4Slack)) {
    const float up = fmaxf(hi, top), down = __builtin_amdgcn_exp2f(top - up);
    top = up;
    sum *= down;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) o[ct] *= down;
  }
}
// Then the weights, as B operand of PV.
__device__ __forceinline__ void tile_weights(const f32x4 (&acc)[4], float scale, float top, f16x8 (&pf)[2]) {
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      pf[w][2 * e] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(acc[2 * w][e], scale, kWeightUp - top));
      pf[w][2 * e + 1] = (f16)__builtin_amdgcn_exp2f(__builtin_fmaf(acc[2 * w + 1][e], scale, kWeightUp - top));
    }
}
// The row sums of the weights, on the matrix pipe: sixteen rows of ones (each result row is the sum).
__device__ __forceinline__ f32x4 add_weights(const f16x8 (&pf)[2], f32x4 sum) {
  f16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = (f16)1.0f;
#pragma unroll
  for (int w = 0; w < 2; ++w) sum = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pf[w], sum, 0, 0, 0);
  return sum;
}

// Values that are not finite (a NaN was stored) are zeros in the products.  The rows that see such a key get a
// NaN in its group's channels, the others must not (0 times NaN would be one).  broken[t]: bit 16 j + i
// for group j of key 16 t + i.
template <int NG, int RT, int CT>
__device__ __forceinline__ void poison_rows(f32x4 (&o)[RT][CT], const uint64_t (&broken)[4], const int (&limit)[RT],
                                            int key0) {
  int at = 4 * ((threadIdx.x & 63) >> 4);
  asm volatile("" : "+v"(at));  // what follows stays in this rare block
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    uint32_t seen = 0;  // groups
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t keys = (1u << min(max(limit[rt] - (key0 + 16 * t + at), 0), 4)) - 1;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const uint32_t bits = (uint32_t)(j < 2 ? broken[t] : broken[t] >> 32) >> (16 * (j & 1) + at);
        seen |= (bits & keys) != 0 ? 1u << j : 0u;
      }
    }
    seen = lanes16_or(seen);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
      if ((seen >> (ct >> 1)) & 1) o[rt][ct] = f32x4{} + __builtin_nanf("");
  }
}

// Eight channels of a key: the word's codes with their group's scale and minimum.
__device__ __forceinline__ f16x8 key_words(uint32_t word, uint32_t param) {
  const f16x2 sm = __builtin_bit_cast(f16x2, param), sc = {sm[0], sm[0]}, mn = {sm[1], sm[1]};
  f16x2 c[4];
  kv4_codes(word, c);
  f16x8 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const f16x2 v = kv4_fma(c[j], sc, mn);
    r[2 * j] = v[0];
    r[2 * j + 1] = v[1];
  }
  return r;
}

// Scales and minima of one group for the lane's 16 keys, as lds_s and lds_m hold them.
struct ValueParams {
  f16x8 s[2], m[2];
  ValueParams() = default;
  __device__ __forceinline__ ValueParams(const f16* lds_s, const f16* lds_m) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      s[w] = *reinterpret_cast<const f16x8*>(lds_s + 8 * w);
      m[w] = *reinterpret_cast<const f16x8*>(lds_m + 8 * w);
    }
  }
  // Word w of a channel: eight keys.
  __device__ __forceinline__ f16x8 values(uint32_t word, int w) const {
    f16x2 c[4];
    kv4_codes(word, c);
    f16x8 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f16x2 v = kv4_fma(c[e], f16x2{s[w][2 * e], s[w][2 * e + 1]}, f16x2{m[w][2 * e], m[w][2 * e + 1]});
      r[2 * e] = v[0];
      r[2 * e + 1] = v[1];
    }
    return r;
  }
};

template <int NG, int RT>
__global__ void __launch_bounds__(kWaves * 64, RT == 1 ? 3 : 2) kv4_attn_kernel(const Kv4Args a) {
  using Tile = Kv4Tile<NG>;
  constexpr int kCT = 2 * NG;  // tiles of 16 channels
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15,
            g = lane >> 4;
  const int rb = fast_div(blockIdx.x, a.by_splits), split = blockIdx.x - rb * a.splits;
  const int first = split * a.split_tiles;
  const Kv4Item it = kv4_item(a, blockIdx.z, blockIdx.y, rb, 16 * RT);
  const int row0 = rb * 16 * RT;
  if (row0 >= it.rows) return;
  const int tiles = it.kmax <= 0 ? 0 : (it.kmax + kTile - 1) / kTile;
  const int last = min(tiles, first + a.split_tiles);
  if (first >= last && split > 0) return;

  // the first keys' places are on their way while the queries come
  Kv4Walk walk;
  walk.table = a.table + it.b * a.s_table;
  walk.key0 = (first + wave) * kTile;
  walk.end = min(it.kmax, last * kTile);
  walk.fetch(a, 0);
  f16x8 qf[RT][NG];
  float scale[RT];
  int limit[RT];
  {
    u32x4 raw[RT][NG];
    load_queries(a, it, row0, raw);
    use_queries(a, it, row0, raw, qf, scale, limit);
  }

  unsigned char* const lds_v = smem + wave * kWaveLds<NG>;
  f16* const lds_s = reinterpret_cast<f16*>(lds_v + 2 * 4 * kBlockLds);
  f16* const lds_m = lds_s + NG * 64;
  const uint32_t v_addr = lds_addr(lds_v);
  Tile x;
  walk.use(a, it.h, 0);
  walk.fetch(a, 16);
  uint32_t there = load_tile(x, a, walk, 0, v_addr);

  f32x4 o[RT][kCT];
  float top[RT];
  f32x4 sum[RT];  // four times the same
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = kNoKey;
    sum[rt] = f32x4{};
#pragma unroll
    for (int ct = 0; ct < kCT; ++ct) o[rt][ct] = f32x4{};
  }

  const int all_see = it.limit0 + (a.causal ? fast_div(row0, a.by_group) : 0);  // keys that every row sees
  // V rows that the lane points at in a transposed read, in LDS
  const int v_at = (i >> 2) * kBlockLds + (4 * g + (i & 3)) * 16;
  const int p_at = 16 * (i >> 2) + 2 * (i & 3);  // of key i of a block in the pairs' order, see below

  int n = 0;
  for (int tile = first + wave; tile < last; tile += kWaves, ++n) {
    const int key0 = tile * kTile;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the copies of V; the other loads are as old
    const bool masked = key0 + kTile > all_see || there != 15u;
    if (masked) {
      // rows without a page and behind the last key that any row sees may hold anything: zeros
#pragma unroll
      for (int t = 0; t < 4; ++t)
        if (!((there >> t) & 1) || key0 + 16 * t + i >= it.kmax) x.vp[t] = 0;
    }
    // groups whose values are not finite: zeros here, see below
    uint64_t broken[4];
    bool any_broken = false;
#pragma unroll
    for (int t = 0; t < 4; ++t) any_broken |= kv4_not_finite(x.vp[t]);
    any_broken = __any(any_broken);
    if (any_broken) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const bool bad = kv4_not_finite(x.vp[t]);
        broken[t] = __ballot(bad);
        if (bad) x.vp[t] = 0;
      }
    }
    // ---- V's parameters to LDS: pairs of the same key of blocks 2 w and 2 w + 1 ----
    if (NG == 4 || g < NG) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const uint32_t p0 = x.vp[2 * w], p1 = x.vp[2 * w + 1];
        *reinterpret_cast<uint32_t*>(lds_s + g * 64 + p_at + 8 * w) = __builtin_amdgcn_perm(p1, p0, 0x05040100u);
        *reinterpret_cast<uint32_t*>(lds_m + g * 64 + p_at + 8 * w) = __builtin_amdgcn_perm(p1, p0, 0x07060302u);
      }
    }
    // ---- S^T = K Q^T ----
    f32x4 acc[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt][t] = f32x4{};
#pragma unroll
      for (int s = 0; s < NG; ++s) {
        const uint32_t p = NG == 3 && (NG * g + s) / 4 != NG * g / 4 ? x.kp[t][Tile::kNP - 1] : x.kp[t][0];
        const f16x8 kf = key_words(x.k[t][s], p);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          acc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[rt][s], acc[rt][t], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    // ---- the next tile is on its way while this one goes on ----
    const uint32_t here = there;
    if (((n + 1) & 15) == 0) {
      walk.use(a, it.h, n + 1);
      walk.fetch(a, n + 17);
    }
    there = load_tile(x, a, walk, n + 1, v_addr + ((n + 1) & 1) * 4 * kBlockLds);
    __builtin_amdgcn_sched_barrier(0);
    // ---- softmax ----
    f16x8 pf[RT][2];
    const int mine = key0 + 4 * g;  // the lane's keys are mine + 16 t + e
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (masked) mask_tile(acc[rt], limit[rt], here, mine);
      raise_max(tile_max(acc[rt], scale[rt]), top[rt], sum[rt], o[rt]);
      tile_weights(acc[rt], scale[rt], top[rt], pf[rt]);
      sum[rt] = add_weights(pf[rt], sum[rt]);
    }
    // ---- O^T += V^T P^T ----
    const unsigned char* const v_tile = lds_v + (n & 1) * 4 * kBlockLds + v_at;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      // (one group's parameters at a time: fetched all ahead they would take 64 registers)
      __builtin_amdgcn_sched_barrier(0);
      const ValueParams params(lds_s + j * 64 + 16 * g, lds_m + j * 64 + 16 * g);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int ct = 2 * j + c;
        const i32x2 words = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
            (__attribute__((address_space(3))) i32x2*)(v_tile + 256 * j + 8 * c));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const f16x8 vf = params.values((uint32_t)words[w], w);
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            o[rt][ct] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[rt][w], o[rt][ct], 0, 0, 0);
        }
      }
    }
    // Values that are not finite (a NaN was stored): the rows that see the key get a NaN in the
    // group's channels, the others must not (0 times NaN would be one).
    if (any_broken) poison_rows<NG>(o, broken, limit, key0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no copy is left that could overwrite what follows

  // ---- the four waves' parts ----
  float2* const lds_ml = reinterpret_cast<float2*>(smem + kv4_lds_bytes<NG, RT>() - kWaves * RT * 16 * 8);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    if (g == 0) lds_ml[(wave * RT + rt) * 16 + i] = make_float2(top[rt], sum[rt][0]);
  }
  const int item = ((it.b * a.hk + it.h) * a.row_blocks + rb) * a.splits + split;
  f32x4* const lds_o = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    __syncthreads();  // the tiles' LDS, or the row tile before, is no longer read
    float all_top = kNoKey, all_sum = 0.0f;
    float2 ml[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      ml[w] = lds_ml[(w * RT + rt) * 16 + i];
      all_top = fmaxf(all_top, ml[w].x);
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all_sum += ml[w].y * __builtin_amdgcn_exp2f(ml[w].x - all_top);
    const float down = __builtin_amdgcn_exp2f(top[rt] - all_top);
#pragma unroll
    for (int ct = 0; ct < kCT; ++ct) lds_o[(wave * kCT + ct) * 64 + lane] = o[rt][ct] * down;
    __syncthreads();
    const int row = row0 + 16 * rt + i, token = fast_div(row, a.by_group), head = row - token * a.group;
    if (row < it.rows) {
      if (a.splits > 1 && wave == 0 && g == 0)
        a.part_ml[(int64_t)item * (16 * RT) + 16 * rt + i] = make_float2(all_top, all_sum);
      const float norm = all_sum == 0.0f ? 0.0f : 1.0f / all_sum;
      for (int ct = wave; ct < kCT; ct += kWaves) {
        f32x4 r = lds_o[ct * 64 + lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) r += lds_o[(w * kCT + ct) * 64 + lane];
        const int c = 16 * ct + 4 * g;
        if (a.splits > 1) {
          *reinterpret_cast<f32x4*>(a.part + ((int64_t)item * (16 * RT) + 16 * rt + i) * (32 * NG) + c) = r;
          continue;
        }
        r *= norm;
        store_out(a.out, (it.start + token) * a.so_t + (it.h * a.group + head) * a.so_h + c, r, a.d - c, a.o_vec,
                  a.bf);
      }
    }
  }
}

// ---- many query rows ---------------------------------------------------------------
// A workgroup takes 32 RT query rows, 16 RT of each wave, and all its waves go through the same
// tiles: each turns a quarter of a tile's codes into fp16 operands, which all read from LDS as they
// lie in the registers (operand [..][lane], no bank conflicts in either direction).
// The loop is skewed so that the matrix pipe and the vector units have independent work side by side:
// iteration n multiplies Q with the keys of tile n + 1 beside the softmax of tile n, then its weights with
// the values of tile n beside the conversion of K's tile n + 2 and V's tile n + 1; the codes after those are
// on their way.  One barrier a tile.  K's codes come in registers (wave t: block t), V's as copies to
// LDS, from which wave t makes the channels ct = t and t + 4.
template <int NG>
struct ChunkLds {
  f16x8 k[2][4 * NG * 64];      // [tile][(t NG + s) 64 + lane]
  f16x8 v[2][4 * NG * 64];      // [tile][(2 ct + w) 64 + lane]
  unsigned char codes[2][4 * kBlockLds];
  f16 scale[2][NG * 64], least[2][NG * 64];
  // Of the tiles n, n + 1, ..: flags[n % 4][t] of block t: 1 it has a page, 2 it has values that are not finite,
  // those of `broken` (poison_rows).
  uint32_t flags[4][4];
  uint64_t broken[4][4];
};

// Asks the scheduler for COUNT matrix instructions with VALU vector and TRANS transcendental ones behind each.
template <int COUNT, int VALU, int TRANS>
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    if (VALU > 0) __builtin_amdgcn_sched_group_barrier(0x2, VALU, 0);
    if (TRANS > 0) __builtin_amdgcn_sched_group_barrier(0x400, TRANS, 0);
  }
}

template <int NG, int RT>
__global__ void __launch_bounds__(kWaves * 64, 2) kv4_chunk_kernel(const Kv4Args a) {
  constexpr int kCT = 2 * NG, kNP = Kv4Tile<NG>::kNP, kRows = kWaves * 16 * RT;
  __shared__ __attribute__((aligned(16))) ChunkLds<NG> lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15,
            g = lane >> 4;
  const int rb = fast_div(blockIdx.y, a.by_splits), split = blockIdx.y - rb * a.splits;
  const int first = split * a.split_tiles;
  // The rows of the pool of block `wave` of the tiles first + 64 c .. + 63, one in each lane (-1: no page).
  const int32_t* const table = a.table + blockIdx.z * a.s_table;
  auto key_of = [&](int n) { return (first + n + lane) * kTile + 16 * wave; };
  int ids = table_entry(a, table, key_of(0)), rows = -1;
  const Kv4Item it = kv4_item(a, blockIdx.z, blockIdx.x, rb, kRows);
  if (rb * kRows >= it.rows) return;
  const int tiles = it.kmax <= 0 ? 0 : (it.kmax + kTile - 1) / kTile;
  const int last = min(tiles, first + a.split_tiles);
  if (first >= last && split > 0) return;
  const int end = min(it.kmax, last * kTile);  // keys

  const int row0 = rb * kRows + wave * 16 * RT;  // of the wave
  // ---- loads ----
  const int gc = g < NG ? g : NG - 1;
  const uint32_t words_at = i * (4 * NG) + NG * g, chunk_at = 16 * (i * NG + gc), group_at = i * NG + gc;
  const uint32_t codes_lds = lds_addr(&lds.codes[0][0]) + wave * kBlockLds;
  struct KeyCodes {
    uint32_t k[NG], kp[kNP];
  } fresh, codes;  // of the tile that is loaded, and of the one that is made
  uint32_t vp;
  auto find = [&](int n) {  // the row of the wave's block of tile n
    if ((n & 63) == 0) {
      rows = block_row(a, ids, it.h, key_of(n), end);
      ids = table_entry(a, table, key_of(n + 64));
    }
    return __builtin_amdgcn_readlane(rows, n & 63);
  };
  auto load_k = [&](int found) {  // (a block without a page reads rows of page 0: they count for nothing)
    const int64_t row = max(found, 0);
    load_words(fresh.k, a.kc + row * (4 * NG) + words_at);
#pragma unroll
    for (int j = 0; j < kNP; ++j) {
      const uint32_t group = NG == 4 ? g : j == 0 ? NG * g / 4 : (NG * g + NG - 1) / 4;
      fresh.kp[j] = (a.kp + row * NG)[i * NG + group];
    }
  };
  auto load_v = [&](int n, int found) {
    const int64_t row = max(found, 0);
    copy16(a.vc + row * (4 * NG), chunk_at, codes_lds + (n & 1) * 4 * kBlockLds);
    vp = (a.vp + row * NG)[group_at];
  };
  // V's parameters of tile n (in vp) to LDS, in the order of the pairs
  const int p_at = 16 * (i >> 2) + 2 * (i & 3) + 8 * (wave >> 1) + (wave & 1);
  auto stage_params = [&](int n, int found) {
    uint32_t p = vp;
    if (found < 0 || (first + n) * kTile + 16 * wave + i >= end) p = 0;
    const bool bad = kv4_not_finite(p);
    const uint64_t broken = __ballot(bad);
    if (bad) p = 0;
    const f16x2 sm = __builtin_bit_cast(f16x2, p);
    if (NG == 4 || g < NG) {
      lds.scale[n & 1][g * 64 + p_at] = sm[0];
      lds.least[n & 1][g * 64 + p_at] = sm[1];
    }
    if (lane == 0) {
      lds.flags[n & 3][wave] = (found >= 0 ? 1u : 0u) | (broken != 0 ? 2u : 0u);
      lds.broken[n & 3][wave] = broken;
    }
  };
  auto make_k = [&](int n, int s) {  // one word of each key
    const uint32_t p = NG == 3 && (NG * g + s) / 4 != NG * g / 4 ? codes.kp[kNP - 1] : codes.kp[0];
    lds.k[n & 1][(wave * NG + s) * 64 + lane] = key_words(codes.k[s], p);
  };
  const int v_at = (i >> 2) * kBlockLds + (4 * g + (i & 3)) * 16;
  // 16 channels ct = wave + 4 c: reads and conversion apart, so that products fit between them
  auto has_v = [&](int c) { return NG == 4 || wave + 4 * c < kCT; };
  auto read_v = [&](int n, int c, i32x2& words) {
    const int ct = wave + 4 * c, j = ct >> 1;
    words = __builtin_amdgcn_ds_read_tr4_b64_v2i32(
        (__attribute__((address_space(3))) i32x2*)(lds.codes[n & 1] + v_at + 256 * j + 8 * (ct & 1)));
    return ValueParams(lds.scale[n & 1] + j * 64 + 16 * g, lds.least[n & 1] + j * 64 + 16 * g);
  };
  auto write_v = [&](int n, int c, const i32x2& words, const ValueParams& params) {
#pragma unroll
    for (int w = 0; w < 2; ++w)
      lds.v[n & 1][(2 * (wave + 4 * c) + w) * 64 + lane] = params.values((uint32_t)words[w], w);
  };
  auto make_v = [&](int n, int c) {
    if (has_v(c)) {
      i32x2 words;
      const ValueParams params = read_v(n, c, words);
      write_v(n, c, words, params);
    }
  };

  u32x4 raw[RT][NG];
  load_queries(a, it, min(row0, it.rows - 1), raw);
  // ---- before tile 0: its scores, its values, K's tile 1, the codes of K's tile 2 and V's tile 1 ----
  const int count = last - first;
  int row[3];  // of the wave's block of tiles n + 1 .. n + 3
  auto wait_loads = [] { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); };
#pragma unroll
  for (int k = 0; k < 3; ++k) row[k] = find(k);
  KeyCodes ahead_codes[3];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    load_k(row[k]);
    ahead_codes[k] = fresh;
  }
  load_v(0, row[0]);
  const uint32_t vp0 = vp;
  load_v(1, row[1]);
  const uint32_t vp1 = vp;
  f16x8 qf[RT][NG];
  float scale[RT];
  int limit[RT];
  use_queries(a, it, min(row0, it.rows - 1), raw, qf, scale, limit);
  const bool rows_there = row0 < it.rows;
  const int all_see = it.limit0 + (a.causal ? fast_div(row0, a.by_group) : 0);  // keys that all rows of the wave see

  f32x4 o[RT][kCT];
  float top[RT];
  f32x4 sum[RT];  // four times the same
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    top[rt] = kNoKey;
    sum[rt] = f32x4{};
#pragma unroll
    for (int ct = 0; ct < kCT; ++ct) o[rt][ct] = f32x4{};
  }

  wait_loads();
  vp = vp0;
  stage_params(0, row[0]);
  vp = vp1;
  stage_params(1, row[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    codes = ahead_codes[k];
#pragma unroll
    for (int s = 0; s < NG; ++s) make_k(k, s);
  }
  codes = ahead_codes[2];
  row[1] = row[2];
  __syncthreads();
  f32x4 acc[RT][4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) acc[rt][t] = f32x4{};
#pragma unroll
    for (int s = 0; s < NG; ++s)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        acc[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lds.k[0][(t * NG + s) * 64 + lane], qf[rt][s], acc[rt][t],
                                                            0, 0, 0);
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) make_v(0, c);
  __syncthreads();

  for (int n = 0; n < count; ++n) {
    const int key0 = (first + n) * kTile;
    const f16x8* const kf = lds.k[(n + 1) & 1] + lane;
    const f16x8* const vf = lds.v[n & 1] + lane;
    f16x8 x[2][4], pf[RT][2];
    auto read_keys = [&](int s) {
#pragma unroll
      for (int t = 0; t < 4; ++t) x[s & 1][t] = kf[(t * NG + s) * 64];
    };
    read_keys(0);
    const u32x4 flags = *reinterpret_cast<const u32x4*>(lds.flags[n & 3]);
    __builtin_amdgcn_sched_barrier(0);
    // in flight: K's tile n + 3, V's tile n + 2
    row[2] = find(n + 3);
    load_v(n + 2, row[1]);
    load_k(row[2]);
    const uint32_t all = __builtin_amdgcn_readfirstlane(flags[0] & flags[1] & flags[2] & flags[3]);
    const uint32_t some = __builtin_amdgcn_readfirstlane(flags[0] | flags[1] | flags[2] | flags[3]);
    if (key0 + kTile > all_see || (all & 1) == 0) {
      const uint32_t there = (flags[0] & 1) | (flags[1] & 1) << 1 | (flags[2] & 1) << 2 | (flags[3] & 1) << 3;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) mask_tile(acc[rt], limit[rt], there, key0 + 4 * g);
    }
    // ---- scores of tile n + 1 beside the softmax of tile n ----
    __builtin_amdgcn_s_setprio(1);
    f32x4 ahead[RT][4];
    auto scores = [&](int s) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          ahead[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[s & 1][t], qf[rt][s], s == 0 ? f32x4{} : ahead[rt][t],
                                                                0, 0, 0);
    };
    float hi[RT];
#pragma unroll
    for (int s = 0; s < (NG + 1) / 2; ++s) {
      if (s + 1 < NG) read_keys(s + 1);
      scores(s);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) hi[rt] = tile_max(acc[rt], scale[rt]);
    interleave<4 * RT * ((NG + 1) / 2), 3, 0>();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) raise_max(hi[rt], top[rt], sum[rt], o[rt]);
#pragma unroll
    for (int s = (NG + 1) / 2; s < NG; ++s) {
      if (s + 1 < NG) read_keys(s + 1);
      scores(s);
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) tile_weights(acc[rt], scale[rt], top[rt], pf[rt]);
    interleave<4 * RT * (NG / 2), 3, 2>();
    // ---- values of tile n beside the conversion of what comes next ----
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    auto read_values = [&](int c) {  // operands 4 c .. 4 c + 3: channels 2 c and 2 c + 1 of 16, two words each
#pragma unroll
      for (int t = 0; t < 4; ++t) x[c & 1][t] = vf[(4 * c + t) * 64];
    };
    read_values(0);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) sum[rt] = add_weights(pf[rt], sum[rt]);
#pragma unroll
    for (int c = 0; c < NG; ++c) {
      if (c + 1 < NG) read_values(c + 1);
      i32x2 words;
      ValueParams params;
      if (NG == 4 && c < 2) params = read_v(n + 1, c, words);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            o[rt][2 * c + k] =
                __builtin_amdgcn_mfma_f32_16x16x32_f16(x[c & 1][2 * k + w], pf[rt][w], o[rt][2 * c + k], 0, 0, 0);
      if (NG == 4 && c < 2) write_v(n + 1, c, words, params);
      if (NG < 4 || c >= 2) {
        make_k(n + 2, NG < 4 ? c : 2 * (c - 2));
        if (NG == 4) make_k(n + 2, 2 * (c - 2) + 1);
      }
      interleave<4 * RT, 4, 0>();
      __builtin_amdgcn_sched_barrier(0);
    }
    if (NG < 4) {
#pragma unroll
      for (int c = 0; c < 2; ++c) make_v(n + 1, c);
    }
    if ((some & 2) != 0) {
      const uint64_t broken[4] = {lds.broken[n & 3][0], lds.broken[n & 3][1], lds.broken[n & 3][2], lds.broken[n & 3][3]};
      poison_rows<NG>(o, broken, limit, key0);
    }
    // V's tile n + 2 has arrived; its parameters take the place of tile n's, whose operands all waves have made
    wait_loads();
    stage_params(n + 2, row[1]);
    codes = fresh;
    row[1] = row[2];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) acc[rt][t] = ahead[rt][t];
    __syncthreads();
  }

  // ---- each wave has its rows for itself ----
  if (!rows_there) return;
  const int64_t item = ((int64_t)(it.b * a.hk + it.h) * a.row_blocks + rb) * a.splits + split;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float all = sum[rt][0];
    const int row = row0 + 16 * rt + i, token = fast_div(row, a.by_group), head = row - token * a.group;
    if (row >= it.rows) continue;
    const int64_t part = item * kRows + wave * 16 * RT + 16 * rt + i;
    if (a.splits > 1 && g == 0) a.part_ml[part] = make_float2(top[rt], all);
    const float norm = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
    for (int ct = 0; ct < kCT; ++ct) {
      const int c = 16 * ct + 4 * g;
      if (a.splits > 1) *reinterpret_cast<f32x4*>(a.part + part * (32 * NG) + c) = o[rt][ct];
      else
        store_out(a.out, (it.start + token) * a.so_t + (it.h * a.group + head) * a.so_h + c, o[rt][ct] * norm, a.d - c,
                  a.o_vec, a.bf);
    }
  }
}

// Adds up the splits of a row.  One thread takes four channels of every `lanes`-th split and keeps
// its own running maximum; the `lanes` threads of a row's channels meet in LDS.
template <int NG>
__global__ void __launch_bounds__(256) kv4_join_kernel(const Kv4Args a, int block_rows, int lanes, int rows) {
  constexpr int kC = 8 * NG;
  __shared__ f32x4 lds_o[256];
  __shared__ float2 lds_ml[256];
  const int unit = threadIdx.x / kC, c = 4 * (threadIdx.x - unit * kC), r = unit / lanes, lane = unit - r * lanes;
  const int groups = (block_rows + rows - 1) / rows, rb = blockIdx.x / groups;
  const int in_block = (blockIdx.x - rb * groups) * rows + r;
  const Kv4Item it = kv4_item(a, blockIdx.z, blockIdx.y, rb, block_rows);
  const int row = rb * block_rows + in_block;
  const bool there = r < rows && in_block < block_rows && row < it.rows;
  f32x4 o = {};
  float2 ml = make_float2(kNoKey, 0.0f);
  if (there) {
    const int tiles = it.kmax <= 0 ? 0 : (it.kmax + kTile - 1) / kTile;
    const int parts = max(1, (tiles + a.split_tiles - 1) / a.split_tiles);
    const int64_t first =
        (int64_t)((it.b * a.hk + it.h) * a.row_blocks + rb) * a.splits * block_rows + in_block;
#pragma unroll 4
    for (int s = lane; s < parts; s += lanes) {
      const int64_t at = first + (int64_t)s * block_rows;
      const float2 part = a.part_ml[at];
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + at * (32 * NG) + c);
      const float up = fmaxf(ml.x, part.x);
      const float mine = __builtin_amdgcn_exp2f(ml.x - up), its = __builtin_amdgcn_exp2f(part.x - up);
      ml = make_float2(up, ml.y * mine + part.y * its);
      o = o * mine + x * its;
    }
  }
  lds_o[threadIdx.x] = o;
  lds_ml[threadIdx.x] = ml;
  __syncthreads();
  if (!there || lane != 0 || c >= a.d) return;
  float top = ml.x;
  for (int i = 1; i < lanes; ++i) top = fmaxf(top, lds_ml[threadIdx.x + i * kC].x);
  const float mine = __builtin_amdgcn_exp2f(ml.x - top);
  o *= mine;
  float sum = ml.y * mine;
  for (int i = 1; i < lanes; ++i) {
    const float2 part = lds_ml[threadIdx.x + i * kC];
    const float its = __builtin_amdgcn_exp2f(part.x - top);
    sum += part.y * its;
    o += lds_o[threadIdx.x + i * kC] * its;
  }
  o *= sum == 0.0f ? 0.0f : 1.0f / sum;
  const int token = fast_div(row, a.by_group), head = row - token * a.group;
  store_out(a.out, (it.start + token) * a.so_t + (it.h * a.group + head) * a.so_h + c, o, a.d - c, a.o_vec, a.bf);
}

constexpr int64_t kMostKeys = 1 << 30;  // of a sequence: places of keys ahead of the last one still fit 32 bits

struct Plan {
  int block_rows, row_blocks, splits, split_tiles;
  int64_t bytes;
};

// Tiles of a split.  A split costs the join (a second launch, 4 us) and each workgroup's start and end (3 us, 10
// with the chunk kernel, of which two fit a CU); too few leave the card waiting for the longest sequence.
// Calls in us (head_dim 128, 24/8 heads unless said), this rule / others:
//   * up to 12 tiles one: 1 x 700 (14/2 heads x 64) 8.2, split 9.5; 16 x 512 10.0 / 11.8;
//   * few (sequence, head) pairs: two workgroups a CU.  1 x 131072 in 64 42.4, 48 45.7, 96 46.6; 3 of 2000 .. 30000
//     in 21 30.1, 16 34.7, 32 31.1; 1 x 1024 in four 11.5, one 12.9;
//   * else 16 tiles each (four a wave), as lengths differ and the longest sequence is waited for: 24 of 700 ..
//     9001 (28/4 heads) in 9 29.6, 6 36.3; 24 of 61 .. 5000 in 5 29.4, 3 36.8; 16 of 61 .. 5000 in 5 25.6, 7
//     26.1; 32 x 1024 in one 14.7, two 18.5;
//   * but no more than three workgroups a CU, all that are resident: 64 x 8192 in one 126, two 131, four
//     134; 48 of 200 .. 6000 in two 62.4, four 67.2; 32 x 4096 in three 42.8, four 44.2.
int64_t plan_split(int64_t items, int64_t tiles, int block_rows) {
  if (block_rows == kChunkRows) {
    const int64_t splits = std::min(std::max<int64_t>(512 / items, 1), std::max<int64_t>(tiles / 8, 1));
    return (tiles + splits - 1) / splits;
  }
  if (tiles <= 12) return tiles;
  int64_t splits;
  if (items < 64) {
    splits = std::min(512 / items, tiles / 4);
  } else {
    splits = (tiles + 15) / 16;
    if (items * splits >= 1024) splits = std::max<int64_t>(768 / items, 1);
  }
  const int64_t each = (tiles + splits - 1) / splits;
  return (each + kWaves - 1) / kWaves * kWaves;  // the waves take whole tiles in turn
}

bool make_plan(const char* what, const tilemix_kv4_attn_params& p, Plan& plan) {
  if (!kv4_pool_ok(what, p.k_codes, p.k_params, p.v_codes, p.v_params, p.pages, p.page_size, p.heads_k, p.head_dim,
                   p.dtype))
    return false;
  if (p.heads_q <= 0 || p.heads_q % p.heads_k != 0 || p.batch < 0 || p.batch > 65535 || p.table_columns < 0 ||
      p.max_seqlen_q < 0 || p.max_seqlen_k < 0 || p.tokens_q < 0 || p.tokens_q > INT32_MAX ||
      std::min<int64_t>(p.max_seqlen_k, (int64_t)p.table_columns * p.page_size) > kMostKeys) {
    set_error("%s: invalid sizes (heads %d/%d, batch %d, table_columns %d, max_seqlen %d/%d, %lld queries)", what,
              p.heads_q, p.heads_k, p.batch, p.table_columns, p.max_seqlen_q, p.max_seqlen_k, (long long)p.tokens_q);
    return false;
  }
  const int64_t rows = (int64_t)p.max_seqlen_q * (p.heads_q / p.heads_k);
  const int64_t keys = std::min<int64_t>(p.max_seqlen_k, (int64_t)p.table_columns * p.page_size);
  const int64_t tiles = std::max<int64_t>((keys + kTile - 1) / kTile, 1);
  // The chunk kernel needs rows to share its conversions among, and work that outweighs its start and end; the
  // other one takes the same rows 32 at a time.  Calls in us, blocks of 32 / chunk kernel (24/8 heads x 128, tiles
  // of blocks of 32): 90 rows 8 x 4000 41.3 / 42.6; 120 rows 1 x 4000 (2016) 17.5 / 29.5, 8 x 4000 (16128) 51.4 /
  // 44.2, 1 x 40000 (20000) 49.5 / 47.0; 300 rows 1 x 4000 (5040) 28.4 / 31.4, 1 x 40000 (50000) 111 / 88.
  const int64_t blocks32 = (rows + 31) / 32;
  const bool few = blocks32 * p.heads_k * p.batch * tiles <= 10000;
  plan.block_rows = rows <= 16 ? 16 : rows <= 96 || few ? 32 : kChunkRows;
  const int64_t blocks = (rows + plan.block_rows - 1) / plan.block_rows;
  const int64_t items = std::max<int64_t>(blocks * p.heads_k * p.batch, 1);
  const int64_t split_tiles = plan_split(items, tiles, plan.block_rows);
  const int64_t splits = (tiles + split_tiles - 1) / split_tiles;
  const int64_t grid = blocks * splits;
  if (rows > INT32_MAX / 2 || grid > (plan.block_rows < kChunkRows ? (1 << 24) - 1 : 65535) || items * splits > INT32_MAX / 64) {
    set_error("%s: too many queries for one call (%lld rows a sequence, batch %d)", what, (long long)rows, p.batch);
    return false;
  }
  plan.row_blocks = (int)blocks;
  plan.splits = (int)splits;
  plan.split_tiles = (int)split_tiles;
  const int width = (p.head_dim + kKv4Group - 1) / kKv4Group * kKv4Group;
  plan.bytes = splits > 1 ? items * splits * plan.block_rows * (width * 4 + 8) : 0;
  return true;
}

template <int NG>
void launch_kv4(const Kv4Args& a, int block_rows, int batch, hipStream_t stream) {
  if (block_rows < kChunkRows) {
    const dim3 grid((unsigned)(a.row_blocks * a.splits), a.hk, batch), block(kWaves * 64);
    constexpr int lds1 = kv4_lds_bytes<NG, 1>(), lds2 = kv4_lds_bytes<NG, 2>();
    if (block_rows == 16) hipLaunchKernelGGL((kv4_attn_kernel<NG, 1>), grid, block, lds1, stream, a);
    else hipLaunchKernelGGL((kv4_attn_kernel<NG, 2>), grid, block, lds2, stream, a);
  } else {
    // Heads are the fastest: the workgroups of a head, which read the same keys, meet on few XCDs.
    hipLaunchKernelGGL((kv4_chunk_kernel<NG, kChunkRT>), dim3(a.hk, (unsigned)(a.row_blocks * a.splits), batch),
                       dim3(kWaves * 64), 0, stream, a);
  }
  if (a.splits > 1) {
    // about four splits a thread
    constexpr int units = 256 / (8 * NG);
    int lanes = 1;
    while (lanes * 2 <= units && lanes * 4 < a.splits) lanes *= 2;
    const int rows = units / lanes;
    const dim3 grid((unsigned)(a.row_blocks * ((block_rows + rows - 1) / rows)), a.hk, batch);
    hipLaunchKernelGGL((kv4_join_kernel<NG>), grid, dim3(256), 0, stream, a, block_rows, lanes, rows);
  }
}

}  // namespace

int64_t kv4_attn_workspace(const tilemix_kv4_attn_params& p) {
  Plan plan;
  return make_plan("tilemix_kv4_attn_workspace", p, plan) ? plan.bytes : -1;
}

int launch_kv4_attn(const tilemix_kv4_attn_params& p, hipStream_t stream) {
  const char* const what = "tilemix_kv4_attn";
  Plan plan;
  if (!make_plan(what, p, plan)) return TILEMIX_E_INVALID;
  if (p.batch == 0 || p.tokens_q == 0 || p.max_seqlen_q == 0) return TILEMIX_OK;
  if (p.q == nullptr || p.out == nullptr || p.seq_lens == nullptr ||
      (p.block_table == nullptr && p.table_columns > 0)) {
    set_error("%s: null pointer", what);
    return TILEMIX_E_INVALID;
  }
  if (plan.bytes > 0 && (p.workspace == nullptr || p.workspace_bytes < plan.bytes ||
                         (reinterpret_cast<uintptr_t>(p.workspace) & 15) != 0)) {
    set_error("%s: needs %lld bytes of 16-byte aligned workspace, got %lld", what, (long long)plan.bytes,
              (long long)p.workspace_bytes);
    return TILEMIX_E_INVALID;
  }
  const int width = (p.head_dim + kKv4Group - 1) / kKv4Group * kKv4Group;
  Kv4Args a{};
  a.q = p.q;
  a.out = p.out;
  a.kc = static_cast<const uint32_t*>(p.k_codes);
  a.kp = static_cast<const uint32_t*>(p.k_params);
  a.vc = static_cast<const uint32_t*>(p.v_codes);
  a.vp = static_cast<const uint32_t*>(p.v_params);
  a.table = p.block_table;
  a.lens = p.seq_lens;
  a.cu = p.cu_seqlens_q;
  a.part = static_cast<float*>(p.workspace);
  const int64_t parts = (int64_t)p.batch * p.heads_k * plan.row_blocks * plan.splits * plan.block_rows;
  if (plan.bytes > 0) a.part_ml = reinterpret_cast<float2*>(a.part + parts * width);
  a.sq_t = p.stride_q_token;
  a.sq_h = p.stride_q_head;
  a.so_t = p.stride_o_token;
  a.so_h = p.stride_o_head;
  a.s_table = p.stride_table;
  a.tokens = p.tokens_q;
  a.scale = p.sm_scale * kLog2eF32;
  a.pages = p.pages;
  a.hq = p.heads_q;
  a.hk = p.heads_k;
  a.group = p.heads_q / p.heads_k;
  a.d = p.head_dim;
  a.columns = p.table_columns;
  a.max_q = p.max_seqlen_q;
  a.max_k = p.max_seqlen_k;
  a.causal = p.causal;
  a.bf = p.dtype;
  a.q_vec = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && ((p.stride_q_token | p.stride_q_head) & 7) == 0;
  a.o_vec = (reinterpret_cast<uintptr_t>(p.out) & 7) == 0 && ((p.stride_o_token | p.stride_o_head) & 3) == 0;
  a.row_blocks = plan.row_blocks;
  a.splits = plan.splits;
  a.split_tiles = plan.split_tiles;
  a.by_page = make_fast_div(p.page_size);
  a.by_group = make_fast_div(a.group);
  a.by_splits = make_fast_div(a.splits);
  switch (width / kKv4Group) {
    case 1:
      launch_kv4<1>(a, plan.block_rows, p.batch, stream);
      break;
    case 2:
      launch_kv4<2>(a, plan.block_rows, p.batch, stream);
      break;
    case 3:
      launch_kv4<3>(a, plan.block_rows, p.batch, stream);
      break;
    default:
      launch_kv4<4>(a, plan.block_rows, p.batch, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return TILEMIX_E_LAUNCH;
  }
  return TILEMIX_OK;
}

}  // namespace tmx
