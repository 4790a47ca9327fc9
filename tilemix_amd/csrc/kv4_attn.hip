// Attention over the paged 4-bit cache (format and arguments: include/tilemix_hip.h).
//
// A workgroup takes one (sequence, KV head), up to 16 RT of its query rows -- a row is a (query token,
// query head of the group) pair -- and one piece of the keys.  Its four waves take the piece's
// 64-key tiles in turn and join their running maxima, sums and outputs in LDS at the end; with
// several pieces the parts go to the workspace and kv4_join_kernel adds them up.
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
// The chunk kernel's query rows, of a wave in 16s and of a workgroup.
constexpr int kChunkRT = 2, kChunkRows = kWaves * 16 * kChunkRT, kChunkShift = 7;
static_assert(1 << kChunkShift == kChunkRows, "rows of a block are a power of two");
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
  float* part;     // [head][unit][row][channel] sums, unnormalised
  float2* part_ml; // [head][unit][row] maximum, sum
  int2* notes;     // [sequence] number of its first workgroup, pieces
  int64_t sq_t, sq_h, so_t, so_h, s_table, tokens;
  float scale;
  int pages, hq, hk, group, d, columns, max_q, max_k, causal, bf, q_vec, o_vec;
  int batch, block_shift, row_blocks;  // rows of a block: 1 << block_shift; blocks of max_q
  int units, least, fit;               // workgroups of a head; see Kv4Splits
  int each;                            // tiles of a piece of an even split
  FastDiv by_page, by_group, by_heads, by_blocks, by_pieces, by_share, by_units;
};

// How a call's keys are split: not at all (an item is one workgroup's), into the same number of tiles everywhere, or
// by the sequences' lengths.
enum Kv4Split { kNoSplit, kEvenSplit, kBalancedSplit };

// The queries and keys of a sequence.
struct Kv4Seq {
  int start, nq, len;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Args& a, int b) {
  int64_t start = (int64_t)b * a.max_q;
  int nq = a.max_q;
  if (a.cu != nullptr) {
    start = a.cu[b];
    nq = a.cu[b + 1] - (int)start;
  }
  const bool inside = start >= 0 && start <= a.tokens;
  const int64_t room = min((int64_t)a.columns * a.by_page.d, (int64_t)a.max_k);
  Kv4Seq s;
  s.start = inside ? (int)start : 0;
  s.nq = inside ? max((int)min((int64_t)min(nq, a.max_q), a.tokens - start), 0) : 0;
  s.len = (int)min((int64_t)max(a.lens[b], 0), room);
  return s;
}

// One (sequence, KV head, block of query rows): its rows and keys.
struct Kv4Item : Kv4Seq {
  int b, h, rb;
  int rows;    // of all blocks
  int limit0;  // keys that query 0 sees (may be <= 0)
  int kmax;    // keys that the block's last row sees
};
__device__ __forceinline__ Kv4Item kv4_item(const Kv4Args& a, const Kv4Seq& seq, int b, int h, int rb) {
  Kv4Item it;
  static_cast<Kv4Seq&>(it) = seq;
  it.b = b;
  it.h = h;
  it.rb = rb;
  it.rows = it.nq * a.group;
  it.limit0 = a.causal ? it.len - it.nq + 1 : it.len;
  const int last = min(it.rows, (rb + 1) << a.block_shift) - 1;
  it.kmax = a.causal ? it.limit0 + fast_div(max(last, 0), a.by_group) : it.len;
  return it;
}

// ---- the keys of a call over the workgroups -----------------------------------------
// How long the sequences of a batch are is known on the device only.  Every wave adds them up (64 at a time, one a
// lane): `share` workgroups a head are to have the same work, `least` units of it at least; a sequence's blocks
// of rows are split into as many pieces as that gives, of one size.  The pieces of all sequences are
// numbered [sequence][block][piece]: a workgroup finds its own in the sums, about 1 us later than from its
// index alone.  That costs batches of one length 0 to 2 us and saves the others the wait for their longest
// sequence: calls in us, pieces of one size for all sequences / by their lengths (head_dim 128):
//   decode, 24/8 heads, 48 of 200 .. 6000 57.6 / 51.5; 24 of 700 .. 9001 (28/4 heads) 29.1 / 26.4; 16 x 2048 (32/8)
//   17.9 / 19.5; 32 x 4096 37.9 / 37.6;
//   8 queries, 16 of 500 .. 6000 43.9 / 35.5, 8 x 4000 22.8 / 24.4; 40 of 300 .. 2500 (6 queries, 24/4) 41.3 / 33.0;
//   256 queries, 4 of 600 .. 6000 122 / 77; 40 .. 100 queries, 8 of 500 .. 4000 87 / 49.
__device__ __forceinline__ int kv4_blocks(const Kv4Args& a, const Kv4Seq& s) {
  return (int)(((int64_t)s.nq * a.group + (1 << a.block_shift) - 1) >> a.block_shift);
}
__device__ __forceinline__ int kv4_tiles(int keys) {
  return keys <= 0 ? 0 : (int)(((uint32_t)keys + kTile - 1) / kTile);
}

// The units: rounds of the four waves, or pairs of tiles that they go through together.
__device__ __forceinline__ int kv4_work(const Kv4Args& a, int keys) {
  const int shift = a.block_shift == kChunkShift ? 1 : 2;
  return (kv4_tiles(keys) + (1 << shift) - 1) >> shift;
}

struct Kv4Splits {
  int unit;     // work of a piece
  Kv4Seq mine;  // of the lane's sequence, among the 64 at hand

  __device__ __forceinline__ Kv4Seq load(const Kv4Args& a, int c0) const {
    const int b = c0 + (threadIdx.x & 63);
    Kv4Seq s{};
    if (b < a.batch) s = kv4_seq(a, b);
    return s;
  }
  __device__ __forceinline__ explicit Kv4Splits(const Kv4Args& a) {
    uint32_t total = 0;
    for (int c0 = (a.batch - 1) & ~63; c0 >= 0; c0 -= 64) {
      mine = load(a, c0);
      const uint32_t work = (uint32_t)kv4_blocks(a, mine) * (uint32_t)kv4_work(a, mine.len);
      total += (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(work), 63);
    }
    // (below 2^31: fewer than 512 blocks of rows, of 2^22 units at most)
    unit = max(fast_div((int)(total + (uint32_t)a.by_share.d - 1), a.by_share), a.least);
    // Larger until the pieces are no more than the card takes at once, if that is asked for: with one more than
    // that on a CU all wait for it (8 queries, 8 of 500 .. 6000: 25.8 us, 29.9 without this).
    while (a.fit > 0 && unit < a.fit) {
      int all = 0;
      for (int c0 = (a.batch - 1) & ~63; c0 >= 0; c0 -= 64) {
        if (a.batch > 64) mine = load(a, c0);
        all += __builtin_amdgcn_readlane((int)wave_scan((uint32_t)pieces(a) * (uint32_t)kv4_blocks(a, mine)), 63);
      }
      if (all <= a.by_share.d) break;
      unit += unit / 8 + 1;
    }
  }
  // ceil(work / unit) = 1 + floor((work - 1/2) / unit), never more (the grid has no room for it): the factor is
  // below 1 by more than the quotient's rounding, and by less than what is left of 1/2 up to 2^19 units.
  __device__ __forceinline__ int pieces(const Kv4Args& a) const {
    const float work = (float)kv4_work(a, mine.len) - 0.5f;  // exact
    return 1 + (int)fmaxf(work * ((1.0f - 0x1p-20f) * __builtin_amdgcn_rcpf((float)unit)), 0.0f);
  }
};

// Where a workgroup stands: a piece of one (sequence, block of rows).
struct Kv4Place {
  Kv4Seq seq;
  int b, rb, split, pieces, in;  // in: number in the sequence
};
__device__ __forceinline__ Kv4Seq read_lane(const Kv4Seq& s, int lane) {
  return Kv4Seq{__builtin_amdgcn_readlane(s.start, lane), __builtin_amdgcn_readlane(s.nq, lane),
                __builtin_amdgcn_readlane(s.len, lane)};
}
// Of workgroup `unit` of a head; b = -1: there is none.
template <Kv4Split kSplit>
__device__ __forceinline__ Kv4Place kv4_place(const Kv4Args& a, int unit, int h) {
  if constexpr (kSplit != kBalancedSplit) {
    Kv4Place at{};
    const int item = fast_div(unit, a.by_pieces);
    at.pieces = a.by_pieces.d;
    at.split = unit - item * at.pieces;
    at.b = fast_div(item, a.by_blocks);
    at.rb = item - at.b * a.row_blocks;
    // The last blocks of rows, which see the most keys, go first (us, before / after: 8192 queries of 2 sequences, 24/8
    // heads x 128, 978 / 882; 4096 of 8 1005 / 955; 1 .. 1030 of 6 over up to 4100 keys, 32/8, 223 / 210).
    if (kSplit == kNoSplit) at.rb = a.row_blocks - 1 - at.rb;
    return at;
  }
  const int whole = unit;
  Kv4Splits s(a);
  Kv4Place at{};
  at.b = -1;
  for (int c0 = 0; c0 < a.batch; c0 += 64) {
    if (c0 > 0) s.mine = s.load(a, c0);
    // (with a cu out of order the sums may pass 32 bits: then no workgroup finds itself here, and whichever does
    // is within its sequence, as none is beyond it)
    const int pieces = s.pieces(a), mine = (int)((uint32_t)pieces * (uint32_t)kv4_blocks(a, s.mine));
    const int behind = (int)wave_scan((uint32_t)mine), all = __builtin_amdgcn_readlane(behind, 63);
    if (unit < all) {
      const int lane = __popcll(__ballot(behind <= unit));
      at.in = unit - __builtin_amdgcn_readlane(behind - mine, lane);
      at.seq = read_lane(s.mine, lane);
      at.pieces = __builtin_amdgcn_readlane(pieces, lane);
      at.b = c0 + lane;
      // (blocks: of the longest sequence, a sequence with one has no quotient to wait for)
      at.rb = a.row_blocks > 1 ? (int)((uint32_t)at.in / (uint32_t)at.pieces) : 0;
      at.split = at.in - at.rb * at.pieces;
      if (at.in == 0 && h == 0 && threadIdx.x == 0) a.notes[at.b] = make_int2(whole, at.pieces);  // for the join
      return at;
    }
    unit -= all;
  }
  return at;
}
// Tiles of a piece; kWhole: whole rounds of the waves.
template <bool kWhole>
__device__ __forceinline__ int piece_tiles(const Kv4Seq& s, int pieces) {
  const int tiles = kv4_tiles(s.len), work = kWhole ? (tiles + 3) / 4 : tiles;  // at most 2^24
  int each = (int)((float)work * __builtin_amdgcn_rcpf((float)pieces));  // (off by one)
  each += each * pieces < work ? 1 : 0;
  each += each * pieces < work ? 1 : 0;
  each = max(each, 1);
  return kWhole ? 4 * each : each;
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
    u32x4 w[NG];
#pragma unroll
    for (int s = 0; s < NG; ++s) w[s] = raw[rt][s];
    // bf16 queries are held as fp16 times a power of two of their row: exact but for elements below
    // 2^-14 of the row's largest, which lose no more than 2^-25 of that one.
    if (a.bf) {
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[s][e] << 16)),
                                 fabsf(__uint_as_float(w[s][e] & 0xffff0000u))));
      const int e2 = __builtin_amdgcn_frexp_expf(lanes16_max(top));
      scale[rt] = ldexpf(scale[rt], e2);
#pragma unroll
      for (int s = 0; s < NG; ++s)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const f16x2 h = {(f16)ldexpf(__uint_as_float(w[s][e] << 16), -e2),
                           (f16)ldexpf(__uint_as_float(w[s][e] & 0xffff0000u), -e2)};
          w[s][e] = __builtin_bit_cast(uint32_t, h);
        }
    }
    // in the pairs' order
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int s = 0; s < NG; ++s) {
      u32x4 r;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        r[2 * j] = __builtin_amdgcn_perm(w[s][j + 2], w[s][j], 0x05040100u) ^ sign;
        r[2 * j + 1] = __builtin_amdgcn_perm(w[s][j + 2], w[s][j], 0x07060302u) ^ sign;
      }
      qf[rt][s] = __builtin_bit_cast(f16x8, r);
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

// Bound by HBM where the card is full (64 x 8192 keys, 24/8 heads x 128: 672 MB in 123 us, 5.4 TB/s; its vector
// instructions, 600 a tile and wave of which the codes take 400, are 60% of that time), and for short or few sequences by
// the chain of loads before the first tile (lengths, table, codes: about 5 us) and the tiles that a wave takes
// one after the other.  Keys over the lanes and codes in registers leave LDS to V alone; waves take whole tiles
// so that none waits for another before the end.
template <int NG, int RT, Kv4Split kSplit>
__global__ void __launch_bounds__(kWaves * 64, RT == 1 ? 3 : 2) kv4_attn_kernel(const Kv4Args a) {
  using Tile = Kv4Tile<NG>;
  constexpr int kCT = 2 * NG;  // tiles of 16 channels
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15,
            g = lane >> 4;
  // KV heads are the fastest (kv4_chunk_kernel), but for one sequence's pieces, which are alike: 1 x 131072 37.5 us
  // with the heads slowest, 38.2 with them fastest.
  const int slow = fast_div(blockIdx.x, kSplit == kEvenSplit ? a.by_units : a.by_heads);
  const int fast = blockIdx.x - slow * (kSplit == kEvenSplit ? a.units : a.hk);
  const int unit = kSplit == kEvenSplit ? fast : slow, h = kSplit == kEvenSplit ? slow : fast;
  const Kv4Place at = kv4_place<kSplit>(a, unit, h);
  if (at.b < 0) return;
  // the first keys' places are on their way while the queries come
  int first = kSplit == kEvenSplit ? at.split * a.each : 0, each = a.each;
  if (kSplit == kBalancedSplit) {
    each = piece_tiles<true>(at.seq, at.pieces);
    first = at.split * each;
  }
  Kv4Walk walk;
  walk.table = a.table + at.b * a.s_table;
  walk.key0 = (first + wave) * kTile;
  walk.fetch(a, 0);
  const Kv4Item it = kv4_item(a, kSplit == kBalancedSplit ? at.seq : kv4_seq(a, at.b), at.b, h, at.rb);
  const int rb = at.rb, row0 = rb * 16 * RT;
  if (row0 >= it.rows) return;
  const bool joined = kSplit != kNoSplit && at.pieces > 1;
  int last = kv4_tiles(it.kmax);
  if (joined) {
    last = min(last, first + each);
    if (first >= last && at.split > 0) return;
  }
  walk.end = min(it.kmax, last * kTile);
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
  const int64_t part0 = ((int64_t)h * a.units + unit) * (16 * RT);
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
      if (joined && wave == 0 && g == 0)
        a.part_ml[part0 + 16 * rt + i] = make_float2(all_top, all_sum);
      const float norm = all_sum == 0.0f ? 0.0f : 1.0f / all_sum;
      for (int ct = wave; ct < kCT; ct += kWaves) {
        f32x4 r = lds_o[ct * 64 + lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) r += lds_o[(w * kCT + ct) * 64 + lane];
        const int c = 16 * ct + 4 * g;
        if (joined) {
          *reinterpret_cast<f32x4*>(a.part + (part0 + 16 * rt + i) * (32 * NG) + c) = r;
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
// With two workgroups a CU a tile of both takes 2.4 us (64000 keys: 815 TFLOP/s, 0.62 of a large GEMM's rate; the
// matrix instructions alone would take 1.5, vector instructions are issued 46% of the time).  512 queries at 8000 keys
// (24/8 heads x 128): 77 us, of which the conversion is 14, exp2 5, the start 10, the partial sums 5.
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

template <int NG, int RT, Kv4Split kSplit>
__global__ void __launch_bounds__(kWaves * 64, 2) kv4_chunk_kernel(const Kv4Args a) {
  constexpr int kCT = 2 * NG, kNP = Kv4Tile<NG>::kNP, kRows = kWaves * 16 * RT;
  __shared__ __attribute__((aligned(16))) ChunkLds<NG> lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15,
            g = lane >> 4;
  const int unit = fast_div(blockIdx.x, a.by_heads), h = blockIdx.x - unit * a.hk;
  const Kv4Place at = kv4_place<kSplit>(a, unit, h);
  if (at.b < 0) return;
  int first = kSplit == kEvenSplit ? at.split * a.each : 0, each = a.each;
  if (kSplit == kBalancedSplit) {
    each = piece_tiles<false>(at.seq, at.pieces);
    first = at.split * each;
  }
  // The rows of the pool of block `wave` of the tiles first + 64 c .. + 63, one in each lane (-1: no page).
  const int32_t* const table = a.table + at.b * a.s_table;
  auto key_of = [&](int n) { return (first + n + lane) * kTile + 16 * wave; };
  int ids = table_entry(a, table, key_of(0)), rows = -1;
  const Kv4Item it = kv4_item(a, kSplit == kBalancedSplit ? at.seq : kv4_seq(a, at.b), at.b, h, at.rb);
  const int rb = at.rb;
  if (rb * kRows >= it.rows) return;
  const bool joined = kSplit != kNoSplit && at.pieces > 1;
  int last = kv4_tiles(it.kmax);
  if (joined) {
    last = min(last, first + each);
    if (first >= last && at.split > 0) return;
  }
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
  const int at_end = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0));  // lane: no register holds it
  const int i_end = at_end & 15, g_end = at_end >> 4;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float all = sum[rt][0];
    const int row = row0 + 16 * rt + i_end, token = fast_div(row, a.by_group), head = row - token * a.group;
    if (row >= it.rows) continue;
    const int64_t part = ((int64_t)h * a.units + unit) * kRows + wave * 16 * RT + 16 * rt + i_end;
    if (joined && g_end == 0) a.part_ml[part] = make_float2(top[rt], all);
    const float norm = all == 0.0f ? 0.0f : 1.0f / all;
#pragma unroll
    for (int ct = 0; ct < kCT; ++ct) {
      const int c = 16 * ct + 4 * g_end;
      if (joined) *reinterpret_cast<f32x4*>(a.part + part * (32 * NG) + c) = o[rt][ct];
      else
        store_out(a.out, (it.start + token) * a.so_t + (it.h * a.group + head) * a.so_h + c, o[rt][ct] * norm, a.d - c,
                  a.o_vec, a.bf);
    }
  }
}

// Adds up the splits of a row.  One thread takes four channels of every `lanes`-th split and keeps
// its own running maximum; the `lanes` threads of a row's channels meet in LDS.
template <int NG>
__global__ void __launch_bounds__(256) kv4_join_kernel(const Kv4Args a, bool balanced, int lanes, int rows) {
  constexpr int kC = 8 * NG;
  __shared__ f32x4 lds_o[256];
  __shared__ float2 lds_ml[256];
  const int unit = threadIdx.x / kC, c = 4 * (threadIdx.x - unit * kC), r = unit / lanes, lane = unit - r * lanes;
  const int block_rows = 1 << a.block_shift, groups = (block_rows + rows - 1) / rows, rb = blockIdx.x / groups;
  const int in_block = (blockIdx.x - rb * groups) * rows + r;
  const Kv4Seq seq = kv4_seq(a, blockIdx.z);
  int before = blockIdx.z * a.row_blocks * a.by_pieces.d, pieces = a.by_pieces.d;
  if (balanced) {
    // (written by a workgroup of the sequence; what stands there if none was launched, with a cu out of order, is
    // bounded here)
    const int2 note = a.notes[blockIdx.z];
    before = note.x;
    pieces = note.y;
    if (pieces <= 1) return;  // it wrote the output
    if ((uint64_t)(uint32_t)before + (uint64_t)rb * (uint32_t)pieces >= (uint64_t)a.units) return;
  }
  const Kv4Item it = kv4_item(a, seq, blockIdx.z, blockIdx.y, rb);
  const int row = rb * block_rows + in_block;
  const bool there = r < rows && in_block < block_rows && row < it.rows;
  f32x4 o = {};
  float2 ml = make_float2(kNoKey, 0.0f);
  if (there) {
    const int each = !balanced                ? a.each
                     : block_rows == kChunkRows ? piece_tiles<false>(it, pieces)
                                                : piece_tiles<true>(it, pieces);
    // (no more than there are workgroups, whatever cu holds)
    const int parts = min(max(1, (kv4_tiles(it.kmax) + each - 1) / each), a.units - before - rb * pieces);
    const int64_t first = ((int64_t)it.h * a.units + before + rb * pieces) * block_rows + in_block;
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
  Kv4Split split;
  int block_shift, row_blocks, units, share, least, fit, each, pieces;
  int64_t bytes;
};


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
  // (rows of a sequence: no more than there are queries, however loose the bound)
  const int64_t group = p.heads_q / p.heads_k, rows = std::min<int64_t>(p.max_seqlen_q, p.tokens_q) * group;
  const int64_t keys = std::min<int64_t>(p.max_seqlen_k, (int64_t)p.table_columns * p.page_size);
  const int64_t tiles = std::max<int64_t>((keys + kTile - 1) / kTile, 1);
  // The chunk kernel needs rows to share its conversions among, and work that outweighs its start and end; the
  // other one takes the same rows 32 at a time.  Calls in us, blocks of 32 / chunk kernel (24/8 heads x 128, tiles
  // of blocks of 32): 90 rows 8 x 4000 41.3 / 42.6; 120 rows 1 x 4000 (2016) 17.5 / 29.5, 8 x 4000 (16128) 51.4 /
  // 44.2, 1 x 40000 (20000) 49.5 / 47.0; 300 rows 1 x 4000 (5040) 28.4 / 31.4, 1 x 40000 (50000) 111 / 88.
  const int64_t blocks32 = (rows + 31) / 32;
  const bool few = blocks32 * p.heads_k * p.batch * tiles <= 10000;
  const bool chunk = rows > 96 && !few;
  plan.block_shift = rows <= 16 ? 4 : chunk ? kChunkShift : 5;
  const int64_t block_rows = (int64_t)1 << plan.block_shift;
  const int64_t blocks = (rows + block_rows - 1) / block_rows;  // of a sequence, at most
  int64_t units = blocks * p.batch;                             // workgroups of a head
  if (p.max_seqlen_q * group > INT32_MAX / 2 || units * p.heads_k >= 1 << 24) {
    set_error("%s: too many queries for one call (%lld rows a sequence, batch %d)", what,
              (long long)(p.max_seqlen_q * group), p.batch);
    return false;
  }
  plan.share = plan.least = plan.fit = plan.each = 0;
  plan.pieces = 1;
  plan.bytes = 0;
  plan.split = kNoSplit;
  const int64_t items = std::max<int64_t>(std::min(units, p.tokens_q * group / block_rows + p.batch) * p.heads_k, 1);
  // A split costs the join (a second launch, 4 us) and each workgroup's start and end (3 us, 10 with the chunk
  // kernel): none for short sequences or where the items fill the card.  Calls in us (24/8 heads x 128 unless
  // said), whole / split: 1 x 700 (14/2 heads x 64) 8.2 / 9.5; 16 x 512 10.0 / 11.8; 8 x 1024 13.0 / 15.3; 32 x 1024
  // 15.2 / 17.4; but 1 x 1024 12.9 / 11.5; 64 x 8192 126 / 131.
  if (chunk ? items < 256 && tiles >= 16 : items < 512 && tiles > (items < 64 ? 12 : 16)) {
    if (p.batch == 1) {
      // Two workgroups a CU: 1 x 131072 in 64 pieces 42.4, 48 45.7, 96 46.6.
      const int64_t whole = chunk ? 1 : kWaves;
      const int64_t pieces = std::max<int64_t>(std::min(512 / items, tiles / (chunk ? 8 : 4)), 1);
      plan.each = (int)(((tiles + pieces - 1) / pieces + whole - 1) / whole * whole);
      plan.pieces = (int)((tiles + plan.each - 1) / plan.each);
      plan.split = plan.pieces > 1 ? kEvenSplit : kNoSplit;
      units *= plan.pieces;
    } else {
      plan.split = kBalancedSplit;
      plan.share = (int)std::max<int64_t>((plan.block_shift == 5 && items <= 96 ? 256 : 512) / p.heads_k, 1);
      // Blocks of 32 rows hold two workgroups a CU, and do best with one where that gives pieces short enough: 8 of
      // 1500 .. 6144 (5 queries, 32/8 heads; 64 items) 26.1 with 256 workgroups, 30.4 with 512; 16 of 500 .. 6000 (8
      // queries, 128 items) 42.9 / 35.5.  Those of 16 rows hold three: room for what is over.
      if (plan.block_shift == 4) {
        plan.least = items < 64 ? 1 : 4;
        units = items / p.heads_k + plan.share;
      } else {
        plan.least = chunk ? 4 : 2;
        plan.fit = (int)((tiles + 1) / 2);  // (no piece has more work)
        units = std::max<int64_t>(items / p.heads_k, plan.share);
      }
      plan.pieces = (int)std::min<int64_t>(units * p.heads_k / items, (tiles + 3) / 4);  // on average
    }
  }
  if (plan.split != kNoSplit) {
    const int64_t width = (p.head_dim + kKv4Group - 1) / kKv4Group * kKv4Group;
    plan.bytes = units * p.heads_k * block_rows * (width * 4 + 8) + p.batch * 8;
  }
  plan.row_blocks = (int)blocks;
  plan.units = (int)units;
  return true;
}

template <int NG, Kv4Split kSplit>
void launch_split(const Kv4Args& a, hipStream_t stream) {
  // KV heads are the fastest: the workgroups of a head, which read the same keys, meet on few XCDs.
  const dim3 grid((unsigned)a.units * a.hk), block(kWaves * 64);
  constexpr int lds1 = kv4_lds_bytes<NG, 1>(), lds2 = kv4_lds_bytes<NG, 2>();
  if (a.block_shift == 4) hipLaunchKernelGGL((kv4_attn_kernel<NG, 1, kSplit>), grid, block, lds1, stream, a);
  else if (a.block_shift == 5) hipLaunchKernelGGL((kv4_attn_kernel<NG, 2, kSplit>), grid, block, lds2, stream, a);
  else hipLaunchKernelGGL((kv4_chunk_kernel<NG, kChunkRT, kSplit>), grid, block, 0, stream, a);
}

template <int NG>
void launch_kv4(const Kv4Args& a, const Plan& plan, hipStream_t stream) {
  if (plan.split == kNoSplit) launch_split<NG, kNoSplit>(a, stream);
  else if (plan.split == kEvenSplit) launch_split<NG, kEvenSplit>(a, stream);
  else launch_split<NG, kBalancedSplit>(a, stream);
  if (plan.split == kNoSplit) return;
  // about four pieces a thread
  constexpr int units = 256 / (8 * NG);
  const int block_rows = 1 << a.block_shift;
  int lanes = 1;
  while (lanes * 2 <= units && lanes * 4 < plan.pieces) lanes *= 2;
  const int rows = units / lanes;
  const dim3 grid((unsigned)(a.row_blocks * ((block_rows + rows - 1) / rows)), a.hk, a.batch);
  hipLaunchKernelGGL((kv4_join_kernel<NG>), grid, dim3(256), 0, stream, a, plan.split == kBalancedSplit, lanes, rows);
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
  if (plan.bytes > 0) {
    const int64_t parts = ((int64_t)plan.units * p.heads_k) << plan.block_shift;
    a.part_ml = reinterpret_cast<float2*>(a.part + parts * width);
    a.notes = reinterpret_cast<int2*>(a.part_ml + parts);
  }
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
  a.batch = p.batch;
  a.block_shift = plan.block_shift;
  a.row_blocks = plan.row_blocks;
  a.units = plan.units;
  a.least = plan.least;
  a.fit = plan.fit;
  a.each = plan.each;
  a.by_page = make_fast_div(p.page_size);
  a.by_group = make_fast_div(a.group);
  a.by_heads = make_fast_div(a.hk);
  a.by_blocks = make_fast_div(a.row_blocks);
  a.by_pieces = make_fast_div(plan.split == kEvenSplit ? plan.pieces : 1);
  a.by_units = make_fast_div(a.units);
  a.by_share = make_fast_div(std::max(plan.share, 1));
  switch (width / kKv4Group) {
    case 1:
      launch_kv4<1>(a, plan, stream);
      break;
    case 2:
      launch_kv4<2>(a, plan, stream);
      break;
    case 3:
      launch_kv4<3>(a, plan, stream);
      break;
    default:
      launch_kv4<4>(a, plan, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) {
    set_error("%s: launch failed: %s", what, hipGetErrorString(e));
    return TILEMIX_E_LAUNCH;
  }
  return TILEMIX_OK;
}

}  // namespace tmx
