// Attention of a ragged batch's new tokens over a paged K/V cache:
//   o_n = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q_n.k_j - m),
// j over the cached positions up to the token's own, all of them or those of
// the 64-key blocks listed for the token's 64-position block; m a running
// maximum, sums in 32 bits, p rounded to the matrix cores' 16 bits (an error of
// half a step a weight, of the size of the output's own rounding; in f16, which
// has few exponents, of 2^-32 of the largest weight for those below 2^-21 of it).
//
// Rows of one (sequence, KV head) are packed token by token, head by head
// (row r: token r / G, query head g G + r % G), so few tokens of a wide group
// fill a matrix tile as many tokens of a narrow one do.  What bounds a row tile
// turns with its height: up to 32 packed rows (a decoding step, a few drafted
// tokens) each key is read for few products and memory is the bound; above,
// the matrix cores are.  A workgroup of eight waves works on one unit (a row
// tile against a range of its keys) in one of two ways:
//   few rows    32 rows; every wave takes 32 keys at a time of its own,
//               without a barrier until the waves' sums are joined;
//   many rows   256 rows, 32 a wave; all waves share each 64-key block in LDS.
// A batch may mix them: a launch each (both in one kernel needed more
// registers than there are).
//
// How the units come about is decided on the host, from the sizes alone (the
// lengths are on the device).  Where there are few keys, or tiles enough for
// all CUs, a workgroup takes a tile whole.  Otherwise the tiles of a head stand
// in one line, each as long as it has keys, and a fixed number of workgroups
// shares the line out evenly, whatever the lengths are; tiles cut by a border
// are joined by a second kernel, in the line's order, so results do not depend
// on timing.  (Equal parts of each sequence instead: 64 sequences of 6 to 32
// thousand keys 590 us rather than 512 at that stage.)
//
// Measured on one MI355X (bf16 but for the drafts, heads of 128 but for theirs):
//   one token of each of 64 sequences of 6554 to 32768 keys, 28/4 heads, pages of 16: 440 us, 5.87 TB/s
//   four drafted tokens of each of 16 sequences of 1800 to 9001 keys, 16/8 heads of 64: 44 us, 4.3 TB/s
//   one token over 517 keys, 8/2 heads: 12 us
//   512 tokens over 33000 keys, 28/4 heads: 260 us, 925 TFLOP/s
//   4096 tokens over 32768 keys, 32/8 heads: 1922 us, 1070 TFLOP/s (pages of 128; of 16 6% longer)
//   2048 tokens over 64 listed blocks each, 28/4 heads: 141 us, 847 TFLOP/s
//   one token of each of 64 sequences over 64 listed blocks, 28/4 heads: 116 us
#pragma once

#include "attention_impl.h"
#include "paged.h"

namespace spruce {

struct PagedAttn {
  const void* q;
  void* out;
  int64_t qs[2], os[2];  // token, head strides
  const void* k;
  const void* v;
  int64_t ks[3], vs[3];  // page, head, slot strides
  PagedBatch batch;
  int Hkv, G;
  Divisor by_heads, by_group;  // by Hkv and G
  float cs;  // scale * log2 e
  const int32_t* idx;  // block lists [S, Hkv, Qc, K], or null
  int64_t is[3];
  int Qc, K;
  int few_limit;   // packed rows of a sequence up to which it goes the few-row way
  int groups;      // workgroups of a head that share its keys out
  float* part_o;   // [groups][32 * D], a 32 x 32 accumulator's order
  float* part_ml;  // [groups][2][32]
  int4* begun;     // what each workgroup's stretch ends within
};

constexpr int kWaves = 8;
constexpr int kCus = 256;       // a workgroup fills a CU's registers

// Unit shapes: packed rows of a tile, and its fixed part (look-ups, first loads,
// last sums, store) in keys.
struct Few {
  static constexpr int rows = 32, cost = 768;
};
struct Many {
  static constexpr int rows = 32 * kWaves, cost = 512;
};

typedef float f32x4v __attribute__((ext_vector_type(4)));
// 16 bytes of a row.  A native vector: copies of the struct uint4 between
// memory spaces have kept arrays of it out of registers.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ u32x4 load16(const uint16_t* p) { return *reinterpret_cast<const u32x4*>(p); }

// The same of what is read but once: not kept in the caches, which a pass over
// a large cache of keys would only fill in vain.
__device__ __forceinline__ u32x4 load16_once(const uint16_t* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

template <bool F16>
__device__ __forceinline__ f32x4v mfma16x16x32(u32x4 a, u32x4 b, f32x4v c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// The kernel's arguments, read from memory again where they are next used:
// kept in scalar registers over a loop that does not need them, they push out
// what it does need.  (PagedAttn is the kernels' only argument.)
template <typename T>
__device__ __forceinline__ T* global(T* p) {
  return (T*)(__attribute__((address_space(1))) T*)p;
}
__device__ __forceinline__ PagedAttn arguments(uintptr_t k) {
  asm volatile("" : "+s"(k));
  PagedAttn p = *(const PagedAttn*)(const __attribute__((address_space(4))) PagedAttn*)k;
  // Pointers read from memory might point anywhere; these are global.
  p.q = global(p.q);
  p.out = global(p.out);
  p.k = global(p.k);
  p.v = global(p.v);
  p.idx = global(p.idx);
  p.part_o = global(p.part_o);
  p.part_ml = global(p.part_ml);
  p.begun = global(p.begun);
  p.batch.table = global(p.batch.table);
  p.batch.q_starts = global(p.batch.q_starts);
  p.batch.kv_lens = global(p.batch.kv_lens);
  return p;
}

// The same value in every lane, for the compiler too: it must branch on the
// scalar unit around matrix instructions, which run whatever EXEC holds.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// The lane below's value by `n` (row shifts within 16 lanes, then the rows'
// last lanes onward), zero from outside: the steps of a prefix sum.
template <int CTRL, int ROWS>
__device__ __forceinline__ int shifted(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t shifted(int64_t v) {
  const int lo = shifted<CTRL, ROWS>((int)v), hi = shifted<CTRL, ROWS>((int)(v >> 32));
  return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
// Sum of v over the lanes up to this one.
template <typename T>
__device__ __forceinline__ T wave_prefix(T v) {
  v += shifted<0x111, 0xf>(v);
  v += shifted<0x112, 0xf>(v);
  v += shifted<0x114, 0xf>(v);
  v += shifted<0x118, 0xf>(v);
  v += shifted<0x142, 0xa>(v);
  v += shifted<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ int64_t lane_of(int64_t v, int l) {
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32) |
                   (uint32_t)__builtin_amdgcn_readlane((int)v, l));
}

// a / b of no negative numbers, by way of 32 bits where both fit.
__device__ __forceinline__ int64_t divided(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  return a / b;
}

// A key of a tile, or the last key below `end` where it lies past that.
__device__ __forceinline__ int nearest(int key, int end) { return key < end ? key : end - 1; }

// A position as an int: -1 for any below zero, the largest int for any past it.
__device__ __forceinline__ int clip(int64_t pos) {
  return pos < 0 ? -1 : (pos < 0x7fffffff ? (int)pos : 0x7fffffff);
}

// The work of one sequence, of one kind: its row tiles per KV head, and how
// they weigh.  Tile j weighs first + slope (j + 1), G to a key: its keys, and
// its fixed part.  (An upper bound of the keys: what a tile does not have,
// nobody walks.)
struct SeqWork {
  int start, n;  // first packed row, new tokens
  int64_t pos0;  // position of the first
  int tiles;     // 0 where the sequence is of the other kind
  int rows;      // packed rows of a tile
  int sub;       // with lists: tiles of one 64-position block
  int64_t first, slope;
  __device__ __forceinline__ int64_t before(int64_t j) const { return first * j + slope * (j * (j + 1) / 2); }
};

// A sequence's lengths as the caller gives them.
struct Lengths {
  int starts, ends, keys;
};
__device__ __forceinline__ Lengths lengths_of(const PagedAttn& p, int s) {
  if (s >= p.batch.S) return Lengths{0, 0, 0};
  return Lengths{p.batch.q_starts[s], p.batch.q_starts[s + 1], p.batch.kv_lens[s]};
}

template <typename SHAPE>
__device__ __forceinline__ SeqWork sequence_work(const PagedAttn& p, const Lengths& len) {
  constexpr bool kMany = SHAPE::rows > Few::rows;
  SeqWork w{};
  const int a = clamp_start(p.batch, len.starts), e = clamp_start(p.batch, len.ends);
  w.start = a;
  w.n = e > a ? e - a : 0;
  // Positions go by the lengths as given; only what they address is bounded.
  w.pos0 = (int64_t)len.keys - ((int64_t)len.ends - len.starts) + ((int64_t)a - len.starts);
  const int64_t packed = (int64_t)w.n * p.G;
  if (w.n == 0 || (packed > p.few_limit) != kMany) return w;
  int64_t base = w.pos0 < 0 ? 0 : (w.pos0 < p.batch.cap ? w.pos0 : p.batch.cap);
  w.rows = SHAPE::rows;
  if (p.idx != nullptr) {
    const int64_t b0 = w.pos0 >> 6, b1 = (w.pos0 + w.n - 1) >> 6;
    const int rows = (w.n < kBlock ? w.n : kBlock) * p.G;
    w.sub = (rows + SHAPE::rows - 1) / SHAPE::rows;
    w.rows = ((rows + 31) / 32 + w.sub - 1) / w.sub * 32;  // shared out evenly
    w.tiles = (int)(b1 - b0 + 1) * w.sub;
    base = (int64_t)p.K * kBlock;
  } else {
    w.tiles = (int)((packed + SHAPE::rows - 1) / SHAPE::rows);
    w.slope = SHAPE::rows;  // the last row of tile j is of token rows (j + 1) / G at most
    base += 1;
  }
  w.first = (base + SHAPE::cost) * p.G;
  return w;
}

// What a workgroup works on: all tiles of all sequences of one kind stand in
// one line per head, each as long as it weighs, and a head's workgroups share
// its line out evenly, whatever the lengths are.  A stretch may end within a
// tile; the sums of such parts go to the workgroup's two slots and are joined
// afterwards.  The heads' workgroups alternate: those of all heads are at the
// same keys at a time, which lie together in memory, and as workgroups go to
// the eight XCDs in turn, each L2 serves one head where their number divides 8.
struct Line {
  int64_t total, share;
};

// `w0`: the work of sequence `lane`, which most batches need no more than.
template <typename SHAPE>
__device__ __forceinline__ Line line_of(const PagedAttn& p, const SeqWork& w0, int lane) {
  Line line{0, 1};
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const SeqWork w = s0 == 0 ? w0 : sequence_work<SHAPE>(p, lengths_of(p, s0 + lane));
    line.total += lane_of(wave_prefix(w.before(w.tiles)), 63);
  }
  // Parts of fewer than 256 keys cost more than they save.
  line.share = divided(line.total + p.groups - 1, p.groups);
  const int64_t least = (int64_t)(SHAPE::cost + 256) * p.G;
  if (line.share < least) line.share = least;
  return line;
}

struct Unit {
  int s, tile, g;
  int64_t start, end;  // of the tile in the line
  SeqWork w;
};

__device__ __forceinline__ void take_sequence(Unit& u, const SeqWork& w, int s0, int l) {
  u.s = s0 + l;
  u.w.start = __builtin_amdgcn_readlane(w.start, l);
  u.w.n = __builtin_amdgcn_readlane(w.n, l);
  u.w.pos0 = lane_of(w.pos0, l);
  u.w.tiles = __builtin_amdgcn_readlane(w.tiles, l);
  u.w.rows = __builtin_amdgcn_readlane(w.rows, l);
  u.w.sub = __builtin_amdgcn_readlane(w.sub, l);
  u.w.first = lane_of(w.first, l);
  u.w.slope = lane_of(w.slope, l);
}

// The at-th of the row tiles, of a sequence the last first: they see the most
// keys.  False behind the last.  (The line is not measured.)
template <typename SHAPE>
__device__ __forceinline__ bool find_tile(const PagedAttn& p, int at, int g, int lane, Unit& u) {
  constexpr int kMost = 1 << 24;  // a call has fewer; starts that overlap may claim any number
  int count = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const SeqWork w = sequence_work<SHAPE>(p, lengths_of(p, s0 + lane));
    const int pc = count + wave_prefix(w.tiles < kMost ? w.tiles : kMost);
    const uint64_t past = __ballot(pc > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      take_sequence(u, w, s0, l);
      u.g = g;
      u.tile = __builtin_amdgcn_readlane(pc, l) - 1 - at;
      u.start = u.end = 0;
      return u.tile < u.w.tiles;
    }
    count = __builtin_amdgcn_readlane(pc, 63);
  }
  return false;
}

// The tile of head g at place `at` of the line.  False behind the last.
template <typename SHAPE>
__device__ __forceinline__ bool find_unit(const PagedAttn& p, const SeqWork& w0, int64_t at, int g, int lane, Unit& u) {
  int64_t places = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const SeqWork w = s0 == 0 ? w0 : sequence_work<SHAPE>(p, lengths_of(p, s0 + lane));
    const int64_t pp = wave_prefix(w.before(w.tiles));
    const uint64_t past = __ballot(places + pp > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      take_sequence(u, w, s0, l);
      u.g = g;
      if (u.w.tiles <= 0) return false;
      const int64_t origin = places + lane_of(pp, l) - u.w.before(u.w.tiles);
      int64_t j;
      if (u.w.slope == 0) {
        j = divided(at - origin, u.w.first);
      } else {
        // The tile j with before(j) <= y < before(j + 1).
        const int64_t y = at - origin;
        const double b = (double)u.w.first + 0.5 * (double)u.w.slope;
        j = (int64_t)((sqrt(b * b + 2.0 * (double)u.w.slope * (double)y) - b) / (double)u.w.slope);
        j = j < 0 ? 0 : (j < u.w.tiles ? j : u.w.tiles - 1);
        while (j > 0 && u.w.before(j) > y) --j;
        while (j + 1 < u.w.tiles && u.w.before(j + 1) <= y) ++j;
      }
      if (j < 0 || j >= u.w.tiles) return false;  // starts that overlap
      u.tile = uniform((int)j);
      u.start = origin + u.w.before(u.tile);
      u.end = origin + u.w.before(u.tile + 1);
      return true;
    }
    places += lane_of(pp, 63);
  }
  return false;
}

// A workgroup's part of a tile: tiles of KEYS keys [lo, hi) of the row's keys
// or list, its slot for the sums (-1: it holds the tile whole), and, of a
// tile's first part, the turn that has the last one (-1: not the first).
struct Part {
  int lo, hi, slot, last;
};
constexpr Part kWhole{0, 0x7fffffff, -1, -1};

// For the join: a tile begun, but not ended, in a workgroup's stretch.
__device__ __forceinline__ void note_begun(const PagedAttn& p, const Part& part, int row0, int rows, int start) {
  if (part.last >= 0 && threadIdx.x == 0) p.begun[blockIdx.x] = int4{row0, rows | (part.slot & 1) << 16, start, part.last};
}

template <typename SHAPE, int KEYS>
__device__ __forceinline__ Part part_of(const Line& line, const Unit& u, int G, int64_t from, int64_t to, int64_t turn) {
  Part part = kWhole;
  if (from > u.start || to < u.end) {
    // Neighbours round the border between them alike.
    auto border = [&](int64_t at) {
      const int64_t key = at - u.start - (int64_t)SHAPE::cost * G;
      const int64_t tiles = key <= 0 ? 0 : divided(key + KEYS * G - 1, KEYS * G);
      return tiles < 1 << 30 ? (int)tiles : 1 << 30;
    };
    part.lo = uniform(border(from));
    if (to < u.end) {
      part.hi = uniform(border(to));
      if (from <= u.start) part.last = uniform((int)divided(u.end - 1, line.share));
    }
    part.slot = uniform((int)(2 * blockIdx.x + (from > turn * line.share ? 1 : 0)));
  }
  return part;
}

// Rows [row0, row0 + rows) of a unit in the sequence's packed rows, the block
// list that they share, and the keys below `end` that the last of them sees.
struct TileRows {
  int row0, rows, end;
  const int32_t* list;
};

__device__ __forceinline__ TileRows tile_rows(const PagedAttn& p, const Unit& u) {
  TileRows t{};
  int left;
  if (p.idx != nullptr) {
    const int bi = u.tile / u.w.sub, sub = u.tile - bi * u.w.sub;
    const int64_t lo = (((u.w.pos0 >> 6) + bi) << 6) - u.w.pos0;
    const int t0 = lo < 0 ? 0 : (int)lo;
    const int t1 = lo + kBlock < u.w.n ? (int)(lo + kBlock) : u.w.n;
    t.row0 = t0 * p.G + sub * u.w.rows;
    left = t1 * p.G - t.row0;
    t.list = bi < p.Qc ? p.idx + (int64_t)u.s * p.is[0] + (int64_t)u.g * p.is[1] + (int64_t)bi * p.is[2] : nullptr;
  } else {
    t.row0 = u.tile * u.w.rows;
    left = u.w.n * p.G - t.row0;
  }
  t.rows = uniform(left < 0 ? 0 : (left < u.w.rows ? left : u.w.rows));
  t.row0 = uniform(t.row0);
  const int64_t last = u.w.pos0 + p.by_group.of(t.row0 + t.rows - 1);
  t.end = uniform(last < 0 || p.batch.pages == 0 ? 0 : (last + 1 < p.batch.cap ? (int)(last + 1) : p.batch.cap));
  return t;
}

// The first keys of the tiles of KEYS keys that a wave (or a workgroup) takes,
// in order: items base, base + stride .. below hi of the row's keys, or of its
// list's blocks without those that are padding or in every row's future.  64
// items of a list are looked up at once, one a lane.
template <int KEYS>
struct KeyWalk {
  const int32_t* list;
  int base, stride, hi, end, lane, found;
  bool lists;
  uint64_t bits;
  __device__ __forceinline__ void init(const PagedAttn& p, const TileRows& t, int base_, int stride_, int hi_, int lane_) {
    lists = p.idx != nullptr;
    list = t.list;
    base = uniform(base_);
    stride = stride_;
    hi = uniform(lists && list == nullptr ? 0 : hi_);
    end = t.end;
    lane = lane_;
    bits = 0;
    found = -1;
  }
  __device__ __forceinline__ int next() {
    if (!lists) {  // hi is at most the tiles below `end`
      if (base >= hi) return -1;
      const int key = base * KEYS;
      base += stride;
      return key;
    }
    while (bits == 0) {
      if (base >= hi) return -1;
      const int item = base + stride * lane;
      int64_t key = end;
      if (item < hi) {
        const int id = list[KEYS == kBlock ? item : item >> 1];
        if (id >= 0) key = (int64_t)id * kBlock + (KEYS == kBlock ? 0 : (item & 1) * KEYS);
      }
      const bool ok = key < end;
      found = ok ? (int)key : -1;
      bits = __ballot(ok);
      base += 64 * stride;
    }
    const int l = __builtin_ctzll(bits);
    bits &= bits - 1;
    return __builtin_amdgcn_readlane(found, l);
  }
};

// Where element (row, d) of a unit's 32-row group lies in its partial sums.
__device__ __forceinline__ int part_at(int row, int d) {
  return ((d >> 3) * 64 + row + 32 * ((d >> 2) & 1)) * 4 + (d & 3);
}

// Weights of f16 are 2^kLift times as large, their sum with them, so that what
// lies far below a row's largest score keeps its bits: normal down to 2^-21 of
// the running maximum, and at 2^(8 + 7), the most above it, still finite.
template <bool F16>
constexpr float kLift = F16 ? 7.f : 0.f;

// fmaf(s, cs, -m cs) is off by the rounding of m cs alone, for all of a row
// alike: nothing, until half a step of it leaves the weights' range.  A unit whose
// maximum reaches this size is done again like one with sums that are not
// finite; there m is taken off first.
constexpr float kLargeScore = 0x1p+22f;

// x combined over the lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float quad_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return half_max(fmaxf(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1)));
}
__device__ __forceinline__ float quad_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return half_sum(__builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1));
}

// Orders a wave's own LDS accesses, for the compiler; the hardware keeps them in order.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Zero, unknown to the compiler.
__device__ __forceinline__ int opaque_zero() {
  int z = 0;
  asm volatile("" : "+v"(z));
  return z;
}

constexpr int kFewKeys = 32;  // keys of a wave's tile
template <int D>
constexpr int few_lds_bytes() {
  // Every wave's V rows, or later its O rows, 16 at a time; then the waves'
  // maxima and sums, and which of the waves has a unit to do again.
  static_assert(16 * (D + 4) * 4 <= kFewKeys * (D + 8) * 2, "a wave's O rows must fit its V rows");
  return kWaves * (kFewKeys * (D + 8) * 2 + 2 * 32 * 4 + 4);
}
template <int D>
constexpr int many_lds_bytes() {
  return 2 * kBlock * ((D + 8) + (D + 32)) * 2;
}

// A few-row unit.  Memory bounds it: a key's 4 D bytes meet at most 32 rows.
// A wave's K and V rows come from memory as whole rows (D / 8 lanes of 16 bytes
// each; 64 bytes of 16 rows a load, the operands' own order, took 496 us where
// this takes 470), past the caches (440), and go through the wave's own LDS,
// K's first: read back row by row they are the A operand of S^T = K Q^T, V's by
// the transposing read that of O^T = V^T P^T; P^T, the B operand, is S^T's
// accumulator as it lies (keys 4 (l / 16) + r).  The next tile's K is in flight
// from this one's LDS write on, its V likewise.  Tiles of 64 keys at D = 64: 57.6
// us where 32 took 55.2 (four drafted tokens of 16 sequences).
//
// A masked key has p = 0, but 0 times a NaN or infinity in its value row is
// NaN.  Where sums come out non-finite, or a maximum is of a size that the usual
// exponent does not hold (kLargeScore), nothing is written and the result is
// true: the unit is then done again, CAREFUL, with the partly masked tiles
// taken one column at a time.
template <int D, bool F16, bool CAREFUL>
__device__ __forceinline__ bool few_rows(uintptr_t args, const Unit& u, const Part& part, char* smem) {
  const PagedAttn p = arguments(args);
  constexpr int KEYS = kFewKeys, KT = KEYS / 16, KH = KEYS / 32;  // 16- and 32-key pieces of a tile
  constexpr int KK = D / 32;   // steps of S^T over d
  constexpr int DT = D / 16;   // 16-row tiles of O^T
  constexpr int VSTR = D + 8;  // V rows in LDS, 16-bit elements
  constexpr int OSTR = D + 4;  // O rows in LDS, floats
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  float* ml = reinterpret_cast<float*>(smem + kWaves * kFewKeys * VSTR * 2);  // [wave][2][32]
  int* odds = reinterpret_cast<int*>(ml + kWaves * 64);                     // [wave]

  const TileRows tr = tile_rows(p, u);
  if (tr.rows == 0) return false;  // uniform: before any barrier
  const int token0 = u.w.start;
  const bool two = tr.rows > 16;  // the second 16 columns hold rows

  // This lane's two rows: position and query fragment.  Columns past the last
  // row repeat it, and keys past the last seen one below: every load has an
  // address, none is under a branch.
  int qpos[2];
  u32x4 qf[2][KK];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = tr.row0 + (16 * c + l16 < tr.rows ? 16 * c + l16 : tr.rows - 1);
    const int t = p.by_group.of(r), h = r - t * p.G;
    qpos[c] = clip(u.w.pos0 + t);
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t)(token0 + t) * p.qs[0] +
                          (int64_t)(u.g * p.G + h) * p.qs[1] + 8 * g4;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[c][kk] = load16(src + 32 * kk);
  }
  const int first_pos = uniform(clip(u.w.pos0 + p.by_group.of(tr.row0)));
  const int items = p.idx ? kBlock / KEYS * p.K : (tr.end + KEYS - 1) / KEYS;
  const int hi = part.hi < items ? part.hi : items;

  // Rows as memory has them: LROWS at a time, this lane's lr-th of those, 16 bytes at 8 lc.
  constexpr int LROWS = 512 / D, LI = KEYS / LROWS;
  const int lr = lane / (D / 8), lc = lane % (D / 8);
  const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + (int64_t)u.g * p.ks[1] + 8 * lc;
  const uint16_t* vbase = static_cast<const uint16_t*>(p.v) + (int64_t)u.g * p.vs[1] + 8 * lc;
  uint16_t* vl = reinterpret_cast<uint16_t*>(smem) + wave * KEYS * VSTR;

  // Table entries of the keys key0 + 16 c + l16.
  auto pages_of = [&](int key0, int (&pg)[KT]) {
#pragma unroll
    for (int c = 0; c < KT; ++c) pg[c] = page_entry(p.batch, u.s, nearest(key0 + 16 * c + l16, tr.end));
  };
  auto load = [&](const uint16_t* base, const int64_t* st, int key0, const int (&pg)[KT], u32x4 (&x)[LI]) {
#pragma unroll
    for (int i = 0; i < LI; ++i) {
      const int entry = __shfl(pg[i * LROWS / 16], i * LROWS % 16 + lr);
      const int key = nearest(key0 + i * LROWS + lr, tr.end);
      const int slot = key - page_of(p.batch, key) * p.batch.page;
      x[i] = load16_once(base + (int64_t)(is_page(p.batch, entry) ? entry : 0) * st[0] + (int64_t)slot * st[2]);
    }
  };
  auto keep = [&](const u32x4 (&x)[LI]) {
#pragma unroll
    for (int i = 0; i < LI; ++i) *reinterpret_cast<u32x4*>(vl + (i * LROWS + lr) * VSTR + 8 * lc) = x[i];
    wave_lds_fence();
  };

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // m: of the scores as products, before cs
  const float threshold = fminf(kRescaleThreshold / p.cs, 0x1.fffffep+127f);  // -inf's distance is past it
  f32x4v acc[2][DT];
  // Zeros that are no constant: constant ones are kept in registers, or worse,
  // for every later use of a zero.
  const float zero = __builtin_bit_cast(float, opaque_zero());
  {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[c][dt] = f32x4v{zero, zero, zero, zero};
    }
    KeyWalk<KEYS> walk;
    walk.init(p, tr, part.lo + wave, kWaves, hi, lane);
    // Keys and table entries of this tile, the next and the one after: entries
    // are looked up a tile before the loads that they address are issued.
    int pg[KT], pn[KT], pa[KT];
    u32x4 kx[LI], vx[LI];
    int key0 = walk.next(), nkey = -1;
    if (key0 >= 0) {
      pages_of(key0, pg);
      nkey = walk.next();
      if (nkey >= 0) pages_of(nkey, pn);
      load(kbase, p.ks, key0, pg, kx);
      load(vbase, p.vs, key0, pg, vx);
    }
    while (key0 >= 0) {
      const int akey = nkey >= 0 ? walk.next() : -1;
      if (akey >= 0) pages_of(akey, pa);
      // Bits of the keys with a page and a position below the end.
      uint32_t have[KH];
      bool masked = key0 + KEYS - 1 > first_pos;
#pragma unroll
      for (int i = 0; i < KH; ++i) {
        have[i] = (uint32_t)(__ballot(is_page(p.batch, pg[2 * i])) & 0xffffu) |
                  (uint32_t)(__ballot(is_page(p.batch, pg[2 * i + 1])) << 16);
        const int left = tr.end - key0 - 32 * i;
        if (left < 32) have[i] &= left <= 0 ? 0u : (1u << left) - 1;
        masked |= have[i] != 0xffffffffu;
      }
      keep(kx);
      if (nkey >= 0) load(kbase, p.ks, nkey, pn, kx);
      f32x4v s[2][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        s[0][kt] = f32x4v{};
        s[1][kt] = f32x4v{};
        u32x4 a[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) a[kk] = load16(vl + (16 * kt + l16) * VSTR + 32 * kk + 8 * g4);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) s[0][kt] = mfma16x16x32<F16>(a[kk], qf[0][kk], s[0][kt]);
        if (two)
#pragma unroll
          for (int kk = 0; kk < KK; ++kk) s[1][kt] = mfma16x16x32<F16>(a[kk], qf[1][kk], s[1][kt]);
      }
      wave_lds_fence();
      u32x4 pk[2][KH];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c == 1 && !two) break;
        if (masked) {
          const int rel = qpos[c] - key0 - 4 * g4;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            const uint32_t mine = have[kt >> 1] >> (4 * g4);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!(mine & (1u << (16 * (kt & 1) + r))) || 16 * kt + r > rel) s[c][kt][r] = -INFINITY;
          }
        }
        float mx = s[c][0][0];
#pragma unroll
        for (int i = 1; i < 4 * KT; ++i) mx = fmaxf(mx, s[c][i >> 2][i & 3]);
        mx = quad_max(mx);
        if (__ballot(mx - m[c] > threshold)) {
          const float mn = fmaxf(m[c], mx);
          const float alpha = mn == -INFINITY ? 1.f : fast_exp2((m[c] - mn) * p.cs);
          m[c] = mn;
          l[c] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[c][dt] *= alpha;
        }
        float nm = m[c] == -INFINITY ? 0.f : fmaf(-m[c], p.cs, kLift<F16>);
        if constexpr (CAREFUL) {
          const float off = m[c] == -INFINITY ? 0.f : m[c];
#pragma unroll
          for (int i = 0; i < 4 * KT; ++i) s[c][i >> 2][i & 3] -= off;
          nm = kLift<F16>;
        }
#pragma unroll
        for (int h2 = 0; h2 < KH; ++h2) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = fast_exp2(fmaf(s[c][2 * h2 + (i >> 2)][i & 3], p.cs, nm));
            l[c] += x[i];
          }
          pk[c][h2] =
              u32x4{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]), pack2<F16>(x[6], x[7])};
        }
      }
      keep(vx);
      if (nkey >= 0) load(vbase, p.vs, nkey, pn, vx);
      const uint16_t* vt = vl + (4 * g4 + (l16 >> 2)) * VSTR + 4 * (l16 & 3);
      if (CAREFUL && masked) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c == 1 && !two) break;
          const int rel = qpos[c] < key0 ? -1 : qpos[c] - key0;  // last key that the row sees
#pragma unroll 1
          for (int q = 0; q < 16; ++q) {
            // Column q alone, with the value rows that it does not see as zeros.
            const int seen = __builtin_amdgcn_readlane(rel, q);
            const uint16_t* vq = vt + opaque_zero();  // reads it again for every column, not 64 registers ahead
#pragma unroll
            for (int h2 = 0; h2 < KH; ++h2) {
              const int s2 = seen - 32 * h2;
              const uint32_t mine = (s2 < 0 ? 0u : (s2 < 31 ? have[h2] & ((2u << s2) - 1) : have[h2])) >> (4 * g4);
              uint32_t w[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int b = 16 * (i >> 1) + 2 * (i & 1);
                w[i] = (mine & (1u << b) ? 0xffffu : 0u) | (mine & (2u << b) ? 0xffff0000u : 0u);
              }
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) {
                const uint2 a = lds_read_tr16(vq + 32 * h2 * VSTR + 16 * dt),
                            b = lds_read_tr16(vq + (32 * h2 + 16) * VSTR + 16 * dt);
                const f32x4v one =
                    mfma16x16x32<F16>(u32x4{a.x & w[0], a.y & w[1], b.x & w[2], b.y & w[3]}, pk[c][h2], f32x4v{});
                if (l16 == q) acc[c][dt] += one;
              }
            }
          }
        }
      } else {
        auto values = [&](int h2, int dt) {
          const uint2 a = lds_read_tr16(vt + 32 * h2 * VSTR + 16 * dt),
                      b = lds_read_tr16(vt + (32 * h2 + 16) * VSTR + 16 * dt);
          return u32x4{a.x, a.y, b.x, b.y};
        };
        if (two) {
#pragma unroll
          for (int h2 = 0; h2 < KH; ++h2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const u32x4 va = values(h2, dt);
              acc[0][dt] = mfma16x16x32<F16>(va, pk[0][h2], acc[0][dt]);
              acc[1][dt] = mfma16x16x32<F16>(va, pk[1][h2], acc[1][dt]);
            }
        } else {
#pragma unroll
          for (int h2 = 0; h2 < KH; ++h2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[0][dt] = mfma16x16x32<F16>(values(h2, dt), pk[0][h2], acc[0][dt]);
        }
      }
      wave_lds_fence();
      key0 = nkey;
      nkey = akey;
#pragma unroll
      for (int c = 0; c < KT; ++c) {
        pg[c] = pn[c];
        pn[c] = pa[c];
      }
    }
  }
  if constexpr (!CAREFUL) {
    bool odd = false;
#pragma unroll
    for (int c = 0; c < 2; ++c) odd |= m[c] != -INFINITY && !(fabsf(m[c] * p.cs) < kLargeScore);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= !(fabsf(acc[c][dt][r]) < INFINITY);
    odds[wave] = __ballot(odd) != 0;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    l[c] = quad_sum(l[c]);
    if (g4 == 0) {
      ml[wave * 64 + 16 * c + l16] = m[c] * p.cs;
      ml[wave * 64 + 32 + 16 * c + l16] = l[c];
    }
  }
  const PagedAttn pe = arguments(args);
  note_begun(pe, part, tr.row0, tr.rows, token0);
  // The waves' sums joined through LDS, 16 rows at a time, each wave's where
  // its V rows were: thread t takes D / 32 values of row t / 32.
  constexpr int OWAVE = kFewKeys * VSTR / 2;  // floats from wave to wave
  float* ol = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (c == 1 && !two) break;
    if (c == 1) __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4v*>(ol + wave * OWAVE + l16 * OSTR + 16 * dt + 4 * g4) = acc[c][dt];
    __syncthreads();
    if (!CAREFUL && c == 0) {
      int any = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) any |= odds[w];
      if (uniform(any)) return true;
    }
    constexpr int PER = D / 32;
    const int r = threadIdx.x >> 5, d0 = (threadIdx.x & 31) * PER, row = 16 * c + r;
    if (row >= tr.rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w * 64 + row]);
    const float nm = top == -INFINITY ? 0.f : -top;
    float sum = 0.f, o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(ml[w * 64 + row] + nm);
      sum += f * ml[w * 64 + 32 + row];
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += f * ol[w * OWAVE + r * OSTR + d0 + i];
    }
    if (part.slot >= 0) {
      const int64_t group = part.slot;
      float* po = pe.part_o + group * 32 * D + part_at(row, d0);
#pragma unroll
      for (int i = 0; i < PER; ++i) po[i] = o[i];
      if (d0 == 0) {
        pe.part_ml[group * 64 + row] = top;
        pe.part_ml[group * 64 + 32 + row] = sum;
      }
      continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int t = pe.by_group.of(tr.row0 + row), h = tr.row0 + row - t * pe.G;
    uint16_t* dst = static_cast<uint16_t*>(pe.out) + (int64_t)(token0 + t) * pe.os[0] +
                    (int64_t)(u.g * pe.G + h) * pe.os[1] + d0;
#pragma unroll
    for (int i = 0; i < PER; i += 2)
      reinterpret_cast<uint32_t*>(dst)[i / 2] = pack2<F16>(o[i] * inv, o[i + 1] * inv);
  }
  return false;
}

// A many-row unit.  The matrix cores bound it, with the softmax's VALU work
// and the LDS reads beside them (each about 2050 cycles a block and SIMD at full
// rate; the matrix cores are busy 50% of the time), so it is laid out like the block-sparse
// prefill: S^T = K Q^T and O^T = V^T P^T on 32 x 32 x 16 with one query row a
// lane column, 64-key blocks double-buffered in LDS by way of registers, the
// next block's loads in flight under the present one's products.  The pages of
// the block after that are looked up meanwhile, one key a lane.  ALIGNED: a
// page holds whole blocks, so a block is one piece of memory behind one buffer
// descriptor; otherwise every row finds its own page.
template <int D, bool F16, bool ALIGNED, bool CAREFUL>
__device__ __forceinline__ bool many_rows(uintptr_t args, const Unit& u, const Part& part, char* smem) {
  const PagedAttn p = arguments(args);
  constexpr int NTHR = kWaves * 64;
  constexpr int KSTR = D + 8, VSTR = D + 32;  // LDS rows; V rows start 16 banks apart
  constexpr int KTILE = kBlock * KSTR, BUF = KTILE + kBlock * VSTR;
  constexpr int ROWCH = D / 8, KCH = kBlock * ROWCH / NTHR;  // 16-byte pieces of a row, and of a thread
  constexpr int DT = D / 32, KS = D / 16;
  uint16_t* lds = reinterpret_cast<uint16_t*>(smem);
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;

  const TileRows tr = tile_rows(p, u);
  if (tr.rows == 0) return false;  // uniform: before any barrier
  const int token0 = u.w.start;
  const int left = tr.rows - 32 * wave;
  const int nrow = left < 0 ? 0 : (left < 32 ? left : 32);  // this wave's rows
  // Columns past the last row repeat it; a wave without rows has the unit's first.
  const int row = tr.row0 + (nrow == 0 ? 0 : 32 * wave + (l32 < nrow ? l32 : nrow - 1));
  const int tok = p.by_group.of(row), head = u.g * p.G + row - tok * p.G;
  const int qpos = clip(u.w.pos0 + tok);
  // Positions of the wave's first and last row.
  const int pos_lo = uniform(clip(u.w.pos0 + p.by_group.of(tr.row0 + 32 * wave)));
  const int pos_hi = uniform(clip(u.w.pos0 + p.by_group.of(tr.row0 + 32 * wave + (nrow > 0 ? nrow - 1 : 0))));

  uint4 qf[KS];
  {
    const uint16_t* src =
        static_cast<const uint16_t*>(p.q) + (int64_t)(token0 + tok) * p.qs[0] + (int64_t)head * p.qs[1] + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk)
      qf[kk] = *reinterpret_cast<const uint4*>(src + 16 * kk);
  }
  const int items = p.idx ? p.K : (tr.end + kBlock - 1) / kBlock;
  const int hi = part.hi < items ? part.hi : items;

  const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + (int64_t)u.g * p.ks[1];
  const uint16_t* vbase = static_cast<const uint16_t*>(p.v) + (int64_t)u.g * p.vs[1];
  const int srow = tid / ROWCH, scol = (tid % ROWCH) * 8;  // this thread's pieces: rows srow + i NTHR / ROWCH
  constexpr int SSTEP = NTHR / ROWCH;
  int koff[KCH], voff[KCH];
#pragma unroll
  for (int i = 0; i < KCH; ++i) {
    koff[i] = ((srow + i * SSTEP) * (int)p.ks[2] + scol) * 2;
    voff[i] = ((srow + i * SSTEP) * (int)p.vs[2] + scol) * 2;
  }
  u32x4 kst[KCH], vst[KCH];
  // The table's entry of key0 + lane.
  auto page_at = [&](int key0) -> int {
    return page_entry(p.batch, u.s, ALIGNED ? key0 : nearest(key0 + lane, tr.end));
  };
  auto load_block = [&](int key0, int pg) {
    if constexpr (ALIGNED) {
      const int page = uniform(is_page(p.batch, pg) ? pg : 0);
      const int slot = key0 - page_of(p.batch, key0) * p.batch.page;
      int nk = tr.end - key0;
      nk = nk > kBlock ? kBlock : nk;
      const __amdgpu_buffer_rsrc_t rk =
          make_rsrc(kbase + (int64_t)page * p.ks[0] + (int64_t)slot * p.ks[2], (uint32_t)(nk * (int)p.ks[2] * 2));
      const __amdgpu_buffer_rsrc_t rv =
          make_rsrc(vbase + (int64_t)page * p.vs[0] + (int64_t)slot * p.vs[2], (uint32_t)(nk * (int)p.vs[2] * 2));
#pragma unroll
      for (int i = 0; i < KCH; ++i)
        kst[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rk, koff[i], 0, 0));
#pragma unroll
      for (int i = 0; i < KCH; ++i)
        vst[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rv, voff[i], 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < KCH; ++i) {
        const int r = srow + i * SSTEP, page = __shfl(is_page(p.batch, pg) ? pg : 0, r);
        const int key = nearest(key0 + r, tr.end), slot = key - page_of(p.batch, key) * p.batch.page;
        kst[i] = load16(kbase + (int64_t)page * p.ks[0] + (int64_t)slot * p.ks[2] + scol);
        vst[i] = load16(vbase + (int64_t)page * p.vs[0] + (int64_t)slot * p.vs[2] + scol);
      }
    }
  };
  auto store_block = [&](int buf) {
    uint16_t* ks = lds + buf * BUF;
#pragma unroll
    for (int i = 0; i < KCH; ++i) {
      *reinterpret_cast<u32x4*>(ks + (srow + i * SSTEP) * KSTR + scol) = kst[i];
      *reinterpret_cast<u32x4*>(ks + KTILE + (srow + i * SSTEP) * VSTR + scol) = vst[i];
    }
  };

  float m = -INFINITY, l = 0.f;  // m: of the scores as products, before cs
  const float threshold = fminf(kRescaleThreshold / p.cs, 0x1.fffffep+127f);  // -inf's distance is past it
  f32x16_t acc[DT];
  uint4 pk[2][2];
  auto scores = [&](const uint16_t* ks, f32x16_t& s0, f32x16_t& s1) {
    const uint16_t* kp = ks + l32 * KSTR + 8 * hl;
    uint4 a0[KS], a1[KS];
    auto rd = [&](int kk) {
      a0[kk] = *reinterpret_cast<const uint4*>(kp + 16 * kk);
      a1[kk] = *reinterpret_cast<const uint4*>(kp + 32 * KSTR + 16 * kk);
    };
#pragma unroll
    for (int kk = 0; kk < kLookahead; ++kk) rd(kk);
    s0 = f32x16_t{};
    s1 = f32x16_t{};
    // The reads of step kk + kLookahead are issued before the products of
    // step kk; without the barriers one register quad serves all reads.
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      if (kk + kLookahead < KS) rd(kk + kLookahead);
      __builtin_amdgcn_sched_barrier(0);
      s0 = mfma32x32x16<F16>(a0[kk], qf[kk], s0);
      s1 = mfma32x32x16<F16>(a1[kk], qf[kk], s1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Register r of key half c holds key 32 c + 8 (r / 4) + 4 (lane / 32) + r % 4.
  auto softmax = [&](f32x16_t& s0, f32x16_t& s1, bool masked, int rel, uint64_t there) {
    if (masked) {
      const uint32_t lo_bits = (uint32_t)there >> (4 * hl), hi_bits = (uint32_t)(there >> 32) >> (4 * hl);
      const int thr = rel - 4 * hl;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int kr = 8 * (r >> 2) + (r & 3);
        if (kr > thr || !(lo_bits & (1u << kr))) s0[r] = -INFINITY;
        if (32 + kr > thr || !(hi_bits & (1u << kr))) s1[r] = -INFINITY;
      }
    }
    float mx = fmaxf(s0[0], s0[1]);
#pragma unroll
    for (int r = 2; r < 16; ++r) mx = fmaxf(mx, s0[r]);
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s1[r]);
    mx = half_max(mx);
    if (__ballot(mx - m > threshold) != 0) {
      const float mn = fmaxf(m, mx);
      const float alpha = mn == -INFINITY ? 1.f : fast_exp2((m - mn) * p.cs);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[dt][r] *= alpha;
    }
    float nm = m == -INFINITY ? 0.f : fmaf(-m, p.cs, kLift<F16>);
    if constexpr (CAREFUL) {
      const float off = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s0[r] -= off;
        s1[r] -= off;
      }
      nm = kLift<F16>;
    }
    float sum = 0.f;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      uint32_t w0[4], w1[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x0 = fast_exp2(fmaf(s0[8 * h2 + 2 * e], p.cs, nm));
        const float x1 = fast_exp2(fmaf(s0[8 * h2 + 2 * e + 1], p.cs, nm));
        const float y0 = fast_exp2(fmaf(s1[8 * h2 + 2 * e], p.cs, nm));
        const float y1 = fast_exp2(fmaf(s1[8 * h2 + 2 * e + 1], p.cs, nm));
        sum += (x0 + x1) + (y0 + y1);
        w0[e] = pack2<F16>(x0, x1);
        w1[e] = pack2<F16>(y0, y1);
      }
      pk[0][h2] = uint4{w0[0], w0[1], w0[2], w0[3]};
      pk[1][h2] = uint4{w1[0], w1[1], w1[2], w1[3]};
    }
    l += sum;
  };
  // P^T fragment pk[c][h2] holds keys K0 + 4 hl + 0..3 and K0 + 8 + 4 hl + 0..3,
  // K0 = 32 c + 16 h2; the V^T fragment of d = 32 dt + l32 is two transposing reads of 4 keys each.
  const int vlane = (4 * hl + ((lane & 15) >> 2)) * VSTR + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  auto value = [&](const uint16_t* vp, int dt, int ch) {
    const uint16_t* a = vp + 16 * ch * VSTR + 32 * dt;
    const uint2 x = lds_read_tr16(a), y = lds_read_tr16(a + 8 * VSTR);
    return uint4{x.x, x.y, y.x, y.y};
  };
  auto pv = [&](const uint16_t* vs) {
    const uint16_t* vp = vs + vlane;
    uint4 va[DT * 4];
#pragma unroll
    for (int i = 0; i < DT * 4; ++i) va[i] = value(vp, i % DT, i / DT);
    __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 4 * kLookahead, 0);
#pragma unroll
    for (int i = 0; i < DT * 4 - 2 * kLookahead; ++i) {
      __builtin_amdgcn_sched_group_barrier(kSchedMfma, 1, 0);
      __builtin_amdgcn_sched_group_barrier(kSchedDsRead, 2, 0);
    }
    __builtin_amdgcn_sched_group_barrier(kSchedMfma, 2 * kLookahead, 0);
#pragma unroll
    for (int i = 0; i < DT * 4; ++i)
      acc[i % DT] = mfma32x32x16<F16>(va[i], pk[(i / DT) >> 1][(i / DT) & 1], acc[i % DT]);
  };
  // The same for one column at a time, with the value rows that it does not
  // see as zeros: 0 times a NaN or infinity there would be NaN.
  auto pv_careful = [&](const uint16_t* vs, int rel, uint64_t there) {
    const uint16_t* vp = vs + vlane;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
      for (int q = 0; q < 32; ++q) {
        const int seen = __builtin_amdgcn_readlane(rel, q);
        // (-1: a row before the block sees nothing of it.)
        const uint64_t mine = seen < 0 ? 0ull : (seen < 63 ? there & ((2ull << seen) - 1) : there);
        const uint16_t* vq = vp + opaque_zero();  // as above
        f32x16_t one = f32x16_t{};
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          const uint4 a = value(vq, dt, ch);
          const uint32_t bits = (uint32_t)(mine >> (16 * ch + 4 * hl));
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int b = 8 * (i >> 1) + 2 * (i & 1);
            w[i] = (bits & (1u << b) ? 0xffffu : 0u) | (bits & (2u << b) ? 0xffff0000u : 0u);
          }
          one = mfma32x32x16<F16>(uint4{a.x & w[0], a.y & w[1], a.z & w[2], a.w & w[3]}, pk[ch >> 1][ch & 1], one);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (l32 == q) {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[dt][r] += one[r];
        }
      }
    }
  };

  {
    m = -INFINITY;
    l = 0.f;
    const float zero = __builtin_bit_cast(float, opaque_zero());
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[dt][r] = zero;
    KeyWalk<kBlock> walk;
    walk.init(p, tr, part.lo, 1, hi, lane);
    auto take = [&](int& key0, int& pg) {
      key0 = walk.next();
      pg = key0 < 0 ? 0 : page_at(key0);
    };
    int key0, pg, nkey, npg;
    take(key0, pg);
    int buf = 0;
    if (key0 >= 0) {
      load_block(key0, pg);
      take(nkey, npg);
      store_block(0);
      __syncthreads();
      while (true) {
        if (nkey >= 0) load_block(nkey, npg);
        int akey = -1, apg = -1;
        if (nkey >= 0) take(akey, apg);
        if (nrow > 0 && key0 <= pos_hi) {
          const uint16_t* ks = lds + buf * BUF;
          // Bits of the keys with a page and a position below the end.
          uint64_t there = __ballot(is_page(p.batch, pg));
          if (tr.end - key0 < kBlock) there &= (1ull << (tr.end - key0)) - 1;
          const bool masked = there != ~0ull || key0 + kBlock - 1 > pos_lo;
          const int rel = qpos < key0 ? -1 : qpos - key0;
          f32x16_t s0, s1;
          scores(ks, s0, s1);
          // The wave that is at its softmax goes first: the other one of its SIMD
          // has the matrix cores busy 32 cycles with each instruction that it
          // gets in (chunk of 4096 rows over 32768 keys: 1903 us, 1941 without).
          __builtin_amdgcn_s_setprio(1);
          softmax(s0, s1, masked, rel, there);
          __builtin_amdgcn_s_setprio(0);
          if (CAREFUL && masked)
            pv_careful(ks + KTILE, rel, there);
          else
            pv(ks + KTILE);
        }
        if (nkey < 0) break;
        store_block(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        key0 = nkey;
        pg = npg;
        nkey = akey;
        npg = apg;
      }
    }
  }
  if constexpr (!CAREFUL) {
    bool odd = m != -INFINITY && !(fabsf(m * p.cs) < kLargeScore);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) odd |= !(fabsf(acc[dt][r]) < INFINITY);
    if (uniform(__syncthreads_or(odd))) return true;  // as in few_rows
  } else {
    __syncthreads();
  }

  l = half_sum(l);
  const PagedAttn pe = arguments(args);
  note_begun(pe, part, tr.row0, tr.rows, token0);
  if (part.slot >= 0) {
    const int64_t group = (int64_t)part.slot * kWaves + wave;
    if (nrow == 0) return false;
    float* po = pe.part_o + group * 32 * D + lane * 4;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(po + (dt * 4 + j) * 256) =
            float4{acc[dt][4 * j], acc[dt][4 * j + 1], acc[dt][4 * j + 2], acc[dt][4 * j + 3]};
    if (hl == 0) {
      pe.part_ml[group * 64 + l32] = m * pe.cs;
      pe.part_ml[group * 64 + 32 + l32] = l;
    }
    return false;
  }
  // Through LDS, so that every store writes 16-byte pieces of whole rows; all
  // readers of the tiles have passed the barrier above.
  constexpr int OSTR = D + 8;
  static_assert(kWaves * 32 * OSTR <= 2 * BUF, "output staging must fit the K/V tiles");
  if (nrow == 0) return false;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* ot = lds + wave * 32 * OSTR;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint2*>(ot + l32 * OSTR + dt * 32 + 8 * j + 4 * hl) =
          uint2{pack2<F16>(acc[dt][4 * j] * inv, acc[dt][4 * j + 1] * inv),
                pack2<F16>(acc[dt][4 * j + 2] * inv, acc[dt][4 * j + 3] * inv)};
  wave_lds_fence();
  const int64_t at = (int64_t)(token0 + tok) * pe.os[0] + (int64_t)head * pe.os[1];  // of row l32
#pragma unroll
  for (int i = 0; i < 32 * ROWCH / 64; ++i) {
    const int c = i * 64 + lane, r = c / ROWCH, ch = c % ROWCH;
    const int lo32 = __shfl((int)at, r), hi32 = __shfl((int)(at >> 32), r);
    if (r < nrow)
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(pe.out) +
                                (int64_t)(((uint64_t)(uint32_t)hi32 << 32) | (uint32_t)lo32) + ch * 8) =
          *reinterpret_cast<const uint4*>(ot + r * OSTR + ch * 8);
  }
  return false;
}

// What the two kinds have for a unit: its shape, the keys of a step, its LDS,
// and the body.
template <int D, bool F16>
struct FewBody {
  typedef Few Shape;
  static constexpr int keys = kFewKeys, lds = few_lds_bytes<D>();
  template <bool CAREFUL>
  static __device__ __forceinline__ bool run(uintptr_t args, const Unit& u, const Part& part, char* smem) {
    return few_rows<D, F16, CAREFUL>(args, u, part, smem);
  }
};
template <int D, bool F16, bool ALIGNED>
struct ManyBody {
  typedef Many Shape;
  static constexpr int keys = kBlock, lds = many_lds_bytes<D>();
  template <bool CAREFUL>
  static __device__ __forceinline__ bool run(uintptr_t args, const Unit& u, const Part& part, char* smem) {
    return many_rows<D, F16, ALIGNED, CAREFUL>(args, u, part, smem);
  }
};

// The stretch [at, end) of head g's line, the turn-th, as far as its first unit.
struct Stretch {
  int64_t at, end, turn;
  int g;
};

// Every wave keeps the lengths of the first 64 sequences behind the body's LDS.
template <typename BODY>
constexpr int lds_bytes() {
  return BODY::lds + kWaves * 64 * (int)sizeof(Lengths);
}
template <typename BODY>
__device__ __forceinline__ Lengths& kept_lengths(char* smem) {
  return reinterpret_cast<Lengths*>(smem + BODY::lds)[threadIdx.x];
}

// The turn of a workgroup among those of its head, and the head.
__device__ __forceinline__ int turn_of(const PagedAttn& p, int& g) {
  const int turn = uniform(p.by_heads.of((int)blockIdx.x));
  g = (int)blockIdx.x - turn * p.Hkv;
  return turn;
}

template <typename BODY, bool CAREFUL>
__device__ __forceinline__ bool run_unit(uintptr_t args, const Line& line, const Stretch& st, char* smem, int64_t& to) {
  Unit u;
  int G;
  {
    const PagedAttn p = arguments(args);
    const SeqWork w0 = sequence_work<typename BODY::Shape>(p, kept_lengths<BODY>(smem));
    if (!find_unit<typename BODY::Shape>(p, w0, st.at, st.g, threadIdx.x & 63, u)) return false;
    G = p.G;
  }
  to = u.end < st.end ? u.end : st.end;
  const Part part = part_of<typename BODY::Shape, BODY::keys>(line, u, G, st.at, to, st.turn);
  return BODY::template run<CAREFUL>(args, u, part, smem);
}

template <typename BODY, bool CAREFUL>
__device__ __forceinline__ bool run_tile(uintptr_t args, char* smem) {
  Unit u;
  {
    const PagedAttn p = arguments(args);
    int g;
    const int turn = turn_of(p, g);
    if (!find_tile<typename BODY::Shape>(p, turn, g, threadIdx.x & 63, u)) return false;
  }
  return BODY::template run<CAREFUL>(args, u, kWhole, smem);
}

// The careful way, looking its unit up again, is a function of its own: what
// it would keep in registers pushed the usual way's out of them.
template <typename BODY>
__device__ __attribute__((noinline)) void run_again(uint64_t args, int64_t share, int64_t at, int64_t end, int64_t turn,
                                                    int g, __attribute__((address_space(3))) char* smem) {
  auto same = [](int64_t x) { return lane_of(x, 0); };
  int64_t to;
  run_unit<BODY, true>((uintptr_t)same((int64_t)args), Line{0, same(share)},
                       Stretch{same(at), same(end), same(turn), uniform(g)}, (char*)smem, to);
}
template <typename BODY>
__device__ __attribute__((noinline)) void run_tile_again(uint64_t args, __attribute__((address_space(3))) char* smem) {
  run_tile<BODY, true>((uintptr_t)lane_of((int64_t)args, 0), (char*)smem);
}

// A launch for either kind: the lengths that tell them apart are on the
// device, so the workgroups of a kind that the batch does not hold find no
// tile and end.  (Both in one kernel needed more registers than there are.)
// One kernel for shares of the line, one for a whole tile a workgroup, which
// has none of the line's arithmetic before its first load.
template <typename BODY>
__global__ __launch_bounds__(kWaves * 64, 2) void paged_attention_kernel(const PagedAttn) {
  typedef typename BODY::Shape SHAPE;
  __shared__ __attribute__((aligned(16))) char smem[lds_bytes<BODY>()];
  const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  Line line;
  Stretch st;
  {
    const PagedAttn p = arguments(args);
    const int lane = threadIdx.x & 63;
    const Lengths len = lengths_of(p, lane);
    kept_lengths<BODY>(smem) = len;
    line = line_of<SHAPE>(p, sequence_work<SHAPE>(p, len), lane);
    st.turn = turn_of(p, st.g);
    if (threadIdx.x == 0) p.begun[blockIdx.x] = int4{0, 0, 0, 0};  // none yet
  }
  st.at = st.turn * line.share;
  st.end = st.at + line.share < line.total ? st.at + line.share : line.total;
  while (st.at < st.end) {
    int64_t to = st.end;
    if (run_unit<BODY, false>(args, line, st, smem, to))
      run_again<BODY>(args, line.share, st.at, st.end, st.turn, st.g, (__attribute__((address_space(3))) char*)smem);
    if (to <= st.at) break;  // lines past 64 bits, of starts that overlap, lead back
    st.at = to;
    if (st.at < st.end) __syncthreads();  // the unit's LDS is free
  }
}

template <typename BODY>
__global__ __launch_bounds__(kWaves * 64, 2) void paged_tile_kernel(const PagedAttn) {
  __shared__ __attribute__((aligned(16))) char smem[BODY::lds];
  const uintptr_t args = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  if (run_tile<BODY, false>(args, smem)) run_tile_again<BODY>(args, (__attribute__((address_space(3))) char*)smem);
}

// Joins the parts of one 32-row group of the tile that a workgroup began and
// others ended: every thread takes 4 values of its row from every eighth of d.
template <typename SHAPE, int D, bool F16>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttn p) {
  constexpr int kTileGroups = SHAPE::rows / 32;
  const int sub = blockIdx.x % kTileGroups, from = blockIdx.x / kTileGroups;
  const int4 tile = p.begun[from];
  const int lane = threadIdx.x & 63, row = lane & 31, hl = lane >> 5, wave = threadIdx.x >> 6;
  const int r = sub * 32 + row;
  const int t0 = p.by_heads.of(from), t1 = tile.w, g = from - t0 * p.Hkv;
  if (r >= (tile.y & 0xffff) || t1 >= p.groups) return;  // (none, or starts that overlap)
  // The part of a turn: the one that starts its stretch, or the one behind.
  auto part = [&](int t) {
    return (2 * ((int64_t)t * p.Hkv + g) + (t == t0 ? tile.y >> 16 : 0)) * kTileGroups + sub;
  };
  constexpr int PIECES = D / 32;  // of 4 values: pieces wave, wave + 4 ..
  float top = -INFINITY, sum = 0.f;
  f32x4v o[PIECES] = {};
  // Two parts at a time, all their loads in flight (a second one behind the
  // last is the last again and weighs nothing).
  for (int t = t0; t <= t1; t += 2) {
    float m[2], l[2];
    f32x4v x[2][PIECES];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = part(t + i < t1 ? t + i : t1);
      m[i] = p.part_ml[at * 64 + row];
      l[i] = p.part_ml[at * 64 + 32 + row];
#pragma unroll
      for (int j = 0; j < PIECES; ++j)
        x[i][j] = *reinterpret_cast<const f32x4v*>(p.part_o + at * 32 * D + (wave + 4 * j) * 256 + lane * 4);
    }
    if (t + 1 > t1) {
      m[1] = -INFINITY;
      l[1] = 0.f;
    }
    const float now = fmaxf(top, fmaxf(m[0], m[1]));
    const float nm = now == -INFINITY ? 0.f : -now;
    const float f = fast_exp2(top + nm), f0 = fast_exp2(m[0] + nm), f1 = fast_exp2(m[1] + nm);
    sum = f * sum + f0 * l[0] + f1 * l[1];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      o[j] = f * o[j] + f0 * x[0][j];
      if (t + 1 <= t1) o[j] += f1 * x[1][j];
    }
    top = now;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int at = tile.x + r, t = p.by_group.of(at), h = at - t * p.G;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)(tile.z + t) * p.os[0] +
                  (int64_t)(g * p.G + h) * p.os[1] + 4 * hl;
#pragma unroll
  for (int j = 0; j < PIECES; ++j)
    *reinterpret_cast<uint2*>(dst + 8 * (wave + 4 * j)) =
        uint2{pack2<F16>(o[j][0] * inv, o[j][1] * inv), pack2<F16>(o[j][2] * inv, o[j][3] * inv)};
}

// The launches of one kind: `tiles` workgroups that take a row tile whole each
// (shares 0), or `shares` that share the line out, and the join.
struct PagedLaunch {
  int64_t tiles, shares;
};

template <typename BODY, int D, bool F16>
int launch_paged(const PagedAttn& p, const PagedLaunch& n, hipStream_t st) {
  typedef typename BODY::Shape Shape;
  if (n.shares == 0) {
    hipLaunchKernelGGL((paged_tile_kernel<BODY>), dim3((unsigned)n.tiles), dim3(kWaves * 64), 0, st, p);
    return check_launch("paged attention");
  }
  hipLaunchKernelGGL((paged_attention_kernel<BODY>), dim3((unsigned)n.shares), dim3(kWaves * 64), 0, st, p);
  const int rc = check_launch("paged attention");
  if (rc) return rc;
  hipLaunchKernelGGL((paged_join_kernel<Shape, D, F16>), dim3((unsigned)(n.shares * (Shape::rows / 32))), dim3(256), 0,
                     st, p);
  return check_launch("paged attention join");
}

// D 64 or 128; one source file each, they take a while to compile.
int launch_paged_few(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st);
int launch_paged_many(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st);
int launch_paged_scattered(const PagedAttn& p, int D, bool f16, const PagedLaunch& n, hipStream_t st);

}  // namespace spruce
