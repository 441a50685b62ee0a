// Attention of a ragged batch's new tokens over a paged K/V cache:
//   o_n = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q_n.k_j - m),
// j over the cached positions up to the token's own, all of them or those of
// the 64-key blocks listed for the token's 64-position block.
//
// Rows of one (sequence, KV head) are packed token by token, head by head
// (row r: token r / G, query head g G + r % G), so few tokens of a wide group
// fill a matrix tile as many tokens of a narrow one do.
#include "attention_impl.h"
#include "paged.h"

using namespace spruce;

namespace {

struct PagedAttn {
  const void* q;
  void* out;
  int64_t qs[2], os[2];  // token, head strides
  const void* k;
  const void* v;
  int64_t ks[3], vs[3];  // page, head, slot strides
  PagedBatch batch;
  int Hkv, G;
  float cs;  // scale * log2 e
  const int32_t* idx;  // block lists [S, Hkv, Qc, K], or null
  int64_t is[3];
  int Qc, K;
  float* part_o;   // [units][kRows][D]
  float* part_ml;  // [units][2][kRows]
  int grid;        // units that have a workgroup and a partial slot
};

constexpr int kRows = 32;      // rows of a unit
constexpr int kKeys = 32;      // keys a wave takes at a time
constexpr int kWaves = 4;      // waves of a workgroup, each with keys of its own
constexpr int kStep = kKeys * kWaves;
constexpr int kSlots = 512;    // units that the splits aim at: two workgroups a CU
constexpr int kMinSteps = 2;   // steps below which a row's keys are not split further

typedef float f32x4v __attribute__((ext_vector_type(4)));

template <bool F16>
__device__ __forceinline__ f32x4v mfma16x16x32(uint4 a, uint4 b, f32x4v c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0,
                                                  0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c,
                                                   0, 0, 0);
}

// The same value in every lane, for the compiler too: it must branch on the
// scalar unit around matrix instructions, which run whatever EXEC holds.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)x));
}

// Sum of v over the lanes up to this one (row shifts within 16 lanes, then
// the rows' last lanes broadcast onward).
__device__ __forceinline__ int wave_prefix(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// The work of one sequence: row tiles per KV head, and 128-key steps of each.
struct SeqWork {
  int n;        // new tokens
  int64_t pos0;  // position of the first
  int tiles, steps, sub;
};

__device__ __forceinline__ SeqWork sequence_work(const PagedAttn& p, int s) {
  SeqWork w{};
  if (s >= p.batch.S) return w;
  const int a = start_at(p.batch, s), e = start_at(p.batch, s + 1);
  w.n = e > a ? e - a : 0;
  // Positions go by the lengths as given; only what they address is bounded.
  w.pos0 = (int64_t)p.batch.kv_lens[s] - ((int64_t)p.batch.q_starts[s + 1] - p.batch.q_starts[s]) +
           (a - p.batch.q_starts[s]);
  if (w.n == 0) return w;
  if (p.idx != nullptr) {
    const int64_t b0 = w.pos0 >> 6, b1 = (w.pos0 + w.n - 1) >> 6;
    const int tok = w.n < kBlock ? w.n : kBlock;
    w.sub = (tok * p.G + kRows - 1) / kRows;
    w.tiles = (int)(b1 - b0 + 1) * w.sub;
    w.steps = (int)(((int64_t)p.K * kBlock + kStep - 1) / kStep);
  } else {
    w.sub = 1;
    w.tiles = (int)(((int64_t)w.n * p.G + kRows - 1) / kRows);
    w.steps = (keys_of(p.batch, s) + kStep - 1) / kStep;
  }
  if (w.steps < 1) w.steps = 1;
  return w;
}

// Keys are split so that about kSlots units of equal size come out: a unit
// takes `per` steps of its row tile at most.  Every workgroup works this out
// from the lengths, 64 sequences at a time.
__device__ __forceinline__ int steps_per_unit(const PagedAttn& p, int lane) {
  int64_t all = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const SeqWork w = sequence_work(p, s0 + lane);
    all += (int64_t)w.tiles * w.steps;
  }
#pragma unroll
  for (int m = 1; m < 64; m *= 2) all += __shfl_xor(all, m);
  const int64_t per = (all * p.Hkv + kSlots - 1) / kSlots;
  return per < kMinSteps ? kMinSteps : uniform((int)(per < (1 << 30) ? per : (1 << 30)));
}

struct Unit {
  int s, tile, g, split, splits, first;  // first: unit of split 0 of this tile and head
  SeqWork w;
};

// The unit `want` counted over units (BY_TILE false), or the (tile, head)
// `want` counted without the splits.  false behind the last.
template <bool BY_TILE>
__device__ __forceinline__ bool find_unit(const PagedAttn& p, int want, int per, int lane, Unit& u) {
  int units = 0, tiles = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const SeqWork w = sequence_work(p, s0 + lane);
    const int splits = (w.steps + per - 1) / per;
    const int mt = w.tiles * p.Hkv, mu = mt * splits;
    const int pt = wave_prefix(mt), pu = wave_prefix(mu);
    const int mine = (BY_TILE ? tiles + pt : units + pu);
    const uint64_t past = __ballot(mine > want);
    if (past) {
      const int l = __builtin_ctzll(past);
      const int th = __builtin_amdgcn_readlane(mt, l);
      u.s = s0 + l;
      u.splits = __builtin_amdgcn_readlane(splits, l);
      u.w.n = __builtin_amdgcn_readlane(w.n, l);
      u.w.pos0 = (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w.pos0 >> 32), l) << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((int)w.pos0, l));
      u.w.tiles = __builtin_amdgcn_readlane(w.tiles, l);
      u.w.steps = __builtin_amdgcn_readlane(w.steps, l);
      u.w.sub = __builtin_amdgcn_readlane(w.sub, l);
      const int before = units + __builtin_amdgcn_readlane(pu, l) - th * u.splits;
      const int in = want - (BY_TILE ? tiles + __builtin_amdgcn_readlane(pt, l) - th : before);
      if (in < 0 || in >= th * (BY_TILE ? 1 : u.splits)) return false;  // starts that overlap
      // Within a sequence: split slowest, then tile, head fastest.
      u.split = BY_TILE ? 0 : in / th;
      const int r = in - u.split * th;
      u.tile = r / p.Hkv;
      u.g = r - u.tile * p.Hkv;
      u.first = before + r;
      return true;
    }
    tiles += __builtin_amdgcn_readlane(pt, 63);
    units += __builtin_amdgcn_readlane(pu, 63);
  }
  return false;
}

// Rows [row0, row0 + rows) of the tile in the sequence's packed rows, and the
// block list that they share.
struct TileRows {
  int row0, rows;
  const int32_t* list;
};

__device__ __forceinline__ TileRows tile_rows(const PagedAttn& p, const Unit& u) {
  TileRows t{};
  if (p.idx == nullptr) {
    t.row0 = u.tile * kRows;
    const int left = u.w.n * p.G - t.row0;
    t.rows = left < kRows ? left : kRows;
    return t;
  }
  const int bi = u.tile / u.w.sub, sub = u.tile - bi * u.w.sub;
  const int64_t lo = (((u.w.pos0 >> 6) + bi) << 6) - u.w.pos0;
  const int t0 = lo < 0 ? 0 : (int)lo;
  const int t1 = lo + kBlock < u.w.n ? (int)(lo + kBlock) : u.w.n;
  t.row0 = t0 * p.G + sub * kRows;
  const int left = t1 * p.G - t.row0;
  t.rows = left < 0 ? 0 : (left < kRows ? left : kRows);
  t.list = bi < p.Qc ? p.idx + (int64_t)u.s * p.is[0] + (int64_t)u.g * p.is[1] + (int64_t)bi * p.is[2] : nullptr;
  return t;
}

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

// One unit: up to 32 packed rows against a range of 32-key tiles, the four
// waves taking every fourth tile each without a barrier between them.
// Memory bounds it: a key's 256 + 256 bytes meet at most 32 rows.  A wave's
// K rows go from memory straight into the A operand of S^T = K Q^T (lane: key
// l % 16, 16 bytes of d at 8 (l / 16) + 32 kk, so a load takes 64 bytes of each of 16
// rows); V rows, loaded alike, pass through the wave's own LDS, whose
// transposing read gives the A operand of O^T = V^T P^T; P^T, the B operand,
// is S^T's accumulator as it lies (keys 4 (l / 16) + r).  The next tile's K
// is in flight from the last S^T on, its V from the LDS write on.
template <int D, bool F16>
__global__ __launch_bounds__(kWaves * 64, 2) void paged_rows_kernel(const PagedAttn p) {
  constexpr int KK = D / 32;   // steps of S^T over d
  constexpr int DT = D / 16;   // 16-row tiles of O^T
  constexpr int VSTR = D + 8;  // V rows in LDS, 16-bit elements
  constexpr int OSTR = D + 4;  // O rows in LDS, floats
  constexpr int kVBytes = kWaves * kKeys * VSTR * 2, kOBytes = kWaves * 16 * OSTR * 4;
  __shared__ __attribute__((aligned(16))) char smem[kVBytes > kOBytes ? kVBytes : kOBytes];
  __shared__ float ml[kWaves][2][kRows];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;

  Unit u;
  const int per = steps_per_unit(p, lane);
  if (!find_unit<false>(p, blockIdx.x, per, lane, u)) return;  // uniform: before any barrier
  const TileRows tr = tile_rows(p, u);
  if (tr.rows == 0) return;
  const int token0 = uniform(start_at(p.batch, u.s));
  const bool two = tr.rows > 16;  // the second 16 columns hold rows

  // This lane's two rows: token, position (-1: no row) and query fragment.
  int64_t qpos[2];
  uint4 qf[2][KK];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int r = tr.row0 + 16 * c + l16;
    const bool have = 16 * c + l16 < tr.rows;
    const int t = r / p.G, h = r - t * p.G;
    qpos[c] = have ? u.w.pos0 + t : -1;
    const uint16_t* src = static_cast<const uint16_t*>(p.q) + (int64_t)(token0 + t) * p.qs[0] +
                          (int64_t)(u.g * p.G + h) * p.qs[1] + 8 * g4;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk)
      qf[c][kk] = have ? *reinterpret_cast<const uint4*>(src + 32 * kk) : uint4{0u, 0u, 0u, 0u};
  }
  // Keys below `end` are read: up to the last row's position.
  const int64_t first_pos = u.w.pos0 + tr.row0 / p.G, last_pos = u.w.pos0 + (tr.row0 + tr.rows - 1) / p.G;
  const int end = last_pos + 1 < p.batch.cap ? (last_pos < 0 ? 0 : (int)(last_pos + 1)) : p.batch.cap;
  // Tiles of this split: of the sequence's positions, or of its list's blocks.
  const int tiles = p.idx ? 2 * p.K : (end + kKeys - 1) / kKeys;
  const int lo = u.split * per * kWaves;
  const int hi = tiles < lo + per * kWaves ? tiles : lo + per * kWaves;

  const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + (int64_t)u.g * p.ks[1] + 8 * g4;
  const uint16_t* vbase = static_cast<const uint16_t*>(p.v) + (int64_t)u.g * p.vs[1] + 8 * g4;
  uint16_t* vl = reinterpret_cast<uint16_t*>(smem) + wave * kKeys * VSTR;

  // First key of tile t, -1 for none: a listed block that is padding or in
  // the future of every row.
  auto key_of = [&](int t) -> int {
    if (t >= hi) return -1;
    if (p.idx == nullptr) return t * kKeys;
    const int id = tr.list != nullptr ? __builtin_amdgcn_readfirstlane(tr.list[t >> 1]) : -1;
    if (id < 0 || (int64_t)id * kBlock >= end) return -1;
    return id * kBlock + (t & 1) * kKeys;
  };
  auto next_key = [&](int& t) -> int {
    for (t += kWaves; t < hi; t += kWaves) {
      const int k = key_of(t);
      if (k >= 0 && k < end) return k;
    }
    return -1;
  };
  // Pages of the keys key0 + l16 and key0 + 16 + l16.
  auto pages_of = [&](int key0, int (&pg)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = key0 + 16 * c + l16;
      pg[c] = key0 >= 0 && key < end ? page_id(p.batch, u.s, key) : -1;
    }
  };
  auto load = [&](const uint16_t* base, const int64_t* st, int key0, const int (&pg)[2], uint4 (&x)[2][KK]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int key = key0 + 16 * c + l16;
      const int slot = key - page_of(p.batch, key) * p.batch.page;
      const uint16_t* src = base + (int64_t)pg[c] * st[0] + (int64_t)slot * st[2];
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        x[c][kk] = pg[c] >= 0 ? *reinterpret_cast<const uint4*>(src + 32 * kk) : uint4{0u, 0u, 0u, 0u};
    }
  };

  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  f32x4v acc[2][DT];
  // A masked key has p = 0, but 0 times a NaN or infinity in its value row is
  // NaN: where the sums come out non-finite, the keys are walked once more
  // with the partly masked tiles taken one column at a time.
  for (bool careful = false;; careful = true) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      m[c] = -INFINITY;
      l[c] = 0.f;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[c][dt] = f32x4v{};
    }
    int t = lo + wave - kWaves, pg[2], pn[2];
    uint4 kx[2][KK], vx[2][KK];
    int key0 = next_key(t);
    pages_of(key0, pg);
    if (key0 >= 0) {
      load(kbase, p.ks, key0, pg, kx);
      load(vbase, p.vs, key0, pg, vx);
    }
    while (key0 >= 0) {
      const int nkey = next_key(t);
      pages_of(nkey, pn);
      const uint32_t have = (uint32_t)(__ballot(pg[0] >= 0) & 0xffffu) | (uint32_t)(__ballot(pg[1] >= 0) << 16);
      f32x4v s[2][2];
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          s[c][kt] = f32x4v{};
          if (c == 0 || two)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) s[c][kt] = mfma16x16x32<F16>(kx[kt][kk], qf[c][kk], s[c][kt]);
        }
      if (nkey >= 0) load(kbase, p.ks, nkey, pn, kx);
      const bool part = have != 0xffffffffu || key0 + kKeys - 1 > first_pos;
      uint4 pk[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (c == 1 && !two) break;
        if (part) {
#pragma unroll
          for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int kr = 16 * kt + 4 * g4 + r;
              if (!((have >> kr) & 1u) || key0 + kr > qpos[c]) s[c][kt][r] = -INFINITY;
            }
        }
        float mx = fmaxf(fmaxf(fmaxf(s[c][0][0], s[c][0][1]), fmaxf(s[c][0][2], s[c][0][3])),
                         fmaxf(fmaxf(s[c][1][0], s[c][1][1]), fmaxf(s[c][1][2], s[c][1][3])));
        mx = quad_max(mx) * p.cs;
        if (__ballot(mx > m[c] + kRescaleThreshold)) {
          const float mn = fmaxf(m[c], mx);
          const float alpha = mn == -INFINITY ? 1.f : fast_exp2(m[c] - mn);
          m[c] = mn;
          l[c] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[c][dt] *= alpha;
        }
        const float nm = m[c] == -INFINITY ? 0.f : -m[c];
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = fast_exp2(fmaf(s[c][i >> 2][i & 3], p.cs, nm));
          l[c] += x[i];
        }
        pk[c] = uint4{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(x[4], x[5]), pack2<F16>(x[6], x[7])};
      }
      // V through the wave's LDS rows; the previous tile's reads of them
      // come before these writes in the wave's own order.
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
          *reinterpret_cast<uint4*>(vl + (16 * kt + l16) * VSTR + 32 * kk + 8 * g4) = vx[kt][kk];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (nkey >= 0) load(vbase, p.vs, nkey, pn, vx);
      const uint16_t* vt = vl + (4 * g4 + (l16 >> 2)) * VSTR + 4 * (l16 & 3);
      if (careful && part) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (c == 1 && !two) break;
          const int64_t off = qpos[c] - key0;
          const int rel = off < -1 ? -1 : (off > kKeys ? kKeys : (int)off);
#pragma unroll 1
          for (int q = 0; q < 16; ++q) {
            // Column q alone, with the value rows that it does not see as zeros.
            const int seen = __builtin_amdgcn_readlane(rel, q);
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int kr = 16 * (i >> 1) + 4 * g4 + 2 * (i & 1);
              w[i] = (((have >> kr) & 1u) && kr <= seen ? 0xffffu : 0u) |
                     (((have >> (kr + 1)) & 1u) && kr + 1 <= seen ? 0xffff0000u : 0u);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const uint2 a = lds_read_tr16(vt + 16 * dt), b = lds_read_tr16(vt + 16 * VSTR + 16 * dt);
              const f32x4v one = mfma16x16x32<F16>(uint4{a.x & w[0], a.y & w[1], b.x & w[2], b.y & w[3]}, pk[c], f32x4v{});
              if (l16 == q) acc[c][dt] += one;
            }
          }
        }
      } else {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint2 a = lds_read_tr16(vt + 16 * dt), b = lds_read_tr16(vt + 16 * VSTR + 16 * dt);
          const uint4 va = {a.x, a.y, b.x, b.y};
          acc[0][dt] = mfma16x16x32<F16>(va, pk[0], acc[0][dt]);
          if (two) acc[1][dt] = mfma16x16x32<F16>(va, pk[1], acc[1][dt]);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      key0 = nkey;
      pg[0] = pn[0];
      pg[1] = pn[1];
    }
    if (careful) break;
    bool odd = false;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) odd |= !(fabsf(acc[c][dt][r]) < INFINITY);
    if (!__ballot(odd)) break;
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    l[c] = quad_sum(l[c]);
    if (g4 == 0) {
      ml[wave][0][16 * c + l16] = m[c];
      ml[wave][1][16 * c + l16] = l[c];
    }
  }
  // The waves' sums joined through LDS, 16 rows at a time: thread t takes
  // D / 16 values of row t / 16.
  float* ol = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (c == 1 && !two) break;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4v*>(ol + (wave * 16 + l16) * OSTR + 16 * dt + 4 * g4) = acc[c][dt];
    __syncthreads();
    constexpr int PER = D / 16;
    const int r = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * PER, row = 16 * c + r;
    if (row >= tr.rows) continue;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w][0][row]);
    const float nm = top == -INFINITY ? 0.f : -top;
    float sum = 0.f, o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) o[i] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = fast_exp2(ml[w][0][row] + nm);
      sum += f * ml[w][1][row];
#pragma unroll
      for (int i = 0; i < PER; ++i) o[i] += f * ol[(w * 16 + r) * OSTR + d0 + i];
    }
    if (u.splits > 1) {
      float* po = p.part_o + ((int64_t)blockIdx.x * kRows + row) * D + d0;
#pragma unroll
      for (int i = 0; i < PER; ++i) po[i] = o[i];
      if (d0 == 0) {
        p.part_ml[(int64_t)blockIdx.x * 2 * kRows + row] = top;
        p.part_ml[(int64_t)blockIdx.x * 2 * kRows + kRows + row] = sum;
      }
      continue;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int t = (tr.row0 + row) / p.G, h = tr.row0 + row - t * p.G;
    uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)(token0 + t) * p.os[0] +
                    (int64_t)(u.g * p.G + h) * p.os[1] + d0;
#pragma unroll
    for (int i = 0; i < PER; i += 2)
      reinterpret_cast<uint32_t*>(dst)[i / 2] = pack2<F16>(o[i] * inv, o[i + 1] * inv);
  }
}

// Joins the splits of one (tile, head): a wave takes every fourth row.
template <int D, bool F16>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttn p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  Unit u;
  const int per = steps_per_unit(p, lane);
  if (!find_unit<true>(p, blockIdx.x, per, lane, u) || u.splits == 1) return;
  const TileRows tr = tile_rows(p, u);
  const int token0 = start_at(p.batch, u.s), stride = u.w.tiles * p.Hkv;
  if (u.first + (int64_t)(u.splits - 1) * stride >= p.grid) return;  // starts that overlap
  constexpr int PER = D / 64;
  for (int row = wave; row < tr.rows; row += 4) {
    float best = -INFINITY;
    for (int i = lane; i < u.splits; i += 64)
      best = fmaxf(best, p.part_ml[((int64_t)u.first + (int64_t)i * stride) * 2 * kRows + row]);
#pragma unroll
    for (int mm = 1; mm < 64; mm *= 2) best = fmaxf(best, __shfl_xor(best, mm));
    const float nm = best == -INFINITY ? 0.f : -best;
    float sum = 0.f, o[PER] = {};
    for (int i = 0; i < u.splits; ++i) {
      const int64_t slot = (int64_t)u.first + (int64_t)i * stride;
      const float f = fast_exp2(p.part_ml[slot * 2 * kRows + row] + nm);
      sum += f * p.part_ml[slot * 2 * kRows + kRows + row];
#pragma unroll
      for (int j = 0; j < PER; ++j) o[j] += f * p.part_o[(slot * kRows + row) * D + PER * lane + j];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int t = (tr.row0 + row) / p.G, h = tr.row0 + row - t * p.G;
    uint16_t* dst = static_cast<uint16_t*>(p.out) + (int64_t)(token0 + t) * p.os[0] +
                    (int64_t)(u.g * p.G + h) * p.os[1] + PER * lane;
    if constexpr (PER == 2)
      *reinterpret_cast<uint32_t*>(dst) = pack2<F16>(o[0] * inv, o[1] * inv);
    else
      *dst = (uint16_t)pack2<F16>(o[0] * inv, 0.f);
  }
}

// Tiles of a (ragged) batch with N new tokens: sequences round up one each.
int64_t tile_bound(int64_t N, int64_t S, int64_t G, bool lists) {
  if (!lists) return (N * G + kRows - 1) / kRows + S;
  // Listed rows also break at every 64 positions.
  const int64_t blocks = N / kBlock + 2 * S < N + S ? N / kBlock + 2 * S : N + S;
  return blocks * ((kBlock * G + kRows - 1) / kRows);
}

}  // namespace

extern "C" int64_t spruce_paged_attention_workspace_bytes(int64_t N, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                                          int64_t K) {
  if (N < 1 || S < 1 || Hkv < 1 || Hq < Hkv || N >= (int64_t)1 << 30 || S >= (int64_t)1 << 20) return 0;
  const int64_t units = tile_bound(N, S, Hq / Hkv, K > 0) * Hkv + kSlots;
  return units * kRows * (D + 2) * 4;
}

extern "C" int spruce_paged_attention(const void* q, const int64_t qs[3], const void* k_pages, const int64_t kps[4],
                                      const void* v_pages, const int64_t vps[4], int64_t pages, int64_t page_size,
                                      const int32_t* page_table, int64_t table_stride, int64_t table_width,
                                      const int32_t* q_starts, const int32_t* kv_lens, int64_t S, int64_t N,
                                      int64_t Hq, int64_t Hkv, int64_t D, float scale, int dtype, const int32_t* idx,
                                      const int64_t is[4], int64_t Qc, int64_t K, void* out, const int64_t os[3],
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  SPRUCE_REQUIRE(qs && kps && vps && os, "stride arrays must be non-null");
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(dtype == SPRUCE_DTYPE_BF16 || dtype == SPRUCE_DTYPE_F16,
                 "the paged attention takes bf16 or f16, got dtype code %d", dtype);
  SPRUCE_REQUIRE(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq < 1 << 16,
                 "query heads (%lld) must be divisible by KV heads (%lld)", (long long)Hq, (long long)Hkv);
  SPRUCE_REQUIRE(Hq / Hkv <= 64, "at most 64 query heads per KV head are supported");
  SPRUCE_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  SPRUCE_REQUIRE(qs[2] == 1 && kps[3] == 1 && vps[3] == 1 && os[2] == 1,
                 "q, the pages and out must have a contiguous final dimension");
  PagedAttn p{};
  const int rc = prepare_batch(p.batch, page_table, table_stride, table_width, q_starts, kv_lens, S, N, page_size, pages);
  if (rc) return rc;
  if (N == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(q && out && (pages == 0 || (k_pages && v_pages)), "q, the pages and out must be non-null device pointers");
  auto rows16 = [](const void* ptr, const int64_t* s, int n) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return false;
    for (int i = 0; i < n; ++i)
      if (s[i] % 8) return false;
    return true;
  };
  SPRUCE_REQUIRE(rows16(q, qs, 2) && rows16(k_pages, kps, 3) && rows16(v_pages, vps, 3) && rows16(out, os, 2),
                 "q, the pages and out must be 16-byte aligned with strides that keep rows 16-byte aligned");
  SPRUCE_REQUIRE(K >= 0 && K < (int64_t)1 << 24, "invalid list width %lld", (long long)K);
  SPRUCE_REQUIRE(K == 0 || (idx && is && Qc >= 0), "indices must be a non-null device pointer");
  SPRUCE_REQUIRE(K == 0 || is[3] == 1, "indices must have a contiguous final dimension");
  const int64_t need = spruce_paged_attention_workspace_bytes(N, S, Hq, Hkv, D, K);
  SPRUCE_REQUIRE(workspace && workspace_bytes >= need, "workspace too small: %lld bytes, need %lld",
                 (long long)workspace_bytes, (long long)need);
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace must be 16-byte aligned");
  p.q = q;
  p.out = out;
  p.k = k_pages;
  p.v = v_pages;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = qs[i];
    p.os[i] = os[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = kps[i];
    p.vs[i] = vps[i];
  }
  p.Hkv = (int)Hkv;
  p.G = (int)(Hq / Hkv);
  p.cs = scale * 1.4426950408889634f;
  if (K > 0) {
    p.idx = idx;
    for (int i = 0; i < 3; ++i) p.is[i] = is[i];
    p.Qc = (int)(Qc < (int64_t)1 << 30 ? Qc : (int64_t)1 << 30);
    p.K = (int)K;
  }
  const int64_t tiles = tile_bound(N, S, p.G, K > 0) * Hkv;
  SPRUCE_REQUIRE(tiles + kSlots < (int64_t)1 << 24, "too many tokens for one call");
  p.grid = (int)(tiles + kSlots);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (int64_t)p.grid * kRows * D;
  const hipStream_t st = (hipStream_t)stream;
  const int64_t most = K > 0 ? K * kBlock : p.batch.cap;  // keys of a row at most
  const bool join = most > kMinSteps * kStep;
#define SPRUCE_PAGED(KERNEL, GRID)                                                                    \
  do {                                                                                                \
    const dim3 g((unsigned)(GRID));                                                                   \
    if (D == 128 && dtype == SPRUCE_DTYPE_BF16)                                                       \
      hipLaunchKernelGGL((KERNEL<128, false>), g, dim3(256), 0, st, p);                               \
    else if (D == 128) hipLaunchKernelGGL((KERNEL<128, true>), g, dim3(256), 0, st, p);               \
    else if (dtype == SPRUCE_DTYPE_BF16) hipLaunchKernelGGL((KERNEL<64, false>), g, dim3(256), 0, st, p); \
    else hipLaunchKernelGGL((KERNEL<64, true>), g, dim3(256), 0, st, p);                              \
    const int e = check_launch(#KERNEL);                                                              \
    if (e) return e;                                                                                  \
  } while (0)
  SPRUCE_PAGED(paged_rows_kernel, join ? p.grid : tiles);
  if (join) SPRUCE_PAGED(paged_join_kernel, tiles);
#undef SPRUCE_PAGED
  return SPRUCE_OK;
}
