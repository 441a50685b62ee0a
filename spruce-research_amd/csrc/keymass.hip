// The attention weight that the cached keys of a paged K/V cache get from a
// ragged batch's new tokens:
//   mass_j (+)= sum over tokens i, heads h of a KV head, of exp(scale q_ih.k_j - lse_ih),
//   lse_ih = log sum_{j <= pos_i} exp(scale q_ih.k_j).
// A weight needs the sum over its row's keys and a mass the sum over its key's
// rows, so there are two passes over the scores, each with one side held in
// registers and the other streamed through LDS:
//   rows  256 packed rows (as in the paged attention: token by token, head by
//         head) against a range of keys: every lane has one row's maximum and
//         sum over its part of the keys, which go to the workspace;
//   keys  256 keys against the rows that see them: every lane has one key's sum.
// Both are S = A B^T on the matrix cores with the streamed side as A, so what is
// held lies in the columns, one a lane, and sums stay within the lane.
//
// Sequences of few packed rows (a decoding step, a few drafted tokens) are bound by
// the read of their keys, which is done once: their scores, 4 bytes against a
// key's 2 D, go to the workspace, with every row's maximum and sum by ranges of keys, and
// a second kernel makes the weights of them.
//
// Measured on one MI355X:
//   one token of each of 64 sequences of 6554 to 32768 keys, 28/4 heads of 128, bf16: 289 to 318 us, 4.1 to
//   4.5 TB/s of keys (by two passes over the keys 952)
//   one token over 517 keys, 8/2 heads: 12 to 14 us
//   windows of 8 to 40 tokens over four prompts of up to 33000 keys, 16/8 heads of 64: 60 us
//   4096 tokens over 32768 keys, 28/4 heads: 2060 to 2090 us, 870 TFLOP/s of its two products
#include "paged_impl.h"

namespace spruce {

struct KeyMass {
  PagedAttn a;     // q, k, the batch; sequences past few_limit packed rows go the many-row way
  float* mass;
  int64_t ms[3];   // page, head, slot strides
  float2* stats;   // [N * Hq][parts]: maximum (of scores as products) and sum, of a whole row its logarithm
  int Hq, parts, accumulate;
  int row_parts;   // of the rows that a key tile sees, where there are few tiles: each a workgroup's
  float* partial;  // their sums, [key tile][KV head][row_parts][256]
  // Sequences of up to few_rows packed rows (all, where no other kernels run): stats by ranges of `range` keys, scores of a (KV head, sequence)
  // as [32 keys][row][key] from its first packed row (of few_tokens, those of such sequences alone where that
  // is fewer than N) times key_room on.
  int few_rows, range, ranges, key_room, few_tokens;
  float* scores;
  float2* few_stats;  // [few_tokens * Hq][ranges]
  float cs_low;       // what scale log2 e has past p.cs
};

namespace {

constexpr int kRowsOf = Many::rows;   // rows, or keys, that a workgroup of 4 waves holds
constexpr int kWave = 64;             // of which a wave
constexpr int kStream = 64;           // rows, or keys, streamed between barriers

// Scores enter the exponential as differences to the row's reference, which the
// matrix cores take off as they accumulate: one product and one exponential an
// element.  The difference is then as exact as a 32-bit score of the reference's
// size; where that is large (times scale log2 e) it is formed from the finished
// score instead, so that the largest weight of a row is one whatever the scores.
constexpr float kLargeReference = 0x1p+10f;
// Scores that the tokens of a call may have for them to go to the workspace; with more all sequences go by two
// passes over the keys.  (1 GiB: one token of 64 sequences over 131072 keys, 28 heads, is 0.88.)
constexpr int64_t kMostScores = (int64_t)1 << 28;
// A tile's sum past this moves the reference.
constexpr float kRescaleSum = 0x1p+60f;

// Rows (or keys) streamed: [kStream][D + 8] 16-bit elements.
template <int D>
struct Stream {
  static constexpr int stride = D + 8, lanes = D / 8, rows = 256 / lanes, passes = kStream / rows;
};

// S^T's 32 x 64 block: streamed rows a (LDS), held columns b, what to begin with c.
template <int D, bool F16>
__device__ __forceinline__ void products(const uint16_t* rows, const u32x4 (&b)[2][D / 16], int lane, const f32x16_t& c0,
                                         const f32x16_t& c1, f32x16_t& x0, f32x16_t& x1) {
  const uint16_t* at = rows + (lane & 31) * Stream<D>::stride + 8 * (lane >> 5);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint4 a = *reinterpret_cast<const uint4*>(at + 16 * kk);
    x0 = mfma32x32x16<F16>(a, __builtin_bit_cast(uint4, b[0][kk]), kk == 0 ? c0 : x0);
    x1 = mfma32x32x16<F16>(a, __builtin_bit_cast(uint4, b[1][kk]), kk == 0 ? c1 : x1);
  }
}

// What is held is there from here on, for the compiler too: in the loop it would wait for all loads in flight,
// the next tile's among them, before the first use.
template <int N>
__device__ __forceinline__ void settle(u32x4 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}

// The streamed row of accumulator register r, within 32.
__device__ __forceinline__ int row_of(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

// One column's running sum of exp2(cs (s - m)); l is 0 until m is set.
struct Sum {
  float m = 0.f, l = 0.f;
  // x: scores less m.
  __device__ __forceinline__ void add(const f32x16_t& x, float cs) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) t += fast_exp2(x[r] * cs);
    if (__ballot(l == 0.f || !(t < kRescaleSum))) {
      float mx = x[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, x[r]);
      if (mx > -INFINITY && (l == 0.f || !(t < kRescaleSum))) {
        l *= l == 0.f ? 0.f : fast_exp2(-mx * cs);
        m += mx;
        t = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) t += fast_exp2((x[r] - mx) * cs);
      }
    }
    l += t;
  }
  // s: the scores.
  __device__ __forceinline__ void add_large(const f32x16_t& s, float cs) {
    float mx = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
    float now = l == 0.f ? mx : fmaxf(m, mx);
    if (now == -INFINITY) now = 0.f;  // nothing yet, but perhaps NaN
    float t = l == 0.f ? 0.f : l * fast_exp2((m - now) * cs);
#pragma unroll
    for (int r = 0; r < 16; ++r) t += fast_exp2((s[r] - now) * cs);
    m = now;
    l = t;
  }
  __device__ __forceinline__ void join(float m2, float l2, float cs) {
    if (l2 == 0.f) return;
    if (l == 0.f) {
      m = m2;
      l = l2;
      return;
    }
    const float now = fmaxf(m, m2);
    l = l * fast_exp2((m - now) * cs) + l2 * fast_exp2((m2 - now) * cs);
    m = now;
  }
};

// What a row's weights are formed with: its maximum, and the logarithm of its sum, infinite where it has no key.
// (With what the instruction's result lacks: the same way in all rows, it was 3e-7 of every mass.)
__device__ __forceinline__ float2 whole_row(const Sum& s) {
  const float lg = __builtin_amdgcn_logf(s.l);
  return float2{s.m, s.l == 0.f ? INFINITY : fmaf(s.l, fast_exp2(-lg), -1.f) * 1.44269504f + lg};
}

// EVEN: pages hold whole passes of the stream's loads, so a pass has one page, and its address but
// for the lane's part is found on the scalar unit (looked up by every lane, as with other pages, a chunk of
// 4096 tokens over 32768 keys took 1342 us here rather than 1282 at that stage, 1000 now).  Three waves a SIMD, without the registers
// that would have a wave's own products and exponentials overlap (two waves: 1395).
template <int D, bool F16, bool EVEN>
__global__ __launch_bounds__(256, 3) void key_mass_rows_kernel(const KeyMass a) {
  typedef Stream<D> ST;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][kStream * ST::stride];
  __shared__ int paged[2][kStream];
  const PagedAttn& p = a.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const uint32_t block = flat_block();
  const int g = (int)(block % (uint32_t)p.Hkv);
  const uint32_t rest = block / (uint32_t)p.Hkv;
  const int part = (int)(rest % (uint32_t)a.parts), at = (int)(rest / (uint32_t)a.parts);
  Unit u;
  if (!find_tile<Many>(p, at, g, lane, u)) return;
  const TileRows tr = tile_rows(p, u);
  if (tr.rows == 0) return;

  // This lane's two columns.
  // Up to two waves' rows: the other two take the second half of every tile's keys.  (Windows of 8 to 40 tokens
  // over four prompts, 16/8 heads of 64: 33 us, 26 so.)
  const bool halves = tr.rows <= 2 * kWave;
  const int group = halves ? wave & 1 : wave, sub0 = halves ? wave >> 1 : 0, sub1 = halves ? sub0 + 1 : kStream / 32;
  const int mine = uniform(tr.rows - kWave * group);  // rows of this wave, if positive
  u32x4 held[2][D / 16];
  int qpos[2];
  int64_t out[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int i = kWave * group + 32 * c + l32;
    const int r = tr.row0 + (i < tr.rows ? i : tr.rows - 1);
    const int t = p.by_group.of(r), h = g * p.G + r - t * p.G;
    qpos[c] = clip(u.w.pos0 + t);
    out[c] = (int64_t)(u.w.start + t) * a.Hq + h;
    const uint16_t* src =
        static_cast<const uint16_t*>(p.q) + (int64_t)(u.w.start + t) * p.qs[0] + (int64_t)h * p.qs[1] + 8 * hl;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) held[c][kk] = load16(src + 16 * kk);
  }
  const int first_pos = uniform(clip(u.w.pos0 + p.by_group.of(tr.row0 + (mine > 0 ? kWave * group : 0))));

  const int tiles = (tr.end + kStream - 1) / kStream, per = (tiles + a.parts - 1) / a.parts;
  const int t0 = part * per < tiles ? part * per : tiles, t1 = t0 + per < tiles ? t0 + per : tiles;
  const int lr = tid / ST::lanes, lc = tid % ST::lanes;
  const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + (int64_t)g * p.ks[1] + 8 * lc;
  int entry[ST::passes];
  u32x4 row[ST::passes];
  int there[ST::passes];
  uint64_t have_next = 0;
  const int64_t lane_part = lr * p.ks[2];
  auto look_up = [&](int tile) {
#pragma unroll
    for (int i = 0; i < ST::passes; ++i) {
      if constexpr (EVEN) {
        const int at_page = uniform(page_of(p.batch, nearest(tile * kStream + i * ST::rows, tr.end)));
        const int32_t* table = p.batch.table + (int64_t)u.s * p.batch.table_stride;
        entry[i] = ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)table)[at_page];
      } else {
        entry[i] = page_entry(p.batch, u.s, nearest(tile * kStream + i * ST::rows + lr, tr.end));
      }
    }
  };
  auto load = [&](int tile) {
    if constexpr (EVEN) {
      have_next = 0;
#pragma unroll
      for (int i = 0; i < ST::passes; ++i) {
        const int key = uniform(nearest(tile * kStream + i * ST::rows, tr.end));
        const int first = key - uniform(page_of(p.batch, key)) * p.batch.page;
        const bool ok = is_page(p.batch, entry[i]);
        // (Past the end the pass begins at the last key: its page's rows are read from that row's pass on.)
        const int slot = first - first % ST::rows;
        row[i] = load16(kbase + ((int64_t)(ok ? entry[i] : 0) * p.ks[0] + (int64_t)slot * p.ks[2]) + lane_part);
        if (ok) have_next |= (ST::rows == 64 ? ~0ull : (1ull << (ST::rows & 63)) - 1) << (i * ST::rows);
      }
      const int left = tr.end - tile * kStream;
      if (left < kStream) have_next &= (1ull << left) - 1;
    } else {
#pragma unroll
      for (int i = 0; i < ST::passes; ++i) {
        const int key = tile * kStream + i * ST::rows + lr, in = nearest(key, tr.end);
        const int slot = in - page_of(p.batch, in) * p.batch.page;
        const bool ok = is_page(p.batch, entry[i]);
        there[i] = ok && key < tr.end;
        row[i] = load16(kbase + (int64_t)(ok ? entry[i] : 0) * p.ks[0] + (int64_t)slot * p.ks[2]);
      }
    }
  };
  Sum sum[2];
  if (t0 < t1) {
    look_up(t0);
    load(t0);
    if (t0 + 1 < t1) look_up(t0 + 1);
  }
  settle(held[0]);
  settle(held[1]);
  for (int t = t0; t < t1; ++t) {
    const int b = t & 1;
#pragma unroll
    for (int i = 0; i < ST::passes; ++i) {
      *reinterpret_cast<u32x4*>(&lds[b][(i * ST::rows + lr) * ST::stride + 8 * lc]) = row[i];
      if (!EVEN && lc == 0) paged[b][i * ST::rows + lr] = there[i];
    }
    const uint64_t have_now = have_next;
    __syncthreads();
    if (t + 1 < t1) {
      load(t + 1);
      if (t + 2 < t1) look_up(t + 2);
    }
    if (mine <= 0) continue;
    const uint64_t have = EVEN ? have_now : __ballot(paged[b][lane] != 0);
    const int key0 = t * kStream;
    const bool masked = have != ~0ull || key0 + kStream - 1 > first_pos;
    const bool large =
        __ballot(fabsf(sum[0].m * p.cs) >= kLargeReference || fabsf(sum[1].m * p.cs) >= kLargeReference) != 0;
#pragma unroll 1
    for (int sub = sub0; sub < sub1; ++sub) {
      f32x16_t x[2];
      if (large) {
        const f32x16_t zero = {};
        products<D, F16>(&lds[b][32 * sub * ST::stride], held, lane, zero, zero, x[0], x[1]);
      } else {
        f32x16_t less[2];
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) less[c][r] = -sum[c].m;
        products<D, F16>(&lds[b][32 * sub * ST::stride], held, lane, less[0], less[1], x[0], x[1]);
      }
      if (masked) {
        const uint32_t in = (uint32_t)(have >> (32 * sub));
        const int lane_now = lane + opaque_zero();  // the keys' bits are found here, not kept in 32 registers
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int k = row_of(r, lane_now);
            if (!(in >> k & 1) || key0 + 32 * sub + k > qpos[c]) x[c][r] = -INFINITY;
          }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (large)
          sum[c].add_large(x[c], p.cs);
        else
          sum[c].add(x[c], p.cs);
      }
      // (A reference that has just become large: the next 64 keys go by it.)
    }
  }
  __syncthreads();
  float2* other = reinterpret_cast<float2*>(lds);  // of the second half's waves
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float m0, m1, s0, s1;
    half_swap(sum[c].m, m0, m1);
    half_swap(sum[c].l, s0, s1);
    Sum all;
    all.join(m0, s0, p.cs);
    all.join(m1, s1, p.cs);
    sum[c] = all;
    if (halves && wave >= 2 && hl == 0) other[(wave - 2) * kWave + 32 * c + l32] = float2{all.m, all.l};
  }
  __syncthreads();
  if (halves && wave >= 2) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    Sum all = sum[c];
    if (halves) {
      const float2 x = other[wave * kWave + 32 * c + l32];
      all.join(x.x, x.y, p.cs);
    }
    if (hl == 0 && 32 * c + l32 < mine)
      a.stats[out[c] * a.parts + part] = a.parts == 1 ? whole_row(all) : float2{all.m, all.l};
  }
}

// Joins the parts of every row's keys: the first part's place has the whole row's afterwards.
__global__ __launch_bounds__(256) void key_mass_join_kernel(float2* stats, int64_t rows, int parts, float cs) {
  const int64_t r = (int64_t)flat_block() * 256 + threadIdx.x;
  if (r >= rows) return;
  float2* st = stats + r * parts;
  Sum all;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) {
    const float2 x = st[i];
    all.join(x.x, x.y, cs);
  }
  st[0] = whole_row(all);
}

// The at-th of the key tiles of all sequences with new tokens.
struct KeyTile {
  int s, tile, len, start, n;
  int row;  // the first of the rows, of a unit that has not all
  int place;  // of the first token among few_tokens
  int64_t pos0;
};
__device__ __forceinline__ bool find_keys(const PagedAttn& p, int64_t at, int lane, KeyTile& k) {
  int64_t count = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const Lengths len = lengths_of(p, s0 + lane);
    const int a = clamp_start(p.batch, len.starts), e = clamp_start(p.batch, len.ends);
    int keys = len.keys < 0 ? 0 : (len.keys < p.batch.cap ? len.keys : p.batch.cap);
    if (e <= a || (int64_t)(e - a) * p.G <= p.few_limit || p.batch.pages == 0) keys = 0;
    const int64_t pc = count + wave_prefix((int64_t)((keys + kRowsOf - 1) / kRowsOf));
    const uint64_t past = __ballot(pc > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      k.s = s0 + l;
      k.len = __builtin_amdgcn_readlane(keys, l);
      k.tile = uniform((int)(at - lane_of(pc, l))) + (k.len + kRowsOf - 1) / kRowsOf;
      k.start = __builtin_amdgcn_readlane(a, l);
      k.n = __builtin_amdgcn_readlane(e, l) - k.start;
      k.pos0 = lane_of((int64_t)len.keys - ((int64_t)len.ends - len.starts) + ((int64_t)a - len.starts), l);
      return true;
    }
    count = lane_of(pc, 63);
  }
  return false;
}

// Key `key` of a sequence, in the table's entry `entry`, has got v.
__device__ __forceinline__ void set_mass(const KeyMass& a, const KeyTile& k, int g, int key, int entry, float v) {
  const int slot = key - page_of(a.a.batch, key) * a.a.batch.page;
  float* to = a.mass + (int64_t)entry * a.ms[0] + (int64_t)g * a.ms[1] + (int64_t)slot * a.ms[2];
  *to = a.accumulate && key < k.pos0 ? *to + v : v;
}

// Joins the sums of key tiles whose rows were shared out, in their order.
__global__ __launch_bounds__(256) void key_mass_add_kernel(const KeyMass a) {
  const PagedAttn& p = a.a;
  const int tid = threadIdx.x, lane = tid & 63;
  for (int64_t tile = blockIdx.x;; tile += gridDim.x) {
    const int64_t at = tile / p.Hkv;
    const int g = (int)(tile - at * p.Hkv);
    KeyTile k;
    if (!find_keys(p, at, lane, k)) return;
    float v = 0.f;
    for (int i = 0; i < a.row_parts; ++i) v += a.partial[(tile * a.row_parts + i) * kRowsOf + tid];
    const int key = k.tile * kRowsOf + tid;
    if (key >= k.len) continue;
    const int entry = page_entry(p.batch, k.s, key);
    if (is_page(p.batch, entry)) set_mass(a, k, g, key, entry, v);
  }
}

template <int D, bool F16>
__global__ __launch_bounds__(256, 2) void key_mass_keys_kernel(const KeyMass a) {
  typedef Stream<D> ST;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][kStream * ST::stride];
  // Of the streamed rows: what to take off the scores, its parts, and the position.
  __shared__ __attribute__((aligned(16))) float less[2][kStream], top[2][kStream], log_sum[2][kStream];
  __shared__ int pos[2][kStream], large[2];
  const PagedAttn& p = a.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, hl = lane >> 5;
  const int lr = tid / ST::lanes, lc = tid % ST::lanes;
  const float per_cs = 1.f / p.cs;
  for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
    const int64_t tile = unit / a.row_parts, at = tile / p.Hkv;
    const int row_part = (int)(unit - tile * a.row_parts), g = (int)(tile - at * p.Hkv);
    KeyTile k;
    if (!find_keys(p, at, lane, k)) return;
    const int key0 = k.tile * kRowsOf + kWave * wave;
    u32x4 held[2][D / 16];
    int key[2], entry[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      key[c] = key0 + 32 * c + l32;
      const int in = nearest(key[c], k.len);
      entry[c] = page_entry(p.batch, k.s, in);
      const bool ok = is_page(p.batch, entry[c]);
      const int slot = in - page_of(p.batch, in) * p.batch.page;
      const uint16_t* src = static_cast<const uint16_t*>(p.k) + (int64_t)(ok ? entry[c] : 0) * p.ks[0] +
                            (int64_t)g * p.ks[1] + (int64_t)slot * p.ks[2] + 8 * hl;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) held[c][kk] = load16(src + 16 * kk);
      if (key[c] >= k.len) entry[c] = -1;
    }
    // Rows from the first that sees the tile's first key on.
    const int64_t skip = (int64_t)k.tile * kRowsOf - k.pos0;
    int rows = k.n * p.G, row0 = skip <= 0 ? 0 : (skip < k.n ? (int)skip * p.G : rows);
    if (a.row_parts > 1) {
      const int steps = (rows - row0 + kStream - 1) / kStream, per = (steps + a.row_parts - 1) / a.row_parts * kStream;
      const int begin = row0 + row_part * per;
      row0 = begin < rows ? begin : rows;
      rows = row0 + per < rows ? row0 + per : rows;
    }
    // The stream's rows follow by kStream packed rows: a row's head goes on by what that leaves of
    // the group, its token by the rest.
    u32x4 row[ST::passes];
    const uint16_t* from[ST::passes];
    int head[ST::passes];
    const int tokens = kStream / p.G, heads = kStream - tokens * p.G;
    const int64_t plain = tokens * p.qs[0] + heads * p.qs[1], wrapped = plain + p.qs[0] - p.G * p.qs[1];
#pragma unroll
    for (int i = 0; i < ST::passes; ++i) {
      const int r = nearest(row0 + i * ST::rows + lr, rows), t = p.by_group.of(r);
      head[i] = r - t * p.G;
      from[i] = static_cast<const uint16_t*>(p.q) + (int64_t)(k.start + t) * p.qs[0] +
                (int64_t)(g * p.G + head[i]) * p.qs[1] + 8 * lc;
    }
    float2 stat{0.f, INFINITY};
    int row_pos = -1;
    auto load = [&](int r0) {
#pragma unroll
      for (int i = 0; i < ST::passes; ++i) {
        if (r0 > row0 && r0 + i * ST::rows + lr < rows) {
          const int next = head[i] + heads;
          const bool wrap = next >= p.G;
          head[i] = wrap ? next - p.G : next;
          from[i] += wrap ? wrapped : plain;
        }
        row[i] = load16(from[i]);
      }
      stat = float2{0.f, INFINITY};
      row_pos = -1;
      if (tid < kStream && r0 + tid < rows) {
        const int t = p.by_group.of(r0 + tid), h = g * p.G + r0 + tid - t * p.G;
        row_pos = clip(k.pos0 + t);
        stat = a.stats[((int64_t)(k.start + t) * a.Hq + h) * a.parts];
      }
    };
    // A key's weights are added up 64 rows at a time, and these sums with what each addition rounds off kept for the
    // next: tens of thousands of rows of about one weight, in one line, were off by 3e-4 of their sum.
    float sum[2] = {0.f, 0.f}, lost[2] = {0.f, 0.f};
    if (row0 < rows) load(row0);
    settle(held[0]);
    settle(held[1]);
    int b = 0;
    for (int r0 = row0; r0 < rows; r0 += kStream, b ^= 1) {
#pragma unroll
      for (int i = 0; i < ST::passes; ++i)
        *reinterpret_cast<u32x4*>(&lds[b][(i * ST::rows + lr) * ST::stride + 8 * lc]) = row[i];
      if (tid < kStream) {  // one wave
        // No key: nothing of it reaches a sum.  (The quotient is mended: its error is the same in all rows.)
        const float lg = stat.y, by = lg * per_cs;
        const float ref = lg == INFINITY ? lg : stat.x + fmaf(fmaf(-by, p.cs, lg), per_cs, by);
        less[b][tid] = -ref;
        top[b][tid] = stat.x;
        log_sum[b][tid] = lg;
        pos[b][tid] = row_pos;
        const uint64_t odd = __ballot(lg != INFINITY && !(fabsf(ref * p.cs) < kLargeReference));
        if (tid == 0) large[b] = odd != 0;
      }
      __syncthreads();
      if (r0 + kStream < rows) load(r0 + kStream);
      if (key0 >= k.len) continue;
      // (Rows go up with their positions.)
      const bool masked = uniform(pos[b][0]) < key0 + kWave - 1;
      const bool is_large = uniform(large[b]) != 0;
      float now[2] = {0.f, 0.f};
#pragma unroll 1
      for (int sub = 0; sub < kStream / 32; ++sub) {
        f32x16_t x[2], c;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4_t v = *reinterpret_cast<const f32x4_t*>(&less[b][32 * sub + 8 * i + 4 * hl]);
#pragma unroll
          for (int j = 0; j < 4; ++j) c[4 * i + j] = v[j];
        }
        if (is_large) c = f32x16_t{};
        products<D, F16>(&lds[b][32 * sub * ST::stride], held, lane, c, c, x[0], x[1]);
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int at_pos = pos[b][32 * sub + row_of(r, lane)];
#pragma unroll
            for (int c = 0; c < 2; ++c)
              if (key[c] > at_pos) x[c][r] = -INFINITY;
          }
        }
        if (is_large) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float m = top[b][32 * sub + row_of(r, lane)], lg = log_sum[b][32 * sub + row_of(r, lane)];
            const int at_pos = pos[b][32 * sub + row_of(r, lane)];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              // No weight is above one, whatever a score's last bits are.
              const float e = (x[c][r] - m) * p.cs - lg, w = fast_exp2(e > 0.f ? 0.f : e);
              now[c] += key[c] <= at_pos ? w : 0.f;  // (of a row whose sum is NaN too)
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int c = 0; c < 2; ++c) now[c] += fast_exp2(x[c][r] * p.cs);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float more = now[c] - lost[c], all = sum[c] + more;
        lost[c] = (all - sum[c]) - more;
        sum[c] = all;
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float v = half_sum(sum[c]);
      if (hl != c) continue;
      if (a.row_parts > 1)
        a.partial[unit * kRowsOf + kWave * wave + 32 * c + l32] = v;
      else if (is_page(p.batch, entry[c]))
        set_mass(a, k, g, key[c], entry[c], v);
    }
    __syncthreads();  // LDS is free
  }
}

// ------------------------------------------------------------------ few rows

constexpr int kFewTile = 32;  // rows, and keys, of a wave's tile
// Keys of a workgroup.  (64 sequences of up to 32768: the scores 285 us, the weights 36; 2048: 290 and 36, 512: 286 and 39.)
constexpr int kMostRange = 1024;

// exp2(cs d) with the product's rounding and cs's made good: the argument is some tens, so that half
// a step of it is some 2^-20 of the result.
__device__ __forceinline__ float weight_of(float d, float cs, float cs_low) {
  const float y = d * cs;
  const float off = fmaf(d, cs, -y) + d * cs_low;
  return y < -150.f ? 0.f : fast_exp2(y) * fmaf(off, 0.69314718f, 1.f);  // (NaN stays NaN)
}

// The at-th range of `keys` keys of all sequences of few rows.
// ROWS: of its rows, so many at a time (0: all).
template <int ROWS>
__device__ __forceinline__ bool find_range(const KeyMass& a, int64_t at, int keys, int lane, KeyTile& k) {
  const PagedAttn& p = a.a;
  const bool own_places = a.few_tokens < p.batch.N;
  int64_t count = 0;
  int tokens = 0;
  for (int s0 = 0; s0 < p.batch.S; s0 += 64) {
    const Lengths len = lengths_of(p, s0 + lane);
    const int first = clamp_start(p.batch, len.starts), e = clamp_start(p.batch, len.ends);
    int n = len.keys < 0 ? 0 : (len.keys < p.batch.cap ? len.keys : p.batch.cap);
    const bool few = e > first && (int64_t)(e - first) * p.G <= a.few_rows;
    if (!few || p.batch.pages == 0) n = 0;
    const int mine = few ? e - first : 0, upto = own_places ? tokens + wave_prefix(mine) : 0;
    const int64_t row_tiles = ROWS && e > first ? ((int64_t)(e - first) * p.G + ROWS - 1) / (ROWS ? ROWS : 1) : 1;
    const int64_t pc = count + wave_prefix((n + keys - 1) / keys * row_tiles);
    const uint64_t past = __ballot(pc > at);
    if (past) {
      const int l = __builtin_ctzll(past);
      k.s = s0 + l;
      k.len = __builtin_amdgcn_readlane(n, l);
      const int ranges = (k.len + keys - 1) / keys, tiles = ROWS ? (int)lane_of(row_tiles, l) : 1;
      k.tile = uniform((int)(at - lane_of(pc, l) + (int64_t)ranges * tiles));
      k.row = 0;
      if (tiles > 1) {
        k.row = k.tile % tiles * ROWS;
        k.tile /= tiles;
      }
      k.start = __builtin_amdgcn_readlane(first, l);
      k.n = __builtin_amdgcn_readlane(e, l) - k.start;
      k.place = own_places ? __builtin_amdgcn_readlane(upto, l) - k.n : k.start;
      k.pos0 = lane_of((int64_t)len.keys - ((int64_t)len.ends - len.starts) + ((int64_t)first - len.starts), l);
      return true;
    }
    count = lane_of(pc, 63);
    tokens = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

__device__ __forceinline__ float* scores_of(const KeyMass& a, const KeyTile& k, int g) {
  return a.scores + ((int64_t)g * a.few_tokens + k.place) * a.a.G * (int64_t)a.key_room;
}

// The scores of a range of keys: every wave takes 32 keys at a time of its own, as in
// the paged attention: whole rows from memory, past the caches, through the wave's own LDS.
// The rows are columns of the products, one a lane: 32, or 16 where sequences have no more, which halves what
// is done for columns without a row.  (One token of each of 64 sequences of 16384 keys, 28/4 heads, by 32 columns and by
// 16: 249 us and 241, of one of 32768 29 and 27, two tokens of 16 of 16384 97 and 89; of four of 131072, 16/8 heads, 234
// and 238.)
template <int D, bool F16, int COLS>
__global__ __launch_bounds__(256, COLS == 16 ? 4 : 3) void key_scores_kernel(const KeyMass a) {
  constexpr int STR = D + 8, LROWS = 512 / D, LI = kFewTile / LROWS;
  constexpr int GROUPS = 64 / COLS, DEPTH = 8 * GROUPS, SCORES = kFewTile / GROUPS;  // scores of a lane
  __shared__ __attribute__((aligned(16))) uint16_t lds[4][kFewTile * STR];
  __shared__ float2 sums[4 * GROUPS][COLS];
  const PagedAttn& p = a.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int l32 = lane & 31, col = lane % COLS, group = lane / COLS, lr = lane / (D / 8), lc = lane % (D / 8);
  uint16_t* mine = lds[wave];
  // Of a lane's i-th score: its key.
  auto key_of = [](int i, int lane) {
    if constexpr (COLS == 32)
      return row_of(i, lane);
    else
      return 16 * (i >> 2) + 4 * (lane >> 4) + (i & 3);
  };
  for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
    const int64_t at = unit / p.Hkv;
    const int g = (int)(unit - at * p.Hkv);
    KeyTile k;
    if (!find_range<COLS>(a, at, a.range, lane, k)) return;
    const int rows = k.n * p.G;
    const int r = k.row + col < rows ? k.row + col : rows - 1, t = p.by_group.of(r), h = g * p.G + r - t * p.G;
    const int qpos = clip(k.pos0 + t);
    const uint16_t* src =
        static_cast<const uint16_t*>(p.q) + (int64_t)(k.start + t) * p.qs[0] + (int64_t)h * p.qs[1] + 8 * group;
    u32x4 held[D / DEPTH];
#pragma unroll
    for (int kk = 0; kk < D / DEPTH; ++kk) held[kk] = load16(src + DEPTH * kk);
    const int k0 = k.tile * a.range + kFewTile * wave;
    const int k1 = (k.tile + 1) * a.range < k.len ? (k.tile + 1) * a.range : k.len;
    const uint16_t* kbase = static_cast<const uint16_t*>(p.k) + (int64_t)g * p.ks[1] + 8 * lc;
    float* out = scores_of(a, k, g) + (k.row + col) * kFewTile + 4 * group;
    const int first_pos = uniform(clip(k.pos0));
    // The next tile of keys in flight, its table entries looked up a tile before.  (Two tiles in
    // flight: 333 us where one took 327.)
    constexpr int STEP = 4 * kFewTile;
    u32x4 x[LI];
    int entry, ahead;
    auto look_up = [&](int key0) { return page_entry(p.batch, k.s, nearest(key0 + l32, k.len)); };
    auto load = [&](int key0, int e) {
#pragma unroll
      for (int i = 0; i < LI; ++i) {
        const int from = __shfl(e, i * LROWS + lr);
        const int key = nearest(key0 + i * LROWS + lr, k.len);
        const int slot = key - page_of(p.batch, key) * p.batch.page;
        x[i] = load16_once(kbase + (int64_t)(is_page(p.batch, from) ? from : 0) * p.ks[0] + (int64_t)slot * p.ks[2]);
      }
    };
    Sum sum;
    if (k0 < k1) {
      entry = look_up(k0);
      load(k0, entry);
      ahead = look_up(k0 + STEP);
    }
    settle(held);
    for (int key0 = k0; key0 < k1; key0 += STEP) {
      uint32_t have = (uint32_t)__ballot(is_page(p.batch, entry));
      if (k.len - key0 < kFewTile) have &= (1u << (k.len - key0)) - 1;
#pragma unroll
      for (int i = 0; i < LI; ++i) *reinterpret_cast<u32x4*>(mine + (i * LROWS + lr) * STR + 8 * lc) = x[i];
      wave_lds_fence();
      entry = ahead;
      if (key0 + STEP < k1) {
        load(key0 + STEP, entry);
        ahead = look_up(key0 + 2 * STEP);
      }
      float s[SCORES];
      if constexpr (COLS == 32) {
        f32x16_t x = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint4 row = *reinterpret_cast<const uint4*>(mine + l32 * STR + 8 * group + 16 * kk);
          x = mfma32x32x16<F16>(row, __builtin_bit_cast(uint4, held[kk]), x);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = x[i];
      } else {
        f32x4v x[2] = {};
#pragma unroll
        for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const u32x4 row = *reinterpret_cast<const u32x4*>(mine + (16 * i + col) * STR + 8 * group + 32 * kk);
            x[i] = mfma16x16x32<F16>(row, held[kk], x[i]);
          }
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = x[i >> 2][i & 3];
      }
      wave_lds_fence();
      if (have != 0xffffffffu || key0 + kFewTile - 1 > first_pos) {
#pragma unroll
        for (int i = 0; i < SCORES; ++i)
          if (!(have >> key_of(i, lane) & 1) || key0 + key_of(i, lane) > qpos) s[i] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < SCORES; ++i) mx = fmaxf(mx, s[i]);
      float now = sum.l == 0.f ? mx : fmaxf(sum.m, mx);
      if (now == -INFINITY) now = 0.f;  // nothing yet, but perhaps NaN
      float l = sum.l == 0.f ? 0.f : sum.l * weight_of(sum.m - now, p.cs, a.cs_low);
#pragma unroll
      for (int i = 0; i < SCORES; ++i) l += weight_of(s[i] - now, p.cs, a.cs_low);
      sum.m = now;
      sum.l = l;
      if (k.row + col < rows) {
        float* to = out + (int64_t)(key0 / kFewTile) * rows * kFewTile;
#pragma unroll
        for (int i = 0; i < SCORES / 4; ++i)
          *reinterpret_cast<f32x4_t*>(to + 4 * GROUPS * i) = f32x4_t{s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]};
      }
    }
    sums[GROUPS * wave + group][col] = float2{sum.m, sum.l};
    __syncthreads();
    if (tid < COLS && k.row + col < rows) {
      Sum all;
#pragma unroll
      for (int i = 0; i < 4 * GROUPS; ++i) all.join(sums[i][col].x, sums[i][col].y, p.cs);
      a.few_stats[((int64_t)(k.place + t) * a.Hq + h) * a.ranges + k.tile] = float2{all.m, all.l};
    }
    __syncthreads();
  }
}

// The weights of 1024 keys, four a thread, from their scores.
constexpr int kWeightKeys = 1024;
__global__ __launch_bounds__(256) void key_weights_kernel(const KeyMass a) {
  __shared__ float2 parts[8][kFewTile], row[kFewTile];
  __shared__ int reach;  // the last position of a row whose sum is NaN
  const PagedAttn& p = a.a;
  const int tid = threadIdx.x, lane = tid & 63;
  for (int64_t unit = blockIdx.x;; unit += gridDim.x) {
    const int64_t at = unit / p.Hkv;
    const int g = (int)(unit - at * p.Hkv);
    KeyTile k;
    if (!find_range<0>(a, at, kWeightKeys, lane, k)) return;
    const int rows = k.n * p.G, ranges = (k.len + a.range - 1) / a.range;
    const float* scores = scores_of(a, k, g);
    int key[4], entry[4];
    const float* from[4];
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      key[i] = k.tile * kWeightKeys + i * 256 + tid;
      const int in = nearest(key[i], k.len);
      entry[i] = page_entry(p.batch, k.s, in);
      from[i] = scores + (int64_t)(in / kFewTile) * rows * kFewTile + in % kFewTile;
    }
    for (int r0 = 0; r0 < rows; r0 += kFewTile) {
      const int n = rows - r0 < kFewTile ? rows - r0 : kFewTile;
      const int of = tid % kFewTile, r = r0 + of, t = p.by_group.of(r), h = g * p.G + r - t * p.G;
      Sum one;
      if (of < n) {
        const float2* st = a.few_stats + ((int64_t)(k.place + t) * a.Hq + h) * a.ranges;
        for (int i = tid / kFewTile; i < ranges; i += 8) one.join(st[i].x, st[i].y, p.cs);
      }
      parts[tid / kFewTile][of] = float2{one.m, one.l};
      __syncthreads();
      if (tid < kFewTile) {
        Sum all;
#pragma unroll
        for (int i = 0; i < 8; ++i) all.join(parts[i][tid].x, parts[i][tid].y, p.cs);
        // Of a row whose sum is NaN the keys that it sees get NaN, by `reach`, and masked ones nothing (their weight
        // of zero times NaN would be NaN).
        const bool none = !(all.l == all.l);
        row[tid] = float2{none ? INFINITY : all.m, none || all.l == 0.f ? 0.f : 1.f / all.l};
        const uint64_t bad = __ballot(none);
        if (tid == 0) reach = bad ? clip(k.pos0 + p.by_group.of(r0 + 63 - __builtin_clzll(bad))) : -1;
      }
      __syncthreads();
#pragma unroll 2
      for (int i = 0; i < n; ++i) {
        const float2 ml = row[i];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sum[j] += weight_of(from[j][(int64_t)(r0 + i) * kFewTile] - ml.x, p.cs, a.cs_low) * ml.y;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (key[j] <= reach) sum[j] = NAN;
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (key[i] >= k.len || !is_page(p.batch, entry[i])) continue;
      set_mass(a, k, g, key[i], entry[i], sum[i]);
    }
  }
}

struct MassPlan {
  bool few, many;
  bool narrow;  // few rows as 16 columns
  int64_t tiles, parts;  // row tiles that a batch can have, and the parts of the keys of each
  int64_t range, ranges, key_room, few_tokens;
  int64_t row_parts;     // of the rows of a key tile
  int64_t many_bytes, partial_bytes, few_stats_bytes, score_bytes;
  int64_t bytes() const { return many_bytes + partial_bytes + few_stats_bytes + score_bytes; }
};
MassPlan mass_plan(int64_t N, int64_t S, int64_t Hq, int64_t Hkv, int64_t keys) {
  const int64_t G = Hq / Hkv;
  MassPlan plan{};
  // As in the attention's plan: the lengths are not known here, but every sequence has a new token
  // in all but odd batches (whose longer ones then go the few-row way, 32 rows at a time).
  const int64_t longest = N > S ? N - S + 1 : 1;
  plan.key_room = (keys + kFewTile - 1) / kFewTile * kFewTile;
  // Where the average is past it too, few sequences are taken to be alike: the launches of the other kind cost more
  // than they save (four windows of 8 to 40 tokens, by these kernels alone then: 69 us, 120 with both).
  plan.few = (N * G <= S * kFewTile || S > 8) && G <= kFewTile && plan.key_room <= kMostScores / (N * Hq);
  plan.many = !plan.few || longest * G > kFewTile;
  plan.narrow = N * G <= S * 16;
  if (plan.few) {
    // Ranges of 1024 keys, fewer where that leaves CUs without one.
    plan.range = kMostRange;
    while (plan.range > 4 * kFewTile && S * Hkv * ((keys + plan.range - 1) / plan.range) < 4 * kCus) plan.range /= 2;
    plan.ranges = (keys + plan.range - 1) / plan.range;
    // Beside longer sequences, room for the tokens that these can have, however many the longer ones do.
    const int64_t most = S * (kFewTile / G);
    plan.few_tokens = plan.many && most < N ? most : N;
    plan.score_bytes = plan.few_tokens * Hq * plan.key_room * 4;
    plan.few_stats_bytes = (plan.few_tokens * Hq * plan.ranges * 8 + 15) / 16 * 16;
  }
  if (plan.many) {
    plan.tiles = N * G / kRowsOf + (S < N ? S : N);
    // Four workgroups a CU, of at least 256 keys; or up to 24 of at least 1024, which even out what a chunk's tiles
    // see.  (4096 tokens over 32768 keys, 28/4 heads: 2307 us with four alone, 2132; with more parts of rows below
    // too, 16384 over themselves, 32/8 heads, 3327 and 2451, 4096 292 and 227.)
    const int64_t tiles = plan.tiles * Hkv > 0 ? plan.tiles * Hkv : 1;
    int64_t parts = 4 * kCus / tiles, more = 24 * kCus / tiles;
    if (parts > (keys + 255) / 256) parts = (keys + 255) / 256;
    if (more > keys / 1024) more = keys / 1024;
    if (parts < more) parts = more;
    if (parts > 64) parts = 64;
    plan.parts = parts < 1 ? 1 : parts;
    plan.many_bytes = (N * Hq * plan.parts * 8 + 15) / 16 * 16;
    // Two workgroups a CU, of at least 256 rows, or up to twelve of at least 2048 on average.  (2048 tokens over
    // themselves, 28/4 heads: 84 us, with whole tiles 497; 1000 over 3000 keys, 8/2 heads: 48 and 154.)
    const int64_t key_tiles = S * ((keys + kRowsOf - 1) / kRowsOf) * Hkv;
    const int64_t each = key_tiles > 0 ? key_tiles : 1;
    plan.row_parts = 2 * kCus / each;
    if (plan.row_parts > longest * G / 256) plan.row_parts = longest * G / 256;
    int64_t more_rows = 12 * kCus / each;
    if (more_rows > N * G / S / 2048) more_rows = N * G / S / 2048;
    if (plan.row_parts < more_rows) plan.row_parts = more_rows;
    if (plan.row_parts > 16) plan.row_parts = 16;
    if (plan.row_parts < 1) plan.row_parts = 1;
    if (plan.row_parts > 1) plan.partial_bytes = key_tiles * plan.row_parts * kRowsOf * 4;
  }
  return plan;
}

}  // namespace
}  // namespace spruce

using namespace spruce;

extern "C" int64_t spruce_paged_key_mass_workspace_bytes(int64_t N, int64_t S, int64_t Hq, int64_t Hkv, int64_t keys) {
  if (N < 1 || S < 1 || Hkv < 1 || Hq < Hkv || N >= (int64_t)1 << 30 || S >= (int64_t)1 << 20 || Hq >= 1 << 16 || keys < 0 ||
      keys >= (int64_t)1 << 31)
    return 0;
  return mass_plan(N, S, Hq, Hkv, keys).bytes();
}

extern "C" int spruce_paged_key_mass(const spruce_paged_key_mass_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_paged_key_mass_args& a = *args;
  const int64_t N = a.N, S = a.S, Hq = a.Hq, Hkv = a.Hkv, D = a.D;
  const int dtype = (int)a.dtype;
  const float scale = (float)a.scale;
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(dtype == SPRUCE_DTYPE_BF16 || dtype == SPRUCE_DTYPE_F16,
                 "the key mass takes bf16 or f16, got dtype code %d", dtype);
  SPRUCE_REQUIRE(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq < 1 << 16,
                 "query heads (%lld) must be divisible by KV heads (%lld)", (long long)Hq, (long long)Hkv);
  SPRUCE_REQUIRE(Hq / Hkv <= 64, "at most 64 query heads per KV head are supported");
  const float cs = scale * 1.4426950408889634f;  // of exp2
  // (The logarithm of a sum over scale log2 e must be finite.)
  SPRUCE_REQUIRE(scale >= 0x1p-100f && cs < INFINITY, "scale must be at least 2^-100, and finite times log2(e)");
  SPRUCE_REQUIRE(a.qs[2] == 1 && a.kps[3] == 1, "q and the pages must have a contiguous final dimension");
  KeyMass m{};
  const int rc = prepare_batch(m.a.batch, a.page_table, a.table_stride, a.table_width, a.q_starts, a.kv_lens, S, N,
                               a.page_size, a.pages);
  if (rc) return rc;
  if (N == 0 || a.pages == 0 || m.a.batch.cap == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(a.q && a.k_pages && a.mass_pages, "q and the pages must be non-null device pointers");
  auto rows16 = [](const void* ptr, const int64_t* s, int n) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return false;
    for (int i = 0; i < n; ++i)
      if (s[i] % 8) return false;
    return true;
  };
  SPRUCE_REQUIRE(rows16(a.q, a.qs, 2) && rows16(a.k_pages, a.kps, 3),
                 "q and the pages must be 16-byte aligned with strides that keep rows 16-byte aligned");
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.mass_pages) % 4 == 0, "mass_pages must be 4-byte aligned");
  const int64_t sizes[3] = {a.pages, Hkv, a.page_size};
  SPRUCE_REQUIRE(rows_apart(a.mps, sizes, 3, 1), "the values of mass_pages overlap");
  const MassPlan plan = mass_plan(N, S, Hq, Hkv, m.a.batch.cap);
  const int64_t need = plan.bytes();
  SPRUCE_REQUIRE(a.workspace && a.workspace_bytes >= need, "workspace too small: %lld bytes, need %lld",
                 (long long)a.workspace_bytes, (long long)need);
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace must be 16-byte aligned");
  SPRUCE_REQUIRE(N * (Hq / Hkv) < (int64_t)1 << 28 && plan.tiles < (int64_t)1 << 23, "too many tokens for one call");
  m.a.q = a.q;
  m.a.k = a.k_pages;
  m.a.qs[0] = a.qs[0];
  m.a.qs[1] = a.qs[1];
  for (int i = 0; i < 3; ++i) {
    m.a.ks[i] = a.kps[i];
    m.ms[i] = a.mps[i];
  }
  m.a.Hkv = (int)Hkv;
  m.a.G = (int)(Hq / Hkv);
  m.a.by_heads = divisor(Hkv);
  m.a.by_group = divisor(Hq / Hkv);
  m.a.cs = cs;
  m.a.few_limit = plan.few ? kFewTile : -1;
  m.mass = a.mass_pages;
  m.Hq = (int)Hq;
  m.accumulate = a.accumulate != 0;
  char* work = static_cast<char*>(a.workspace);
  m.stats = reinterpret_cast<float2*>(work);
  m.parts = (int)plan.parts;
  m.row_parts = (int)plan.row_parts;
  m.partial = reinterpret_cast<float*>(work += plan.many_bytes);
  m.few_stats = reinterpret_cast<float2*>(work += plan.partial_bytes);
  m.scores = reinterpret_cast<float*>(work += plan.few_stats_bytes);
  m.few_rows = plan.many ? kFewTile : 0x7fffffff;
  m.range = (int)plan.range;
  m.ranges = (int)plan.ranges;
  m.key_room = (int)plan.key_room;
  m.few_tokens = (int)plan.few_tokens;
  m.cs_low = (float)(a.scale * 1.44269504088896340736 - (double)cs);
  const hipStream_t st = (hipStream_t)stream;
  const int64_t units = plan.tiles * plan.parts * Hkv;
  SPRUCE_REQUIRE(units < (int64_t)1 << 31, "too many tokens for one call");
  // Workgroups take more than one unit where there are more.
  auto grid = [&](int64_t keys, int64_t most, int64_t times = 1) {
    const int64_t all = S * ((m.a.batch.cap + keys - 1) / keys) * Hkv * times;
    return dim3((unsigned)(all < most ? all : most));
  };
#define SPRUCE_KEY_MASS(D_, F16_)                                                                              \
  do {                                                                                                         \
    if (plan.many) {                                                                                           \
      if (a.page_size % Stream<D_>::rows == 0)                                                                 \
        hipLaunchKernelGGL((key_mass_rows_kernel<D_, F16_, true>), flat_grid(units), dim3(256), 0, st, m);     \
      else                                                                                                     \
        hipLaunchKernelGGL((key_mass_rows_kernel<D_, F16_, false>), flat_grid(units), dim3(256), 0, st, m);    \
      if (plan.parts > 1)                                                                                      \
        hipLaunchKernelGGL(key_mass_join_kernel, flat_grid((N * Hq + 255) / 256), dim3(256), 0, st, m.stats,   \
                           N * Hq, m.parts, cs);                                                               \
      hipLaunchKernelGGL((key_mass_keys_kernel<D_, F16_>), grid(kRowsOf, 8 * kCus, plan.row_parts), dim3(256), \
                         0, st, m);                                                                            \
      if (plan.row_parts > 1)                                                                                  \
        hipLaunchKernelGGL(key_mass_add_kernel, grid(kRowsOf, 8 * kCus), dim3(256), 0, st, m);                 \
    }                                                                                                          \
    if (plan.few && plan.narrow)                                                                               \
      hipLaunchKernelGGL((key_scores_kernel<D_, F16_, 16>), grid(plan.range, 16 * kCus), dim3(256), 0, st, m); \
    else if (plan.few)                                                                                         \
      hipLaunchKernelGGL((key_scores_kernel<D_, F16_, 32>), grid(plan.range, 16 * kCus), dim3(256), 0, st, m); \
  } while (0)
  if (D == 128) {
    if (dtype == SPRUCE_DTYPE_F16) SPRUCE_KEY_MASS(128, true);
    else SPRUCE_KEY_MASS(128, false);
  } else {
    if (dtype == SPRUCE_DTYPE_F16) SPRUCE_KEY_MASS(64, true);
    else SPRUCE_KEY_MASS(64, false);
  }
#undef SPRUCE_KEY_MASS
  if (plan.few) hipLaunchKernelGGL(key_weights_kernel, grid(kWeightKeys, 16 * kCus), dim3(256), 0, st, m);
  return check_launch("paged key mass");
}
