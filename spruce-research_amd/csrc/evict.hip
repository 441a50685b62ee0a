// Eviction from a paged K/V cache: of every sequence and KV head the first and
// the most recent positions and, of those between, the ones with the largest
// masses are kept (`keep` in all, ties to the lowest position), and their rows
// move in order into other pages.
//
// The smallest mass that is kept is found digit by digit from the top: histograms of 11, 11
// and 10 bits of the masses' bits, ordered as numbers.  Where a table has no more
// than 32768 positions, one workgroup holds the masses in registers, does all of it, and
// writes the kept positions in order (read again for every digit, 64 sequences of up to 16384 took 48 us of
// selection, 19 held).  Longer ones are shared out: the first
// histogram part by part, the members of the bin that holds the end listed, and the end found
// among these by one workgroup.  Then the rows move, 16 bytes a lane.
#include "paged_impl.h"

namespace spruce {

struct Evict {
  PagedBatch batch;  // (no new tokens)
  const int32_t* out_table;
  int64_t out_stride;
  int out_cap;
  const char* k;
  const char* v;
  char* ko;
  char* vo;
  int64_t ks[3], vs[3];  // page, head, slot strides in bytes
  float* mass;
  int64_t ms[3];
  int Hkv, keep, first, recent;
  int32_t* kept;      // [S, Hkv, keep]
  int32_t* new_lens;  // [S]
  // Of long tables, per (sequence, KV head): masses by part, those within the first digit's bin,
  // and the first digit's histogram.
  int parts;
  uint32_t* keys;
  uint32_t* listed;
  uint32_t* hists;     // [parts][2048]
  struct EvictPart* part_of;
  struct EvictEnd* end_of;
};
struct EvictPart {
  int larger, listed;                // masses in higher bins, and in the end's
  int larger_before, equal_before;   // than the end's, in the parts before
};
struct EvictEnd {
  uint32_t bin, key;
  int need, unused;  // of the bin's; then of those equal to key
};

namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

__device__ __forceinline__ int kept_length(const PagedBatch& b, int s) {
  const int len = b.kv_lens[s];
  return len < 0 ? 0 : (len < b.cap ? len : b.cap);
}

// A mass as a number to compare: ascending, both zeros alike, NaN and what has no page the lowest.
constexpr uint32_t kLowest = 0x007fffffu;  // -inf's
__device__ __forceinline__ uint32_t order_of(float x) {
  if (!(x == x)) return kLowest;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// That one workgroup holds.  (In parts, and held: a head of 20000 positions 28 us and 25, 64 sequences of them, 8 heads,
// 90 and 61, 64 of 32768, 4 heads, 69 and 45, but 8 heads of 32768 31 and 33.)
constexpr int kWholeKeys = 32 * kSelectThreads;
// Of a longer table, in parts.  (One sequence of 131072 positions, 4 heads, with the kernels of that stage: 65 us in
// all, with twice as many a part 70, half as many 72; 54 to 57 now.)
constexpr int kPartKeys = 8 * kSelectThreads;

// What a (sequence, KV head) has to choose from.
struct Choice {
  int s, g, len, begin, n, need;  // positions begin .. begin + n - 1, of which `need` are kept
  int32_t* kept;
};
// False where everything, or nothing of the middle, is kept; the kept positions are then written by
// `part` 0, as are those outside of the middle.
__device__ __forceinline__ bool choose(const Evict& e, uint32_t pair, int part, Choice& c) {
  const int tid = threadIdx.x;
  c.g = (int)(pair % (uint32_t)e.Hkv);
  c.s = (int)(pair / (uint32_t)e.Hkv);
  c.len = kept_length(e.batch, c.s);
  c.kept = e.kept + ((int64_t)c.s * e.Hkv + c.g) * e.keep;
  c.begin = e.first;
  c.n = c.len - e.recent - e.first;
  c.need = e.keep - e.first - e.recent;
  const bool all = c.len <= e.keep;
  if (part == 0) {
    if (c.g == 0 && tid == 0) e.new_lens[c.s] = all ? c.len : e.keep;
    if (all) {
      for (int i = tid; i < e.keep; i += kSelectThreads) c.kept[i] = i < c.len ? i : -1;
    } else {
      for (int i = tid; i < e.first; i += kSelectThreads) c.kept[i] = i;
      for (int i = tid; i < e.recent; i += kSelectThreads) c.kept[e.keep - e.recent + i] = c.len - e.recent + i;
    }
  }
  return !all && c.need > 0;
}

// A workgroup's masses, 1024 neighbours at a time: key[i] is position from + 1024 i + thread's.
template <int E>
__device__ __forceinline__ void load_keys(const Evict& e, const Choice& c, int from, uint32_t (&key)[E]) {
  int entry[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int at = from + i * kSelectThreads + (int)threadIdx.x;
    entry[i] = page_entry(e.batch, c.s, c.begin + nearest(at, c.n));
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int pos = c.begin + nearest(from + i * kSelectThreads + (int)threadIdx.x, c.n);
    const int slot = pos - page_of(e.batch, pos) * e.batch.page;
    const bool ok = is_page(e.batch, entry[i]);
    const float m = e.mass[(int64_t)(ok ? entry[i] : 0) * e.ms[0] + (int64_t)c.g * e.ms[1] + (int64_t)slot * e.ms[2]];
    key[i] = ok ? order_of(m) : kLowest;
  }
}

struct SelectLds {
  uint32_t hist[2048];
  uint32_t waves[kSelectWaves];
  uint32_t found[2];
  uint32_t counts[kWholeKeys / 64];
};

// From the top: the bin of the histogram within which the need-th lies; need goes on to its place there.
__device__ __forceinline__ uint32_t find_digit(SelectLds& sh, int& need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int top = 2047 - 2 * tid;
  const int c0 = (int)sh.hist[top], c1 = (int)sh.hist[top - 1];
  const int upto = wave_prefix(c0 + c1);
  if (lane == 63) sh.waves[wave] = (uint32_t)upto;
  __syncthreads();
  int above = upto - c0 - c1;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) above += w < wave ? (int)sh.waves[w] : 0;
  if (above < need && need <= above + c0 + c1) {
    const bool second = need > above + c0;
    sh.found[0] = (uint32_t)(top - (second ? 1 : 0));
    sh.found[1] = (uint32_t)(need - above - (second ? c0 : 0));
  }
  __syncthreads();
  need = (int)sh.found[1];
  return sh.found[0];
}
__device__ __forceinline__ void clear_hist(SelectLds& sh) {
  sh.hist[threadIdx.x] = 0;
  sh.hist[threadIdx.x + 1024] = 0;
  __syncthreads();
}
constexpr int kShift[3] = {21, 10, 0};

// Writes the kept ones of a workgroup's masses: all above `end`, and the equal ones as long as `need`
// are not yet taken; larger and equal ones come before, in other parts.
template <int E>
__device__ __forceinline__ void write_kept(SelectLds& sh, const Evict& e, const Choice& c, int from,
                                           const uint32_t (&key)[E], uint32_t end, int need, int larger, int equal) {
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  uint64_t is_larger[E], is_equal[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const bool in = from + i * kSelectThreads + tid < c.n;
    is_larger[i] = __ballot(in && key[i] > end);
    is_equal[i] = __ballot(in && key[i] == end);
    if (lane == 0)
      sh.counts[i * kSelectWaves + wave] =
          (uint32_t)__builtin_popcountll(is_larger[i]) | (uint32_t)__builtin_popcountll(is_equal[i]) << 16;
  }
  __syncthreads();
  if (wave == 0) {
    // Sums before each 64 of them: E / 4 a lane.  (Up to 32768 of either, so the halves hold.)
    constexpr int EACH = E * kSelectWaves / 64;
    uint32_t v[EACH], mine = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      v[i] = sh.counts[lane * EACH + i];
      mine += v[i];
    }
    uint32_t upto = (uint32_t)wave_prefix((int)mine) - mine;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      sh.counts[lane * EACH + i] = upto;
      upto += v[i];
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const uint32_t before = sh.counts[i * kSelectWaves + wave];
    const int lg = larger + (int)(before & 0xffffu) + __builtin_popcountll(is_larger[i] & below);
    const int eq = equal + (int)(before >> 16) + __builtin_popcountll(is_equal[i] & below);
    if ((is_larger[i] >> lane & 1) || ((is_equal[i] >> lane & 1) && eq < need))
      c.kept[c.begin + lg + (eq < need ? eq : need)] = c.begin + from + i * kSelectThreads + tid;
  }
}

// A table of up to E * 1024 positions.
template <int E>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const Evict e) {
  __shared__ SelectLds sh;
  Choice c;
  if (!choose(e, blockIdx.x, 0, c)) return;
  const int tid = threadIdx.x;
  uint32_t key[E];
  load_keys<E>(e, c, 0, key);
  uint32_t prefix = 0, mask = 0;
  int need = c.need;
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? kShift[0] : (level == 1 ? kShift[1] : kShift[2]);
    const uint32_t bits = level == 2 ? 1023u : 2047u;
    clear_hist(sh);
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i * kSelectThreads + tid < c.n && (key[i] & mask) == prefix) atomicAdd(&sh.hist[key[i] >> shift & bits], 1u);
    __syncthreads();
    prefix |= find_digit(sh, need) << shift;
    mask |= bits << shift;
  }
  write_kept<E>(sh, e, c, 0, key, prefix, need, 0, 0);
}

// Longer tables, part by part: the masses in order of position, and the first digit's histogram.
__global__ __launch_bounds__(kSelectThreads) void evict_count_kernel(const Evict e) {
  constexpr int E = kPartKeys / kSelectThreads;
  __shared__ SelectLds sh;
  const uint32_t pair = flat_block() / (uint32_t)e.parts;
  const int part = (int)(flat_block() % (uint32_t)e.parts), tid = threadIdx.x;
  Choice c;
  if (pair >= (uint32_t)(e.batch.S * e.Hkv) || !choose(e, pair, part, c) || part * kPartKeys >= c.n) return;
  uint32_t key[E];
  load_keys<E>(e, c, part * kPartKeys, key);
  clear_hist(sh);
  uint32_t* keys = e.keys + ((int64_t)pair * e.parts + part) * kPartKeys;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    keys[i * kSelectThreads + tid] = key[i];
    if (part * kPartKeys + i * kSelectThreads + tid < c.n) atomicAdd(&sh.hist[key[i] >> kShift[0]], 1u);
  }
  __syncthreads();
  uint32_t* hist = e.hists + ((int64_t)pair * e.parts + part) * 2048;
  hist[tid] = sh.hist[tid];
  hist[tid + 1024] = sh.hist[tid + 1024];
}

// The members of the bin that holds the end, listed part by part.
__global__ __launch_bounds__(kSelectThreads) void evict_list_kernel(const Evict e) {
  constexpr int E = kPartKeys / kSelectThreads;
  __shared__ SelectLds sh;
  __shared__ int larger, listed;
  const uint32_t pair = flat_block() / (uint32_t)e.parts;
  const int part = (int)(flat_block() % (uint32_t)e.parts), tid = threadIdx.x;
  Choice c;
  if (pair >= (uint32_t)(e.batch.S * e.Hkv) || !choose(e, pair, 1, c) || part * kPartKeys >= c.n) return;
  const int parts = (c.n + kPartKeys - 1) / kPartKeys;
  const uint32_t* hists = e.hists + (int64_t)pair * e.parts * 2048;
  uint32_t a = 0, b = 0;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    a += hists[(int64_t)i * 2048 + tid];
    b += hists[(int64_t)i * 2048 + tid + 1024];
  }
  sh.hist[tid] = a;
  sh.hist[tid + 1024] = b;
  if (tid == 0) larger = listed = 0;
  __syncthreads();
  int need = c.need;
  const uint32_t bin = find_digit(sh, need);
  const int64_t at = ((int64_t)pair * e.parts + part) * kPartKeys;
  int mine = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (part * kPartKeys + i * kSelectThreads + tid >= c.n) continue;
    const uint32_t key = e.keys[at + i * kSelectThreads + tid];
    mine += key >> kShift[0] > bin;
    if (key >> kShift[0] == bin) e.listed[at + atomicAdd(&listed, 1)] = key;  // in any order: they are counted
  }
  mine = wave_prefix(mine);
  if ((tid & 63) == 63) atomicAdd(&larger, mine);
  __syncthreads();
  if (tid == 0) {
    e.part_of[(int64_t)pair * e.parts + part] = EvictPart{larger, listed, 0, 0};
    if (part == 0) e.end_of[pair] = EvictEnd{bin, 0, need, 0};
  }
}

// The end among the listed, and what of each part is before it.
__global__ __launch_bounds__(kSelectThreads) void evict_end_kernel(const Evict e) {
  __shared__ SelectLds sh;
  const uint32_t pair = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Choice c;
  if (!choose(e, pair, 1, c)) return;
  const int parts = (c.n + kPartKeys - 1) / kPartKeys;
  EvictPart* part_of = e.part_of + (int64_t)pair * e.parts;
  const uint32_t* listed = e.listed + (int64_t)pair * e.parts * kPartKeys;
  uint32_t prefix = e.end_of[pair].bin << kShift[0], mask = 2047u << kShift[0];
  int need = e.end_of[pair].need;
#pragma unroll 1
  for (int level = 1; level < 3; ++level) {
    const int shift = level == 1 ? kShift[1] : kShift[2];
    const uint32_t bits = level == 2 ? 1023u : 2047u;
    clear_hist(sh);
    for (int p = wave; p < parts; p += kSelectWaves) {
      const int n = part_of[p].listed;
#pragma unroll 4
      for (int i = lane; i < n; i += 64) {
        const uint32_t key = listed[(int64_t)p * kPartKeys + i];
        if ((key & mask) == prefix) atomicAdd(&sh.hist[key >> shift & bits], 1u);
      }
    }
    __syncthreads();
    prefix |= find_digit(sh, need) << shift;
    mask |= bits << shift;
  }
  for (int p = wave; p < parts; p += kSelectWaves) {
    int larger = 0, equal = 0;
    const int n = part_of[p].listed;
#pragma unroll 4
    for (int i = lane; i < n; i += 64) {
      const uint32_t key = listed[(int64_t)p * kPartKeys + i];
      larger += key > prefix;
      equal += key == prefix;
    }
    larger = wave_prefix(larger);
    equal = wave_prefix(equal);
    if (lane == 63) {
      part_of[p].larger_before = larger + part_of[p].larger;
      part_of[p].equal_before = equal;
    }
  }
  __threadfence_block();
  __syncthreads();
  if (wave == 0) {
    int larger = 0, equal = 0;
    for (int p0 = 0; p0 < parts; p0 += 64) {
      const int p = p0 + lane;
      const int lg = p < parts ? part_of[p].larger_before : 0, eq = p < parts ? part_of[p].equal_before : 0;
      const int upto_lg = wave_prefix(lg), upto_eq = wave_prefix(eq);
      if (p < parts) {
        part_of[p].larger_before = larger + upto_lg - lg;
        part_of[p].equal_before = equal + upto_eq - eq;
      }
      larger += __builtin_amdgcn_readlane(upto_lg, 63);
      equal += __builtin_amdgcn_readlane(upto_eq, 63);
    }
  }
  if (tid == 0) {
    e.end_of[pair].key = prefix;
    e.end_of[pair].need = need;
  }
}

__global__ __launch_bounds__(kSelectThreads) void evict_write_kernel(const Evict e) {
  constexpr int E = kPartKeys / kSelectThreads;
  __shared__ SelectLds sh;
  const uint32_t pair = flat_block() / (uint32_t)e.parts;
  const int part = (int)(flat_block() % (uint32_t)e.parts), tid = threadIdx.x;
  Choice c;
  if (pair >= (uint32_t)(e.batch.S * e.Hkv) || !choose(e, pair, 1, c) || part * kPartKeys >= c.n) return;
  uint32_t key[E];
  const uint32_t* keys = e.keys + ((int64_t)pair * e.parts + part) * kPartKeys;
#pragma unroll
  for (int i = 0; i < E; ++i) key[i] = keys[i * kSelectThreads + tid];
  const EvictEnd end = e.end_of[pair];
  const EvictPart p = e.part_of[(int64_t)pair * e.parts + part];
  write_kept<E>(sh, e, c, part * kPartKeys, key, end.key, end.need, p.larger_before, p.equal_before);
}

// Rows of ROW bytes: a workgroup moves kMoveRows of one (sequence, KV head).  HBM bounds it, and rows are
// used once: past the caches 243 us in all for 64 sequences that keep 4096, 256 through them (32 rows a
// workgroup: 246; on a faster card 206).
constexpr int kMoveRows = 16;
template <int ROW>
__global__ __launch_bounds__(256) void evict_move_kernel(const Evict e, int tiles) {
  constexpr int LANES = ROW / 16, ROWS = 256 / LANES, PASSES = (kMoveRows + ROWS - 1) / ROWS;
  const uint32_t block = flat_block();
  const int g = (int)(block % (uint32_t)e.Hkv);
  const uint32_t rest = block / (uint32_t)e.Hkv;
  const int tile = (int)(rest % (uint32_t)tiles), s = (int)(rest / (uint32_t)tiles);
  if (s >= e.batch.S) return;
  const int lr = threadIdx.x / LANES, lc = threadIdx.x % LANES;
  const int32_t* kept = e.kept + ((int64_t)s * e.Hkv + g) * e.keep;
  u32x4 kx[PASSES], vx[PASSES];
  float m[PASSES];
  int64_t to[PASSES];  // page, and slot below; -1: nothing to move
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = tile * kMoveRows + i * ROWS + lr;
    to[i] = -1;
    const int pos = r < e.keep && i * ROWS + lr < kMoveRows ? kept[r] : -1;
    if (pos < 0 || r >= e.out_cap) continue;
    const int entry = page_entry(e.batch, s, pos), out = e.out_table[(int64_t)s * e.out_stride + page_of(e.batch, r)];
    if (!is_page(e.batch, entry) || !is_page(e.batch, out)) continue;
    const int slot = pos - page_of(e.batch, pos) * e.batch.page;
    to[i] = (int64_t)out << 32 | (uint32_t)(r - page_of(e.batch, r) * e.batch.page);
    kx[i] = load16_once(reinterpret_cast<const uint16_t*>(e.k + (int64_t)entry * e.ks[0] + (int64_t)g * e.ks[1] +
                                                          (int64_t)slot * e.ks[2] + 16 * lc));
    vx[i] = load16_once(reinterpret_cast<const uint16_t*>(e.v + (int64_t)entry * e.vs[0] + (int64_t)g * e.vs[1] +
                                                          (int64_t)slot * e.vs[2] + 16 * lc));
    if (lc == 0) m[i] = e.mass[(int64_t)entry * e.ms[0] + (int64_t)g * e.ms[1] + (int64_t)slot * e.ms[2]];
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (to[i] < 0) continue;
    const int64_t out = to[i] >> 32, slot = (uint32_t)to[i];
    __builtin_nontemporal_store(
        kx[i], reinterpret_cast<u32x4*>(e.ko + out * e.ks[0] + (int64_t)g * e.ks[1] + slot * e.ks[2] + 16 * lc));
    __builtin_nontemporal_store(
        vx[i], reinterpret_cast<u32x4*>(e.vo + out * e.vs[0] + (int64_t)g * e.vs[1] + slot * e.vs[2] + 16 * lc));
    if (lc == 0) e.mass[out * e.ms[0] + (int64_t)g * e.ms[1] + slot * e.ms[2]] = m[i];
  }
}

}  // namespace
}  // namespace spruce

using namespace spruce;

namespace {

// Of tables that one workgroup does not hold.
struct EvictPlan {
  int64_t parts, keys, hists, part_of, end_of;
  int64_t bytes() const { return 2 * keys + hists + part_of + end_of; }
};
EvictPlan evict_plan(int64_t S, int64_t Hkv, int64_t cap) {
  EvictPlan p{};
  if (cap <= kWholeKeys) return p;
  p.parts = (cap + kPartKeys - 1) / kPartKeys;
  const int64_t all = S * Hkv * p.parts;
  p.keys = all * kPartKeys * 4;
  p.hists = all * 2048 * 4;
  p.part_of = all * (int64_t)sizeof(EvictPart);
  p.end_of = S * Hkv * (int64_t)sizeof(EvictEnd);
  return p;
}

}  // namespace

extern "C" int64_t spruce_paged_evict_workspace_bytes(int64_t S, int64_t Hkv, int64_t keys) {
  if (S < 1 || Hkv < 1 || keys < 0 || S >= (int64_t)1 << 20 || Hkv >= 1 << 16 || keys >= (int64_t)1 << 31) return 0;
  return evict_plan(S, Hkv, keys).bytes();
}

extern "C" int spruce_paged_evict(const spruce_paged_evict_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_paged_evict_args& a = *args;
  const int64_t S = a.S, Hkv = a.Hkv, D = a.D;
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "unsupported dtype code %lld", (long long)a.dtype);
  SPRUCE_REQUIRE(Hkv >= 1 && Hkv < 1 << 16, "invalid KV head count %lld", (long long)Hkv);
  SPRUCE_REQUIRE(a.keep >= 1 && a.keep < (int64_t)1 << 30, "keep must be in [1, 2^30), got %lld", (long long)a.keep);
  SPRUCE_REQUIRE(a.first >= 0 && a.recent >= 0 && a.first <= a.keep && a.recent <= a.keep - a.first,
                 "first (%lld) and recent (%lld) must not be negative or together above keep (%lld)", (long long)a.first,
                 (long long)a.recent, (long long)a.keep);
  SPRUCE_REQUIRE(a.kps[3] == 1 && a.vps[3] == 1, "the pages must have a contiguous final dimension");
  Evict e{};
  // (No packed rows: what stands for q_starts is not read.)
  const int rc = prepare_batch(e.batch, a.page_table, a.table_stride, a.table_width, a.kv_lens, a.kv_lens, S, 0,
                               a.page_size, a.pages);
  if (rc) return rc;
  const int64_t width = (a.keep + a.page_size - 1) / a.page_size, most = width < a.table_width ? width : a.table_width;
  SPRUCE_REQUIRE(a.out_width >= most, "out_table must hold keep positions: %lld pages, need %lld", (long long)a.out_width,
                 (long long)most);
  SPRUCE_REQUIRE(a.out_table || a.out_width == 0, "out_table must be a non-null device pointer");
  SPRUCE_REQUIRE(S == 1 || a.out_stride >= a.out_width, "out_table rows (%lld) overlap (stride %lld)",
                 (long long)a.out_width, (long long)a.out_stride);
  SPRUCE_REQUIRE(a.kept && a.new_lens, "kept and new_lens must be non-null device pointers");
  SPRUCE_REQUIRE(a.pages == 0 || (a.k_pages && a.v_pages && a.mass_pages), "the pages must be non-null device pointers");
  const int eb = a.dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  auto rows16 = [&](const void* ptr, const int64_t* s) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && s[0] * eb % 16 == 0 && s[1] * eb % 16 == 0 && s[2] * eb % 16 == 0;
  };
  SPRUCE_REQUIRE(rows16(a.k_pages, a.kps) && rows16(a.v_pages, a.vps),
                 "the pages must be 16-byte aligned with strides that keep rows 16-byte aligned");
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.mass_pages) % 4 == 0, "mass_pages must be 4-byte aligned");
  const int64_t sizes[3] = {a.pages, Hkv, a.page_size};
  SPRUCE_REQUIRE(rows_apart(a.kps, sizes, 3, D) && rows_apart(a.vps, sizes, 3, D), "the rows of the pages overlap");
  SPRUCE_REQUIRE(rows_apart(a.mps, sizes, 3, 1), "the values of mass_pages overlap");
  e.out_table = a.out_table;
  e.out_stride = a.out_stride;
  e.out_cap = (int)(a.out_width < ((int64_t)1 << 31) / a.page_size ? a.out_width * a.page_size : 0x7fffffff);
  e.k = e.ko = static_cast<char*>(a.k_pages);
  e.v = e.vo = static_cast<char*>(a.v_pages);
  for (int i = 0; i < 3; ++i) {
    e.ks[i] = a.kps[i] * eb;
    e.vs[i] = a.vps[i] * eb;
    e.ms[i] = a.mps[i];
  }
  e.mass = a.mass_pages;
  if (a.pages == 0) {  // what is read in place of masses without a page, and not used, has to be memory
    e.mass = reinterpret_cast<float*>(a.kept);
    e.ms[0] = e.ms[1] = e.ms[2] = 0;
  }
  e.Hkv = (int)Hkv;
  e.keep = (int)a.keep;
  e.first = (int)a.first;
  e.recent = (int)a.recent;
  e.kept = a.kept;
  e.new_lens = a.new_lens;
  // No sequence keeps more than the table holds.
  const int64_t rows = a.keep < e.batch.cap ? a.keep : e.batch.cap, tiles = (rows + kMoveRows - 1) / kMoveRows;
  SPRUCE_REQUIRE(S * Hkv <= kGridX && S * Hkv * tiles < (int64_t)1 << 31, "too many rows for one call");
  const EvictPlan plan = evict_plan(S, Hkv, e.batch.cap);
  SPRUCE_REQUIRE(plan.bytes() == 0 || (a.workspace && a.workspace_bytes >= plan.bytes()),
                 "workspace too small: %lld bytes, need %lld", (long long)a.workspace_bytes, (long long)plan.bytes());
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace must be 16-byte aligned");
  SPRUCE_REQUIRE(S * Hkv * plan.parts < (int64_t)1 << 31, "too many rows for one call");
  const hipStream_t st = (hipStream_t)stream;
  const dim3 pairs((unsigned)(S * Hkv));
  if (plan.parts == 0) {
    if (e.batch.cap <= 4 * kSelectThreads)
      hipLaunchKernelGGL(evict_select_kernel<4>, pairs, dim3(kSelectThreads), 0, st, e);
    else if (e.batch.cap <= 16 * kSelectThreads)
      hipLaunchKernelGGL(evict_select_kernel<16>, pairs, dim3(kSelectThreads), 0, st, e);
    else if (e.batch.cap <= 24 * kSelectThreads)
      hipLaunchKernelGGL(evict_select_kernel<24>, pairs, dim3(kSelectThreads), 0, st, e);
    else
      hipLaunchKernelGGL(evict_select_kernel<32>, pairs, dim3(kSelectThreads), 0, st, e);
  } else {
    char* work = static_cast<char*>(a.workspace);
    e.parts = (int)plan.parts;
    e.keys = reinterpret_cast<uint32_t*>(work);
    e.listed = reinterpret_cast<uint32_t*>(work += plan.keys);
    e.hists = reinterpret_cast<uint32_t*>(work += plan.keys);
    e.part_of = reinterpret_cast<EvictPart*>(work += plan.hists);
    e.end_of = reinterpret_cast<EvictEnd*>(work += plan.part_of);
    const dim3 all = flat_grid(S * Hkv * plan.parts);
    hipLaunchKernelGGL(evict_count_kernel, all, dim3(kSelectThreads), 0, st, e);
    hipLaunchKernelGGL(evict_list_kernel, all, dim3(kSelectThreads), 0, st, e);
    hipLaunchKernelGGL(evict_end_kernel, pairs, dim3(kSelectThreads), 0, st, e);
    hipLaunchKernelGGL(evict_write_kernel, all, dim3(kSelectThreads), 0, st, e);
  }
  const int rc2 = check_launch("paged eviction");
  if (rc2 || tiles == 0 || a.pages == 0) return rc2;
  const dim3 grid = flat_grid(S * Hkv * tiles);
  switch (D * eb) {
    case 128: hipLaunchKernelGGL(evict_move_kernel<128>, grid, dim3(256), 0, st, e, (int)tiles); break;
    case 256: hipLaunchKernelGGL(evict_move_kernel<256>, grid, dim3(256), 0, st, e, (int)tiles); break;
    default: hipLaunchKernelGGL(evict_move_kernel<512>, grid, dim3(256), 0, st, e, (int)tiles); break;
  }
  return check_launch("paged eviction");
}
