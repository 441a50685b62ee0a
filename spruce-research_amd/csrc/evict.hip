// Eviction from a paged K/V cache: of every sequence and KV head the first and
// the most recent positions and, of those between, the ones with the largest
// masses are kept (`keep` in all, ties to the lowest position), and their rows
// move in order into other pages.
//
// Two steps: one workgroup per (sequence, KV head) finds the smallest mass that
// is kept, digit by digit from the top (a histogram of 11, 11 and 10 bits of
// the masses' bits, ordered as numbers), and writes the kept positions in order;
// then the rows move, 16 bytes a lane.
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

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const Evict e) {
  __shared__ uint32_t hist[2048];
  __shared__ int wave_sum[kSelectWaves], found[2], counts[2][kSelectWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int g = (int)(flat_block() % (uint32_t)e.Hkv), s = (int)(flat_block() / (uint32_t)e.Hkv);
  if (s >= e.batch.S) return;
  const int len = kept_length(e.batch, s);
  int32_t* kept = e.kept + ((int64_t)s * e.Hkv + g) * e.keep;
  const int new_len = len < e.keep ? len : e.keep;
  if (g == 0 && tid == 0) e.new_lens[s] = new_len;
  if (len <= e.keep) {
    for (int i = tid; i < e.keep; i += kSelectThreads) kept[i] = i < len ? i : -1;
    return;
  }
  const int begin = e.first, n = len - e.recent - begin;  // the positions to choose from
  int need = e.keep - e.first - e.recent;
  for (int i = tid; i < e.first; i += kSelectThreads) kept[i] = i;
  for (int i = tid; i < e.recent; i += kSelectThreads) kept[e.keep - e.recent + i] = len - e.recent + i;
  if (need == 0) return;
  auto key_of = [&](int i) {
    const int pos = begin + i, entry = page_entry(e.batch, s, pos);
    if (!is_page(e.batch, entry)) return kLowest;
    const int slot = pos - page_of(e.batch, pos) * e.batch.page;
    return order_of(e.mass[(int64_t)entry * e.ms[0] + (int64_t)g * e.ms[1] + (int64_t)slot * e.ms[2]]);
  };

  uint32_t prefix = 0, mask = 0;
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : (level == 1 ? 10 : 0), bins = level == 2 ? 1024 : 2048;
    hist[tid] = 0;
    hist[tid + 1024] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < n; i += kSelectThreads) {
      const uint32_t key = key_of(i);
      if ((key & mask) == prefix) atomicAdd(&hist[key >> shift & (bins - 1)], 1u);
    }
    __syncthreads();
    // From the top: the bin within which the need-th lies.
    const int top = 2047 - 2 * tid;
    const int c0 = (int)hist[top], c1 = (int)hist[top - 1];
    const int upto = wave_prefix(c0 + c1);
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    int above = upto - c0 - c1;
    for (int w = 0; w < wave; ++w) above += wave_sum[w];
    if (above < need && need <= above + c0 + c1) {
      const bool second = need > above + c0;
      found[0] = top - (second ? 1 : 0);
      found[1] = need - above - (second ? c0 : 0);
    }
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    need = found[1];
  }
  // Larger masses than `prefix` are kept, and the first `need` equal ones.  Every wave has a run of positions.
  const int run = (((n + kSelectWaves - 1) / kSelectWaves) + 63) & ~63;
  const int lo = wave * run < n ? wave * run : n, hi = lo + run < n ? lo + run : n;
  int larger = 0, equal = 0;
  for (int i = lo; i < hi; i += 64) {
    const uint32_t key = i + lane < hi ? key_of(i + lane) : 0;
    larger += __builtin_popcountll(__ballot(i + lane < hi && key > prefix));
    equal += __builtin_popcountll(__ballot(i + lane < hi && key == prefix));
  }
  if (lane == 0) {
    counts[0][wave] = larger;
    counts[1][wave] = equal;
  }
  __syncthreads();
  larger = equal = 0;
  for (int w = 0; w < wave; ++w) {
    larger += counts[0][w];
    equal += counts[1][w];
  }
  for (int i = lo; i < hi; i += 64) {
    const uint32_t key = i + lane < hi ? key_of(i + lane) : 0;
    const uint64_t is_larger = __ballot(i + lane < hi && key > prefix), is_equal = __ballot(i + lane < hi && key == prefix);
    const uint64_t below = (1ull << lane) - 1;
    const int eq = equal + __builtin_popcountll(is_equal & below);
    const bool take = (is_larger >> lane & 1) || ((is_equal >> lane & 1) && eq < need);
    if (take)
      kept[e.first + larger + __builtin_popcountll(is_larger & below) + (eq < need ? eq : need)] = begin + i + lane;
    larger += __builtin_popcountll(is_larger);
    equal += __builtin_popcountll(is_equal);
  }
}

// Rows of ROW bytes: a workgroup moves kMoveRows of one (sequence, KV head).
constexpr int kMoveRows = 32;
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
    kx[i] = *reinterpret_cast<const u32x4*>(e.k + (int64_t)entry * e.ks[0] + (int64_t)g * e.ks[1] +
                                            (int64_t)slot * e.ks[2] + 16 * lc);
    vx[i] = *reinterpret_cast<const u32x4*>(e.v + (int64_t)entry * e.vs[0] + (int64_t)g * e.vs[1] +
                                            (int64_t)slot * e.vs[2] + 16 * lc);
    if (lc == 0) m[i] = e.mass[(int64_t)entry * e.ms[0] + (int64_t)g * e.ms[1] + (int64_t)slot * e.ms[2]];
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    if (to[i] < 0) continue;
    const int64_t out = to[i] >> 32, slot = (uint32_t)to[i];
    *reinterpret_cast<u32x4*>(e.ko + out * e.ks[0] + (int64_t)g * e.ks[1] + slot * e.ks[2] + 16 * lc) = kx[i];
    *reinterpret_cast<u32x4*>(e.vo + out * e.vs[0] + (int64_t)g * e.vs[1] + slot * e.vs[2] + 16 * lc) = vx[i];
    if (lc == 0) e.mass[out * e.ms[0] + (int64_t)g * e.ms[1] + slot * e.ms[2]] = m[i];
  }
}

}  // namespace
}  // namespace spruce

using namespace spruce;

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
  e.Hkv = (int)Hkv;
  e.keep = (int)a.keep;
  e.first = (int)a.first;
  e.recent = (int)a.recent;
  e.kept = a.kept;
  e.new_lens = a.new_lens;
  // No sequence keeps more than the table holds.
  const int64_t rows = a.keep < e.batch.cap ? a.keep : e.batch.cap, tiles = (rows + kMoveRows - 1) / kMoveRows;
  SPRUCE_REQUIRE(S * Hkv < (int64_t)1 << 31 && S * Hkv * tiles < (int64_t)1 << 31, "too many rows for one call");
  const hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(evict_select_kernel, flat_grid(S * Hkv), dim3(kSelectThreads), 0, st, e);
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
