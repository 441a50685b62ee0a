// One token a row from logits x, given a random number u a row:
//   w_i = exp((x_i - max x) / T);
//   kept: in the order of x descending, ties by index ascending, the shortest
//   of three prefixes: the first top_k; of those the fewest whose weights reach
//   top_p of all of theirs; those with w_i >= min_p (the first one always);
//   token: the first i, by index, with sum_{kept j <= i} w_j > u sum_{kept} w_j.
//
// A token is a whole number, and either side of a border between two is
// another one: weights are formed in 64 bits, rounded to whole multiples of a unit
// (2^-45 of the largest for 2^18 logits) and added as whole numbers, so sums are
// exact and no order of additions, of atomics among them, changes a result.  What
// lies below half a unit weighs nothing.
//
// One workgroup has a row: its largest logit (pass A); with top_k or top_p a
// histogram of counts and weights over 2048 equal ranges of logits (pass B),
// the range within which a prefix ends, its members sorted (pass C); then sums
// of the kept weights per 512 logits in index order (pass D), and the draw.
#include "paged_impl.h"

namespace spruce {

struct Sampling {
  const void* logits;
  int64_t stride;  // of rows, in elements
  int V;
  const void* uniform;
  int uniform64;
  // Per-row values where the pointers are given, one for all otherwise.
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  double temperature1, top_p1, min_p1;
  int64_t top_k1;
  double shift;  // of weights
  int64_t* tokens;
  float* logprobs;  // or null
};

namespace {

constexpr int kThreads = 1024, kRowWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 4096;        // candidates that are sorted in LDS
constexpr int kChunk = 8;          // logits of a lane
constexpr int kPart = 64 * kChunk; // logits of a wave, and of one sum of pass D
constexpr int kParts = 4096;       // such sums
constexpr int kTable = 64;

// A unit is the smallest power of two of which V weights of one stay within 2^63,
// and 2^-52 at the least.
constexpr int kMostUnitBits = 52;
constexpr float kNothing = 54.f;  // below 2^-54 a weight is zero units

// A logit's bits as a number that goes up with it.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Eight logits from virtual place `at` on: NaN, and what lies outside of the
// row, as -inf.  Places count from the last 16-byte border at or before the row,
// so that all but the row's two ends are read 16 bytes at a time.
template <typename T>
struct Row {
  const char* base;
  int first, end;  // places of the row's logits
  __device__ __forceinline__ void init(const void* logits, int64_t element, int V) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(logits) + element * T::bytes;
    first = (int)(p % 16) / T::bytes;
    end = first + V;
    base = reinterpret_cast<const char*>(p - p % 16);
  }
  __device__ __forceinline__ static float widen(uint32_t bits) { return unpack1<T::code == SPRUCE_DTYPE_F16>(bits); }
  __device__ __forceinline__ float one(int at) const {
    if constexpr (T::bytes == 4)
      return reinterpret_cast<const float*>(base)[at];
    else
      return widen(reinterpret_cast<const uint16_t*>(base)[at]);
  }
  __device__ __forceinline__ void load(int at, float (&x)[kChunk]) const {
    if (at >= first && at + kChunk <= end) {
      if constexpr (T::bytes == 4) {
        const f32x4v a = *reinterpret_cast<const f32x4v*>(base + (int64_t)at * 4),
                     b = *reinterpret_cast<const f32x4v*>(base + (int64_t)at * 4 + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = a[i];
          x[4 + i] = b[i];
        }
      } else {
        const u32x4 a = *reinterpret_cast<const u32x4*>(base + (int64_t)at * 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[2 * i] = widen(a[i] & 0xffffu);
          x[2 * i + 1] = widen(a[i] >> 16);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) x[i] = at + i >= first && at + i < end ? one(at + i) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kChunk; ++i) x[i] = x[i] == x[i] ? x[i] : -INFINITY;
  }
};

// exp2(y) for y <= 0 in units, by 2^(n / 64) from a table and a polynomial in the rest: |z| <=
// ln 2 / 128, so that z^5 / 120 is below 2^-44.
struct Weights {
  double max, c2;
  const double* table;
  double shift;  // 2^52 units
  __device__ __forceinline__ double exact(float x) const {
    // The difference first: of the largest logit it is zero whatever c2 is.
    const double y = fmax(((double)x - max) * c2, -64.0);
    const double n = __builtin_rint(y * kTable);
    const double z = fma(n, -1.0 / kTable, y) * 0.69314718055994530942;
    const int k = (int)n;
    const double e = fma(z, fma(z, fma(z, fma(z, 1.0 / 24, 1.0 / 6), 0.5), 1.0), 1.0);
    return __builtin_ldexp(e * table[k & (kTable - 1)], k >> 6);
  }
  __device__ __forceinline__ double of(float x) const {
    if (max == INFINITY) return x == INFINITY ? 1.0 : 0.0;
    return exact(x);
  }
  __device__ __forceinline__ uint64_t units(double w) const {
    // Rounded to units as it is added to what has one as its last bit.
    return __builtin_bit_cast(uint64_t, w + shift) - __builtin_bit_cast(uint64_t, shift);
  }
};

struct Shared {
  double table[kTable];
  uint64_t weight[kBins];
  uint32_t count[kBins];
  uint64_t list[kList];     // order << 32 | ~place
  uint64_t part[kParts];
  uint64_t waves[kRowWaves];
  uint32_t wave_count[kRowWaves];
  uint64_t result[4];
  uint32_t size, lo, hi;
};

// Prefix sums over the workgroup's threads of a and b (up to and with this
// one's), and their totals.
__device__ __forceinline__ void block_prefix(Shared& sh, uint64_t& a, uint32_t& b, uint64_t& total_a, uint32_t& total_b) {
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  a = (uint64_t)wave_prefix((int64_t)a);
  b = (uint32_t)wave_prefix((int)b);
  __syncthreads();
  if (lane == 63) {
    sh.waves[wave] = a;
    sh.wave_count[wave] = b;
  }
  __syncthreads();
  uint64_t before_a = 0;
  uint32_t before_b = 0;
  total_a = total_b = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const uint64_t wa = sh.waves[w];
    const uint32_t wb = sh.wave_count[w];
    if (w < wave) {
      before_a += wa;
      before_b += wb;
    }
    total_a += wa;
    total_b += wb;
  }
  a += before_a;
  b += before_b;
}

// The list's first n entries, in descending order (zeros behind them).
__device__ __forceinline__ void sort_list(Shared& sh, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) sh.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int t = threadIdx.x; t < size / 2; t += kThreads) {
        const int i = 2 * t - (t & (j - 1));
        const uint64_t a = sh.list[i], b = sh.list[i + j];
        if ((a < b) == ((i & k) == 0)) {
          sh.list[i] = b;
          sh.list[i + j] = a;
        }
      }
      __syncthreads();
    }
}

// Where a prefix of the order ends: with the place `last` of the value `key`.
struct Cut {
  uint32_t key;
  uint32_t last;
};
__device__ __forceinline__ bool within(const Cut& c, uint32_t key, uint32_t place) {
  return key > c.key || (key == c.key && place <= c.last);
}

template <typename T>
struct Sampler {
  Shared& sh;
  Row<T> row;
  Weights w;
  int steps;  // of kThreads * kChunk places
  float top, per_bin;

  __device__ __forceinline__ int bin_of(float x) const {
    const float d = x == top ? 0.f : top - x;
    const float b = d * per_bin;
    return b < (float)(kBins - 1) ? (int)b : kBins - 1;
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int s = 0; s < steps; ++s) {
      const int at = (s * kThreads + (int)threadIdx.x) * kChunk;
      float x[kChunk];
      row.load(at, x);
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (x[i] > -INFINITY) f(x[i], at + i);
    }
  }

  // Where the prefix ends that has the first `rank` (by_count), or as few as reach
  // `mass` units: within bin `bin`, `above` and `above_mass` before it.  Its own
  // weight in *total.  The bin holds what is asked for.
  __device__ Cut resolve(int bin, bool by_count, uint32_t rank, double mass, uint32_t above, uint64_t above_mass,
                         const Cut& limit, uint64_t* total) {
    // Members of the bin as a range of orders.
    if (threadIdx.x == 0) {
      sh.lo = 0xffffffffu;
      sh.hi = 0;
      sh.size = 0;
    }
    __syncthreads();
    each([&](float x, int at) {
      if (bin_of(x) == bin) {
        const uint32_t key = ordered(x);
        if (!within(limit, key, (uint32_t)at)) return;
        const uint32_t i = atomicAdd(&sh.size, 1u);
        if (i < kList) sh.list[i] = (uint64_t)key << 32 | (uint32_t)~at;
        atomicMin(&sh.lo, key);
        atomicMax(&sh.hi, key);
      }
    });
    __syncthreads();
    uint32_t lo = sh.lo, hi = sh.hi, n = sh.size;
    // Too many to sort: narrowed to the range of orders that holds the end, or to one value.
    while (n > kList && lo < hi) {
      int shift = 0;
      while ((hi - lo) >> shift >= kBins) ++shift;
      __syncthreads();
      for (int i = threadIdx.x; i < kBins; i += kThreads) {
        sh.count[i] = 0;
        sh.weight[i] = 0;
      }
      __syncthreads();
      each([&](float x, int at) {
        const uint32_t key = ordered(x);
        if (key < lo || key > hi || !within(limit, key, (uint32_t)at)) return;
        const int b = (int)((hi - key) >> shift);
        atomicAdd(&sh.count[b], 1u);
        atomicAdd((unsigned long long*)&sh.weight[b], (unsigned long long)w.units(w.of(x)));
      });
      __syncthreads();
      const int b = find_bin(by_count, rank, mass, above, above_mass);
      const uint32_t top_key = hi - ((uint32_t)b << shift);
      const uint32_t low_key = b == (int)((hi - lo) >> shift) ? lo : top_key - ((1u << shift) - 1);
      hi = top_key;
      lo = low_key;
      n = sh.count[b];
      __syncthreads();
      if (n <= kList) {
        if (threadIdx.x == 0) sh.size = 0;
        __syncthreads();
        each([&](float x, int at) {
          const uint32_t key = ordered(x);
          if (key < lo || key > hi || !within(limit, key, (uint32_t)at)) return;
          sh.list[atomicAdd(&sh.size, 1u)] = (uint64_t)key << 32 | (uint32_t)~at;
        });
        __syncthreads();
      }
    }
    if (n > kList) {
      // One value: the first so many by place.
      const uint64_t one = w.units(w.of(unordered(hi)));
      uint64_t want;
      if (by_count)
        want = rank - above;
      else
        want = one == 0 ? 1 : (uint64_t)ceil((mass - (double)above_mass) / (double)one);
      if (want < 1) want = 1;
      if (want > n) want = n;
      *total = above_mass + want * one;
      return Cut{hi, nth_equal(hi, (uint32_t)want, limit)};
    }
    sort_list(sh, (int)n);
    // The entry with which the prefix ends, four a thread.
    uint64_t each_w[4], a = 0;
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * threadIdx.x + i;
      each_w[i] = at < (int)n ? w.units(w.of(unordered((uint32_t)(sh.list[at] >> 32)))) : 0;
      a += each_w[i];
    }
    const uint64_t mine = a;
    uint64_t all_a;
    uint32_t all_b;
    block_prefix(sh, a, b, all_a, all_b);
    if (threadIdx.x == 0) {
      sh.result[0] = sh.list[n - 1];
      sh.result[1] = above_mass + all_a;
    }
    __syncthreads();
    uint64_t before = above_mass + a - mine;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 4 * threadIdx.x + i;
      // The last of the prefix: what is before it falls short, what is with it does not.
      const bool last = by_count ? above + at + 1 == rank
                                 : ((double)before < mass || (above == 0 && at == 0)) &&
                                       !((double)(before + each_w[i]) < mass);
      if (at < (int)n && last && (by_count || each_w[i] > 0)) {
        sh.result[0] = sh.list[at];
        sh.result[1] = before + each_w[i];
      }
      before += each_w[i];
    }
    __syncthreads();
    const uint64_t end = sh.result[0];
    *total = sh.result[1];
    __syncthreads();
    return Cut{(uint32_t)(end >> 32), ~(uint32_t)end};
  }

  // The bin of the histogram in which the prefix ends; above and above_mass go on to
  // what is before it.  (The last bin that holds anything, where none reaches.)
  __device__ int find_bin(bool by_count, uint32_t rank, double mass, uint32_t& above, uint64_t& above_mass) {
    const int at = 2 * threadIdx.x;
    const uint32_t c0 = sh.count[at], c1 = sh.count[at + 1];
    const uint64_t w0 = sh.weight[at], w1 = sh.weight[at + 1];
    uint64_t a = w0 + w1, all_a;
    uint32_t b = c0 + c1, all_b;
    block_prefix(sh, a, b, all_a, all_b);
    const uint64_t a0 = above_mass + a - w0 - w1;
    const uint32_t b0 = above + b - c0 - c1;
    if (threadIdx.x == 0) sh.result[0] = 0xffffffffull;
    if (threadIdx.x == 0) sh.result[3] = 0;
    __syncthreads();
    auto look = [&](int bin, uint32_t c, uint64_t wt, uint32_t before, uint64_t before_mass) {
      if (c == 0) return;
      atomicMax((unsigned long long*)&sh.result[3], (unsigned long long)bin);
      const bool reaches = by_count ? before + c >= rank : !((double)(before_mass + wt) < mass);
      if (reaches) atomicMin((unsigned long long*)&sh.result[0], (unsigned long long)bin);
    };
    look(at, c0, w0, b0, a0);
    look(at + 1, c1, w1, b0 + c0, a0 + w0);
    __syncthreads();
    const int bin = (int)(sh.result[0] == 0xffffffffull ? sh.result[3] : sh.result[0]);
    if (bin == at || bin == at + 1) {
      sh.result[1] = bin == at ? a0 : a0 + w0;
      sh.result[2] = bin == at ? b0 : b0 + c0;
    }
    __syncthreads();
    above_mass = sh.result[1];
    above = (uint32_t)sh.result[2];
    __syncthreads();
    return bin;
  }

  // The place of the want-th logit of one value.
  __device__ uint32_t nth_equal(uint32_t key, uint32_t want, const Cut& limit) {
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    for (int s = 0; s < steps; ++s) {
      const int at = (s * kThreads + (int)threadIdx.x) * kChunk;
      float x[kChunk];
      row.load(at, x);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) c += x[i] > -INFINITY && ordered(x[i]) == key && within(limit, key, at + i);
      const int all = wave_prefix(c);
      if (lane == 63) sh.part[s * kRowWaves + wave] = (uint64_t)all;
    }
    uint64_t before;
    const int part = find_part(want - 1, before);
    if (wave == 0) {
      const int at = part * kPart + lane * kChunk;
      float x[kChunk];
      row.load(at, x);
      int c = 0, hit = -1;
      bool is[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        is[i] = x[i] > -INFINITY && ordered(x[i]) == key && within(limit, key, at + i);
        c += is[i];
      }
      int upto = (int)before + wave_prefix(c) - c;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        if (is[i] && ++upto == (int)want) hit = at + i;
      }
      if (hit >= 0) sh.result[0] = (uint64_t)hit;
    }
    __syncthreads();
    const uint32_t place = (uint32_t)sh.result[0];
    __syncthreads();
    return place;
  }

  // The first part whose sums, added up in order, are past `target`, and what is before it
  // (the last part with anything where none is).
  __device__ int find_part(uint64_t target, uint64_t& before) {
    const int n = steps * kRowWaves;
    constexpr int EACH = kParts / kThreads;
    __syncthreads();
    uint64_t v[EACH], a = 0;
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = EACH * threadIdx.x + i;
      v[i] = at < n ? sh.part[at] : 0;
      a += v[i];
    }
    const uint64_t mine = a;
    uint64_t all_a;
    uint32_t all_b;
    block_prefix(sh, a, b, all_a, all_b);
    if (target >= all_a) target = all_a - 1;
    uint64_t upto = a - mine;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      if (upto <= target && target < upto + v[i]) {
        sh.result[0] = EACH * threadIdx.x + i;
        sh.result[1] = upto;
      }
      upto += v[i];
    }
    __syncthreads();
    const int part = (int)sh.result[0];
    before = sh.result[1];
    __syncthreads();
    return part;
  }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)flat_block(), tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  Sampler<T> s{sh};
  s.row.init(p.logits, (int64_t)b * p.stride, p.V);
  s.steps = (s.row.end + kThreads * kChunk - 1) / (kThreads * kChunk);
  const double temperature = p.temperature ? (double)p.temperature[b] : p.temperature1;
  const int64_t top_k = p.top_k ? (int64_t)p.top_k[b] : p.top_k1;
  const double top_p = p.top_p ? (double)p.top_p[b] : p.top_p1;
  double min_p = p.min_p ? (double)p.min_p[b] : p.min_p1;
  min_p = min_p < 1.0 ? min_p : 1.0;
  if (tid < kTable) sh.table[tid] = exp2((double)tid / kTable);

  // Pass A: the largest logit with its first place, and the smallest.
  uint64_t best = 0;
  float least = INFINITY;
  s.each([&](float x, int at) {
    const uint64_t v = (uint64_t)ordered(x) << 32 | (uint32_t)~at;
    best = v > best ? v : best;
    least = fminf(least, x);
  });
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const uint64_t o = __shfl_xor(best, i);
    best = o > best ? o : best;
    least = fminf(least, __shfl_xor(least, i));
  }
  if (lane == 0) {
    sh.waves[wave] = best;
    sh.wave_count[wave] = __builtin_bit_cast(uint32_t, least);
  }
  __syncthreads();
  for (int i = 0; i < kRowWaves; ++i) {
    best = sh.waves[i] > best ? sh.waves[i] : best;
    least = fminf(least, __builtin_bit_cast(float, sh.wave_count[i]));
  }
  __syncthreads();
  const uint32_t first_place = ~(uint32_t)best;
  if (best == 0 || !(temperature > 0)) {  // nothing to choose from, or the largest
    if (tid == 0) {
      p.tokens[b] = best == 0 ? -1 : (int64_t)(first_place - (uint32_t)s.row.first);
      if (p.logprobs) p.logprobs[b] = best == 0 ? -INFINITY : 0.f;
    }
    return;
  }
  s.top = unordered((uint32_t)(best >> 32));
  // (An infinite temperature: all weights one, but those of -inf.)
  s.w = Weights{(double)s.top, fmax(1.44269504088896340736 / temperature, 1e-300), sh.table, p.shift};

  Cut cut{0, 0};  // all
  const bool by_k = top_k > 0 && top_k < p.V, by_p = top_p < 1.0;
  if (by_k || by_p) {
    // Pass B.  Bins of equal width down to the smallest logit, or to where weights end.
    float range = fminf(s.top - least, (float)(kNothing / s.w.c2));
    range = range > 1e-30f ? (range < 1e30f ? range : 1e30f) : 1e-30f;
    s.per_bin = (float)(kBins - 1) / range;
    for (int i = tid; i < kBins; i += kThreads) {
      sh.count[i] = 0;
      sh.weight[i] = 0;
    }
    __syncthreads();
    s.each([&](float x, int) {
      const int bin = s.bin_of(x);
      atomicAdd(&sh.count[bin], 1u);
      atomicAdd((unsigned long long*)&sh.weight[bin], (unsigned long long)s.w.units(s.w.of(x)));
    });
    __syncthreads();
    uint64_t a = sh.weight[2 * tid] + sh.weight[2 * tid + 1], total;
    uint32_t c = sh.count[2 * tid] + sh.count[2 * tid + 1], all;
    block_prefix(sh, a, c, total, all);
    if (by_k && top_k < (int64_t)all) {
      uint32_t above = 0;
      uint64_t above_mass = 0;
      const int bin = s.find_bin(true, (uint32_t)top_k, 0.0, above, above_mass);
      // (What is behind the last weight has none to choose by.)
      if (above_mass < total) {
        cut = s.resolve(bin, true, (uint32_t)top_k, 0.0, above, above_mass, cut, &total);
        if (by_p) {  // the histogram again, of what is left
          __syncthreads();
          for (int i = tid; i < kBins; i += kThreads) {
            sh.count[i] = 0;
            sh.weight[i] = 0;
          }
          __syncthreads();
          s.each([&](float x, int at) {
            if (!within(cut, ordered(x), (uint32_t)at)) return;
            const int bin2 = s.bin_of(x);
            atomicAdd(&sh.count[bin2], 1u);
            atomicAdd((unsigned long long*)&sh.weight[bin2], (unsigned long long)s.w.units(s.w.of(x)));
          });
          __syncthreads();
        }
      }
    }
    if (by_p) {
      const double mass = fmax(top_p, 0.0) * (double)total;
      uint32_t above = 0;
      uint64_t above_mass = 0;
      const int bin = s.find_bin(false, 0, mass, above, above_mass);
      uint64_t left;
      cut = s.resolve(bin, false, 0, mass, above, above_mass, cut, &left);
    }
  }

  // Pass D.
  const double least_weight = fmin(min_p, 1.0);
  auto weight_at = [&](float x, int at) -> uint64_t {
    if (!(x > -INFINITY) || !within(cut, ordered(x), (uint32_t)at)) return 0;
    const double wt = s.w.of(x);
    return wt >= least_weight ? s.w.units(wt) : 0;
  };
  for (int i = 0; i < s.steps; ++i) {
    const int at = (i * kThreads + tid) * kChunk;
    float x[kChunk];
    s.row.load(at, x);
    uint64_t sum = 0;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) sum += weight_at(x[j], at + j);
    const int64_t upto = wave_prefix((int64_t)sum);
    if (lane == 63) sh.part[i * kRowWaves + wave] = (uint64_t)upto;
  }
  __syncthreads();
  uint64_t total = 0;
  {
    uint64_t a = 0;
    uint32_t c = 0, all;
    for (int i = tid; i < s.steps * kRowWaves; i += kThreads) a += sh.part[i];
    block_prefix(sh, a, c, total, all);
  }
  double u = p.uniform64 ? static_cast<const double*>(p.uniform)[b] : (double)static_cast<const float*>(p.uniform)[b];
  u = u > 0.0 ? u : 0.0;
  const double wanted = u * (double)total;
  const uint64_t target = wanted < (double)(total - 1) ? (uint64_t)wanted : total - 1;
  uint64_t before;
  const int part = s.find_part(target, before);
  if (wave == 0) {
    const int at = part * kPart + lane * kChunk;
    float x[kChunk];
    s.row.load(at, x);
    uint64_t each_w[kChunk], sum = 0;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      each_w[j] = weight_at(x[j], at + j);
      sum += each_w[j];
    }
    uint64_t upto = before + (uint64_t)wave_prefix((int64_t)sum) - sum;
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      if (upto <= target && target < upto + each_w[j]) {
        p.tokens[b] = at + j - s.row.first;
        if (p.logprobs) p.logprobs[b] = (float)log(s.w.of(x[j]) / ((double)total * (p.shift * 0x1p-52)));
      }
      upto += each_w[j];
    }
  }
}

}  // namespace
}  // namespace spruce

using namespace spruce;

extern "C" int spruce_sample_tokens(const spruce_sample_tokens_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_sample_tokens_args& a = *args;
  SPRUCE_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "unsupported dtype code %lld", (long long)a.dtype);
  SPRUCE_REQUIRE(a.B >= 0 && a.B < (int64_t)1 << 30, "invalid row count %lld", (long long)a.B);
  constexpr int64_t kMostV = (int64_t)kParts * kPart - kThreads * kChunk;
  SPRUCE_REQUIRE(a.V >= 1 && a.V <= kMostV, "the vocabulary must be in [1, %lld], got %lld", (long long)kMostV,
                 (long long)a.V);
  if (a.B == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(a.logits && a.uniform && a.tokens, "logits, uniform and tokens must be non-null device pointers");
  const int eb = a.dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % eb == 0, "logits must be aligned to their type");
  SPRUCE_REQUIRE(a.temperature || a.temperature1 >= 0, "temperature must not be negative");
  SPRUCE_REQUIRE(a.top_k || a.top_k1 >= 0, "top_k must not be negative");
  SPRUCE_REQUIRE(a.top_p || (a.top_p1 >= 0 && a.top_p1 <= 1), "top_p must be in [0, 1]");
  SPRUCE_REQUIRE(a.min_p || (a.min_p1 >= 0 && a.min_p1 <= 1), "min_p must be in [0, 1]");
  Sampling p{};
  p.logits = a.logits;
  p.stride = a.stride;
  p.V = (int)a.V;
  p.uniform = a.uniform;
  p.uniform64 = a.uniform64 != 0;
  p.temperature = a.temperature;
  p.top_k = a.top_k;
  p.top_p = a.top_p;
  p.min_p = a.min_p;
  p.temperature1 = a.temperature1;
  p.top_k1 = a.top_k1;
  p.top_p1 = a.top_p1;
  p.min_p1 = a.min_p1;
  int bits = 63;
  while (bits > 0 && ((int64_t)1 << (63 - bits)) < a.V) --bits;
  p.shift = __builtin_ldexp(1.0, kMostUnitBits - (bits < kMostUnitBits ? bits : kMostUnitBits));
  p.tokens = a.tokens;
  p.logprobs = a.logprobs;
  const hipStream_t st = (hipStream_t)stream;
  SPRUCE_REQUIRE(a.B <= kGridX, "too many rows for one call");
  const dim3 grid((unsigned)a.B);
  switch (a.dtype) {
    case SPRUCE_DTYPE_BF16: hipLaunchKernelGGL(sample_kernel<InBF16>, grid, dim3(kThreads), 0, st, p); break;
    case SPRUCE_DTYPE_F16: hipLaunchKernelGGL(sample_kernel<InF16>, grid, dim3(kThreads), 0, st, p); break;
    default: hipLaunchKernelGGL(sample_kernel<InF32>, grid, dim3(kThreads), 0, st, p); break;
  }
  return check_launch("token sampling");
}
