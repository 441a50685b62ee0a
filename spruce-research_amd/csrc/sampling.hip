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
// One workgroup has a row.  Its first pass finds the largest logit.  What can be
// kept is then mostly few logits: a second pass lists those above a bound
// (of top_k, from the threads' own largest; of min_p; of top_p, from a
// histogram of the weights that needs a pass of its own), and the ends of the
// prefixes and the draw are found among them: each is the first entry of some
// order whose running sum passes a target, which select() narrows down digit by digit.
// Rows that keep more than the list holds go the long way: the end of a prefix
// within one range of the histogram, then sums of 512 logits each, in index order.
//
// What bounds it: a row's logits pass one CU, where every instruction on each of 150016 logits takes about
// a microsecond, and the steps after the lists are chains of a few dozen barriers; the bytes are nothing to it (19 MB
// take 4 us).  So a weight is two additions, a fused one and a polynomial of four terms, only rows of a histogram
// need all of them, and few long rows without top_k and min_p are shared by workgroups.
// Measured: top_k 50, top_p 0.95 of [1, 32003] f16 20 us; rows of all kinds up to top_k 1000, top_p 0.9 of [24, 50021]
// bf16 46 to 68, by the inputs; top_p 0.95 of [64, 150016] bf16 89; min_p 0.001 of [256, 131072] f32 77 to 82.
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
  // Rows that more than one workgroup shares: parts of part_places places, and what they leave each other.
  int parts, part_places;
  uint64_t* best;             // [B][parts] the largest logit's order << 32 | ~place of its chunk
  uint64_t* hists;            // [B][parts][2048]
  uint64_t* lists;            // [B][parts][4096]
  struct PartList* part_list; // [B][parts]
  uint64_t* sums;             // [B][4096]
  struct RowState* states;    // [B]
};
// kind: everything from the bound on; the members of the bin that holds an end (kMembers: the rest did not
// fit); or not even those (kTooMany).
struct PartList {
  uint32_t size;
  int kind;
};
struct RowState {
  int stage, bin;            // that the end is in
  uint64_t before, total;    // of the bin, and of all weights
  float low, high;           // logits that lists begin and the bin's end with
  uint32_t cut_key, cut_last;
};

namespace {

constexpr int kThreads = 1024, kRowWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kList = 4096, kEach = kList / kThreads;
constexpr int kChunk = 8;           // logits that a lane reads at once
constexpr int kPart = 64 * kChunk;  // logits of one sum of the long way
constexpr int kParts = 4096;        // such sums
constexpr int kTable = 64;
constexpr int kMostParts = 16;      // of a row
// Rows that are shared out, to as many workgroups: of so many logits at the least, with top_p and without.
// Shared and not, in us: top_p 0.95 of bf16 [1, 100000] 55 and 95, [8, 150016] 64 and 130, [64, 150016]
// 89 and 130, [128, 256000] 149 and 216, [128, 100000] 93 and 109; at 50021 logits the launches' own latency
// takes all that is gained; without top_p [1, 50021] 18 and 26, [128, 150016] 38 and 56.
// (With top_k or min_p the lists are short, and it lost at every size: top_k 50 of [1, 150016] 40 and 34.)
constexpr int kSharers = kCus;
constexpr int64_t kLeastByP = 65536, kLeastPlain = 32768;
constexpr int kWhole = 0, kMembers = 1, kTooMany = 2;              // of a PartList
constexpr int kWeighed = 0, kSummed = 1;                           // of a RowState: what it waits for next

// A unit is the smallest power of two of which V weights of one stay within 2^63,
// and 2^-52 at the least.
constexpr int kMostUnitBits = 52;
constexpr double kNothing = 54.0;  // below 2^-54 a weight is zero units

// A logit's bits as a number that goes up with it.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// A row's logits by place.  Places count from the last 16-byte border at or
// before the row, so that all but its two ends are read 16 bytes at a time; what lies
// outside of it, and NaN, are -inf.
template <typename T>
struct Row {
  typedef struct { u32x4 v[T::bytes / 2]; } Raw;  // eight logits
  const char* base;
  int first, end;  // places of the row's logits
  __device__ __forceinline__ void init(const void* logits, int64_t element, int V) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(logits) + element * T::bytes;
    first = (int)(p % 16) / T::bytes;
    end = first + V;
    base = reinterpret_cast<const char*>(p - p % 16);
  }
  __device__ __forceinline__ static float widen(uint32_t bits) { return unpack1<T::code == SPRUCE_DTYPE_F16>(bits); }
  __device__ __forceinline__ Raw load(int at) const {
    constexpr uint32_t kInf = T::bytes == 4 ? 0xff800000u : (T::code == SPRUCE_DTYPE_F16 ? 0xfc00fc00u : 0xff80ff80u);
    Raw r;
#pragma unroll
    for (int i = 0; i < T::bytes / 2; ++i) r.v[i] = u32x4{kInf, kInf, kInf, kInf};
    if (at >= first && at + kChunk <= end) {
#pragma unroll
      for (int i = 0; i < T::bytes / 2; ++i)
        r.v[i] = *reinterpret_cast<const u32x4*>(base + (int64_t)at * T::bytes + 16 * i);
    } else if (at + kChunk > first && at < end) {  // the row's two ends, a 32-bit word at a time
#pragma unroll 1
      for (int i = 0; i < kChunk; ++i) {
        if (at + i < first || at + i >= end) continue;
        const int word = i * T::bytes / 4;
        uint32_t x, old = kInf;
        if constexpr (T::bytes == 4) {
          x = reinterpret_cast<const uint32_t*>(base)[at + i];
        } else {
          x = reinterpret_cast<const uint16_t*>(base)[at + i];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j == word) old = r.v[0][j];
          x = i & 1 ? (old & 0xffffu) | x << 16 : (old & 0xffff0000u) | x;
        }
#pragma unroll
        for (int j = 0; j < 2 * T::bytes; ++j)
          if (j == word) r.v[j >> 2][j & 3] = x;
      }
    }
    return r;
  }
  static __device__ __forceinline__ void decode(const Raw& r, float (&x)[kChunk]) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) {
      float y;
      if constexpr (T::bytes == 4) {
        const uint32_t bits = r.v[i >> 2][i & 3];  // (a bit cast of the element itself reads element 0)
        y = __builtin_bit_cast(float, bits);
      } else
        y = widen(i & 1 ? r.v[0][i >> 1] >> 16 : r.v[0][i >> 1] & 0xffffu);
      // (The maximum of a number and NaN is the number.)
      x[i] = fmaxf(y, -INFINITY);
    }
  }
};

// exp((x - max) / T) = 2^(n / 64) 2^(r / 64): n by adding what leaves no bits for a fraction, its power
// from a table, with n's upper bits added to the exponent (and its lower six taken off in the table), and a
// polynomial in r, |r| <= 1 / 2, of ln 2 / 64 so small that the next term is below 2^-44.
struct Weights {
  double max, steps, lowest;  // 64 log2(e) / T, and the difference past which weights are nothing
  double shift;               // 2^52 units
  const uint2* table;
  // (-inf comes out below half a unit.  No product is fused with the sum of units(): a weight's units are the same
  // wherever they are formed, so that sums of some hold against sums of all.)
  __device__ __forceinline__ double of(float x) const {
#pragma clang fp contract(off)
    // The difference first: of the largest logit it is zero whatever T is.
    const double d = fmax((double)x - max, lowest);
    constexpr double kRound = 0x1.8p+52, kStep = 0.69314718055994530942 / kTable;
    const double t = fma(d, steps, kRound);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, t);
    const double r = fma(d, steps, kRound - t);
    const double e = fma(r, fma(r, fma(r, fma(r, kStep * kStep * kStep * kStep / 24, kStep * kStep * kStep / 6), kStep * kStep / 2), kStep), 1.0);
    const uint2 p = table[n & (kTable - 1)];
    return e * __builtin_bit_cast(double, (uint64_t)(p.y + (n << 14)) << 32 | p.x);
  }
  __device__ __forceinline__ uint64_t units(double w) const {
#pragma clang fp contract(off)
    // Rounded to units as it is added to what has one as its last bit.
    return __builtin_bit_cast(uint64_t, w + shift) - __builtin_bit_cast(uint64_t, shift);
  }
  // Those of eight, kept where they are for the compiler: moved under the conditions
  // of their use they follow one another, each with its chain's latency.
  __device__ __forceinline__ void of8(const float (&x)[kChunk], double (&w)[kChunk]) const {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) w[i] = of(x[i]);
#pragma unroll
    for (int i = 0; i < kChunk; ++i) asm volatile("" : "+v"(w[i]));
  }
};

struct Small {
  uint64_t key, weight;
};

// The same in every lane: kept in scalar registers.
__device__ __forceinline__ double uniform(double x) {
  return __builtin_bit_cast(double, lane_of(__builtin_bit_cast(int64_t, x), 0));
}
__device__ __forceinline__ float uniform(float x) {
  return __builtin_bit_cast(float, spruce::uniform(__builtin_bit_cast(int, x)));
}

struct Shared {
  uint2 table[kTable];
  uint64_t weight[kBins];
  uint64_t list[kList];     // order << 32 | ~place
  uint64_t part[kParts];
  Small small[64];
  uint64_t waves[kRowWaves];
  uint64_t result[3];
  uint32_t size;
  uint32_t starts[kMostParts];
  // What the long way goes on with.
  float top;
  int infinite, bin;        // of the first end by weight or count; -1: none yet
  uint64_t before, total;   // of the bin, and of all weights (of an end by count: the number of logits)
};

// Sums of a over the threads up to and with this one, and their total.  Ends with a barrier to come.
__device__ __forceinline__ uint64_t block_prefix(Shared& sh, uint64_t a, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = spruce::uniform(threadIdx.x >> 6);
  a = (uint64_t)wave_prefix((int64_t)a);
  __syncthreads();
  if (lane == 63) sh.waves[wave] = a;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kRowWaves; ++w) {
    const uint64_t x = sh.waves[w];
    if (w < wave) before += x;
    total += x;
  }
  return a + before;
}

// Of up to kEach entries a thread, all keys different and those of a weight within [lo, hi],
// the one that comes first, in descending order of the keys, with a sum of weights
// (its own included) above `target`: its key.  target must be below the sum of all.
__device__ __forceinline__ uint64_t select(Shared& sh, const uint64_t (&key)[kEach], const uint64_t (&weight)[kEach],
                                           uint64_t lo, uint64_t hi, uint64_t target) {
  const int tid = threadIdx.x, lane = tid & 63, wave = spruce::uniform(tid >> 6);
  uint64_t before = 0;
  __syncthreads();
  while (true) {
    // A digit of what is left: as many bits as there are threads.
    const int bits = 64 - __builtin_clzll((hi - lo) | 1);
    const int shift = bits > 10 ? bits - 10 : 0;
    sh.weight[tid] = 0;
    if (tid < 64) sh.part[tid] = 0;
    if (tid == 0) sh.size = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (weight[i] && key[i] >= lo && key[i] <= hi)
        atomicAdd((unsigned long long*)&sh.weight[(hi - key[i]) >> shift], (unsigned long long)weight[i]);
    __syncthreads();
    const uint64_t mine = sh.weight[tid];
    uint64_t total;
    const uint64_t upto = before + block_prefix(sh, mine, total);
    if (upto - mine <= target && target < upto) {
      sh.result[0] = tid;
      sh.result[1] = upto - mine;
    }
    __syncthreads();
    before = sh.result[1];
    hi -= sh.result[0] << shift;
    lo = hi - lo < (1ull << shift) ? lo : hi - ((1ull << shift) - 1);
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (weight[i] && key[i] >= lo && key[i] <= hi) {
        const uint32_t at = atomicAdd(&sh.size, 1u);
        if (at < 64) sh.small[at] = Small{key[i], weight[i]};
      }
    __syncthreads();
    if (sh.size <= 64) break;
    __syncthreads();
  }
  // Few are left: each one's sum by comparison with all, every wave with some of them.
  const int n = (int)sh.size;
  if (lane < n) {
    const uint64_t me = sh.small[lane].key;
    uint64_t sum = 0;
    for (int j = wave; j < n; j += kRowWaves) {
      const Small o = sh.small[j];
      if (o.key > me) sum += o.weight;
    }
    if (sum) atomicAdd((unsigned long long*)&sh.part[lane], (unsigned long long)sum);
  }
  __syncthreads();
  if (tid < n) {
    const Small me = sh.small[tid];
    const uint64_t sum = before + sh.part[tid];
    if (sum <= target && target < sum + me.weight) sh.result[2] = me.key;
  }
  __syncthreads();
  return sh.result[2];
}

// Where a prefix of the order ends: with the place `last` of the value `key`.
struct Cut {
  uint32_t key;
  uint32_t last;
};
__device__ __forceinline__ bool within(const Cut& c, uint32_t key, uint32_t place) {
  return ((uint64_t)key << 32 | (uint32_t)~place) >= ((uint64_t)c.key << 32 | (uint32_t)~c.last);
}

// The target of the smallest prefix that reaches a mass.
__device__ __forceinline__ uint64_t target_of(double mass) { return mass > 1.0 ? (uint64_t)ceil(mass) - 1 : 0; }

template <typename T>
struct Sampler {
  Shared& sh;
  Row<T> row;
  Weights w;
  int begin, steps;  // the first place, and steps of kThreads * kChunk from there on
  bool infinite;   // the largest logit is +inf: such are taken as 0, all others as -inf
  float top, per_bin;

  // Ranges of logits that the histogram tells apart, from the top down.
  __device__ __forceinline__ int bin_of(float x) const {
    return (int)fminf((top - x) * per_bin, (float)(kBins - 1));
  }
  // The smallest logit in a bin, or above it: 64 orders tried at once.
  __device__ __forceinline__ float bin_end(int bin) const {
    if (bin >= kBins - 1) return -3.402823466e+38f;
    uint32_t lo = ordered(-INFINITY), hi = ordered(top);  // lo is past the bin, hi is not
    while (hi - lo > 1) {
      const uint32_t step = (hi - lo) / 65 + 1, rest = hi - lo, mine = step * ((threadIdx.x & 63) + 1);
      const uint64_t in = __ballot(mine >= rest || bin_of(unordered(lo + mine)) <= bin);
      // (step * 64 may fall short of hi, which is within.)
      const uint32_t first = in ? (uint32_t)__builtin_ctzll(in) : 64;
      const uint32_t to = step * (first + 1);
      hi = to < rest ? lo + to : hi;
      lo += step * first;
    }
    return uniform(unordered(hi));
  }
  __device__ __forceinline__ void decode(const typename Row<T>::Raw& raw, float (&x)[kChunk]) const {
    Row<T>::decode(raw, x);
    if (infinite) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
    }
  }
  // f(eight logits, the place of the first); the loads of AHEAD and up to twice as many in flight.
  template <int AHEAD, typename F>
  __device__ __forceinline__ void chunks(F f) const {
    chunks_while<AHEAD>(f, [] { return true; });
  }
  template <int AHEAD, typename F, typename G>
  __device__ __forceinline__ void chunks_while(F f, G more) const {
    typename Row<T>::Raw raw[AHEAD], next[AHEAD];
    const int mine = begin + (int)threadIdx.x * kChunk;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) raw[i] = row.load(mine + i * kThreads * kChunk);
    for (int s = 0; s < steps && more(); s += AHEAD) {
      const int at = s * kThreads * kChunk + mine;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) next[i] = row.load(at + (AHEAD + i) * kThreads * kChunk);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        float x[kChunk];
        decode(raw[i], x);
        f(x, at + i * kThreads * kChunk);
        raw[i] = next[i];
      }
    }
  }
  static __device__ __forceinline__ float largest(const float (&x)[kChunk]) {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < kChunk; ++i) m = fmaxf(m, x[i]);
    return m;
  }
  // Appends a chunk's logits named by `bits` to the list: one addition to its length a wave.
  __device__ __forceinline__ void append(const float (&x)[kChunk], int at, uint32_t bits) const {
    if (__ballot(bits != 0) == 0) return;
    const int mine = __builtin_popcount(bits), upto = wave_prefix(mine);
    uint32_t to = 0;
    if ((threadIdx.x & 63) == 63) to = atomicAdd(&sh.size, (uint32_t)upto);
    to = (uint32_t)__builtin_amdgcn_readlane((int)to, 63) + upto - mine;
    if (bits) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (bits >> i & 1) {
          if (to < kList) sh.list[to] = (uint64_t)ordered(x[i]) << 32 | (uint32_t)~(at + i);
          ++to;
        }
    }
  }
  // Lists the logits from `low` to `high`, within `limit`; false where there are more than fit.
  __device__ __forceinline__ bool collect(float low, float high, const Cut& limit) const {
    __syncthreads();
    if (threadIdx.x == 0) sh.size = 0;
    __syncthreads();
    const bool limited = limit.key != 0;
    chunks_while<T::bytes == 2 ? 4 : 2>([&](const float (&x)[kChunk], int at) {
      uint32_t bits = 0;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) bits |= (uint32_t)((x[i] >= low) & (x[i] <= high)) << i;
      if (limited && bits) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          if (!within(limit, ordered(x[i]), (uint32_t)(at + i))) bits &= ~(1u << i);
      }
      append(x, at, bits);
    }, [&] { return *(volatile uint32_t*)&sh.size <= kList; });
    __syncthreads();
    return sh.size <= kList;
  }
  __device__ __forceinline__ void clear_bins() const {
    __syncthreads();
    sh.weight[threadIdx.x] = 0;
    sh.weight[threadIdx.x + kThreads] = 0;
    __syncthreads();
  }
  // This thread's entries of the list.
  // An entry without the bits that all entries have alike, the lower ones of 16-bit logits and the upper ones of
  // places: select() would go through them a digit at a time, with all additions in one place.  ([24, 50021] bf16 of
  // up to top_k 1000: 75 us, 68 without; the end within a bin of [64, 150016] bf16: 31 and 26.)
  static constexpr int kSame = T::bytes == 4 ? 0 : (T::code == SPRUCE_DTYPE_F16 ? 13 : 16), kPlaceBits = 22;
  static constexpr uint64_t kPlace = ((uint64_t)1 << kPlaceBits) - 1;
  static __device__ __forceinline__ uint64_t tight(uint64_t entry) {
    return entry >> (32 + kSame) << kPlaceBits | (entry & kPlace);
  }
  static __device__ __forceinline__ uint64_t tight(uint32_t order, bool last) {
    return tight((uint64_t)order << 32 | (last ? 0xffffffffu : 0));
  }
  static __device__ __forceinline__ uint32_t place_of(uint64_t tightened) { return (uint32_t)(kPlace - (tightened & kPlace)); }
  static __device__ __forceinline__ uint32_t order_of(uint64_t tightened) {
    const uint32_t order = (uint32_t)(tightened >> kPlaceBits) << kSame;
    return order & 0x80000000u ? order : order | ((1u << kSame) - 1);
  }
  __device__ __forceinline__ void entries(uint64_t (&key)[kEach]) const {
    const uint32_t n = sh.size;
#pragma unroll
    for (int i = 0; i < kEach; ++i) key[i] = i * kThreads + threadIdx.x < n ? sh.list[i * kThreads + threadIdx.x] : 0;
  }

  // The first bin with which the histogram's sum, `before` it, is above `target`, or the last that holds
  // anything; `before` goes on to what is before the bin, `all` gets the whole.
  __device__ __forceinline__ int find_bin(uint64_t target, uint64_t& before, uint64_t& all) {
    const int at = 2 * threadIdx.x;
    const uint64_t w0 = sh.weight[at], w1 = sh.weight[at + 1];
    const uint64_t from = before + block_prefix(sh, w0 + w1, all) - w0 - w1;
    all += before;
    if (target >= all) target = all - 1;
    if (from <= target && target < from + w0 + w1) {
      const bool second = target >= from + w0;
      sh.result[0] = at + (second ? 1 : 0);
      sh.result[1] = from + (second ? w0 : 0);
    }
    __syncthreads();
    const int bin = (int)sh.result[0];
    before = sh.result[1];
    __syncthreads();
    return bin;
  }

  // Weights of the logits within `limit`, or their number.
  __device__ __forceinline__ void weigh(const Cut& limit) {
    clear_bins();
    const bool limited = limit.key != 0;
    chunks<2>([&](const float (&x)[kChunk], int at) {
      double weight[kChunk];
      w.of8(x, weight);
      if (limited) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i)
          if (!within(limit, ordered(x[i]), (uint32_t)(at + i))) weight[i] = 0.0;
      }
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        const uint64_t units = w.units(weight[i]);
        if (units) atomicAdd((unsigned long long*)&sh.weight[bin_of(x[i])], (unsigned long long)units);
      }
    });
    __syncthreads();
  }
  __device__ __forceinline__ void count() {
    clear_bins();
    chunks<T::bytes == 2 ? 4 : 2>([&](const float (&x)[kChunk], int) {
#pragma unroll
      for (int i = 0; i < kChunk; ++i)
        if (x[i] > -INFINITY) atomicAdd((unsigned long long*)&sh.weight[bin_of(x[i])], 1ull);
    });
    __syncthreads();
  }

  // The long way to the end of a prefix: that of the logits within `limit` whose number (by_count), or
  // weight, is the first above `target`.  It ends in bin `bin`, `before` before it.
  __device__ __forceinline__ Cut resolve(int bin, bool by_count, uint64_t target, uint64_t before, const Cut& limit) {
    uint32_t lo = ordered(bin_end(bin)), hi = bin == 0 ? ordered(top) : ordered(bin_end(bin - 1)) - 1;
    // Narrowed until its members can be listed, or are of one value.
    bool fits;
    while (!(fits = collect(unordered(lo), unordered(hi), limit)) && lo < hi) {
      int shift = 0;
      while ((hi - lo) >> shift >= kBins) ++shift;
      clear_bins();
      const float low = unordered(lo), high = unordered(hi);
      chunks<2>([&](const float (&x)[kChunk], int at) {
#pragma unroll
        for (int i = 0; i < kChunk; ++i) {
          const uint32_t key = ordered(x[i]);
          if (!((x[i] >= low) & (x[i] <= high)) || !within(limit, key, (uint32_t)(at + i))) continue;
          const uint64_t units = by_count ? 1 : w.units(w.of(x[i]));
          atomicAdd((unsigned long long*)&sh.weight[(hi - key) >> shift], (unsigned long long)units);
        }
      });
      __syncthreads();
      uint64_t all;
      const uint32_t b = (uint32_t)find_bin(target, before, all);
      hi -= b << shift;
      lo = hi - lo < (1u << shift) ? lo : hi - ((1u << shift) - 1);
    }
    if (!fits) {
      // One value: the first so many by place.
      const uint64_t one = by_count ? 1 : w.units(w.of(unordered(hi)));
      const uint64_t more = one == 0 ? 0 : (target - before) / one;
      return Cut{hi, nth_equal(hi, more, limit)};
    }
    return end_among(by_count, target, before, lo, hi);
  }
  // The same among the list, of orders from lo to hi.
  __device__ __forceinline__ Cut end_among(bool by_count, uint64_t target, uint64_t before, uint32_t lo, uint32_t hi) const {
    uint64_t key[kEach], ones[kEach], all = 0;
    entries(key);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      ones[i] = key[i] == 0 ? 0 : (by_count ? 1 : w.units(w.of(unordered((uint32_t)(key[i] >> 32)))));
      key[i] = tight(key[i]);
      all += ones[i];
    }
    block_prefix(sh, all, all);
    if (all == 0) return Cut{lo, 0xffffffffu};  // no weight to choose by
    target = target - before < all ? target - before : all - 1;
    const uint64_t last = select(sh, key, ones, tight(lo, false), tight(hi, true), target);
    return Cut{order_of(last), place_of(last)};
  }

  // The place of the nth (from 0) logit of one value.
  __device__ __forceinline__ uint32_t nth_equal(uint32_t key, uint64_t nth, const Cut& limit) {
    const int lane = threadIdx.x & 63, wave = spruce::uniform(threadIdx.x >> 6);
    for (int s = 0; s < steps; ++s) {
      const int at = (s * kThreads + (int)threadIdx.x) * kChunk;
      float x[kChunk];
      decode(row.load(at), x);
      int c = 0;
#pragma unroll
      for (int i = 0; i < kChunk; ++i) c += x[i] > -INFINITY && ordered(x[i]) == key && within(limit, key, at + i);
      const int all = wave_prefix(c);
      if (lane == 63) sh.part[s * kRowWaves + wave] = (uint64_t)all;
    }
    uint64_t before;
    const int part = find_part(nth, before);  // (the last of them where there are no more than nth)
    if (wave == 0) {
      const int at = part * kPart + lane * kChunk;
      float x[kChunk];
      decode(row.load(at), x);
      int c = 0;
      bool is[kChunk];
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        is[i] = x[i] > -INFINITY && ordered(x[i]) == key && within(limit, key, at + i);
        c += is[i];
      }
      uint64_t upto = before + (uint64_t)(wave_prefix(c) - c);
#pragma unroll
      for (int i = 0; i < kChunk; ++i) {
        if (is[i] && upto == nth) sh.result[0] = (uint64_t)(at + i);
        upto += is[i];
      }
    }
    __syncthreads();
    const uint32_t place = (uint32_t)sh.result[0];
    __syncthreads();
    return place;
  }

  // The first of the sums with which they are above `target`, and what is before it.  A target past them all
  // becomes the last within them.
  __device__ __forceinline__ int find_part(uint64_t& target, uint64_t& before) {
    const int n = steps * kRowWaves;
    constexpr int EACH = kParts / kThreads;
    __syncthreads();
    uint64_t v[EACH], mine = 0, all;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int at = EACH * threadIdx.x + i;
      v[i] = at < n ? sh.part[at] : 0;
      mine += v[i];
    }
    uint64_t upto = block_prefix(sh, mine, all) - mine;
    if (target >= all) target = all - 1;
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

// floor(u times a sum), below it.
__device__ __forceinline__ uint64_t drawn(double u, uint64_t total) {
  const double wanted = (u > 0.0 ? u : 0.0) * (double)total;
  return wanted < (double)(total - 1) ? (uint64_t)wanted : total - 1;
}

// A row's settings.
struct Settings {
  double temperature, top_p, min_p, u;
  int64_t top_k;
  bool by_k, by_p;
  __device__ __forceinline__ void init(const Sampling& p, int b) {
    temperature = p.temperature ? (double)p.temperature[b] : p.temperature1;
    top_k = p.top_k ? (int64_t)p.top_k[b] : p.top_k1;
    top_p = p.top_p ? (double)p.top_p[b] : p.top_p1;
    min_p = p.min_p ? (double)p.min_p[b] : p.min_p1;
    min_p = min_p < 1.0 ? min_p : 1.0;
    u = p.uniform64 ? static_cast<const double*>(p.uniform)[b] : (double)static_cast<const float*>(p.uniform)[b];
    by_k = top_k > 0 && top_k < p.V;
    by_p = top_p < 1.0;
  }
  // Of rows that parts share.
  __device__ __forceinline__ void init_shared(const Sampling& p, int b) {
    init(p, b);
    by_k = false;
    min_p = 0.0;
  }
};

template <typename T>
__device__ __forceinline__ void set_up(Sampler<T>& s, const Sampling& p, int b) {
  s.row.init(p.logits, (int64_t)b * p.stride, p.V);
  s.begin = 0;
  s.steps = (s.row.end + kThreads * kChunk - 1) / (kThreads * kChunk);
  s.infinite = false;
}
// Of a part of the row alone: what is behind it counts as behind the row.
template <typename T>
__device__ __forceinline__ void set_up(Sampler<T>& s, const Sampling& p, int b, int part) {
  set_up(s, p, b);
  s.begin = part * p.part_places;
  const int end = s.begin + p.part_places;
  s.row.end = end < s.row.end ? end : s.row.end;
  s.steps = s.row.end > s.begin ? (s.row.end - s.begin + kThreads * kChunk - 1) / (kThreads * kChunk) : 0;
}
__device__ __forceinline__ void fill_table(Shared& sh) {
  if (threadIdx.x < kTable) {
    const uint64_t power = __builtin_bit_cast(uint64_t, exp2((double)threadIdx.x / kTable));
    sh.table[threadIdx.x] = uint2{(uint32_t)power, (uint32_t)(power >> 32) - (threadIdx.x << 14)};
  }
}

template <typename T>
__device__ __forceinline__ void set_weights(Sampler<T>& s, const Sampling& p, double temperature, float top) {
  s.top = uniform(top);
  // (An infinite temperature: all weights one, but those of -inf.)
  const double inv = fmin(fmax(1.0 / temperature, 1e-300), 1e+300);
  constexpr double kLog2e = 1.44269504088896340736;
  s.w = Weights{uniform((double)top), uniform(kTable * kLog2e * inv), uniform(-60.0 / (kLog2e * inv)), p.shift,
                s.sh.table};
  // Bins of equal width down to where weights end.
  const float range = (float)(kNothing / (kLog2e * inv));
  s.per_bin = uniform((float)(kBins - 1) / (range > 1e-30f ? (range < 1e30f ? range : 1e30f) : 1e-30f));
}

// The weights of eight logits, zero where they are not kept.
template <typename T>
__device__ __forceinline__ void weights_at(const Sampler<T>& s, const Settings& set, const Cut& cut,
                                           const float (&x)[kChunk], int at, double (&weight)[kChunk]) {
  s.w.of8(x, weight);
  if (cut.key) {
    const float end = unordered(cut.key);
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
      if (!((x[j] > end) | ((x[j] == end) & ((uint32_t)(at + j) <= cut.last)))) weight[j] = 0.0;
  }
  if (set.min_p > 0.0) {
#pragma unroll
    for (int j = 0; j < kChunk; ++j)
      if (weight[j] < set.min_p) weight[j] = 0.0;
  }
}

// The kept weights' sums of 512 logits each.
template <typename T, typename F>
__device__ __forceinline__ void sum_up(const Sampler<T>& s, const Settings& set, const Cut& cut, F store) {
  const int lane = threadIdx.x & 63, most = (s.begin + s.steps * kThreads * kChunk) / kPart;
  const float end = unordered(cut.key);
  s.template chunks<2>([&](const float (&x)[kChunk], int at) {
    uint64_t sum = 0;
    if (cut.key == 0 || __ballot(s.largest(x) >= end)) {
      double weight[kChunk];
      weights_at(s, set, cut, x, at, weight);
      // (What the units are rounded against is taken off once.)
#pragma unroll
      for (int j = 0; j < kChunk; ++j) sum += __builtin_bit_cast(uint64_t, weight[j] + s.w.shift);
      sum -= kChunk * __builtin_bit_cast(uint64_t, s.w.shift);
    }
    const int64_t upto = wave_prefix((int64_t)sum);
    if (lane == 63 && at / kPart < most) store(at / kPart, (uint64_t)upto);
  });
}

// The draw from the row's sums in LDS.
template <typename T>
__device__ __forceinline__ void draw_summed(Shared& sh, Sampler<T>& s, const Sampling& p, const Settings& set,
                                            const Cut& cut, int b) {
  const int tid = threadIdx.x, lane = tid & 63, wave = spruce::uniform(tid >> 6);
  __syncthreads();
  uint64_t a = 0, total, before;
  for (int i = tid; i < s.steps * kRowWaves; i += kThreads) a += sh.part[i];
  block_prefix(sh, a, total);
  uint64_t target = drawn(set.u, total);
  const int part = s.find_part(target, before);
  if (wave != 0) return;
  const int at = part * kPart + lane * kChunk;
  float x[kChunk];
  s.decode(s.row.load(at), x);
  double weight[kChunk];
  uint64_t units[kChunk], sum = 0;
  weights_at(s, set, cut, x, at, weight);
#pragma unroll
  for (int j = 0; j < kChunk; ++j) sum += units[j] = s.w.units(weight[j]);
  uint64_t upto = before + (uint64_t)wave_prefix((int64_t)sum) - sum;
#pragma unroll
  for (int j = 0; j < kChunk; ++j) {
    if (upto <= target && target < upto + units[j]) {
      p.tokens[b] = at + j - s.row.first;
      if (p.logprobs) p.logprobs[b] = (float)log(s.w.of(x[j]) / ((double)total * (p.shift * 0x1p-52)));
    }
    upto += units[j];
  }
}

// A row that keeps more than the list holds, by one workgroup.  A function of its own, which sets
// everything up again: what it would keep in registers pushed the usual way's out of them.  (And one for each
// of its two callers: with both, 74 us of sample_kernel were 79.)
template <typename T, bool SHARED>
__device__ __attribute__((noinline)) void sample_far(uint64_t args, __attribute__((address_space(3))) Shared* lds) {
  const Sampling p = *(const Sampling*)(const __attribute__((address_space(4))) Sampling*)lane_of((int64_t)args, 0);
  Shared& sh = *(Shared*)lds;
  const int b = (int)blockIdx.x, tid = threadIdx.x;
  Settings set;
  set.init(p, b);
  Sampler<T> s{sh};
  set_up(s, p, b);
  __syncthreads();
  s.infinite = spruce::uniform(sh.infinite) != 0;
  set_weights(s, p, set.temperature, sh.top);
  Cut cut{0, 0xffffffffu};  // all
  int bin = spruce::uniform(sh.bin);
  uint64_t total = sh.total, before = sh.before;
  if (set.by_k) {
    const uint64_t target = (uint64_t)set.top_k - 1;
    uint64_t all = total;
    if (bin < 0) {
      s.count();
      before = 0;
      bin = s.find_bin(target, before, all);
    }
    if (target < all) cut = s.resolve(bin, true, target, before, cut);  // else all there are
    if (set.by_p) {
      s.weigh(cut);
      before = 0;
      uint64_t mine = sh.weight[tid] + sh.weight[tid + kThreads];
      block_prefix(sh, mine, total);
      bin = s.find_bin(target_of(fmax(set.top_p, 0.0) * (double)total), before, all);
    }
  }
  if (set.by_p) cut = s.resolve(bin, false, target_of(fmax(set.top_p, 0.0) * (double)total), before, cut);
  sum_up(s, set, cut, [&](int i, uint64_t sum) { sh.part[i] = sum; });
  draw_summed(sh, s, p, set, cut, b);
}

// The largest logit of the sampler's places: its order << 32 | ~place of its chunk, 0 for none; and this thread's
// own.
template <typename T>
__device__ __forceinline__ uint64_t largest_logit(Shared& sh, const Sampler<T>& s, float& most) {
  const int lane = threadIdx.x & 63, wave = spruce::uniform(threadIdx.x >> 6);
  most = -INFINITY;
  int place = 0;
  s.template chunks<4>([&](const float (&x)[kChunk], int at) {
    const float m = s.largest(x);
    place = m > most ? at : place;
    most = fmaxf(most, m);
  });
  uint64_t best = most > -INFINITY ? (uint64_t)ordered(most) << 32 | (uint32_t)~place : 0;
#pragma unroll
  for (int i = 1; i < 64; i <<= 1) {
    const uint64_t o = __shfl_xor(best, i);
    best = o > best ? o : best;
  }
  if (lane == 0) sh.waves[wave] = best;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowWaves; ++i) best = sh.waves[i] > best ? sh.waves[i] : best;
  __syncthreads();
  return best;
}

// The token of a row with nothing to choose: the first of its largest logits, or -1.
template <typename T>
__device__ __forceinline__ void take_largest(const Sampler<T>& s, const Sampling& p, uint64_t best, int b) {
  if (threadIdx.x != 0) return;
  int64_t token = -1;
  if (best != 0) {
    float x[kChunk];
    const int at = (int)~(uint32_t)best;
    Row<T>::decode(s.row.load(at), x);
#pragma unroll
    for (int i = kChunk - 1; i >= 0; --i)
      if (x[i] == unordered((uint32_t)(best >> 32))) token = at + i - s.row.first;
  }
  p.tokens[b] = token;
  if (p.logprobs) p.logprobs[b] = best == 0 ? -INFINITY : 0.f;
}

// What a row's list begins with by min_p, a little lower than it is, for the roundings: a weight's own, of
// less than 2^-43, is all that counts where the temperature is so high, or min_p so near to one, that weights do not
// tell logits apart.
template <typename T>
__device__ __forceinline__ float least_by_share(const Sampler<T>& s, double min_p) {
  const float bound = s.top + (float)((log(min_p) * 1.000001 - 0x1p-40) * (kTable * 1.44269504088896340736) / s.w.steps);
  return fmaxf(-3.402823466e+38f, bound - (fabsf(bound) + fabsf(s.top)) * 0x1p-20f);
}

// The ends and the draw of a row whose kept logits are all in LDS: those from `low` on.
// total: all weights, where the ends go by them alone.
template <typename T>
__device__ __forceinline__ void draw_listed(Shared& sh, const Sampler<T>& s, const Sampling& p, const Settings& set,
                                            float low, uint64_t total, int b) {
  const int lane = threadIdx.x & 63, wave = spruce::uniform(threadIdx.x >> 6);
  const uint32_t n = sh.size;
  auto done = [&](uint32_t place, double weight, uint64_t sum) {
    p.tokens[b] = (int64_t)(place - (uint32_t)s.row.first);
    if (p.logprobs) p.logprobs[b] = (float)log(weight / ((double)sum * (p.shift * 0x1p-52)));
  };
  if (n <= 64) {
    // One wave: an entry a lane, its rank and the weight before it by comparison with all.
    if (wave != 0) return;
    const uint64_t mine = lane < (int)n ? sh.list[lane] : 0;
    const double exact = lane < (int)n ? s.w.of(unordered((uint32_t)(mine >> 32))) : 0.0;
    uint64_t units = s.w.units(exact);
    sh.weight[lane] = units;
    wave_lds_fence();
    uint32_t rank = 0;
    uint64_t before = 0;
    if (set.by_k || set.by_p) {
#pragma unroll 8
      for (uint32_t j = 0; j < n; ++j) {
        const bool first = sh.list[j] > mine;
        rank += first;
        before += first ? sh.weight[j] : 0;
      }
      if (set.by_k && rank >= set.top_k) units = 0;
      if (set.by_p) {
        const uint64_t all = (uint64_t)lane_of(wave_prefix((int64_t)units), 63);
        if (before > target_of(fmax(set.top_p, 0.0) * (double)(set.by_k ? all : total))) units = 0;
      }
    }
    if (!(exact >= set.min_p)) units = 0;
    const uint64_t sum = (uint64_t)lane_of(wave_prefix((int64_t)units), 63), target = drawn(set.u, sum);
    wave_lds_fence();
    sh.weight[lane] = units;
    wave_lds_fence();
    before = 0;
#pragma unroll 8
    for (uint32_t j = 0; j < n; ++j) before += (uint32_t)sh.list[j] > (uint32_t)mine ? sh.weight[j] : 0;
    if (before <= target && target < before + units) done(~(uint32_t)mine, exact, sum);
    return;
  }
  uint64_t key[kEach], units[kEach], weight[kEach], sum = 0;
  double exact[kEach];
  s.entries(key);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    exact[i] = key[i] ? s.w.of(unordered((uint32_t)(key[i] >> 32))) : 0.0;
    units[i] = s.w.units(exact[i]);
    weight[i] = key[i] ? 1 : 0;
    key[i] = s.tight(key[i]);
  }
  // The ends by count and by weight, then the draw: three selections.
  const uint64_t lowest = s.tight(ordered(low), false), highest = s.tight(ordered(s.top), true);
  for (int turn = set.by_k && (uint64_t)set.top_k < n ? 0 : (set.by_p ? 1 : 2);; turn = turn == 0 && set.by_p ? 1 : 2) {
    uint64_t target = (uint64_t)set.top_k - 1;
    if (turn > 0) {
      sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        if (turn == 2) {
          if (!(exact[i] >= set.min_p)) units[i] = 0;
          key[i] &= s.kPlace;  // goes down as the place goes up
        }
        weight[i] = units[i];
        sum += units[i];
      }
      block_prefix(sh, sum, sum);
      target = turn == 2 ? drawn(set.u, sum) : target_of(fmax(set.top_p, 0.0) * (double)(set.by_k ? sum : total));
      if (target >= sum) target = sum - 1;
    }
    const uint64_t found = turn == 2 ? select(sh, key, weight, s.kPlace - s.row.end, s.kPlace, target)
                                     : select(sh, key, weight, lowest, highest, target);
    if (turn == 2) {
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (units[i] && key[i] == found) done(s.place_of(found), exact[i], sum);
      return;
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i)
      if (key[i] < found) units[i] = 0;
  }
}

// The bound of a row's (or a part's) list by top_k, from the threads' own largest: at least so many threads have
// a logit in that bin or above; everything where fewer have any.
template <typename T>
__device__ __forceinline__ float least_by_rank(Shared& sh, Sampler<T>& s, int64_t top_k, float most) {
  s.clear_bins();
  if (most > -INFINITY) atomicAdd((unsigned long long*)&sh.weight[s.bin_of(most)], 1ull);
  __syncthreads();
  uint64_t before = 0, all;
  uint64_t mine = sh.weight[threadIdx.x] + sh.weight[threadIdx.x + kThreads];
  block_prefix(sh, mine, all);
  if ((uint64_t)top_k > all) return -3.402823466e+38f;
  return s.bin_end(s.find_bin((uint64_t)top_k - 1, before, all));
}

// A row by one workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.x, tid = threadIdx.x;
  Settings set;
  set.init(p, b);
  Sampler<T> s{sh};
  set_up(s, p, b);
  fill_table(sh);
  float most;
  const uint64_t best = largest_logit(sh, s, most);
  if (best == 0 || !(set.temperature > 0)) {
    take_largest(s, p, best, b);
    return;
  }
  s.infinite = unordered((uint32_t)(best >> 32)) == INFINITY;
  if (s.infinite) most = most == INFINITY ? 0.f : -INFINITY;
  set_weights(s, p, set.temperature, s.infinite ? 0.f : unordered((uint32_t)(best >> 32)));

  // The list: everything from `low` on.
  uint64_t total = 0, before = 0;
  int bin = -1;
  float low = -3.402823466e+38f;
  bool far = false;
  if (set.by_k && set.top_k <= kThreads / 2) {
    low = least_by_rank(sh, s, set.top_k, most);
  } else if (set.by_k) {
    s.count();
    bin = s.find_bin((uint64_t)set.top_k - 1, before, total);
    low = s.bin_end(bin);
  } else if (set.by_p) {
    s.weigh(Cut{0, 0xffffffffu});
    uint64_t mine = sh.weight[tid] + sh.weight[tid + kThreads];
    block_prefix(sh, mine, total);
    bin = s.find_bin(target_of(fmax(set.top_p, 0.0) * (double)total), before, mine);
    low = s.bin_end(bin);
  } else if (set.min_p > 0.0) {
    low = least_by_share(s, set.min_p);
  } else {
    far = true;
  }
  if (!far) far = !s.collect(low, INFINITY, Cut{0, 0xffffffffu});
  if (!far) {
    draw_listed(sh, s, p, set, low, total, b);
    return;
  }
  if (tid == 0) {
    sh.top = s.top;
    sh.infinite = s.infinite;
    sh.bin = bin;
    sh.before = before;
    sh.total = total;
  }
  sample_far<T, false>((uint64_t)__builtin_amdgcn_kernarg_segment_ptr(), (__attribute__((address_space(3))) Shared*)&sh);
}

// ------------------------------------------------------------------ rows by more than one workgroup
// Rows without top_k and min_p, whose lists are long or none: the same steps, the passes over a row part by part, a
// launch each.  (An instruction on each of 150016 logits is a microsecond of one workgroup.  Steps between them in
// whichever workgroup of a row is done last need every wave's stores written back from its L2 before: top_p 0.95 of
// bf16 [64, 150016] took 258 us so, 89 in launches of their own.)

template <typename T>
__global__ __launch_bounds__(kThreads) void part_largest_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.y, part = (int)blockIdx.x;
  Sampler<T> s{sh};
  set_up(s, p, b, part);
  float most;
  const uint64_t best = largest_logit(sh, s, most);
  if (threadIdx.x == 0) p.best[(int64_t)b * p.parts + part] = best;
  if (part == 0 && threadIdx.x == 0) p.states[b] = RowState{kSummed, 0, 0, 0, 0.f, 0.f, 0, 0xffffffffu};
}

// Sets a part up behind its row's largest logit; the largest, 0 where there is none.
template <typename T>
__device__ __forceinline__ uint64_t set_up_behind(Sampler<T>& s, const Sampling& p, const Settings& set, int b, int part) {
  set_up(s, p, b, part);
  uint64_t best = 0;
  for (int i = 0; i < p.parts; ++i) {
    const uint64_t x = p.best[(int64_t)b * p.parts + i];
    best = x > best ? x : best;
  }
  if (best == 0 || !(set.temperature > 0)) return best;
  s.infinite = unordered((uint32_t)(best >> 32)) == INFINITY;
  set_weights(s, p, set.temperature, s.infinite ? 0.f : unordered((uint32_t)(best >> 32)));
  fill_table(s.sh);
  __syncthreads();
  return best;
}
// The whole row in its place.
template <typename T>
__device__ __forceinline__ void widen(Sampler<T>& s, const Sampling& p, int b) {
  const bool infinite = s.infinite;
  set_up(s, p, b);
  s.infinite = infinite;
}

// The weights' histogram.
template <typename T>
__global__ __launch_bounds__(kThreads) void part_weights_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.y, part = (int)blockIdx.x, tid = threadIdx.x;
  Settings set;
  set.init_shared(p, b);
  if (!set.by_p) return;
  Sampler<T> s{sh};
  const uint64_t best = set_up_behind(s, p, set, b, part);
  if (best == 0 || !(set.temperature > 0)) return;
  s.weigh(Cut{0, 0xffffffffu});
  uint64_t* hists = p.hists + (int64_t)b * p.parts * kBins;
#pragma unroll
  for (int i = 0; i < 2; ++i) hists[(int64_t)part * kBins + tid + i * kThreads] = sh.weight[tid + i * kThreads];
}

// The bin of the end by top_p, and the lists of what is before it and in it, or of the bin alone.
template <typename T>
__global__ __launch_bounds__(kThreads) void part_list_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.y, part = (int)blockIdx.x, tid = threadIdx.x;
  Settings set;
  set.init_shared(p, b);
  if (!set.by_p) return;
  Sampler<T> s{sh};
  const uint64_t best = set_up_behind(s, p, set, b, part);
  if (best == 0 || !(set.temperature > 0)) return;
  const uint64_t* hists = p.hists + (int64_t)b * p.parts * kBins;
  uint64_t h0 = 0, h1 = 0;
#pragma unroll 4
  for (int i = 0; i < p.parts; ++i) {
    h0 += hists[(int64_t)i * kBins + tid];
    h1 += hists[(int64_t)i * kBins + tid + kThreads];
  }
  sh.weight[tid] = h0;
  sh.weight[tid + kThreads] = h1;
  uint64_t total, before = 0, all;
  block_prefix(sh, h0 + h1, total);
  const int bin = s.find_bin(target_of(fmax(set.top_p, 0.0) * (double)total), before, all);
  // About as many logits are before the bin or in it: a list of them all is not tried if they are too many.
  uint64_t many = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = tid + i * kThreads;
    if (at <= bin) many += (uint64_t)((double)(i ? h1 : h0) / (double)(s.w.units(s.w.of(s.top - (float)at / s.per_bin)) + 1));
  }
  block_prefix(sh, many, many);
  const float low = s.bin_end(bin), high = bin == 0 ? INFINITY : unordered(ordered(s.bin_end(bin - 1)) - 1);
  if (part == 0 && tid == 0) p.states[b] = RowState{kWeighed, bin, before, total, low, high, 0, 0xffffffffu};
  int kind = kWhole;
  if (many > kList || !s.collect(low, INFINITY, Cut{0, 0xffffffffu}))
    kind = s.collect(low, high, Cut{0, 0xffffffffu}) ? kMembers : kTooMany;
  const int64_t at = (int64_t)b * p.parts + part;
  const uint32_t n = kind == kTooMany ? 0 : sh.size;
  for (uint32_t i = tid; i < n; i += kThreads) p.lists[at * kList + i] = sh.list[i];
  if (tid == 0) p.part_list[at] = PartList{n, kind};
}

// The end of a row whose parts have left their lists: the draw, where they hold all that is kept; the end by
// weight, where they hold its bin; by this workgroup alone everything where they do not.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_end_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.x, tid = threadIdx.x;
  const RowState state = p.states[b];
  if (state.stage != kWeighed) return;
  Settings set;
  set.init_shared(p, b);
  Sampler<T> s{sh};
  set_up_behind(s, p, set, b, 0);
  widen(s, p, b);
  const PartList* lists = p.part_list + (int64_t)b * p.parts;
  int worst = kWhole;
  uint32_t all = 0;
  for (int i = 0; i < p.parts; ++i) {
    const PartList x = lists[i];
    worst = x.kind > worst ? x.kind : worst;
    if (tid == 0) sh.starts[i] = all;
    all += x.size;
  }
  const bool listed = worst == kWhole && all <= kList;
  bool members = !listed && worst != kTooMany;
  const uint32_t most = ordered(members ? state.high : INFINITY);
  if (tid == 0) sh.size = 0;
  __syncthreads();
  if (listed || members) {
    for (uint32_t i = 0; i < all; i += kThreads * 4) {
      uint64_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = i + j * kThreads + tid;
        int part = 0;
        for (int k = 1; k < p.parts; ++k) part = sh.starts[k] <= at ? k : part;
        x[j] = at < all ? p.lists[((int64_t)b * p.parts + part) * kList + (at - sh.starts[part])] : 0;
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = x[j] && (uint32_t)(x[j] >> 32) <= most;
        const uint64_t mask = __ballot(in);
        if (mask == 0) continue;
        uint32_t to = 0;
        if ((tid & 63) == 0) to = atomicAdd(&sh.size, (uint32_t)__builtin_popcountll(mask));
        to = (uint32_t)lane_of((int)to, 0) + (uint32_t)__builtin_popcountll(mask & ((1ull << (tid & 63)) - 1));
        if (in && to < kList) sh.list[to] = x[j];
      }
    }
    __syncthreads();
    members = members && sh.size <= kList;
  }
  if (listed) {
    draw_listed(sh, s, p, set, state.low, state.total, b);
    return;
  }
  if (members) {
    const uint64_t target = target_of(fmax(set.top_p, 0.0) * (double)state.total);
    const Cut cut = s.end_among(false, target, state.before, ordered(state.low), most);
    if (tid == 0) {
      p.states[b].cut_key = cut.key;
      p.states[b].cut_last = cut.last;
      p.states[b].stage = kSummed;
    }
    return;
  }
  if (tid == 0) {
    sh.top = s.top;
    sh.infinite = s.infinite;
    sh.bin = state.bin;
    sh.before = state.before;
    sh.total = state.total;
  }
  sample_far<T, true>((uint64_t)__builtin_amdgcn_kernarg_segment_ptr(), (__attribute__((address_space(3))) Shared*)&sh);
}

// The sums of rows whose ends are known.
template <typename T>
__global__ __launch_bounds__(kThreads) void part_sums_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.y, part = (int)blockIdx.x;
  const RowState state = p.states[b];
  if (state.stage != kSummed) return;
  Settings set;
  set.init_shared(p, b);
  Sampler<T> s{sh};
  const uint64_t best = set_up_behind(s, p, set, b, part);
  if (best == 0 || !(set.temperature > 0)) return;
  uint64_t* sums = p.sums + (int64_t)b * kParts;
  sum_up(s, set, Cut{state.cut_key, state.cut_last}, [&](int i, uint64_t sum) { sums[i] = sum; });
}

// The draw by them.
template <typename T>
__global__ __launch_bounds__(kThreads) void row_draw_kernel(const Sampling p) {
  __shared__ Shared sh;
  const int b = (int)blockIdx.x;
  const RowState state = p.states[b];
  if (state.stage != kSummed) return;
  Settings set;
  set.init_shared(p, b);
  Sampler<T> s{sh};
  const uint64_t best = set_up_behind(s, p, set, b, 0);
  widen(s, p, b);
  if (best == 0 || !(set.temperature > 0)) {
    take_largest(s, p, best, b);
    return;
  }
  for (int i = threadIdx.x; i < s.steps * kRowWaves; i += kThreads)
    sh.part[i] = i * kPart < s.row.end ? p.sums[(int64_t)b * kParts + i] : 0;
  draw_summed(sh, s, p, set, Cut{state.cut_key, state.cut_last}, b);
}

struct SamplePlan {
  int64_t parts, places;  // 1: a workgroup a row
  int64_t best, hists, lists, part_list, sums, states;
  int64_t bytes() const { return best + hists + lists + part_list + sums + states; }
};
// Parts of whole steps of a workgroup, a workgroup a CU at the most.
SamplePlan sample_plan(int64_t B, int64_t V, bool by_p) {
  constexpr int64_t kStep = kThreads * kChunk;
  SamplePlan plan{};
  const int64_t steps = (V + 7 + kStep - 1) / kStep;
  int64_t parts = V >= (by_p ? kLeastByP : kLeastPlain) ? kSharers / B : 1;
  if (parts > kMostParts) parts = kMostParts;
  if (parts > steps) parts = steps;
  if (parts < 2) {
    plan.parts = 1;
    return plan;
  }
  const int64_t each = (steps + parts - 1) / parts;
  plan.parts = (steps + each - 1) / each;
  plan.places = each * kStep;
  const int64_t all = B * plan.parts;
  plan.best = (all * 8 + 15) / 16 * 16;
  plan.hists = all * kBins * 8;
  plan.lists = all * kList * 8;
  plan.part_list = (all * (int64_t)sizeof(PartList) + 15) / 16 * 16;
  plan.sums = B * kParts * 8;
  plan.states = B * (int64_t)sizeof(RowState);
  return plan;
}

template <typename T>
void launch_parts(const Sampling& p, int64_t B, bool ends, hipStream_t st) {
  const dim3 parts((unsigned)p.parts, (unsigned)B), rows((unsigned)B), threads(kThreads);
  hipLaunchKernelGGL(part_largest_kernel<T>, parts, threads, 0, st, p);
  if (ends) {
    hipLaunchKernelGGL(part_weights_kernel<T>, parts, threads, 0, st, p);
    hipLaunchKernelGGL(part_list_kernel<T>, parts, threads, 0, st, p);
    hipLaunchKernelGGL(row_end_kernel<T>, rows, threads, 0, st, p);
  }
  hipLaunchKernelGGL(part_sums_kernel<T>, parts, threads, 0, st, p);
  hipLaunchKernelGGL(row_draw_kernel<T>, rows, threads, 0, st, p);
}

}  // namespace
}  // namespace spruce

using namespace spruce;

extern "C" int64_t spruce_sample_tokens_workspace_bytes(int64_t B, int64_t V, int64_t by_p) {
  return B < 1 || V < 1 || B >= (int64_t)1 << 30 || V >= (int64_t)1 << 31 ? 0 : sample_plan(B, V, by_p != 0).bytes();
}

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
  SPRUCE_REQUIRE(a.B <= kGridX, "too many rows for one call");
  const bool by_k = a.top_k || (a.top_k1 > 0 && a.top_k1 < a.V), by_p = a.top_p || a.top_p1 < 1;
  const bool by_share = a.min_p || a.min_p1 > 0, greedy = !a.temperature && a.temperature1 == 0;
  SamplePlan plan{};
  if (!by_k && !by_share && !greedy) plan = sample_plan(a.B, a.V, by_p);
  SPRUCE_REQUIRE(plan.bytes() == 0 || (a.workspace && a.workspace_bytes >= plan.bytes()),
                 "workspace too small: %lld bytes, need %lld", (long long)a.workspace_bytes, (long long)plan.bytes());
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace must be 16-byte aligned");
  const hipStream_t st = (hipStream_t)stream;
  if (plan.parts > 1) {
    char* work = static_cast<char*>(a.workspace);
    p.parts = (int)plan.parts;
    p.part_places = (int)plan.places;
    p.best = reinterpret_cast<uint64_t*>(work);
    p.hists = reinterpret_cast<uint64_t*>(work += plan.best);
    p.lists = reinterpret_cast<uint64_t*>(work += plan.hists);
    p.part_list = reinterpret_cast<PartList*>(work += plan.lists);
    p.sums = reinterpret_cast<uint64_t*>(work += plan.part_list);
    p.states = reinterpret_cast<RowState*>(work += plan.sums);
    switch (a.dtype) {
      case SPRUCE_DTYPE_BF16: launch_parts<InBF16>(p, a.B, by_p, st); break;
      case SPRUCE_DTYPE_F16: launch_parts<InF16>(p, a.B, by_p, st); break;
      default: launch_parts<InF32>(p, a.B, by_p, st); break;
    }
    return check_launch("token sampling");
  }
  const dim3 grid((unsigned)a.B);
  switch (a.dtype) {
    case SPRUCE_DTYPE_BF16: hipLaunchKernelGGL(sample_kernel<InBF16>, grid, dim3(kThreads), 0, st, p); break;
    case SPRUCE_DTYPE_F16: hipLaunchKernelGGL(sample_kernel<InF16>, grid, dim3(kThreads), 0, st, p); break;
    default: hipLaunchKernelGGL(sample_kernel<InF32>, grid, dim3(kThreads), 0, st, p); break;
  }
  return check_launch("token sampling");
}
