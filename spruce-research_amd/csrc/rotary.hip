// Per-head norms and rotary positions of queries and keys, in place of a
// model's own elementwise passes, and the same on the way into a paged cache.
//
// For a head row x of D values at position p, with w the norm's weights:
//   y = x * (mean(x^2) + eps)^(-1/2) * w            (y = x without a norm)
//   (a, b) <- s * (a cos t_i - b sin t_i, b cos t_i + a sin t_i),
//   t_i = p * inv_freq[i],  i < R / 2
// over the pairs (a, b) = (y_i, y_{i + R/2}) of the half layout or
// (y_{2i}, y_{2i+1}) of the interleaved one; y_R.. stay as they are.
//
// An angle in 32 bits is off by up to p * 2^-24 radians, 0.06 at p = 10^6, so
// t_i / (2 pi) is formed in 64 bits and its fraction alone goes to 32; all
// else is 32-bit, rounded once.
//
// Bytes bound it (each value read and written once).  A wave owns one token,
// or some of its heads where tokens are few: its lanes work out one pair's sine
// and cosine each, once for all heads, and hand them over through LDS; then
// D/16 lanes take a head row, 16 values a lane chosen so that both members of
// every pair are in the lane.  The rows of four passes (two of float32) are in
// flight before the look-ups (sequence, position, page) and the sines begin.
//
// Measured on one MI355X: 32768 tokens of 28 + 4 heads of 128, normed, bf16, 103 us
// (5.23 TB/s); the append of 16384 tokens of 32 + 8 + 8 heads 80 us (5.05 TB/s), 162 in float32; 8170
// tokens of 16 + 8 heads of 64 in float32, interleaved, 25 us (4.0 TB/s); one token of each of
// 64 sequences 4.9 us of kernel.  (Weights kept in LDS instead of registers: 119 us for 114.)
#include "paged.h"

using namespace spruce;

namespace {

struct RotaryRows {
  const void* src;
  void* dst;
  int64_t ss[3], ds[3];  // batch, head, token strides; of pages: page, head, slot
  int heads;
};

struct RotaryParams {
  RotaryRows q, k, v;    // v only with PAGED, whose k and v go to the pages
  const void* positions;  // int32 or int64
  int64_t pos_stride;    // per batch
  int pos64;
  const double* inv_freq;
  int rot, interleaved;
  float factor;
  const void* q_weight;
  const void* k_weight;
  int weight_f32;
  float eps;
  int tokens;    // per batch
  int64_t rows;  // batches * tokens
  int groups;    // waves that share a token's passes
  PagedBatch batch;
};

constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Eight values as they lie in memory.
template <int EB>
struct Raw8 {
  u32x4 w[EB / 2];
};
template <int EB, bool PAST = false>
__device__ __forceinline__ Raw8<EB> raw8(const char* p) {
  Raw8<EB> r;
#pragma unroll
  for (int i = 0; i < EB / 2; ++i) {
    const u32x4* at = reinterpret_cast<const u32x4*>(p) + i;
    r.w[i] = PAST ? __builtin_nontemporal_load(at) : *at;
  }
  return r;
}

template <int EB, bool F16>
__device__ __forceinline__ void widen8(const Raw8<EB>& r, float* v) {
  if constexpr (EB == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __builtin_bit_cast(float, (uint32_t)r.w[i >> 2][i & 3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = unpack1<F16>(r.w[0][i] & 0xffffu);
      v[2 * i + 1] = unpack1<F16>(r.w[0][i] >> 16);
    }
  }
}

template <int EB, bool F16, bool PAST>
__device__ __forceinline__ void store8(char* p, const float* v) {
  if constexpr (PAST) {
    static_assert(EB == 2, "16-byte pieces");
    __builtin_nontemporal_store(
        u32x4{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7])},
        reinterpret_cast<u32x4*>(p));
  } else if constexpr (EB == 4) {
    reinterpret_cast<float4*>(p)[0] = float4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<float4*>(p)[1] = float4{v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<u32x4*>(p) =
        u32x4{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7])};
  }
}

// PAST: rows go past the caches (see launch_rotary).
// Four waves a SIMD for every type: at five the float32 append kept 22 registers
// in scratch (16384 tokens of 32 + 8 + 8 heads of 128 176 us rather than 162, 8192 of
// 16 + 8 + 8 heads of 64 47 rather than 38), and the float32 rotation was no faster.
template <int EB, bool F16, int D, bool PAGED, bool PAST>
__global__ __launch_bounds__(256, 4) void head_rotary_kernel(const RotaryParams p) {
  constexpr int LPH = D / 16, HPW = 64 / LPH;  // lanes of a head row, head rows of a pass
  constexpr int kFlight = 8 / EB;              // passes in flight: 32 registers
  __shared__ float2 turns[4][D / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)flat_block() * 4 + wave;
  int64_t row = item;
  int grp = 0;
  if (p.groups > 1) {  // few tokens: the product fits 32 bits
    row = (uint32_t)item / (uint32_t)p.groups;
    grp = (int)((uint32_t)item - (uint32_t)row * (uint32_t)p.groups);
  }
  if (row >= p.rows) return;  // no barrier below
  int b = 0, t = (int)row;
  if (!PAGED && p.rows > p.tokens) {
    b = (int)(row / p.tokens);
    t = (int)(row - (int64_t)b * p.tokens);
  }
  const int j = lane % LPH;
  const bool turned = j < p.rot / 16;
  const int e0 = turned && !p.interleaved ? 8 * j : 16 * j;
  const int e1 = turned && !p.interleaved ? 8 * j + p.rot / 2 : 16 * j + 8;

  // Passes of HPW heads each: the queries', the keys', the values'.
  const int nq = (p.q.heads + HPW - 1) / HPW, nk = (p.k.heads + HPW - 1) / HPW;
  const int passes = nq + nk + (PAGED ? nk : 0);
  const int per = (passes + p.groups - 1) / p.groups;
  const int first = grp * per, last = first + per < passes ? first + per : passes;
  auto rows_of = [&](int pass) -> const RotaryRows& { return pass < nq ? p.q : (pass < nq + nk ? p.k : p.v); };
  auto head_of = [&](int pass) {
    return (pass < nq ? pass : (pass < nq + nk ? pass - nq : pass - nq - nk)) * HPW + lane / LPH;
  };

  float cs[8], sn[8], qw[16], kw[16];
  int64_t position = 0;
  int page = -1, slot = 0;
  for (int base = first; base < last; base += kFlight) {
    Raw8<EB> x[kFlight][2];
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      if (base + i < last) {
        const RotaryRows& r = rows_of(base + i);
        int h = head_of(base + i);
        h = h < r.heads ? h : r.heads - 1;  // lanes without a head repeat the last
        const char* src = static_cast<const char*>(r.src) +
                          ((int64_t)b * r.ss[0] + (int64_t)h * r.ss[1] + (int64_t)t * r.ss[2]) * EB;
        x[i][0] = raw8<EB, PAST>(src + e0 * EB);
        x[i][1] = raw8<EB, PAST>(src + e1 * EB);
      }
    }
    if (base == first) {
      auto weights = [&](const void* w, float* out) {
        if (w == nullptr) return;
        if (p.weight_f32) {
          widen8<4, false>(raw8<4>(static_cast<const char*>(w) + e0 * 4), out);
          widen8<4, false>(raw8<4>(static_cast<const char*>(w) + e1 * 4), out + 8);
        } else {
          widen8<EB, F16>(raw8<EB>(static_cast<const char*>(w) + e0 * EB), out);
          widen8<EB, F16>(raw8<EB>(static_cast<const char*>(w) + e1 * EB), out + 8);
        }
      };
      weights(p.q_weight, qw);
      weights(p.k_weight, kw);
      double freq = 0.0;
      if (lane < p.rot / 2) freq = p.inv_freq[lane];
      if constexpr (PAGED) {
        const int s = sequence_of(p.batch, t, lane);
        if (s < 0) return;
        position = (int64_t)p.batch.kv_lens[s] - p.batch.q_starts[s + 1] + t;
        if (position >= 0 && position < p.batch.cap) {
          const int at = (int)position;
          page = page_entry(p.batch, s, at);
          if (!is_page(p.batch, page)) page = -1;
          slot = at - page_of(p.batch, at) * p.batch.page;
        }
      }
      if (!PAGED || p.positions != nullptr) {
        const int64_t i = (int64_t)b * p.pos_stride + t;
        position = p.pos64 ? static_cast<const int64_t*>(p.positions)[i] : static_cast<const int32_t*>(p.positions)[i];
      }
      if (p.rot > 0) {
        if (lane < p.rot / 2) {
          double turn = (double)position * freq * kTurn;
          turn -= rint(turn);
          float s, c;
          sincospif(2.f * (float)turn, &s, &c);
          turns[wave][lane] = float2{c * p.factor, s * p.factor};
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (turned) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 y = turns[wave][8 * j + i];
            cs[i] = y.x;
            sn[i] = y.y;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const int pass = base + i;
      if (pass >= last) break;
      const RotaryRows& r = rows_of(pass);
      const int h = head_of(pass);
      float v[16];
      widen8<EB, F16>(x[i][0], v);
      widen8<EB, F16>(x[i][1], v + 8);
      if (pass < nq + nk) {
        const bool is_q = pass < nq;
        if ((is_q ? p.q_weight : p.k_weight) != nullptr) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) ss += v[e] * v[e];
#pragma unroll
          for (int m = 1; m < LPH; m *= 2) ss += __shfl_xor(ss, m);
          const float rn = 1.f / sqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = v[e] * rn * (is_q ? qw[e] : kw[e]);
        }
        if (turned) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            // Pairs: (v[e], v[e + 8]), or neighbours.
            float& a = p.interleaved ? v[2 * e] : v[e];
            float& c = p.interleaved ? v[2 * e + 1] : v[e + 8];
            const float a0 = a, c0 = c;
            a = a0 * cs[e] - c0 * sn[e];
            c = c0 * cs[e] + a0 * sn[e];
          }
        }
      }
      const bool paged = PAGED && pass >= nq;
      if (h >= r.heads || (paged && page < 0)) continue;
      char* dst = static_cast<char*>(r.dst) +
                  ((int64_t)(paged ? page : b) * r.ds[0] + (int64_t)h * r.ds[1] + (int64_t)(paged ? slot : t) * r.ds[2]) *
                      EB;
      store8<EB, F16, PAST>(dst + e0 * EB, v);
      store8<EB, F16, PAST>(dst + e1 * EB, v + 8);
    }
  }
}

template <bool PAGED>
int launch_rotary(RotaryParams& p, int64_t D, int dtype, hipStream_t stream) {
  const int hpw = D == 128 ? 8 : 16;
  const int nk = (p.k.heads + hpw - 1) / hpw, passes = (p.q.heads + hpw - 1) / hpw + nk + (PAGED ? nk : 0);
  // Few tokens: their heads are shared out until 4096 waves (four a SIMD) are up.
  p.groups = 1;
  if (p.rows < 4096) {
    const int64_t g = 4096 / p.rows;
    p.groups = g < passes ? (int)g : passes;
  }
  const int64_t blocks = (p.rows * p.groups + 3) / 4;
  SPRUCE_REQUIRE(blocks < (int64_t)1 << 31, "too many tokens");
  const dim3 grid = flat_grid(blocks);
  // Rows that the 256 MB behind the L2s cannot hold until someone reads them
  // again go past the caches, where the lanes of a head take 128 bytes at a
  // time (a whole line): 32768 tokens of 28 + 4 heads of 128 in 102 us rather than 113, the append
  // of 16384 tokens in 80 rather than 88.  Pieces of a line come from memory more than once so (8170
  // tokens in float32 in 35 us rather than 25), and small outputs serve their readers from the caches.
  auto lines = [](const RotaryRows& r) {
    bool whole = (reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst)) % 128 == 0;
    for (int i = 0; i < 3; ++i) whole = whole && (r.ss[i] | r.ds[i]) % 64 == 0;
    return whole;  // (rows that are not there have zeros)
  };
  const int64_t values = p.rows * (p.q.heads + p.k.heads + (PAGED ? p.k.heads : 0)) * D;
  const bool past = values * 4 > (int64_t)256 << 20 && dtype != SPRUCE_DTYPE_F32 && D == 128 && p.rot == D &&
                    !p.interleaved && lines(p.q) && lines(p.k) && lines(p.v);
#define SPRUCE_ROTARY(EB, F16, DD, PAST) \
  hipLaunchKernelGGL((head_rotary_kernel<EB, F16, DD, PAGED, PAST>), grid, dim3(256), 0, stream, p)
  if (past) {
    if (dtype == SPRUCE_DTYPE_BF16) SPRUCE_ROTARY(2, false, 128, true);
    else SPRUCE_ROTARY(2, true, 128, true);
  } else if (D == 128) {
    if (dtype == SPRUCE_DTYPE_BF16) SPRUCE_ROTARY(2, false, 128, false);
    else if (dtype == SPRUCE_DTYPE_F16) SPRUCE_ROTARY(2, true, 128, false);
    else SPRUCE_ROTARY(4, false, 128, false);
  } else {
    if (dtype == SPRUCE_DTYPE_BF16) SPRUCE_ROTARY(2, false, 64, false);
    else if (dtype == SPRUCE_DTYPE_F16) SPRUCE_ROTARY(2, true, 64, false);
    else SPRUCE_ROTARY(4, false, 64, false);
  }
#undef SPRUCE_ROTARY
  return check_launch("head_rotary_kernel");
}

// Rows of 16-byte pieces: the base and every stride but the last.
bool rows16(const void* p, const int64_t s[3], int eb) {
  if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (s[i] * eb % 16) return false;
  return true;
}

int set_rotary(RotaryParams& p, int64_t D, int dtype, const double* inv_freq, int64_t rotary_dim, int64_t layout,
               double factor, const void* q_weight, const void* k_weight, int64_t weight_dtype, double eps) {
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(dtype == SPRUCE_DTYPE_BF16 || dtype == SPRUCE_DTYPE_F16 || dtype == SPRUCE_DTYPE_F32,
                 "unsupported dtype code %d", dtype);
  SPRUCE_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0,
                 "rotary_dim must be a multiple of 16 up to head_dim, got %lld", (long long)rotary_dim);
  SPRUCE_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq must be a non-null device pointer");
  SPRUCE_REQUIRE(layout == SPRUCE_ROTARY_HALF || layout == SPRUCE_ROTARY_INTERLEAVED, "unknown rotary layout %lld",
                 (long long)layout);
  SPRUCE_REQUIRE(weight_dtype == SPRUCE_DTYPE_F32 || weight_dtype == dtype,
                 "norm weights must be float32 or the input dtype (code %d), got code %d", dtype, (int)weight_dtype);
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(q_weight) % 16 == 0 && reinterpret_cast<uintptr_t>(k_weight) % 16 == 0,
                 "norm weights must be 16-byte aligned");
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(inv_freq) % 8 == 0, "inv_freq must be 8-byte aligned");
  p.inv_freq = inv_freq;
  p.rot = (int)rotary_dim;
  p.interleaved = layout == SPRUCE_ROTARY_INTERLEAVED;
  p.factor = (float)factor;
  p.q_weight = q_weight;
  p.k_weight = k_weight;
  p.weight_f32 = weight_dtype == SPRUCE_DTYPE_F32;
  p.eps = (float)eps;
  return SPRUCE_OK;
}

}  // namespace

extern "C" int spruce_rotate_heads(const spruce_rotate_heads_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_rotate_heads_args& a = *args;
  const int64_t B = a.B, Hq = a.Hq, Hkv = a.Hkv, T = a.T, D = a.D;
  const int dtype = (int)a.dtype;
  SPRUCE_REQUIRE(B >= 0 && T >= 0 && Hq >= 1 && Hkv >= 1 && Hq < 1 << 16 && Hkv < 1 << 16, "invalid shape");
  SPRUCE_REQUIRE(T < (int64_t)1 << 30 && B < (int64_t)1 << 30, "too many tokens");
  SPRUCE_REQUIRE(a.qs[3] == 1 && a.ks[3] == 1 && a.qos[3] == 1 && a.kos[3] == 1,
                 "q, k and the outputs must have a contiguous final dimension");
  RotaryParams p{};
  const int rc = set_rotary(p, D, dtype, a.inv_freq, a.rotary_dim, a.layout, a.factor, a.q_weight, a.k_weight,
                            a.weight_dtype, a.eps);
  if (rc) return rc;
  if (B == 0 || T == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(a.q && a.k && a.q_out && a.k_out && a.positions, "q, k, positions and the outputs must be non-null device pointers");
  const int eb = dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  SPRUCE_REQUIRE(rows16(a.q, a.qs, eb) && rows16(a.k, a.ks, eb) && rows16(a.q_out, a.qos, eb) &&
                     rows16(a.k_out, a.kos, eb),
                 "q, k and the outputs must be 16-byte aligned with strides that keep rows 16-byte aligned");
  const int64_t q_rows[3] = {B, Hq, T}, k_rows[3] = {B, Hkv, T};
  SPRUCE_REQUIRE(rows_apart(a.qos, q_rows, 3, D) && rows_apart(a.kos, k_rows, 3, D), "the rows of the outputs overlap");
  auto rows = [](RotaryRows& r, const void* src, const int64_t* ss, void* dst, const int64_t* ds, int64_t heads) {
    r.src = src;
    r.dst = dst;
    for (int i = 0; i < 3; ++i) {
      r.ss[i] = ss[i];
      r.ds[i] = ds[i];
    }
    r.heads = (int)heads;
  };
  rows(p.q, a.q, a.qs, a.q_out, a.qos, Hq);
  rows(p.k, a.k, a.ks, a.k_out, a.kos, Hkv);
  p.positions = a.positions;
  p.pos_stride = a.pos_stride;
  p.pos64 = a.pos64 != 0;
  p.tokens = (int)T;
  p.rows = B * T;
  return launch_rotary<false>(p, D, dtype, (hipStream_t)stream);
}

extern "C" int spruce_paged_append(const spruce_paged_append_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_paged_append_args& a = *args;
  const int64_t N = a.N, Hq = a.Hq, Hkv = a.Hkv, D = a.D;
  const int dtype = (int)a.dtype;
  SPRUCE_REQUIRE(Hq >= 0 && Hkv >= 1 && Hq < 1 << 16 && Hkv < 1 << 16, "invalid shape");
  SPRUCE_REQUIRE((Hq == 0 || (a.qs[2] == 1 && a.qos[2] == 1)) && a.ks[2] == 1 && a.vs[2] == 1 && a.kps[3] == 1 &&
                     a.vps[3] == 1,
                 "q, k, v, the pages and the output must have a contiguous final dimension");
  RotaryParams p{};
  int rc = set_rotary(p, D, dtype, a.inv_freq, a.rotary_dim, a.layout, a.factor, a.q_weight, a.k_weight, a.weight_dtype,
                      a.eps);
  if (rc) return rc;
  rc = prepare_batch(p.batch, a.page_table, a.table_stride, a.table_width, a.q_starts, a.kv_lens, a.S, N, a.page_size,
                     a.pages);
  if (rc) return rc;
  if (N == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(a.k && a.v && (a.pages == 0 || (a.k_pages && a.v_pages)),
                 "k, v and the pages must be non-null device pointers");
  SPRUCE_REQUIRE(Hq == 0 || (a.q && a.q_out), "q and its output must be non-null device pointers");
  // Packed [N, H, D] rows as one batch; the pages' strides as they are.
  auto rows = [&](RotaryRows& r, const void* src, const int64_t* ss, void* dst, const int64_t* ds, bool paged, int64_t heads) {
    r.src = src;
    r.dst = dst;
    r.ss[1] = ss[1];
    r.ss[2] = ss[0];
    r.ds[0] = paged ? ds[0] : 0;
    r.ds[1] = ds[1];
    r.ds[2] = paged ? ds[2] : ds[0];
    r.heads = (int)heads;
  };
  const int eb = dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  if (Hq) rows(p.q, a.q, a.qs, a.q_out, a.qos, false, Hq);
  rows(p.k, a.k, a.ks, a.k_pages, a.kps, true, Hkv);
  rows(p.v, a.v, a.vs, a.v_pages, a.vps, true, Hkv);
  auto fits = [&](const RotaryRows& r) { return rows16(r.src, r.ss, eb) && rows16(r.dst, r.ds, eb); };
  SPRUCE_REQUIRE((Hq == 0 || fits(p.q)) && fits(p.k) && fits(p.v),
                 "q, k, v, the pages and the output must be 16-byte aligned with strides that keep rows 16-byte "
                 "aligned");
  const int64_t pages[3] = {a.pages, Hkv, a.page_size}, tokens[2] = {N, Hq};
  SPRUCE_REQUIRE(rows_apart(a.kps, pages, 3, D) && rows_apart(a.vps, pages, 3, D), "the rows of the pages overlap");
  SPRUCE_REQUIRE(Hq == 0 || rows_apart(a.qos, tokens, 2, D), "the rows of the output overlap");
  p.positions = a.positions;
  p.pos64 = a.pos64 != 0;
  p.tokens = (int)N;
  p.rows = N;
  return launch_rotary<true>(p, D, dtype, (hipStream_t)stream);
}
