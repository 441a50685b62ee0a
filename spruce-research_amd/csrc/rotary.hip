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
// Bytes bound it (each value read and written once).  A wave owns one token:
// its lanes work out one pair's sine and cosine each, once for all heads, and
// hand them over through LDS; then D/16 lanes take a head row, 16 values a
// lane chosen so that both members of every pair are in the lane.
#include "paged.h"

using namespace spruce;

namespace {

struct RotaryParams {
  const void* src[3];    // q, k, v rows; v only with PAGED
  void* dst[3];          // q and k rows, or the key and value pages
  int64_t ss[3][3];      // batch, head, token strides of src
  int64_t ds[3][3];      // the same of dst; for pages: page, head, slot
  const void* positions;  // int32 or int64
  int64_t pos_stride;    // per batch
  int pos64;
  const double* inv_freq;
  int rot, interleaved;
  float factor;
  const void* weight[2];
  int weight_f32;
  float eps;
  int heads[3];
  int tokens;   // per batch
  int64_t rows;  // batches * tokens
  int groups, passes;  // passes over the heads, and in how many waves' hands
  PagedBatch batch;
};

constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

template <int EB, bool F16>
__device__ __forceinline__ void widen8(const char* p, float (&v)[8]) {
  if constexpr (EB == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 r = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = unpack1<F16>(w[i] & 0xffffu);
      v[2 * i + 1] = unpack1<F16>(w[i] >> 16);
    }
  }
}

template <int EB, bool F16>
__device__ __forceinline__ void narrow8(char* p, const float (&v)[8]) {
  if constexpr (EB == 4) {
    reinterpret_cast<float4*>(p)[0] = float4{v[0], v[1], v[2], v[3]};
    reinterpret_cast<float4*>(p)[1] = float4{v[4], v[5], v[6], v[7]};
  } else {
    *reinterpret_cast<uint4*>(p) =
        uint4{pack2<F16>(v[0], v[1]), pack2<F16>(v[2], v[3]), pack2<F16>(v[4], v[5]), pack2<F16>(v[6], v[7])};
  }
}

template <int EB, bool F16, int D, bool PAGED>
__global__ __launch_bounds__(256) void head_rotary_kernel(const RotaryParams p) {
  constexpr int LPH = D / 16, HPW = 64 / LPH;  // lanes of a head row, head rows of a pass
  __shared__ float2 turns[4][D / 2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = (int64_t)flat_block() * 4 + wave;
  const int64_t row = item / p.groups;
  const int grp = (int)(item - row * p.groups);
  if (row >= p.rows) return;  // no barrier below
  const int b = (int)(row / p.tokens), t = (int)(row - (int64_t)b * p.tokens);

  int64_t position;
  int page = -1, slot = 0;
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
  if (lane < p.rot / 2) {
    double turn = (double)position * p.inv_freq[lane] * kTurn;
    turn -= rint(turn);
    float s, c;
    sincospif(2.f * (float)turn, &s, &c);
    turns[wave][lane] = float2{c * p.factor, s * p.factor};
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

  const int j = lane % LPH;
  const bool turned = j < p.rot / 16;
  const int e0 = turned && !p.interleaved ? 8 * j : 16 * j;
  const int e1 = turned && !p.interleaved ? 8 * j + p.rot / 2 : 16 * j + 8;
  float cs[8], sn[8];
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 x = turns[wave][8 * j + i];
      cs[i] = x.x;
      sn[i] = x.y;
    }
  }
  const int total = p.heads[0] + p.heads[1] + (PAGED ? p.heads[2] : 0);
  const int per = (p.passes + p.groups - 1) / p.groups;
  for (int pass = grp * per; pass < (grp + 1) * per && pass < p.passes; ++pass) {
    int h = pass * HPW + lane / LPH;
    if (h >= total) continue;
    int what = 0;
    if (h >= p.heads[0]) {
      h -= p.heads[0];
      what = 1;
      if (PAGED && h >= p.heads[1]) {
        h -= p.heads[1];
        what = 2;
      }
    }
    if (PAGED && what > 0 && page < 0) continue;
    const char* src = static_cast<const char*>(p.src[what]) +
                      ((int64_t)b * p.ss[what][0] + (int64_t)h * p.ss[what][1] + (int64_t)t * p.ss[what][2]) * EB;
    const bool paged = PAGED && what > 0;
    char* dst = static_cast<char*>(p.dst[what]) +
                ((int64_t)(paged ? page : b) * p.ds[what][0] + (int64_t)h * p.ds[what][1] +
                 (int64_t)(paged ? slot : t) * p.ds[what][2]) * EB;
    float x[8], y[8];
    widen8<EB, F16>(src + e0 * EB, x);
    widen8<EB, F16>(src + e1 * EB, y);
    if (what < 2) {
      const void* weight = p.weight[what];
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += x[i] * x[i] + y[i] * y[i];
      // Every lane of the row takes part; rows of one pass may differ in
      // `what`, so the sums are formed before the branch on the weight.
#pragma unroll
      for (int m = 1; m < LPH; m *= 2) ss += __shfl_xor(ss, m);
      if (weight != nullptr) {
        const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
        float w0[8], w1[8];
        if (p.weight_f32) {
          widen8<4, false>(static_cast<const char*>(weight) + e0 * 4, w0);
          widen8<4, false>(static_cast<const char*>(weight) + e1 * 4, w1);
        } else {
          widen8<EB, F16>(static_cast<const char*>(weight) + e0 * EB, w0);
          widen8<EB, F16>(static_cast<const char*>(weight) + e1 * EB, w1);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = x[i] * r * w0[i];
          y[i] = y[i] * r * w1[i];
        }
      }
      if (turned) {
        if (p.interleaved) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = x[2 * i], c = x[2 * i + 1], d = y[2 * i], f = y[2 * i + 1];
            x[2 * i] = a * cs[i] - c * sn[i];
            x[2 * i + 1] = c * cs[i] + a * sn[i];
            y[2 * i] = d * cs[4 + i] - f * sn[4 + i];
            y[2 * i + 1] = f * cs[4 + i] + d * sn[4 + i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float a = x[i], c = y[i];
            x[i] = a * cs[i] - c * sn[i];
            y[i] = c * cs[i] + a * sn[i];
          }
        }
      }
    }
    narrow8<EB, F16>(dst + e0 * EB, x);
    narrow8<EB, F16>(dst + e1 * EB, y);
  }
}

template <bool PAGED>
int launch_rotary(RotaryParams& p, int64_t D, int dtype, hipStream_t stream) {
  const int total = p.heads[0] + p.heads[1] + (PAGED ? p.heads[2] : 0);
  const int hpw = D == 128 ? 8 : 16;
  p.passes = (total + hpw - 1) / hpw;
  p.groups = 1;
  const int64_t blocks = (p.rows * p.groups + 3) / 4;
  SPRUCE_REQUIRE(blocks < (int64_t)1 << 31, "too many tokens");
  const dim3 grid = flat_grid(blocks);
#define SPRUCE_ROTARY(EB, F16, DD) \
  hipLaunchKernelGGL((head_rotary_kernel<EB, F16, DD, PAGED>), grid, dim3(256), 0, stream, p)
  if (D == 128) {
    if (dtype == SPRUCE_DTYPE_BF16) SPRUCE_ROTARY(2, false, 128);
    else if (dtype == SPRUCE_DTYPE_F16) SPRUCE_ROTARY(2, true, 128);
    else SPRUCE_ROTARY(4, false, 128);
  } else {
    if (dtype == SPRUCE_DTYPE_BF16) SPRUCE_ROTARY(2, false, 64);
    else if (dtype == SPRUCE_DTYPE_F16) SPRUCE_ROTARY(2, true, 64);
    else SPRUCE_ROTARY(4, false, 64);
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

int set_rotary(RotaryParams& p, int64_t D, int dtype, const double* inv_freq, int64_t rotary_dim, int layout,
               float factor, const void* q_weight, const void* k_weight, int weight_dtype, float eps) {
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(dtype == SPRUCE_DTYPE_BF16 || dtype == SPRUCE_DTYPE_F16 || dtype == SPRUCE_DTYPE_F32,
                 "unsupported dtype code %d", dtype);
  SPRUCE_REQUIRE(rotary_dim >= 0 && rotary_dim <= D && rotary_dim % 16 == 0,
                 "rotary_dim must be a multiple of 16 up to head_dim, got %lld", (long long)rotary_dim);
  SPRUCE_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "inv_freq must be a non-null device pointer");
  SPRUCE_REQUIRE(layout == SPRUCE_ROTARY_HALF || layout == SPRUCE_ROTARY_INTERLEAVED, "unknown rotary layout %d",
                 layout);
  SPRUCE_REQUIRE(weight_dtype == SPRUCE_DTYPE_F32 || weight_dtype == dtype,
                 "norm weights must be float32 or the input dtype (code %d), got code %d", dtype, weight_dtype);
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(q_weight) % 16 == 0 && reinterpret_cast<uintptr_t>(k_weight) % 16 == 0,
                 "norm weights must be 16-byte aligned");
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(inv_freq) % 8 == 0, "inv_freq must be 8-byte aligned");
  p.inv_freq = inv_freq;
  p.rot = (int)rotary_dim;
  p.interleaved = layout == SPRUCE_ROTARY_INTERLEAVED;
  p.factor = factor;
  p.weight[0] = q_weight;
  p.weight[1] = k_weight;
  p.weight_f32 = weight_dtype == SPRUCE_DTYPE_F32;
  p.eps = eps;
  return SPRUCE_OK;
}

}  // namespace

extern "C" int spruce_rotate_heads(const void* q, const int64_t qs[4], const void* k, const int64_t ks[4], int64_t B,
                                   int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int dtype, const void* positions,
                                   int64_t pos_stride, int pos64, const double* inv_freq, int64_t rotary_dim,
                                   int layout, float factor, const void* q_weight, const void* k_weight,
                                   int weight_dtype, float eps, void* qo, const int64_t qos[4], void* ko,
                                   const int64_t kos[4], void* stream) {
  SPRUCE_REQUIRE(qs && ks && qos && kos, "stride arrays must be non-null");
  SPRUCE_REQUIRE(B >= 0 && T >= 0 && Hq >= 1 && Hkv >= 1 && Hq < 1 << 16 && Hkv < 1 << 16, "invalid shape");
  SPRUCE_REQUIRE(T < (int64_t)1 << 30 && B < (int64_t)1 << 30, "too many tokens");
  SPRUCE_REQUIRE(qs[3] == 1 && ks[3] == 1 && qos[3] == 1 && kos[3] == 1,
                 "q, k and the outputs must have a contiguous final dimension");
  RotaryParams p{};
  const int rc = set_rotary(p, D, dtype, inv_freq, rotary_dim, layout, factor, q_weight, k_weight, weight_dtype, eps);
  if (rc) return rc;
  if (B == 0 || T == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(q && k && qo && ko && positions, "q, k, positions and the outputs must be non-null device pointers");
  const int eb = dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  SPRUCE_REQUIRE(rows16(q, qs, eb) && rows16(k, ks, eb) && rows16(qo, qos, eb) && rows16(ko, kos, eb),
                 "q, k and the outputs must be 16-byte aligned with strides that keep rows 16-byte aligned");
  p.src[0] = q;
  p.src[1] = k;
  p.dst[0] = qo;
  p.dst[1] = ko;
  for (int i = 0; i < 3; ++i) {
    p.ss[0][i] = qs[i];
    p.ss[1][i] = ks[i];
    p.ds[0][i] = qos[i];
    p.ds[1][i] = kos[i];
  }
  p.positions = positions;
  p.pos_stride = pos_stride;
  p.pos64 = pos64;
  p.heads[0] = (int)Hq;
  p.heads[1] = (int)Hkv;
  p.tokens = (int)T;
  p.rows = B * T;
  return launch_rotary<false>(p, D, dtype, (hipStream_t)stream);
}

extern "C" int spruce_paged_append(const void* q, const int64_t qs[3], void* qo, const int64_t qos[3], const void* k,
                                   const int64_t ks[3], const void* v, const int64_t vs[3], int64_t N, int64_t Hq,
                                   int64_t Hkv, int64_t D, int dtype, void* k_pages, const int64_t kps[4],
                                   void* v_pages, const int64_t vps[4], int64_t pages, int64_t page_size,
                                   const int32_t* page_table, int64_t table_stride, int64_t table_width,
                                   const int32_t* q_starts, const int32_t* kv_lens, int64_t S, const void* positions,
                                   int pos64, const double* inv_freq, int64_t rotary_dim, int layout, float factor,
                                   const void* q_weight, const void* k_weight, int weight_dtype, float eps,
                                   void* stream) {
  SPRUCE_REQUIRE(ks && vs && kps && vps, "stride arrays must be non-null");
  SPRUCE_REQUIRE(Hq == 0 || (qs && qos), "stride arrays must be non-null");
  SPRUCE_REQUIRE(Hq >= 0 && Hkv >= 1 && Hq < 1 << 16 && Hkv < 1 << 16, "invalid shape");
  SPRUCE_REQUIRE((Hq == 0 || (qs[2] == 1 && qos[2] == 1)) && ks[2] == 1 && vs[2] == 1 && kps[3] == 1 && vps[3] == 1,
                 "q, k, v, the pages and the output must have a contiguous final dimension");
  RotaryParams p{};
  int rc = set_rotary(p, D, dtype, inv_freq, rotary_dim, layout, factor, q_weight, k_weight, weight_dtype, eps);
  if (rc) return rc;
  rc = prepare_batch(p.batch, page_table, table_stride, table_width, q_starts, kv_lens, S, N, page_size, pages);
  if (rc) return rc;
  if (N == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(k && v && (pages == 0 || (k_pages && v_pages)), "k, v and the pages must be non-null device pointers");
  SPRUCE_REQUIRE(Hq == 0 || (q && qo), "q and its output must be non-null device pointers");
  // Packed [N, H, D] rows: batch stride 0, head, token.
  const int64_t* packed[3] = {qs, ks, vs};
  for (int i = 0; i < 3; ++i) {
    if (i == 0 && Hq == 0) continue;
    p.ss[i][1] = packed[i][1];
    p.ss[i][2] = packed[i][0];
  }
  if (Hq) {
    p.ds[0][1] = qos[1];
    p.ds[0][2] = qos[0];
  }
  for (int i = 0; i < 3; ++i) {
    p.ds[1][i] = kps[i];
    p.ds[2][i] = vps[i];
  }
  p.src[0] = q;
  p.src[1] = k;
  p.src[2] = v;
  p.dst[0] = qo;
  p.dst[1] = k_pages;
  p.dst[2] = v_pages;
  const int eb = dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  for (int i = Hq ? 0 : 1; i < 3; ++i)
    SPRUCE_REQUIRE(rows16(p.src[i], p.ss[i], eb) && rows16(p.dst[i], p.ds[i], eb),
                   "q, k, v, the pages and the output must be 16-byte aligned with strides that keep rows 16-byte "
                   "aligned");
  p.positions = positions;
  p.pos64 = pos64;
  p.heads[0] = (int)Hq;
  p.heads[1] = p.heads[2] = (int)Hkv;
  p.tokens = (int)N;
  p.rows = N;
  return launch_rotary<true>(p, D, dtype, (hipStream_t)stream);
}
