// Attention over a paged K/V cache: the arguments' checks and the plan of a
// call (the kernels are in paged_impl.h).
#include "paged_impl.h"

using namespace spruce;

namespace {

// How a call is launched, and the most row tiles that a batch with N new
// tokens of S sequences can hold of either kind, whatever its lengths are.
struct Plan {
  bool few, many, few_whole, many_whole;
  int few_limit;
  int64_t few_tiles, many_tiles, groups;
  int64_t slots;  // for sums of 32 rows each
};

template <typename SHAPE>
int64_t tiles_bound(int64_t N, int64_t S, int64_t G, int64_t most, bool lists) {
  // `most`: packed rows that a sequence of this kind has at most, and so its
  // tokens; a sequence rounds up by one tile.  (By all tokens alone a large chunk
  // passes for thousands of few-row tiles, which the rules below take whole:
  // 16384 tokens of one sequence beside one token over 131072 keys, 32/8 heads
  // of 128, 4031 us rather than 2564.)
  const int64_t seqs = S < N ? S : N, tokens = most / G;
  if (tokens == 0) return 0;
  auto least = [](int64_t x, int64_t y) { return x < y ? x : y; };
  auto tiles = [](int64_t rows) { return (rows + SHAPE::rows - 1) / SHAPE::rows; };
  if (!lists) return least(N * G / SHAPE::rows + seqs, seqs * tiles(most));
  // Rows break at every 64 positions too; n tokens touch (n - 2) / 64 + 2 such blocks at most, one token one.
  return least(N / kBlock + 2 * seqs, seqs * ((tokens + kBlock - 2) / kBlock + 1)) * tiles(least(most, kBlock * G));
}

// The rules below go by sizes that the host knows; figures are of bf16 and f16,
// 28/4 heads of 128 and 16/8 heads of 64, keys between a fifth and the whole of
// the table's.
Plan plan_of(int64_t N, int64_t S, int64_t G, int64_t Hkv, int64_t keys, bool lists) {
  Plan plan{};
  // Packed rows of a sequence up to which it goes the few-row way.  More than 32
  // make a second tile, which reads every key again (64 sequences of 42 rows and
  // 8000 keys: 358 us, 228 the many-row way; 16 of 4000: 63 and 54); where there
  // are few workgroups that costs less than the many-row way's longer steps (one
  // sequence of 35 rows: 13 us rather than 19 over 600 keys, 42 rather than 47
  // over 32000).
  const int64_t few_rows = S * Hkv >= 32 ? 32 : 64;
  // The lengths are not known here, but every sequence has a new token in all
  // but odd batches: where even one that has all others' is two tiles at most,
  // the few-row way is launched alone and takes whatever there is; likewise the
  // many-row way where one sequence has all tokens.  (An idle launch is 4 to 15
  // us: 48 us rather than 44 for one to four tokens of each of 16 sequences.)
  const int64_t longest = N > S ? N - S + 1 : 1;
  plan.few = S > 1 || N * G <= few_rows;
  plan.many = !plan.few || longest * G > 64;
  if (plan.many && G > few_rows) plan.few = false;  // one token is past it
  plan.few_limit = !plan.many ? 0x7fffffff : (plan.few ? (int)few_rows : -1);
  if (plan.few) plan.few_tiles = tiles_bound<Few>(N, S, G, plan.many ? few_rows : N * G, lists) * Hkv;
  if (plan.many) plan.many_tiles = tiles_bound<Many>(N, S, G, N * G, lists) * Hkv;
  // Whole tiles save the line's arithmetic and the join, shares even the lengths
  // out.  Few rows: 16 sequences, 1024 keys: 16 us whole, 25 shared; 2048: 27
  // and 26; 4096: 50 and 28.  64 sequences (a tile a CU), 4096 keys: 66 and 75;
  // 8192: 130 and 127; 16384: 254 and 233.  Many rows: 8 sequences of 256 tokens
  // (224 tiles), 1536 keys: 59 and 67, 4096: 131 and 111; 32 of 128 tokens, 8192
  // keys: 422 and 400.  Tiles of one sequence are alike: 4096 tokens (512 tiles)
  // over 16384 keys 985 and 1018; but 2560 (320 tiles) 874 and 672.
  plan.few_whole = keys <= 1024 || (plan.few_tiles >= kCus && keys <= 4096) || plan.few_tiles > 64 * kCus;
  plan.many_whole =
      keys <= 1024 || (plan.many_tiles >= kCus && keys <= 2048) || plan.many_tiles >= (S == 1 ? 2 : 16) * kCus;
  // A workgroup fills a CU's registers.  (40 heads, 4 sequences of 4000 keys: six
  // workgroups a head on 256 CUs 70 us, 25 a head in rounds 79.)
  plan.groups = kCus / Hkv;
  if (plan.groups < 1) plan.groups = 1;
  if (plan.few && !plan.few_whole) plan.slots = 2 * plan.groups * Hkv;
  if (plan.many && !plan.many_whole) plan.slots = 2 * plan.groups * Hkv * kWaves;
  return plan;
}

// Sums of the slots, then what the workgroups have begun.
int64_t workspace_of(const Plan& plan, int64_t Hkv, int64_t D) {
  return plan.slots * 32 * (D + 2) * 4 + plan.groups * Hkv * 16;
}

}  // namespace

extern "C" int64_t spruce_paged_attention_workspace_bytes(int64_t N, int64_t S, int64_t Hq, int64_t Hkv, int64_t D,
                                                          int64_t keys, int64_t K) {
  if (N < 1 || S < 1 || Hkv < 1 || Hq < Hkv || N >= (int64_t)1 << 30 || S >= (int64_t)1 << 20 || Hq >= 1 << 16 ||
      D < 1 || D > 128)
    return 0;
  return workspace_of(plan_of(N, S, Hq / Hkv, Hkv, K > 0 ? K * kBlock : keys, K > 0), Hkv, D);
}

extern "C" int spruce_paged_attention(const spruce_paged_attention_args* args, void* stream) {
  SPRUCE_REQUIRE(args != nullptr, "args must be non-null");
  const spruce_paged_attention_args& a = *args;
  const int64_t N = a.N, S = a.S, Hq = a.Hq, Hkv = a.Hkv, D = a.D, K = a.K;
  const int dtype = (int)a.dtype;
  const float scale = (float)a.scale;
  SPRUCE_REQUIRE(D == 64 || D == 128, "kernel supports head_dim 64 or 128, got %lld", (long long)D);
  SPRUCE_REQUIRE(dtype == SPRUCE_DTYPE_BF16 || dtype == SPRUCE_DTYPE_F16,
                 "the paged attention takes bf16 or f16, got dtype code %d", dtype);
  SPRUCE_REQUIRE(Hq >= 1 && Hkv >= 1 && Hq % Hkv == 0 && Hq < 1 << 16,
                 "query heads (%lld) must be divisible by KV heads (%lld)", (long long)Hq, (long long)Hkv);
  SPRUCE_REQUIRE(Hq / Hkv <= 64, "at most 64 query heads per KV head are supported");
  const float cs = scale * 1.4426950408889634f;  // of exp2
  SPRUCE_REQUIRE(scale > 0.f && cs < INFINITY, "scale must be positive, and finite times log2(e)");
  SPRUCE_REQUIRE(a.qs[2] == 1 && a.kps[3] == 1 && a.vps[3] == 1 && a.os[2] == 1,
                 "q, the pages and out must have a contiguous final dimension");
  PagedAttn p{};
  const int rc = prepare_batch(p.batch, a.page_table, a.table_stride, a.table_width, a.q_starts, a.kv_lens, S, N,
                               a.page_size, a.pages);
  if (rc) return rc;
  if (N == 0) return SPRUCE_OK;
  SPRUCE_REQUIRE(a.q && a.out && (a.pages == 0 || (a.k_pages && a.v_pages)),
                 "q, the pages and out must be non-null device pointers");
  auto rows16 = [](const void* ptr, const int64_t* s, int n) {
    if (reinterpret_cast<uintptr_t>(ptr) % 16) return false;
    for (int i = 0; i < n; ++i)
      if (s[i] % 8) return false;
    return true;
  };
  SPRUCE_REQUIRE(rows16(a.q, a.qs, 2) && rows16(a.k_pages, a.kps, 3) && rows16(a.v_pages, a.vps, 3) && rows16(a.out, a.os, 2),
                 "q, the pages and out must be 16-byte aligned with strides that keep rows 16-byte aligned");
  const int64_t rows[2] = {N, Hq};
  SPRUCE_REQUIRE(rows_apart(a.os, rows, 2, D), "the rows of out overlap");
  SPRUCE_REQUIRE(K >= 0 && K < (int64_t)1 << 24, "invalid list width %lld", (long long)K);
  SPRUCE_REQUIRE(K == 0 || (a.idx && a.Qc >= 0), "indices must be a non-null device pointer");
  SPRUCE_REQUIRE(K == 0 || a.is[3] == 1, "indices must have a contiguous final dimension");
  const Plan plan = plan_of(N, S, Hq / Hkv, Hkv, K > 0 ? K * kBlock : p.batch.cap, K > 0);
  const int64_t need = workspace_of(plan, Hkv, D);
  SPRUCE_REQUIRE(a.workspace && a.workspace_bytes >= need, "workspace too small: %lld bytes, need %lld",
                 (long long)a.workspace_bytes, (long long)need);
  SPRUCE_REQUIRE(reinterpret_cast<uintptr_t>(a.workspace) % 16 == 0, "workspace must be 16-byte aligned");
  p.q = a.q;
  p.out = a.out;
  p.k = a.k_pages;
  p.v = a.v_pages;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.qs[i];
    p.os[i] = a.os[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = a.kps[i];
    p.vs[i] = a.vps[i];
  }
  p.Hkv = (int)Hkv;
  p.by_heads = divisor(Hkv);
  p.by_group = divisor(Hq / Hkv);
  p.G = (int)(Hq / Hkv);
  p.cs = cs;
  if (K > 0) {
    p.idx = a.idx;
    for (int i = 0; i < 3; ++i) p.is[i] = a.is[i];
    p.Qc = (int)(a.Qc < (int64_t)1 << 30 ? a.Qc : (int64_t)1 << 30);
    p.K = (int)K;
  }
  // Grids of fewer than 2^32 threads, rows of a sequence in 32 bits with room for the tiles' ends.
  SPRUCE_REQUIRE(N * (Hq / Hkv) < (int64_t)1 << 28 && plan.few_tiles < (int64_t)1 << 23 &&
                     plan.many_tiles < (int64_t)1 << 23,
                 "too many tokens for one call");
  p.few_limit = plan.few_limit;
  p.groups = (int)plan.groups;
  // The kinds' launches follow one another, so they share the slots.
  p.part_o = static_cast<float*>(a.workspace);
  p.part_ml = p.part_o + plan.slots * 32 * D;
  p.begun = reinterpret_cast<int4*>(p.part_ml + plan.slots * 64);
  // Rows of a page's block behind one 32-bit buffer offset, bounded by the last row's end.
  const bool aligned = a.page_size % kBlock == 0 && a.kps[2] >= D && a.vps[2] >= D && a.kps[2] < 1 << 22 &&
                       a.vps[2] < 1 << 22;
  const hipStream_t st = (hipStream_t)stream;
  const bool f16 = dtype == SPRUCE_DTYPE_F16;
  if (plan.many) {
    const PagedLaunch n{plan.many_tiles, plan.many_whole ? 0 : plan.groups * Hkv};
    const int e = aligned ? launch_paged_many(p, (int)D, f16, n, st) : launch_paged_scattered(p, (int)D, f16, n, st);
    if (e) return e;
  }
  if (plan.few) {
    const int e = launch_paged_few(p, (int)D, f16, PagedLaunch{plan.few_tiles, plan.few_whole ? 0 : plan.groups * Hkv}, st);
    if (e) return e;
  }
  return SPRUCE_OK;
}
