// Choice and launch of the W8A8 products over ragged groups of rows (grouped_gemm.h).
#include "grouped_gemm.h"

namespace xgen {

namespace {

// (waves x, waves y, fragments x, fragments y, pair slots)
#define XGEN_GROUPED_TILES(X) \
  X(1, 4, 1, 1, 6) /*  32 x 128 */ \
  X(2, 2, 1, 2, 4) /*  64 x 128 */ \
  X(2, 2, 1, 3, 3) /*  64 x 192 */ \
  X(2, 2, 2, 2, 4) /* 128 x 128 */ \
  X(2, 2, 2, 3, 3) /* 128 x 192 */ \
  X(2, 2, 4, 3, 2) /* 256 x 192 */ \
  X(2, 2, 4, 4, 2) /* 256 x 256 */

constexpr int kTiles = 7;
struct TileSize {
  int m, n, slots;
};
#define XGEN_TILE_SIZE(WM, WN, FM, FN, S) {GroupedCfg<WM, WN, FM, FN, S>::kM, GroupedCfg<WM, WN, FM, FN, S>::kN, S},
constexpr TileSize kTileSizes[kTiles] = {XGEN_GROUPED_TILES(XGEN_TILE_SIZE)};
// (the exact kind's widened fragments do not fit the registers beside the accumulators of 256 x 256)
constexpr bool has_tile(int kind, int tile) { return kind != kFp8Exact || kTileSizes[tile].m * kTileSizes[tile].n < 256 * 256; }

// What a call takes on a tile, in us: start + (c^4 + m^4)^(1/4), c = rounds * (pairs * per_pair + per_tile) on the
// matrix cores and through LDS, m the operands' and the output's bytes at 5.4 TB/s.  Fitted to the times of
// every tile on 300 calls (2 to 256 groups, 1 to 31,000 rows, N and K 512 to 5,376) with weights that no
// cache holds, rounds taken from their group sizes.
struct TileCost {
  float start, per_pair, per_tile;
};
constexpr TileCost kTileCosts[3][kTiles] = {
    // INT8
    {{5.2f, 0.354f, 0.40f}, {4.7f, 0.438f, 0.82f}, {4.5f, 0.597f, 0.93f}, {3.2f, 0.585f, 2.1f},
     {2.6f, 0.758f, 3.2f}, {0.00f, 1.27f, 6.9f}, {0.00f, 1.52f, 7.6f}},
    // FP8
    {{5.1f, 0.354f, 0.47f}, {4.0f, 0.446f, 0.81f}, {4.1f, 0.628f, 0.91f}, {2.6f, 0.582f, 2.4f},
     {2.0f, 0.724f, 4.0f}, {0.00f, 1.31f, 6.7f}, {0.00f, 1.49f, 9.0f}},
    // FP8 exact
    {{5.5f, 0.445f, 0.95f}, {4.6f, 0.559f, 1.5f}, {4.5f, 0.76f, 2.0f}, {4.1f, 0.783f, 2.8f},
     {2.9f, 1.04f, 4.1f}, {1.8f, 1.73f, 7.2f}, {}},
};
constexpr float kBytesPerUs = 5.4e6f;

// P(x > v) of a normal x
float above(float v, float mean, float deviation) { return 0.5f * erfcf((v - mean) / (deviation * 1.41421356f)); }

// The host does not know the groups' sizes.  They are taken to spread as a router's do: log-normal, deviation 0.4 of
// the logarithm, and each its Poisson count.  Over those 300 calls the tile rows so come within 8% of the real
// ones, and the choice within 1.7% of the best tile on the average (1.3% by the real ones; taking even groups
// that end half way in a tile, 7%).  In all of them every row belongs to a group: in the plan of a rank that holds some of
// the experts M counts rows that have no tile, and the choice is the one for that many more rows.
float expected_tile_rows(int m, float M, float groups) {
  const float mean = M / groups;
  if (mean > 8.0f * (float)m) return M / (float)m + 0.5f * groups;
  const float s2 = 0.16f + 1.0f / mean, s = sqrtf(s2);
  float rows = groups * (1.0f - expf(-mean));  // groups that are not empty: one tile row at least
  for (int j = 1; j < 64; ++j) {               // those of more than j m rows: one more
    const float p = above(logf((float)(j * m) / mean), -0.5f * s2, s);
    rows += groups * p;
    if (p < 1e-3f) break;
  }
  const float least = ceilf(M / (float)m);
  return rows > least ? rows : least;
}

// Expected rounds of the CUs over that many tiles (of a normal count: the groups end anywhere in their last tile).
float expected_rounds(float tile_rows, float tiles_n, float groups, float cus) {
  const float mean = tile_rows * tiles_n / cus;
  if (mean <= 1.0f) return mean < 0.9f ? 1.0f : 0.1f + mean;
  if (mean > 16.0f) return mean + 0.5f;
  float deviation = groups > 1.0f ? sqrtf(groups / 12.0f) * tiles_n / cus : 0.0f;
  deviation = deviation > 0.02f ? deviation : 0.02f;
  float rounds = 0.0f;
  for (int j = 0; j < 64; ++j) {  // sum of P(count > j)
    const float p = above((float)j, mean, deviation);
    rounds += p;
    if (p < 1e-3f && (float)j > mean) break;
  }
  return rounds;
}

int choose_tile(int kind, int64_t M, int64_t N, int64_t K, int64_t groups) {
  const float rows = (float)M, count = (float)groups, cus = (float)device_cu_count();
  const float filled = count * (1.0f - expf(-rows / count));
  const float bytes = filled * (float)N * (float)K + 2.0f * rows * (float)N + rows * (float)K;
  const float mem = bytes / kBytesPerUs, mem2 = mem * mem;
  int best = 0;
  float cost = 0.0f;
  for (int t = 0; t < kTiles; ++t) {
    if (!has_tile(kind, t)) continue;
    const TileSize ts = kTileSizes[t];
    const float tiles_n = (float)((N + ts.n - 1) / ts.n);
    const float rounds = expected_rounds(expected_tile_rows(ts.m, rows, count), tiles_n, count, cus);
    const int64_t steps = (K + 127) / 128;
    const TileCost tc = kTileCosts[kind][t];
    const float c = rounds * ((float)(steps > ts.slots ? steps : ts.slots) * tc.per_pair + tc.per_tile), c2 = c * c;
    const float us = tc.start + sqrtf(sqrtf(c2 * c2 + mem2 * mem2));
    if (t == 0 || us < cost) best = t, cost = us;
  }
  return best;
}

template <int KIND, int WM, int WN, int FM, int FN, int SLOTS>
int launch(GroupedArgs g, hipStream_t stream) {
  typedef GroupedCfg<WM, WN, FM, FN, SLOTS> C;
  g.tiles_n = (g.N + C::kN - 1) / C::kN;
  g.group_m = 8 * kTileM / C::kM;
  // at most one tile row per group ends short of kM rows
  const int64_t parts = g.M < g.groups ? g.M : g.groups;
  const int64_t tiles = (g.M / C::kM + parts) * g.tiles_n;
  if (tiles > 0x3fffffffLL) return fail(XGEN_ERR_UNSUPPORTED, "xgen_grouped_matmul: too many output tiles");
  const int64_t need = (tiles + 7) / 8 * 8;
  auto run = [&](auto PLAIN, auto ONCE) {
    constexpr bool plain = decltype(PLAIN)::value, once = decltype(ONCE)::value;
    static const int per_cu = resident_blocks_per_cu(grouped_gemm_kernel<KIND, WM, WN, FM, FN, SLOTS, plain, once>, C::kThreads);
    const int64_t resident = (int64_t)device_cu_count() * per_cu / 8 * 8;
    grouped_gemm_kernel<KIND, WM, WN, FM, FN, SLOTS, plain, once>
        <<<dim3((unsigned)(need < resident ? need : resident)), dim3(C::kThreads), 0, stream>>>(g);
  };
  const bool plain = g.out_dtype == XGEN_DTYPE_BF16 && g.act == XGEN_ACT_NONE;
  // Weights that the call reads about once, in a call that passes the last-level cache, are read past the caches.  Both
  // ways in turn, us past and through them, by rows an expert: 128 experts of 1,536 x 2,048 (FP8) 8 rows 65.0 / 72.4, 37
  // 77.1 / 82.6, 60 84.1 / 86.5, 90 88.4 / 91.0, 110 101.0 / 100.8, 128 (1.45 tile rows) 108.0 / 107.7, 140 (1.56) 114.5 /
  // 113.7, 160 119.6 / 117.0, 180 132.1 / 128.0; 64 of 2,816 x 2,048 60 rows 72.0 / 77.8, 110 88.2 / 90.3, 140 102.6 /
  // 102.6.  Of 29 calls below the bound two lose more than 1%: 64 INT8 experts of 2,048 x 2,048 with 90 rows on 128 x 128
  // tiles (67.0 / 64.7), 256 FP8 ones of 2,048 x 1,024 with 60 (135.0 / 130.1).
  bool once = false;
  if constexpr (C::kM <= 128) {
    const float rows = (float)g.M, groups = (float)g.groups;
    once = g.past && expected_tile_rows(C::kM, rows, groups) < 1.5f * groups * (1.0f - expf(-rows / groups));
    if (once && plain) run(std::true_type(), std::true_type());
    else if (once) run(std::false_type(), std::true_type());
  }
  if (!once && plain) run(std::true_type(), std::false_type());
  else if (!once) run(std::false_type(), std::false_type());
  return launch_status("xgen_grouped_matmul");
}

typedef int (*Launch)(GroupedArgs, hipStream_t);
template <int KIND, int WM, int WN, int FM, int FN, int SLOTS>
constexpr Launch tile_launch() {
  if constexpr (KIND == kFp8Exact && FM * FN >= 16) return nullptr;
  else return launch<KIND, WM, WN, FM, FN, SLOTS>;
}

template <int KIND>
int launch_kind(int tile, const GroupedArgs &g, hipStream_t stream) {
#define XGEN_TILE_LAUNCH(WM, WN, FM, FN, S) tile_launch<KIND, WM, WN, FM, FN, S>(),
  static constexpr Launch fns[kTiles] = {XGEN_GROUPED_TILES(XGEN_TILE_LAUNCH)};
  return fns[tile](g, stream);
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" int xgen_grouped_matmul(int in_dtype, int exact, const void *a, int64_t lda, int64_t a_rows, const void *w,
                                   int64_t ldw, int64_t w_group_stride, int64_t M, int64_t N, int64_t K,
                                   int64_t groups, const int32_t *ends, const int32_t *rows, const float *a_scale,
                                   int64_t a_scale_stride, const float *w_scale, int64_t w_scale_stride,
                                   const void *bias, int bias_dtype, int activation, void *out, int out_dtype,
                                   int64_t ldo, hipStream_t stream) {
  const char *fn = "xgen_grouped_matmul";
  if (!is_quant_dtype(in_dtype)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: operand dtype must be E4M3 or I8", fn);
  if (exact && in_dtype != XGEN_DTYPE_E4M3)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: exact accumulation applies to E4M3 operands", fn);
  if (M < 0 || N <= 0 || K <= 0 || groups <= 0 || a_rows < 0)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape M=%lld N=%lld K=%lld groups=%lld a_rows=%lld", fn,
                (long long)M, (long long)N, (long long)K, (long long)groups, (long long)a_rows);
  if (!rows && a_rows != M)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: without a row index the activation has M rows", fn);
  if (lda < K || ldw < K || ldo < N)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: leading dimensions must cover the rows", fn);
  if (a_scale_stride != 0 && a_scale_stride != 1)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: activation scale stride must be 0 or 1", fn);
  if (w_scale_stride != 0 && w_scale_stride != 1)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: weight scale stride must be 0 or 1", fn);
  if (bias && bias_dtype != XGEN_DTYPE_BF16 && bias_dtype != XGEN_DTYPE_F16 && bias_dtype != XGEN_DTYPE_F32)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bias dtype must be BF16, F16 or F32", fn);
  if (activation != XGEN_ACT_NONE && activation != XGEN_ACT_GELU_TANH)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", fn, activation);
  if (out_dtype != XGEN_DTYPE_BF16 && out_dtype != XGEN_DTYPE_F16)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: output dtype must be BF16 or F16", fn);
  if (groups > XGEN_ROUTE_MAX_EXPERTS)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: up to %d groups", fn, XGEN_ROUTE_MAX_EXPERTS);
  if (M == 0) return ok();
  if ((a_rows && !a) || !w || !ends || (a_rows && !a_scale) || !w_scale || !out)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (K % 16 || N % 16) return fail(XGEN_ERR_UNSUPPORTED, "%s: K and N must be multiples of 16", fn);
  if (lda % 16 || ldw % 16 || w_group_stride % 16 || !aligned16(a) || !aligned16(w))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: operand rows must be 16-byte aligned", fn);
  if (ldo % 8 || !aligned16(out)) return fail(XGEN_ERR_UNSUPPORTED, "%s: output rows must be 16-byte aligned", fn);
  if (!aligned16(bias)) return fail(XGEN_ERR_UNSUPPORTED, "%s: the bias must be 16-byte aligned", fn);
  // 32-bit offsets: within one group's weight, one tile's rows and, gathered, the whole activation
  constexpr int64_t kLimit = 0x7fffffffLL;
  // (rows are counted in tiles of up to 256, rounded up, in 32 bits)
  if (M > kLimit - 256 || N > kLimit / 2 || K > kLimit || ldw > 0xffffffffLL / (N + 512) || (N - 1) * ldw + K > kLimit)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: a group's weight above 2 GiB, or too many rows", fn);
  if (lda > kLimit / 512 || ldo > kLimit / 1024)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: rows too long for 32-bit offsets", fn);
  if (rows && a_rows && (a_rows - 1) * lda + K > kLimit)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: an activation above 2 GiB cannot be indexed", fn);

  GroupedArgs g{};
  g.a = static_cast<const uint8_t *>(a);
  g.w = static_cast<const uint8_t *>(w);
  g.lda = (int)lda;
  g.ldw = (int)ldw;
  g.M = (int)M;
  g.N = (int)N;
  g.K = (int)K;
  g.sa = a_scale;
  g.sa_stride = a_rows ? (int)a_scale_stride : 1;  // (of no rows there is no scale, not even a common one, to read)
  g.sw = w_scale;
  g.sw_stride = (int)w_scale_stride;
  g.bias = bias;
  g.bias_dtype = bias_dtype;
  g.act = activation;
  g.out_dtype = out_dtype;
  g.out = out;
  g.ldo = ldo;
  g.a_bytes = rows && a_rows ? (uint32_t)((a_rows - 1) * lda + K) : 0;
  g.w_bytes = (uint32_t)((N - 1) * ldw + K);
  g.ends = ends;
  g.rows = rows;
  g.groups = (int)groups;
  g.a_rows = a_rows;
  g.w_group = w_group_stride;
  // (at most: groups may be empty)
  g.past = (M < groups ? M : groups) * N * K + M * (2 * N + K) > kLastLevelCacheBytes;
  const int kind = in_dtype == XGEN_DTYPE_I8 ? kInt8 : exact ? kFp8Exact : kFp8;
  const int tile = choose_tile(kind, M, N, K, groups);
  if (kind == kInt8) return launch_kind<kInt8>(tile, g, stream);
  if (kind == kFp8) return launch_kind<kFp8>(tile, g, stream);
  return launch_kind<kFp8Exact>(tile, g, stream);
}

// The rows (and columns, in *n) of the output tiles that a call runs on.  Not part of the C ABI: for the tests,
// which choose their shapes by it.
extern "C" int xgen_grouped_tile_choice(int kind, int64_t M, int64_t N, int64_t K, int64_t groups, int *n) {
  const TileSize t = kTileSizes[choose_tile(kind, M, N, K, groups)];
  *n = t.n;
  return t.m;
}
