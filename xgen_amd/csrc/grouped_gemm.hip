// W8A8 products over ragged groups of rows, each group with a weight of its own (gfx950): the experts of
// a feed-forward, the streams of a dual-stream block.  The kernel is the tile kernel of gemm_tile.h: an output
// tile never spans two groups, a workgroup finds its tile from the group ends on the device (no host
// synchronization), and reads its activation rows through an index where one is given (each token's row is
// read where it lies; no permuted copy).  An output's accumulator is the same bits as in the
// product of its group alone.
#include "gemm_tile.h"

namespace xgen {

namespace {

// (waves x, waves y, fragments x, fragments y, pair slots), as in gemm_tile.hip
#define XGEN_GROUPED_TILES(X) \
  X(1, 2, 1, 1, 6) /*  32 x  64 */ \
  X(2, 2, 1, 1, 6) /*  64 x  64 */ \
  X(2, 2, 1, 2, 4) /*  64 x 128 */ \
  X(2, 2, 2, 2, 4) /* 128 x 128 */ \
  X(2, 2, 2, 3, 3) /* 128 x 192 */ \
  X(2, 2, 4, 2, 3) /* 256 x 128 */ \
  X(2, 2, 4, 3, 2) /* 256 x 192 */

constexpr int kTiles = 7;
struct TileSize {
  int m, n, slots;
};
#define XGEN_TILE_SIZE(WM, WN, FM, FN, S) {TileCfg<WM, WN, FM, FN, S>::kM, TileCfg<WM, WN, FM, FN, S>::kN, S},
constexpr TileSize kTileSizes[kTiles] = {XGEN_GROUPED_TILES(XGEN_TILE_SIZE)};

// us: start + rounds * (pairs * per_pair + per_tile), as in gemm_tile.hip
struct TileCost {
  float per_pair, per_tile, start;
};
constexpr TileCost kTileCosts[3][kTiles] = {
    // INT8
    {{0.203f, 0.1f, 3.1f}, {0.242f, 2.1f, 1.3f}, {0.39f, 1.3f, 3.3f}, {0.503f, 3.9f, 1.8f}, {0.668f, 5.2f, 1.8f},
     {0.751f, 7.3f, 0.0f}, {1.18f, 8.5f, 0.0f}},
    // FP8
    {{0.202f, 0.1f, 3.0f}, {0.241f, 2.1f, 1.4f}, {0.389f, 1.0f, 3.4f}, {0.499f, 3.0f, 2.4f}, {0.643f, 4.8f, 2.3f},
     {0.72f, 6.6f, 0.5f}, {1.14f, 7.4f, 0.7f}},
    // FP8 exact
    {{0.266f, 0.0f, 4.0f}, {0.367f, 2.2f, 1.5f}, {0.492f, 3.0f, 1.2f}, {0.771f, 4.7f, 0.0f}, {1.06f, 4.8f, 0.0f},
     {1.35f, 6.4f, 0.0f}, {1.92f, 7.8f, 0.0f}},
};

// Tiles that a call's groups come to at m rows a tile, from what the host knows: M rows in `groups` groups.
// Groups of few rows are one tile each (those that are not empty); larger ones end inside a tile, half way on
// the average.
float expected_tile_rows(int m, int64_t M, int64_t groups) {
  const float mean = (float)M / (float)groups;
  const float filled = (float)groups * (1.0f - expf(-mean));
  return filled * (mean > 0.5f * (float)m ? mean / (float)m + 0.5f : 1.0f);
}

int choose_tile(int kind, int64_t M, int64_t N, int64_t K, int64_t groups) {
  int best = 0;
  float cost = 0.0f;
  for (int t = 0; t < kTiles; ++t) {
    const float tiles = expected_tile_rows(kTileSizes[t].m, M, groups) * (float)((N + kTileSizes[t].n - 1) / kTileSizes[t].n);
    const float rounds = ceilf(tiles / (float)device_cu_count());
    const int64_t steps = (K + 127) / 128;
    const float pairs = (float)(steps > kTileSizes[t].slots ? steps : kTileSizes[t].slots);
    const TileCost c = kTileCosts[kind][t];
    const float us = c.start + rounds * (pairs * c.per_pair + c.per_tile);
    if (t == 0 || us < cost) best = t, cost = us;
  }
  return best;
}

template <int KIND, int WM, int WN, int FM, int FN, int SLOTS>
int launch(GroupedArgs g, hipStream_t stream) {
  typedef TileCfg<WM, WN, FM, FN, SLOTS> C;
  g.tiles_n = (g.N + C::kN - 1) / C::kN;
  g.group_m = 8 * kTileM / C::kM;
  // at most one tile per group ends short of kM rows (the rows behind the last group count as one)
  const int64_t parts = g.M < g.groups + 1 ? g.M : g.groups + 1;
  const int64_t tiles = (g.M / C::kM + parts) * g.tiles_n;
  if (tiles > 0x3fffffffLL) return fail(XGEN_ERR_UNSUPPORTED, "xgen_grouped_matmul: too many output tiles");
  gemm_tile_kernel<KIND, WM, WN, FM, FN, SLOTS, false, GroupedArgs>
      <<<dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(C::kThreads), 0, stream>>>(g);
  return launch_status("xgen_grouped_matmul");
}

template <int KIND>
int launch_kind(int tile, const GroupedArgs &g, hipStream_t stream) {
  typedef int (*Fn)(GroupedArgs, hipStream_t);
#define XGEN_TILE_LAUNCH(WM, WN, FM, FN, S) launch<KIND, WM, WN, FM, FN, S>,
  static constexpr Fn fns[kTiles] = {XGEN_GROUPED_TILES(XGEN_TILE_LAUNCH)};
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
  // 32-bit offsets: within one group's weight, one tile's rows and, gathered, the whole activation
  constexpr int64_t kLimit = 0x7fffffffLL;
  if (M > kLimit || N > kLimit / 2 || K > kLimit || ldw > 0xffffffffLL / (N + 512) || (N - 1) * ldw + K > kLimit)
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
  g.sa_stride = (int)a_scale_stride;
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
  const int kind = in_dtype == XGEN_DTYPE_I8 ? kInt8 : exact ? kFp8Exact : kFp8;
  const int tile = choose_tile(kind, M, N, K, groups);
  if (kind == kInt8) return launch_kind<kInt8>(tile, g, stream);
  if (kind == kFp8) return launch_kind<kFp8>(tile, g, stream);
  return launch_kind<kFp8Exact>(tile, g, stream);
}
