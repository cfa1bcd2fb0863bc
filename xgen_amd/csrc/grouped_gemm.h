// The W8A8 product over ragged groups of rows (gfx950): persistent workgroups that stream the output tiles of
// all groups.
//
// A tile is (32 WM FM) rows of one group x (32 WN FN) features, 4 waves of FM x FN MFMA fragments of
// 32 x 32, K in pairs of 64-byte sub-stages through a ring of SLOTS pair slots, as in gemm_tile.h: the same LDS
// rows, MFMA and K order, so an output's accumulator is the same bits as in the product of its group alone.
// What differs is the stream: a workgroup's tiles are one sequence of pairs.  The DMA runs SLOTS pairs
// ahead of the MFMAs and across the tile's end, so a tile's start-up (group search, row indices, first
// loads from memory) passes behind the tile before it, and the epilogue behind loads in flight; one
// tile per workgroup (gemm_tile.h's form) paid 4 to 8 us of those per tile.
//
//   sub-stage 0 of pair p: MFMAs on buffer 0; the fragments of sub-stage 1 are read
//   wait for this thread's DMA of pair p + 1; barrier
//   sub-stage 1 of pair p: MFMAs on buffer 1; the fragments of pair p + 1 are read (not across the
//     tile's end: the epilogue takes their registers); the DMA of pair p + SLOTS
//
// Per tile, in front of its first pair's DMA: its row indices are in LDS already (loaded with the tile
// before), give the rows' offsets, and its scales and bias go to LDS behind them; the indices of the
// tile after it are loaded.
//
// Groups: ends[e] within [0, M] and no less than the end before; rows behind the last end are zeros.  The tile
// rows of all groups, numbered in order, are dealt out as the ungrouped kernel's tiles are: a contiguous
// range per XCD, walked in groups of group_m tile rows of one expert.
//
// Few rows are bound by the weights (8 tokens x 6 of 64 experts, 2,816 x 2,048: 35 us, 5.8 TB/s), many by the matrix
// cores (31,248 rows of 8 experts, 14,336 x 5,376, FP8: 2.0 ms, 2.4 PFLOP/s, what one group of as many rows reaches).
// Between them (2,049 tokens x 8 of 128 experts, 1,536 x 2,048: 105 us; with the weights read through the caches, which
// takes as long, 89 without MFMAs and stores and 56 without memory) it is mostly memory: 449 MB read past the L2, 403 of
// them the weights, and 57 written, 4.8 TB/s, with the matrix cores busy for 35% of the cycles.
#pragma once

#include <utility>

#include "gemm_tile.h"

namespace xgen {

// 4 bytes per lane on the LDS-DMA path: lane l's land at lds + 4 * l.
__device__ __forceinline__ void dma_load4(__amdgpu_buffer_rsrc_t rsrc, uint8_t *lds, uint32_t offset) {
  typedef __attribute__((address_space(3))) void *lds_ptr_t;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 4, offset, 0, 0, 0);
}

// dma_load16 of what the call reads once: non-temporal.
__device__ __forceinline__ void dma_load16_once(__amdgpu_buffer_rsrc_t rsrc, uint8_t *lds, uint32_t offset) {
  typedef __attribute__((address_space(3))) void *lds_ptr_t;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, offset, 0, 0, kCachePolicyNT);
}

// f(0), f(1), .. f(N - 1) with the index a constant.
template <int... I, class F>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F f) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F f) {
  each_of(std::make_integer_sequence<int, N>(), f);
}

template <int WM, int WN, int FM, int FN, int SLOTS>
struct GroupedCfg {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kM = 32 * WM * FM, kN = 32 * WN * FN;
  static constexpr int kLoadsA = kM / 8 / kWaves, kLoadsW = kN / 8 / kWaves, kLoads = kLoadsA + kLoadsW;
  static constexpr int kSlotBytes = (kM + kN) * 128;
  static constexpr int kRing = SLOTS * kSlotBytes;
  // one parameter set: scales of the rows, scales and bias of the features.  A tile's set is filled while the
  // tile before it is multiplied
  static constexpr int kParamSets = 2;
  // (rows: 64 at least, the DMA's lanes)
  static constexpr int kRows = kM < 64 ? 64 : kM, kParamSet = (kRows + 2 * kN) * 4;
  static constexpr int kParamBase = kRing;
  // row indices: loaded a tile ahead of the parameters, read by the epilogue too
  static constexpr int kIndexSets = 3;
  static constexpr int kIndexBase = kParamBase + kParamSets * kParamSet;
  // a wave's transpose area: 32 rows of kXFrags fragments' features, rows 8 bytes apart in banks
  static constexpr int kXFrags = FN > 3 ? 2 : FN, kXPitch = kXFrags * 64 + 8, kXpose = 32 * kXPitch;
  static constexpr int kXposeBase = kIndexBase + kIndexSets * kRows * 4;
  // the groups' first tile rows and first rows
  static constexpr int kTableBase = kXposeBase + kWaves * kXpose;
  static constexpr int kTable = (XGEN_ROUTE_MAX_EXPERTS + 2) * 8;
  // a workgroup's next tiles, filled half by half
  static constexpr int kListed = 64, kListBase = (kTableBase + kTable + 15) / 16 * 16;
  static constexpr int kLdsBytes = kListBase + kListed * 16;
  static constexpr int kStores = FM * FN * 2;  // 16-byte stores per thread and tile
  // pairs per tile at least: a first and a last one, and the ring's (the DMA then reaches the next tile at most)
  static constexpr int kMinPairs = SLOTS > 2 ? SLOTS : 2;
  static_assert(kWaves == 4 && kM % (8 * kWaves) == 0 && kN % (8 * kWaves) == 0 && kM <= 256 && kN <= 256, "DMA split");
  static_assert(FN % kXFrags == 0 && kXposeBase % 8 == 0 && kTableBase % 8 == 0, "epilogue split");
  static_assert(kLdsBytes <= 160 * 1024, "LDS");
};

struct GroupTile {
  int group, row0, rows, n0;  // wave-uniform
};

// PLAIN: a bf16 output without activation; otherwise p.out_dtype and p.act say.  ONCE: the weights are read past the
// caches (a branch on it at every load takes 1 us of 33).
// (every lambda below is inlined: one that is not would hold what it captures in scratch memory)
#define XGEN_INLINE __attribute__((always_inline))
template <int KIND, int WM, int WN, int FM, int FN, int SLOTS, bool PLAIN, bool ONCE>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * WM * WN, 64 * WM * WN), amdgpu_waves_per_eu(1)))
void grouped_gemm_kernel(GroupedArgs p) {
  typedef GroupedCfg<WM, WN, FM, FN, SLOTS> C;
  typedef Mfma<KIND> T;
  typedef typename T::frag_t frag_t;
  constexpr int KS = T::kSteps;
  constexpr int kMfmas = KS * FM * FN;
  constexpr bool kSpread = SLOTS > 2;
  constexpr bool kWeightsOuter = FM <= 2;
  constexpr int kFrags = KS * (FM + FN);
  __shared__ __attribute__((aligned(1024))) uint8_t smem[C::kLdsBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave % WM, wn = wave / WM;
  auto rsrc = [](const void *base, int64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, kBufferFlags);
  };

  // --- the groups' table: first tile row and first row of group e (and of the end) -------------------
  int32_t *tile_row = reinterpret_cast<int32_t *>(smem + C::kTableBase), *first_row = tile_row + XGEN_ROUTE_MAX_EXPERTS + 2;
  const int per = (p.groups + 63) >> 6;  // consecutive groups of a lane
  int tile_rows, last_row;
  {
    constexpr int kMaxPer = XGEN_ROUTE_MAX_EXPERTS / 64;
    // end[i + 1]: of group lane * per + i (past the last group: the last one's, or a lane's padding: the one before);
    // end[0]: of the group before
    int end[kMaxPer + 1] = {}, sum = 0;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) {
      end[i + 1] = 0;
      if (i < per) end[i + 1] = p.ends[lane * per + i < p.groups ? lane * per + i : p.groups - 1];
    }
    // within [0, M], and none below the one before: no row has two groups, and the tiles are as many as the host assumed
#pragma unroll
    for (int i = 1; i <= kMaxPer; ++i) {
      end[i] = end[i] < 0 ? 0 : end[i] > p.M ? p.M : end[i];
      end[i] = end[i] > end[i - 1] ? end[i] : end[i - 1];
    }
    uint32_t top = (uint32_t)end[kMaxPer];  // inclusive prefix maximum over the lanes
    top = max_u32(top, dpp_u32<0x111>(0, top));  // row_shr 1, 2, 4, 8
    top = max_u32(top, dpp_u32<0x112>(0, top));
    top = max_u32(top, dpp_u32<0x114>(0, top));
    top = max_u32(top, dpp_u32<0x118>(0, top));
    top = max_u32(top, dpp_u32<kDppRowBcast15, 0xa>(0, top));
    top = max_u32(top, dpp_u32<kDppRowBcast31, 0xc>(0, top));
    const int up = __shfl_up((int)top, 1), before = lane ? up : 0;
#pragma unroll
    for (int i = 0; i <= kMaxPer; ++i) end[i] = end[i] > before ? end[i] : before;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i)
      if (i < per && end[i + 1] > end[i]) sum += (end[i + 1] - end[i] + C::kM - 1) / C::kM;
    uint32_t incl = (uint32_t)sum;  // inclusive prefix sum over the lanes
    incl += dpp_u32<0x111>(0, incl);
    incl += dpp_u32<0x112>(0, incl);
    incl += dpp_u32<0x114>(0, incl);
    incl += dpp_u32<0x118>(0, incl);
    incl += dpp_u32<kDppRowBcast15, 0xa>(0, incl);
    incl += dpp_u32<kDppRowBcast31, 0xc>(0, incl);
    int at = (int)incl - sum;
    tile_rows = __builtin_amdgcn_readlane((int)incl, 63);
    int last = 0;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) {
      if (i < per) {
        if (wave == 0 && lane * per + i < p.groups) {
          tile_row[lane * per + i] = at;
          first_row[lane * per + i] = end[i];
        }
        if (end[i + 1] > end[i]) at += (end[i + 1] - end[i] + C::kM - 1) / C::kM;
        last = end[i + 1];
      }
    }
    last_row = __builtin_amdgcn_readlane(last, 63);
    if (tid == 0) {
      tile_row[p.groups] = tile_rows;
      first_row[p.groups] = last_row;
    }
  }
  // --- rows behind the last group: zeros, dealt over the workgroups ----------------------------------
  for (int64_t r = last_row + blockIdx.x; r < p.M; r += gridDim.x) {
    uint16_t *o = static_cast<uint16_t *>(p.out) + r * p.ldo;
    for (int c = tid; c < p.N / 8; c += C::kThreads) reinterpret_cast<u32x4 *>(o)[c] = u32x4{0, 0, 0, 0};
  }
  // --- this workgroup's tiles: a contiguous range per XCD, dealt round-robin to its workgroups --------
  const int total = tile_rows * p.tiles_n, per_xcd = (total + 7) >> 3;
  const int xcd = blockIdx.x & 7, wgs_per_xcd = gridDim.x >> 3;
  const int t_first = xcd * per_xcd + (blockIdx.x >> 3);
  const int t_end = (xcd + 1) * per_xcd < total ? (xcd + 1) * per_xcd : total;
  const int n_my = t_first < t_end ? (t_end - t_first + wgs_per_xcd - 1) / wgs_per_xcd : 0;
  if (n_my == 0) return;
  __syncthreads();
  // tiles i .. i + count - 1 of mine, a thread each: into the list
  auto list_tiles = [&](int i, int count) XGEN_INLINE {
    if (tid < count && i + tid < n_my) {
      const int t = t_first + (i + tid) * wgs_per_xcd, mt = t / p.tiles_n;
      int lo = 0, hi = p.groups;  // the group with tile_row[lo] <= mt < tile_row[lo + 1]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile_row[mid] <= mt) lo = mid;
        else hi = mid;
      }
      const int first = tile_row[lo], begin = first_row[lo], end = first_row[lo + 1];
      int m0, n0;
      tile_origin<C::kM, C::kN>(t - first * p.tiles_n, tile_row[lo + 1] - first, p.tiles_n, p.group_m, m0, n0);
      const int left = end - begin - m0;
      *reinterpret_cast<i32x4 *>(smem + C::kListBase + (i + tid) % C::kListed * 16) = i32x4{lo, begin + m0, left < C::kM ? left : C::kM, n0};
    }
  };
  auto find = [&](int i) XGEN_INLINE {  // tile i of mine
    const i32x4 v = *reinterpret_cast<const i32x4 *>(smem + C::kListBase + i % C::kListed * 16);
    return GroupTile{__builtin_amdgcn_readfirstlane(v[0]), __builtin_amdgcn_readfirstlane(v[1]),
                     __builtin_amdgcn_readfirstlane(v[2]), __builtin_amdgcn_readfirstlane(v[3])};
  };

  // --- global -> LDS DMA: lane l fills row (l >> 3) of an 8-row load, physical chunk l & 7, i.e. logical
  // chunk (l & 7) ^ ((row >> 1) & 7); load q of wave w fills rows 8 (q kWaves + w) .. + 7 of its operand ---
  const int ch = ((lane & 7) ^ (((wave & 1) << 2) | (lane >> 4))) * 16;
  const int KP = (p.K + 127) / 128 > C::kMinPairs ? (p.K + 127) / 128 : C::kMinPairs;  // pairs per tile; those past K are zeros
  GroupTile dt{}, nt{};           // the DMA's tile, and the one after it
  int dma_i = 0, dma_k = 0;       // dt's position among mine; K byte of the next pair to load
  uint32_t dma_slot = 0;          // its slot's LDS offset
  uint32_t offa[C::kLoadsA], offw = 0;
  __amdgpu_buffer_rsrc_t ra = rsrc(p.a, 0), rw = rsrc(p.w, 0);
  auto index_set = [&](int i) { return reinterpret_cast<const int32_t *>(smem + C::kIndexBase + i % C::kIndexSets * (C::kRows * 4)); };
  auto load_indices = [&](const GroupTile &g, int i) {
    if (p.rows && wave * 64 < C::kM)
      dma_load4(rsrc(p.rows + g.row0, g.rows * 4), smem + C::kIndexBase + i % C::kIndexSets * (C::kRows * 4) + wave * 256, tid * 4);
  };
  auto row_ok = [&](int at) { return (uint32_t)at < (uint32_t)p.a_rows; };
  // dt's first pair is next: its row offsets, its scales and bias, the indices of the tile after it
  auto next_dma_tile = [&]() XGEN_INLINE {
    const int32_t *index = index_set(dma_i);
#pragma unroll
    for (int q = 0; q < C::kLoadsA; ++q) {
      const int r = wave * 8 + (lane >> 3) + q * C::kWaves * 8;
      const int at = p.rows ? index[r] : r;
      offa[q] = r < dt.rows && (!p.rows || row_ok(at)) ? (uint32_t)at * (uint32_t)p.lda + ch : kOutOfRange;
    }
    ra = p.rows ? rsrc(p.a, p.a_bytes) : rsrc(p.a + (int64_t)dt.row0 * p.lda, (int64_t)(dt.rows - 1) * p.lda + p.K);
    rw = rsrc(p.w + (int64_t)dt.group * p.w_group, p.w_bytes);
    offw = (uint32_t)(dt.n0 + wave * 8 + (lane >> 3)) * (uint32_t)p.ldw + ch;
    uint8_t *prm = smem + C::kParamBase + dma_i % C::kParamSets * C::kParamSet + wave * 256;
    if (wave * 64 < C::kM) {
      const bool one = p.sa_stride == 0;
      const int at = p.rows ? index[tid] : tid;
      const __amdgpu_buffer_rsrc_t r = one ? rsrc(p.sa, 4) : p.rows ? rsrc(p.sa, p.a_rows * 4) : rsrc(p.sa + dt.row0, dt.rows * 4);
      dma_load4(r, prm, one ? 0u : p.rows && !row_ok(at) ? kOutOfRange : (uint32_t)at * 4);
    }
    if (wave * 64 < C::kN) {
      const __amdgpu_buffer_rsrc_t r = p.sw_stride ? rsrc(p.sw + (int64_t)dt.group * p.N, p.N * 4) : rsrc(p.sw + dt.group, 4);
      dma_load4(r, prm + C::kRows * 4, p.sw_stride ? (uint32_t)(dt.n0 + tid) * 4 : 0u);
    }
    if (p.bias && wave * 64 < (p.bias_dtype == XGEN_DTYPE_F32 ? C::kN : C::kN / 2)) {
      const int size = p.bias_dtype == XGEN_DTYPE_F32 ? 4 : 2;
      const uint8_t *b = static_cast<const uint8_t *>(p.bias) + (int64_t)dt.group * p.N * size;
      dma_load4(rsrc(b, p.N * size), prm + (C::kRows + C::kN) * 4, (uint32_t)(dt.n0 * size + tid * 4));
    }
    if (dma_i + 1 < n_my) {
      nt = find(dma_i + 1);
      // the list's other half: every wave is past its tiles
      if ((dma_i + 1) % (C::kListed / 2) == 0) list_tiles(dma_i + 1 + C::kListed / 2, C::kListed / 2);
      load_indices(nt, dma_i + 1);
    }
  };
  bool live = false;
  auto issue_begin = [&]() XGEN_INLINE {
    live = dma_i < n_my && dma_k + ch < p.K;
  };
  // (offsets in range and dma_k are below 2^31, so an offset out of range stays out of it)
  auto issue_load = [&](int q) XGEN_INLINE {
    uint8_t *dst = smem + dma_slot + wave * 1024;
    if (q < C::kLoadsA) {
      dma_load16(ra, dst + q * C::kWaves * 1024, live ? offa[q] + dma_k : kOutOfRange);
    } else {
      const int r = q - C::kLoadsA;
      (ONCE ? dma_load16_once : dma_load16)(rw, dst + C::kM * 128 + r * C::kWaves * 1024,
                                            live ? offw + dma_k + (uint32_t)(r * C::kWaves * 8 * p.ldw) : kOutOfRange);
    }
  };
  auto issue_end = [&]() XGEN_INLINE {
    dma_k += 128;
    if (dma_k == KP * 128) dma_k = 0, ++dma_i;
    dma_slot = dma_slot + C::kSlotBytes == C::kRing ? 0 : dma_slot + C::kSlotBytes;
  };

  // --- fragments: [register buffer = sub-stage][k step][fragment] ---
  // (row block j of a wave: rows 32 (j WM + wm) ..; feature block i: features 32 (wn FN + i) ..)
  const int row_x = wm * 32 + (lane & 31), row_w = wn * 32 * FN + (lane & 31);
  frag_t xf[2][KS][FM], wf[2][KS][FN];
  uint32_t rd_slot = 0;  // LDS offset of the pair being multiplied
  auto read_frag = [&](int b, uint32_t slot, int r) {  // fragment r of sub-stage b, weights first
    const int ks = r / (FM + FN), f = r % (FM + FN);
    if (f < FN) wf[b][ks][f] = load_pair<KIND>(smem + slot + C::kM * 128, row_w + f * 32, b, ks, lane);
    else xf[b][ks][f - FN] = load_pair<KIND>(smem + slot, row_x + (f - FN) * 32 * WM, b, ks, lane);
  };
  auto read_first = [&]() XGEN_INLINE {
#pragma unroll
    for (int r = 0; r < kFrags; ++r) read_frag(0, rd_slot, r);
  };

  typename T::acc_t acc[FN][FM];  // defined by each tile's first sub-stage (mma0)

  // --- epilogue: dequant, bias, activation; a wave's rows through its transpose area into 16-byte pieces ---
  // acc[i][j] element e: feature n0 + (wn*FN + i)*32 + (e/4)*8 + (lane/32)*4 + e%4,
  //                      row     m0 + (j*WM + wm)*32 + lane%32
  auto pin = [](typename T::acc_t &a) XGEN_INLINE { asm volatile("" : "+a"(a)); };  // not read ahead of this
  auto epilogue = [&](const GroupTile &g, int set) XGEN_INLINE {
    constexpr int XF = C::kXFrags, kPieces = XF * 4, kBack = kPieces / 2;
    // 24 wait states behind the last MFMAs before any accumulator is read
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+a"(acc[0][0]));
    each<FN * FM>([&](auto S) XGEN_INLINE {
      constexpr int s = decltype(S)::value;
      pin(acc[s / FM][s % FM]);
    });
    const uint8_t *prm = smem + C::kParamBase + set % C::kParamSets * C::kParamSet;
    const float *psa = reinterpret_cast<const float *>(prm), *psw = psa + C::kRows;
    const uint8_t *pb = prm + (C::kRows + C::kN) * 4;
    int el = lane;  // opaque: the epilogue's addresses are formed here, not held through the stages
    asm volatile("" : "+v"(el));
    const int row = el & 31, half = el >> 5;
    uint8_t *xb = smem + C::kXposeBase + wave * C::kXpose, *xw = xb + row * C::kXPitch + half * 8;
    const __amdgpu_buffer_rsrc_t ro =
        rsrc(static_cast<uint8_t *>(p.out) + (int64_t)g.row0 * p.ldo * 2, ((int64_t)(g.rows - 1) * p.ldo + p.N) * 2);
    float sa[FM];
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const int ml = (j * WM + wm) * 32 + row;
      sa[j] = psa[p.sa_stride ? ml : 0];
      if (p.rows && !row_ok(index_set(set)[ml])) sa[j] = __builtin_nanf("");  // no such row
    }
    // The rows of a step (row block j, fragments i0 ..) are read back behind its writes and stored behind the next
    // step's values: a wave's LDS operations complete in order.  Non-temporal where the call's bytes pass the
    // last-level cache (2,049 tokens x 8 of 128 experts, 2,048 x 1,536: 110 us, 105 so)
    u32x4 back[kBack];
    auto store = [&](int i0, int j) XGEN_INLINE {
#pragma unroll
      for (int q = 0; q < kBack; ++q) {
        const int c = q * 64 + el, r = c / kPieces, col = c % kPieces;
        const int m = (j * WM + wm) * 32 + r, n = g.n0 + (wn * FN + i0) * 32 + col * 8;
        const uint32_t at = m < g.rows && n < p.N ? ((uint32_t)m * (uint32_t)p.ldo + (uint32_t)n) * 2 : kOutOfRange;
        if (p.past) __builtin_amdgcn_raw_buffer_store_b128(back[q], ro, at, 0, kCachePolicyNT);  // uniform
        else __builtin_amdgcn_raw_buffer_store_b128(back[q], ro, at, 0, 0);
      }
    };
    each<FN / XF>([&](auto G) XGEN_INLINE {
      constexpr int i0 = decltype(G)::value * XF;
      f32x4 sw[XF][4], bi[XF][4];  // this lane's 4 features of each group of 8
      const int nl = (wn * FN + i0) * 32 + half * 4;
#pragma unroll
      for (int c = 0; c < XF * 4; ++c) sw[c >> 2][c & 3] = *reinterpret_cast<const f32x4 *>(psw + nl + c * 8);
      if (!p.bias) {
#pragma unroll
        for (int c = 0; c < XF * 4; ++c) bi[c >> 2][c & 3] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      } else if (p.bias_dtype == XGEN_DTYPE_F32) {
#pragma unroll
        for (int c = 0; c < XF * 4; ++c) bi[c >> 2][c & 3] = *reinterpret_cast<const f32x4 *>(pb + (nl + c * 8) * 4);
      } else {
        u32x2 w[XF * 4];
#pragma unroll
        for (int c = 0; c < XF * 4; ++c) w[c] = *reinterpret_cast<const u32x2 *>(pb + (nl + c * 8) * 2);
#pragma unroll
        for (int c = 0; c < XF * 4; ++c)
          bi[c >> 2][c & 3] = p.bias_dtype == XGEN_DTYPE_F16
                                  ? f32x4{Half2<XGEN_DTYPE_F16>::lo(w[c].x), Half2<XGEN_DTYPE_F16>::hi(w[c].x),
                                          Half2<XGEN_DTYPE_F16>::lo(w[c].y), Half2<XGEN_DTYPE_F16>::hi(w[c].y)}
                                  : f32x4{Half2<XGEN_DTYPE_BF16>::lo(w[c].x), Half2<XGEN_DTYPE_BF16>::hi(w[c].x),
                                          Half2<XGEN_DTYPE_BF16>::lo(w[c].y), Half2<XGEN_DTYPE_BF16>::hi(w[c].y)};
      }
      each<FM>([&](auto J) XGEN_INLINE {
        constexpr int j = decltype(J)::value;
        each<XF>([&](auto I) XGEN_INLINE {
          constexpr int ii = decltype(I)::value;
          typename T::acc_t &a = acc[i0 + ii][j];
          pin(a);
#pragma unroll
          for (int gq = 0; gq < 4; ++gq) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(T::to_f32(a[gq * 4 + e]), sa[j] * sw[ii][gq][e], bi[ii][gq][e]);
            u32x2 o;
            if constexpr (PLAIN) {
              o = u32x2{pack_out<XGEN_DTYPE_BF16>(y[0], y[1]), pack_out<XGEN_DTYPE_BF16>(y[2], y[3])};
            } else {
              const bool bf16 = p.out_dtype == XGEN_DTYPE_BF16;
              if (p.act == XGEN_ACT_GELU_TANH) {  // uniform
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  y[e] = gelu_tanh(bf16 ? round_out<XGEN_DTYPE_BF16>(y[e]) : round_out<XGEN_DTYPE_F16>(y[e]));
              }
              const u32x2 ob = {pack_out<XGEN_DTYPE_BF16>(y[0], y[1]), pack_out<XGEN_DTYPE_BF16>(y[2], y[3])};
              const u32x2 oh = {pack_out<XGEN_DTYPE_F16>(y[0], y[1]), pack_out<XGEN_DTYPE_F16>(y[2], y[3])};
              o = u32x2{bf16 ? ob.x : oh.x, bf16 ? ob.y : oh.y};
            }
            *reinterpret_cast<u32x2 *>(xw + (ii * 32 + gq * 8) * 2) = o;
          }
        });
        if constexpr (j > 0) store(i0, j - 1);
        else if constexpr (i0 > 0) store(i0 - XF, FM - 1);
#pragma unroll
        for (int q = 0; q < kBack; ++q) {
          const int c = q * 64 + el;
          const uint8_t *x = xb + c / kPieces * C::kXPitch + c % kPieces * 16;
          const u32x2 lo = *reinterpret_cast<const u32x2 *>(x), hi = *reinterpret_cast<const u32x2 *>(x + 8);
          back[q] = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
      });
    });
    store(FN - XF, FM - 1);
  };

  // one sub-stage: its MFMAs, with the next sub-stage's fragment reads (READ) and a share of a later pair's DMA
  // loads between them; FRESH: the tile's first
  auto sub_stage = [&](auto B, auto FRESH, auto READ, uint32_t next_slot) XGEN_INLINE {
    constexpr int b = decltype(B)::value;
    constexpr bool fresh = decltype(FRESH)::value, read = decltype(READ)::value;
    if constexpr (b == 1) {
      if (dma_k == 0 && dma_i < n_my) {
        dt = nt;
        next_dma_tile();
      }
      issue_begin();
    }
    // the MFMAs are volatile asm statements: the loads written between them stay there
    [[maybe_unused]] typename std::conditional<KIND == kFp8Exact, MfmaA<kFp8Exact>::xw_t, int>::type xw[FM] = {}, ww{};
    each<kMfmas>([&](auto S) XGEN_INLINE {
      constexpr int s = decltype(S)::value, ks = s / (FM * FN);
      constexpr bool outer = KIND == kFp8Exact && kWeightsOuter;
      constexpr int i = outer ? s / FM : s % FN, j = outer ? s % FM : s / FN % FM;
      if constexpr (outer) {
        if constexpr (j == 0) ww = MfmaA<KIND>::widen_x(wf[b][ks][i]);
        if constexpr (i == 0) xw[j] = MfmaA<KIND>::widen_x(xf[b][ks][j]);
      } else if constexpr (KIND == kFp8Exact) {
        if constexpr (i == 0) xw[0] = MfmaA<KIND>::widen_x(xf[b][ks][j]);
      }
      auto mma = [&](auto &w, auto &x) XGEN_INLINE {
        if constexpr (fresh && ks == 0) MfmaA<KIND>::mma0(acc[i][j], w, x);
        else MfmaA<KIND>::mma(acc[i][j], w, x);
      };
      if constexpr (outer) mma(ww, xw[j]);
      else if constexpr (KIND == kFp8Exact) mma(wf[b][ks][i], xw[0]);
      else mma(wf[b][ks][i], xf[b][ks][j]);
      if constexpr (read) {
        constexpr int r0 = spread_first(s, kFrags, kMfmas), r1 = spread_first(s + 1, kFrags, kMfmas);
        each<r1 - r0>([&](auto R) XGEN_INLINE { read_frag(b ^ 1, next_slot, r0 + decltype(R)::value); });
      }
      if constexpr (kSpread || b == 1) {
        // spread: sub-stage 1 takes the first half of a pair's loads, the next sub-stage 0 the rest
        constexpr int kFirst = kSpread ? (C::kLoads + 1) / 2 : C::kLoads, n = b == 1 ? kFirst : C::kLoads - kFirst;
        constexpr int l0 = spread_first(s, n, kMfmas), l1 = spread_first(s + 1, n, kMfmas);
        each<l1 - l0>([&](auto L) XGEN_INLINE { issue_load((b == 1 ? 0 : kFirst) + l0 + decltype(L)::value); });
      }
    });
    if constexpr (b == (kSpread ? 0 : 1)) issue_end();
  };
  typedef std::integral_constant<int, 0> B0;
  typedef std::integral_constant<int, 1> B1;
  typedef std::integral_constant<bool, true> Yes;
  typedef std::integral_constant<bool, false> No;
  // waits for this thread's loads of the next pair (those of SLOTS - 2 pairs, and `stores` stores, were issued after
  // them; the counter retires in issue order), then publishes every wave's and retires the reads of this one
  auto publish = [&](auto STORES) XGEN_INLINE {
    constexpr int n = (SLOTS - 2) * C::kLoads + decltype(STORES)::value;
    wait_vmcnt<(n < 63 ? n : 63)>();
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    lds_barrier();
  };
  auto next_slot = [&]() { return rd_slot + C::kSlotBytes == C::kRing ? 0u : rd_slot + C::kSlotBytes; };

  // --- prologue: the first tile's row indices, SLOTS pairs in flight, pair 0's first fragments ---
  list_tiles(0, C::kListed);
  __syncthreads();
  dt = find(0);
  load_indices(dt, 0);
  wait_vmcnt<0>();
  lds_barrier();
  next_dma_tile();  // (the others' come in the stream: SLOTS pairs are a tile's at most)
#pragma unroll
  for (int s = 0; s < SLOTS; ++s) {
    issue_begin();
#pragma unroll
    for (int q = 0; q < (kSpread && s == SLOTS - 1 ? (C::kLoads + 1) / 2 : C::kLoads); ++q) issue_load(q);
    if (!(kSpread && s == SLOTS - 1)) issue_end();
  }
  wait_vmcnt<(SLOTS - 1) * C::kLoads - (kSpread ? C::kLoads / 2 : 0)>();
  lds_barrier();
  read_first();

  typedef std::integral_constant<int, 0> NoStores;
  auto pair = [&](auto FRESH, auto READ, auto STORES) XGEN_INLINE {
    sub_stage(B0(), FRESH, Yes(), rd_slot);
    publish(STORES);
    const uint32_t next = next_slot();
    sub_stage(B1(), No(), READ, next);
    rd_slot = next;
  };
  for (int i = 0; i < n_my; ++i) {
    const GroupTile g = dt;  // (the DMA reaches the next tile within this one)
    // (the wait of a tile's first pair lets the stores of the epilogue before it be)
    if (i > 0) pair(Yes(), Yes(), std::integral_constant<int, C::kStores>());
    else pair(Yes(), Yes(), NoStores());
    for (int k = 2; k < KP; ++k) pair(No(), Yes(), NoStores());
    pair(No(), No(), NoStores());
    epilogue(g, i);
    if (i + 1 < n_my) read_first();
  }
  // the loads past my last tile may still be writing LDS
  wait_vmcnt<0>();
}

#undef XGEN_INLINE

}  // namespace xgen
