// The MXFP4 GEMM on 256 x 256 tiles (gfx950): one persistent workgroup per CU, four waves (2 x 2), each with a
// 128 x 128 block of 4 x 4 fragments of v_mfma_scale_f32_32x32x64_f8f6f4, whose 256 accumulators live in AGPRs.
//
// K advances in pairs of stages, 128 bytes (256 values) of each row, through two LDS slots; pair p + 2 is loaded into
// pair p's slot, so a pair's products take two barriers:
//
//   stage A of pair p: its first 128 values' products (32 MFMAs a wave); under the first 16, the second values' fragments
//     are read; release: every wave has read all of pair p's slot, and pair p + 2's DMA begins, a load every other MFMA
//   stage B of pair p: the second 128 values' products; the rest of that DMA; publish: every wave's DMA of pair p + 1
//     (issued a pair before) has landed, and its scales and first fragments are read
//
// A workgroup's tiles follow each other without a gap in this: a tile's last stage B is followed by its epilogue, which
// is the next tile's first stage A too: a fragment's accumulators are read, the next tile's first products on them issued,
// and the values rounded.
//
// Epilogue: the DMA places the weight rows so that a lane's accumulators are runs of eight consecutive features; they
// pass through a 4.5 KB area of LDS of the wave's own, 32 tokens of 64 features at a time, so that each row is stored as one
// 128-byte line (stored from the accumulators' places, 32 bytes of a row at a time, the call below took 142 us
// more).  Past the caches: the output is more than they hold wherever this kernel's tiles fill the card.
//
// What bounds it: the matrix units' power.  15,624 x 14,336 x 5,376, back to back, on normally distributed values takes 517 to
// 550 us, 4.4 to 4.7 PFLOP/s, and twice the K twice that; with zeros in both operands, the same instructions, 423 us (5.7): 341
// in the loop over K (from twice the K: 1.16 us a pair, 7.1 PFLOP/s) and 82 beside it, 5.9 us a round of tiles for the
// epilogues and the waits behind them.  On values those cost little, since the power that they leave is the loop's.  A loop of
// these MFMAs alone does 6.2 to 6.7 PFLOP/s on random codes, 9.65 on zeros.  GELU there 570 to 600 (its arithmetic
// stands between the MFMAs of an epilogue).  15,360 x 5,376 x 14,336 and 264 rows more in a launch of their own: 493 to 530 us, with
// the gated residual 574 to 587 (its reads are waited for; that kernel keeps 68 scalars in lanes of vector registers over the
// loop, the others none).
//
// The same on the fragments of 16 x 16 x 128, which draw less power (7.3 PFLOP/s in the loop): 575 us; there are twice
// as many MFMAs and reads of scales to issue, and the power saved is not what it gained.
#include <utility>

#include "gemm_w8a8.h"

namespace xgen {

namespace {

constexpr int kThreads = 256;
constexpr int kWaveRows = 128;                   // of a wave's block, both dimensions
constexpr int kRowsPerWave = 64;                 // DMA rows per operand and wave
constexpr int F = kWaveRows / 32;                // fragments of a wave's block, both dimensions
constexpr int kSteps = 2;                        // of 64 values, a stage
constexpr int kSlots = kSteps * F * F;           // MFMAs of a stage
constexpr int kFrags = kSteps * 2 * F;           // fragment reads of a stage
constexpr int kTileBytes = 256 * 128;            // one operand of one pair
constexpr int kSlotBytes = 2 * kTileBytes;       // activations, then weights
constexpr int kScaleBase = 2 * kSlotBytes;       // per slot: 8 scale bytes of 256 activation and 256 weight rows
constexpr int kScaleSlot = 2 * 256 * 8;
// the bias as stored, a set per tile: tile t + 3's is issued behind a barrier that follows tile t's epilogue, at
// the earliest (tiles of one pair)
constexpr int kBiasBase = kScaleBase + 2 * kScaleSlot;
constexpr int kBiasSets = 4, kBiasBytes = 1024;
// a wave's transpose area of the epilogue: 32 tokens of 64 features, rows 144 bytes apart (16-byte writes of 16
// consecutive rows fall on 64 different banks)
constexpr int kXposeRow = 144, kXpose = 32 * kXposeRow;
constexpr int kXposeBase = kBiasBase + kBiasSets * kBiasBytes;
constexpr int kLdsBytes = kXposeBase + 4 * kXpose;
constexpr int kLoads = 16;                       // 1 KB loads (8 rows) per wave and pair, and one of scales
constexpr int kStores = 8 * 4;                   // of an epilogue, per wave
static_assert(kLdsBytes <= 160 * 1024, "LDS");

// dma_load16 with a scalar offset, and the instruction's own offset (added to both addresses): plain device functions,
// as dma_load16 is, one per offset.
#define XGEN_DMA_AT(KB)                                                                                              \
  __device__ __forceinline__ void dma_load16_at##KB(__amdgpu_buffer_rsrc_t rsrc, uint8_t *lds, uint32_t offset, int scalar) { \
    typedef __attribute__((address_space(3))) void *lds_ptr_t;                                                       \
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, offset, scalar, KB * 1024, 0);                \
  }
XGEN_DMA_AT(0)
XGEN_DMA_AT(1)
XGEN_DMA_AT(2)
XGEN_DMA_AT(3)
#undef XGEN_DMA_AT

// --- the accumulators: fragment (i, j) of a wave's block, weights i and activations j, is AGPRs 16 (4 i + j) .. + 15, all
// 256 of them, by name.  As variables, the compiler moves some of them where the epilogue joins the loop, right behind
// the instructions that write them; the rest of the kernel fits the VGPRs, so it has no use for AGPRs of its own.  The compiler does
// not know that they hold values between two statements: the build reads this file's assembly, and fails where an
// instruction other than these statements' names one, or scratch is used.
constexpr int acc_reg(int i, int j) { return 16 * (F * i + j); }

#define XGEN_MX4(ADDEND, OPSEL) \
  asm volatile("v_mfma_scale_f32_32x32x64_f8f6f4 a[%0:%1], %2, %3, " ADDEND ", %4, %5 " OPSEL " cbsz:4 blgp:4" ::"n"(R), \
               "n"(R + 15), "v"(w), "v"(x), "v"(sw), "v"(sx))
// c += w x of a pair's step STEP of 64 values, whose scales are that byte of sw and sx; FRESH: c = w x (a tile's first)
template <int R, int STEP, bool FRESH>
__device__ __forceinline__ void mma(const i32x4 &w, const i32x4 &x, uint32_t sw, uint32_t sx) {
  static_assert(R % 16 == 0 && R >= 0 && R < 256 && !(FRESH && STEP), "accumulator");
  if constexpr (FRESH) XGEN_MX4("0", "op_sel_hi:[0,0,0]");
  else if constexpr (STEP == 0) XGEN_MX4("a[%0:%1]", "op_sel_hi:[0,0,0]");
  else if constexpr (STEP == 1) XGEN_MX4("a[%0:%1]", "op_sel:[1,1,0] op_sel_hi:[0,0,0]");
  else if constexpr (STEP == 2) XGEN_MX4("a[%0:%1]", "op_sel_hi:[1,1,0]");
  else XGEN_MX4("a[%0:%1]", "op_sel:[1,1,0] op_sel_hi:[1,1,0]");
}
#undef XGEN_MX4
template <int R>
__device__ __forceinline__ float read_acc() {
  float v;
  asm volatile("v_accvgpr_read_b32 %0, a[%1]" : "=v"(v) : "n"(R));
  return v;
}
// Counts all of them in the kernel's registers (it keeps the compiler off them at this place alone).
__device__ __forceinline__ void take_accumulators() {
#define XGEN_A(N) "a" #N
#define XGEN_A10(T) XGEN_A(T##0), XGEN_A(T##1), XGEN_A(T##2), XGEN_A(T##3), XGEN_A(T##4), XGEN_A(T##5), XGEN_A(T##6), XGEN_A(T##7), XGEN_A(T##8), XGEN_A(T##9)
  asm volatile("" ::: XGEN_A10(), XGEN_A10(1), XGEN_A10(2), XGEN_A10(3), XGEN_A10(4), XGEN_A10(5), XGEN_A10(6), XGEN_A10(7),
               XGEN_A10(8), XGEN_A10(9), XGEN_A10(10), XGEN_A10(11), XGEN_A10(12), XGEN_A10(13), XGEN_A10(14), XGEN_A10(15),
               XGEN_A10(16), XGEN_A10(17), XGEN_A10(18), XGEN_A10(19), XGEN_A10(20), XGEN_A10(21), XGEN_A10(22), XGEN_A10(23),
               XGEN_A10(24), XGEN_A(250), XGEN_A(251), XGEN_A(252), XGEN_A(253), XGEN_A(254), XGEN_A(255));
#undef XGEN_A10
#undef XGEN_A
}

// f(0) .. f(N - 1), each with its index as a constant
template <class Fn, int... I>
__device__ __forceinline__ void unrolled_list(Fn &&f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class Fn>
__device__ __forceinline__ void unrolled(Fn &&f) {
  unrolled_list(f, std::make_integer_sequence<int, N>());
}

template <int ACT, int OUT_DT, bool GATED>
__global__ __attribute__((amdgpu_flat_work_group_size(kThreads, kThreads), amdgpu_waves_per_eu(1, 1)))
void mx4_gemm_kernel(GemmArgs p) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kLdsBytes];

  // --- this workgroup's tiles: a contiguous range per XCD, strided by workgroup ---
  const int ntiles = p.tiles_m * p.tiles_n;
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3, wgs_per_xcd = gridDim.x >> 3;
  const int t_first = xcd * p.per_xcd + local;
  const int t_end = min((xcd + 1) * p.per_xcd, ntiles);
  const int n_my = t_first < t_end ? (t_end - t_first + wgs_per_xcd - 1) / wgs_per_xcd : 0;
  if (n_my == 0) return;
  const int KP = (p.K + 127) / 128;  // pairs per tile

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int half = lane >> 5, r32 = lane & 31;

  auto rsrc = [](const void *base, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)bytes, kBufferFlags);
  };
  const int bias_elem = p.bias_dtype == XGEN_DTYPE_F32 ? 4 : 2;
  const __amdgpu_buffer_rsrc_t rb = rsrc(p.bias, p.bias ? p.N * bias_elem : 0);  // (without a bias: zeros)
  const __amdgpu_buffer_rsrc_t ro = rsrc(p.out, p.out_bytes);

  // --- global -> LDS DMA: wave w fills LDS rows [64 w, 64 w + 64) of both tiles, load l rows 8 l .. 8 l + 7 of them.
  // Lane i fills row i / 8 of a load, physical chunk i % 8, which holds logical chunk (i % 8) ^ ((row / 2) % 8).
  // Row r of a weight fragment's 32 is feature (r / 16) * 16 + (r / 4 % 2) * 8 + (r / 8 % 2) * 4 + r % 4 of its 32: the
  // accumulators of a lane (rows 8 g + 4 half .. + 3, g = 0 .. 3) are then features (g / 2) * 16 + half * 8 + (g % 2) * 4
  // .. + 3, two runs of eight.  Load l's rows start at (l / 4) * 32 + (l / 2 % 2) * 16 + (l % 2) * 4, its upper
  // four 8 features behind the lower. ---
  const int ch_e = ((lane & 7) ^ (lane >> 4)) * 16, ch_o = ((lane & 7) ^ (4 | (lane >> 4))) * 16;
  const int row8 = lane >> 3, wrow8 = (row8 >> 2) * 8 + (row8 & 3);
  // Byte offsets of a tile's 16 loads, each 1 KB further in LDS; four share an LDS base, their place behind it being the
  // instruction's own offset, which the hardware adds to both addresses (so it is taken off here, from offsets that start
  // kBefore bytes ahead of the operands and so stay positive).  A pair's place in K is the scalar offset.  Buffers check
  // the other two's sum alone: it holds the row, and rows past M or N read as zeros.
  constexpr int kBefore = 3 * 1024;
  constexpr uint32_t kNowhere = 0xf0000000u;  // (operands end below 2^31 + kBefore)
  const __amdgpu_buffer_rsrc_t ra = rsrc(p.a - kBefore, p.a_bytes + kBefore), rw = rsrc(p.w - kBefore, p.w_bytes + kBefore);
  uint32_t va[8], vw[8];
  int dma_m0 = 0, dma_n0 = 0;
  auto set_dma_tile = [&](int i) {
    tile_origin<256, 256>(t_first + i * wgs_per_xcd, p.tiles_m, p.tiles_n, p.group_m, dma_m0, dma_n0);
    const uint32_t a = (uint32_t)(dma_m0 + wave * kRowsPerWave + row8) * (uint32_t)p.lda;
    const uint32_t w = (uint32_t)(dma_n0 + wave * kRowsPerWave + wrow8) * (uint32_t)p.ldw;
#pragma unroll
    for (int l = 0; l < 8; ++l) {
      const int ch = (l & 1 ? ch_o : ch_e) + kBefore - (l & 3) * 1024;
      va[l] = a + (uint32_t)(l * 8 * p.lda + ch);
      vw[l] = w + (uint32_t)(((l >> 2) * 32 + (l >> 1 & 1) * 16 + (l & 1) * 4) * p.ldw + ch);
    }
  };
  // lanes whose chunk lies past `left` bytes of K: out of range
  auto mask = [&](int left) {
#pragma unroll
    for (int l = 0; l < 8; ++l)
      if ((l & 1 ? ch_o : ch_e) >= left) va[l] = vw[l] = kNowhere;
  };
  const int sub = (wave & 1) * 128;
  const bool act = wave < 2;  // waves 0 and 1 load the scales of the activations' rows, 2 and 3 of the weights'
  const uint8_t *const scales = act ? p.xs : p.ws;
  const int64_t scale_block = act ? p.xs_block : p.ws_block;
  const uint32_t scale_bytes = act ? p.xs_rows : p.ws_rows;
  int dma_k = 0, dma_i = 0;  // next pair to load: pair dma_k of my tile dma_i
  struct Pair {
    int k0;                  // its place in K, bytes
    uint32_t scale;          // this lane's scales in its block
    __amdgpu_buffer_rsrc_t block;
    int bias_set, bias_offset;  // set -1: not a tile's first pair
  };
  auto prepare = [&]() {
    Pair q;
    const bool live = dma_i < n_my;
    if (dma_k == 0) {
      asm volatile("");  // (the tile's place, with its divisions, stays behind the branch)
      if (live) set_dma_tile(dma_i);
      else mask(0);
    }
    q.k0 = dma_k * 128;
    if (p.K - q.k0 < 128) mask(p.K - q.k0);  // (a tile's last pair)
    q.block = rsrc(scales + dma_k * scale_block, live ? scale_bytes : 0);
    q.scale = (uint32_t)((act ? dma_m0 : dma_n0) + sub + lane * 2) * 8;
    q.bias_set = live && dma_k == 0 ? dma_i % kBiasSets : -1;
    q.bias_offset = dma_n0 * bias_elem;
    if (++dma_k == KP) dma_k = 0, ++dma_i;
    return q;
  };
  // load n of a pair into LDS slot `slot`: 0 the scales (and a tile's bias), then activations and weights by fours
  auto issue = [&](const Pair &q, uint32_t slot, auto N) {
    constexpr int n = decltype(N)::value;
    if constexpr (n == 0) {
      if (q.bias_set >= 0 && wave == 2)
        dma_load16(rb, smem + kBiasBase + q.bias_set * kBiasBytes, (uint32_t)q.bias_offset + lane * 16);
      dma_load16(q.block, smem + kScaleBase + slot * kScaleSlot + wave * 1024, q.scale);
    } else {
      constexpr int l = (n - 1) % 8;
      constexpr bool weights = n > 8;
      uint8_t *dst = smem + slot * kSlotBytes + wave * (kRowsPerWave * 128) + (l & 4) * 1024 + (weights ? kTileBytes : 0);
      const __amdgpu_buffer_rsrc_t r = weights ? rw : ra;
      const uint32_t offset = weights ? vw[l] : va[l];
      if constexpr ((l & 3) == 0) dma_load16_at0(r, dst, offset, q.k0);
      else if constexpr ((l & 3) == 1) dma_load16_at1(r, dst, offset, q.k0);
      else if constexpr ((l & 3) == 2) dma_load16_at2(r, dst, offset, q.k0);
      else dma_load16_at3(r, dst, offset, q.k0);
    }
  };

  // --- fragments and scales: LDS offsets of this lane, of the slot whose pair is read ---
  const int key = (r32 >> 1) & 7;
  uint32_t fx = (uint32_t)(wm * kWaveRows + r32) * 128 + ((half ^ key) << 4);  // step 0's; the others': ^ 32, 64, 96
  uint32_t fw = (uint32_t)(wn * kWaveRows + r32) * 128 + ((half ^ key) << 4) + kTileBytes;
  const int wfeature = (r32 >> 4) * 16 + (r32 >> 2 & 1) * 8 + (r32 >> 3 & 1) * 4 + (r32 & 3);  // of fragment 0's rows
  uint32_t sx = kScaleBase + (uint32_t)(wm * kWaveRows + r32) * 8 + half * 4;
  uint32_t sw = kScaleBase + 2048 + (uint32_t)(wn * kWaveRows + wfeature) * 8 + half * 4;
  i32x4 xf[2][kSteps][F], wf[2][kSteps][F];  // [stage][step][fragment]
  uint32_t sc[2][2 * F];                     // scales: weights, then activations; stage B's are copies
  auto read = [&](int stage, int r) {        // step by step, weights first
    const int ks = r / (2 * F), f = r % (2 * F);
    const uint32_t flip = (stage * 2 + ks) * 32;
    if (f < F) wf[stage][ks][f] = *reinterpret_cast<const i32x4 *>(smem + (fw ^ flip) + f * 4096);
    else xf[stage][ks][f - F] = *reinterpret_cast<const i32x4 *>(smem + (fx ^ flip) + (f - F) * 4096);
  };
  auto read_scale = [&](int f) {  // a row's dword of this lane's half: its blocks half, half + 2, half + 4, half + 6
    sc[0][f] = *reinterpret_cast<const uint32_t *>(smem + (f < F ? sw + f * 256 : sx + (f - F) * 256));
  };
  auto copy_scale = [&](int f) { asm volatile("v_mov_b32 %0, %1" : "=v"(sc[1][f]) : "v"(sc[0][f])); };
  auto next_slot = [&]() { fx ^= kSlotBytes, fw ^= kSlotBytes, sx ^= kScaleSlot, sw ^= kScaleSlot; };

  take_accumulators();
  uint32_t slot = 0;  // of the pair that is multiplied
  Pair q;

  // Slots (MFMAs) of the two stages: stage B waits and publishes at kPublish, stage A releases at kRelease; the DMA's
  // loads follow the release, one every kSpacing slots, through stage A and on into stage B.
  constexpr int kPublish = 10, kRelease = 19, kSpacing = 2;
  constexpr int kLoadsA = (kSlots - kRelease - 1 + kSpacing - 1) / kSpacing;  // issued in stage A (or behind an epilogue)
  constexpr int kFirstB = kSpacing - (kSlots - kRelease - 1 - (kLoadsA - 1) * kSpacing);  // stage B's first slot with one
  constexpr int kNewer = kLoadsA + (kPublish - kFirstB + kSpacing - 1) / kSpacing;        // in flight at kPublish that may stay so
  static_assert(kFirstB >= 0 && kFirstB + (kLoads - kLoadsA) * kSpacing < kSlots, "the loads fit");
  static_assert(kFrags < kRelease && kPublish + 1 + kFrags <= kSlots, "the reads fit");

  // this wave's reads of stage B's fragments are done: with every wave's, the pair's slot is free
  auto release = [&]() {
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    lds_barrier();
  };
  // The MFMAs are volatile asm statements: what is written between them stays there.
  auto stage_a = [&](auto FRESH) {
    unrolled<kSlots>([&](auto S) {
      constexpr int s = decltype(S)::value, ks = s / (F * F), j = s / F % F, i = s % F;
      mma<acc_reg(i, j), ks, decltype(FRESH)::value && ks == 0>(wf[0][ks][i], xf[0][ks][j], sc[0][i], sc[0][F + j]);
      if constexpr (s < kFrags) read(1, s);
      if constexpr (s < 2 * F) copy_scale(s);
      if constexpr (s == kFrags) q = prepare();
      if constexpr (s == kRelease) release();
      if constexpr (s > kRelease && (s - kRelease - 1) % kSpacing == 0) issue(q, slot, std::integral_constant<int, (s - kRelease - 1) / kSpacing>());
    });
  };
  bool stores = false;  // an epilogue's are in flight, issued behind the DMA that is waited for
  auto stage_b = [&]() {
    next_slot();
    unrolled<kSlots>([&](auto S) {
      constexpr int s = decltype(S)::value, ks = s / (F * F), j = s / F % F, i = s % F;
      if constexpr (s == kPublish) {
        if (stores) wait_vmcnt<kNewer + kStores>();
        else wait_vmcnt<kNewer>();
        stores = false;
        lds_barrier();
      }
      mma<acc_reg(i, j), 2 + ks, false>(wf[1][ks][i], xf[1][ks][j], sc[1][i], sc[1][F + j]);
      if constexpr (s >= kFirstB && (s - kFirstB) % kSpacing == 0 && kLoadsA + (s - kFirstB) / kSpacing <= kLoads)
        issue(q, slot, std::integral_constant<int, kLoadsA + (s - kFirstB) / kSpacing>());
      if constexpr (s >= kPublish && s < kPublish + 2 * F) read_scale(s - kPublish);
      if constexpr (s > kPublish && s <= kPublish + kFrags) read(0, s - kPublish - 1);
    });
    slot ^= 1;
  };

  // eight biases from `feature` on and eight from feature + 16 on (without a bias: zeros)
  auto read_bias = [&](const uint8_t *pb, int feature, float (&bias)[16]) {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      float v[8];
      if (p.bias_dtype == XGEN_DTYPE_F32) {
        const f32x4 *b = reinterpret_cast<const f32x4 *>(pb + (feature + m * 16) * 4);
        const f32x4 lo = b[0], hi = b[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lo[e], v[4 + e] = hi[e];
      } else {
        const u32x4 b = *reinterpret_cast<const u32x4 *>(pb + (feature + m * 16) * 2);
        if (p.bias_dtype == XGEN_DTYPE_F16) unpack8<XGEN_DTYPE_F16>(b, v);
        else unpack8<XGEN_DTYPE_BF16>(b, v);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[m * 8 + e] = v[e];
    }
  };

  int tile_i = 0;
  // accumulators (i, j), values 8 m .. 8 m + 7: features n0 + wn*128 + i*32 + m*16 + (lane/32)*8 + 0 .. 7, token m0 + wm*128 + j*32 + lane%32
  auto epilogue = [&]() {
    int m0, n0;
    tile_origin<256, 256>(t_first + tile_i * wgs_per_xcd, p.tiles_m, p.tiles_n, p.group_m, m0, n0);
    // (opaque: the epilogue's addresses are formed here, not held through the loop)
    int el = lane;
    asm volatile("" : "+v"(el));
    const int feature = wn * kWaveRows + (el >> 5) * 8;  // + i * 32 + m * 16
    const uint8_t *pb = smem + kBiasBase + (tile_i % kBiasSets) * kBiasBytes;
    uint8_t *xb = smem + kXposeBase + wave * kXpose;
    uint8_t *xw = xb + (el & 31) * kXposeRow + (el >> 5) * (GATED ? 32 : 16);
    // this lane's pieces of what is read back: 8 features of kPieces rows of each 32 tokens, kBetween apart
    constexpr int kLanes = GATED ? 4 : 8, kBetween = 64 / kLanes, kPieces = 32 / kBetween;
    const uint8_t *xr = xb + el / kLanes * kXposeRow + el % kLanes * (GATED ? 32 : 16);
    const int col = n0 + wn * kWaveRows + el % kLanes * 8;                   // + the block's first feature
    const uint32_t row = (uint32_t)(m0 + wm * kWaveRows + el / kLanes);      // + j * 32 + q * kBetween
    const uint32_t at = (row * (uint32_t)p.ldo + (uint32_t)col) * 2;         // rows past M lie past the output's bytes
    const uint32_t step = kBetween * 2 * (uint32_t)p.ldo;                    // bytes of kBetween rows
    [[maybe_unused]] __amdgpu_buffer_rsrc_t rres, rgate;
    [[maybe_unused]] uint32_t gate_row[F][kPieces];  // byte offset, or kOutOfRange: an index outside the table
    [[maybe_unused]] u32x4 res[kPieces], gate[kPieces];
    if constexpr (GATED) {
      rres = rsrc(p.residual, p.residual_bytes);
      rgate = rsrc(p.gate, p.gate_bytes);
      const __amdgpu_buffer_rsrc_t rind = rsrc(p.indices, p.seq * 8);
#pragma unroll
      for (int n = 0; n < kPieces * F; ++n) {
        const uint32_t m = row + n * kBetween + p.seq_first, mq = (__umulhi(m, p.seq_magic) + m) >> p.seq_shift;
        const u32x2 index = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rind, (m - mq * p.seq) * 8, 0, 0));
        gate_row[n / kPieces][n % kPieces] = index.y == 0 && index.x < (uint32_t)p.gate_rows ? index.x * (uint32_t)p.gate_stride * 2 : kOutOfRange;
      }
    }
    u32x4 pending[kPieces][GATED ? 2 : 1];  // as read back: rounded, or with a gated residual in fp32
    auto store = [&](int first, int j) {
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        u32x4 v = pending[q][0];
        if constexpr (GATED) {
          const f32x4 lo = __builtin_bit_cast(f32x4, pending[q][0]), hi = __builtin_bit_cast(f32x4, pending[q][1]);
          const float y[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          v = gate_row[j][q] != kOutOfRange ? gate_residual8(res[q], y, gate[q])
                                            : u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
        }
        __builtin_amdgcn_raw_buffer_store_b128(v, ro, col + first < p.N ? at + (j * kPieces + q) * step + first * 2 : kOutOfRange, 0,
                                               kCachePolicyNT);
      }
    };
    // what has passed the transpose area: 32 tokens (j) of the features from `first` on; the step before is stored while
    // this one's rows are read back (a wave's LDS operations complete in order)
    auto read_back = [&](int first, int j) {
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const u32x4 *from = reinterpret_cast<const u32x4 *>(xr + q * kBetween * kXposeRow);
        pending[q][0] = from[0];
        if constexpr (GATED) {
          pending[q][1] = from[1];
          const uint32_t c = (uint32_t)(col + first);
          const bool in = c < (uint32_t)p.N;
          res[q] = __builtin_amdgcn_raw_buffer_load_b128(
              rres, in ? ((row + j * 32 + q * kBetween) * (uint32_t)p.ld_residual + c) * 2 : kOutOfRange, 0, 0);
          gate[q] = __builtin_amdgcn_raw_buffer_load_b128(
              rgate, in && gate_row[j][q] != kOutOfRange ? gate_row[j][q] + c * 2 : kOutOfRange, 0, 0);
        }
      }
    };
    float bias[2][16];
    unrolled<F * F>([&](auto B) {
      // 32 tokens (j) of 64 features (h) after the others: fragments 2 h and 2 h + 1
      constexpr int n = decltype(B)::value, h = n / 8, j = n / 2 % 4, ii = n % 2, i = 2 * h + ii, R = acc_reg(i, j);
      if constexpr (j == 0) read_bias(pb, feature + i * 32, bias[ii]);
      float y[16];
      unrolled<16>([&](auto E) { y[E] = read_acc<R + decltype(E)::value>(); });
      mma<R, 0, true>(wf[0][0][i], xf[0][0][j], sc[0][i], sc[0][F + j]);
      // (a block's second products behind the next one's first: they add to the same registers)
      if constexpr (n > 0) {
        constexpr int b1 = n - 1, i1 = b1 / 8 * 2 + b1 % 2, j1 = b1 / 2 % 4;
        mma<acc_reg(i1, j1), 1, false>(wf[0][1][i1], xf[0][1][j1], sc[0][i1], sc[0][F + j1]);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        y[e] += bias[ii][e];
        if constexpr (ACT == XGEN_ACT_GELU_TANH) y[e] = gelu_tanh(y[e]);
      }
      if constexpr (GATED) {
        // in fp32, a fragment's 32 features at a time: the product with the gate and the sum are rounded once
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *reinterpret_cast<f32x4 *>(xw + e / 8 * 64 + e % 8 * 4) = f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]};
        if constexpr (n > 0) store(((n - 1) / 8 * 2 + (n - 1) % 2) * 32, (n - 1) / 2 % 4);
        read_back(i * 32, j);
      } else {
#pragma unroll
        for (int m = 0; m < 2; ++m)
          *reinterpret_cast<u32x4 *>(xw + ii * 64 + m * 32) =
              u32x4{pack_out<OUT_DT>(y[8 * m], y[8 * m + 1]), pack_out<OUT_DT>(y[8 * m + 2], y[8 * m + 3]),
                    pack_out<OUT_DT>(y[8 * m + 4], y[8 * m + 5]), pack_out<OUT_DT>(y[8 * m + 6], y[8 * m + 7])};
        if constexpr (ii == 1) {
          if constexpr (n > 1) store((n - 2) / 8 * 64, (n - 2) / 2 % 4);
          read_back(h * 64, j);
        }
      }
    });
    store(GATED ? (F - 1) * 32 : 64, F - 1);
    mma<acc_reg(F - 1, F - 1), 1, false>(wf[0][1][F - 1], xf[0][1][F - 1], sc[0][F - 1], sc[0][2 * F - 1]);
    // the rest of a stage A, for the next tile's first pair (behind the epilogue, which needs the fragments' registers)
#pragma unroll
    for (int r = 0; r < kFrags; ++r) read(1, r);
#pragma unroll
    for (int f = 0; f < 2 * F; ++f) copy_scale(f);
    q = prepare();
    release();
    unrolled<kLoadsA>([&](auto N) { issue(q, slot, N); });
    ++tile_i;
  };

  // --- prologue: pairs 0 and 1 in flight, pair 0's first fragments in registers ---
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    q = prepare();
    unrolled<kLoads + 1>([&](auto N) { issue(q, s, N); });
  }
  wait_vmcnt<kLoads + 1>();
  lds_barrier();
#pragma unroll
  for (int r = 0; r < kFrags; ++r) read(0, r);
#pragma unroll
  for (int f = 0; f < 2 * F; ++f) read_scale(f);

  typedef std::integral_constant<bool, true> Fresh;
  typedef std::integral_constant<bool, false> Sum;
  stage_a(Fresh());  // the first tile's; the others' run with the epilogues
  int left = KP;
  for (int h = n_my * KP; h > 0; --h) {
    stage_b();
    if (--left > 0) {
      stage_a(Sum());
    } else {
      // 24 wait states behind the last MFMAs before any accumulator is read
      asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7");
      // after the last tile too: the "next tile" is then zeros, and its products are unused
      epilogue();
      stores = true;
      left = KP;
    }
  }
  // the loads of the pairs past my last may still be writing LDS
  wait_vmcnt<0>();
}

template <int ACT, int OUT_DT, bool GATED>
void launch(const GemmArgs &g, hipStream_t stream) {
  const int ntiles = g.tiles_m * g.tiles_n, need = (ntiles + 7) / 8 * 8;
  int wgs = device_cu_count() / 8 * 8;
  if (wgs > need) wgs = need;
  if (wgs < 8) wgs = 8;
  mx4_gemm_kernel<ACT, OUT_DT, GATED><<<dim3((unsigned)wgs), dim3(kThreads), 0, stream>>>(g);
}

}  // namespace

void launch_mx4_gemm(const GemmArgs &g, hipStream_t stream) {
  if (g.residual) launch<XGEN_ACT_NONE, XGEN_DTYPE_BF16, true>(g, stream);
  else if (g.act == XGEN_ACT_NONE && g.out_dtype == XGEN_DTYPE_BF16) launch<XGEN_ACT_NONE, XGEN_DTYPE_BF16, false>(g, stream);
  else if (g.act == XGEN_ACT_NONE) launch<XGEN_ACT_NONE, XGEN_DTYPE_F16, false>(g, stream);
  else if (g.out_dtype == XGEN_DTYPE_BF16) launch<XGEN_ACT_GELU_TANH, XGEN_DTYPE_BF16, false>(g, stream);
  else launch<XGEN_ACT_GELU_TANH, XGEN_DTYPE_F16, false>(g, stream);
}

}  // namespace xgen
