// The norms of queries and keys over each head and their position rotation, in one pass (gfx950), and the
// table of cosines and sines that it reads.
//
//   v = norm(x) * w                          over the head's `dim` values (RMS, layer, or x as it is)
//   the first 2 * pairs values in pairs (a, b), (i, i + pairs) or (2 i, 2 i + 1):
//   a' = a cos[p, i] - b sin[p, i],   b' = b cos[p, i] + a sin[p, i],   p the token's position
//   the head's other values are normed only
//
// With x' the partner of x and m, s the head's mean and 1 / deviation, every value is
//   out = s ((x - m) cw + (x' - m) sw),   cw = w cos,  sw = -+ w' sin   (w and 0 past the pairs),
// and cw, sw belong to the token: a wave forms them once for all of the heads it takes.  fp32 throughout, one
// rounding at the store; layer statistics are two-pass in registers.
//
// Layout: a lane holds 8 consecutive values (16 bytes), a power of two of lanes a head, so its reductions are
// lane shuffles; a wave takes GROUPS such groups of heads of one token.  The halves' partner is another
// lane's chunk (or, where the pairs are no multiple of 8, read again from memory).
//
// Memory bounds it: 15,624 tokens of 112 heads of 128, 904 MB, 172 us (5.2 TB/s, a copy's rate; a wave that took queries and
// keys in turn and read its weights value by value took 366); 3,910 tokens of 40 heads of 64 11 us; one token of each of 4
// requests 3.3 us.  Halves whose pairs are no multiple of 8 read every partner by itself: 422 to 488 us at the
// first of these (10, 60 or 63 pairs; 16, 48 or 64: 166); pairs side by side whose number is none of 4, 162 to 166 (150).
#include <utility>

#include "fastdiv.h"
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Heads that a wave takes, in groups of 64 / LANES: four groups past the caches (15,624 tokens of 112 heads of 128: 172 us,
// 175 with two), one in calls of few groups (64 tokens of those: 3.7 us against 3.9 with two; 128 tokens, 3,584
// groups: 4.9 against 4.7), two in the others (2,000 tokens: 31 us, 35 with one).
constexpr int64_t kFewGroups = 2560;

// Where a chunk's partners come from: halves by whole chunks, side by side, or halves of any length.
enum Pairing { kHalves = 0, kBeside = 1, kHalvesAny = 2 };

struct Heads {
  const uint8_t *x;
  int64_t sb, ss, sh;  // bytes
  const void *w;
  uint8_t *out;
  int heads;
};

struct RotateArgs {
  Heads t[2];          // queries, keys
  uint32_t first, end; // the tokens of this launch
  FastDiv seq;         // token t = b * seq + s
  FastDiv waves;       // wave i = (token - first) * waves + part: GROUPS groups of 64 / LANES heads
  int query_waves;     // the parts that are queries'
  int dim, pairs;
  int norm, weight_dtype;
  bool aligned_tables;
  float eps;
  const float *cos, *sin;
  int64_t places;
  const int64_t *positions;
  int64_t position_batch;  // elements between two batches' positions
};

template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  auto dpp = [](float x, auto ctrl) { return __uint_as_float(dpp_u32<decltype(ctrl)::value>(0, __float_as_uint(x))); };
  if constexpr (LANES >= 2) v += dpp(v, std::integral_constant<int, kDppQuad1032>{});
  if constexpr (LANES >= 4) v += dpp(v, std::integral_constant<int, kDppQuad2301>{});
  if constexpr (LANES >= 8) v += dpp(v, std::integral_constant<int, kDppRowHalfMirror>{});
  if constexpr (LANES >= 16) v += dpp(v, std::integral_constant<int, kDppRowMirror>{});
  if constexpr (LANES >= 32) v += __shfl_xor(v, 16);
  if constexpr (LANES >= 64) v += __shfl_xor(v, 32);
  return v;
}

template <int DT>
__device__ __forceinline__ float load_value(const uint8_t *p) {
  if constexpr (DT == XGEN_DTYPE_BF16) return Half2<DT>::lo(*reinterpret_cast<const uint16_t *>(p));
  else return (float)*reinterpret_cast<const _Float16 *>(p);
}

__device__ __forceinline__ float load_weight(const void *w, int dtype, int i) {
  if (dtype == XGEN_DTYPE_F32) return static_cast<const float *>(w)[i];
  if (dtype == XGEN_DTYPE_BF16) return Half2<XGEN_DTYPE_BF16>::lo(static_cast<const uint16_t *>(w)[i]);
  return (float)static_cast<const _Float16 *>(w)[i];
}

// Eight weights from a multiple of 8 on.
__device__ __forceinline__ void load_weights(const void *w, int dtype, int i, float (&v)[8]) {
  if (dtype == XGEN_DTYPE_F32) {
    const f32x4 *q = reinterpret_cast<const f32x4 *>(static_cast<const float *>(w) + i);
    const f32x4 a = q[0], b = q[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[4 + j] = b[j];
  } else {
    const u32x4 c = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(w) + i);
    if (dtype == XGEN_DTYPE_BF16) unpack8<XGEN_DTYPE_BF16>(c, v);
    else unpack8<XGEN_DTYPE_F16>(c, v);
  }
}

template <int DT, int LANES, int PAIRING, int GROUPS, bool PAST>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs p) {
  const int lane = threadIdx.x & 63;
  const uint32_t id = (uint32_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x * kWaves + (threadIdx.x >> 6)));
  const uint32_t nth = fast_div(id, p.waves), token = p.first + nth;
  if (token >= p.end) return;
  // (queries' waves first: a wave's groups are of one set)
  const int part = (int)(id - nth * p.waves.d);
  const bool keys = part >= p.query_waves;
  const Heads &t = p.t[keys];
  const uint32_t b = fast_div(token, p.seq), s = token - b * p.seq.d;
  constexpr int kHeads = 64 / LANES;  // heads of a group
  const int chunk = lane & (LANES - 1), sub = lane / LANES;
  const int e0 = chunk * 8;
  const bool in = e0 < p.dim;
  const int head0 = (keys ? part - p.query_waves : part) * (GROUPS * kHeads);

  // this lane's chunks, all in flight at once
  const uint8_t *src = t.x + b * t.sb + s * t.ss + (int64_t)(head0 + sub) * t.sh + e0 * 2;
  u32x4 c[GROUPS];
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    c[g] = u32x4{0, 0, 0, 0};
    if (in && head0 + g * kHeads + sub < t.heads) c[g] = stream_load<PAST>(reinterpret_cast<const u32x4 *>(src + g * kHeads * t.sh));
  }

  const int64_t place = p.positions ? p.positions[b * p.position_batch + s] : (int64_t)s;
  const bool known = (uint64_t)place < (uint64_t)p.places;
  // place of value e's partner in its head
  const int rotary = 2 * p.pairs;
  auto partner = [&](int e) {
    if (e >= rotary) return e;
    if constexpr (PAIRING == kBeside) return e ^ 1;
    else return e < p.pairs ? e + p.pairs : e - p.pairs;
  };
  // this lane's values' weights on the cosines, and their partners' on the sines with the product's sign (1 and 0 past the pairs)
  float cw[8], sw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) cw[i] = 1.0f, sw[i] = 0.0f;
  if (known && e0 < rotary) {
    const float *pc = p.cos + place * p.pairs, *ps = p.sin + place * p.pairs;
    if (PAIRING == kBeside && p.aligned_tables) {  // four pairs (their number a multiple of 4)
      const f32x4 a = *reinterpret_cast<const f32x4 *>(pc + e0 / 2), d = *reinterpret_cast<const f32x4 *>(ps + e0 / 2);
#pragma unroll
      for (int i = 0; i < 8; ++i) cw[i] = a[i / 2], sw[i] = i & 1 ? d[i / 2] : -d[i / 2];
    } else if (PAIRING == kHalves && p.aligned_tables) {  // eight pairs' first or second values
      const bool second = e0 >= p.pairs;
      const int i0 = second ? e0 - p.pairs : e0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(pc + i0 + h * 4), d = *reinterpret_cast<const f32x4 *>(ps + i0 + h * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) cw[h * 4 + i] = a[i], sw[h * 4 + i] = second ? d[i] : -d[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (e0 + i < rotary) {
          const bool second = PAIRING == kBeside ? i & 1 : e0 + i >= p.pairs;
          const int at = PAIRING == kBeside ? (e0 + i) / 2 : second ? e0 + i - p.pairs : e0 + i;
          cw[i] = pc[at], sw[i] = second ? ps[at] : -ps[at];
        }
    }
  }
  if (t.w && in) {
    float w[8];
    load_weights(t.w, p.weight_dtype, e0, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) cw[i] *= w[i];
    if constexpr (PAIRING == kBeside) {
#pragma unroll
      for (int i = 0; i < 8; ++i) sw[i] *= w[i ^ 1];
    } else if constexpr (PAIRING == kHalves) {
      load_weights(t.w, p.weight_dtype, partner(e0), w);
#pragma unroll
      for (int i = 0; i < 8; ++i) sw[i] *= w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) sw[i] *= load_weight(t.w, p.weight_dtype, partner(e0 + i));
    }
  }

  // the lane whose chunk holds this chunk's partners (kHalves; its own past the pairs)
  const int other = PAIRING == kHalves ? lane + (partner(e0) - e0) / 8 : lane;
  const float inv_dim = 1.0f / (float)p.dim;
  uint8_t *out = t.out + (((int64_t)token * t.heads + head0 + sub) * p.dim + e0) * 2;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    // (a group's values are formed behind the one before's: all at once take three times the registers)
    __builtin_amdgcn_sched_barrier(0);
    if (head0 + g * kHeads >= t.heads) break;  // (uniform)
    const bool mine = in && head0 + g * kHeads + sub < t.heads;
    float v[8], o[8];
    unpack8<DT>(c[g], v);
    if constexpr (PAIRING == kBeside) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[i ^ 1];
    } else if constexpr (PAIRING == kHalves) {
      u32x4 x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (uint32_t)__shfl((int)c[g][i], other);
      unpack8<DT>(x, o);
    } else {
      const uint8_t *head = src + g * kHeads * t.sh - e0 * 2;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = mine && e0 + i < rotary ? load_value<DT>(head + partner(e0 + i) * 2) : 0.0f;
    }
    // (an unknown place: NaN throughout)
    float mean = 0.0f, scale = known ? 1.0f : __builtin_nanf("");
    if (p.norm != XGEN_NORM_NONE) {
      if (p.norm == XGEN_NORM_LAYER) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += v[i];
        mean = head_sum<LANES>(sum) * inv_dim;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= mean, o[i] -= mean;
      }
      float sum = 0.0f;
      if (in) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(v[i], v[i], sum);
      }
      scale *= __builtin_amdgcn_rsqf(__builtin_fmaf(head_sum<LANES>(sum), inv_dim, p.eps));
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (past the pairs the partner's product is none: a partner of inf would make it NaN)
      const float turn = e0 + i < rotary ? o[i] * sw[i] : 0.0f;
      y[i] = __builtin_fmaf(v[i], cw[i], turn) * scale;
    }
    if (mine) {
      u32x4 r;
      if constexpr (DT == XGEN_DTYPE_BF16)
        r = u32x4{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7])};
      else
        r = u32x4{pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7])};
      stream_store<PAST>(reinterpret_cast<u32x4 *>(out + g * kHeads * p.dim * 2), r);
    }
  }
}

template <int DT, int LANES, int PAIRING>
void launch_rotate(const RotateArgs &p, int groups, bool past, unsigned blocks, hipStream_t stream) {
  if (groups == 1) rotate_kernel<DT, LANES, PAIRING, 1, false><<<blocks, kThreads, 0, stream>>>(p);
  else if (past) rotate_kernel<DT, LANES, PAIRING, 4, true><<<blocks, kThreads, 0, stream>>>(p);
  else rotate_kernel<DT, LANES, PAIRING, 2, false><<<blocks, kThreads, 0, stream>>>(p);
}

template <int DT, int LANES>
void launch_rotate(const RotateArgs &p, int pairing, int groups, bool past, unsigned blocks, hipStream_t stream) {
  if (pairing == kHalves) launch_rotate<DT, LANES, kHalves>(p, groups, past, blocks, stream);
  else if (pairing == kBeside) launch_rotate<DT, LANES, kBeside>(p, groups, past, blocks, stream);
  else launch_rotate<DT, LANES, kHalvesAny>(p, groups, past, blocks, stream);
}

template <int DT>
void launch_rotate(const RotateArgs &p, int lanes, int pairing, int groups, bool past, unsigned blocks, hipStream_t stream) {
  switch (lanes) {
    case 2: return launch_rotate<DT, 2>(p, pairing, groups, past, blocks, stream);
    case 4: return launch_rotate<DT, 4>(p, pairing, groups, past, blocks, stream);
    case 8: return launch_rotate<DT, 8>(p, pairing, groups, past, blocks, stream);
    case 16: return launch_rotate<DT, 16>(p, pairing, groups, past, blocks, stream);
    case 32: return launch_rotate<DT, 32>(p, pairing, groups, past, blocks, stream);
    default: return launch_rotate<DT, 64>(p, pairing, groups, past, blocks, stream);
  }
}

// ---------------------------------------------------------------------------
// cos and sin of positions[p, axis[i]] * f[i], times a factor.  The angle is formed and brought into
// [-pi/4, pi/4] in 64 bits (pi/2 in two parts), where series up to r^13 and r^12 are right to 2^-38 of the value:
// at position 10^6 a 32-bit angle would be off by 0.03.  One rounding, to fp32.  A value a thread: its chain of 64-bit
// operations bounds it: 96 vector instructions a wave, 2.4 us of the card's issue for 15,624 x 64 pairs, which take 5.2 us in a
// graph (a launch of 4 x 64 1.9); the waves wait for the axis and for the position behind it two thirds of their time.  Of
// 249,984 places, 51 us, the issue is 39.
// ---------------------------------------------------------------------------
struct TableArgs {
  const int64_t *positions;
  int axes;
  const double *f;
  const int32_t *axis;
  FastDiv pairs;
  uint32_t values;
  double factor;
  float *cos, *sin;
};

__global__ __launch_bounds__(kThreads) void table_kernel(TableArgs p) {
  const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
  if (at >= p.values) return;
  const uint32_t place = fast_div(at, p.pairs), i = at - place * p.pairs.d;
  const int axis = p.axis ? p.axis[i] : 0;
  double c = __builtin_nan(""), s = c;
  if ((uint32_t)axis < (uint32_t)p.axes) {
    const double t = (double)p.positions[(int64_t)place * p.axes + axis] * p.f[i];
    if (__builtin_fabs(t) < 0x1p36) {  // (false for NaN)
      const double n = __builtin_rint(t * 0.63661977236758134308);  // 2 / pi
      double r = __builtin_fma(-n, 1.57079632679489655800, t);
      r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
      const double q = r * r;
      double a = 1.0 / 6227020800.0, b = 1.0 / 479001600.0;  // 1 / 13!, 1 / 12!
      a = __builtin_fma(a, q, -1.0 / 39916800.0);
      b = __builtin_fma(b, q, -1.0 / 3628800.0);
      a = __builtin_fma(a, q, 1.0 / 362880.0);
      b = __builtin_fma(b, q, 1.0 / 40320.0);
      a = __builtin_fma(a, q, -1.0 / 5040.0);
      b = __builtin_fma(b, q, -1.0 / 720.0);
      a = __builtin_fma(a, q, 1.0 / 120.0);
      b = __builtin_fma(b, q, 1.0 / 24.0);
      a = __builtin_fma(a, q, -1.0 / 6.0);
      b = __builtin_fma(b, q, -0.5);
      a = __builtin_fma(a * q, r, r);
      b = __builtin_fma(b, q, 1.0);
      const int quarter = (int)((int64_t)n & 3);
      c = quarter & 1 ? a : b;
      s = quarter & 1 ? b : a;
      if (quarter == 1 || quarter == 2) c = -c;
      if (quarter >= 2) s = -s;
    }
  }
  p.cos[at] = (float)(c * p.factor);
  p.sin[at] = (float)(s * p.factor);
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" int xgen_qk_norm_rope(int dtype, const void *q, int64_t q_stride_batch, int64_t q_stride_seq, int64_t q_stride_head,
                                 int64_t q_heads, const void *k, int64_t k_stride_batch, int64_t k_stride_seq,
                                 int64_t k_stride_head, int64_t k_heads, int64_t batch, int64_t seq, int64_t dim,
                                 int norm_kind, const void *q_weight, const void *k_weight, int weight_dtype, float eps,
                                 const float *cos, const float *sin, int64_t places, int64_t pairs, int interleaved,
                                 const int64_t *positions, int64_t position_stride_batch, void *q_out, void *k_out,
                                 hipStream_t stream) {
  const char *fn = "xgen_qk_norm_rope";
  if (!is_input_dtype(dtype)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: dtype must be BF16 or F16", fn);
  if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0 || dim <= 0 || pairs <= 0 || pairs > dim / 2 || places < 0)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape", fn);
  if (dim % 8 || dim > XGEN_HEAD_MAX_DIM)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: dim must be a multiple of 8, up to %d", fn, XGEN_HEAD_MAX_DIM);
  if (norm_kind != XGEN_NORM_NONE && norm_kind != XGEN_NORM_LAYER && norm_kind != XGEN_NORM_RMS)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown norm kind %d", fn, norm_kind);
  if ((q_weight || k_weight) && (norm_kind == XGEN_NORM_NONE || (!is_input_dtype(weight_dtype) && weight_dtype != XGEN_DTYPE_F32)))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: weights need a norm, and BF16, F16 or F32 values", fn);
  if (!(eps >= kFltMin && eps < 1.0f)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: eps must be in [2^-126, 1)", fn);
  if (batch == 0 || seq == 0 || q_heads + k_heads == 0) return ok();
  if ((q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out)) || (places && (!cos || !sin)))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  for (const auto &t : {std::make_pair(q_heads ? q : nullptr, q_heads ? q_out : nullptr),
                        std::make_pair(k_heads ? k : nullptr, k_heads ? k_out : nullptr)})
    if (!aligned16(t.first) || !aligned16(t.second)) return fail(XGEN_ERR_UNSUPPORTED, "%s: heads must be 16-byte aligned", fn);
  if ((q_weight && !aligned16(q_weight)) || (k_weight && !aligned16(k_weight)))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: weights must be 16-byte aligned", fn);
  if ((q_heads && (q_stride_batch % 8 || q_stride_seq % 8 || q_stride_head % 8)) ||
      (k_heads && (k_stride_batch % 8 || k_stride_seq % 8 || k_stride_head % 8)))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: strides must be multiples of 8", fn);
  if (q_heads >= (1 << 24) || k_heads >= (1 << 24) || batch >= (1ll << 31) || seq >= (1ll << 31) || batch * seq >= (1ll << 31))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: too many tokens or heads", fn);
  int lanes = 2;
  while (lanes * 8 < dim) lanes *= 2;
  const int64_t per = 64 / lanes, groups_q = (q_heads + per - 1) / per, groups_k = (k_heads + per - 1) / per;
  const bool past = batch * seq * (q_heads + k_heads) * dim * 4 > kLastLevelCacheBytes;  // read and written
  const int groups = past ? 4 : batch * seq * (groups_q + groups_k) <= kFewGroups ? 1 : 2;
  const int64_t waves_q = (groups_q + groups - 1) / groups, waves = waves_q + (groups_k + groups - 1) / groups;
  RotateArgs p;
  p.t[0] = {static_cast<const uint8_t *>(q), q_stride_batch * 2, q_stride_seq * 2, q_stride_head * 2, q_weight,
            static_cast<uint8_t *>(q_out), (int)q_heads};
  p.t[1] = {static_cast<const uint8_t *>(k), k_stride_batch * 2, k_stride_seq * 2, k_stride_head * 2, k_weight,
            static_cast<uint8_t *>(k_out), (int)k_heads};
  p.seq = make_fastdiv((uint32_t)seq);
  p.waves = make_fastdiv((uint32_t)waves);
  p.query_waves = (int)waves_q;
  p.dim = (int)dim;
  p.pairs = (int)pairs;
  p.norm = norm_kind;
  p.weight_dtype = weight_dtype;
  p.aligned_tables = pairs % 4 == 0 && aligned16(cos) && aligned16(sin);
  p.eps = eps;
  p.cos = cos;
  p.sin = sin;
  p.places = places;
  p.positions = positions;
  p.position_batch = position_stride_batch;
  const int pairing = interleaved ? kBeside : pairs % 8 == 0 ? kHalves : kHalvesAny;
  // (a grid's threads are counted in 32 bits; waves is 2^25 at most)
  const int64_t tokens = batch * seq, step = (1ll << 25) / waves;
  for (int64_t first = 0; first < tokens; first += step) {
    const int64_t end = tokens - first < step ? tokens : first + step;
    p.first = (uint32_t)first;
    p.end = (uint32_t)end;
    const unsigned blocks = (unsigned)(((end - first) * waves + kWaves - 1) / kWaves);
    if (dtype == XGEN_DTYPE_BF16) launch_rotate<XGEN_DTYPE_BF16>(p, lanes, pairing, groups, past, blocks, stream);
    else launch_rotate<XGEN_DTYPE_F16>(p, lanes, pairing, groups, past, blocks, stream);
  }
  return launch_status(fn);
}

extern "C" int xgen_rotary_table(const int64_t *positions, int64_t places, int64_t axes, const double *frequencies,
                                 const int32_t *axis, int64_t pairs, double factor, float *cos, float *sin, hipStream_t stream) {
  const char *fn = "xgen_rotary_table";
  if (places < 0 || axes <= 0 || pairs < 0) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape", fn);
  if (places == 0 || pairs == 0) return ok();
  if (!positions || !frequencies || !cos || !sin) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (axes >= (1ll << 31) || places >= (1ll << 31) || pairs >= (1ll << 31) || places * pairs >= (1ll << 31))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: places * pairs must be below 2^31", fn);
  const TableArgs p = {positions, (int)axes, frequencies, axis, make_fastdiv((uint32_t)pairs),
                       (uint32_t)(places * pairs), factor, cos, sin};
  table_kernel<<<(p.values + kThreads - 1) / kThreads, kThreads, 0, stream>>>(p);
  return launch_status(fn);
}
