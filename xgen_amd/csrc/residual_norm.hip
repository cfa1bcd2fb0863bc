// The norms behind and in front of a block's branch, fused with its gate, its residual scale, the
// AdaLN-table modulation and the next projection's per-row quantization (gfx950):
//
//   stream = a * x + gate[g] * (norm_b(y) * w_b)
//   h      = norm(stream) * w * (1 + scale[g]) + shift[g],   g = indices[s]
//   out    = bf16(h), or (q, s) = quantize_row(h)
//
// Everything between the loads and the stores is fp32: the stream's rounding to bf16 and the rows'
// rounding are the only ones (the rows are normed from the unrounded stream; of the eager bf16 form's
// nine roundings per value seven are gone).
//
// One pass: a row stays in registers between its one read of x and y and its writes.  Layer statistics are
// two-pass there (mean, then squared deviations): no cancellation whatever the row's offset.
//
// Layout: rows up to 1,024 values take a wave each, wider ones a workgroup of four waves, whose
// reductions meet in LDS with one barrier each.  Workgroups as are resident at once walk the
// rows; both norm weights stay in registers over the walk.  Memory bound: 15,624 x 5,376 with gate, scale and shift
// tables, bf16 out: 129 us, 5.2 TB/s (the rate of a large copy); e4m3fn out 120 us.  That call reads and writes past
// the caches (129 us; through them 136).  Smaller ones go through them: at 4,000 rows past them is faster alone
// (31 against 38 us), but slower with a kernel behind that reads both outputs (62.5 against 60).  One row takes
// 4 us (the launch, its loads and reductions), and further rows what their bytes do: 256 rows 6, 501 rows 8.
#include "fastdiv.h"
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kThreads = 256;

struct ResNormArgs {
  const uint8_t *x, *y;
  int64_t xsb, xss, ysb, yss;  // bytes
  FastDiv seq;                 // row r = b * seq + s
  int64_t rows;
  int width;
  int branch_norm, norm;  // XGEN_NORM_LAYER, XGEN_NORM_RMS; branch_norm also XGEN_NORM_NONE
  const void *branch_weight, *weight;  // of dtype WT (kernel template), or null
  const uint8_t *gate, *scale, *shift;
  int64_t gate_stride, scale_stride, shift_stride;  // bytes
  int64_t table_rows;
  const int64_t *indices;  // null without tables
  float residual_scale, eps;
  uint8_t *stream, *out;
  float *token_scale;
};

// Slots of the cross-wave reductions: one set per reduction of a row step, alternating between even and odd
// steps (a wave writes a set again two steps later, behind a barrier that every wave passed after reading it).
constexpr int kReductions = 5;
struct Slots {
  float v[kReductions][4];
};

template <int WPR>
__device__ __forceinline__ float row_sum(float v, int wave, int lane, float (&red)[4]) {
  v = wave_sum_f32(v);
  if constexpr (WPR > 1) {
    if (lane == 0) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}
template <int WPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, int wave, int lane, float (&red)[4]) {
  v = wave_max_u32(v);
  if constexpr (WPR > 1) {
    if (lane == 0) red[wave] = __uint_as_float(v);
    __syncthreads();
    const uint32_t a = max_u32(__float_as_uint(red[0]), __float_as_uint(red[1]));
    const uint32_t b = max_u32(__float_as_uint(red[2]), __float_as_uint(red[3]));
    v = max_u32(a, b);
  }
  return v;
}

// The 8 norm weights of one chunk, kept over the row walk (ones where there is no weight).
template <int WT>
struct NormWeight {
  u32x4 w[WT == XGEN_DTYPE_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *base, int chunk) {
    constexpr int kParts = WT == XGEN_DTYPE_F32 ? 2 : 1;
    const uint32_t one = WT == XGEN_DTYPE_F32 ? 0x3f800000u : 0x3f803f80u;
#pragma unroll
    for (int i = 0; i < kParts; ++i)
      w[i] = base ? static_cast<const u32x4 *>(base)[kParts * chunk + i] : u32x4{one, one, one, one};
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (WT == XGEN_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i >> 2][i & 3]);
    } else {
      unpack8<XGEN_DTYPE_BF16>(w[0], v);
    }
  }
};

__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
  return u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}

// PAST: the call's reads and writes pass the last-level cache
template <int OUT, int WT, int WPR, int CH, bool PAST>
__global__ __launch_bounds__(kThreads) void residual_norm_kernel(ResNormArgs a) {
  static_assert(WPR == 1 || WPR == 4, "a wave or a workgroup per row");
  constexpr int kRowsPerBlock = 4 / WPR;
  __shared__ Slots slots[2];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int first = (wave % WPR) * 64 + lane;  // this lane's first chunk of a row
  const float inv_w = 1.0f / (float)a.width;
  const int chunks = a.width >> 3;
  // Every lane has its first CH - 1 chunks (a row's width is above what CH - 1 hold); the last may lie past the row's
  // end: then the row's last chunk is read in its place, and counts nowhere.
  const bool last = first + (CH - 1) * 64 * WPR < chunks;
  const int last_at = last ? first + (CH - 1) * 64 * WPR : chunks - 1;
  auto at = [&](int j) { return j < CH - 1 ? first + j * 64 * WPR : last_at; };
  auto live = [&](int j) { return j < CH - 1 || last; };

  // (rows past the end redo the last one, writing what its owner writes: the barriers stay in step)
  auto row_at = [&](int64_t base) {
    const int64_t want = base + wave / WPR;
    return (uint32_t)(want < a.rows ? want : a.rows - 1);
  };
  // a row's table index: a scalar load (constant address space), a row ahead of the table rows it selects
  auto index_of = [&](uint32_t row) -> int64_t {
    const uint32_t s = row - fast_div(row, a.seq) * a.seq.d;
    return a.indices ? ((const __attribute__((address_space(4))) int64_t *)a.indices)[s] : 0;
  };
  const int64_t step = (int64_t)gridDim.x * kRowsPerBlock;
  int64_t next_g = index_of(row_at((int64_t)blockIdx.x * kRowsPerBlock));

  NormWeight<WT> wb[CH], wn[CH];
#pragma unroll
  for (int j = 0; j < CH; ++j) {
    wb[j].load(a.branch_weight, at(j));
    wn[j].load(a.weight, at(j));
  }

  int parity = 0;
  for (int64_t base = (int64_t)blockIdx.x * kRowsPerBlock; base < a.rows; base += step) {
    const uint32_t row = row_at(base);
    const uint32_t b = fast_div(row, a.seq), s = row - b * a.seq.d;
    const u32x4 *xr = reinterpret_cast<const u32x4 *>(a.x + (int64_t)b * a.xsb + (int64_t)s * a.xss);
    const u32x4 *yr = reinterpret_cast<const u32x4 *>(a.y + (int64_t)b * a.ysb + (int64_t)s * a.yss);
    u32x4 xc[CH], yc[CH], gc[CH], sc[CH], tc[CH];
#pragma unroll
    for (int j = 0; j < CH; ++j) yc[j] = stream_load<PAST>(yr + at(j));
#pragma unroll
    for (int j = 0; j < CH; ++j) xc[j] = stream_load<PAST>(xr + at(j));
    // table rows: gate 1, scale 0, shift 0 without a table; an index outside the tables makes what they
    // reach NaN (nothing outside is read)
    const int64_t g = next_g;
    next_g = index_of(row_at(base + step));
    const bool g_ok = g >= 0 && g < a.table_rows;
    auto table = [&](const uint8_t *tab, int64_t stride, uint32_t none, u32x4 (&c)[CH]) {
      if (tab && g_ok) {  // uniform
        const u32x4 *r = reinterpret_cast<const u32x4 *>(tab + g * stride);
#pragma unroll
        for (int j = 0; j < CH; ++j) c[j] = r[at(j)];
      } else {
        const uint32_t fill = tab ? 0x7fc07fc0u : none;
#pragma unroll
        for (int j = 0; j < CH; ++j) c[j] = u32x4{fill, fill, fill, fill};
      }
    };
    table(a.gate, a.gate_stride, 0x3f803f80u, gc);
    table(a.scale, a.scale_stride, 0u, sc);
    table(a.shift, a.shift_stride, 0u, tc);
    Slots &red = slots[parity];
    parity ^= 1;

    // statistics of v: mean (layer norm) and 1 / sqrt(mean square + eps)
    auto statistics = [&](const float (&v)[CH][8], int kind, int slot, float &mean, float &rstd) {
      mean = 0.0f;
      float t[2] = {0.0f, 0.0f}, q[2] = {0.0f, 0.0f};
      if (kind == XGEN_NORM_LAYER) {
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          float u[2] = {t[0], t[1]};
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i & 1] += v[j][i];
#pragma unroll
          for (int i = 0; i < 2; ++i) t[i] = live(j) ? u[i] : t[i];
        }
        mean = row_sum<WPR>(t[0] + t[1], wave, lane, red.v[slot]) * inv_w;
      }
#pragma unroll
      for (int j = 0; j < CH; ++j) {
        float u[2] = {q[0], q[1]};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = v[j][i] - mean;
          u[i & 1] = __builtin_fmaf(d, d, u[i & 1]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) q[i] = live(j) ? u[i] : q[i];
      }
      rstd = __builtin_amdgcn_rsqf(row_sum<WPR>(q[0] + q[1], wave, lane, red.v[slot + 1]) * inv_w + a.eps);
    };

    float v[CH][8];
#pragma unroll
    for (int j = 0; j < CH; ++j) unpack8<XGEN_DTYPE_BF16>(yc[j], v[j]);
    float mean = 0.0f, rstd = 1.0f;
    if (a.branch_norm != XGEN_NORM_NONE) statistics(v, a.branch_norm, 0, mean, rstd);
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float xv[8], wv[8], gv[8];
      unpack8<XGEN_DTYPE_BF16>(xc[j], xv);
      wb[j].get(wv);
      unpack8<XGEN_DTYPE_BF16>(gc[j], gv);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        v[j][i] = __builtin_fmaf(a.residual_scale, xv[i], (v[j][i] - mean) * rstd * (wv[i] * gv[i]));
    }
    uint8_t *so = a.stream + (int64_t)row * a.width * 2;
#pragma unroll
    for (int j = 0; j < CH; ++j)
      if (live(j)) stream_store<PAST>(reinterpret_cast<u32x4 *>(so) + at(j), pack8(v[j]));
    statistics(v, a.norm, 2, mean, rstd);
    float am = 0.0f;
#pragma unroll
    for (int j = 0; j < CH; ++j) {
      float wv[8], sv[8], tv[8];
      wn[j].get(wv);
      unpack8<XGEN_DTYPE_BF16>(sc[j], sv);
      unpack8<XGEN_DTYPE_BF16>(tc[j], tv);
      float top = am;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[j][i] = __builtin_fmaf((v[j][i] - mean) * rstd * wv[i], 1.0f + sv[i], tv[i]);
        top = __builtin_elementwise_maximum(top, __builtin_fabsf(v[j][i]));  // NaN-propagating
      }
      am = live(j) ? top : am;
    }
    if constexpr (OUT == XGEN_DTYPE_BF16) {
      uint8_t *o = a.out + (int64_t)row * a.width * 2;
#pragma unroll
      for (int j = 0; j < CH; ++j)
        if (live(j)) stream_store<PAST>(reinterpret_cast<u32x4 *>(o) + at(j), pack8(v[j]));
    } else {
      const float amax = __uint_as_float(row_max<WPR>(__float_as_uint(am) & 0x7fffffffu, wave, lane, red.v[4]));
      RowQuant p;
      if constexpr (OUT == XGEN_DTYPE_E4M3) {
        const float sr = amax / kE4M3Max;
        p = fp8_scale_params(sr < kFltMin ? kFltMin : sr);
      } else {
        p = i8_row_params(amax);
      }
      uint8_t *o = a.out + (int64_t)row * a.width;
#pragma unroll
      for (int j = 0; j < CH; ++j)
        if (live(j)) stream_store<PAST>(reinterpret_cast<u32x2 *>(o) + at(j), quant8<OUT>(v[j], p));
      if (lane == 0 && wave % WPR == 0) a.token_scale[row] = p.s;
    }
  }
}

template <int OUT, int WT, int WPR, int CH, bool PAST>
void launch_walk(const ResNormArgs &a, hipStream_t stream) {
  constexpr int kRowsPerBlock = 4 / WPR;
  static const int per_cu = resident_blocks_per_cu(residual_norm_kernel<OUT, WT, WPR, CH, PAST>, kThreads);
  const int64_t need = (a.rows + kRowsPerBlock - 1) / kRowsPerBlock;
  const int64_t cap = (int64_t)device_cu_count() * per_cu;
  residual_norm_kernel<OUT, WT, WPR, CH, PAST>
      <<<dim3((unsigned)(need < cap ? need : cap)), dim3(kThreads), 0, stream>>>(a);
}

template <int OUT, int WT, int WPR, int CH>
void launch(const ResNormArgs &a, hipStream_t stream) {
  // x, y and the stream, and the rows
  if (a.rows * a.width * (OUT == XGEN_DTYPE_BF16 ? 8 : 7) > kLastLevelCacheBytes) launch_walk<OUT, WT, WPR, CH, true>(a, stream);
  else launch_walk<OUT, WT, WPR, CH, false>(a, stream);
}

template <int OUT, int WT>
void dispatch_width(const ResNormArgs &a, hipStream_t stream) {
  const int w = a.width;
  if (w <= 512) launch<OUT, WT, 1, 1>(a, stream);
  else if (w <= 1024) launch<OUT, WT, 1, 2>(a, stream);
  else if (w <= 2048) launch<OUT, WT, 4, 1>(a, stream);
  else if (w <= 4096) launch<OUT, WT, 4, 2>(a, stream);
  else if (w <= 6144) launch<OUT, WT, 4, 3>(a, stream);
  else launch<OUT, WT, 4, 4>(a, stream);
}

template <int OUT>
void dispatch_weight(const ResNormArgs &a, int weight_dtype, hipStream_t stream) {
  if (weight_dtype == XGEN_DTYPE_F32) dispatch_width<OUT, XGEN_DTYPE_F32>(a, stream);
  else dispatch_width<OUT, XGEN_DTYPE_BF16>(a, stream);
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" int xgen_residual_norm(const void *x, int64_t x_stride_batch, int64_t x_stride_seq, const void *branch,
                                  int64_t br_stride_batch, int64_t br_stride_seq, int64_t batch, int64_t seq,
                                  int64_t width, int branch_norm, const void *branch_weight, int norm_kind,
                                  const void *norm_weight, int norm_weight_dtype, float residual_scale, float eps,
                                  const void *gate_table, int64_t gate_row_stride, const void *scale_table,
                                  int64_t scale_row_stride, const void *shift_table, int64_t shift_row_stride,
                                  int64_t table_rows, const int64_t *indices, void *stream_out, int out_dtype,
                                  void *out, float *token_scale, hipStream_t stream) {
  const char *fn = "xgen_residual_norm";
  if (branch_norm != XGEN_NORM_NONE && branch_norm != XGEN_NORM_LAYER && branch_norm != XGEN_NORM_RMS)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown branch norm kind %d", fn, branch_norm);
  if (norm_kind != XGEN_NORM_LAYER && norm_kind != XGEN_NORM_RMS)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown norm kind %d", fn, norm_kind);
  if (out_dtype != XGEN_DTYPE_BF16 && !is_quant_dtype(out_dtype))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: output dtype must be BF16, E4M3 or I8", fn);
  if (norm_weight_dtype != XGEN_DTYPE_NONE && norm_weight_dtype != XGEN_DTYPE_BF16 &&
      norm_weight_dtype != XGEN_DTYPE_F32)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: norm weight dtype must be NONE, BF16 or F32", fn);
  if ((norm_weight_dtype == XGEN_DTYPE_NONE) != (!norm_weight && !branch_weight))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: norm weight pointers and dtype disagree", fn);
  if (branch_weight && branch_norm == XGEN_NORM_NONE)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: a branch weight needs a branch norm", fn);
  const bool tables = gate_table || scale_table || shift_table;
  if (batch < 0 || seq < 0 || width <= 0 || (tables && table_rows <= 0))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape batch=%lld seq=%lld width=%lld tables=%lld", fn,
                (long long)batch, (long long)seq, (long long)width, (long long)table_rows);
  // (v_rsq_f32 takes a subnormal for 0: a row of zeros would be 0 * inf)
  if (!(eps >= kFltMin && eps < 1.0f)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: eps must be in [2^-126, 1)", fn);
  if (!__builtin_isfinite(residual_scale))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: residual scale must be finite", fn);
  if (width > XGEN_NORM_MAX_WIDTH)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: width %lld exceeds %d", fn, (long long)width, XGEN_NORM_MAX_WIDTH);
  if (x_stride_seq < width || br_stride_seq < width || x_stride_batch < 0 || br_stride_batch < 0 ||
      (gate_table && gate_row_stride < width) || (scale_table && scale_row_stride < width) ||
      (shift_table && shift_row_stride < width))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: row strides must be >= width and batch strides >= 0", fn);
  if ((scale_table == nullptr) != (shift_table == nullptr))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: scale and shift tables come together", fn);
  if (batch != 0 && seq > 0x3fffffffLL / batch) return fail(XGEN_ERR_UNSUPPORTED, "%s: too many rows", fn);
  const int64_t rows = batch * seq;
  if (rows == 0) return ok();
  if (!x || !branch || !stream_out || !out || (tables && !indices) || (out_dtype != XGEN_DTYPE_BF16 && !token_scale))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (width % 8 || x_stride_seq % 8 || x_stride_batch % 8 || br_stride_seq % 8 || br_stride_batch % 8 ||
      (gate_table && gate_row_stride % 8) || (scale_table && (scale_row_stride % 8 || shift_row_stride % 8)) ||
      !aligned16(x) || !aligned16(branch) || !aligned16(gate_table) || !aligned16(scale_table) ||
      !aligned16(shift_table) || !aligned16(branch_weight) || !aligned16(norm_weight) || !aligned16(stream_out) ||
      !aligned16(out))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: width and strides must be multiples of 8 elements and buffers "
                "16-byte aligned", fn);

  ResNormArgs a;
  a.x = static_cast<const uint8_t *>(x);
  a.y = static_cast<const uint8_t *>(branch);
  a.xsb = x_stride_batch * 2;
  a.xss = x_stride_seq * 2;
  a.ysb = br_stride_batch * 2;
  a.yss = br_stride_seq * 2;
  a.seq = make_fastdiv((uint32_t)seq);
  a.rows = rows;
  a.width = (int)width;
  a.branch_norm = branch_norm;
  a.norm = norm_kind;
  a.branch_weight = branch_weight;
  a.weight = norm_weight;
  a.gate = static_cast<const uint8_t *>(gate_table);
  a.scale = static_cast<const uint8_t *>(scale_table);
  a.shift = static_cast<const uint8_t *>(shift_table);
  a.gate_stride = gate_row_stride * 2;
  a.scale_stride = scale_row_stride * 2;
  a.shift_stride = shift_row_stride * 2;
  a.table_rows = table_rows;
  a.indices = tables ? indices : nullptr;
  a.residual_scale = residual_scale;
  a.eps = eps;
  a.stream = static_cast<uint8_t *>(stream_out);
  a.out = static_cast<uint8_t *>(out);
  a.token_scale = token_scale;
  if (out_dtype == XGEN_DTYPE_BF16) dispatch_weight<XGEN_DTYPE_BF16>(a, norm_weight_dtype, stream);
  else if (out_dtype == XGEN_DTYPE_E4M3) dispatch_weight<XGEN_DTYPE_E4M3>(a, norm_weight_dtype, stream);
  else dispatch_weight<XGEN_DTYPE_I8>(a, norm_weight_dtype, stream);
  return launch_status(fn);
}
