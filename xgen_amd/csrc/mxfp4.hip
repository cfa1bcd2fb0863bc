// MXFP4 rows (gfx950): e2m1 codes, two per byte, with one power-of-two scale (e8m0) per 32 consecutive values.
//
//   E = floor(log2 max|x|) - 2, or the least E with max|x| <= 6 * 2^E;  E >= -127
//   code = e2m1(x / 2^E), to nearest with ties to the even code, saturated at 6;  value = code * 2^E
//
// A division by a power of two rounds nothing (fp32 holds x / 2^E of every bf16 and f16 x that does not vanish
// below 2^-126 by a wide margin), so the code's rounding is the only one, and a row has the same bytes in every
// implementation.  A block with an inf or NaN takes the scale byte 255 (NaN) and codes 0.
//
// Scale bytes lie as the matrix product's lanes read them (gemm_w8a8.h): [256 values][row][8], block i of a
// row's 256 values at (i mod 2) * 4 + i / 2, so that 16 rows share a line and a lane's four blocks a dword.
//
// Memory bounds both directions: 15,624 x 5,376 of bf16 takes 40 us either way, 5.3 TB/s, as a copy of as many bytes (to float32
// 83 us, 4.6 TB/s); 2 x 2,048
// 2.4 us, a launch and one load's way.  A wave takes 4 rows of 512 values, so that four loads are in flight in each
// lane, and a workgroup 16 rows, whose scale bytes are whole lines.
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kCols = 512;                    // values of a row that a wave takes at once: 8 per lane
constexpr int kRows = 4;                      // rows a wave takes: that many loads in flight per lane
constexpr int kTileRows = kWaves * kRows;     // a workgroup's rows: their scale bytes fill whole lines
// rows of a launch: a grid's threads are counted in 32 bits
constexpr int64_t kLaunchRows = (int64_t)kTileRows * ((1ll << 32) / kThreads / 2);

struct RowsArgs {
  const uint8_t *x;       // values, or codes (dequantize)
  int64_t ldx;            // bytes
  int64_t rows;
  int K, blocks256;       // values of a row, and their blocks of 256
  uint8_t *out;           // codes, or values (dequantize)
  int64_t ldo;            // bytes
  uint8_t *scales;        // written, or read (dequantize)
  int64_t block_stride;
  int ceil_scale;
};

// Byte of block `block` of a row: its offset in the scales of its row's 256 values.
__device__ __forceinline__ int scale_at(int block) { return (block & 1) * 4 + ((block >> 1) & 3); }

// The scale byte of a block whose largest |x| has the fp32 bits `most` (NaN above inf).
__device__ __forceinline__ uint32_t scale_byte(uint32_t most, bool ceil_scale) {
  const uint32_t e = most >> 23;
  if (e == 255) return 255;
  const int up = ceil_scale && (most & 0x7fffffu) > 0x400000u;  // above 1.5 * 2^(e - 127) = 6 * 2^(e - 2 - 127)
  const int b = (int)e - 2 + up;
  return (uint32_t)(b > 0 ? b : 0);
}

// Eight values of one 16-byte chunk as codes, divided by 2^(byte - 127).
template <int DT>
__device__ __forceinline__ uint32_t codes8(const u32x4 &c, uint32_t byte) {
  float v[8];
  unpack8<DT>(c, v);
  uint32_t r = 0;
  const int e = 127 - (int)byte;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __builtin_ldexpf(v[i], e);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[0], v[1], 1.0f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], 1.0f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], 1.0f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], 1.0f, 3);
  return byte == 255 ? 0u : r;
}

template <int DT>
__global__ __launch_bounds__(kThreads) void quantize_kernel(RowsArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * kTileRows + wave * kRows;
  const int col = blockIdx.y * kCols + lane * 8;
  const bool in = col < p.K, mine = (lane & 3) == 0 && (col >> 8) < p.blocks256;
  u32x4 c[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    c[r] = u32x4{0, 0, 0, 0};
    if (in && row0 + r < p.rows) c[r] = *reinterpret_cast<const u32x4 *>(p.x + (row0 + r) * p.ldx + (int64_t)col * 2);
  }
  uint8_t *sc = p.scales + (int64_t)(col >> 8) * p.block_stride + scale_at(col >> 5);
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + r;
    // the block's four lanes: the largest |x|, as the 16-bit pattern (ordered like |x|, NaN above inf)
    uint32_t m = hmax_u16x2(absmax_chunk<DT>(c[r], u16x2{0, 0}));
    m = max_u32(m, dpp_u32<kDppQuad1032>(0, m));
    m = max_u32(m, dpp_u32<kDppQuad2301>(0, m));
    const uint32_t byte = scale_byte(__float_as_uint(Half2<DT>::from_absbits(m)), p.ceil_scale);
    if (in && row < p.rows) *reinterpret_cast<uint32_t *>(p.out + row * p.ldo + (col >> 1)) = codes8<DT>(c[r], byte);
    // (the row that makes their number even, and the blocks past K: zeros)
    if (mine && row < p.rows + (p.rows & 1)) sc[row * 8] = (uint8_t)byte;
  }
}

template <int OUT>
__global__ __launch_bounds__(kThreads) void dequantize_kernel(RowsArgs p) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row0 = (int64_t)blockIdx.x * kTileRows + wave * kRows;
  const int col = blockIdx.y * kCols + lane * 8;
  if (col >= p.K) return;
  const uint8_t *sc = p.scales + (int64_t)(col >> 8) * p.block_stride + scale_at(col >> 5);
  uint32_t c[kRows], b[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + r;
    c[r] = b[r] = 0;
    if (row < p.rows) {
      c[r] = *reinterpret_cast<const uint32_t *>(p.x + row * p.ldx + (col >> 1));
      b[r] = sc[row * 8];
    }
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int64_t row = row0 + r;
    if (row >= p.rows) return;
    float v[8];
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[r], 1.0f, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[r], 1.0f, 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[r], 1.0f, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[r], 1.0f, 3);
    v[0] = p0.x, v[1] = p0.y, v[2] = p1.x, v[3] = p1.y, v[4] = p2.x, v[5] = p2.y, v[6] = p3.x, v[7] = p3.y;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = b[r] == 255 ? __builtin_nanf("") : __builtin_ldexpf(v[i], (int)b[r] - 127);
    uint8_t *o = p.out + row * p.ldo;
    if constexpr (OUT == XGEN_DTYPE_F32) {
      f32x4 *q = reinterpret_cast<f32x4 *>(o + (int64_t)col * 4);
      q[0] = f32x4{v[0], v[1], v[2], v[3]};
      q[1] = f32x4{v[4], v[5], v[6], v[7]};
    } else if constexpr (OUT == XGEN_DTYPE_BF16) {
      *reinterpret_cast<u32x4 *>(o + (int64_t)col * 2) =
          u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    } else {
      *reinterpret_cast<u32x4 *>(o + (int64_t)col * 2) =
          u32x4{pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7])};
    }
  }
}

// What both directions check: `dense` the 16-bit or 32-bit rows (elements of `size` bytes), `codes` the packed ones.
int check_rows(const char *fn, int64_t rows, int64_t K, const void *dense, int64_t ld_dense, int size, const void *codes,
               int64_t ld_codes, const void *scales, int64_t block_stride) {
  if (rows < 0 || K <= 0) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape rows=%lld K=%lld", fn, (long long)rows, (long long)K);
  if (K % 32) return fail(XGEN_ERR_UNSUPPORTED, "%s: K must be a multiple of 32", fn);
  if (ld_dense < K || ld_codes < K / 2) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: leading dimensions must cover the rows", fn);
  if (K > (int64_t)kCols * 65535 || rows >= (1ll << 31) * kTileRows - kTileRows)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: too many rows or values", fn);
  if (block_stride < (rows + (rows & 1)) * 8) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: the scales' blocks must cover the rows", fn);
  if (rows == 0) return XGEN_OK;
  if (!dense || !codes || !scales) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (!aligned16(dense) || ld_dense * size % 16 || !aligned16(codes) || ld_codes % 16)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: rows must be 16-byte aligned", fn);
  if (!aligned16(scales) || block_stride % 16) return fail(XGEN_ERR_UNSUPPORTED, "%s: the scales' blocks must be 16-byte aligned", fn);
  return XGEN_OK;
}

// launch(args, grid) for the rows of each launch (whole workgroups, so that the scales' last row stays the last launch's)
template <class Launch>
void each_launch(const RowsArgs &p, Launch launch) {
  for (int64_t first = 0; first < p.rows; first += kLaunchRows) {
    RowsArgs q = p;
    q.x += first * p.ldx;
    q.out += first * p.ldo;
    q.scales += first * 8;
    q.rows = p.rows - first < kLaunchRows ? p.rows - first : kLaunchRows;
    launch(q, dim3((unsigned)((q.rows + kTileRows - 1) / kTileRows), (unsigned)(((int64_t)p.K + kCols - 1) / kCols)));
  }
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" int xgen_mxfp4_quantize(int in_dtype, const void *x, int64_t rows, int64_t K, int64_t ldx, int rounding,
                                   void *codes, int64_t ld_codes, void *scales, int64_t block_stride, hipStream_t stream) {
  const char *fn = "xgen_mxfp4_quantize";
  if (!is_input_dtype(in_dtype)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: input dtype must be BF16 or F16", fn);
  if (rounding != XGEN_MX_FLOOR && rounding != XGEN_MX_CEIL)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown scale rounding %d", fn, rounding);
  const int st = check_rows(fn, rows, K, x, ldx, 2, codes, ld_codes, scales, block_stride);
  if (st != XGEN_OK) return st;
  if (rows == 0) return ok();
  const RowsArgs p = {static_cast<const uint8_t *>(x), ldx * 2, rows, (int)K, (int)((K + 255) / 256),
                      static_cast<uint8_t *>(codes), ld_codes, static_cast<uint8_t *>(scales), block_stride,
                      rounding == XGEN_MX_CEIL};
  each_launch(p, [&](const RowsArgs &q, dim3 grid) {
    if (in_dtype == XGEN_DTYPE_BF16) quantize_kernel<XGEN_DTYPE_BF16><<<grid, kThreads, 0, stream>>>(q);
    else quantize_kernel<XGEN_DTYPE_F16><<<grid, kThreads, 0, stream>>>(q);
  });
  return launch_status(fn);
}

extern "C" int xgen_mxfp4_dequantize(const void *codes, int64_t ld_codes, const void *scales, int64_t block_stride,
                                     int64_t rows, int64_t K, int out_dtype, void *out, int64_t ldo, hipStream_t stream) {
  const char *fn = "xgen_mxfp4_dequantize";
  if (!is_input_dtype(out_dtype) && out_dtype != XGEN_DTYPE_F32)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: output dtype must be BF16, F16 or F32", fn);
  const int size = out_dtype == XGEN_DTYPE_F32 ? 4 : 2;
  const int st = check_rows(fn, rows, K, out, ldo, size, codes, ld_codes, scales, block_stride);
  if (st != XGEN_OK) return st;
  if (rows == 0) return ok();
  const RowsArgs p = {static_cast<const uint8_t *>(codes), ld_codes, rows, (int)K, (int)((K + 255) / 256),
                      static_cast<uint8_t *>(out), ldo * size, static_cast<uint8_t *>(const_cast<void *>(scales)),
                      block_stride, 0};
  each_launch(p, [&](const RowsArgs &q, dim3 grid) {
    if (out_dtype == XGEN_DTYPE_BF16) dequantize_kernel<XGEN_DTYPE_BF16><<<grid, kThreads, 0, stream>>>(q);
    else if (out_dtype == XGEN_DTYPE_F16) dequantize_kernel<XGEN_DTYPE_F16><<<grid, kThreads, 0, stream>>>(q);
    else dequantize_kernel<XGEN_DTYPE_F32><<<grid, kThreads, 0, stream>>>(q);
  });
  return launch_status(fn);
}
