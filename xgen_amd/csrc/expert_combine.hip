// Sum of each token's expert rows, weighted, with the gated residual behind it (gfx950):
//
//   out[t] = dtype(residual[t] + gate[indices[t % seq]] * sum_j weights[t, j] * y[slots[t, j]])
//
// summed in fp32 in the order of j and rounded once: the result does not depend on how rows were
// dealt to experts.  A slot of -1 (a choice that no expert here takes) adds nothing, and its row is not
// read: a token without experts is residual[t], or zeros.
//
// Memory bound: k gathered rows in, one row out.  A wave takes 64 16-byte pieces of a token's row and loads
// the pieces of up to four experts at once; the token's slots and weights are wave-uniform (scalar loads).
// 15,624 tokens x 2 experts x 5,376 with the gated residual: 125 us, 5.4 TB/s (through the caches 133); 8,000 x 8 x
// 2,048: 51 us, 5.8 TB/s (62).  8 tokens x 6: 3.7 us.
#include "fastdiv.h"
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kThreads = 256;

struct CombineArgs {
  const uint8_t *y;
  int64_t ldy;  // bytes
  int64_t y_rows;
  const float *weights;
  const int32_t *slots;
  int64_t tokens;
  int k;
  int chunks;       // 16-byte chunks per row
  FastDiv blocks;   // waves per token: 64 chunks each
  int64_t items;    // tokens * blocks
  const uint8_t *residual;
  int64_t ld_residual;  // bytes
  const uint8_t *gate;
  int64_t gate_stride;  // bytes
  int64_t gate_rows;
  const int64_t *indices;
  FastDiv seq;
  uint8_t *out;
};

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == XGEN_DTYPE_BF16) return pack_bf16x2(a, b);
  else return pack_f16x2(a, b);
}

// PAST: the call's reads and writes pass the last-level cache
template <int DT, bool PAST>
__global__ __launch_bounds__(kThreads) void expert_combine_kernel(CombineArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t step = (int64_t)gridDim.x * (kThreads / 64);
  constexpr uint32_t kNaN2 = DT == XGEN_DTYPE_BF16 ? 0x7fc07fc0u : 0x7e007e00u;
  for (int64_t item = (int64_t)blockIdx.x * (kThreads / 64) + wave; item < a.items; item += step) {
    const uint32_t t = fast_div((uint32_t)item, a.blocks);
    const int c = (int)((uint32_t)item - t * a.blocks.d) * 64 + lane;
    if (c >= a.chunks) continue;
    const int32_t *slots = a.slots + (int64_t)t * a.k;
    const float *weights = a.weights + (int64_t)t * a.k;
    float acc[8] = {};
    bool bad = false;
    for (int j0 = 0; j0 < a.k; j0 += 4) {
      u32x4 v[4];
      float w[4];
      bool on[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int j = j0 + u < a.k ? j0 + u : a.k - 1;
        const int32_t slot = slots[j];
        w[u] = weights[j];
        on[u] = j0 + u < a.k && slot >= 0 && slot < a.y_rows;
        bad |= slot >= a.y_rows;
        v[u] = u32x4{0, 0, 0, 0};
        if (on[u]) v[u] = stream_load<PAST>(reinterpret_cast<const u32x4 *>(a.y + (int64_t)slot * a.ldy + (int64_t)c * 16));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (on[u]) {
          float y[8];
          unpack8<DT>(v[u], y);
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(w[u], y[i], acc[i]);
        }
      }
    }
    if (a.residual) {
      float r[8];
      unpack8<DT>(stream_load<PAST>(reinterpret_cast<const u32x4 *>(a.residual + (int64_t)t * a.ld_residual + (int64_t)c * 16)), r);
      if (a.gate) {
        const int64_t g = a.indices[t - fast_div(t, a.seq) * a.seq.d];
        const bool g_ok = g >= 0 && g < a.gate_rows;
        bad |= !g_ok;
        float gv[8];
        unpack8<DT>(*reinterpret_cast<const u32x4 *>(a.gate + (g_ok ? g : 0) * a.gate_stride + (int64_t)c * 16), gv);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = __builtin_fmaf(gv[i], acc[i], r[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += r[i];
      }
    }
    u32x4 o = {pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3]), pack2<DT>(acc[4], acc[5]), pack2<DT>(acc[6], acc[7])};
    if (bad) o = u32x4{kNaN2, kNaN2, kNaN2, kNaN2};
    stream_store<PAST>(reinterpret_cast<u32x4 *>(a.out + ((int64_t)t * a.chunks + c) * 16), o);
  }
}

template <int DT, bool PAST>
void launch(const CombineArgs &a, hipStream_t stream) {
  static const int per_cu = resident_blocks_per_cu(expert_combine_kernel<DT, PAST>, kThreads);
  const int64_t need = (a.items + kThreads / 64 - 1) / (kThreads / 64);
  const int64_t cap = (int64_t)device_cu_count() * per_cu;
  expert_combine_kernel<DT, PAST><<<dim3((unsigned)(need < cap ? need : cap)), dim3(kThreads), 0, stream>>>(a);
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" int xgen_expert_combine(int dtype, const void *y, int64_t ldy, int64_t y_rows, const float *weights,
                                   const int32_t *slots, int64_t tokens, int64_t k, int64_t width,
                                   const void *residual, int64_t ld_residual, const void *gate_table,
                                   int64_t gate_row_stride, int64_t gate_rows, const int64_t *indices, int64_t seq,
                                   void *out, hipStream_t stream) {
  const char *fn = "xgen_expert_combine";
  if (!is_input_dtype(dtype)) return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: dtype must be BF16 or F16", fn);
  if (tokens < 0 || k <= 0 || width <= 0 || y_rows < 0)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape tokens=%lld k=%lld width=%lld rows=%lld", fn,
                (long long)tokens, (long long)k, (long long)width, (long long)y_rows);
  if (ldy < width || (residual && ld_residual < width) || (gate_table && gate_row_stride < width))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: row strides must be >= width", fn);
  if (gate_table && (!residual || gate_rows <= 0 || seq <= 0 || tokens % seq))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: a gate needs a residual, table rows and tokens a multiple of seq", fn);
  if (tokens == 0) return ok();
  if ((y_rows && !y) || !weights || !slots || !out || (gate_table && !indices))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (width % 8 || ldy % 8 || (residual && ld_residual % 8) || (gate_table && gate_row_stride % 8) || !aligned16(y) ||
      !aligned16(residual) || !aligned16(gate_table) || !aligned16(out))
    return fail(XGEN_ERR_UNSUPPORTED, "%s: width and strides must be multiples of 8 elements and buffers "
                "16-byte aligned", fn);
  const int64_t blocks = (width / 8 + 63) / 64;
  // (the kernel steps through the choices by four in 32 bits)
  if (width > 0x3fffffffLL || k > 0x3fffffffLL || y_rows > 0x7fffffffLL || tokens > 0x7fffffffLL / blocks)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: too many rows or choices", fn);
  CombineArgs a;
  a.y = static_cast<const uint8_t *>(y);
  a.ldy = ldy * 2;
  a.y_rows = y_rows;
  a.weights = weights;
  a.slots = slots;
  a.tokens = tokens;
  a.k = (int)k;
  a.chunks = (int)(width / 8);
  a.blocks = make_fastdiv((uint32_t)blocks);
  a.items = tokens * blocks;
  a.residual = static_cast<const uint8_t *>(residual);
  a.ld_residual = ld_residual * 2;
  a.gate = static_cast<const uint8_t *>(gate_table);
  a.gate_stride = gate_row_stride * 2;
  a.gate_rows = gate_rows;
  a.indices = indices;
  a.seq = make_fastdiv((uint32_t)(gate_table ? seq : 1));
  a.out = static_cast<uint8_t *>(out);
  const bool past = (double)tokens * width * 2 * (k + 1 + (residual ? 1 : 0)) > (double)kLastLevelCacheBytes;
  if (dtype == XGEN_DTYPE_BF16) {
    if (past) launch<XGEN_DTYPE_BF16, true>(a, stream);
    else launch<XGEN_DTYPE_BF16, false>(a, stream);
  } else {
    if (past) launch<XGEN_DTYPE_F16, true>(a, stream);
    else launch<XGEN_DTYPE_F16, false>(a, stream);
  }
  return launch_status(fn);
}
