// Expert router (gfx950): the k experts of each token, their weights, and the plan that groups the
// (token, choice) pairs by expert for the grouped products and the sum behind them.
//
//   score[e]   = float(logit[e]) + bias[e]; the k largest scores, ties to the lowest expert; a score of
//                -inf or NaN is never taken (a token masked in every expert takes none)
//   weight     = exp(logit[e]) / sum exp(logit) over all experts, or 1 / (1 + exp(-logit[e])); then, if
//                renormalised, divided by the sum over the taken experts
//   plan       pairs of the experts [first, first + local) in the order (expert, token, choice):
//                ends[e]    pairs of experts up to and including first + e
//                rows[i]    token of pair i (-1 behind the last pair)
//                slots[t,j] place of pair (t, j), or -1
//
// A chunk of tokens (64, more from 32,768 tokens on) is a workgroup's.  One chunk takes a single launch
// that chooses, counts and places; more take two: every chunk's choices and its count per expert, then, from
// all counts, every chunk's places.  Places are ranks (ballots within a wave, per-wave counts in LDS), never the order that an
// atomic happened to take: the plan is the same on every run.
//
// A token is a group of G lanes with V logits each; a choice is a maximum over the group and a
// ballot for the lowest expert that has it.
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChunk = 64;        // tokens that a workgroup takes at once
constexpr int kMaxChunks = 512;   // every workgroup reads all chunks' counts: a chunk is several kChunk beyond
constexpr int kMaxPairs = kChunk * XGEN_ROUTE_MAX_CHOICES;

struct RouteArgs {
  const void *logits;
  int dtype;
  int64_t ld;  // elements
  int64_t tokens;
  int experts, k;
  const float *bias;
  int sigmoid, renormalize;
  int first, local;
  float *weights;
  int32_t *chosen, *ends, *rows, *slots;
  int32_t *counts;  // [chunks][local]
  int chunks;
  int64_t chunk_tokens;  // a multiple of kChunk
};

__device__ __forceinline__ float load_logit(const RouteArgs &a, int64_t t, int e) {
  const int64_t i = t * a.ld + e;
  if (a.dtype == XGEN_DTYPE_F32) return static_cast<const float *>(a.logits)[i];
  const uint32_t w = static_cast<const uint16_t *>(a.logits)[i];
  return a.dtype == XGEN_DTYPE_BF16 ? Half2<XGEN_DTYPE_BF16>::lo(w) : Half2<XGEN_DTYPE_F16>::lo(w);
}

// Reductions over groups of G lanes (every lane active), the result in every lane: quad
// permutes and mirrors within 16 lanes, row swaps beyond.
template <int G, class F>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, F f) {
  v = f(v, dpp_u32<kDppQuad1032>(0, v));
  v = f(v, dpp_u32<kDppQuad2301>(0, v));
  v = f(v, dpp_u32<kDppRowHalfMirror>(0, v));
  if constexpr (G >= 16) v = f(v, dpp_u32<kDppRowMirror>(0, v));
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r[0], r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = f(r[0], r[1]);
  }
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  return group_reduce<G>(v, [](uint32_t a, uint32_t b) { return max_u32(a, b); });
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return __uint_as_float(group_reduce<G>(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}

// A float's bits as an unsigned integer of the same order; above 0 for every value above -inf.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// The choices of tokens [t0, t0 + kChunk), counted per expert into hist[local]; ids also into `ids`
// ([token in chunk][k]) if given.
template <int G, int V>
__device__ __forceinline__ void choose(const RouteArgs &a, int64_t t0, int32_t *hist, int32_t *ids) {
  const int gl = threadIdx.x % G, lane = threadIdx.x & 63;
  constexpr int kGroups = kThreads / G;
  const float ninf = -__builtin_inff();
  const int n = (int)(a.tokens - t0 < kChunk ? a.tokens - t0 : kChunk);
  float bias[V];
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = a.bias && v * G + gl < a.experts ? a.bias[v * G + gl] : 0.0f;
  for (int i0 = 0; i0 < n; i0 += kGroups) {  // (every lane stays active: tokens past the end redo the last one)
    const int i = i0 + (int)threadIdx.x / G;
    const int64_t t = t0 + (i < n ? i : n - 1);
    float x[V];
    uint32_t key[V];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = v * G + gl < a.experts ? load_logit(a, t, v * G + gl) : ninf;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float s = a.bias ? x[v] + bias[v] : x[v];
      if (s == 0.0f) s = 0.0f;  // -0 ranks with 0
      key[v] = v * G + gl < a.experts && s > ninf ? order_key(s) : 0u;
      nan |= !(x[v] == x[v]);
    }
    int mine = -1;  // lane j of the group: the group's choice j
    for (int j = 0; j < a.k; ++j) {
      uint32_t m = key[0];
#pragma unroll
      for (int v = 1; v < V; ++v) m = max_u32(m, key[v]);
      m = group_max<G>(m);
      int e = -1;
#pragma unroll
      for (int v = V - 1; v >= 0; --v) {
        uint64_t at = __ballot(key[v] == m) >> (lane & ~(G - 1));
        if constexpr (G < 64) at &= (1ull << G) - 1;
        if (at) e = v * G + __builtin_ctzll(at);
      }
      if (m == 0) e = -1;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (e == v * G + gl) key[v] = 0;
      if (gl == j) mine = e;
    }
    // weights: the chosen experts' logits again (cached), one per lane
    const bool taken = gl < a.k && mine >= 0;
    const float xe = taken ? load_logit(a, t, mine) : ninf;
    float p, total = 1.0f;
    if (a.sigmoid) {
      p = taken ? 1.0f / (1.0f + expf(-xe)) : 0.0f;
      if (a.renormalize) total = group_sum<G>(p);
    } else {
      // the peak over what is summed: the sum is 1 at least
      float peak = xe;
      if (!a.renormalize) {
#pragma unroll
        for (int v = 0; v < V; ++v) peak = __builtin_fmaxf(peak, x[v]);
      }
      peak = from_order_key(group_max<G>(order_key(peak)));
      p = taken ? expf(xe - peak) : 0.0f;
      if (a.renormalize) {
        total = group_sum<G>(p);
      } else {
        float part = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) part += x[v] > ninf ? expf(x[v] - peak) : 0.0f;
        total = group_sum<G>(part);
      }
    }
    // a NaN logit makes its token's weights NaN
    nan = (__ballot(nan) >> (lane & ~(G - 1)) & (G < 64 ? (1ull << (G & 63)) - 1 : ~0ull)) != 0;
    float w = taken ? (total > 0.0f ? p / total : total) : 0.0f;
    if (nan && taken) w = __builtin_nanf("");
    if (gl < a.k && i < n) {
      a.chosen[t * a.k + gl] = mine;
      a.weights[t * a.k + gl] = w;
      if (ids) ids[i * a.k + gl] = mine;
      const int le = mine - a.first;
      if (mine >= 0 && le >= 0 && le < a.local) atomicAdd(&hist[le], 1);
    }
  }
}

// LDS of the placement.
struct PlaceShared {
  int32_t count[kWaves][XGEN_ROUTE_MAX_EXPERTS];  // pairs of the wave's segment per expert; then its first place
  int32_t base[XGEN_ROUTE_MAX_EXPERTS];           // the chunk's first place per expert
  int32_t total[XGEN_ROUTE_MAX_EXPERTS];
  int32_t ids[kMaxPairs];
  int32_t routed;                                 // pairs of all experts here
};

// Lanes of this wave with the same group (0 <= group <= 512; every lane active).
__device__ __forceinline__ uint64_t same_group(int group, int bits) {
  uint64_t mask = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const bool set = (group >> b) & 1;
    const uint64_t on = __ballot(set);
    mask &= set ? on : ~on;
  }
  return mask;
}

// From every expert's pairs (sh.total) and those of the chunks before this one (sh.base): the group ends, and
// the chunk's first place per expert into sh.base.
__device__ __forceinline__ void first_places(const RouteArgs &a, bool write_ends, PlaceShared &sh) {
  const int lane = threadIdx.x & 63;
  __syncthreads();
  if (threadIdx.x < 64) {
    constexpr int kPer = XGEN_ROUTE_MAX_EXPERTS / 64;
    int32_t t[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane * kPer + i;
      t[i] = e < a.local ? sh.total[e] : 0;
      sum += t[i];
    }
    int32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int32_t up = __shfl_up(incl, d);
      if (lane >= d) incl += up;
    }
    int32_t at = incl - sum;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane * kPer + i;
      if (e < a.local) {
        sh.base[e] += at;
        if (write_ends) a.ends[e] = at + t[i];
      }
      at += t[i];
    }
    if (lane == 63) sh.routed = incl;
  }
}

// The places of tokens [t0, t0 + kChunk), whose choices are in sh.ids; sh.base moves on past them.
__device__ __forceinline__ void place(const RouteArgs &a, int64_t t0, PlaceShared &sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int n = (int)(a.tokens - t0 < kChunk ? a.tokens - t0 : kChunk) * a.k;
  for (int i = tid; i < kWaves * XGEN_ROUTE_MAX_EXPERTS; i += kThreads) (&sh.count[0][0])[i] = 0;
  __syncthreads();
  // each wave a contiguous segment of the pairs, 64 at a time
  const int seg = ((n + kWaves - 1) / kWaves + 63) / 64 * 64, begin = wave * seg;
  const int bits = 32 - __builtin_clz(a.local);  // groups 0 .. local (local: no expert here)
  auto group_of = [&](int i) {
    const int id = i < n ? sh.ids[i] : -1, g = id - a.first;
    return id >= 0 && g >= 0 && g < a.local ? g : a.local;
  };
  for (int i0 = begin; i0 < begin + seg && i0 < n; i0 += 64) {
    const int g = group_of(i0 + lane);
    const uint64_t same = same_group(g, bits);
    if (g < a.local && lane == __builtin_ctzll(same)) atomicAdd(&sh.count[wave][g], __builtin_popcountll(same));
  }
  __syncthreads();
  for (int e = tid; e < a.local; e += kThreads) {
    int32_t at = sh.base[e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int32_t c = sh.count[w][e];
      sh.count[w][e] = at;
      at += c;
    }
    sh.base[e] = at;
  }
  __syncthreads();
  for (int i0 = begin; i0 < begin + seg && i0 < n; i0 += 64) {
    const int i = i0 + lane, g = group_of(i);
    const uint64_t same = same_group(g, bits);
    const int leader = __builtin_ctzll(same);
    int32_t at = 0;
    if (g < a.local && lane == leader) at = atomicAdd(&sh.count[wave][g], __builtin_popcountll(same));
    at = __shfl(at, leader) + (int32_t)__builtin_popcountll(same & ((1ull << lane) - 1));
    if (i < n) {
      const bool routed = g < a.local;
      a.slots[t0 * a.k + i] = routed ? at : -1;
      if (routed) a.rows[at] = (int32_t)(t0 + i / a.k);
    }
  }
  // rows behind the last pair: each chunk the part at its own pairs' positions
  for (int64_t i = t0 * a.k + tid; i < t0 * a.k + n; i += kThreads)
    if (i >= sh.routed) a.rows[i] = -1;
}

template <int G, int V>
__global__ __launch_bounds__(kThreads) void route_one_kernel(RouteArgs a) {
  __shared__ PlaceShared sh;
  for (int e = threadIdx.x; e < a.local; e += kThreads) sh.total[e] = sh.base[e] = 0;
  __syncthreads();
  choose<G, V>(a, 0, sh.total, sh.ids);
  first_places(a, true, sh);
  __syncthreads();
  place(a, 0, sh);
}

template <int G, int V>
__global__ __launch_bounds__(kThreads) void route_choose_kernel(RouteArgs a) {
  __shared__ int32_t hist[XGEN_ROUTE_MAX_EXPERTS];
  for (int e = threadIdx.x; e < a.local; e += kThreads) hist[e] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * a.chunk_tokens;
  const int64_t end = begin + a.chunk_tokens < a.tokens ? begin + a.chunk_tokens : a.tokens;
  for (int64_t t0 = begin; t0 < end; t0 += kChunk) choose<G, V>(a, t0, hist, nullptr);
  __syncthreads();
  for (int e = threadIdx.x; e < a.local; e += kThreads) a.counts[(int64_t)blockIdx.x * a.local + e] = hist[e];
}

__global__ __launch_bounds__(kThreads) void route_place_kernel(RouteArgs a) {
  __shared__ PlaceShared sh;
  const int tid = threadIdx.x;
  for (int e = tid; e < a.local; e += kThreads) sh.total[e] = sh.base[e] = 0;
  __syncthreads();
  // counts of all chunks and of those before this one: the threads share out the chunks
  int span = 1;
  while (span < a.local) span <<= 1;
  const int e = tid & (span - 1), part = tid / span, parts = kThreads / span;
  if (e < a.local) {
    int32_t all = 0, before = 0;
    for (int c = part; c < a.chunks; c += parts) {
      const int32_t v = a.counts[(int64_t)c * a.local + e];
      all += v;
      before += c < (int)blockIdx.x ? v : 0;
    }
    if (all) atomicAdd(&sh.total[e], all);
    if (before) atomicAdd(&sh.base[e], before);
  }
  first_places(a, blockIdx.x == 0, sh);
  const int64_t begin = (int64_t)blockIdx.x * a.chunk_tokens;
  const int64_t end = begin + a.chunk_tokens < a.tokens ? begin + a.chunk_tokens : a.tokens;
  for (int64_t t0 = begin; t0 < end; t0 += kChunk) {
    const int n = (int)(end - t0 < kChunk ? end - t0 : kChunk) * a.k;
    __syncthreads();  // the places before are done with sh.ids
    for (int i = tid; i < n; i += kThreads) sh.ids[i] = a.chosen[t0 * a.k + i];
    __syncthreads();
    place(a, t0, sh);
  }
}

template <int G, int V>
void launch(const RouteArgs &a, hipStream_t stream) {
  if (a.chunks == 1) {
    route_one_kernel<G, V><<<dim3(1), dim3(kThreads), 0, stream>>>(a);
    return;
  }
  route_choose_kernel<G, V><<<dim3((unsigned)a.chunks), dim3(kThreads), 0, stream>>>(a);
  route_place_kernel<<<dim3((unsigned)a.chunks), dim3(kThreads), 0, stream>>>(a);
}

int64_t chunk_tokens_of(int64_t tokens) {
  const int64_t pieces = (tokens + kChunk - 1) / kChunk;
  return (pieces + kMaxChunks - 1) / kMaxChunks * kChunk;
}
int64_t chunks_of(int64_t tokens) { return (tokens + chunk_tokens_of(tokens) - 1) / chunk_tokens_of(tokens); }

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" size_t xgen_route_workspace_bytes(int64_t tokens, int64_t local_experts) {
  if (tokens <= kChunk || local_experts <= 0) return 0;
  return (size_t)chunks_of(tokens) * (size_t)local_experts * 4;
}

extern "C" int xgen_route(int in_dtype, const void *logits, int64_t ld, int64_t tokens, int64_t experts, int64_t k,
                          const float *bias, int scoring, int renormalize, int64_t first_expert,
                          int64_t local_experts, float *weights, int32_t *chosen, int32_t *ends, int32_t *rows,
                          int32_t *slots, void *workspace, size_t workspace_bytes, hipStream_t stream) {
  const char *fn = "xgen_route";
  if (in_dtype != XGEN_DTYPE_BF16 && in_dtype != XGEN_DTYPE_F16 && in_dtype != XGEN_DTYPE_F32)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: logits dtype must be BF16, F16 or F32", fn);
  if (scoring != XGEN_ROUTE_SOFTMAX && scoring != XGEN_ROUTE_SIGMOID)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: unknown scoring %d", fn, scoring);
  if (tokens <= 0 || experts <= 0 || k <= 0 || k > experts || ld < experts)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: bad shape tokens=%lld experts=%lld k=%lld ld=%lld", fn,
                (long long)tokens, (long long)experts, (long long)k, (long long)ld);
  if (experts > XGEN_ROUTE_MAX_EXPERTS || k > XGEN_ROUTE_MAX_CHOICES)
    return fail(XGEN_ERR_UNSUPPORTED, "%s: up to %d experts and %d choices", fn, XGEN_ROUTE_MAX_EXPERTS,
                XGEN_ROUTE_MAX_CHOICES);
  if (first_expert < 0 || local_experts <= 0 || first_expert > experts - local_experts)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: experts [%lld, %lld) are not among %lld", fn, (long long)first_expert,
                (long long)(first_expert + local_experts), (long long)experts);
  if (!logits || !weights || !chosen || !ends || !rows || !slots)
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: null pointer", fn);
  if (tokens > 0x7fffffffLL / k) return fail(XGEN_ERR_UNSUPPORTED, "%s: tokens * k must be below 2^31", fn);
  const size_t need = xgen_route_workspace_bytes(tokens, local_experts);
  if (need && (!workspace || workspace_bytes < need))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required", fn, need);

  RouteArgs a;
  a.logits = logits;
  a.dtype = in_dtype;
  a.ld = ld;
  a.tokens = tokens;
  a.experts = (int)experts;
  a.k = (int)k;
  a.bias = bias;
  a.sigmoid = scoring == XGEN_ROUTE_SIGMOID;
  a.renormalize = renormalize != 0;
  a.first = (int)first_expert;
  a.local = (int)local_experts;
  a.weights = weights;
  a.chosen = chosen;
  a.ends = ends;
  a.rows = rows;
  a.slots = slots;
  a.counts = static_cast<int32_t *>(workspace);
  a.chunks = (int)chunks_of(tokens);
  a.chunk_tokens = chunk_tokens_of(tokens);
  // the fewest lanes that hold the experts, and the choices (one per lane)
  const int64_t lanes = experts > k ? experts : k;
  if (lanes <= 8) launch<8, 1>(a, stream);
  else if (lanes <= 16) launch<16, 1>(a, stream);
  else if (lanes <= 32) launch<32, 1>(a, stream);
  else if (lanes <= 64) launch<64, 1>(a, stream);
  else if (lanes <= 128) launch<64, 2>(a, stream);
  else if (lanes <= 256) launch<64, 4>(a, stream);
  else launch<64, 8>(a, stream);
  return launch_status(fn);
}
