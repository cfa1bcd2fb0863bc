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
// As many tokens as 4 waves choose for at once (32 of up to 64 experts, 4 of 512) take one launch that chooses, counts
// and places; more take two: chunks of tokens choose and count their pairs per expert; then, from all counts, each
// chunk places its own.  (16 tokens of 128 experts: 7.4 us, in two launches 5.2 + 4.2; 64 tokens: 11.3 us in one
// launch of 16 waves, in two 5.8 + 4.4.)  Up to 4096 tokens a chunk is 16 tokens and a workgroup 4 waves, beyond 64
// and 16: small workgroups spread the choosing over more CUs (4096 tokens 6.5 us against 10), but every one reads the
// counts of all (7.2 us against 6).  Places are ranks (ballots within a wave, per-wave counts in LDS), never the order
// that an atomic happened to take: the plan is the same on every run.
//
// A token is a group of G lanes, a lane V consecutive experts.  A choice is the maximum over the group, the lowest
// lane that has it and that lane's lowest expert with it, which it notes in LDS: nothing but the maximum crosses
// lanes in the loop.  15,624 tokens, 128 experts, bf16: 8.2 us for one choice and 10.8 for eight, and the placement 6.8
// (a wave per token, a ballot per logit and the counts read one by one took 14 and 12).  So a choice costs 0.4 us of
// vector issue, and most of the time does not depend on them: 5.0 us at 501 tokens and 5.1 at 4,096 (the launch and two
// dependent reads), 14.4 at 32,768.
#include "xgen_common.h"

namespace xgen {

namespace {

constexpr int kOneWaves = 4;      // one launch: waves of its workgroup
constexpr int kPerWave = 4;       // two launches: tokens of a chunk per wave
constexpr int kMaxChunks = 512;   // every workgroup reads all chunks' counts: a chunk is several passes beyond

struct RouteArgs {
  const void *logits;
  int64_t ld;  // elements
  int64_t tokens;
  int experts, k;
  const float *bias;
  int sigmoid, renormalize;
  int whole;  // logits can be read 8 at a time
  int first, local;
  float *weights;
  int32_t *chosen, *ends, *rows, *slots;
  int32_t *counts;  // [chunks][local]
  int chunks;
  int64_t chunk_tokens;  // a multiple of kPerWave * waves
};

// V consecutive logits of a token's row from expert e0 on (those from `experts` on: -inf).  Whole: the row's pieces
// are 16-byte aligned and no piece passes the experts.
template <int DT, int V>
__device__ __forceinline__ void load_logits(const RouteArgs &a, int64_t t, int e0, float (&x)[V]) {
  using T = std::conditional_t<DT == XGEN_DTYPE_F32, float, uint16_t>;
  const T *row = static_cast<const T *>(a.logits) + t * a.ld;
  if constexpr (V == 8) {
    if (a.whole) {  // uniform
      // (the last piece's in place of those past it)
      const T *piece = row + min(e0, a.experts - 8);
      const u32x4 w = *reinterpret_cast<const u32x4 *>(piece);
      if constexpr (DT == XGEN_DTYPE_F32) {
        const u32x4 u = *reinterpret_cast<const u32x4 *>(piece + 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) x[v] = __uint_as_float(w[v]), x[v + 4] = __uint_as_float(u[v]);
      } else {
#pragma unroll
        for (int v = 0; v < 4; ++v) x[2 * v] = Half2<DT>::lo(w[v]), x[2 * v + 1] = Half2<DT>::hi(w[v]);
      }
#pragma unroll
      for (int v = 0; v < V; ++v) x[v] = e0 < a.experts ? x[v] : -__builtin_inff();
      return;
    }
  }
  // (the last expert's in place of those past it: loads under a condition each would wait for each other)
  T w[V];
#pragma unroll
  for (int v = 0; v < V; ++v) w[v] = row[min(e0 + v, a.experts - 1)];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if constexpr (DT == XGEN_DTYPE_F32) x[v] = w[v];
    else x[v] = Half2<DT>::lo((uint32_t)w[v]);
    if (e0 + v >= a.experts) x[v] = -__builtin_inff();
  }
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

// What an expert's logit adds to its token's sum (-inf: nothing), over a factor that is the same for all of a token:
// softmax e^top; sigmoid 1 / (1 + e^-x) over e^min(top, 0), so that the sum of the taken ones is a half at least, however
// low all of them are (1 / (1 + e^-x) itself is 0 from -88.8 on).  Without a sum, top is 0 and the factor 1.
__device__ __forceinline__ float score(float x, float top, int sigmoid) {
  if (sigmoid && x >= 0.0f) return 1.0f / (1.0f + expf(-x));
  const float e = x > -__builtin_inff() ? expf(x - (sigmoid ? __builtin_fminf(top, 0.0f) : top)) : 0.0f;
  return sigmoid ? e / (1.0f + expf(x)) : e;
}

// The choices of tokens [t0, t0 + n): expert j of token i at choice[i * k + j] (LDS), weights and experts out; pairs
// counted per expert into hist[local].  logits: V per thread in LDS, a token's in the order of its experts.
template <int DT, int G, int V, int WAVES>
__device__ __forceinline__ void choose(const RouteArgs &a, int64_t t0, int n, int32_t *choice, float *logits,
                                       int32_t *hist) {
  const int gl = threadIdx.x % G, lane = threadIdx.x & 63;
  constexpr int kGroups = 64 * WAVES / G;
  const uint64_t group = (G < 64 ? (1ull << (G & 63)) - 1 : ~0ull) << (lane & ~(G - 1));
  const uint64_t before = group & ((1ull << lane) - 1);  // lanes of the group in front of this one
  const float ninf = -__builtin_inff();
  float bias[V] = {};
  if (a.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias[min(gl * V + v, a.experts - 1)] + 0.0f;  // (never -0)
  }
  for (int i0 = 0; i0 < n; i0 += kGroups) {  // (every lane stays active: groups past the end redo the last token, unseen)
    const int i = i0 + (int)threadIdx.x / G;
    const bool live = i < n;
    if (!__any(live)) break;
    const int64_t t = t0 + (live ? i : n - 1);
    float x[V];
    uint32_t key[V];
    load_logits<DT, V>(a, t, gl * V, x);
#pragma unroll
    for (int v = 0; v < V; ++v) logits[threadIdx.x * V + v] = x[v];
    bool nan = false;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float s = x[v] + bias[v];  // (never -0, so that 0 and -0 rank alike)
      key[v] = s > ninf ? order_key(s) : 0u;  // (-inf, NaN, no expert: 0)
      nan |= !(x[v] == x[v]);
    }
    nan = (__ballot(nan) & group) != 0;  // a NaN logit makes its token's weights NaN
    int32_t *ids = choice + i * a.k;
    uint32_t own = key[0];
#pragma unroll
    for (int v = 1; v < V; ++v) own = max_u32(own, key[v]);
    for (int j = 0; j < a.k; ++j) {
      const uint32_t m = group_max<G>(own);
      const uint64_t has = __ballot(own == m);
      if (own == m && (has & before) == 0) {
        int e = 0;
        bool open = true;
        own = 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const bool hit = open && key[v] == m;
          e = hit ? v : e;
          key[v] = hit ? 0 : key[v];
          open = open && !hit;
          own = max_u32(own, key[v]);
        }
        if (live) ids[j] = m ? gl * V + e : -1;
      }
    }
    // the group's notes in LDS are in front of its reads: one wave, in order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    auto logit = [&](int j) {  // of choice j, -inf for none
      const int e = live && j < a.k ? ids[j] : -1;
      return e < 0 ? ninf : logits[(threadIdx.x - gl) * V + e];
    };
    float top = a.sigmoid ? 0.0f : ninf, total = 0.0f;
    if (a.renormalize) {
      // over the choices; the peak is one of them
      top = ninf;
      for (int j = gl; j < a.k; j += G) top = __builtin_fmaxf(top, logit(j));
      top = from_order_key(group_max<G>(order_key(top)));
      for (int j = gl; j < a.k; j += G) total += score(logit(j), top, a.sigmoid);
      total = group_sum<G>(total);
    } else if (!a.sigmoid) {  // over all experts
      float high = x[0];
#pragma unroll
      for (int v = 1; v < V; ++v) high = __builtin_fmaxf(high, x[v]);
      top = from_order_key(group_max<G>(order_key(high)));
#pragma unroll
      for (int v = 0; v < V; ++v) total += x[v] > ninf ? expf(x[v] - top) : 0.0f;
      total = group_sum<G>(total);
    }
    if (!live) continue;
    for (int j = gl; j < a.k; j += G) {
      const int e = ids[j];
      float w = 0.0f;
      if (e >= 0) {
        w = score(logit(j), top, a.sigmoid);
        if (a.renormalize || !a.sigmoid) w = total > 0.0f ? w / total : total;
        if (nan) w = __builtin_nanf("");
        const int le = e - a.first;
        if (le >= 0 && le < a.local) atomicAdd(&hist[le], 1);
      }
      a.chosen[t * a.k + j] = e;
      a.weights[t * a.k + j] = w;
    }
  }
}

// What the placement keeps in LDS.
template <int WAVES, int TOKENS>
struct RouteShared {
  static constexpr int kWaves = WAVES, kThreads = 64 * WAVES;
  int32_t ids[TOKENS * XGEN_ROUTE_MAX_CHOICES];
  int32_t count[WAVES * XGEN_ROUTE_MAX_EXPERTS];  // [wave][local]: pairs of the wave's segment; then its first place
  int32_t base[XGEN_ROUTE_MAX_EXPERTS];           // the chunk's first place per expert
  int32_t total[XGEN_ROUTE_MAX_EXPERTS];
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
template <class Shared>
__device__ __forceinline__ void first_places(const RouteArgs &a, bool write_ends, Shared &sh) {
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

// The places of the n pairs from token t0 on, whose choices are in sh.ids; sh.base moves on past them.
template <class Shared>
__device__ __forceinline__ void place(const RouteArgs &a, int64_t t0, int n, Shared &sh) {
  constexpr int kWaves = Shared::kWaves, kThreads = Shared::kThreads;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kWaves * a.local; i += kThreads) sh.count[i] = 0;
  __syncthreads();
  int32_t *count = sh.count + wave * a.local;
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
    if (g < a.local && lane == __builtin_ctzll(same)) atomicAdd(&count[g], __builtin_popcountll(same));
  }
  __syncthreads();
  for (int e = tid; e < a.local; e += kThreads) {
    int32_t at = sh.base[e];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int32_t c = sh.count[w * a.local + e];
      sh.count[w * a.local + e] = at;
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
    if (g < a.local && lane == leader) at = atomicAdd(&count[g], __builtin_popcountll(same));
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

template <int DT, int G, int V>
__global__ __launch_bounds__(64 * kOneWaves) void route_one_kernel(RouteArgs a) {
  __shared__ RouteShared<kOneWaves, 64 * kOneWaves / G> sh;
  __shared__ __align__(16) float logits[64 * kOneWaves * V];
  for (int e = threadIdx.x; e < a.local; e += 64 * kOneWaves) sh.total[e] = sh.base[e] = 0;
  __syncthreads();
  choose<DT, G, V, kOneWaves>(a, 0, (int)a.tokens, sh.ids, logits, sh.total);
  first_places(a, true, sh);
  place(a, 0, (int)a.tokens * a.k, sh);
}

template <int DT, int G, int V, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void route_choose_kernel(RouteArgs a) {
  constexpr int kThreads = 64 * WAVES, kChunk = kPerWave * WAVES;
  __shared__ int32_t ids[kChunk * XGEN_ROUTE_MAX_CHOICES], total[XGEN_ROUTE_MAX_EXPERTS];
  __shared__ __align__(16) float logits[kThreads * V];
  for (int e = threadIdx.x; e < a.local; e += kThreads) total[e] = 0;
  __syncthreads();
  const int64_t begin = (int64_t)blockIdx.x * a.chunk_tokens;
  const int64_t end = begin + a.chunk_tokens < a.tokens ? begin + a.chunk_tokens : a.tokens;
  // (a wave's tokens are its own in LDS: no barrier between passes)
  for (int64_t t0 = begin; t0 < end; t0 += kChunk)
    choose<DT, G, V, WAVES>(a, t0, (int)(end - t0 < kChunk ? end - t0 : kChunk), ids, logits, total);
  __syncthreads();
  for (int e = threadIdx.x; e < a.local; e += kThreads) a.counts[(int64_t)blockIdx.x * a.local + e] = total[e];
}

template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void route_place_kernel(RouteArgs a) {
  constexpr int kThreads = 64 * WAVES, kChunk = kPerWave * WAVES;
  __shared__ RouteShared<WAVES, kChunk> sh;
  const int tid = threadIdx.x;
  for (int e = tid; e < a.local; e += kThreads) sh.total[e] = sh.base[e] = 0;
  __syncthreads();
  // counts of all chunks and of those before this one: the threads share out the experts, four each where they
  // divide, and the chunks
  auto sum = [&](auto WIDTH) {
    constexpr int W = decltype(WIDTH)::value;
    using Counts = std::conditional_t<W == 4, i32x4, int32_t>;
    const int columns = a.local / W;
    int span = 1;
    while (span < columns && span < kThreads) span <<= 1;
    const int part = tid / span, parts = kThreads / span;
    for (int c0 = 0; c0 < columns; c0 += span) {
      const int c = c0 + (tid & (span - 1));
      int32_t all[W] = {}, before[W] = {};
      if (c < columns) {
        constexpr int kDeep = 8;  // reads in flight (a missing chunk: one that is there, uncounted)
        for (int i0 = part; i0 < a.chunks; i0 += kDeep * parts) {
          Counts v[kDeep];
#pragma unroll
          for (int d = 0; d < kDeep; ++d)
            v[d] = *reinterpret_cast<const Counts *>(a.counts + (int64_t)min(i0 + d * parts, a.chunks - 1) * a.local + c * W);
#pragma unroll
          for (int d = 0; d < kDeep; ++d) {
            const int i = i0 + d * parts;
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const int32_t n = reinterpret_cast<const int32_t *>(&v[d])[w];
              all[w] += i < a.chunks ? n : 0;
              before[w] += i < (int)blockIdx.x ? n : 0;
            }
          }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (all[w]) atomicAdd(&sh.total[c * W + w], all[w]);
          if (before[w]) atomicAdd(&sh.base[c * W + w], before[w]);
        }
      }
    }
  };
  if (a.local % 4 == 0 && (reinterpret_cast<uintptr_t>(a.counts) & 15) == 0) sum(std::integral_constant<int, 4>());
  else sum(std::integral_constant<int, 1>());
  first_places(a, blockIdx.x == 0, sh);
  const int64_t begin = (int64_t)blockIdx.x * a.chunk_tokens;
  const int64_t end = begin + a.chunk_tokens < a.tokens ? begin + a.chunk_tokens : a.tokens;
  for (int64_t t0 = begin; t0 < end; t0 += kChunk) {
    const int n = (int)(end - t0 < kChunk ? end - t0 : kChunk) * a.k;
    __syncthreads();  // the places before are done with sh.ids
    for (int i = tid; i < n; i += kThreads) sh.ids[i] = a.chosen[t0 * a.k + i];
    place(a, t0, n, sh);
  }
}

// Lanes of a token: 8 experts each, 8 lanes at least.
int lanes_of(int64_t experts) { return experts <= 64 ? 8 : experts <= 128 ? 16 : experts <= 256 ? 32 : 64; }
bool one_launch(int64_t tokens, int64_t experts) { return tokens <= kOneWaves * 64 / lanes_of(experts); }
int waves_of(int64_t tokens) { return tokens <= 4096 ? 4 : 16; }
int64_t chunk_tokens_of(int64_t tokens) {
  const int64_t pass = kPerWave * waves_of(tokens), pieces = (tokens + pass - 1) / pass;
  return (pieces + kMaxChunks - 1) / kMaxChunks * pass;
}
int64_t chunks_of(int64_t tokens) { return (tokens + chunk_tokens_of(tokens) - 1) / chunk_tokens_of(tokens); }

template <int DT, int G, int V>
void launch(const RouteArgs &a, hipStream_t stream) {
  const dim3 grid((unsigned)a.chunks);
  if (one_launch(a.tokens, a.experts)) {
    route_one_kernel<DT, G, V><<<dim3(1), dim3(64 * kOneWaves), 0, stream>>>(a);
  } else if (waves_of(a.tokens) == 4) {
    route_choose_kernel<DT, G, V, 4><<<grid, dim3(256), 0, stream>>>(a);
    route_place_kernel<4><<<grid, dim3(256), 0, stream>>>(a);
  } else {
    route_choose_kernel<DT, G, V, 16><<<grid, dim3(1024), 0, stream>>>(a);
    route_place_kernel<16><<<grid, dim3(1024), 0, stream>>>(a);
  }
}
template <int DT>
void launch(const RouteArgs &a, hipStream_t stream) {
  if (a.experts <= 8) launch<DT, 8, 1>(a, stream);
  else if (a.experts <= 16) launch<DT, 8, 2>(a, stream);
  else if (a.experts <= 32) launch<DT, 8, 4>(a, stream);
  else if (a.experts <= 64) launch<DT, 8, 8>(a, stream);
  else if (a.experts <= 128) launch<DT, 16, 8>(a, stream);
  else if (a.experts <= 256) launch<DT, 32, 8>(a, stream);
  else launch<DT, 64, 8>(a, stream);
}

}  // namespace

}  // namespace xgen

using namespace xgen;

extern "C" size_t xgen_route_workspace_bytes(int64_t tokens, int64_t experts, int64_t local_experts) {
  if (tokens <= 0 || local_experts <= 0 || one_launch(tokens, experts)) return 0;
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
  const size_t need = xgen_route_workspace_bytes(tokens, experts, local_experts);
  if (need && (!workspace || workspace_bytes < need))
    return fail(XGEN_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes required", fn, need);

  RouteArgs a;
  a.logits = logits;
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
  a.whole = aligned16(logits) && ld % 8 == 0 && experts % 8 == 0;
  if (in_dtype == XGEN_DTYPE_F32) launch<XGEN_DTYPE_F32>(a, stream);
  else if (in_dtype == XGEN_DTYPE_BF16) launch<XGEN_DTYPE_BF16>(a, stream);
  else launch<XGEN_DTYPE_F16>(a, stream);
  return launch_status(fn);
}
