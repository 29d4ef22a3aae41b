// Routing to experts: every token's scores, its best experts and their weights, and the pairs in the order of their experts.
//
//   s = softmax(l) or 1 / (1 + exp(-l));   c = s + bias, or l itself without a bias (the order of the scores is that of the logits)
//   groups: a group is worth the sum of its best two c (without a bias: of their s); the best of them stay, the others' c are out
//   the `top` best c, descending, the lowest index where equal; weights = their s, over their sum if asked for, times `scale`
//
// A logit (or a bias) that is NaN counts as -infinity, and an expert of -infinity has the score 0; a row of nothing else gets the
// first experts with weights of 0. All in fp32.
//
// A wavefront takes a token, its logits in registers, V neighbours to a lane; a choice is a maximum over the wavefront, of the
// values as sortable integers, and the first lane that has it. The pairs are sorted by counting:
// tokens are dealt in order to workgroups and their wavefronts, and a wavefront places its tokens one after the other -- a
// token's experts are all different, so its lanes can place them at once. That makes the order stable and the same every time.
// What bounds it are latencies: 8 tokens of 32 experts 3.2 us in one launch; 8191 of 256, 4.2 MB of logits, 14.6 + 9.2 us in two
// (branches around single loads, one wait each, had made the first 19.5; counts summed one load at a time the second 60). In the second each
// of 256 workgroups reads every workgroup's counts, 67 MB in all, and one wavefront of it scans them; of 32 experts, softmax, 4.4 + 6.6.
#include "mx_common.h"

namespace tllm {

constexpr int ROUTE_E = 512, ROUTE_TOP = 32, ROUTE_GROUPS = 64;
constexpr int ROUTE_WAVES = 16;           // wavefronts of a workgroup
constexpr int ROUTE_RUNS = 256;           // most workgroups that count
constexpr int ROUTE_ALONE = 64;           // tokens that one workgroup routes and sorts in one launch

struct RouteArgs {
  const void* logits;
  int64_t row_stride;
  const float* bias;
  int* experts;
  float* weights;
  int* order;
  int* offsets;
  int* counts;                            // [runs][n_experts]
  int64_t tokens;
  int n_experts, top, groups, kept, renorm;
  float scale;
  int per_wave, runs;                     // tokens of a wavefront; workgroups
};

__device__ __forceinline__ unsigned wave_max_u32(unsigned v) {
  auto dpp = [](unsigned x, auto ctrl) { return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));
  v = max(v, dpp(v, std::integral_constant<int, 0x140>{}));
  const unsigned r0 = __builtin_amdgcn_readlane(v, 0), r1 = __builtin_amdgcn_readlane(v, 16), r2 = __builtin_amdgcn_readlane(v, 32), r3 = __builtin_amdgcn_readlane(v, 48);
  return max(max(r0, r1), max(r2, r3));
}

// Lanes of one wavefront see each other's LDS writes in the order of the program; this keeps the compiler to it.
__device__ __forceinline__ void lds_in_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); }

// fp32 as an unsigned integer of the same order; -0 is 0 and NaN -infinity. No float gives 0.
__device__ __forceinline__ unsigned sortable(float v) {
  v = v != v ? -__builtin_inff() : v + 0.0f;
  const unsigned b = __builtin_bit_cast(unsigned, v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The largest key of the wavefront and its expert V lane + v, the lowest where several have it; it is taken out.
template <int V>
__device__ __forceinline__ int take_best(unsigned (&key)[V], int lane) {
  unsigned best = key[0];
#pragma unroll
  for (int v = 1; v < V; ++v) best = max(best, key[v]);
  const unsigned top = wave_max_u32(best);
  int at = V - 1;
#pragma unroll
  for (int v = V - 2; v >= 0; --v) at = key[v] == top ? v : at;
  const int l = __builtin_ctzll(__ballot(best == top));
  const int e = V * l + __builtin_amdgcn_readlane(at, l);
#pragma unroll
  for (int v = 0; v < V; ++v) key[v] = V * lane + v == e ? 0 : key[v];
  return e;
}

// The best two of a pair of values and another's
__device__ __forceinline__ void best_two(float& one, float& two, float a, float b) {
  two = fmaxf(fminf(one, a), fmaxf(two, b));
  one = fmaxf(one, a);
}

// One token: lane j < top has its j-th expert in the result, and writes that and the weight.
template <int V, bool SIGMOID, class T>
__device__ __forceinline__ int route_token(const RouteArgs& a, const float (&bias)[V], int64_t t, int lane, float* mine) {
  const float ninf = -__builtin_inff();
  const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
  float score[V];
  unsigned key[V];
  T l[V];
#pragma unroll
  for (int v = 0; v < V; ++v) l[v] = row[min(V * lane + v, a.n_experts - 1)];   // (no branch: the loads leave together)
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float f = static_cast<float>(l[v]);
    score[v] = V * lane + v >= a.n_experts || f != f ? ninf : f;
  }
  float best = ninf, sum = 0.f;
  if constexpr (!SIGMOID) {
#pragma unroll
    for (int v = 0; v < V; ++v) best = fmaxf(best, score[v]);
    best = wave_max(best);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float l = score[v];
    key[v] = V * lane + v < a.n_experts ? sortable(l) : 0;
    if constexpr (SIGMOID) score[v] = 1.0f / (1.0f + expf(-l));
    else score[v] = l == ninf ? 0.f : l == best ? 1.f : expf(l - best);     // (an infinite logit takes all)
    sum += score[v];
  }
  if constexpr (!SIGMOID) {
    sum = wave_sum(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) score[v] = sum > 0.f ? score[v] / sum : 0.f;
  }
  if (a.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (V * lane + v < a.n_experts) key[v] = sortable(score[v] + bias[v]);
  }
  if (a.groups > 1) {
    const int size = a.n_experts / a.groups, lanes = size / V;
    float c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      c[v] = a.bias ? score[v] + bias[v] : score[v];
      c[v] = c[v] != c[v] ? ninf : c[v];
    }
    float value;                                            // of this lane's group, or of group `lane`
    const bool spans = size == lanes * V && lanes > 0 && (lanes & (lanes - 1)) == 0;
    if (spans) {                                            // a group is a power of two of whole lanes
      float one = c[0], two = ninf;
#pragma unroll
      for (int v = 1; v < V; ++v) best_two(one, two, c[v], ninf);
#pragma unroll
      for (int d = 1; d < 64; d *= 2)
        if (d < lanes) best_two(one, two, __shfl_xor(one, d), __shfl_xor(two, d));
      value = size > 1 ? one + two : one;
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (V * lane + v < a.n_experts) mine[V * lane + v] = c[v];
      lds_in_order();
      float one = ninf, two = ninf;
      if (lane < a.groups)
        for (int i = 0; i < size; ++i) best_two(one, two, mine[lane * size + i], ninf);
      value = size > 1 ? one + two : one;
      lds_in_order();
    }
    // a group stays if fewer than `kept` are worth more, or as much with a lower number
    const unsigned gk = sortable(value);
    const int step = spans ? lanes : 1, group = lane / step;
    int ahead = 0;
    for (int j = 0; j < a.groups; ++j) {
      const unsigned o = __builtin_amdgcn_readlane(gk, j * step);
      ahead += o > gk || (o == gk && j < group);
    }
    const unsigned long long stay = __ballot(ahead < a.kept);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int of = spans ? lane : (V * lane + v) / size;  // the lane that knows of the group
      if (of > 63 || !(stay >> (of & 63) & 1)) key[v] = 0;
    }
  }
  int expert = 0;
  float weight = 0.f, total = 0.f;
  for (int j = 0; j < a.top; ++j) {
    const int e = take_best<V>(key, lane);
    float s = score[0];
#pragma unroll
    for (int v = 1; v < V; ++v) s = e % V == v ? score[v] : s;
    s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), e / V));
    total += s;
    expert = lane == j ? e : expert;
    weight = lane == j ? s : weight;
  }
  if (lane < a.top) {
    if (a.renorm) weight = total > 0.f ? weight / total : 0.f;
    a.experts[t * a.top + lane] = expert;
    a.weights[t * a.top + lane] = weight * a.scale;
  }
  return expert;
}

// Counts of a workgroup's wavefronts become their first places: each expert's `start` (the pairs before its own, of all experts
// before and of the workgroups before), then the wavefronts one after the other.
__device__ __forceinline__ void first_places(int* count, int pitch, const int* start, int n_experts) {
  for (int e = threadIdx.x; e < n_experts; e += ROUTE_WAVES * 64) {
    int at = start[e], c[ROUTE_WAVES];
#pragma unroll
    for (int w = 0; w < ROUTE_WAVES; ++w) c[w] = count[w * pitch + e];
#pragma unroll
    for (int w = 0; w < ROUTE_WAVES; ++w) {
      count[w * pitch + e] = at;
      at += c[w];
    }
  }
}

// Sum over the lanes up to this one: inside the rows of sixteen, then the first row's last to the second and the third's to the
// fourth, then the second's to the upper half.
__device__ __forceinline__ int wave_upto(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

// One wavefront: all[e], pairs of expert e, becomes the pairs of the experts before it; so do the offsets, if they are to be written.
__device__ __forceinline__ void scan_experts(int* all, int n_experts, int lane, int* offsets) {
  int before = 0;
  for (int e0 = 0; e0 < n_experts; e0 += 64) {
    const int e = e0 + lane, n = e < n_experts ? all[e] : 0;
    const int upto = wave_upto(n), start = before + upto - n;
    if (e < n_experts) {
      all[e] = start;
      if (offsets) offsets[e] = start;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  if (offsets && lane == 0) offsets[n_experts] = before;
}

// Many tokens: four to a wavefront, a token's experts in the sixteen lanes of a DPP row, V neighbours to a lane. All of a choice is
// then vector work of four tokens at once -- a maximum inside the row, the first lane that has it, its first value. A wavefront takes
// longer over its tokens that way, but there is a quarter as much to issue: of 256 experts in groups, the best 8, both launches,
// 32768 tokens 61.5 us with a token to a wavefront, 51.0 so, 8191 24.4 and 23.3, 2048 15.2 and 18.5. Groups have to be whole
// lanes, a power of two of them, and `top` at most sixteen, one to a lane. The tokens of workgroup b are those of the kernel below, so
// that the pairs are placed by the same counts.
constexpr int FOURS_WAVES = 8, FOURS_FROM = 6000;
__device__ __forceinline__ unsigned row_max_u32(unsigned v) {
  auto dpp = [](unsigned x, auto ctrl) { return static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));
  return max(v, dpp(v, std::integral_constant<int, 0x140>{}));
}
template <class Op>
__device__ __forceinline__ float row_all(float v, Op op) {
  auto dpp = [](float x, auto ctrl) { return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  v = op(v, dpp(v, std::integral_constant<int, 0xB1>{}));
  v = op(v, dpp(v, std::integral_constant<int, 0x4E>{}));
  v = op(v, dpp(v, std::integral_constant<int, 0x141>{}));
  return op(v, dpp(v, std::integral_constant<int, 0x140>{}));
}
template <int V, bool SIGMOID, class T>
__global__ __launch_bounds__(FOURS_WAVES * 64) void moe_route_fours_kernel(RouteArgs a) {
  __shared__ int count[16 * V];
  const float ninf = -__builtin_inff();
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, base = lane & 48;
  for (int i = tid; i < 16 * V; i += FOURS_WAVES * 64) count[i] = 0;
  float bias[V] = {};
  if (a.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias[min(V * l16 + v, a.n_experts - 1)];
  }
  __syncthreads();
  const int64_t first = static_cast<int64_t>(blockIdx.x) * ROUTE_WAVES * a.per_wave;
  const int per_run = ROUTE_WAVES * a.per_wave;
  // rows of whole sixteens come in as such
  const bool whole = a.n_experts == 16 * V && V * sizeof(T) % 16 == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.row_stride * sizeof(T) % 16 == 0;
  for (int i0 = 4 * wave; i0 < per_run && first + i0 < a.tokens; i0 += 4 * FOURS_WAVES) {
    const int64_t mine = first + i0 + (lane >> 4);
    const bool there = mine < a.tokens;
    const int64_t t = there ? mine : a.tokens - 1;
    const T* const row = static_cast<const T*>(a.logits) + t * a.row_stride;
    T l[V];
    if (whole) {
      typedef __attribute__((__vector_size__(16))) T T16;
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int v = 0; v + N <= V; v += N) {
        const T16 x = *reinterpret_cast<const T16*>(row + V * l16 + v);
#pragma unroll
        for (int i = 0; i < N; ++i) l[v + i] = x[i];
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) l[v] = row[min(V * l16 + v, a.n_experts - 1)];
    }
    float s[V];                                             // logits, then scores
    float best = ninf, sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float f = static_cast<float>(l[v]);
      s[v] = V * l16 + v >= a.n_experts || f != f ? ninf : f;
      best = fmaxf(best, s[v]);
    }
    unsigned key[V];
    if constexpr (!SIGMOID) best = row_all(best, [](float x, float y) { return fmaxf(x, y); });
    // the scores of all are needed for softmax's sum, a bias or groups; otherwise the chosen ones' alone, below
    auto score_of = [&](float x) {
      if constexpr (SIGMOID) return 1.0f / (1.0f + expf(-x));
      else return x == ninf ? 0.f : x == best ? 1.f : expf(x - best);       // (an infinite logit takes all)
    };
    const bool all = !SIGMOID || a.bias || a.groups > 1;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      key[v] = V * l16 + v < a.n_experts ? sortable(s[v]) : 0;
      if (all) {
        s[v] = score_of(s[v]);
        sum += s[v];
      }
    }
    if constexpr (!SIGMOID) {
      sum = row_all(sum, [](float x, float y) { return x + y; });
      if (a.bias || a.groups > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) s[v] = sum > 0.f ? s[v] / sum : 0.f;
      }
    }
    if (a.bias) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        s[v] += bias[v];
        key[v] = V * l16 + v < a.n_experts ? sortable(s[v]) : 0;
      }
    }
    if (a.groups > 1) {
      const int lanes = a.n_experts / a.groups / V;
      float one = ninf, two = ninf;
#pragma unroll
      for (int v = 0; v < V; ++v) best_two(one, two, s[v] != s[v] ? ninf : s[v], ninf);
#pragma unroll
      for (int d = 1; d < 16; d *= 2)
        if (d < lanes) best_two(one, two, __shfl_xor(one, d), __shfl_xor(two, d));
      const unsigned gk = sortable(V * lanes > 1 ? one + two : one);
      const int group = l16 / lanes;
      int ahead = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const unsigned o = __shfl(gk, base + ((j * lanes) & 15));
        ahead += j < a.groups && (o > gk || (o == gk && j < group));
      }
      if (ahead >= a.kept) {
#pragma unroll
        for (int v = 0; v < V; ++v) key[v] = 0;
      }
    }
    int expert = 0;
    T chosen = static_cast<T>(0.f);
    for (int j = 0; j < a.top; ++j) {
      unsigned half[V];                                     // (a tree: the steps of a chain would wait for one another)
#pragma unroll
      for (int v = 0; v < V; ++v) half[v] = key[v];
#pragma unroll
      for (int d = V / 2; d >= 1; d /= 2)
#pragma unroll
        for (int v = 0; v < d; ++v) half[v] = max(half[v], half[v + d]);
      const unsigned own = half[0], top = row_max_u32(own);
      const unsigned has = static_cast<unsigned>(__ballot(own == top) >> base) & 0xffffu;
      const int who = __builtin_ctz(has);
      unsigned hits[V];
#pragma unroll
      for (int v = 0; v < V; ++v) hits[v] = key[v] == top ? 1u << v : 0u;
#pragma unroll
      for (int d = V / 2; d >= 1; d /= 2)
#pragma unroll
        for (int v = 0; v < d; ++v) hits[v] |= hits[v + d];
      const int at = __builtin_ctz(hits[0] | 0x80000000u);
      const int gone = l16 == who ? at : -1;
#pragma unroll
      for (int v = 0; v < V; ++v) key[v] = v == gone ? 0 : key[v];
      const int e = V * who + __shfl(at, base + who);
      if (l16 == j) {
        expert = e;
        chosen = row[e];
      }
    }
    float weight = 0.f;
    if (l16 < a.top) {
      const float f = static_cast<float>(chosen);
      weight = score_of(f != f ? ninf : f);
      if (!SIGMOID) weight = sum > 0.f ? weight / sum : 0.f;
    }
    const float total = row_all(weight, [](float x, float y) { return x + y; });
    if (a.renorm) weight = total > 0.f ? weight / total : 0.f;
    if (there && l16 < a.top) {
      a.experts[t * a.top + l16] = expert;
      a.weights[t * a.top + l16] = weight * a.scale;
      atomicAdd(&count[expert], 1);
    }
  }
  __syncthreads();
  for (int e = tid; e < a.n_experts; e += FOURS_WAVES * 64) a.counts[static_cast<int64_t>(blockIdx.x) * a.n_experts + e] = count[e];
}

// The tokens of workgroup b, wavefront w: per_wave of them from (b ROUTE_WAVES + w) per_wave on.
template <int V, bool SIGMOID, class T, bool ALONE>
__global__ __launch_bounds__(ROUTE_WAVES * 64) void moe_route_kernel(RouteArgs a) {
  __shared__ float choices[ROUTE_WAVES][V * 64];
  __shared__ int count[ALONE ? ROUTE_WAVES : 1][V * 64], start[ALONE ? V * 64 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int i = threadIdx.x; i < static_cast<int>(sizeof(count) / 4); i += ROUTE_WAVES * 64) count[0][i] = 0;
  __syncthreads();
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * ROUTE_WAVES + wave) * a.per_wave;
  float bias[V] = {};
  if (a.bias) {
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = a.bias[min(V * lane + v, a.n_experts - 1)];
  }
  int chosen[ALONE ? ROUTE_ALONE / ROUTE_WAVES : 1];
  if constexpr (ALONE) {
#pragma unroll
    for (int i = 0; i < ROUTE_ALONE / ROUTE_WAVES; ++i)
      if (i < a.per_wave && t0 + i < a.tokens) {
        chosen[i] = route_token<V, SIGMOID, T>(a, bias, t0 + i, lane, choices[wave]);
        if (lane < a.top) count[wave][chosen[i]] += 1;      // (a token's experts are different ones)
        lds_in_order();
      }
  } else {
    for (int i = 0; i < a.per_wave && t0 + i < a.tokens; ++i) {
      const int e = route_token<V, SIGMOID, T>(a, bias, t0 + i, lane, choices[wave]);
      if (lane < a.top) atomicAdd(&count[0][e], 1);
    }
  }
  __syncthreads();
  if constexpr (!ALONE) {
    for (int e = threadIdx.x; e < a.n_experts; e += ROUTE_WAVES * 64) a.counts[static_cast<int64_t>(blockIdx.x) * a.n_experts + e] = count[0][e];
  } else {
    for (int e = threadIdx.x; e < a.n_experts; e += ROUTE_WAVES * 64) {
      int n = 0;
#pragma unroll
      for (int w = 0; w < ROUTE_WAVES; ++w) n += count[w][e];
      start[e] = n;
    }
    __syncthreads();
    if (wave == 0) scan_experts(start, a.n_experts, lane, a.offsets);
    __syncthreads();
    first_places(count[0], V * 64, start, a.n_experts);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ROUTE_ALONE / ROUTE_WAVES; ++i)
      if (i < a.per_wave && t0 + i < a.tokens && lane < a.top) {
        lds_in_order();
        const int at = count[wave][chosen[i]];
        count[wave][chosen[i]] = at + 1;
        a.order[at] = static_cast<int>((t0 + i) * a.top + lane);
      }
  }
}

// Places the pairs of a run (the tokens of one workgroup of the kernel before): behind the experts before theirs, the runs
// before this one, and the wavefronts before this one.
__global__ __launch_bounds__(ROUTE_WAVES * 64) void moe_place_kernel(RouteArgs a) {
  __shared__ int all[ROUTE_E], earlier[ROUTE_E], count[ROUTE_WAVES][ROUTE_E];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int E = a.n_experts, run = blockIdx.x;
  constexpr int THREADS = ROUTE_WAVES * 64;
  for (int i = tid; i < ROUTE_WAVES * ROUTE_E; i += THREADS) count[0][i] = 0;
  for (int e = tid; e < ROUTE_E; e += THREADS) all[e] = earlier[e] = 0;
  __syncthreads();
  // this wavefront's first tokens' experts, read once where there are few
  constexpr int HELD = 4;
  const int64_t t0 = (static_cast<int64_t>(run) * ROUTE_WAVES + wave) * a.per_wave;
  int held[HELD];
#pragma unroll
  for (int i = 0; i < HELD; ++i) {
    const int64_t t = t0 + i < a.tokens ? t0 + i : a.tokens - 1;
    held[i] = a.experts[t * a.top + (lane < a.top ? lane : 0)];
  }
  auto expert_of = [&](int i) { return i == 0 ? held[0] : i == 1 ? held[1] : i == 2 ? held[2] : i == 3 ? held[3] : a.experts[(t0 + i) * a.top + lane]; };
  // the runs' counts, dealt to the threads by expert and by run, thirty-two of a thread's on their way at a time
  const int parts = THREADS / E, part = tid / E, mine = tid - part * E;
  if (part < parts) {
    int total = 0, before = 0;
    for (int r0 = part; r0 < a.runs; r0 += 32 * parts) {
      int c[32];
#pragma unroll
      for (int j = 0; j < 32; ++j) c[j] = r0 + j * parts < a.runs ? a.counts[static_cast<int64_t>(r0 + j * parts) * E + mine] : 0;
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        total += c[j];
        before += r0 + j * parts < run ? c[j] : 0;
      }
    }
    atomicAdd(&all[mine], total);
    atomicAdd(&earlier[mine], before);
  }
  for (int i = 0; i < a.per_wave && t0 + i < a.tokens; ++i) {
    if (lane < a.top) count[wave][expert_of(i)] += 1;
    lds_in_order();
  }
  __syncthreads();
  if (wave == 0) scan_experts(all, E, lane, run == 0 ? a.offsets : nullptr);
  __syncthreads();
  for (int e = tid; e < E; e += THREADS) all[e] += earlier[e];
  __syncthreads();
  first_places(count[0], ROUTE_E, all, E);
  __syncthreads();
  for (int i = 0; i < a.per_wave && t0 + i < a.tokens; ++i) {
    lds_in_order();
    if (lane < a.top) {
      const int64_t p = (t0 + i) * a.top + lane;
      int* const c = &count[wave][expert_of(i)];
      const int at = *c;
      *c = at + 1;
      a.order[at] = static_cast<int>(p);
    }
  }
}

// Whether the choice can be made in a row of sixteen lanes with V experts each
static bool in_fours(const RouteArgs& a, int V) {
  if (a.top > 16) return false;
  if (a.groups == 1) return true;
  const int size = a.n_experts / a.groups, lanes = size / V;
  return size % V == 0 && lanes > 0 && (lanes & (lanes - 1)) == 0;
}
template <int V>
static int launch_fours(const RouteArgs& a, bool sigmoid, bool is_f32, hipStream_t st) {
  auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, dim3(a.runs), dim3(FOURS_WAVES * 64), 0, st, a); };
  if (sigmoid) is_f32 ? go(moe_route_fours_kernel<V, true, float>) : go(moe_route_fours_kernel<V, true, bf16>);
  else is_f32 ? go(moe_route_fours_kernel<V, false, float>) : go(moe_route_fours_kernel<V, false, bf16>);
  return check_launch("moe_route");
}

template <int V>
static int launch_route(const RouteArgs& a, bool sigmoid, bool is_f32, bool alone, hipStream_t st) {
  auto go = [&](auto* kernel) { hipLaunchKernelGGL(kernel, dim3(a.runs), dim3(ROUTE_WAVES * 64), 0, st, a); };
  auto type = [&](auto sig, auto one) {
    constexpr bool S = decltype(sig)::value, A = decltype(one)::value;
    if (is_f32) go(moe_route_kernel<V, S, float, A>);
    else go(moe_route_kernel<V, S, bf16, A>);
  };
  if (sigmoid) alone ? type(std::true_type{}, std::true_type{}) : type(std::true_type{}, std::false_type{});
  else alone ? type(std::false_type{}, std::true_type{}) : type(std::false_type{}, std::false_type{});
  return check_launch("moe_route");
}

static int route_runs(int64_t tokens, int* per_wave) {
  const int64_t per = (tokens + ROUTE_RUNS * ROUTE_WAVES - 1) / (ROUTE_RUNS * ROUTE_WAVES);
  *per_wave = static_cast<int>(tokens > ROUTE_ALONE ? per : tokens > 0 ? (tokens + ROUTE_WAVES - 1) / ROUTE_WAVES : 1);
  return static_cast<int>((tokens + static_cast<int64_t>(*per_wave) * ROUTE_WAVES - 1) / (static_cast<int64_t>(*per_wave) * ROUTE_WAVES));
}

}  // namespace tllm

using namespace tllm;

extern "C" int64_t tllm_moe_route_workspace_bytes(int64_t tokens, int n_experts) {
  if (tokens <= ROUTE_ALONE || n_experts < 1) return 0;
  int per;
  return static_cast<int64_t>(route_runs(tokens, &per)) * n_experts * 4;
}

extern "C" int tllm_moe_route(const void* logits, int logits_is_f32, int64_t logits_row_stride, const float* bias, int sigmoid, int n_groups, int topk_groups,
                              int renormalize, float scale, int32_t* experts, float* weights, int32_t* order, int32_t* offsets, void* workspace,
                              int64_t workspace_bytes, int64_t tokens, int n_experts, int top, void* stream) {
  TLLM_REQUIRE(tokens >= 0, TLLM_E_ARG, "moe_route: tokens %lld", (long long)tokens);
  TLLM_REQUIRE(n_experts >= 1 && n_experts <= ROUTE_E, TLLM_E_SHAPE, "moe_route: %d experts, 1 to %d are supported", n_experts, ROUTE_E);
  TLLM_REQUIRE(n_groups >= 1 && n_groups <= ROUTE_GROUPS && n_experts % n_groups == 0, TLLM_E_SHAPE, "moe_route: %d experts in %d groups", n_experts, n_groups);
  TLLM_REQUIRE(topk_groups >= 1 && topk_groups <= n_groups, TLLM_E_SHAPE, "moe_route: %d of %d groups", topk_groups, n_groups);
  TLLM_REQUIRE(top >= 1 && top <= ROUTE_TOP && top <= n_experts / n_groups * topk_groups, TLLM_E_SHAPE,
               "moe_route: top %d of %d experts (%d of %d groups); at most %d", top, n_experts, topk_groups, n_groups, ROUTE_TOP);
  TLLM_REQUIRE(tokens * top < (1ll << 31), TLLM_E_SHAPE, "moe_route: %lld tokens x %d are too many", (long long)tokens, top);
  TLLM_REQUIRE(offsets, TLLM_E_ARG, "moe_route: null pointer");
  TLLM_REQUIRE(tokens == 0 || (logits && experts && weights && order), TLLM_E_ARG, "moe_route: null pointer");
  TLLM_REQUIRE(logits_row_stride >= n_experts || tokens <= 1, TLLM_E_ARG, "moe_route: logits_row_stride %lld < %d experts", (long long)logits_row_stride, n_experts);
  const int64_t need = tllm_moe_route_workspace_bytes(tokens, n_experts);
  TLLM_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), TLLM_E_ARG, "moe_route: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes,
               (long long)need);
  RouteArgs a{logits, logits_row_stride, bias, experts, weights, order, offsets, static_cast<int*>(workspace), tokens, n_experts, top, n_groups, topk_groups,
              renormalize, scale, 0, 0};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool alone = tokens <= ROUTE_ALONE;
  a.runs = route_runs(tokens, &a.per_wave);
  if (tokens == 0) a.runs = 1;                             // (the offsets alone, all 0)
  const bool s = sigmoid != 0, f = logits_is_f32 != 0;
  const int per_lane = n_experts <= 32 ? 2 : n_experts <= 64 ? 4 : n_experts <= 128 ? 8 : n_experts <= 256 ? 16 : 32;
  const bool fours = tokens >= FOURS_FROM && in_fours(a, per_lane);
  const int rc = fours ? (per_lane == 2   ? launch_fours<2>(a, s, f, st)
                          : per_lane == 4  ? launch_fours<4>(a, s, f, st)
                          : per_lane == 8  ? launch_fours<8>(a, s, f, st)
                          : per_lane == 16 ? launch_fours<16>(a, s, f, st)
                                           : launch_fours<32>(a, s, f, st))
               : n_experts <= 64 ? launch_route<1>(a, s, f, alone, st) : n_experts <= 128 ? launch_route<2>(a, s, f, alone, st)
               : n_experts <= 256 ? launch_route<4>(a, s, f, alone, st) : launch_route<8>(a, s, f, alone, st);
  if (rc != TLLM_OK || alone) return rc;
  hipLaunchKernelGGL(moe_place_kernel, dim3(a.runs), dim3(ROUTE_WAVES * 64), 0, st, a);
  return check_launch("moe_route");
}
