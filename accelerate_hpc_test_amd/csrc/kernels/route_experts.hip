// Routing to experts: from router logits [T, E] the k experts of each token and their weights, and the logits' gradient.
//   s = softmax(logits) or sigmoid(logits);  key = s + bias
//   with groups: a group's rating is the sum of its two largest keys; only the experts of the best groups stay open
//   experts = the k largest open keys (equal keys: the lower index);  w = s[experts] [/ their sum] * scale
// Backward, with u = dw * scale, h_j = w_j / scale (the shares) and U = sum u_j h_j:
//   renormalised   softmax: dl_j = h_j (u_j - U)              sigmoid: dl_j = h_j (u_j - U) (1 - s_j)
//   as they are    softmax: dl_e = s_e (u_e - sum u_j s_j)    sigmoid: dl_j = u_j s_j (1 - s_j)
// (u_e = 0 for experts that were not chosen; the bias steers the choice alone and has no gradient.)
// What bounds the kernel is how many instructions a choice takes, not the bytes. A wave chooses for one token, each lane holding
// 1 to 16 neighbouring experts:
//   * keys are order-preserving unsigned integers; NaN sorts as -inf, a closed expert is 0;
//   * a bisection over key values, counting by ballots, finds a bound that a few more than k keys reach (a handful of steps);
//   * those are compacted in the order of their experts, and each counts the ones before it: that is its rank.
// 16384 tokens with 256 experts in 8 groups, k = 8: 20.3 us (k rounds of a maximum over the lanes: 28.9 us; keys in 64 bits
// throughout: 32.7 us), 64 tokens: 5.1 us. The order must not hang on a rounding of exp: where keys are sums of scores and a bias,
// a wave chooses by keys in 32 bits, and does it again in 64 where two neighbours of the order, or the last open and the first
// closed group, lie within the rounding errors of 32 (6 tokens in 10000 with distinct logits). Where keys are scores alone (no
// bias, no closed groups) their order is the logits' own, and exact.
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <type_traits>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr int kMaxExperts = 1024, kMaxTop = 64, kMaxGroups = 64;
constexpr int kThreads = 256;
constexpr float kNoScore = -103.972077f;  // ln 2^-150: the sigmoid of a logit below it is 0 in 32 bits

struct RouteArgs {
  long rows, stride;
  int E, k, groups, top_groups;
  int softmax, renorm;
  float scale;
};

// Order-preserving keys above 0.
__device__ __forceinline__ uint32_t order_key(float f) {
  if (f != f) f = -INFINITY;
  const uint32_t u = __float_as_uint(f + 0.f);
  return u ^ ((u & 0x80000000u) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t order_key(double d) {
  if (d != d) d = -INFINITY;
  const uint64_t u = __double_as_longlong(d + 0.0);
  return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double key_value(uint64_t k) {
  return __longlong_as_double(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull));
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu)); }

__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896340736f); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }
__device__ __forceinline__ float sigmoid_of(float x) { return __builtin_amdgcn_rcpf(1.f + exp_of(-x)); }
__device__ __forceinline__ double sigmoid_of(double x) { return 1.0 / (1.0 + exp(-x)); }

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ float wave_sum_of(float v) { return wave_reduce<OpSum>(v); }
__device__ __forceinline__ double wave_sum_of(double v) { return wave_sum64(v); }

// Values at .. at + V - 1 of a row of n (`fill` past its end). `full`: the row has a value for every lane.
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* __restrict__ row, int at, int n, bool full, float fill, float (&f)[V]) {
  constexpr int C = V * sizeof(T) <= 16 ? V : 16 / sizeof(T);
  if (full) {
#pragma unroll
    for (int i = 0; i < V; i += C) {
      const Pack<T, C> x = load_any<T, C>(row + at + i);
#pragma unroll
      for (int v = 0; v < C; ++v) f[i + v] = x.get(v);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = to_f<T>(row[min(at + v, n - 1)]);
#pragma unroll
    for (int v = 0; v < V; ++v) f[v] = at + v < n ? f[v] : fill;
  }
}

// The scores of f[V], sigmoid, or softmax over the wave; 0 where f is -inf for want of an expert.
template <int V, typename F>
__device__ __forceinline__ void scores_of(const float (&f)[V], bool softmax, F (&s)[V]) {
  if (softmax) {
    float hi = f[0];  // -inf where there is no expert
#pragma unroll
    for (int v = 1; v < V; ++v) hi = fmaxf(hi, f[v]);
    hi = wave_reduce<OpMax>(hi);
    F sum = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      s[v] = exp_of((F)f[v] - (F)hi);
      sum += s[v];
    }
    const F inv = (F)1 / wave_sum_of(sum);
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] *= inv;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = sigmoid_of((F)f[v]);
  }
}

// What a 32-bit key (a score and a bias) may be off: `noise` for its score, and one rounding of the sum. A sigmoid is within
// 2^-22 (the exponent's rounding moves s by at most s (1 - s) |x| 2^-23 < 2^-25; exp, sum and reciprocal by a step of s each),
// a softmax within 2^-19 of itself (exponent and exp, a sum of up to 1024 by lanes of 16, a reciprocal and a product: 30 half
// steps where it matters: a score e^-d has d 2^-24 e^-d < 2^-25).
__device__ __forceinline__ float key_margin(float key, float noise) { return noise + fabsf(key) * 0x1p-23f; }

// This wave's writes to its shared memory are there for its other lanes.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's shared memory.
template <int V>
struct Scratch {
  uint64_t keys[64 * V];  // every expert's, for the ratings; then the candidates'
  int ids[64 * V];        // the candidates' experts
  uint64_t sorted[kMaxTop + 1];
  int chosen[kMaxTop + 1];
};

// The two best values of a group's lanes, an aligned power of two of them.
template <typename F>
__device__ __forceinline__ void merge_two(F& first, F& second, F of, F os) {
  const F low = of > first ? first : of, high = second > os ? second : os;
  first = of > first ? of : first;
  second = low > high ? low : high;
}
__device__ __forceinline__ void best_two(float& first, float& second, int lanes) {
  auto step = [&](auto move) { merge_two(first, second, move(first), move(second)); };
  if (lanes >= 2) step([](float v) { return __uint_as_float(dpp_move<0xB1>(__float_as_uint(v))); });
  if (lanes >= 4) step([](float v) { return __uint_as_float(dpp_move<0x4E>(__float_as_uint(v))); });
  if (lanes >= 8) step([](float v) { return __uint_as_float(dpp_move<0x141>(__float_as_uint(v))); });
  if (lanes >= 16) step([](float v) { return __uint_as_float(dpp_move<0x140>(__float_as_uint(v))); });
  if (lanes >= 32) step([](float v) { return __shfl_xor(v, 16, 64); });
}
__device__ __forceinline__ void best_two(double& first, double& second, int lanes) {
  for (int o = 1; o < lanes; o <<= 1) merge_two(first, second, __shfl_xor(first, o, 64), __shfl_xor(second, o, 64));
}

__device__ __forceinline__ float lane_value(float v, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane)); }
__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t u = __double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(u >> 32), lane);
  return __longlong_as_double(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ uint32_t high_of(uint32_t k) { return k; }
__device__ __forceinline__ uint32_t high_of(uint64_t k) { return (uint32_t)(k >> 32); }

// Lane l holds experts l * V .. l * V + V - 1 of a token. Leaves the k experts that keys of type F choose in `sh.chosen`, in order.
// False (F = float): two keys are too close to call. `by_logit`: the logits are the keys, and exact.
template <int V, typename F>
__device__ __forceinline__ bool choose(const float (&f)[V], const float* __restrict__ bias, Scratch<V>& sh, bool by_logit,
                                       const RouteArgs& a) {
  constexpr bool kWide = sizeof(F) == 8;
  using Key = typename std::conditional<kWide, uint64_t, uint32_t>::type;
  const int lane = threadIdx.x & 63, e0 = lane * V;
  Key* const keys = reinterpret_cast<Key*>(sh.keys);
  Key* const sorted = reinterpret_cast<Key*>(sh.sorted);
  Key key[V];
  float noise = 0x1p-22f;
  {
    F d[V];
    if (by_logit) {
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] = f[v];
    } else {
      scores_of<V, F>(f, a.softmax, d);
      if (!kWide && a.softmax) {
        float most = (float)d[0];
#pragma unroll
        for (int v = 1; v < V; ++v) most = fmaxf(most, (float)d[v]);
        noise = wave_reduce<OpMax>(most) * 0x1p-19f;
      }
      if (bias != nullptr) {
        float b[V];
        load_values<float, V>(bias, e0, a.E, a.E == 64 * V, 0.f, b);
#pragma unroll
        for (int v = 0; v < V; ++v) d[v] += (F)b[v];
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) key[v] = e0 + v < a.E ? order_key(d[v]) : (Key)0;
  }
  if (a.top_groups < a.groups) {
    // Ratings: the lanes share out over the groups, a power of two for each.
    const int size = a.E / a.groups, per = 64 >> (32 - __clz(a.groups - 1)), g = lane / per;
#pragma unroll
    for (int v = 0; v < V; ++v) keys[e0 + v] = key[v];
    wave_sync();
    F first = (F)-INFINITY, second = (F)-INFINITY;
    if (g < a.groups)
      for (int q = lane & (per - 1); q < size; q += per) merge_two(first, second, key_value(keys[g * size + q]), (F)-INFINITY);
    best_two(first, second, per);
    const F rating = size > 1 ? first + second : first;
    int above = 0;
    for (int i = 0; i < a.groups; ++i) {
      const F other = lane_value(rating, i * per);
      above += other > rating || (other == rating && i < g);
    }
    const bool in = g < a.groups && above < a.top_groups;
    if constexpr (!kWide) {
      // A rating is off by its two keys' errors, each of the key's own size (large keys of opposite signs make a small rating), and by
      // one rounding. An infinite one is exact.
      float off = size > 1 ? key_margin(first, noise) + key_margin(second, noise) + fabsf(rating) * 0x1p-23f : key_margin(first, noise);
      off = wave_reduce<OpMax>(g < a.groups && fabsf(rating) < INFINITY ? off : 0.f);
      const float worst = -wave_reduce<OpMax>(in ? -rating : -INFINITY), best = wave_reduce<OpMax>(g < a.groups && !in ? rating : -INFINITY);
      if (!(worst - best > 2.f * off)) return false;
    }
    const uint64_t open = __ballot(in);
    const float inv = 1.f / (float)size;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int eg = (int)(((float)(e0 + v) + 0.5f) * inv);  // exact: E <= 1024
      if (!((open >> (eg * per & 63)) & 1)) key[v] = 0;
    }
    wave_sync();  // the keys are read: the candidates' may take their place
  }

  // A bound that at least `need` keys reach (one more than k shows how far the first one left out is), and few exceed it.
  uint32_t hi_key = 0;
  int open_count = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    hi_key = high_of(key[v]) > hi_key ? high_of(key[v]) : hi_key;
    open_count += __popcll(__ballot(key[v] != 0));
  }
  const int need = kWide || by_logit || a.k == open_count ? a.k : a.k + 1;
  // the least of the lanes' best keys is reached by as many keys as there are lanes that have one
  const uint64_t holders = __ballot(hi_key != 0);
  uint32_t low = 1;  // reached by all
  if (__popcll(holders) >= need) low = ~lanes_max_u32<64>(hi_key != 0 ? ~hi_key : 0);
  uint32_t high = lanes_max_u32<64>(hi_key);  // the bound is at most this
  low = __builtin_amdgcn_readfirstlane(low);
  high = __builtin_amdgcn_readfirstlane(high);
  while (low < high) {
    const uint32_t mid = low + (high - low + 1) / 2;
    int reach = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) reach += __popcll(__ballot(high_of(key[v]) >= mid));
    if (reach >= need) {
      low = mid;
      if (reach <= need + 8) break;
    } else {
      high = mid - 1;
    }
  }

  // The candidates, in the order of their experts.
  int at = 0, n = 0;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const uint64_t m = __ballot(high_of(key[v]) >= low);
    n += __popcll(m);
    at = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, at));
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (high_of(key[v]) >= low) {
      keys[at] = key[v];
      sh.ids[at++] = e0 + v;
    }
  wave_sync();
  for (int i = lane; i < n; i += 64) {
    const Key mine = keys[i];
    int rank = 0;
#pragma unroll 4
    for (int q = 0; q < n; ++q) {
      const Key other = keys[q];
      rank += other > mine || (other == mine && q < i);
    }
    if (rank < need) {
      sorted[rank] = mine;
      sh.chosen[rank] = sh.ids[i];
    }
  }
  wave_sync();
  if constexpr (!kWide) {
    if (!by_logit) {
      bool close = false;
      if (lane + 1 < need) {
        const float one = key_value(sorted[lane]), next = key_value(sorted[lane + 1]);
        close = !(one - next > key_margin(one, noise) + key_margin(next, noise));
      }
      if (__any(close)) return false;
    }
  }
  return true;
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void route_fwd_kernel(const T* __restrict__ logits, const float* __restrict__ bias,
                                                             float* __restrict__ weights, int64_t* __restrict__ experts,
                                                             const RouteArgs a) {
  __shared__ Scratch<V> scratch[kThreads / 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const long row = (long)blockIdx.x * (kThreads / 64) + wave;
  if (row >= a.rows) return;  // the whole wave: nothing below waits for the block
  const T* x = logits + row * a.stride;
  Scratch<V>& sh = scratch[wave];
  float f[V];
  load_values<T, V>(x, lane * V, a.E, a.E == 64 * V, -INFINITY, f);
  const bool by_logit = bias == nullptr && a.top_groups == a.groups;
  if (!choose<V, float>(f, bias, sh, by_logit, a)) {
    wave_sync();
    choose<V, double>(f, bias, sh, false, a);
  }

  // The weights, a choice in each lane. Shares are of the chosen alone, formed against the largest logit among them (`top`): that may
  // lie any distance below the row's (`hi`), where a bias or closed groups keep others out. Else the first choice has both.
  const int id = lane < a.k ? sh.chosen[lane] : 0;
  const float v = to_f<T>(x[id]);
  float top = lane_value(v, 0);
  if (a.renorm && !by_logit) top = wave_reduce<OpMax>(lane < a.k ? v : -INFINITY);
  float w;
  if (a.softmax) {
    float hi = top;
    if (!by_logit) {
      hi = f[0];
#pragma unroll
      for (int i = 1; i < V; ++i) hi = fmaxf(hi, f[i]);
      hi = wave_reduce<OpMax>(hi);
    }
    float all = 0.f;  // also: NaN where a logit is NaN or +inf, or all are -inf
#pragma unroll
    for (int i = 0; i < V; ++i) all += exp_of(f[i] - hi);
    all = wave_reduce<OpSum>(all);
    // chosen scores that are all zero share nothing: 0, not 0 / 0
    const bool none = a.renorm && top == -INFINITY;
    w = lane < a.k && !none ? exp_of(v - (a.renorm ? top : hi)) : 0.f;
    const float sum = a.renorm ? wave_reduce<OpSum>(w) : all;
    w = all == all ? (none ? 0.f : w / sum) : NAN;
  } else if (a.renorm) {
    // s_j over the best score, up to a factor that all share: e^(v - min(top, 0)) / (1 + e^v)
    const bool none = top < kNoScore && !__any(lane < a.k && v != v);
    w = lane < a.k && !none ? (v > 0.f ? 1.f : exp_of(v - fminf(top, 0.f))) * __builtin_amdgcn_rcpf(1.f + exp_of(-fabsf(v))) : 0.f;
    const float sum = wave_reduce<OpSum>(w);
    w = none ? 0.f : w / sum;
  } else {
    w = lane < a.k ? sigmoid_of(v) : 0.f;
  }
  if (lane < a.k) {
    weights[row * a.k + lane] = w * a.scale;
    experts[row * a.k + lane] = id;
  }
}

template <typename T, int L, int V>
__global__ __launch_bounds__(kThreads) void route_bwd_kernel(const T* __restrict__ logits, const float* __restrict__ weights,
                                                             const int64_t* __restrict__ experts, const float* __restrict__ dw,
                                                             T* __restrict__ out, const RouteArgs a) {
  constexpr int PER = kThreads / L;
  const int lane = threadIdx.x % L, base = (threadIdx.x & 63) - lane;
  const long row = (long)blockIdx.x * PER + threadIdx.x / L;
  const bool live = row < a.rows;
  const T* x = logits + (live ? row : 0) * a.stride;
  const bool chosen = live && lane < a.k;
  const int id = chosen ? (int)experts[row * a.k + lane] : -1;
  const float u = chosen ? dw[row * a.k + lane] * a.scale : 0.f;
  float score[V];
  float h = 0.f;  // the chosen expert's share, or its score where shares are not taken
  if (a.softmax && !a.renorm) {
    float hi = -INFINITY, sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      score[v] = v * L + lane < a.E ? to_f<T>(x[v * L + lane]) : -INFINITY;
      hi = fmaxf(hi, score[v]);
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor(hi, o, 64));
#pragma unroll
    for (int v = 0; v < V; ++v) {
      score[v] = expf(score[v] - hi);
      sum += score[v];
    }
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int v = 0; v < V; ++v) score[v] /= sum;
    if (chosen) h = expf(to_f<T>(x[id]) - hi) / sum;
  } else if (a.renorm) {
    h = chosen ? weights[row * a.k + lane] / a.scale : 0.f;
  } else {
    h = chosen ? 1.f / (1.f + expf(-to_f<T>(x[id]))) : 0.f;
  }
  float all = u * h;
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) all += __shfl_xor(all, o, 64);
  float value = 0.f;  // the chosen expert's gradient
  if (chosen) {
    value = a.renorm ? h * (u - all) : a.softmax ? h * (u - all) : u * h;
    if (!a.softmax) value *= 1.f / (1.f + expf(to_f<T>(x[id])));  // 1 - s, without cancellation
  }
  float g[V];
#pragma unroll
  for (int v = 0; v < V; ++v) g[v] = a.softmax && !a.renorm ? -score[v] * all : 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int e = __shfl(id, base + j, 64);
    const float q = __shfl(value, base + j, 64);
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane == e) g[v] = q;
  }
  if (!live) return;
  T* o = out + row * a.E;
#pragma unroll
  for (int v = 0; v < V; ++v)
    if (v * L + lane < a.E) o[v * L + lane] = from_f<T>(g[v]);
}

template <int N> using Const = std::integral_constant<int, N>;
// Calls go(experts per lane of a wave).
template <typename F>
void by_experts(int E, F go) {
  if (E <= 64) go(Const<1>{});
  else if (E <= 128) go(Const<2>{});
  else if (E <= 256) go(Const<4>{});
  else if (E <= 512) go(Const<8>{});
  else go(Const<16>{});
}

RouteArgs args_of(const torch::Tensor& logits, int64_t k, bool softmax, int64_t groups, int64_t top_groups, bool renorm, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1 || logits.numel() == 0),
              "route_experts: logits must be a 2-D HIP tensor with contiguous rows");
  const long E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= kMaxExperts, "route_experts: 1 to ", kMaxExperts, " experts expected");
  TORCH_CHECK(groups >= 1 && groups <= kMaxGroups && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
              "route_experts: groups must divide the experts, at most ", kMaxGroups, " of them");
  TORCH_CHECK(k >= 1 && k <= kMaxTop && k <= E / groups * top_groups, "route_experts: more choices than open experts, or than ", kMaxTop);
  // a wave for each row, whole blocks: fewer than 2^32 threads to a launch (the backward has at most as many)
  constexpr long per = kThreads / 64;
  TORCH_CHECK((logits.size(0) + per - 1) / per * kThreads < (1L << 32), "route_experts: too many rows in one call");
  return RouteArgs{logits.size(0), logits.stride(0), (int)E, (int)k, (int)groups, (int)top_groups, softmax, renorm, (float)scale};
}

}  // namespace

ACC_DEBUG_TAKE_FN(acc_dbg_take_route_experts)

// weights fp32 [T, k], experts int64 [T, k] in falling order of their keys.
std::vector<torch::Tensor> route_experts_fwd(torch::Tensor logits, int64_t k, bool softmax, c10::optional<torch::Tensor> bias,
                                             int64_t groups, int64_t top_groups, bool renorm, double scale) {
  const RouteArgs a = args_of(logits, k, softmax, groups, top_groups, renorm, scale);
  TORCH_CHECK(!bias.has_value() || (bias->dim() == 1 && bias->size(0) == a.E && bias->scalar_type() == at::kFloat &&
                                    bias->is_contiguous() && bias->device() == logits.device()),
              "route_experts: bias must be a contiguous fp32 [experts] tensor on the logits' device");
  const c10::DeviceGuard guard(logits.device());
  auto w = torch::empty({a.rows, k}, logits.options().dtype(torch::kFloat32));
  auto ids = torch::empty({a.rows, k}, logits.options().dtype(torch::kInt64));
  if (a.rows == 0) return {w, ids};
  auto stream = at::hip::getCurrentHIPStream();
  ACC_FOR_FLOAT_TYPES(logits.scalar_type(), "route_experts", {
    by_experts(a.E, [&](auto v) {
      constexpr int V = decltype(v)::value, per = kThreads / 64;
      hipLaunchKernelGGL((route_fwd_kernel<scalar, V>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream,
                         reinterpret_cast<const scalar*>(logits.data_ptr()), bias.has_value() ? bias->data_ptr<float>() : nullptr,
                         w.data_ptr<float>(), ids.data_ptr<int64_t>(), a);
    });
  });
  return {w, ids};
}

torch::Tensor route_experts_bwd(torch::Tensor logits, torch::Tensor weights, torch::Tensor experts, torch::Tensor dw, bool softmax,
                                bool renorm, double scale) {
  const RouteArgs a = args_of(logits, dw.size(-1), softmax, 1, 1, renorm, scale);
  for (const auto& t : {weights, dw})
    TORCH_CHECK(t.dim() == 2 && t.size(0) == a.rows && t.size(1) == a.k && t.scalar_type() == at::kFloat && t.is_contiguous() &&
                    t.device() == logits.device(), "route_experts: weights and their gradient must be fp32 [rows, k]");
  TORCH_CHECK(experts.sizes() == dw.sizes() && experts.scalar_type() == at::kLong && experts.is_contiguous(), "route_experts: experts");
  const c10::DeviceGuard guard(logits.device());
  auto out = torch::empty({a.rows, (long)a.E}, logits.options());
  if (a.rows == 0) return out;
  auto stream = at::hip::getCurrentHIPStream();
  ACC_FOR_FLOAT_TYPES(logits.scalar_type(), "route_experts", {
    auto go = [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value, per = kThreads / L;
      hipLaunchKernelGGL((route_bwd_kernel<scalar, L, V>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream,
                         reinterpret_cast<const scalar*>(logits.data_ptr()), weights.data_ptr<float>(), experts.data_ptr<int64_t>(),
                         dw.data_ptr<float>(), reinterpret_cast<scalar*>(out.data_ptr()), a);
    };
    // up to 32 experts several tokens share a wave; a token's lanes hold a choice each, so they are as many as the experts
    if (a.E <= 8) go(Const<8>{}, Const<1>{});
    else if (a.E <= 16) go(Const<16>{}, Const<1>{});
    else if (a.E <= 32) go(Const<32>{}, Const<1>{});
    else by_experts(a.E, [&](auto v) { go(Const<64>{}, v); });
  });
  return out;
}
