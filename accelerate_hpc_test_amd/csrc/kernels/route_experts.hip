// Routing to experts: from router logits [T, E] the k experts of each token and their weights, and the logits' gradient.
//   s = softmax(logits) or sigmoid(logits);  key = s + bias
//   with groups: a group's rating is the sum of its two largest keys; only the experts of the best groups stay open
//   experts = the k largest open keys (equal keys: the lower index);  w = s[experts] [/ their sum] * scale
// Backward, with u = dw * scale, h_j = w_j / scale (the shares) and U = sum u_j h_j:
//   renormalised   softmax: dl_j = h_j (u_j - U)              sigmoid: dl_j = h_j (u_j - U) (1 - s_j)
//   as they are    softmax: dl_e = s_e (u_e - sum u_j s_j)    sigmoid: dl_j = u_j s_j (1 - s_j)
// (u_e = 0 for experts that were not chosen; the bias steers the choice alone and has no gradient.)
// Bound by latency: a token's logits are a few hundred values, held by 8 to 64 lanes of one wave from the load to the last
// choice. The order must not hang on a rounding of exp, so keys are computed in 64 bits where they are sums of scores and a
// bias; where they are not (no bias, no groups) the scores' order is the logits' own and is taken from them. Keys become
// unsigned integers of the same order: choosing is an integer maximum, NaN sorts below every number and cannot be chosen
// twice.
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr int kMaxExperts = 1024, kMaxTop = 64, kMaxGroups = 64;
constexpr int kThreads = 256;

struct RouteArgs {
  long rows, stride;
  int E, k, groups, top_groups;
  int softmax, renorm;
  float scale;
};

// Order-preserving keys; 0 is below all of them (taken, or not there), 1 a closed expert, 2 NaN.
__device__ __forceinline__ uint64_t order_key(double d) {
  if (d != d) return 2;
  uint64_t u = __double_as_longlong(d + 0.0);
  return u ^ ((u >> 63) ? ~0ull : 0x8000000000000000ull);
}

template <int L>
__device__ __forceinline__ double lanes_sum(double v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
template <int L>
__device__ __forceinline__ double lanes_max(double v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
  return v;
}

// L lanes hold a token, V experts each: expert v * L + lane.
template <typename T, int L, int V>
__global__ __launch_bounds__(kThreads) void route_fwd_kernel(const T* __restrict__ logits, const float* __restrict__ bias,
                                                             float* __restrict__ weights, int64_t* __restrict__ experts,
                                                             const RouteArgs a) {
  constexpr int PER = kThreads / L;
  __shared__ double rating_of[kThreads / 64][kMaxGroups];
  __shared__ double keys_of[kThreads / 64][L == 64 ? V * 64 : 1];
  const int lane = threadIdx.x % L, wave = threadIdx.x >> 6;
  const long row = (long)blockIdx.x * PER + threadIdx.x / L;
  const bool live = row < a.rows;  // lanes of rows past the end walk along: no lane leaves before the last exchange
  const T* x = logits + (live ? row : 0) * a.stride;
  float f[V];
#pragma unroll
  for (int v = 0; v < V; ++v) f[v] = v * L + lane < a.E ? to_f<T>(x[v * L + lane]) : -INFINITY;

  uint64_t key[V];
  float score[V];
  const bool by_logit = bias == nullptr && a.top_groups == a.groups;
  double hi = -INFINITY, total = 0.0;
  if (a.softmax) {
#pragma unroll
    for (int v = 0; v < V; ++v) hi = (v * L + lane < a.E) ? fmax(hi, (double)f[v]) : hi;
    hi = lanes_max<L>(hi);
  }
  if (by_logit) {
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool there = v * L + lane < a.E;
      score[v] = a.softmax ? expf(f[v] - (float)hi) : 1.f / (1.f + expf(-f[v]));
      if (there) sum += score[v];
      key[v] = there ? order_key((double)f[v]) : 0;
    }
    if (a.softmax) {
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
#pragma unroll
      for (int v = 0; v < V; ++v) score[v] /= sum;
    }
  } else {
    double d[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const bool there = v * L + lane < a.E;
      d[v] = a.softmax ? exp((double)f[v] - hi) : 1.0 / (1.0 + exp(-(double)f[v]));
      if (there) total += d[v];
    }
    if (a.softmax) {
      total = lanes_sum<L>(total);
#pragma unroll
      for (int v = 0; v < V; ++v) d[v] /= total;
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int e = v * L + lane;
      const bool there = e < a.E;
      score[v] = (float)d[v];
      if (there && bias != nullptr) d[v] += (double)bias[e];
      key[v] = there ? order_key(d[v]) : 0;
      if constexpr (L == 64)
        if (there && a.top_groups < a.groups) keys_of[wave][e] = d[v];
    }
    if constexpr (L == 64) {
      if (a.top_groups < a.groups) {
        const int size = a.E / a.groups;
        __syncthreads();
        uint64_t mine = 0;
        if (lane < a.groups) {
          // two largest by their order, summed in 64 bits
          double first = 0.0, second = 0.0;
          uint64_t kf = 0, ks = 0;
          for (int i = 0; i < size; ++i) {
            const double q = keys_of[wave][lane * size + i];
            const uint64_t kq = order_key(q);
            if (kq > kf) {
              second = first;
              ks = kf;
              first = q;
              kf = kq;
            } else if (kq > ks) {
              second = q;
              ks = kq;
            }
          }
          const double rating = size > 1 ? first + second : first;
          rating_of[wave][lane] = rating;
          mine = order_key(rating);
        }
        __syncthreads();
        int above = 0;
        if (lane < a.groups)
          for (int g = 0; g < a.groups; ++g) {
            const uint64_t other = order_key(rating_of[wave][g]);
            above += other > mine || (other == mine && g < lane);
          }
        const uint64_t open = __ballot(lane < a.groups && above < a.top_groups);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const int e = v * L + lane;
          if (e < a.E && !((open >> (e / size)) & 1)) key[v] = 1;
        }
      }
    }
  }

  // k times the best key of the token's lanes; lane j keeps choice j
  float my_score = 0.f, sum = 0.f;
  int my_expert = 0;
  for (int j = 0; j < a.k; ++j) {
    uint64_t best = 0;
    int at = 0;
    float s = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (key[v] > best) {
        best = key[v];
        at = v * L + lane;
        s = score[v];
      }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) {
      const uint64_t ob = __shfl_xor((unsigned long long)best, o, 64);
      const int oa = __shfl_xor(at, o, 64);
      const float os = __shfl_xor(s, o, 64);
      if (ob > best || (ob == best && oa < at)) {
        best = ob;
        at = oa;
        s = os;
      }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * L + lane == at) key[v] = 0;
    sum += s;
    if (lane == j) {
      my_score = s;
      my_expert = at;
    }
  }
  if (live && lane < a.k) {
    // scores that are all zero share nothing: 0, not 0 / 0
    const float share = a.renorm ? my_score / fmaxf(sum, 1.17549435e-38f) : my_score;
    weights[row * a.k + lane] = (sum != sum ? NAN : share) * a.scale;
    experts[row * a.k + lane] = my_expert;
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

// Calls go(lanes of a token, experts per lane). A token with groups takes a whole wave.
template <int N> using Const = std::integral_constant<int, N>;
template <typename F>
void by_experts(int E, bool whole_wave, F go) {
  if (E <= 8 && !whole_wave) go(Const<8>{}, Const<1>{});
  else if (E <= 16 && !whole_wave) go(Const<16>{}, Const<1>{});
  else if (E <= 32 && !whole_wave) go(Const<32>{}, Const<1>{});
  else if (E <= 64) go(Const<64>{}, Const<1>{});
  else if (E <= 128) go(Const<64>{}, Const<2>{});
  else if (E <= 256) go(Const<64>{}, Const<4>{});
  else if (E <= 512) go(Const<64>{}, Const<8>{});
  else go(Const<64>{}, Const<16>{});
}

RouteArgs args_of(const torch::Tensor& logits, int64_t k, bool softmax, int64_t groups, int64_t top_groups, bool renorm, double scale) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1 || logits.numel() == 0),
              "route_experts: logits must be a 2-D HIP tensor with contiguous rows");
  const long E = logits.size(1);
  TORCH_CHECK(E >= 1 && E <= kMaxExperts, "route_experts: 1 to ", kMaxExperts, " experts expected");
  TORCH_CHECK(groups >= 1 && groups <= kMaxGroups && E % groups == 0 && top_groups >= 1 && top_groups <= groups,
              "route_experts: groups must divide the experts, at most ", kMaxGroups, " of them");
  TORCH_CHECK(k >= 1 && k <= kMaxTop && k <= E / groups * top_groups, "route_experts: more choices than open experts, or than ", kMaxTop);
  TORCH_CHECK(logits.size(0) < (1L << 31), "route_experts: too many rows");
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
    by_experts(a.E, a.top_groups < a.groups, [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value;
      constexpr int per = kThreads / L;
      hipLaunchKernelGGL((route_fwd_kernel<scalar, L, V>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream,
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
    by_experts(a.E, false, [&](auto l, auto v) {
      constexpr int L = decltype(l)::value, V = decltype(v)::value;
      constexpr int per = kThreads / L;
      hipLaunchKernelGGL((route_bwd_kernel<scalar, L, V>), dim3((unsigned)((a.rows + per - 1) / per)), dim3(kThreads), 0, stream,
                         reinterpret_cast<const scalar*>(logits.data_ptr()), weights.data_ptr<float>(), experts.data_ptr<int64_t>(),
                         dw.data_ptr<float>(), reinterpret_cast<scalar*>(out.data_ptr()), a);
    });
  });
  return out;
}
