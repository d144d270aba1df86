// Rotary positions in every layout: half pairs (i, i + R/2) or interleaved pairs (2i, 2i + 1) of the first R of D values of
// heads [0, n_rot), the rest of the head and the other heads copied; bf16 / fp16 / fp32, fp32 cos / sin tables [S, R/2]:
//   out_a = a cos - b sin,  out_b = b cos + a sin;  the gradient turns back (sin negated).
// Bound by memory: one read and one write of every value. A head is cut into windows of 16 bytes, the last one moved back to
// end with the head (windows that overlap write the same bytes), so every load and store is whole and all lanes of a wave
// move data, whatever R and D are: out = x cos + partner (+-sin) needs the partners of a window's values beside them, which
// are a swap in registers (interleaved) or a second load of a line that is in flight anyway (half layout: each half is cut
// into windows of its own, the last one moved back to end with the half; a few loads where a half is shorter than a window).
// A thread keeps one window position for all the
// (token, head) units that it walks, so a token's cos / sin are loaded once and serve all its heads from registers. The
// source may have any strides over batch, sequence and heads. 8192 tokens with 192 heads of 96 bf16, 24 turned in halves: 109 us,
// 5.5 TB/s (one unit per thread: 138 us). 8192 x 48 heads of 128, 126 turned in halves: 45 us (82 with windows that hold values
// of both halves and single loads of their partners). Heads with odd halves shorter than a window take such loads still, at
// half the copy's rate.
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <algorithm>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // units in flight per thread
constexpr int kPasses = 4;  // units a thread walks in a long call
constexpr int kMaxHead = 1000;  // a head's windows fit kThreads at any width

// n of N angles (all of them in whole windows); the rest is not looked up
template <int N>
__device__ __forceinline__ void load_angles(const float* __restrict__ p, float (&f)[N], int n) {
  const Pack<float, N> v = n == N ? load_any<float, N>(p) : load_part<float, N>(p, n);
#pragma unroll
  for (int j = 0; j < N; ++j) f[j] = v.get(j);
}

struct RopeArgs {
  long sb, ss, sh;  // source strides in elements: batch, sequence, head
  long pb, ps;      // position strides
  long units;       // batch * seq * heads
  int seq, heads, n_rot, D, R, S;
  int windows;  // of a head
  int units_per_block;
  float sign;
};

// The pairs of a window that starts with one, exchanged.
template <typename T, int M>
__device__ __forceinline__ Pack<T, M> swap_pairs(const Pack<T, M>& x) {
  Pack<T, M> p;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < M; ++j) p.u[j] = x.u[j ^ 1];
  } else {
#pragma unroll
    for (int i = 0; i < M / 2; ++i) p.u[i] = (x.u[i] << 16) | (x.u[i] >> 16);
  }
  return p;
}

// G: a window falls into pieces of G values that turn together, with partners side by side. Half layout: the whole window where
// a half has room for one, else the largest power of two that divides the half and the head; interleaved: the whole window
// where the head is even, else 1.
template <typename T, int G, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_any_kernel(const T* __restrict__ src, T* __restrict__ dst,
                                                            const float* __restrict__ cosb, const float* __restrict__ sinb,
                                                            const int64_t* __restrict__ pos, const RopeArgs a) {
  constexpr int M = 16 / sizeof(T);
  constexpr bool kSwap = INTERLEAVED && G > 1;  // partners within the window
  constexpr bool kHalves = !INTERLEAVED && G == M;  // no window holds values of both halves
  const int windows = a.windows;
  const int slots = kThreads / windows;  // units walked side by side by a block
  const int slot = threadIdx.x / windows, item = threadIdx.x - slot * windows;
  if (slot >= slots) return;
  const int half = a.R >> 1;
  const bool short_head = a.D < M;
  int d0 = short_head ? 0 : min(item * M, a.D - M);
  if constexpr (kHalves) {
    const int per = (half + M - 1) / M;
    if (item < 2 * per) d0 = item < per ? min(item * M, half - M) : half + min((item - per) * M, half - M);
    else d0 = min(a.R + (item - 2 * per) * M, a.D - M);  // may begin in the second half, where the rest is shorter than it
  }
  const bool turns = d0 < a.R;
  const long first = (long)blockIdx.x * a.units_per_block;
  const int count = (int)min((long)a.units_per_block, a.units - first);

  // (batch, position, head) of this thread's next unit, stepped by `slots` without divisions
  const long t0 = (first + slot) / a.heads;
  int head = (int)(first + slot - t0 * a.heads);
  long bi = t0 / a.seq;
  int si = (int)(t0 - bi * a.seq);
  const int step_tok = slots / a.heads, step_head = slots - step_tok * a.heads;
  auto advance = [&]() {
    head += step_head;
    si += step_tok;
    if (head >= a.heads) {
      head -= a.heads;
      ++si;
    }
    while (si >= a.seq) {
      si -= a.seq;
      ++bi;
    }
  };

  long have_b = -1;
  int have_s = -1;
  float c[M], s[M];  // of this window's values; s has the partner's sign
  for (int u0 = slot; u0 < count; u0 += slots * kUnroll) {
    Pack<T, M> x[kUnroll], z[kUnroll];
    long ub[kUnroll];
    int us[kUnroll];
    bool turn[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (u0 + k * slots < count) {
        const T* p = src + bi * a.sb + si * a.ss + head * a.sh + d0;
        x[k] = short_head ? load_part<T, M>(p, a.D) : load_any<T, M>(p);
        turn[k] = turns && head < a.n_rot;
        if constexpr (!kSwap) {
          z[k] = Pack<T, M>::zero();
          if (turn[k]) {
#pragma unroll
            for (int i = 0; i < M; i += G) {
              const int d = d0 + i, other = INTERLEAVED ? d ^ 1 : d < half ? d + half : d - half;
              if (d < a.R) z[k].template put<G>(i, load_any<T, G>(p + (other - d0)));
            }
          }
        }
        ub[k] = bi;
        us[k] = si;
        advance();
      }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (u0 + k * slots < count) {
        if (turn[k]) {
          if (have_s != us[k] || have_b != ub[k]) {
            have_s = us[k];
            have_b = ub[k];
            const long at = pos != nullptr ? pos[ub[k] * a.pb + us[k] * a.ps] : us[k];
            const bool inside = at >= 0 && at < a.S;  // a position outside the tables is never looked up: NaN
            ACC_CHECK(inside, kChkRopePos);
            const long row = inside ? at * half : 0;
            if constexpr (kSwap) {
              float cc[M / 2], ss[M / 2];
              load_angles<M / 2>(cosb + row + d0 / 2, cc, min(M / 2, half - d0 / 2));
              load_angles<M / 2>(sinb + row + d0 / 2, ss, min(M / 2, half - d0 / 2));
#pragma unroll
              for (int j = 0; j < M; ++j) {
                c[j] = cc[j / 2];
                s[j] = j & 1 ? ss[j / 2] : -ss[j / 2];
              }
            } else {
#pragma unroll
              for (int i = 0; i < M; i += G) {
                const int d = d0 + i, angle = INTERLEAVED ? d / 2 : d < half ? d : d - half;
                const bool minus = INTERLEAVED ? (d & 1) == 0 : d < half;
                float cc[G], ss[G];
                const int n = kHalves ? min(G, half - angle) : d < a.R ? G : 0;
                load_angles<G>(cosb + row + angle, cc, n);
                load_angles<G>(sinb + row + angle, ss, n);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                  c[i + j] = cc[j];
                  s[i + j] = minus ? -ss[j] : ss[j];
                }
              }
            }
#pragma unroll
            for (int j = 0; j < M; ++j) {
              c[j] = inside ? c[j] : NAN;
              s[j] *= a.sign;
            }
          }
          if constexpr (kSwap) z[k] = swap_pairs<T, M>(x[k]);
          float o[M];
#pragma unroll
          for (int j = 0; j < M; ++j) {
            const float v = x[k].get(j);
            o[j] = v * c[j] + z[k].get(j) * s[j];
            if (d0 + j >= a.R) o[j] = v;
          }
          x[k] = Pack<T, M>::of(o);
        }
        T* q = dst + (first + u0 + k * slots) * a.D + d0;
        if (short_head) store_part<T, M>(q, x[k], a.D);
        else store_any<T, M>(q, x[k]);
      }
    }
  }
}

template <typename T, int G, bool INTERLEAVED>
void launch(const torch::Tensor& src, const torch::Tensor& dst, const torch::Tensor& cos, const torch::Tensor& sin,
            const int64_t* pos, RopeArgs a, hipStream_t stream) {
  constexpr int M = 16 / sizeof(T);
  const auto cut = [](int n) { return (n + M - 1) / M; };
  a.windows = !INTERLEAVED && G == M ? 2 * cut(a.R / 2) + cut(a.D - a.R) : cut(a.D);
  TORCH_CHECK(a.windows <= kThreads, "rope: head size");
  const int slots = kThreads / a.windows;
  // Each block walks a few units of every slot: enough to reuse a token's angles, few enough to fill the chip.
  const long passes = std::min<long>(kPasses, std::max<long>(1, a.units / ((long)slots * 2048)));
  a.units_per_block = (int)(passes * slots);
  const long blocks = (a.units + a.units_per_block - 1) / a.units_per_block;
  TORCH_CHECK(blocks * kThreads < (1L << 32), "rope: too many heads in one call");
  hipLaunchKernelGGL((rope_any_kernel<T, G, INTERLEAVED>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, reinterpret_cast<const T*>(src.data_ptr()),
                     reinterpret_cast<T*>(dst.data_ptr()), cos.data_ptr<float>(), sin.data_ptr<float>(), pos, a);
}

}  // namespace

ACC_DEBUG_TAKE_FN(acc_dbg_take_rope)

// src [B, S, heads, D] (last dimension contiguous) -> a new contiguous tensor; cos / sin fp32 [positions, R / 2]; pos int64
// [B, S] of any strides, or none for 0 .. S - 1.
torch::Tensor rope_any(torch::Tensor src, torch::Tensor cos, torch::Tensor sin, c10::optional<torch::Tensor> pos, int64_t n_rot,
                       bool interleaved, double sign) {
  TORCH_CHECK(src.is_cuda() && src.dim() == 4, "rope: a 4-D HIP tensor expected");
  const long B = src.size(0), S = src.size(1), Hn = src.size(2), D = src.size(3);
  TORCH_CHECK(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.is_contiguous() && sin.is_contiguous() &&
                  cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.device() == src.device() &&
                  sin.device() == src.device(),
              "rope: cos and sin must be contiguous fp32 [positions, rotary_dim / 2] tensors on the input's device");
  const long R = 2 * cos.size(1);
  TORCH_CHECK(R >= 2 && R <= D && D <= kMaxHead && n_rot >= 0 && n_rot <= Hn, "rope: rotary part, head size or head count");
  TORCH_CHECK(src.stride(3) == 1 || D == 1 || src.numel() == 0, "rope: the last dimension must be contiguous");
  TORCH_CHECK(Hn < (1L << 24) && S < (1L << 31) && cos.size(0) < (1L << 31), "rope: sizes");
  const c10::DeviceGuard guard(src.device());
  auto out = torch::empty({B, S, Hn, D}, src.options());
  if (out.numel() == 0) return out;
  RopeArgs a{};
  a.sb = src.stride(0); a.ss = src.stride(1); a.sh = src.stride(2);
  a.units = B * S * Hn;
  a.seq = (int)S; a.heads = (int)Hn; a.n_rot = (int)n_rot; a.D = (int)D; a.R = (int)R; a.S = (int)cos.size(0);
  a.sign = (float)sign;
  const int64_t* pp = nullptr;
  if (pos.has_value()) {
    TORCH_CHECK(pos->dim() == 2 && pos->size(0) == B && pos->size(1) == S && pos->scalar_type() == at::kLong &&
                    pos->device() == src.device(), "rope: positions must be int64 [B, S] on the input's device");
    a.pb = pos->stride(0); a.ps = pos->stride(1);
    pp = pos->data_ptr<int64_t>();
  } else {
    TORCH_CHECK(S <= cos.size(0), "rope: the sequence is longer than the cos / sin tables");
  }
  auto stream = at::hip::getCurrentHIPStream();
  ACC_FOR_FLOAT_TYPES(src.scalar_type(), "rope", {
    constexpr int M = 16 / sizeof(scalar);
    const auto fits = [&](long g) { return R / 2 % g == 0 && D % g == 0; };
    auto go = [&](auto kind) { kind(src, out, cos, sin, pp, a, stream); };
    if (interleaved) go(D % 2 == 0 ? launch<scalar, M, true> : launch<scalar, 1, true>);
    else if (R / 2 >= M) go(launch<scalar, M, false>);
    else if (M > 4 && fits(4)) go(launch<scalar, (M > 4 ? 4 : 1), false>);
    else if (fits(2)) go(launch<scalar, 2, false>);
    else go(launch<scalar, 1, false>);
  });
  return out;
}
