// Rotary positions in every layout: half pairs (i, i + R/2) or interleaved pairs (2i, 2i + 1) of the first R of D values of
// heads [0, n_rot), the rest of the head and the other heads copied; bf16 / fp16 / fp32, fp32 cos / sin tables [S, R/2]:
//   out_a = a cos - b sin,  out_b = b cos + a sin;  the gradient turns back (sin negated).
// Bound by memory: one read and one write of every value. A head is cut into items of W values (pairs of W-value chunks in
// the half layout), and a thread keeps one item position for all the (token, head) units it walks, so the cos / sin of a
// token are loaded once and serve all its heads from registers. Where a part is no multiple of W its last item starts early
// and overlaps the one before: both write the same bytes, and every access stays W wide at any even R and any D. The source
// may have any strides over batch, sequence and heads.
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <algorithm>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 2;  // units in flight per thread
constexpr int kMaxHead = 1000;  // a head's items fit kThreads at any width

template <int N>
__device__ __forceinline__ void load_angles(const float* __restrict__ p, float (&f)[N]) {
  if constexpr (N >= 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const Pack<float, 4> v = load_any<float, 4>(p + j);
#pragma unroll
      for (int q = 0; q < 4; ++q) f[j + q] = v.v[q];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = p[j];
  }
}

struct RopeArgs {
  long sb, ss, sh;  // source strides in elements: batch, sequence, head
  long pb, ps;      // position strides
  long units;       // batch * seq * heads
  int seq, heads, n_rot, D, R, S;
  int n_pair, n_copy;  // items of the rotated part (pairs of chunks in the half layout), items of the rest
  int units_per_block;
  float sign;
};

// W: values of a rotated item, M: of a copied one (16 bytes).
template <typename T, int W, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_any_kernel(const T* __restrict__ src, T* __restrict__ dst,
                                                            const float* __restrict__ cosb, const float* __restrict__ sinb,
                                                            const int64_t* __restrict__ pos, const RopeArgs a) {
  constexpr int NC = INTERLEAVED ? W / 2 : W, M = 16 / sizeof(T);
  const int items = a.n_pair + a.n_copy;
  const int slots = kThreads / items;  // units walked side by side by a block
  const int slot = threadIdx.x / items, item = threadIdx.x - slot * items;
  if (slot >= slots) return;
  const int half = a.R >> 1, rest = a.D - a.R;
  const bool pair = item < a.n_pair;
  const int part = !pair && rest < M ? rest : 0;  // a rest too short for one access
  const int span = INTERLEAVED ? a.R : half;
  const int d0 = pair ? min(item * W, span - W) : part > 0 ? a.R : min(a.R + (item - a.n_pair) * M, a.D - M);
  const int angle0 = INTERLEAVED ? d0 >> 1 : d0;
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
  float c[NC], s[NC];
  for (int u0 = slot; u0 < count; u0 += slots * kUnroll) {
    Pack<T, W> x[kUnroll], z[kUnroll];
    Pack<T, M> y[kUnroll];
    long ub[kUnroll];
    int us[kUnroll], uh[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (u0 + k * slots < count) {
        ub[k] = bi;
        us[k] = si;
        uh[k] = head;
        const T* p = src + bi * a.sb + si * a.ss + head * a.sh + d0;
        if (pair) {
          x[k] = load_any<T, W>(p);
          if (!INTERLEAVED) z[k] = load_any<T, W>(p + half);
        } else {
          y[k] = part > 0 ? load_part<T, M>(p, part) : load_any<T, M>(p);
        }
        advance();
      }
    }
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (u0 + k * slots < count) {
        T* q = dst + (first + u0 + k * slots) * a.D + d0;
        if (pair) {
          if (uh[k] < a.n_rot) {
            if (have_s != us[k] || have_b != ub[k]) {
              have_s = us[k];
              have_b = ub[k];
              const long at = pos != nullptr ? pos[ub[k] * a.pb + us[k] * a.ps] : us[k];
              const bool inside = at >= 0 && at < a.S;  // a position outside the tables is never looked up: NaN
              ACC_CHECK(inside, kChkRopePos);
              const long row = inside ? at * half + angle0 : 0;
              if (inside) {
                load_angles<NC>(cosb + row, c);
                load_angles<NC>(sinb + row, s);
              }
#pragma unroll
              for (int j = 0; j < NC; ++j) {
                c[j] = inside ? c[j] : NAN;
                s[j] = inside ? s[j] * a.sign : NAN;
              }
            }
            if constexpr (INTERLEAVED) {
#pragma unroll
              for (int j = 0; j < NC; ++j) {
                const float p0 = to_f<T>(x[k].v[2 * j]), p1 = to_f<T>(x[k].v[2 * j + 1]);
                x[k].v[2 * j] = from_f<T>(p0 * c[j] - p1 * s[j]);
                x[k].v[2 * j + 1] = from_f<T>(p1 * c[j] + p0 * s[j]);
              }
            } else {
#pragma unroll
              for (int j = 0; j < W; ++j) {
                const float p0 = to_f<T>(x[k].v[j]), p1 = to_f<T>(z[k].v[j]);
                x[k].v[j] = from_f<T>(p0 * c[j] - p1 * s[j]);
                z[k].v[j] = from_f<T>(p1 * c[j] + p0 * s[j]);
              }
            }
          }
          store_any<T, W>(q, x[k]);
          if (!INTERLEAVED) store_any<T, W>(q + half, z[k]);
        } else if (part > 0) {
          store_part<T, M>(q, y[k], part);
        } else {
          store_any<T, M>(q, y[k]);
        }
      }
    }
  }
}

template <typename T, int W>
void launch(const torch::Tensor& src, const torch::Tensor& dst, const torch::Tensor& cos, const torch::Tensor& sin,
            const int64_t* pos, RopeArgs a, bool interleaved, hipStream_t stream) {
  constexpr int M = 16 / sizeof(T);
  const int span = interleaved ? a.R : a.R / 2;
  a.n_pair = (span + W - 1) / W;
  a.n_copy = (a.D - a.R + M - 1) / M;
  TORCH_CHECK(a.n_pair + a.n_copy <= kThreads, "rope: head size");
  const int slots = kThreads / (a.n_pair + a.n_copy);
  // Each block walks a few units of every slot: enough to reuse a token's angles, few enough to fill the chip.
  const long passes = std::min<long>(8, std::max<long>(1, a.units / ((long)slots * 2048)));
  a.units_per_block = (int)(passes * slots);
  const long blocks = (a.units + a.units_per_block - 1) / a.units_per_block;
  TORCH_CHECK(blocks < (1L << 31), "rope: too many heads in one call");
  const T* sp = reinterpret_cast<const T*>(src.data_ptr());
  T* dp = reinterpret_cast<T*>(dst.data_ptr());
  if constexpr (W > 1) {
    if (interleaved) {
      hipLaunchKernelGGL((rope_any_kernel<T, W, true>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, sp, dp,
                         cos.data_ptr<float>(), sin.data_ptr<float>(), pos, a);
      return;
    }
  }
  hipLaunchKernelGGL((rope_any_kernel<T, W, false>), dim3((unsigned)blocks), dim3(kThreads), 0, stream, sp, dp,
                     cos.data_ptr<float>(), sin.data_ptr<float>(), pos, a);
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
    // the widest item that the rotated part holds, up to 16 bytes; the rest of the head follows it
    constexpr int most = 16 / sizeof(scalar);
    const long span = interleaved ? R : R / 2;
    if (most == 8 && span >= 8) launch<scalar, most>(src, out, cos, sin, pp, a, interleaved, stream);
    else if (span >= 4) launch<scalar, 4>(src, out, cos, sin, pp, a, interleaved, stream);
    else if (span >= 2) launch<scalar, 2>(src, out, cos, sin, pp, a, interleaved, stream);
    else launch<scalar, 1>(src, out, cos, sin, pp, a, interleaved, stream);
  });
  return out;
}
