// Log-probabilities of given tokens, the entropy of their distributions and the k best alternatives, over logits [rows, V]
// (bf16 / fp16 / fp32, all sums in fp32), and the gradient of all three. With b the row's largest logit and
// t_i = (x_i - b) log2(e) / temperature, one pass keeps the running b, S = sum 2^t and U = sum t 2^t of each row:
//   log p_i = (x_i - b) / temperature - ln S,   H = ln S - ln 2 U / S
//   dlogits_i = (1/T) [ -p_i (G + dH (log p_i + H)) + sum of the gradients of the outputs that name i ],
//   G = the sum of the row's log-probability gradients.
// Bound by memory: the forward reads the logits once, the backward reads them once and writes the gradient once. A block takes
// a row; few rows are cut into slices for several blocks, and a second small kernel joins their sums and best keys. An -inf
// logit has p = 0 and adds nothing. A row whose token is `ignore` gives 0, 0, 0 and -1, and a zero gradient, whatever it holds. A row
// without a distribution (NaN, +inf, all -inf) gives NaN and alternatives -1; a token outside [0, V) gives a NaN constant, whose
// gradient is dropped.
// 4096 x 128256 bf16: 224 us forward (4.7 TB/s), 380 us backward (5.5 TB/s); 16 rows with 20 alternatives: 9.5 us and 4.3 us
// for the join (whole rows: 19.9 us).
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <algorithm>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr float kLn2 = 0.693147180559945309417f;
constexpr float kFar = -256.f;  // stands for all exponents below it where they are multiplied with 2^t, which is 0 there: finite, and
                                // small enough for a product with any gradient
constexpr int kMaxTop = 64;
constexpr int kList = 2048;  // candidates of a row kept in shared memory
constexpr int kMaxParts = 8;  // slices of a row
constexpr long kBlocks = 512, kSlice = 32768;
constexpr int kJoinThreads = kMaxParts * kMaxTop;  // a thread for every key of a row's slices
constexpr int kBwdThreads = 256, kBwdUnroll = 4;

// Keys ordered as (value, then lower index): the larger key is the better alternative. Equal values, -0 and +0 among them,
// differ in the index alone, so all keys of a row are distinct.
__device__ __forceinline__ uint64_t key_of(float x, int index) {
  uint32_t u = __float_as_uint(x + 0.f);
  u ^= (u & 0x80000000u) ? 0xffffffffu : 0x80000000u;
  return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  uint32_t u = (uint32_t)(k >> 32);
  u ^= (u & 0x80000000u) ? 0x80000000u : 0xffffffffu;
  return __uint_as_float(u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

__device__ __forceinline__ uint64_t key_max(uint64_t a, uint64_t b) { return a > b ? a : b; }

__device__ __forceinline__ float exp2_of(float t) { return __builtin_amdgcn_exp2f(t); }

struct Sums { float b, s, u; };  // of a part of a row: its largest logit, sum 2^t and sum t 2^t against it

// `x` as if its sums were against `b`, at least as large
__device__ __forceinline__ Sums against(Sums x, float b, float scale) {
  if (x.b > -INFINITY && b < INFINITY) {
    const float d = fmaxf((x.b - b) * scale, kFar), f = exp2_of(d);
    x.u = (x.u + d * x.s) * f;
    x.s *= f;
  }
  return x;
}

// 1 / temperature; `scale` is it times log2(e) rounded to 32 bits, `slack` the relative error of that. All exponents of a row
// are off by the same share, so S is off by slack ln 2 U to first order, and corrected by it.
struct Temper {
  double inv_t;
  float scale, slack;
};

struct RowOut {
  float *lp, *ent, *top_lp, *stats;
  int64_t* top_id;
};

// The row's log-probability, entropy and, for the backward, b, 1 / S, ln S and the entropy. Returns ln S, NaN for a row without
// a distribution.
template <typename T>
__device__ __forceinline__ float finish_row(const Sums& r, const T* __restrict__ x, int64_t tok, long row, int V, const Temper& w,
                                            const RowOut& out, bool write) {
  const bool sound = r.s > 0.f && r.s < INFINITY;  // false for NaN too
  const float sum = sound ? fmaf(w.slack * kLn2, r.u, r.s) : NAN, ln_s = logf(sum);
  if (write) {
    const bool named = tok >= 0 && tok < V;
    ACC_CHECK(named, kChkXentLabel);
    const float ent = sound ? logf(r.s) - kLn2 * (r.u / r.s) : NAN;
    out.lp[row] = named ? (float)((double)(to_f<T>(x[named ? tok : 0]) - r.b) * w.inv_t) - ln_s : NAN;
    out.ent[row] = ent;
    if (out.stats != nullptr) *reinterpret_cast<float4*>(out.stats + row * 4) = make_float4(r.b, 1.f / sum, ln_s, ent);
  }
  return ln_s;
}

__device__ __forceinline__ void put_alternative(const RowOut& out, long at, uint64_t key, const Temper& w, float b, float ln_s) {
  out.top_lp[at] = (float)((double)(key_value(key) - b) * w.inv_t) - ln_s;
  out.top_id[at] = key_index(key);
}

template <int NT>
__device__ __forceinline__ void put_no_row(const RowOut& out, long row, int K, float value) {
  for (int j = threadIdx.x; j < K; j += NT) {
    out.top_lp[row * K + j] = value;
    out.top_id[row * K + j] = -1;
  }
}

// blockIdx.x: row * parts + the slice of it. With one slice the block writes the row's outputs, else its sums and its K best
// keys (falling, 0 where the slice has fewer elements) for token_logprobs_join_kernel.
template <typename T, int NT, int UNROLL>
__global__ __launch_bounds__(NT) void token_logprobs_fwd_kernel(const T* __restrict__ logits, long stride,
                                                                const int64_t* __restrict__ tokens, const RowOut out,
                                                                Sums* __restrict__ part_sums, uint64_t* __restrict__ part_keys,
                                                                int parts, int V, int K, const Temper w, int64_t ignore) {
  constexpr int VEC = 16 / sizeof(T), GROUPS = NT / 4;
  __shared__ float slots[3][16];
  __shared__ uint64_t group_key[GROUPS];
  __shared__ uint64_t list[kList];
  __shared__ uint64_t threshold, round_key[NT / 64];
  __shared__ int n_list, n_threads, threads_list[NT];
  const long row = parts == 1 ? blockIdx.x : blockIdx.x / parts;
  const int part = parts == 1 ? 0 : blockIdx.x - (int)row * parts, tid = threadIdx.x;
  int64_t tok = 0;
  if (parts == 1) {  // slices do not wait for their row's token: the join writes a row that is ignored
    tok = tokens[row];
    if (tok == ignore) {  // uniform over the block
      if (tid == 0) out.lp[row] = out.ent[row] = 0.f;
      put_no_row<NT>(out, row, K, 0.f);
      return;
    }
  }
  const T* x = logits + row * stride;
  const float scale = w.scale;
  const int nfull = V / VEC, tail = V % VEC, chunks = nfull + (tail > 0);
  const int span = (chunks + parts - 1) / parts, c_lo = min(part * span, chunks), c_hi = min(c_lo + span, chunks);
  const int c_full = min(c_hi, nfull);

  // one pass: running sums per thread, and the chunk that holds the thread's maximum
  Sums r{-INFINITY, 0.f, 0.f};
  // Sums of a turn's UNROLL chunks, against the same b, added to the thread's at its end: one by one, hundreds of terms below half a step
  // of a sum that holds the largest would be lost (S low by 3e-7 in rows of 50257 with few likely tokens, by 2e-5 at worst).
  float turn_s = 0.f, turn_u = 0.f;
  auto end_turn = [&]() {
    r.s += turn_s;
    r.u += turn_u;
    turn_s = turn_u = 0.f;
  };
  int best = c_lo + tid;  // nothing above -inf: the first chunk stands for the thread
  Pack<T, VEC> best_chunk;
  auto take = [&](const float (&f)[VEC], const Pack<T, VEC>& p, int c) {
    float hi = f[0];
#pragma unroll
    for (int j = 1; j < VEC; ++j) hi = fmaxf(hi, f[j]);
    if (hi > r.b) {
      const Sums turn = against(Sums{r.b, turn_s, turn_u}, hi, scale);
      turn_s = turn.s;
      turn_u = turn.u;
      r = against(r, hi, scale);
      r.b = hi;
      best = c;
      best_chunk = p;
    }
    const float b = r.b > -INFINITY ? r.b : 0.f;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float t = (f[j] - b) * scale, e = exp2_of(t);
      turn_s += e;
      turn_u = fmaf(fmaxf(t, kFar), e, turn_u);
    }
  };
  for (int c = c_lo + tid; c < c_full; c += UNROLL * NT) {
    Pack<T, VEC> p[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) p[u] = load_any<T, VEC>(x + (long)min(c + u * NT, c_full - 1) * VEC);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      float f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) f[j] = p[u].get(j);
      if (c + u * NT < c_full) take(f, p[u], c + u * NT);
    }
    end_turn();
  }
  if (c_hi > c_full && tid == (nfull - c_lo) % NT) {  // the row's last, smaller chunk: the thread whose turn it is
    const Pack<T, VEC> p = load_tail<T, VEC>(x + (long)nfull * VEC, tail, nfull * VEC);
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = j < tail ? p.get(j) : -INFINITY;
    take(f, p, nfull);
    end_turn();
  }
  const float m = r.b, b = row_reduce<OpMax, NT>(m, slots[0]);
  r = against(r, b, scale);
  r.b = b;
  r.s = row_reduce<OpSum, NT>(r.s, slots[1]);
  r.u = row_reduce<OpSum, NT>(r.u, slots[2]);
  float ln_s = 0.f;
  uint64_t* keys_out = nullptr;
  if (parts == 1) {
    ln_s = finish_row<T>(r, x, tok, row, V, w, out, tid == 0);
    if (K == 0) return;
    if (ln_s != ln_s) {
      put_no_row<NT>(out, row, K, NAN);
      return;
    }
  } else {
    if (tid == 0) part_sums[blockIdx.x] = r;
    if (K == 0) return;
    keys_out = part_keys + (long)blockIdx.x * K;
    if (r.s != r.s || c_lo >= c_hi) {  // the row has no distribution, or this slice no elements
      for (int j = tid; j < K; j += NT) keys_out[j] = 0;
      return;
    }
  }
  auto put = [&](int rank, uint64_t key) {
    if (keys_out != nullptr) keys_out[rank] = key;
    else put_alternative(out, row * K + rank, key, w, r.b, ln_s);
  };

  // The K best alternatives. Each group of four threads has its best key; the K-th best of those is a bound that K elements
  // at least reach and few exceed. The threads whose own best reaches it read their chunks again (a few of them, from the
  // cache) and list every element that does; the list is ranked by counting.
  uint64_t mine = 0;
  if (c_lo + tid < c_hi) {
    const int n = best < nfull ? VEC : tail;
    if (m == -INFINITY) {
      mine = key_of(m, best * VEC);  // NaN apart, which no sound row has, the first chunk holds nothing else
    } else {
#pragma unroll
      for (int j = VEC - 1; j >= 0; --j)
        if (j < n && best_chunk.get(j) == m) mine = key_of(m, best * VEC + j);
    }
  }
  uint64_t g = mine;
  g = key_max(g, (uint64_t)__shfl_xor((unsigned long long)g, 1, 64));
  g = key_max(g, (uint64_t)__shfl_xor((unsigned long long)g, 2, 64));
  if ((tid & 3) == 0) group_key[tid >> 2] = g;
  if (tid == 0) {
    threshold = 0;
    n_list = 0;
    n_threads = 0;
  }
  __syncthreads();
  {
    int above = 0;
    for (int i = 0; i < GROUPS / 4; ++i) above += group_key[(tid & 3) * (GROUPS / 4) + i] > g;
    above += __shfl_xor(above, 1, 64);
    above += __shfl_xor(above, 2, 64);
    if ((tid & 3) == 0 && above == K - 1 && g != 0) threshold = g;  // one group: the keys differ
  }
  __syncthreads();
  const uint64_t bound = threshold;
  if (mine != 0 && mine >= bound) threads_list[atomicAdd(&n_threads, 1)] = tid;
  __syncthreads();
  {
    const int lane = tid & 63, waves = NT / 64, nt = n_threads;
    for (int i = tid >> 6; i < nt; i += waves) {
      for (int cc = c_lo + threads_list[i] + lane * NT; cc < c_hi; cc += 64 * NT) {
        const int n = cc < nfull ? VEC : tail;
        const Pack<T, VEC> p = n == VEC ? load_any<T, VEC>(x + (long)cc * VEC) : load_tail<T, VEC>(x + (long)cc * VEC, n, cc * VEC);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const uint64_t k = key_of(p.get(j), cc * VEC + j);
          if (j < n && k >= bound) {
            const int at = atomicAdd(&n_list, 1);
            if (at < kList) list[at] = k;
          }
        }
      }
    }
  }
  __syncthreads();
  const int n = n_list;
  if (n <= kList) {
    for (int i = tid; i < n; i += NT) {
      const uint64_t k = list[i];
      int rank = 0;
#pragma unroll 8
      for (int q = 0; q < n; ++q) rank += list[q] > k;
      if (rank < K) put(rank, k);
    }
    for (int j = n + tid; j < K; j += NT) keys_out[j] = 0;  // a slice with fewer elements; a row has K at least
    return;
  }
  // More elements of a few threads than the list holds reach the bound (a row whose largest values all lie one thread's
  // stride apart): the best one below the last, K times over the slice.
  uint64_t last = ~0ull;
  for (int rank = 0; rank < K; ++rank) {
    uint64_t k = 0;
    for (int cc = c_lo + tid; cc < c_hi; cc += NT) {
      const int nn = cc < nfull ? VEC : tail;
      for (int j = 0; j < nn; ++j) {
        const uint64_t q = key_of(to_f<T>(x[(long)cc * VEC + j]), cc * VEC + j);
        if (q < last) k = key_max(k, q);
      }
    }
    for (int o = 1; o < 64; o <<= 1) k = key_max(k, (uint64_t)__shfl_xor((unsigned long long)k, o, 64));
    __syncthreads();
    if ((tid & 63) == 0) round_key[tid >> 6] = k;
    __syncthreads();
    for (int i = 0; i < NT / 64; ++i) k = key_max(k, round_key[i]);
    last = k;
    if (tid == 0) put(rank, k);
  }
}

// A block per row: the sums of its slices and the K best of their keys, ranked by counting.
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void token_logprobs_join_kernel(const T* __restrict__ logits, long stride,
                                                                  const int64_t* __restrict__ tokens, const RowOut out,
                                                                  const Sums* __restrict__ part_sums,
                                                                  const uint64_t* __restrict__ part_keys, int parts, int V, int K,
                                                                  const Temper w, int64_t ignore) {
  __shared__ uint64_t keys[kJoinThreads];
  const long row = blockIdx.x;
  const int tid = threadIdx.x, n = parts * K;
  const int64_t tok = tokens[row];
  if (tok == ignore) {
    if (tid == 0) out.lp[row] = out.ent[row] = 0.f;
    put_no_row<kJoinThreads>(out, row, K, 0.f);
    return;
  }
  if (tid < n) keys[tid] = part_keys[row * n + tid];
  // 8 lanes hold the slices' sums, every 8 lanes the same
  static_assert(kMaxParts == 8, "a slice per lane");
  Sums r{-INFINITY, 0.f, 0.f};
  if ((tid & 7) < parts) r = part_sums[row * parts + (tid & 7)];
  const float b = lanes_reduce<8, OpMax>(r.b);
  r = against(r, b, w.scale);
  r = Sums{b, lanes_reduce<8, OpSum>(r.s), lanes_reduce<8, OpSum>(r.u)};
  const float ln_s = finish_row<T>(r, logits + row * stride, tok, row, V, w, out, tid == 0);
  if (K == 0) return;
  if (ln_s != ln_s) {
    put_no_row<kJoinThreads>(out, row, K, NAN);
    return;
  }
  __syncthreads();
  if (tid < n) {
    const uint64_t k = keys[tid];
    int rank = 0;
#pragma unroll 8
    for (int q = 0; q < n; ++q) rank += keys[q] > k;
    if (k != 0 && rank < K) put_alternative(out, row * K + rank, k, w, r.b, ln_s);
  }
}

// blockIdx.x: a span of kBwdThreads * kBwdUnroll chunks, blockIdx.y / z: the row.
template <typename T>
__global__ __launch_bounds__(kBwdThreads) void token_logprobs_bwd_kernel(
    const T* __restrict__ logits, long stride, const int64_t* __restrict__ tokens, const float* __restrict__ stats,
    const int64_t* __restrict__ top_id, const float* __restrict__ g_lp, long g_lp_stride, const float* __restrict__ g_ent,
    long g_ent_stride, const float* __restrict__ g_top, T* __restrict__ out, int V, int K, const Temper w, int64_t ignore, int spans) {
  constexpr int VEC = 16 / sizeof(T);
  const long row = blockIdx.x / spans;
  const int span = (int)(blockIdx.x - row * spans), tid = threadIdx.x;
  const int nfull = V / VEC, tail = V % VEC, chunks = nfull + (tail > 0);
  const int64_t tok = tokens[row];
  const int c0 = span * kBwdThreads * kBwdUnroll;
  T* o = out + row * (long)V;
  if (tok == ignore) {
    const Pack<T, VEC> z = Pack<T, VEC>::zero();
    for (int u = 0; u < kBwdUnroll; ++u) {
      const int c = c0 + u * kBwdThreads + tid;
      if (c < nfull) store_any<T, VEC>(o + (long)c * VEC, z);
      else if (c < chunks) store_part<T, VEC>(o + (long)c * VEC, z, tail);
    }
    return;
  }
  const T* x = logits + row * stride;
  Pack<T, VEC> p[kBwdUnroll];
#pragma unroll
  for (int u = 0; u < kBwdUnroll; ++u) {
    const int c = c0 + u * kBwdThreads + tid;
    if (c < nfull) p[u] = load_any<T, VEC>(x + (long)c * VEC);
    else if (c < chunks) p[u] = load_tail<T, VEC>(x + (long)c * VEC, tail, c * VEC);
  }
  const float4 st = *reinterpret_cast<const float4*>(stats + row * 4);  // b, 1 / S, ln S, entropy
  // a token outside [0, V) has a NaN constant for a log-probability: nothing of its gradient reaches the logits
  const float gl = g_lp != nullptr && tok >= 0 && tok < V ? g_lp[row * g_lp_stride] : 0.f;
  const float gh = g_ent != nullptr ? g_ent[row * g_ent_stride] : 0.f;
  float total = gl;
  if (g_top != nullptr)
    for (int j = 0; j < K; ++j) total += g_top[row * K + j];
  // -p (G + dH (log p + H)) / T = 2^t (c + d t)
  const float inv_t = (float)w.inv_t, share = -st.y * inv_t, cc = share * (total + gh * (st.w - st.z)), dd = share * gh * kLn2;
  // The exponent's product and its scale are rounded: p is off by up to 1.5 |ln p| 2^-24 of itself. 16-bit gradients do not show it;
  // in fp32 what the rounding left out multiplies p (777 rows of 50257: 46 to 47 us with and without).
  auto value = [&](float f) {
    const float far = kFar / w.scale, d = sizeof(T) == 4 ? fmaxf(f - st.x, far) : f - st.x, t = d * w.scale;
    float p = exp2_of(t);
    if constexpr (sizeof(T) == 4) p = fmaf(p, kLn2 * fmaf(t, w.slack, fmaf(d, w.scale, -t)), p);
    return p * fmaf(dd, fmaxf(t, kFar), cc);
  };
#pragma unroll
  for (int u = 0; u < kBwdUnroll; ++u) {
    const int c = c0 + u * kBwdThreads + tid;
    if (c >= chunks) continue;
    float f[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) f[j] = value(p[u].get(j));
    const Pack<T, VEC> q = Pack<T, VEC>::of(f);
    if (c < nfull) store_any<T, VEC>(o + (long)c * VEC, q);
    else store_part<T, VEC>(o + (long)c * VEC, q, tail);
  }
  // the named elements of this span, each written again by one thread with all its terms and one rounding
  __syncthreads();
  const int named = g_top != nullptr ? K : 0;
  if (tid > named) return;
  const int64_t id = tid < named ? top_id[row * K + tid] : tok;
  const long lo = (long)c0 * VEC, hi = lo + (long)kBwdThreads * kBwdUnroll * VEC;
  if (id < lo || id >= hi || id >= V) return;  // -1 (no alternatives in this row) falls out here
  float extra = 0.f;
  if (tid < named) {
    extra = g_top[row * K + tid] + (id == tok ? gl : 0.f);
  } else {
    for (int j = 0; j < named; ++j)
      if (top_id[row * K + j] == tok) return;  // that alternative's thread writes it
    extra = gl;
  }
  o[id] = from_f<T>(fmaf(extra, inv_t, value(to_f<T>(x[id]))));
}

Temper temper_of(double inv_t) {
  const double scale = inv_t * 1.4426950408889634074;
  const float rounded = (float)scale;
  return Temper{inv_t, rounded, (float)((scale - rounded) / rounded)};
}

void check_logits(const torch::Tensor& logits, const torch::Tensor& tokens) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) == 1 || logits.numel() == 0),
              "token_logprobs: logits must be a 2-D HIP tensor with contiguous rows");
  TORCH_CHECK(logits.size(1) >= 1 && logits.size(1) < (1L << 31) - 65536, "token_logprobs: 1 to 2^31 - 65536 columns expected");
  TORCH_CHECK(tokens.dim() == 1 && tokens.size(0) == logits.size(0) && tokens.scalar_type() == at::kLong &&
                  tokens.is_contiguous() && tokens.device() == logits.device(),
              "token_logprobs: tokens must be a contiguous int64 [rows] tensor on the logits' device");
}

}  // namespace

ACC_DEBUG_TAKE_FN(acc_dbg_take_token_logprobs)

// logprobs [rows], entropy [rows], top log-probabilities and tokens [rows, K] (K > 0), stats [rows, 4] (`want_stats`).
std::vector<torch::Tensor> token_logprobs_fwd(torch::Tensor logits, torch::Tensor tokens, int64_t K, double inv_t, int64_t ignore,
                                              bool want_stats) {
  check_logits(logits, tokens);
  const long rows = logits.size(0), V = logits.size(1);
  TORCH_CHECK(K >= 0 && K <= kMaxTop && K <= V, "token_logprobs: 0 to ", kMaxTop, " alternatives, no more than the vocabulary");
  const c10::DeviceGuard guard(logits.device());
  const auto fopt = logits.options().dtype(torch::kFloat32);
  auto lp = torch::empty({rows}, fopt), ent = torch::empty({rows}, fopt);
  torch::Tensor top_lp, top_id, stats, work;
  if (K > 0) {
    top_lp = torch::empty({rows, K}, fopt);
    top_id = torch::empty({rows, K}, fopt.dtype(torch::kInt64));
  }
  if (want_stats) stats = torch::empty({rows, 4}, fopt);
  if (rows > 0) {
    // Few rows leave most of the chip idle: slices of at least kSlice bytes, as many as give kBlocks blocks.
    const long bytes = V * logits.element_size();
    const int parts = (int)std::max(1L, std::min({(long)kMaxParts, kBlocks / rows, bytes / kSlice}));
    TORCH_CHECK(rows * parts * 256 < (1L << 32), "token_logprobs: too many rows in one call");
    if (parts > 1) work = torch::empty({rows * parts * (K * 8 + (long)sizeof(Sums))}, fopt.dtype(torch::kUInt8));
    const RowOut out{lp.data_ptr<float>(), ent.data_ptr<float>(), K > 0 ? top_lp.data_ptr<float>() : nullptr,
                     want_stats ? stats.data_ptr<float>() : nullptr, K > 0 ? top_id.data_ptr<int64_t>() : nullptr};
    uint64_t* kp = parts > 1 ? reinterpret_cast<uint64_t*>(work.data_ptr()) : nullptr;
    Sums* sp = parts > 1 ? reinterpret_cast<Sums*>(kp + rows * parts * K) : nullptr;
    auto stream = at::hip::getCurrentHIPStream();
    ACC_FOR_FLOAT_TYPES(logits.scalar_type(), "token_logprobs", {
      const scalar* x = reinterpret_cast<const scalar*>(logits.data_ptr());
      // slices: twice the threads for the shortest way through one
      const int nt = parts > 1 ? 512 : 256;
      auto kernel = parts > 1 ? token_logprobs_fwd_kernel<scalar, 512, 4> : token_logprobs_fwd_kernel<scalar, 256, 4>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * parts)), dim3(nt), 0, stream, x,
                         logits.stride(0), tokens.data_ptr<int64_t>(), out, sp, kp, parts, (int)V, (int)K, temper_of(inv_t), ignore);
      if (parts > 1)
        hipLaunchKernelGGL((token_logprobs_join_kernel<scalar>), dim3((unsigned)rows), dim3(kJoinThreads), 0, stream, x, logits.stride(0),
                           tokens.data_ptr<int64_t>(), out, sp, kp, parts, (int)V, (int)K, temper_of(inv_t), ignore);
    });
  }
  return {lp, ent, top_lp, top_id, stats};
}

torch::Tensor token_logprobs_bwd(torch::Tensor logits, torch::Tensor tokens, torch::Tensor stats,
                                 c10::optional<torch::Tensor> top_id, c10::optional<torch::Tensor> g_lp,
                                 c10::optional<torch::Tensor> g_ent, c10::optional<torch::Tensor> g_top, double inv_t,
                                 int64_t ignore) {
  check_logits(logits, tokens);
  const long rows = logits.size(0), V = logits.size(1);
  const c10::DeviceGuard guard(logits.device());
  TORCH_CHECK(stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == rows * 4, "token_logprobs: stats");
  for (const auto& g : {g_lp, g_ent})
    TORCH_CHECK(!g.has_value() || (g->scalar_type() == at::kFloat && g->dim() == 1 && g->size(0) == rows && g->device() == logits.device()),
                "token_logprobs: gradients must be fp32 [rows]");
  long K = 0;
  if (g_top.has_value()) {
    TORCH_CHECK(top_id.has_value() && top_id->dim() == 2 && top_id->scalar_type() == at::kLong && top_id->is_contiguous() &&
                    g_top->scalar_type() == at::kFloat && g_top->is_contiguous() && g_top->sizes() == top_id->sizes() &&
                    top_id->size(0) == rows && top_id->size(1) <= kMaxTop && g_top->device() == logits.device(),
                "token_logprobs: the alternatives' gradients must be fp32 [rows, K]");
    K = top_id->size(1);
  }
  auto out = torch::empty({rows, V}, logits.options());
  if (rows == 0) return out;
  auto stream = at::hip::getCurrentHIPStream();
  ACC_FOR_FLOAT_TYPES(logits.scalar_type(), "token_logprobs", {
    constexpr long per = 16 / sizeof(scalar) * kBwdThreads * kBwdUnroll;
    const long spans = (V + per - 1) / per;
    TORCH_CHECK(rows * spans * kBwdThreads < (1L << 32), "token_logprobs: too many rows in one call");
    hipLaunchKernelGGL((token_logprobs_bwd_kernel<scalar>), dim3((unsigned)(rows * spans)), dim3(kBwdThreads), 0, stream,
                       reinterpret_cast<const scalar*>(logits.data_ptr()), logits.stride(0), tokens.data_ptr<int64_t>(),
                       stats.data_ptr<float>(), K > 0 ? top_id->data_ptr<int64_t>() : nullptr,
                       g_lp.has_value() ? g_lp->data_ptr<float>() : nullptr, g_lp.has_value() ? g_lp->stride(0) : 0,
                       g_ent.has_value() ? g_ent->data_ptr<float>() : nullptr, g_ent.has_value() ? g_ent->stride(0) : 0,
                       K > 0 ? g_top->data_ptr<float>() : nullptr, reinterpret_cast<scalar*>(out.data_ptr()), (int)V, (int)K,
                       temper_of(inv_t), ignore, (int)spans);
  });
  return out;
}
