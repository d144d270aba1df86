// Layer norm, forward and backward, with the residual add fused in (bf16 / fp16 / fp32, statistics in fp32):
//   s = round(x + residual),  y = (s - mean) * rstd * w + b,  rstd = 1 / sqrt(var + eps)
//   g = dy * w,  dx = rstd * (g - mean(g) - h * mean(g * h)) (+ dres),  h = (s - mean) * rstd
//   dw = sum over rows of dy * h,  db = sum over rows of dy
// Both are bound by memory. The row stays in registers between its sums and its output, so x is read once; the variance
// is the mean of squared distances from the mean, not a difference of two large sums. The threads of a row are chosen by
// its width and, in the forward, the number of rows: 8 lanes for a 128-byte row (32 rows to a block) up to 1024 threads.
// 8192 x 4096 bf16 with a residual: 48 us forward and 44 us backward (5.5 and 6.1 TB/s). 200000 x 64 bf16: 12 and 31 us (a wave
// for each row: 65 and 97), 60000 x 256: 14 and 22 us (23 and 35).
#include <hip/hip_runtime.h>
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <algorithm>
#include <type_traits>

#include "row_ops.h"

using namespace acc;

namespace {

constexpr int kMaxChunks = 4096;  // 16-byte chunks in a row: 32768 elements of 16 bits, 16384 of 32

// Chunk c of a row has n = VEC elements, the few at the end of a row whose width is no multiple of VEC, or 0 past it. The few
// (RAGGED kernels only) are loaded as the last VEC elements of the row, and moved to the front by settle() where they are
// used: a load that something waits for at once would hold up all the loads behind it. Rows of one chunk or less, shorter
// than VEC, are loaded element by element.
template <bool RAGGED, int VEC>
__device__ __forceinline__ int chunk_size(int c, int nfull, int tail) {
  return c < nfull ? VEC : RAGGED && c == nfull ? tail : 0;
}
template <bool RAGGED, typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> get_chunk(const T* row, int c, int n) {
  if (n == 0) return Pack<T, VEC>::zero();
  if constexpr (RAGGED) {
    if (c == 0 && n < VEC) return load_part<T, VEC>(row, n);
    return load_any<T, VEC>(row + c * VEC - (VEC - n));
  }
  return load_any<T, VEC>(row + c * VEC);
}
template <bool RAGGED, typename T, int VEC>
__device__ __forceinline__ void settle(Pack<T, VEC>& x, int c, int n) {
  if constexpr (RAGGED)
    if (n > 0 && n < VEC && c > 0) x = drop_front<T, VEC>(x, VEC - n);
}
template <bool RAGGED, typename T, int VEC>
__device__ __forceinline__ void put_chunk(T* p, const Pack<T, VEC>& x, int n) {
  if (n == VEC) store_any<T, VEC>(p, x);
  else if constexpr (RAGGED) store_part<T, VEC>(p, x, n);
}

// Where a whole wave works on one row, the row and its addresses are kept in scalar registers.
template <int TPR, int ROWS>
__device__ __forceinline__ long first_row() {
  if (ROWS == 1) return blockIdx.x;
  const int slot = threadIdx.x / TPR;
  return (long)blockIdx.x * ROWS + (TPR < 64 ? slot : __builtin_amdgcn_readfirstlane(slot));
}

template <typename T, typename W, int TPR, int VPT, bool RAGGED>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layer_norm_fwd_kernel(
    const T* __restrict__ x, long x_stride, const T* __restrict__ res, long res_stride, const W* __restrict__ w,
    const W* __restrict__ b, T* __restrict__ y, T* __restrict__ sum_out, float* __restrict__ mean_out,
    float* __restrict__ rstd_out, long rows, int H, float eps) {
  constexpr int VEC = 16 / sizeof(T), NT = TPR < 256 ? 256 : TPR, ROWS = NT / TPR;
  __shared__ float slots[2][16];
  const int li = ROWS == 1 ? threadIdx.x : threadIdx.x % TPR, nfull = H / VEC, tail = H % VEC;
  const float width = (float)H;
  // Up to two chunks per thread the parameters are loaded once, ahead of the first row's sums; wider rows load them again
  // for each row, from the cache.
  constexpr bool kHold = VPT <= 2;
  Pack<W, VEC> wv[VPT], bv[VPT];
  auto load_params = [&](int i) {
    const int c = li + i * TPR, n = chunk_size<RAGGED, VEC>(c, nfull, tail);
    if (w != nullptr) {
      wv[i] = get_chunk<RAGGED, W, VEC>(w, c, n);
      settle<RAGGED, W, VEC>(wv[i], c, n);
    }
    if (b != nullptr) {
      bv[i] = get_chunk<RAGGED, W, VEC>(b, c, n);
      settle<RAGGED, W, VEC>(bv[i], c, n);
    }
  };
  if constexpr (kHold) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) load_params(i);
  }
  // the trip count is uniform over each row's threads: lanes of a wave, or the whole block where barriers are used
  for (long row = first_row<TPR, ROWS>(); row < rows; row += (long)gridDim.x * ROWS) {
    const T* xr = x + row * x_stride;
    const T* rr = res == nullptr ? nullptr : res + row * res_stride;
    Pack<T, VEC> xa[VPT], xb[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = li + i * TPR, n = chunk_size<RAGGED, VEC>(c, nfull, tail);
      xa[i] = get_chunk<RAGGED, T, VEC>(xr, c, n);
      if (rr != nullptr) xb[i] = get_chunk<RAGGED, T, VEC>(rr, c, n);
    }
    float v[VPT][VEC];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = li + i * TPR;
      const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
      Pack<T, VEC> a = xa[i];
      settle<RAGGED, T, VEC>(a, c, n);
      if (rr != nullptr) {
        Pack<T, VEC> r = xb[i];
        settle<RAGGED, T, VEC>(r, c, n);
        float f[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) f[j] = a.get(j) + r.get(j);
        a = Pack<T, VEC>::of(f);
        // what is normalised is what the residual stream stores
        put_chunk<RAGGED, T, VEC>(sum_out + row * H + c * VEC, a, n);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] = a.get(j);
        sum += v[i][j];
      }
    }
    const float mean = row_reduce<OpSum, TPR>(sum, slots[0]) / width;
    float sq = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = li + i * TPR;
      const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        v[i][j] = (RAGGED ? j < n : n != 0) ? v[i][j] - mean : 0.f;
        sq = fmaf(v[i][j], v[i][j], sq);
      }
    }
    const float rstd = 1.f / sqrtf(row_reduce<OpSum, TPR>(sq, slots[1]) / width + eps);
    if (mean_out != nullptr && li == 0) {
      mean_out[row] = mean;
      rstd_out[row] = rstd;
    }
    T* yr = y + row * H;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = li + i * TPR;
      const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
      if (n == 0) continue;
      float o[VEC];
      if constexpr (!kHold) load_params(i);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float f = v[i][j] * rstd;
        if (w != nullptr) f *= wv[i].get(j);
        if (b != nullptr) f += bv[i].get(j);
        o[j] = f;
      }
      put_chunk<RAGGED, T, VEC>(yr + c * VEC, Pack<T, VEC>::of(o), n);
    }
  }
}

// One pass over the rows: dx, and each block's share of the column sums of dw and db in registers. The blocks' shares
// (fp32, [blocks, 2, chunks * VEC]) are added up in a fixed order by layer_norm_colsum_kernel, so results repeat.
template <typename T, typename W, int TPR, int VPT, bool RAGGED>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void layer_norm_bwd_kernel(
    const T* __restrict__ dy, long dy_stride, const T* __restrict__ s, long s_stride, const W* __restrict__ w,
    const float* __restrict__ mean, const float* __restrict__ rstd, const T* __restrict__ dres, long dres_stride,
    T* __restrict__ dx, float* __restrict__ part, long rows, int H) {
  constexpr int VEC = 16 / sizeof(T), NT = TPR < 256 ? 256 : TPR, ROWS = NT / TPR;
  __shared__ float slots[2][2][16];
  extern __shared__ float combine[];  // ROWS > 1: [2, chunks * VEC]
  const int li = ROWS == 1 ? threadIdx.x : threadIdx.x % TPR, nfull = H / VEC, tail = H % VEC, chunks = (H + VEC - 1) / VEC;
  const float width = (float)H;
  float dw[VPT][VEC], db[VPT][VEC];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dw[i][j] = db[i][j] = 0.f;
  // Up to two chunks per thread the weight stays in registers and the next row is loaded while this one is summed: a block
  // walks its rows in sequence, and each would pay the memory's latency after the last one's barrier. Wider rows have no
  // registers for that, and 64 elements per thread none for the row either, beside its columns' sums: the second reading
  // comes from the cache, in a loop that is not unrolled (2048 rows of 32768 bf16: 301 us, and 424 with the row kept).
  constexpr bool kHold = VPT <= 2, kKeep = VPT * VEC <= 32;
  auto load_w = [&](int c) {
    const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
    Pack<W, VEC> p = get_chunk<RAGGED, W, VEC>(w, c, n);
    settle<RAGGED, W, VEC>(p, c, n);
    return p;
  };
  Pack<W, VEC> wv[VPT];
  if (kHold && w != nullptr) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) wv[i] = load_w(li + i * TPR);
  }
  struct Chunk {
    Pack<T, VEC> s, dy, dres;
  };
  auto load_chunk = [&](long row, int c) {
    Chunk p;
    const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
    p.s = get_chunk<RAGGED, T, VEC>(s + row * s_stride, c, n);
    p.dy = get_chunk<RAGGED, T, VEC>(dy + row * dy_stride, c, n);  // zero past the row: adds nothing below
    if (dres != nullptr) p.dres = get_chunk<RAGGED, T, VEC>(dres + row * dres_stride, c, n);
    return p;
  };
  auto settle_chunk = [&](Chunk& p, int c) {
    const int n = chunk_size<RAGGED, VEC>(c, nfull, tail);
    settle<RAGGED, T, VEC>(p.s, c, n);
    settle<RAGGED, T, VEC>(p.dy, c, n);
    if (dres != nullptr) settle<RAGGED, T, VEC>(p.dres, c, n);
  };
  auto put_dx = [&](long row, int c, const Chunk& p, const Pack<W, VEC>& wc, float mu, float r, float s1, float s2) {
    float o[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float dd = p.dy.get(j), h = (p.s.get(j) - mu) * r;
      const float g = w != nullptr ? dd * wc.get(j) : dd;
      float f = r * (g - s1 - h * s2);
      if (dres != nullptr) f += p.dres.get(j);
      o[j] = f;
    }
    put_chunk<RAGGED, T, VEC>(dx + row * H + c * VEC, Pack<T, VEC>::of(o), chunk_size<RAGGED, VEC>(c, nfull, tail));
  };
  struct Row {
    Chunk at[VPT];
    float mean, rstd;
  };
  auto load_row = [&](long row, Row& r) {
    r.mean = mean[row];
    r.rstd = rstd[row];
    if constexpr (kKeep) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) r.at[i] = load_chunk(row, li + i * TPR);
    }
  };
  const long step = (long)gridDim.x * ROWS;
  long row = first_row<TPR, ROWS>();
  Row next;
  if (kHold && row < rows) load_row(row, next);
  int parity = 0;
  for (; row < rows; row += step, parity ^= 1) {
    Row cur;
    if constexpr (kHold) {
      cur = next;
      if (row + step < rows) load_row(row + step, next);
    } else {
      load_row(row, cur);
    }
    const float mu = cur.mean, r = cur.rstd;
    float s1 = 0.f, s2 = 0.f, s1_before = 0.f, s2_before = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      int c = li + i * TPR;
      if constexpr (!kKeep) {
        if (i % 2 == 0) {  // two chunks at a time, which keeps the chains of additions as short as those of narrower rows, and
          s1_before += s1;  // their loads behind the last two's sums: the compiler would start all of them and spill
          s2_before += s2;
          s1 = s2 = 0.f;
          asm volatile("" : "+v"(c), "+v"(s1_before), "+v"(s2_before));
        } else {
          asm volatile("" : "+v"(c));
        }
      }
      if (!kHold && w != nullptr) wv[i] = load_w(c);
      if constexpr (!kKeep) cur.at[i] = load_chunk(row, c);
      settle_chunk(cur.at[i], c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dd = cur.at[i].dy.get(j), h = (cur.at[i].s.get(j) - mu) * r;
        const float g = w != nullptr ? dd * wv[i].get(j) : dd;
        dw[i][j] = fmaf(dd, h, dw[i][j]);
        db[i][j] += dd;
        s1 += g;
        s2 = fmaf(g, h, s2);
      }
    }
    if constexpr (!kKeep) {
      s1 += s1_before;
      s2 += s2_before;
    }
    s1 = lanes_reduce<(TPR < 64 ? TPR : 64), OpSum>(s1);
    s2 = lanes_reduce<(TPR < 64 ? TPR : 64), OpSum>(s2);
    if constexpr (TPR > 64) {  // both sums behind one barrier; the other parity's slots serve the next row
      if ((threadIdx.x & 63) == 0) {
        slots[parity][0][threadIdx.x >> 6] = s1;
        slots[parity][1][threadIdx.x >> 6] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int k = 0; k < TPR / 64; ++k) {
        s1 += slots[parity][0][k];
        s2 += slots[parity][1][k];
      }
    }
    s1 /= width;
    s2 /= width;
    if constexpr (kKeep) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = li + i * TPR;
        if (c < chunks) put_dx(row, c, cur.at[i], wv[i], mu, r, s1, s2);
      }
    } else {
      for (int c = li; c < chunks; c += TPR) {
        Chunk p = load_chunk(row, c);
        settle_chunk(p, c);
        put_dx(row, c, p, w != nullptr ? load_w(c) : Pack<W, VEC>::zero(), mu, r, s1, s2);
      }
    }
  }
  if (part == nullptr) return;
  const long pitch = (long)chunks * VEC;
  float* out = part + (long)blockIdx.x * 2 * pitch;
  if constexpr (ROWS > 1) {  // the block's rows add into shared memory one after another: a fixed order
    for (int k = 0; k < ROWS; ++k) {
      if ((int)threadIdx.x / TPR == k) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const int c = li + i * TPR;
          if (c < chunks) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const int at = c * VEC + j;
              combine[at] = k == 0 ? dw[i][j] : combine[at] + dw[i][j];
              combine[pitch + at] = k == 0 ? db[i][j] : combine[pitch + at] + db[i][j];
            }
          }
        }
      }
      __syncthreads();
    }
    for (long at = threadIdx.x; at < 2 * pitch; at += NT) out[at] = combine[at];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = li + i * TPR;
      if (c < chunks) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
          *reinterpret_cast<float4*>(out + c * VEC + j) = make_float4(dw[i][j], dw[i][j + 1], dw[i][j + 2], dw[i][j + 3]);
          *reinterpret_cast<float4*>(out + pitch + c * VEC + j) =
              make_float4(db[i][j], db[i][j + 1], db[i][j + 2], db[i][j + 3]);
        }
      }
    }
  }
}

// Column sums of the blocks' shares: 32 columns x 32 row groups per block, eight loads in flight per thread.
template <typename W>
__global__ __launch_bounds__(1024) void layer_norm_colsum_kernel(const float* __restrict__ part, W* __restrict__ dw,
                                                                 W* __restrict__ db, int blocks, int H, long pitch) {
  __shared__ float red[32][33];
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const long col = (long)blockIdx.x * 32 + c;
  const float* src = part + blockIdx.y * pitch + col;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (col < H) {
    int p = rg;
    for (; p + 7 * 32 < blocks; p += 8 * 32)
#pragma unroll
      for (int u = 0; u < 8; ++u) acc[u] += src[(long)(p + 32 * u) * 2 * pitch];
    for (; p < blocks; p += 32) acc[0] += src[(long)p * 2 * pitch];
  }
  red[rg][c] = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
  __syncthreads();
  if (rg == 0 && col < H) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][c];
    W* out = blockIdx.y == 0 ? dw : db;
    if (out != nullptr) out[col] = from_f<W>(t);
  }
}

void check_rows(const torch::Tensor& t, const char* name, const torch::Tensor& like) {
  TORCH_CHECK(t.dim() == 2 && t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type() && t.device() == like.device() &&
                  (t.stride(1) == 1 || t.size(1) == 1 || t.numel() == 0),
              "layer_norm: ", name, " must be a 2-D tensor of x's shape, type and device with contiguous rows");
}

void check_param(const c10::optional<torch::Tensor>& p, const char* name, const torch::Tensor& x) {
  if (!p.has_value()) return;
  TORCH_CHECK(p->dim() == 1 && p->size(0) == x.size(1) && p->is_contiguous() && p->device() == x.device() &&
                  (p->scalar_type() == x.scalar_type() || p->scalar_type() == at::kFloat),
              "layer_norm: ", name, " must be a contiguous [hidden] tensor in x's type or fp32, on x's device");
}

template <typename T>
const T* ptr(const c10::optional<torch::Tensor>& t) { return t.has_value() ? reinterpret_cast<const T*>(t->data_ptr()) : nullptr; }
template <typename T>
T* out_ptr(const torch::Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }
long row_stride(const c10::optional<torch::Tensor>& t) { return t.has_value() ? t->stride(0) : 0; }

// Calls go(threads of a row, chunks of each) for a row of `chunks` 16-byte chunks.
template <int N> using Const = std::integral_constant<int, N>;
template <typename F>
void by_width_fwd(long chunks, long rows, F go) {
  if (chunks <= 8) return go(Const<8>{}, Const<1>{});
  if (chunks <= 16) return go(Const<16>{}, Const<1>{});
  if (chunks <= 32) return go(Const<32>{}, Const<1>{});
  if (chunks <= 64) return go(Const<64>{}, Const<1>{});
  if (rows >= 1024) {  // enough rows to fill the chip: few threads for each, and no barriers up to 256 chunks
    if (chunks <= 128) return go(Const<64>{}, Const<2>{});
    if (chunks <= 256) return go(Const<64>{}, Const<4>{});
    if (chunks <= 512) return go(Const<256>{}, Const<2>{});
    if (chunks <= 1024) return go(Const<256>{}, Const<4>{});
  }
  // few rows: as many threads as a row feeds, for the shortest way through one
  if (chunks <= 256) return go(Const<256>{}, Const<1>{});
  if (chunks <= 512) return go(Const<512>{}, Const<1>{});
  if (chunks <= 1024) return go(Const<1024>{}, Const<1>{});
  if (chunks <= 2048) return go(Const<1024>{}, Const<2>{});
  go(Const<1024>{}, Const<4>{});
}
template <typename F>
void by_width_bwd(long chunks, F go) {
  if (chunks <= 8) go(Const<8>{}, Const<1>{});
  else if (chunks <= 16) go(Const<16>{}, Const<1>{});
  else if (chunks <= 32) go(Const<32>{}, Const<1>{});
  else if (chunks <= 64) go(Const<64>{}, Const<1>{});
  else if (chunks <= 128) go(Const<64>{}, Const<2>{});
  else if (chunks <= 256) go(Const<256>{}, Const<1>{});
  else if (chunks <= 512) go(Const<256>{}, Const<2>{});
  else if (chunks <= 1024) go(Const<512>{}, Const<2>{});
  else if (chunks <= 2048) go(Const<512>{}, Const<4>{});
  else go(Const<512>{}, Const<8>{});
}

template <typename T, typename W>
void launch_fwd(const torch::Tensor& x, const c10::optional<torch::Tensor>& res, const c10::optional<torch::Tensor>& w,
                const c10::optional<torch::Tensor>& b, const torch::Tensor& y, const torch::Tensor& sum,
                const torch::Tensor& mean, const torch::Tensor& rstd, float eps, hipStream_t stream) {
  const long rows = x.size(0), H = x.size(1);
  by_width_fwd((H * (long)sizeof(T) + 15) / 16, rows, [&](auto tpr, auto vpt) {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value, NT = TPR < 256 ? 256 : TPR, per = NT / TPR;
    const long want = (rows + per - 1) / per, most = 1024L * 256 / NT;
    auto kernel = H % (16 / sizeof(T)) ? layer_norm_fwd_kernel<T, W, TPR, VPT, true> : layer_norm_fwd_kernel<T, W, TPR, VPT, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)std::min(want, most)), dim3(NT), 0, stream,
                       reinterpret_cast<const T*>(x.data_ptr()), x.stride(0), ptr<T>(res), row_stride(res), ptr<W>(w), ptr<W>(b),
                       out_ptr<T>(y), out_ptr<T>(sum), out_ptr<float>(mean), out_ptr<float>(rstd), rows, (int)H, eps);
  });
}

template <typename T, typename W>
void launch_bwd(const torch::Tensor& dy, const torch::Tensor& s, const c10::optional<torch::Tensor>& w, const torch::Tensor& mean,
                const torch::Tensor& rstd, const c10::optional<torch::Tensor>& dres, const torch::Tensor& dx,
                const torch::Tensor& dw, const torch::Tensor& db, hipStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  const long rows = s.size(0), H = s.size(1), chunks = (H + VEC - 1) / VEC, pitch = chunks * VEC;
  const bool sums = dw.defined() || db.defined();
  torch::Tensor part;
  long blocks = 0;
  by_width_bwd(chunks, [&](auto tpr, auto vpt) {
    constexpr int TPR = decltype(tpr)::value, VPT = decltype(vpt)::value, NT = TPR < 256 ? 256 : TPR, per = NT / TPR;
    // two blocks for each of the 256 units, or one of 512 and more threads: every block leaves a share to add up
    blocks = std::min((rows + per - 1) / per, NT == 256 ? 512L : 256L);
    if (sums) part = torch::empty({blocks, 2, pitch}, s.options().dtype(at::kFloat));
    auto kernel = H % VEC ? layer_norm_bwd_kernel<T, W, TPR, VPT, true> : layer_norm_bwd_kernel<T, W, TPR, VPT, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(NT),
                       per > 1 && sums ? 2 * pitch * sizeof(float) : 0, stream, reinterpret_cast<const T*>(dy.data_ptr()),
                       dy.stride(0), reinterpret_cast<const T*>(s.data_ptr()), s.stride(0), ptr<W>(w), mean.data_ptr<float>(),
                       rstd.data_ptr<float>(), ptr<T>(dres), row_stride(dres), out_ptr<T>(dx), out_ptr<float>(part), rows, (int)H);
  });
  if (sums)
    hipLaunchKernelGGL((layer_norm_colsum_kernel<W>), dim3((unsigned)((H + 31) / 32), 2), dim3(1024), 0, stream,
                       part.data_ptr<float>(), out_ptr<W>(dw), out_ptr<W>(db), (int)blocks, (int)H, pitch);
}

}  // namespace

ACC_DEBUG_TAKE_FN(acc_dbg_take_layer_norm)

// y [, s] [, mean, rstd (`stats`)] for x [rows, hidden].
std::vector<torch::Tensor> layer_norm_fwd(torch::Tensor x, c10::optional<torch::Tensor> residual, c10::optional<torch::Tensor> w,
                                          c10::optional<torch::Tensor> b, double eps, bool stats) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "layer_norm: x must be a 2-D HIP tensor");
  check_rows(x, "x", x);
  if (residual.has_value()) check_rows(*residual, "residual", x);
  check_param(w, "weight", x);
  check_param(b, "bias", x);
  TORCH_CHECK(!w.has_value() || !b.has_value() || w->scalar_type() == b->scalar_type(), "layer_norm: weight and bias of one type");
  const long rows = x.size(0);
  const int H = (int)x.size(1);
  const long chunks = (x.size(1) * x.element_size() + 15) / 16;
  TORCH_CHECK(x.size(1) >= 1 && chunks <= kMaxChunks, "layer_norm: 1 to ", kMaxChunks * 16 / x.element_size(), " columns expected");
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty({rows, H}, x.options());
  torch::Tensor sum, mean, rstd;
  if (residual.has_value()) sum = torch::empty({rows, H}, x.options());
  if (stats) {
    mean = torch::empty({rows}, x.options().dtype(torch::kFloat32));
    rstd = torch::empty({rows}, x.options().dtype(torch::kFloat32));
  }
  if (rows == 0) return {y, sum, mean, rstd};
  auto stream = at::hip::getCurrentHIPStream();
  const bool wide = (w.has_value() ? w->scalar_type() : b.has_value() ? b->scalar_type() : x.scalar_type()) == at::kFloat;
  ACC_FOR_FLOAT_TYPES(x.scalar_type(), "layer_norm", {
    if (wide) launch_fwd<scalar, float>(x, residual, w, b, y, sum, mean, rstd, (float)eps, stream);
    else launch_fwd<scalar, scalar>(x, residual, w, b, y, sum, mean, rstd, (float)eps, stream);
  });
  return {y, sum, mean, rstd};
}

// dx [, dw] [, db] as `want_dw` / `want_db` ask for them, in fp32 (`wide_params`) or the input's type. `w`, where given, has
// that type too.
std::vector<torch::Tensor> layer_norm_bwd(torch::Tensor dy, torch::Tensor s, c10::optional<torch::Tensor> w, torch::Tensor mean,
                                          torch::Tensor rstd, c10::optional<torch::Tensor> dres, bool want_dw, bool want_db,
                                          bool wide_params) {
  TORCH_CHECK(s.is_cuda() && s.dim() == 2, "layer_norm: the normalised input must be a 2-D HIP tensor");
  check_rows(s, "input", s);
  check_rows(dy, "dy", s);
  if (dres.has_value()) check_rows(*dres, "dres", s);
  check_param(w, "weight", s);
  TORCH_CHECK(!w.has_value() || (w->scalar_type() == at::kFloat) == (wide_params || s.scalar_type() == at::kFloat),
              "layer_norm: the weight's type and wide_params differ");
  const long rows = s.size(0);
  for (const auto& t : {mean, rstd})
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == rows && t.device() == s.device(),
                "layer_norm: mean and rstd must be fp32 [rows]");
  const int H = (int)s.size(1);
  const long chunks = (s.size(1) * s.element_size() + 15) / 16;
  TORCH_CHECK(s.size(1) >= 1 && chunks <= kMaxChunks, "layer_norm: 1 to ", kMaxChunks * 16 / s.element_size(), " columns expected");
  const c10::DeviceGuard guard(s.device());
  auto dx = torch::empty({rows, H}, s.options());
  const auto popt = s.options().dtype(wide_params ? at::kFloat : s.scalar_type());
  torch::Tensor dw, db;
  if (rows == 0) {
    if (want_dw) dw = torch::zeros({H}, popt);
    if (want_db) db = torch::zeros({H}, popt);
    return {dx, dw, db};
  }
  if (want_dw) dw = torch::empty({H}, popt);
  if (want_db) db = torch::empty({H}, popt);
  auto stream = at::hip::getCurrentHIPStream();
  ACC_FOR_FLOAT_TYPES(s.scalar_type(), "layer_norm", {
    if (wide_params) launch_bwd<scalar, float>(dy, s, w, mean, rstd, dres, dx, dw, db, stream);
    else launch_bwd<scalar, scalar>(dy, s, w, mean, rstd, dres, dx, dw, db, stream);
  });
  return {dx, dw, db};
}
