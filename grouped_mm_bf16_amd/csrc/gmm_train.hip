// What stands around the grouped products of an expert layer that is trained (declared in include/grouped_mm_hip.h): rows of tokens sorted by
// expert and back, with the router's weights, the activation between the products, and the derivatives of all three.
//   sort       xs[row(t, j)] = x[t]                        its gradient   dx[t] = sum over j of dxs[row(t, j)]
//   combine    out[t] = sum over j of w[t, j] y[row(t, j)]
//              its gradients   dy[row(t, j)] = w[t, j] dout[t],   dw[t, j] = <dout[t], y[row(t, j)]>
//   route      w = softmax of the chosen logits, or of all:  dl[e] = p[e] ([e chosen] dw[e] - sum over the chosen of p dw)
//   gated      out = g s(g) u,  s(g) = 1 / (1 + e^-g):  dg = dout u s(g) (1 + g (1 - s(g))),  du = dout g s(g)
// Memory bounds all of them.  Everything goes token by token, not row by row: what a token has once (x, dout, the sums) is read or written
// once, its choices' rows once each, and the sums over choices need no atomics.  16 bytes to an access, at any address; what is read or written
// once goes past the caches (below: without / with).
//   16384 tokens, 8 of 128 experts, bf16 rows of 2048   sort 115 / 103 us (5.9 TB/s; its one read through them, past them 114), sums 120 / 98 (6.2),
//                                                       combine's gradients 283 / 219 (5.2)
//   16384 x 14336 bf16                                  activation 265 / 251 (5.6), its gradient 446 / 428 (5.5)
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_elem.h"

namespace {

using namespace gmm;

constexpr int kMaxTopK = 32, kMaxExperts = 1023;
constexpr int kBlock = 256;

struct RowArgs {
  const void* x;              // of tokens (sort; combine's gradient: dout) or of sorted rows (sum)
  const void* y;              // combine's gradient: the sorted rows
  void* out;                  // sorted rows (sort, dy), or tokens (sum); dy: null if not wanted
  const int32_t* token_rows;
  const float* weight;        // null: ones
  float* dweight;             // null: not wanted
  int64_t tokens, rows, x_stride, y_stride, out_stride;
  int32_t top_k, width;
  int32_t lanes;              // that share a token: a power of two
};

template <typename T> __device__ __forceinline__ const T* row_of(const void* base, int64_t row, int64_t stride) {
  return static_cast<const T*>(base) + row * stride;
}
template <typename T> __device__ __forceinline__ T* row_of(void* base, int64_t row, int64_t stride) { return static_cast<T*>(base) + row * stride; }

// N elements from chunk c on.  Where rows are no WHOLE number of accesses the last one begins earlier, and two lanes write the same values to the same
// place.
template <typename T, int N, bool WHOLE>
__global__ void __launch_bounds__(kBlock) sort_rows_kernel(const RowArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1);
  const int64_t t = int64_t(blockIdx.x) * (kBlock / a.lanes) + threadIdx.x / a.lanes;
  if (t >= a.tokens) return;
  for (int c = lane * N; c < a.width; c += a.lanes * N) {
    const int at = Chunk<N, !WHOLE>(c, a.width).at;
    const Pack<T, N> v = unaligned<Pack<T, N>>(row_of<T>(a.x, t, a.x_stride) + at);
    for (int j = 0; j < a.top_k; ++j) {
      const int64_t r = a.token_rows[t * a.top_k + j];
      if (r >= 0 && r < a.rows) stream_out<WHOLE>(row_of<T>(a.out, r, a.out_stride) + at, v);
    }
  }
}

constexpr int kAtOnce = 8;      // choices whose rows are on their way together

// Rows of T, sums rounded to O: of the same type, or rows of fp32 (4001 tokens, 8 rows of 2048 each to bf16, 54 us, 5.2 TB/s; bf16 rows 26).
template <typename T, typename O, int N, bool WHOLE>
__global__ void __launch_bounds__(kBlock) sum_rows_kernel(const RowArgs a) {
  constexpr int M = N < kVector<T> ? N : kVector<T>;      // elements to a load
  const int lane = threadIdx.x & (a.lanes - 1);
  const int64_t t = int64_t(blockIdx.x) * (kBlock / a.lanes) + threadIdx.x / a.lanes;
  if (t >= a.tokens) return;
  for (int c = lane * N; c < a.width; c += a.lanes * N) {
    const int at = Chunk<N, !WHOLE>(c, a.width).at;
    float s[N] = {};
    for (int first = 0; first < a.top_k; first += kAtOnce) {
      Pack<T, M> v[kAtOnce][N / M];
      float w[kAtOnce];
      bool in[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int64_t slot = t * a.top_k + min(first + j, a.top_k - 1), r = a.token_rows[slot];
        in[j] = first + j < a.top_k && r >= 0 && r < a.rows;
        w[j] = a.weight ? a.weight[slot] : 1.0f;
        if (in[j])
#pragma unroll
          for (int q = 0; q < N / M; ++q) v[j][q] = stream_in<Pack<T, M>, WHOLE>(row_of<T>(a.x, r, a.x_stride) + at + q * M);
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j)
        if (in[j])
#pragma unroll
          for (int i = 0; i < N; ++i) s[i] += w[j] * v[j][i / M].get(i % M);
    }
    stream_out<WHOLE>(row_of<O>(a.out, t, a.out_stride) + at, Pack<O, N>::of(s));
  }
}

// The sums of products of kAtOnce choices stay in registers over all of the row, then go over its lanes; those of several waves meet in LDS.  A wave to
// a token, its row in pieces, takes an eighth longer.
template <typename T, int N, bool WHOLE>
__global__ void __launch_bounds__(kBlock) combine_backward_kernel(const RowArgs a) {
  constexpr int J = kAtOnce, WAVES = kBlock / 64;
  __shared__ float dots[WAVES][J];
  const int lane = threadIdx.x & (a.lanes - 1);
  const int64_t t = int64_t(blockIdx.x) * (kBlock / a.lanes) + threadIdx.x / a.lanes;
  const bool live = t < a.tokens;
  for (int first = 0; first < a.top_k; first += J) {
    int64_t row[J];
    float w[J], dot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const bool in = live && first + j < a.top_k;
      row[j] = in ? a.token_rows[t * a.top_k + first + j] : -1;
      if (row[j] >= a.rows) row[j] = -1;
      w[j] = in ? a.weight[t * a.top_k + first + j] : 0.0f;
      dot[j] = 0;
    }
    for (int c = lane * N; live && c < a.width; c += a.lanes * N) {
      const Chunk<N, !WHOLE> chunk(c, a.width);
      const Pack<T, N> d = stream_in<Pack<T, N>, WHOLE>(row_of<T>(a.x, t, a.x_stride) + chunk.at);
      Pack<T, N> y[J];
      if (a.dweight)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (row[j] >= 0) y[j] = stream_in<Pack<T, N>, WHOLE>(row_of<T>(a.y, row[j], a.y_stride) + chunk.at);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (row[j] < 0) continue;
        float dy[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (a.dweight) dot[j] += chunk.own(i) ? d.get(i) * y[j].get(i) : 0.0f;
          dy[i] = w[j] * d.get(i);
        }
        if (a.out) stream_out<WHOLE>(row_of<T>(a.out, row[j], a.out_stride) + chunk.at, Pack<T, N>::of(dy));
      }
    }
    if (!a.dweight) continue;
#pragma unroll
    for (int j = 0; j < J; ++j)
      for (int o = min(a.lanes, 64) / 2; o > 0; o >>= 1) dot[j] += __shfl_xor(dot[j], o);
    if (a.lanes > 64) {      // the same for the whole workgroup
      __syncthreads();
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int j = 0; j < J; ++j) dots[threadIdx.x >> 6][j] = dot[j];
      __syncthreads();
      const int waves = a.lanes / 64, wave0 = threadIdx.x / a.lanes * waves;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        dot[j] = 0;
        for (int i = 0; i < waves; ++i) dot[j] += dots[wave0 + i][j];
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane == 0 && live && first + j < a.top_k) a.dweight[t * a.top_k + first + j] = dot[j];
  }
}

// One wave to a token.  The weights that were softmax's results are what the derivative is made of; over all experts, those that were not
// chosen take part, and their shares are computed again from the logits: an infinite largest logit has equal shares with its equals.
template <typename T>
__global__ void __launch_bounds__(kBlock) route_backward_kernel(const float* __restrict__ dweight, const int32_t* __restrict__ slot_expert,
                                                                const float* __restrict__ slot_weight, const T* __restrict__ logits, int64_t ld,
                                                                T* __restrict__ dlogits, int64_t tokens, int E, int k) {
  const int lane = threadIdx.x & 63;
  const int64_t t = int64_t(blockIdx.x) * (kBlock / 64) + (threadIdx.x >> 6);
  if (t >= tokens) return;
  const bool in = lane < k;
  const int mine = in ? slot_expert[t * k + lane] : -1;
  const float w = in ? slot_weight[t * k + lane] : 0.0f, g = in ? dweight[t * k + lane] : 0.0f;
  float s = w * g;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  float most = 0, total = 1;
  if (logits) {
    most = -INFINITY;
    for (int e = lane; e < E; e += 64) most = fmaxf(most, widen(logits[t * ld + e]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
    total = 0;
    for (int e = lane; e < E; e += 64) {
      const float l = widen(logits[t * ld + e]);
      total += l == most ? 1.0f : expf(l - most);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o);
  }
  for (int first = 0; first < E; first += 64) {
    const int e = first + lane;
    float p = 0, d = 0;
    bool chosen = false;
    for (int j = 0; j < k; ++j) {
      const int ej = __builtin_amdgcn_readlane(mine, j);
      const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j)), gj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g), j));
      if (ej == e) { p = wj; d = gj; chosen = true; }
    }
    if (e >= E) continue;
    if (logits && !chosen) {
      const float l = widen(logits[t * ld + e]);
      p = (l == most ? 1.0f : expf(l - most)) / total;
    }
    dlogits[t * E + e] = rounded<T>(p * (d - s));
  }
}

// ---------------------------------------------------------------- activation
struct GatedArgs {
  const void* h;
  const void* dout;     // null: forward
  void* out;            // result, or dh
  int64_t rows, h_stride, dout_stride, out_stride;
  int32_t inner, lanes;
};

// e^-g, accurate for fp32 values, the hardware's for 16-bit ones, whose rounding is 2^13 times as large.
template <typename T> __device__ __forceinline__ float exp_minus(float g) { return sizeof(T) == 4 ? expf(-g) : __expf(-g); }

template <typename T, int N, bool WHOLE, bool SWIGLU, bool BACK>
__global__ void __launch_bounds__(kBlock) gated_kernel(const GatedArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1);
  const int64_t r = int64_t(blockIdx.x) * (kBlock / a.lanes) + threadIdx.x / a.lanes;
  if (r >= a.rows) return;
  const T* h = row_of<T>(a.h, r, a.h_stride);
  T* out = row_of<T>(a.out, r, a.out_stride);
  for (int c = lane * N; c < a.inner; c += a.lanes * N) {
    const int at = Chunk<N, !WHOLE>(c, a.inner).at;
    const Pack<T, N> gate = stream_in<Pack<T, N>, WHOLE>(h + at);
    Pack<T, N> up, d;
    if constexpr (SWIGLU) up = stream_in<Pack<T, N>, WHOLE>(h + a.inner + at);
    if constexpr (BACK) d = stream_in<Pack<T, N>, WHOLE>(row_of<T>(a.dout, r, a.dout_stride) + at);
    float first[N], second[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // g s(g) as one quotient where the result is fp32: as a product with a reciprocal it is a rounding further off.  The slope s(g) (1 + g (1 - s(g))) is
      // g s(g) (1 - s(g)) + s(g): a difference and a fused sum, three roundings fewer than with e^-g s(g) for 1 - s(g), after which the gradient of
      // normal values in fp32 was 6.0e-8 off (the formula in elementary operations 5.6e-8, this 5.0e-8).  Neither takes longer: memory bounds it.
      const float g = gate.get(i), t = 1.0f + exp_minus<T>(g), part = 1.0f / t, silu = sizeof(T) == 4 ? g / t : g * part;
      if constexpr (!BACK) {
        first[i] = silu;
        if constexpr (SWIGLU) first[i] *= up.get(i);
      } else {
        const float slope = __builtin_fmaf(silu, 1.0f - part, part);
        if constexpr (SWIGLU) {
          second[i] = d.get(i) * silu;
          first[i] = d.get(i) * slope * up.get(i);      // a slope of zero makes it zero, however large the partner
        } else {
          first[i] = d.get(i) * slope;
        }
      }
    }
    stream_out<WHOLE>(out + at, Pack<T, N>::of(first));
    if constexpr (BACK && SWIGLU) stream_out<WHOLE>(out + a.inner + at, Pack<T, N>::of(second));
  }
}

// ---------------------------------------------------------------- host side
// Lanes that share a row of `chunks` accesses.
int lanes_for(int64_t chunks, int most) {
  int n = 1;
  while (n < chunks && n < most) n *= 2;
  return n;
}

bool stride_fits(int64_t stride, int64_t rows, int64_t width) { return stride >= width || rows <= 1; }

// f(element type, elements to an access, whether rows are whole numbers of them) for rows of `width` elements.
template <typename F>
int by_type(int32_t dtype, int64_t width, F&& f) {
  const auto go = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (width >= kVector<T> && width % kVector<T> == 0) f(t, std::integral_constant<int, kVector<T>>{}, std::true_type{});
    else if (width >= kVector<T>) f(t, std::integral_constant<int, kVector<T>>{}, std::false_type{});
    else f(t, std::integral_constant<int, 1>{}, std::false_type{});
  };
  if (dtype == GMM_DT_BF16) go(static_cast<Bf16*>(nullptr));
  else if (dtype == GMM_DT_F16) go(static_cast<F16*>(nullptr));
  else go(static_cast<float*>(nullptr));
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

int check_rows(int64_t tokens, int64_t top_k, int64_t width, int64_t rows, int32_t dtype) {
  constexpr int64_t limit = int64_t(1) << 31;
  if (tokens < 0 || tokens >= limit || top_k < 1 || top_k > kMaxTopK || width < 0 || width > limit - kBlock * 8 || rows < 0 || rows >= limit)
    return GMM_ERR_BAD_ARGUMENT;
  return dtype < GMM_DT_BF16 || dtype > GMM_DT_F32 ? GMM_ERR_UNSUPPORTED : GMM_OK;
}

unsigned groups_of(int64_t rows, int lanes) { return unsigned((rows + kBlock / lanes - 1) / (kBlock / lanes)); }

// Rows of `dtype`, their sums of `out_dtype`: the same, or rows of fp32.
int sum_rows(const void* y, const int32_t* token_rows, const float* slot_weight, void* out, int64_t tokens, int64_t top_k, int64_t hidden,
             int64_t y_rows, int64_t y_stride, int64_t out_stride, int32_t dtype, int32_t out_dtype, void* stream) {
  const int bad = check_rows(tokens, top_k, hidden, y_rows, out_dtype);
  if (bad) return bad;
  if (tokens == 0 || hidden == 0) return GMM_OK;
  if ((y_rows > 0 && !y) || !token_rows || !out || !stride_fits(y_stride, y_rows, hidden) || !stride_fits(out_stride, tokens, hidden)) return GMM_ERR_BAD_ARGUMENT;
  RowArgs a{};
  a.x = y; a.out = out; a.token_rows = token_rows; a.weight = slot_weight; a.tokens = tokens; a.rows = y_rows; a.x_stride = y_stride;
  a.out_stride = out_stride; a.top_k = int32_t(top_k); a.width = int32_t(hidden);
  return by_type(out_dtype, hidden, [&](auto* t, auto n, auto whole) {
    using O = std::remove_pointer_t<decltype(t)>;
    constexpr int N = decltype(n)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    a.lanes = lanes_for((hidden + N - 1) / N, kBlock);
    const dim3 grid(groups_of(tokens, a.lanes)), block(kBlock);
    if (dtype == out_dtype) hipLaunchKernelGGL((sum_rows_kernel<O, O, N, WHOLE>), grid, block, 0, static_cast<hipStream_t>(stream), a);
    else hipLaunchKernelGGL((sum_rows_kernel<float, O, N, WHOLE>), grid, block, 0, static_cast<hipStream_t>(stream), a);
  });
}

int gated(GatedArgs a, int64_t inner, int32_t kind, int32_t dtype, void* stream) {
  constexpr int64_t limit = int64_t(1) << 31;
  const int64_t parts = kind == GMM_ACT_SWIGLU ? 2 : 1;
  if (a.rows < 0 || a.rows >= limit || inner < 0 || inner > (limit - kBlock * 8) / 2 || kind < GMM_ACT_SILU || kind > GMM_ACT_SWIGLU) return GMM_ERR_BAD_ARGUMENT;
  if (dtype < GMM_DT_BF16 || dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
  if (a.rows == 0 || inner == 0) return GMM_OK;
  if (!a.h || !a.out || !stride_fits(a.h_stride, a.rows, parts * inner) || !stride_fits(a.out_stride, a.rows, (a.dout ? parts : 1) * inner) ||
      (a.dout && !stride_fits(a.dout_stride, a.rows, inner))) return GMM_ERR_BAD_ARGUMENT;
  a.inner = int32_t(inner);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return by_type(dtype, inner, [&](auto* t, auto n, auto whole) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int N = decltype(n)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    GatedArgs b = a;
    b.lanes = lanes_for((inner + N - 1) / N, kBlock);
    const dim3 grid(groups_of(a.rows, b.lanes)), block(kBlock);
    if (a.dout && parts == 2) hipLaunchKernelGGL((gated_kernel<T, N, WHOLE, true, true>), grid, block, 0, s, b);
    else if (a.dout) hipLaunchKernelGGL((gated_kernel<T, N, WHOLE, false, true>), grid, block, 0, s, b);
    else if (parts == 2) hipLaunchKernelGGL((gated_kernel<T, N, WHOLE, true, false>), grid, block, 0, s, b);
    else hipLaunchKernelGGL((gated_kernel<T, N, WHOLE, false, false>), grid, block, 0, s, b);
  });
}

}  // namespace

extern "C" {

int gmm_moe_sort_rows(const void* x, const int32_t* token_rows, void* out, int64_t tokens, int64_t top_k, int64_t hidden, int64_t out_rows,
                      int64_t x_stride, int64_t out_stride, int32_t dtype, void* stream) {
  const int bad = check_rows(tokens, top_k, hidden, out_rows, dtype);
  if (bad) return bad;
  if (tokens == 0 || hidden == 0 || out_rows == 0) return GMM_OK;
  if (!x || !token_rows || !out || !stride_fits(x_stride, tokens, hidden) || !stride_fits(out_stride, out_rows, hidden)) return GMM_ERR_BAD_ARGUMENT;
  RowArgs a{};
  a.x = x; a.out = out; a.token_rows = token_rows; a.tokens = tokens; a.rows = out_rows; a.x_stride = x_stride; a.out_stride = out_stride;
  a.top_k = int32_t(top_k); a.width = int32_t(hidden);
  return by_type(dtype, hidden, [&](auto* t, auto n, auto whole) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int N = decltype(n)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    a.lanes = lanes_for((hidden + N - 1) / N, kBlock);
    hipLaunchKernelGGL((sort_rows_kernel<T, N, WHOLE>), dim3(groups_of(tokens, a.lanes)), dim3(kBlock), 0, static_cast<hipStream_t>(stream), a);
  });
}

int gmm_moe_sum_rows(const void* y, const int32_t* token_rows, const float* slot_weight, void* out, int64_t tokens, int64_t top_k, int64_t hidden,
                     int64_t y_rows, int64_t y_stride, int64_t out_stride, int32_t dtype, void* stream) {
  return sum_rows(y, token_rows, slot_weight, out, tokens, top_k, hidden, y_rows, y_stride, out_stride, dtype, dtype, stream);
}

int gmm_moe_sum_rows_f32(const float* y, const int32_t* token_rows, const float* slot_weight, void* out, int64_t tokens, int64_t top_k, int64_t hidden,
                         int64_t y_rows, int64_t y_stride, int64_t out_stride, int32_t out_dtype, void* stream) {
  return sum_rows(y, token_rows, slot_weight, out, tokens, top_k, hidden, y_rows, y_stride, out_stride, GMM_DT_F32, out_dtype, stream);
}

int gmm_moe_combine_backward(const void* dout, const void* y, const int32_t* token_rows, const float* slot_weight, void* dy, float* dweight,
                             int64_t tokens, int64_t top_k, int64_t hidden, int64_t y_rows, int64_t dout_stride, int64_t y_stride,
                             int64_t dy_stride, int32_t dtype, void* stream) {
  const int bad = check_rows(tokens, top_k, hidden, y_rows, dtype);
  if (bad) return bad;
  if (tokens == 0 || (!dy && !dweight)) return GMM_OK;
  if (!token_rows || !slot_weight) return GMM_ERR_BAD_ARGUMENT;
  if (hidden > 0 && (!dout || (dweight && y_rows > 0 && !y) || !stride_fits(dout_stride, tokens, hidden) ||
                     (dweight && !stride_fits(y_stride, y_rows, hidden)) || (dy && !stride_fits(dy_stride, y_rows, hidden)))) return GMM_ERR_BAD_ARGUMENT;
  RowArgs a{};
  a.x = dout; a.y = y; a.out = dy; a.token_rows = token_rows; a.weight = slot_weight; a.dweight = dweight; a.tokens = tokens; a.rows = y_rows;
  a.x_stride = dout_stride; a.y_stride = y_stride; a.out_stride = dy_stride; a.top_k = int32_t(top_k); a.width = int32_t(hidden);
  return by_type(dtype, hidden, [&](auto* t, auto n, auto whole) {
    using T = std::remove_pointer_t<decltype(t)>;
    constexpr int N = decltype(n)::value;
    constexpr bool WHOLE = decltype(whole)::value;
    a.lanes = lanes_for((hidden + N - 1) / N, kBlock);
    hipLaunchKernelGGL((combine_backward_kernel<T, N, WHOLE>), dim3(groups_of(tokens, a.lanes)), dim3(kBlock), 0, static_cast<hipStream_t>(stream), a);
  });
}

int gmm_moe_route_backward(const float* dweight, const int32_t* slot_expert, const float* slot_weight, const void* logits, void* dlogits,
                           int64_t tokens, int64_t experts, int64_t top_k, int64_t logits_stride, int32_t logits_dtype, void* stream) {
  if (tokens < 0 || tokens >= (int64_t(1) << 31) || experts < 1 || experts > kMaxExperts || top_k < 1 || top_k > kMaxTopK || top_k > experts)
    return GMM_ERR_BAD_ARGUMENT;
  if (logits_dtype < GMM_DT_BF16 || logits_dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
  if (tokens == 0) return GMM_OK;
  if (!dweight || !slot_expert || !slot_weight || !dlogits || (logits && !stride_fits(logits_stride, tokens, experts))) return GMM_ERR_BAD_ARGUMENT;
  const dim3 grid(unsigned((tokens + kBlock / 64 - 1) / (kBlock / 64))), block(kBlock);
  const auto launch = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    hipLaunchKernelGGL(route_backward_kernel<T>, grid, block, 0, static_cast<hipStream_t>(stream), dweight, slot_expert, slot_weight,
                       static_cast<const T*>(logits), logits_stride, static_cast<T*>(dlogits), tokens, int(experts), int(top_k));
  };
  if (logits_dtype == GMM_DT_BF16) launch(static_cast<Bf16*>(nullptr));
  else if (logits_dtype == GMM_DT_F16) launch(static_cast<F16*>(nullptr));
  else launch(static_cast<float*>(nullptr));
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

int gmm_gated(const void* h, void* out, int64_t rows, int64_t inner, int64_t h_stride, int64_t out_stride, int32_t kind, int32_t dtype, void* stream) {
  GatedArgs a{};
  a.h = h; a.out = out; a.rows = rows; a.h_stride = h_stride; a.out_stride = out_stride;
  return gated(a, inner, kind, dtype, stream);
}

int gmm_gated_backward(const void* dout, const void* h, void* dh, int64_t rows, int64_t inner, int64_t dout_stride, int64_t h_stride,
                       int64_t dh_stride, int32_t kind, int32_t dtype, void* stream) {
  if (!dout && rows > 0 && inner > 0) return GMM_ERR_BAD_ARGUMENT;
  GatedArgs a{};
  a.h = h; a.dout = dout; a.out = dh; a.rows = rows; a.h_stride = h_stride; a.dout_stride = dout_stride; a.out_stride = dh_stride;
  return gated(a, inner, kind, dtype, stream);
}

}  // extern "C"
