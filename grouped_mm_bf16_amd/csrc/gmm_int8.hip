// Rows rounded to 8-bit integers with a scale each (declared in include/grouped_mm_hip.h):
//   scale[r] = max(max |x[r]|, 2^-100) / 127,   q[r, c] = x[r, c] / scale[r], rounded to a whole number, ties to even
// of x as it is, or of the activation between an expert layer's products, which is computed here from their fp32 result: no rounding to 16 bits
// stands between the two.  A row with an infinity or NaN in it has that as its scale and zeros for values: products with it are NaN.  Memory
// bounds it: a row is read once and stays in registers between its maximum and its rounding, 16 to 256 lanes to a row by its length.
//   8192 rows of 4096 bf16   16.6 us (6.0 TB/s)      32008 rows of 768 fp32   20.9 us (5.9 TB/s)
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_elem.h"
#include "gmm_launch.h"

namespace {

using namespace gmm;

constexpr int kSpan = 16;      // elements that a lane turns into one store of 16 bytes
constexpr int kGroup = 256;

struct QuantArgs {
  const void* x;
  int8_t* values;
  float* scale;
  int64_t rows, x_stride, values_stride;
  int32_t width;
  int32_t parts;          // of the activation's operand, each `plane` elements behind the one before: it is their sum
  int64_t plane;
};

// 16 elements from column c on; zeros past the row's end.
template <typename T>
struct Plain {
  typedef T Elem;
  static __device__ __forceinline__ void load(const QuantArgs& a, const T* row, int c, float (&v)[kSpan]) { get(row, c, a.width, v); }
  static __device__ __forceinline__ void get(const T* row, int c, int width, float (&v)[kSpan]) {
    constexpr int N = kVector<T>;
    if (c + kSpan <= width) {
#pragma unroll
      for (int q = 0; q < kSpan / N; ++q) {
        const Pack<T, N> p = unaligned<Pack<T, N>>(row + c + q * N);
#pragma unroll
        for (int i = 0; i < N; ++i) v[q * N + i] = p.get(i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kSpan; ++i) v[i] = c + i < width ? widen(row[c + i]) : 0.0f;
    }
  }
};

// silu(h), or silu(h[c]) * h[width + c].
template <bool SWIGLU>
struct Gated {
  typedef float Elem;
  static __device__ __forceinline__ void load(const QuantArgs& a, const float* row, int c, float (&v)[kSpan]) {
    float u[kSpan];
    Plain<float>::get(row, c, a.width, v);
    if constexpr (SWIGLU) Plain<float>::get(row + a.width, c, a.width, u);
    for (int p = 1; p < a.parts; ++p) {
      float more[kSpan];
      Plain<float>::get(row + p * a.plane, c, a.width, more);
#pragma unroll
      for (int i = 0; i < kSpan; ++i) v[i] += more[i];
      if constexpr (SWIGLU) {
        Plain<float>::get(row + p * a.plane + a.width, c, a.width, more);
#pragma unroll
        for (int i = 0; i < kSpan; ++i) u[i] += more[i];
      }
    }
#pragma unroll
    for (int i = 0; i < kSpan; ++i) {
      v[i] = v[i] / (1.0f + __expf(-v[i]));
      if constexpr (SWIGLU) v[i] *= u[i];
    }
  }
};

// The larger of two magnitudes, NaN above all, by their bits.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// PER spans to a lane, LANES lanes to a row; PER = 0: rows of any length, read twice.
template <typename S, int LANES, int PER>
__global__ void __launch_bounds__(kGroup) quantize_kernel(const QuantArgs a) {
  constexpr int ROWS = kGroup / LANES, WAVES = LANES > 64 ? LANES / 64 : 1;
  __shared__ uint32_t slots[WAVES];
  const int lane = threadIdx.x % LANES;
  const int64_t r = int64_t(blockIdx.x) * ROWS + threadIdx.x / LANES;
  const bool live = r < a.rows;      // whole rows of lanes; a workgroup of several waves has one row
  const auto* x = static_cast<const typename S::Elem*>(a.x) + (live ? r : 0) * a.x_stride;
  float v[PER ? PER : 1][kSpan];
  uint32_t most = 0;
  if constexpr (PER > 0) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int c = (p * LANES + lane) * kSpan;
      if (live && c < a.width) S::load(a, x, c, v[p]);
      else
#pragma unroll
        for (int i = 0; i < kSpan; ++i) v[p][i] = 0;
    }
#pragma unroll
    for (int p = 0; p < PER; ++p)
#pragma unroll
      for (int i = 0; i < kSpan; ++i) most = max(most, magnitude(v[p][i]));
  } else {
    for (int c = lane * kSpan; live && c < a.width; c += LANES * kSpan) {
      S::load(a, x, c, v[0]);
#pragma unroll
      for (int i = 0; i < kSpan; ++i) most = max(most, magnitude(v[0][i]));
    }
  }
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) most = max(most, uint32_t(__shfl_xor(int(most), o)));
  if constexpr (LANES > 64) {
    if ((threadIdx.x & 63) == 0) slots[threadIdx.x >> 6] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) most = max(most, slots[w]);
  }
  if (!live) return;
  const RowScale s(most);
  if (lane == 0) a.scale[r] = s.scale;
  int8_t* const to = a.values + r * a.values_stride;
  const auto store = [&](int c, const float (&f)[kSpan]) {
    u32x4 w;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      w[q] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[q] |= s.rounded_bits(f[4 * q + i]) << 8 * i;
      if (!s.finite) w[q] = 0;
    }
    *reinterpret_cast<u32x4*>(to + c) = w;
  };
  if constexpr (PER > 0) {
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const int c = (p * LANES + lane) * kSpan;
      if (c < a.width) store(c, v[p]);
    }
  } else {
    for (int c = lane * kSpan; c < a.width; c += LANES * kSpan) {
      S::load(a, x, c, v[0]);
      store(c, v[0]);
    }
  }
}

template <typename S>
int launch(const QuantArgs& a, hipStream_t stream) {
#define GMM_SHAPE(lanes, per)                                                                                                              \
  if (a.width <= lanes * per * kSpan || per == 0) {                                                                                        \
    constexpr int rows = kGroup / lanes;                                                                                                   \
    hipLaunchKernelGGL((quantize_kernel<S, lanes, per>), dim3(unsigned((a.rows + rows - 1) / rows)), dim3(kGroup), 0, stream, a);           \
    return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;                                                                      \
  }
  GMM_SHAPE(16, 1)
  GMM_SHAPE(64, 1)
  GMM_SHAPE(64, 2)
  GMM_SHAPE(256, 1)
  GMM_SHAPE(256, 2)
  GMM_SHAPE(256, 4)
  GMM_SHAPE(256, 0)
#undef GMM_SHAPE
  return GMM_ERR_BAD_ARGUMENT;
}

int check(const void* x, int8_t* values, float* scale, int64_t rows, int64_t width, int64_t columns, int64_t x_stride, int64_t values_stride) {
  if (rows < 0 || rows >= (int64_t(1) << 31) || width < 0 || width >= (int64_t(1) << 30)) return GMM_ERR_BAD_ARGUMENT;
  if (rows == 0) return GMM_OK;
  if (!scale || (width > 0 && (!x || !values)) || (x_stride < columns && rows > 1)) return GMM_ERR_BAD_ARGUMENT;
  if ((values_stride & 15) || values_stride < width || !aligned16(values)) return GMM_ERR_BAD_ARGUMENT;
  return GMM_OK;
}

}  // namespace

int gmm_int8_gated_parts(const float* h, int parts, int64_t plane, int8_t* values, float* scale, int64_t rows, int64_t inner, int64_t h_stride,
                         int64_t values_stride, int32_t kind, hipStream_t stream) {
  if (kind < GMM_ACT_SILU || kind > GMM_ACT_SWIGLU) return GMM_ERR_BAD_ARGUMENT;
  const int bad = check(h, values, scale, rows, inner, (kind == GMM_ACT_SWIGLU ? 2 : 1) * inner, h_stride, values_stride);
  if (bad || rows == 0) return bad;
  const QuantArgs a{h, values, scale, rows, h_stride, values_stride, int32_t(inner), parts, plane};
  return kind == GMM_ACT_SWIGLU ? launch<Gated<true>>(a, stream) : launch<Gated<false>>(a, stream);
}

extern "C" {

int gmm_int8_quantize(const void* x, int8_t* values, float* scale, int64_t rows, int64_t width, int64_t x_stride, int64_t values_stride,
                      int32_t dtype, void* stream) {
  if (dtype < GMM_DT_BF16 || dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
  const int bad = check(x, values, scale, rows, width, width, x_stride, values_stride);
  if (bad || rows == 0) return bad;
  const QuantArgs a{x, values, scale, rows, x_stride, values_stride, int32_t(width), 1, 0};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GMM_DT_BF16) return launch<Plain<Bf16>>(a, s);
  if (dtype == GMM_DT_F16) return launch<Plain<F16>>(a, s);
  return launch<Plain<float>>(a, s);
}

int gmm_int8_gated(const float* h, int8_t* values, float* scale, int64_t rows, int64_t inner, int64_t h_stride, int64_t values_stride,
                   int32_t kind, void* stream) {
  return gmm_int8_gated_parts(h, 1, 0, values, scale, rows, inner, h_stride, values_stride, kind, static_cast<hipStream_t>(stream));
}

}  // extern "C"
