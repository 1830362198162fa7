// Layer norm, forward and backward (declared in include/grouped_mm_hip.h).
//   z = (x - mean) * rstd,  rstd = 1 / sqrt(var + eps),  y = z * w + b
//   g = dy * w:  dx = rstd * (g - mean(g) - z * mean(g * z));   dw = sum over the rows of dy * z;   db = sum over the rows of dy
// Memory bounds both directions: forward reads x and writes y, backward reads x and dy and writes dx.  A row is read once and stays
// in registers between its sums; mean and variance are two sums over registers (no cancellation as with the sum of squares), and
// what the first mean's rounding left is added up and taken back: of a constant row of 1e4 the result was 0.3 off.  All
// sums are fp32.  8 to 1024 lanes share a row, 16 bytes to an access, so that short rows fill a wave and long ones fit into
// registers; the next row is on its way while one is summed.
//   forward   16384 x 4096 bf16 47 us, 8192 x 14336 fp16 91 us, 4096 x 16384 fp32 83 us (5.2 to 6.5 TB/s; a copy of that size 5.0)
//   backward  16384 x 4096 bf16 70 us, 8192 x 14336 fp16 143 us (5.7 and 4.9 TB/s), with the sums over the rows
// Rows that are no whole number of vectors cost about half as much again for an element: 4320 x 4397 bf16 27 and 40 us.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_elem.h"

namespace {

using namespace gmm;

constexpr int kMaxWidth = 16384;

struct NormArgs {
  const void* x;
  const void* dy;        // backward
  const void* weight;    // null: ones
  const void* bias;      // null: zeros
  void* out;             // y, or dx (null: not wanted)
  float* mean;           // forward: written unless null; backward: read
  float* rstd;
  float* partial;        // backward: [workgroups][2][width], null: neither dw nor db is wanted
  int64_t rows, x_stride, dy_stride, out_stride;
  int32_t width, weight_f32;
  float eps;
};

// Eight (fp32: four) elements to an access, which may begin anywhere.  Where fewer are left in a row (TAIL) the last eight are loaded: `skip`
// of them are another lane's.
template <int N, bool TAIL>
struct Chunk {
  int at, skip;
  bool in;
  __device__ __forceinline__ Chunk(int c, int width) : at(c), skip(0), in(c < width) {
    if constexpr (TAIL) {
      at = min(c, width - N);
      skip = c - at;
    }
  }
  __device__ __forceinline__ bool own(int i) const { return in && (!TAIL || i >= skip); }
};

// A chunk of a row that is read once.  Non-temporal, which keeps it from driving out what is written (4096 x 16384 fp32 99 -> 81 us; rows that
// lie at odd addresses too: 8192 x 14336 fp16, 14337 apart, 111 -> 103), but not where a row ends inside a chunk: two lanes then read its
// last cache line, one after the other (21800 x 329 fp32 11.8, non-temporal 15.3 us).
template <typename T, int N, bool TAIL>
__device__ __forceinline__ Pack<T, N> load_row(const T* row, const Chunk<N, TAIL>& c) {
  if constexpr (TAIL || N == 1) {
    return unaligned<Pack<T, N>>(row + c.at);
  } else {
    typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
    return __builtin_bit_cast(Pack<T, N>, u32x4(__builtin_nontemporal_load(reinterpret_cast<const Words*>(row + c.at))));
  }
}

// A parameter vector's elements c .. c + N - 1: of x's type, or fp32 beside 16-bit rows.
template <typename T, int N>
__device__ __forceinline__ void load_params(const void* p, int f32, int c, bool in, float none, float (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = none;
  if (!p || !in) return;
  if (f32) {
    const Pack<float, N> v = unaligned<Pack<float, N>>(static_cast<const float*>(p) + c);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v.get(i);
  } else {
    const Pack<T, N> v = unaligned<Pack<T, N>>(static_cast<const T*>(p) + c);
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = v.get(i);
  }
}

template <typename T, int N, bool TAIL>
__device__ __forceinline__ void store_row(T* row, const Chunk<N, TAIL>& c, const float (&v)[N]) {
  const Pack<T, N> p = Pack<T, N>::of(v);
  if (!TAIL || c.skip == 0) {
    if (c.in) __builtin_memcpy(row + c.at, &p, sizeof(p));
  } else if (c.in) {
#pragma unroll
    for (int i = 1; i < N; ++i) if (i >= c.skip) row[c.at + i] = rounded<T>(v[i]);
  }
}

// Sum over the LANES lanes that share a row.  Up to a wave: butterfly.  More: one slot per wave in LDS; `turn` alternates between two
// sets of slots, so that one barrier a sum is enough (whoever writes a set again has passed the barrier of the other one, behind
// which nobody reads it any more).
template <int LANES>
__device__ __forceinline__ void row_sum(float (&v)[2], int n, float* slots, int& turn) {
  constexpr int STEPS = LANES < 64 ? LANES : 64;
#pragma unroll
  for (int o = STEPS / 2; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) if (i < n) v[i] += __shfl_xor(v[i], o);
  if constexpr (LANES > 64) {
    constexpr int WAVES = LANES / 64;
    float* const at = slots + turn * 2 * WAVES;
    turn ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < 2; ++i) if (i < n) at[i * WAVES + wave] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (i >= n) continue;
      float s = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += at[i * WAVES + w];
      v[i] = s;
    }
  }
}

// N elements to an access, LANES lanes to a row, PER accesses to a lane: LANES * PER * N >= width.
template <int LANES> constexpr int kBlock = LANES < 256 ? 256 : LANES;

template <typename T, int N, int LANES, int PER, bool TAIL>
__global__ void __launch_bounds__(kBlock<LANES>) norm_forward_kernel(const NormArgs a) {
  constexpr int ROWS = kBlock<LANES> / LANES;
  __shared__ float slots[LANES > 64 ? 4 * (LANES / 64) : 1];
  const int lane = threadIdx.x % LANES, sub = ROWS > 1 ? threadIdx.x / LANES : 0;
  const float inv = 1.0f / float(a.width);
  float w[PER][N], b[PER][N];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
    load_params<T, N>(a.weight, a.weight_f32, c.at, c.in, 1.0f, w[p]);
    load_params<T, N>(a.bias, a.weight_f32, c.at, c.in, 0.0f, b[p]);
  }
  const int64_t step = int64_t(gridDim.x) * ROWS;
  Pack<T, N> next[PER];
  const auto fetch = [&](int64_t row) {
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
      if (row < a.rows && c.in) next[p] = load_row<T>(x, c);
    }
  };
  int turn = 0;
  // all lanes of the workgroup make the same number of turns (barriers, shuffles)
  int64_t row = int64_t(blockIdx.x) * ROWS + sub;
  fetch(row);
  for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += step, row += step) {
    float x[PER][N];
    float s[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[p][i] = c.own(i) ? next[p].get(i) : 0.0f;
        s[0] += x[p][i];
      }
    }
    fetch(row + step);
    row_sum<LANES>(s, 1, slots, turn);
    float mean = s[0] * inv;
    asm volatile("" : "+v"(mean));      // rounded: what is subtracted is what `rest` is added to (and not the product, in a fused operation)
    s[0] = s[1] = 0;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x[p][i] -= mean;
        const float d = c.own(i) ? x[p][i] : 0.0f;
        s[0] += d * d;
        if constexpr (sizeof(T) == 4) s[1] += d;
      }
    }
    row_sum<LANES>(s, sizeof(T) == 4 ? 2 : 1, slots, turn);
    // What the mean's rounding left: of 16-bit rows only where it shows, the same for all lanes of a row (always: 8192 x 14336 fp16 89 -> 98 us)
    float var = s[0] * inv;
    if (sizeof(T) == 2 && mean * mean > 256.0f * (var + a.eps)) {
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
#pragma unroll
        for (int i = 0; i < N; ++i) s[1] += c.own(i) ? x[p][i] : 0.0f;
      }
      s[0] = s[1];
      row_sum<LANES>(s, 1, slots, turn);
      s[1] = s[0];
    }
    const float rest = s[1] * inv;
    var -= rest * rest;
    const float rstd = 1.0f / sqrtf((var < 0 ? 0.0f : var) + a.eps);
    if (row >= a.rows) continue;
    if (lane == 0 && a.mean) {
      a.mean[row] = mean + rest;
      a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.out) + row * a.out_stride;
    const float shift = -rest * rstd;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
#pragma unroll
      for (int i = 0; i < N; ++i) x[p][i] = (x[p][i] * rstd + shift) * w[p][i] + b[p][i];
      store_row(y, Chunk<N, TAIL>((p * LANES + lane) * N, a.width), x[p]);
    }
  }
}

// Each workgroup sums dy * z and dy of its rows in registers, column by column, and leaves them in `partial`: no atomics, the sums do
// not depend on timing.
template <typename T, int N, int LANES, int PER, bool TAIL>
__global__ void __launch_bounds__(kBlock<LANES>) norm_backward_kernel(const NormArgs a) {
  constexpr int ROWS = kBlock<LANES> / LANES;
  constexpr int SPAN = LANES * PER * N;     // columns that a row's lanes cover
  // The next row's x is loaded ahead, its dy as well where the registers allow: 6001 x 10935 fp16 179 us with, 133 without; 8192 x 14336 (no
  // tail) 143 with, 163 without; 4320 x 4397 40 with, 43 without.
  constexpr bool AHEAD = 3 * PER * N + int(sizeof(T)) * PER * N + (TAIL ? 32 : 0) <= (LANES > 256 ? 160 : 256);
  __shared__ float slots[LANES > 64 ? 4 * (LANES / 64) : 1];
  __shared__ float shared_sums[ROWS > 1 ? ROWS * SPAN : 1];
  const int lane = threadIdx.x % LANES, sub = ROWS > 1 ? threadIdx.x / LANES : 0;
  const float inv = 1.0f / float(a.width);
  float w[PER][N], dw[PER][N], db[PER][N];
#pragma unroll
  for (int p = 0; p < PER; ++p) {
    const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
    load_params<T, N>(a.weight, a.weight_f32, c.at, c.in, 1.0f, w[p]);
#pragma unroll
    for (int i = 0; i < N; ++i) dw[p][i] = db[p][i] = 0.0f;
  }
  const int64_t step = int64_t(gridDim.x) * ROWS;
  Pack<T, N> next_x[PER], next_dy[PER];
  float next_mean = 0, next_rstd = 0;
  const auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const T* dy = static_cast<const T*>(a.dy) + row * a.dy_stride;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
      if (c.in) {
        next_x[p] = load_row<T>(x, c);
        if constexpr (AHEAD) next_dy[p] = load_row<T>(dy, c);
      }
    }
    next_mean = a.mean[row];
    next_rstd = a.rstd[row];
  };
  int turn = 0;
  int64_t row = int64_t(blockIdx.x) * ROWS + sub;
  fetch(row);
  for (int64_t first = int64_t(blockIdx.x) * ROWS; first < a.rows; first += step, row += step) {
    const bool live = row < a.rows;
    const float mean = next_mean, rstd = next_rstd;
    Pack<T, N> x[PER], dy[PER];
    if constexpr (!AHEAD) {
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
        if (live && c.in) next_dy[p] = load_row<T>(static_cast<const T*>(a.dy) + row * a.dy_stride, c);
      }
    }
    float s[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
      x[p] = next_x[p];
      dy[p] = next_dy[p];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const bool in = live && c.own(i);
        const float z = in ? (x[p].get(i) - mean) * rstd : 0.0f, d = in ? dy[p].get(i) : 0.0f, g = d * w[p][i];
        s[0] += g;
        s[1] += g * z;
        dw[p][i] += d * z;
        db[p][i] += d;
      }
      if constexpr (PER >= 4) __builtin_amdgcn_sched_barrier(0);      // chunk by chunk, for want of registers
    }
    fetch(row + step);
    if (!a.out) continue;
    row_sum<LANES>(s, 2, slots, turn);
    const float c1 = s[0] * inv, c2 = s[1] * inv;
    if (!live) continue;
    T* dx = static_cast<T*>(a.out) + row * a.out_stride;
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      // 16-bit values are kept as they were loaded and widened again, not kept twice as wide: rows of 14336 209 -> 143 us, with what follows
      // from it (next to no scratch memory, both operands ahead)
      if constexpr (sizeof(T) == 2 && N > 1) asm volatile("" : "+v"(x[p].w), "+v"(dy[p].w));
      float v[N];
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = rstd * (dy[p].get(i) * w[p][i] - c1 - (x[p].get(i) - mean) * rstd * c2);
      store_row(dx, Chunk<N, TAIL>((p * LANES + lane) * N, a.width), v);
      if constexpr (PER >= 4) __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (!a.partial) return;
  float* const mine = a.partial + int64_t(blockIdx.x) * 2 * a.width;
  const auto leave = [&](const float (&v)[PER][N], float* to) {
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int p = 0; p < PER; ++p)
        store_row(to, Chunk<N, TAIL>((p * LANES + lane) * N, a.width), v[p]);
    } else {
      __syncthreads();
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const Chunk<N, TAIL> c((p * LANES + lane) * N, a.width);
#pragma unroll
        for (int i = 0; i < N; ++i) if (c.own(i)) shared_sums[sub * SPAN + c.at + i] = v[p][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.width; c += kBlock<LANES>) {
        float s = 0;
        for (int r = 0; r < ROWS; ++r) s += shared_sums[r * SPAN + c];
        to[c] = s;
      }
    }
  };
  leave(dw, mine);
  leave(db, mine + a.width);
}

// Sums of the workgroups' partial sums: 64 columns to a workgroup, 16 waves share the rows of `partial`.
template <typename W>
__global__ void __launch_bounds__(1024) norm_reduce_kernel(const float* __restrict__ partial, int parts, int width, W* __restrict__ dw,
                                                           W* __restrict__ db) {
  constexpr int AHEAD = 16;
  __shared__ float sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + lane;     // of 2 * width: dw, then db
  float s[4] = {0, 0, 0, 0};
  if (c < 2 * width)
    for (int r = wave; r < parts; r += 16 * AHEAD)
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)      // past the end the last part again, and not used: so many loads are on their way at once
        s[u % 4] += r + 16 * u < parts ? partial[int64_t(min(r + 16 * u, parts - 1)) * 2 * width + c] : 0.0f;
  sums[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (wave || c >= 2 * width) return;
  float total = 0;
#pragma unroll
  for (int w = 0; w < 16; ++w) total += sums[w][lane];
  W* const out = c < width ? dw : db;
  if (out) out[c < width ? c : c - width] = rounded<W>(total);
}

// ---------------------------------------------------------------- host side
// Calls f(N, LANES, PER) as constants for rows of `width` elements.
template <typename T, int LONG, typename F>
void by_shape(int width, F&& f) {
#define GMM_SHAPE(n, lanes, per) \
  if (width <= (n) * (lanes) * (per)) return f(std::integral_constant<int, n>{}, std::integral_constant<int, lanes>{}, std::integral_constant<int, per>{});
  constexpr int V = kVector<T>;
  if (width < V) {
    GMM_SHAPE(1, 8, 1)
  }
  GMM_SHAPE(V, 8, 1)
  GMM_SHAPE(V, 16, 1)
  GMM_SHAPE(V, 32, 1)
  GMM_SHAPE(V, 64, 1)
  GMM_SHAPE(V, 64, 2)
  GMM_SHAPE(V, 256, 1)
  GMM_SHAPE(V, 256, 2)
  GMM_SHAPE(V, 256, 4)
  if constexpr (V == 8) {
    GMM_SHAPE(V, LONG, 2048 / LONG)
  } else {
    GMM_SHAPE(V, 512, 4)
    GMM_SHAPE(V, LONG, 4096 / LONG)
  }
#undef GMM_SHAPE
}

// Workgroups of the backward kernel, each of which leaves 2 * width sums: two to a compute unit.
int64_t backward_groups(int64_t rows) {
  const int64_t most = 2 * gmm_num_cus();
  return rows < most ? rows : most;
}

template <typename T>
int launch_norm(const NormArgs& a, bool backward, int64_t groups_used, hipStream_t stream) {
  const auto tail = [&](auto n, auto&& launch) {
    if constexpr (decltype(n)::value > 1) {
      if (a.width % decltype(n)::value) return launch(std::true_type{});
    }
    launch(std::false_type{});
  };
  if (backward) {
    by_shape<T, 512>(a.width, [&](auto n, auto lanes, auto per) {
      constexpr int N = decltype(n)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
      tail(n, [&](auto t) {
        // workgroups that a row at a time would need and several rows at a time do not: their sums are zero
        hipLaunchKernelGGL((norm_backward_kernel<T, N, LANES, PER, decltype(t)::value>), dim3(unsigned(groups_used)), dim3(kBlock<LANES>), 0, stream, a);
      });
    });
  } else {
    // the longest rows take 1024 lanes, which here have registers enough: 4096 x 16384 bf16 61 -> 51 us; backward 131 -> 158, spilled
    by_shape<T, 1024>(a.width, [&](auto n, auto lanes, auto per) {
      constexpr int N = decltype(n)::value, LANES = decltype(lanes)::value, PER = decltype(per)::value;
      constexpr int block = kBlock<LANES>, rows_at_once = block / LANES;
      const int64_t groups = (a.rows + rows_at_once - 1) / rows_at_once, most = int64_t(gmm_num_cus()) * (2048 / block);
      tail(n, [&](auto t) {
        hipLaunchKernelGGL((norm_forward_kernel<T, N, LANES, PER, decltype(t)::value>), dim3(unsigned(groups < most ? groups : most)), dim3(block), 0, stream, a);
      });
    });
  }
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

bool stride_fits(int64_t stride, int64_t rows, int64_t width) { return stride >= width || rows <= 1; }

int check_norm(int64_t rows, int64_t width, int32_t dtype, int32_t weight_dtype) {
  if (rows < 0 || width < 0 || width > kMaxWidth) return GMM_ERR_BAD_ARGUMENT;
  if (dtype < GMM_DT_BF16 || dtype > GMM_DT_F32 || (weight_dtype != dtype && weight_dtype != GMM_DT_F32)) return GMM_ERR_UNSUPPORTED;
  return GMM_OK;
}

}  // namespace

extern "C" {

int gmm_layer_norm(const void* x, const void* weight, const void* bias, void* y, float* mean, float* rstd, int64_t rows, int64_t width,
                   int64_t x_stride, int64_t y_stride, float eps, int32_t dtype, int32_t weight_dtype, void* stream) {
  const int bad = check_norm(rows, width, dtype, weight_dtype);
  if (bad) return bad;
  if (rows == 0 || width == 0) return GMM_OK;
  if (!x || !y || !mean != !rstd || !stride_fits(x_stride, rows, width) || !stride_fits(y_stride, rows, width)) return GMM_ERR_BAD_ARGUMENT;
  NormArgs a{};
  a.x = x; a.weight = weight; a.bias = bias; a.out = y; a.mean = mean; a.rstd = rstd;
  a.rows = rows; a.width = int32_t(width); a.x_stride = x_stride; a.out_stride = y_stride;
  a.eps = eps; a.weight_f32 = weight_dtype == GMM_DT_F32;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GMM_DT_BF16) return launch_norm<Bf16>(a, false, 0, s);
  if (dtype == GMM_DT_F16) return launch_norm<F16>(a, false, 0, s);
  return launch_norm<float>(a, false, 0, s);
}

int64_t gmm_layer_norm_workspace_bytes(int64_t rows, int64_t width) {
  if (rows < 0 || width < 0 || width > kMaxWidth) return -1;
  return backward_groups(rows) * 2 * width * int64_t(sizeof(float));
}

int gmm_layer_norm_backward(const void* dy, const void* x, const void* weight, const float* mean, const float* rstd, void* dx,
                            void* dweight, void* dbias, int64_t rows, int64_t width, int64_t dy_stride, int64_t x_stride,
                            int64_t dx_stride, int32_t dtype, int32_t weight_dtype, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  const int bad = check_norm(rows, width, dtype, weight_dtype);
  if (bad) return bad;
  if (width == 0 || (!dx && !dweight && !dbias)) return GMM_OK;
  const bool sums = dweight || dbias;
  if (rows > 0 && (!x || !dy || !mean || !rstd || !stride_fits(x_stride, rows, width) || !stride_fits(dy_stride, rows, width) ||
                   (dx && !stride_fits(dx_stride, rows, width)))) return GMM_ERR_BAD_ARGUMENT;
  if (sums && (workspace_bytes < gmm_layer_norm_workspace_bytes(rows, width) || (rows > 0 && !workspace))) return GMM_ERR_WORKSPACE;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t groups = backward_groups(rows);
  if (rows > 0) {
    NormArgs a{};
    a.x = x; a.dy = dy; a.weight = weight; a.out = dx; a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd);
    a.partial = sums ? static_cast<float*>(workspace) : nullptr;
    a.rows = rows; a.width = int32_t(width); a.x_stride = x_stride; a.dy_stride = dy_stride; a.out_stride = dx_stride;
    a.weight_f32 = weight_dtype == GMM_DT_F32;
    int rc;
    if (dtype == GMM_DT_BF16) rc = launch_norm<Bf16>(a, true, groups, s);
    else if (dtype == GMM_DT_F16) rc = launch_norm<F16>(a, true, groups, s);
    else rc = launch_norm<float>(a, true, groups, s);
    if (rc != GMM_OK) return rc;
  }
  if (sums) {
    const dim3 grid(unsigned((2 * width + 63) / 64)), block(1024);
    const float* partial = static_cast<const float*>(workspace);
    const auto reduce = [&](auto* dw, auto* db) {
      hipLaunchKernelGGL((norm_reduce_kernel<std::remove_pointer_t<decltype(dw)>>), grid, block, 0, s, partial, int(groups), int(width), dw, db);
    };
    if (weight_dtype == GMM_DT_BF16) reduce(static_cast<Bf16*>(dweight), static_cast<Bf16*>(dbias));
    else if (weight_dtype == GMM_DT_F16) reduce(static_cast<F16*>(dweight), static_cast<F16*>(dbias));
    else reduce(static_cast<float*>(dweight), static_cast<float*>(dbias));
  }
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

}  // extern "C"
