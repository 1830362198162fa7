// Dropout from a counter-based generator (declared in include/grouped_mm_hip.h): out = residual + x * [bits >= limit] * 65536 / (65536 - limit).
// The mask is never stored: the backward pass makes the same bits again.  Element i of x, rows one after the other, has bits 16 (i % 8) ..
// of block i / 8 of Philox 4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers, as easy as 1, 2, 3, 2011): key rng[0], counter
// (i / 8, rng[1]), the call's site in the counter's bits 48 .. 63.  16 bits to an element make a block's ten rounds, 20 products of 32 bits,
// serve eight elements: with 32 bits each the rounds, not memory, would bound 16-bit rows.  What is read or written once goes past the caches.
//   16384 x 4096 bf16   with a residual 63 us (6.4 TB/s), its gradient 43 (6.2)
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_elem.h"

namespace {

using namespace gmm;

constexpr int kBlock = 256;

struct DropoutArgs {
  const void* x;
  const void* residual;    // null: none
  void* out;
  const int64_t* rng;      // key, offset
  int64_t* used;           // gets what rng held (null: not wanted)
  int64_t rows, width, x_stride, residual_stride, out_stride;
  uint32_t limit, site;
  float factor;
};

struct Bits { uint32_t w[4]; };

__device__ __forceinline__ Bits philox(uint64_t block, uint64_t offset, uint64_t key) {
  uint32_t c0 = uint32_t(block), c1 = uint32_t(block >> 32), c2 = uint32_t(offset), c3 = uint32_t(offset >> 32);
  uint32_t k0 = uint32_t(key), k1 = uint32_t(key >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p0 = uint64_t(c0) * 0xD2511F53u, p1 = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(p1 >> 32) ^ c1 ^ k0;
    c1 = uint32_t(p1);
    c2 = uint32_t(p0 >> 32) ^ c3 ^ k1;
    c3 = uint32_t(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Bits{{c0, c1, c2, c3}};
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  constexpr int N = kVector<T>;
#pragma unroll
  for (int q = 0; q < 8 / N; ++q) {
    const Pack<T, N> a = stream_in<Pack<T, N>, true>(p + q * N);
#pragma unroll
    for (int i = 0; i < N; ++i) v[q * N + i] = a.get(i);
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  constexpr int N = kVector<T>;
#pragma unroll
  for (int q = 0; q < 8 / N; ++q) {
    float part[N];
#pragma unroll
    for (int i = 0; i < N; ++i) part[i] = v[q * N + i];
    stream_out<true>(p + q * N, Pack<T, N>::of(part));
  }
}

// A thread takes eight elements that share a block of random bits.  FLAT: all tensors are one row.
template <typename T, bool FLAT>
__global__ void __launch_bounds__(kBlock) dropout_kernel(const DropoutArgs a) {
  const uint64_t key = uint64_t(a.rng[0]), offset = uint64_t(a.rng[1]);
  if (a.used && blockIdx.x == 0 && threadIdx.x == 0) {
    a.used[0] = int64_t(key);
    a.used[1] = int64_t(offset);
  }
  const T* x = static_cast<const T*>(a.x);
  const T* residual = static_cast<const T*>(a.residual);
  T* out = static_cast<T*>(a.out);
  const int64_t n = a.rows * a.width, blocks = (n + 7) / 8;
  for (int64_t b = int64_t(blockIdx.x) * kBlock + threadIdx.x; b < blocks; b += int64_t(gridDim.x) * kBlock) {
    int64_t r = 0, c = 8 * b;
    if constexpr (!FLAT) {
      r = n <= 0xffffffff ? uint32_t(8 * b) / uint32_t(a.width) : 8 * b / a.width;
      c = 8 * b - r * a.width;
    }
    const Bits bits = philox(uint64_t(b) | uint64_t(a.site) << 48, offset, key);
    const auto kept = [&](int i) { return (i & 1 ? bits.w[i / 2] >> 16 : bits.w[i / 2] & 0xffffu) >= a.limit; };
    if (c + 8 <= a.width) {
      float v[8], s[8];
      load8(x + r * a.x_stride + c, v);
      if (residual) load8(residual + r * a.residual_stride + c, s);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = kept(i) ? v[i] * a.factor : 0.0f;
        if (residual) v[i] += s[i];
      }
      store8(out + r * a.out_stride + c, v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (8 * b + i < n) {
          float v = kept(i) ? widen(x[r * a.x_stride + c]) * a.factor : 0.0f;
          if (residual) v += widen(residual[r * a.residual_stride + c]);
          out[r * a.out_stride + c] = rounded<T>(v);
        }
        if (++c == a.width) { c = 0; ++r; }
      }
    }
  }
}

bool stride_fits(int64_t stride, int64_t rows, int64_t width) { return stride >= width || rows <= 1; }

}  // namespace

extern "C" int gmm_dropout(const void* x, const void* residual, void* out, const int64_t* rng, int64_t* used, int64_t rows, int64_t width,
                           int64_t x_stride, int64_t residual_stride, int64_t out_stride, int32_t limit, int32_t site, int32_t dtype, void* stream) {
  if (rows < 0 || width < 0 || limit < 0 || limit > 65536 || site < 0 || site > 65535) return GMM_ERR_BAD_ARGUMENT;
  if (width > 0 && rows > (int64_t(1) << 50) / width) return GMM_ERR_BAD_ARGUMENT;      // block numbers stay below the site's bits
  if (dtype < GMM_DT_BF16 || dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
  if (!rng) return GMM_ERR_BAD_ARGUMENT;
  if (rows == 0 || width == 0) rows = width = 0;
  else if (!x || !out || !stride_fits(x_stride, rows, width) || !stride_fits(out_stride, rows, width) ||
           (residual && !stride_fits(residual_stride, rows, width))) return GMM_ERR_BAD_ARGUMENT;
  if (rows == 0 && !used) return GMM_OK;
  DropoutArgs a{};
  a.x = x; a.residual = residual; a.out = out; a.rng = rng; a.used = used; a.rows = rows; a.width = width;
  a.x_stride = x_stride; a.residual_stride = residual_stride; a.out_stride = out_stride;
  a.limit = uint32_t(limit); a.site = uint32_t(site);
  a.factor = limit < 65536 ? 65536.0f / float(65536 - limit) : 0.0f;
  const bool flat = rows <= 1 || (x_stride == width && out_stride == width && (!residual || residual_stride == width));
  if (flat) { a.width = rows * width; a.rows = 1; }
  const int64_t blocks = (rows * width + 7) / 8, most = int64_t(gmm_num_cus()) * 32;
  int64_t groups = (blocks + kBlock - 1) / kBlock;
  groups = groups < 1 ? 1 : groups > most ? most : groups;
  const auto launch = [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    const dim3 grid{unsigned(groups)}, block(kBlock);
    if (flat) hipLaunchKernelGGL((dropout_kernel<T, true>), grid, block, 0, static_cast<hipStream_t>(stream), a);
    else hipLaunchKernelGGL((dropout_kernel<T, false>), grid, block, 0, static_cast<hipStream_t>(stream), a);
  };
  if (dtype == GMM_DT_BF16) launch(static_cast<Bf16*>(nullptr));
  else if (dtype == GMM_DT_F16) launch(static_cast<F16*>(nullptr));
  else launch(static_cast<float*>(nullptr));
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}
