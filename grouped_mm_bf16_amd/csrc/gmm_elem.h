// Elements of the operators around the grouped product: 16-bit and fp32 values as they lie in memory, read and rounded 8 (16-bit)
// or 4 (fp32) to a 16-byte access, or one by one where nothing is aligned.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gmm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

struct Bf16 { uint16_t bits; };
struct F16 { uint16_t bits; };

__device__ __forceinline__ float widen(Bf16 x) { return __uint_as_float(uint32_t(x.bits) << 16); }
__device__ __forceinline__ float widen(F16 x) { return float(__builtin_bit_cast(_Float16, x.bits)); }
__device__ __forceinline__ float widen(float x) { return x; }

// Round to nearest even (v_cvt_pk_bf16_f32, v_cvt_f16_f32).
template <typename T> __device__ __forceinline__ T rounded(float f);
template <> __device__ __forceinline__ Bf16 rounded<Bf16>(float f) { return Bf16{__builtin_bit_cast(uint16_t, static_cast<__bf16>(f))}; }
template <> __device__ __forceinline__ F16 rounded<F16>(float f) { return F16{__builtin_bit_cast(uint16_t, static_cast<_Float16>(f))}; }
template <> __device__ __forceinline__ float rounded<float>(float f) { return f; }

// N adjacent elements as they lie in memory: one, or a 16-byte aligned vector, whose 16-bit elements stay two to a register.
template <typename T, int N> struct alignas(N > 1 ? 16 : sizeof(T)) Pack {
  T v[N];
  __device__ __forceinline__ float get(int i) const { return widen(v[i]); }
  static __device__ __forceinline__ Pack of(const float (&f)[N]) {
    Pack p;
#pragma unroll
    for (int i = 0; i < N; ++i) p.v[i] = rounded<T>(f[i]);
    return p;
  }
};

template <typename T> struct alignas(16) Half8 {
  u32x4 w;
  __device__ __forceinline__ float get(int i) const { return widen(T{uint16_t(w[i / 2] >> 16 * (i & 1))}); }
  static __device__ __forceinline__ Half8 of(const float (&f)[8]) {
    Half8 p;
#pragma unroll
    for (int q = 0; q < 4; ++q) p.w[q] = uint32_t(rounded<T>(f[2 * q]).bits) | uint32_t(rounded<T>(f[2 * q + 1]).bits) << 16;
    return p;
  }
};
template <> struct Pack<Bf16, 8> : Half8<Bf16> {
  __device__ Pack() = default;
  __device__ __forceinline__ Pack(const Half8<Bf16>& h) : Half8<Bf16>(h) {}
};
template <> struct Pack<F16, 8> : Half8<F16> {
  __device__ Pack() = default;
  __device__ __forceinline__ Pack(const Half8<F16>& h) : Half8<F16>(h) {}
};

// What lies at any address: the hardware asks for no alignment.
template <typename V>
__device__ __forceinline__ V unaligned(const void* p) {
  V v;
  __builtin_memcpy(&v, p, sizeof(V));
  return v;
}

template <typename T> constexpr int kVector = 16 / int(sizeof(T));

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace gmm

// Compute units of the current device (a multiple of 8), 0 if there is none (gmm_api.hip).
int gmm_num_cus();
