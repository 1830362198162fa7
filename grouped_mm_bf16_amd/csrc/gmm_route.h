// Top-k choice of one token by one wave, for the routing (gmm_moe.hip) and the kernels that route for themselves (gmm_few.hip).
#pragma once
#include "gmm_elem.h"

namespace gmm {

// ---------------------------------------------------------------- wave helpers (64 lanes)
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
// Maximum over the wave with data-parallel-primitive moves: prefix maxima inside each row of 16 lanes
// (row_shr 1, 2, 4, 8), then lane 15 of a row into the next row (row_bcast15 into rows 1 and 3) and lane 31
// into rows 2 and 3 (row_bcast31); lane 63 ends up with the maximum of all 64.  Lanes a move does not reach
// take 0, the identity.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#define GMM_DPP_UMAX(ctrl, rows)                                                        \
  {                                                                                     \
    const uint32_t t = uint32_t(__builtin_amdgcn_update_dpp(0, int(v), ctrl, rows, 0xf, false)); \
    v = t > v ? t : v;                                                                  \
  }
  GMM_DPP_UMAX(0x111, 0xf)
  GMM_DPP_UMAX(0x112, 0xf)
  GMM_DPP_UMAX(0x114, 0xf)
  GMM_DPP_UMAX(0x118, 0xf)
  GMM_DPP_UMAX(0x142, 0xa)
  GMM_DPP_UMAX(0x143, 0xc)
#undef GMM_DPP_UMAX
  return uint32_t(__builtin_amdgcn_readlane(int(v), 63));
}

// fp32 -> uint32 whose unsigned order is the numeric order (NaN with a clear sign bit sorts above +inf)
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);   // -0 becomes +0: the two compare equal
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// ---------------------------------------------------------------- routing: top-k and weights
// One wave per token.  Choice j of token t is slot t * k + j.  Ties go to the lower expert index (a stable
// descending sort).  weight = softmax over the chosen k logits (renorm) or over all E logits.
// Lane l holds the order keys of experts l, l + 64, ...: kPer of them, in registers (in LDS, with an index loop per round, a
// token's 8 of 128 choices took a wave 2.3 us).  The wave's best key is found first, then the first expert that holds it.  A
// choice looks at all kPer keys, there or not: 4096 tokens with 32 of 260 experts take 79 us with 16 of them, 52 with 8 (64 from
// LDS).
template <typename T, int kPer>
struct MoeTopk {
  uint32_t key[kPer];   // 0 beyond the last expert

  __device__ __forceinline__ void load(const T* row, int E, int lane) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + (i << 6);
      key[i] = e < E ? order_key(widen(row[e])) : 0u;
    }
  }

  // Lane j < k returns choice j and its weight.
  __device__ __forceinline__ void choose(int E, int k, int renorm, int lane, int& my_e, float& weight) const {
    uint32_t free_keys = 0, my_key = 0, top_key = 0;   // free_keys: bit i: the lane's i-th expert exists and is not chosen yet
#pragma unroll
    for (int i = 0; i < kPer; ++i) free_keys |= lane + (i << 6) < E ? 1u << i : 0u;
    my_e = 0;
    for (int j = 0; j < k; ++j) {
      uint32_t best = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint32_t v = (free_keys >> i) & 1u ? key[i] : 0u;
        best = v > best ? v : best;
      }
      const uint32_t win = wave_umax(best);
      int e_win = 0;
      bool found = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const uint64_t holders = __ballot(((free_keys >> i) & 1u) && key[i] == win);
        if (!found && holders) {
          e_win = (i << 6) + __ffsll((unsigned long long)holders) - 1;
          found = true;
        }
      }
      if ((e_win & 63) == lane) free_keys &= ~(1u << (e_win >> 6));
      if (lane == j) { my_e = e_win; my_key = win; }
      if (j == 0) top_key = win;
    }
    // exp(x - m) with an infinite maximum m (a +inf logit, or a row of -inf: every expert masked) is the limit
    // of the softmax: all weight, in equal shares, on the entries that equal the maximum (inf - inf is NaN)
    const float m = key_value(top_key);
    const bool inf_max = (__float_as_uint(m) & 0x7fffffffu) == 0x7f800000u;
    const float p = lane < k ? (inf_max ? (my_key == top_key ? 1.0f : 0.0f) : __expf(key_value(my_key) - m)) : 0.0f;
    float den;
    if (renorm) {
      den = wave_sum(p);
    } else {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        if (lane + (i << 6) < E) s += inf_max ? (key[i] == top_key ? 1.0f : 0.0f) : __expf(key_value(key[i]) - m);
      den = wave_sum(s);
    }
    weight = p / den;
  }
};

}  // namespace gmm
