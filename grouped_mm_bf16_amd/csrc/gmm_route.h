// Top-k choice of one token by one wave, for the routing (gmm_moe.hip) and the kernels that route for themselves (gmm_few.hip,
// gmm_int8_few.hip).
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

// Slots (choices of all tokens; at most a wave's lanes) and experts up to which a workgroup routes for itself, one wave to a token.  1 token, 1 of
// 8 experts of 3674 -> 2 x 151 18 us, with a launch for the routing 20; 64 slots, 4 of 8 experts of 432 -> 2 x 10752 87 and 81.
constexpr int kRouteSlots = 32, kRouteKeys = 4, kRouteExperts = 64 * kRouteKeys;

// Routing by every workgroup for itself: up to kRouteSlots slots, kRouteExperts experts, a wave to a token.  The first workgroup leaves the
// results for the kernels behind.  Rows are sorted by expert, stably, as gmm_moe_route has them.
struct RouteHere {
  const void* logits;
  int64_t logits_ld;
  int32_t* offs;
  int32_t* token_rows;
  float* slot_weight;
  int32_t tokens, experts, top_k, slots, renormalize, logits_dtype;
};

struct FewRouting {
  int32_t expert[kRouteSlots];
  float weight[kRouteSlots];
  int32_t token[kRouteSlots];     // of a row of the expert that this workgroup looks for
  int32_t found, row0, rows;
};

template <int WAVES>
__device__ __forceinline__ bool route_here(const RouteHere& a, FewRouting& r, int which, int& expert, int& row0, int& rows) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int t = wave; t < a.tokens; t += WAVES) {
    int e;
    float w;
    const auto choose = [&](auto zero) {
      using L = decltype(zero);
      MoeTopk<L, kRouteKeys> token;
      token.load(static_cast<const L*>(a.logits) + t * a.logits_ld, a.experts, lane);
      token.choose(a.experts, a.top_k, a.renormalize, lane, e, w);
    };
    if (a.logits_dtype == GMM_DT_BF16) choose(Bf16{});
    else if (a.logits_dtype == GMM_DT_F16) choose(F16{});
    else choose(0.0f);
    if (lane < a.top_k) {
      r.expert[t * a.top_k + lane] = e;
      r.weight[t * a.top_k + lane] = w;
    }
  }
  __syncthreads();
  if (wave == 0) {
    const int e = lane < a.slots ? r.expert[lane] : a.experts;
    int row = 0, before = 0;     // slots ahead of the lane's; experts ahead of its own
    bool head = lane < a.slots;  // the first slot of its expert
    for (int s = 0; s < a.slots; ++s) {
      const int other = __builtin_amdgcn_readlane(e, s);
      row += other < e || (other == e && s < lane);
      head = head && !(other == e && s < lane);
    }
    const uint64_t heads = __ballot(head);
    for (uint64_t todo = heads; todo; todo &= todo - 1)
      before += __builtin_amdgcn_readlane(e, __ffsll(static_cast<unsigned long long>(todo)) - 1) < e;
    const uint64_t it = __ballot(head && before == which);
    if (it) {
      const int at = __ffsll(static_cast<unsigned long long>(it)) - 1;
      const int mine = __builtin_amdgcn_readlane(e, at), first = __builtin_amdgcn_readlane(row, at);
      const uint64_t same = __ballot(e == mine);
      if (e == mine) r.token[row - first] = lane / a.top_k;
      if (lane == 0) { r.expert[0] = mine; r.row0 = first; r.rows = __popcll(same); }
    }
    if (lane == 0) r.found = it != 0;
    if (blockIdx.x == 0 && lane < a.slots) {
      a.token_rows[lane] = row;
      a.slot_weight[lane] = r.weight[lane];
    }
    if (blockIdx.x == 0)
      for (int i = lane; i < a.experts; i += 64) {
        int to = 0;
        for (int s = 0; s < a.slots; ++s) to += __builtin_amdgcn_readlane(e, s) <= i;
        a.offs[i] = to;
      }
  }
  __syncthreads();
  if (!r.found) return false;
  expert = __builtin_amdgcn_readfirstlane(r.expert[0]);
  row0 = __builtin_amdgcn_readfirstlane(r.row0);
  rows = __builtin_amdgcn_readfirstlane(r.rows);
  return true;
}

}  // namespace gmm
