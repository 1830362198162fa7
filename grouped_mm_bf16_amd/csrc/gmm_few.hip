// A mixture-of-experts layer for a few tokens (gmm_moe_few in include/grouped_mm_hip.h):
//   out[t] = sum over the choices j of w_tj * act(x[t] @ w_up[e_tj]) @ w_down[e_tj]
// Routing as gmm_moe_route, then every chosen expert's matrices are read once, past a few rows (gmm_skinny.h).  Reading them bounds
// it.  Between the two products the activations stay in 32 bits (two 16-bit values each), the second products in fp32: the result is
// rounded once.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_skinny.h"

namespace {

using namespace gmm;

constexpr int kMaxTokens = 64;
constexpr int kWaves = 4, kThreads = 64 * kWaves;

struct FewArgs {
  const void* x;
  const void* w;            // w_up or w_down
  const int32_t* offs;      // routing
  const int32_t* row_token;
  const int32_t* token_rows;
  const float* slot_weight;
  void* act;                // [2][slots][act_ld]: high and low halves
  float* y;                 // [parts][slots][H]
  void* out;
  int64_t w_sg;             // elements from one expert to the next
  int64_t x_ld, out_ld;
  uint32_t w_sk, w_sn;      // elements
  uint32_t w_bytes;         // of one expert's matrix
  int32_t tokens, experts, top_k, slots, H, inner, act_ld;
  int32_t tiles, parts, k_part;   // strips of columns; parts along k and their length
  int32_t kind;
};

// The `which`-th expert that has rows: its number, first row, number of rows.
__device__ __forceinline__ bool find_expert(const FewArgs& a, int which, int& expert, int& row0, int& rows) {
  const int lane = threadIdx.x & 63;
  for (int base = 0; base < a.experts; base += 64) {
    const int e = base + lane;
    const int to = e < a.experts ? a.offs[e] : 0, from = e < a.experts && e > 0 ? a.offs[e - 1] : 0;
    const uint64_t used = __ballot(to > from);
    const int n = __popcll(used);
    if (which < n) {
      const uint64_t it = __ballot(to > from && __popcll(used & ((uint64_t(1) << lane) - 1)) == which);
      const int at = __ffsll(static_cast<unsigned long long>(it)) - 1;
      expert = base + at;
      row0 = __builtin_amdgcn_readlane(from, at);
      rows = __builtin_amdgcn_readlane(to, at) - row0;
      return true;
    }
    which -= n;
  }
  return false;
}

// act[r] = act(x[token of row r] @ w_up[e]).  GLU: a strip is 8 * FR gate columns and their partners.
template <typename T, int LAY, int MF, bool GLU>
__global__ void __launch_bounds__(kThreads, MF <= 2 && LAY != GMM_W_ANY ? 2 : 1) few_up_kernel(const FewArgs a) {
  using S = Strip<T, LAY, MF, 1>;
  constexpr int FR = S::FR, OUT = GLU ? 8 * FR : 16 * FR;
  __shared__ SkinnyShared<S, kWaves> shared;
  int expert, row0, rows;
  if (!find_expert(a, blockIdx.x / a.tiles, expert, row0, rows)) return;
  const int tile = blockIdx.x % a.tiles;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.w_buf = buffer(static_cast<const T*>(a.w) + expert * a.w_sg, a.w_bytes);
  s.a_buf = buffer(a.x, uint32_t((int64_t(a.tokens - 1) * a.x_ld + a.H) * 2));
  s.a_plane = 0;
  const int c = tile * OUT;     // of the result
  if constexpr (GLU) {
    if (a.kind == GMM_ACT_SWIGLU) s.set_columns(c, a.inner - c, a.w_sk, a.w_sn, OUT, a.inner + c);
    else s.set_columns(c / 64 * 128 + c % 64, a.inner - c, a.w_sk, a.w_sn, OUT, c / 64 * 128 + c % 64 + 64);
  } else {
    s.set_columns(c, a.inner - c, a.w_sk, a.w_sn);
  }
  s.set_rows([&](int r) { return r < rows ? uint32_t(a.row_token[row0 + r]) * uint32_t(a.x_ld) * 2 : kNowhere; });
  f32x4 acc[MF][FR];
  clear(acc);
  s.template run<kWaves>(rows, 0, a.H, wave, acc);

  T* const high = static_cast<T*>(a.act);
  T* const low = high + int64_t(a.slots) * a.act_ld;
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (16 * m >= rows) break;
    __syncthreads();
    shared.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = threadIdx.x; u < OUT * 4; u += kThreads) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.inner) continue;
      const f32x4 h = shared.sums.get(S::product_of(oc), S::lane_of(oc), og);
      const f32x4 partner = GLU ? shared.sums.get(S::product_of(OUT + oc), S::lane_of(OUT + oc), og) : f32x4{1, 1, 1, 1};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 16 * m + 4 * og + v;
        if (r >= rows) break;
        const float value = h[v] / (1.0f + __expf(-h[v])) * partner[v];
        const int64_t to = int64_t(row0 + r) * a.act_ld + col;
        split(value, high[to], low[to]);
      }
    }
  }
}

// y[part][r] = act[r] @ w_down[e], over the part's range of k.
template <typename T, int LAY, int MF>
__global__ void __launch_bounds__(kThreads, MF <= 2 && LAY != GMM_W_ANY ? 2 : 1) few_down_kernel(const FewArgs a) {
  using S = Strip<T, LAY, MF, 2>;
  constexpr int FR = S::FR, OUT = 16 * FR;
  __shared__ SkinnyShared<S, kWaves> shared;
  const int part = blockIdx.x % a.parts, item = blockIdx.x / a.parts, tile = item % a.tiles;
  int expert, row0, rows;
  if (!find_expert(a, item / a.tiles, expert, row0, rows)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.w_buf = buffer(static_cast<const T*>(a.w) + expert * a.w_sg, a.w_bytes);
  s.a_plane = uint32_t(a.slots) * a.act_ld * 2;
  s.a_buf = buffer(a.act, 2 * s.a_plane);
  s.set_columns(tile * OUT, a.H - tile * OUT, a.w_sk, a.w_sn);
  s.set_rows([&](int r) { return r < rows ? uint32_t(row0 + r) * a.act_ld * 2 : kNowhere; });
  f32x4 acc[MF][FR];
  clear(acc);
  s.template run<kWaves>(rows, part * a.k_part, min(a.inner, (part + 1) * a.k_part), wave, acc);

  float* const y = a.y + int64_t(part) * a.slots * a.H;
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (16 * m >= rows) break;
    __syncthreads();
    shared.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = threadIdx.x; u < OUT * 4; u += kThreads) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.H) continue;
      const f32x4 h = shared.sums.get(S::product_of(oc), S::lane_of(oc), og);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 16 * m + 4 * og + v;
        if (r < rows) y[int64_t(row0 + r) * a.H + col] = h[v];
      }
    }
  }
}

// out[t] = sum over j of weight * sum over the parts of y, in that order.
template <typename T>
__global__ void __launch_bounds__(kThreads) few_combine_kernel(const FewArgs a) {
  const int t = blockIdx.y, c = blockIdx.x * kThreads + threadIdx.x;
  if (c >= a.H) return;
  float sum = 0;
  for (int j = 0; j < a.top_k; ++j) {
    const int64_t row = a.token_rows[t * a.top_k + j];
    float v = 0;
    for (int p = 0; p < a.parts; ++p) v += a.y[(int64_t(p) * a.slots + row) * a.H + c];
    sum += a.slot_weight[t * a.top_k + j] * v;
  }
  static_cast<T*>(a.out)[t * a.out_ld + c] = rounded<T>(sum);
}

// ---------------------------------------------------------------- host side
struct FewPlan {
  int64_t slots, used;              // used: the most experts that can have rows
  int64_t act_ld, route_bytes, ints_at, act_at, y_at, bytes;
  int parts, k_part;
};

// Parts along k of the second product: enough workgroups for every compute unit to have several, none shorter than two steps of all
// waves.
bool plan_few(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I, FewPlan& p) {
  if (T < 0 || T > kMaxTokens || E < 1 || H < 0 || I < 0 || H >= (1 << 30) || I >= (1 << 30)) return false;
  p.route_bytes = gmm_moe_route_workspace_bytes(T, E, k);
  if (p.route_bytes < 0 || k > 32 || k > E) return false;
  p.slots = T * k;
  p.used = p.slots < E ? p.slots : E;
  p.act_ld = round_up(I, 8);
  p.ints_at = 0;
  p.act_at = round_up((E + 4 * p.slots) * 4 + p.route_bytes, 256);
  p.y_at = round_up(p.act_at + 2 * p.slots * p.act_ld * 2, 256);
  const int64_t items = p.used * ((H + 127) / 128), cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  int64_t parts = items ? 4 * cus / items : 1;
  const int64_t most = (I + 511) / 512;
  parts = parts < 1 ? 1 : parts > 8 ? 8 : parts;
  if (parts > most) parts = most > 0 ? most : 1;
  p.k_part = int(round_up((I + parts - 1) / parts, 64));
  p.parts = p.k_part ? int((I + p.k_part - 1) / p.k_part) : 1;
  p.bytes = p.y_at + p.parts * p.slots * H * 4;
  return p.bytes < (int64_t(1) << 31);
}

template <typename F>
void by_layout(int lay, int64_t tokens, F&& f) {
  const auto rows = [&](auto l) {
    if (tokens <= 16) f(l, std::integral_constant<int, 1>{});
    else if (tokens <= 32) f(l, std::integral_constant<int, 2>{});
    else f(l, std::integral_constant<int, 4>{});
  };
  if (lay == GMM_W_ROWS) rows(std::integral_constant<int, GMM_W_ROWS>{});
  else if (lay == GMM_W_COLS) rows(std::integral_constant<int, GMM_W_COLS>{});
  else rows(std::integral_constant<int, GMM_W_ANY>{});
}

template <typename T>
int launch_few(FewArgs a, const FewPlan& p, int64_t I, const void* w_up, const int64_t* up, const void* w_down, const int64_t* down,
               uint32_t up_bytes, uint32_t down_bytes, hipStream_t stream) {
  const bool x_whole = aligned16(a.x) && multiple8(a.x_ld);
  const bool glu = a.kind != GMM_ACT_SILU;
  FewArgs u = a;
  u.w = w_up; u.w_sg = up[0]; u.w_sk = uint32_t(up[1]); u.w_sn = uint32_t(up[2]); u.w_bytes = up_bytes;
  by_layout(layout_of(w_up, up[0], up[1], up[2], a.H, multiple8(I), x_whole), a.tokens, [&](auto l, auto m) {
    constexpr int LAY = decltype(l)::value, MF = decltype(m)::value, FR = LAY == GMM_W_COLS ? 4 : 8;
    const int out = (glu ? 8 : 16) * FR;
    u.tiles = int((I + out - 1) / out);
    const dim3 grid(unsigned(p.used * u.tiles));
    if (!u.tiles) return;
    if (glu) hipLaunchKernelGGL((few_up_kernel<T, LAY, MF, true>), grid, dim3(kThreads), 0, stream, u);
    else hipLaunchKernelGGL((few_up_kernel<T, LAY, MF, false>), grid, dim3(kThreads), 0, stream, u);
  });
  FewArgs d = a;
  d.w = w_down; d.w_sg = down[0]; d.w_sk = uint32_t(down[1]); d.w_sn = uint32_t(down[2]); d.w_bytes = down_bytes;
  by_layout(layout_of(w_down, down[0], down[1], down[2], I, multiple8(a.H), true), a.tokens, [&](auto l, auto m) {
    constexpr int LAY = decltype(l)::value, MF = decltype(m)::value, FR = LAY == GMM_W_COLS ? 4 : 8;
    d.tiles = (a.H + 16 * FR - 1) / (16 * FR);
    hipLaunchKernelGGL((few_down_kernel<T, LAY, MF>), dim3(unsigned(p.used * d.tiles * p.parts)), dim3(kThreads), 0, stream, d);
  });
  hipLaunchKernelGGL((few_combine_kernel<T>), dim3(unsigned((a.H + kThreads - 1) / kThreads), unsigned(a.tokens)), dim3(kThreads), 0, stream, d);
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

}  // namespace

extern "C" {

int64_t gmm_moe_few_workspace_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t inner) {
  FewPlan p;
  return plan_few(tokens, experts, top_k, hidden, inner, p) ? p.bytes : -1;
}

int gmm_moe_few(const void* x, const void* logits, const void* w_up, const void* w_down, void* out, int64_t tokens, int64_t experts,
                int64_t top_k, int64_t hidden, int64_t inner, int64_t x_stride, int64_t logits_stride, int64_t up_stride_g,
                int64_t up_stride_k, int64_t up_stride_n, int64_t down_stride_g, int64_t down_stride_k, int64_t down_stride_n,
                int64_t out_stride, int32_t kind, int32_t renormalize, int32_t dtype, int32_t logits_dtype, void* workspace,
                int64_t workspace_bytes, void* stream) {
  FewPlan p;
  if (!plan_few(tokens, experts, top_k, hidden, inner, p) || kind < GMM_ACT_SILU || kind > GMM_ACT_SWIGLU_INTERLEAVED) return GMM_ERR_BAD_ARGUMENT;
  if (dtype != GMM_DT_BF16 && dtype != GMM_DT_F16) return GMM_ERR_UNSUPPORTED;
  if (kind == GMM_ACT_SWIGLU_INTERLEAVED && inner % 64) return GMM_ERR_BAD_ARGUMENT;
  if (tokens == 0 || hidden == 0) return GMM_OK;
  if (!x || !logits || !out || (inner && (!w_up || !w_down))) return GMM_ERR_BAD_ARGUMENT;
  if (tokens > 1 && (x_stride < hidden || out_stride < hidden)) return GMM_ERR_BAD_ARGUMENT;
  if (tokens > 1 && x_stride > (int64_t(1) << 30) / kMaxTokens - hidden) return GMM_ERR_BAD_ARGUMENT;
  if (up_stride_g < 0 || down_stride_g < 0) return GMM_ERR_BAD_ARGUMENT;
  if (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)) return GMM_ERR_WORKSPACE;
  const int64_t N = kind == GMM_ACT_SILU ? inner : 2 * inner;
  const uint32_t up_bytes = inner ? matrix_bytes(hidden, N, up_stride_k, up_stride_n) : 2;
  const uint32_t down_bytes = inner ? matrix_bytes(inner, hidden, down_stride_k, down_stride_n) : 2;
  if (!up_bytes || !down_bytes) return GMM_ERR_BAD_ARGUMENT;
  char* const ws = static_cast<char*>(workspace);
  int32_t* const ints = reinterpret_cast<int32_t*>(ws);
  const int64_t S = p.slots;
  float* const weight = reinterpret_cast<float*>(ints + experts + S);
  const int rc = gmm_moe_route(logits, logits_stride, logits_dtype, tokens, experts, top_k, renormalize, ints, ints + experts, weight,
                               ints + experts + 2 * S, ints + experts + 3 * S, ints + experts + 4 * S, p.route_bytes, stream);
  if (rc != GMM_OK) return rc;
  FewArgs a{};
  a.x = x; a.out = out; a.offs = ints; a.slot_weight = weight; a.row_token = ints + experts + 2 * S; a.token_rows = ints + experts + 3 * S;
  a.act = ws + p.act_at; a.y = reinterpret_cast<float*>(ws + p.y_at);
  a.x_ld = tokens > 1 ? x_stride : round_up(hidden, 8); a.out_ld = out_stride;
  a.tokens = int(tokens); a.experts = int(experts); a.top_k = int(top_k); a.slots = int(S); a.H = int(hidden); a.inner = int(inner);
  a.act_ld = int(p.act_ld); a.parts = p.parts; a.k_part = p.k_part; a.kind = kind;
  const int64_t up[3] = {up_stride_g, up_stride_k, up_stride_n}, down[3] = {down_stride_g, down_stride_k, down_stride_n};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GMM_DT_BF16) return launch_few<Bf16>(a, p, inner, w_up, up, w_down, down, up_bytes, down_bytes, s);
  return launch_few<F16>(a, p, inner, w_up, up, w_down, down, up_bytes, down_bytes, s);
}

}  // extern "C"
