// A mixture-of-experts layer for a few tokens (gmm_moe_few in include/grouped_mm_hip.h):
//   out[t] = sum over the choices j of w_tj * act(x[t] @ w_up[e_tj]) @ w_down[e_tj]
// Routing as gmm_moe_route, then every chosen expert's matrices are read once, past a few rows (gmm_skinny.h).  Reading them bounds
// it: 8 tokens, 2 of 8 experts of 4096 -> 2 x 14336 361 to 397 us by card (7.0 to 6.4 TB/s), 32 tokens, 8 of 128 experts of 2048 -> 2 x 768 151 to 160 us (7.0 to 6.6).
// Between the two products the activations are two 16-bit values each (bf16: 2^-16 of them is lost, fp16: 2^-22 or, below 2^-3, 2^-25;
// past 65504 fp16 has infinity, as the layer of many launches), the second products fp32: the result is rounded once.
// Of very few tokens the time is that of the launches and of the trips to memory behind one another (1 token, 8 of 128 experts of
// 2048 -> 2 x 768 25 us, of which the weights are 11).  Then there are two launches: every workgroup of the first routes for
// itself, and of the second's, the last that is done with some columns adds them up.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_route.h"
#include "gmm_skinny.h"

namespace {

using namespace gmm;

constexpr int kMaxTokens = 64;
constexpr int kWaves = 4, kThreads = 64 * kWaves;

// Slots up to which the second product's last workgroup of some columns adds them up: a launch less, but one workgroup reads what otherwise
// all of them would.  2 tokens, 6 of 34 experts of 280 -> 600 16 us, with a launch for the sums 17 (1 token of small experts 15 and 16); 6
// tokens, 4 of 8 experts of 432 -> 2 x 10752 60 and 56.
constexpr int kJoinSlots = 16;
// Words from one counter to the next.  2 tokens, 6 of 64 experts of 2048 -> 2 x 1408 38 to 41 us, with the counters side by side 60 (1 token, 8 of
// 128 of 2 x 768 25 and 26).
constexpr int kLine = 32;

// Workgroups that a compute unit is to hold: two where their sums leave the registers.  Column-major, 33 tokens and more (strips of half as many
// columns): 64 tokens through 8 of 128 experts of 2048 -> 2 x 768 214 us, held to two 202; 40 through 4 of 8 of 432 -> 2 x 10752 108 and 88.
constexpr int few_groups(int lay, int MF) { return lay == GMM_W_COLS || (lay == GMM_W_ROWS && MF <= 2) ? 2 : 1; }

struct FewArgs {
  const void* x;
  const void* w;            // w_up or w_down
  const void* logits;
  int32_t* offs;            // routing
  int32_t* row_token;
  int32_t* token_rows;
  float* slot_weight;
  uint32_t* arrived;        // of each strip of the result's columns: workgroups that are done with it
  void* act;                // [2][slots][act_ld]: high and low halves
  float* y;                 // [parts][slots][H]
  float* part;              // [up_parts][slots][columns of w_up]: parts of x @ w_up, where they are more than one
  void* out;
  int64_t w_sg;             // elements from one expert to the next
  int64_t x_ld, out_ld, logits_ld;
  uint32_t w_sk, w_sn;      // elements
  uint32_t w_bytes;         // of one expert's matrix
  int32_t tokens, experts, top_k, slots, H, inner, act_ld;
  int32_t tiles, parts, k_part;   // strips of columns; parts along k of the second product and their length
  int32_t up_parts, up_k;         // of the first
  int32_t kind, renormalize, logits_dtype;
  int32_t join;             // the second product's workgroups add up the result themselves
  int32_t strips;           // counters of `arrived`
};

// The `which`-th expert that has rows: its number, first row, number of rows; used: how many experts have any.
__device__ __forceinline__ bool find_expert(const FewArgs& a, int which, int& expert, int& row0, int& rows, int& used) {
  constexpr int AT_ONCE = 4;      // trips to memory for 256 experts are one
  const int lane = threadIdx.x & 63;
  bool found = false;
  int start = 0;
  used = 0;
  for (int base = 0; base < a.experts; base += 64 * AT_ONCE) {
    int ends[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) ends[i] = a.offs[min(base + 64 * i + lane, a.experts - 1)];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int to = ends[i], before = __shfl_up(to, 1), from = lane ? before : start;
      start = __builtin_amdgcn_readlane(to, 63);
      const uint64_t with = __ballot(to > from);      // the last expert again: no rows
      const int n = __popcll(with);
      if (!found && which < used + n) {
        const uint64_t it = __ballot(to > from && __popcll(with & ((uint64_t(1) << lane) - 1)) == which - used);
        const int at = __ffsll(static_cast<unsigned long long>(it)) - 1;
        expert = base + 64 * i + at;
        row0 = __builtin_amdgcn_readlane(from, at);
        rows = __builtin_amdgcn_readlane(to, at) - row0;
        found = true;
      }
      used += n;
    }
    if (found && !a.join) break;      // nobody wants to know the rest
  }
  return found;
}

// The parts of the choices of a token, one after the other; behind the last one that one's first part again.
struct Choice {
  int j, part;
  __device__ __forceinline__ void next(const FewArgs& a) {
    const bool last = ++part == a.parts;
    part = last ? 0 : part;
    j = min(j + last, a.top_k - 1);
  }
};

__device__ __forceinline__ float silu(float x) { return x / (1.0f + __expf(-x)); }

// act[r] = act(x[token of row r] @ w_up[e]), or parts of the product.  GLU: a strip is 8 * FR gate columns and their partners.
// SIDE: the waves of a workgroup take strips side by side and all of k, and have no sums to share.
template <typename T, int LAY, int MF, bool GLU, bool ROUTE, bool SIDE>
__global__ void __launch_bounds__(kThreads, few_groups(LAY, MF)) few_up_kernel(const FewArgs a) {
  using S = Strip<T, LAY, MF, 1>;
  constexpr int FR = S::FR, OUT = GLU ? 8 * FR : 16 * FR;
  __shared__ SkinnyShared<S, kWaves> shared;
  const int part = blockIdx.x % a.up_parts, item = blockIdx.x / a.up_parts;
  int expert, row0, rows;
  const int32_t* row_token;
  if (a.join && blockIdx.x == 0)      // for the kernel behind
    for (int i = threadIdx.x; i < a.strips; i += kThreads) a.arrived[i * kLine] = 0;
  if constexpr (ROUTE) {
    __shared__ FewRouting routing;
    const RouteHere here{a.logits, a.logits_ld, a.offs, a.token_rows, a.slot_weight, a.tokens, a.experts, a.top_k, a.slots, a.renormalize, a.logits_dtype};
    if (!route_here<kWaves>(here, routing, item / a.tiles, expert, row0, rows)) return;
    row_token = routing.token;
  } else {
    int used;
    if (!find_expert(a, item / a.tiles, expert, row0, rows, used)) return;
    row_token = a.row_token + row0;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tile = SIDE ? item % a.tiles * kWaves + wave : item % a.tiles;
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
  s.set_rows([&](int r) { return r < rows ? uint32_t(row_token[r]) * uint32_t(a.x_ld) * 2 : kNowhere; });
  f32x4 acc[MF][FR];
  clear(acc);
  s.template run<SIDE ? 1 : kWaves>(rows, part * a.up_k, min(a.H, (part + 1) * a.up_k), SIDE ? 0 : wave, acc);

  T* const high = static_cast<T*>(a.act);
  T* const low = high + int64_t(a.slots) * a.act_ld;
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (16 * m >= rows) break;
    __syncthreads();
    shared.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = SIDE ? lane : threadIdx.x; u < OUT * 4; u += SIDE ? 64 : kThreads) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.inner) continue;
      const auto result = [&](int c) {
        const int at = S::position(c, a.inner - col);
        return SIDE ? shared.sums.of(wave, S::product_of(at), S::lane_of(at), og) : shared.sums.get(S::product_of(at), S::lane_of(at), og);
      };
      const f32x4 h = result(oc), partner = GLU ? result(OUT + oc) : f32x4{1, 1, 1, 1};
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 16 * m + 4 * og + v;
        if (r >= rows) break;
        if (a.up_parts > 1) {
          float* const to = a.part + (int64_t(part) * a.slots + row0 + r) * (GLU ? 2 : 1) * a.inner + col;
          to[0] = h[v];
          if constexpr (GLU) to[a.inner] = partner[v];
        } else {
          const int64_t to = int64_t(row0 + r) * a.act_ld + col;
          split(silu(h[v]) * partner[v], high[to], low[to]);
        }
      }
    }
  }
}

constexpr int kDeviceScope = 16;   // sc1

// y[part][r] = act[r] @ w_down[e], over the part's range of k; with a.join the result as well.
// PARTS: the first product lies in parts; a workgroup adds up those that it needs, and keeps their activations in LDS.
template <typename T, int LAY, int MF, bool PARTS>
__global__ void __launch_bounds__(kThreads, few_groups(LAY, MF)) few_down_kernel(const FewArgs a) {
  using S = Strip<T, LAY, MF, 2, PARTS ? GMM_A_RESIDENT : LAY == GMM_W_ANY ? GMM_A_ELEMENTS : GMM_A_STAGED>;
  constexpr int FR = S::FR, OUT = 16 * FR;
  __shared__ SkinnyShared<S, kWaves> shared;
  __shared__ int last;
  __shared__ int32_t slot_row[kJoinSlots];
  __shared__ float slot_weight[kJoinSlots];
  extern __shared__ __align__(16) char resident[];      // PARTS: [2][rows][k_part + 8]
  const int part = blockIdx.x % a.parts, item = blockIdx.x / a.parts, tile = item % a.tiles;
  if (a.join && int(threadIdx.x) < a.slots) {
    slot_row[threadIdx.x] = a.token_rows[threadIdx.x];
    slot_weight[threadIdx.x] = a.slot_weight[threadIdx.x];
  }
  int expert, row0, rows, used;
  if (!find_expert(a, item / a.tiles, expert, row0, rows, used)) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int from = part * a.k_part, to = min(a.inner, from + a.k_part);
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.w_buf = buffer(static_cast<const T*>(a.w) + expert * a.w_sg, a.w_bytes);
  s.set_columns(tile * OUT, a.H - tile * OUT, a.w_sk, a.w_sn);
  typename S::Step step[S::STEPS];
  if constexpr (PARTS) {
    s.pitch = (a.k_part + 8) * 2;
    s.a_plane = uint32_t(a.tokens) * s.pitch;
    s.resident = resident;
    s.resident_k = from;
    s.resident_rows = rows;
    s.template prime<1, kWaves>(step, from + wave * S::KS, to);      // on their way while the activations are computed
    const int columns = a.kind == GMM_ACT_SILU ? a.inner : 2 * a.inner;
    for (int u = threadIdx.x; u < rows * a.k_part; u += kThreads) {
      const int r = u / a.k_part, c = u % a.k_part;
      float gate = 0, partner = 0;
      if (from + c < to) {
        const float* at = a.part + int64_t(row0 + r) * columns + from + c;
        in_fours(a.up_parts, [&](int p, bool in) {
          const float* const here = at + int64_t(p) * a.slots * columns;
          const float g = here[0], u = a.kind == GMM_ACT_SILU ? 0.0f : here[a.inner];
          gate += in ? g : 0.0f;
          partner += in ? u : 0.0f;
        });
      }
      T* const keep = reinterpret_cast<T*>(resident + r * s.pitch) + c;
      split(silu(gate) * (a.kind == GMM_ACT_SILU ? 1.0f : partner), keep[0], *reinterpret_cast<T*>(reinterpret_cast<char*>(keep) + s.a_plane));
    }
    __syncthreads();
  } else {
    s.a_plane = uint32_t(a.slots) * a.act_ld * 2;
    s.a_buf = buffer(a.act, 2 * s.a_plane);
    s.set_rows([&](int r) { return r < rows ? uint32_t(row0 + r) * a.act_ld * 2 : kNowhere; });
  }
  f32x4 acc[MF][FR];
  clear(acc);
  if constexpr (PARTS) s.template primed<1, kWaves>(step, from + wave * S::KS, to, acc);
  else s.template run<kWaves>(rows, from, to, wave, acc);

  // stored through to memory at device scope where another workgroup reads it in this launch
  const __amdgpu_buffer_rsrc_t y = buffer(a.y, uint32_t(a.parts) * a.slots * a.H * 4);
  const uint32_t y_at = (uint32_t(part) * a.slots + row0) * a.H;
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (16 * m >= rows) break;
    __syncthreads();
    shared.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = threadIdx.x; u < OUT * 4; u += kThreads) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.H) continue;
      const int at = S::position(oc, a.H - col);
      const f32x4 h = shared.sums.get(S::product_of(at), S::lane_of(at), og);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 16 * m + 4 * og + v;
        if (r >= rows) break;
        const int to = int((y_at + uint32_t(r) * a.H + col) * 4);
        if (a.join) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(h[v]), y, to, 0, kDeviceScope);
        else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(h[v]), y, to, 0, 0);
      }
    }
  }
  if (!a.join) return;
  // The last workgroup of these columns adds up what all of them left, in the order of the choices and parts whichever it is.  Nobody
  // waits for anybody.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(&a.arrived[tile * kLine], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(used * a.parts) - 1;
  __syncthreads();
  if (!last) return;
  for (int u = threadIdx.x; u < a.tokens * OUT; u += kThreads) {
    const int t = u / OUT, col = tile * OUT + u % OUT;
    if (col >= a.H) continue;
    float sum = 0;
    Choice q{0, 0};
    in_fours(a.top_k * a.parts, [&](int, bool in) {
      const int slot = t * a.top_k + q.j;
      const uint32_t at = (uint32_t(q.part) * a.slots + slot_row[slot]) * a.H + col;
      const float v = slot_weight[slot] * __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(y, int(at * 4), 0, kDeviceScope));
      sum += in ? v : 0.0f;
      q.next(a);
    });
    static_cast<T*>(a.out)[t * a.out_ld + col] = rounded<T>(sum);
  }
}

// out[t] = sum over j of weight * sum over the parts of y, in that order.  Where they lie is looked up at once, and eight of them are on their
// way together: one after the other 6 of 32 tokens took 14 us.
template <typename T>
__global__ void __launch_bounds__(kThreads) few_combine_kernel(const FewArgs a) {
  const int t = blockIdx.y, c = blockIdx.x * kThreads + threadIdx.x, lane = threadIdx.x & 63;
  // of choice j: in lane j
  const int mine = t * a.top_k + min(lane, a.top_k - 1);
  const int from = a.token_rows[mine] * a.H, weight = __builtin_bit_cast(int, a.slot_weight[mine]);
  const uint32_t next = uint32_t(a.slots) * a.H;
  const float* const y = a.y + min(c, a.H - 1);      // every lane has its part in the lookup
  float sum = 0, v = 0;
  Choice q{0, 0};
  in_fours(a.top_k * a.parts, [&](int, bool in) {
    const float one = (y + uint32_t(__builtin_amdgcn_readlane(from, q.j)))[q.part * next];
    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(weight, q.j));
    v = in ? (q.part ? v : 0.0f) + one : v;
    if (in && q.part == a.parts - 1) sum += w * v;
    q.next(a);
  });
  if (c >= a.H) return;
  static_cast<T*>(a.out)[t * a.out_ld + c] = rounded<T>(sum);
}

// ---------------------------------------------------------------- host side
struct FewPlan {
  int64_t slots, used;              // used: the most experts that can have rows
  int64_t act_ld, route_bytes, arrived_at, act_at, y_at, bytes;
  int32_t parts, k_part, up_parts, up_k, join;
};

constexpr int64_t kResident = 1024;      // elements of a row of activations that a workgroup keeps

// `want` parts of k elements, each a multiple of 64 and at least 256 long.
void cut(int64_t k, int64_t want, int32_t& parts, int32_t& each) {
  const int64_t most = k / 256;
  if (want > most) want = most;
  if (want < 1) want = 1;
  each = int32_t(round_up((k + want - 1) / want, 64));
  parts = each ? int32_t((k + each - 1) / each) : 1;
}

// Where the strips of the first product are fewer than compute units they are cut along k, and the second product's workgroups add the
// parts up: 1 token, 8 of 128 experts of 2048 -> 2 x 768 30.8 -> 28.2 us, 4 of 32 of 4096 -> 2 x 2048 58 -> 49.5.  (More strips, cut as
// well: within 2 us either way.)
bool plan_few(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I, FewPlan& p) {
  if (T < 0 || T > kMaxTokens || E < 1 || H < 0 || I < 0 || H >= (1 << 30) || I >= (1 << 30)) return false;
  p.route_bytes = gmm_moe_route_workspace_bytes(T, E, k);
  if (p.route_bytes < 0 || k > 32 || k > E) return false;
  const int64_t cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  p.slots = T * k;
  p.used = p.slots < E ? p.slots : E;
  p.act_ld = round_up(I, 8);
  p.join = p.slots <= kJoinSlots && I > 0;
  const int64_t ups = p.used * ((I + 63) / 64), downs = p.used * ((H + 127) / 128);
  cut(H, T <= 16 && ups && ups <= cus ? 3 * cus / ups : 1, p.up_parts, p.up_k);
  int64_t parts = downs ? 4 * cus / downs : 1;
  if (parts > 8) parts = 8;
  if (p.up_parts > 1 && parts < (I + kResident - 1) / kResident) parts = (I + kResident - 1) / kResident;
  cut(I, parts, p.parts, p.k_part);
  p.arrived_at = round_up((E + 4 * p.slots) * 4 + p.route_bytes, 256);
  p.act_at = round_up(p.arrived_at + (H + 63) / 64 * kLine * 4, 256);
  p.y_at = round_up(p.act_at + (p.up_parts > 1 ? p.up_parts * p.slots * 2 * I * 4 : 2 * p.slots * p.act_ld * 2), 256);
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
               uint32_t up_bytes, uint32_t down_bytes, hipStream_t stream, void* table) {
  const bool glu = a.kind != GMM_ACT_SILU;
  const int64_t cus = gmm_num_cus();
  int rc = GMM_OK;
  bool routed = false;
  FewArgs u = a;
  u.w = w_up; u.w_sg = up[0]; u.w_sk = uint32_t(up[1]); u.w_sn = uint32_t(up[2]); u.w_bytes = up_bytes;
  by_layout(layout_of(up[1], up[2], a.H, I), a.tokens, [&](auto l, auto m) {
    constexpr int LAY = decltype(l)::value, MF = decltype(m)::value, FR = LAY == GMM_W_COLS ? 4 : 8;
    const int out = (glu ? 8 : 16) * FR;
    u.tiles = int((I + out - 1) / out);
    // Strips side by side (512 bytes and more of a row of w_up for a workgroup) where that leaves every compute unit one and rows are long:
    // 8 of 8 experts of 4096 -> 2 x 14336, 8 tokens 419 -> 387 us, 64 537 -> 493; 16 experts of 2048 -> 2 x 4096, 8 tokens 144 -> 122; but
    // 128 experts of 2048 -> 2 x 768, 64 tokens 191 -> 206; 32 of 4096 -> 2 x 2048 16 tokens 231 -> 214, 4 tokens 118 -> 132.
    const bool side = LAY == GMM_W_ROWS && p.up_parts == 1 && 2 * p.used * u.tiles >= 7 * cus && (u.tiles >= 64 || (u.tiles >= 32 && a.tokens >= 16));
    if (side) u.tiles = (u.tiles + kWaves - 1) / kWaves;
    const int64_t groups = p.used * u.tiles * p.up_parts;
    // one round of workgroups: routing is as long in all of them as in one
    routed = MF == 1 && groups && groups <= 4 * cus && a.slots <= kRouteSlots && a.experts <= kRouteExperts;
    if (!routed) {
      rc = gmm_moe_route(a.logits, a.logits_ld, a.logits_dtype, a.tokens, a.experts, a.top_k, a.renormalize, a.offs, a.offs + a.experts, a.slot_weight,
                         a.row_token, a.token_rows, table, p.route_bytes, stream);
      if (rc != GMM_OK) return;
    }
    if (!groups) return;
    const auto launch = [&](auto g, auto r, auto sd) {
      constexpr bool GLU = decltype(g)::value, ROUTE = decltype(r)::value, SIDE = decltype(sd)::value;
      hipLaunchKernelGGL((few_up_kernel<T, LAY, MF, GLU, ROUTE, SIDE>), dim3(unsigned(groups)), dim3(kThreads), 0, stream, u);
    };
    const auto sided = [&](auto g, auto r) {
      if constexpr (LAY == GMM_W_ROWS) {
        if (side) return launch(g, r, std::true_type{});
      }
      launch(g, r, std::false_type{});
    };
    const auto routing = [&](auto g) {
      if constexpr (MF == 1) {
        if (routed) return sided(g, std::true_type{});
      }
      sided(g, std::false_type{});
    };
    glu ? routing(std::true_type{}) : routing(std::false_type{});
  });
  if (rc != GMM_OK) return rc;
  FewArgs d = a;
  d.w = w_down; d.w_sg = down[0]; d.w_sk = uint32_t(down[1]); d.w_sn = uint32_t(down[2]); d.w_bytes = down_bytes;
  by_layout(layout_of(down[1], down[2], I, a.H), a.tokens, [&](auto l, auto m) {
    constexpr int LAY = decltype(l)::value, MF = decltype(m)::value, FR = LAY == GMM_W_COLS ? 4 : 8;
    d.tiles = (a.H + 16 * FR - 1) / (16 * FR);
    const dim3 grid(unsigned(p.used * d.tiles * p.parts));
    if constexpr (MF == 1) {
      if (p.up_parts > 1) {
        const int lds = 2 * a.tokens * (p.k_part + 8) * 2;
        hipLaunchKernelGGL((few_down_kernel<T, LAY, MF, true>), grid, dim3(kThreads), lds, stream, d);
        return;
      }
    }
    hipLaunchKernelGGL((few_down_kernel<T, LAY, MF, false>), grid, dim3(kThreads), 0, stream, d);
  });
  if (!a.join)
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
  if (tokens > 1 && (x_stride < hidden || out_stride < hidden || logits_stride < experts)) return GMM_ERR_BAD_ARGUMENT;
  if (logits_dtype < GMM_DT_BF16 || logits_dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
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
  FewArgs a{};
  a.x = x; a.logits = logits; a.out = out; a.offs = ints; a.slot_weight = weight; a.row_token = ints + experts + 2 * S; a.token_rows = ints + experts + 3 * S;
  a.arrived = reinterpret_cast<uint32_t*>(ws + p.arrived_at); a.act = ws + p.act_at; a.part = reinterpret_cast<float*>(ws + p.act_at); a.y = reinterpret_cast<float*>(ws + p.y_at);
  a.x_ld = tokens > 1 ? x_stride : round_up(hidden, 8); a.out_ld = out_stride; a.logits_ld = tokens > 1 ? logits_stride : experts;
  a.tokens = int(tokens); a.experts = int(experts); a.top_k = int(top_k); a.slots = int(S); a.H = int(hidden); a.inner = int(inner);
  a.act_ld = int(p.act_ld); a.parts = p.parts; a.k_part = p.k_part; a.kind = kind; a.renormalize = renormalize; a.logits_dtype = logits_dtype;
  a.up_parts = p.up_parts; a.up_k = p.up_k; a.join = p.join; a.strips = int((hidden + 63) / 64);
  const int64_t up[3] = {up_stride_g, up_stride_k, up_stride_n}, down[3] = {down_stride_g, down_stride_k, down_stride_n};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == GMM_DT_BF16) return launch_few<Bf16>(a, p, inner, w_up, up, w_down, down, up_bytes, down_bytes, s, ints + experts + 4 * S);
  return launch_few<F16>(a, p, inner, w_up, up, w_down, down, up_bytes, down_bytes, s, ints + experts + 4 * S);
}

}  // extern "C"
