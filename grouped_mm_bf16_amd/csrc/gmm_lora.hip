// A projection that all rows share beside low-rank adapters of which each row has its own (declared in include/grouped_mm_hip.h):
//   y[t] = x[t] @ W + scale[i] * (x[t] @ A[i]) @ B[i],  i = adapter[t]; a number outside [0, L): no adapter
// and the adapters' gradients.
//   A few rows (gmm_lora_linear): W and the adapters are read once, past the rows (gmm_skinny.h), in one launch; a second one adds the
//     parts up.  Reading W bounds it: 48 rows of 64 adapters of rank 16, 4096 -> 8192, 23 us, of which W takes 9.5 at the fastest reads; of one
//     row, 4096 -> 4096, 12 us, mostly the two launches and the trips to memory behind one another.
//   Many rows (gmm_lora_sum): W's product is a grouped product of one group, in fp32; what the adapters add is two thin products, bound by
//     reading x, by reading that product and by writing y: 8192 rows of 4096 -> 4096, rank 16, 69 us (268 MB, 3.9 TB/s).
//   Gradients (gmm_lora_grad): dA[i] = scale[i] * sum of x[t]^T u[t], dB[i] = scale[i] * sum of low[t]^T dy[t] over the rows t that have
//     adapter i: thin products along the rows, bound by reading x and dy: of those 8192 rows 30 us (134 MB, 4.5 TB/s), and 20 for the sort before
//     and the sums behind; in fp16 6 more for the powers of two.
// The rank-sized values x @ A and dy @ B^T stay in fp32; where they are operands of a 16-bit product they are two values each, in fp16 behind
// a power of two that brings them into its range.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_launch.h"
#include "gmm_skinny.h"

namespace {

using namespace gmm;

constexpr int kFewRows = 64;
// Rows up to which they are taken one at a time: they are likely to be of different adapters.  4096 -> 4096 in all, one at a time and in strips of
// 16 rows: 128 rows of different adapters of rank 16 40 and 78 us, of one 40 and 42; 256 of rank 64 61 and 104, of one 57 and 52.
constexpr int kSingleRows = 256;
constexpr int kMaxRank = 256;
constexpr int kMaxAdapters = 1022;     // one more bin of the sort holds the rows without an adapter
constexpr int kWaves = 4, kThreads = 64 * kWaves;
// Waves of a workgroup of a few rows' launch: eight, four where the sums of 64 rows by 128 columns, or what is loaded element by element,
// need half of the registers.
constexpr int few_waves(int MF, int lay) { return MF == 4 || (MF == 2 && lay == GMM_W_ANY) ? 4 : 8; }

// ... and how many of four waves a compute unit is to hold: two where half of the registers do (48 rows, 64 adapters, column-major 4096 -> 8192
// 24.5 -> 23.2 us: all workgroups, those of the adapters and those of W, then run at once).
constexpr int few_at_once(int MF, int lay) { return MF == 4 && lay == GMM_W_COLS ? 2 : 1; }

struct Matrices {          // a stack [L, K, N] of 16-bit matrices, or one
  const void* at;
  int64_t sg;              // elements from one to the next
  uint32_t sk, sn;         // elements
  uint32_t bytes;          // of one
};

struct LoraArgs {
  const void* x;
  Matrices w, a, b;
  const int32_t* adapter;
  const float* scale;      // null: 1
  void* out;
  float* low;              // [low_parts][rows][R]: parts of x @ A
  float* low_out;          // [rows][R]: their sums, null: not wanted
  float* sums;             // many rows: [rows][pitch], x @ A times scale, zeros past the rank; null: not wanted
  float* base;             // [base_parts][rows][N]: parts of x @ W; without any: it lies in `out`
  int64_t x_ld, out_ld;
  int32_t rows, K, N, R, L;
  int32_t strip_rows, low_parts, low_k, low_tiles;   // rows of a strip; parts of K and their length; strips of columns of A
  int32_t base_parts, base_k, base_tiles, low_groups, pitch, strips;
  int32_t keep;            // x @ A of one part goes where the second product wants it
};

__device__ __forceinline__ bool has_adapter(int id, int L) { return id >= 0 && id < L; }

template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t matrix(const Matrices& m, int which) {
  return buffer(static_cast<const T*>(m.at) + which * m.sg, m.bytes);
}

// Many rows: low of a row for the second product, times scale, zeros past the rank; and as it is where that is wanted.
__device__ __forceinline__ void keep_low(const LoraArgs& a, int row, int r, float v, float scale) {
  if (a.low_out && r < a.R) a.low_out[int64_t(row) * a.R + r] = v;
  if (a.sums) a.sums[int64_t(row) * a.pitch + r] = v * scale;
}

// low[part][t] = x[t] @ A[adapter[t]] over a part of K, for a strip of up to 16 rows.  Of rows with different adapters one adapter comes
// after the other; their steps are one sequence, so that the next adapter's loads are on their way while the last one's are
// multiplied (1024
// rows of 64 adapters, rank 64, with W's product: drained each time 233 us, as one sequence 167).
template <typename T, int LAY, int FR, bool AE>
using LowSkinny = Skinny<T, LAY, FR, 1, 1, AE ? GMM_A_ELEMENTS : GMM_A_STAGED, FR <= 2 ? 4 : 2>;

// The adapters of a strip's rows, one after the other.
struct Adapters {
  uint32_t todo, mine;      // rows of adapters to come; of this one
  int which;

  __device__ __forceinline__ void next(int id) {
    which = __builtin_amdgcn_readlane(id, __ffs(todo) - 1);
    mine = uint32_t(__ballot(id == which)) & 0xffffu;
    todo &= ~mine;
  }
};

template <typename T, typename S, int WAVES, int ST>
__device__ __forceinline__ void low_product(const LoraArgs& a, int item, SkinnyShared<S, WAVES>& shared) {
  constexpr int FR = S::FR, OUT = S::COLUMNS, NEXT = WAVES * S::KS;
  const int part = item % a.low_parts, tile = item / a.low_parts % a.low_tiles, row0 = item / a.low_parts / a.low_tiles * a.strip_rows;
  const int rows = min(a.strip_rows, a.rows - row0);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int id = j < rows ? a.adapter[row0 + j] : -1;
  const uint32_t with = uint32_t(__ballot(has_adapter(id, a.L))) & 0xffffu;
  if (!with) return;
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.a_buf = buffer(static_cast<const T*>(a.x) + row0 * a.x_ld, uint32_t(((rows - 1) * a.x_ld + a.K) * 2));
  s.a_plane = 0;
  s.set_columns(tile * OUT, a.R - tile * OUT, a.a.sk, a.a.sn);
  const int to = min(a.K, (part + 1) * a.low_k), begin = part * a.low_k + wave * S::KS;
  const int steps = max(1, (to - begin + NEXT - 1) / NEXT);      // of an adapter, of this wave
  Adapters loading{with, 0, 0}, adding{with, 0, 0};
  int load_step = 0, add_step = 0;
  const auto open = [&] {
    loading.next(id);
    s.w_buf = matrix<T>(a.a, loading.which);
    s.set_rows([&](int r) { return loading.mine >> r & 1 ? uint32_t(r) * uint32_t(a.x_ld) * 2 : kNowhere; });
    load_step = 0;
  };
  const auto load = [&](typename S::Step& step) {
    s.template load<1>(step, begin + load_step * NEXT, load_step < steps ? to : 0);
    if (++load_step >= steps && loading.todo) open();
    __builtin_amdgcn_sched_barrier(0);
  };
  typename S::Step step[ST];
  f32x4 acc[1][FR], low[FR];
  clear(acc);
#pragma unroll
  for (int i = 0; i < FR; ++i) low[i] = f32x4{0, 0, 0, 0};
  open();
#pragma unroll
  for (int u = 0; u < ST; ++u) load(step[u]);
  adding.next(id);
  for (bool more = true; more;) {
#pragma unroll
    for (int u = 0; u < ST; ++u) {
      s.template multiply<1>(step[u], begin + add_step * NEXT, to, acc);
      // behind an adapter's last step its rows are taken over: what is no number in it stays with them.  (Steps behind all of them
      // add zeros to a row that has been taken.)
      if (++add_step == steps) {
#pragma unroll
        for (int i = 0; i < FR; ++i)
#pragma unroll
          for (int v = 0; v < 4; ++v) low[i][v] = adding.mine >> (4 * g + v) & 1 ? acc[0][i][v] : low[i][v];
        clear(acc);
        add_step = 0;
        if (adding.todo) adding.next(id);
        else { adding.mine = 0; more = false; }
      }
      __builtin_amdgcn_sched_barrier(0);
      load(step[u]);
    }
  }
  __syncthreads();
  shared.sums.put(wave, lane, low);
  __syncthreads();
  float* const out = a.low + (int64_t(part) * a.rows + row0) * a.R;
  for (int u = threadIdx.x; u < OUT * 4; u += 64 * WAVES) {
    const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
    const int at = S::position(oc, max(1, a.R - col));
    const f32x4 h = shared.sums.get(S::product_of(at), S::lane_of(at), og);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = 4 * og + v;
      if (!(with >> r & 1)) continue;
      if (a.low_parts > 1 || !a.keep) {
        if (col < a.R) out[r * a.R + col] = h[v];
      } else if (col < a.pitch) {
        keep_low(a, row0 + r, col, col < a.R ? h[v] : 0.0f, a.scale ? a.scale[a.adapter[row0 + r]] : 1.0f);
      }
    }
  }
}

// Up to rank 16 (FR 1) eight waves share K, which then needs few parts or none, and no launch for their sums: 615 rows of 1031 -> 519 with
// gradients 158 -> 151 us, 96 rows of 4096 -> 4096 with column-major W 37 -> 34 (but 8192 rows with gradients 569 -> 572).  Above, four
// waves and more parts: with the steps of many adapters one after the other, 257 rows of 64 adapters of rank 64 94 us, with 16 waves 108.
constexpr int low_waves(int FR) { return FR == 1 ? 8 : 4; }

template <typename T, int LAY, int FR, bool AE>
__global__ void __launch_bounds__(64 * low_waves(FR), FR == 1 ? 4 : FR == 2 ? 3 : 2) lora_low_kernel(const LoraArgs a) {
  constexpr int WAVES = low_waves(FR);
  using S = LowSkinny<T, LAY, FR, AE>;
  __shared__ SkinnyShared<S, WAVES> shared;
  low_product<T, S, WAVES, FR <= 2 ? 4 : 2>(a, blockIdx.x, shared);
}

// A few rows: workgroups for x @ A first, then those for x @ W: base[part][t] over a part of K.
template <typename T, int LAY_W, int LAY_A, int MF>
__global__ void __launch_bounds__(64 * few_waves(MF, LAY_W), few_at_once(MF, LAY_W)) lora_few_kernel(const LoraArgs a) {
  constexpr int WAVES = few_waves(MF, LAY_W);
  using S = Strip<T, LAY_W, MF, 1>;
  using SA = LowSkinny<T, LAY_A, 1, LAY_W == GMM_W_ANY>;
  constexpr int FR = S::FR, OUT = S::COLUMNS;
  __shared__ union Shared {
    SkinnyShared<SA, WAVES> low;
    SkinnyShared<S, WAVES> base;
    __device__ Shared() {}
  } shared;
  if (int(blockIdx.x) < a.low_groups) return low_product<T, SA, WAVES, 4>(a, blockIdx.x, shared.low);
  const int item = blockIdx.x - a.low_groups, part = item % a.base_parts, tile = item / a.base_parts;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  S s;
  s.lane = lane;
  s.lds = shared.base.wave[wave];
  s.w_buf = matrix<T>(a.w, 0);
  s.a_buf = buffer(a.x, uint32_t(((a.rows - 1) * a.x_ld + a.K) * 2));
  s.a_plane = 0;
  s.set_columns(tile * OUT, a.N - tile * OUT, a.w.sk, a.w.sn);
  s.set_rows([&](int r) { return r < a.rows ? uint32_t(r) * uint32_t(a.x_ld) * 2 : kNowhere; });
  f32x4 acc[MF][FR];
  clear(acc);
  s.template run<WAVES>(a.rows, part * a.base_k, min(a.K, (part + 1) * a.base_k), wave, acc);
  float* const base = a.base + int64_t(part) * a.rows * a.N;
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (16 * m >= a.rows) break;
    __syncthreads();
    shared.base.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = threadIdx.x; u < OUT * 4; u += 64 * WAVES) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.N) continue;
      const int at = S::position(oc, a.N - col);
      const f32x4 h = shared.base.sums.get(S::product_of(at), S::lane_of(at), og);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const int r = 16 * m + 4 * og + v;
        if (r < a.rows) base[int64_t(r) * a.N + col] = h[v];
      }
    }
  }
}

// Sums of the parts of x @ A of one row, times its adapter's scale.
__device__ __forceinline__ float low_sum(const LoraArgs& a, int row, int r) {
  float s = 0;
  in_fours(a.low_parts, [&](int p, bool in) {
    const float v = a.low[(int64_t(p) * a.rows + row) * a.R + r];
    s += in ? v : 0.0f;
  });
  return s;
}

// One row after the other: y[t] = sum of the parts of x @ W (without any: what lies in y) + scale * low @ B.  A wave for 64 lanes' columns
// of one row: eight columns to a lane where B is contiguous along them (where fewer are left the last eight, of which the lane writes its
// own), else one.
template <typename T, int LAY>
__global__ void __launch_bounds__(64) lora_finish_kernel(const LoraArgs a) {
  constexpr int W = LAY == GMM_W_ROWS ? 8 : 1;
  __shared__ float low[kMaxRank];
  const int t = blockIdx.y, lane = threadIdx.x, own = (blockIdx.x * 64 + lane) * W, c = W == 8 ? min(own, max(0, a.N - 8)) : own;
  const int id = a.adapter[t];
  float y[W];
#pragma unroll
  for (int i = 0; i < W; ++i) y[i] = 0;
  T* const out = static_cast<T*>(a.out) + t * a.out_ld + c;
  if (own < a.N && a.base_parts == 0) {
    if constexpr (W == 8) {
      const Pack<T, 8> there = unaligned<Pack<T, 8>>(out);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = there.get(i);
    } else {
      y[0] = widen(out[0]);
    }
  }
  if (own < a.N) {
    const float* base = a.base + int64_t(t) * a.N + c;
    const int64_t next = int64_t(a.rows) * a.N;
    in_fours(a.base_parts, [&](int p, bool in) {
      const float* const at = base + p * next;
      if constexpr (W == 8) {
        const f32x4 lo = unaligned<f32x4>(at), hi = unaligned<f32x4>(at + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) { y[i] += in ? lo[i] : 0.0f; y[4 + i] += in ? hi[i] : 0.0f; }
      } else {
        const float v = at[0];
        y[0] += in ? v : 0.0f;
      }
    });
  }
  const bool has = has_adapter(id, a.L);
  const float scale = has && a.scale ? a.scale[id] : 1.0f;
  if (has)
    for (int r = lane; r < a.R; r += 64) {
      const float s = low_sum(a, t, r);
      if (a.low_out && blockIdx.x == 0) a.low_out[int64_t(t) * a.R + r] = s;
      low[r] = s * scale;
    }
  __syncthreads();
  if (own >= a.N) return;
  if (has) {
    const T* b = static_cast<const T*>(a.b.at) + id * a.b.sg + int64_t(c) * a.b.sn;
    float add[W];
#pragma unroll
    for (int i = 0; i < W; ++i) add[i] = 0;
    if constexpr (LAY == GMM_W_ROWS) {
#pragma unroll 8
      for (int r = 0; r < a.R; ++r) {
        const Pack<T, 8> v = unaligned<Pack<T, 8>>(b + int64_t(r) * a.b.sk);
#pragma unroll
        for (int i = 0; i < 8; ++i) add[i] += low[r] * v.get(i);
      }
    } else if constexpr (LAY == GMM_W_COLS) {
#pragma unroll 4
      for (int r = 0; r + 8 <= a.R; r += 8) {
        const Pack<T, 8> v = unaligned<Pack<T, 8>>(b + r);
#pragma unroll
        for (int i = 0; i < 8; ++i) add[0] += low[r + i] * v.get(i);
      }
      for (int r = a.R / 8 * 8; r < a.R; ++r) add[0] += low[r] * widen(b[r]);
    } else {
#pragma unroll 4
      for (int r = 0; r < a.R; ++r) add[0] += low[r] * widen(b[int64_t(r) * a.b.sk]);
    }
#pragma unroll
    for (int i = 0; i < W; ++i) y[i] += add[i];
  }
  if constexpr (W == 8) {
    const Pack<T, 8> now = Pack<T, 8>::of(y);
    if (c == own) {
      __builtin_memcpy(out, &now, 16);
    } else {
#pragma unroll
      for (int i = 1; i < 8; ++i) if (c + i >= own) out[i] = rounded<T>(y[i]);
    }
  } else {
    out[0] = rounded<T>(y[0]);
  }
}

// The parts of x @ A of many rows summed.
__global__ void __launch_bounds__(kThreads) lora_low_sum_kernel(const LoraArgs a) {
  const int64_t u = int64_t(blockIdx.x) * kThreads + threadIdx.x;
  const int row = int(u / a.pitch), r = int(u % a.pitch);
  if (row >= a.rows) return;
  const int id = a.adapter[row];
  if (has_adapter(id, a.L)) keep_low(a, row, r, r < a.R ? low_sum(a, row, r) : 0.0f, a.scale ? a.scale[id] : 1.0f);
}

// The power of two that brings the largest of some values between 2^14 and 2^15 (as near as fp32 has one).  Two fp16 values then hold each
// of them to 2^-22 of it, or 2^-39 of the largest; without it, what is smaller than 2^-3 would lose bits (of 1e-6 all but five) and what
// is past 65504 would be infinite.  Values that are no finite numbers do not count.
struct Exponent {
  uint32_t most = 0;      // bits of the largest absolute value

  __device__ __forceinline__ void take(float v) {
    const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
    most = max(most, bits < 0x7f800000u ? bits : 0u);
  }
  __device__ __forceinline__ void join(int distance) { most = max(most, uint32_t(__shfl_xor(int(most), distance))); }
  __device__ __forceinline__ uint32_t field() const { return max(most >> 23, 15u); }      // at most 254
  __device__ __forceinline__ float down() const { return __uint_as_float((268 - field()) << 23); }
  __device__ __forceinline__ float up() const { return __uint_as_float((field() - 14) << 23); }
};

// Eight values of x @ W on their way: two to a register where they lie in y, fp32 elsewhere.
template <typename T> struct OnTheWay {
  u32x4 w;
  __device__ __forceinline__ float get(int i) const { return widen(T{uint16_t(w[i / 2] >> 16 * (i & 1))}); }
};
template <> struct OnTheWay<float> {
  u32x4 w[2];
  __device__ __forceinline__ float get(int i) const { return __uint_as_float(w[i / 4][i % 4]); }
};

// Many rows: y[t] = x @ W + scale * low @ B, for x @ W in fp32 (P float: all rows are written, and rounded once) or in y as it is (P = T: the
// rows that have an adapter).  A wave takes 16 rows and strips of 128 columns, one after the other, 16 bytes to a lane.  The next strip's
// x @ W and B are on their way while one is written: of 4 waves and one strip at a time 8192 x 4096 took 65 us, five trips to memory one after the other for each.
// NK: steps of 32 of the rank that are held.
// ALIGNED: y's rows begin at whole 16 bytes; its accesses are then non-temporal (P = T, 8192 x 4096, with x @ A 57 -> 52 us).  Elsewhere
// neighbours share cache lines, and are not (8192 x 4099 72 us, non-temporal 75).  Nor is x @ W in fp32, which the product has just
// written (8192 rows of 4096 -> 4096 with the product 285 -> 282 us).
// that a compute unit holds; of fp32 rows three would spill (column-major B) or give nothing (282 us both ways)
constexpr int add_groups(int NK, bool here) { return NK == 1 && here ? 3 : 2; }

template <typename T, typename P, int LAY, int NK, bool ALIGNED>
__global__ void __launch_bounds__(kThreads, add_groups(NK, sizeof(P) == 2)) lora_add_kernel(const LoraArgs a) {
  using S = Skinny<T, GMM_W_ROWS, 8, 1, 2, GMM_A_STAGED, 1>;
  constexpr int FR = S::FR, OUT = S::COLUMNS, POLICY = ALIGNED ? kStream : 0;
  constexpr bool HERE = sizeof(P) == 2;      // x @ W lies in y
  constexpr bool FP16 = std::is_same_v<T, F16>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int first = (blockIdx.x * kWaves + wave) * 16;
  const int id = first + j < a.rows ? a.adapter[first + j] : -1;
  const uint32_t with = uint32_t(__ballot(has_adapter(id, a.L))) & 0xffffu;
  const int there = min(16, a.rows - first);
  if (HERE ? !with : there <= 0) return;
  const uint32_t none = HERE ? 0 : ~with & ((1u << there) - 1);      // rows that only have to be rounded
  const float* const low = a.sums + int64_t(min(first + j, a.rows - 1)) * a.pitch + 8 * g;
  const int tile0 = blockIdx.y * a.strips, tiles = min(a.strips, (a.N + OUT - 1) / OUT - tile0);
  // y from row `first` on; what is not to be read or written lies nowhere, so that no branch stands around an access
  const __amdgpu_buffer_rsrc_t y = buffer(static_cast<T*>(a.out) + first * a.out_ld, uint32_t(((there - 1) * a.out_ld + a.N) * 2));
  const uint32_t y_at = uint32_t(4 * g) * uint32_t(a.out_ld) * 2, y_step = uint32_t(a.out_ld) * 2;
  const __amdgpu_buffer_rsrc_t base = HERE ? y : buffer(a.base + int64_t(first) * a.N, uint32_t(there) * a.N * 4);
  const auto load_y = [&](OnTheWay<P> (&old)[4], int tile, uint32_t mine) {
    const int c = (tile0 + tile) * OUT + FR * j;
    const uint32_t step = HERE ? y_step : uint32_t(a.N) * 4, at = 4 * g * step + uint32_t(min(c, a.N - FR)) * uint32_t(sizeof(P));
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int from = int(mine >> (4 * g + v) & 1 && c < a.N ? at + v * step : kNowhere);
      if constexpr (HERE) {
        old[v].w = __builtin_amdgcn_raw_buffer_load_b128(base, from, 0, POLICY);
      } else {
        old[v].w[0] = __builtin_amdgcn_raw_buffer_load_b128(base, from, 0, 0);
        old[v].w[1] = __builtin_amdgcn_raw_buffer_load_b128(base, from, 16, 0);
      }
    }
  };
  const auto store_y = [&](const u32x4 (&now)[4], int tile, uint32_t mine) {
    const int c = (tile0 + tile) * OUT + FR * j, left = a.N - c;
    const uint32_t at = y_at + uint32_t(c) * 2;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const u32x4 p = now[v];
      const bool in = mine >> (4 * g + v) & 1;
      __builtin_amdgcn_raw_buffer_store_b128(p, y, int(in && left >= FR ? at + v * y_step : kNowhere), 0, POLICY);
      if (in && left > 0 && left < FR) {      // the lane that has fewer than eight: they are the last ones of what it loaded
        const uint32_t last = at + v * y_step + 2 * left - 2;
#pragma unroll
        for (int i = 1; i < FR; ++i)
          if (i >= FR - left) __builtin_amdgcn_raw_buffer_store_b16(uint16_t(p[i / 2] >> 16 * (i & 1)), y, int(last - 2 * (FR - 1 - i)), 0, 0);
      }
    }
  };
  S s;
  s.lane = lane;
  const auto load_b = [&](u32x4 (&w)[8], int tile, int k) {
    s.set_columns((tile0 + tile) * OUT, a.N - (tile0 + tile) * OUT, a.b.sk, a.b.sn);
    if constexpr (LAY == GMM_W_ROWS) {
      s.load_w(w, k, a.R);
    } else {      // a rank's values of a column lie side by side: the operands as they are
#pragma unroll
      for (int i = 0; i < FR; ++i)
        w[i] = __builtin_amdgcn_raw_buffer_load_b128(
            s.w_buf, int(s.columns && k + 8 * g < a.R ? s.w_at + i * s.w_step_n + (k + 8 * g) * 2 - S::back(k + 8 * g, a.R) : kNowhere), 0, 0);
    }
  };
  const auto multiply = [&](u32x4 (&w)[8], int k, u32x4 h, u32x4 l, f32x4 (&acc)[FR]) {
    if (LAY != GMM_W_ROWS && k + 32 > a.R) {
#pragma unroll
      for (int i = 0; i < FR; ++i) w[i] = S::tail(w[i], k + 8 * g, a.R);
    }
#pragma unroll
    for (int i = 0; i < FR; ++i) {
      const u32x4 b = LAY == GMM_W_ROWS ? S::turned(w, i) : w[i];
      acc[i] = mfma(T{}, h, b, acc[i]);
      acc[i] = mfma(T{}, l, b, acc[i]);
    }
  };
  // strips, and in a strip the adapters of the rows, one after the other: one sequence
  u32x4 h[NK], l[NK], w[NK][8];
  OnTheWay<P> next[4];
  Exponent exponent;
  const auto load_low = [&](int k) {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int at = k + 32 * n;      // of a lane's eight values none are there, or all
      const bool in = at + 8 * g < a.pitch;
      const Pack<float, 8> v = *reinterpret_cast<const Pack<float, 8>*>(low + (in ? at : -8 * g));
      T high[8], rest[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) split(in ? (FP16 ? v.get(i) * exponent.down() : v.get(i)) : 0.0f, high[i], rest[i]);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        h[n][q] = uint32_t(high[2 * q].bits) | uint32_t(high[2 * q + 1].bits) << 16;
        l[n][q] = uint32_t(rest[2 * q].bits) | uint32_t(rest[2 * q + 1].bits) << 16;
      }
    }
  };
  Adapters ahead{with, 0, 0};
  int tile = 0;
  const auto go_on = [&] {      // rows without an adapter come with a strip's first adapter, or alone
    const bool first_one = ahead.todo == with;
    if (HERE || with) ahead.next(id);
    ahead.mine = first_one ? ahead.mine | none : ahead.mine;
    s.w_buf = HERE || with ? matrix<T>(a.b, ahead.which) : buffer(a.b.at, 0);
  };
  go_on();
#pragma unroll
  for (int n = 0; n < NK; ++n) load_b(w[n], 0, 32 * n);
  load_y(next, 0, ahead.mine);
  __builtin_amdgcn_sched_barrier(0);
  float up[4];      // of the lane's rows of the result
  if constexpr (FP16) {
    for (int k = 0; k + 8 * g < a.pitch; k += 32)
#pragma unroll
      for (int i = 0; i < 8; ++i) exponent.take(low[k + i]);
    exponent.join(16);
    exponent.join(32);
#pragma unroll
    for (int v = 0; v < 4; ++v) up[v] = __shfl(exponent.up(), 4 * g + v);
  }
  load_low(0);
#pragma unroll 1
  while (tile < tiles) {
    const uint32_t mine = ahead.mine;
    const int here = tile;
    f32x4 acc[FR];
#pragma unroll
    for (int i = 0; i < FR; ++i) acc[i] = f32x4{0, 0, 0, 0};
#pragma unroll 1
    for (int k = 0;;) {
#pragma unroll
      for (int n = 0; n < NK; ++n) multiply(w[n], k + 32 * n, h[n], l[n], acc);
      k += 32 * NK;
      if (k >= a.R) break;
      load_low(k);
#pragma unroll
      for (int n = 0; n < NK; ++n) load_b(w[n], here, k + 32 * n);
    }
    if (a.R > 32 * NK) load_low(0);
    if (!ahead.todo) {
      ahead.todo = with;
      ++tile;
    }
    go_on();
    const int then = min(tile, tiles - 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < NK; ++n) load_b(w[n], then, 32 * n);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 now[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      float sum[FR];
#pragma unroll
      for (int i = 0; i < FR; ++i) sum[i] = next[v].get(i) + (HERE || with >> (4 * g + v) & 1 ? (FP16 ? acc[i][v] * up[v] : acc[i][v]) : 0.0f);
      now[v] = Pack<T, 8>::of(sum).w;
    }
    load_y(next, then, tile < tiles ? ahead.mine : 0);
    __builtin_amdgcn_sched_barrier(0);
    store_y(now, here, mine);
  }
}

// The same where neither step of B is one element, or there are fewer than eight columns: a thread has one column and 16 rows, and multiplies on the vector units, in fp32.
constexpr int kAnyRows = 16;

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) lora_add_any_kernel(const LoraArgs a) {
  constexpr bool HERE = sizeof(P) == 2;      // as above
  __shared__ f32x4 low[kAnyRows][kMaxRank / 4 + 1];
  const int row0 = blockIdx.x * kAnyRows, c = blockIdx.y * kThreads + threadIdx.x, lane = threadIdx.x & 63;
  const int span = int(a.R + 3) / 4 * 4;
  for (int u = threadIdx.x; u < kAnyRows * span; u += kThreads) {
    reinterpret_cast<float*>(low[u / span])[u % span] = a.sums[int64_t(min(row0 + u / span, a.rows - 1)) * a.pitch + u % span];
  }
  __syncthreads();
  const int id = lane < kAnyRows && row0 + lane < a.rows ? a.adapter[row0 + lane] : -1;
  const uint32_t with = uint32_t(__ballot(has_adapter(id, a.L)));
  if (c >= a.N) return;
  T* const y = static_cast<T*>(a.out) + int64_t(row0) * a.out_ld + c;
  const float* const base = HERE ? nullptr : a.base + int64_t(row0) * a.N + c;
  if constexpr (!HERE)
    for (int t = 0; t < min(kAnyRows, a.rows - row0); ++t)
      if (!(with >> t & 1)) y[t * a.out_ld] = rounded<T>(base[int64_t(t) * a.N]);
  for (uint32_t todo = with; todo;) {
    const int which = __builtin_amdgcn_readlane(id, __ffs(todo) - 1);
    uint32_t mine = 0;
    for (int t = 0; t < kAnyRows; ++t) mine |= __builtin_amdgcn_readlane(id, t) == which ? 1u << t : 0u;
    todo &= ~mine;
    const T* b = static_cast<const T*>(a.b.at) + which * a.b.sg + int64_t(c) * a.b.sn;
    float acc[kAnyRows];
#pragma unroll
    for (int t = 0; t < kAnyRows; ++t) acc[t] = 0;
    for (int r = 0; r < a.R; r += 4) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = r + i < a.R ? widen(b[int64_t(r + i) * a.b.sk]) : 0.0f;
#pragma unroll
      for (int t = 0; t < kAnyRows; ++t) {
        const f32x4 l = low[t][r / 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t] += l[i] * v[i];
      }
    }
#pragma unroll
    for (int t = 0; t < kAnyRows; ++t)
      if (mine >> t & 1) y[t * a.out_ld] = rounded<T>((HERE ? widen(y[t * a.out_ld]) : base[int64_t(t) * a.N]) + acc[t]);
  }
}

// ---------------------------------------------------------------- gradients
// Rows are sorted by adapter; adapter i's begin at place(i) of the sorted operands: a multiple of 8, so that 8 rows' values can be read
// 16 bytes at a time, and past all that earlier adapters have.
__device__ __forceinline__ int place(const int32_t* offs, int i) { return ((i ? offs[i - 1] : 0) + 7) / 8 * 8 + 8 * i; }

// One of the two gradients: out[i] = q^T p over adapter i's rows.
struct GradOf {
  const void* p;            // [rows][C]: x or dy
  const void* q;            // [2][R][places]: u or low by place, times scale (fp16: and an Exponent's power of two): high and low halves
  const uint32_t* peak;     // fp16: [peak_parts][L][R]: what an Exponent takes of the adapter's rows
  void* out;                // [L][R][C] with the strides below
  float* partial;           // [slots][R * C] as `out` has it: of adapters whose rows are more than one chunk
  int64_t p_ld, out_sg, out_sr, out_sc;
  int32_t C, tiles;
  int32_t r_first;          // out is contiguous along R (of partial: always along one of the two)
};

struct GradArgs {
  GradOf of[2];
  const int32_t* row_at;    // [places] the row at a place
  const int32_t* offs;      // [L + 1] ends of the adapters' rows
  int32_t places, R, L, chunk, groups0;   // groups0: workgroups of of[0]
  int32_t peak_parts;
};

// fp16: the power of two that rank r of adapter i's values are brought down by, all rows alike, as the sum over them needs it.
__device__ __forceinline__ Exponent exponent_of(const uint32_t* peak, int parts, int L, int R, int i, int r) {
  Exponent e;
  in_fours(parts, [&](int p, bool) { e.most = max(e.most, peak[(int64_t(p) * L + i) * R + r]); });
  return e;
}

// An adapter's n rows are dealt evenly to as many chunks as are needed (one for no rows: its gradient is zero).
__device__ __forceinline__ int chunks_of(int n, int chunk) { return n > chunk ? (n + chunk - 1) / chunk : 1; }

// The `which`-th chunk of all adapters' rows: its adapter, first place, number of rows; slot: of its partial sums, -1: it is the only one.
__device__ __forceinline__ bool find_chunk(const GradArgs& a, int which, int& adapter, int& first, int& rows, int& slot) {
  const int lane = threadIdx.x & 63;
  int slots = 0;
  for (int base = 0; base < a.L; base += 64) {
    const int i = base + lane;
    const int from = i < a.L && i ? a.offs[i - 1] : 0, n = i < a.L ? a.offs[i] - from : 0;
    const int chunks = i < a.L ? chunks_of(n, a.chunk) : 0, own = chunks > 1 ? chunks : 0;
    int sum = chunks, slot_sum = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int s = __shfl_up(sum, o), t = __shfl_up(slot_sum, o);
      if (lane >= o) { sum += s; slot_sum += t; }
    }
    const uint64_t it = __ballot(which < sum);
    if (it) {
      const int at = __ffsll(static_cast<unsigned long long>(it)) - 1;
      const int count = __builtin_amdgcn_readlane(chunks, at), all = __builtin_amdgcn_readlane(n, at);
      const int c = which - (__builtin_amdgcn_readlane(sum, at) - count), each = ((all + count - 1) / count + 7) / 8 * 8;
      adapter = base + at;
      first = place(a.offs, adapter) + c * each;
      rows = max(0, min(each, all - c * each));
      slot = count > 1 ? slots + __builtin_amdgcn_readlane(slot_sum, at) - count + c : -1;
      return true;
    }
    which -= __builtin_amdgcn_readlane(sum, 63);
    slots += __builtin_amdgcn_readlane(slot_sum, 63);
  }
  return false;
}

constexpr int kPiece = 4096;      // rows of a chunk whose places are in LDS at a time

// out[i] += q^T p over a chunk of adapter i's rows: R rows, a strip of 128 columns of p, the contraction along p's rows.
// WHOLE: there are eight columns.
template <typename T, int MF, bool WHOLE>
__global__ void __launch_bounds__(kThreads) lora_grad_kernel(const GradArgs args) {
  using S = Skinny<T, GMM_W_ROWS, 8, MF, 2, GMM_A_STAGED, 2>;
  constexpr int FR = S::FR, OUT = S::COLUMNS;
  __shared__ SkinnyShared<S, kWaves> shared;
  __shared__ int32_t row_at[kPiece];
  __shared__ __align__(16) float up[16 * MF];
  constexpr bool FP16 = std::is_same_v<T, F16>;
  const bool second = int(blockIdx.x) >= args.groups0;
  const GradOf& a = args.of[second];
  const int item = blockIdx.x - (second ? args.groups0 : 0);
  int adapter, first, rows, slot;
  if (!find_chunk(args, item / a.tiles, adapter, first, rows, slot)) return;
  const int tile = item % a.tiles, r0 = blockIdx.y * 16 * MF;
  if constexpr (FP16)
    if (int(threadIdx.x) < 16 * MF)
      up[threadIdx.x] = exponent_of(a.peak, args.peak_parts, args.L, args.R, adapter, min(r0 + int(threadIdx.x), args.R - 1)).up();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, g = lane >> 4;
  const int c = tile * OUT + FR * j, columns = max(0, min(FR, a.C - c)), R = args.R, end = (rows + 7) / 8 * 8;   // zeros behind the last row
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.a_plane = uint32_t(R) * args.places * 2;
  s.a_buf = buffer(a.q, 2 * s.a_plane);
  s.set_rows([&](int r) { return r0 + r < R ? (uint32_t(r0 + r) * args.places + first) * 2 : kNowhere; });
  // Steps as Skinny has them, from rows that are anywhere (64-bit addresses).  Past the end of a piece its last row is read again and not used.
  const T* const p = static_cast<const T*>(a.p) + (WHOLE ? min(c, a.C - FR) : columns ? c : 0);
  int piece = 0, piece_end = 0;
  const auto load = [&](typename S::Step& step, int k) {
    const int kl = k + 8 * g - piece;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const T* at = p + int64_t(row_at[min(kl + r, piece_end - piece - 1)]) * a.p_ld;
      u32x4 v = {0, 0, 0, 0};
      if constexpr (WHOLE) {
        v = unaligned<u32x4>(at);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i / 2] |= uint32_t(at[max(0, min(i, columns - 1))].bits) << 16 * (i & 1);
      }
      step.w[r] = v;
    }
    s.template load_a<MF>(step, k, end);
    __builtin_amdgcn_sched_barrier(0);
  };
  const auto multiply = [&](typename S::Step& step, int k, f32x4 (&acc)[MF][FR]) {
    if (k >= piece_end) return;
    if (k + 32 > rows) {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) step.w[r][q] = k + 8 * g + r < rows ? step.w[r][q] : 0u;
    }
    s.template multiply<MF>(step, k, end, acc);
    __builtin_amdgcn_sched_barrier(0);
  };
  f32x4 acc[MF][FR];
  clear(acc);
  for (; piece < rows; piece = piece_end) {
    constexpr int NEXT = 32 * kWaves;
    static_assert(kPiece % (2 * NEXT) == 0);
    piece_end = min(rows, piece + kPiece);
    __syncthreads();
    for (int u = threadIdx.x; u < piece_end - piece; u += kThreads) row_at[u] = args.row_at[first + piece + u];
    __syncthreads();
    typename S::Step step[2];
    load(step[0], piece + 32 * wave);
    load(step[1], piece + 32 * wave + NEXT);
    for (int k = piece + 32 * wave; k < piece_end; k += 2 * NEXT)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        multiply(step[u], k + u * NEXT, acc);
        load(step[u], k + (2 + u) * NEXT);
      }
  }
#pragma unroll
  for (int m = 0; m < MF; ++m) {
    if (r0 + 16 * m >= R) break;
    __syncthreads();
    shared.sums.put(wave, lane, acc[m]);
    __syncthreads();
    for (int u = threadIdx.x; u < OUT * 4; u += kThreads) {
      const int oc = u % OUT, og = u / OUT, col = tile * OUT + oc;
      if (col >= a.C) continue;
      const int at = WHOLE ? S::position(oc, a.C - col) : oc;
      f32x4 h = shared.sums.get(S::product_of(at), S::lane_of(at), og);
      if constexpr (FP16) h *= *reinterpret_cast<const f32x4*>(up + 16 * m + 4 * og);
      const int r = r0 + 16 * m + 4 * og;
      if (slot >= 0) {
        float* const to = a.partial + int64_t(slot) * R * a.C + (a.r_first ? int64_t(col) * R + r : int64_t(r) * a.C + col);
#pragma unroll
        for (int v = 0; v < 4; ++v) if (r + v < R) to[a.r_first ? v : int64_t(v) * a.C] = h[v];
      } else {
        T* const to = static_cast<T*>(a.out) + adapter * a.out_sg + r * a.out_sr + col * a.out_sc;
        if (a.r_first == 2 && r < R) {
          const uint64_t v = uint64_t(rounded<T>(h[0]).bits) | uint64_t(rounded<T>(h[1]).bits) << 16 | uint64_t(rounded<T>(h[2]).bits) << 32 |
                             uint64_t(rounded<T>(h[3]).bits) << 48;
          *reinterpret_cast<uint64_t*>(to) = v;
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) if (r + v < R) to[v * a.out_sr] = rounded<T>(h[v]);
        }
      }
    }
  }
}

// Gradients of adapters whose rows were more than one chunk: the sum of the chunks, in order.
template <typename T>
__global__ void __launch_bounds__(kThreads) lora_grad_sum_kernel(const GradArgs args) {
  const GradOf& a = args.of[blockIdx.z];
  const int adapter = blockIdx.y, lane = threadIdx.x & 63;
  const int chunks = chunks_of(args.offs[adapter] - (adapter ? args.offs[adapter - 1] : 0), args.chunk);
  if (chunks == 1) return;
  int slot = 0;      // chunks of earlier adapters that have several
  for (int i = lane; i < adapter; i += 64) {
    const int m = chunks_of(args.offs[i] - (i ? args.offs[i - 1] : 0), args.chunk);
    slot += m > 1 ? m : 0;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) slot += __shfl_xor(slot, o);
  const int inner = a.r_first ? args.R : a.C, each = args.R * a.C;
  const int64_t s_outer = a.r_first ? a.out_sc : a.out_sr, s_inner = a.r_first ? a.out_sr : a.out_sc;
  for (int u = blockIdx.x * kThreads + threadIdx.x; u < each; u += gridDim.x * kThreads) {
    float s = 0;
#pragma unroll 4
    for (int k = 0; k < chunks; ++k) s += a.partial[int64_t(slot + k) * each + u];
    static_cast<T*>(a.out)[adapter * a.out_sg + u / inner * s_outer + u % inner * s_inner] = rounded<T>(s);
  }
}

// The largest absolute values of each adapter's rows of q1 and q2 [rows][R] times scale (either may be null), for exponent_of: part `y` of them,
// q1 or q2 by `z`.
__global__ void __launch_bounds__(kThreads) lora_peak_kernel(const float* __restrict__ q1, const float* __restrict__ q2,
                                                             const float* __restrict__ scale, const int32_t* __restrict__ row_token,
                                                             const int32_t* __restrict__ offs, int R, int L, uint32_t* __restrict__ peak1,
                                                             uint32_t* __restrict__ peak2) {
  __shared__ uint32_t most[kThreads];
  const float* const q = blockIdx.z ? q2 : q1;
  const int i = blockIdx.x, part = blockIdx.y, parts = gridDim.y;
  const int begin = i ? offs[i - 1] : 0, n = q ? offs[i] - begin : 0;
  const int from = begin + int(int64_t(n) * part / parts), to = begin + int(int64_t(n) * (part + 1) / parts);
  const int columns = 1 << (32 - __clz(R - 1)), lines = kThreads / columns;      // (of one column: 1 << 0)
  const int r = threadIdx.x % columns;
  const float by = scale ? scale[i] : 1.0f;
  Exponent e;
  if (r < R)
    for (int k = from + int(threadIdx.x) / columns; k < to; k += 8 * lines)
#pragma unroll
      for (int u = 0; u < 8; ++u) e.take(q[int64_t(row_token[min(k + u * lines, to - 1)]) * R + r] * by);      // past the end the last one again
  most[threadIdx.x] = e.most;
  __syncthreads();
  if (int(threadIdx.x) >= R) return;
  for (int k = 1; k < lines; ++k) e.most = max(e.most, most[threadIdx.x + k * columns]);
  (blockIdx.z ? peak2 : peak1)[(int64_t(part) * L + i) * R + r] = e.most;
}

// Sorted operands: q1 and q2 [rows][R] fp32 (either may be null) as [2][R][places] 16-bit halves, times scale; rows by place.
template <typename T>
__global__ void __launch_bounds__(kThreads) lora_sorted_kernel(const float* __restrict__ q1, const float* __restrict__ q2,
                                                               const float* __restrict__ scale, const int32_t* __restrict__ adapter,
                                                               const int32_t* __restrict__ row_token, const int32_t* __restrict__ offs,
                                                               int rows, int R, int L, int places, T* __restrict__ s1, T* __restrict__ s2,
                                                               int32_t* __restrict__ row_at, const uint32_t* __restrict__ peak1,
                                                               const uint32_t* __restrict__ peak2, int peak_parts) {
  const int at = blockIdx.x * kThreads + threadIdx.x, r = blockIdx.y;
  const int row = row_token[min(at, rows - 1)], id = adapter[row];
  float down[2] = {1.0f, 1.0f};
  if constexpr (std::is_same_v<T, F16>) {
    // a wave of one adapter's rows looks the parts up together (gradients of 8192 rows of one adapter of rank 64 115 -> 111 us)
    const int lead = __builtin_amdgcn_readfirstlane(id), lane = threadIdx.x & 63;
    const bool together = __all(id == lead);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t* const peak = i ? peak2 : peak1;
      if (!(i ? q2 : q1) || !has_adapter(id, L)) continue;
      Exponent e;
      if (together) {
        e.most = peak[(int64_t(min(lane, peak_parts - 1)) * L + lead) * R + r];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) e.join(o);
      } else {
        e = exponent_of(peak, peak_parts, L, R, id, r);
      }
      down[i] = e.down();
    }
  }
  if (at >= rows || !has_adapter(id, L)) return;
  const int to = place(offs, id) + at - (id ? offs[id - 1] : 0);
  const float by = scale ? scale[id] : 1.0f;
  if (r == 0) row_at[to] = row;
  const int64_t plane = int64_t(R) * places, slot = int64_t(r) * places + to;
  if (q1) split(q1[int64_t(row) * R + r] * by * down[0], s1[slot], s1[plane + slot]);
  if (q2) split(q2[int64_t(row) * R + r] * by * down[1], s2[slot], s2[plane + slot]);
  // the adapter's last row: the places behind it, up to a multiple of 8, are read with it
  if (at == offs[id] - 1)
    for (int64_t t = slot + 1; t % 8; ++t) {
      if (q1) s1[t] = s1[plane + t] = T{};
      if (q2) s2[t] = s2[plane + t] = T{};
    }
}

// ---------------------------------------------------------------- host side
int clamp(int64_t v, int64_t lo, int64_t hi) { return int(v > hi ? (hi < lo ? lo : hi) : v < lo ? lo : v); }

// `want` parts of k elements, each a multiple of 64 and at least `least` long.
void cut(int64_t k, int64_t want, int64_t least, int32_t& parts, int32_t& each) {
  parts = clamp(want, 1, k / least);
  each = int32_t(round_up((k + parts - 1) / parts, 64));
  parts = each ? int32_t((k + each - 1) / each) : 1;
}


struct LowPlan { int32_t strip_rows, parts, each; };

LowPlan plan_low(int64_t rows, int64_t K, int64_t R) {
  LowPlan p;
  p.strip_rows = rows <= kSingleRows ? 1 : 16;
  const int64_t strips = (rows + p.strip_rows - 1) / p.strip_rows;
  if (rows <= kFewRows) cut(K, strips ? 128 / strips : 1, 512, p.parts, p.each);
  else if (R <= 16) cut(K, 256 / strips, 1024, p.parts, p.each);
  else cut(K, 2048 / strips, 256, p.parts, p.each);
  return p;
}

struct BasePlan { int32_t parts, each; };

// A workgroup for each compute unit.
BasePlan plan_base(int64_t K, int64_t N, int columns) {
  BasePlan p;
  const int64_t strips = (N + columns - 1) / columns, cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  cut(K, strips ? (cus + strips / 2) / strips : 1, 512, p.parts, p.each);
  return p;
}

template <typename F>
void by_layout(int lay, F&& f) {
  if (lay == GMM_W_ROWS) f(std::integral_constant<int, GMM_W_ROWS>{});
  else if (lay == GMM_W_COLS) f(std::integral_constant<int, GMM_W_COLS>{});
  else f(std::integral_constant<int, GMM_W_ANY>{});
}

int strip_columns(int lay) { return lay == GMM_W_COLS ? 64 : 128; }

int layout_of(const Matrices& m, int64_t K, int64_t N) { return gmm::layout_of(m.sk, m.sn, K, N); }

// B's layout: nothing is asked of the rank where it is contiguous along its columns.
int layout_of_b(const Matrices& b, int64_t R, int64_t N) {
  if (N < 8) return GMM_W_ANY;
  return b.sn == 1 ? GMM_W_ROWS : b.sk == 1 && R >= 8 ? GMM_W_COLS : GMM_W_ANY;
}

bool set(Matrices& m, const void* at, int64_t sg, int64_t sk, int64_t sn, int64_t K, int64_t N) {
  if (sg < 0 || sk < 0 || sn < 0) return false;
  m.at = at; m.sg = sg;
  m.bytes = K && N ? matrix_bytes(K, N, sk, sn) : 2;
  m.sk = K > 1 ? uint32_t(sk) : sk == 1 ? 1 : uint32_t(round_up(N, 8));      // of no matter: such that it does not decide the layout
  m.sn = N > 1 ? uint32_t(sn) : sn == 1 ? 1 : uint32_t(round_up(K, 8));
  return m.bytes != 0;
}

int check_sizes(int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int32_t dtype) {
  constexpr int64_t most = int64_t(1) << 22, most_rows = int64_t(1) << 26;
  if (rows < 0 || K < 0 || N < 0 || R < 1 || L < 0 || rows >= most_rows || K >= most || N >= most || R > kMaxRank || L > kMaxAdapters) return GMM_ERR_BAD_ARGUMENT;
  return dtype == GMM_DT_BF16 || dtype == GMM_DT_F16 ? GMM_OK : GMM_ERR_UNSUPPORTED;
}

// Rows that are read (or written) a strip of them at a time, from one base.
bool x_fits(int64_t x_ld, int64_t rows, int64_t K) {
  return rows <= 1 || (x_ld >= K && x_ld <= ((int64_t(1) << 30) - 64 - K) / (rows < kFewRows ? rows : kFewRows));
}

void set_low(LoraArgs& a, int columns) {
  const LowPlan lp = plan_low(a.rows, a.K, a.R);
  a.strip_rows = lp.strip_rows; a.low_parts = lp.parts; a.low_k = lp.each;
  a.low_tiles = (a.R + columns - 1) / columns;
  a.low_groups = (a.rows + a.strip_rows - 1) / a.strip_rows * a.low_tiles * a.low_parts;
}

template <typename T>
int launch_finish(const LoraArgs& a, hipStream_t stream) {
  by_layout(layout_of_b(a.b, a.R, a.N), [&](auto l) {
    constexpr int B = decltype(l)::value, W = B == GMM_W_ROWS ? 8 : 1;
    hipLaunchKernelGGL((lora_finish_kernel<T, B>), dim3(unsigned(a.N ? (a.N + 64 * W - 1) / (64 * W) : 1), unsigned(a.rows)), dim3(64), 0, stream, a);
  });
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

template <typename T>
int launch_few(LoraArgs a, hipStream_t stream) {
  const int lay_w = layout_of(a.w, a.K, a.N);
  const int lay_a = lay_w == GMM_W_ANY ? GMM_W_ANY : layout_of(a.a, a.K, a.R);
  set_low(a, 16);
  const BasePlan bp = plan_base(a.K, a.N, strip_columns(lay_w));
  a.base_parts = bp.parts; a.base_k = bp.each;
  a.base_tiles = (a.N + strip_columns(lay_w) - 1) / strip_columns(lay_w);
  if (a.L == 0) a.low_groups = 0;
  const dim3 grid(unsigned(a.low_groups + a.base_tiles * a.base_parts));
  const auto launch = [&](auto w, auto l) {
    constexpr int W = decltype(w)::value, A = decltype(l)::value;
    if (a.rows <= 16) hipLaunchKernelGGL((lora_few_kernel<T, W, A, 1>), grid, dim3(64 * few_waves(1, W)), 0, stream, a);
    else if (a.rows <= 32) hipLaunchKernelGGL((lora_few_kernel<T, W, A, 2>), grid, dim3(64 * few_waves(2, W)), 0, stream, a);
    else hipLaunchKernelGGL((lora_few_kernel<T, W, A, 4>), grid, dim3(64 * few_waves(4, W)), 0, stream, a);
  };
  constexpr std::integral_constant<int, GMM_W_ROWS> rows{};
  constexpr std::integral_constant<int, GMM_W_COLS> cols{};
  constexpr std::integral_constant<int, GMM_W_ANY> any{};
  constexpr std::integral_constant<int, GMM_W_THIN> thin{};
  const auto with_a = [&](auto w) {
    if (lay_a == GMM_W_COLS) launch(w, cols);
    else if (lay_a == GMM_W_ROWS) launch(w, thin);
    else launch(w, any);
  };
  if (lay_w == GMM_W_ROWS) with_a(rows);
  else if (lay_w == GMM_W_COLS) with_a(cols);
  else launch(any, any);
  return launch_finish<T>(a, stream);
}

// Columns of a strip: as few as hold the rank.
template <typename T>
int launch_low(LoraArgs& a, hipStream_t stream) {
  const int lay = layout_of(a.a, a.K, a.R);
  int fr = a.R <= 16 ? 1 : a.R <= 32 ? 2 : a.R <= 64 || lay == GMM_W_COLS ? 4 : 8;
  if (lay == GMM_W_ANY) fr = 1;
  set_low(a, 16 * fr);
  const dim3 grid(unsigned(a.low_groups));
  const bool edge = a.K < 8;
  const auto launch = [&](auto l, auto n, auto e) {
    constexpr int LAY = decltype(l)::value, FR = decltype(n)::value;
    hipLaunchKernelGGL((lora_low_kernel<T, LAY, FR, decltype(e)::value>), grid, dim3(64 * low_waves(FR)), 0, stream, a);
  };
  constexpr std::integral_constant<int, 1> one{};
  constexpr std::integral_constant<int, 2> two{};
  constexpr std::integral_constant<int, 4> four{};
  if (lay == GMM_W_COLS) {
    constexpr std::integral_constant<int, GMM_W_COLS> cols{};
    if (fr == 1) launch(cols, one, std::false_type{});
    else if (fr == 2) launch(cols, two, std::false_type{});
    else launch(cols, four, std::false_type{});
  } else if (lay == GMM_W_ROWS) {
    constexpr std::integral_constant<int, GMM_W_THIN> thin{};
    if (fr == 1) launch(thin, one, std::false_type{});
    else if (fr == 2) launch(thin, two, std::false_type{});
    else if (fr == 4) launch(thin, four, std::false_type{});
    else launch(std::integral_constant<int, GMM_W_ROWS>{}, std::integral_constant<int, 8>{}, std::false_type{});
  } else {
    constexpr std::integral_constant<int, GMM_W_ANY> any{};
    if (edge) launch(any, one, std::true_type{});
    else launch(any, one, std::false_type{});
  }
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

int64_t pitch_of(int64_t R) { return round_up(R, 16); }

template <typename T, typename P>
int launch_add(LoraArgs a, hipStream_t stream) {
  a.pitch = int(pitch_of(a.R));
  a.keep = a.rows > kSingleRows;
  const int rc = a.L ? launch_low<T>(a, stream) : GMM_OK;
  if (rc != GMM_OK) return rc;
  if (!a.keep) return launch_finish<T>(a, stream);
  const unsigned blocks = unsigned((int64_t(a.rows) * a.pitch + kThreads - 1) / kThreads);
  if (a.L && a.low_parts > 1) hipLaunchKernelGGL(lora_low_sum_kernel, dim3(blocks), dim3(kThreads), 0, stream, a);
  if (a.N) {
    const int lay = layout_of_b(a.b, a.R, a.N);
    const dim3 any((a.rows + kAnyRows - 1) / kAnyRows, (a.N + kThreads - 1) / kThreads);
    // strips to a wave: as many as leave every place for one a wave (rank 64: for three groups 54 us, for the two that there is room for 50)
    const int tiles = (a.N + 127) / 128, row_groups = (a.rows + 16 * kWaves - 1) / (16 * kWaves);
    a.strips = clamp(int64_t(row_groups) * tiles / (add_groups(a.R <= 32 ? 1 : 2, sizeof(P) == 2) * gmm_num_cus()), 1, tiles);
    const dim3 grid(row_groups, (tiles + a.strips - 1) / a.strips);
    const auto launch = [&](auto lay, auto nk) {
      constexpr int B = decltype(lay)::value, NK = decltype(nk)::value;
      if (aligned16(a.out) && a.out_ld % 8 == 0) hipLaunchKernelGGL((lora_add_kernel<T, P, B, NK, true>), grid, dim3(kThreads), 0, stream, a);
      else hipLaunchKernelGGL((lora_add_kernel<T, P, B, NK, false>), grid, dim3(kThreads), 0, stream, a);
    };
    const auto rank = [&](auto lay) {
      if (a.R <= 32) launch(lay, std::integral_constant<int, 1>{});
      else launch(lay, std::integral_constant<int, 2>{});
    };
    if (lay == GMM_W_ANY) hipLaunchKernelGGL((lora_add_any_kernel<T, P>), any, dim3(kThreads), 0, stream, a);
    else if (lay == GMM_W_ROWS) rank(std::integral_constant<int, GMM_W_ROWS>{});
    else rank(std::integral_constant<int, GMM_W_COLS>{});
  }
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

// Where the operands of gmm_lora_grad lie in its workspace.
struct GradPlan {
  int64_t places, offs_at, token_at, rows_at, table_at, row_at, q_at[2], partial_at[2], peak_at[2], bytes;
  int32_t chunk, peak_parts;
};

bool plan_grad(int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, GradPlan& p) {
  const int64_t table = gmm_moe_route_workspace_bytes(rows, L + 1, 1);
  if (table < 0) return false;
  // chunks: as long as leaves some workgroups, one for a chunk and 128 columns, to a compute unit, up to 4096 rows; or a 32nd of all rows, so
  // that the partial sums stay few (1 million rows of 4096 -> 4096, rank 64: 0.7 GB with the operands, in chunks of 4096 rows 1.6)
  const int64_t tiles = (K + 127) / 128 + (N + 127) / 128, least = round_up(rows / 32, 128);
  p.chunk = clamp(round_up(rows * tiles / 1024 > rows / 32 ? rows * tiles / 1024 : rows / 32, 128), 256, least > 4096 ? least : 4096);
  p.places = round_up(rows, 8) + 8 * (L + 1);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) { const int64_t here = at; at = round_up(at + bytes, 256); return here; };
  p.offs_at = take((L + 1) * 4);
  p.token_at = take(rows * 4);
  p.rows_at = take(rows * 4);
  p.table_at = take(table);
  p.row_at = take(p.places * 4);
  for (int i = 0; i < 2; ++i) p.q_at[i] = take(2 * R * p.places * 2);
  for (int i = 0; i < 2; ++i)      // adapters of several chunks have fewer than two for each chunk of all rows
    p.partial_at[i] = take(2 * (rows / p.chunk) * R * (i ? N : K) * 4);
  // as many as leave a thread two trips to memory or so (8192 rows of one adapter, rank 64, in 8 parts: 28 us), while there are few adapters
  p.peak_parts = clamp(rows * R / 8192, 1, clamp(1024 / (L + 1), 1, 32));
  for (int i = 0; i < 2; ++i) p.peak_at[i] = take(int64_t(p.peak_parts) * L * R * 4);
  p.bytes = at;
  return 2 * R * p.places * 2 < (int64_t(1) << 31) && R * K < (int64_t(1) << 30) && R * N < (int64_t(1) << 30);
}

void set_grad(GradOf& g, const void* p, int64_t p_ld, const void* q, void* out, float* partial, int64_t C, int64_t R, int64_t sg, int64_t sr,
              int64_t sc) {
  g.p = p; g.q = q; g.out = out; g.partial = partial; g.p_ld = p_ld;
  g.out_sg = sg; g.out_sr = sr; g.out_sc = sc;
  g.C = int32_t(C);
  g.tiles = out ? int32_t((C + 127) / 128) : 0;
  const bool four = (reinterpret_cast<uintptr_t>(out) & 7) == 0 && R % 4 == 0 && sg % 4 == 0 && sc % 4 == 0;   // four of R in 8 bytes
  g.r_first = sr != 1 || R == 1 ? 0 : four ? 2 : 1;
}

template <typename T>
int launch_grad(GradArgs& g, int64_t rows, hipStream_t stream) {
  const int64_t chunks = rows / g.chunk + g.L;
  g.groups0 = int32_t(chunks * g.of[0].tiles);
  const int64_t groups = g.groups0 + chunks * g.of[1].tiles;
  if (groups == 0) return GMM_OK;
  const bool whole = (!g.of[0].tiles || g.of[0].C >= 8) && (!g.of[1].tiles || g.of[1].C >= 8);
  const auto launch = [&](auto mf) {
    constexpr int MF = decltype(mf)::value;
    const dim3 grid(unsigned(groups), unsigned((g.R + 16 * MF - 1) / (16 * MF)));
    if (whole) hipLaunchKernelGGL((lora_grad_kernel<T, MF, true>), grid, dim3(kThreads), 0, stream, g);
    else hipLaunchKernelGGL((lora_grad_kernel<T, MF, false>), grid, dim3(kThreads), 0, stream, g);
  };
  if (g.R <= 16) launch(std::integral_constant<int, 1>{});
  else if (g.R <= 32) launch(std::integral_constant<int, 2>{});
  else launch(std::integral_constant<int, 4>{});
  if (rows > g.chunk) {      // an adapter may have several chunks
    if (!g.of[0].tiles) g.of[0] = g.of[1];
    const int64_t widest = g.of[1].tiles && g.of[1].C > g.of[0].C ? g.of[1].C : g.of[0].C;
    const int64_t blocks = (int64_t(g.R) * widest + 4 * kThreads - 1) / (4 * kThreads);
    const bool both = g.of[1].tiles && g.of[0].out != g.of[1].out;
    hipLaunchKernelGGL((lora_grad_sum_kernel<T>), dim3(unsigned(blocks < 256 ? blocks : 256), unsigned(g.L), both ? 2 : 1), dim3(kThreads), 0, stream, g);
  }
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

}  // namespace

// Bytes of the parts of x @ A.
static int64_t low_bytes(int64_t rows, int64_t K, int64_t R) { return round_up(int64_t(plan_low(rows, K, R).parts) * rows * R * 4, 256); }

// gmm_lora_sum, and with `base` null gmm_lora_add.
static int lora_add(const void* x, const void* a, const void* b, const int32_t* adapter, const float* scale, const float* base, void* out,
                    float* low, int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int64_t x_stride, int64_t a_stride_l,
                    int64_t a_stride_k, int64_t a_stride_r, int64_t b_stride_l, int64_t b_stride_r, int64_t b_stride_n, int64_t out_stride,
                    int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int bad = check_sizes(rows, K, N, R, L, dtype);
  if (bad) return bad;
  if (!out) N = 0;
  if (rows == 0 || (N == 0 && (!low || L == 0))) return GMM_OK;
  LoraArgs g{};
  if (!adapter || (L && ((N && !b) || (K && (!x || !a)))) || !x_fits(x_stride, rows, K) || !x_fits(out_stride, rows, N)) return GMM_ERR_BAD_ARGUMENT;
  if (!set(g.a, a, a_stride_l, a_stride_k, a_stride_r, K, R) || !set(g.b, b, b_stride_l, b_stride_r, b_stride_n, R, N)) return GMM_ERR_BAD_ARGUMENT;
  if (!workspace || !aligned16(workspace) || workspace_bytes < low_bytes(rows, K, R) + rows * pitch_of(R) * 4) return GMM_ERR_WORKSPACE;
  g.x = x; g.adapter = adapter; g.scale = scale; g.out = out; g.low_out = low; g.low = static_cast<float*>(workspace);
  g.sums = N ? reinterpret_cast<float*>(static_cast<char*>(workspace) + low_bytes(rows, K, R)) : nullptr;
  g.base = const_cast<float*>(base); g.base_parts = base ? 1 : 0;
  g.x_ld = rows > 1 ? x_stride : round_up(K, 8); g.out_ld = rows > 1 ? out_stride : round_up(N, 8);
  g.rows = int(rows); g.K = int(K); g.N = int(N); g.R = int(R); g.L = int(L);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (base) return dtype == GMM_DT_BF16 ? launch_add<Bf16, float>(g, s) : launch_add<F16, float>(g, s);
  return dtype == GMM_DT_BF16 ? launch_add<Bf16, Bf16>(g, s) : launch_add<F16, F16>(g, s);
}

extern "C" {

int64_t gmm_lora_workspace_bytes(int64_t rows, int64_t K, int64_t N, int64_t R) {
  if (check_sizes(rows, K, N, R, 0, GMM_DT_BF16) != GMM_OK) return -1;
  int64_t bytes = low_bytes(rows, K, R) + round_up(rows * pitch_of(R) * 4, 256);
  if (rows <= kFewRows) bytes += int64_t(plan_base(K, N, 128).parts) * rows * N * 4;     // the layout with the more parts
  return bytes;
}

int gmm_lora_linear(const void* x, const void* w, const void* a, const void* b, const int32_t* adapter, const float* scale, void* out,
                    float* low, int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int64_t x_stride, int64_t w_stride_k,
                    int64_t w_stride_n, int64_t a_stride_l, int64_t a_stride_k, int64_t a_stride_r, int64_t b_stride_l, int64_t b_stride_r,
                    int64_t b_stride_n, int64_t out_stride, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int bad = check_sizes(rows, K, N, R, L, dtype);
  if (bad) return bad;
  if (rows > kFewRows) return GMM_ERR_UNSUPPORTED;
  if (rows == 0 || N == 0) return GMM_OK;
  LoraArgs g{};
  if (!out || !adapter || (K && (!x || !w)) || (L && (!b || (K && !a))) || !x_fits(x_stride, rows, K) || !x_fits(out_stride, rows, N)) return GMM_ERR_BAD_ARGUMENT;
  if (!set(g.a, a, a_stride_l, a_stride_k, a_stride_r, K, R) || !set(g.b, b, b_stride_l, b_stride_r, b_stride_n, R, N)) return GMM_ERR_BAD_ARGUMENT;
  if (!set(g.w, w, 0, w_stride_k, w_stride_n, K, N)) return w_stride_k < 0 || w_stride_n < 0 ? GMM_ERR_BAD_ARGUMENT : GMM_ERR_UNSUPPORTED;
  if (!workspace || !aligned16(workspace) || workspace_bytes < gmm_lora_workspace_bytes(rows, K, N, R)) return GMM_ERR_WORKSPACE;
  g.x = x; g.adapter = adapter; g.scale = scale; g.out = out; g.low_out = low;
  g.low = static_cast<float*>(workspace);
  g.base = reinterpret_cast<float*>(static_cast<char*>(workspace) + low_bytes(rows, K, R));
  g.x_ld = rows > 1 ? x_stride : round_up(K, 8); g.out_ld = rows > 1 ? out_stride : round_up(N, 8);
  g.rows = int(rows); g.K = int(K); g.N = int(N); g.R = int(R); g.L = int(L);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GMM_DT_BF16 ? launch_few<Bf16>(g, s) : launch_few<F16>(g, s);
}

int gmm_lora_add(const void* x, const void* a, const void* b, const int32_t* adapter, const float* scale, void* out, float* low,
                 int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int64_t x_stride, int64_t a_stride_l, int64_t a_stride_k,
                 int64_t a_stride_r, int64_t b_stride_l, int64_t b_stride_r, int64_t b_stride_n, int64_t out_stride, int32_t dtype,
                 void* workspace, int64_t workspace_bytes, void* stream) {
  if (L == 0) return check_sizes(rows, K, N, R, L, dtype);
  return lora_add(x, a, b, adapter, scale, nullptr, out, low, rows, K, N, R, L, x_stride, a_stride_l, a_stride_k, a_stride_r, b_stride_l,
                  b_stride_r, b_stride_n, out_stride, dtype, workspace, workspace_bytes, stream);
}

int gmm_lora_sum(const void* x, const void* a, const void* b, const int32_t* adapter, const float* scale, const float* base, void* out,
                 float* low, int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int64_t x_stride, int64_t a_stride_l,
                 int64_t a_stride_k, int64_t a_stride_r, int64_t b_stride_l, int64_t b_stride_r, int64_t b_stride_n, int64_t out_stride,
                 int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int bad = check_sizes(rows, K, N, R, L, dtype);
  if (bad) return bad;
  if (rows && N && (!base || !out)) return GMM_ERR_BAD_ARGUMENT;
  return lora_add(x, a, b, adapter, scale, base, out, low, rows, K, N, R, L, x_stride, a_stride_l, a_stride_k, a_stride_r, b_stride_l,
                  b_stride_r, b_stride_n, out_stride, dtype, workspace, workspace_bytes, stream);
}

int64_t gmm_lora_grad_workspace_bytes(int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L) {
  GradPlan p;
  return check_sizes(rows, K, N, R, L, GMM_DT_BF16) == GMM_OK && plan_grad(rows, K, N, R, L, p) ? p.bytes : -1;
}

int gmm_lora_grad(const void* x, const void* dy, const float* low, const float* u, const int32_t* adapter, const float* scale, void* da,
                  void* db, int64_t rows, int64_t K, int64_t N, int64_t R, int64_t L, int64_t x_stride, int64_t dy_stride,
                  int64_t da_stride_l, int64_t da_stride_k, int64_t da_stride_r, int64_t db_stride_l, int64_t db_stride_r,
                  int64_t db_stride_n, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const int bad = check_sizes(rows, K, N, R, L, dtype);
  if (bad) return bad;
  if (L == 0 || (!da && !db)) return GMM_OK;
  GradPlan p;
  if (!plan_grad(rows, K, N, R, L, p)) return GMM_ERR_BAD_ARGUMENT;
  if (rows && (!adapter || (da && (!u || (K && !x))) || (db && (!low || (N && !dy))))) return GMM_ERR_BAD_ARGUMENT;
  if (rows > 1 && ((da && x_stride < K) || (db && dy_stride < N))) return GMM_ERR_BAD_ARGUMENT;
  if (!workspace || !aligned16(workspace) || workspace_bytes < p.bytes) return GMM_ERR_WORKSPACE;
  char* const ws = static_cast<char*>(workspace);
  const auto ints = [&](int64_t at) { return reinterpret_cast<int32_t*>(ws + at); };
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int rc = gmm_sort_slots(adapter, rows, L + 1, ints(p.offs_at), ints(p.token_at), ints(p.rows_at), ws + p.table_at, s);
  if (rc != GMM_OK) return rc;
  GradArgs g{};
  g.row_at = ints(p.row_at); g.offs = ints(p.offs_at);
  g.places = int(p.places); g.R = int(R); g.L = int(L); g.chunk = p.chunk; g.peak_parts = p.peak_parts;
  uint32_t* const peak[2] = {reinterpret_cast<uint32_t*>(ws + p.peak_at[0]), reinterpret_cast<uint32_t*>(ws + p.peak_at[1])};
  for (int i = 0; i < 2; ++i) g.of[i].peak = peak[i];
  const float* const q1 = da ? u : nullptr;
  const float* const q2 = db ? low : nullptr;
  if (dtype == GMM_DT_F16)
    hipLaunchKernelGGL(lora_peak_kernel, dim3(unsigned(L), unsigned(p.peak_parts), 2), dim3(kThreads), 0, s, q1, q2, scale, ints(p.token_at), ints(p.offs_at),
                       int(R), int(L), peak[0], peak[1]);
  set_grad(g.of[0], x, x_stride, ws + p.q_at[0], da, reinterpret_cast<float*>(ws + p.partial_at[0]), K, R, da_stride_l, da_stride_r, da_stride_k);
  set_grad(g.of[1], dy, dy_stride, ws + p.q_at[1], db, reinterpret_cast<float*>(ws + p.partial_at[1]), N, R, db_stride_l, db_stride_r, db_stride_n);
  const auto both = [&](auto zero) {
    using T = decltype(zero);
    if (rows)
      hipLaunchKernelGGL((lora_sorted_kernel<T>), dim3(unsigned((rows + kThreads - 1) / kThreads), unsigned(R)), dim3(kThreads), 0, s, q1, q2, scale,
                         adapter, ints(p.token_at), ints(p.offs_at), int(rows), int(R), int(L), int(p.places), reinterpret_cast<T*>(ws + p.q_at[0]),
                         reinterpret_cast<T*>(ws + p.q_at[1]), ints(p.row_at), peak[0], peak[1], p.peak_parts);
    return launch_grad<T>(g, rows, s);
  };
  return dtype == GMM_DT_BF16 ? both(Bf16{}) : both(F16{});
}

}  // extern "C"
