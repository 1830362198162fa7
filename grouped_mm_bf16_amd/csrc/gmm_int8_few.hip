// Products of 8-bit integers for a few rows, a linear layer for a few tokens and the expert layer for them (gmm_int8_linear, gmm_int8_moe_few in
// include/grouped_mm_hip.h).  Reading the weights bounds them: they are streamed past the rows as the 16-bit ones are (gmm_skinny.h), 16 to 64 columns
// to a workgroup, whose waves share k (few_shape); where that leaves compute units idle, k is cut into parts as well.
//   one matrix        parts are planes of integer sums, which a second kernel adds up and scales: exact, as in one part
//   expert layer      route, rows of x to 8 bits, first product, activation to 8 bits, second product, sum over choices and parts.  The planes
//                     between its launches are scaled fp32 values; SwiGLU is computed by the first product where k is in one part
// Of a few short rows every workgroup makes the 8-bit ones itself, while its first weights are on their way (rounds_here), and the layer's routing
// (routes_here) and sums (kJoinSlots) as well: of one token two launches are left.
// Columns of 4096 values lie in the same memory channels, so workgroups that run side by side begin at different places along k (Cycle): 1 x 14336 x
// 4096 12.8 -> 11.4 us, 48 rows 18.1 -> 17.2 (16.6 since their scales are loaded ahead; 15.6 to 17.4 by the profiler), 1 x 28672 x 4096 21.3 -> 19.5.
// One layer of 24 tokens, all 8 experts of 4096 -> 2 x 14336 (1.41 GB of weights): 199 to 232 us, 6.1 to 7.1 TB/s (a copy reaches 5.1, which writes as well).
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/grouped_mm_hip.h"
#include "gmm_device.h"
#include "gmm_launch.h"
#include "gmm_route.h"
#include "gmm_skinny.h"

namespace {

using namespace gmm;

constexpr int kThreads = 256;      // of the kernels behind the products
constexpr int kMaxRows = 64;       // of a block
constexpr int kMostRows = 256;     // of one matrix; tokens of an expert layer
constexpr int kMostSlots = 1024;   // rows of many matrices

enum Result : int { kOut, kSums, kScaled, kActivated, kJoined };

// Slots up to which the last workgroup of a strip adds up its columns of the layer's result: a launch less.  1 token, 8 of 128 experts of 2048 -> 2 x
// 768 24.2 us, with a launch for the sums 25.4.
constexpr int kJoinSlots = 16;
constexpr int kLine = 32;            // words from one counter to the next
constexpr int kDeviceScope = 16;     // cache policy: stored through to memory, loaded from there

struct FewArgs {
  const void* a;
  const void* b;
  const float* a_scale;
  const float* b_scale;
  const int32_t* offs;        // null: one group
  const int32_t* row_index;   // null: rows as they are
  void* out;                  // kOut: [M][out_ld] of out_dtype; kSums: int32 [parts][M][N]; kScaled: float [parts][M][N]; kActivated: float [M][N / 2]
  int64_t a_ld, b_sg, b_ld, out_ld;      // pairs of integers (out_ld: elements)
  uint32_t a_bytes, b_bytes;
  int32_t G, M, N, K, a_rows; // K: pairs
  int32_t most, block, items; // rows that a group can have; rows of a block, a multiple of 16; blocks of one group's rows that there can be
  int32_t columns, tiles, parts, k_part;      // of a strip (with its partners); strips; parts along k and their length
  int32_t result, out_dtype;
  int32_t x_dtype;            // of rows that are rounded here: a is x, a_ld its elements from one row to the next
  // kJoined: out float [M][N], and behind it the layer's result from its slots' rows and weights.  The product in front has cleared the counters.
  void* sum;                  // [tokens][sum_ld] of out_dtype
  const int32_t* token_rows;
  const float* slot_weight;
  uint32_t* arrived;          // of each strip, kLine words apart: workgroups that are done with it
  int64_t sum_ld;
  int32_t tokens, top_k;
  int32_t clear;              // counters that this launch clears
  RouteHere route;            // where the workgroups route for themselves
};

constexpr int kNotRounded = -1;

// The `which`-th block of up to BLOCK rows of a group, found by every wave for itself.  A row is its that first has a higher offset: where offsets go down
// as well as up the highest so far takes their place, so groups share no rows and have no more blocks than the launch.
template <int BLOCK>
__device__ __forceinline__ bool find_group(const FewArgs& a, int which, int& g, int& row0, int& rows) {
  constexpr int AT_ONCE = 4;
  const int lane = threadIdx.x & 63;
  int used = 0, start = 0;
  for (int base = 0; base < a.G; base += 64 * AT_ONCE) {
    int ends[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) ends[i] = a.offs[min(base + 64 * i + lane, a.G - 1)];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const bool there = base + 64 * i + lane < a.G;
      int to = min(max(ends[i], 0), a.M), before = __shfl_up(to, 1), from = lane ? before : start;
      if (__ballot(to < from)) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int up = __shfl_up(to, o);
          to = max(to, lane >= o ? up : start);
        }
        before = __shfl_up(to, 1);
        from = lane ? before : start;
      }
      start = __builtin_amdgcn_readlane(to, 63);
      const uint64_t with = __ballot(there && to > from);
      int ahead = __popcll(with & ((uint64_t(1) << lane) - 1)), n = __popcll(with), own = there && to > from;      // blocks of lanes before the own
      if (a.most > BLOCK) {      // a group may have several
        own = own ? (to - from + BLOCK - 1) / BLOCK : 0;
        ahead = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int up = __shfl_up(ahead, o);
          ahead += lane >= o ? up : 0;
        }
        n = __builtin_amdgcn_readlane(ahead, 63);
        ahead -= own;
      }
      if (which < used + n) {
        const uint64_t it = __ballot(ahead <= which - used && which - used < ahead + own);
        const int at = __ffsll(static_cast<unsigned long long>(it)) - 1;
        g = base + 64 * i + at;
        const int skip = (which - used - __builtin_amdgcn_readlane(ahead, at)) * BLOCK;
        row0 = __builtin_amdgcn_readlane(from, at) + skip;
        rows = min(__builtin_amdgcn_readlane(to, at) - row0, BLOCK);
        return true;
      }
      used += n;
    }
  }
  return false;
}

__device__ __forceinline__ void put(void* out, int dtype, int64_t at, float v) {
  if (dtype == GMM_DT_BF16) static_cast<Bf16*>(out)[at] = rounded<Bf16>(v);
  else if (dtype == GMM_DT_F16) static_cast<F16*>(out)[at] = rounded<F16>(v);
  else static_cast<float*>(out)[at] = v;
}

// A sum in fp32, by its column's scale, then by its row's: no product fused with the rounding to 16 bits that follows.
__device__ __forceinline__ float scaled(int sum, float column, float row) {
  float v = float(sum) * column * row;
  asm volatile("" : "+v"(v));
  return v;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t joined(const FewArgs& a) { return buffer(a.out, uint32_t(a.M) * uint32_t(a.N) * 4); }

// The last workgroup of a strip adds up what all of them left, in the order of the choices whichever it is.  Nobody waits for anybody.  Choices
// that are not there take part as zeros: asked for each, the compiler makes every load wait for the one before it.
template <int OUT, int THREADS>
__device__ __forceinline__ void join(const FewArgs& a, int tile) {
  __shared__ int last, rows[kJoinSlots];
  __shared__ float weights[kJoinSlots];
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(&a.arrived[tile * kLine], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == uint32_t(a.items) - 1;
  if (int(threadIdx.x) < a.M) {
    rows[threadIdx.x] = a.token_rows[threadIdx.x];
    weights[threadIdx.x] = a.slot_weight[threadIdx.x];
  }
  __syncthreads();
  if (!last) return;
  const __amdgpu_buffer_rsrc_t y = joined(a);
  for (int u = threadIdx.x; u < a.tokens * OUT; u += THREADS) {
    const int t = u / OUT, col = tile * OUT + u % OUT;
    if (col >= a.N) continue;
    float sum = 0;
    for (int j = 0; j < a.top_k; j += 8) {
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = rows[t * a.top_k + min(j + i, a.top_k - 1)];
        v[i] = __builtin_amdgcn_raw_buffer_load_b32(y, int((uint32_t(row) * a.N + col) * 4), 0, kDeviceScope);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t there = j + i < a.top_k ? ~0u : 0u;
        const float w = __uint_as_float(__float_as_uint(weights[t * a.top_k + min(j + i, a.top_k - 1)]) & there);
        sum += w * __uint_as_float(v[i] & there);
      }
    }
    put(a.sum, a.out_dtype, t * a.sum_ld + col, sum);
  }
}

// Eight values of x to an access, so many accesses to a thread, as many elements of all rows as leave LDS for other workgroups.
template <typename X> constexpr int kAccesses = sizeof(X) == 2 ? 8 : 4;
constexpr int64_t kMostRounded = 16384;

// Rows of x that a workgroup rounds for itself, as gmm_int8_quantize does.
template <typename X, int WAVES>
struct RowsHere {
  static constexpr int THREADS = 64 * WAVES, N = kAccesses<X>;
  Pack<X, kVector<X>> v[N][8 / kVector<X>];

  // f(access, row, column of the first of eight elements, how many of them are the one before's) for the thread's accesses.
  template <typename F>
  static __device__ __forceinline__ void each(int rows, int K, F&& f) {
    const int per_row = (K + 7) / 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int at = int(threadIdx.x) + i * THREADS, r = at / per_row;
      if (r >= rows) break;
      const Chunk<8, true> c((at - r * per_row) * 8, K);
      f(i, r, c.at, c.skip);
    }
  }

  // row(r): where row r of x is, null: zeros.
  template <typename R>
  __device__ __forceinline__ void load(int rows, int K, R&& row) {
    each(rows, K, [&](int i, int r, int c, int) {
      const X* from = row(r);
#pragma unroll
      for (int q = 0; q < 8 / kVector<X>; ++q)
        if (from) v[i][q] = unaligned<Pack<X, kVector<X>>>(from + c + q * kVector<X>);
    });
  }

  // Into LDS, row r from to + r * pitch on, and the scales.  All threads; ends with a barrier.  most[]: zeros, behind a barrier.
  template <typename R>
  __device__ __forceinline__ void round(int rows, int K, R&& row, char* to, int pitch, uint32_t* most, float* scale) {
    const int lane = threadIdx.x & 63;
    each(rows, K, [&](int i, int r, int, int) {
      uint32_t m = 0;
#pragma unroll
      for (int q = 0; q < 8; ++q) m = max(m, __float_as_uint(v[i][q / kVector<X>].get(q % kVector<X>)) & 0x7fffffffu);
      if (!row(r)) m = 0;
      // one row in all of the wave's lanes: they have one maximum
      if (__all(r == __builtin_amdgcn_readfirstlane(r)) && __popcll(__ballot(1)) == 64) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, uint32_t(__shfl_xor(int(m), o)));
        if (lane == 0) atomicMax(&most[r], m);
      } else {
        atomicMax(&most[r], m);
      }
    });
    __syncthreads();
    each(rows, K, [&](int i, int r, int c, int skip) {
      const uint32_t bits = most[r];
      const RowScale s(bits);
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int q = 0; q < 8; ++q) w[q / 4] |= s.rounded_bits(v[i][q / kVector<X>].get(q % kVector<X>)) << q % 4 * 8;
      if (!s.finite || !row(r)) w[0] = w[1] = 0;
      if (skip == 0) *reinterpret_cast<uint2*>(to + r * pitch + c) = make_uint2(w[0], w[1]);
      else
#pragma unroll
        for (int q = 1; q < 8; ++q) if (q >= skip) to[r * pitch + c + q] = char(w[q / 4] >> q % 4 * 8);
    });
    if (int(threadIdx.x) < rows) scale[threadIdx.x] = row(threadIdx.x) ? RowScale(most[threadIdx.x]).scale : 0.0f;
    __syncthreads();
  }
};

// LDS of a workgroup: the waves' own parts while they multiply, then the sums.
template <typename S, int MF, int WAVES>
union FewShared {
  char wave[WAVES][S::LDS_BYTES > 0 ? S::LDS_BYTES : 16];
  SkinnySums<WAVES, S::FR> sums[MF];
  __device__ FewShared() {}
};

// FR: a strip is 16 FR columns.  GLU: half of them gate columns, the others their partners, N / 2 further on; the result is silu(gate) * partner.
// X: the rows are values of this type, rounded here (up to 16 of them, k in one part); void: 8-bit integers.
// ROUTE: every workgroup routes for itself (GLU and X alone).
template <typename X, int MF, int FR, int WAVES, bool GLU, bool ROUTE>
__global__ void __launch_bounds__(64 * WAVES, WAVES >= 8 || MF == 4 ? 1 : 2) int8_few_kernel(const FewArgs a) {
  constexpr bool HERE = !std::is_void_v<X>;
  static_assert(!HERE || MF == 1, "");
  using S = Skinny<I8x2, GMM_W_COLS, FR, MF, 1, HERE ? GMM_A_RESIDENT : GMM_A_STAGED, 2>;
  constexpr int OUT = GLU ? 8 * FR : 16 * FR, THREADS = 64 * WAVES;
  __shared__ FewShared<S, MF, WAVES> shared;
  __shared__ float column_scales[16 * FR], row_scales[16 * MF];
  extern __shared__ __align__(16) char rows_here[];      // HERE: 8-bit rows
  __shared__ uint32_t most_here[16];
  if constexpr (HERE) {
    if (threadIdx.x < 16) most_here[threadIdx.x] = 0;
    __syncthreads();
  }
  if (GLU && blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.clear; i += THREADS) a.arrived[i * kLine] = 0;
  const int part = blockIdx.x % a.parts, item = blockIdx.x / a.parts, tile = item % a.tiles;
  int g = 0, row0 = a.offs ? 0 : item / a.tiles * 16 * MF, rows = min(a.M - row0, 16 * MF);
  const int32_t* row_index = a.row_index;      // of the group's rows
  if constexpr (ROUTE) {
    __shared__ FewRouting routing;
    if (!route_here<WAVES>(a.route, routing, item / a.tiles, g, row0, rows)) return;
    row_index = routing.token;
  } else if (a.offs && !find_group<16 * MF>(a, item / a.tiles, g, row0, rows)) {
    if constexpr (!GLU && MF == 1) if (a.result == kJoined) join<OUT, THREADS>(a, tile);      // it is counted as well
    return;
  }
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int width = GLU ? a.N / 2 : a.N, first = tile * OUT;
  S s;
  s.lane = lane;
  s.lds = shared.wave[wave];
  s.w_buf = buffer(static_cast<const uint16_t*>(a.b) + g * a.b_sg, a.b_bytes);
  s.a_plane = 0;
  s.turn = (g * a.tiles + tile) * a.parts / 8;      // the same for all blocks of rows
  if constexpr (GLU) s.set_columns(first, width - first, 1, uint32_t(a.b_ld), OUT, width + first);
  else s.set_columns(first, width - first, 1, uint32_t(a.b_ld));
  const float* const columns = a.b_scale + int64_t(g) * a.N;
  const auto source = [&](int r) {      // row of a, or -1
    const int at = ROUTE ? row_index[r] : row_index ? row_index[row0 + r] : row0 + r;
    return uint32_t(at) < uint32_t(a.a_rows) ? at : -1;
  };
  // the scales are on their way during the product: asked for behind it they took a trip to memory each, one behind the other
  const int mine = threadIdx.x;
  float column_scale = 0, row_scale = 0;
  if (mine < 16 * FR && first + mine % OUT < width) column_scale = columns[mine / OUT * width + first + mine % OUT];
  if constexpr (!HERE) {
    if (mine < rows) {
      const int from = source(mine);
      if (from >= 0) row_scale = a.a_scale[from];
    }
  }
  f32x4 acc[MF][FR];
  clear(acc);
  if constexpr (HERE) {
    const auto row = [&](int r) {
      const int at = source(r);
      return at < 0 ? static_cast<const X*>(nullptr) : static_cast<const X*>(a.a) + at * a.a_ld;
    };
    RowsHere<X, WAVES> x;
    typename S::Step step[S::STEPS];
    s.pitch = (a.K * 2 + 31) & ~15;      // rows in other banks
    s.resident = rows_here;
    s.resident_k = 0;
    s.resident_rows = rows;
    x.load(rows, 2 * a.K, row);
    typename S::template Cycle<1, WAVES> cycle(wave * S::KS, a.K, s.turn);
    cycle.prime(s, step);
    x.round(rows, 2 * a.K, row, rows_here, s.pitch, most_here, row_scales);
    cycle.primed(s, step, acc);
  } else {
    s.a_buf = buffer(a.a, a.a_bytes);
    s.set_rows([&](int r) {
      const int at = r < rows ? source(r) : -1;
      return at < 0 ? kNowhere : uint32_t(at) * uint32_t(a.a_ld) * 2;
    });
    s.template run<WAVES>(rows, part * a.k_part, min(a.K, (part + 1) * a.k_part), wave, acc);
  }
  __syncthreads();
#pragma unroll
  for (int m = 0; m < MF; ++m) shared.sums[m].put(wave, lane, acc[m]);
  if (mine < 16 * FR) column_scales[mine] = column_scale;
  if (!HERE && mine < 16 * MF) row_scales[mine] = row_scale;
  __syncthreads();
  const int blocks = (rows + 15) / 16;
  for (int u = threadIdx.x; u < OUT * 4 * blocks; u += THREADS) {
    const int oc = u % OUT, og = u / OUT % 4, m = u / OUT / 4, col = first + oc;
    if (col >= width) continue;
    const auto sums = [&](int c) { return shared.sums[m].whole(S::product_of(c), S::lane_of(c), og); };
    const i32x4 h = sums(oc), partner = GLU ? sums(OUT + oc) : i32x4{0, 0, 0, 0};
    const float cs = column_scales[oc], ps = GLU ? column_scales[OUT + oc] : 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = 16 * m + 4 * og + v;
      if (r >= rows) break;
      const int64_t row = row0 + r;
      if (a.result == kSums) {
        static_cast<int32_t*>(a.out)[(int64_t(part) * a.M + row) * a.N + col] = h[v];
        continue;
      }
      const float rs = row_scales[r], f = scaled(h[v], cs, rs);
      if constexpr (GLU) {
        static_cast<float*>(a.out)[row * width + col] = f / (1.0f + __expf(-f)) * scaled(partner[v], ps, rs);
      } else if (a.result == kJoined) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(f), joined(a), int((uint32_t(row) * a.N + col) * 4), 0, kDeviceScope);
      } else if (a.result == kScaled) {
        static_cast<float*>(a.out)[(int64_t(part) * a.M + row) * a.N + col] = f;
      } else {
        put(a.out, a.out_dtype, row * a.out_ld + col, f);
      }
    }
  }
  if constexpr (!GLU && MF == 1) if (a.result == kJoined) join<OUT, THREADS>(a, tile);
}

// Planes of integer sums added up and scaled.
__global__ void __launch_bounds__(kThreads) int8_finish_kernel(const FewArgs a, const int32_t* __restrict__ planes) {
  const int col = blockIdx.x * kThreads + threadIdx.x, row = blockIdx.y;
  if (col >= a.N) return;
  const int32_t* at = planes + int64_t(row) * a.N + col;
  int sum = 0;
  in_fours(a.parts, [&](int p, bool in) {
    const int v = at[int64_t(p) * a.M * a.N];
    sum += in ? v : 0;
  });
  put(a.out, a.out_dtype, row * a.out_ld + col, scaled(sum, a.b_scale[col], a.a_scale[row]));
}

// out[t] = sum over j of weight * sum over the parts of y, in that order.
template <typename T>
__global__ void __launch_bounds__(kThreads) int8_combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ token_rows,
                                                                const float* __restrict__ slot_weight, T* __restrict__ out, int top_k, int parts,
                                                                int slots, int H, int64_t out_ld) {
  const int t = blockIdx.y, c = blockIdx.x * kThreads + threadIdx.x, lane = threadIdx.x & 63;
  const int mine = t * top_k + min(lane, top_k - 1);
  const int row = token_rows[mine], weight = __builtin_bit_cast(int, slot_weight[mine]);      // of choice j: in lane j
  const float* const from = y + min(c, H - 1);
  float sum = 0, v = 0;
  int j = 0, part = 0;
  in_fours(top_k * parts, [&](int, bool in) {
    const float one = from[(int64_t(part) * slots + __builtin_amdgcn_readlane(row, j)) * H];
    const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(weight, j));
    v = in ? (part ? v : 0.0f) + one : v;
    const bool last = part == parts - 1;
    if (in && last) sum += w * v;
    part = last ? 0 : part + 1;
    j = min(j + last, top_k - 1);
  });
  if (c < H) out[t * out_ld + c] = rounded<T>(sum);
}

// ---------------------------------------------------------------- host side
// How a product of up to `rows` rows of a group is laid out.  Measured alone, us, for rows x N x K of one matrix, weights from memory (8-bit rows unless
// said otherwise):
//   64 columns, 4 waves    where such strips fill half the compute units and more: 1 x 14336 x 4096 11.6 (32 columns 12.2), 1 x 9216 x 2048 6.4 (7.8),
//                          48 x 14336 x 4096 16.6 (21.3; 64 in two parts 23.2), 48 x 9216 x 2048 11.2 (14.9); but 1 x 8192 x 8192 14.4 (14.4), 1 x 7168 x
//                          7168 13.5 (11.1), 48 x 8192 x 8192 23.1 (18.8)
//   16 columns, 16 waves   up to 16 rows, one round of long strips: 1 x 4096 x 14336 12.7 (32 columns 14.7, in two parts 13.8), 1 x 1024 x 8192 7.0 (8.5),
//                          1 x 4096 x 4096 6.4 (6.4); but 1 x 4608 x 4608, more than a round, 10.5 (7.0), 1 x 2048 x 2048 5.3 (4.6)
//   32 columns, 8 waves    what is left; of more rows and long columns in as many parts of k as fill the compute units: 48 x 4096 x 8192 14.0 in two
//                          parts, 16.5 in one, 48 x 2048 x 8192 11.3 in four; 64 x 1024 x 4096 10.3, 11.5 in one; but 48
//                          x 4096 x 4096 11.4 and 10.7, 48 x 1536 x 2048 8.4 in four and 7.8
//   64 columns in parts    the longest, where four or more parts fill the compute units: 48 x 4096 x 28672 27.7 (32 columns in two parts 30.3), x 14336
//                          19.3 (20.1), x 11008 17.1 (17.2); but 32 x 6144 x 16384 25.3 (32 columns 23.5), 64 x 2048 x 14336 16.3 in eight (15.7 in four)
// Rows that every workgroup rounds for itself are rounded by more threads where it has more waves: 1 x 14336 x 4096 11.9 with 32 columns (64 14.4), 4 rows
// 16.3 (19.8), 1 x 6144 x 4096 8.6 (16 columns 10.5), 1 x 2048 x 2048 5.3 with 16 (32 5.7); but 1 x 28672 x 2048 15.5 with 32 (64 12.2).
struct Shape { int32_t columns, parts, k_part; };

constexpr int64_t kStep = 64;      // k of a wave's step

Shape few_shape(int64_t used, int64_t rows, int64_t N, int64_t K) {
  const int64_t cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  const auto strips = [&](int64_t columns) { return used * ((N + columns - 1) / columns); };
  Shape s{64, 1, int32_t(round_up(K, kStep))};
  if (16 * strips(64) >= 9 * cus) return s;
  s.columns = rows <= 16 && K >= 2048 && strips(16) <= cus ? 16 : 32;
  if (rows <= 16 || K <= 1024 || (K <= 2048 && 4 * strips(32) > cus)) return s;
  if (K >= 6144 && 8 * strips(64) > cus && 4 * strips(64) <= cus) s.columns = 64;
  int64_t want = strips(s.columns) > 0 ? cus / strips(s.columns) : 1;
  if (want > K / (8 * kStep)) want = K / (8 * kStep);      // a step for each wave
  if (want <= 1) return s;
  s.k_part = int32_t(round_up((K + want - 1) / want, kStep));
  s.parts = int32_t((K + s.k_part - 1) / s.k_part);
  return s;
}

// Are the rows rounded by every workgroup for itself?  1 x 4096 x 4096 with its rounding 6.0 us, in a launch of its own 2.3 and 5.4.
bool rounds_here(int64_t rows, int64_t K, const Shape& s, int32_t x_dtype) {
  const int64_t threads = s.columns == 64 ? 256 : s.columns == 32 ? 512 : 1024, each = x_dtype == GMM_DT_F32 ? kAccesses<float> : kAccesses<Bf16>;
  return rows <= 16 && s.parts == 1 && rows * K <= kMostRounded && rows * ((K + 7) / 8) <= threads * each;
}

// The same of rows of x_dtype that may be rounded here.
Shape few_shape(int64_t used, int64_t rows, int64_t N, int64_t K, int32_t x_dtype) {
  const int64_t cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  const auto strips = [&](int64_t columns) { return used * ((N + columns - 1) / columns); };
  const Shape s = few_shape(used, rows, N, K);
  Shape h{64, 1, int32_t(round_up(K, kStep))};
  if (K >= 1024 && strips(16) <= cus) h.columns = 16;
  else if (K >= 2048 && strips(32) <= 2 * cus) h.columns = 32;      // all of them at once
  else h.columns = s.columns;
  return rounds_here(rows, 2 * K, h, x_dtype) ? h : s;
}

void set_shape(FewArgs& a, const Shape& s, bool glu = false) {
  a.columns = s.columns;
  a.parts = s.parts;
  a.k_part = s.k_part;
  a.tiles = glu ? gmm_cdiv(a.N / 2, s.columns / 2) : gmm_cdiv(a.N, s.columns);
}

// Rows of a block for `slots` rows over `used` groups, which have about as many as each other: one and a half times that, and what a group has more is
// another block.  us by rows of a block (and through tiles), expert layers: 64 tokens, 8 of 128 experts of 2048 -> 2 x 768, 4 rows 16: 121, 32: 123, 64: 186
// (144), 192 tokens, 12 rows 144, 138, 220 (150); 2 of 8 of 4096 -> 2 x 14336, 96 tokens, 24 rows 32: 257, 48: 264 (335), 128, 32 rows 347, 283 (343),
// 192, 48 rows 490, 394 (352); 6 of 64 of 2048 -> 2 x 1408, 256 tokens, 24 rows 140, 151 (139).
bool few_each(int64_t slots, int64_t used) { return slots <= 32 * used; }
int64_t block_of(int64_t slots, int64_t used, int64_t most) {
  const int64_t block = slots <= 24 * used ? 32 : few_each(slots, used) ? 48 : kMaxRows, all = round_up(most, 16);
  return block < all ? block : all;
}
int64_t items_of(int64_t slots, int64_t used, int64_t most, int64_t block) { return most <= block ? used : used + slots / block; }

FewArgs from_params(const GmmInt8Params& p) {
  FewArgs a{};
  a.a = p.a; a.b = p.b; a.a_scale = p.a_scale; a.b_scale = p.b_scale; a.offs = p.jag == GMM_JAG_M ? p.offs : nullptr; a.row_index = p.gather;
  a.out = p.c; a.a_ld = p.a_sm; a.b_sg = p.b_sg; a.b_ld = p.b_sn; a.out_ld = p.c_sm;
  a.G = p.G; a.M = p.M; a.N = p.N; a.K = p.K; a.a_rows = p.gather ? p.a_rows : p.M;
  a.x_dtype = kNotRounded;
  a.most = p.M;
  if (a.offs) {
    const int used = gmm_min(p.G, p.M);
    a.block = int32_t(p.M <= kMaxRows ? round_up(p.M, 16) : block_of(p.M, used, p.M));
    a.items = int32_t(items_of(p.M, used, p.M, a.block));
    set_shape(a, few_shape(used, gmm_min(a.most, a.block), a.N, a.K));
  } else {      // one matrix: blocks of the same length
    a.items = (p.M + kMaxRows - 1) / kMaxRows;
    a.block = int32_t(round_up(a.items ? (p.M + a.items - 1) / a.items : 0, 16));
    set_shape(a, few_shape(a.items, gmm_min(a.most, a.block), a.N, a.K));
  }
  return a;
}

bool sizes_fit(FewArgs& a) {
  if (a.a_rows > 0 && int64_t(a.a_rows) * a.a_ld >= (int64_t(1) << 30)) return false;
  a.a_bytes = uint32_t(gmm_rows_bytes(a.a_rows, a.a_ld, a.K));      // a row that does not exist is asked for behind it
  a.b_bytes = matrix_bytes(a.K, a.N, 1, a.b_ld);
  return a.K >= 8 && a.b_bytes != 0;
}

// Do the workgroups of this product route for themselves?  In one round of them, in which that is as long in all as in one.  1 token, 8 of 128 experts
// of 2048 -> 2 x 768 19.6 us, with a launch for the routing 22.5.
bool routes_here(int64_t used, int64_t tiles, int64_t slots, int64_t experts) {
  const int64_t cus = gmm_num_cus() > 0 ? gmm_num_cus() : 256;
  return used * tiles <= 4 * cus && slots <= kRouteSlots && experts <= kRouteExperts;
}

template <typename X, bool GLU, bool ROUTE = false>
int launch_rows(const FewArgs& a, hipStream_t stream) {
  constexpr bool HERE = !std::is_void_v<X>;
  const dim3 grid(unsigned(int64_t(a.items) * a.tiles * a.parts));
  const int lds = HERE ? a.most * ((a.K * 2 + 31) & ~15) : 0;
  const auto go = [&](auto mf, auto fr, auto waves) {
    constexpr int MF = decltype(mf)::value, FR = decltype(fr)::value, WAVES = decltype(waves)::value;
    hipLaunchKernelGGL((int8_few_kernel<X, MF, FR, WAVES, GLU, ROUTE>), grid, dim3(64 * WAVES), lds, stream, a);
  };
  const auto by_rows = [&](auto fr, auto waves) {
    if constexpr (!HERE) {
      if (a.block > 48) return go(std::integral_constant<int, 4>{}, fr, waves);
      if (a.block > 32) return go(std::integral_constant<int, 3>{}, fr, waves);
      if (a.block > 16) return go(std::integral_constant<int, 2>{}, fr, waves);
    }
    go(std::integral_constant<int, 1>{}, fr, waves);
  };
  if (a.columns == 64) by_rows(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{});
  else if (a.columns == 32) by_rows(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
  else go(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 16>{});
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

template <bool GLU>
int launch(const FewArgs& a, hipStream_t stream) {
  if constexpr (GLU) {
    if (a.route.logits) return a.x_dtype == GMM_DT_BF16 ? launch_rows<Bf16, true, true>(a, stream) : launch_rows<F16, true, true>(a, stream);
  }
  if (a.x_dtype == GMM_DT_BF16) return launch_rows<Bf16, GLU>(a, stream);
  if (a.x_dtype == GMM_DT_F16) return launch_rows<F16, GLU>(a, stream);
  if constexpr (!GLU) {
    if (a.x_dtype == GMM_DT_F32) return launch_rows<float, GLU>(a, stream);
  }
  return launch_rows<void, GLU>(a, stream);
}

}  // namespace

bool gmm_int8_few_preferred(const GmmInt8Params& p) {
  FewArgs a = from_params(p);
  if (p.k_odd || !sizes_fit(a) || int64_t(a.items) * a.tiles >= (int64_t(1) << 27)) return false;
  if (p.M <= kMaxRows) return true;
  // us, tile / here, by all groups' rows: 128 groups of 2048 -> 1536 65 40.8 / 27.2, 256 67.1 / 53.5, 1024 73.5 / 65.8, 2048 73.5 / 72.4; 64 of 2048 -> 2816
  // 256 69.3 / 56.5, 2048 70.6 / 85.1; 8 of 14336 -> 4096 65 108 / 76, 256 (32 each) 108 / 82; 32 of 1024 -> 1024 1024 (32 each) 16.4 / 14.5
  if (a.offs) return p.M <= kMostSlots && few_each(p.M, gmm_min(p.G, p.M));
  // Blocks of rows read the weights again, from the caches at best, where the tile has fewer tiles than compute units.  us, tile / here: 65 x 4096 x 4096
  // 31.6 / 10.6, 256 34.1 / 17.4; 96 x 14336 x 4096 34.5 / 27.3, 128 35.6 / 36.2; 256 x 4096 x 14336 74.3 / 40.2; 160 x 6144 x 1024 15.1 / 14.3, 192 15.3
  // / 20.1; 96 x 9216 x 2048 21.3 / 15.9, 128 21.8 / 24.8; 65 x 28672 x 4096 41.6 / 45.8.
  const int64_t work = int64_t((p.N + 63) / 64) * ((p.M + 15) / 16);
  return p.M <= kMostRows && (work <= 1024 || (work <= 1536 && p.K >= 2048));
}

int64_t gmm_int8_few_bytes(const GmmInt8Params& p) {
  const FewArgs a = from_params(p);
  return !a.offs && a.parts > 1 ? int64_t(a.parts) * a.M * a.N * 4 : 0;
}

int gmm_launch_int8_few(const GmmInt8Params& p, void* planes, int64_t planes_bytes, int out_dtype, hipStream_t stream) {
  FewArgs a = from_params(p);
  if (!sizes_fit(a)) return GMM_ERR_UNSUPPORTED;
  a.out_dtype = out_dtype;
  a.result = kOut;
  if (a.offs || !planes || planes_bytes < gmm_int8_few_bytes(p)) {      // the planes do not say whose scales their rows take
    if (a.parts > 1) set_shape(a, Shape{32, 1, int32_t(round_up(a.K, kStep))});
  }
  if (a.parts == 1) return launch<false>(a, stream);
  FewArgs u = a;
  u.out = planes;
  u.result = kSums;
  const int rc = launch<false>(u, stream);
  if (rc != GMM_OK) return rc;
  hipLaunchKernelGGL(int8_finish_kernel, dim3(unsigned(gmm_cdiv(a.N, kThreads)), unsigned(a.M)), dim3(kThreads), 0, stream, a,
                     static_cast<const int32_t*>(planes));
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

namespace {

// ---------------------------------------------------------------- linear layer
struct LinearPlan { int64_t pitch, scale_at, planes_at, bytes; Shape shape; bool here; };

bool plan_linear(int64_t T, int64_t K, int64_t N, int32_t dtype, LinearPlan& p) {
  if (T < 0 || T > kMaxRows || K < 0 || K >= 131072 || N < 0 || N >= (int64_t(1) << 31)) return false;
  p.shape = few_shape(1, T, N, K / 2, dtype);
  const int64_t parts = p.shape.parts;
  p.here = rounds_here(T, K, p.shape, dtype);
  p.pitch = round_up(K > 0 ? K : 1, 16);
  p.scale_at = T * p.pitch;
  p.planes_at = round_up(p.scale_at + 4 * T, 16);
  p.bytes = p.here ? 0 : p.planes_at + (parts > 1 ? parts * T * N * 4 : 0);
  return true;
}

// ---------------------------------------------------------------- expert layer
struct LayerPlan {
  int64_t slots, used, block, items, x_pitch, act_pitch, table_bytes;
  int64_t table_at, arrived_at, x_at, x_scale_at, h_at, act_at, act_scale_at, y_at, bytes;
  Shape up, down;
  bool activated;      // by the first product
  bool x_here, act_here;      // rows that the products round themselves
  bool join;                  // the second product's workgroups add up the result
};

bool plan_layer(int64_t T, int64_t E, int64_t k, int64_t H, int64_t I, int64_t kind, LayerPlan& p) {
  if (T < 0 || T > kMostRows || E < 1 || H < 1 || I < 1 || H >= 131072 || I >= 131072 || k < 1) return false;
  p.table_bytes = gmm_moe_route_workspace_bytes(T, E, k);
  if (p.table_bytes < 0 || k > 32 || k > E) return false;
  const int64_t N = kind == GMM_ACT_SWIGLU ? 2 * I : I;
  p.slots = T * k;
  p.used = p.slots < E ? p.slots : E;
  if (T > kMaxRows && !few_each(p.slots, p.used)) return false;
  p.block = block_of(p.slots, p.used, T);
  p.items = items_of(p.slots, p.used, T, p.block);
  p.up = few_shape(p.used, T, N, H / 2, GMM_DT_BF16);
  p.activated = p.up.parts == 1 && kind == GMM_ACT_SWIGLU;
  p.down = p.activated ? few_shape(p.used, T, H, I / 2, GMM_DT_F32) : few_shape(p.used, T, H, I / 2);
  p.x_here = rounds_here(T, H, p.up, GMM_DT_BF16);
  p.act_here = p.activated && rounds_here(T, I, p.down, GMM_DT_F32);
  p.join = p.activated && p.slots <= kJoinSlots && p.down.parts == 1;
  p.x_pitch = round_up(H, 16);
  p.act_pitch = round_up(I, 16);
  int64_t at = 0;
  const auto take = [&](int64_t bytes) { const int64_t from = at; at = round_up(at + bytes, 256); return from; };
  take((E + 4 * p.slots) * 4);
  p.table_at = take(p.table_bytes);
  p.arrived_at = take(p.join ? (H + p.down.columns - 1) / p.down.columns * kLine * 4 : 0);
  p.x_at = take(T * p.x_pitch);
  p.x_scale_at = take(4 * T);
  p.h_at = take((p.activated ? I : p.up.parts * N) * p.slots * 4);
  p.act_at = take(p.slots * p.act_pitch);
  p.act_scale_at = take(4 * p.slots);
  p.y_at = take(p.down.parts * p.slots * H * 4);
  p.bytes = at;
  return true;
}

bool lies(const void* p, int64_t stride, int64_t width, int64_t count) {
  return aligned16(p) && (stride & 15) == 0 && stride >= 0 && (stride >= width || count <= 1) && stride < (int64_t(1) << 23);
}

}  // namespace

extern "C" {

int64_t gmm_int8_linear_workspace_bytes(int64_t rows, int64_t K, int64_t N, int32_t dtype) {
  LinearPlan p;
  return plan_linear(rows, K, N, dtype, p) ? p.bytes : -1;
}

int gmm_int8_linear(const void* x, const int8_t* b, const float* b_scale, void* out, int64_t rows, int64_t K, int64_t N, int64_t x_stride,
                    int64_t b_stride_n, int64_t out_stride, int32_t dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  LinearPlan plan;
  if (rows < 0 || K < 0 || N < 0) return GMM_ERR_BAD_ARGUMENT;
  if (dtype < GMM_DT_BF16 || dtype > GMM_DT_F32 || !plan_linear(rows, K, N, dtype, plan) || (K & 1) || K < 16) return GMM_ERR_UNSUPPORTED;
  if (rows == 0 || N == 0) return GMM_OK;
  if (!x || !b || !b_scale || !out || (rows > 1 && (x_stride < K || out_stride < N)) || !lies(b, b_stride_n, K, N)) return GMM_ERR_BAD_ARGUMENT;
  if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || !aligned16(workspace))) return GMM_ERR_WORKSPACE;
  char* const ws = static_cast<char*>(workspace);
  GmmInt8Params p{};
  p.a = ws; p.b = b; p.c = out; p.G = 1; p.jag = GMM_JAG_NONE; p.M = int32_t(rows); p.N = int32_t(N); p.K = int32_t(K / 2);
  p.a_sm = plan.pitch / 2; p.a_sk = 1; p.b_sk = 1; p.b_sn = b_stride_n / 2; p.c_sm = out_stride; p.c_sn = 1; p.a_rows = int32_t(rows);
  p.a_scale = reinterpret_cast<float*>(ws + plan.scale_at);
  p.b_scale = b_scale;
  if (!gmm_int8_few_preferred(p)) return GMM_ERR_UNSUPPORTED;
  if (plan.here) {
    FewArgs f = from_params(p);
    f.a = x; f.a_ld = rows > 1 ? x_stride : K; f.x_dtype = dtype; f.out_dtype = dtype; f.result = kOut;
    set_shape(f, plan.shape);
    return sizes_fit(f) ? launch<false>(f, static_cast<hipStream_t>(stream)) : GMM_ERR_UNSUPPORTED;
  }
  const int rc = gmm_int8_quantize(x, reinterpret_cast<int8_t*>(ws), reinterpret_cast<float*>(ws + plan.scale_at), rows, K, x_stride, plan.pitch,
                                   dtype, stream);
  return rc == GMM_OK ? gmm_launch_int8_few(p, ws + plan.planes_at, plan.bytes - plan.planes_at, dtype, static_cast<hipStream_t>(stream)) : rc;
}

int64_t gmm_int8_moe_few_workspace_bytes(int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t inner, int32_t kind) {
  LayerPlan p;
  return plan_layer(tokens, experts, top_k, hidden, inner, kind, p) ? p.bytes : -1;
}

int gmm_int8_moe_few(const void* x, const void* logits, const int8_t* w_up, const float* up_scale, const int8_t* w_down, const float* down_scale,
                     void* out, int64_t tokens, int64_t experts, int64_t top_k, int64_t hidden, int64_t inner, int64_t x_stride, int64_t logits_stride,
                     int64_t up_stride_g, int64_t up_stride_n, int64_t down_stride_g, int64_t down_stride_n, int64_t out_stride, int32_t kind,
                     int32_t renormalize, int32_t dtype, int32_t logits_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  LayerPlan p;
  if (kind < GMM_ACT_SILU || kind > GMM_ACT_SWIGLU || tokens < 0 || experts < 1 || top_k < 1 || top_k > experts) return GMM_ERR_BAD_ARGUMENT;
  if ((dtype != GMM_DT_BF16 && dtype != GMM_DT_F16) || logits_dtype < GMM_DT_BF16 || logits_dtype > GMM_DT_F32) return GMM_ERR_UNSUPPORTED;
  if (!plan_layer(tokens, experts, top_k, hidden, inner, kind, p) || (hidden & 1) || (inner & 1) || hidden < 16 || inner < 16) return GMM_ERR_UNSUPPORTED;
  if (tokens == 0) return GMM_OK;
  const int64_t N = kind == GMM_ACT_SWIGLU ? 2 * inner : inner;
  if (!x || !logits || !w_up || !up_scale || !w_down || !down_scale || !out) return GMM_ERR_BAD_ARGUMENT;
  if (tokens > 1 && (x_stride < hidden || out_stride < hidden || logits_stride < experts)) return GMM_ERR_BAD_ARGUMENT;
  if (!lies(w_up, up_stride_n, hidden, N) || !lies(w_down, down_stride_n, inner, hidden) || up_stride_g < 0 || down_stride_g < 0 ||
      (up_stride_g & 15) || (down_stride_g & 15)) return GMM_ERR_BAD_ARGUMENT;
  if (!workspace || workspace_bytes < p.bytes || !aligned16(workspace)) return GMM_ERR_WORKSPACE;
  char* const ws = static_cast<char*>(workspace);
  int32_t* const offs = reinterpret_cast<int32_t*>(ws);
  int32_t* const slot_expert = offs + experts;
  float* const slot_weight = reinterpret_cast<float*>(slot_expert + p.slots);
  int32_t* const row_token = slot_expert + 2 * p.slots;
  int32_t* const token_rows = slot_expert + 3 * p.slots;
  const auto at = [&](int64_t offset) { return reinterpret_cast<float*>(ws + offset); };
  hipStream_t s = static_cast<hipStream_t>(stream);

  FewArgs u{};
  u.a = ws + p.x_at; u.a_scale = at(p.x_scale_at); u.a_ld = p.x_pitch / 2; u.a_rows = int32_t(tokens); u.row_index = row_token;
  u.b = w_up; u.b_scale = up_scale; u.b_sg = up_stride_g / 2; u.b_ld = up_stride_n / 2; u.offs = offs; u.out = ws + p.h_at;
  u.G = int32_t(experts); u.M = int32_t(p.slots); u.N = int32_t(N); u.K = int32_t(hidden / 2);
  u.most = int32_t(tokens); u.block = int32_t(p.block); u.items = int32_t(p.items);      // a token chooses an expert once
  u.x_dtype = kNotRounded;
  if (p.x_here) { u.a = x; u.a_ld = tokens > 1 ? x_stride : hidden; u.x_dtype = dtype; }
  set_shape(u, p.up, p.activated);
  u.result = p.activated ? kActivated : kScaled;
  FewArgs d{};
  d.a = ws + p.act_at; d.a_scale = at(p.act_scale_at); d.a_ld = p.act_pitch / 2; d.a_rows = int32_t(p.slots);
  d.b = w_down; d.b_scale = down_scale; d.b_sg = down_stride_g / 2; d.b_ld = down_stride_n / 2; d.offs = offs; d.out = ws + p.y_at;
  d.G = int32_t(experts); d.M = int32_t(p.slots); d.N = int32_t(hidden); d.K = int32_t(inner / 2);
  d.most = int32_t(tokens); d.block = int32_t(p.block); d.items = int32_t(p.items);
  d.x_dtype = kNotRounded;
  if (p.act_here) { d.a = ws + p.h_at; d.a_ld = inner; d.x_dtype = GMM_DT_F32; }
  set_shape(d, p.down);
  d.result = kScaled;
  if (p.join) {
    d.result = kJoined;
    d.sum = out; d.sum_ld = out_stride; d.out_dtype = dtype; d.token_rows = token_rows; d.slot_weight = slot_weight; d.tokens = int32_t(tokens); d.top_k = int32_t(top_k);
    d.arrived = u.arrived = reinterpret_cast<uint32_t*>(ws + p.arrived_at);
    u.clear = d.tiles;
  }
  if (!sizes_fit(u) || !sizes_fit(d)) return GMM_ERR_UNSUPPORTED;
  if (p.items * u.tiles * u.parts >= (int64_t(1) << 31) || p.items * d.tiles * d.parts >= (int64_t(1) << 31)) return GMM_ERR_UNSUPPORTED;

  int rc = GMM_OK;
  const int64_t logits_ld = tokens > 1 ? logits_stride : experts;
  if (p.x_here && p.activated && routes_here(p.used, u.tiles, p.slots, experts))
    u.route = {logits, logits_ld, offs, token_rows, slot_weight, int32_t(tokens), int32_t(experts), int32_t(top_k), int32_t(p.slots), renormalize, logits_dtype};
  else
    rc = gmm_moe_route(logits, logits_ld, logits_dtype, tokens, experts, top_k, renormalize, offs, slot_expert, slot_weight, row_token, token_rows,
                       ws + p.table_at, p.table_bytes, stream);
  if (rc == GMM_OK && !p.x_here) rc = gmm_int8_quantize(x, reinterpret_cast<int8_t*>(ws + p.x_at), at(p.x_scale_at), tokens, hidden, x_stride, p.x_pitch, dtype, stream);
  if (rc == GMM_OK) rc = p.activated ? launch<true>(u, s) : launch<false>(u, s);
  if (rc == GMM_OK && !p.act_here)
    rc = p.activated ? gmm_int8_quantize(ws + p.h_at, reinterpret_cast<int8_t*>(ws + p.act_at), at(p.act_scale_at), p.slots, inner, inner, p.act_pitch,
                                         GMM_DT_F32, stream)
                     : gmm_int8_gated_parts(at(p.h_at), p.up.parts, p.slots * N, reinterpret_cast<int8_t*>(ws + p.act_at), at(p.act_scale_at), p.slots,
                                            inner, N, p.act_pitch, kind, s);
  if (rc == GMM_OK) rc = launch<false>(d, s);
  if (rc != GMM_OK || p.join) return rc;
  const dim3 grid(unsigned((hidden + kThreads - 1) / kThreads), unsigned(tokens));
  if (dtype == GMM_DT_BF16)
    hipLaunchKernelGGL(int8_combine_kernel<Bf16>, grid, dim3(kThreads), 0, s, at(p.y_at), token_rows, slot_weight, static_cast<Bf16*>(out), int(top_k),
                       p.down.parts, int(p.slots), int(hidden), out_stride);
  else
    hipLaunchKernelGGL(int8_combine_kernel<F16>, grid, dim3(kThreads), 0, s, at(p.y_at), token_rows, slot_weight, static_cast<F16*>(out), int(top_k),
                       p.down.parts, int(p.slots), int(hidden), out_stride);
  return hipGetLastError() == hipSuccess ? GMM_OK : GMM_ERR_LAUNCH;
}

}  // extern "C"
