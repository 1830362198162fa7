// Products of a few rows with a matrix that is read once: D[m, n] = sum over k of A[m, k] * W[k, n], m < 64.
//
// Reading W bounds them (2 bytes for 2 * m operations).  A wave takes a strip of columns and a range of k, loads both operands 16 bytes
// to a lane, some steps ahead, into registers, and multiplies with v_mfma_f32_16x16x32, whose operands want 8 values of k for one column
// (or row) in a lane.  How they get there, by the way W lies in memory:
//   along n, in strips of 128 columns (GMM_W_ROWS): a lane (j = lane & 15, g = lane >> 4) loads columns 8 j .. 8 j + 7 of rows
//     k + 8 g .. k + 8 g + 7; byte permutes of pairs of rows, half an instruction an element, make them the operands of eight
//     products, product i having columns i, 8 + i, 16 + i, ...  Nothing has to be undone: a column of the result is one of its product.
//   along k (GMM_W_COLS): eight lanes load 64 values of k of a column, and the lanes swap through LDS.  Loaded as the operand wants it, four
//     neighbouring lanes would ask for four cache lines: such a load takes the unit that looks lines up 64 cycles, not 16, and that
//     is what bounded these products (67 MB past 64 rows 27 us).
//   along n, 16 to 64 columns (GMM_W_THIN): rows of k side by side, turned by LDS reads that transpose.
//   anything else (GMM_W_ANY: neither step is one element, or fewer than eight of a kind): as GMM_W_ROWS, or 16 columns, element by element.
// Nothing is asked of alignment: a load of 16 bytes may begin at any element.  Where fewer than eight are left, along n as along k, the
// last eight are loaded: so no load leaves the matrix.  Along n, columns then lie elsewhere in the result (`position`); along k, the
// ones that were there already are shifted out (`tail`), in a range's last step.
// A goes through LDS as well, for the same reason.  Its rows that do not exist read as zeros and cost no access.  LDS is a wave's own
// here: its instructions run in order, nobody waits for anybody.  The waves of a workgroup share the range of k and add up in LDS.
#pragma once
#include <type_traits>

#include "gmm_elem.h"

namespace gmm {

constexpr int GMM_W_ROWS = 0, GMM_W_COLS = 1, GMM_W_ANY = 2, GMM_W_THIN = 3;
constexpr uint32_t kNowhere = 0x80000000u;   // an offset past every buffer: reads as zeros
constexpr int kStream = 2;                   // cache policy of loads of what is read once: non-temporal

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma(Bf16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(F16, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Two 8-bit integers: everything that counts elements counts pairs of them, and a product of 32 values of k is one of 64.  Its sums are 32-bit
// integers, kept as the bits of the registers that hold fp32 sums otherwise.
struct I8x2 { uint16_t bits; };
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma(I8x2, u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b),
                                                                          __builtin_bit_cast(i32x4, c), 0, 0, 0));
}

// Buffer of `bytes` bytes (below 2^31) at a base that all lanes share.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(at)), hi = __builtin_amdgcn_readfirstlane(uint32_t(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(hi) << 32 | lo), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// Value f as the sum of two 16-bit values: an operand that is held in 32 bits takes part in a product of 16-bit operands as two, and
// its error is then 2^-16 of it (bf16), or 2^-22 of it and 2^-25 at least (fp16, whose second value is below its normal range for |f| < 2^-3).
// Where the first overflows there is no second (fp16: |f| >= 65520).
template <typename T>
__device__ __forceinline__ void split(float f, T& high, T& low) {
  high = rounded<T>(f);
  const float back = widen(high);
  low = rounded<T>(__builtin_isfinite(back) ? f - back : 0.0f);
}

// Order of a wave's LDS accesses for the compiler; the hardware keeps it.
__device__ __forceinline__ void lds_order() { asm volatile("" ::: "memory"); }

// One strip of columns of one product, by one wave.
//   FR: products of 16 columns (GMM_W_ROWS: 8; GMM_W_COLS, GMM_W_THIN: 1, 2, 4; GMM_W_ANY: 1, 8).
//   MF: sixteens of rows.  NA: planes of A (2: A = high + low).  AM: how A comes (GMM_A_..).  ST: steps in flight.
constexpr int GMM_A_STAGED = 0;      // from memory, 16 bytes at a time
constexpr int GMM_A_ELEMENTS = 1;    // from memory, element by element (no alignment)
constexpr int GMM_A_RESIDENT = 2;    // lies in LDS

template <typename T, int LAY, int FR_, int MF, int NA, int AM, int ST>
struct Skinny {
  static constexpr int FR = FR_, STEPS = ST;
  static constexpr bool CYCLIC = std::is_same_v<T, I8x2>;     // sums of integers, which no order changes
  static constexpr int KS = LAY == GMM_W_COLS ? 64 : 32;      // k of a step
  static constexpr int KH = KS / 32;                          // products' halves of it
  static constexpr int COLUMNS = 16 * FR;
  static constexpr int CH = KS / 8;                           // 16-byte chunks of a row (or column) in a step
  static constexpr int ROWS_AT_ONCE = 64 / CH;                // that a load has
  static constexpr int WL = LAY == GMM_W_COLS ? 2 * FR : LAY == GMM_W_THIN ? FR : LAY == GMM_W_ROWS || FR == 8 ? 8 : 1;   // loads of W
  static constexpr int AL = MF * KH;                          // loads of a plane of A
  static constexpr int W_BYTES = LAY == GMM_W_COLS ? 128 * COLUMNS : LAY == GMM_W_THIN ? 1024 * FR : 0;
  static constexpr int PLANE_BYTES = AM == GMM_A_STAGED ? 32 * MF * KS : 0;
  static constexpr int LDS_BYTES = W_BYTES + NA * PLANE_BYTES;      // of a wave
  static_assert(LAY != GMM_W_ROWS || FR == 8, "");
  static_assert(LAY != GMM_W_ANY || FR == 1 || FR == 8, "");

  __amdgpu_buffer_rsrc_t w_buf, a_buf;
  char* lds;
  int lane;
  uint32_t w_at;          // byte offset of what the lane loads first, k = 0
  uint32_t w_step_k, w_step_n;   // bytes from one k, one column, to the next
  int columns;            // the lane's columns that exist (GMM_W_ROWS, GMM_W_THIN: all or none); GMM_W_COLS: the strip's (of either half)
  uint32_t w_jump;        // GMM_W_COLS: bytes that the second half of the columns lies further away than it would
  int w_half;             // and where it begins
  uint32_t a_at[AL];      // byte offset of the lane's rows of A, kNowhere: no such row
  uint32_t a_plane;       // bytes from the high to the low plane
  const char* resident;   // GMM_A_RESIDENT: row 0 of the high plane, from k = resident_k on,
  int pitch, resident_k, resident_rows;   // bytes from one row to the next, number of rows
  uint32_t turn;          // CYCLIC: the step that is the first
  uint32_t w_col[CYCLIC ? WL : 1];   // and byte offsets of the lane's columns, k = 0

  struct Step { u32x4 w[WL]; u32x4 a[AM == GMM_A_RESIDENT ? 1 : NA][AL]; };

  static __device__ __forceinline__ uint32_t element(__amdgpu_buffer_rsrc_t buf, uint32_t at) {
    return uint32_t(uint16_t(__builtin_amdgcn_raw_buffer_load_b16(buf, int(at), 0, 0)));
  }

  // Where a column of the strip is: in the lanes j, 16 + j, ... of product i.  left: how many columns there are from it on.
  static __device__ __forceinline__ int position(int column, int left) {
    return LAY == GMM_W_ROWS || LAY == GMM_W_THIN ? column - column % 8 + max(column % 8, 8 - left) : column;
  }
  static __device__ __forceinline__ int product_of(int position) { return LAY == GMM_W_ROWS || LAY == GMM_W_ANY ? position % FR : position / 16; }
  static __device__ __forceinline__ int lane_of(int position) { return LAY == GMM_W_ROWS || LAY == GMM_W_ANY ? position / FR : position % 16; }

  // Eight values of k from `from` on of a row, of which those before `end` exist: where they are loaded, relative to it; and, loaded, the
  // ones that exist, zeros behind them.
  static __device__ __forceinline__ uint32_t back(int from, int end) { return uint32_t(max(0, from + 8 - end)) * 2; }
  static __device__ __forceinline__ u32x4 tail(u32x4 v, int from, int end) {
    const int over = from + 8 - end;      // nothing was loaded: zeros
    const bool four = over & 4, two = over & 2, one = over & 1, any = over > 0;
    if (any) {
      v = four ? u32x4{v[2], v[3], 0, 0} : v;
      v = two ? u32x4{v[1], v[2], v[3], 0} : v;
      v = one ? u32x4{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16} : v;
    }
    return v;
  }

  // The strip of columns from `first` on, of which `count` (or more than the strip holds) exist; steps in elements.  With `half` > 0 it is
  // that many columns from `first` on and as many from `other` on, `count` of each.
  __device__ __forceinline__ void set_columns(int first, int count, uint32_t sk, uint32_t sn, int half = 0, int other = 0) {
    const int j = lane & 15;
    w_step_k = sk * 2;
    w_step_n = sn * 2;
    if constexpr (LAY == GMM_W_COLS) {
      columns = count;
      w_half = half ? half : COLUMNS;
      w_jump = half ? uint32_t(other - first - half) * w_step_n : 0;
      w_at = uint32_t(first + (lane >> 3)) * w_step_n + (lane & 7) * 16;
      if constexpr (CYCLIC)
#pragma unroll
        for (int i = 0; i < WL; ++i) {
          const bool second = 8 * i >= w_half;
          w_col[i] = 8 * i + (lane >> 3) - (second ? w_half : 0) < columns ? w_at + 8 * i * w_step_n + (second ? w_jump : 0) : kNowhere;
        }
    } else if constexpr (LAY == GMM_W_THIN) {
      const int c = lane % (2 * FR) * 8;
      columns = count - c;
      w_at = uint32_t(lane / (2 * FR)) * w_step_k + uint32_t(first + c - max(0, 8 - max(1, columns))) * 2;
    } else {
      const int c = FR * j, in = half ? c % half : c;
      columns = max(0, min(FR, count - in));
      w_at = uint32_t((half && c >= half ? other : first) + in - (LAY == GMM_W_ROWS ? 8 - max(1, columns) : 0)) * w_step_n;
    }
  }

  // at(r): byte offset of row r of A, kNowhere if there is none.
  template <typename F>
  __device__ __forceinline__ void set_rows(F&& at) {
#pragma unroll
    for (int i = 0; i < AL; ++i) {
      const uint32_t from = at(AM == GMM_A_ELEMENTS ? 16 * i + (lane & 15) : ROWS_AT_ONCE * i + lane / CH);
      a_at[i] = from == kNowhere || AM == GMM_A_ELEMENTS ? from : from + lane % CH * 16;
    }
  }

  // CYCLIC: what k adds to an offset; past the end, past every buffer (of columns and rows that do not exist it may lead back into it: their sums go
  // nowhere).  Not asked for each load, or the compiler branches around them, and they wait for one another.
  static __device__ __forceinline__ uint32_t from_k(bool in, int k, int at, int end) {
    uint32_t along = in ? uint32_t(k) * 2 - back(at, end) : kNowhere;
    asm volatile("" : "+v"(along));
    return along;
  }

  // Loads k .. k + KS - 1, of which those before `end` exist, and the first M of the sixteens of rows.
  template <int M>
  __device__ __forceinline__ void load(Step& s, int k, int end) const {
    load_w(s.w, k, end);
    load_a<M>(s, k, end);
  }

  __device__ __forceinline__ void load_w(u32x4 (&w)[WL], int k, int end) const {
    const int kl = k + 8 * (lane >> 4);
    if constexpr (LAY == GMM_W_ROWS) {
      const uint32_t at = w_at + uint32_t(kl) * w_step_k;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        w[r] = __builtin_amdgcn_raw_buffer_load_b128(w_buf, int(columns && kl + r < end ? at + r * w_step_k : kNowhere), 0, kStream);
    } else if constexpr (LAY == GMM_W_COLS) {
      const bool in = k + 8 * (lane & 7) < end;
      if constexpr (CYCLIC) {
        const uint32_t along = from_k(in, k, k + 8 * (lane & 7), end);
#pragma unroll
        for (int i = 0; i < WL; ++i) w[i] = __builtin_amdgcn_raw_buffer_load_b128(w_buf, int(w_col[i] + along), 0, kStream);
        return;
      }
      const uint32_t at = w_at + uint32_t(k) * 2 - back(k + 8 * (lane & 7), end);
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        const int c = 8 * i + (lane >> 3);
        const bool second = 8 * i >= w_half;
        w[i] = __builtin_amdgcn_raw_buffer_load_b128(
            w_buf, int(in && c - (second ? w_half : 0) < columns ? at + 8 * i * w_step_n + (second ? w_jump : 0) : kNowhere), 0, kStream);
      }
    } else if constexpr (LAY == GMM_W_THIN) {
#pragma unroll
      for (int i = 0; i < WL; ++i) {
        const int row = k + 32 / FR * i;
        w[i] = __builtin_amdgcn_raw_buffer_load_b128(
            w_buf, int(columns > 0 && row + lane / (2 * FR) < end ? w_at + uint32_t(row) * w_step_k : kNowhere), 0, 0);
      }
    } else if constexpr (FR == 1) {
      const uint32_t at = w_at + uint32_t(kl) * w_step_k;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t lo = element(w_buf, columns && kl + 2 * q < end ? at + 2 * q * w_step_k : kNowhere);
        const uint32_t hi = element(w_buf, columns && kl + 2 * q + 1 < end ? at + (2 * q + 1) * w_step_k : kNowhere);
        w[0][q] = lo | hi << 16;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t at = w_at + uint32_t(kl + r) * w_step_k + 2 * q * w_step_n;
          const bool in = kl + r < end;
          const uint32_t lo = element(w_buf, in && 2 * q < columns ? at : kNowhere);
          const uint32_t hi = element(w_buf, in && 2 * q + 1 < columns ? at + w_step_n : kNowhere);
          w[r][q] = lo | hi << 16;
        }
    }
  }

  template <int M>
  __device__ __forceinline__ void load_a(Step& s, int k, int end) const {
    if constexpr (AM == GMM_A_RESIDENT) return;
#pragma unroll
    for (int i = 0; i < M * KH; ++i)
#pragma unroll
      for (int p = 0; p < NA; ++p) {
        if constexpr (AM == GMM_A_ELEMENTS) {
          const int kl = k + 8 * (lane >> 4);
          const uint32_t at = a_at[i] + p * a_plane + uint32_t(kl) * 2;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t lo = element(a_buf, a_at[i] != kNowhere && kl + 2 * q < end ? at + 4 * q : kNowhere);
            const uint32_t hi = element(a_buf, a_at[i] != kNowhere && kl + 2 * q + 1 < end ? at + 4 * q + 2 : kNowhere);
            s.a[p][i][q] = lo | hi << 16;
          }
        } else if constexpr (CYCLIC) {
          const uint32_t along = from_k(k + 8 * (lane % CH) < end, k, k + 8 * (lane % CH), end);
          s.a[p][i] = __builtin_amdgcn_raw_buffer_load_b128(a_buf, int(a_at[i] + p * a_plane + along), 0, 0);
        } else {
          const bool in = a_at[i] != kNowhere && k + 8 * (lane % CH) < end;
          const uint32_t at = a_at[i] + p * a_plane + uint32_t(k) * 2 - back(k + 8 * (lane % CH), end);
          s.a[p][i] = __builtin_amdgcn_raw_buffer_load_b128(a_buf, int(in ? at : kNowhere), 0, 0);
        }
      }
  }

  // GMM_W_ROWS: the second operand of product i.
  static __device__ __forceinline__ u32x4 turned(const u32x4 (&w)[WL], int i) {
    u32x4 b;
#pragma unroll
    for (int q = 0; q < 4; ++q) b[q] = __builtin_amdgcn_perm(w[2 * q + 1][i / 2], w[2 * q][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
    return b;
  }

  // Where chunk c of row (or column) r of a step lies: such that 16 rows' chunks lie in different banks.
  static __device__ __forceinline__ int chunk_at(int r, int c) { return r * 16 * CH + 16 * (CH == 8 ? c ^ (r >> 1 & 7) : c ^ (r >> 2 & 3)); }

  template <int M>
  __device__ __forceinline__ void multiply(Step& s, int k, int end, f32x4 (&acc)[MF][FR]) const {
    const int j = lane & 15, g = lane >> 4;
    if ((end & 7) && k + KS > end) {      // asked of every product it cost 2 %
      if constexpr (LAY == GMM_W_COLS)
#pragma unroll
        for (int i = 0; i < WL; ++i) s.w[i] = tail(s.w[i], k + 8 * (lane & 7), end);
      if constexpr (AM == GMM_A_STAGED)
#pragma unroll
        for (int i = 0; i < M * KH; ++i)
#pragma unroll
          for (int p = 0; p < NA; ++p) s.a[p][i] = tail(s.a[p][i], k + 8 * (lane % CH), end);
    }
    lds_order();
    if constexpr (LAY == GMM_W_COLS)
#pragma unroll
      for (int i = 0; i < WL; ++i) *reinterpret_cast<u32x4*>(lds + chunk_at(8 * i + (lane >> 3), lane & 7)) = s.w[i];
    if constexpr (LAY == GMM_W_THIN)
#pragma unroll
      for (int i = 0; i < WL; ++i) *reinterpret_cast<u32x4*>(lds + 1024 * i + 16 * lane) = s.w[i];
    if constexpr (AM == GMM_A_STAGED)
#pragma unroll
      for (int i = 0; i < M * KH; ++i)
#pragma unroll
        for (int p = 0; p < NA; ++p)
          *reinterpret_cast<u32x4*>(lds + W_BYTES + p * PLANE_BYTES + chunk_at(ROWS_AT_ONCE * i + lane / CH, lane % CH)) = s.a[p][i];
    lds_order();
#pragma unroll
    for (int h = 0; h < KH; ++h) {
      u32x4 a[M][NA];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int p = 0; p < NA; ++p) {
          if constexpr (AM == GMM_A_ELEMENTS) a[m][p] = s.a[p][KH * m + h];
          else if constexpr (AM == GMM_A_RESIDENT) {
            const int at = k + 8 * (4 * h + g);      // zeros behind the end, whose W reads as zeros: what lies there may be no number
            a[m][p] = *reinterpret_cast<const u32x4*>(resident + p * a_plane + min(16 * m + j, resident_rows - 1) * pitch + (at < end ? at - resident_k : 0) * 2);
            a[m][p] = at < end ? a[m][p] : u32x4{0, 0, 0, 0};
          }
          else a[m][p] = *reinterpret_cast<const u32x4*>(lds + W_BYTES + p * PLANE_BYTES + chunk_at(16 * m + j, 4 * h + g));
        }
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        u32x4 b;
        if constexpr (LAY == GMM_W_COLS) {
          b = *reinterpret_cast<const u32x4*>(lds + chunk_at(16 * i + j, 4 * h + g));
        } else if constexpr (LAY == GMM_W_THIN) {
          typedef short s16x4 __attribute__((ext_vector_type(4)));
          typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
          char* const from = lds + (8 * g + j / 4) * 32 * FR + 32 * i + j % 4 * 8;
          const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from)));
          const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(from + 4 * 32 * FR)));
          b = u32x4{lo[0], lo[1], hi[0], hi[1]};
        } else if constexpr (FR == 1) {
          b = s.w[0];
        } else {
          b = turned(s.w, i);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
          for (int p = 0; p < NA; ++p) acc[m][i] = mfma(T{}, a[m][p], b, acc[m][i]);
      }
    }
  }

  // acc += A[:, k] W[k] over every WAVES-th step of begin .. end.  Steps past the end load nothing: no branch stands between the loads in
  // flight, and nothing moves past the barriers: moved loads would be waited for together.
  template <int M, int WAVES>
  __device__ __forceinline__ void prime(Step (&step)[ST], int begin, int end) const {
#pragma unroll
    for (int u = 0; u < ST; ++u) {
      load<M>(step[u], begin + u * WAVES * KS, end);
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  template <int M, int WAVES>
  __device__ __forceinline__ void primed(Step (&step)[ST], int begin, int end, f32x4 (&acc)[MF][FR]) const {
    constexpr int NEXT = WAVES * KS;
    for (int k = begin; k < end; k += ST * NEXT)
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        multiply<M>(step[u], k + u * NEXT, end, acc);
        __builtin_amdgcn_sched_barrier(0);
        load<M>(step[u], k + (ST + u) * NEXT, end);
        __builtin_amdgcn_sched_barrier(0);
      }
  }

  // The same from the `turn`-th step on and round to the one before it (CYCLIC).
  template <int M, int WAVES>
  struct Cycle {
    int next, begin, last, end, left, at[ST];
    __device__ __forceinline__ Cycle(int begin_, int end_, uint32_t turn) : begin(begin_), end(end_) {
      constexpr int NEXT = WAVES * KS;
      left = begin < end ? (end - begin + NEXT - 1) / NEXT : 0;
      last = begin + left * NEXT;
      next = begin + (left ? int(turn % uint32_t(left)) * NEXT : 0);
    }
    __device__ __forceinline__ int advance() {      // past the last step: to the end
      const int k = left > 0 ? next : end;
      --left;
      next += WAVES * KS;
      next = next >= last ? begin : next;
      return k;
    }
    __device__ __forceinline__ void prime(const Skinny& s, Step (&step)[ST]) {
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        at[u] = advance();
        s.load<M>(step[u], at[u], end);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    __device__ __forceinline__ void primed(const Skinny& s, Step (&step)[ST], f32x4 (&acc)[MF][FR]) {
      for (int todo = (last - begin) / (WAVES * KS); todo > 0; todo -= ST)
#pragma unroll
        for (int u = 0; u < ST; ++u) {
          s.multiply<M>(step[u], at[u], end, acc);
          __builtin_amdgcn_sched_barrier(0);
          at[u] = advance();
          s.load<M>(step[u], at[u], end);
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  };

  template <int M, int WAVES>
  __device__ __forceinline__ void steps(int begin, int end, f32x4 (&acc)[MF][FR]) const {
    Step step[ST];
    if constexpr (CYCLIC) {
      Cycle<M, WAVES> c(begin, end, turn);
      c.prime(*this, step);
      c.primed(*this, step, acc);
    } else {
      prime<M, WAVES>(step, begin, end);
      primed<M, WAVES>(step, begin, end, acc);
    }
  }

  // The part of wave `wave` of WAVES of the product over begin .. end: the waves' steps lie side by side in memory.  rows: how many there
  // are; sixteens that hold none take no part.
  template <int WAVES>
  __device__ __forceinline__ void run(int rows, int begin, int end, int wave, f32x4 (&acc)[MF][FR]) const {
    begin += wave * KS;
    if constexpr (MF >= 2) {
      if (rows <= 16) return steps<1, WAVES>(begin, end, acc);
    }
    if constexpr (MF >= 4) {
      if (rows <= 32) return steps<2, WAVES>(begin, end, acc);
    }
    steps<MF, WAVES>(begin, end, acc);
  }
};

// A strip of a matrix that is large.
template <typename T, int LAY, int MF, int NA, int AM = LAY == GMM_W_ANY ? GMM_A_ELEMENTS : GMM_A_STAGED>
using Strip = Skinny<T, LAY, LAY == GMM_W_COLS ? 4 : 8, MF, NA, AM, 2>;

template <int MF, int FR>
__device__ __forceinline__ void clear(f32x4 (&acc)[MF][FR]) {
#pragma unroll
  for (int m = 0; m < MF; ++m)
#pragma unroll
    for (int i = 0; i < FR; ++i) acc[m][i] = f32x4{0, 0, 0, 0};
}

// Sums over the waves of a workgroup, one sixteen of rows at a time: sums[wave][product i][lane].
template <int WAVES, int FR>
struct SkinnySums {
  static constexpr int PITCH = 64 + 4;       // of a product's 64 lanes: neighbours in a row of the result lie in other banks
  f32x4 at[WAVES][FR][PITCH];

  __device__ __forceinline__ void put(int wave, int lane, const f32x4 (&acc)[FR]) {
#pragma unroll
    for (int i = 0; i < FR; ++i) at[wave][i][lane] = acc[i];
  }
  // Rows 4 g .. 4 g + 3 of the column that product i has in lane j; of one wave alone, or the sum over all.
  __device__ __forceinline__ f32x4 of(int wave, int i, int j, int g) const { return at[wave][i][16 * g + j]; }
  __device__ __forceinline__ f32x4 get(int i, int j, int g) const {
    f32x4 s = of(0, i, j, g);
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += of(w, i, j, g);
    return s;
  }
  // The same of integers.
  __device__ __forceinline__ i32x4 whole(int i, int j, int g) const {
    i32x4 s = __builtin_bit_cast(i32x4, of(0, i, j, g));
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += __builtin_bit_cast(i32x4, of(w, i, j, g));
    return s;
  }
};

// LDS of a workgroup: the waves' own parts while they multiply, then (behind a barrier) the sums.
template <typename S, int WAVES>
union SkinnyShared {
  char wave[WAVES][S::LDS_BYTES > 0 ? S::LDS_BYTES : 16];
  SkinnySums<WAVES, S::FR> sums;
  __device__ SkinnyShared() {}
};

// f(i, in) for all i < n, eight and then four at a time: as many loads are on their way together.  Past the end the last one again, `in` false.
// (A loop that the compiler unrolls takes what is left over one by one: a trip to memory each.)
template <typename F>
__device__ __forceinline__ void in_fours(int n, F&& f) {
  int i = 0;
  for (; i + 4 < n; i += 8)
#pragma unroll
    for (int u = 0; u < 8; ++u) f(min(i + u, n - 1), i + u < n);
  if (i < n)
#pragma unroll
    for (int u = 0; u < 4; ++u) f(min(i + u, n - 1), i + u < n);
}

// ---------------------------------------------------------------- host side
inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Layout of matrices [K, N] with the steps sk and sn of which eight columns belong together.
inline int layout_of(int64_t sk, int64_t sn, int64_t K, int64_t N) {
  if (K < 8) return GMM_W_ANY;
  return sn == 1 && N >= 8 ? GMM_W_ROWS : sk == 1 ? GMM_W_COLS : GMM_W_ANY;
}

// Bytes from the first to behind the last element of a matrix of 16-bit elements; 0: strides that do not fit or 2 GiB and more.
inline uint32_t matrix_bytes(int64_t K, int64_t N, int64_t sk, int64_t sn) {
  constexpr int64_t most = (int64_t(1) << 30) - 64;
  if (sk < 0 || sn < 0 || (sk > 0 && K - 1 > most / sk) || (sn > 0 && N - 1 > most / sn)) return 0;
  const int64_t n = (K - 1) * sk + (N - 1) * sn + 1;
  return n > most ? 0 : uint32_t(n * 2);
}

}  // namespace gmm
