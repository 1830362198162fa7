// Products of a few rows with a matrix that is read once: D[m, n] = sum over k of A[m, k] * W[k, n], m < 64.
//
// Reading W bounds them (2 bytes for 2 * m operations).  So W goes from memory into registers past no LDS: a wave takes a strip of
// columns and a range of k, and what it loads is the second operand of v_mfma_f32_16x16x32 as it is, or nearly so:
//   W contiguous along n (GMM_W_ROWS): the operand wants 8 values of k for one column in a lane, memory gives 8 columns for one k.  Lane
//     (j = lane & 15, g = lane >> 4) loads columns 8 j .. 8 j + 7 of rows k + 8 g .. k + 8 g + 7 (16 bytes each, 256 side by side over the
//     lanes); byte permutes of pairs of rows, half an instruction an element, make them the operands of eight products, product i having
//     columns i, 8 + i, 16 + i, ...  Nothing has to be undone: a column of the result is a column of its product.
//   W contiguous along k (GMM_W_COLS): a lane loads 16 values of k of each of 4 columns, 128 bytes side by side over the four g's.
//   anything else (GMM_W_ANY): as GMM_W_ROWS, element by element.
// Rows of A are the first operand: 16 rows to a product, rows that do not exist read as zeros and cost no access.  The waves of a
// workgroup share the range of k and add their results up in LDS.
#pragma once
#include "gmm_elem.h"

namespace gmm {

constexpr int GMM_W_ROWS = 0, GMM_W_COLS = 1, GMM_W_ANY = 2;
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

// Buffer of `bytes` bytes (below 2^31) at a base that all lanes share.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const void* base, uint32_t bytes) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(at)), hi = __builtin_amdgcn_readfirstlane(uint32_t(at >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uint64_t(hi) << 32 | lo), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// Value f as the sum of two 16-bit values: an operand that is held in 32 bits takes part in a product of 16-bit operands as two, and
// its error is then 2^-16 (bf16) or 2^-22 (fp16) of it.  Where the first overflows there is no second (fp16: |f| >= 65520).
template <typename T>
__device__ __forceinline__ void split(float f, T& high, T& low) {
  high = rounded<T>(f);
  const float back = widen(high);
  low = rounded<T>(__builtin_isfinite(back) ? f - back : 0.0f);
}

// One strip of columns of one product, by one wave.
//   FR: columns of a lane, which is products of 16 columns (GMM_W_ROWS: 2, 4, 8; GMM_W_COLS: any; GMM_W_ANY: 1, 8).
//   KH: 32s of k in a step (2 for GMM_W_COLS where k is long: whole cache lines).
//   AE: rows of A are read element by element (no alignment).
//   MF: sixteens of rows.  NA: planes of A (2: A = high + low).  ST: steps in flight.
template <typename T, int LAY, int FR_, int KH, bool AE, int MF, int NA, int ST>
struct Skinny {
  static constexpr int FR = FR_;
  static constexpr int KS = 32 * KH;          // k of a step
  static constexpr int KG = KS / 4;           // of them a lane's
  static constexpr int COLUMNS = 16 * FR;
  static constexpr int WORDS = LAY == GMM_W_COLS ? 4 * FR * KH : FR == 1 ? 4 : 4 * FR;   // of W in a step, of a lane
  static_assert(LAY == GMM_W_COLS || KH == 1, "");
  static_assert(LAY != GMM_W_ANY || FR == 1 || FR == 8, "");
  static_assert(LAY != GMM_W_ROWS || FR == 2 || FR == 4 || FR == 8, "");

  __amdgpu_buffer_rsrc_t w_buf, a_buf;
  uint32_t w_at;          // byte offset of the lane's first column
  uint32_t w_step_k, w_step_n;   // bytes from one k, one column, to the next
  int columns;            // the lane's columns that exist (GMM_W_ROWS: all or none)
  uint32_t a_at[MF];      // byte offset of the lane's rows of A, kNowhere: no such row
  uint32_t a_plane;       // bytes from the high to the low plane

  struct Step { uint32_t w[WORDS]; u32x4 a[MF][NA][KH]; };

  static __device__ __forceinline__ uint32_t element(__amdgpu_buffer_rsrc_t buf, uint32_t at) {
    return uint32_t(uint16_t(__builtin_amdgcn_raw_buffer_load_b16(buf, int(at), 0, 0)));
  }

  // Loads k .. k + KS - 1, of which those before `end` exist.
  template <int M>
  __device__ __forceinline__ void load(Step& s, int k, int end, int g) const {
    load_w(s, k, end, g);
    load_a<M>(s, k, end, g);
  }

  __device__ __forceinline__ void load_w(Step& s, int k, int end, int g) const {
    const int kl = k + KG * g;
    if constexpr (LAY == GMM_W_ROWS) {
      const uint32_t at = w_at + uint32_t(kl) * w_step_k;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int from = int(columns && kl + r < end ? at + r * w_step_k : kNowhere);
        if constexpr (FR == 8) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(w_buf, from, 0, kStream);
#pragma unroll
          for (int i = 0; i < 4; ++i) s.w[4 * r + i] = v[i];
        } else if constexpr (FR == 4) {
          const auto v = __builtin_amdgcn_raw_buffer_load_b64(w_buf, from, 0, 0);
          s.w[2 * r] = v[0];
          s.w[2 * r + 1] = v[1];
        } else {
          s.w[r] = __builtin_amdgcn_raw_buffer_load_b32(w_buf, from, 0, 0);
        }
      }
    } else if constexpr (LAY == GMM_W_COLS) {
      const uint32_t at = w_at + uint32_t(kl) * 2;
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(
              w_buf, int(i < columns && kl + 8 * h < end ? at + i * w_step_n + 16 * h : kNowhere), 0, kStream);
#pragma unroll
          for (int q = 0; q < 4; ++q) s.w[4 * (KH * i + h) + q] = v[q];
        }
    } else if constexpr (FR == 1) {
      const uint32_t at = w_at + uint32_t(kl) * w_step_k;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t lo = element(w_buf, columns && kl + 2 * q < end ? at + 2 * q * w_step_k : kNowhere);
        const uint32_t hi = element(w_buf, columns && kl + 2 * q + 1 < end ? at + (2 * q + 1) * w_step_k : kNowhere);
        s.w[q] = lo | hi << 16;
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
          s.w[4 * r + q] = lo | hi << 16;
        }
    }
  }

  // The first M of the sixteens of rows.
  template <int M>
  __device__ __forceinline__ void load_a(Step& s, int k, int end, int g) const {
    const int kl = k + KG * g;
#pragma unroll
    for (int m = 0; m < M; ++m) {
#pragma unroll
      for (int p = 0; p < NA; ++p)
#pragma unroll
        for (int h = 0; h < KH; ++h) {
          const uint32_t at = a_at[m] + p * a_plane + uint32_t(kl + 8 * h) * 2;
          if constexpr (AE) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const int kq = kl + 8 * h + 2 * q;
              const uint32_t lo = element(a_buf, a_at[m] != kNowhere && kq < end ? at + 4 * q : kNowhere);
              const uint32_t hi = element(a_buf, a_at[m] != kNowhere && kq + 1 < end ? at + 4 * q + 2 : kNowhere);
              s.a[m][p][h][q] = lo | hi << 16;
            }
          } else {
            s.a[m][p][h] = __builtin_amdgcn_raw_buffer_load_b128(a_buf, int(a_at[m] != kNowhere && kl + 8 * h < end ? at : kNowhere), 0, 0);
          }
        }
    }
  }

  // Second operand of product i, half h of the step.
  static __device__ __forceinline__ u32x4 operand(const Step& s, int i, int h) {
    u32x4 b;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (LAY == GMM_W_COLS) b[q] = s.w[4 * (KH * i + h) + q];
      else if constexpr (FR == 1) b[q] = s.w[q];
      else b[q] = __builtin_amdgcn_perm(s.w[(2 * q + 1) * (FR / 2) + i / 2], s.w[2 * q * (FR / 2) + i / 2], i & 1 ? 0x07060302u : 0x05040100u);
    }
    return b;
  }

  template <int M>
  __device__ __forceinline__ void multiply(const Step& s, f32x4 (&acc)[MF][FR]) const {
#pragma unroll
    for (int i = 0; i < FR; ++i)
#pragma unroll
      for (int h = 0; h < KH; ++h) {
        const u32x4 b = operand(s, i, h);
#pragma unroll
        for (int m = 0; m < M; ++m) {
#pragma unroll
          for (int p = 0; p < NA; ++p) acc[m][i] = mfma(T{}, s.a[m][p][h], b, acc[m][i]);
        }
      }
  }

  // acc += A[:, begin .. end) W[begin .. end).  Steps past the end load nothing: no branch stands between the loads in flight.
  template <int M>
  __device__ __forceinline__ void steps(int begin, int end, int g, f32x4 (&acc)[MF][FR]) const {
    Step step[ST];
#pragma unroll
    for (int u = 0; u < ST; ++u) load<M>(step[u], begin + u * KS, end, g);
    for (int k = begin; k < end; k += ST * KS)
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        multiply<M>(step[u], acc);
        load<M>(step[u], k + (ST + u) * KS, end, g);
      }
  }

  // rows: how many there are; sixteens that hold none take no part.
  __device__ __forceinline__ void run(int rows, int begin, int end, int g, f32x4 (&acc)[MF][FR]) const {
    if constexpr (MF >= 2) {
      if (rows <= 16) return steps<1>(begin, end, g, acc);
    }
    if constexpr (MF >= 4) {
      if (rows <= 32) return steps<2>(begin, end, g, acc);
    }
    steps<MF>(begin, end, g, acc);
  }
};

// A strip of a matrix that is large: all columns of a lane in 16-byte loads, whole cache lines.
template <typename T, int LAY, int MF, int NA, int ST>
using Strip = Skinny<T, LAY, LAY == GMM_W_COLS ? 4 : 8, LAY == GMM_W_COLS ? 2 : 1, LAY == GMM_W_ANY, MF, NA, ST>;

// Range of k of one of WAVES waves: whole steps of KS, dealt evenly.
template <int KS, int WAVES>
__device__ __forceinline__ void wave_range(int begin, int end, int wave, int& from, int& to) {
  const int steps = (end - begin + KS - 1) / KS, each = (steps + WAVES - 1) / WAVES;
  from = begin + wave * each * KS;
  to = min(end, from + each * KS);
}

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
  // Rows 4 g .. 4 g + 3 of column FR * j + i of the strip.
  __device__ __forceinline__ f32x4 get(int i, int j, int g) const {
    f32x4 s = at[0][i][16 * g + j];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) s += at[w][i][16 * g + j];
    return s;
  }
};

// ---------------------------------------------------------------- host side
inline bool multiple8(int64_t v) { return (v & 7) == 0; }
inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// Layout of a stack of matrices [G, K, N].  n_whole: columns come in whole eights; whole: 16 bytes of A can be read at a time.
inline int layout_of(const void* w, int64_t sg, int64_t sk, int64_t sn, int64_t K, bool n_whole, bool whole) {
  if (!whole || !aligned16(w) || !multiple8(sg) || !multiple8(K)) return GMM_W_ANY;
  if (sn == 1 && multiple8(sk) && n_whole) return GMM_W_ROWS;
  if (sk == 1 && multiple8(sn)) return GMM_W_COLS;
  return GMM_W_ANY;
}

// Bytes from the first to behind the last element of a matrix of 16-bit elements; 0: strides that do not fit or 2 GiB and more.
inline uint32_t matrix_bytes(int64_t K, int64_t N, int64_t sk, int64_t sn) {
  constexpr int64_t most = (int64_t(1) << 30) - 64;
  if (sk < 0 || sn < 0 || (sk > 0 && K - 1 > most / sk) || (sn > 0 && N - 1 > most / sn)) return 0;
  const int64_t n = (K - 1) * sk + (N - 1) * sn + 1;
  return n > most ? 0 : uint32_t(n * 2);
}

}  // namespace gmm
