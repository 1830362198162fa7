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

// One strip of columns of one product, by one wave.  MF: sixteens of rows.  NA: planes of A (2: A = high + low).  ST: steps in flight.
template <typename T, int LAY, int MF, int NA, int ST>
struct Skinny {
  static constexpr int FR = LAY == GMM_W_COLS ? 4 : 8;        // columns of a lane: products of 16 columns
  static constexpr int KS = LAY == GMM_W_COLS ? 64 : 32;      // k of a step
  static constexpr int KG = KS / 4;                           // of them a lane's
  static constexpr int COLUMNS = 16 * FR;

  __amdgpu_buffer_rsrc_t w_buf, a_buf;
  uint32_t w_at;          // byte offset of the lane's first column
  uint32_t w_step_k, w_step_n;   // bytes from one k, one column, to the next
  int columns;            // the lane's columns that exist (GMM_W_ROWS: all or none)
  uint32_t a_at[MF];      // byte offset of the lane's rows of A, kNowhere: no such row
  uint32_t a_plane;       // bytes from the high to the low plane
  int rows16;             // sixteens of rows that hold any

  struct Step { u32x4 w[8]; u32x4 a[MF][NA][KS / 32]; };

  __device__ __forceinline__ uint32_t element(__amdgpu_buffer_rsrc_t buf, uint32_t at) const {
    return uint32_t(uint16_t(__builtin_amdgcn_raw_buffer_load_b16(buf, int(at), 0, 0)));
  }

  // Loads k .. k + KS - 1, of which those before `end` exist.
  __device__ __forceinline__ void load(Step& s, int k, int end, int g) const {
    load_w(s, k, end, g);
    load_a(s, k, end, g);
  }

  __device__ __forceinline__ void load_w(Step& s, int k, int end, int g) const {
    const int kl = k + KG * g;
    if constexpr (LAY == GMM_W_ROWS) {
      const uint32_t at = w_at + uint32_t(kl) * w_step_k;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        s.w[r] = __builtin_amdgcn_raw_buffer_load_b128(w_buf, int(columns && kl + r < end ? at + r * w_step_k : kNowhere), 0, kStream);
    } else if constexpr (LAY == GMM_W_COLS) {
      const uint32_t at = w_at + uint32_t(kl) * 2;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          s.w[2 * i + h] = __builtin_amdgcn_raw_buffer_load_b128(
              w_buf, int(i < columns && kl + 8 * h < end ? at + i * w_step_n + 16 * h : kNowhere), 0, kStream);
    } else {
#pragma unroll
      for (int r = 0; r < 8; ++r)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t at = w_at + uint32_t(kl + r) * w_step_k + 2 * q * w_step_n;
          const bool in = kl + r < end;
          const uint32_t lo = element(w_buf, in && 2 * q < columns ? at : kNowhere);
          const uint32_t hi = element(w_buf, in && 2 * q + 1 < columns ? at + w_step_n : kNowhere);
          s.w[r][q] = lo | hi << 16;
        }
    }
  }

  __device__ __forceinline__ void load_a(Step& s, int k, int end, int g) const {
    const int kl = k + KG * g;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
      if (m >= rows16) break;
#pragma unroll
      for (int p = 0; p < NA; ++p)
#pragma unroll
        for (int h = 0; h < KS / 32; ++h) {
          const uint32_t at = a_at[m] + p * a_plane + uint32_t(kl + 8 * h) * 2;
          if constexpr (LAY == GMM_W_ANY) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t lo = element(a_buf, a_at[m] != kNowhere && kl + 2 * q < end ? at + 4 * q : kNowhere);
              const uint32_t hi = element(a_buf, a_at[m] != kNowhere && kl + 2 * q + 1 < end ? at + 4 * q + 2 : kNowhere);
              s.a[m][p][h][q] = lo | hi << 16;
            }
          } else {
            s.a[m][p][h] = __builtin_amdgcn_raw_buffer_load_b128(a_buf, int(a_at[m] != kNowhere && kl + 8 * h < end ? at : kNowhere), 0, 0);
          }
        }
    }
  }

  __device__ __forceinline__ void multiply(const Step& s, f32x4 (&acc)[MF][FR]) const {
    if constexpr (LAY == GMM_W_COLS) {
#pragma unroll
      for (int i = 0; i < FR; ++i)
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          if (m >= rows16) break;
#pragma unroll
          for (int p = 0; p < NA; ++p)
#pragma unroll
            for (int h = 0; h < 2; ++h) acc[m][i] = mfma(T{}, s.a[m][p][h], s.w[2 * i + h], acc[m][i]);
        }
    } else {
#pragma unroll
      for (int i = 0; i < FR; ++i) {
        u32x4 b;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          b[q] = __builtin_amdgcn_perm(s.w[2 * q + 1][i / 2], s.w[2 * q][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int m = 0; m < MF; ++m) {
          if (m >= rows16) break;
#pragma unroll
          for (int p = 0; p < NA; ++p) acc[m][i] = mfma(T{}, s.a[m][p][0], b, acc[m][i]);
        }
      }
    }
  }

  // acc += A[:, begin .. end) W[begin .. end).  Steps past the end load nothing: no branch stands between the loads in flight.
  __device__ __forceinline__ void run(int begin, int end, int g, f32x4 (&acc)[MF][FR]) const {
    Step step[ST];
#pragma unroll
    for (int u = 0; u < ST; ++u) load(step[u], begin + u * KS, end, g);
    for (int k = begin; k < end; k += ST * KS)
#pragma unroll
      for (int u = 0; u < ST; ++u) {
        multiply(step[u], acc);
        load(step[u], k + (ST + u) * KS, end, g);
      }
  }
};

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
