// rows.h — what the operators over rows share: vectors of a row at any
// alignment, and the sum of partial rows.
#ifndef TCA_HIP_ROWS_H_
#define TCA_HIP_ROWS_H_

#include "tca/hip/device.h"

namespace tca {
namespace hip {

template <typename T>
constexpr int kRowE = 16 / static_cast<int>(sizeof(T));  // values per 16-byte vector

// E values of a row of C from column c on, as they lie in memory: 16 bytes a
// load, unaligned, with no test of a lane's own. A piece that would run past
// the end of the row is loaded from the end's last 16 bytes instead and is
// moved into place by row_fix, which waits for it and so is called where the
// values are used. Rows of less than 16 bytes are gathered. WHOLE: all of the
// values lie in the row. NT: not kept in the caches.
template <typename T>
__device__ __forceinline__ uint32_t row_at(uint32_t c, uint32_t C) {
  const uint32_t last = C >= static_cast<uint32_t>(kRowE<T>) ? C - kRowE<T> : 0u;
  return c < last ? c : last;
}
template <int E, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ vec<T, E> row_raw(const T* row, uint32_t c, uint32_t C) {
  constexpr int P = kRowE<T>;
  static_assert(E % P == 0, "whole pieces");
  struct {
    vec<T, P> piece[E / P];
  } r;
#pragma unroll
  for (int k = 0; k < E / P; ++k) {
    if (WHOLE || C >= static_cast<uint32_t>(P)) {
      r.piece[k] = load_vec_any<T, P, NT>(row + (WHOLE ? c + k * P : row_at<T>(c + k * P, C)));
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) r.piece[k].set(e, static_cast<uint32_t>(e) < C ? row[e] : static_cast<T>(0.0f));
    }
  }
  return __builtin_bit_cast(vec<T, E>, r);
}
// The values of row_raw moved down to their places, zeros past the end.
template <int E, typename T>
__device__ __forceinline__ void row_fix(vec<T, E>& v, uint32_t c, uint32_t C) {
  constexpr int P = kRowE<T>;
  struct Words {
    uint32_t w[E / P][4];
  };
  Words x = __builtin_bit_cast(Words, v);
#pragma unroll
  for (int k = 0; k < E / P; ++k) {
    const uint32_t n = c + k * P - row_at<T>(c + k * P, C);  // places
    if (n == 0u) continue;
    uint32_t(&w)[4] = x.w[k];
    const uint32_t words = sizeof(T) == 2 ? n >> 1 : n;
    if (words & 1u) {
      w[0] = w[1];
      w[1] = w[2];
      w[2] = w[3];
      w[3] = 0u;
    }
    if (words & 2u) {
      w[0] = w[2];
      w[1] = w[3];
      w[2] = w[3] = 0u;
    }
    if (words >= 4u) w[0] = w[1] = w[2] = w[3] = 0u;
    if (sizeof(T) == 2 && (n & 1u)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (w[i] >> 16) | (i < 3 ? w[i + 1] << 16 : 0u);
    }
  }
  v = __builtin_bit_cast(vec<T, E>, x);
}
// Both at once.
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ vec<T, E> row_vec(const T* row, uint32_t c, uint32_t C) {
  vec<T, E> v = row_raw<E, WHOLE>(row, c, C);
  if constexpr (!WHOLE) row_fix<E>(v, c, C);
  return v;
}
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ void row_load(const T* row, uint32_t c, uint32_t C, float (&f)[E]) {
  const vec<T, E> v = row_vec<E, WHOLE>(row, c, C);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = static_cast<float>(v[e]);
}
// ... and back, rounded to nearest once.
template <int E, bool WHOLE = false, bool NT = false, typename T>
__device__ __forceinline__ void row_store(T* row, uint32_t c, uint32_t C, const float (&f)[E]) {
  if (WHOLE || (c < C && C - c >= static_cast<uint32_t>(E))) {
    vec<T, E> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.set(e, static_cast<T>(f[e]));
    store_vec_any<T, E, NT>(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < C) row[c + e] = static_cast<T>(f[e]);
  }
}

// Partial rows of a sum over R rows: one for each `rows` of them, at most
// `most` (the plan's grid term R/rows:most).
__host__ __device__ __forceinline__ uint32_t partial_rows(uint32_t R, uint32_t rows, uint32_t most) {
  const uint32_t p = R == 0u ? 0u : (R - 1u) / rows + 1u;
  return p < most ? p : most;
}

// out_q[c] = the sum of the P partials of column c, q < Q (out_1 may be null
// with Q = 1): 32 columns by 32 slices of partials a workgroup of 1024 lanes,
// eight partials of a lane in flight (past the end, the last one again), the
// slices joined in order. P = 0 (no rows): zeros.
template <typename W>
__device__ __forceinline__ void join_partials(const float* __restrict__ part, W* __restrict__ out0, W* __restrict__ out1,
                                              uint32_t Q, uint32_t C, uint32_t P) {
  __shared__ float join[32][33];
  const uint32_t blocks = (C - 1u) / 32u + 1u, q = blockIdx.x / blocks, i = threadIdx.x & 31u, slot = threadIdx.x >> 5;
  const uint32_t c = (blockIdx.x - q * blocks) * 32u + i;
  float v = 0.0f;
  if (c < C)
    for (uint32_t p = slot; p < P; p += 256u) {
      float s[8];
#pragma unroll
      for (uint32_t k = 0; k < 8u; ++k) {
        const uint32_t r = p + 32u * k < P ? p + 32u * k : P - 1u;
        s[k] = part[(static_cast<uint64_t>(r) * Q + q) * C + c];
      }
#pragma unroll
      for (uint32_t k = 0; k < 8u; ++k) v = p + 32u * k < P ? v + s[k] : v;
    }
  join[slot][i] = v;
  __syncthreads();
  if (slot != 0u || c >= C) return;
#pragma unroll
  for (int s = 1; s < 32; ++s) v += join[s][i];
  (q == 0u ? out0 : out1)[c] = static_cast<W>(v);
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_ROWS_H_
