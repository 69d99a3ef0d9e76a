// rows.h — what the operators over rows share: vectors of a row at any
// alignment, and the sum of partial rows.
#ifndef TCA_HIP_ROWS_H_
#define TCA_HIP_ROWS_H_

#include "tca/hip/device.h"

namespace tca {
namespace hip {

template <typename T>
constexpr int kRowE = 16 / static_cast<int>(sizeof(T));  // values per 16-byte vector

// E values of a row from column c on, as f32; zeros past the end. WHOLE: all
// of them lie before it.
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ void row_load(const T* row, uint32_t c, uint32_t C, float (&f)[E]) {
  if (WHOLE || (c < C && C - c >= static_cast<uint32_t>(E))) {
    const vec<T, E> v = load_vec_any<T, E, false>(row + c);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = static_cast<float>(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = c + e < C ? static_cast<float>(row[c + e]) : 0.0f;
  }
}
// ... and back, rounded to nearest once.
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ void row_store(T* row, uint32_t c, uint32_t C, const float (&f)[E]) {
  if (WHOLE || (c < C && C - c >= static_cast<uint32_t>(E))) {
    vec<T, E> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.set(e, static_cast<T>(f[e]));
    store_vec_any<T, E, false>(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + e < C) row[c + e] = static_cast<T>(f[e]);
  }
}

// The same values as they lie in memory, for loads ahead of their use.
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ vec<T, E> row_raw(const T* row, uint32_t c, uint32_t C) {
  if (WHOLE || (c < C && C - c >= static_cast<uint32_t>(E))) return load_vec_any<T, E, false>(row + c);
  vec<T, E> v;
#pragma unroll
  for (int e = 0; e < E; ++e) v.set(e, c + e < C ? row[c + e] : static_cast<T>(0.0f));
  return v;
}

// Partial rows of a sum over R rows: one for each `rows` of them, at most
// `most` (the plan's grid term R/rows:most).
__host__ __device__ __forceinline__ uint32_t partial_rows(uint32_t R, uint32_t rows, uint32_t most) {
  const uint32_t p = R == 0u ? 0u : (R - 1u) / rows + 1u;
  return p < most ? p : most;
}

// out_q[c] = the sum of the P partials of column c, q < Q (out_1 may be null
// with Q = 1): 32 columns by 8 slices of partials a workgroup of 256 lanes,
// the slices joined in order. P = 0 (no rows): zeros.
template <typename W>
__device__ __forceinline__ void join_partials(const float* __restrict__ part, W* __restrict__ out0, W* __restrict__ out1,
                                          uint32_t Q, uint32_t C, uint32_t P) {
  __shared__ float join[8][33];
  const uint32_t blocks = (C - 1u) / 32u + 1u, q = blockIdx.x / blocks, i = threadIdx.x & 31u, slot = threadIdx.x >> 5;
  const uint32_t c = (blockIdx.x - q * blocks) * 32u + i;
  float v = 0.0f;
  if (c < C)
    for (uint32_t p = slot; p < P; p += 8u) v += part[(static_cast<uint64_t>(p) * Q + q) * C + c];
  join[slot][i] = v;
  __syncthreads();
  if (slot != 0u || c >= C) return;
#pragma unroll
  for (int s = 1; s < 8; ++s) v += join[s][i];
  (q == 0u ? out0 : out1)[c] = static_cast<W>(v);
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_ROWS_H_
