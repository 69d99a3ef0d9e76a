// norm.h — layer norm over the last axis and its backward pass (family N).
//
//   forward   m = sum_c x / C,  v = sum_c (x - m)^2 / C,  s = 1 / sqrt(v + eps)
//             y = (x - m) s gamma + beta
//   backward  h = (x - m) s,  t = dy gamma
//             dx = s (t - sum_c t / C - h sum_c (t h) / C)  [+ dres]
//             dgamma = sum_r dy h,  dbeta = sum_r dy
//
// Both are bound by HBM: every operand is read once, every result written
// once. A row is held in registers by a group of G lanes (16, a wave, or 4 or
// 16 waves), NV vectors of 16 bytes a lane, so that the variance is the
// centred sum of squares with no second read; longer rows are read twice
// (norm_long), their mean and variance merged pairwise in the first read. All
// sums are 32-bit. Rows may start at any element: vectors are loaded and
// stored unaligned, and the last, partial vector of a row element by element.
//
// The weights' gradients are sums over rows, so a workgroup walks rows with
// the grid as its stride, sums its rows' terms in registers, joins its groups
// in LDS and writes one partial row; join_partials adds the partial rows, always
// in the same order.
#ifndef TCA_HIP_NORM_H_
#define TCA_HIP_NORM_H_

#include "tca/hip/rows.h"

namespace tca {
namespace hip {

// The sum of v over the G lanes of a group; G > 64: over the G / 64 waves of
// it too, through `lds` (one slot per wave of the workgroup). `lds` must not
// be written again before a barrier: callers alternate between two.
template <int G>
__device__ __forceinline__ float norm_group_sum(float v, float* lds) {
  v = seg_allreduce<(G < 64 ? G : 64)>(v, [](float a, float b) { return a + b; });
  if constexpr (G > 64) {
    constexpr uint32_t kWaves = G / 64;
    if (lane_id() == 0u) lds[wave_id()] = v;
    __syncthreads();
    const float* g = lds + wave_id() / kWaves * kWaves;
    v = g[0];
#pragma unroll
    for (uint32_t i = 1; i < kWaves; ++i) v += g[i];
  }
  return v;
}

// One row per group of G lanes, at most NV vectors per lane (C <= G NV E).
template <typename T, typename W, int G, int NV, bool BIAS, bool STATS>
__device__ __forceinline__ void norm_rows(const T* x, const W* __restrict__ gamma, const W* __restrict__ beta, T* y,
                                          float* __restrict__ mean, float* __restrict__ rstd, uint32_t R, uint32_t C,
                                          float eps) {
  constexpr int E = kRowE<T>, BLOCK = G < 256 ? 256 : G;
  __shared__ float lds[2][BLOCK / 64];
  const uint32_t lane = threadIdx.x % G, row = blockIdx.x * (BLOCK / G) + threadIdx.x / G;
  const bool live = row < R;
  const uint64_t at = static_cast<uint64_t>(live ? row : 0u) * C;
  float v[NV][E];
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    row_load<E>(x + at, (i * G + lane) * E, C, v[i]);
#pragma unroll
    for (int e = 0; e < E; ++e) s += v[i][e];
  }
  const float m = norm_group_sum<G>(s, lds[0]) / static_cast<float>(C);
  float q = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[i][e] -= m;
      if ((i * G + lane) * E + e < C) q = __builtin_fmaf(v[i][e], v[i][e], q);
    }
  const float r = 1.0f / __builtin_sqrtf(norm_group_sum<G>(q, lds[1]) / static_cast<float>(C) + eps);
  if (!live) return;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (i * G + lane) * E;
    float g[E], b[E];
    row_load<E>(gamma, c, C, g);
    if constexpr (BIAS) row_load<E>(beta, c, C, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[i][e] = v[i][e] * r * g[e];
      if constexpr (BIAS) v[i][e] += b[e];
    }
    row_store<E>(y + at, c, C, v[i]);
  }
  if constexpr (STATS) {
    if (lane == 0u) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

// (s, m2, n) of the whole workgroup of WAVES waves, in every lane.
template <int WAVES>
__device__ __forceinline__ void norm_merge_block(float& s, float& m2, float& n, float (*lds)[3]) {
  for (int off = 1; off < 64; off <<= 1)
    chan_merge_present(s, m2, n, xor_lanes(s, off), xor_lanes(m2, off), xor_lanes(n, off));
  if (lane_id() == 0u) {
    lds[wave_id()][0] = s;
    lds[wave_id()][1] = m2;
    lds[wave_id()][2] = n;
  }
  __syncthreads();
  s = lds[0][0];
  m2 = lds[0][1];
  n = lds[0][2];
  for (int w = 1; w < WAVES; ++w) chan_merge_present(s, m2, n, lds[w][0], lds[w][1], lds[w][2]);
}

// Rows longer than the registers of a workgroup hold: one per workgroup of
// 1024 lanes, read once for the mean and the centred sum of squares (whole
// vectors merged pairwise) and once more for the map.
template <typename T, typename W, bool BIAS, bool STATS>
__device__ __forceinline__ void norm_long(const T* x, const W* __restrict__ gamma, const W* __restrict__ beta, T* y,
                                          float* __restrict__ mean, float* __restrict__ rstd, uint32_t R, uint32_t C,
                                          float eps) {
  constexpr int E = kRowE<T>;
  __shared__ float lds[16][3];
  const uint32_t row = blockIdx.x;
  if (row >= R) return;
  const T* xr = x + static_cast<uint64_t>(row) * C;
  T* yr = y + static_cast<uint64_t>(row) * C;
  const uint32_t whole = C / E * E;
  float s = 0.0f, m2 = 0.0f, n = 0.0f;
  for (uint32_t c = threadIdx.x * E; c < whole; c += 1024u * E) {
    float v[E];
    row_load<E>(xr, c, C, v);
    chan_add<E>(s, m2, n, v);
  }
  if (whole + threadIdx.x < C) chan_merge_present(s, m2, n, static_cast<float>(xr[whole + threadIdx.x]), 0.0f, 1.0f);
  norm_merge_block<16>(s, m2, n, lds);
  const float m = s / static_cast<float>(C), r = 1.0f / __builtin_sqrtf(m2 / static_cast<float>(C) + eps);
  for (uint32_t c = threadIdx.x * E; c < C; c += 1024u * E) {
    float v[E], g[E], b[E];
    row_load<E>(xr, c, C, v);
    row_load<E>(gamma, c, C, g);
    if constexpr (BIAS) row_load<E>(beta, c, C, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = (v[e] - m) * r * g[e];
      if constexpr (BIAS) v[e] += b[e];
    }
    row_store<E>(yr, c, C, v);
  }
  if constexpr (STATS) {
    if (threadIdx.x == 0u) {
      mean[row] = m;
      rstd[row] = r;
    }
  }
}

// ------------------------------------------------------------- backward pass

// Workgroups of 1024 lanes, 1024 / G groups; `part` is [workgroups][1 + BIAS][C].
template <typename T, typename W, int G, int NV, bool BIAS, bool RES>
__device__ __forceinline__ void norm_backward_rows(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const W* __restrict__ gamma, const float* __restrict__ mean,
                                                   const float* __restrict__ rstd, const T* dres, T* dx,
                                                   float* __restrict__ part, uint32_t R, uint32_t C) {
  constexpr int E = kRowE<T>, BLOCK = 1024, GROUPS = BLOCK / G;
  constexpr uint32_t SPAN = G * NV * E;
  __shared__ float sums[2][2][BLOCK / 64];
  __shared__ __attribute__((aligned(16))) float join[GROUPS * SPAN];
  const uint32_t lane = threadIdx.x % G, grp = threadIdx.x / G;
  const float inv = 1.0f / static_cast<float>(C);
  float dg[NV][E], db[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dg[i][e] = db[i][e] = 0.0f;
  uint32_t turn = 0u;
  // r0 < R is the same for every group: all of them reach the barriers.
  for (uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * GROUPS; r0 < R; r0 += static_cast<uint64_t>(gridDim.x) * GROUPS) {
    const uint64_t row = r0 + grp;
    const bool live = row < R;
    const uint64_t at = live ? row * C : 0u;
    const float m = live ? mean[row] : 0.0f, rs = live ? rstd[row] : 0.0f;
    float h[NV][E], t[NV][E];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (i * G + lane) * E;
      float g[E];
      row_load<E>(x + at, c, C, h[i]);
      row_load<E>(dy + at, c, C, t[i]);
      row_load<E>(gamma, c, C, g);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[i][e] = (h[i][e] - m) * rs;
        if (live) {  // a group past the last row adds nothing, whatever row 0 holds
          dg[i][e] = __builtin_fmaf(t[i][e], h[i][e], dg[i][e]);
          db[i][e] += t[i][e];
        }
        t[i][e] *= g[e];
        s1 += t[i][e];
        if (c + e < C) s2 = __builtin_fmaf(t[i][e], h[i][e], s2);
      }
    }
    s1 = norm_group_sum<G>(s1, sums[turn & 1u][0]);
    s2 = norm_group_sum<G>(s2, sums[turn & 1u][1]);
    ++turn;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (i * G + lane) * E;
      float o[E];
      if constexpr (RES) row_load<E>(dres + at, c, C, o);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = (t[i][e] - (s1 + h[i][e] * s2) * inv) * rs;
        o[e] = RES ? d + o[e] : d;
      }
      row_store<E>(dx + at, c, C, o);
    }
  }
  // The groups' sums, in group order.
  float* to = part + static_cast<uint64_t>(blockIdx.x) * (BIAS ? 2u : 1u) * C;
#pragma unroll
  for (int q = 0; q < (BIAS ? 2 : 1); ++q) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) join[grp * SPAN + (i * G + lane) * E + e] = q == 0 ? dg[i][e] : db[i][e];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < C && c < SPAN; c += BLOCK) {
      float v = join[c];
#pragma unroll
      for (int g = 1; g < GROUPS; ++g) v += join[g * SPAN + c];
      to[static_cast<uint64_t>(q) * C + c] = v;
    }
  }
}

// dx of rows longer than norm_backward_rows takes, one per workgroup of 1024
// lanes: the two sums in one read, the map in a second.
template <typename T, typename W, bool RES>
__device__ __forceinline__ void norm_backward_long(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const W* __restrict__ gamma, const float* __restrict__ mean,
                                                   const float* __restrict__ rstd, const T* dres, T* dx, uint32_t R,
                                                   uint32_t C) {
  constexpr int E = kRowE<T>;
  __shared__ float sums[2][16];
  const uint32_t row = blockIdx.x;
  if (row >= R) return;
  const uint64_t at = static_cast<uint64_t>(row) * C;
  const float m = mean[row], rs = rstd[row], inv = 1.0f / static_cast<float>(C);
  float s1 = 0.0f, s2 = 0.0f;
  for (uint32_t c = threadIdx.x * E; c < C; c += 1024u * E) {
    float h[E], t[E], g[E];
    row_load<E>(x + at, c, C, h);
    row_load<E>(dy + at, c, C, t);
    row_load<E>(gamma, c, C, g);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s1 = __builtin_fmaf(t[e], g[e], s1);
      if (c + e < C) s2 = __builtin_fmaf(t[e] * g[e], (h[e] - m) * rs, s2);
    }
  }
  s1 = norm_group_sum<1024>(s1, sums[0]);
  s2 = norm_group_sum<1024>(s2, sums[1]);
  for (uint32_t c = threadIdx.x * E; c < C; c += 1024u * E) {
    float h[E], t[E], g[E], o[E];
    row_load<E>(x + at, c, C, h);
    row_load<E>(dy + at, c, C, t);
    row_load<E>(gamma, c, C, g);
    if constexpr (RES) row_load<E>(dres + at, c, C, o);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = (t[e] * g[e] - (s1 + (h[e] - m) * rs * s2) * inv) * rs;
      o[e] = RES ? d + o[e] : d;
    }
    row_store<E>(dx + at, c, C, o);
  }
}

// The weights' gradients of those rows: 64 vectors of columns by 4 rows a
// workgroup of 256 lanes, over row chunk p of P; `part` is [P][1 + BIAS][C].
template <typename T, bool BIAS>
__device__ __forceinline__ void norm_backward_columns(const T* __restrict__ dy, const T* __restrict__ x,
                                                      const float* __restrict__ mean, const float* __restrict__ rstd,
                                                      float* __restrict__ part, uint32_t R, uint32_t C, uint32_t P) {
  constexpr int E = kRowE<T>;
  __shared__ float join[4][64 * E];
  const uint32_t p = blockIdx.x % P, c = (blockIdx.x / P * 64u + lane_id()) * E, slot = wave_id();
  const uint64_t rows = (R - 1u) / P + 1u, first = p * rows, last = first + rows < R ? first + rows : R;
  float dg[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dg[e] = db[e] = 0.0f;
  for (uint64_t r = first + slot; r < last; r += 4u) {
    const float m = mean[r], rs = rstd[r];
    float h[E], t[E];
    row_load<E>(x + r * C, c, C, h);
    row_load<E>(dy + r * C, c, C, t);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dg[e] = __builtin_fmaf(t[e], (h[e] - m) * rs, dg[e]);
      db[e] += t[e];
    }
  }
  float* to = part + static_cast<uint64_t>(p) * (BIAS ? 2u : 1u) * C;
#pragma unroll
  for (int q = 0; q < (BIAS ? 2 : 1); ++q) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) join[slot][lane_id() * E + e] = q == 0 ? dg[e] : db[e];
    __syncthreads();
    const uint32_t c0 = blockIdx.x / P * 64u * E;
    for (uint32_t i = threadIdx.x; i < 64u * E && c0 + i < C; i += 256u)
      to[static_cast<uint64_t>(q) * C + c0 + i] = ((join[0][i] + join[1][i]) + join[2][i]) + join[3][i];
  }
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_NORM_H_
