// norm.h — layer norm over the last axis and its backward pass (family N).
//
//   forward   m = sum_c x / C,  v = sum_c (x - m)^2 / C,  s = 1 / sqrt(v + eps)
//             y = (x - m) s gamma + beta
//   backward  h = (x - m) s,  t = dy gamma
//             dx = s (t - sum_c t / C - h sum_c (t h) / C)  [+ dres]
//             dgamma = sum_r dy h,  dbeta = sum_r dy
//
// The maps are chains of fused multiply-adds, so that a result is few roundings
// away from its sums (-0 where there is nothing to add: it leaves -0 as it is).
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
//
// Measured: forward f32 [32768, 1024] with the statistics 46 to 48 us (268 MB, 5.6 to
// 5.8 TB/s), bf16 [16384, 4096] 51, f16 [3000, 8000] 24, [1618, 16880] 29; backward
// bf16 [8192, 4096] with a residual 43 to 45 us (268 MB, 6.0 TB/s) and 4 to 5 for
// the join. Streaming stores (forward) and loads (backward) took 5 and 8% off,
// loads a row ahead and joins of 1024 lanes 10 and 30%.
#ifndef TCA_HIP_NORM_H_
#define TCA_HIP_NORM_H_

#include "tca/hip/rows.h"

namespace tca {
namespace hip {

// The sums of v[0] .. v[S - 1] over the G lanes of a group; G > 64: over the G /
// 64 waves of it too, through `lds` (S floats for each wave of the workgroup).
// `lds` must not be written again before a barrier: callers alternate
// between two.
template <int G, int S>
__device__ __forceinline__ void norm_group_sums(float (&v)[S], float* lds) {
#pragma unroll
  for (int i = 0; i < S; ++i) v[i] = seg_allreduce<(G < 64 ? G : 64)>(v[i], [](float a, float b) { return a + b; });
  if constexpr (G > 64) {
    constexpr uint32_t kWaves = G / 64;
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (lane_id() == 0u) lds[wave_id() * S + i] = v[i];
    __syncthreads();
    const float* g = lds + wave_id() / kWaves * kWaves * S;
#pragma unroll
    for (int i = 0; i < S; ++i) {
      v[i] = g[i];
#pragma unroll
      for (uint32_t k = 1; k < kWaves; ++k) v[i] += g[k * S + i];
    }
  }
}

// What vector i of a wave's lanes, of groups of G, holds of rows of C: nothing,
// part of its places, or all. The same for every lane of the wave.
enum { kNormNone, kNormPart, kNormAll };
template <int G, int E>
__device__ __forceinline__ int norm_holds(int i, uint32_t C) {
  const uint32_t wave = G > 64 ? static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) % (G > 64 ? G / 64 : 1) : 0u;
  const uint32_t first = (i * G + wave * 64u) * E, span = (G < 64 ? G : 64) * E;
  return first >= C ? kNormNone : C - first < span ? kNormPart : kNormAll;
}

// Rows by groups of G lanes, at most NV vectors per lane (C <= G NV E), the
// workgroups walking them with the grid as their stride: a row's loads are
// issued a row ahead, and gamma and beta are read once (in rows of 32 16-bit
// values a lane again for every row, out of the L2: registers for both spill).
template <typename T, typename W, int G, int NV, bool BIAS, bool STATS>
__device__ __forceinline__ void norm_rows(const T* x, const W* __restrict__ gamma, const W* __restrict__ beta, T* y,
                                          float* __restrict__ mean, float* __restrict__ rstd, uint32_t R, uint32_t C,
                                          float eps) {
  constexpr int E = kRowE<T>, BLOCK = G < 256 ? 256 : G, GROUPS = BLOCK / G;
  constexpr bool HELD = BLOCK < 1024 || NV * E < 32;
  __shared__ float lds[2][2][BLOCK / 64];
  const uint32_t lane = threadIdx.x % G;
  uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * GROUPS;  // the workgroup's first row
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * GROUPS, grp = threadIdx.x / G;
  vec<T, E> next[NV];
  vec<W, E> g[NV], b[NV];
  int holds[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) holds[i] = norm_holds<G, E>(i, C);
  auto load = [&](uint64_t row) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (holds[i] != kNormNone) next[i] = row_raw<E>(x + row * C, (i * G + lane) * E, C);
  };
  auto weights = [&](int i) {
    g[i] = row_vec<E>(gamma, (i * G + lane) * E, C);
    if constexpr (BIAS) b[i] = row_vec<E>(beta, (i * G + lane) * E, C);
  };
  if (r0 + grp < R) load(r0 + grp);
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < NV; ++i) weights(i);
  }
  // r0 is the same for every group: all of them reach the barriers.
  for (uint32_t turn = 0u; r0 < R; r0 += step, ++turn) {
    const uint64_t row = r0 + grp;
    float v[NV][E];
    float s[1] = {0.0f}, q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (holds[i] == kNormPart) row_fix<E>(next[i], (i * G + lane) * E, C);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] = static_cast<float>(next[i][e]);
    }
    if (row + step < R) load(row + step);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (holds[i] != kNormNone) {
#pragma unroll
        for (int e = 0; e < E; ++e) s[0] += v[i][e];
      }
    norm_group_sums<G>(s, lds[turn & 1u][0]);
    const float m = s[0] / static_cast<float>(C);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (holds[i] == kNormNone) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] -= m;
      if (holds[i] == kNormPart) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if ((i * G + lane) * E + e >= C) v[i][e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) q[0] = __builtin_fmaf(v[i][e], v[i][e], q[0]);
    }
    norm_group_sums<G>(q, lds[turn & 1u][1]);
    const float r = 1.0f / __builtin_sqrtf(q[0] / static_cast<float>(C) + eps);
    if (row >= R) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (holds[i] == kNormNone) continue;
      if constexpr (!HELD) weights(i);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[i][e] = __builtin_fmaf(v[i][e] * r, static_cast<float>(g[i][e]), BIAS ? static_cast<float>(b[i][e]) : -0.0f);
      }
      if (holds[i] == kNormAll) row_store<E, true, true>(y + row * C, (i * G + lane) * E, C, v[i]);
      else row_store<E, false, true>(y + row * C, (i * G + lane) * E, C, v[i]);
    }
    if constexpr (STATS) {
      if (lane == 0u) {
        mean[row] = m;
        rstd[row] = r;
      }
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
      v[e] = __builtin_fmaf((v[e] - m) * r, g[e], BIAS ? b[e] : -0.0f);
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

// Workgroups of 512 lanes, 512 / G groups, walking the rows with the grid as
// their stride, a row's loads issued a row ahead; `part` is [workgroups][1 + BIAS][C].
template <typename T, typename W, int G, int NV, bool BIAS, bool RES>
__device__ __forceinline__ void norm_backward_rows(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const W* __restrict__ gamma, const float* __restrict__ mean,
                                                   const float* __restrict__ rstd, const T* dres, T* dx,
                                                   float* __restrict__ part, uint32_t R, uint32_t C) {
  constexpr int E = kRowE<T>, BLOCK = 512, GROUPS = BLOCK / G;
  constexpr uint32_t SPAN = G * NV * E;
  __shared__ float sums[2][2 * BLOCK / 64];
  __shared__ __attribute__((aligned(16))) float join[GROUPS * SPAN];
  const uint32_t lane = threadIdx.x % G, grp = threadIdx.x / G;
  const float inv = 1.0f / static_cast<float>(C);
  struct Row {
    vec<T, E> x[NV], dy[NV], res[RES ? NV : 1];
    float m, rs;
  };
  uint64_t r0 = static_cast<uint64_t>(blockIdx.x) * GROUPS;
  const uint64_t step = static_cast<uint64_t>(gridDim.x) * GROUPS;
  int holds[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) holds[i] = norm_holds<G, E>(i, C);
  auto load = [&](Row& w, uint64_t row) {
    w.m = mean[row];
    w.rs = rstd[row];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (i * G + lane) * E;
      if (holds[i] == kNormNone) continue;
      w.x[i] = row_raw<E, false, true>(x + row * C, c, C);
      w.dy[i] = row_raw<E, false, true>(dy + row * C, c, C);
      // dres may be dx: this row's elements are written by the lanes that read them.
      if constexpr (RES) w.res[i] = row_raw<E, false, true>(dres + row * C, c, C);
    }
  };
  Row next;
  if (r0 + grp < R) load(next, r0 + grp);
  vec<W, E> g[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) g[i] = row_vec<E>(gamma, (i * G + lane) * E, C);
  float dg[NV][E], db[NV][E];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dg[i][e] = db[i][e] = 0.0f;
  // r0 is the same for every group: all of them reach the barriers.
  for (uint32_t turn = 0u; r0 < R; r0 += step, ++turn) {
    const uint64_t row = r0 + grp;
    const bool live = row < R;
    Row now = next;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (i * G + lane) * E;
      if (holds[i] != kNormPart) continue;
      row_fix<E>(now.x[i], c, C);
      row_fix<E>(now.dy[i], c, C);
      if constexpr (RES) row_fix<E>(now.res[i], c, C);
    }
    if (row + step < R) load(next, row + step);
    float s[2] = {0.0f, 0.0f};
    if (live) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (holds[i] == kNormNone) continue;
#pragma unroll
        for (int e = 0; e < E; ++e) {  // (past the end of the row dy is 0, and so are t and t h)
          const float h = (static_cast<float>(now.x[i][e]) - now.m) * now.rs, d = static_cast<float>(now.dy[i][e]);
          dg[i][e] = __builtin_fmaf(d, h, dg[i][e]);
          db[i][e] += d;
          const float t = d * static_cast<float>(g[i][e]);
          s[0] += t;
          s[1] = __builtin_fmaf(t, h, s[1]);
        }
      }
    }
    norm_group_sums<G>(s, sums[turn & 1u]);
    if (!live) continue;
    const float mt = s[0] * inv, mth = s[1] * inv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (holds[i] == kNormNone) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float h = (static_cast<float>(now.x[i][e]) - now.m) * now.rs;
        const float t = __builtin_fmaf(static_cast<float>(now.dy[i][e]), static_cast<float>(g[i][e]), -mt);
        o[e] = __builtin_fmaf(__builtin_fmaf(-h, mth, t), now.rs, RES ? static_cast<float>(now.res[i][e]) : -0.0f);
      }
      if (holds[i] == kNormAll) row_store<E, true>(dx + row * C, (i * G + lane) * E, C, o);
      else row_store<E>(dx + row * C, (i * G + lane) * E, C, o);
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
// lanes: the two sums in one read, the map in a second. (f16 [1901, 24912] with a
// residual 88 us, and 38 for the columns' pass over the same rows.)
template <typename T, typename W, bool RES>
__device__ __forceinline__ void norm_backward_long(const T* __restrict__ dy, const T* __restrict__ x,
                                                   const W* __restrict__ gamma, const float* __restrict__ mean,
                                                   const float* __restrict__ rstd, const T* dres, T* dx, uint32_t R,
                                                   uint32_t C) {
  constexpr int E = kRowE<T>;
  __shared__ float sums[2 * 16];
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
  float both[2] = {s1, s2};
  norm_group_sums<1024>(both, sums);
  s1 = both[0] * inv;
  s2 = both[1] * inv;
  for (uint32_t c = threadIdx.x * E; c < C; c += 1024u * E) {
    float h[E], t[E], g[E], o[E];
    row_load<E>(x + at, c, C, h);
    row_load<E>(dy + at, c, C, t);
    row_load<E>(gamma, c, C, g);
    if constexpr (RES) row_load<E>(dres + at, c, C, o);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = __builtin_fmaf(-(h[e] - m) * rs, s2, __builtin_fmaf(t[e], g[e], -s1));
      o[e] = __builtin_fmaf(d, rs, RES ? o[e] : -0.0f);
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
