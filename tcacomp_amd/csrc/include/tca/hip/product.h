// product.h — 16-bit matrix products of a dense sublayer (family P): a
// projection with bias, activation and residual in its epilogue, two
// projections whose results meet in the epilogue (gated), and the gradients
// of both.
//
//   C[m, n] = sum_k A[m, k] B[k, n], 32-bit sums on the matrix cores
//   (v_mfma_f32_16x16x32), rounded once when the epilogue stores
//
// An operand is K-contiguous (rows of k, as x [M][K] in a forward product) or
// row-contiguous (rows of its own index, as a weight [K][N]; as x and dz in
// dW = x^T dz, whose reduction runs over their rows). The B side of a tile has
// two halves. In a plain product they are neighbouring columns of one matrix;
// in a pair (PAIR) the same columns of two matrices, so that a lane holds both
// products of an output element and the epilogue combines them. A product
// may run over two segments of k (SEGS), each with its own pair of operands:
// dx = dg Wg^T + du Wu^T is one chain of sums.
#ifndef TCA_HIP_PRODUCT_H_
#define TCA_HIP_PRODUCT_H_

#include "tca/hip/gemm.h"
#include "tca/hip/rows.h"

namespace tca {
namespace hip {

// ----------------------------------------------------------- activations
// Results are rounded to 16 bits by every caller, so the hardware's exp2 and
// reciprocal (1 ulp each) stand in for the rounded ones.
enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4 };

__device__ __forceinline__ float act_sigmoid(float z) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}
// The tail Q(x) = 1 - Phi(x) of the normal distribution over e = exp(-x^2 / 2),
// x >= 0: t P(t), t = 1 / (1 + 0.36 x), P of degree 6 fitted to erfcx(x /
// sqrt 2) / 2 over x <= 13.5 by reweighted least squares, 8e-7 off relative to
// the value. No branches: erfcf has some, and a lane's eight columns wait for each
// other at them (linear 4096^3 with gelu took 16 us more than without, now none
// that a run's noise of 2 us shows).
__device__ __forceinline__ float act_tail(float x) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.36f, x, 1.0f));
  float p = __builtin_fmaf(0.04734482616186142f, t, -0.18075250089168549f);
  p = __builtin_fmaf(p, t, 0.1822986900806427f);
  p = __builtin_fmaf(p, t, 0.02562311850488186f);
  p = __builtin_fmaf(p, t, 0.14005766808986664f);
  p = __builtin_fmaf(p, t, 0.14171062409877777f);
  p = __builtin_fmaf(p, t, 0.1437174379825592f);
  return p * t;
}
// exp(-x^2 / 2); 0 from x = 14 on, where callers hold x.
__device__ __forceinline__ float act_bell(float x) { return __builtin_amdgcn_exp2f(-0.72134752044448170f * x * x); }
__device__ __forceinline__ float act_far(float z) { return __builtin_fminf(__builtin_fabsf(z), 14.0f); }

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == kActRelu) return z < 0.0f ? 0.0f : z;
  else if constexpr (ACT == kActSilu) return z * act_sigmoid(z);
  else if constexpr (ACT == kActGelu) {  // z Phi(z) = max(z, 0) - |z| Q(|z|)
    const float x = act_far(z);
    return (z < 0.0f ? 0.0f : z) - x * (act_tail(x) * act_bell(x));
  } else if constexpr (ACT == kActGeluTanh)  // 1 + tanh(u) = 2 sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3)
    return z * act_sigmoid(1.59576912160573071f * z * __builtin_fmaf(0.044715f * z, z, 1.0f));
  else return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == kActRelu) {
    return z <= 0.0f ? 0.0f : 1.0f;
  } else if constexpr (ACT == kActSilu) {
    const float s = act_sigmoid(z);
    return s * __builtin_fmaf(z, 1.0f - s, 1.0f);
  } else if constexpr (ACT == kActGelu) {
    const float x = act_far(z), e = act_bell(x), q = act_tail(x) * e;
    const float d = 0.39894228040143268f * (x * e);  // |z| phi(z)
    return z < 0.0f ? q - d : z == z ? (1.0f - q) + d : z;
  } else if constexpr (ACT == kActGeluTanh) {
    // Held where s is 0 or 1 exactly: z^3 would pass the range, and 0 times that.
    const float x = __builtin_fminf(__builtin_fmaxf(z, -32.0f), 32.0f);
    const float s = act_sigmoid(1.59576912160573071f * x * __builtin_fmaf(0.044715f * x, x, 1.0f));
    const float du = 1.59576912160573071f * __builtin_fmaf(3.0f * 0.044715f * x, x, 1.0f);
    return z == z ? s * __builtin_fmaf(x * du, 1.0f - s, 1.0f) : z;
  } else {
    return 1.0f;
  }
}

// ------------------------------------------------------------- epilogues
// Each takes eight consecutive columns n .. n + 7 of row m < M, n < N, and
// stores those before N (WHOLE: all of them); fetch() loads what it reads of
// memory, ahead of the call.
struct NoFetch {};

// y = res + act(z), z = v + b [z stored too]. res may be y: an element is
// read by the lane that then writes it.
template <typename T, int ACT, bool BIAS, bool RES, bool SAVE>
struct LinearStore {
  const T* b;
  const T* res;
  T* y;
  T* z;
  uint32_t N;
  struct Fetch {
    vec<T, 8> res, b;
  };
  template <bool WHOLE>
  __device__ __forceinline__ Fetch fetch(uint32_t m, uint32_t n) const {
    Fetch f;
    if constexpr (RES) f.res = row_vec<8, WHOLE>(res + static_cast<uint64_t>(m) * N, n, N);
    if constexpr (BIAS) f.b = row_vec<8, WHOLE>(b, n, N);
    return f;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(uint32_t m, uint32_t n, const Fetch& f, float (&v)[8]) const {
    const uint64_t row = static_cast<uint64_t>(m) * N;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if constexpr (BIAS) v[e] += static_cast<float>(f.b[e]);
    if constexpr (SAVE) row_store<8, WHOLE>(z + row, n, N, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = act<ACT>(v[e]);
      if constexpr (RES) v[e] += static_cast<float>(f.res[e]);
    }
    row_store<8, WHOLE>(y + row, n, N, v);
  }
};
// h = act(g) u, g = v0 + bg, u = v1 + bu [g and u stored too].
template <typename T, int ACT, bool BIAS, bool SAVE>
struct GatedStore {
  const T* bg;
  const T* bu;
  T* h;
  T* g;
  T* u;
  uint32_t N;
  struct Fetch {
    vec<T, 8> bg, bu;
  };
  template <bool WHOLE>
  __device__ __forceinline__ Fetch fetch(uint32_t, uint32_t n) const {
    Fetch f;
    if constexpr (BIAS) {
      f.bg = row_vec<8, WHOLE>(bg, n, N);
      f.bu = row_vec<8, WHOLE>(bu, n, N);
    }
    return f;
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(uint32_t m, uint32_t n, const Fetch& f, float (&v0)[8], float (&v1)[8]) const {
    const uint64_t row = static_cast<uint64_t>(m) * N;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if constexpr (BIAS) {
        v0[e] += static_cast<float>(f.bg[e]);
        v1[e] += static_cast<float>(f.bu[e]);
      }
    if constexpr (SAVE) {
      row_store<8, WHOLE>(g + row, n, N, v0);
      row_store<8, WHOLE>(u + row, n, N, v1);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v0[e] = act<ACT>(v0[e]) * v1[e];
    row_store<8, WHOLE>(h + row, n, N, v0);
  }
};
// The results themselves: of one product, or of a pair.
template <typename T>
struct PlainStore {
  T* c;
  T* c1;
  uint32_t N;
  using Fetch = NoFetch;
  template <bool WHOLE>
  __device__ __forceinline__ Fetch fetch(uint32_t, uint32_t) const {
    return {};
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(uint32_t m, uint32_t n, const Fetch&, float (&v)[8]) const {
    row_store<8, WHOLE>(c + static_cast<uint64_t>(m) * N, n, N, v);
  }
  template <bool WHOLE>
  __device__ __forceinline__ void store(uint32_t m, uint32_t n, const Fetch&, float (&v0)[8], float (&v1)[8]) const {
    row_store<8, WHOLE>(c + static_cast<uint64_t>(m) * N, n, N, v0);
    row_store<8, WHOLE>(c1 + static_cast<uint64_t>(m) * N, n, N, v1);
  }
};

// The epilogue of a product whose k is split over P workgroups: P == 1 the
// product's own, otherwise the partial sums of chunk c as rows of f32
// (`part` is [P][1 or 2][M][N]; join_parts adds them in order).
template <typename Epi>
struct SplitStore {
  const Epi& epi;
  PlainStore<float> part;
  bool direct;
  using Fetch = typename Epi::Fetch;
  template <bool WHOLE>
  __device__ __forceinline__ Fetch fetch(uint32_t m, uint32_t n) const {
    return direct ? epi.template fetch<WHOLE>(m, n) : Fetch{};
  }
  template <bool WHOLE, typename... V>
  __device__ __forceinline__ void store(uint32_t m, uint32_t n, const Fetch& f, V&... v) const {
    if (direct) epi.template store<WHOLE>(m, n, f, v...);
    else part.template store<WHOLE>(m, n, NoFetch{}, v...);
  }
};
template <bool PAIR, typename Epi>
__device__ __forceinline__ SplitStore<Epi> split_store(const Epi& epi, float* part, uint32_t chunk, uint32_t P, uint32_t M, uint32_t N) {
  const uint64_t plane = static_cast<uint64_t>(M) * N;
  float* at = part + chunk * (PAIR ? 2u : 1u) * plane;
  return SplitStore<Epi>{epi, PlainStore<float>{at, at + plane, N}, P == 1u};
}

// A wave's results to the epilogue: IM blocks of 16 rows by JH blocks of 16
// columns of either half (acc[i][j], j < JH the first half), at most 64 rows at a
// time through `lds` (those rows by 32 JH floats, the wave's own), so that a lane
// takes eight consecutive columns, the memory accesses of a row are whole
// lines, and the epilogue's code is there once and not once for each block.
// 16-byte slot c of row r lies at c ^ store_swizzle(r): the writes of a
// block's 16 rows cover the banks once. Four chunks a turn, the next turn's loads
// issued before this one's stores: a wave has its SIMD to itself, nothing else
// covers their latency (4096^3 with bias, gelu and residual 161 us with the
// accumulators stored as they lie, 16 blocks of code and 8-byte rows; 131 so). WHOLE: every
// chunk lies inside the plane.
template <uint32_t SLOTS>
__device__ __forceinline__ uint32_t store_swizzle(uint32_t r) {
  return SLOTS >= 16u ? r & 15u : (r >> 1) & 7u;  // rows of 128 bytes: two to the banks
}
template <int IM, int JH, bool PAIR, bool WHOLE, typename Epi>
__device__ __forceinline__ void product_store(const f32x4_t (&acc)[IM][2 * JH], float* lds, uint32_t m0, uint32_t n0,
                                              uint32_t half, uint32_t M, uint32_t N, const Epi& epi, uint32_t lane) {
  constexpr uint32_t TH = 16u * JH, PITCH = 2u * TH, CHUNKS = PAIR ? TH / 8u : TH / 4u;  // of a row
  constexpr int IP = IM < 4 ? IM : 4;  // blocks of rows at a time
  constexpr uint32_t ROWS = 16u * IP, COUNT = ROWS * CHUNKS / 64u, TURN = COUNT < 4u ? COUNT : 4u, TURNS = COUNT / TURN;
  constexpr uint32_t PASSES = IM / IP, SLOTS = PITCH / 4u;
  static_assert(IM % IP == 0 && ROWS * CHUNKS % 64u == 0u && COUNT % TURN == 0u && SLOTS >= 8u, "whole turns");
  typename Epi::Fetch now[TURN], next[TURN];
  auto row_of = [&](uint32_t t) { return (t * 64u + lane) / CHUNKS; };  // of a pass
  auto col_of = [&](uint32_t t) { return (t * 64u + lane) % CHUNKS; };
  auto fetch = [&](uint32_t turn, typename Epi::Fetch (&f)[TURN]) {  // turns counted over the passes
#pragma unroll
    for (uint32_t i = 0; i < TURN; ++i) {
      const uint32_t t = turn % TURNS * TURN + i, k = col_of(t);
      const uint32_t m = m0 + ROWS * (turn / TURNS) + row_of(t), n = n0 + k / (TH / 8u) * half + k % (TH / 8u) * 8u;
      if (WHOLE || (m < M && n < N)) f[i] = epi.template fetch<WHOLE>(m, n);
    }
  };
  fetch(0u, now);
#pragma unroll 1
  for (uint32_t pass = 0; pass < PASSES; ++pass) {
    wave_exchange();
#pragma unroll
    for (int p = 0; p < static_cast<int>(PASSES); ++p) {
      if (pass != static_cast<uint32_t>(p)) continue;
#pragma unroll
      for (int i = 0; i < IP; ++i)
#pragma unroll
        for (int j = 0; j < 2 * JH; ++j) {
          const uint32_t r = 16u * i + (lane & 15u), c = 4u * j + (lane >> 4);
          *reinterpret_cast<f32x4_t*>(&lds[r * PITCH + ((c ^ store_swizzle<SLOTS>(r)) << 2)]) = acc[IP * p + i][j];
        }
    }
    wave_exchange();
#pragma unroll 1
    for (uint32_t b = 0; b < TURNS; ++b) {
      const uint32_t turn = pass * TURNS + b;
      if (turn + 1u < PASSES * TURNS) fetch(turn + 1u, next);
#pragma unroll
      for (uint32_t i = 0; i < TURN; ++i) {
        const uint32_t t = b * TURN + i, r = row_of(t), k = col_of(t), h = k / (TH / 8u), c = h * (TH / 4u) + k % (TH / 8u) * 2u;
        const uint32_t m = m0 + ROWS * pass + r, n = n0 + h * half + k % (TH / 8u) * 8u;
        const float* row = &lds[r * PITCH];
        auto take = [&](uint32_t s, float (&v)[8]) {
          const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(&row[(s ^ store_swizzle<SLOTS>(r)) << 2]);
          const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(&row[((s + 1u) ^ store_swizzle<SLOTS>(r)) << 2]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = lo[e];
            v[4 + e] = hi[e];
          }
        };
        float v0[8], v1[8];
        take(c, v0);
        if constexpr (PAIR) take(c + TH / 4u, v1);
        if (WHOLE || (m < M && n < N)) {
          if constexpr (PAIR) epi.template store<WHOLE>(m, n, now[i], v0, v1);
          else epi.template store<WHOLE>(m, n, now[i], v0);
        }
      }
#pragma unroll
      for (uint32_t i = 0; i < TURN; ++i) now[i] = next[i];
    }
  }
}

// ------------------------------------------------------------- operands
// M x N results over SEGS segments of K. a[s]: [M][K] or, A_RC, [K][M]; b[h][s]
// [N][K] or, B_RC, [K][N], b[1] the second matrix of a pair. Rows are packed.
template <int SEGS>
struct Operands {
  const uint16_t* a[SEGS];
  const uint16_t* b[2][SEGS];
  uint32_t M, N, K;
};

// n <= 8 values at p, zeros after them.
__device__ __forceinline__ u32x4 gather16(const uint16_t* p, uint32_t n) {
  uint64_t lo = 0u, hi = 0u;
#pragma unroll 1
  for (uint32_t e = 0; e < n; ++e) {
    const uint64_t v = p[e];
    if (e < 4u) lo |= v << (16u * e);
    else hi |= v << (16u * (e - 4u));
  }
  return u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
               static_cast<uint32_t>(hi >> 32)};
}

// ------------------------------------- any shape, any alignment
// Tiles of BM x 128 (a pair: BM x 64 of each product), 8 waves, 2 x 4 of them,
// 64-deep slices of K: global memory -> registers (16 bytes a lane, two slices
// ahead, unguarded: rows and chunks past the end re-read the last ones) -> LDS
// (two buffers, one barrier a slice). A chunk that runs past the end of its row
// is loaded from 8 elements before that end and moved into place, so the tail
// of k adds zeros. Slices first .. end - 1 of all segments'. Loads
// of rows that start anywhere span a line more, and go through registers: about
// half the ring's rate (bf16 4001 x 2049 x 3203 97 us; 4000 x 2048 x 3200 in the ring
// 54. f16 1001 x 1003 x 1501 with gelu, saved, 15.0).
template <bool F16, bool A_RC, bool B_RC, bool PAIR, int SEGS, uint32_t BM, typename Epi>
__device__ __forceinline__ void product_any(const Operands<SEGS>& p, const Epi& epi, uint32_t tile, uint32_t first, uint32_t end) {
  constexpr uint32_t HB = 64, THREADS = 512, SLICE = BM * 64u, HALF = HB * 64u, BUF = SLICE + 2u * HALF;
  constexpr int IM = BM / 32, CA = BM * 8 / THREADS;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * BUF];
  const uint32_t M = p.M, N = p.N, K = p.K, width = PAIR ? HB : 2u * HB;
  uint32_t tm, tn;
  gemm_tile_coords((M - 1u) / BM + 1u, (N - 1u) / width + 1u, &tm, &tn, tile);
  const uint32_t m0 = tm * BM, n0 = tn * width;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = (wave >> 2) * (BM / 2u), wn = (wave & 3u) * 16u;

  // One chunk of 8 of a K-contiguous panel row, or of row k of a row-contiguous
  // panel, and its values in place. TINY: rows of less than 8 values may occur,
  // and are gathered; otherwise a load has no branch, so that the waits for the
  // loads of one slice can leave those of the next in flight.
  auto kc_load = [&](auto tiny, const uint16_t* base, uint32_t row, uint32_t rows, uint32_t k) -> u32x4 {
    const uint16_t* r = base + static_cast<uint64_t>(row < rows ? row : rows - 1u) * K;
    if constexpr (decltype(tiny)::value)
      if (K < 8u) return gather16(r + (k < K ? k : 0u), k < K ? K - k : 0u);
    return load16_any(r + (k < K - 8u ? k : K - 8u));
  };
  auto kc_fix = [&](u32x4 v, uint32_t k) -> u32x4 {
    return K < 8u || k + 8u <= K ? v : shift_down16(v, k - (K - 8u));
  };
  auto rc_load = [&](auto tiny, const uint16_t* base, uint32_t c, uint32_t cols, uint32_t k) -> u32x4 {
    const uint16_t* r = base + static_cast<uint64_t>(k < K ? k : K - 1u) * cols;
    if constexpr (decltype(tiny)::value)
      if (cols < 8u) return gather16(r + (c < cols ? c : 0u), c < cols ? cols - c : 0u);
    return load16_any(r + (c < cols - 8u ? c : cols - 8u));
  };
  auto rc_fix = [&](u32x4 v, uint32_t c, uint32_t cols, uint32_t k) -> u32x4 {
    if (k >= K) return u32x4{0u, 0u, 0u, 0u};
    return cols < 8u || c + 8u <= cols ? v : shift_down16(v, c - (cols - 8u));
  };
  // A panel of W columns has W / 8 chunks a row of k; HB = 64: 8, as a row of k has.
  constexpr uint32_t kAC = A_RC ? BM / 8u : 8u;
  struct Regs {
    u32x4 a[CA], b[2];
  };
  Regs regs[2];
  const uint32_t ns = (K + 63u) / 64u;
  // Slice t, past the last one that again: every slice issues the same loads.
  auto load = [&](auto tiny, Regs& r, uint32_t at) {
    const uint32_t t = at < end ? at : end - 1u;
    const uint32_t seg = SEGS == 1 || t < ns ? 0u : 1u, k0 = (t - seg * ns) * 64u;
    const uint16_t* a = seg == 0u ? p.a[0] : p.a[SEGS - 1];
#pragma unroll
    for (uint32_t i = 0; i < CA; ++i) {
      const uint32_t c = i * THREADS + tid;
      r.a[i] = A_RC ? rc_load(tiny, a, m0 + c % kAC * 8u, M, k0 + c / kAC) : kc_load(tiny, a, m0 + (c >> 3), M, k0 + (c & 7u) * 8u);
    }
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
      const uint32_t hp = PAIR ? h : 0u, nh = PAIR ? n0 : n0 + HB * h;
      const uint16_t* b = seg == 0u ? p.b[hp][0] : p.b[hp][SEGS - 1];
      r.b[h] = B_RC ? rc_load(tiny, b, nh + (tid & 7u) * 8u, N, k0 + (tid >> 3)) : kc_load(tiny, b, nh + (tid >> 3), N, k0 + (tid & 7u) * 8u);
    }
  };
  auto write = [&](Regs& r, uint32_t t, uint32_t buf) {
    const uint32_t k0 = (SEGS == 1 || t < ns ? t : t - ns) * 64u;
    uint16_t* As = lds + buf * BUF;
    const bool ktail = k0 + 64u > K;
#pragma unroll
    for (uint32_t i = 0; i < CA; ++i) {
      const uint32_t c = i * THREADS + tid;
      if constexpr (A_RC) {
        const uint32_t k = c / kAC, m = c % kAC * 8u;
        if (ktail || m0 + BM > M) r.a[i] = rc_fix(r.a[i], m0 + m, M, k0 + k);
        *reinterpret_cast<u32x4*>(&As[swz_kn<BM>(k, m)]) = r.a[i];
      } else {
        if (ktail) r.a[i] = kc_fix(r.a[i], k0 + (c & 7u) * 8u);
        *reinterpret_cast<u32x4*>(&As[swz_rows64(c >> 3, c & 7u)]) = r.a[i];
      }
    }
#pragma unroll
    for (uint32_t h = 0; h < 2u; ++h) {
      uint16_t* Bs = As + SLICE + h * HALF;
      const uint32_t nh = PAIR ? n0 : n0 + HB * h;
      if constexpr (B_RC) {
        const uint32_t k = tid >> 3, n = (tid & 7u) * 8u;
        if (ktail || nh + HB > N) r.b[h] = rc_fix(r.b[h], nh + n, N, k0 + k);
        *reinterpret_cast<u32x4*>(&Bs[swz_kn<HB>(k, n)]) = r.b[h];
      } else {
        if (ktail) r.b[h] = kc_fix(r.b[h], k0 + (tid & 7u) * 8u);
        *reinterpret_cast<u32x4*>(&Bs[swz_rows64(tid >> 3, tid & 7u)]) = r.b[h];
      }
    }
  };
  f32x4_t acc[IM][2];  // [block of rows][half]
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) acc[i][h] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](uint32_t buf) {
    const uint16_t* As = lds + buf * BUF;
#pragma unroll
    for (uint32_t s = 0; s < 2u; ++s) {
      bf16x8 fa[IM], fb[2];
#pragma unroll
      for (uint32_t i = 0; i < IM; ++i) {
        if constexpr (A_RC) fa[i] = frag_b16_tr<BM>(As, wm + 16u * i, lane, 32u * s);
        else fa[i] = *reinterpret_cast<const bf16x8*>(&As[swz_rows64(wm + 16u * i + (lane & 15u), 4u * s + (lane >> 4))]);
      }
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        const uint16_t* Bs = As + SLICE + h * HALF;
        if constexpr (B_RC) fb[h] = frag_b16_tr<HB>(Bs, wn, lane, 32u * s);
        else fb[h] = *reinterpret_cast<const bf16x8*>(&Bs[swz_rows64(wn + (lane & 15u), 4u * s + (lane >> 4))]);
      }
      // Operands swapped: a lane ends with four consecutive columns of one row.
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < IM; ++i) acc[i][h] = mfma_16x16x32_16b<F16>(fb[h], fa[i], acc[i][h]);
    }
  };
  auto run = [&](auto tiny) {
    auto fence = []() { __builtin_amdgcn_sched_barrier(0); };  // loads stay in the order that the waits count
    load(tiny, regs[0], first);
    fence();
    load(tiny, regs[1], first + 1u);
    fence();
    write(regs[0], first, 0u);
    fence();
    load(tiny, regs[0], first + 2u);
    fence();
    __syncthreads();
    // Slice t, in buffer i; the next one (past the last: that again, read by
    // no one) in the registers of its parity.
    auto slice = [&](uint32_t t, uint32_t i) {
      compute(i);
      write(regs[1u - i], t + 1u < end ? t + 1u : t, 1u - i);
      load(tiny, regs[1u - i], t + 3u);
      __syncthreads();
    };
    // (Whole pairs: a way out between the two would make every wait one for all loads.)
    uint32_t t = first;
    for (; t + 2u <= end; t += 2u) {
      slice(t, 0u);
      slice(t + 1u, 1u);
    }
    if (t < end) {
      compute(0u);
      __syncthreads();
    }
  };
  if (first < end) {
    if ((A_RC ? M : K) < 8u || (B_RC ? N : K) < 8u) run(std::true_type{});
    else run(std::false_type{});
  }
  // (the last slice's barrier: no wave reads the slices any more)
  product_store<IM, 1, PAIR, false>(acc, reinterpret_cast<float*>(lds) + wave * (32u * (IM < 4 ? 16u * IM : 64u)), m0 + wm, n0 + wn, HB, M, N,
                                    epi, lane);
}

// The 64-deep slices of all segments' that chunk c of P takes: a run of them.
struct Run {
  uint32_t first, end;
};
__device__ __forceinline__ Run run_of(uint32_t K, uint32_t segs, uint32_t chunk, uint32_t P) {
  const uint32_t total = (K + 63u) / 64u * segs, per = (total + P - 1u) / P, first = chunk * per;
  return Run{first < total ? first : total, first + per < total ? first + per : total};
}

// ------------------------- rows of whole 16-byte chunks: straight into LDS
// What chunks that lie outside an operand read (a static constant of the code
// object): rows past the end and slices past the last add zeros to the sums.
static __device__ __attribute__((aligned(16))) const uint32_t kZeroChunk[4] = {0u, 0u, 0u, 0u};

// Extents up to here keep a lane's offset in a panel (256 rows of K, or 64
// rows of M or N, in bytes) within 32 bits.
constexpr uint32_t kInnerMost = 1u << 22;

// How a lane reads the MFMA operands of a 64-deep panel of W rows
// (K-contiguous) or W columns (RC), `blocks` of 16 from `first` on: for k 32 h ..
// 32 h + 31 of block i, a byte offset in the panel, of which only few depend on
// the lane (one for each h, or for each block), the rest being constants of
// the instruction. (RC: ds_read_b64_tr_b16 as at frag_b16_tr; the swizzle of row
// k leaves out bits 2, 4 and 5 of k.)
template <bool RC, uint32_t W, int BLOCKS>
struct Frags {
  uint32_t off[RC ? BLOCKS : 2];
  __device__ __forceinline__ Frags(uint32_t first, uint32_t lane) {
    const uint32_t g = lane >> 4, j = lane & 15u;
    if constexpr (RC) {
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) off[i] = 2u * swz_kn<W>(8u * g + (j >> 2), first + 16u * i + 4u * (j & 3u));
    } else {
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) off[h] = 2u * swz_rows64(first + j, 4u * h + g);
    }
  }
  // `panel`: bytes from `lds`, a scalar.
  __device__ __forceinline__ bf16x8 read(const uint16_t* lds, uint32_t panel, int h, int i) const {
    if constexpr (RC) {
      const char* p = reinterpret_cast<const char*>(lds) + (panel + off[i]) + 64 * static_cast<int>(W) * h;
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p + 8 * static_cast<int>(W)));
      typedef short i16x8 __attribute__((ext_vector_type(8)));
      const i16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(bf16x8, v);
    } else {
      return *reinterpret_cast<const bf16x8*>(reinterpret_cast<const char*>(lds) + (panel + off[h]) + 2048 * i);
    }
  }
};

// How the lanes of WAVES waves fill a 64-deep panel of W rows (K-contiguous)
// or W columns (RC): chunk q of a wave is chunk q WAVES + wave of the panel, so
// that a lane's places in them differ by a multiple of the pitch, a scalar
// (and, for 256 columns, by a swizzle that alternates with q).
template <bool RC, uint32_t W, uint32_t WAVES>
struct Fill {
  static constexpr uint32_t kRows = RC ? 512u / W : 8u;  // rows of memory in a chunk
  static constexpr bool kTwo = RC && WAVES * kRows == 8u;
  static_assert(!RC || WAVES * kRows % 8u == 0u, "the swizzle of row k alternates with q at most");
  uint32_t off[kTwo ? 2 : 1], row, col[kTwo ? 2 : 1];  // elements from the panel's first, row and column in it
  __device__ __forceinline__ Fill(uint32_t wave, uint32_t lane, uint32_t pitch) {
    row = wave * kRows + lane / (RC ? W / 8u : 8u);
#pragma unroll
    for (uint32_t i = 0; i < (kTwo ? 2u : 1u); ++i) {
      if constexpr (RC) col[i] = ((lane % (W / 8u)) ^ kn_slot_xor<W>(row + 8u * i)) * 8u;
      else col[i] = ((lane & 7u) ^ (row & 6u)) * 8u;  // the inverse of swz_rows64
      off[i] = row * pitch + col[i];
    }
  }
  // Chunk q of the panel at p, its first element (k0, c0) in k and its own
  // index, K and C their ends.
  template <bool FAST>
  __device__ __forceinline__ void load(const uint16_t* p, const uint16_t* zero, uint16_t* lds, int q, uint32_t pitch, uint32_t wave,
                                       uint32_t k0, uint32_t c0, uint32_t K, uint32_t C) const {
    constexpr uint32_t kStep = WAVES * kRows;
    const uint32_t i = kTwo ? q & 1 : 0u, k = RC ? row + q * kStep : col[0], c = RC ? col[i] : row + q * kStep;
    const uint16_t* at = p + static_cast<uint64_t>(q) * kStep * pitch;
    asm volatile("" : "+s"(at));  // a scalar: not one sum of it and the lane's offset kept for every q
    const uint16_t* g = at + off[i];
    if constexpr (FAST) g = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(at) + 2u * off[i]);
    else g = ((k0 + k < K) & (c0 + c < C)) ? g : zero;  // (no branch)
    __builtin_amdgcn_global_load_lds(g, (lds_void*)(lds + (q * WAVES + wave) * 512u), 16, 0, 0);
  }
};

// Loads of the steps after step `at` up to step 0: qa in an even one, qb in an odd one.
constexpr int loads_after(int at, int qa, int qb) {
  int n = 0;
  for (int s = at + 1; s <= 0; ++s) n += s % 2 == 0 ? qa : qb;
  return n;
}

// A tile of BM x 2 HB (a pair: BM x HB of each product), WGM x WGN waves, each
// (BM / WGM) rows by HB / WGN columns of either half, for operands whose rows
// are whole chunks of 8 (K % 8 == 0 where K-contiguous, M or N % 8 == 0 where
// row-contiguous).
//
// K advances in turns of 64 through rings of SA slots of A and SB of B, filled
// by global_load_lds (lane i of a load writes 16 bytes at 16 i of a 1 KiB
// chunk, from any global address: each lane's address is the inverse of the
// LDS swizzle). 64 deep, a K-contiguous row is a whole 128-byte line of memory
// (in slices of 32, loads of half lines cost 4096^3 of [M][K] by [N][K] a third of
// its time), and one barrier serves two MFMA steps (a 128x128 tile needs 256
// cycles for its MFMAs of 32 k and 450 for a barrier and the waits at it).
// Turn t:
//   step 0: MFMAs of k 0..31 on registers, while the fragments of k 32..63 are
//           read into the other register set and A of turn t - 1 + SA is loaded
//           into the slot of turn t - 1;
//   wait until turn t + 1 has landed and every read of turn t has completed,
//   barrier;
//   step 1: MFMAs of k 32..63, reads of turn t + 1, k 0..31, and B of turn
//           t + SB is loaded into the slot of turn t.
// Every turn issues the same loads: a chunk outside its operand, or past the
// last turn, is read from kZeroChunk, so no tail of k, edge of the plane or
// border between segments needs code of its own, and the count of loads in
// flight is static. Turns first .. end - 1 of all segments'. (The operands are
// __restrict__ parameters: without them the compiler takes a transposing read
// of LDS to depend on every load into it and waits for all of them.)
//
// bf16 4096^3 with bias, gelu and residual 118 to 128 us on three cards, 1.07 to 1.16
// PFLOP/s, the library's bare product 119; a pair 4096 x 2048 x 8192 that saves both
// 243 to 250. The matrix cores are busy for half of the cycles, no bank of LDS
// conflicts; with operands that stay in the L2 4096^3 takes 110 us, with no
// loads at all 86: what is left is the loads into LDS beside its reads, at the
// clock that the power leaves.
template <bool F16, bool A_RC, bool B_RC, bool PAIR, int SEGS, uint32_t BM, uint32_t HB, uint32_t WGM, uint32_t WGN, int SA, int SB,
          typename Epi>
__device__ __forceinline__ void product_ring_of(const uint16_t* __restrict__ pa0, const uint16_t* __restrict__ pa1,
                                                const uint16_t* __restrict__ pb00, const uint16_t* __restrict__ pb01,
                                                const uint16_t* __restrict__ pb10, const uint16_t* __restrict__ pb11,
                                                const uint16_t* __restrict__ zero, uint32_t M, uint32_t N, uint32_t K,
                                                const Epi& epi, uint32_t tile, uint32_t first, uint32_t end) {
  constexpr uint32_t WAVES = WGM * WGN, TM = BM / WGM, TH = HB / WGN, ASL = BM * 64u, BSL = HB * 64u;
  constexpr int IM = TM / 16, JH = TH / 16, JN = 2 * JH, QA = BM / 8 / WAVES, QB = 2 * HB / 8 / WAVES;
  static_assert(BM / 8 % WAVES == 0 && HB / 8 % WAVES == 0, "whole chunks, of either half, per wave");
  static_assert(SA >= 3 && SB >= 2, "A is loaded a turn later than B");
  __shared__ __attribute__((aligned(16))) uint16_t lds[SA * ASL + SB * 2u * BSL];
  const uint32_t width = PAIR ? HB : 2u * HB;
  uint32_t tm, tn;
  gemm_tile_coords((M - 1u) / BM + 1u, (N - 1u) / width + 1u, &tm, &tn, tile);
  const uint32_t m0 = tm * BM, n0 = tn * width;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t wm = (wave / WGN) * TM, wn = (wave % WGN) * TH;
  const uint32_t pitch_a = A_RC ? M : K, pitch_b = B_RC ? N : K;
  const Fill<A_RC, BM, WAVES> fill_a(wave, lane, pitch_a);
  const Fill<B_RC, HB, WAVES> fill_b(wave, lane, pitch_b);
  const uint32_t ns = (K + 63u) / 64u;
  uint16_t* ldsp = lds;
  // Turns whose chunks all lie inside the operands, for a tile that does:
  // their loads take the panel's address from scalar registers and a 32-bit
  // offset a lane, with no test (which costs a tenth of the whole time).
  const bool inner = m0 + BM <= M && n0 + width <= N && M <= kInnerMost && N <= kInnerMost && K <= kInnerMost;
  const uint32_t full = K % 64u == 0u ? end : SEGS == 1 ? K / 64u : 0u, whole = !inner ? 0u : full < end ? full : end;
  // The first k of turn t in its segment; past the last turn every chunk is zeros.
  auto first_k = [&](uint32_t t) { return t < end ? (SEGS == 1 || t < ns ? t : t - ns) * 64u : K; };
  auto load_a = [&](auto fast, uint32_t t, uint32_t slot, int q) {
    const uint32_t k0 = first_k(t);
    const uint16_t* p = (SEGS == 1 || t < ns ? pa0 : pa1) +
                        (A_RC ? static_cast<uint64_t>(k0) * M + m0 : static_cast<uint64_t>(m0) * K + k0);
    fill_a.template load<decltype(fast)::value>(p, zero, ldsp + slot / 2u, q, pitch_a, wave, k0, m0, K, M);
  };
  auto load_b = [&](auto fast, uint32_t t, uint32_t slot, int q) {  // q < QB / 2: the first half
    const uint32_t k0 = first_k(t), h = q / (QB / 2), nh = PAIR ? n0 : n0 + h * HB;
    const uint16_t* b = (PAIR && h != 0u) ? (SEGS == 1 || t < ns ? pb10 : pb11) : (SEGS == 1 || t < ns ? pb00 : pb01);
    const uint16_t* p = b + (B_RC ? static_cast<uint64_t>(k0) * N + nh : static_cast<uint64_t>(nh) * K + k0);
    fill_b.template load<decltype(fast)::value>(p, zero, ldsp + slot / 2u + h * BSL, q % (QB / 2), pitch_b, wave, k0, nh, K, N);
  };
  const Frags<A_RC, BM, IM> frags_a(wm, lane);
  const Frags<B_RC, HB, JH> frags_b(wn, lane);
  auto rd_a = [&](uint32_t slot, int h, int i) { return frags_a.read(ldsp, slot, h, i); };
  auto rd_b = [&](uint32_t slot, int h, int j) {  // j < JH: the first half
    return frags_b.read(ldsp, slot + (j / JH) * 2u * BSL, h, j % JH);
  };
  f32x4_t acc[IM][JN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < JN; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto fence = []() { __builtin_amdgcn_sched_barrier(0); };
  // The accumulators are tied to AGPRs by inline-asm MFMAs (the compiler's own
  // move them from one AGPR to another, 64 moves a turn of 128x128, and a third
  // of the time at 256x128), with the hazards covered as at gemm_bf16_4w: the
  // operands are results of LDS reads only; wait states before the first and
  // after the last.
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < JN; ++j) asm volatile("" : "+a"(acc[i][j]));
  asm volatile("s_nop 7\n\ts_nop 7" ::: "memory");
  fence();
  using Fast = std::true_type;
  using Checked = std::false_type;
  bf16x8 a0[IM], b0[JN], a1[IM], b1[JN];
  // Loads that may be in flight at turn t's barrier: those issued after the
  // later one of A and B of turn t + 1. With the steps numbered 2t and 2t + 1, A
  // of turn j is issued in step 2 (j + 1 - SA), B in step 2 (j - SB) + 1.
  constexpr int kAt = 4 - 2 * SA > 3 - 2 * SB ? 4 - 2 * SA : 3 - 2 * SB;
  constexpr int kFlight = loads_after(kAt, QA, QB);
  constexpr int kStart = (SA - 1) * QA + SB * QB;  // the first turns' loads
  static_assert(kStart < 64, "vmcnt holds the loads in flight");
  // One 32-deep step: the MFMAs of one register set, with the reads of the
  // other and then `n` loads evenly over them but the last few: in a burst,
  // four SIMDs ask for twice what LDS gives. MFMA c takes block (i, j), i
  // snaking, so that consecutive ones share an operand; operands swapped, so
  // that a lane ends with four columns of one row.
  auto step = [&](const bf16x8* ca, const bf16x8* cb, auto&& rd, auto n, auto&& ld) {
    constexpr int kOps = IM + JN + decltype(n)::value, kOver = IM * JN - 4;
    fence();
#pragma unroll
    for (int c = 0; c < IM * JN; ++c) {
      const int j = c / IM, i = (j & 1) ? IM - 1 - c % IM : c % IM;
      mfma16_bf16_acc<F16>(acc[i][j], cb[j], ca[i]);
      fence();
      for (int o = c * kOps / kOver; o < (c + 1) * kOps / kOver && o < kOps; ++o) {
        if (o < IM + JN) rd(o);
        else ld(o - IM - JN);
      }
      fence();
    }
  };
  // The slots of turns t - 1, t and t + 1 (bytes of LDS), kept as scalars.
  constexpr uint32_t kA = 2u * ASL, kB = 4u * BSL, kB0 = SA * kA;
  uint32_t a_last = (SA - 1) * kA, a_this = 0u, a_next = kA, b_this = kB0, b_next = kB0 + kB;
  auto turn = [&](auto fast, uint32_t t) {
    step(a0, b0, [&](int o) { if (o < IM) a1[o] = rd_a(a_this, 1, o); else b1[o - IM] = rd_b(b_this, 1, o - IM); },
         std::integral_constant<int, QA>{}, [&](int q) { load_a(fast, t + SA - 1, a_last, q); });
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(kFlight, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    step(a1, b1, [&](int o) { if (o < IM) a0[o] = rd_a(a_next, 0, o); else b0[o - IM] = rd_b(b_next, 0, o - IM); },
         std::integral_constant<int, QB>{}, [&](int q) { load_b(fast, t + SB, b_this, q); });
    a_last = a_this;
    a_this = a_next;
    a_next = a_next == (SA - 1) * kA ? 0u : a_next + kA;
    b_this = b_next;
    b_next = b_next == kB0 + (SB - 1) * kB ? kB0 : b_next + kB;
  };
#pragma unroll
  for (int t = 0; t < (SA - 1 > SB ? SA - 1 : SB); ++t) {
    if (t < SA - 1)
#pragma unroll
      for (int q = 0; q < QA; ++q) load_a(Checked{}, first + t, t * kA, q);
    if (t < SB)
#pragma unroll
      for (int q = 0; q < QB; ++q) load_b(Checked{}, first + t, kB0 + t * kB, q);
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(kStart - QA - QB, 0));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < IM; ++i) a0[i] = rd_a(a_this, 0, i);
#pragma unroll
  for (int j = 0; j < JN; ++j) b0[j] = rd_b(b_this, 0, j);
  // No turns at all (K = 0) is one of zeros: a branch round the loop would hold
  // the accumulators in two places, and spill.
  uint32_t t = first;
  constexpr uint32_t kAhead = SA - 1 > SB ? SA - 1 : SB;
  for (; t + kAhead < whole; ++t) turn(Fast{}, t);
  do turn(Checked{}, t++);
  while (t < end);
  // No load into LDS is in flight past the loop, in any wave.
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  fence();
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory");
  fence();
  static_assert(WAVES * 64u * 2u * TH * 4u <= sizeof(lds), "64 rows of every wave");
  float* own = reinterpret_cast<float*>(lds) + wave * (64u * 2u * TH);
  if (m0 + BM <= M && n0 + width <= N) product_store<IM, JH, PAIR, true>(acc, own, m0 + wm, n0 + wn, HB, M, N, epi, lane);
  else product_store<IM, JH, PAIR, false>(acc, own, m0 + wm, n0 + wn, HB, M, N, epi, lane);
}

template <bool F16, bool A_RC, bool B_RC, bool PAIR, int SEGS, uint32_t BM, uint32_t HB, uint32_t WGM, uint32_t WGN, int SA, int SB,
          typename Epi>
__device__ __forceinline__ void product_ring(const Operands<SEGS>& p, const Epi& epi, uint32_t tile, uint32_t first, uint32_t end) {
  product_ring_of<F16, A_RC, B_RC, PAIR, SEGS, BM, HB, WGM, WGN, SA, SB>(
      p.a[0], p.a[SEGS - 1], p.b[0][0], p.b[0][SEGS - 1], p.b[1][0], p.b[1][SEGS - 1],
      reinterpret_cast<const uint16_t*>(kZeroChunk), p.M, p.N, p.K, epi, tile, first, end);
}

// ----------------------------------------------- few rows: the weight is read
// At most 64 rows of x [M][K] by a row-contiguous weight (of a pair: two): bound by
// the weight's bytes. Nothing of it goes through LDS: a lane reads 4 columns
// of the 8 rows of k that an MFMA operand holds, 16 lanes a whole 128-byte
// line of a row, and transposes them in registers (one byte permute for two values);
// column j of every lane makes one operand, so that operand's 16 columns are 4
// apart, which the result only has to know. Eight waves of a workgroup take
// every eighth 32-deep step of a strip of 64 columns and meet in LDS in wave
// order; where strips are few, P workgroups share one, each a run of steps, and
// join_parts adds their partial sums in order (`part`, [P][1 or 2][M][N]).
//
// One row by 4096 x 4096 7.4 to 9.5 us (33.5 MB, 3.5 to 4.5 TB/s) and 3.9 for the
// join; 16 rows by a pair of 4096 x 8192 27.6 us (134 MB, 4.9 TB/s) and 4.7. Strips
// of 32 and of 16 columns, of which these need no join, take 12.9 and 16.9, and
// 38 and 55 us: the time goes with the number of loads. Lanes of 8 columns spill.
constexpr uint32_t kFewColumns = 64, kFewWaves = 8;

template <bool F16, bool PAIR, int MB, typename Epi>
__device__ __forceinline__ void product_few(const Operands<1>& p, const Epi& epi, float* __restrict__ part, uint32_t strips,
                                            uint32_t P) {
  constexpr int H = PAIR ? 2 : 1, D = H * MB > 4 ? 2 : 4;  // steps in registers
  constexpr int VEC = 4;                                   // columns a lane
  constexpr uint32_t COLS = kFewColumns, PITCH = H * COLS, CHUNKS = COLS / 8u;
  typedef uint32_t Row __attribute__((ext_vector_type(VEC / 2)));
  typedef uint32_t RowAny __attribute__((ext_vector_type(VEC / 2), aligned(2)));
  __shared__ __attribute__((aligned(16))) float lds[kFewWaves * 16u * PITCH];
  const uint32_t M = p.M, N = p.N, K = p.K;
  const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = lane & 15u, g = lane >> 4, strip = blockIdx.x % strips, chunk = blockIdx.x / strips;
  const uint32_t n0 = strip * COLS, n = n0 + VEC * c;
  // A lane's columns: past the end, the last VEC (stored where they are its own).
  const uint32_t at = n + VEC <= N ? n : N >= VEC ? N - VEC : 0u;
  const uint32_t ns = (K + 31u) / 32u, per = (ns + P - 1u) / P, first = chunk * per;
  const uint32_t end = first + per < ns ? first + per : ns;
  struct Step {
    Row w[H][8];
    u32x4 x[MB];
  };
  Step st[D];
  auto load = [&](Step& s, uint32_t t) {
    const uint32_t k0 = t * 32u + 8u * g;
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (uint32_t e = 0; e < 8u; ++e) {
        const uint32_t k = k0 + e < K ? k0 + e : K - 1u;
        const uint16_t* row = p.b[h][0] + static_cast<uint64_t>(k) * N + at;
        if (N >= VEC) {
          // Read once by the whole grid: not kept in the caches (5% of the time).
          s.w[h][e] = __builtin_nontemporal_load(reinterpret_cast<const RowAny*>(row));
        } else {
          const u32x4 v = gather16(row, N);
#pragma unroll
          for (int d = 0; d < VEC / 2; ++d) s.w[h][e][d] = v[d];
        }
      }
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const uint32_t m = 16u * i + c;
      const uint16_t* row = p.a[0] + static_cast<uint64_t>(m < M ? m : M - 1u) * K;
      if (K >= 8u) s.x[i] = load16_any(row + (k0 < K - 8u ? k0 : K - 8u));
      else s.x[i] = gather16(row + (k0 < K ? k0 : 0u), k0 < K ? K - k0 : 0u);
    }
  };
  f32x4_t acc[H][MB][VEC];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[h][i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto compute = [&](Step& s, uint32_t t) {
    const uint32_t k0 = t * 32u + 8u * g;
    if (t * 32u + 32u > K) {  // the last, short step: zeros past K in both operands
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (uint32_t e = 0; e < 8u; ++e)
#pragma unroll
          for (int d = 0; d < VEC / 2; ++d)
            if (k0 + e >= K) s.w[h][e][d] = 0u;
#pragma unroll
      for (int i = 0; i < MB; ++i)
        if (K >= 8u && k0 + 8u > K) s.x[i] = shift_down16(s.x[i], k0 - (K - 8u));
    }
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        u32x4 w;
#pragma unroll
        for (int d = 0; d < 4; ++d)  // k 2d and 2d + 1 of column j
          w[d] = __builtin_amdgcn_perm(s.w[h][2 * d + 1][j / 2], s.w[h][2 * d][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int i = 0; i < MB; ++i)
          acc[h][i][j] = mfma_16x16x32_16b<F16>(__builtin_bit_cast(bf16x8, s.x[i]), __builtin_bit_cast(bf16x8, w), acc[h][i][j]);
      }
  };
  const uint32_t t0 = first + wave;
  if (t0 < end) {
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (t0 + d * kFewWaves < end) load(st[d], t0 + d * kFewWaves);
    for (uint32_t t = t0; t < end; t += D * kFewWaves) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        const uint32_t s = t + d * kFewWaves;
        if (s < end) compute(st[d], s);
        if (s + D * kFewWaves < end) load(st[d], s + D * kFewWaves);
      }
    }
  }
  // acc[h][i][j][e] is the sum of row 16 i + 4 g + e, column at + j.
  const bool direct = P == 1u;
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    if (16u * i >= M) break;
    if (i > 0) __syncthreads();
    float* own = lds + wave * (16u * PITCH);
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (uint32_t e = 0; e < 4u; ++e) {
        float* row = own + (4u * g + e) * PITCH + h * COLS;
        if (at == n) {
#pragma unroll
          for (int j = 0; j < VEC; j += 4)
            *reinterpret_cast<f32x4_t*>(row + VEC * c + j) =
                f32x4_t{acc[h][i][j][e], acc[h][i][j + 1][e], acc[h][i][j + 2][e], acc[h][i][j + 3][e]};
        } else if (n < N) {
#pragma unroll
          for (uint32_t j = 0; j < VEC; ++j)
            if (at + j >= n && at + j < N) row[at + j - n0] = acc[h][i][j][e];
        }
      }
    __syncthreads();
    const uint32_t r = threadIdx.x / CHUNKS, k = threadIdx.x % CHUNKS, m = 16u * i + r, nk = n0 + 8u * k;
    if (r < 16u && m < M && nk < N) {
      float v[H][8];
#pragma unroll
      for (int h = 0; h < H; ++h) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[h][e] = 0.0f;
        const float* from = lds + r * PITCH + h * COLS + 8u * k;
#pragma unroll
        for (uint32_t w = 0; w < kFewWaves; ++w) {
          const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(from + w * (16u * PITCH));
          const f32x4_t hi = *reinterpret_cast<const f32x4_t*>(from + w * (16u * PITCH) + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[h][e] += lo[e];
            v[h][4 + e] += hi[e];
          }
        }
      }
      if (direct) {
        const auto f = epi.template fetch<false>(m, nk);
        if constexpr (PAIR) epi.template store<false>(m, nk, f, v[0], v[1]);
        else epi.template store<false>(m, nk, f, v[0]);
      } else {
#pragma unroll
        for (int h = 0; h < H; ++h) row_store<8>(part + (static_cast<uint64_t>(chunk * H + h) * M + m) * N, nk, N, v[h]);
      }
    }
  }
}

// The P partial sums of eight columns a lane, in order, to the epilogue: 32
// chunks of row blockIdx.x % M by SLICES slices of the partials a workgroup,
// four partials of a lane in flight (past the end, the last one again). With a
// lane adding all of them, 25 partials of one row took 22 us (8 slices: 6);
// planes of tiles have fewer partials and many rows (940 x 1040 by 4: 8.2 us with
// 8 slices, 5 with 4).
template <bool PAIR, uint32_t SLICES, typename Epi>
__device__ __forceinline__ void join_parts(const float* __restrict__ part, const Epi& epi, uint32_t M, uint32_t N, uint32_t P) {
  constexpr int H = PAIR ? 2 : 1;
  __shared__ __attribute__((aligned(16))) float join[SLICES][H][32][8];
  const uint32_t i = threadIdx.x & 31u, slot = threadIdx.x >> 5;
  const uint32_t m = blockIdx.x % M, n = (blockIdx.x / M * 32u + i) * 8u;
  float v[H][8];
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[h][e] = 0.0f;
  if (n < N)
    for (uint32_t p = slot; p < P; p += 4u * SLICES) {
      vec<float, 8> s[4][H];
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k)
#pragma unroll
        for (int h = 0; h < H; ++h)
          s[k][h] = row_raw<8>(part + (static_cast<uint64_t>((p + SLICES * k < P ? p + SLICES * k : P - 1u) * H + h) * M + m) * N, n, N);
#pragma unroll
      for (uint32_t k = 0; k < 4u; ++k)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          row_fix<8>(s[k][h], n, N);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[h][e] = p + SLICES * k < P ? v[h][e] + s[k][h][e] : v[h][e];
        }
    }
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int e = 0; e < 8; ++e) join[slot][h][i][e] = v[h][e];
  __syncthreads();
  if (slot != 0u || n >= N) return;
  const auto f = epi.template fetch<false>(m, n);
#pragma unroll
  for (uint32_t s = 1; s < SLICES; ++s)
#pragma unroll
    for (int h = 0; h < H; ++h)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[h][e] += join[s][h][i][e];
  if constexpr (PAIR) epi.template store<false>(m, n, f, v[0], v[1]);
  else epi.template store<false>(m, n, f, v[0]);
}

// ------------------------------------------ gradients of the pre-activations
// One element each: dz = dy act'(z) of a projection, dg = dh u act'(g) and
// du = dh act(g) of a gated pair.
template <typename T, int ACT, bool GATED>
struct Slope {
  const T* dy;
  const T* z;  // g of a pair
  const T* u;
  T* dz;  // dg of a pair; no store where ACT is none
  T* du;
  static constexpr bool kZ = ACT != kActNone || GATED;
  struct Raw {
    vec<T, 8> dy, z, u;
  };
  // The vector from element c of the row at `at`, of C.
  __device__ __forceinline__ Raw load(uint64_t at, uint32_t c, uint32_t C) const {
    Raw r;
    r.dy = row_raw<8>(dy + at, c, C);
    if constexpr (kZ) r.z = row_raw<8>(z + at, c, C);
    if constexpr (GATED) r.u = row_raw<8>(u + at, c, C);
    return r;
  }
  // f0 = dz or dg, f1 = du, stored.
  __device__ __forceinline__ void store(Raw r, uint64_t at, uint32_t c, uint32_t C, float (&f0)[8], float (&f1)[8]) const {
    row_fix<8>(r.dy, c, C);
    if constexpr (kZ) row_fix<8>(r.z, c, C);
    if constexpr (GATED) row_fix<8>(r.u, c, C);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = static_cast<float>(r.dy[e]);
      if constexpr (GATED) {
        const float a = static_cast<float>(r.z[e]);
        f0[e] = d * static_cast<float>(r.u[e]) * act_slope<ACT>(a);
        f1[e] = d * act<ACT>(a);
      } else if constexpr (ACT != kActNone) {
        f0[e] = d * act_slope<ACT>(static_cast<float>(r.z[e]));
      } else {
        f0[e] = d;
      }
    }
    if constexpr (kZ) row_store<8>(dz + at, c, C, f0);
    if constexpr (GATED) row_store<8>(du + at, c, C, f1);
  }
};

// Over the whole plane as one row of `n` elements, 8 a lane. Bound by HBM: five
// planes of 4096 x 8192 52 to 55 us, 6.1 to 6.4 TB/s.
template <typename T, int ACT, bool GATED>
__device__ __forceinline__ void slope_flat(const Slope<T, ACT, GATED>& f, uint32_t n) {
  const uint32_t c = (blockIdx.x * 256u + threadIdx.x) * 8u;
  if (c >= n) return;
  float f0[8], f1[8];
  f.store(f.load(0u, c, n), 0u, c, n, f0, f1);
}

// ... with the column sums of a bias' gradient, of the values before they are
// rounded: 512 columns by 16 rows a workgroup of 1024 lanes, over row chunk p of
// P, two rows of a lane in flight; `part` is [P][1 + GATED][N]. (Four rows a lane one
// after the other take a wave 9 us, however few there are.) Three planes of 2048 x
// 4096 13 us, 3.9 TB/s: one round of workgroups, whose start and join show.
template <typename T, int ACT, bool GATED>
__device__ __forceinline__ void slope_columns(const Slope<T, ACT, GATED>& f, float* __restrict__ part, uint32_t M,
                                              uint32_t N, uint32_t P) {
  constexpr uint32_t AHEAD = 2, SLOTS = 16;
  __shared__ float join[SLOTS][512];
  const uint32_t p = blockIdx.x % P, c0 = blockIdx.x / P * 512u, c = c0 + lane_id() * 8u, slot = wave_id();
  const uint64_t rows = (M - 1u) / P + 1u, first = p * rows, last = first + rows < M ? first + rows : M;
  float s0[8], s1[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) s0[e] = s1[e] = 0.0f;
  if (c < N)
    for (uint64_t r = first + slot; r < last; r += SLOTS * AHEAD) {
      typename Slope<T, ACT, GATED>::Raw raw[AHEAD];
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; ++k)
        if (r + SLOTS * k < last) raw[k] = f.load((r + SLOTS * k) * N, c, N);
#pragma unroll
      for (uint32_t k = 0; k < AHEAD; ++k) {
        if (r + SLOTS * k >= last) break;
        float f0[8], f1[8];
        f.store(raw[k], (r + SLOTS * k) * N, c, N, f0, f1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s0[e] += f0[e];
          if constexpr (GATED) s1[e] += f1[e];
        }
      }
    }
  constexpr uint32_t Q = GATED ? 2u : 1u;
#pragma unroll
  for (uint32_t q = 0; q < Q; ++q) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) join[slot][lane_id() * 8u + e] = q == 0u ? s0[e] : s1[e];
    __syncthreads();
    if (threadIdx.x < 512u && c0 + threadIdx.x < N) {
      float v = join[0][threadIdx.x];
#pragma unroll
      for (uint32_t s = 1; s < SLOTS; ++s) v += join[s][threadIdx.x];
      part[(static_cast<uint64_t>(p) * Q + q) * N + c0 + threadIdx.x] = v;
    }
  }
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_PRODUCT_H_
