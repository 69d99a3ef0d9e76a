// positions.h — where new tokens stand: block tables and slot maps from request
// lengths, rotary positions, and the same while keys and values are stored into a
// paged cache.
#ifndef TCA_HIP_POSITIONS_H_
#define TCA_HIP_POSITIONS_H_

#include "tca/hip/rows.h"

namespace tca {
namespace hip {

// ------------------------------------------------- block tables, slot maps
// have = ceil(held / page), need = ceil((held + new) / page) of a sequence, at most
// the table's P columns; columns have .. need - 1 take the free pages from
// free[first + pages taken by earlier sequences] on.
//
// Every workgroup adds up all sequences (1024 runs of them, a scan in LDS) and
// then places tokens, a grid's stride apart: one launch, no sums between
// workgroups. A page's first token is always a new one, and stores its column, or, where
// the batch has no room for that token, a lane of its own does: nobody reads a column
// that this launch stores. Bound by the chain of loads, scan and
// search: 256 sequences of one token 4.9 us, 37 prompts of 23 k tokens 6.1, 4096 sequences
// of 107 k tokens 10.5 (18 with four tokens a lane).
struct PageSeq {
  uint32_t held, fresh, have, take;
};
__device__ __forceinline__ PageSeq page_seq(const int32_t* held, const int32_t* fresh, uint64_t s, uint32_t page, uint32_t P) {
  PageSeq q;
  const int32_t h = held[s], n = fresh[s];
  q.held = h < 0 ? 0u : static_cast<uint32_t>(h);
  q.fresh = n < 0 ? 0u : static_cast<uint32_t>(n);
  q.have = ceil_div(q.held, page);
  const uint32_t need = ceil_div(q.held + q.fresh, page), most = need < P ? need : P;
  q.take = most > q.have ? most - q.have : 0u;
  return q;
}
// The page that column `col` of a sequence takes, `taken` pages after the first.
__device__ __forceinline__ int32_t page_taken(const int32_t* free_pages, uint32_t F, int64_t from, uint64_t taken) {
  const int64_t f = from + static_cast<int64_t>(taken);
  return f >= 0 && f < static_cast<int64_t>(F) ? free_pages[f] : -1;
}
// Of 1024 runs whose sums end in ends[1 .. 1024], the one that holds unit t: ends[lo] <= t < ends[lo + 1].
__device__ __forceinline__ uint32_t page_run(const uint64_t* ends, uint64_t t) {
  uint32_t lo = 0u, hi = 1024u;
  while (hi - lo > 1u) {
    const uint32_t mid = (lo + hi) / 2u;
    if (ends[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int32_t page_int(uint64_t v) { return v > 0x7fffffffu ? 0x7fffffff : static_cast<int32_t>(v); }

__device__ __forceinline__ void page_table(const int32_t* held, const int32_t* fresh, const int32_t* free_pages, const int32_t* first,
                                           int32_t* table, int32_t* starts, int32_t* lens, int32_t* pos, int32_t* slot, int32_t* next,
                                           uint32_t S, uint32_t F, uint32_t P, uint32_t T, uint32_t page) {
  __shared__ uint64_t tokens[1025], pages[1025];
  const uint32_t tid = threadIdx.x, run = ceil_div(S, 1024u);
  uint64_t n = 0u, k = 0u;
  for (uint32_t i = 0u; i < run; ++i) {
    const uint64_t s = static_cast<uint64_t>(tid) * run + i;
    if (s >= S) break;
    const PageSeq q = page_seq(held, fresh, s, page, P);
    n += q.fresh;
    k += q.take;
  }
  // a scan of the waves, then of their sums
  uint64_t in = n, ik = k;
#pragma unroll
  for (uint32_t off = 1u; off < 64u; off <<= 1) {
    const uint64_t un = __shfl_up(in, off, 64), uk = __shfl_up(ik, off, 64);
    if ((tid & 63u) >= off) {
      in += un;
      ik += uk;
    }
  }
  __shared__ uint64_t sums[2][16];
  if ((tid & 63u) == 63u) {
    sums[0][tid >> 6] = in;
    sums[1][tid >> 6] = ik;
  }
  __syncthreads();
  for (uint32_t w = 0u; w < (tid >> 6); ++w) {
    in += sums[0][w];
    ik += sums[1][w];
  }
  tokens[tid + 1u] = in;
  pages[tid + 1u] = ik;
  if (tid == 0u) tokens[0] = pages[0] = 0u;
  __syncthreads();
  const int64_t from = first[0];
  if (blockIdx.x == 0u) {
    uint64_t at = in - n;
    for (uint32_t i = 0u; i < run; ++i) {
      const uint64_t s = static_cast<uint64_t>(tid) * run + i;
      if (s >= S) break;
      const PageSeq q = page_seq(held, fresh, s, page, P);
      starts[s] = page_int(at);
      lens[s] = page_int(static_cast<uint64_t>(q.held) + q.fresh);
      at += q.fresh;
    }
    if (tid == 0u) {
      starts[S] = page_int(tokens[1024]);
      next[0] = page_int(static_cast<uint64_t>(from < 0 ? 0 : from) + pages[1024]);
    }
  }
  for (uint64_t t = blockIdx.x * 1024ull + tid; t < T; t += gridDim.x * 1024ull) {
    if (t >= tokens[1024]) {
      pos[t] = slot[t] = -1;
      continue;
    }
    const uint32_t lo = page_run(tokens, t);
    uint64_t at = tokens[lo], taken = pages[lo];
    uint64_t s = static_cast<uint64_t>(lo) * run;
    PageSeq q = page_seq(held, fresh, s, page, P);
    while (t >= at + q.fresh && s + 1u < S) {  // ends: the run holds token t
      at += q.fresh;
      taken += q.take;
      q = page_seq(held, fresh, ++s, page, P);
    }
    const uint32_t p = q.held + static_cast<uint32_t>(t - at), col = p / page, in_page = p - col * page;
    int32_t e = -1;
    if (col < P) {
      if (col < q.have) {
        e = table[s * P + col];
      } else {
        e = page_taken(free_pages, F, from, taken + (col - q.have));
        if (in_page == 0u) table[s * P + col] = e;
      }
    }
    pos[t] = static_cast<int32_t>(p);
    slot[t] = e < 0 ? -1 : static_cast<int32_t>(static_cast<uint32_t>(e) * page + in_page);
  }
  if (tokens[1024] <= T) return;
  // The columns whose first token is none of the batch's.
  for (uint64_t k = blockIdx.x * 1024ull + tid; k < pages[1024]; k += gridDim.x * 1024ull) {
    const uint32_t lo = page_run(pages, k);
    uint64_t at = tokens[lo], taken = pages[lo];
    uint64_t s = static_cast<uint64_t>(lo) * run;
    PageSeq q = page_seq(held, fresh, s, page, P);
    while (k >= taken + q.take && s + 1u < S) {  // ends: the run holds column k
      at += q.fresh;
      taken += q.take;
      q = page_seq(held, fresh, ++s, page, P);
    }
    const uint32_t col = q.have + static_cast<uint32_t>(k - taken);
    if (at + (static_cast<uint64_t>(col) * page - q.held) >= T) table[s * P + col] = page_taken(free_pages, F, from, k);
  }
}

// ---------------------------------------------------------------- rotary
// A pair (a, b) of a head turned by pos freq_i: scale (a c - b s, b c + a s); the
// gradient's turn is the other way round. The angle's product and its turns are
// in 64 bits (in 32, a position of a million is off by 0.06 of a radian); what
// is left of an eighth of a turn goes through the Taylor series of sine and
// cosine, 2e-9 off.
__device__ __forceinline__ float2 rotary_angle(int32_t pos, float freq) {
  const double turns = static_cast<double>(pos) * static_cast<double>(freq) * 0.15915494309189533577;
  const double r = turns - __builtin_rint(turns);  // within half a turn
  const double quarter = __builtin_rint(4.0 * r);
  const float x = static_cast<float>((r - 0.25 * quarter) * 6.28318530717958647693), z = x * x;
  float s = fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = fmaf(z, s, 1.0f / 120.0f);
  s = fmaf(z, s, -1.0f / 6.0f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = fmaf(z, c, -1.0f / 720.0f);
  c = fmaf(z, c, 1.0f / 24.0f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.0f);
  const int k = static_cast<int>(quarter) & 3;
  const float cs = (k & 1) != 0 ? s : c, sn = (k & 1) != 0 ? c : s;
  return float2{k == 1 || k == 2 ? -cs : cs, k >= 2 ? -sn : sn};
}

constexpr uint32_t kRotaryMost = 512;  // frequencies

// The cosines and sines of TOKENS tokens, in LDS.
template <uint32_t TOKENS>
struct RotaryTurns {
  float2 v[TOKENS][kRotaryMost];
  __device__ __forceinline__ void fill(const int32_t* pos, const float* freq, uint32_t t0, uint32_t T, uint32_t F, float scale, bool inverse) {
    for (uint32_t i = threadIdx.x; i < TOKENS * F; i += 256u) {
      const uint32_t n = i / F, f = i - n * F;
      if (t0 + n >= T) break;
      float2 a = rotary_angle(pos[t0 + n], freq[f]);
      a.x *= scale;
      a.y *= inverse ? -scale : scale;
      v[n][f] = a;
    }
    __syncthreads();
  }
};

// Part j of a row of D: V pairs (2 V values), or behind them V values as they
// are. Rows lie at any alignment; a lane reads both halves of its pairs before it
// stores them, so `to` may be `from`.
template <typename T, bool INTER>
struct RotaryRow {
  static constexpr uint32_t V = kRowE<T>;
  uint32_t F, D, pairs, parts;
  __device__ __forceinline__ RotaryRow(uint32_t F_, uint32_t D_) : F(F_), D(D_) {
    pairs = (F + V - 1u) / V;
    parts = pairs + (D - 2u * F + V - 1u) / V;
  }
  // turn nullptr: as they are
  __device__ __forceinline__ void part(const T* from, T* to, uint32_t j, const float2* turn) const {
    if (j >= pairs) {
      const uint32_t c = 2u * F + (j - pairs) * V;
      if (c + V <= D) {
        store_vec_any<T, V, false>(to + c, load_vec_any<T, V, false>(from + c));
      } else {
        for (uint32_t e = c; e < D; ++e) to[e] = from[e];
      }
      return;
    }
    const uint32_t f = j * V;
    if (f + V <= F) {
      vec<T, V> a, b;
      if constexpr (INTER) {
        a = load_vec_any<T, V, false>(from + 2u * f);
        b = load_vec_any<T, V, false>(from + 2u * f + V);
      } else {
        a = load_vec_any<T, V, false>(from + f);
        b = load_vec_any<T, V, false>(from + F + f);
      }
      if (turn != nullptr) {
#pragma unroll
        for (uint32_t e = 0; e < V; ++e) {
          if constexpr (INTER) {
            if (e % 2u != 0u) continue;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              vec<T, V>& w = half ? b : a;
              const float2 t = turn[f + half * (V / 2u) + e / 2u];
              const float x = static_cast<float>(w[e]), y = static_cast<float>(w[e + 1]);
              w.set(e, static_cast<T>(fmaf(x, t.x, -(y * t.y))));
              w.set(e + 1, static_cast<T>(fmaf(y, t.x, x * t.y)));
            }
          } else {
            const float2 t = turn[f + e];
            const float x = static_cast<float>(a[e]), y = static_cast<float>(b[e]);
            a.set(e, static_cast<T>(fmaf(x, t.x, -(y * t.y))));
            b.set(e, static_cast<T>(fmaf(y, t.x, x * t.y)));
          }
        }
      }
      if constexpr (INTER) {
        store_vec_any<T, V, false>(to + 2u * f, a);
        store_vec_any<T, V, false>(to + 2u * f + V, b);
      } else {
        store_vec_any<T, V, false>(to + f, a);
        store_vec_any<T, V, false>(to + F + f, b);
      }
      return;
    }
    for (uint32_t i = f; i < F; ++i) {
      const uint32_t p = INTER ? 2u * i : i, q = INTER ? 2u * i + 1u : F + i;
      const T a = from[p], b = from[q];
      if (turn == nullptr) {
        to[p] = a;
        to[q] = b;
        continue;
      }
      const float2 t = turn[i];
      const float x = static_cast<float>(a), y = static_cast<float>(b);
      to[p] = static_cast<T>(fmaf(x, t.x, -(y * t.y)));
      to[q] = static_cast<T>(fmaf(y, t.x, x * t.y));
    }
  }
};

// A workgroup takes TOKENS tokens: their angles once, then all of their heads. Bound by
// HBM: bf16 [8192, 32, 128] 21.0 us (6.4 TB/s), f32 of as many values 43.6 (6.2), heads of
// 77 with 3 pairs 4.4 TB/s (their pieces of 16 bytes lie across lines, the 3 pairs and the
// row's last 7 values move one by one); stores into pages, f16 [4096, 48, 128] 18.2 us (5.5 TB/s).
template <typename T, bool INTER, bool INVERSE, uint32_t TOKENS>
__device__ __forceinline__ void rotary(const T* x, const int32_t* pos, const float* freq, T* y, uint32_t Tn, uint32_t H, uint32_t D,
                                       uint32_t F, float scale) {
  __shared__ RotaryTurns<TOKENS> turns;
  const uint32_t t0 = blockIdx.x * TOKENS;
  turns.fill(pos, freq, t0, Tn, F, scale, INVERSE);
  const RotaryRow<T, INTER> row(F, D);
  const uint32_t some = Tn - t0 < TOKENS ? Tn - t0 : TOKENS, all = some * H * row.parts;
  for (uint32_t i = threadIdx.x; i < all; i += 256u) {
    const uint32_t r = i / row.parts, n = r / H;
    const uint64_t at = (static_cast<uint64_t>(t0) * H + r) * D;
    row.part(x + at, y + at, i - r * row.parts, turns.v[n]);
  }
}

// The same of a fused projection [T][HK G queries, HK keys, HK values][D]: queries
// to q, keys (turned) and values to their slot of the pages [PAGES][HK][PAGE][D].
template <typename T, bool INTER, uint32_t TOKENS>
__device__ __forceinline__ void rotary_cache(const T* x, const int32_t* pos, const int32_t* slot, const float* freq, T* q, T* k, T* v,
                                             uint32_t Tn, uint32_t HK, uint32_t G, uint32_t D, uint32_t F, uint32_t PAGES, uint32_t PAGE,
                                             float scale) {
  __shared__ RotaryTurns<TOKENS> turns;
  const uint32_t t0 = blockIdx.x * TOKENS;
  turns.fill(pos, freq, t0, Tn, F, scale, false);
  const RotaryRow<T, INTER> row(F, D);
  const uint32_t H = HK * (G + 2u), some = Tn - t0 < TOKENS ? Tn - t0 : TOKENS, all = some * H * row.parts;
  for (uint32_t i = threadIdx.x; i < all; i += 256u) {
    const uint32_t r = i / row.parts, n = r / H, h = r - n * H;
    const T* from = x + (static_cast<uint64_t>(t0) * H + r) * D;
    if (h < HK * G) {
      row.part(from, q + (static_cast<uint64_t>(t0 + n) * HK * G + h) * D, i - r * row.parts, turns.v[n]);
      continue;
    }
    const int32_t at = slot[t0 + n];
    if (at < 0 || PAGE == 0u) continue;  // pages of no tokens have no slot
    const uint32_t p = static_cast<uint32_t>(at) / PAGE, o = static_cast<uint32_t>(at) - p * PAGE;
    if (p >= PAGES) continue;
    const bool value = h >= HK * (G + 1u);
    const uint32_t head = h - HK * G - (value ? HK : 0u);
    T* to = (value ? v : k) + ((static_cast<uint64_t>(p) * HK + head) * PAGE + o) * D;
    row.part(from, to, i - r * row.parts, value ? nullptr : turns.v[n]);
  }
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_POSITIONS_H_
