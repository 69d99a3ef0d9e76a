// attention.h — attention of new tokens over a paged cache (family A).
//
//   y[r] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q_r . k_j - m),  over the keys j that row r sees
//
// Rows of a sequence and a key head: r = i G + g, query i of its n new tokens,
// head g of the group that shares the key head, so that one read of the keys
// serves the whole group. Query i of a cache of L tokens sits at L - n + i and
// sees the keys up to its own position (the last `window` of them).
//
// Scores are computed transposed, S^T = K Q^T (v_mfma_f32_32x32x16): a lane
// then holds 16 keys of ONE row, so that the softmax is a chain within the
// lane and one exchange with lane ^ 32, the running maximum and sum are a
// register each, and the probabilities are already the B operand of O^T = V^T
// P^T: its k slots of a lane half are keys 4h + {0..3, 8..11} of 16, which the
// transposing LDS read of V takes in the same order. Only the
// softmax passes through the vector ALU.
//
// One token over 8000 to 16000 keys of 8 heads of 128 (bf16): 21-22 us and 8.4-8.8 of the
// join for HBM's 6; 64 sequences of half as many keys: 272-278 and 6, 5.7 TB/s. Four chunks of
// 512 over 8000 to 16000 keys, 8 heads of a group: 409-440 us and 16 (the matrix cores busy for
// 49% of the cycles; calls, whose clocks are higher than a trace's, 413 in all, 0.97 PFLOP/s);
// prompts of 4096 (f16) 395-406 and 16 (calls 392, 0.70). Heads of 256, one wave a SIMD: as
// many bytes of single tokens 273-278 and 8, prompts of as many operations 559-567 and 15.
// Everything runs once, but rows of a tile that a value which is not finite has got into
// though they do not see it: without the matrix cores (redo_rows).
//
// Lengths lie on the GPU, so the launch knows shapes only: every workgroup of
// a fixed grid reads the lengths, counts the work of all sequences in units
// (a tile of rows by a block of keys) and takes an equal run of them. A run
// may end inside a tile: its sums go to the workspace, and join_attention adds
// the parts of such tiles, in the order of their keys (no atomics; the same
// bits every time).
#ifndef TCA_HIP_ATTENTION_H_
#define TCA_HIP_ATTENTION_H_

#include "tca/hip/device.h"
#include "tca/hip/gemm.h"

namespace tca {
namespace hip {

constexpr uint32_t kAttendGroups = 256;  // workgroups: one a CU
// Rows of a sequence and key head that waves split the keys of. (bf16, 8 key heads of 128: 8
// sequences of 16 rows over 4000 to 8000 keys 45 us so and 49 as tiles of many rows, of 32
// rows 49 both, 64 of 4 rows 291 and 288, one of 32 over 16000 36.4 and 36.9. Calls of 64
// sequences with 4, 16, 32 rows 293, 339, 358, with 36, 64, 128, 256 as tiles 357, 364, 383, 518:
// waves of a tile that have no rows cost nothing while the keys come from HBM.)
constexpr uint32_t kAttendFew = 32;
// Waves of a workgroup: two on a SIMD, each the softmax beside the other's matrix
// products, in 256 registers; one where a wave's sums and queries need more. (One
// wave a SIMD of 64 rows: chunks of 512 1866 us before the loads were counted by
// hand; 32 rows of eight waves 581, with loads and operands ahead 471, in the two
// phases of attend_many 426.)
template <uint32_t DP>
constexpr uint32_t kAttendWaves = DP <= 128u ? 8u : 4u;
template <uint32_t DP>
constexpr uint32_t kFewKeys = 32u * kAttendWaves<DP>;  // a unit of few rows: 32 keys for each wave
template <uint32_t DP>
constexpr uint32_t kAttendRows = 32u * kAttendWaves<DP>;  // a tile of many rows: 32 for each wave
constexpr uint32_t kManyKeys = 64;       // a unit of many rows
constexpr uint32_t kNoRow = 0xffffffffu;

// What is not loaded of a cache: rows behind a sequence, of no page, columns past D.
static __device__ __attribute__((aligned(16))) const uint32_t kAttendZero[4] = {0u, 0u, 0u, 0u};

__device__ __forceinline__ uint32_t attend_uniform(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); }

// One launch's sizes and lengths.
struct AttendShape {
  const int32_t* table;   // [S][P]
  const int32_t* starts;  // [S + 1]
  const int32_t* lens;    // [S]
  uint32_t T, HK, G, D, PAGES, PAGE, S, P, window;  // window 0: none
};

// One sequence: its rows in the batch and its place in the cache.
struct AttendSeq {
  uint32_t start, n, limit;  // first row, rows in the batch, keys that the table can name
  int32_t base;              // the first new token's position
};
__device__ __forceinline__ AttendSeq attend_seq(const AttendShape& a, uint32_t s) {
  AttendSeq q;
  const int32_t b = a.starts[s], e = a.starts[s + 1u], len = a.lens[s];
  const uint32_t T = a.T < 0x7fffffffu ? a.T : 0x7fffffffu;
  q.start = b < 0 ? 0u : static_cast<uint32_t>(b) < T ? static_cast<uint32_t>(b) : T;
  const uint32_t end = e < 0 ? 0u : static_cast<uint32_t>(e) < T ? static_cast<uint32_t>(e) : T;
  q.n = end > q.start ? end - q.start : 0u;
  const uint32_t L = len < 0 ? 0u : static_cast<uint32_t>(len);
  const uint64_t room = a.PAGES == 0u ? 0u : static_cast<uint64_t>(a.P) * a.PAGE;
  q.limit = L < room ? L : static_cast<uint32_t>(room);
  // Rows behind the batch are none of it but count for the others' positions. (Those
  // before row 0 do not: positions are counted from the last row.)
  q.base = q.n == 0u ? 0 : static_cast<int32_t>(L) - (e - static_cast<int32_t>(q.start));
  return q;
}

// Key blocks of KB that tokens t0 .. t1 - 1 of a sequence see. (A position is
// below 2^31 and above -2^31, so that differences of positions fit.)
struct AttendSpan {
  uint32_t first, blocks;
};
__device__ __forceinline__ uint32_t attend_end(const AttendSeq& q, uint32_t t1) {  // keys below it are seen by token t1 - 1 at most
  const int32_t last = q.base + static_cast<int32_t>(t1);
  return last <= 0 ? 0u : static_cast<uint32_t>(last) < q.limit ? static_cast<uint32_t>(last) : q.limit;
}
__device__ __forceinline__ uint32_t attend_begin(const AttendShape& a, const AttendSeq& q, uint32_t t0) {  // keys from it on are seen by token t0
  const int32_t last = q.base + static_cast<int32_t>(t0) + 1;
  return a.window == 0u || last <= 0 || static_cast<uint32_t>(last) <= a.window ? 0u : static_cast<uint32_t>(last) - a.window;
}
template <uint32_t KB>
__device__ __forceinline__ AttendSpan attend_span(const AttendShape& a, const AttendSeq& q, uint32_t t0, uint32_t t1) {
  const uint32_t hi = attend_end(q, t1), lo = attend_begin(a, q, t0);
  AttendSpan p = {lo / KB, 0u};
  if (hi > lo) p.blocks = (hi - 1u) / KB + 1u - p.first;
  return p;
}

// The rows of tiles: `tokens` of a sequence by `heads` of a group, `groups` such parts of it.
struct AttendRows {
  uint32_t tokens, heads, groups;
};
__device__ __forceinline__ AttendRows attend_rows(uint32_t G, uint32_t BM) {
  AttendRows r;
  r.heads = G < BM ? G : BM;
  r.groups = (G - 1u) / r.heads + 1u;
  r.tokens = BM / r.heads;
  return r;
}

// Units of a sequence: a tile that sees no key is one too, since its rows are
// stored. Few rows (MANY false) are one tile a key head.
__device__ __forceinline__ bool attend_is_many(const AttendShape& a, const AttendSeq& q) {
  return static_cast<uint64_t>(q.n) * a.G > kAttendFew;
}
// Of one key head (and part of a group): the tiles j, j + lanes, .. of a sequence.
template <bool MANY, uint32_t DP>
__device__ __forceinline__ uint64_t attend_units(const AttendShape& a, const AttendSeq& q, uint32_t j, uint32_t lanes) {
  if (q.n == 0u || attend_is_many(a, q) != MANY) return 0u;
  const uint32_t tokens = MANY ? attend_rows(a.G, kAttendRows<DP>).tokens : q.n, tiles = (q.n - 1u) / tokens + 1u;
  uint64_t sum = 0u;
  for (uint32_t i = j; i < tiles; i += lanes) {
    const uint32_t t0 = i * tokens, t1 = q.n - t0 < tokens ? q.n : t0 + tokens;
    const uint32_t b = attend_span<MANY ? kManyKeys : kFewKeys<DP>>(a, q, t0, t1).blocks;
    sum += b == 0u ? 1u : b;
  }
  return sum;
}

// Units before each of 256 entries. Up to 256 sequences have `lanes` entries each,
// whose tiles they share; of more, an entry has `run`.
struct AttendCount {
  uint64_t before[2][257], sums[2][4];
  uint32_t odd[2];  // whether sums of a run were not finite
};
struct AttendRuns {
  uint32_t run, lanes;
};
__device__ __forceinline__ AttendRuns attend_runs(uint32_t S) {
  AttendRuns r = {ceil_div(S, 256u), 1u};
  while (r.run <= 1u && S != 0u && S * r.lanes * 2u <= 256u) r.lanes *= 2u;
  return r;
}
template <uint32_t DP>
__device__ __forceinline__ void attend_count(const AttendShape& a, AttendCount* c) {
  const uint32_t tid = threadIdx.x;
  const AttendRuns r = attend_runs(a.S);
  const bool counts = tid < 256u;
  uint64_t few = 0u, many = 0u;
  const bool any = static_cast<uint64_t>(a.T) * a.G > kAttendFew;  // whether a sequence can have many rows
  const uint64_t heads = any ? a.HK * static_cast<uint64_t>(attend_rows(a.G, kAttendRows<DP>).groups) : 0u;
  for (uint32_t i = 0u; counts && i < r.run; ++i) {
    const uint64_t s = static_cast<uint64_t>(tid / r.lanes) * r.run + i;
    if (s >= a.S) break;
    const AttendSeq q = attend_seq(a, static_cast<uint32_t>(s));
    few += attend_units<false, DP>(a, q, tid % r.lanes, r.lanes) * a.HK;
    if (any) many += attend_units<true, DP>(a, q, tid % r.lanes, r.lanes) * heads;
  }
  // a scan of each wave, then the sums of the waves before it
#pragma unroll
  for (uint32_t off = 1u; off < 64u; off <<= 1) {
    const uint64_t f = __shfl_up(few, off, 64), m = __shfl_up(many, off, 64);
    if ((tid & 63u) >= off) {
      few += f;
      many += m;
    }
  }
  if (counts && (tid & 63u) == 63u) {
    c->sums[0][tid >> 6] = few;
    c->sums[1][tid >> 6] = many;
  }
  __syncthreads();
  if (counts) {
    for (uint32_t w = 0u; w < (tid >> 6); ++w) {
      few += c->sums[0][w];
      many += c->sums[1][w];
    }
    c->before[0][tid + 1u] = few;
    c->before[1][tid + 1u] = many;
  }
  if (tid == 0u) {
    c->before[0][0] = c->before[1][0] = 0u;
    c->odd[0] = c->odd[1] = 0u;
  }
  __syncthreads();
}

// The tile that holds unit u.
struct AttendTile {
  AttendSeq q;
  uint32_t s, h, g0, heads, stride;  // sequence, key head, first head of the group, their number, rows a token
  uint32_t t0, t1;                   // its tokens
  uint64_t first, end;               // its units
  AttendSpan span;
};
// The rest of a tile from its sequence, heads, t0 and first unit.
template <bool MANY, uint32_t DP>
__device__ __forceinline__ void attend_place(const AttendShape& a, const AttendRows& r, AttendTile& t) {
  t.stride = MANY ? r.heads : a.G;
  t.heads = a.G - t.g0 < t.stride ? a.G - t.g0 : t.stride;
  t.t1 = MANY && t.q.n - t.t0 > r.tokens ? t.t0 + r.tokens : t.q.n;
  t.span = attend_span<MANY ? kManyKeys : kFewKeys<DP>>(a, t.q, t.t0, t.t1);
  t.end = t.first + (t.span.blocks == 0u ? 1u : t.span.blocks);
}
__device__ __forceinline__ uint64_t attend_uniform64(uint64_t v) {
  return static_cast<uint64_t>(attend_uniform(static_cast<uint32_t>(v))) |
         (static_cast<uint64_t>(attend_uniform(static_cast<uint32_t>(v >> 32))) << 32);
}
__device__ __forceinline__ uint64_t attend_divide(uint64_t a, uint64_t b) {
  return ((a | b) >> 32) == 0u ? static_cast<uint32_t>(a) / static_cast<uint32_t>(b) : a / b;
}
template <bool MANY, uint32_t DP>
__device__ __forceinline__ AttendTile attend_tile(const AttendShape& a, const AttendCount& c, uint64_t u) {
  const uint64_t* before = c.before[MANY ? 1 : 0];
  const AttendRuns runs = attend_runs(a.S);
  uint32_t lo = 0u;  // the entries from 1 on that begin at u or before it
#pragma unroll
  for (uint32_t e = 0u; e < 256u; e += 64u) {
    const uint32_t i = e + (threadIdx.x & 63u) + 1u;
    lo += static_cast<uint32_t>(__popcll(__builtin_amdgcn_ballot_w64(i * runs.lanes < 256u && before[i * runs.lanes < 256u ? i * runs.lanes : 0u] <= u)));
  }
  lo = attend_uniform(lo);
  uint64_t at = attend_uniform64(before[lo * runs.lanes]);
  const uint64_t entry = attend_uniform64(before[(lo + 1u) * runs.lanes]) - at;
  const AttendRows r = attend_rows(a.G, kAttendRows<DP>);
  const uint32_t parts = MANY ? r.groups : 1u;
  AttendTile t = {};
  for (t.s = lo * runs.run;; ++t.s) {  // ends: the run holds unit u
    t.q = attend_seq(a, t.s);
    const uint64_t heads = static_cast<uint64_t>(a.HK) * parts;
    const uint64_t one = runs.run == 1u ? attend_divide(entry, heads) : attend_units<MANY, DP>(a, t.q, 0u, 1u), all = one * heads;
    if (u >= at + all && t.s + 1u < a.S) {
      at += all;
      continue;
    }
    const uint32_t which = static_cast<uint32_t>(attend_divide(u - at, one));
    t.h = which / parts;
    t.g0 = which % parts * r.heads;
    at += one * which;
    break;
  }
  for (t.first = at;; t.first = t.end, t.t0 = t.t1) {
    attend_place<MANY, DP>(a, r, t);
    if (u < t.end || t.t1 == t.q.n) break;
  }
  return t;
}
// The tile after t, which holds unit t.end.
template <bool MANY, uint32_t DP>
__device__ __forceinline__ void attend_next(const AttendShape& a, const AttendCount& c, AttendTile& t) {
  const AttendRows r = attend_rows(a.G, kAttendRows<DP>);
  const bool more = t.t1 < t.q.n, group = MANY && t.g0 + t.stride < a.G;
  if (!more && !group && t.h + 1u == a.HK) {
    t = attend_tile<MANY, DP>(a, c, t.end);
    return;
  }
  t.t0 = more ? t.t1 : 0u;
  if (!more) {
    t.h += group ? 0u : 1u;
    t.g0 = group ? t.g0 + t.stride : 0u;
  }
  t.first = t.end;
  attend_place<MANY, DP>(a, r, t);
}
// Units of a workgroup.
__device__ __forceinline__ uint64_t attend_run(uint64_t units) { return (units + kAttendGroups - 1u) / kAttendGroups; }

// The rows of a tile in memory (in rows of D): tokens from `token` on by heads from g0 on.
struct AttendPlace {
  uint32_t token, tokens, stride, heads, g0, h;
  // row r, or kNoRow
  __device__ __forceinline__ uint32_t row(const AttendShape& a, uint32_t r) const {
    const uint32_t i = r / stride, g = r - i * stride;
    if (i >= tokens || g >= heads) return kNoRow;
    return ((token + i) * a.HK + h) * a.G + g0 + g;
  }
};
__device__ __forceinline__ AttendPlace attend_place_of(const AttendTile& t) {
  return {t.q.start + t.t0, t.t1 - t.t0, t.stride, t.heads, t.g0, t.h};
}
__device__ __forceinline__ uint32_t attend_row(const AttendShape& a, const AttendTile& t, uint32_t r) { return attend_place_of(t).row(a, r); }
// Its position.
__device__ __forceinline__ int32_t attend_pos(const AttendTile& t, uint32_t r) {
  const uint32_t i = r / t.stride, last = t.t1 - t.t0 - 1u;
  return t.q.base + static_cast<int32_t>(t.t0 + (i < last ? i : last));
}

// -------------------------------------------------------------- operands

typedef short i16x8_t __attribute__((ext_vector_type(8)));

template <bool F16>
__device__ __forceinline__ f32x16 mfma_32x32x16(const bf16x8& a, const bf16x8& b, const f32x16& c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t attend_lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) void*)p));
}

// Rows of DP elements (NC chunks of 16 bytes) in LDS. A lane reads a chunk of
// its own row of K: 16 rows of a phase cover the banks when the chunk is XORed
// with the row (rows of 128 and 384 bytes: pairs of rows do already). The
// transposing read takes 64 bytes of four rows: their 64-byte groups are XORed.
template <uint32_t DP>
struct AttendLds {
  static constexpr uint32_t NC = DP / 8u;
  static constexpr bool kPairs = NC % 16u != 0u;
  // Chunk pairs of K and 64-byte groups of V whose place differs from the first's in
  // the XORed bits alone: rows start at multiples of those bits.
  static constexpr uint32_t kXorK = kPairs ? 4u : 8u, kXorV = kPairs ? 2u : 4u;
  static __device__ __forceinline__ uint32_t swz_k(uint32_t row) { return kPairs ? (row >> 1) & 7u : row & 15u; }
  static __device__ __forceinline__ uint32_t swz_v(uint32_t row) { return kPairs ? ((row >> 1) & 1u) << 2 : (row & 3u) << 2; }
};

// 16 bytes a lane from global memory into a 1 KiB chunk of LDS, counted by vmcnt
// alone: the wave that waits for its count (attend_wait) reads them. In asm,
// since the compiler has every read of LDS wait for every such load before it.
// (M0 is read a state after it is written, and put back as the compiler had it.)
__device__ __forceinline__ void attend_load(const uint4* g, uint16_t* lds) {
  const uint32_t to = attend_uniform(attend_lds_address(lds));
  uint32_t kept;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, off\n\ts_mov_b32 m0, %0"
               : "=&s"(kept) : "s"(to), "v"(g) : "memory");
}
// At most VM of the wave's loads are left in flight, and no read of LDS.
template <int VM>
__device__ __forceinline__ void attend_wait() {
  static_assert(VM < 64, "counted loads");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(VM) : "memory");
}

// Chunks i WAVES + wave of a block of KEYS rows of the cache, into LDS: rows[]
// has each key's row in 16-byte units, or kNoRow.
template <uint32_t DP, uint32_t KEYS, uint32_t WAVES>
struct AttendFill {
  using L = AttendLds<DP>;
  static constexpr uint32_t N = KEYS * L::NC / 64u / WAVES;
  static_assert(KEYS * L::NC % (64u * WAVES) == 0u, "whole loads");
  uint32_t off[N];
  __device__ __forceinline__ AttendFill(const uint32_t* rows, uint32_t wave, uint32_t lane) {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) off[i] = rows[((i * WAVES + wave) * 64u + lane) / L::NC];
  }
  template <bool VALUES>
  __device__ __forceinline__ void load_one(uint32_t i, const uint4* __restrict__ cache, const uint4* __restrict__ zero, uint16_t* lds,
                                           uint32_t chunks, uint32_t wave, uint32_t lane) const {
    const uint32_t at = (i * WAVES + wave) * 64u + lane, row = at / L::NC, slot = at % L::NC;
    const uint32_t chunk = slot ^ (VALUES ? L::swz_v(row) : L::swz_k(row));
    attend_load(((off[i] != kNoRow) & (chunk < chunks)) ? cache + (static_cast<uint64_t>(off[i]) + chunk) : zero, lds + (i * WAVES + wave) * 512u);
  }
  template <bool VALUES>
  __device__ __forceinline__ void load(const uint4* __restrict__ cache, const uint4* __restrict__ zero, uint16_t* lds, uint32_t chunks,
                                       uint32_t wave, uint32_t lane) const {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) load_one<VALUES>(i, cache, zero, lds, chunks, wave, lane);
  }
};
template <uint32_t DP, uint32_t KEYS, uint32_t WAVES>
constexpr int attend_loads() {
  return static_cast<int>(KEYS * (DP / 8u) / 64u / WAVES);
}

// The row of key j in the cache, in 16-byte units.
__device__ __forceinline__ uint32_t attend_key(const AttendShape& a, const AttendTile& t, uint32_t j, uint32_t lo, uint32_t hi) {
  if (j < lo || j >= hi) return kNoRow;
  const uint32_t p = j / a.PAGE, o = j - p * a.PAGE;
  const int32_t e = a.table[static_cast<uint64_t>(t.s) * a.P + p];
  if (e < 0 || static_cast<uint32_t>(e) >= a.PAGES) return kNoRow;
  return ((static_cast<uint32_t>(e) * a.HK + t.h) * a.PAGE + o) * (a.D / 8u);
}

// The queries of 32 rows as the B operand of every 16 columns.
template <uint32_t DP>
struct AttendQ {
  bf16x8 v[DP / 16u];
  // All signs changed where `sign` has the two of a word set: once other loads have been waited for.
  __device__ __forceinline__ void turn(uint32_t sign) {
#pragma unroll
    for (uint32_t c = 0; c < DP / 16u; ++c) {
      const uint4 w = __builtin_bit_cast(uint4, v[c]);
      v[c] = __builtin_bit_cast(bf16x8, uint4{w.x ^ sign, w.y ^ sign, w.z ^ sign, w.w ^ sign});
    }
  }
};
template <uint32_t DP>
__device__ __forceinline__ void attend_load_q(AttendQ<DP>& q, const uint4* __restrict__ x, uint32_t row, uint32_t chunks, uint32_t lane) {
#pragma unroll
  for (uint32_t c = 0; c < DP / 16u; ++c) {
    const uint32_t chunk = 2u * c + (lane >> 5);
    uint4 w = {0u, 0u, 0u, 0u};
    if (row != kNoRow && chunk < chunks) w = x[static_cast<uint64_t>(row) * chunks + chunk];
    q.v[c] = __builtin_bit_cast(bf16x8, w);
  }
}

// The state of 32 rows: O^T, the reference of the exponents (log2), the lane's part
// of the sum.
template <uint32_t DP>
struct AttendAcc {
  f32x16 o[DP / 32u];
  float m, l;
};

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
// Probabilities are rounded to the inputs' type for the second product, as its
// operands are: an error of at most half a step (bf16 2^-8, f16 2^-11) of each, which averages out
// over the keys (outputs are off by 0.0023 of their size in bf16, 0.0017 of it
// their own rounding; f16 0.00026 and 0.0002). Their sum is of the unrounded ones.
// The reference of the exponents follows the running maximum only where that is
// more than 8 (a factor of 256) above it: rescaling O is then rare, and a
// probability is at most 256. f16 probabilities are 2^6 larger: less than
// 2^14, and what is lost below f16's smallest number is 2^-30 of the largest.
template <bool F16>
constexpr float kBoost = F16 ? 6.0f : 0.0f;

// Scores of KT x 32 keys for 32 rows.
template <bool F16, uint32_t DP, int KT>
__device__ __forceinline__ void attend_scores(f32x16 (&s)[KT], const AttendQ<DP>& q, const uint16_t* k, uint32_t lane) {
  using L = AttendLds<DP>;
  const uint32_t row = lane & 31u, h = lane >> 5;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) s[kt][i] = 0.0f;
  // Operands are read a group of chunks ahead of the products that take them.
  constexpr uint32_t C = 2u, N = DP / 16u / C;
  bf16x8 f[2][C][KT];
  const uint32_t at = attend_lds_address(k) + row * (2u * DP) + ((h ^ L::swz_k(row)) << 4);
  auto read = [&](uint32_t g) {
#pragma unroll
    for (uint32_t c = 0; c < C; ++c)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        const uint32_t j = g * C + c;
        f[g & 1u][c][kt] = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8*>((at ^ ((j % L::kXorK) << 5)) + j / L::kXorK * (L::kXorK * 32u) + 64u * DP * kt);
      }
  };
  read(0u);
#pragma unroll
  for (uint32_t g = 0; g < N; ++g) {
    if (g + 1u < N) read(g + 1u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t c = 0; c < C; ++c)
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) s[kt] = mfma_32x32x16<F16>(f[g & 1u][c][kt], q.v[g * C + c], s[kt]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Of a lane and lane ^ 32.
__device__ __forceinline__ float attend_halves_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float attend_halves_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Scores to probabilities, in 16 bits: p[kt][m] is the B operand of keys 16 m .. 16 m + 15.
// seen[kt]: which of 32 keys have a row (bits); whole: every key is seen by every row.
template <bool F16, uint32_t DP, int KT>
__device__ __forceinline__ void attend_softmax(const f32x16 (&s)[KT], bf16x8 (&p)[KT][2], AttendAcc<DP>& acc, float scale2,
                                               bool whole, const uint32_t (&seen)[KT], uint32_t key0, int32_t pos,
                                               uint32_t window, uint32_t lane) {
  const uint32_t h = lane >> 5;
  float v[KT][16];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) v[kt][i] = s[kt][i];
  if (!whole) {
    // Key key0 + 4 h + c of the lane's 32 kt + {0..3, 8..11, ..}: constants c against the row's place.
    int32_t last = pos - static_cast<int32_t>(key0 + 4u * h);
    asm volatile("" : "+v"(last));  // nothing of this is kept outside of the branch
    const int32_t before = window == 0u || window > 0x7fffffffu ? -1 : last - static_cast<int32_t>(window);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
      const uint32_t bits = seen[kt] >> (4u * h);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int32_t c = 8 * (i / 4) + i % 4;
        const bool sees = (bits & (1u << c)) != 0u && 32 * kt + c <= last && 32 * kt + c > before;
        v[kt][i] = sees ? v[kt][i] : -__builtin_inff();
      }
    }
  }
  float top = v[0][0];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, v[kt][i]);
  top = attend_halves_max(top) * scale2;
  if (__builtin_amdgcn_ballot_w64(top > acc.m + 8.0f) != 0u) {
    const float m = fmaxf(acc.m, top);
    const float f = m == acc.m ? 1.0f : __builtin_amdgcn_exp2f(acc.m - m);
    acc.m = m;
    acc.l *= f;
#pragma unroll
    for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc.o[d][i] *= f;
  }
  const float sh = (acc.m == -__builtin_inff() ? 0.0f : acc.m) - kBoost<F16>;
  float sum = 0.0f;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if constexpr (F16) {
        f16x8 w;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_amdgcn_exp2f(fmaf(v[kt][8 * m + e], scale2, -sh));
          sum += x;
          w[e] = static_cast<_Float16>(x);
        }
        p[kt][m] = __builtin_bit_cast(bf16x8, w);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = __builtin_amdgcn_exp2f(fmaf(v[kt][8 * m + e], scale2, -sh));
          sum += x;
          p[kt][m][e] = static_cast<__bf16>(x);
        }
      }
    }
  acc.l += sum;
}

// O^T += V^T P^T. The operands of 32 columns at a time, read ahead as those of the scores.
template <bool F16, uint32_t DP, int KT>
struct AttendV {
  using L = AttendLds<DP>;
  uint32_t at;
  bf16x8 f[2][KT][2];
  __device__ __forceinline__ AttendV(const uint16_t* v, uint32_t lane) {
    const uint32_t t = lane >> 4, j = lane & 15u, row = 4u * (t >> 1) + (j >> 2);
    at = attend_lds_address(v) + row * (2u * DP) + (j & 1u) * 8u + (((2u * (t & 1u) + ((j & 3u) >> 1)) ^ L::swz_v(row)) << 4);
  }
  __device__ __forceinline__ void read(uint32_t d) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    const uint32_t from = (at ^ ((d % L::kXorV) << 6)) + d / L::kXorV * (L::kXorV * 64u);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t r = from + (32u * kt + 16u * m) * (2u * DP);
        const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(r));
        const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(r + 16u * DP));
        const i16x8_t w = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        f[d & 1u][kt][m] = __builtin_bit_cast(bf16x8, w);
      }
  }
  // read(0) has been called.
  __device__ __forceinline__ void add(AttendAcc<DP>& acc, const bf16x8 (&p)[KT][2]) {
#pragma unroll
    for (uint32_t d = 0; d < DP / 32u; ++d) {
      if (d + 1u < DP / 32u) read(d + 1u);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int m = 0; m < 2; ++m) acc.o[d] = mfma_32x32x16<F16>(f[d & 1u][kt][m], p[kt][m], acc.o[d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// Whether sums of a row are not finite. A row that does not see a key has
// probability 0 for it, and the product of 0 and a value that is not finite is NaN:
// where rows of different positions share a block, a flag of the workgroup has those
// that this has happened to done again (redo_rows).
template <uint32_t DP>
__device__ __forceinline__ bool attend_odd(const AttendAcc<DP>& acc) {
  float z = 0.0f;
#pragma unroll
  for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) z += acc.o[d][i] - acc.o[d][i];
  return !(z == 0.0f);
}

// Both products of a phase, of 64 keys each and one tile of rows: O^T += V^T P^T of a
// block, S^T = K Q^T of the next. Groups of four products, their operands read two
// groups ahead, the first two of V ahead of the phase (`begin`): one group ahead, a
// phase took 1840 cycles, of which the products are 1024.
template <bool F16, uint32_t DP>
struct AttendPhase {
  using L = AttendLds<DP>;
  static constexpr uint32_t NV = DP / 32u, NK = DP / 32u, N = NV + NK;
  uint32_t v, k;  // the lane's places in the blocks
  bf16x8 f[3][4];
  __device__ __forceinline__ void begin(const uint16_t* vb, uint32_t lane) {
    const uint32_t t = lane >> 4, j = lane & 15u, row = 4u * (t >> 1) + (j >> 2);
    v = attend_lds_address(vb) + row * (2u * DP) + (j & 1u) * 8u + (((2u * (t & 1u) + ((j & 3u) >> 1)) ^ L::swz_v(row)) << 4);
#pragma unroll
    for (uint32_t j = 0; j < 8u; ++j) read(j / 4u, j % 4u);
  }
  __device__ __forceinline__ void keys(const uint16_t* kb, uint32_t lane) {
    const uint32_t row = lane & 31u;
    k = attend_lds_address(kb) + row * (2u * DP) + (((lane >> 5) ^ L::swz_k(row)) << 4);
  }
  // Operand j of group i. V: 32 keys (i odd: the upper ones) of 64 columns, those of one product after the other's.
  __device__ __forceinline__ void read(uint32_t i, uint32_t j) {
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    if (i < NV) {
      const uint32_t d = i / 2u * 2u + (j & 1u);
      const uint32_t r = (v ^ ((d % L::kXorV) << 6)) + d / L::kXorV * (L::kXorV * 64u) + (32u * (i & 1u) + 16u * (j >> 1)) * (2u * DP);
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(r));
      const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_i16x4*>(r + 16u * DP));
      const i16x8_t w = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      f[i % 3u][j] = __builtin_bit_cast(bf16x8, w);
    } else {
      const uint32_t c = (i - NV) * 2u + (j >> 1);
      f[i % 3u][j] = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8*>((k ^ ((c % L::kXorK) << 5)) + c / L::kXorK * (L::kXorK * 32u) +
                                                                                        64u * DP * (j & 1u));
    }
  }
  // FIRST: no V yet; LAST: no K any more. beside(i): issued beside the products of
  // group i. What is issued between two products fits the 32 cycles that one takes:
  // four products and then all else took 1660 cycles for 1024.
  template <bool FIRST, bool LAST, typename Beside>
  __device__ __forceinline__ void run(AttendAcc<DP>& acc, const bf16x8 (&p)[2][2], f32x16 (&s)[2], const AttendQ<DP>& q,
                                      const Beside& beside) {
    constexpr uint32_t from = FIRST ? NV : 0u, to = LAST ? NV : N;
    if constexpr (FIRST) {
#pragma unroll
      for (uint32_t j = 0; j < 8u; ++j) read(NV + j / 4u, j % 4u);
    }
#pragma unroll
    for (uint32_t i = from; i < to; ++i) {
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j) {
        __builtin_amdgcn_sched_barrier(0);
        if (i < NV) {
          const uint32_t d = i / 2u * 2u + (j & 1u);
          acc.o[d] = mfma_32x32x16<F16>(f[i % 3u][j], p[i & 1u][j >> 1], acc.o[d]);
        } else {
          const uint32_t c = (i - NV) * 2u + (j >> 1), kt = j & 1u;
          if (c == 0u) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[kt][e] = 0.0f;
          }
          s[kt] = mfma_32x32x16<F16>(f[i % 3u][j], q.v[c], s[kt]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (i + 2u < to) read(i + 2u, j);
        if (j == 1u) beside(i);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
};

// -------------------------------------------------------------- results

// What a launch writes: y, the statistics (or nullptr), the parts of tiles that
// several workgroups share: sums [2 kAttendGroups][rows][D], (reference, sum) of each row.
template <typename T>
struct AttendOut {
  T* y;
  float* lse;
  float* part;
  float2* ml;
  uint32_t* join;  // [kAttendGroups][8]: of the tile that starts in a workgroup's run and goes on in others', its parts and place; [7] is the flag of attend_odd
  uint32_t rows;
};
__device__ __forceinline__ uint32_t attend_part_rows(uint32_t T, uint32_t G, uint32_t most) {
  const uint64_t n = static_cast<uint64_t>(T) * G;
  return n < most ? static_cast<uint32_t>(n) : most;
}
template <bool F16>
__device__ __forceinline__ float attend_lse(float m, float l) {
  return l == 0.0f ? -__builtin_inff() : (m + (__builtin_log2f(l) - kBoost<F16>)) * kLn2;
}
// slot < 0: the rows themselves
template <bool F16, typename T>
__device__ __forceinline__ void attend_store(const AttendShape& a, const AttendPlace& t, const AttendOut<T>& out, int slot, uint32_t r,
                                             uint32_t d, const float (&v)[4], float m, float l) {
  const uint32_t row = t.row(a, r);
  if (row == kNoRow || d >= a.D) return;
  if (slot >= 0) {
    const uint64_t at = static_cast<uint64_t>(slot) * out.rows + r;
    *reinterpret_cast<float4*>(out.part + at * a.D + d) = float4{v[0], v[1], v[2], v[3]};
    if (d == 0u) out.ml[at] = float2{m, l};
    return;
  }
  const float f = l == 0.0f ? 0.0f : 1.0f / l;
  vec<T, 4> w;
#pragma unroll
  for (int e = 0; e < 4; ++e) w.set(e, static_cast<T>(v[e] * f));
  store_vec<T, 4>(out.y + static_cast<uint64_t>(row) * a.D + d, w);
  if (d == 0u && out.lse != nullptr) out.lse[row] = attend_lse<F16>(m, l);
}

__device__ __forceinline__ void attend_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ void attend_fence_reads() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }

// ------------------------------------------------------------- few rows
// At most 32 rows, the keys split over the waves too: each streams 32 keys of a
// unit through a ring of its own, without a barrier, and the waves' sums meet in LDS.
template <uint32_t DP>
struct FewLds {
  static constexpr uint32_t W = kAttendWaves<DP>;
  static constexpr int NS = DP <= 64u ? 2 : 1;
  static constexpr uint32_t kBlock = 32u * DP;                               // elements of K or V of a step
  static constexpr uint32_t kRing = W * NS * 2u * kBlock * 2u;               // bytes
  static constexpr uint32_t kSums = W * 32u * (DP + 4u) * 4u + W * 32u * 8u;  // the waves' sums, (m, l)
  static constexpr uint32_t kRows = 256u;                                    // keys whose rows a wave holds
  static constexpr uint32_t kHeld = kRing > kSums ? kRing : kSums;
  static constexpr uint32_t kBytes = kHeld + W * kRows * 4u + W * 32u * 4u;
};
template <bool F16, uint32_t DP, typename T>
__device__ __forceinline__ void attend_few(const AttendShape& a, const AttendTile& t, const AttendOut<T>& out, int slot,
                                           const uint4* __restrict__ q, const uint4* __restrict__ k, const uint4* __restrict__ v,
                                           const uint4* __restrict__ zero, float scale2, uint32_t sign, uint32_t first, uint32_t steps,
                                           unsigned char* lds, uint32_t* odd) {
  using F = FewLds<DP>;
  constexpr int kLoads = attend_loads<DP, 32u, 1u>(), kFlight = (2 * F::NS - 1) * kLoads;
  static_assert(kFlight < 64, "counted loads");
  constexpr uint32_t kSteps = F::kRows / 32u;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint16_t* ring = reinterpret_cast<uint16_t*>(lds) + wave * F::NS * 2u * F::kBlock;
  uint32_t* rows = reinterpret_cast<uint32_t*>(lds + F::kHeld) + wave * F::kRows;
  uint32_t* seen = reinterpret_cast<uint32_t*>(lds + F::kHeld + F::W * F::kRows * 4u) + wave * 32u;
  const uint32_t chunks = a.D / 8u;
  const uint32_t hi = attend_end(t.q, t.t1), lo = attend_begin(a, t.q, t.t0);

  AttendQ<DP> qv;
  attend_load_q<DP>(qv, q, attend_row(a, t, lane & 31u), chunks, lane);
  const int32_t pos = attend_pos(t, lane & 31u);
  const int32_t pos_min = t.q.base + static_cast<int32_t>(t.t0), pos_max = t.q.base + static_cast<int32_t>(t.t1) - 1;
  AttendAcc<DP> acc;
  acc.m = -__builtin_inff();
  acc.l = 0.0f;
#pragma unroll
  for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc.o[d][i] = 0.0f;

  // The rows of the next kSteps steps from step f on.
  auto refill = [&](uint32_t f) {
    attend_fence();
#pragma unroll
    for (uint32_t e = 0; e < F::kRows; e += 64u) {
      const uint32_t i = e + lane, step = f + i / 32u;
      const uint32_t r = step < steps ? attend_key(a, t, (first + step) * kFewKeys<DP> + wave * 32u + i % 32u, lo, hi) : kNoRow;
      rows[i] = r;
      const uint64_t has = __builtin_amdgcn_ballot_w64(r != kNoRow);
      if (lane < 2u) seen[(f + e / 32u + lane) % 32u] = lane == 0u ? static_cast<uint32_t>(has) : static_cast<uint32_t>(has >> 32);
    }
    attend_fence();
  };
  auto k_slot = [&](uint32_t n) { return ring + (n % F::NS) * 2u * F::kBlock; };
  auto fill_k = [&](uint32_t n) {
    AttendFill<DP, 32u, 1u>(rows + n % kSteps * 32u, 0u, lane).template load<false>(k, zero, k_slot(n), chunks, 0u, lane);
  };
  auto fill_v = [&](uint32_t n) {
    AttendFill<DP, 32u, 1u>(rows + n % kSteps * 32u, 0u, lane).template load<true>(v, zero, k_slot(n) + F::kBlock, chunks, 0u, lane);
  };
  refill(0u);
  qv.turn(sign);
#pragma unroll
  for (int n = 0; n < F::NS; ++n) {
    fill_k(n);
    fill_v(n);
  }
  for (uint32_t n = 0; n < steps; ++n) {
    const uint32_t next = n + F::NS, key0 = (first + n) * kFewKeys<DP> + wave * 32u;
    attend_wait<kFlight>();
    f32x16 s[1];
    attend_scores<F16, DP, 1>(s, qv, k_slot(n), lane);
    attend_fence_reads();  // the block's reads, before its slot is loaded again
    if (next % kSteps == 0u) refill(next);
    fill_k(next);
    const uint32_t has[1] = {attend_uniform(seen[n % 32u])};
    const bool whole = has[0] == 0xffffffffu && static_cast<int32_t>(key0 + 31u) <= pos_min &&
                       (a.window == 0u || static_cast<int64_t>(key0) + a.window > pos_max);
    bf16x8 p[1][2];
    attend_softmax<F16, DP, 1>(s, p, acc, scale2, whole, has, key0, pos, a.window, lane);
    attend_wait<kFlight>();
    AttendV<F16, DP, 1> vv(k_slot(n) + F::kBlock, lane);
    vv.read(0u);
    vv.add(acc, p);
    attend_fence_reads();
    fill_v(next);
  }
  attend_wait<0>();  // nothing in flight into LDS that is used again
  __syncthreads();
  constexpr uint32_t W = DP + 4u;
  float* sums = reinterpret_cast<float*>(lds);
  float2* ml = reinterpret_cast<float2*>(lds + F::W * 32u * W * 4u);
  acc.l = attend_halves_sum(acc.l);
  const uint32_t rows_here = (t.t1 - t.t0) * t.stride;
  if (t.t1 - t.t0 > 1u && (lane & 31u) < rows_here && attend_odd<DP>(acc)) *odd = 1u;
  if (lane < 32u) ml[wave * 32u + lane] = float2{acc.m, acc.l};
#pragma unroll
  for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((lane & 31u) < rows_here) *reinterpret_cast<float4*>(sums + (wave * 32u + (lane & 31u)) * W + 32u * d + 8u * i + 4u * (lane >> 5)) =
          float4{acc.o[d][4 * i], acc.o[d][4 * i + 1], acc.o[d][4 * i + 2], acc.o[d][4 * i + 3]};
  __syncthreads();
  const AttendPlace place = attend_place_of(t);
  const uint32_t count = rows_here * (DP / 4u);
  for (uint32_t i = tid; i < count; i += 64u * F::W) {
    const uint32_t r = i / (DP / 4u), d = i % (DP / 4u) * 4u;
    float m = -__builtin_inff(), l = 0.0f, f[F::W], o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t w = 0; w < F::W; ++w) m = fmaxf(m, ml[w * 32u + r].x);
#pragma unroll
    for (uint32_t w = 0; w < F::W; ++w) {
      const float2 p = ml[w * 32u + r];
      f[w] = p.x == m ? 1.0f : __builtin_amdgcn_exp2f(p.x - m);
      l += f[w] * p.y;
      const float4 x = *reinterpret_cast<const float4*>(sums + (w * 32u + r) * W + d);
      o[0] += f[w] * x.x;
      o[1] += f[w] * x.y;
      o[2] += f[w] * x.z;
      o[3] += f[w] * x.w;
    }
    attend_store<F16>(a, place, out, slot, r, d, o, m, l);
  }
  __syncthreads();
}

// ------------------------------------------------------------ many rows
// Waves of 32 rows, blocks of 64 keys in a ring that all of them read.
template <uint32_t DP>
struct ManyLds {
  static constexpr uint32_t W = kAttendWaves<DP>;
  static constexpr bool kTwo = W == 8u;  // two waves on a SIMD
  static constexpr int NS = kTwo ? 4 : DP <= 192u ? 3 : 2;
  static constexpr uint32_t kBlock = kManyKeys * DP;
  static constexpr uint32_t kRing = NS * 2u * kBlock * 2u;
  static constexpr uint32_t kRows = 1024u;
  static constexpr uint32_t kBytes = kRing + kRows * 4u + 64u * 4u;
};
template <bool F16, uint32_t DP, typename T>
__device__ __forceinline__ void attend_many(const AttendShape& a, const AttendTile& t, const AttendOut<T>& out, int slot,
                                            const uint4* __restrict__ q, const uint4* __restrict__ k, const uint4* __restrict__ v,
                                            const uint4* __restrict__ zero, float scale2, uint32_t sign, uint32_t first, uint32_t steps,
                                            unsigned char* lds, uint32_t* odd) {
  using M = ManyLds<DP>;
  constexpr int kLoads = 2 * attend_loads<DP, kManyKeys, M::W>();
  constexpr uint32_t kSteps = M::kRows / kManyKeys;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint16_t* ring = reinterpret_cast<uint16_t*>(lds);
  uint32_t* rows = reinterpret_cast<uint32_t*>(lds + M::kRing);
  uint32_t* seen = rows + M::kRows;  // of two times 16 steps
  const uint32_t chunks = a.D / 8u, mine = wave * 32u, all = (t.t1 - t.t0) * t.stride;
  const uint32_t hi = attend_end(t.q, t.t1), lo = attend_begin(a, t.q, t.t0);
  AttendQ<DP> qv;
  attend_load_q<DP>(qv, q, attend_row(a, t, mine + (lane & 31u)), chunks, lane);
  const int32_t pos = attend_pos(t, mine + (lane & 31u));
  AttendAcc<DP> acc;
  acc.m = -__builtin_inff();
  acc.l = 0.0f;
#pragma unroll
  for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc.o[d][e] = 0.0f;
  const int32_t pos_min = attend_pos(t, mine), pos_max = attend_pos(t, mine + 31u);

  // The rows of kSteps / 2 blocks from f on, in one half of rows[]: looked up, and stored when they have come.
  constexpr uint32_t kLook = M::kRows / 2u / (64u * M::W);
  uint32_t found[kLook];
  auto look = [&](uint32_t f) {
#pragma unroll
    for (uint32_t e = 0; e < kLook; ++e) {
      const uint32_t i = e * 64u * M::W + tid, step = f + i / kManyKeys;
      found[e] = step < steps ? attend_key(a, t, (first + step) * kManyKeys + i % kManyKeys, lo, hi) : kNoRow;
    }
  };
  auto keep = [&](uint32_t f) {
#pragma unroll
    for (uint32_t e = 0; e < kLook; ++e) {
      const uint32_t i = e * 64u * M::W + tid, step = f + i / kManyKeys;
      rows[f % kSteps * kManyKeys + i] = found[e];
      const uint64_t has = __builtin_amdgcn_ballot_w64(found[e] != kNoRow);
      if (lane < 2u) seen[2u * (step % 32u) + lane] = lane == 0u ? static_cast<uint32_t>(has) : static_cast<uint32_t>(has >> 32);
    }
  };
  auto refill = [&](uint32_t f) {
    look(f);
    keep(f);
  };
  // A step that ends with the rows of the blocks from n + 4 on.
  auto looks = [&](uint32_t n) { return (n + 4u) % (kSteps / 2u) == 0u; };
  auto block = [&](uint32_t n) { return ring + (n % M::NS) * 2u * M::kBlock; };
  using Fill = AttendFill<DP, kManyKeys, M::W>;
  auto rows_of = [&](uint32_t n) { return Fill(rows + n % kSteps * kManyKeys, wave, lane); };
  auto issue = [&](const Fill& f, uint32_t n) {
    f.template load<false>(k, zero, block(n), chunks, wave, lane);
    f.template load<true>(v, zero, block(n) + M::kBlock, chunks, wave, lane);
  };
  auto fill = [&](uint32_t n) { issue(rows_of(n), n); };
  auto barrier = [&]() {
    asm volatile("" : : : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
  };
  f32x16 s[2];
  bf16x8 p[2][2];
  // Whether any of the wave's rows sees block n.
  auto live = [&](uint32_t n) { return mine < all && static_cast<int32_t>((first + n) * kManyKeys) <= pos_max; };
  auto soften = [&](uint32_t n) {
    const uint32_t key0 = (first + n) * kManyKeys;
    const uint32_t has[2] = {attend_uniform(seen[2u * (n % 32u)]), attend_uniform(seen[2u * (n % 32u) + 1u])};
    const bool whole = (has[0] & has[1]) == 0xffffffffu && static_cast<int32_t>(key0 + kManyKeys - 1u) <= pos_min &&
                       (a.window == 0u || static_cast<int64_t>(key0) + a.window > pos_max);
    attend_softmax<F16, DP, 2>(s, p, acc, scale2, whole, has, key0, pos, a.window, lane);
  };
  auto nothing = [](uint32_t) {};
  refill(0u);
  qv.turn(sign);
  __syncthreads();
  if (steps == 0u) {
    // no key at all
  } else if constexpr (M::kTwo) {
    // Two phases a block: matrix products (of V with the last block's probabilities,
    // of K), then the softmax. Waves 4 to 7 run a phase behind waves 0 to 3, one of
    // either on each SIMD, so that the products of one stand beside the softmax of
    // the other, whatever the barriers align.
    // Block n is read from phase 2 n on and last in phase 2 n + 3 (its V, by the
    // waves behind). A wave issues block n + 2 at its step n, when block n - 2, whose
    // slot that is, has been read; waits, at the end of each phase of step n, until
    // its part of block n + 1 has landed; and looks up the rows of blocks from n + 4 on,
    // eight at a time, two steps before they are used. The loads are issued beside
    // the products (before them they took 500 cycles of a step of 4500).
    // (Blocks that a wave's rows do not see are masked, not skipped: a branch round the
    // products has the sums copied on both ways.)
    static_assert(!M::kTwo || 2u * Fill::N <= AttendPhase<F16, DP>::N, "a load beside each group");
    const bool behind = wave >= 4u;
    fill(0u);
    fill(1u);
    attend_wait<kLoads>();
    barrier();
    if (behind) barrier();
    auto turn = [&]() {
      attend_wait<kLoads>();
      barrier();
    };
    if (mine < all) {
      AttendPhase<F16, DP> phase;
      phase.keys(block(0u), lane);
      fill(2u);
      phase.template run<true, false>(acc, p, s, qv, nothing);
      turn();
      soften(0u);
      phase.begin(block(0u) + M::kBlock, lane);
      turn();
      for (uint32_t n = 1; n < steps; ++n) {
        const Fill f = rows_of(n + 2u);
        if (looks(n)) look(n + 4u);
        phase.keys(block(n), lane);
        uint16_t* to = block(n + 2u);
        __builtin_amdgcn_s_setprio(1);
        phase.template run<false, false>(acc, p, s, qv, [&](uint32_t i) {
          if (i < Fill::N) f.template load_one<false>(i, k, zero, to, chunks, wave, lane);
          else if (i < 2u * Fill::N) f.template load_one<true>(i - Fill::N, v, zero, to + M::kBlock, chunks, wave, lane);
        });
        __builtin_amdgcn_s_setprio(0);
        turn();
        soften(n);
        if (looks(n)) keep(n + 4u);
        phase.begin(block(n) + M::kBlock, lane);
        turn();
      }
      phase.template run<false, true>(acc, p, s, qv, nothing);
    } else {  // no rows: its loads alone
      fill(2u);
      turn();
      turn();
      for (uint32_t n = 1; n < steps; ++n) {
        if (looks(n)) look(n + 4u);
        fill(n + 2u);
        turn();
        if (looks(n)) keep(n + 4u);
        turn();
      }
    }
    if (!behind) barrier();
  } else {
#pragma unroll
    for (int n = 0; n < M::NS - 1; ++n) fill(n);
    for (uint32_t n = 0; n < steps; ++n) {
      attend_wait<(M::NS - 2) * kLoads>();
      barrier();
      if ((n + M::NS) % (kSteps / 2u) == 0u) refill(n + M::NS);
      fill(n + M::NS - 1u);
      if (live(n)) {
        attend_scores<F16, DP, 2>(s, qv, block(n), lane);
        soften(n);
        AttendV<F16, DP, 2> vv(block(n) + M::kBlock, lane);
        vv.read(0u);
        vv.add(acc, p);
      }
    }
  }
  attend_wait<0>();  // nothing in flight into LDS that is used again
  __syncthreads();
  const AttendPlace place = attend_place_of(t);
  acc.l = attend_halves_sum(acc.l);
  const uint32_t r = mine + (lane & 31u);
  if (t.t1 - t.t0 > 1u && r < all && attend_odd<DP>(acc)) *odd = 1u;
  if (slot >= 0) {
#pragma unroll
    for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float o[4] = {acc.o[d][4 * e], acc.o[d][4 * e + 1], acc.o[d][4 * e + 2], acc.o[d][4 * e + 3]};
        attend_store<F16>(a, place, out, slot, r, 32u * d + 8u * e + 4u * (lane >> 5), o, acc.m, acc.l);
      }
    return;
  }
  // A lane and lane ^ 32 hold four columns each of every eight of a row: they
  // exchange those of two eights, so that each stores 16 bytes.
  const uint32_t row = place.row(a, r);
  const float f = acc.l == 0.0f ? 0.0f : 1.0f / acc.l;
#pragma unroll
  for (uint32_t d = 0; d < DP / 32u; ++d)
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      vec<T, 4> x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) x[i].set(c, static_cast<T>(acc.o[d][4 * (e + i) + c] * f));
      const auto lo = __builtin_amdgcn_permlane32_swap(x[0].w[0], x[1].w[0], false, false);
      const auto hi = __builtin_amdgcn_permlane32_swap(x[0].w[1], x[1].w[1], false, false);
      const uint32_t c = 32u * d + 8u * (e + (lane >> 5));
      if (row != kNoRow && c < a.D)
        *reinterpret_cast<uint4*>(out.y + static_cast<uint64_t>(row) * a.D + c) = uint4{lo[0], hi[0], lo[1], hi[1]};
    }
  if (row != kNoRow && lane < 32u && out.lse != nullptr) out.lse[row] = attend_lse<F16>(acc.m, acc.l);
}

// ---------------------------------------------------------------- kernels

// Workgroups are dealt over the 8 XCDs in turn: neighbouring runs of units, which
// mostly read the same keys, go to one of them.
__device__ __forceinline__ uint32_t attend_group() { return blockIdx.x % 8u * (kAttendGroups / 8u) + blockIdx.x / 8u; }

template <bool F16, uint32_t DP, bool MANY, typename T>
__device__ __forceinline__ void attend_kind(const AttendShape& a, AttendCount& c, const AttendOut<T>& out, const uint4* __restrict__ q,
                                            const uint4* __restrict__ k, const uint4* __restrict__ v, const uint4* __restrict__ zero,
                                            float scale2, uint32_t sign, unsigned char* lds) {
  const uint32_t g = attend_group();
  const uint64_t units = c.before[MANY ? 1 : 0][256], run = attend_run(units), begin = run * g;
  const uint64_t end = begin + run < units ? begin + run : units;
  uint32_t* join = out.join + 8u * g;
  if (begin >= end) {
    if (threadIdx.x == 0u) join[0] = join[7] = 0u;
    return;
  }
  AttendTile t = attend_tile<MANY, DP>(a, c, begin);
  for (uint64_t u = begin;;) {
    const uint64_t stop = t.end < end ? t.end : end;
    // the rows themselves, or a part: of a tile from an earlier workgroup, or of one that goes on in the next
    const int slot = u == t.first && stop == t.end ? -1 : static_cast<int>(2u * g + (u == t.first ? 1u : 0u));
    const uint32_t first = t.span.first + static_cast<uint32_t>(u - t.first);
    const uint32_t steps = t.span.blocks == 0u ? 0u : static_cast<uint32_t>(stop - u);
    if constexpr (MANY) attend_many<F16, DP>(a, t, out, slot, q, k, v, zero, scale2, sign, first, steps, lds, c.odd + 1);
    else attend_few<F16, DP>(a, t, out, slot, q, k, v, zero, scale2, sign, first, steps, lds, c.odd);
    u = stop;
    if (u >= end) break;
    attend_next<MANY, DP>(a, c, t);
  }
  __syncthreads();
  if (threadIdx.x == 0u) {
    join[7] = c.odd[MANY ? 1 : 0];
    const bool shared = t.first >= begin && t.end > end;
    join[0] = shared ? static_cast<uint32_t>((t.end - end + run - 1u) / run) + 1u : 0u;
    if (shared) {
      const AttendPlace p = attend_place_of(t);
      const uint32_t w[6] = {p.token, p.tokens, p.stride, p.heads, p.g0, p.h};
#pragma unroll
      for (int i = 0; i < 6; ++i) join[1 + i] = w[i];
    }
  }
}

template <uint32_t DP>
constexpr uint32_t attend_lds() {
  return FewLds<DP>::kBytes > ManyLds<DP>::kBytes ? FewLds<DP>::kBytes : ManyLds<DP>::kBytes;
}

template <bool F16, uint32_t DP, typename T>
__device__ __forceinline__ void attend(const AttendShape& a, const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                       const uint4* __restrict__ zero, const AttendOut<T>& few, const AttendOut<T>& many, float scale) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[attend_lds<DP>()];  // (rows start at multiples of the XORed bits)
  __shared__ AttendCount c;
  attend_count<DP>(a, &c);
  const uint4 *q4 = reinterpret_cast<const uint4*>(q), *k4 = reinterpret_cast<const uint4*>(k), *v4 = reinterpret_cast<const uint4*>(v);
  // Its sign goes to the queries, so that the largest score stays the largest; 0
  // is a number so small that it makes every score 0, but leaves what is hidden -inf.
  const float size = __builtin_fabsf(scale) * kLog2e, scale2 = size < 1.17549435e-38f ? 1.17549435e-38f : size;
  const uint32_t sign = scale < 0.0f ? 0x80008000u : 0u;
  attend_kind<F16, DP, true>(a, c, many, q4, k4, v4, zero, scale2, sign, lds);
  attend_kind<F16, DP, false>(a, c, few, q4, k4, v4, zero, scale2, sign, lds);
}

// AT parts more of four columns of a row, from part p on: loaded together, then added.
struct JoinSum {
  float m = -__builtin_inff(), l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  template <uint32_t AT, typename T>
  __device__ __forceinline__ void add(const AttendOut<T>& out, uint32_t D, uint32_t g, uint32_t p, uint32_t parts, uint32_t r, uint32_t d) {
    float2 x[AT];
    float4 y[AT];
#pragma unroll
    for (uint32_t i = 0; i < AT; ++i) {
      const uint32_t which = p + i < parts ? p + i : parts - 1u;
      const uint64_t at = static_cast<uint64_t>(which == 0u ? 2u * g + 1u : 2u * (g + which)) * out.rows + r;
      x[i] = out.ml[at];
      y[i] = *reinterpret_cast<const float4*>(out.part + at * D + d);
    }
    float top = m;
#pragma unroll
    for (uint32_t i = 0; i < AT; ++i) top = fmaxf(top, x[i].x);
    const float f0 = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    m = top;
    l *= f0;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= f0;
#pragma unroll
    for (uint32_t i = 0; i < AT; ++i) {
      if (p + i >= parts) break;
      const float f = x[i].x == m ? 1.0f : __builtin_amdgcn_exp2f(x[i].x - m);
      l += f * x[i].y;
      o[0] += f * y[i].x;
      o[1] += f * y[i].y;
      o[2] += f * y[i].z;
      o[3] += f * y[i].w;
    }
  }
  template <typename T>
  __device__ __forceinline__ void all(const AttendOut<T>& out, uint32_t D, uint32_t g, uint32_t parts, uint32_t r, uint32_t d) {
    uint32_t p = 0u;
    for (; p + 8u <= parts; p += 8u) add<8u>(out, D, g, p, parts, r, d);
    for (; p < parts; p += 2u) add<2u>(out, D, g, p, parts, r, d);
  }
};
// The parts of the tile that starts in workgroup g's run and goes on in others',
// `slices` workgroups to a tile. Eight parts at a time, since one token over 16000 keys
// has 32 of them, and two where there are less: most tiles have two or three, and 16 at
// a time took 22 us for 5.
template <bool F16, typename T>
__device__ __forceinline__ void join_kind(const AttendShape& a, const AttendOut<T>& out) {
  const uint32_t slices = gridDim.x / kAttendGroups, g = blockIdx.x / slices, slice = blockIdx.x % slices;
  const uint32_t* w = out.join + 8u * g;
  const uint32_t parts = w[0];
  if (parts == 0u) return;
  if (w[2] > 1u) {  // redo_rows does what a flagged workgroup has a part of
    uint32_t odd = 0u;
    for (uint32_t p = 0u; p < parts; ++p) odd |= w[8u * p + 7u];
    if (odd != 0u) return;
  }
  const AttendPlace t = {w[1], w[2], w[3], w[4], w[5], w[6]};
  const uint32_t D4 = a.D / 4u, count = t.tokens * t.stride * D4;
  for (uint32_t i = slice * 256u + threadIdx.x; i < count; i += 256u * slices) {
    const uint32_t r = i / D4, d = i % D4 * 4u;
    if (t.row(a, r) == kNoRow) continue;
    JoinSum s;
    s.all(out, a.D, g, parts, r, d);
    attend_store<F16>(a, t, out, -1, r, d, s.o, s.m, s.l);
  }
}
// Which columns of the keys that some of a tile's rows see and others do not hold values
// that are not finite: the least such key and the one after the greatest, of all of them
// ([0], [1]) and of NaN alone.
struct AttendOdd {
  uint32_t bad[2][256], nan[2][256], rows[512];
};
// Whether what row's keys [lo, hi) give column d can be off: a key that it does not see
// holds such a value there, and none that it sees is known to be NaN (as its own key's is
// where a whole sequence is).
__device__ __forceinline__ bool attend_off(const AttendOdd& odd, uint32_t d, uint32_t lo, uint32_t hi) {
  if (odd.bad[0][d] >= lo && odd.bad[1][d] <= hi) return false;
  const uint32_t first = odd.nan[0][d], last = odd.nan[1][d];
  return !((first >= lo && first < hi) || (last > lo && last <= hi));
}
template <typename T>
__device__ __forceinline__ void attend_find_odd(const AttendShape& a, const AttendTile& t, const T* v, AttendOdd* odd) {
  const uint32_t tid = threadIdx.x, D4 = a.D / 4u;
  const uint32_t lo = attend_begin(a, t.q, t.t0), hi = attend_end(t.q, t.t1);
  // Every row sees the keys from `from` to `to` (the first row's own, which is looked at
  // all the same); there are less than 256 on either side.
  const uint32_t from = attend_begin(a, t.q, t.t1 - 1u), to = attend_end(t.q, t.t0 + 1u);
  const uint32_t back = to > lo ? to - 1u : lo;
  __syncthreads();  // the last tile's have been read
  odd->bad[0][tid] = odd->nan[0][tid] = 0xffffffffu;
  odd->bad[1][tid] = odd->nan[1][tid] = 0u;
  const uint32_t low = from < hi ? from : hi, before = low > lo ? low - lo : 0u, after = hi > back ? hi - back : 0u;
  for (uint32_t i = tid; i < before + after; i += 256u)
    odd->rows[i] = attend_key(a, t, i < before ? lo + i : back + (i - before), lo, hi);
  __syncthreads();
  for (uint32_t i = tid; i < (before + after) * D4; i += 256u) {
    const uint32_t n = i / D4, d = (i - n * D4) * 4u, off = odd->rows[n], key = n < before ? lo + n : back + (n - before);
    if (off == kNoRow) continue;
    const vec<T, 4> x = load_vec<T, 4>(v + static_cast<uint64_t>(off) * 8u + d);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = static_cast<float>(x[e]);
      if (f - f == 0.0f) continue;
      atomicMin(&odd->bad[0][d + e], key);
      atomicMax(&odd->bad[1][d + e], key + 1u);
      if (f == f) continue;
      atomicMin(&odd->nan[0][d + e], key);
      atomicMax(&odd->nan[1][d + e], key + 1u);
    }
  }
  __syncthreads();
}
// Of kRedo rows from r0 on, those of `which` by a wave over all that they see: 64 scores
// at a time, a lane each, then their values, four columns a lane. Bound by the latency of
// the loads: 30 us for 64 keys, by 32 waves a tile. (What stands here takes registers from
// the join of every launch: four rows at a time are 1.2 times as fast, in 88 to 98
// registers, with which the join of 64 single tokens takes 6.9 us for 6.1.)
constexpr uint32_t kRedo = 2;
template <bool F16, typename T>
__device__ __forceinline__ void redo_some(const AttendShape& a, const AttendTile& t, uint32_t r0, uint32_t which, const AttendOut<T>& out, const T* q,
                                          const T* k, const T* v, float scale2, uint32_t lane) {
  const uint32_t D8 = a.D / 8u, any = r0 + static_cast<uint32_t>(__builtin_ctz(which));
  uint32_t row[kRedo], lo[kRedo], hi[kRedo], least = 0xffffffffu, most = 0u;
  float m[kRedo], l[kRedo], o[kRedo][4];
#pragma unroll
  for (uint32_t i = 0; i < kRedo; ++i) {  // a row that is not asked for sees nothing
    const bool asked = (which >> i & 1u) != 0u;
    const uint32_t r = asked ? r0 + i : any, token = t.t0 + r / t.stride;
    row[i] = attend_uniform(attend_row(a, t, r));
    lo[i] = attend_uniform(attend_begin(a, t.q, token));
    hi[i] = asked ? attend_uniform(attend_end(t.q, token + 1u)) : 0u;
    if (hi[i] > lo[i]) {
      least = lo[i] < least ? lo[i] : least;
      most = hi[i] > most ? hi[i] : most;
    }
    m[i] = -__builtin_inff();
    l[i] = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
  }
  for (uint32_t j0 = least; j0 < most; j0 += 64u) {
    const uint32_t j = j0 + lane, off = attend_key(a, t, j, least, most);
    float p[kRedo] = {};
    if (off != kNoRow) {
#pragma unroll 2
      for (uint32_t c = 0u; c < D8; ++c) {
        const vec<T, 8> y = __builtin_bit_cast(vec<T, 8>, reinterpret_cast<const uint4*>(k)[static_cast<uint64_t>(off) + c]);
#pragma unroll
        for (uint32_t i = 0; i < kRedo; ++i) {
          const vec<T, 8> x = __builtin_bit_cast(vec<T, 8>, reinterpret_cast<const uint4*>(q)[static_cast<uint64_t>(row[i]) * D8 + c]);
#pragma unroll
          for (int e = 0; e < 8; ++e) p[i] = fmaf(static_cast<float>(x[e]), static_cast<float>(y[e]), p[i]);
        }
      }
    }
#pragma unroll
    for (uint32_t i = 0; i < kRedo; ++i) {
      const bool sees = off != kNoRow && j >= lo[i] && j < hi[i];
      const float s = sees ? p[i] * scale2 : -__builtin_inff();
      const float top = fmaxf(m[i], seg_allreduce<64>(s, [](float x, float y) { return fmaxf(x, y); }));
      const float f = m[i] == top ? 1.0f : __builtin_amdgcn_exp2f(m[i] - top);
      m[i] = top;
      p[i] = sees ? __builtin_amdgcn_exp2f(s - (top == -__builtin_inff() ? 0.0f : top)) : 0.0f;
      l[i] = l[i] * f + p[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] *= f;
    }
    constexpr uint32_t kAhead = 8u;
    for (uint32_t n = 0u; n < 64u && j0 + n < most; n += kAhead) {
      vec<T, 4> x[kAhead];
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
        const uint32_t at = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(off), static_cast<int>(n + u)));
        x[u] = vec<T, 4>{};
        if (at != kNoRow && lane < a.D / 4u) x[u] = load_vec<T, 4>(v + static_cast<uint64_t>(at) * 8u + lane * 4u);
      }
#pragma unroll
      for (uint32_t u = 0; u < kAhead; ++u) {
#pragma unroll
        for (uint32_t i = 0; i < kRedo; ++i) {
          const float w = __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(p[i])), static_cast<int>(n + u))));
          if (j0 + n + u < lo[i] || j0 + n + u >= hi[i]) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][e] += w * static_cast<float>(x[u][e]);
        }
      }
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kRedo; ++i) {
    l[i] = seg_allreduce<64>(l[i], [](float x, float y) { return x + y; });
    if ((which >> i & 1u) == 0u) continue;
    const float g = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
    if (lane < a.D / 4u) {
      vec<T, 4> w;
#pragma unroll
      for (int e = 0; e < 4; ++e) w.set(e, static_cast<T>(o[i][e] * g));
      store_vec<T, 4>(out.y + static_cast<uint64_t>(row[i]) * a.D + lane * 4u, w);
    }
    if (lane == 0u && out.lse != nullptr) out.lse[row[i]] = l[i] == 0.0f ? -__builtin_inff() : (m[i] + __builtin_log2f(l[i])) * kLn2;
  }
}
// The rows of the tiles that a flagged workgroup has units of, but those of one
// position: those that a value which they do not see has got into are done again, the
// others stay as their sums (or the join of their parts) have them. So a sequence of NaN
// costs a look at each of its tiles, and its first NaN the rows before it in a tile: f16
// prompts of 4096 take 0.42 ms, 0.65 with a NaN at the first token, 5.8 at the last (54
// and 17 where each row that is not finite was done again).
template <bool F16, uint32_t DP, bool MANY, typename T>
__device__ __forceinline__ void redo_rows(const AttendShape& a, const AttendCount& c, AttendOdd* odd, const AttendOut<T>& out, const T* q, const T* k,
                                          const T* v, float scale2) {
  const uint32_t slices = gridDim.x / kAttendGroups, g = blockIdx.x / slices, slice = blockIdx.x % slices;
  if (out.join[8u * g + 7u] == 0u) return;
  const uint64_t units = c.before[MANY ? 1 : 0][256], run = attend_run(units), begin = run * g;
  const uint64_t end = begin + run < units ? begin + run : units;
  if (begin >= end) return;
  AttendTile t = attend_tile<MANY, DP>(a, c, begin);
  for (;;) {
    const uint32_t rows = t.t1 - t.t0 > 1u ? (t.t1 - t.t0) * t.stride : 0u, lane = threadIdx.x & 63u;
    const AttendPlace place = attend_place_of(t);
    const uint32_t from = static_cast<uint32_t>(t.first / run), parts = static_cast<uint32_t>((t.end - 1u) / run) - from + 1u;
    if (rows != 0u) attend_find_odd(a, t, v, odd);
    for (uint32_t r0 = (slice * 4u + (threadIdx.x >> 6)) * kRedo; r0 < rows; r0 += 4u * kRedo * slices) {
      uint32_t which = 0u;
      for (uint32_t i = 0u; i < kRedo && r0 + i < rows; ++i) {
        const uint32_t row = place.row(a, r0 + i), token = t.t0 + (r0 + i) / t.stride;
        if (row == kNoRow) continue;
        const uint32_t lo = attend_begin(a, t.q, token), hi = attend_end(t.q, token + 1u);
        JoinSum s;
        bool off = false;
        if (lane < a.D / 4u) {
          if (parts > 1u) {
            s.all(out, a.D, from, parts, r0 + i, lane * 4u);
          } else {
            const vec<T, 4> x = load_vec<T, 4>(out.y + static_cast<uint64_t>(row) * a.D + lane * 4u);
#pragma unroll
            for (int e = 0; e < 4; ++e) s.o[e] = static_cast<float>(x[e]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) off |= !(s.o[e] - s.o[e] == 0.0f) && attend_off(*odd, lane * 4u + e, lo, hi);
        }
        if (__builtin_amdgcn_ballot_w64(off) != 0u) which |= 1u << i;
        else if (parts > 1u && lane < a.D / 4u) attend_store<F16>(a, place, out, -1, r0 + i, lane * 4u, s.o, s.m, s.l);
      }
      if (which != 0u) redo_some<F16>(a, t, r0, which, out, q, k, v, scale2, lane);
    }
    if (t.end >= end) break;
    attend_next<MANY, DP>(a, c, t);
  }
}

template <bool F16, uint32_t DP, typename T>
__device__ __forceinline__ void join_attention(const AttendShape& a, const T* q, const T* k, const T* v, const AttendOut<T>& few,
                                               const AttendOut<T>& many, float scale) {
  join_kind<F16>(a, many);
  join_kind<F16>(a, few);
  const uint32_t g = blockIdx.x / (gridDim.x / kAttendGroups);
  if ((many.join[8u * g + 7u] | few.join[8u * g + 7u]) == 0u) return;
  __shared__ AttendCount c;
  __shared__ AttendOdd odd;
  attend_count<DP>(a, &c);
  redo_rows<F16, DP, true>(a, c, &odd, many, q, k, v, scale * kLog2e);
  redo_rows<F16, DP, false>(a, c, &odd, few, q, k, v, scale * kLog2e);
}

}  // namespace hip
}  // namespace tca

#endif  // TCA_HIP_ATTENTION_H_
