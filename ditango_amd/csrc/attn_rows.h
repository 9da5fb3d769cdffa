// Attention of 32 query rows a wavefront over tiles of keys, for the kernels whose rows see a window of them (attn_window.hip, attn_pages.hip): the
// rows' state and its arithmetic, which tiles there are, the phases in which two groups of wavefronts share them.  `Args` is a kernel's own
// table, with the names of attn_window.hip's.
#pragma once

#include "attn_tiles.h"

namespace dt {
namespace {

constexpr int kWavesShared = 8;
constexpr int kRowsShared = kWavesShared * 32;   // rows of a workgroup, shared tiles
constexpr int kRowsFew = 32;                     // ... few rows, 4 or 8 wavefronts
// A tile's sum of a lane's probabilities above which the tile is redone with its exact maximum: below it no probability exceeds 2^12,
// which the 16-bit operand and the fp32 sums hold as well as one below 1.
constexpr float kSumLimit = 4096.0f;

struct Span {
  int lo, hi;
};
template <typename Args>
__device__ __forceinline__ Span span_of(const Args& a, int len, int s) {
  const int p = (a.q_begin >= 0 ? a.q_begin : len - a.Sq) + s;
  const int x = p - a.sinks;
  const int f = x >= 0 ? (int)quotient(x, a.by_frame) : -1 - (int)quotient(-1 - x, a.by_frame);
  const int start = a.sinks + f * a.frame;
  Span r;
  r.lo = a.left < 0 ? 0 : max(start - a.left, 0);
  r.hi = a.right < 0 ? len : min(max(start + a.right, 0), len);
  return r;
}
// The same for a query of all lanes, in scalar registers.
template <typename Args>
__device__ __forceinline__ Span uniform_span(const Args& a, int len, int s) {
  const Span r = span_of(a, len, __builtin_amdgcn_readfirstlane(s));
  return {__builtin_amdgcn_readfirstlane(r.lo), __builtin_amdgcn_readfirstlane(r.hi)};
}
template <typename Args>
__device__ __forceinline__ int query_of(const Args& a, int row) { return (int)quotient(row, a.by_group); }

// Tiles of kTile keys that rows between two queries see, [0, n_sink) and [w0, ...), and of that list a part, [begin, end).
template <int kTile>
struct TileList {
  int n_sink, w0, begin, end;
  template <typename Args>
  __device__ __forceinline__ TileList(const Args& a, const Span& first, const Span& last, int part, int ways) {
    n_sink = (min(a.sinks, last.hi) + kTile - 1) / kTile;
    w0 = max(first.lo / kTile, n_sink);
    const int n = n_sink + max((last.hi + kTile - 1) / kTile - w0, 0);
    begin = (int)((int64_t)n * part / ways);
    end = (int)((int64_t)n * (part + 1) / ways);
  }
  __device__ __forceinline__ int key(int t) const { return (t < n_sink ? t : w0 + t - n_sink) * kTile; }
};

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_lds_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int D, int NKB>
struct Tiles {
  static constexpr int kKeys = 32 * NKB;
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kBytes = kKeys * kRowBytes;       // of a K or V tile
  static constexpr int kSegs = D / 32;                   // 64-byte segments of a row
  static constexpr int kRowLanes = D / 8;                // lanes of a row in a 1 KB block
  static constexpr int kBlockRows = 1024 / kRowBytes;
  static constexpr int kBlocks = kBytes / 1024;
  // Rows lie in the LDS without padding (a load to the LDS writes 1 KB in a run), their 16-byte chunks (K) or 64-byte segments (V)
  // permuted by the row, so that the lanes of an operand read are in distinct banks.
  __device__ static constexpr int swz_k(int row) { return D == 128 ? (row & 15) : ((row >> 1) & 7); }
  __device__ static constexpr int swz_v(int row) { return D == 128 ? (row & 3) : ((row >> 1) & 1); }
  static constexpr int kBlockXor = D == 128 ? 3 : 1;     // a K block's rows have swz_k of the first block's ^ 4 (block & this)
};

// The state of 32 rows: lane col + 32 hh holds query col, of O^T[d][query] the d = 32 db + 8 (r / 4) + 4 hh + r % 4.
template <int D, bool kHalf, int NKB>
struct RowState {
  typedef Elem<kHalf> E;
  typedef typename E::x8 ex8;
  typedef typename E::x2 ex2;
  typedef Tiles<D, NKB> T;

  ex8 qf[D / 16];
  f32x16 o[D / 32];
  float m_ref, l_run, c;        // reference of the sums (raw scores), this lane's part of the sum, scale in powers of two
  uint32_t kld[D / 16], vld[T::kSegs];
  Span mine, first, last;       // of this lane's query, of the wavefront's first and last (spans never go back along the rows)
  int sinks;

  template <typename Args>
  __device__ __forceinline__ void open(const Args& a, int b, int hk, int row0, int len, int lane, bool read_q) {
    const int col = lane & 31, hh = lane >> 5;
    const int row = min(row0 + col, a.rows - 1);
    const int s = query_of(a, row), g = row - s * a.group;
    mine = span_of(a, len, s);
    first = uniform_span(a, len, query_of(a, min(row0, a.rows - 1)));
    last = uniform_span(a, len, query_of(a, min(row0 + 31, a.rows - 1)));
    sinks = a.sinks;
    if (read_q) {
      const uint16_t* q = a.q + b * a.q_sb + s * a.q_ss + (int64_t)(hk * a.group + g) * a.q_sh + 8 * hh;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) qf[i] = *reinterpret_cast<const ex8*>(q + 16 * i);
    }
    c = a.scale_log2;
    m_ref = -INFINITY;
    l_run = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    const int krow = key_of_row(col);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) kld[i] = krow * T::kRowBytes + 16 * ((2 * i + hh) ^ T::swz_k(krow));
    const int vrow = 8 * hh + ((lane & 15) >> 2);
#pragma unroll
    for (int g2 = 0; g2 < T::kSegs; ++g2)
      vld[g2] = vrow * T::kRowBytes + 64 * (g2 ^ T::swz_v(vrow)) + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
  }

  // Whether a row of the wavefront sees a key of [k0, k0 + kKeys); whether all of them see all.
  __device__ __forceinline__ bool needs(int k0) const { return (k0 < last.hi) & ((k0 + T::kKeys > first.lo) | (k0 < sinks)); }
  __device__ __forceinline__ bool whole(int k0) const {
    return (k0 + T::kKeys <= first.hi) & ((k0 >= last.lo) | (k0 + T::kKeys <= sinks));
  }

  __device__ __forceinline__ ex8 v_frag(const uint8_t* vt, int db, int step) const {
    const uint8_t* p = vt + vld[db] + 16 * step * T::kRowBytes;
    const s16x4 lo = lds_read_tr(p);
    const s16x4 hi = lds_read_tr(p + 4 * T::kRowBytes);
    return __builtin_bit_cast(ex8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  __device__ __forceinline__ void softmax_pass(const f32x16 (&s)[NKB], float mc, ex8 (&p)[NKB][2], float& sum) const {
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          f32x2 e;
          e.x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * half + r], c, -mc));
          e.y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][8 * half + r + 1], c, -mc));
          s0 += e.x;
          s1 += e.y;
          // P goes to the second product in the tensors' 16 bits, as q, k and v come: half a step relative to each probability.  The
          // sum is that of the fp32 values.
          const ex2 h = __builtin_convertvector(e, ex2);
          p[kb][half][r] = h.x;
          p[kb][half][r + 1] = h.y;
        }
        // (rounded and added here: the compiler otherwise holds them in fp32, beside the scores, until the sum's branch is decided)
        asm volatile("" : "+v"(p[kb][half]), "+v"(s0), "+v"(s1));
      }
    sum = s0 + s1;
  }

  // S^T = K Q^T of the tile at kt.
  __device__ __forceinline__ void scores(const uint8_t* kt, f32x16 (&s)[NKB]) const {
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) s[kb] = E::mfma(*reinterpret_cast<const ex8*>(kt + kld[i] + kb * 32 * T::kRowBytes), qf[i], s[kb]);
  }

  // Scores of the keys k0 .. -> probabilities.
  __device__ __forceinline__ void softmax(f32x16 (&s)[NKB], ex8 (&p)[NKB][2], int k0, bool masked, int lane) {
    if (masked) {
      asm volatile("" ::: "memory");   // keeps this a real branch
      // One border after the other, as most such tiles have only one of them.  Keys in front of the window but for the sinks are hidden: the place
      // behind the last sink, as an unsigned number, is then below that of the window.
      const int at = k0 + 8 * (lane >> 5);
      if (k0 < last.lo) {
        int some = max(sinks - at, 0);
        uint32_t hidden = (uint32_t)max(mine.lo - at - some, 0);
        asm volatile("" : "+v"(some), "+v"(hidden));     // (their sums with the keys' places would otherwise be kept through the loop)
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 32 * kb + 16 * (r >> 3) + (r & 7);
            s[kb][r] = (uint32_t)(key - some) < hidden ? -INFINITY : s[kb][r];
            asm volatile("" : "+v"(s[kb][r]));     // one comparison and choice after the other: 90 spilled scalars otherwise
          }
      }
      if (k0 + T::kKeys > first.hi) {
        int end = mine.hi - at;
        asm volatile("" : "+v"(end));
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = 32 * kb + 16 * (r >> 3) + (r & 7);
            s[kb][r] = key < end ? s[kb][r] : -INFINITY;
            asm volatile("" : "+v"(s[kb][r]));
          }
      }
    }
    // Probabilities relative to the reference that the sums are scaled to.  The tile's own maximum is looked for only where the sum of
    // the probabilities, needed anyway, says that the reference lags too far behind (or is not there yet: the sum is inf or NaN).
    float sum;
    softmax_pass(s, m_ref * c, p, sum);
    if (__builtin_expect(__any(!(sum <= kSumLimit)), 0)) {
      float mx = s[0][0];
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m_ref, mx);
      const float alpha = m_new > -INFINITY ? __builtin_amdgcn_exp2f((m_ref - m_new) * c) : 1.f;
      m_ref = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= alpha;
      softmax_pass(s, m_new > -INFINITY ? m_new * c : 0.f, p, sum);
    }
    l_run += sum;
  }

  // O^T += V^T P^T of the tile at vt.
  __device__ __forceinline__ void values(const uint8_t* vt, const ex8 (&p)[NKB][2]) {
#pragma unroll
    for (int step = 0; step < 2 * NKB; ++step)
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] = E::mfma(v_frag(vt, db, step), p[step >> 1][step & 1], o[db]);
  }

  // A masked key's probability is 0, which an infinite or undefined value of V would turn into NaN.  Few rows look tiles with masked keys through
  // (3 instructions for 8 values); where there is such a value, they multiply the tile with zeros in their place and then add them, as they are, to
  // the rows that see them (the weight of a visible key is above 0).  Shared tiles look at the sums instead, once: where one of a defined weight is
  // not finite and a tile with masked keys holds such a value, they compute the 32 rows once more (rows_one_by_one).
  static constexpr uint32_t kExp = kHalf ? 0x7c007c00u : 0x7f807f80u, kOne = kHalf ? 0x04000400u : 0x00800080u;
  __device__ __forceinline__ static uint32_t ones(const u32x4& x) {     // sign bits where an element's exponent is all ones, whose carry they are
    uint32_t over = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) over |= (x[e] & kExp) + kOne;
    return over;
  }
  __device__ __forceinline__ bool any_not_finite(const uint8_t* vt, int lane) const {
    uint32_t over = 0;
#pragma unroll 2
    for (int i = 0; i < T::kBlocks; ++i) over |= ones(*reinterpret_cast<const u32x4*>(vt + i * 1024 + lane * 16));
    return __any((over & 0x80008000u) != 0);
  }
  // What the rows see of such values, added as it is.
  __device__ __forceinline__ void add_not_finite(const uint8_t* vt, int k0, int lane) {
    const int hh = lane >> 5;
#pragma unroll 1
    for (int key = 0; key < T::kKeys; ++key) {
      const int j = k0 + key;
      const bool seen = j < mine.hi && (j >= mine.lo || j < sinks);
      const uint8_t* row = vt + key * T::kRowBytes;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const typename E::x4 v = *reinterpret_cast<const typename E::x4*>(row + 64 * (db ^ T::swz_v(key)) + 16 * g + 8 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = (float)v[e];
            if (seen && !(__builtin_fabsf(f) < INFINITY)) o[db][4 * g + e] += f;
          }
        }
    }
  }
  // The same ahead of the products: what the rows see of such values is added as it is, and the tile holds zeros for all of them.  (With products of its own
  // the rare case made the compiler move all of O^T from registers to others and back in every turn.)
  __device__ __forceinline__ void take_out_not_finite(uint8_t* vt, int k0, int lane) {
    add_not_finite(vt, k0, lane);
#pragma unroll 1
    for (int i = 0; i < T::kBlocks; ++i) {
      u32x4* at = reinterpret_cast<u32x4*>(vt + i * 1024 + lane * 16);
      u32x4 v = *at;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t bad = ((v[e] & kExp) + kOne) & 0x80008000u;
        v[e] &= ~((bad << 1) - (bad >> 15));
      }
      *at = v;
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  __device__ __forceinline__ void values_not_finite(const uint8_t* vt, const ex8 (&p)[NKB][2], int k0, int lane) {
#pragma unroll
    for (int step = 0; step < 2 * NKB; ++step)
#pragma unroll
      for (int db = 0; db < D / 32; ++db) {
        u32x4 v = __builtin_bit_cast(u32x4, v_frag(vt, db, step));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = ((v[e] & kExp) + kOne) & 0x80008000u;     // sign bits of the elements to leave out
          v[e] &= ~((bad << 1) - (bad >> 15));
        }
        o[db] = E::mfma(__builtin_bit_cast(ex8, v), p[step >> 1][step & 1], o[db]);
      }
    add_not_finite(vt, k0, lane);
  }
};

typedef __attribute__((address_space(3))) uint8_t* lds_ptr_t;

// The weight of a state with maximum m and sum l beside others of which the largest maximum is `top`.  Without a maximum there was no key and the
// sum is 0, or only undefined scores, and the sum is undefined: it is then the weight.
__device__ __forceinline__ float weight_of(float m, float l, float top) { return m > -INFINITY ? __builtin_amdgcn_exp2f(m - top) : l; }

// Phases of the shared tiles.  Group g (0 or 1) does the softmax of tile t in phase 2t + g and its products -- O^T += V^T P^T of tile t, then
// S^T = K Q^T of tile t + 1 -- in phase 2t + g + 1; a barrier ends every phase.  V of tile t and K of tile t + 1, read together, are pair t:
//   * read in phases 2t (the products' first fragments, ahead of the barrier) to 2t + 2;
//   * in buffer t % 4.  A softmax phase of tile t begins with the loads of pair t + 2, whose buffer was last read in phase 2t - 2 (pair t - 2);
//   * waited for by both groups at the end of phase 2t - 1, where the pair behind it, t + 1, may still be on its way: a barrier lies between
//     every wavefront's wait and anybody's read.
// The first scores' K, tile 0, is the second half of pair -1, in buffer 3.  Past the last tile, loads go on with empty descriptors.
constexpr int kPairs = 4;

template <int D>
struct SharedLds {
  typedef Tiles<D, 2> T;
  static constexpr int kPair = 2 * T::kBytes;            // V, then K
  static constexpr int kStage = kPairs * kPair;          // rows of the result, half of the columns, 32 x D bytes a wavefront
  static constexpr int kBytes = kStage + kWavesShared * 32 * D;
  static constexpr int kLoads = 2 * T::kBlocks / kWavesShared;   // of a wavefront, a pair
  // a row's 16-byte chunks in the staging rows
  __device__ static constexpr int swz_o(int row) { return D == 128 ? ((row >> 1) & 7) : ((row >> 2) & 3); }
};

template <int N>
__device__ __forceinline__ void wait_all_but() {
  static_assert(N == 2 || N == 4 || N == 8, "loads of a pair or two");
  if constexpr (N == 2) asm volatile("s_waitcnt vmcnt(2)" ::: "memory");
  else if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
}
// Ends a phase: what it has made goes through the statement, so that the compiler keeps the work on its side of the barrier.
template <typename V>
__device__ __forceinline__ void end_softmax(V (&p)[2][2]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : "+v"(p[0][0]), "+v"(p[0][1]), "+v"(p[1][0]), "+v"(p[1][1]) : : "memory");
  __builtin_amdgcn_sched_barrier(0);
}
template <int NO>
__device__ __forceinline__ void end_products(f32x16 (&s)[2], f32x16 (&o)[NO]) {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s[0]), "+v"(s[1]) : : "memory");
  if constexpr (NO == 4) asm volatile("s_barrier" : "+v"(o[0]), "+v"(o[1]), "+v"(o[2]), "+v"(o[3]) : : "memory");
  else asm volatile("s_barrier" : "+v"(o[0]), "+v"(o[1]) : : "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int D>
__device__ __forceinline__ int pair_at(int t) { return (t & (kPairs - 1)) * SharedLds<D>::kPair; }

// The wavefront's rows of Q come as whole lines through the LDS: half of them through its staging rows, a quarter each through its own shares
// of V of pairs 3 and 2, which nothing but its own later loads writes.  (As fragments from memory, a load instruction touches 32 lines for 32
// bytes each, and the compiler's wait for them would be one for every tile load behind them.)
// Block i of the wavefront's share of a tile: every eighth, or (kRun) kPer neighbours.
template <int D, bool kRun>
__device__ __forceinline__ int share_at(int wave, int i) { return kRun ? Tiles<D, 2>::kBlocks / kWavesShared * wave + i : wave + kWavesShared * i; }
template <int D, bool kRun = false>
__device__ __forceinline__ int query_at(int wave, int r) {      // row r; a quarter is kPer blocks of 1 KB
  typedef Tiles<D, 2> T;
  typedef SharedLds<D> S;
  constexpr int kPer = T::kBlocks / kWavesShared, kQRows = T::kBlockRows;
  const int in_half = S::kStage + wave * 32 * D + r * T::kRowBytes;
  const int blk = r / kQRows, i = blk % kPer;
  const int apart = (blk / kPer == 2 ? pair_at<D>(3) : pair_at<D>(2)) + share_at<D, kRun>(wave, i) * 1024 + r % kQRows * T::kRowBytes;
  return r < 16 ? in_half : apart;
}
// from(r): where row r of the batch and key head begins.
template <int D, bool kRun = false, typename From>
__device__ __forceinline__ void queries_to_lds(uint32_t lds0, int row0, int wave, int lane, From from) {
  typedef Tiles<D, 2> T;
  typedef SharedLds<D> S;
  constexpr int kPer = T::kBlocks / kWavesShared;
#pragma unroll
  for (int blk = 0; blk < 4 * kPer; ++blk) {
    const int quarter = blk / kPer, i = blk % kPer;
    const int to = quarter < 2 ? S::kStage + wave * 32 * D + blk * 1024 : pair_at<D>(5 - quarter) + share_at<D, kRun>(wave, i) * 1024;
    const int r = blk * T::kBlockRows + lane / T::kRowLanes;
    load_rows_to_lds(from(row0 + r) + 8 * ((lane % T::kRowLanes) ^ T::swz_k(r)), lds0 + to);
  }
}

// The rows of a wavefront over the tiles of a list that is not empty.  In front of it go the loads of Q, K of tile 0 and pairs 0 and 1, in this order, of
// kLoads / 2 and kLoads loads a wavefront; load_pair(t) sends for pair t.
template <int D, bool kHalf, bool kRun = false, typename LoadPair>
__device__ __forceinline__ void walk_tiles(RowState<D, kHalf, 2>& st, const uint8_t* lds, TileList<64> list, Span all_first, Span all_last,
                                           int n, int wave, int lane, LoadPair load_pair) {
  typedef Tiles<D, 2> T;
  typedef SharedLds<D> S;
  typedef Elem<kHalf> E;
  typedef typename E::x8 ex8;
  const int group = wave >> 2;
  f32x16 s[2];
  ex8 p[2][2];
  // The products of a tile and the scores of the next as one stream of MFMAs, fed by reads from the LDS that run kRing fragments ahead.
  constexpr int kPV = D / 32 * 4, kQK = D / 16 * 2, kRing = 4;
  ex8 ring[kRing];
  auto products = [&](const uint8_t* vt) __attribute__((always_inline)) {
    const uint8_t* kt = vt + T::kBytes;
    auto frag = [&](int i) __attribute__((always_inline)) -> ex8 {
      if (i < kPV) return st.v_frag(vt, i % (D / 32), i / (D / 32));
      return *reinterpret_cast<const ex8*>(kt + st.kld[(i - kPV) >> 1] + ((i - kPV) & 1) * 32 * T::kRowBytes);
    };
#pragma unroll
    for (int i = 0; i < kPV + kQK; ++i) {
      const ex8 cur = ring[i % kRing];
      if (i + kRing < kPV + kQK) ring[i % kRing] = frag(i + kRing);
      if (i < kPV) {
        const int step = i / (D / 32);
        st.o[i % (D / 32)] = E::mfma(cur, p[step >> 1][step & 1], st.o[i % (D / 32)]);
      } else {
        const int kb = (i - kPV) & 1, at = (i - kPV) >> 1;
        if (at == 0) {
          f32x16 zero;
#pragma unroll
          for (int r = 0; r < 16; ++r) zero[r] = 0.f;
          s[kb] = E::mfma(cur, st.qf[at], zero);
        } else {
          s[kb] = E::mfma(cur, st.qf[at], s[kb]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kPV - kRing; ++i) {   // behind an MFMA the two reads of a fragment of V, or the one of a fragment of K
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
#pragma unroll
    for (int i = 0; i < kQK; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, kRing, 0);
  };
  auto prefill = [&](const uint8_t* vt) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) ring[i] = st.v_frag(vt, i % (D / 32), i / (D / 32));
  };
  // Q and K of tile 0 are here, pairs 0 and 1 on their way
  wait_all_but<2 * S::kLoads>();
  {
    const int r = lane & 31, hh = lane >> 5;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) st.qf[i] = *reinterpret_cast<const ex8*>(lds + query_at<D, kRun>(wave, r) + 16 * ((2 * i + hh) ^ T::swz_k(r)));
  }
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(st.qf[i]));
  wait_lds_barrier();
  if (group == 1) {
    wait_all_but<S::kLoads>();
    wait_lds_barrier();
  }
  st.scores(lds + pair_at<D>(-1) + T::kBytes, s);
  if (group == 0) wait_all_but<S::kLoads>();
  end_products(s, st.o);
  int k0 = list.key(list.begin);
  // keys from which on, and up to which, a tile is seen whole by all rows of the workgroup
  const uint32_t inside = (uint32_t)max(all_first.hi - (T::kKeys - 1) - all_last.lo, 0);
  auto probabilities = [&](bool need, bool masked) __attribute__((always_inline)) {
    if (__builtin_expect(need, 1)) {
      st.softmax(s, p, k0, masked, lane);
    } else {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i >> 1][i & 1] = __builtin_bit_cast(ex8, u32x4{0u, 0u, 0u, 0u});
    }
  };
  // (the last tile is apart: with a way out in the middle of the loop, the compiler moves O^T to other registers and back in every turn)
  // Where the loop begins does not go by the code in front of it: 16 bytes off, the windowed attention's same instructions with heads of 64 take 1.2 % longer
  // (4096 rows over 8192 keys of 24 heads 225.0 against 227.7 us).  Over pages no place was better than another by more than cards differ.
  if constexpr (!kRun) asm volatile(".p2align 6" ::: "memory");
  for (int t = 0; t < n - 1; ++t) {
    __builtin_amdgcn_s_setprio(D == 64 ? 0 : 1);
    load_pair(t + 2);
    const uint8_t* vt = lds + pair_at<D>(t);
    bool masked = false, need = true;
    if (__builtin_expect((uint32_t)(k0 - all_last.lo) >= inside, 0)) {
      masked = !st.whole(k0);
      need = st.needs(k0);
    }
    probabilities(need, masked);
    prefill(vt);
    if (group == 1) wait_all_but<S::kLoads>();
    end_softmax(p);
    __builtin_amdgcn_s_setprio(0);
    products(vt);
    if (group == 0) wait_all_but<S::kLoads>();
    end_products(s, st.o);
    k0 = list.begin + t + 1 == list.n_sink ? list.w0 * T::kKeys : k0 + T::kKeys;
  }
  const bool masked = !st.whole(k0);
  const uint8_t* vt = lds + pair_at<D>(n - 1);
  probabilities(st.needs(k0), masked);
  end_softmax(p);
  st.values(vt, p);
  // group 1's last products are the last thing that happens in the buffers
  if (group == 0) wait_lds_barrier();
  wait_loads();     // those past the last tile, which store zeros: before the LDS is another workgroup's (and not behind the result's stores)
}

// A wavefront without rows among others that walk: its share of the loads, and everybody's barriers.
template <int D, typename LoadPair>
__device__ __forceinline__ void walk_idle(int n, int wave, LoadPair load_pair) {
  typedef SharedLds<D> S;
  const int group = wave >> 2;
  wait_all_but<2 * S::kLoads>();
  wait_lds_barrier();
  wait_all_but<S::kLoads>();
  if (group == 1) wait_lds_barrier();
  wait_lds_barrier();
  for (int t = 0; t < n - 1; ++t) {
    load_pair(t + 2);
    if (group == 1) wait_all_but<S::kLoads>();
    wait_lds_barrier();
    if (group == 0) wait_all_but<S::kLoads>();
    wait_lds_barrier();
  }
  wait_lds_barrier();
  if (group == 0) wait_lds_barrier();
  wait_loads();
}

template <int D, int W>
struct FewLds {
  static constexpr int kTile = 2 * Tiles<D, 1>::kBytes;
  static constexpr int kBytes = W * kTile;
  static_assert(32 * D * 4 <= kTile, "a state fits its wavefront's tile");
  static constexpr int kFlag = kBytes + W * 256;             // behind a maximum and a sum a row and wavefront
  static constexpr int kAll = kFlag + 16;
};
template <int N>
__device__ __forceinline__ void wait_oldest() {     // all loads but those of the newest half tile
  static_assert(N == 4 || N == 8, "blocks of a half tile");
  if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
}


}  // namespace
}  // namespace dt
