// Attention in a window (gfx950): a query sees the frames (or tokens) around its own and the first keys of the sequence, and leaves a
// state (out, lse) like every other attention launch, so that it merges with them.
//
// With p the query's position among the keys and frames of `frame` tokens counted from key `sinks`:
//   start = sinks + floor((p - sinks) / frame) * frame           its frame's first token
//   lo = start - left, hi = start + right                        (left = frames before x frame; right = frames behind + 1, x frame)
//   key j is visible:  j < min(hi, len)  and  (j >= lo or j < sinks)
//   out = sum_j e_j v_j / sum_j e_j,  lse = log sum_j e_j,  e_j = exp(scale q.k_j);  no key visible: out = 0, lse = -inf
//
// Work: rows of one key head are the queries of all query heads that share it (row = query * group + head in group), so shared heads
// fill the matrix instructions of a single token.  Two forms:
//   * shared tiles: a workgroup of 8 wavefronts, 32 rows each, walks the 64-key tiles that some of its 256 rows see: the sinks' tiles,
//     then the window's.  Its two groups of 4 run a phase apart: while one has its products on the matrix pipe, the other does its softmax.
//   * few rows: the 8 (or 4) wavefronts of a workgroup share 32 rows and take 32-key tiles of their own in turn; their states meet in the LDS.
// Only a tile with a border in it is masked.  The last round of workgroups, or all of them, may be cut into parts along the keys, whose states the
// last one of an item adds up (few rows, with counters) or a kernel behind the launch.
//
// Large launches are bound by the package's power cap: 14 400 queries of 24 heads of 128 over 8 frames of 3600 of 57 600 keys and the first frame 4.69 ms, 1.22
// PFLOP/s of visible pairs at 1.65 GHz, MFMAs busy 71 % of the cycles (a library product of 16384^3: 1.36 PFLOP/s); 48 heads of 64, 17 550 queries over 5 frames of 1350
// 1.41 ms, 0.97 PFLOP/s (vector ALU 76 %).  Single tokens by HBM: 4 x 24 heads of 128 over 4160 keys 44.3 us, 4.6 TB/s with the launch, of 64 29.0 us, 3.5 TB/s.
#include <algorithm>
#include <cmath>

#include "attn_rows.h"
#include "dt_common.h"

namespace dt {
namespace {

constexpr int kXcds = 8;
constexpr int64_t kMostItems = (1 << 23) - (1 << 17);      // a grid holds fewer than 2^32 lanes, 512 a workgroup; 2^17 workgroups for parts
constexpr int32_t kMostTokens = 1 << 29;   // positions, spans and lengths: their sums stay in 32 bits

struct WindowArgs {
  const uint16_t *q, *k, *v;
  uint16_t* out;
  float* lse;
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  int32_t Sq, Sk, H, Hk, group;
  int32_t left, right;          // spans in tokens; -1: no border
  int32_t frame, sinks, q_begin;
  const int32_t* kv_lens;       // device [B], or null: Sk
  float scale_log2;
  int32_t rows, row_tiles, items, per_xcd;
  Quotient by_group, by_frame, by_tiles, by_heads, by_ways;
  // An XCD's items from tail_start on, tail of them, are cut along the keys into `ways` workgroups each
  int32_t tail_start, tail, ways;
  float* part_out;              // [part][row of a tile][D] sums, and [part][row] (maximum in powers of two, sum)
  float* part_ml;
  uint32_t* counters;           // of an item's parts that are done, zero before and after the launch; null: a kernel adds them up
};

__device__ __forceinline__ int keys_of(const WindowArgs& a, int b) {
  return a.kv_lens ? min(max(a.kv_lens[b], 0), a.Sk) : a.Sk;   // nothing on the host has looked at the list
}

// What a lane needs to bring its 16 bytes of every 1 KB block of a tile.
template <int D, int NKB>
struct Loader {
  typedef Tiles<D, NKB> T;
  const uint16_t *k, *v;       // of this batch and key head
  int64_t k_ss, v_ss;
  uint32_t k_row, k_chunk, v_off;     // lane's bytes within block 0; of K the row's and, apart from them, those inside the row

  __device__ __forceinline__ void open(const WindowArgs& a, int b, int hk, int lane) {
    k = a.k + b * a.k_sb + hk * a.k_sh;
    v = a.v + b * a.v_sb + hk * a.v_sh;
    k_ss = a.k_ss;
    v_ss = a.v_ss;
    const int row = lane / T::kRowLanes, chunk = lane % T::kRowLanes;
    k_row = row * (uint32_t)(2 * k_ss);
    k_chunk = 16 * (chunk ^ T::swz_k(row));
    v_off = row * (uint32_t)(2 * v_ss) + 64 * ((chunk >> 2) ^ T::swz_v(row)) + 16 * (chunk & 3);
  }
  // Bytes of a tile in front of key `left` of the sample's: rows behind the last key arrive as zeros.
  __device__ __forceinline__ static uint32_t bytes(int left, int64_t ss) {
    return left > 0 ? (uint32_t)(min(left, T::kKeys) - 1) * (2 * (uint32_t)ss) + T::kRowBytes : 0u;
  }
  // Blocks b0, b0 + step .. of the tile at `from`, of which `valid` bytes are there, into the LDS at `to`.  The descriptor's base is the tile's, so
  // that no offset needs more than 32 bits however long the cache is.  (The row is part of the lane's offset: a scalar offset beyond the
  // descriptor's end would wrap its range check.)
  template <int kCount>
  __device__ __forceinline__ void issue_k(const uint16_t* from, uint32_t valid, int b0, int step, uint32_t to) const {
    const u32x4 r = make_rsrc(from, valid);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int blk = b0 + i * step;
      // (the block permutes the chunks of a row, whose own place may have any multiple of 16 bytes in it)
      const uint32_t chunk = k_chunk ^ (64u * (blk & T::kBlockXor));
      load_block_to_lds(r, k_row + chunk + blk * T::kBlockRows * (2 * (uint32_t)k_ss), 0, to + blk * 1024);
    }
  }
  template <int kCount>
  __device__ __forceinline__ void issue_v(const uint16_t* from, uint32_t valid, int b0, int step, uint32_t to) const {
    const u32x4 r = make_rsrc(from, valid);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int blk = b0 + i * step;
      load_block_to_lds(r, v_off + blk * T::kBlockRows * (2 * (uint32_t)v_ss), 0, to + blk * 1024);
    }
  }
};

// Walks a list's tiles: where a tile lies and how many bytes of it there are, 0 behind the last one.  Between two stops -- the first tile of the
// window, the last one, which may end early -- a step is an addition and a comparison.
template <int D, int NKB>
struct Cursor {
  typedef Tiles<D, NKB> T;
  const uint16_t* from;
  uint32_t valid;
  int t, stop;
  __device__ __forceinline__ void open(const TileList<T::kKeys>& list, const uint16_t* base, int64_t ss, int len) {
    t = list.begin;
    seek(list, base, ss, len);
  }
  __device__ __forceinline__ void next(const TileList<T::kKeys>& list, const uint16_t* base, int64_t ss, int len) {
    from += T::kKeys * ss;
    if (__builtin_expect(++t == stop, 0)) seek(list, base, ss, len);
  }
  __device__ __forceinline__ void seek(const TileList<T::kKeys>& list, const uint16_t* base, int64_t ss, int len) {
    const int key = t < list.end ? list.key(t) : 0;
    from = base + key * ss;
    valid = t < list.end ? Loader<D, NKB>::bytes(len - key, ss) : 0u;
    stop = t >= list.end - 1 ? t + 1 : t < list.n_sink ? min(list.n_sink, list.end - 1) : list.end - 1;
  }
};

// The workgroup's item: rows (the last ones first: under a causal border without a window they see most), batch and key head, and of its tiles
// the part [n part / ways, n (part + 1) / ways).
struct Item {
  int row0, b, hk, part, ways, slot;    // slot: of the part's state in the workspace
};
__device__ __forceinline__ bool item_at(const WindowArgs& a, int xcd, int idx, int rows, Item& it) {
  const int item = xcd * a.per_xcd + idx;      // an XCD works through neighbouring items, which share keys in its L2
  if (idx >= a.per_xcd || item >= a.items) return false;
  const int unit = (int)quotient(item, a.by_tiles);
  it.row0 = (a.row_tiles - 1 - (item - unit * a.row_tiles)) * rows;
  it.b = (int)quotient(unit, a.by_heads);
  it.hk = unit - it.b * a.Hk;
  return true;
}
__device__ __forceinline__ bool item_of(const WindowArgs& a, int rows, Item& it) {
  const int xcd = blockIdx.x % kXcds;
  int idx = blockIdx.x / kXcds;
  it.part = 0;
  it.ways = 1;
  it.slot = 0;
  if (idx >= a.tail_start) {
    const int k = idx - a.tail_start;
    const int whole = (int)quotient(k, a.by_ways);
    idx = a.tail_start + whole;
    it.part = k - whole * a.ways;
    it.ways = a.ways;
    it.slot = xcd * a.tail * a.ways + k;
  }
  if (!item_at(a, xcd, idx, rows, it)) return false;
  for (int* x : {&it.row0, &it.b, &it.hk, &it.part, &it.ways, &it.slot}) *x = __builtin_amdgcn_readfirstlane(*x);
  return true;
}

// The 32 rows of a wavefront without matrix instructions, visible keys only, from the maxima (in powers of two) and inverse sums that lane r and
// r + 32 hold of row r: a lane has a key's score, then its columns.
template <int D, bool kHalf>
__device__ __forceinline__ void rows_one_by_one(const WindowArgs& a, const Item& it, int len, int row0, float m, float inv, int begin, int end, int lane) {
  typedef Elem<kHalf> E;
  constexpr int kCols = D / 64;
  const uint16_t* k = a.k + it.b * a.k_sb + it.hk * a.k_sh;
  const uint16_t* v = a.v + it.b * a.v_sb + it.hk * a.v_sh + lane * kCols;
#pragma unroll 1
  for (int r = 0; r < 32 && row0 + r < a.rows; ++r) {
    const int s = query_of(a, row0 + r), head = it.hk * a.group + row0 + r - s * a.group;
    const Span span = uniform_span(a, len, s);
    const uint16_t* q = a.q + it.b * a.q_sb + s * a.q_ss + head * a.q_sh;
    const float top = __shfl(m, r), norm = __shfl(inv, r);
    float acc[kCols] = {};
    // keys [begin, end) of them: in front of the window, and in it
    const int lo = max(span.lo, begin), hi = min(span.hi, end);
    const int sinks = min(min(a.sinks, end), min(span.lo, span.hi));
#pragma unroll 1
    for (int j0 = begin < sinks ? begin : lo; j0 < hi || j0 < sinks; j0 = j0 < sinks && j0 + 64 >= sinks ? max(lo, sinks) : j0 + 64) {
      const int stop = min(j0 < sinks ? sinks : hi, j0 + 64);
      float score = 0.f;
      if (j0 + lane < stop) {
        const uint16_t* row = k + (int64_t)(j0 + lane) * a.k_ss;
#pragma unroll 1
        for (int d = 0; d < D; d += 8) {
          const typename E::x8 x = *reinterpret_cast<const typename E::x8*>(q + d), y = *reinterpret_cast<const typename E::x8*>(row + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) score = __builtin_fmaf((float)x[e], (float)y[e], score);
        }
      }
      const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale_log2, -top));
      for (int j = j0; j < stop; j += 8) {
        typename E::t x[8][kCols];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int e = 0; e < kCols; ++e) x[i][e] = reinterpret_cast<const typename E::t*>(v + (int64_t)min(j + i, stop - 1) * a.v_ss)[e];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wj = __shfl(w, j + i - j0);
#pragma unroll
          for (int e = 0; e < kCols; ++e)
            if (j + i < stop) acc[e] = __builtin_fmaf(wj, (float)x[i][e], acc[e]);
        }
      }
    }
    if (it.ways > 1) {
      float* part = a.part_out + ((int64_t)it.slot * kRowsShared + row0 % kRowsShared + r) * D + lane * kCols;
#pragma unroll
      for (int e = 0; e < kCols; ++e) part[e] = acc[e];
    } else {
      typename E::t* out = reinterpret_cast<typename E::t*>(a.out) + (((int64_t)it.b * a.Sq + s) * a.H + head) * D + lane * kCols;
#pragma unroll
      for (int e = 0; e < kCols; ++e) out[e] = (typename E::t)(acc[e] * norm);
    }
  }
}

// Whether a tile that some row of the wavefront does not see whole holds infinite or undefined values.
template <int D, bool kHalf>
__device__ __forceinline__ bool masked_not_finite(const WindowArgs& a, const Item& it, const RowState<D, kHalf, 2>& st, const TileList<64>& list, int len, int lane) {
  typedef RowState<D, kHalf, 2> State;
  typedef Tiles<D, 2> T;
  const uint16_t* v = a.v + it.b * a.v_sb + it.hk * a.v_sh + 8 * (lane % T::kRowLanes);
  uint32_t over = 0;
#pragma unroll 1
  for (int t = list.begin; t < list.end; ++t) {
    const int k0 = list.key(t);
    if (st.whole(k0)) continue;
#pragma unroll 1
    for (int j = k0 + lane / T::kRowLanes; j < min(k0 + T::kKeys, len); j += T::kBlockRows) over |= State::ones(*reinterpret_cast<const u32x4*>(v + j * a.v_ss));
  }
  return __any((over & 0x80008000u) != 0);
}

template <int D, bool kHalf>
__global__ __launch_bounds__(kWavesShared * 64, D == 64 ? 4 : 2) void attn_window_kernel(const WindowArgs a) {
  typedef Tiles<D, 2> T;
  typedef SharedLds<D> S;
  typedef Elem<kHalf> E;
  typedef typename E::x8 ex8;
  extern __shared__ __align__(1024) uint8_t lds[];
  Item it;
  if (!item_of(a, kRowsShared, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int len = keys_of(a, it.b);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const Span all_first = uniform_span(a, len, query_of(a, it.row0)), all_last = uniform_span(a, len, query_of(a, min(it.row0 + kRowsShared - 1, a.rows - 1)));
  const TileList<T::kKeys> list(a, all_first, all_last, it.part, it.ways);
  const int n = list.end - list.begin;
  Loader<D, 2> ld;
  ld.open(a, it.b, it.hk, lane);
  constexpr int kPer = T::kBlocks / kWavesShared;
  Cursor<D, 2> kc, vc;
  kc.open(list, ld.k, ld.k_ss, len);
  vc.open(list, ld.v, ld.v_ss, len);
  auto load_k = [&](int pair) __attribute__((always_inline)) {
    ld.template issue_k<kPer>(kc.from, kc.valid, wave, kWavesShared, lds0 + pair_at<D>(pair) + T::kBytes);
    kc.next(list, ld.k, ld.k_ss, len);
  };
  auto load_pair = [&](int t) __attribute__((always_inline)) {
    ld.template issue_v<kPer>(vc.from, vc.valid, wave, kWavesShared, lds0 + pair_at<D>(t));
    vc.next(list, ld.v, ld.v_ss, len);
    load_k(t);
  };
  RowState<D, kHalf, 2> st;
  const int row0 = it.row0 + 32 * wave;
  if (n > 0) {
    const uint16_t* q = a.q + it.b * a.q_sb + (int64_t)it.hk * a.group * a.q_sh;
    queries_to_lds<D>(lds0, row0, wave, lane, [&](int r) __attribute__((always_inline)) {
      const int row = min(r, a.rows - 1);
      const int s = query_of(a, row), g = row - s * a.group;
      return q + s * a.q_ss + g * a.q_sh;
    });
    load_k(-1);
    load_pair(0);
    load_pair(1);
  }
  st.open(a, it.b, it.hk, row0, len, lane, false);
  if (n > 0) walk_tiles<D, kHalf>(st, lds, list, all_first, all_last, n, wave, lane, load_pair);
  // Rows of the result through the LDS, so that a store covers whole lines: half of the columns at a time.
  const int col = lane & 31, hh = lane >> 5;
  const float l = st.l_run + __shfl_xor(st.l_run, 32);
  const float inv = l != 0.f ? 1.f / l : 0.f;      // (an undefined sum stays one)
  float undefined = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) undefined = __builtin_fmaf(st.o[i][r], 0.f, undefined);
  const bool hurt = __builtin_expect(__any(undefined != 0.f && l == l), 0) && masked_not_finite<D, kHalf>(a, it, st, list, len, lane);
  if (it.ways > 1) {
    // A part's sums, fp32.  (Where they have to be computed once more, they are those of the keys of the part.)
    const int64_t at = (int64_t)it.slot * kRowsShared + 32 * wave + col;
    if (__builtin_expect(hurt, 0)) {
      rows_one_by_one<D, kHalf>(a, it, len, row0, st.m_ref * st.c, inv, list.begin < list.end ? list.key(list.begin) : 0, list.begin < list.end ? list.key(list.end - 1) + T::kKeys : 0, lane);
    } else if (row0 + col < a.rows) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = st.o[db][4 * g + e];
          *reinterpret_cast<f32x4*>(a.part_out + at * D + 32 * db + 8 * g + 4 * hh) = x;
        }
    }
    if (hh == 0 && row0 + col < a.rows) {
      a.part_ml[at * 2] = st.m_ref * st.c;
      a.part_ml[at * 2 + 1] = l;
    }
    return;
  }
  if (hh == 0 && row0 + col < a.rows) {
    const int s = query_of(a, row0 + col), g = row0 + col - s * a.group;
    a.lse[((int64_t)it.b * a.H + it.hk * a.group + g) * a.Sq + s] =
        l != 0.f ? (st.m_ref * st.c + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
  }
  if (__builtin_expect(hurt, 0)) {
    rows_one_by_one<D, kHalf>(a, it, len, row0, st.m_ref * st.c, inv, 0, len, lane);
    return;
  }
  uint8_t* stage = lds + S::kStage + wave * 32 * D;
  constexpr int kChunks = D / 16, kPass = 64 / kChunks;       // 16-byte chunks of half a row, rows of a store
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        typename E::x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(st.o[half * (D / 64) + i][4 * g + e] * inv);
        *reinterpret_cast<typename E::x4*>(stage + col * D + (((4 * i + g) ^ S::swz_o(col)) << 4) + 8 * hh) = h;
      }
#pragma unroll
    for (int i = 0; i < 32 / kPass; ++i) {
      const int r = i * kPass + lane / kChunks, chunk = lane % kChunks;
      const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * D + ((chunk ^ S::swz_o(r)) << 4));
      const int row = row0 + r;
      if (row < a.rows) {
        const int s = query_of(a, row), g = row - s * a.group;
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(a.out + (((int64_t)it.b * a.Sq + s) * a.H + it.hk * a.group + g) * D + half * (D / 2) + 8 * chunk));
      }
    }
  }
}

// Few rows, W wavefronts.  The LDS holds a tile (K and V) of each wavefront, then its state.  A wavefront needs nobody: K of its next tile is sent for
// before the softmax of this one, V of the next behind its values, and while it waits the others have theirs (8 x 16 KB a
// CU at D = 128; four wavefronts with two tiles each were 48 KB a us and CU, this is 70).
// As the compiler builds the loop, more is waited for than that needs.  Q comes by loads that it counts, the tiles by loads that it does not, and its wait for
// Q stands in front of the score MFMAs, in the loop: at D = 128 vmcnt(7) .. vmcnt(0) of every tile, so that V of a tile has landed before its softmax begins and K of
// the next comes alone.  At D = 64, where four wavefronts a SIMD leave 128 registers, 4 to 6 are spilled around the loop, whose stores, counted as well, leave these
// waits at vmcnt(8) .. vmcnt(4); the branch of the exact maximum, which the first tile takes, brings one of them back and waits for all loads.
template <int D, bool kHalf, int W>
__global__ __launch_bounds__(W * 64, D == 64 ? 4 : 2) void attn_window_few_kernel(const WindowArgs a) {
  typedef Tiles<D, 1> T;
  typedef Elem<kHalf> E;
  extern __shared__ __align__(1024) uint8_t lds[];
  Item it;
  if (!item_of(a, kRowsFew, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, hh = lane >> 5;
  const int len = keys_of(a, it.b);
  RowState<D, kHalf, 1> st;
  st.open(a, it.b, it.hk, it.row0, len, lane, true);
  const TileList<T::kKeys> list(a, st.first, st.last, it.part, it.ways);   // and of the part every W-th tile
  const uint8_t* kt = lds + wave * FewLds<D, W>::kTile;
  const uint8_t* vt = kt + T::kBytes;
  const uint32_t kt0 = (uint32_t)(uintptr_t)(lds_ptr_t)(lds + wave * FewLds<D, W>::kTile);
  Loader<D, 1> ld;
  ld.open(a, it.b, it.hk, lane);
  auto load_k = [&](int t) __attribute__((always_inline)) {     // (past the end, with an empty descriptor: the waits count loads)
    const int k0 = list.key(t);
    ld.template issue_k<T::kBlocks>(ld.k + k0 * ld.k_ss, t < list.end ? ld.bytes(len - k0, ld.k_ss) : 0u, 0, 1, kt0);
  };
  auto load_v = [&](int t) __attribute__((always_inline)) {
    const int k0 = list.key(t);
    ld.template issue_v<T::kBlocks>(ld.v + k0 * ld.v_ss, t < list.end ? ld.bytes(len - k0, ld.v_ss) : 0u, 0, 1, kt0 + T::kBytes);
  };
  int t = list.begin + wave;
  if (t < list.end) {
    load_k(t);
    load_v(t);
  }
  for (; t < list.end; t += W) {
    const int k0 = list.key(t);
    const bool masked = !st.whole(k0);
    f32x16 s[1];
    typename E::x8 p[1][2];
    wait_oldest<T::kBlocks>();
    st.scores(kt, s);
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s[0]) : : "memory");      // (the tile has been read)
    load_k(t + W);
    st.softmax(s, p, k0, masked, lane);
    wait_oldest<T::kBlocks>();
    if (masked && st.any_not_finite(vt, lane)) st.values_not_finite(vt, p, k0, lane);
    else st.values(vt, p);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    load_v(t + W);
  }
  // The states as they lie in the registers; a wavefront then adds up its share of the columns.
  float l = st.l_run + __shfl_xor(st.l_run, 32);
  wait_loads();
  float* slot = reinterpret_cast<float*>(lds + wave * FewLds<D, W>::kTile) + lane * 4;
  float* ml = reinterpret_cast<float*>(lds + FewLds<D, W>::kBytes);
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = st.o[i][4 * g + e];
      *reinterpret_cast<f32x4*>(slot + (4 * i + g) * 256) = x;
    }
  if (hh == 0) {
    ml[wave * 64 + col] = st.m_ref * st.c;
    ml[wave * 64 + 32 + col] = l;
  }
  __syncthreads();
  float m[W], w[W], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    m[i] = ml[i * 64 + col];
    top = fmaxf(top, m[i]);
  }
  l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float li = ml[i * 64 + 32 + col];
    w[i] = weight_of(m[i], li, top);
    l = __builtin_fmaf(w[i], li, l);
  }
  const int row = it.row0 + col;
  const bool live = row < a.rows;
  const int s = query_of(a, min(row, a.rows - 1)), g0 = min(row, a.rows - 1) - s * a.group;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int64_t head = it.hk * a.group + g0;
  uint16_t* out = a.out + (((int64_t)it.b * a.Sq + s) * a.H + head) * D;
  const bool meet = it.ways > 1 && a.counters != nullptr;
  const int64_t part_row = (int64_t)it.slot * kRowsFew + col;
  constexpr uint32_t kPartBytes = kRowsFew * D * 4;
  const Rsrc part = buffer_of(a.part_out + (int64_t)it.slot * (kRowsFew * D), kPartBytes);
#pragma unroll
  for (int i = 0; i < D / 8 / W; ++i) {
    const int q = wave * (D / 8 / W) + i;  // group of 4 registers: d = 8 q + 4 hh ..
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + j * FewLds<D, W>::kTile) + lane * 4 + q * 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w[j], x[e], sum[e]);     // (a weight of 0 keeps what is undefined: some row's visible key is)
    }
    if (!live) continue;
    if (it.ways > 1) {
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum), part, (col * D + 8 * q + 4 * hh) * 4, 0, kDevice);
    } else {
      typename E::x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(sum[e] * inv);
      *reinterpret_cast<typename E::x4*>(out + 8 * q + 4 * hh) = h;
    }
  }
  if (wave == 0 && hh == 0 && live) {
    if (it.ways > 1) {
      store_device(a.part_ml + part_row * 2, top);
      store_device(a.part_ml + part_row * 2 + 1, l);
    } else {
      a.lse[((int64_t)it.b * a.H + head) * a.Sq + s] = l != 0.f ? (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
    }
  }
  if (!meet) return;
  // The last of the item's parts adds them all up, each lane the columns it has stored of its own part's.
  int* flag = reinterpret_cast<int*>(lds + FewLds<D, W>::kFlag);
  wait_loads();                // (stores as well)
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* counter = a.counters + it.slot / it.ways;
    const bool last = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == it.ways;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  if (!*flag || !live) return;
  const int slot0 = it.slot - it.part;
  const float* mls = a.part_ml + ((int64_t)slot0 * kRowsFew + col) * 2;
  const float* parts = a.part_out + (int64_t)slot0 * (kRowsFew * D);
  constexpr int kCols = D / 8 / W, kSome = 4;          // parts under way together
  top = -INFINITY;
  for (int p0 = 0; p0 < it.ways; p0 += kSome) {
    float x[kSome];
#pragma unroll
    for (int p = 0; p < kSome; ++p) x[p] = load_device(mls + min(p0 + p, it.ways - 1) * (2 * kRowsFew));
#pragma unroll
    for (int p = 0; p < kSome; ++p) top = fmaxf(top, x[p]);
  }
  f32x4 sum[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  l = 0.f;
  for (int p0 = 0; p0 < it.ways; p0 += kSome) {
    float pm[kSome], pl[kSome];
    f32x4 x[kSome][kCols];
#pragma unroll
    for (int p = 0; p < kSome; ++p) {
      const int at = min(p0 + p, it.ways - 1);
      pm[p] = load_device(mls + at * (2 * kRowsFew));
      pl[p] = load_device(mls + at * (2 * kRowsFew) + 1);
      const Rsrc from = buffer_of(parts + (int64_t)at * (kRowsFew * D), kPartBytes);
#pragma unroll
      for (int i = 0; i < kCols; ++i)
        x[p][i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, (col * D + 8 * (wave * kCols + i) + 4 * hh) * 4, 0, kDevice));
    }
#pragma unroll
    for (int p = 0; p < kSome; ++p) {
      if (p0 + p >= it.ways) continue;
      const float wp = weight_of(pm[p], pl[p], top);
      l = __builtin_fmaf(wp, pl[p], l);
#pragma unroll
      for (int i = 0; i < kCols; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][e] = __builtin_fmaf(wp, x[p][i][e], sum[i][e]);
    }
  }
  const float norm = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    typename E::x4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(sum[i][e] * norm);
    *reinterpret_cast<typename E::x4*>(out + 8 * (wave * kCols + i) + 4 * hh) = h;
  }
  if (wave == 0 && hh == 0)
    a.lse[((int64_t)it.b * a.H + head) * a.Sq + s] = l != 0.f ? (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

// Adds up the parts of a row: a lane group of D / 4 lanes a row.
template <int D, bool kHalf>
__global__ __launch_bounds__(256) void attn_window_fold_kernel(const WindowArgs a, int tile_rows) {
  typedef Elem<kHalf> E;
  constexpr int kLanes = D / 4;
  const int c = threadIdx.x % kLanes;
  const int64_t at = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int unit = (int)(at / tile_rows), r = (int)(at % tile_rows);     // of the items that are cut
  if (unit >= kXcds * a.tail) return;
  Item it;
  if (!item_at(a, unit / a.tail, a.tail_start + unit % a.tail, tile_rows, it)) return;
  const int row = it.row0 + r;
  if (row >= a.rows) return;
  float top = -INFINITY, l = 0.f;
  const int64_t first = (int64_t)unit * a.ways * tile_rows + r;
  for (int p = 0; p < a.ways; ++p) top = fmaxf(top, a.part_ml[(first + tile_rows * p) * 2]);
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < a.ways; ++p) {
    const int64_t i = first + tile_rows * p;
    const float li = a.part_ml[i * 2 + 1], w = weight_of(a.part_ml[i * 2], li, top);
    l = __builtin_fmaf(w, li, l);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_out + i * D + 4 * c);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w, x[e], sum[e]);
  }
  const int s = query_of(a, row), b = it.b, h = it.hk * a.group + row - s * a.group;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  typename E::x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (typename E::t)(sum[e] * inv);
  *reinterpret_cast<typename E::x4*>(a.out + (((int64_t)b * a.Sq + s) * a.H + h) * D + 4 * c) = o;
  if (c == 0) a.lse[((int64_t)b * a.H + h) * a.Sq + s] = l != 0.f ? (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

int cus() {
  static thread_local int cached_dev = -1, cached = 0;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 0;
  if (dev != cached_dev) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
    cached = n;
    cached_dev = dev;
  }
  return cached;
}

template <void (*kernel)(const WindowArgs)>
int launch(const WindowArgs& a, unsigned grid, int waves, int lds, hipStream_t stream) {
  // more than 64 KB of LDS has to be allowed once per kernel and device
  static thread_local int allowed_dev = -1;
  int dev = 0;
  if (int rc = hip_fail(hipGetDevice(&dev), "hipGetDevice")) return rc;
  if (lds > 65536 && allowed_dev != dev) {
    if (int rc = hip_fail(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds),
                          "hipFuncSetAttribute"))
      return rc;
    allowed_dev = dev;
  }
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(waves * 64), lds, stream, a);
  return hip_fail(hipGetLastError(), "attn_window launch");
}

// How a launch runs: the form, and how the last round of workgroups (all of them, in a launch of less than one) is cut along the keys.  By
// estimate, from what the forms take here, in us: a step -- 64 keys of shared tiles, a 32-key tile of every wavefront of few rows -- with up to
// eight wavefronts a CU, and with more (D = 64); an item beside its steps; parts, their states' way to memory and back, 2 bytes / 6.7 TB/s, and the
// kernel that adds them up, or the last of them that does, 0.4 us a part (2 heads of 64, a token over 20 000: 20.9 us without that term, 13.3 with).
// The constants lie inside what launches of one round measure (8 heads, no border, 8 to 32 steps; a workgroup on every fourth CU .. on every one, then as many as fit):
//   us a step: shared tiles, D = 64 0.92 .. 1.19, then 2.1; D = 128 1.1 .. 1.7;  few rows, 8 wavefronts, D = 64 0.76 .. 0.92, then 1.6; D = 128 1.1 .. 1.5;
//   4 wavefronts, D = 64 0.7 .. 0.78, then 1.6; D = 128 0.75 .. 1.0, then 1.5.  Beside the steps, with the launch's 4 to 5: 7 .. 12; 5 .. 10; 4 .. 9.
// Keys that no two workgroups share cost more, from 128 workgroups on what HBM gives them, and rounds at the power cap do (1.86 a step of D = 128): both change all forms alike.
struct Form {
  int rows, keys, per_cu;       // rows of a workgroup, keys of its step, workgroups a CU
  double step, full, once;
};
template <int D>
constexpr Form kForms[3] = {
    {kRowsShared, 64, D == 64 ? 2 : 1, D == 64 ? 1.15 : 1.4, D == 64 ? 2.0 : 1.4, 8.0},
    {kRowsFew, 256, D == 64 ? 2 : 1, D == 64 ? 1.0 : 1.6, D == 64 ? 2.0 : 1.6, 5.0},
    {kRowsFew, 128, D == 64 ? 4 : 2, D == 64 ? 1.0 : 1.6, D == 64 ? 2.0 : 1.6, 4.0},
};
struct Plan {
  int form, ways;
  int64_t tail;
  double us;
};

template <int D>
Plan plan_form(const WindowArgs& a, int form, int64_t units, int n_cus, int64_t workspace_bytes) {
  const Form& f = kForms<D>[form];
  const int64_t row_tiles = (a.rows + f.rows - 1) / f.rows, per_xcd = (units * row_tiles + kXcds - 1) / kXcds, cus = std::max(n_cus / kXcds, 1);
  const int64_t slots = cus * f.per_cu;
  // keys that a row tile sees, at most
  const int64_t queries = std::min<int64_t>(f.rows / a.group + 1, a.Sq);
  const int64_t seen = a.left < 0 || a.right < 0 ? a.Sk : std::min<int64_t>(a.Sk, (int64_t)a.left + a.right + a.sinks + queries / a.frame * a.frame);
  const int64_t steps = (seen + f.keys - 1) / f.keys;
  auto item = [&](int64_t n, int64_t workgroups) {     // us of an item of n steps, that many at once on an XCD
    return (2 * workgroups > slots ? f.full : f.step) * n + f.once;
  };
  const int64_t tail = (per_xcd - 1) % slots + 1;
  const double before = (double)((per_xcd - tail) / slots) * item(steps, slots);
  Plan best{form, 1, 0, before + item(steps, tail)};
  for (int ways = 2; ways <= 64 && steps >= 2 * ways; ++ways) {
    const int64_t bytes = kXcds * tail * ways * f.rows * (D + 2) * 4;
    if (bytes > workspace_bytes) break;
    const double fold = form != 0 && a.counters ? 2.0 + 0.4 * ways : 8.0;
    const double us = before + (double)((tail * ways + slots - 1) / slots) * item((steps + ways - 1) / ways, std::min(tail * ways, slots)) + fold +
                      2.0 * bytes / 6.7e6;
    if (us < best.us) best = Plan{form, ways, tail, us};
  }
  return best;
}

template <int D, bool kHalf>
int launch_dim(WindowArgs& a, int64_t units, int n_cus, void* workspace, int64_t workspace_bytes, int64_t n_counters, hipStream_t stream) {
  Plan plan = plan_form<D>(a, 0, units, n_cus, workspace ? workspace_bytes : 0);
  for (int form : {1, 2}) {
    if (units * ((a.rows + kRowsFew - 1) / kRowsFew) > kMostItems) break;
    const Plan other = plan_form<D>(a, form, units, n_cus, workspace ? workspace_bytes : 0);
    if (other.us < plan.us) plan = other;
  }
  const int tile_rows = kForms<D>[plan.form].rows;
  a.row_tiles = (a.rows + tile_rows - 1) / tile_rows;
  a.items = (int32_t)(units * a.row_tiles);
  a.per_xcd = (a.items + kXcds - 1) / kXcds;
  a.ways = plan.ways;
  a.by_ways = quotient_by(a.ways);
  a.by_tiles = quotient_by(a.row_tiles);
  a.by_heads = quotient_by(a.Hk);
  a.tail = (int32_t)plan.tail;
  a.tail_start = a.per_xcd - a.tail;
  if (a.ways > 1) {
    a.part_out = static_cast<float*>(workspace);
    a.part_ml = a.part_out + kXcds * plan.tail * a.ways * tile_rows * D;
  }
  if (plan.form == 0 || kXcds * plan.tail > n_counters) a.counters = nullptr;
  const unsigned grid = (unsigned)(kXcds * (a.tail_start + a.tail * a.ways));
  std::unique_lock<std::mutex> lock;
  if (a.ways > 1) lock = std::unique_lock<std::mutex>(workspace_lock(workspace));
  const int rc = plan.form == 0   ? launch<attn_window_kernel<D, kHalf>>(a, grid, kWavesShared, SharedLds<D>::kBytes, stream)
                 : plan.form == 1 ? launch<attn_window_few_kernel<D, kHalf, 8>>(a, grid, 8, FewLds<D, 8>::kAll, stream)
                                  : launch<attn_window_few_kernel<D, kHalf, 4>>(a, grid, 4, FewLds<D, 4>::kAll, stream);
  if (rc != DT_OK || a.ways == 1 || a.counters) return rc;
  const int64_t folded = (int64_t)kXcds * a.tail * tile_rows;
  hipLaunchKernelGGL((attn_window_fold_kernel<D, kHalf>), dim3((unsigned)((folded * (D / 4) + 255) / 256)), dim3(256), 0, stream, a, tile_rows);
  return hip_fail(hipGetLastError(), "attn_window fold launch");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_attn_window_fwd(const void* q, const void* k, const void* v, void* out, float* lse, int32_t B, int32_t Sq, int32_t Sk,
                                  int32_t H, int32_t Hk, int32_t D, const int64_t* q_strides, const int64_t* k_strides,
                                  const int64_t* v_strides, const dt_window* window, float softmax_scale, int32_t flags, void* workspace,
                                  int64_t workspace_bytes, uint32_t* counters, int64_t n_counters, void* stream) {
  if (B <= 0 || Sq <= 0 || Sk < 0 || H <= 0 || Hk <= 0 || H % Hk) {
    set_error("B, Sq, H, Hk must be positive, Sk not negative and H a multiple of Hk (got %d, %d, %d, %d, %d)", B, Sq, Sk, H, Hk);
    return DT_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    set_error("head dim %d not built (64 and 128 are)", D);
    return DT_ERR_UNSUPPORTED;
  }
  if (!q || !out || !lse || !q_strides || !k_strides || !v_strides || !window || !aligned16(q) || !aligned16(out) ||
      (Sk > 0 && (!k || !v || !aligned16(k) || !aligned16(v)))) {
    set_error("q, k, v and out must be non-null and 16-byte aligned, lse, strides and window non-null");
    return DT_ERR_INVALID;
  }
  for (int i = 0; i < 3; ++i)
    if ((q_strides[i] | k_strides[i] | v_strides[i]) & 7) {
      set_error("strides must be multiples of 8 elements");
      return DT_ERR_INVALID;
    }
  // (a tile's rows are addressed with 32 bits)
  if (k_strides[1] < 0 || v_strides[1] < 0 || k_strides[1] > (1 << 23) || v_strides[1] > (1 << 23)) {
    set_error("token strides of k and v must be in 0..2^23 elements");
    return DT_ERR_INVALID;
  }
  const dt_window& w = *window;
  if (w.left < -1 || w.right < -1 || w.frame < 1 || w.sinks < 0 || w.q_begin < -1) {
    set_error("window: left and right must be -1 (no border) or frames, frame at least 1, sinks and q_begin not negative (q_begin -1: behind the keys)");
    return DT_ERR_INVALID;
  }
  if (Sk > kMostTokens || Sq > kMostTokens || w.q_begin > kMostTokens || w.sinks > kMostTokens || w.frame > kMostTokens) {
    set_error("lengths, positions, sinks and frames beyond 2^29 tokens are not supported");
    return DT_ERR_UNSUPPORTED;
  }
  if (flags & ~DT_ATTN_FP16) {
    set_error("flags 0x%x: only DT_ATTN_FP16 is known here", (unsigned)flags);
    return DT_ERR_INVALID;
  }
  if (workspace && (!aligned16(workspace) || workspace_bytes < 0)) {
    set_error("workspace must be 16-byte aligned with a non-negative size");
    return DT_ERR_INVALID;
  }
  if (counters && ((reinterpret_cast<uintptr_t>(counters) & 3) || n_counters < 0)) {
    set_error("counters must be 4-byte aligned with a non-negative number");
    return DT_ERR_INVALID;
  }
  const int64_t rows = (int64_t)Sq * (H / Hk), units = (int64_t)B * Hk;
  if (rows > (1ll << 30) || units > kMostItems || units * ((rows + kRowsShared - 1) / kRowsShared) > kMostItems) {
    set_error("too many query rows");
    return DT_ERR_INVALID;
  }
  WindowArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.q_sb = q_strides[0]; a.q_ss = q_strides[1]; a.q_sh = q_strides[2];
  a.k_sb = k_strides[0]; a.k_ss = k_strides[1]; a.k_sh = k_strides[2];
  a.v_sb = v_strides[0]; a.v_ss = v_strides[1]; a.v_sh = v_strides[2];
  a.Sq = Sq; a.Sk = Sk; a.H = H; a.Hk = Hk; a.group = H / Hk;
  a.frame = w.frame; a.sinks = w.sinks; a.q_begin = w.q_begin;
  // (a span of 2^30 reaches past every key from every position)
  a.left = w.left < 0 ? -1 : (int32_t)std::min<int64_t>((int64_t)w.left * w.frame, 1 << 30);
  a.right = w.right < 0 ? -1 : (int32_t)std::min<int64_t>(((int64_t)w.right + 1) * w.frame, 1 << 30);
  a.kv_lens = w.kv_lens;
  a.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  a.rows = (int32_t)rows;
  a.by_group = quotient_by(a.group);
  a.by_frame = quotient_by(a.frame);
  a.counters = counters;
  const int n_cus = cus();
  if (n_cus <= 0) {
    set_error("no current device");
    return DT_ERR_HIP;
  }
  const hipStream_t st = (hipStream_t)stream;
  const bool half = (flags & DT_ATTN_FP16) != 0;
  if (D == 128)
    return half ? launch_dim<128, true>(a, units, n_cus, workspace, workspace_bytes, n_counters, st)
                : launch_dim<128, false>(a, units, n_cus, workspace, workspace_bytes, n_counters, st);
  return half ? launch_dim<64, true>(a, units, n_cus, workspace, workspace_bytes, n_counters, st)
              : launch_dim<64, false>(a, units, n_cus, workspace, workspace_bytes, n_counters, st);
}
