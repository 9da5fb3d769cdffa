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
//   * shared tiles: a workgroup of 4 wavefronts, 32 rows each, walks the 64-key tiles that some of its 128 rows see: the sinks' tiles,
//     then the window's.  Two workgroups a CU; one does its softmax while the other has the matrix pipe.
//   * few rows: the 4 wavefronts of a workgroup share 32 rows and take 32-key tiles of their own in turn, and the window is cut into
//     `parts` workgroups; states meet in the LDS, those of the parts in a fold kernel behind the launch.
// A wavefront leaves out tiles that none of its rows sees, and only a tile with a border in it is masked.
#include <algorithm>
#include <cmath>

#include "attn_tiles.h"
#include "dt_common.h"

namespace dt {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kRowsShared = kWaves * 32;   // rows of a workgroup, shared tiles
constexpr int kRowsFew = 32;               // ... few rows
constexpr int kXcds = 8;
// A tile's sum of a lane's probabilities above which the tile is redone with its exact maximum: below it no probability exceeds 2^12,
// which the 16-bit operand and the fp32 sums hold as well as one below 1.
constexpr float kSumLimit = 4096.0f;
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
  int32_t rows, row_tiles, parts, items, per_xcd;
  float* part_out;              // parts > 1: [item][row 32][D] sums, and [item][row 32] (maximum in powers of two, sum)
  float* part_ml;
};

struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span span_of(const WindowArgs& a, int len, int s) {
  const int p = (a.q_begin >= 0 ? a.q_begin : len - a.Sq) + s;
  const int x = p - a.sinks;
  int f = x / a.frame;
  if (f * a.frame > x) --f;
  const int start = a.sinks + f * a.frame;
  Span r;
  r.lo = a.left < 0 ? 0 : max(start - a.left, 0);
  r.hi = a.right < 0 ? len : min(max(start + a.right, 0), len);
  return r;
}
__device__ __forceinline__ int keys_of(const WindowArgs& a, int b) {
  return a.kv_lens ? min(max(a.kv_lens[b], 0), a.Sk) : a.Sk;   // nothing on the host has looked at the list
}

// Tiles of kTile keys that rows between two queries see: [0, n_sink) and [w0, w0 + n - n_sink).
struct TileList {
  int n_sink, w0, n;
};
template <int kTile>
__device__ __forceinline__ TileList tiles_of(const WindowArgs& a, const Span& first, const Span& last) {
  TileList t;
  t.n_sink = (min(a.sinks, last.hi) + kTile - 1) / kTile;
  t.w0 = max(first.lo / kTile, t.n_sink);
  t.n = t.n_sink + max((last.hi + kTile - 1) / kTile - t.w0, 0);
  return t;
}

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void wait_loads_barrier() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

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

  __device__ __forceinline__ void open(const WindowArgs& a, int b, int hk, int row0, int len, int lane) {
    const int col = lane & 31, hh = lane >> 5;
    const int row = min(row0 + col, a.rows - 1);
    const int s = row / a.group, g = row - s * a.group;
    mine = span_of(a, len, s);
    first = span_of(a, len, __builtin_amdgcn_readfirstlane(min(row0, a.rows - 1) / a.group));
    last = span_of(a, len, __builtin_amdgcn_readfirstlane(min(row0 + 31, a.rows - 1) / a.group));
    sinks = a.sinks;
    const uint16_t* q = a.q + b * a.q_sb + s * a.q_ss + (int64_t)(hk * a.group + g) * a.q_sh + 8 * hh;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) qf[i] = *reinterpret_cast<const ex8*>(q + 16 * i);
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
  __device__ __forceinline__ bool needs(int k0) const { return k0 < last.hi && (k0 + T::kKeys > first.lo || k0 < sinks); }
  __device__ __forceinline__ bool whole(int k0) const {
    return k0 + T::kKeys <= first.hi && (k0 >= last.lo || k0 + T::kKeys <= sinks);
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
      for (int r = 0; r < 16; r += 2) {
        f32x2 e;
        e.x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], c, -mc));
        e.y = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], c, -mc));
        s0 += e.x;
        s1 += e.y;
        // P goes to the second product in the tensors' 16 bits, as q, k and v come: half a step relative to each probability.  The sum
        // is that of the fp32 values.
        const ex2 h = __builtin_convertvector(e, ex2);
        p[kb][r >> 3][r & 7] = h.x;
        p[kb][r >> 3][(r & 7) + 1] = h.y;
      }
    sum = s0 + s1;
  }

  // The tile of keys k0 .. in the LDS at kt and vt.
  __device__ __forceinline__ void tile(const uint8_t* kt, const uint8_t* vt, int k0, int lane) {
    const int hh = lane >> 5;
    f32x16 s[NKB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb) {
        const ex8 ka = *reinterpret_cast<const ex8*>(kt + kld[i] + kb * 32 * T::kRowBytes);
        s[kb] = E::mfma(ka, qf[i], s[kb]);
      }
    const bool masked = !whole(k0);   // uniform
    if (masked) {
      asm volatile("" ::: "memory");   // keeps this a real branch
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = k0 + 32 * kb + 16 * (r >> 3) + 8 * hh + (r & 7);
          if (!(key < mine.hi && (key >= mine.lo || key < sinks))) s[kb][r] = -INFINITY;
        }
    }
    // Probabilities relative to the reference that the sums are scaled to.  The tile's own maximum is looked for only where the sum of
    // the probabilities, needed anyway, says that the reference lags too far behind (or is not there yet: the sum is inf or NaN).
    ex8 p[NKB][2];
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
    if (masked && any_not_finite(vt, lane)) {
      visible_only(vt, p, k0, lane);
      return;
    }
#pragma unroll
    for (int step = 0; step < 2 * NKB; ++step)
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] = E::mfma(v_frag(vt, db, step), p[step >> 1][step & 1], o[db]);
  }

  // A masked key's probability is 0, which an infinite or undefined value of V would turn into NaN.  Tiles with masked keys are looked
  // through (a wavefront reads all of the tile: 192 more vector instructions), and one with such a value adds up visible keys only.
  __device__ __forceinline__ bool any_not_finite(const uint8_t* vt, int lane) const {
    constexpr uint32_t kExp = kHalf ? 0x7c007c00u : 0x7f807f80u, kOne = kHalf ? 0x04000400u : 0x00800080u;
    uint32_t over = 0;
#pragma unroll
    for (int i = 0; i < T::kBytes / 1024; ++i) {
      const u32x4 x = *reinterpret_cast<const u32x4*>(vt + i * 1024 + lane * 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) over |= (x[e] & kExp) + kOne;   // an exponent of ones carries into the sign's bit
    }
    return __any((over & 0x80008000u) != 0);
  }
  __device__ __forceinline__ void visible_only(const uint8_t* vt, const ex8 (&p)[NKB][2], int k0, int lane) {
    const int hh = lane >> 5;
#pragma unroll 1
    for (int key = 0; key < T::kKeys; ++key) {
      const int at = (key >> 5) * 16 + ((key >> 4) & 1) * 8 + (key & 7), from = (key >> 3) & 1;
      float w = 0.f;
#pragma unroll
      for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (at == kb * 16 + r) w = (float)p[kb][r >> 3][r & 7];
      w = __shfl(w, (lane & 31) + 32 * from);
      const int j = k0 + key;
      const bool seen = j < mine.hi && (j >= mine.lo || j < sinks);
      const uint8_t* row = vt + key * T::kRowBytes;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const typename E::x4 v = *reinterpret_cast<const typename E::x4*>(row + 64 * (db ^ T::swz_v(key)) + 16 * g + 8 * hh);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (seen) o[db][4 * g + e] = __builtin_fmaf(w, (float)v[e], o[db][4 * g + e]);
        }
    }
  }
};

// What a lane needs to bring its 16 bytes of every 1 KB block of a tile.
template <int D, int NKB>
struct Loader {
  typedef Tiles<D, NKB> T;
  const uint16_t *k, *v;       // of this batch and key head
  int64_t k_ss, v_ss;
  uint32_t k_off, v_off;       // lane's bytes within block 0
  int len;

  __device__ __forceinline__ void open(const WindowArgs& a, int b, int hk, int keys, int lane) {
    k = a.k + b * a.k_sb + hk * a.k_sh;
    v = a.v + b * a.v_sb + hk * a.v_sh;
    k_ss = a.k_ss;
    v_ss = a.v_ss;
    len = keys;
    const int row = lane / T::kRowLanes, chunk = lane % T::kRowLanes;
    k_off = row * (uint32_t)(2 * k_ss) + 16 * (chunk ^ T::swz_k(row));
    v_off = row * (uint32_t)(2 * v_ss) + 64 * ((chunk >> 2) ^ T::swz_v(row)) + 16 * (chunk & 3);
  }
  // Blocks b0, b0 + step .. of the tile at key k0 into the LDS at kt and vt.  The descriptor ends behind the last key there is, rows
  // behind it arrive as zeros; its base is the tile's, so that no offset needs more than 32 bits however long the cache is.
  template <int kCount>
  __device__ __forceinline__ void issue(int k0, int b0, int step, uint32_t kt, uint32_t vt) const {
    const int valid = min(len - k0, T::kKeys);
    const uint32_t kb = 2 * (uint32_t)k_ss, vb = 2 * (uint32_t)v_ss;
    const u32x4 rk = make_rsrc(k + (int64_t)k0 * k_ss, valid > 0 ? (valid - 1) * kb + T::kRowBytes : 0u);
    const u32x4 rv = make_rsrc(v + (int64_t)k0 * v_ss, valid > 0 ? (valid - 1) * vb + T::kRowBytes : 0u);
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int blk = b0 + i * step;
      load_block_to_lds(rk, (k_off ^ (64u * (blk & T::kBlockXor))) + blk * T::kBlockRows * kb, 0, kt + blk * 1024);
    }
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      const int blk = b0 + i * step;
      load_block_to_lds(rv, v_off + blk * T::kBlockRows * vb, 0, vt + blk * 1024);
    }
  }
};

// The workgroup's item: part, rows (the last ones first: under a causal border without a window they see most), batch and key head.
struct Item {
  int index, part, row0, b, hk;
};
__device__ __forceinline__ bool item_of(const WindowArgs& a, int rows, Item& it) {
  const int xcd = blockIdx.x % kXcds, at = blockIdx.x / kXcds;
  it.index = xcd * a.per_xcd + at;      // an XCD works through neighbouring items, which share keys in its L2
  if (it.index >= a.items) return false;
  const int t = it.index / a.parts;
  it.part = it.index - t * a.parts;
  const int unit = t / a.row_tiles;
  it.row0 = (a.row_tiles - 1 - (t - unit * a.row_tiles)) * rows;
  it.b = unit / a.Hk;
  it.hk = unit - it.b * a.Hk;
  return true;
}

typedef __attribute__((address_space(3))) uint8_t* lds_ptr_t;

template <int D>
struct SharedLds {
  static constexpr int kStagePitch = 2 * D + 16;
  static constexpr int kBytes = 4 * Tiles<D, 2>::kBytes;
  static_assert(kWaves * 32 * kStagePitch <= kBytes, "the epilogue's rows fit the tile buffers");
};

template <int D, bool kHalf>
__global__ __launch_bounds__(kThreads, D == 64 ? 4 : 2) void attn_window_kernel(const WindowArgs a) {
  typedef Tiles<D, 2> T;
  typedef Elem<kHalf> E;
  extern __shared__ __align__(1024) uint8_t lds[];
  Item it;
  if (!item_of(a, kRowsShared, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int len = keys_of(a, it.b);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const Span first = span_of(a, len, it.row0 / a.group);
  const Span last = span_of(a, len, min(it.row0 + kRowsShared - 1, a.rows - 1) / a.group);
  const TileList list = tiles_of<T::kKeys>(a, first, last);
  auto key_of = [&](int t) __attribute__((always_inline)) { return (t < list.n_sink ? t : list.w0 + t - list.n_sink) * T::kKeys; };
  Loader<D, 2> ld;
  ld.open(a, it.b, it.hk, len, lane);
  constexpr int kPer = T::kBlocks / kWaves;
  auto issue = [&](int t) __attribute__((always_inline)) {
    const uint32_t at = lds0 + (t & 1) * 2 * T::kBytes;
    ld.template issue<kPer>(key_of(t), wave, kWaves, at, at + T::kBytes);
  };
  if (list.n > 0) issue(0);
  RowState<D, kHalf, 2> st;
  const int row0 = it.row0 + 32 * wave;
  st.open(a, it.b, it.hk, row0, len, lane);
  for (int t = 0; t < list.n; ++t) {
    wait_loads_barrier();        // the tile is there, and nobody reads the one before any more
    if (t + 1 < list.n) issue(t + 1);
    const int k0 = key_of(t);
    if (st.needs(k0)) {
      const uint8_t* kt = lds + (t & 1) * 2 * T::kBytes;
      st.tile(kt, kt + T::kBytes, k0, lane);
    }
  }
  // Rows of the result through the LDS, so that a store covers whole lines.
  const int col = lane & 31, hh = lane >> 5;
  const float l = st.l_run + __shfl_xor(st.l_run, 32);
  const float inv = l != 0.f ? 1.f / l : 0.f;      // (an undefined sum stays one)
  wait_loads_barrier();
  constexpr int kPitch = SharedLds<D>::kStagePitch;
  uint8_t* stage = lds + wave * 32 * kPitch;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typename E::x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(st.o[db][4 * g + e] * inv);
      *reinterpret_cast<typename E::x4*>(stage + col * kPitch + 64 * db + 16 * g + 8 * hh) = h;
    }
  __builtin_amdgcn_wave_barrier();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (hh == 0 && row0 + col < a.rows) {
    const int s = (row0 + col) / a.group, g = row0 + col - s * a.group;
    a.lse[((int64_t)it.b * a.H + it.hk * a.group + g) * a.Sq + s] =
        l != 0.f ? (st.m_ref * st.c + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 32 / (64 / T::kRowLanes); ++i) {
    const int r = i * (64 / T::kRowLanes) + lane / T::kRowLanes, chunk = lane % T::kRowLanes;
    const int row = row0 + r;
    if (row < a.rows) {
      const int s = row / a.group, g = row - s * a.group;
      const u32x4 x = *reinterpret_cast<const u32x4*>(stage + r * kPitch + 16 * chunk);
      __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(a.out + (((int64_t)it.b * a.Sq + s) * a.H + it.hk * a.group + g) * D + 8 * chunk));
    }
  }
}

// Few rows.  The LDS holds two tiles (K and V) of each wavefront, then the four states.
template <int D>
struct FewLds {
  static constexpr int kBytes = kWaves * 4 * Tiles<D, 1>::kBytes;
  static_assert(kWaves * 32 * D * 4 <= kBytes, "the states fit the tile buffers");
  static constexpr int kAll = kBytes + kWaves * 256;      // and a maximum and a sum a row and wavefront
};

template <int D, bool kHalf>
__global__ __launch_bounds__(kThreads) void attn_window_few_kernel(const WindowArgs a) {
  typedef Tiles<D, 1> T;
  typedef Elem<kHalf> E;
  extern __shared__ __align__(1024) uint8_t lds[];
  Item it;
  if (!item_of(a, kRowsFew, it)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, hh = lane >> 5;
  const int len = keys_of(a, it.b);
  RowState<D, kHalf, 1> st;
  st.open(a, it.b, it.hk, it.row0, len, lane);
  const TileList list = tiles_of<T::kKeys>(a, st.first, st.last);
  auto key_of = [&](int t) __attribute__((always_inline)) { return (t < list.n_sink ? t : list.w0 + t - list.n_sink) * T::kKeys; };
  // the part's tiles, and of them every fourth
  const int t0 = (int)((int64_t)list.n * it.part / a.parts), t1 = (int)((int64_t)list.n * (it.part + 1) / a.parts);
  uint8_t* mine = lds + wave * 4 * T::kBytes;
  const uint32_t mine0 = (uint32_t)(uintptr_t)(lds_ptr_t)mine;
  Loader<D, 1> ld;
  ld.open(a, it.b, it.hk, len, lane);
  auto issue = [&](int t, int buf) __attribute__((always_inline)) {
    const uint32_t at = mine0 + buf * 2 * T::kBytes;
    ld.template issue<T::kBlocks>(key_of(t), 0, 1, at, at + T::kBytes);
  };
  int buf = 0;
  if (t0 + wave < t1) issue(t0 + wave, 0);
  for (int t = t0 + wave; t < t1; t += kWaves, buf ^= 1) {
    wait_loads();
    if (t + kWaves < t1) issue(t + kWaves, buf ^ 1);
    const uint8_t* kt = mine + buf * 2 * T::kBytes;
    st.tile(kt, kt + T::kBytes, key_of(t), lane);
  }
  // The four states as they lie in the registers; a wavefront then adds up its quarter of the columns.
  float l = st.l_run + __shfl_xor(st.l_run, 32);
  wait_loads();
  float* slot = reinterpret_cast<float*>(lds + wave * (32 * D * 4)) + lane * 4;
  float* ml = reinterpret_cast<float*>(lds + FewLds<D>::kBytes);
  __syncthreads();
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
  float m[kWaves], w[kWaves], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    m[i] = ml[i * 64 + col];
    top = fmaxf(top, m[i]);
  }
  l = 0.f;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    w[i] = m[i] > -INFINITY ? __builtin_amdgcn_exp2f(m[i] - top) : 0.f;    // a state without a key
    if (m[i] > -INFINITY) l = __builtin_fmaf(w[i], ml[i * 64 + 32 + col], l);
  }
  const int row = it.row0 + col;
  const bool live = row < a.rows;
  const int s = min(row, a.rows - 1) / a.group, g0 = min(row, a.rows - 1) - s * a.group;
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const int64_t head = it.hk * a.group + g0;
  uint16_t* out = a.out + (((int64_t)it.b * a.Sq + s) * a.H + head) * D;
  const int64_t part_row = (int64_t)it.index * 32 + col;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) {
    const int q = wave * (D / 32) + i;             // group of 4 registers: d = 8 q + 4 hh ..
    f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < kWaves; ++j) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + j * (32 * D * 4)) + lane * 4 + q * 256);
      if (m[j] > -INFINITY)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w[j], x[e], sum[e]);
    }
    if (!live) continue;
    if (a.parts > 1) {
      *reinterpret_cast<f32x4*>(a.part_out + part_row * D + 8 * q + 4 * hh) = sum;
    } else {
      typename E::x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(sum[e] * inv);
      *reinterpret_cast<typename E::x4*>(out + 8 * q + 4 * hh) = h;
    }
  }
  if (wave == 0 && hh == 0 && live) {
    if (a.parts > 1) {
      a.part_ml[part_row * 2] = top;
      a.part_ml[part_row * 2 + 1] = l;
    } else {
      a.lse[((int64_t)it.b * a.H + head) * a.Sq + s] = l != 0.f ? (top + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
    }
  }
}

// Adds up the parts of a row: a lane group of D / 4 lanes a row.
template <int D, bool kHalf>
__global__ __launch_bounds__(256) void attn_window_fold_kernel(const WindowArgs a) {
  typedef Elem<kHalf> E;
  constexpr int kLanes = D / 4;
  const int c = threadIdx.x % kLanes;
  const int64_t at = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
  const int tile = (int)(at / 32), r = (int)(at % 32);
  if (tile >= a.items / a.parts) return;
  const int unit = tile / a.row_tiles;
  const int row = (a.row_tiles - 1 - (tile - unit * a.row_tiles)) * kRowsFew + r;
  if (row >= a.rows) return;
  float top = -INFINITY, l = 0.f;
  const int64_t first = (int64_t)tile * a.parts * 32 + r;
  for (int p = 0; p < a.parts; ++p) top = fmaxf(top, a.part_ml[(first + 32 * p) * 2]);
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < a.parts; ++p) {
    const int64_t i = first + 32 * p;
    const float m = a.part_ml[i * 2];
    if (!(m > -INFINITY)) continue;
    const float w = __builtin_amdgcn_exp2f(m - top);
    l = __builtin_fmaf(w, a.part_ml[i * 2 + 1], l);
    const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_out + i * D + 4 * c);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w, x[e], sum[e]);
  }
  const int s = row / a.group, b = unit / a.Hk, h = (unit - b * a.Hk) * a.group + row - s * a.group;
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

template <typename Kernel>
int launch(Kernel kernel, const WindowArgs& a, unsigned grid, int lds, hipStream_t stream) {
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
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(kThreads), lds, stream, a);
  return hip_fail(hipGetLastError(), "attn_window launch");
}

template <int D, bool kHalf>
int launch_dim(WindowArgs& a, int64_t units, int n_cus, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  const int64_t shared = units * ((a.rows + kRowsShared - 1) / kRowsShared);
  const bool few = shared < 2 * n_cus;
  a.row_tiles = (a.rows + (few ? kRowsFew : kRowsShared) - 1) / (few ? kRowsFew : kRowsShared);
  int64_t items = units * a.row_tiles;
  a.parts = 1;
  if (few) {
    // keys that a row tile may see, in tiles
    const int64_t seen = a.left < 0 || a.right < 0 ? a.Sk : std::min<int64_t>(a.Sk, (int64_t)a.left + a.right + a.sinks + kRowsFew + 2 * a.frame);
    const int64_t tiles = (seen + 31) / 32;
    const int64_t slots = (int64_t)n_cus * (D == 64 ? 2 : 1);
    const int64_t bytes = items * (32 * (D + 2) * 4);
    int64_t most = std::min<int64_t>(64, tiles / (2 * kWaves));
    if (!workspace || bytes <= 0) most = 1;
    else most = std::min(most, workspace_bytes / bytes);
    // rounds of the chip x tiles of a workgroup
    int64_t best = (items + slots - 1) / slots * ((tiles + kWaves - 1) / kWaves);
    for (int64_t p = 2; p <= most; ++p) {
      const int64_t cost = (items * p + slots - 1) / slots * ((tiles + kWaves * p - 1) / (kWaves * p) + 2) + 4;
      if (cost < best) {
        best = cost;
        a.parts = (int)p;
      }
    }
    items *= a.parts;
  }
  if (items > (1 << 28)) {
    set_error("too many query tiles (%lld)", (long long)items);
    return DT_ERR_INVALID;
  }
  a.items = (int32_t)items;
  a.per_xcd = (a.items + kXcds - 1) / kXcds;
  if (a.parts > 1) {
    a.part_out = static_cast<float*>(workspace);
    a.part_ml = a.part_out + items * 32 * D;
  }
  const unsigned grid = (unsigned)(a.per_xcd * kXcds);
  if (!few) return launch(attn_window_kernel<D, kHalf>, a, grid, SharedLds<D>::kBytes, stream);
  if (int rc = launch(attn_window_few_kernel<D, kHalf>, a, grid, FewLds<D>::kAll, stream)) return rc;
  if (a.parts == 1) return DT_OK;
  const int64_t rows = items / a.parts * 32;
  const unsigned fold = (unsigned)((rows * (D / 4) + 255) / 256);
  hipLaunchKernelGGL((attn_window_fold_kernel<D, kHalf>), dim3(fold), dim3(256), 0, stream, a);
  return hip_fail(hipGetLastError(), "attn_window fold launch");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_attn_window_fwd(const void* q, const void* k, const void* v, void* out, float* lse, int32_t B, int32_t Sq, int32_t Sk,
                                  int32_t H, int32_t Hk, int32_t D, const int64_t* q_strides, const int64_t* k_strides,
                                  const int64_t* v_strides, const dt_window* window, float softmax_scale, int32_t flags, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
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
  const int64_t rows = (int64_t)Sq * (H / Hk), units = (int64_t)B * Hk;
  if (rows > (1ll << 30) || units > (1ll << 28) || units * ((rows + 31) / 32) > (1ll << 28)) {
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
  const int n_cus = cus();
  if (n_cus <= 0) {
    set_error("no current device");
    return DT_ERR_HIP;
  }
  const hipStream_t st = (hipStream_t)stream;
  const bool half = (flags & DT_ATTN_FP16) != 0;
  if (D == 128)
    return half ? launch_dim<128, true>(a, units, n_cus, workspace, workspace_bytes, st)
                : launch_dim<128, false>(a, units, n_cus, workspace, workspace_bytes, st);
  return half ? launch_dim<64, true>(a, units, n_cus, workspace, workspace_bytes, st)
              : launch_dim<64, false>(a, units, n_cus, workspace, workspace_bytes, st);
}
