// Attention states in 8 bits (gfx950): stored, read back, and merged with states of any other format.
//
// Blocks of 32 elements along D carry one scale byte.  With M the largest element of the format (448 for e4m3, 127 for int8) and amax the
// block's largest magnitude,
//   e = the smallest integer >= -127 with amax <= M 2^e,   scale byte = e + 127,   element = rne(x 2^-e),   value = element 2^e,
// so nothing saturates, the scaling itself is exact and any arithmetic gives the same elements.  A block that holds an infinite or
// undefined value has scale byte 255 and reads as undefined (a format without such values must not make numbers of them).
//
// The merge is that of the 16-bit states: lse = log sum_i exp(lse_i), out = sum_i exp(lse_i - lse) out_i, fp32 sums, one pass; a single
// state is copied.  Bound by HBM: D + D / 32 + 4 bytes a row and 8-bit state instead of 2 D + 4.
// 6 of 8 bits and 2 of 16 of 14 882 x 24 heads of 128 into fp32: 101.4 us, 6.5 TB/s; one stored and loaded 51.7 us, 5.5 TB/s; four merged into the first, in 8 bits, 49.4 us, 4.9 TB/s.
//
// A lane owns 8 consecutive elements, so 4 lanes hold a block and its maximum is two exchanges inside a quad; a row's lanes are
// neighbours in a wavefront.  States come sorted by the size of their elements, each size in batches whose loads are in flight together.
#include <algorithm>

#include "dt_common.h"
#include "state_rows.h"

namespace dt {
namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
constexpr int kBlock = 32;   // elements of a scale

struct BlockArgs {
  const void* out[DT_MAX_MERGE];        // 8-bit states first, then 16-bit ones, then fp32 ones
  const uint8_t* scales[DT_MAX_MERGE];  // [B,Sq,H,D/32] of the 8-bit ones
  const float* lse[DT_MAX_MERGE];
  uint64_t bsh_mask;    // bit i: lse[i] is [B,Sq,H] (else [B,H,Sq])
  uint64_t kind_mask;   // bit i: int8 instead of e4m3, IEEE half instead of bfloat16
  int32_t n8, n16, n;   // states below n8 are 8-bit, below n16 at most 16-bit
  void* dst;
  uint8_t* dst_scales;
  float* dst_lse;
  int32_t dst_dtype, dst_bsh;
  RowIndex at;
  Quotient by_h_tiles, by_s_tiles;      // tiles of rows (merges)
};

// The arguments where they arrive, in the kernarg segment: indexed in unrolled batches of a by-value parameter, the optimiser makes a private copy
// of the tables for every lane (8 states a batch: 122 -> 1950 us).
typedef const BlockArgs __attribute__((address_space(4))) KernArgs;
__device__ __forceinline__ KernArgs& kernel_args() { return *(KernArgs*)__builtin_amdgcn_kernarg_segment_ptr(); }

__device__ __forceinline__ float scale_of(uint32_t byte) {   // 2^(byte - 127); byte 0 is below the normal numbers, 255 infinite
  return __uint_as_float(byte ? byte << 23 : 0x00400000u);
}

// Raw 8 elements of a lane.
template <int kBytes> struct Raw;
template <> struct Raw<1> { u32x2 x; uint32_t scale; };
template <> struct Raw<2> { u32x4 x; };
template <> struct Raw<4> { u32x4 x, y; };

template <int kBytes>
__device__ __forceinline__ void load(KernArgs& a, int i, int64_t elem, Raw<kBytes>& r) {
  const uint8_t* p = static_cast<const uint8_t*>(a.out[i]) + elem * kBytes;
  if constexpr (kBytes == 1) {
    r.x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    r.scale = a.scales[i][elem / kBlock];
  } else {
    r.x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
    if constexpr (kBytes == 4) r.y = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + 1);
  }
}

// acc += w x.  A state that is not there (an lse of -inf) is left out, whatever it holds.  The weight of one that is there is above 0, so its undefined
// values stay undefined, also where fp32 has no number for the weight: in whatever order the states come.
template <int kBytes>
__device__ __forceinline__ void add(const Raw<kBytes>& r, bool kind, bool there, float w, float (&acc)[8]) {
  float x[8];
  if constexpr (kBytes == 1) {
    w = there ? w * scale_of(r.scale) : 0.f;       // (the scale may be infinite)
    const uint32_t word[2] = {there ? r.x.x : 0u, there ? r.x.y : 0u};     // (e4m3 has undefined elements of its own)
    if (kind) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)((int32_t)(word[e / 4] << (24 - 8 * (e % 4))) >> 24);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)word[e / 4], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)word[e / 4], true);
        x[e] = lo.x;
        x[e + 1] = lo.y;
        x[e + 2] = hi.x;
        x[e + 3] = hi.y;
      }
    }
  } else if constexpr (kBytes == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t word = there ? r.x[e] : 0u;   // (a bit cast of the vector's element itself reads its first one)
      if (kind) {
        const f32x2 f = __builtin_convertvector(__builtin_bit_cast(f16x2, word), f32x2);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
      } else {
        x[2 * e] = __uint_as_float(word << 16);
        x[2 * e + 1] = __uint_as_float(word & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = there ? __uint_as_float(r.x[e]) : 0.f;
      x[4 + e] = there ? __uint_as_float(r.y[e]) : 0.f;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(w, x[e], acc[e]);
}

struct Sums {
  float acc[8], m, den;
};
// Where a lane's elements are, and their row's lse: in the states' own memory, or of all states in the LDS (kRows values a state), where the workgroup
// brings them while the first states' elements are on their way.
constexpr int kWaves = kThreads / 64;
template <int kRows>
struct Place {
  int64_t elem;
  uint32_t row, bhs;
  float* lses;                  // lse of state i at [i * kRows + mine]
  int mine;
  bool staged;
  static constexpr int kAhead = 2;
  float ahead[kAhead];          // of the states wave and wave + kWaves, row `lane` of the tile
  uint32_t as_bsh, as_bhs;      // that row's place

  __device__ __forceinline__ float brought(KernArgs& a, int i) const { return a.lse[i][(a.bsh_mask >> i) & 1 ? as_bsh : as_bhs]; }
  __device__ __forceinline__ void begin(KernArgs& a, int wave, int lane) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = wave + k * kWaves;
      if (i < a.n && lane < kRows) ahead[k] = brought(a, i);
    }
  }
  __device__ __forceinline__ void stage(KernArgs& a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (lane < kRows) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (wave + k * kWaves < a.n) lses[(wave + k * kWaves) * kRows + lane] = ahead[k];
      for (int i = wave + kAhead * kWaves; i < a.n; i += kWaves) lses[i * kRows + lane] = brought(a, i);
    }
    // (the elements stay on their way: a __syncthreads() would wait for them)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    staged = true;
  }
};

// NB states' loads are in flight together, and nothing between them and the folding branches: behind a branch on the lse the compiler would issue
// the other loads after the lse's have come.
template <int kBytes, int NB, int kRows>
__device__ __forceinline__ void batch(int i0, Place<kRows>& at, Sums& s) {
  KernArgs& a = kernel_args();
  Raw<kBytes> r[NB];
  float l[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if constexpr (kRows == 0) l[j] = a.lse[i0 + j][(a.bsh_mask >> (i0 + j)) & 1 ? at.row : at.bhs];
    load<kBytes>(a, i0 + j, at.elem, r[j]);
  }
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (kRows > 0) {
    if (!at.staged) at.stage(a);
#pragma unroll
    for (int j = 0; j < NB; ++j) l[j] = at.lses[(i0 + j) * kRows + at.mine];
  }
  const uint32_t kinds = (uint32_t)(a.kind_mask >> i0);
  float m = s.m;
#pragma unroll
  for (int j = 0; j < NB; ++j) m = fmaxf(m, l[j]);
  const float top = m > -INFINITY ? m : 0.f;       // (no state with a key so far: all weights are 0; an undefined lse stays one)
  const float rescale = __expf(s.m - top);
  s.den *= rescale;
#pragma unroll
  for (int e = 0; e < 8; ++e) s.acc[e] *= rescale;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const float w = __expf(l[j] - top);
    s.den += w;
    add<kBytes>(r[j], (kinds >> j) & 1, l[j] != -INFINITY, w, s.acc);
  }
  s.m = m;
}
template <int kBytes, int NB, int kRows>
__device__ __forceinline__ void rest(int i0, int n, Place<kRows>& at, Sums& s) {
  if constexpr (NB >= 1) {
    if (n == NB) batch<kBytes, NB>(i0, at, s);
    else rest<kBytes, NB - 1>(i0, n, at, s);
  }
}
template <int kBytes, int kBatch, int kRows>
__device__ __forceinline__ void states(int i0, int i1, Place<kRows>& at, Sums& s) {
  for (; i0 + kBatch <= i1; i0 += kBatch) batch<kBytes, kBatch>(i0, at, s);
  rest<kBytes, kBatch - 1>(i0, i1 - i0, at, s);
}

// The other lanes of a quad: lane ^ 1, lane ^ 2.
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, kCtrl, 0xf, 0xf, true);
}

// 8 elements in the destination's format; all lanes of a wavefront, `live` those whose row is there (a quad's are, or are not, together).
__device__ __forceinline__ void store(KernArgs& a, int64_t elem, bool live, int64_t elems, const float (&x)[8]) {
  uint8_t* p = static_cast<uint8_t*>(a.dst);
  if (a.dst_dtype == DT_FP32) {
    // A lane's 32 bytes as two stores would each write every other 16 bytes of a line (9 % more bytes written): through the LDS, whole kilobytes.
    __shared__ f32x4 stage[kThreads / 64][128];
    f32x4 lo, hi;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[e] = x[e];
      hi[e] = x[4 + e];
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    stage[wave][2 * lane] = lo;
    stage[wave][2 * lane + 1] = hi;
    __builtin_amdgcn_wave_barrier();
    const int64_t first = elem - 8 * lane;       // of the wavefront
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 y = stage[wave][64 * i + lane];
      if (first + 256 * i + 4 * lane < elems) __builtin_nontemporal_store(y, reinterpret_cast<f32x4*>(p + (first + 256 * i + 4 * lane) * 4));
    }
  } else if (!live) {
    return;
  } else if (a.dst_dtype == DT_BF16 || a.dst_dtype == DT_FP16) {
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f32x2 f;
      f.x = x[2 * e];
      f.y = x[2 * e + 1];
      w[e] = a.dst_dtype == DT_FP16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2))
                                    : __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
    }
    __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(p + elem * 2));
  } else {
    uint32_t top = 0;     // magnitudes compare like their bits, infinite and undefined ones above all others
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
    top = max(top, dpp<0xb1>(top));
    top = max(top, dpp<0x4e>(top));
    const bool int8 = a.dst_dtype == DT_BLOCK_INT8, finite = top < 0x7f800000u;
    // amax = 1.f 2^n is at most M 2^(n - 8) with M = 1.75 2^8, at most M 2^(n - 6) with M = 1.984375 2^6, or needs one more
    const int n = (int)(top >> 23) - 127;
    const int e = max(n - (int8 ? 6 : 8) + ((top & 0x7fffffu) > (int8 ? 0x7e0000u : 0x600000u) ? 1 : 0), -127);
    const float inv = finite ? __uint_as_float((uint32_t)(127 - e) << 23) : 0.f;
    u32x2 w;
    if (int8) {
      // 1.5 2^23 added, a float's lowest bits are the nearest even integer
      uint32_t v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __float_as_uint(__builtin_fmaf(x[i], inv, 12582912.f));
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[4 * i + 3], v[4 * i + 2], 0x0c0c0400u), __builtin_amdgcn_perm(v[4 * i + 1], v[4 * i], 0x0c0c0400u), 0x05040100u);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
        w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, v, true);
      }
    }
    if (!finite) w = u32x2{0u, 0u};
    __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(p + elem));
    if ((threadIdx.x & 3) == 0) a.dst_scales[elem / kBlock] = finite ? (uint8_t)(e + 127) : 255;
  }
}

// This workgroup's place, and the first element of this lane.  The lse of consecutive queries share a line of the [B,H,Sq] layout, and workgroups go to the 8 XCDs in turn: so
// that a line is read into one L2 only, kGroup workgroups that follow each other in memory are of one XCD.
constexpr int kGroup = 64;
__device__ __forceinline__ uint32_t workgroup() {
  const uint32_t wg = blockIdx.x;
  constexpr uint32_t kSpan = 8 * kGroup;
  return (wg / kSpan + 1) * kSpan <= gridDim.x ? wg / kSpan * kSpan + (wg & 7u) * kGroup + (wg % kSpan >> 3) : wg;
}
template <int kUnits>
__device__ __forceinline__ int64_t first_elem() {
  return ((int64_t)workgroup() * (kThreads * kUnits) + threadIdx.x) * 8;
}

__device__ __forceinline__ RowIndex rows_of(KernArgs& a) {
  RowIndex at;
  at.Sq = a.at.Sq;
  at.H = a.at.H;
  at.rows = a.at.rows;
  at.by_h = {a.at.by_h.mul, a.at.by_h.shift};
  at.by_s = {a.at.by_s.mul, a.at.by_s.shift};
  return at;
}

// kTiles: a workgroup has the rows of kTileQueries queries and 512 / D heads, a wavefront one query's.  In the [B,H,Sq] layout the lse of neighbouring rows
// are a sequence apart, and fetched by the rows' own lanes they cost as many requests as the elements; those of a tile come in 16-byte
// runs, once for the four wavefronts, through the LDS.  us without and with: 14 882 x 24 heads of 128, 8 states of 8 bits 87.7 / 81.5, 6 and 2 of 16 bits
// 111.8 / 104.8, 6 69.7 / 68.3, 2 38.4 / 42.2 (shorter runs of elements); heads of 64, 9000 x 48, 6 states 51.6 / 43.0, 2 25.5 / 24.8; 2222 x 48, 5 and 3 21.5 /
// 18.5.  So heads of 64 always, heads of 128 from six states on.  From 16 queries on: 16 x 24 heads x 32 samples, 2 and 8 states of 64 3.40 / 3.21 and 5.93 / 5.62, 6 and 8
// of 128 5.62 / 5.21 and 6.62 / 6.13; with 8 queries -0.3 .. 0, with 1 to 4 -0.6 .. +0.3 us.
constexpr int kTileQueries = kThreads / 64;
// (Seven wavefronts a SIMD are asked for, but for tiles of heads of 128, which take 74 registers: with six, 5 + 3 states of 2222 x 48 heads of 64 take 18.5 us instead of 17.9.)
template <int D, bool kTiles>
__global__ __launch_bounds__(kThreads, D == 128 && kTiles ? 6 : 7) void merge_blocks_kernel(const BlockArgs args_by_value) {
  (void)args_by_value;
  constexpr int kHeads = 512 / D, kRows = kTiles ? kTileQueries * kHeads : 0;
  KernArgs& a = kernel_args();
  const RowIndex at = rows_of(a);
  const int64_t elems = (int64_t)at.rows * D;
  int64_t elem;
  Place<kRows> place;
  bool live;
  if constexpr (kTiles) {
    __shared__ float lses[DT_MAX_MERGE * kRows];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const uint32_t wg = workgroup();
    const Quotient by_h = {a.by_h_tiles.mul, a.by_h_tiles.shift}, by_s = {a.by_s_tiles.mul, a.by_s_tiles.shift};
    const uint32_t h_tiles = (uint32_t)at.H / kHeads, s_tiles = ((uint32_t)at.Sq + kTileQueries - 1) / kTileQueries;
    const uint32_t bs = quotient(wg, by_h), h0 = (wg - bs * h_tiles) * kHeads, b = quotient(bs, by_s), s0 = (bs - b * s_tiles) * kTileQueries;
    // lane r of a wavefront brings row r of every fourth state: query r % kTileQueries, head r / kTileQueries
    const uint32_t q = min(s0 + lane % kTileQueries, (uint32_t)at.Sq - 1), h = h0 + lane / kTileQueries;
    place.as_bsh = (b * (uint32_t)at.Sq + q) * (uint32_t)at.H + h;
    place.as_bhs = (b * (uint32_t)at.H + h) * (uint32_t)at.Sq + q;
    place.begin(a, wave, lane);
    const uint32_t s = s0 + wave, mine = lane / (D / 8);
    live = s < (uint32_t)at.Sq;
    place.row = (b * (uint32_t)at.Sq + min(s, (uint32_t)at.Sq - 1)) * (uint32_t)at.H + h0 + mine;
    place.bhs = (b * (uint32_t)at.H + h0 + mine) * (uint32_t)at.Sq + min(s, (uint32_t)at.Sq - 1);
    place.elem = elem = (int64_t)place.row * D + 8 * (lane % (D / 8));
    place.lses = lses;
    place.mine = kTileQueries * mine + wave;
    place.staged = false;
  } else {
    elem = first_elem<1>();
    live = elem < elems;
    place.elem = live ? elem : 0;          // (lanes behind the last row read the first one's and store nothing)
    place.row = (uint32_t)(place.elem / D);
    place.bhs = bhs_of(at, place.row);
  }
  Sums s;
#pragma unroll
  for (int e = 0; e < 8; ++e) s.acc[e] = 0.f;
  s.m = -INFINITY;
  s.den = 0.f;
  states<1, 4>(0, a.n8, place, s);
  states<2, 4>(a.n8, a.n16, place, s);
  states<4, 2>(a.n16, a.n, place, s);
  const float inv = s.den != 0.f ? 1.f / s.den : 0.f;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = s.acc[e] * inv;
  store(a, elem, live, live ? elems : kTiles ? 0 : elems, x);
  if (live && elem % D == 0) a.dst_lse[a.dst_bsh ? place.row : place.bhs] = s.den != 0.f ? s.m + __logf(s.den) : -INFINITY;
}

// One state into another format, its lse bit for bit.  From kManyWorkgroups workgroups on, with twice the elements each.  A state of 14 882 x 24 heads of
// 128, int8, stored and loaded: 52.6 us (one unit a lane 54.0, four 54.7; with the lse in the rows' first lanes 56.0).  us with one unit a lane and with two, a store of 24 heads of
// 64, by workgroups: 750 2.71 / 3.02, 1500 3.27 / 3.42, 2048 4.21 / 3.77, 3000 5.41 / 4.98, 4095 6.77 / 6.39, 6000 8.77 / 8.79; of 128: 1500 3.29 / 3.45, 2250 4.63 / 4.28,
// 4096 6.75 / 6.44, 6000 8.69 / 8.77, 22 323 25.35 / 25.05; loads alike.
constexpr unsigned kManyWorkgroups = 2048;
constexpr int kCopyUnits = 2;
// kUnits times kThreads lanes' elements a workgroup.
template <int D, int kBytes, int kUnits>
__global__ __launch_bounds__(kThreads) void copy_blocks_kernel(const BlockArgs args_by_value) {
  (void)args_by_value;
  KernArgs& a = kernel_args();
  const RowIndex at = rows_of(a);
  const int64_t elems = (int64_t)at.rows * D, elem = first_elem<kUnits>();
  // an lse in one layout on both sides is a flat range of its own, of which a workgroup moves what its elements' rows are in number
  constexpr uint32_t kRows = kThreads * 8 * kUnits / D;
  const bool flat = (a.bsh_mask & 1) == (a.dst_bsh ? 1u : 0u);
  const uint32_t mine = (uint32_t)((elem - 8 * (int64_t)threadIdx.x) / D) + threadIdx.x;
  const bool moves = flat && threadIdx.x < kRows && mine < at.rows;
  Raw<kBytes> r[kUnits];
  float l[kUnits];
  uint32_t bhs[kUnits];
  if (moves) l[0] = a.lse[0][mine];
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t e = elem + u * (kThreads * 8), from = e < elems ? e : 0;
    load<kBytes>(a, 0, from, r[u]);
    if (!flat) {
      bhs[u] = bhs_of(at, (uint32_t)(from / D));
      if (e % D == 0) l[u] = a.lse[0][a.bsh_mask & 1 ? (uint32_t)(from / D) : bhs[u]];
    }
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int u = 0; u < kUnits; ++u) {
    const int64_t e = elem + u * (kThreads * 8);
    const bool live = e < elems;
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = -0.f;       // (-0 + -0 keeps its sign)
    add<kBytes>(r[u], a.kind_mask & 1, true, 1.f, x);
    store(a, e, live, elems, x);
    if (!flat && live && e % D == 0) a.dst_lse[a.dst_bsh ? (uint32_t)(e / D) : bhs[u]] = l[u];
  }
  if (moves) a.dst_lse[mine] = l[0];
}

bool is_block(int dtype) { return dtype == DT_BLOCK_E4M3 || dtype == DT_BLOCK_INT8; }
int element_bytes(int dtype) { return is_block(dtype) ? 1 : dtype == DT_FP32 ? 4 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_state(const dt_state& s, const char* what, int i) {
  if (s.dtype < DT_BF16 || s.dtype > DT_BLOCK_INT8 || (s.lse_layout != DT_LSE_BHS && s.lse_layout != DT_LSE_BSH)) {
    set_error("%s %d: bad dtype %d or lse layout %d", what, i, s.dtype, s.lse_layout);
    return DT_ERR_INVALID;
  }
  if (!s.out || !aligned16(s.out) || !s.lse || (is_block(s.dtype) && !s.scales)) {
    set_error("%s %d: out must be non-null and 16-byte aligned, lse and the scales of an 8-bit state non-null", what, i);
    return DT_ERR_INVALID;
  }
  return DT_OK;
}

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_merge_block_states(int32_t n, const dt_state* states, const dt_state* dst, int32_t B, int32_t Sq, int32_t H, int32_t D,
                                     void* stream) {
  if (n < 1 || n > DT_MAX_MERGE || !states || !dst) {
    set_error("%d states: need 1..%d, and a destination", n, DT_MAX_MERGE);
    return DT_ERR_INVALID;
  }
  if (B <= 0 || Sq <= 0 || H <= 0) {
    set_error("B, Sq, H must be positive (got %d, %d, %d)", B, Sq, H);
    return DT_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    set_error("head dim %d not built (64 and 128 are)", D);
    return DT_ERR_UNSUPPORTED;
  }
  // (a grid holds fewer than 2^32 lanes)
  const __int128 rows = (__int128)B * Sq * H;
  if (rows * (D / 8) > (1ll << 32) - kThreads || rows >= (1ll << 31)) {
    set_error("too many rows (%d x %d x %d)", B, Sq, H);
    return DT_ERR_INVALID;
  }
  if (int rc = check_state(*dst, "destination", 0)) return rc;
  for (int i = 0; i < n; ++i)
    if (int rc = check_state(states[i], "state", i)) return rc;
  BlockArgs a{};
  int at = 0;
  for (const int bytes : {1, 2, 4}) {
    for (int i = 0; i < n; ++i) {
      const dt_state& s = states[i];
      if (element_bytes(s.dtype) != bytes) continue;
      a.out[at] = s.out;
      a.scales[at] = s.scales;
      a.lse[at] = s.lse;
      if (s.lse_layout == DT_LSE_BSH) a.bsh_mask |= 1ull << at;
      if (s.dtype == DT_BLOCK_INT8 || s.dtype == DT_FP16) a.kind_mask |= 1ull << at;
      ++at;
    }
    if (bytes == 1) a.n8 = at;
    if (bytes == 2) a.n16 = at;
  }
  a.n = n;
  a.dst = dst->out;
  a.dst_scales = dst->scales;
  a.dst_lse = dst->lse;
  a.dst_dtype = dst->dtype;
  a.dst_bsh = dst->lse_layout == DT_LSE_BSH;
  a.at = row_index(B, Sq, H);
  const dim3 grid((unsigned)(((int64_t)a.at.rows * (D / 8) + kThreads - 1) / kThreads)), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
  const bool some = grid.x >= kManyWorkgroups;
  const dim3 fewer((grid.x + kCopyUnits - 1) / kCopyUnits);
#define DT_LAUNCH(kernel) hipLaunchKernelGGL(kernel, grid, block, 0, st, a)
#define DT_COPY(D, bytes)                                                                                     \
  do {                                                                                                        \
    if (some) hipLaunchKernelGGL((copy_blocks_kernel<D, bytes, kCopyUnits>), fewer, block, 0, st, a);         \
    else DT_LAUNCH((copy_blocks_kernel<D, bytes, 1>));                                                        \
  } while (0)
  const int heads = 512 / D;
  const uint64_t all = n == 64 ? ~0ull : (1ull << n) - 1;
  const int s_tiles = (Sq - 1) / kTileQueries + 1;
  if (n >= (D == 64 ? 2 : 6) && H % heads == 0 && Sq >= 16 && a.bsh_mask != all && (int64_t)B * s_tiles * (H / heads) < 1 << 24) {
    a.by_h_tiles = quotient_by(H / heads);
    a.by_s_tiles = quotient_by(s_tiles);
    const dim3 tiles((unsigned)((int64_t)B * s_tiles * (H / heads)));
    if (D == 128) hipLaunchKernelGGL((merge_blocks_kernel<128, true>), tiles, block, 0, st, a);
    else hipLaunchKernelGGL((merge_blocks_kernel<64, true>), tiles, block, 0, st, a);
  } else if (n > 1) {
    if (D == 128) DT_LAUNCH((merge_blocks_kernel<128, false>));
    else DT_LAUNCH((merge_blocks_kernel<64, false>));
  } else {
    const int bytes = element_bytes(states[0].dtype);
    if (D == 128) {
      if (bytes == 1) DT_COPY(128, 1);
      else if (bytes == 2) DT_COPY(128, 2);
      else DT_COPY(128, 4);
    } else {
      if (bytes == 1) DT_COPY(64, 1);
      else if (bytes == 2) DT_COPY(64, 2);
      else DT_COPY(64, 4);
    }
  }
#undef DT_COPY
#undef DT_LAUNCH
  return hip_fail(hipGetLastError(), "merge_blocks launch");
}
