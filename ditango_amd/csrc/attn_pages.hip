// Attention of requests' new tokens over the pages of a cache that they share (gfx950).
//
// Row i of the n new tokens of a request with len tokens stands at position len - n + i among its keys; which of them it sees is a window as of
// attn_window.hip, and the result is a state (out, lse) like its.  The rows' arithmetic is attn_rows.h's, in the same two forms:
//   * shared tiles: 256 rows of one request and key head a workgroup, which walks the 64-key tiles that some row sees;
//   * few rows: 32 rows, whose four or eight wavefronts take 32-key tiles in turn.
// A request's rows (new tokens x query heads of a key head) go in tiles of 256, and what is left over in tiles of 32 where that is at most 64 or 96.
// Batches of requests that have no more rows than that run in a kernel with few rows only; in the other one both forms run side by side.
//
// Many rows are bound by the matrix instructions at the power cap: two frames of 3600 tokens, 24 heads of 128, 32 400 keys each, 2.54 .. 2.64 ms, 1.1
// PFLOP/s at 1.66 GHz (on contiguous keys 2.47 .. 2.49); heads of 64 by softmax and products in turn (a frame of 1350 of two rollouts, 48 heads, 0.51 ..
// 0.55 ms, 0.83 .. 0.90 PFLOP/s).  Single tokens are bound by the memory: 8 over 3000 to 17 776 keys of 24 heads of 128, 176 .. 190 us, 5.4 .. 5.8 TB/s; of
// 24 heads of 64, over 8192 keys each, 79 us, 5.1 TB/s.  Small calls wait: 3 requests of 4 tokens 9.3 us, of which 2.4 are an empty launch's, 2 go by until
// a workgroup has found its work, 3 until its first tile is there.
//
// Which page holds a tile is read by scalar loads one tile ahead, so that no tile waits for it; a page is a multiple of 16 tokens, and 16 rows of a tile
// are what a load's descriptor covers.  No host knows the lengths, so every workgroup finds its share of the work by itself: it reads all lengths and
// boundaries, a lane a request, settles how long a part of the keys is, and numbers row tiles, parts and key heads through (`find`).
#include <algorithm>
#include <cmath>

#include "attn_rows.h"
#include "dt_common.h"

namespace dt {
namespace {

constexpr int32_t kMostTokens = 1 << 29;   // positions, spans and lengths: their sums stay in 32 bits
constexpr int kXcds = 8;
constexpr int kWavesFew = 4;
constexpr int kMostWays = 64;              // parts of an item
constexpr int kOneMeeting = 8;             // parts of 256 rows that meet all at once
constexpr int kMostRequests = 2048;        // every workgroup reads all lengths

struct PagesArgs {
  const uint16_t* q;
  int64_t q_ss, q_sh;
  uint16_t* out;
  float* lse;
  Pages kv;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *lens, *cu;
  int32_t width, most_len, B, T, H, Hk, group;
  int32_t left, right;          // spans in tokens; -1: no border
  int32_t frame, sinks;
  Quotient by_group, by_frame;
  float scale_log2;
  // ---- how the launch runs
  int32_t few_rows;             // rows that are left over of tiles of 256 go in tiles of 32 up to here
  int32_t all_few;              // whether a grid with tiles of 256 rows has room for all rows as few rows
  int32_t groups;               // workgroups of the grid
  int32_t most_parts[2];        // for how many of them, of 256 rows (0) and of few (1), there is room for parts
  float slots;                  // workgroups at once
  float step[2], once[2], part[2];     // us: of 64 keys, of a workgroup beside them, of a part's way to memory and back
  float join;                   // ... of one of 256 rows that one CU adds to others
  float least;                  // ... of a part of few rows
  float cached;                 // ... of as many keys of all key heads as the last cache holds
  float* part_out[2];           // of slot s: sums of its rows, and (maximum in powers of two, sum) of each
  float* part_ml[2];
  uint32_t* counters[2];        // of an item's parts that are done, zero before and after the launch
  const uint8_t* served;        // 0: a request without keys, whatever its length
  int32_t all_served;           // ... but for launches without `served`, which read any bytes there: a branch around the load waits for it by itself
};

// The rows of a request, by the names of attn_rows.h
struct Queries {
  const uint16_t* q;
  int64_t q_sb, q_ss, q_sh;
  int32_t Sq, rows, group, left, right, frame, sinks, q_begin;
  Quotient by_group, by_frame;
  float scale_log2;
};
__device__ __forceinline__ Queries queries_of(const PagesArgs& a, int begin, int n) {
  return Queries{a.q + begin * a.q_ss, 0, a.q_ss, a.q_sh, n, n * a.group, a.group, a.left, a.right, a.frame, a.sinks, -1, a.by_group, a.by_frame, a.scale_log2};
}

// A workgroup's work: row tile `row0` .. of a request and key head, and of its keys the part [tiles part / ways, tiles (part + 1) / ways)
struct Work {
  int b, begin, n, len;         // request, its first row, its rows' and its keys' number
  int few, once;                // 32 rows, not 256; whose keys are read by this item only, of a launch of many
  int hk, row0, part, ways;
  int first, apart;             // slot of the item's first part, slots between its parts
  template <typename List>
  __device__ __forceinline__ void share(List& list) const {      // (2^24 tiles, 64 parts: 32 bits hold the products)
    const uint32_t n = list.end;
    if (ways > 1) {
      list.begin = (int)(n * part / ways);
      list.end = (int)(n * (part + 1) / ways);
    }
  }
};

// A lane's request: its rows, keys, tiles of 256 rows (0) and of 32 (1), and about how long one of them takes.
struct Request {
  int begin, n, len;
  int tiles[2];
  float us[2];
};
template <bool kMixed>
__device__ __forceinline__ Request request_of(const PagesArgs& a, int b) {
  Request r = {};
  if (b >= a.B) return r;
  const int from = a.cu[b], to = a.cu[b + 1], len = a.lens[b], served = a.served[b] | a.all_served;
  r.begin = min(max(from, 0), a.T);
  r.n = max(min(max(to, 0), a.T) - r.begin, 0);
  r.len = served ? min(max(len, 0), a.most_len) : 0;
  const int rows = r.n * a.group;
  int whole = 0;
  if (kMixed) {
    r.tiles[0] = rows / kRowsShared + (rows % kRowsShared > a.few_rows);
    whole = min(r.tiles[0] * kRowsShared, rows);
  }
  r.tiles[1] = (rows - whole + kRowsFew - 1) / kRowsFew;
#pragma unroll
  for (int i = kMixed ? 0 : 1; i < 2; ++i) {      // 64-key tiles that its last tile sees, the most that one does but where the window has a left border only
    const Queries qs = queries_of(a, 0, r.n);
    const int end = i ? rows : whole;
    const int hi = a.right < 0 ? r.len : span_of(qs, r.len, query_of(qs, max(end - 1, 0))).hi;
    int keys = hi;
    if (a.left >= 0) {
      const int sinks = min(a.sinks, hi);
      keys = sinks + max(hi - max(span_of(qs, r.len, query_of(qs, i ? whole : max(end - kRowsShared, 0))).lo, sinks), 0);
    }
    r.us[i] = r.tiles[i] > 0 ? (float)((keys + 63) / 64) * a.step[i] : 0.f;
  }
  return r;
}
__device__ __forceinline__ int lane_value(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
// Reductions and sums along the wavefront inside the vector instructions (__shfl is an LDS access): lane i of a row of 16 reads lane i - n, then the
// rows behind the first read the row in front of them, or the half.
template <int kCtrl, int kRows>
__device__ __forceinline__ int moved(int x, int none) { return __builtin_amdgcn_update_dpp(none, x, kCtrl, kRows, 0xf, false); }
template <typename Op>
__device__ __forceinline__ int along(int x, int none, Op op) {      // lane i: of lanes 0 .. i
  x = op(x, moved<0x111, 0xf>(x, none));
  x = op(x, moved<0x112, 0xf>(x, none));
  x = op(x, moved<0x114, 0xf>(x, none));
  x = op(x, moved<0x118, 0xf>(x, none));
  x = op(x, moved<0x142, 0xa>(x, none));
  return op(x, moved<0x143, 0xc>(x, none));
}
constexpr int kMost = 1 << 24;      // sums stop here, beyond every workgroup of a grid
__device__ __forceinline__ int sums_along(int x) {
  return along(x, 0, [](int u, int v) { return min(u + v, kMost); });
}
__device__ __forceinline__ int wave_max(int x) {
  return lane_value(along(x, INT32_MIN, [](int u, int v) { return max(u, v); }), 63);
}
__device__ __forceinline__ float as_float(int x) { return __builtin_bit_cast(float, x); }
__device__ __forceinline__ int as_int(float x) { return __builtin_bit_cast(int, x); }
__device__ __forceinline__ float wave_sum(float x) {
  return as_float(lane_value(along(as_int(x), 0, [](int u, int v) { return as_int(as_float(u) + as_float(v)); }), 63));
}
__device__ __forceinline__ float wave_max(float x) {
  return as_float(lane_value(along(as_int(x), 0, [](int u, int v) { return as_int(fmaxf(as_float(u), as_float(v))); }), 63));
}
__device__ __forceinline__ float wave_min(float x) {
  return as_float(lane_value(along(as_int(x), as_int(INFINITY), [](int u, int v) { return as_int(fminf(as_float(u), as_float(v))); }), 63));
}
// n / d and n % d, n < 2^23
__device__ __forceinline__ int divided(int n, int d, int* rest) {
  int q = (int)((float)n * __builtin_amdgcn_rcpf((float)d));
  q -= q * d > n;
  q += (q + 1) * d <= n;
  q = __builtin_amdgcn_readfirstlane(q);
  *rest = n - q * d;
  return q;
}
// Parts of an item that takes `us`, where a part takes 1 / inv of them.  (In floating point: nothing depends on it but that all agree.)
__device__ __forceinline__ int ways_of(float us, float inv) { return min(max((int)__builtin_ceilf(us * inv - 0.001f), 1), kMostWays); }
__device__ __forceinline__ float over(float x, float y) { return x * __builtin_amdgcn_rcpf(y); }      // to 2^-22 or so

// Finds workgroup blockIdx.x's work; false: it has none.  *none: whether there are rows that no request owns.
template <bool kMixed>
__device__ __forceinline__ bool find(const PagesArgs& a, Work& w, bool* none) {
  const int lane = threadIdx.x & 63;
  // (workgroups are dealt round the XCDs)
  int g = blockIdx.x;
  Request r = request_of<kMixed>(a, lane);
  uint32_t owned = r.n;
  float most = r.us[0], keys = r.us[1], work[2] = {}, items[2] = {};
#pragma unroll
  for (int i = kMixed ? 0 : 1; i < 2; ++i) {
    work[i] = (float)r.tiles[i] * r.us[i];
    items[i] = (float)r.tiles[i];
  }
  for (int b0 = 64; b0 < a.B; b0 += 64) {
    const Request x = request_of<kMixed>(a, b0 + lane);
    owned += x.n;
    most = max(most, x.us[0]);
    keys += x.us[1];
#pragma unroll
    for (int i = kMixed ? 0 : 1; i < 2; ++i) {
      work[i] += (float)x.tiles[i] * x.us[i];
      items[i] += (float)x.tiles[i];
    }
  }
  *none = lane_value(along((int)owned, 0, [](int u, int v) { return (int)((uint32_t)u + (uint32_t)v); }), 63) != a.T;
#pragma unroll
  for (int i = kMixed ? 0 : 1; i < 2; ++i) {
    work[i] = wave_sum(work[i]) * (float)a.Hk;
    items[i] = wave_sum(items[i]) * (float)a.Hk;
  }
  keys = wave_sum(keys);
  float inv[2] = {0.f, 0.f};                // 1 / us of a part
  int tail = INT32_MAX, tail_ways = 1, tail_end = 0;      // items of 256 rows from `tail` on are cut into that many
  // Few rows: as many parts a slot as make their own time and the wait for the last of them least.  (What there is room for, below by more than the
  // sums' roundings: an item makes at most its time over that of a part, and one more.)
  const float per_slot = over(work[0] + work[1], a.slots);
  if (items[1] > 0.f) {
    const float room = 0.99f * min((float)a.most_parts[1], (float)a.groups - items[0]) - items[1];
    float us = 0.03f * per_slot;
    if (!kMixed) {
      const float rounds = __builtin_amdgcn_sqrtf(0.05f * over(keys * (float)a.Hk, a.slots));
      us = rounds > 2.f ? over(per_slot, rounds) : over(work[1], max(a.slots - items[1], 0.3f * a.slots));
    }
    us = max(us, a.least);
    if (room > 0.f) inv[1] = __builtin_amdgcn_rcpf(max(us, over(work[1], room)));
  }
  if (kMixed && items[0] > 0.f) {
    // Tiles of 256 rows: a lane prices 1 .. 64 parts of those of the last round, or of the longest where there is but one.
    most = wave_max(most);
    const float ways = (float)(lane + 1), whole = __builtin_floorf(over(items[0], a.slots) + 1e-4f), rest = items[0] - whole * a.slots;
    const float each = whole > 0.f ? over(work[0], items[0]) : most;
    // (unlike items, cut to one length: half a part more each, at most a whole one)
    const float like = over(work[0], most), parts = whole > 0.f ? rest * ways : lane == 0 ? rest : like * ways + 0.5f * (rest - like);
    const float at_most = whole > 0.f ? parts : like * ways + rest;
    float cost = __builtin_ceilf(over(parts, a.slots) - 1e-4f) * (each * __builtin_amdgcn_rcpf(ways) + a.once[0]);
    if (lane > 0) cost += 2.f + a.join * (lane < kOneMeeting ? ways : 2.f * __builtin_amdgcn_sqrtf(ways)) + parts * a.part[0];
    if (lane > 0 && at_most > 0.99f * min((float)a.most_parts[0], (float)a.groups - whole * a.slots - items[1])) cost = INFINITY;
    const float best = wave_min(cost);
    const uint64_t these = __ballot(cost == best);
    const int at = these ? __builtin_ctzll(these) : 0;
    bool all_few = false;
    if (a.all_few && whole == 0.f) {
      // Little work: all of it as few rows, which twice as many CUs share.
      const Request f = request_of<false>(a, lane);
      const float all = wave_sum((float)f.tiles[1] * f.us[1]) * (float)a.Hk, n = wave_sum((float)f.tiles[1]) * (float)a.Hk, longest = wave_max(f.us[1]);
      all_few = a.once[1] + max(min(longest, a.least), over(all, a.slots)) + (longest > a.least ? 5.f : 0.f) < best;
      if (all_few) {
        r = f;
        const float room = 0.99f * min((float)a.most_parts[1], (float)a.groups) - n;
        inv[1] = room > 0.f ? __builtin_amdgcn_rcpf(max(max(over(all, max(a.slots - n, 0.3f * a.slots)), a.least), over(all, room))) : 0.f;
      }
    }
    if (at > 0 && whole > 0.f) {
      tail = (int)(whole * a.slots);
      tail_ways = 1 + at;
      tail_end = tail + (int)rest * tail_ways;
      inv[1] = min(inv[1], over(0.99f * min((float)a.most_parts[1], (float)a.groups - (float)tail_end) - items[1], work[1] + 1e-9f));
      inv[1] = max(inv[1], 0.f);
    } else if (at > 0 && !all_few) {
      inv[0] = (float)(at + 1) * __builtin_amdgcn_rcpf(most);
      inv[1] = max(min(inv[1], over(0.99f * ((float)a.groups - (over(work[0] * (float)(at + 1), most) + items[0])) - items[1], work[1] + 1e-9f)), 0.f);
    }
  }
  w.ways = 1;
  w.part = 0;
  int slot = -1;
  if (kMixed && g >= tail && g < tail_end) {
    int part;
    const int item = divided(g - tail, tail_ways, &part);
    slot = item * tail_ways;
    g = tail + item;
    w.part = part;
    w.ways = tail_ways;
  } else if (kMixed && g >= tail) {
    g += tail + (tail_end - tail) / tail_ways - tail_end;      // among the few rows, as if none of the others were cut
  }
  // items, or their parts, in front of a lane's request: those of 256 rows, then the few rows
  int before = 0;
#pragma unroll
  for (int i = kMixed ? 0 : 1; i < 2; ++i) {
    const int first = before;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      if (a.B > 64) r = request_of<kMixed>(a, b0 + lane);
      const int ways = ways_of(r.us[i], inv[i]), sum = sums_along((int)min((int64_t)a.Hk * r.tiles[i] * ways, (int64_t)kMost));
      const uint64_t passed = __ballot(before + sum <= g);
      if (passed == ~0ull) {
        before += lane_value(sum, 63);
        continue;
      }
      const int at = __builtin_ctzll(~passed);
      const int group0 = before + (at > 0 ? lane_value(sum, at - 1) : 0);
      w.b = b0 + at;
      w.begin = lane_value(r.begin, at);
      w.n = lane_value(r.n, at);
      w.len = lane_value(r.len, at);
      w.few = i;
      // Keys that no other workgroup reads go past the caches where all of them are more than the last one holds: 8 tokens over 10 000 keys of 24 heads of 128
      // each 187 -> 167 us.  Of keys that the last call has left there, 64 tokens over 300 keys of 24 heads, 45 -> 48; with two row tiles to a head 120 -> 140.
      w.once = i && keys > a.cached && lane_value(r.tiles[0] * 2 + r.tiles[1], at) == 1;
      const int tiles = lane_value(r.tiles[i], at), cuts = lane_value(ways, at);
      // Of tiles of 256 rows key heads are counted first, then parts, then row tiles, from those with the most keys on: a multiple of eight key heads stay on
      // an XCD each, whose L2 its tiles share; else every other eight go back, or the first XCD would always get the longer one.  Of few rows the tiles of a
      // part are eight apart, on one XCD, which reads their keys once: 16 requests x 80 rows of 6 heads of 128 over 13 600 keys 298 -> 205 us.
      int at_g = g - group0, part, tile;
      const int units = a.Hk * cuts;
      if (i == 0 || tiles == 1) {
        if (a.Hk % kXcds && (at_g & kXcds) && (at_g | (kXcds - 1)) < units * tiles) at_g ^= kXcds - 1;
        tile = divided(divided(at_g, a.Hk, &w.hk), cuts, &part);
      } else {
        const int eights = units / kXcds * kXcds;
        int unit, rest;
        if (at_g < eights * tiles) {
          unit = divided(at_g, kXcds * tiles, &rest) * kXcds + rest % kXcds;
          tile = rest / kXcds;
        } else {
          tile = divided(at_g - eights * tiles, units - eights, &rest);
          unit = eights + rest;
        }
        part = divided(unit, a.Hk, &w.hk);
      }
      w.apart = 1;
      if (slot < 0) {
        w.ways = cuts;
        w.part = part;
        w.apart = a.Hk;
        slot = group0 - first + tile * units + w.hk;
      }
      tile = tiles - 1 - tile;
      w.first = slot;
      w.row0 = i ? (kMixed ? lane_value(r.tiles[0], at) * kRowsShared : 0) + tile * kRowsFew : tile * kRowsShared;
      return true;
    }
  }
  return false;
}

// Zeros, and -inf, in the rows that no request owns: those in front of the first one's and behind the last one's.
__device__ __forceinline__ void fill_rows(const PagesArgs& a, int D) {
  const int lane = threadIdx.x & 63;
  int lo = a.T, hi = 0;
  for (int b = lane; b < a.B; b += 64) {
    const int from = min(max(a.cu[b], 0), a.T), to = min(max(a.cu[b + 1], 0), a.T);
    if (to > from) {
      lo = min(lo, from);
      hi = max(hi, to);
    }
  }
  const int to = wave_max(hi), from = min(-wave_max(-lo), to);
  const int row = a.H * D / 8;          // 16-byte chunks
  for (int r = blockIdx.x; r < a.T - (to - from); r += gridDim.x) {
    const int64_t t = r < from ? r : r + (to - from);
    for (int c = threadIdx.x; c < row; c += blockDim.x) *reinterpret_cast<u32x4*>(a.out + (t * row + c) * 8) = u32x4{0, 0, 0, 0};
    for (int h = threadIdx.x; h < a.H; h += blockDim.x) a.lse[(int64_t)h * a.T + t] = -INFINITY;
  }
}

// A request's keys (0) and values (1) of a key head.
struct Keys {
  const uint16_t* base[2];
  uint32_t sp[2], ss[2];        // bytes
  const __attribute__((address_space(4))) int32_t* table;      // (constant while the launch runs: scalar loads)
  int len, page, n_pages, width;
  Quotient by_page;
  __device__ __forceinline__ Keys(const PagesArgs& a, const Work& w) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      base[i] = a.kv.base[i] + w.hk * a.kv.sh[i];
      sp[i] = 2 * (uint32_t)a.kv.sp[i];
      ss[i] = 2 * (uint32_t)a.kv.ss[i];
    }
    table = (const __attribute__((address_space(4))) int32_t*)(a.tables + w.b * a.table_stride);
    len = w.len;
    page = a.kv.page;
    n_pages = a.kv.n_pages;
    width = a.width;
    by_page = a.kv.by_page;
  }
  __device__ __forceinline__ const uint16_t* at(int i, uint32_t p, uint32_t place) const {
    return reinterpret_cast<const uint16_t*>(reinterpret_cast<const uint8_t*>(base[i]) + (uint64_t)p * sp[i] + (uint64_t)place * ss[i]);
  }
  // Row of key j < len, each lane's own; null where its entry is no page.
  __device__ __forceinline__ const uint16_t* row(int i, int j) const {
    const int e = (int)quotient(j, by_page), p = reinterpret_cast<const int32_t*>(reinterpret_cast<uintptr_t>(table))[e];
    return (uint32_t)p < (uint32_t)n_pages ? at(i, p, j - e * page) : nullptr;
  }
};

// kCount times 16 keys of a tile; each sixteen is in one page.
template <int kCount>
struct Sixteens {
  int id[kCount], place[kCount];      // page, and the first key's place in it
  int left;                           // keys from the first one to the last of the request; not above 0: none of them is there
  // (rows behind the last key, and those of no page, arrive as zeros)
  template <int D>
  __device__ __forceinline__ void rsrc(const Keys& ks, int i, u32x4 (&r)[kCount]) const {
    uint32_t valid[kCount];
#pragma unroll
    for (int j = 0; j < kCount; ++j) valid[j] = 15 * ks.ss[i] + 2 * D;
    if (__builtin_expect(left < 16 * kCount, 0)) {
      asm volatile("" ::: "memory");
#pragma unroll
      for (int j = 0; j < kCount; ++j) valid[j] = left > 16 * j ? (uint32_t)(min(left - 16 * j, 16) - 1) * ks.ss[i] + 2 * D : 0u;
    }
#pragma unroll
    for (int j = 0; j < kCount; ++j) r[j] = make_rsrc(ks.at(i, id[j], place[j]), (uint32_t)id[j] < (uint32_t)ks.n_pages ? valid[j] : 0u);
  }
};
// Finds the sixteens of each tile of a list, every kStep keys between two stops: the first key of the window, the list's end.  An entry is asked for when it
// is found, and used a tile later.
template <int kKeys, int kTiles, int kCount>
struct Finder {
  int entry, place, left, t, stop;      // of the next one: its first sixteen's table entry, ...
  int over, more;                       // kStep % page, kStep / page
  static constexpr int kStep = kKeys * kTiles;
  __device__ __forceinline__ void open(const Keys& ks, const TileList<kKeys>& list, int first, int offset) {
    t = first;
    more = (int)quotient(kStep, ks.by_page);
    over = kStep - more * ks.page;
    seek(ks, list, offset);
  }
  __device__ __forceinline__ void seek(const Keys& ks, const TileList<kKeys>& list, int offset) {
    const int key = list.key(t) + offset;
    left = t < list.end ? ks.len - key : 0;
    entry = left > 0 ? (int)quotient(key, ks.by_page) : 0;
    place = left > 0 ? key - entry * ks.page : 0;
    stop = t < list.n_sink ? min(list.n_sink, list.end) : t < list.end ? list.end : INT32_MAX;
    for (int* x : {&entry, &place, &left, &stop}) *x = __builtin_amdgcn_readfirstlane(*x);
  }
  __device__ __forceinline__ Sixteens<kCount> next(const Keys& ks, const TileList<kKeys>& list, int offset) {
    Sixteens<kCount> x;
    x.left = left;
    int e = entry, p = place;
#pragma unroll
    for (int j = 0; j < kCount; ++j) {
      if (j > 0) {
        p += 16;
        if (p >= ks.page) {
          p = 0;
          ++e;
        }
      }
      x.place[j] = p;
      x.id[j] = *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(
          reinterpret_cast<const __attribute__((address_space(4))) char*>(ks.table) + 4u * (uint32_t)min(e, ks.width - 1));
    }
    t += kTiles;
    entry += more;
    place += over;
    left -= kStep;
    if (place >= ks.page) {
      place -= ks.page;
      ++entry;
    }
    if (__builtin_expect(t >= stop, 0)) seek(ks, list, offset);
    return x;
  }
};

// What a lane needs to bring its 16 bytes of every 1 KB block of a tile; blocks are numbered through the tile, kOf of them a sixteen.
template <int D, int NKB>
struct PageLoader {
  typedef Tiles<D, NKB> T;
  static constexpr int kOf = 16 / T::kBlockRows;
  uint32_t k_row, k_chunk, v_off, k_block, v_block;
  __device__ __forceinline__ void open(const Keys& ks, int lane) {
    const int row = lane / T::kRowLanes, chunk = lane % T::kRowLanes;
    k_row = row * ks.ss[0];
    k_chunk = 16 * (chunk ^ T::swz_k(row));
    v_off = row * ks.ss[1] + 64 * ((chunk >> 2) ^ T::swz_v(row)) + 16 * (chunk & 3);
    k_block = T::kBlockRows * ks.ss[0];
    v_block = T::kBlockRows * ks.ss[1];
  }
  template <bool kOnce = false>
  __device__ __forceinline__ static void load(const u32x4& r, uint32_t off, uint32_t to) {
    if constexpr (kOnce) load_block_once_to_lds(r, off, to);
    else load_block_to_lds(r, off, 0, to);
  }
  template <bool kOnce = false>
  __device__ __forceinline__ void issue_k(const u32x4& r, int blk, uint32_t to) const {
    load<kOnce>(r, k_row + (k_chunk ^ (64u * (blk & T::kBlockXor))) + (blk % kOf) * k_block, to + blk * 1024);
  }
  template <bool kOnce = false>
  __device__ __forceinline__ void issue_v(const u32x4& r, int blk, uint32_t to) const { load<kOnce>(r, v_off + (blk % kOf) * v_block, to + blk * 1024); }
};

// Parts as they lie in the registers: 4 floats a lane, (register group) x (lane).  `at`: of a row's column d.
template <int D>
__device__ __forceinline__ int part_at(int row, int d) { return ((d >> 3) * 64 + 32 * ((d >> 2) & 1) + row) * 4 + (d & 3); }

// The 32 rows of a wavefront without matrix instructions, visible keys of [begin, end) only, from the maxima (in powers of two) and inverse sums that lane r
// and r + 32 hold of row r: a lane has a key's score, then its columns.
template <int D, bool kHalf>
__device__ __forceinline__ void rows_one_by_one(const PagesArgs& a, const Work& w, const Queries& qs, const Keys& ks, int row0, float m, float inv, int begin,
                                                int end, float* part, int lane) {
  typedef Elem<kHalf> E;
  constexpr int kCols = D / 64;
#pragma unroll 1
  for (int r = 0; r < 32 && row0 + r < qs.rows; ++r) {
    const int s = query_of(qs, row0 + r), head = w.hk * a.group + row0 + r - s * a.group;
    const Span span = uniform_span(qs, ks.len, s);
    const uint16_t* q = qs.q + s * a.q_ss + head * a.q_sh;
    const float top = __shfl(m, r), norm = __shfl(inv, r);
    float acc[kCols] = {};
#pragma unroll 1
    for (int j0 = begin; j0 < min(end, span.hi); j0 += 64) {
      if (j0 + 64 <= span.lo && j0 >= a.sinks) continue;
      const int j = j0 + lane;
      const bool seen = j < min(end, span.hi) && (j >= span.lo || j < a.sinks);
      float weight = 0.f;
      if (seen) {
        float score = 0.f;
        if (const uint16_t* k = ks.row(0, j))
#pragma unroll 1
          for (int d = 0; d < D; d += 8) {
            const typename E::x8 x = *reinterpret_cast<const typename E::x8*>(q + d), y = *reinterpret_cast<const typename E::x8*>(k + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) score = __builtin_fmaf((float)x[e], (float)y[e], score);
          }
        weight = __builtin_amdgcn_exp2f(__builtin_fmaf(score, a.scale_log2, -top));
      }
      uint64_t some = __ballot(seen);
#pragma unroll 1
      while (some) {
        const int i = __builtin_ctzll(some);
        some &= some - 1;
        const float wi = __shfl(weight, i);
        if (const uint16_t* v = ks.row(1, j0 + i))
#pragma unroll
          for (int e = 0; e < kCols; ++e) acc[e] = __builtin_fmaf(wi, (float)reinterpret_cast<const typename E::t*>(v)[lane * kCols + e], acc[e]);
      }
    }
    if (part) {
#pragma unroll
      for (int e = 0; e < kCols; ++e) store_device(part + part_at<D>(r, lane * kCols + e), acc[e]);
    } else {
      typename E::t* out = reinterpret_cast<typename E::t*>(a.out) + ((int64_t)(w.begin + s) * a.H + head) * D + lane * kCols;
#pragma unroll
      for (int e = 0; e < kCols; ++e) out[e] = (typename E::t)(acc[e] * norm);
    }
  }
}

// Whether a tile that some row of the wavefront does not see whole holds infinite or undefined values.
template <int D, bool kHalf>
__device__ __forceinline__ bool masked_not_finite(const Keys& ks, const RowState<D, kHalf, 2>& st, const TileList<64>& list, int lane) {
  typedef RowState<D, kHalf, 2> State;
  typedef Tiles<D, 2> T;
  uint32_t over = 0;
#pragma unroll 1
  for (int t = list.begin; t < list.end; ++t) {
    const int k0 = list.key(t);
    if (st.whole(k0)) continue;
#pragma unroll 1
    for (int j = k0 + lane / T::kRowLanes; j < min(k0 + T::kKeys, ks.len); j += T::kBlockRows)
      if (const uint16_t* v = ks.row(1, j)) over |= State::ones(*reinterpret_cast<const u32x4*>(v + 8 * (lane % T::kRowLanes)));
  }
  return __any((over & 0x80008000u) != 0);
}

constexpr float kLn2 = 0.6931471805599453f;

// A wavefront's share of the tiles of 256 rows: kPer neighbouring blocks of each, which are of one sixteen.  Tile t + 1 of K goes with tile t of V.
template <int D>
struct SharedLoads {
  typedef Tiles<D, 2> T;
  typedef PageLoader<D, 2> L;
  static constexpr int kPer = T::kBlocks / kWavesShared;
  const Keys ks;
  const TileList<64>& list;
  const int wave, offset;
  const uint32_t lds0;
  L ld;
  Finder<64, 1, 1> finder;
  Sixteens<1> of_v, of_k, of_next;
  __device__ __forceinline__ SharedLoads(const PagesArgs& a, const Work& w, const TileList<64>& tiles, uint32_t lds_at, int wave_at, int lane)
      : ks(a, w), list(tiles), wave(wave_at), offset(16 * (kPer * wave_at / L::kOf)), lds0(lds_at) {
    ld.open(ks, lane);
  }
  __device__ __forceinline__ void open() {
    finder.open(ks, list, list.begin, offset);
    of_k = finder.next(ks, list, offset);
    of_next = finder.next(ks, list, offset);
  }
  __device__ __forceinline__ void load_k(int pair) {
    u32x4 r[1];
    of_k.template rsrc<D>(ks, 0, r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) ld.issue_k(r[0], kPer * wave + i, lds0 + pair_at<D>(pair) + T::kBytes);
    of_v = of_k;
    of_k = of_next;
    of_next = finder.next(ks, list, offset);
  }
  __device__ __forceinline__ void load_pair(int t) {
    u32x4 r[1];
    of_v.template rsrc<D>(ks, 1, r);
#pragma unroll
    for (int i = 0; i < kPer; ++i) ld.issue_v(r[0], kPer * wave + i, lds0 + pair_at<D>(t));
    load_k(t);
  }
};

template <int D, bool kHalf>
__device__ __forceinline__ void shared_tiles(const PagesArgs& a, const Work& w, uint8_t* lds) {
  typedef Tiles<D, 2> T;
  typedef SharedLds<D> S;
  typedef Elem<kHalf> E;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds;
  const Queries qs = queries_of(a, w.begin, w.n);
  const Span all_first = uniform_span(qs, w.len, query_of(qs, w.row0)), all_last = uniform_span(qs, w.len, query_of(qs, min(w.row0 + kRowsShared - 1, qs.rows - 1)));
  TileList<64> list(qs, all_first, all_last, 0, 1);
  w.share(list);
  const int n = list.end - list.begin;
  const int row0 = w.row0 + 32 * wave;
  if (__builtin_expect(row0 >= qs.rows, 0)) {      // (11 requests x 114 rows of 8 key heads of 128 over 8000 keys 158 -> 118 us: the others have the SIMDs, and the power)
    if (n > 0) {
      SharedLoads<D> loads(a, w, list, lds0, wave, lane);
      loads.open();
      loads.load_k(-1);
      loads.load_pair(0);
      loads.load_pair(1);
      walk_idle<D>(n, wave, [&](int t) __attribute__((always_inline)) { loads.load_pair(t); });
    }
    return;
  }
  SharedLoads<D> loads(a, w, list, lds0, wave, lane);
  const Keys& ks = loads.ks;
  RowState<D, kHalf, 2> st;
  if (n > 0) {
    loads.open();
    const uint16_t* q = qs.q + (int64_t)w.hk * a.group * a.q_sh;
    queries_to_lds<D, true>(lds0, row0, wave, lane, [&](int r) __attribute__((always_inline)) {
      const int row = min(r, qs.rows - 1);
      const int s = query_of(qs, row), g = row - s * a.group;
      return q + s * a.q_ss + g * a.q_sh;
    });
    loads.load_k(-1);
    loads.load_pair(0);
    loads.load_pair(1);
  }
  st.open(qs, 0, w.hk, row0, w.len, lane, false);
  if (n > 0) walk_tiles<D, kHalf, true>(st, lds, list, all_first, all_last, n, wave, lane, [&](int t) __attribute__((always_inline)) { loads.load_pair(t); });
  const int col = lane & 31, hh = lane >> 5;
  float m = st.m_ref * st.c, l = st.l_run + __shfl_xor(st.l_run, 32);
  float undefined = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) undefined = __builtin_fmaf(st.o[i][r], 0.f, undefined);
  bool hurt = __builtin_expect(__any(undefined != 0.f && l == l), 0) && masked_not_finite<D, kHalf>(ks, st, list, lane);
  const bool live = row0 + col < qs.rows;
  if (w.ways > 1) {
    // A part's sums, fp32; the wavefront that completes the parts of its rows adds them up, in order: of more than eight, neighbours in groups first, and what
    // the groups come to then, so that several CUs read them (one reads 100 KB a us): 617 rows of 2 key heads of 128 over 38 000 keys, 39 parts, 97 -> 61 us.  A
    // group's counter is its first part's, that of the groups part 1's.
    constexpr int kPartFloats = 32 * D;
    auto part_of = [&](int at) __attribute__((always_inline)) { return (int64_t)(w.first + at * w.apart) * kWavesShared + wave; };
    auto store_sums = [&](int64_t at) __attribute__((always_inline)) {
      float* ml = a.part_ml[0] + (at * 32 + col) * 2;
      if (hh == 0) {
        store_device(ml, m);
        store_device(ml + 1, l);
      }
    };
    auto store_part = [&](int64_t at) __attribute__((always_inline)) {
      const Rsrc to = buffer_of(a.part_out[0] + at * kPartFloats, kPartFloats * 4);
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          u32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = __builtin_bit_cast(uint32_t, (float)st.o[i][4 * g + e]);
          __builtin_amdgcn_raw_buffer_store_b128(x, to, (4 * i + g) * 1024 + lane * 16, 0, kDevice);
        }
    };
    const int64_t mine = part_of(w.part);
    if (hurt)
      rows_one_by_one<D, kHalf>(a, w, qs, ks, row0, m, 0.f, list.begin < list.end ? list.key(list.begin) : 0,
                                list.begin < list.end ? list.key(list.end - 1) + T::kKeys : 0, a.part_out[0] + mine * kPartFloats, lane);
    else store_part(mine);
    store_sums(mine);
    const int group = w.ways <= kOneMeeting ? w.ways : (int)__builtin_ceilf(__builtin_amdgcn_sqrtf((float)w.ways));
    int lead = w.part / group * group, count = min(group, w.ways - lead), step = 1, counter_of = lead;
#pragma unroll 1
    for (;;) {
      wait_loads();                // (stores as well)
      int done = 0;
      if (lane == 0) {
        uint32_t* counter = a.counters[0] + part_of(counter_of);
        done = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == count;
        if (done) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      if (!__builtin_amdgcn_readfirstlane(done)) return;
      asm volatile("" ::: "memory");
      const int64_t first = part_of(lead), apart = (int64_t)step * w.apart * kWavesShared;
      const float* mls = a.part_ml[0] + (first * 32 + col) * 2;
      m = -INFINITY;
      for (int p = 0; p < count; ++p) m = fmaxf(m, load_device(mls + p * apart * 64));
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) st.o[i][r] = 0.f;
      l = 0.f;
#pragma unroll 1
      for (int p = 0; p < count; ++p) {
        const float lp = load_device(mls + p * apart * 64 + 1), wp = weight_of(load_device(mls + p * apart * 64), lp, m);
        const Rsrc from = buffer_of(a.part_out[0] + (first + p * apart) * kPartFloats, kPartFloats * 4);
        l = __builtin_fmaf(wp, lp, l);
        f32x4 x[D / 8];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) x[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, i * 1024 + lane * 16, 0, kDevice));
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) st.o[i / 4][4 * (i % 4) + e] = __builtin_fmaf(wp, x[i][e], st.o[i / 4][4 * (i % 4) + e]);
      }
      if (step > 1 || group == w.ways) break;
      store_part(first);
      store_sums(first);
      lead = 0;
      step = group;
      count = (w.ways + group - 1) / group;
      counter_of = 1;
    }
    hurt = false;
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;      // (an undefined sum stays one)
  if (hh == 0 && live) {
    const int s = query_of(qs, row0 + col), g = row0 + col - s * a.group;
    a.lse[(int64_t)(w.hk * a.group + g) * a.T + w.begin + s] = l != 0.f ? (m + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
  }
  if (__builtin_expect(hurt, 0)) {
    rows_one_by_one<D, kHalf>(a, w, qs, ks, row0, m, inv, 0, w.len, nullptr, lane);
    return;
  }
  // Rows of the result through the LDS, so that a store covers whole lines: half of the columns at a time.
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
      if (row < qs.rows) {
        const int s = query_of(qs, row), g = row - s * a.group;
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(a.out + ((int64_t)(w.begin + s) * a.H + w.hk * a.group + g) * D + half * (D / 2) + 8 * chunk));
      }
    }
  }
}

template <int N>
__device__ __forceinline__ void wait_q() {     // all loads but those of a tile's K and V, of N each
  static_assert(N == 4 || N == 8, "blocks of a half tile");
  if constexpr (N == 4) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
}
// Few rows: as attn_window.hip's, a wavefront takes every fourth tile of its item, or of a part of it, K of the next tile sent for before the softmax of
// this one, V of the next behind its values; the states of the four meet in the LDS, those of parts in memory, where the last part adds them up.
// Q comes once for all of them, through the LDS: loaded as fragments, by loads that the compiler counts among the tiles' that it does not know, it would be
// waited for in the loop, and V of a tile with it.
template <int D, int W>
struct FewPagesLds {
  typedef FewLds<D, W> F;
  static constexpr int kQ = (F::kAll + 1023) / 1024 * 1024, kAll = kQ + 32 * 2 * D;
};
template <int D, bool kHalf, int W>
__device__ __forceinline__ void few_rows(const PagesArgs& a, const Work& w, uint8_t* lds) {
  typedef Tiles<D, 1> T;
  typedef Elem<kHalf> E;
  typedef PageLoader<D, 1> L;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 31, hh = lane >> 5;
  const Queries qs = queries_of(a, w.begin, w.n);
  RowState<D, kHalf, 1> st;
  // (4 or 8 blocks of 1 KB: none, one or two a wavefront)
  const uint32_t qt0 = (uint32_t)(uintptr_t)(lds_ptr_t)lds + FewPagesLds<D, W>::kQ;
#pragma unroll
  for (int i = 0; i < (T::kBlocks + W - 1) / W; ++i) {
    const int blk = wave + W * i, r = blk * T::kBlockRows + lane / T::kRowLanes;
    if (blk < T::kBlocks) {
      const int row = min(w.row0 + r, qs.rows - 1), s = query_of(qs, row);
      load_rows_to_lds(qs.q + s * a.q_ss + (w.hk * a.group + row - s * a.group) * a.q_sh + 8 * ((lane % T::kRowLanes) ^ T::swz_k(r)), qt0 + blk * 1024);
    }
  }
  st.open(qs, 0, w.hk, w.row0, w.len, lane, false);
  TileList<T::kKeys> list(qs, st.first, st.last, 0, 1);
  w.share(list);                // ... every W-th tile
  const uint8_t* kt = lds + wave * FewLds<D, W>::kTile;
  const uint8_t* vt = kt + T::kBytes;
  const uint32_t kt0 = (uint32_t)(uintptr_t)(lds_ptr_t)(lds + wave * FewLds<D, W>::kTile);
  const Keys ks(a, w);
  L ld;
  ld.open(ks, lane);
  const bool once = __builtin_amdgcn_readfirstlane(w.once);
  Finder<T::kKeys, W, 2> finder;
  Sixteens<2> here, next;
  auto load_k = [&](const Sixteens<2>& x) __attribute__((always_inline)) {     // (past the end, with an empty descriptor: the waits count loads)
    u32x4 r[2];
    x.template rsrc<D>(ks, 0, r);
    if (once) {
#pragma unroll
      for (int blk = 0; blk < T::kBlocks; ++blk) ld.template issue_k<true>(r[blk / L::kOf], blk, kt0);
    } else {
#pragma unroll
      for (int blk = 0; blk < T::kBlocks; ++blk) ld.issue_k(r[blk / L::kOf], blk, kt0);
    }
  };
  auto load_v = [&](const Sixteens<2>& x) __attribute__((always_inline)) {
    u32x4 r[2];
    x.template rsrc<D>(ks, 1, r);
    if (once) {
#pragma unroll
      for (int blk = 0; blk < T::kBlocks; ++blk) ld.template issue_v<true>(r[blk / L::kOf], blk, kt0 + T::kBytes);
    } else {
#pragma unroll
      for (int blk = 0; blk < T::kBlocks; ++blk) ld.issue_v(r[blk / L::kOf], blk, kt0 + T::kBytes);
    }
  };
  int t = list.begin + wave;
  if (t < list.end) {
    finder.open(ks, list, t, 0);
    here = finder.next(ks, list, 0);
    next = finder.next(ks, list, 0);
    load_k(here);
    load_v(here);
    wait_q<T::kBlocks>();
  } else {
    wait_loads();
  }
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_barrier" ::: "memory");
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
    st.qf[i] = *reinterpret_cast<const typename E::x8*>(lds + FewPagesLds<D, W>::kQ + col * T::kRowBytes + 16 * ((2 * i + hh) ^ T::swz_k(col)));
#pragma unroll
  for (int i = 0; i < D / 16; ++i) asm volatile("" : "+v"(st.qf[i]));
  for (; t < list.end; t += W) {
    const int k0 = list.key(t);
    const bool masked = !st.whole(k0);
    f32x16 s[1];
    typename E::x8 p[1][2];
    wait_oldest<T::kBlocks>();
    st.scores(kt, s);
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s[0]) : : "memory");      // (the tile has been read)
    load_k(next);
    here = next;
    next = finder.next(ks, list, 0);
    st.softmax(s, p, k0, masked, lane);
    wait_oldest<T::kBlocks>();
    if (masked && st.any_not_finite(vt, lane)) st.take_out_not_finite(const_cast<uint8_t*>(vt), k0, lane);
    st.values(vt, p);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    load_v(here);
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
  float m[W], weight[W], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    m[i] = ml[i * 64 + col];
    top = fmaxf(top, m[i]);
  }
  l = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float li = ml[i * 64 + 32 + col];
    weight[i] = weight_of(m[i], li, top);
    l = __builtin_fmaf(weight[i], li, l);
  }
  constexpr int kCols = D / 8 / W;          // register groups of a wavefront's share
  const int row = w.row0 + col;
  const bool live = row < qs.rows;
  f32x4 sum[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + j * FewLds<D, W>::kTile) + lane * 4 + (wave * kCols + i) * 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[i][e] = __builtin_fmaf(weight[j], x[e], sum[i][e]);     // (a weight of 0 keeps what is undefined: some row's visible key is)
    }
  }
  if (w.ways == 1) {
    if (!live) return;
    const int s = query_of(qs, row), g0 = row - s * a.group;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int64_t head = w.hk * a.group + g0;
    uint16_t* out = a.out + ((int64_t)(w.begin + s) * a.H + head) * D;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      typename E::x4 h;
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = (typename E::t)(sum[i][e] * inv);
      *reinterpret_cast<typename E::x4*>(out + 8 * (wave * kCols + i) + 4 * hh) = h;
    }
    if (wave == 0 && hh == 0) a.lse[head * a.T + w.begin + s] = l != 0.f ? (top + __builtin_amdgcn_logf(l)) * kLn2 : -INFINITY;
    return;
  }
  // A part's rows, [row][D]; the workgroup that completes an item's parts adds them all up, in an order of the sizes' own.
  constexpr int kPartFloats = kRowsFew * D, kThreads = W * 64;
  const int64_t mine = w.first + w.part * w.apart;
  const Rsrc to = buffer_of(a.part_out[1] + mine * kPartFloats, kPartFloats * 4);
#pragma unroll
  for (int i = 0; i < kCols; ++i)
    if (live) __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, sum[i]), to, (col * D + 8 * (wave * kCols + i) + 4 * hh) * 4, 0, kDevice);
  if (wave == 0 && hh == 0 && live) {
    store_device(a.part_ml[1] + (mine * kRowsFew + col) * 2, top);
    store_device(a.part_ml[1] + (mine * kRowsFew + col) * 2 + 1, l);
  }
  int* flag = reinterpret_cast<int*>(lds + FewLds<D, W>::kFlag);
  wait_loads();                // (stores as well)
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* counter = a.counters[1] + w.first;
    const bool last = (int)__hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == w.ways;
    if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  if (!*flag) return;
  // Everything that is asked for comes from memory, so as much of it as there is is under way together: maxima and sums of all parts, a thread each, then
  // 16 bytes of a row a thread, of every `by`-th part where the rows are fewer than the threads.
  const int tid = threadIdx.x, rows = min(qs.rows - w.row0, kRowsFew);
  float* weights = reinterpret_cast<float*>(lds);                  // [part][row] maxima, then weights
  float* sums = weights + kMostWays * kRowsFew;                    // [part][row]
  float* norms = sums + kMostWays * kRowsFew;                      // [row]
  f32x4* halves = reinterpret_cast<f32x4*>(norms + kRowsFew);      // [by][16 bytes of the rows]
  static_assert((2 * kMostWays * kRowsFew + kRowsFew) * 4 + kThreads * 16 <= FewLds<D, W>::kBytes, "the parts' meeting fits the tiles");
  float pm[kMostWays * kRowsFew / kThreads], pl[kMostWays * kRowsFew / kThreads];
#pragma unroll
  for (int i = 0; i < kMostWays * kRowsFew / kThreads; ++i) {
    const int at = tid + i * kThreads, p = at / kRowsFew, r = at % kRowsFew;
    if (p < w.ways && r < rows) {
      const float* ml = a.part_ml[1] + ((w.first + (int64_t)p * w.apart) * kRowsFew + r) * 2;
      pm[i] = load_device(ml);
      pl[i] = load_device(ml + 1);
    }
  }
#pragma unroll
  for (int i = 0; i < kMostWays * kRowsFew / kThreads; ++i) {
    const int at = tid + i * kThreads;
    if (at / kRowsFew < w.ways && at % kRowsFew < rows) {
      weights[at] = pm[i];
      sums[at] = pl[i];
    }
  }
  __syncthreads();
  if (tid < rows) {
    float high = -INFINITY, all = 0.f;
    for (int p = 0; p < w.ways; ++p) high = fmaxf(high, weights[p * kRowsFew + tid]);
    for (int p = 0; p < w.ways; ++p) {
      const float lp = sums[p * kRowsFew + tid], wp = weight_of(weights[p * kRowsFew + tid], lp, high);
      all = __builtin_fmaf(wp, lp, all);
      weights[p * kRowsFew + tid] = wp;
    }
    norms[tid] = all != 0.f ? 1.f / all : 0.f;
    const int s = query_of(qs, w.row0 + tid), head = w.hk * a.group + w.row0 + tid - s * a.group;
    a.lse[(int64_t)head * a.T + w.begin + s] = all != 0.f ? (high + __builtin_amdgcn_logf(all)) * kLn2 : -INFINITY;
  }
  __syncthreads();
  constexpr int kSixteens = D / 4, kSome = 8;          // 16-byte pieces of a row, parts under way together
  const int pieces = rows * kSixteens;
  auto added = [&](int e, int first, int by) {      // piece e of the parts first, first + by ..
    const Rsrc from = buffer_of(a.part_out[1] + (int64_t)w.first * kPartFloats, 0x7fffffff);
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int p0 = first; p0 < w.ways; p0 += kSome * by) {
      f32x4 x[kSome];
#pragma unroll
      for (int i = 0; i < kSome; ++i) {
        const uint32_t at = (uint32_t)min(p0 + i * by, w.ways - 1) * (uint32_t)w.apart * (kPartFloats * 4);
        x[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(from, at + e * 16, 0, kDevice));
      }
#pragma unroll
      for (int i = 0; i < kSome; ++i)
        if (p0 + i * by < w.ways) {
          const float wp = weights[(p0 + i * by) * kRowsFew + e / kSixteens];
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(wp, x[i][c], acc[c]);
        }
    }
    return acc;
  };
  auto store = [&](int e, const f32x4& acc) {
    const int r = e / kSixteens, s = query_of(qs, w.row0 + r), head = w.hk * a.group + w.row0 + r - s * a.group;
    typename E::x4 h;
#pragma unroll
    for (int c = 0; c < 4; ++c) h[c] = (typename E::t)(acc[c] * norms[r]);
    *reinterpret_cast<typename E::x4*>(a.out + ((int64_t)(w.begin + s) * a.H + head) * D + 4 * (e % kSixteens)) = h;
  };
  if (2 * pieces <= kThreads) {
    const int by = kThreads / pieces, first = tid / pieces, e = tid - first * pieces;
    if (first < by) halves[first * pieces + e] = added(e, first, by);
    __syncthreads();
    if (tid < pieces) {
      f32x4 acc = halves[tid];
      for (int i = 1; i < by; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] += halves[i * pieces + tid][c];
      store(tid, acc);
    }
  } else {
    for (int e = tid; e < pieces; e += kThreads) store(e, added(e, 0, 1));
  }
}

template <int D, bool kHalf, int W>
__global__ __launch_bounds__(W * 64, D == 64 ? 4 : 2) void attn_pages_few_kernel(const PagesArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  Work w;
  bool none;
  const bool some = find<false>(a, w, &none);
  if (none) fill_rows(a, D);
  if (some) few_rows<D, kHalf, W>(a, w, lds);
}
static_assert(FewPagesLds<64, kWavesShared>::kAll <= SharedLds<64>::kBytes && FewPagesLds<128, kWavesShared>::kAll <= SharedLds<128>::kBytes, "both forms fit");
template <int D, bool kHalf>
__global__ __launch_bounds__(kWavesShared * 64, D == 64 ? 4 : 2) void attn_pages_kernel(const PagesArgs a) {
  extern __shared__ __align__(1024) uint8_t lds[];
  Work w;
  bool none;
  const bool some = find<true>(a, w, &none);
  if (none) fill_rows(a, D);
  if (!some) return;
  if (w.few) few_rows<D, kHalf, kWavesShared>(a, w, lds);
  else shared_tiles<D, kHalf>(a, w, lds);
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

template <void (*kernel)(const PagesArgs)>
int launch(const PagesArgs& a, int64_t grid, int waves, int lds, hipStream_t stream) {
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
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(waves * 64), lds, stream, a);
  return hip_fail(hipGetLastError(), "attn_pages launch");
}

struct Scratch {
  void* workspace;
  int64_t bytes;
  uint32_t* counters;
  int64_t n_counters;
};

// The grid holds what there can be, cut or not.  `step` is the time of 64 keys as traces of launches that fill the chip show it: 256 rows 1.6 us with heads
// of 128 (alone on a CU), 2.2 with heads of 64 (two on a CU); 32 rows by the memory, of which eight wavefronts draw twice what four do.  `once` is a workgroup's
// time beside them.  They only decide how keys are cut.  Each of them halved and doubled, 45 launches of all sizes: -2.1 .. +2.6 % over all of them, most of
// them within 3 % (single ones: `step` doubled +56 % at 25 us, the shortest part of few rows `least` halved +22 % at 13 us or doubled +53 % at 16 us, a meeting's price
// halved +54 % at 25 us).  A window with a left border and none on the right is priced by its last tile (`request_of`), which then sees the fewest keys: 2030 rows
// of 3 heads of 64 beside 44 requests of 8, 50 keys back and all ahead, 53 us as tiles of 256 rows, 20 as few rows.
template <int D, bool kHalf>
int launch_dim(PagesArgs& a, int64_t most_rows, int n_cus, const Scratch& scratch, hipStream_t stream) {
  const int64_t rows = (int64_t)a.T * a.group, requests = std::min<int64_t>(a.B, a.T);
  // What is left over of tiles of 256 rows: as few rows up to 64 (heads of 128) or 96, else as a tile of 256 some of whose wavefronts have none.  Heads of 128,
  // 16 requests x 80 rows of 8 key heads over 13 600 keys: with 96 270 us, with 64 174; 313 rows over 20 000 keys of 40 heads with 64 420, with 32 369, but over all
  // sizes alike.  Heads of 64, 6 requests x 72 rows beside a prompt: with 96 1154, with 64 1541.  Little work goes by few rows alone up to 96: 63 requests x 96
  // rows over 50 keys 9.5, with tiles of 256 13.8.
  a.few_rows = D == 64 ? 96 : 64;
  const int64_t as_few = a.Hk * (rows / kRowsFew + requests);
  const bool mixed = std::min(most_rows, rows) > (as_few > n_cus ? a.few_rows : 96);
  const int64_t big = mixed ? rows / kRowsShared + std::min(requests, rows / (a.few_rows + 1)) : 0;
  const int64_t small = std::min(rows / kRowsFew + requests, mixed ? requests * (a.few_rows / kRowsFew) : INT64_MAX);
  const int64_t uncut = a.Hk * (big + small);
  // Few rows of few requests, which leave CUs without one, have eight wavefronts each: 40 items of 30 rows, heads of 64, over 20 000 keys 40 us, with four 47;
  // 144 items of a row, heads of 128, over 5000 keys 82, with four 69.
  const bool eight = !mixed && uncut <= n_cus / 2;
  const int64_t slots = (int64_t)n_cus * (mixed || eight ? 1 : 2) * (D == 64 ? 2 : 1);
  a.slots = (float)slots;
  a.step[0] = D == 64 ? 2.2f : 1.6f;
  a.step[1] = mixed ? (D == 64 ? 0.5f : 0.6f) : eight ? 1.6f : 3.2f;
  a.least = mixed ? 8.f : 16 * a.step[1];
  a.once[0] = 8.f;
  a.once[1] = 4.f;
  a.cached = 268435456.f / (256 * D) / a.Hk * a.step[1];      // (256 MB; 64 keys and values of a head are 256 D bytes)
  constexpr int64_t kBytes[2] = {(int64_t)kRowsShared * (D + 2) * 4, (int64_t)kRowsFew * (D + 2) * 4};
  for (int i = 0; i < 2; ++i) a.part[i] = (float)(2.0 * kBytes[i] / 6.7e6);
  a.join = (float)(kBytes[0] / 1e5);
  a.all_few = mixed && a.B <= 64 && as_few <= slots;
  // few rows first, whose parts are small
  int64_t bytes = scratch.workspace && scratch.counters ? scratch.bytes : 0, counters = scratch.counters ? scratch.n_counters : 0;
  // (an empty workgroup takes a slot for 1.1 us: there are no more than what the longest row of the tables could be cut into)
  int64_t groups = uncut + std::min<int64_t>((mixed ? 3 : 6) * slots / 2, uncut * std::min<int64_t>(a.most_len / 512, kMostWays - 1));
  if (a.all_few) groups = std::max(groups, as_few + slots);
  int64_t parts[2];
  parts[1] = std::min({bytes / 2 / kBytes[1], counters / 2, groups, (int64_t)INT32_MAX / kBytes[1]});      // (a part's place in 32 bits)
  parts[0] = mixed ? std::min({(bytes - parts[1] * kBytes[1]) / kBytes[0], (counters - parts[1]) / kWavesShared, groups}) : 0;
  float* at = static_cast<float*>(scratch.workspace);
  uint32_t* counter = scratch.counters;
  for (int i : {1, 0}) {
    const int64_t floats = parts[i] * kBytes[i] / 4, sums = floats / (D + 2) * D;
    a.most_parts[i] = (int32_t)parts[i];
    a.part_out[i] = at;
    a.part_ml[i] = at + sums;
    a.counters[i] = counter;
    at += floats;
    counter += parts[i] * (i ? 1 : kWavesShared);
  }
  const int64_t grid = (parts[1] > 0 || a.all_few ? groups : uncut) + kXcds - 1;
  if (grid > (1 << 23) - 1) {
    set_error("too many query rows");
    return DT_ERR_INVALID;
  }
  a.groups = (int32_t)(grid / kXcds * kXcds);
  return mixed ? launch<attn_pages_kernel<D, kHalf>>(a, a.groups, kWavesShared, SharedLds<D>::kBytes, stream)
         : eight ? launch<attn_pages_few_kernel<D, kHalf, kWavesShared>>(a, a.groups, kWavesShared, FewPagesLds<D, kWavesShared>::kAll, stream)
                 : launch<attn_pages_few_kernel<D, kHalf, kWavesFew>>(a, a.groups, kWavesFew, FewPagesLds<D, kWavesFew>::kAll, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_attn_pages_served_fwd(const void* q, const int64_t* q_strides, void* out, float* lse, int32_t T, int32_t H, int32_t Hk, int32_t D,
                                        const dt_pages* pages, const int32_t* tables, int64_t table_stride, int32_t width, int32_t B, const int32_t* lens,
                                        const uint8_t* served, const int32_t* cu_seqlens, int32_t max_seqlen_q, const dt_window* window, float softmax_scale,
                                        int32_t flags, void* workspace, int64_t workspace_bytes, uint32_t* counters, int64_t n_counters, void* stream) {
  if (T <= 0 || B <= 0 || H <= 0 || Hk <= 0 || H % Hk) {
    set_error("T, B, H, Hk must be positive and H a multiple of Hk (got %d, %d, %d, %d)", T, B, H, Hk);
    return DT_ERR_INVALID;
  }
  PagesArgs a{};
  if (int rc = check_pages(pages, D, a.kv)) return rc;
  if (!q || !out || !lse || !q_strides || !lens || !cu_seqlens || !window || (width > 0 && !tables) || !aligned16(q) || !aligned16(out)) {
    set_error("q and out must be non-null and 16-byte aligned, lse, strides, tables, lens, cu_seqlens and window non-null");
    return DT_ERR_INVALID;
  }
  if ((q_strides[0] | q_strides[1]) & 7) {
    set_error("strides must be multiples of 8 elements");
    return DT_ERR_INVALID;
  }
  if (width < 0 || table_stride < width) {
    set_error("width must not be negative, table rows at least `width` apart");
    return DT_ERR_INVALID;
  }
  const dt_window& w = *window;
  if (w.left < -1 || w.right < -1 || w.frame < 1 || w.sinks < 0) {
    set_error("window: left and right must be -1 (no border) or frames, frame at least 1, sinks not negative");
    return DT_ERR_INVALID;
  }
  if (B > kMostRequests) {
    set_error("more than %d requests are not supported", kMostRequests);
    return DT_ERR_UNSUPPORTED;
  }
  if ((int64_t)width * pages->page_size > kMostTokens || T > kMostTokens || w.sinks > kMostTokens || w.frame > kMostTokens) {
    set_error("lengths, sinks and frames beyond 2^29 tokens are not supported");
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
  if ((int64_t)T * (H / Hk) > (1ll << 30) || (int64_t)T * H * D > (1ll << 40)) {
    set_error("too many query rows");
    return DT_ERR_INVALID;
  }
  a.q = static_cast<const uint16_t*>(q);
  a.q_ss = q_strides[0];
  a.q_sh = q_strides[1];
  a.out = static_cast<uint16_t*>(out);
  a.lse = lse;
  a.tables = tables;
  a.table_stride = table_stride;
  a.lens = lens;
  a.served = served ? served : reinterpret_cast<const uint8_t*>(lens);
  a.all_served = !served;
  a.cu = cu_seqlens;
  a.width = width;
  a.most_len = width * pages->page_size;
  a.B = B;
  a.T = T;
  a.H = H;
  a.Hk = Hk;
  a.group = H / Hk;
  a.frame = w.frame;
  a.sinks = w.sinks;
  // (a span of 2^30 reaches past every key from every position)
  a.left = w.left < 0 ? -1 : (int32_t)std::min<int64_t>((int64_t)w.left * w.frame, 1 << 30);
  a.right = w.right < 0 ? -1 : (int32_t)std::min<int64_t>(((int64_t)w.right + 1) * w.frame, 1 << 30);
  a.by_frame = quotient_by(a.frame);
  a.by_group = quotient_by(a.group);
  a.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  const hipStream_t st = (hipStream_t)stream;
  const bool half = (flags & DT_ATTN_FP16) != 0;
  const int n_cus = cus();
  if (n_cus <= 0) {
    set_error("no current device");
    return DT_ERR_HIP;
  }
  const Scratch scratch = {workspace, workspace_bytes, counters, n_counters};
  const int64_t most_rows = (int64_t)std::max(max_seqlen_q, 0) * a.group;
  if (D == 128) return half ? launch_dim<128, true>(a, most_rows, n_cus, scratch, st) : launch_dim<128, false>(a, most_rows, n_cus, scratch, st);
  return half ? launch_dim<64, true>(a, most_rows, n_cus, scratch, st) : launch_dim<64, false>(a, most_rows, n_cus, scratch, st);
}

extern "C" int dt_attn_pages_fwd(const void* q, const int64_t* q_strides, void* out, float* lse, int32_t T, int32_t H, int32_t Hk, int32_t D,
                                 const dt_pages* pages, const int32_t* tables, int64_t table_stride, int32_t width, int32_t B, const int32_t* lens,
                                 const int32_t* cu_seqlens, int32_t max_seqlen_q, const dt_window* window, float softmax_scale, int32_t flags,
                                 void* workspace, int64_t workspace_bytes, uint32_t* counters, int64_t n_counters, void* stream) {
  return dt_attn_pages_served_fwd(q, q_strides, out, lse, T, H, Hk, D, pages, tables, table_stride, width, B, lens, nullptr, cu_seqlens, max_seqlen_q, window,
                                  softmax_scale, flags, workspace, workspace_bytes, counters, n_counters, stream);
}
