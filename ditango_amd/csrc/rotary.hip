// QK norm and rotation by positions on several axes (gfx950): what producer.hip does with cos / sin tables, for q and k in one launch and
// from the tokens' int32 positions.
//
// A pair (a, b) of a head row at position n on its axis turns by t = n f / 2 pi full turns.  f / 2 pi comes as a 64-bit fraction F of a
// turn, so n F mod 2^64 is the angle of any 32-bit position to 2^-32 of a turn: integers have no range reduction to lose bits in.  Its upper half, as
// a signed fraction of a turn in fp32, is what the sine and cosine instructions take; they are off by 1.9e-7 at most, the fraction's rounding
// included (4 million fractions all round the turn), where the row's 16 bits are off by 2^-9 to 2^-12 of a value.
//
// HBM-bound: rows x D x 2 bytes in and out, 12 bytes of positions a token.  A lane owns 4 pairs of a row: 8 neighbours with interleaved pairs, two
// runs of 4 half a section apart with rotate-half.  It has their angles once for the heads of its lane group.  14 882 tokens x (24 + 24) heads of
// 128 with an RMS norm: 64.4 us, 5.7 TB/s (two launches of the kernel with tables: 68.2, and the tables' making).
#include "producer_math.h"

namespace dt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;
// A lane group takes 4 heads of a token, or 8: the angles and the loads in front of them are then shared by twice as many rows.  Eight where groups of four
// make more than kManyWorkgroups workgroups and eight leave no more lanes idle.  us with 4 and with 8, q and k of 24 heads of 128: 600 tokens (450 workgroups)
// 6.0 / 6.0, 1200 8.3 / 7.8, 2400 15.6 / 12.0, 4800 25.8 / 23.2, 14 882 69.1 / 66.2; of 12 heads, 2400 tokens 8.2 / 9.2.  Twelve need scratch.
constexpr unsigned kManyWorkgroups = 640;
constexpr int kMostAxes = 8;

struct Rows {
  const uint16_t* x;
  uint16_t* y;
  int64_t sb, ss, sh;
  const void *w, *bias;
  float scale;
  int32_t H, groups;              // groups of heads that a lane group takes
};
struct RotaryArgs {
  Rows rows[2];
  const int32_t* pos;
  int64_t pos_sb;
  int32_t S, n_axes, norm, w16, halves;
  float eps;
  uint32_t items;                 // B * S * groups of both
  Quotient by_groups, by_s;
  uint8_t a0[16], b0[16];         // first element of a lane's two runs of 4 (halves)
  uint8_t axis[64];               // of pair 4 lane + i
  uint64_t turns[64];
};

template <bool kHalf>
__device__ __forceinline__ void load_weights4(const void* base, bool w16, int d, float* v) {
  if (w16) {   // uniform
    const u32x2 r = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(base) + d);
    float u[8];
    unpack8<kHalf>(u32x4{r.x, r.y, 0u, 0u}, u);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = u[i];
  } else {
    const f32x4 r = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + d);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = r[i];
  }
}

// kRms: with an RMS norm, which does without the 20 registers of means and biases (14 882 x 48 heads of 128 66.6 -> 64.4 us; a form of its own for rows
// without a norm, with as few, is 3 % slower than the common one).
template <int D, bool kHalf, bool kHalves, int kHeads, bool kRms>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_axes_kernel(const RotaryArgs a) {
  constexpr int G = D / 8;
  const int c = threadIdx.x % G;
  const uint32_t item = blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (item >= a.items) return;   // a lane group leaves as a whole; the exchanges below stay inside a group
  const uint32_t bs = quotient(item, a.by_groups);
  int hg = (int)(item - bs * (uint32_t)(a.rows[0].groups + a.rows[1].groups));
  const bool second = hg >= a.rows[0].groups;
  if (second) hg -= a.rows[0].groups;
  const Rows& t = second ? a.rows[1] : a.rows[0];
  const uint32_t b = quotient(bs, a.by_s), s = bs - b * (uint32_t)a.S;
  const int h0 = hg * kHeads, nh = min(t.H - h0, kHeads);
  const int ea = kHalves ? a.a0[c] : 8 * c, eb = kHalves ? a.b0[c] : 8 * c + 4;

  const uint16_t* xp = t.x + (int64_t)b * t.sb + (int64_t)s * t.ss + (int64_t)h0 * t.sh;
  u32x4 raw[kHeads];
#pragma unroll
  for (int r = 0; r < kHeads; ++r) {
    raw[r] = u32x4{0, 0, 0, 0};
    if (r < nh) {
      const uint16_t* p = xp + (int64_t)r * t.sh;
      if constexpr (kHalves) {
        const u32x2 lo = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p + ea));
        const u32x2 hi = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p + eb));
        raw[r] = u32x4{lo.x, lo.y, hi.x, hi.y};
      } else {
        raw[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + ea));
      }
    }
  }
  // the angles of this lane's pairs; t mod 2^32 of the upper half of n F
  float sn[4], cs[4];
  {
    const int32_t* pos = a.pos + (int64_t)b * a.pos_sb + (int64_t)s * a.n_axes;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t n = pos[a.axis[4 * c + i]];
      const uint64_t f = a.turns[4 * c + i];
      const uint32_t lo = (uint32_t)f, hi = (uint32_t)(f >> 32);
      const uint32_t t32 = __umulhi((uint32_t)n, lo) + (uint32_t)n * hi - (n < 0 ? lo : 0u);
      const float turn = (float)(int32_t)t32 * 2.3283064365386963e-10f;     // 2^-32
      sn[i] = __builtin_amdgcn_sinf(turn);
      cs[i] = __builtin_amdgcn_cosf(turn);
    }
  }
  float w[8], bias[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = 1.f;
    bias[i] = 0.f;
  }
  if ((kRms || a.norm != DT_NORM_NONE) && t.w) {
    load_weights4<kHalf>(t.w, a.w16 != 0, ea, w);
    load_weights4<kHalf>(t.w, a.w16 != 0, eb, w + 4);
  }
  if (!kRms && a.norm == DT_NORM_LAYER && t.bias) {
    load_weights4<kHalf>(t.bias, a.w16 != 0, ea, bias);
    load_weights4<kHalf>(t.bias, a.w16 != 0, eb, bias + 4);
  }
  float mean[kHeads] = {}, rs[kHeads] = {}, ss[kHeads];
  if (kRms || a.norm != DT_NORM_NONE) {   // uniform
#pragma unroll
    for (int r = 0; r < kHeads; ++r) {
      float v[8];
      unpack8<kHalf>(raw[r], v);
      if (!kRms && a.norm == DT_NORM_LAYER) {
        mean[r] = row_sum<G>(v) * (1.0f / D);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] -= mean[r];
      }
      ss[r] = row_squares<G>(v);
    }
#pragma unroll
    for (int r = 0; r < kHeads; r += 4) {
      float four[4];
      inverse_rms4<D>(ss[r], ss[r + 1], ss[r + 2], ss[r + 3], a.eps, four);
#pragma unroll
      for (int i = 0; i < 4; ++i) rs[r + i] = four[i];
    }
  }
  uint16_t* yp = t.y + ((int64_t)bs * t.H + h0) * D;
#pragma unroll
  for (int r = 0; r < kHeads; ++r) {
    if (r >= nh) break;
    float v[8];
    unpack8<kHalf>(raw[r], v);
    if (kRms || a.norm != DT_NORM_NONE) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = kRms ? v[i] * rs[r] * w[i] : layer_norm(v[i], mean[r], rs[r], w[i], bias[i]);
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int ia = kHalves ? i : 2 * i, ib = kHalves ? 4 + i : 2 * i + 1;
      y[ia] = rotated(v[ia], -v[ib], cs[i], sn[i]) * t.scale;
      y[ib] = rotated(v[ib], v[ia], cs[i], sn[i]) * t.scale;
    }
    const u32x4 o = u32x4{pack2<kHalf>(y[0], y[1]), pack2<kHalf>(y[2], y[3]), pack2<kHalf>(y[4], y[5]), pack2<kHalf>(y[6], y[7])};
    uint16_t* q = yp + r * D;
    if constexpr (kHalves) {
      __builtin_nontemporal_store(u32x2{o.x, o.y}, reinterpret_cast<u32x2*>(q + ea));
      __builtin_nontemporal_store(u32x2{o.z, o.w}, reinterpret_cast<u32x2*>(q + eb));
    } else {
      __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(q + ea));
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_qk_norm_rope_axes(const dt_rotary_rows* rows, int32_t n_rows, int32_t B, int32_t S, int32_t D, int32_t norm, float eps,
                                    const int32_t* positions, int64_t pos_stride_b, int32_t n_axes, const uint64_t* turns,
                                    const uint8_t* axis_of_pair, int32_t rope, const int32_t* sections, int32_t n_sections,
                                    int32_t rounding, void* stream) {
  if (!rows || n_rows < 1 || n_rows > 2 || B <= 0 || S <= 0) {
    set_error("need one or two tensors and positive B and S (got %d, %d, %d)", n_rows, B, S);
    return DT_ERR_INVALID;
  }
  if (D != 64 && D != 128) {
    set_error("head dim %d not built (64 and 128 are)", D);
    return DT_ERR_UNSUPPORTED;
  }
  if (norm < DT_NORM_NONE || norm > DT_NORM_LAYER || (rope != DT_ROPE_INTERLEAVED && rope != DT_ROPE_HALVES) ||
      (rounding & ~(DT_IO_FP16 | DT_WEIGHTS_16))) {
    set_error("bad norm / rope / rounding code (%d, %d, %d)", norm, rope, rounding);
    return DT_ERR_INVALID;
  }
  if (!positions || n_axes < 1 || n_axes > kMostAxes || !turns || !axis_of_pair || pos_stride_b < 0) {
    set_error("positions, turns and axis_of_pair must be non-null, with 1..%d axes and a stride that is not negative", kMostAxes);
    return DT_ERR_INVALID;
  }
  RotaryArgs a{};
  for (int j = 0; j < D / 2; ++j)
    if (axis_of_pair[j] >= n_axes) {
      set_error("pair %d is on axis %d of %d", j, axis_of_pair[j], n_axes);
      return DT_ERR_INVALID;
    }
  int pair_of[64];      // of run element 4 lane + i
  if (rope == DT_ROPE_HALVES) {
    const int32_t whole[1] = {D};
    if (n_sections == 0) {
      sections = whole;
      n_sections = 1;
    }
    if (n_sections < 0 || n_sections > DT_MAX_SECTIONS || !sections) {
      set_error("rotate-half RoPE takes 0..%d sections", DT_MAX_SECTIONS);
      return DT_ERR_INVALID;
    }
    int lo = 0, lane = 0;
    for (int i = 0; i < n_sections; ++i) {
      if (sections[i] <= 0 || (sections[i] & 7) || sections[i] > D - lo) {
        set_error("section %d has %d elements: need positive multiples of 8 that sum to %d", i, sections[i], D);
        return DT_ERR_INVALID;
      }
      for (int e = 0; e < sections[i] / 2; e += 4, ++lane) {
        a.a0[lane] = (uint8_t)(lo + e);
        a.b0[lane] = (uint8_t)(lo + sections[i] / 2 + e);
        for (int k = 0; k < 4; ++k) pair_of[4 * lane + k] = lo / 2 + e + k;
      }
      lo += sections[i];
    }
    if (lo != D) {
      set_error("sections sum to %d, head dim is %d", lo, D);
      return DT_ERR_INVALID;
    }
  } else {
    for (int j = 0; j < D / 2; ++j) pair_of[j] = j;
  }
  for (int j = 0; j < D / 2; ++j) {
    a.axis[j] = axis_of_pair[pair_of[j]];
    a.turns[j] = turns[pair_of[j]];
  }
  for (int i = 0; i < n_rows; ++i) {
    const dt_rotary_rows& r = rows[i];
    if (r.H <= 0 || !r.x || !r.y || !aligned16(r.x) || !aligned16(r.y) || ((r.stride_b | r.stride_s | r.stride_h) & 7)) {
      set_error("tensor %d: x and y must be non-null, 16-byte aligned, with strides that are multiples of 8 elements and a positive number of heads", i);
      return DT_ERR_INVALID;
    }
    if (!(r.out_scale > 0.0f) || !(r.out_scale < INFINITY)) {
      set_error("out_scale must be positive and finite (1 for none)");
      return DT_ERR_INVALID;
    }
    if ((r.weight && !aligned16(r.weight)) || (r.bias && !aligned16(r.bias))) {
      set_error("weight and bias must be 16-byte aligned");
      return DT_ERR_INVALID;
    }
    Rows& d = a.rows[i];
    d.x = static_cast<const uint16_t*>(r.x);
    d.y = static_cast<uint16_t*>(r.y);
    d.sb = r.stride_b; d.ss = r.stride_s; d.sh = r.stride_h;
    d.w = r.weight; d.bias = r.bias;
    d.scale = r.out_scale;
    d.H = r.H;
    d.groups = (r.H - 1) / 4 + 1;
  }
  int64_t groups = (int64_t)a.rows[0].groups + a.rows[1].groups;
  __int128 items = (__int128)B * S * groups;
  if (items * (D / 8) > (1ll << 32) - kThreads || items >= (1ll << 31)) {      // (a grid holds fewer than 2^32 lanes)
    set_error("too many rows");
    return DT_ERR_INVALID;
  }
  const int per_wg = kThreads / (D / 8);
  const bool eight = items > (int64_t)kManyWorkgroups * per_wg && a.rows[0].groups % 2 == 0 && a.rows[1].groups % 2 == 0;
  if (eight) {
    for (Rows& r : a.rows) r.groups /= 2;
    groups /= 2;
    items /= 2;
  }
  a.pos = positions;
  a.pos_sb = pos_stride_b;
  a.S = S;
  a.n_axes = n_axes;
  a.norm = norm;
  a.w16 = (rounding & DT_WEIGHTS_16) != 0;
  a.eps = eps;
  a.items = (uint32_t)items;
  a.by_groups = quotient_by((int32_t)groups);
  a.by_s = quotient_by(S);
  const dim3 grid((unsigned)((items + per_wg - 1) / per_wg)), block(kThreads);
  const hipStream_t st = (hipStream_t)stream;
  const bool half = (rounding & DT_IO_FP16) != 0, halves = rope == DT_ROPE_HALVES;
  const bool rms = norm == DT_NORM_RMS;
#define DT_LAUNCH_L(D, half, halves, rms)                                                                                  \
  do {                                                                                                                       \
    if (eight) hipLaunchKernelGGL((qk_norm_rope_axes_kernel<D, half, halves, 8, rms>), grid, block, 0, st, a);             \
    else hipLaunchKernelGGL((qk_norm_rope_axes_kernel<D, half, halves, 4, rms>), grid, block, 0, st, a);                   \
  } while (0)
#define DT_LAUNCH(D, half, halves)                          \
  do {                                                      \
    if (rms) DT_LAUNCH_L(D, half, halves, true);          \
    else DT_LAUNCH_L(D, half, halves, false);               \
  } while (0)
#define DT_LAUNCH_D(D)                                                           \
  do {                                                                           \
    if (half && halves) DT_LAUNCH(D, true, true);                                \
    else if (half) DT_LAUNCH(D, true, false);                                    \
    else if (halves) DT_LAUNCH(D, false, true);                                  \
    else DT_LAUNCH(D, false, false);                                             \
  } while (0)
  if (D == 128) DT_LAUNCH_D(128);
  else DT_LAUNCH_D(64);
#undef DT_LAUNCH_D
#undef DT_LAUNCH
#undef DT_LAUNCH_L
  return hip_fail(hipGetLastError(), "qk_norm_rope_axes launch");
}
