// Attention of requests' new tokens over the pages of a cache that they share (gfx950).
//
// Row i of the n new tokens of a request with len tokens stands at position len - n + i among its keys; which of them it sees is a window as of
// attn_window.hip, and the result is a state (out, lse) like its.
#include <algorithm>
#include <cmath>

#include "attn_tiles.h"
#include "dt_common.h"

namespace dt {
namespace {

constexpr int32_t kMostTokens = 1 << 29;   // positions, spans and lengths: their sums stay in 32 bits

struct PagesArgs {
  const uint16_t* q;
  int64_t q_ss, q_sh;
  uint16_t* out;
  float* lse;
  Pages kv;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t *lens, *cu;
  int32_t width, B, T, H, Hk, group;
  int32_t left, right;          // spans in tokens; -1: no border
  int32_t frame, sinks;
  Quotient by_frame;
  float scale_log2;
};

// One wavefront a row and head: a lane has a key's score, then its columns.
template <int D, bool kHalf>
__global__ __launch_bounds__(64) void attn_pages_kernel(const PagesArgs a) {
  typedef Elem<kHalf> E;
  constexpr int kCols = D / 64;
  const int lane = threadIdx.x, row = blockIdx.x, head = blockIdx.y;
  int b = -1, begin = 0, n = 0;
  for (int i = 0; i < a.B; ++i) {
    const int lo = min(max(a.cu[i], 0), a.T), hi = min(max(a.cu[i + 1], 0), a.T);
    if (row >= lo && row < hi) {
      b = i;
      begin = lo;
      n = hi - lo;
      break;
    }
  }
  typename E::t* out = reinterpret_cast<typename E::t*>(a.out) + ((int64_t)row * a.H + head) * D + lane * kCols;
  float m = -INFINITY, l = 0.f, acc[kCols] = {};
  if (b >= 0) {
    const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.width * a.kv.page);
    const int x = len - n + row - begin - a.sinks;
    const int f = x >= 0 ? (int)quotient(x, a.by_frame) : -1 - (int)quotient(-1 - x, a.by_frame);
    const int start = a.sinks + f * a.frame;
    const int lo = a.left < 0 ? 0 : max(start - a.left, 0), hi = a.right < 0 ? len : min(max(start + a.right, 0), len);
    const int hk = head / a.group;
    const uint16_t* q = a.q + row * a.q_ss + head * a.q_sh;
    auto place = [&](int j, int i) -> const uint16_t* {      // of key j (0) or its value (1), null where it has no page
      const int at = (int)quotient(j, a.kv.by_page), p = a.tables[b * a.table_stride + at];
      if ((uint32_t)p >= (uint32_t)a.kv.n_pages) return nullptr;
      return a.kv.base[i] + p * a.kv.sp[i] + (int64_t)(j - at * a.kv.page) * a.kv.ss[i] + hk * a.kv.sh[i];
    };
    for (int j0 = 0; j0 < hi; j0 += 64) {
      if (j0 + 64 <= lo && j0 >= a.sinks) continue;
      const int j = j0 + lane;
      const bool seen = j < hi && (j >= lo || j < a.sinks);
      float s = -INFINITY;
      if (seen) {
        s = 0.f;
        if (const uint16_t* k = place(j, 0))
          for (int d = 0; d < D; d += 8) {
            const typename E::x8 u = *reinterpret_cast<const typename E::x8*>(q + d), w = *reinterpret_cast<const typename E::x8*>(k + d);
#pragma unroll
            for (int e = 0; e < 8; ++e) s = __builtin_fmaf((float)u[e], (float)w[e], s);
          }
        s *= a.scale_log2;
      }
      float top = s;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
      const float m_new = fmaxf(m, top), ref = m_new > -INFINITY ? m_new : 0.f;
      const float alpha = __builtin_amdgcn_exp2f(m - ref), w = seen ? __builtin_amdgcn_exp2f(s - ref) : 0.f;
      m = m_new;
      float sum = w;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d);
      l = l * alpha + sum;
#pragma unroll
      for (int e = 0; e < kCols; ++e) acc[e] *= alpha;
      for (int i = 0; i < 64; ++i) {
        const int key = j0 + i;
        if (key >= hi || !(key >= lo || key < a.sinks)) continue;
        const float wi = __shfl(w, i);
        if (const uint16_t* v = place(key, 1))
#pragma unroll
          for (int e = 0; e < kCols; ++e) acc[e] = __builtin_fmaf(wi, (float)reinterpret_cast<const typename E::t*>(v + lane * kCols)[e], acc[e]);
      }
    }
  }
  const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int e = 0; e < kCols; ++e) out[e] = (typename E::t)(acc[e] * inv);
  if (lane == 0) a.lse[(int64_t)head * a.T + row] = l != 0.f ? (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f : -INFINITY;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace dt

using namespace dt;

extern "C" int dt_attn_pages_fwd(const void* q, const int64_t* q_strides, void* out, float* lse, int32_t T, int32_t H, int32_t Hk, int32_t D,
                                 const dt_pages* pages, const int32_t* tables, int64_t table_stride, int32_t width, int32_t B, const int32_t* lens,
                                 const int32_t* cu_seqlens, int32_t max_seqlen_q, const dt_window* window, float softmax_scale, int32_t flags,
                                 void* workspace, int64_t workspace_bytes, uint32_t* counters, int64_t n_counters, void* stream) {
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
  if ((int64_t)T * (H / Hk) > (1ll << 30) || H > 65535 || T > (1 << 25)) {
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
  a.cu = cu_seqlens;
  a.width = width;
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
  a.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / std::sqrt((float)D)) * 1.4426950408889634f;
  const hipStream_t st = (hipStream_t)stream;
  const bool half = (flags & DT_ATTN_FP16) != 0;
  const dim3 grid(T, H), block(64);
  if (D == 128 && half) hipLaunchKernelGGL((attn_pages_kernel<128, true>), grid, block, 0, st, a);
  else if (D == 128) hipLaunchKernelGGL((attn_pages_kernel<128, false>), grid, block, 0, st, a);
  else if (half) hipLaunchKernelGGL((attn_pages_kernel<64, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((attn_pages_kernel<64, false>), grid, block, 0, st, a);
  return hip_fail(hipGetLastError(), "attn_pages launch");
}
