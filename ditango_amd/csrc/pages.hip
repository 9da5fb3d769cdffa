// Pages of a cache that several requests share (gfx950): which page holds which tokens, and new keys and values into their places.
//
// dt_plan_pages.  A request of len tokens holds the first ceil(len / page) entries of its row of the tables; a page that no request holds is free, so
// tables and lengths are all the state there is: no list of free pages to keep, a request ends by its length going to 0, and requests may share
// pages.  New tokens n come to
//   need = ceil((len + n) / page) - ceil(len / page)
// free pages, lowest ids first, requests in order; the slot of token j of a request is table[j / page] * page + j % page.
//
// dt_append_pages.  Rows of k and v into their slots: bound by the memory.
#include <algorithm>

#include "dt_common.h"

namespace dt {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- plan ---------------------------------------------------------------------------------------------------------

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kMostRequests = 2048;
constexpr int kMostPages = 1 << 20;

struct PlanArgs {
  int32_t* tables;
  int64_t table_stride;
  const int32_t *lens, *new_lens;
  int32_t B, width, n_pages, page;
  int32_t n_tokens;
  int32_t* lens_out;
  int32_t* cu;
  int64_t* slots;
  uint8_t* served;
  Quotient by_page;
  int32_t words;               // of the bitmap
  int32_t lanes;               // that read a request's entries, a power of two
};

__device__ __forceinline__ int held_pages(const PlanArgs& a, int tokens) { return (int)quotient(tokens + a.page - 1, a.by_page); }

// Sums along the threads that stop at `most`, and are still sums then: of x, 0 .. 2^30, over the lanes up to this one, or over the threads in front of it;
// *total over all.
template <int kCtrl, int kRows>
__device__ __forceinline__ int moved(int x) { return __builtin_amdgcn_update_dpp(0, x, kCtrl, kRows, 0xf, false); }
__device__ __forceinline__ int wave_scan(int sum, int most) {      // rows of 16 lanes, then across them
  sum = min(sum + moved<0x111, 0xf>(sum), most);
  sum = min(sum + moved<0x112, 0xf>(sum), most);
  sum = min(sum + moved<0x114, 0xf>(sum), most);
  sum = min(sum + moved<0x118, 0xf>(sum), most);
  sum = min(sum + moved<0x142, 0xa>(sum), most);
  return min(sum + moved<0x143, 0xc>(sum), most);
}
__device__ __forceinline__ int block_scan(int x, int most, int* waves, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sum = wave_scan(x, most);
  if (lane == 63) waves[wave] = sum;
  const int mine = __shfl_up(sum, 1);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    const int w = waves[i];
    if (i < wave) before = min(before + w, most);
    all = min(all + w, most);
  }
  __syncthreads();
  *total = all;
  return min(before + (lane > 0 ? mine : 0), most);
}

// The last of the n values of x, which never fall, that is at most v (x[0] is): a quarter of them each time, as three reads under way together take no longer
// than one.
__device__ __forceinline__ int last_at_most(const int32_t* x, int n, int v) {
  int lo = 0;
  while (n > 1) {
    const int quarter = (n + 3) >> 2, last = lo + n - 1;
    const int p = min(lo + quarter, last), q = min(lo + 2 * quarter, last), r = min(lo + 3 * quarter, last);
    const int u = x[p], w = x[q], y = x[r];
    const int from = y <= v ? r : w <= v ? q : u <= v ? p : lo;
    n = min(quarter, last + 1 - from);
    lo = from;
  }
  return lo;
}

__device__ __forceinline__ int64_t slot_of(const PlanArgs& a, int b, int j) {
  const int i = (int)quotient(j, a.by_page);
  const int p = a.tables[b * a.table_stride + i];
  return (uint32_t)p < (uint32_t)a.n_pages ? (int64_t)p * a.page + (j - i * a.page) : -1;
}

// One workgroup: the free pages are in its LDS, a bit a page.  Latency all the way: 8 requests' next tokens 5.7 us, of which an empty launch is 2.4, lengths and
// their sums 1.2, the tables' entries 1.6; 64 requests that hold 29 300 pages and get 1250 11.8, of which the entries are 4.5 and what is given away 2.5 (their
// 86 400 slots, by a launch behind it, 4.0).
__global__ __launch_bounds__(kPlanThreads) void plan_pages_kernel(const PlanArgs a, int slots_too) {
  extern __shared__ __align__(16) uint8_t lds[];
  __shared__ int32_t waves[kPlanWaves];
  __shared__ int32_t before[kPlanThreads];          // free pages in front of a thread's words
  uint32_t* taken = reinterpret_cast<uint32_t*>(lds);
  int32_t* cu = reinterpret_cast<int32_t*>(taken + a.words);      // [B + 1]
  int32_t* start = cu + a.B + 1;                                  // [B]: pages that the requests in front of it need
  int32_t* len = start + a.B;                                     // [B], its complement where the request is not served
  const int tid = threadIdx.x, most_len = a.width * a.page;
  int tokens = 0, pages = 0;
  const bool one_wave = a.B <= 64;        // then every wavefront sums by itself, and none waits for another
  for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
    const int b = one_wave ? tid & 63 : b0 + tid;
    const bool there = b < a.B;
    const int l = there ? min(max(a.lens[b], 0), most_len) : 0, asked = there ? min(max(a.new_lens[b], 0), a.n_tokens) : 0;
    if (b0 == 0)
      for (int i = tid; i < a.words; i += kPlanThreads) taken[i] = 0;
    int total;
    auto in_front = [&](int x, int most) __attribute__((always_inline)) {
      if (!one_wave) return block_scan(x, most, waves, &total);
      const int sum = wave_scan(x, most);
      total = __builtin_amdgcn_readlane(sum, 63);
      return moved<0x138, 0xf>(sum);      // of the lane in front
    };
    const int from = min(tokens + in_front(asked, a.n_tokens), a.n_tokens), n = min(asked, a.n_tokens - from);
    tokens = min(tokens + total, a.n_tokens);
    const bool fits = n <= most_len - l;
    const int before_me = in_front(there && fits ? min(held_pages(a, l + n) - held_pages(a, l), kMostPages + 1) : 0, kMostPages + 1);
    if (there && (tid < 64 || !one_wave)) {
      cu[b] = from;
      len[b] = fits ? l : ~l;
      start[b] = min(pages + before_me, kMostPages + 1);
    }
    pages = min(pages + total, kMostPages + 1);
  }
  if (tid == 0) cu[a.B] = tokens;
  __syncthreads();
  // the pages that somebody holds; a.lanes threads a request, up to 32 entries of each under way together
  constexpr int kSome = 8, kTimes = 4;
  for (int b = tid / a.lanes; b < a.B; b += kPlanThreads / a.lanes) {
    const int l = len[b], n = held_pages(a, l < 0 ? ~l : l);
    const int32_t* row = a.tables + b * a.table_stride;
    for (int i = tid % a.lanes; i < n; i += kTimes * kSome * a.lanes) {
      int p[kTimes][kSome];
#pragma unroll
      for (int k = 0; k < kTimes; ++k)
        if (i + k * kSome * a.lanes < n)
#pragma unroll
          for (int j = 0; j < kSome; ++j) p[k][j] = row[min(i + (k * kSome + j) * a.lanes, n - 1)];
#pragma unroll
      for (int k = 0; k < kTimes; ++k)
        if (i + k * kSome * a.lanes < n)
#pragma unroll
          for (int j = 0; j < kSome; ++j)
            if (i + (k * kSome + j) * a.lanes < n && (uint32_t)p[k][j] < (uint32_t)a.n_pages) atomicOr(&taken[p[k][j] >> 5], 1u << (p[k][j] & 31));
    }
  }
  // behind the last page there is none
  if (tid == 0 && (a.n_pages & 31)) atomicOr(&taken[a.words - 1], ~0u << (a.n_pages & 31));
  __syncthreads();
  const int each = (a.words + kPlanThreads - 1) / kPlanThreads;
  int mine = 0;
  for (int i = 0; i < each; ++i) {
    const int w = tid * each + i;
    if (w < a.words) mine += __popc(~taken[w]);
  }
  int n_free;
  before[tid] = block_scan(mine, kMostPages + 1, waves, &n_free);
  // who is served: in order, from the first one that finds too few on none that needs any
  int granted = 0;
  for (int b = tid; b < a.B; b += kPlanThreads) {
    const int l = len[b], at = l < 0 ? ~l : l, n = cu[b + 1] - cu[b];
    const int need = l < 0 ? 0 : held_pages(a, at + n) - held_pages(a, at);
    const bool yes = l >= 0 && (need == 0 || need <= n_free - start[b]);
    if (!yes) len[b] = ~at;
    else if (need > 0) granted = max(granted, start[b] + need);
    a.served[b] = yes;
    a.lens_out[b] = yes ? at + n : at;
    a.cu[b] = cu[b];
  }
  if (tid == 0) a.cu[a.B] = cu[a.B];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) granted = max(granted, __shfl_xor(granted, d));
  if ((tid & 63) == 0) waves[tid >> 6] = granted;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) granted = max(granted, waves[i]);
  // the r-th free page, for every r that is given away
  const bool kept = granted <= kPlanThreads;      // then `before` keeps them for the slots
  int page = 0, entry_of = 0, entry = 0;
  for (int r = tid; r < granted; r += kPlanThreads) {
    const int t = last_at_most(before, kPlanThreads, r);
    int k = r - before[t], w = t * each;
    for (; k >= __popc(~taken[w]); ++w) k -= __popc(~taken[w]);
    uint32_t bits = ~taken[w];
    for (; k > 0; --k) bits &= bits - 1;
    entry_of = last_at_most(start, a.B, r);
    entry = held_pages(a, len[entry_of]) + r - start[entry_of];
    page = 32 * w + __ffs(bits) - 1;
    if (!kept || !slots_too) a.tables[entry_of * a.table_stride + entry] = page;
  }
  if (!slots_too) return;
  __syncthreads();
  if (kept) {
    if (tid < granted) before[tid] = page;
    __syncthreads();
    if (tid < granted) a.tables[entry_of * a.table_stride + entry] = page;
  }
  for (int t = tid; t < a.n_tokens; t += kPlanThreads) {
    int64_t slot = -1;
    if (t < cu[a.B]) {
      const int b = last_at_most(cu, a.B, t);
      if (len[b] >= 0) {
        const int j = len[b] + t - cu[b], held = held_pages(a, len[b]), i = (int)quotient(j, a.by_page);
        slot = kept && i >= held ? (int64_t)before[start[b] + i - held] * a.page + (j - i * a.page) : slot_of(a, b, j);
      }
    }
    a.slots[t] = slot;
  }
}

// Slots of many tokens, from what the kernel above has left.
__global__ __launch_bounds__(256) void plan_slots_kernel(const PlanArgs a) {
  extern __shared__ __align__(16) int32_t cu[];
  for (int i = threadIdx.x; i <= a.B; i += 256) cu[i] = a.cu[i];
  __syncthreads();
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= a.n_tokens) return;
  int64_t slot = -1;
  if (t < cu[a.B]) {
    const int b = last_at_most(cu, a.B, t);
    if (a.served[b]) slot = slot_of(a, b, a.lens_out[b] + t - cu[b + 1]);      // (lens may be lens_out)
  }
  a.slots[t] = slot;
}

// Slots by the one workgroup up to here, else by a launch of their own: 2560 tokens 9.5 us against 10.8, 4096 9.5 .. 10.4 against 10.6 .. 11.1, 6400 12.0
// against 10.9, 16 384 19.2 against 11.2 (64 requests).
constexpr int kSlotsInPlan = 4096;

// ---- append -------------------------------------------------------------------------------------------------------

struct AppendArgs {
  const uint16_t* x[2];
  int64_t x_ss[2], x_sh[2];
  Pages to;
  const int64_t* slots;
  uint32_t items;              // tokens x chunks of 8 elements of a token's heads
  Quotient by_chunks;
  int32_t chunks, row_shift;   // of a head: log2(D / 8)
};

// A lane copies two pieces of k and two of v, past the caches: 14 882 tokens of 24 heads of 128 63.6 us, 5.8 TB/s (one piece 63.9, through the caches 68.9); 2 x
// 2222 of 48 heads of 64 20.3 (21.3, 21.2).
constexpr int kCopies = 2;
__global__ __launch_bounds__(256) void append_pages_kernel(const AppendArgs a) {
  const uint32_t first = blockIdx.x * (256 * kCopies) + threadIdx.x;
  u32x4 x[kCopies][2];
  int64_t slot[kCopies];
  int h[kCopies], d[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const uint32_t item = min(first + j * 256, a.items - 1), t = quotient(item, a.by_chunks), c = item - t * a.chunks;
    slot[j] = first + j * 256 < a.items ? a.slots[t] : -1;
    h[j] = c >> a.row_shift;
    d[j] = 8 * (c & ((1 << a.row_shift) - 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) x[j][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(a.x[i] + t * a.x_ss[i] + h[j] * a.x_sh[i] + d[j]));
  }
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    if (!a.to.has(slot[j])) continue;
#pragma unroll
    for (int i = 0; i < 2; ++i) __builtin_nontemporal_store(x[j][i], reinterpret_cast<u32x4*>(a.to.row(i, slot[j]) + h[j] * a.to.sh[i] + d[j]));
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

int check_pages(const dt_pages* p, int D, Pages& out) {
  if (D != 64 && D != 128) {
    set_error("head dim %d not built (64 and 128 are)", D);
    return DT_ERR_UNSUPPORTED;
  }
  if (!p || p->n_pages < 0 || p->page_size <= 0 || p->page_size % 16) {
    set_error("pages must be given, not negative in number, and of a positive multiple of 16 tokens");
    return DT_ERR_INVALID;
  }
  if ((int64_t)p->n_pages * p->page_size > INT32_MAX) {
    set_error("%d pages of %d tokens: more than 2^31 - 1 tokens are not supported", p->n_pages, p->page_size);
    return DT_ERR_UNSUPPORTED;
  }
  if (p->n_pages > 0 && (!p->k || !p->v || !aligned16(p->k) || !aligned16(p->v))) {
    set_error("key and value pages must be non-null and 16-byte aligned");
    return DT_ERR_INVALID;
  }
  const int64_t* strides[2] = {p->k_strides, p->v_strides};
  for (int i = 0; i < 2; ++i) {
    if ((strides[i][0] | strides[i][1] | strides[i][2]) & 7) {
      set_error("strides of the pages must be multiples of 8 elements");
      return DT_ERR_INVALID;
    }
    // (a tile's rows are addressed with 32 bits)
    if (strides[i][1] < 0 || strides[i][1] > (1 << 23)) {
      set_error("token strides of the pages must be in 0..2^23 elements");
      return DT_ERR_INVALID;
    }
    if (strides[i][0] < 0 || strides[i][0] > INT32_MAX) {
      set_error("page strides must be in 0..2^31 - 1 elements");
      return DT_ERR_INVALID;
    }
    out.base[i] = static_cast<uint16_t*>(i ? p->v : p->k);
    out.sp[i] = strides[i][0];
    out.ss[i] = strides[i][1];
    out.sh[i] = strides[i][2];
  }
  out.n_pages = p->n_pages;
  out.page = p->page_size;
  out.by_page = quotient_by(p->page_size);
  return DT_OK;
}

}  // namespace dt

using namespace dt;

extern "C" int dt_plan_pages(int32_t* tables, int64_t table_stride, int32_t width, const int32_t* lens, const int32_t* new_lens, int32_t B,
                             int32_t n_pages, int32_t page_size, int32_t n_tokens, int32_t* lens_out, int32_t* cu_seqlens, int64_t* slots,
                             uint8_t* served, void* stream) {
  if (B <= 0 || width < 0 || n_pages < 0 || n_tokens < 0 || page_size <= 0 || page_size % 16) {
    set_error("B must be positive, width, n_pages and n_tokens not negative, page_size a positive multiple of 16 (got %d, %d, %d, %d, %d)", B, width, n_pages,
              n_tokens, page_size);
    return DT_ERR_INVALID;
  }
  if (!lens || !new_lens || !lens_out || !cu_seqlens || !served || (width > 0 && !tables) || (n_tokens > 0 && !slots) || table_stride < width) {
    set_error("tables, lens, new_lens and the results must be non-null, table rows at least `width` apart");
    return DT_ERR_INVALID;
  }
  if (B > kMostRequests || n_pages > kMostPages || (int64_t)width * page_size > (1 << 29) || (int64_t)n_pages * page_size > INT32_MAX ||
      n_tokens > (1 << 29)) {
    set_error("more than %d requests, %d pages, 2^29 tokens of a request, 2^31 - 1 of the pool or 2^29 new ones are not supported", kMostRequests, kMostPages);
    return DT_ERR_UNSUPPORTED;
  }
  PlanArgs a{};
  a.tables = tables;
  a.table_stride = table_stride;
  a.lens = lens;
  a.new_lens = new_lens;
  a.B = B;
  a.width = width;
  a.n_pages = n_pages;
  a.page = page_size;
  a.n_tokens = n_tokens;
  a.lens_out = lens_out;
  a.cu = cu_seqlens;
  a.slots = slots;
  a.served = served;
  a.by_page = quotient_by(page_size);
  a.words = (n_pages + 31) / 32;
  a.lanes = kPlanThreads;
  while (a.lanes > 1 && (int64_t)a.lanes * B > kPlanThreads) a.lanes /= 2;
  const int lds = 4 * (a.words + 3 * B + 1);
  static thread_local int allowed_dev = -1;
  int dev = 0;
  if (int rc = hip_fail(hipGetDevice(&dev), "hipGetDevice")) return rc;
  if (allowed_dev != dev) {      // more than 64 KB of LDS has to be allowed once per kernel and device
    if (int rc = hip_fail(hipFuncSetAttribute(reinterpret_cast<const void*>(plan_pages_kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                              4 * (kMostPages / 32 + 3 * kMostRequests + 1)), "hipFuncSetAttribute"))
      return rc;
    allowed_dev = dev;
  }
  const hipStream_t st = (hipStream_t)stream;
  const int here = n_tokens <= kSlotsInPlan;
  hipLaunchKernelGGL(plan_pages_kernel, dim3(1), dim3(kPlanThreads), lds, st, a, here);
  if (int rc = hip_fail(hipGetLastError(), "plan_pages launch")) return rc;
  if (here) return DT_OK;
  hipLaunchKernelGGL(plan_slots_kernel, dim3((n_tokens + 255) / 256), dim3(256), 4 * (B + 1), st, a);
  return hip_fail(hipGetLastError(), "plan_slots launch");
}

extern "C" int dt_append_pages(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides, int32_t T, int32_t Hk, int32_t D,
                               const dt_pages* pages, const int64_t* slots, void* stream) {
  if (T <= 0 || Hk <= 0) {
    set_error("T and Hk must be positive (got %d, %d)", T, Hk);
    return DT_ERR_INVALID;
  }
  AppendArgs a{};
  if (int rc = check_pages(pages, D, a.to)) return rc;
  if (!k || !v || !k_strides || !v_strides || !slots || !aligned16(k) || !aligned16(v)) {
    set_error("k, v, their strides and slots must be non-null, k and v 16-byte aligned");
    return DT_ERR_INVALID;
  }
  if ((k_strides[0] | k_strides[1] | v_strides[0] | v_strides[1]) & 7) {
    set_error("strides must be multiples of 8 elements");
    return DT_ERR_INVALID;
  }
  const int64_t items = (int64_t)T * Hk * (D / 8);
  if (items >= (1ll << 31)) {
    set_error("too many rows");
    return DT_ERR_INVALID;
  }
  a.x[0] = static_cast<const uint16_t*>(k);
  a.x[1] = static_cast<const uint16_t*>(v);
  a.x_ss[0] = k_strides[0];
  a.x_ss[1] = v_strides[0];
  a.x_sh[0] = k_strides[1];
  a.x_sh[1] = v_strides[1];
  a.slots = slots;
  a.items = (uint32_t)items;
  a.chunks = Hk * (D / 8);
  a.by_chunks = quotient_by(a.chunks);
  a.row_shift = D == 128 ? 4 : 3;
  hipLaunchKernelGGL(append_pages_kernel, dim3((unsigned)((items + 256 * kCopies - 1) / (256 * kCopies))), dim3(256), 0, (hipStream_t)stream, a);
  return hip_fail(hipGetLastError(), "append_pages launch");
}
