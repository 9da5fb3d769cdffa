// Building blocks of the attention kernels: element types and their MFMA, LDS operand reads, tile loads that go straight into the LDS.
#pragma once

#include "dt_common.h"

namespace dt {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// The 16-bit element type of q, K, V, P and the output states: bfloat16, or IEEE half (kHalf).  Loads, LDS
// layout, swizzles and the transposing reads only see 16-bit elements; the type decides the MFMA and the
// roundings of P and of the output.
template <bool kHalf>
struct Elem {
  typedef __bf16 t;
  typedef __bf16 x8 __attribute__((ext_vector_type(8)));
  typedef __bf16 x4 __attribute__((ext_vector_type(4)));
  typedef __bf16 x2 __attribute__((ext_vector_type(2)));
  __device__ static __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // two packed elements of a 32-bit word, widened
  __device__ static __forceinline__ f32x2 widen(uint32_t w) {
    f32x2 f;
    f.x = __builtin_bit_cast(float, w << 16);
    f.y = __builtin_bit_cast(float, w & 0xffff0000u);
    return f;
  }
};
template <>
struct Elem<true> {
  typedef _Float16 t;
  typedef _Float16 x8 __attribute__((ext_vector_type(8)));
  typedef _Float16 x4 __attribute__((ext_vector_type(4)));
  typedef _Float16 x2 __attribute__((ext_vector_type(2)));
  __device__ static __forceinline__ f32x16 mfma(x8 a, x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  __device__ static __forceinline__ f32x2 widen(uint32_t w) {
    return __builtin_convertvector(__builtin_bit_cast(x2, w), f32x2);
  }
};

// Row permutation of the K operand: MFMA row i -> key (within a 32-key half tile).
__device__ __forceinline__ int key_of_row(int i) {
  return (i & 19) | ((i & 4) << 1) | ((i & 8) >> 1);
}

// Raw buffer descriptor word 3 for gfx9-family targets (32-bit data format, no swizzle).
constexpr int kRsrcFlags = 0x00020000;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
// Transposing LDS read (ds_read_b64_tr_b16).  Within each block of 16 lanes the 16 x 4 matrix of
// 16-bit elements [source lane][element] is read as 4 rows of 16 (source lane 4j+m supplies
// row j, columns 4m..4m+3) and lane i receives column i: element j = row j, column i.
__device__ __forceinline__ s16x4 lds_read_tr(const uint8_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (s16x4 __attribute__((address_space(3)))*)(p));
}

// Raw buffer descriptor: base address, stride 0, number of valid bytes, flags.
__device__ __forceinline__ u32x4 make_rsrc(const void* base, uint32_t valid_bytes) {
  const uint64_t p = reinterpret_cast<uint64_t>(base);
  u32x4 r;   // uniform by construction; say so, the descriptor then lives in scalar registers
  r.x = __builtin_amdgcn_readfirstlane((uint32_t)p);
  r.y = __builtin_amdgcn_readfirstlane((uint32_t)(p >> 32) & 0xffffu);
  r.z = __builtin_amdgcn_readfirstlane(valid_bytes);
  r.w = (uint32_t)kRsrcFlags;
  return r;
}
// One 16-byte-per-lane buffer load whose destination is the LDS: lane L's bytes land at
// lds_addr + 16 L (lds_addr, through M0, is uniform).  Written as inline assembly on purpose: the
// compiler, when it sees such a load, makes every later LDS read of the wavefront wait for ALL
// outstanding loads (it cannot tell that the reads touch other buffers), which turns a prefetch
// several phases deep into one that must land within the phase.  Here the waits are the explicit
// vmcnt in front of the barriers.  (Loads the compiler does not know of only make its own vmcnt
// waits for other loads stricter, never too weak: the counter retires in order.)
__device__ __forceinline__ void load_block_to_lds(u32x4 rsrc, uint32_t lane_off, uint32_t uniform_off, uint32_t lds_addr) {
  // (the uniform operands are uniform by construction; say so, or a value the compiler happens to
  // hold in a vector register ends up in the instruction as one)
  u32x4 r;
  r.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  r.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  r.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  r.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
               :
               : "v"(lane_off), "s"(r), "s"(__builtin_amdgcn_readfirstlane(uniform_off)),
                 "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory", "m0");
}

// The same for bytes that nobody else reads: past the caches, which keep what others do.
__device__ __forceinline__ void load_block_once_to_lds(u32x4 rsrc, uint32_t lane_off, uint32_t lds_addr) {
  u32x4 r;
  r.x = __builtin_amdgcn_readfirstlane(rsrc.x);
  r.y = __builtin_amdgcn_readfirstlane(rsrc.y);
  r.z = __builtin_amdgcn_readfirstlane(rsrc.z);
  r.w = __builtin_amdgcn_readfirstlane(rsrc.w);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen nt lds"
               :
               : "v"(lane_off), "s"(r), "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory", "m0");
}

// The same from an address of each lane's own.
__device__ __forceinline__ void load_rows_to_lds(const uint16_t* from, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(from), "s"(__builtin_amdgcn_readfirstlane(lds_addr))
               : "memory", "m0");
}

// ---- states that meet inside a launch ----------------------------------------------------------
// What another workgroup of the launch reads (states and partial states of a merging launch) is stored and loaded with the
// device-scope bit: past the L1 and the XCD's L2, so that behind the writer's s_waitcnt vmcnt(0) it is where every XCD finds
// it.  The fences of an acquire and release at device scope do the same to whole caches: the invalidation alone, executed by
// one wavefront per merge, took the keys and values of the XCD's other workgroups out of its L2 and cost 4 us per work
// item (two samples of 24 heads x 1861 queries x 3 of 8 chunks 242 -> 261 us); counting and waiting cost nothing that shows.
constexpr int kNt = 2, kDevice = 16, kDeviceNt = kDevice | kNt;   // cache-policy bits of a raw buffer access: nt, sc1
typedef __amdgpu_buffer_rsrc_t Rsrc;
__device__ __forceinline__ Rsrc buffer_of(const void* base, uint32_t valid_bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, valid_bytes, kRsrcFlags);
}
__device__ __forceinline__ void store_device(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_device(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace dt
