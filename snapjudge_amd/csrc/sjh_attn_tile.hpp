// sjh_attn_tile.hpp -- LDS tile access shared by the bf16 attention kernels.
#pragma once

#include <type_traits>

#include "sjh_common.hpp"

namespace sjh {

namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((ext_vector_type(8))) short s16x8_t;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2_t;

__device__ __forceinline__ float wave_max32(float v) {
  // lanes l and l^32 hold the two halves of one query's keys: one
  // v_permlane32_swap hands each half the other's value (no LDS round trip)
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Chunk position of 16-byte chunk c of tile row r is c ^ kv_swz(r), a
// permutation of (r >> 1) & 7 (rows r and r + 16 share the key).  LDS serves
// 256 bytes (64 banks) per cycle and a 128-byte row covers half of them, so
// even and odd rows fall in different halves: 16 consecutive rows read at one
// logical chunk (K fragments) then hit 16 distinct bank groups, and the four
// rows r0 + [0, 4) that half a wave's transposed V reads cover (chunks
// 4 db + [0, 4) of each) do too, since rows r0 and r0 + 2 differ in the
// key's bit 2.
__device__ __forceinline__ int kv_swz(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }

// LDS byte offset of element (row, col) of a 64 x 64 bf16 tile.
__device__ __forceinline__ int kv_off(int row, int col) {
  return row * 128 + (((col >> 3) ^ kv_swz(row)) << 4) + ((col & 7) << 1);
}

// Buffer descriptor over the n_bytes bytes from p on (untyped dword loads:
// word 3 carries gfx9's 32-bit data format).  A load at or past n_bytes
// returns zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t seq_rsrc(const bf16_t* p, uint32_t n_bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16_t*>(p), static_cast<short>(0),
                                           static_cast<int>(n_bytes), 0x00020000);
}

// 16 bytes per lane from buffer r at voff + soff into LDS at lds + 16 * lane
// (buffer_load_dwordx4 ... lds; the LDS base goes through M0).
__device__ __forceinline__ void load_lds16_buf(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds), 16,
                                           static_cast<int>(voff), static_cast<int>(soff), 0, 0);
}

// Transposed 8-byte LDS read (ds_read_b64_tr_b16) at LDS byte address
// addr + OFF.  Within each 16-lane group, if lane q + 4k addresses element
// (r0 + k, c0 + 4q) of a row-major tile, lane i of the group receives
// elements (r0 + k, c0 + i), k = 0..3.
//
// Inline asm rather than the builtin: before the builtin's read the compiler
// waits for every direct-to-LDS load in flight (vmcnt(0)), which would hold
// each tile's P.V phase until the next tile's K/V loads (into the other ring
// slot) have landed.  The asm is invisible to the compiler's wait insertion,
// so its results are claimed with lgkm_claim before their first use.
template <int OFF>
__device__ __forceinline__ s16x4_t lds_read_tr(uint32_t addr) {
  static_assert(OFF >= 0 && OFF < 65536, "ds offset field");
  s16x4_t r;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  return r;
}
// Waits until at most N LDS operations of this wave are outstanding, tied to
// the four registers it makes valid (the compiler cannot move their uses
// above it).  LDS operations complete in issue order, so N = the number of
// LDS reads issued after the four means those four have returned; LDS
// operations the compiler issues in between only make the wait longer.
template <int N>
__device__ __forceinline__ void lgkm_claim(s16x4_t& a, s16x4_t& b, s16x4_t& c, s16x4_t& d) {
  static_assert(N >= 0 && N <= 15, "lgkmcnt immediate");
  asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : "n"(N));
}
// f(integral_constant<int, I>) for I = B .. E - 1 in turn: loop indices that
// the asm operands above need as compile-time constants.
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (B < E) {
    f(std::integral_constant<int, B>{});
    static_for<B + 1, E>(f);
  }
}
// LDS byte address of a pointer into the workgroup's LDS.
__device__ __forceinline__ uint32_t lds_addr(const char* p) {
  return static_cast<uint32_t>(
      reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)(p)));
}

}  // namespace

}  // namespace sjh
