// lds_tiles.h -- key and value tiles in LDS: 16-byte copies from global memory
// straight into LDS, the waits that go with them, the swizzles of the rows and the
// transposed reads (2-byte types). Used by paged_prefill.hip and paged_shared.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mgi_common.h"

namespace mgi {

// Rows store their 16-byte chunk c at c ^ k_swz(r) (K) and c ^ v_swz(r) (V), swizzles
// chosen by measuring the read sequences of paged_prefill_tr on MI355X. CPR: chunks
// per row.
template <int CPR>
__device__ __forceinline__ int k_swz(int row) {
  return (row & 3) | ((row >> 1) & (CPR - 4));
}
template <int CPR>
__device__ __forceinline__ int v_swz(int row) {
  return CPR == 16 ? (2 * (row & 3)) | (8 * ((row >> 3) & 1)) : 2 * (row & 3);
}

// Source of the zero rows the copies read for keys that must contribute nothing.
__device__ __align__(16) const unsigned char kZeroRow[512] = {0};

template <typename T> struct TrRead;
template <> struct TrRead<bf16_t> {
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  // From an LDS byte address: constant terms added to it fold into the
  // instruction's offset field.
  __device__ static __forceinline__ uint2 at(uint32_t addr) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
                                         (__attribute__((address_space(3))) v4*)(uintptr_t)addr));
  }
};
template <> struct TrRead<f16_t> {
  typedef __fp16 v4 __attribute__((__vector_size__(4 * sizeof(__fp16))));
  __device__ static __forceinline__ uint2 at(uint32_t addr) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                                         (__attribute__((address_space(3))) v4*)(uintptr_t)addr));
  }
};

// One 16-byte copy per lane from global memory into LDS at lds_base + 16 *
// lane (lds_base wave-uniform): global_load_lds_dwordx4 from a per-lane
// address, or from a wave-uniform base plus a per-lane 32-bit offset. The
// instruction takes its LDS base from M0; the "{m0}" operand has the compiler
// set M0 to lds_base before the statement (the asm only reads it), and the
// s_nop is the wait state an LDS copy needs after an SALU write of M0. The
// copy stays opaque to the compiler's wait-count tracking: the pipeline below
// counts its copies itself (wait_and_barrier). With the compiler's own
// __builtin_amdgcn_global_load_lds the kernel measured 4% slower on MI355X
// (2048 rows after 2048: 70.5-71.1 against 67.8-68.0 us on one box), as the
// compiler then drains every LDS read (lgkmcnt(0)) before MFMAs that use
// them.
__device__ __forceinline__ void copy16_to_lds(const void* src, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds_base) : "memory");
}
__device__ __forceinline__ void copy16_to_lds(const void* sbase, uint32_t voff, uint32_t lds_base) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_base)
               : "memory");
}

// Waits until at most N of this wave's vector-memory instructions are
// outstanding and all its LDS and scalar memory instructions are done, then
// joins the workgroup barrier.
template <int N>
__device__ __forceinline__ void wait_and_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt immediate");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));  // vmcnt(N) expcnt(7) lgkmcnt(0)
  asm volatile("s_barrier" ::: "memory");
}

__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)(p);
}

template <int V> struct Stage {
  static constexpr int value = V;
};

// Calls f(Stage<I>{}) for I = B .. E - 1.
template <int B, int E, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  if constexpr (B < E) {
    f(Stage<B>{});
    static_for<B + 1, E>(f);
  }
}

}  // namespace mgi
