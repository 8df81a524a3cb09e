// Device building blocks that the attention kernels share: fragment types,
// matrix and cross-lane instructions, direct-to-LDS loads, waits and barriers.
#ifndef FA_DEVICE_H
#define FA_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Maximum of two scores or of two parts' lse. IEEE-754 maximum lowers to a
// single v_maximum3_f32 with no operand canonicalization, and a NaN on either
// side stays one.
__device__ __forceinline__ float smax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Combine a per-lane value with the lane 32 apart (same query row, other
// half of the keys).
__device__ __forceinline__ float half_max(float x) {
  auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return smax(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// acc + the FP16 value in half HI (0 = low, 1 = high) of x, one rounding:
// v_fma_mix_f32 with the FP16 operand converted exactly and multiplied by
// 1.0. It runs on the plain VALU pipe; the FP16 dot product v_dot2c_f32_f16
// (one instruction per pair) measured 3-4 % slower as the softmax's row sum,
// beside the matrix products of the other wave on the SIMD.
template <int HI>
__device__ __forceinline__ float add_f16(float acc, h2 x) {
  if constexpr (HI)
    asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(acc) : "v"(x));
  else
    asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel_hi:[1,0,0]" : "+v"(acc) : "v"(x));
  return acc;
}

__device__ __forceinline__ f32x16 mfma32(h8 a, h8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// The LDS word a transposing read returns: ds_read_b64_tr_b16 with lane j
// pointing at 4 consecutive FP16 values gives, in each group of 16 lanes,
// lane l the values at offset l % 4 of the 4 lanes 4e + (l % 16) / 4 of its
// group (e = 0..3): the 4 x 16 block those lanes address, read by column.
typedef __attribute__((__vector_size__(4 * sizeof(__fp16)))) __fp16 tr_h4;
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ h4 lds_read_tr(const char* p) {
  const tr_h4 r = __builtin_amdgcn_ds_read_tr16_b64_v4f16(
      (__attribute__((address_space(3))) tr_h4*)(p));
  return __builtin_bit_cast(h4, r);
}

// Raw-buffer descriptor (gfx9 layout: base address, stride 0, range in
// bytes, 32-bit data format) for loads from `base`; the hardware returns
// zeros for any 32-bit word whose offset (per-lane plus scalar) lies at or
// past `bytes`, also into LDS (direct-to-LDS loads write the zeros).
__device__ __forceinline__ i32x4 buffer_rsrc(const void* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  return i32x4{(int)(uint32_t)a, (int)(uint32_t)(a >> 32), bytes, 0x00020000};
}

// One direct-to-LDS load: 64 lanes x 16 bytes from the buffer `rsrc` at byte
// offset voff (per lane) + soff (wave-uniform) into the 1 KiB of LDS at byte
// address lds_addr (wave-uniform; M0 holds it for the load). Written as
// inline assembly so that the compiler does not track these loads: it
// orders a transposing LDS read (ds_read_b64_tr_b16) after every load into
// LDS still in flight (vmcnt(0)), which would stall each MFMA step on the
// loads meant for later blocks. The attention body orders its loads and
// operand reads itself (explicit vmcnt waits before the barriers that
// publish a block). M0 is declared clobbered, so code the compiler places
// after the load never assumes M0 still holds a value it set earlier; M0 is
// a reserved register to the compiler, which warns about naming it, and the
// pragma silences that warning for this function alone.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma_to_lds(i32x4 rsrc, uint32_t lds_addr, int voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc), "s"(soff) : "memory", "m0");
}
// dma_to_lds() of a descriptor that a vector instruction may have written just
// before (v_readfirstlane): a vector-memory instruction may read such a scalar
// register five wait states later, which the compiler does not see to inside
// inline assembly.
__device__ __forceinline__ void dma_to_lds_late(i32x4 rsrc, uint32_t lds_addr, int voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc), "s"(soff) : "memory", "m0");
}
#pragma clang diagnostic pop

// Workgroup barrier that also drains this wave's outstanding LDS operations,
// so LDS writes issued before it are visible to every wave after it. The
// memory clobber keeps the compiler from moving memory accesses across it,
// and the scheduling fences keep arithmetic on its own side too: the
// ping-pong schedule depends on a phase's work not leaking into the next.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// Every LDS read this wave has issued has returned: its slot can be refilled.
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

}  // namespace

#endif  // FA_DEVICE_H
