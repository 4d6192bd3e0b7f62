// Element types of the sequence operators: a value of any of them is widened to f32 when it is loaded and rounded once, to nearest even, when it is stored (one
// conversion instruction on gfx950: v_cvt_pk_bf16_f32, v_cvt_f16_f32), and the two fast transcendental instructions.  The host emulation has its own copy of this file.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>

namespace half_types {

__device__ __forceinline__ float widen_bf16(uint16_t u) { return __uint_as_float((unsigned)u << 16); }
__device__ __forceinline__ uint16_t round_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ float widen_f16(uint16_t u) { return (float)__builtin_bit_cast(_Float16, u); }
__device__ __forceinline__ uint16_t round_f16(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }      // v_exp_f32: 1 ulp, 0 below -126
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }        // v_rcp_f32: 1 ulp
__device__ __forceinline__ float sqrt_fast(float x) { return __builtin_amdgcn_sqrtf(x); }      // v_sqrt_f32: 1 ulp

// accesses that leave the caches to others (macros: a template parameter would lose the alignment of the pointer's type)
#define APX_PASSING(p) __builtin_nontemporal_load(p)
#define APX_PASS(p, x) __builtin_nontemporal_store(x, p)
// the value of the first lane, for what is the same in all lanes of a wave (a scalar register then)
__device__ __forceinline__ int wave_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// an address in global memory that is the same in all lanes, kept in scalar registers (the compiler would rather add a lane's offset to it first and have 64-bit vector additions
// from then on)
#define APX_GLOBAL __attribute__((address_space(1)))
template <class T> __device__ __forceinline__ APX_GLOBAL T* wave_address(T* p) { APX_GLOBAL T* q = (APX_GLOBAL T*)p; asm("" : "+s"(q)); return q; }
// a lane's 32-bit offset, made where it is used (widened to 64 bits outside a loop it would take the vector additions again)
__device__ __forceinline__ unsigned lane_offset(unsigned x) { asm("" : "+v"(x)); return x; }

}  // namespace half_types
