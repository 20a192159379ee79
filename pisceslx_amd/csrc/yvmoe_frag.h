// Register types and conversions that the GEMM translation units share (gfx950 only).
#pragma once

#include <hip/hip_runtime.h>

namespace yvmoe {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));  // staging registers (plain vector)
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Weight loads of the streaming kernel: at decode sizes every weight byte is read by one
// work-group (a few for the shared experts, right after each other), so the loads are
// non-temporal — they do not push the activation rows, which every work-group of a tile
// reads again, out of L2.
__device__ __forceinline__ uint4 nt_load16(const char* p) {
    const u32x4 v = __builtin_nontemporal_load((const u32x4*)p);
    return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ uint2 nt_load8(const char* p) {
    const u32x2 v = __builtin_nontemporal_load((const u32x2*)p);
    return make_uint2(v.x, v.y);
}

// Round-to-nearest-even fp32 -> bf16 pair (v_cvt_pk_bf16_f32), lo in bits 0..15.
__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const bf16x2 v = __builtin_convertvector(f32x2{lo, hi}, bf16x2);
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned short f32_to_bf16_rne(float f) {
    return (unsigned short)(pack_bf16(f, 0.0f) & 0xffffu);
}
__device__ __forceinline__ float bf16_to_f32(unsigned short h) {
    return __uint_as_float((unsigned)h << 16);
}
__device__ __forceinline__ float round_bf16(float f) { return bf16_to_f32(f32_to_bf16_rne(f)); }

union Frag16 {  // 16 bf16 = two MFMA operands
    uint4 u[2];
    bf16x8 v[2];
};

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

}  // namespace
}  // namespace yvmoe
