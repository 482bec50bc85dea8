// Softmax arithmetic, barrier and tensor-map helpers shared by the tcgen05
// attention kernels (sage_attn.cu, sparse_attn.cu).  Included after
// TB_TRY_WAIT_NO_HINT is chosen.
#pragma once

#include <type_traits>

#include "tb_capi_internal.h"

namespace tb {
namespace {

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(addr, parity)) {
    if (globaltimer_ns() - t0 > TB_WAIT_TIMEOUT_NS) {
      record_device_error(kDevWaitTimeoutDrain);
      return;
    }
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Exact int32 -> float for |v| < 2^22 (|S| <= 127 * 127 * 128 < 2^21).
__device__ __forceinline__ float i2f_exact(int32_t v) {
  return __int_as_float(v + 0x4B400000) - 12582912.0f;
}

__device__ __forceinline__ uint64_t f2_pack(float lo, float hi) {
  return (static_cast<uint64_t>(__float_as_uint(hi)) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float f2_lo(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float f2_hi(uint64_t v) {
  return __uint_as_float(static_cast<uint32_t>(v >> 32));
}
__device__ __forceinline__ uint64_t f2_sub(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// The helpers below keep each key pair in one 64-bit register pair built
// inside a single asm block (mov.b64 {lo, hi}), so the packed f32x2
// arithmetic needs no moves to assemble its operands.

// 2^x of both halves on the MUFU unit.
__device__ __forceinline__ uint64_t ex2_pair(uint64_t x2) {
  uint64_t r;
  asm("{\n\t.reg .f32 a, b;\n\t"
      "mov.b64 {a, b}, %1;\n\t"
      "ex2.approx.ftz.f32 a, a;\n\t"
      "ex2.approx.ftz.f32 b, b;\n\t"
      "mov.b64 %0, {a, b};\n\t}"
      : "=l"(r)
      : "l"(x2));
  return r;
}

template <typename TV>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<TV, __nv_bfloat16>::value) return pack_bf16x2(lo, hi);
  else return pack_f16x2(lo, hi);
}

// Both halves of a pair rounded to TV and packed (low half = even key).
template <typename TV>
__device__ __forceinline__ uint32_t pack_pair(uint64_t p2) {
  uint32_t r;
  if constexpr (std::is_same<TV, __nv_bfloat16>::value) {
    asm("{\n\t.reg .f32 a, b;\n\tmov.b64 {a, b}, %1;\n\tcvt.rn.bf16x2.f32 %0, b, a;\n\t}"
        : "=r"(r)
        : "l"(p2));
  } else {
    asm("{\n\t.reg .f32 a, b;\n\tmov.b64 {a, b}, %1;\n\tcvt.rn.f16x2.f32 %0, b, a;\n\t}"
        : "=r"(r)
        : "l"(p2));
  }
  return r;
}

// Exact floats of a pair of int32 scores (for fma(s, c, -m) with s itself).
__device__ __forceinline__ uint64_t score_pair_f32(uint32_t s0, uint32_t s1) {
  uint64_t r;
  asm("{\n\t.reg .f32 a, b;\n\t"
      "cvt.rn.f32.s32 a, %1;\n\t"
      "cvt.rn.f32.s32 b, %2;\n\t"
      "mov.b64 %0, {a, b};\n\t}"
      : "=l"(r)
      : "r"(s0), "r"(s1));
  return r;
}

void make_map_4d(CUtensorMap* map, CUtensorMapDataType dt, const void* base, int64_t d_elems,
                 int64_t L, int64_t H, int64_t B, int64_t sl, int64_t sh, int64_t sb,
                 int elem_bytes, uint32_t box_inner, uint32_t box_rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d_elems), static_cast<uint64_t>(L),
                            static_cast<uint64_t>(H), static_cast<uint64_t>(B)};
  const uint64_t strides[3] = {static_cast<uint64_t>(sl * elem_bytes),
                               static_cast<uint64_t>(sh * elem_bytes),
                               static_cast<uint64_t>(sb * elem_bytes)};
  const uint32_t box[4] = {box_inner, box_rows, 1, 1};
  encode_tensor_map(map, dt, 4, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace
}  // namespace tb
