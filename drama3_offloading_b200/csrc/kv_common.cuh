// What the paged K/V cache's kernels share: the element types, one row of a
// head spread over a group of lanes, and the e4m3 form of a cached row.
#pragma once

#include "d3_common.cuh"

#include <cuda_fp16.h>

namespace d3 {

// one 16-bit element type: bf16 or fp16
template <typename T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float2 to_f2(uint32_t w) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
  }
  static __device__ __forceinline__ uint32_t from_f2(float a, float b) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float2 to_f2(uint32_t w) {
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ uint32_t from_f2(float a, float b) {
    const __half2 p = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
};

// 8 elements <-> 16 bytes
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Elem<T>::to_f2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(Elem<T>::from_f2(x[0], x[1]), Elem<T>::from_f2(x[2], x[3]),
                    Elem<T>::from_f2(x[4], x[5]), Elem<T>::from_f2(x[6], x[7]));
}

// two e4m3 codes of (a, b): round to nearest even, saturating at +-448
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
// two codes -> fp16 (exact: every e4m3 value is an fp16 value)
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_f2(uint16_t c) {
  const uint32_t h = e4m3x2_to_h2(c);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// a pair of fp32 operations in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b) {   // (x, y) * a + b
  asm("{\n\t.reg .b64 v, m, n;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %2};\n\tmov.b64 n, {%3, %3};\n\t"
      "fma.rn.f32x2 v, v, m, n;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float n) {   // (x * a + n, y * b + n)
  asm("{\n\t.reg .b64 v, m, n;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %3};\n\tmov.b64 n, {%4, %4};\n\t"
      "fma.rn.f32x2 v, v, m, n;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(n));
}
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {   // (x * a, y * b)
  asm("{\n\t.reg .b64 v, m;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %3};\n\t"
      "mul.rn.f32x2 v, v, m;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {   // (x + a, y + b)
  asm("{\n\t.reg .b64 v, m;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %3};\n\t"
      "add.rn.f32x2 v, v, m;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void fma2v(float& x, float& y, float a, float b, float c, float e) {   // (a * b + x, c * e + y)
  asm("{\n\t.reg .b64 v, m, n;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 m, {%2, %4};\n\tmov.b64 n, {%3, %5};\n\t"
      "fma.rn.f32x2 v, m, n, v;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b), "f"(c), "f"(e));
}

constexpr float kE4m3Max = 448.f;

// Reads of what an earlier launch wrote go through L2 (__ldcg): under
// programmatic launch a kernel may share an SM with an earlier reader of the
// same memory, whose L1 lines are older than the write.

// an index read as 4 or 8 bytes
__device__ __forceinline__ long long load_index(const void* p, int bytes, long long i) {
  return bytes == 8 ? __ldcg(static_cast<const long long*>(p) + i)
                    : (long long)__ldcg(static_cast<const int*>(p) + i);
}

// host: the checks every entry point makes of a cache descriptor
int check_kv_cache(const d3_kv_cache* c, const char* who);

}  // namespace d3
