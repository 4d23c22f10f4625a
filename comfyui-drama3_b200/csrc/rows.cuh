// The row types of the kernels over a model's rows (bfloat16, float16, float32): 16-byte vectors of them to 32-bit values and
// back, and weights that are of the rows' type or float32.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace d3 {

enum { QR_BF16 = 0, QR_F16 = 1, QR_F32 = 2 };

struct QrTensor {  // rows [T, heads, D], the last dimension contiguous
  const void* p;
  long long token, head;  // strides in elements
};

template <int TYPE> struct QrType;
template <> struct QrType<QR_BF16> {
  using T = uint16_t;
  static D3_DEV void get2(uint32_t w, float& lo, float& hi) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
  static D3_DEV uint32_t put2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static D3_DEV float get(uint16_t v) { return bf16_to_f32(v); }
  static D3_DEV uint16_t put(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
};
template <> struct QrType<QR_F16> {
  using T = uint16_t;
  static D3_DEV void get2(uint32_t w, float& lo, float& hi) {
    lo = h_lo(w);
    hi = h_hi(w);
  }
  static D3_DEV uint32_t put2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static D3_DEV float get(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static D3_DEV uint16_t put(float v) { return __half_as_ushort(__float2half_rn(v)); }
};
template <> struct QrType<QR_F32> {
  using T = float;
  static D3_DEV float get(float v) { return v; }
  static D3_DEV float put(float v) { return v; }
};

// The values of a 16-byte vector, and back (rounded to nearest).
template <int TYPE, int VEC>
D3_DEV void qr_unpack(const uint32_t* w, float* x) {
  if constexpr (TYPE == QR_F32) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = __uint_as_float(w[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) QrType<TYPE>::get2(w[e / 2], x[e], x[e + 1]);
  }
}
template <int TYPE, int VEC>
D3_DEV void qr_pack(const float* y, uint32_t* w) {
  if constexpr (TYPE == QR_F32) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) w[e] = __float_as_uint(y[e]);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; e += 2) w[e / 2] = QrType<TYPE>::put2(y[e], y[e + 1]);
  }
}

template <int TYPE> D3_DEV float qr_weight(const void* w, bool f32, float add, int d) {
  if (!w) return 1.0f;
  return (f32 ? ((const float*)w)[d] : QrType<TYPE>::get(((const typename QrType<TYPE>::T*)w)[d])) + add;
}

// A vector's weights: of 16 bytes' columns from d on (aligned, or fp32 and aligned).
template <int TYPE, int VEC>
D3_DEV void qr_weights(const void* w, bool f32, float add, int d, float* out) {
  if (!w) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) out[e] = 1.0f;
    return;
  }
  if (f32) {
#pragma unroll
    for (int e = 0; e < VEC; e += 4) {
      const float4 x = __ldg((const float4*)((const float*)w + d + e));
      out[e] = x.x, out[e + 1] = x.y, out[e + 2] = x.z, out[e + 3] = x.w;
    }
  } else {
    const uint4 x = __ldg((const uint4*)((const typename QrType<TYPE>::T*)w + d));
    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
    qr_unpack<TYPE, VEC>(words, out);
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) out[e] += add;
}

// 1 / (1 + e^-z). Rows of 16 bits take the fast exponential and reciprocal: off by about (2 + |z|) 2^-22 of the value, and half a step of
// bf16 and fp16 is 2^-8 and 2^-11.
template <int TYPE> D3_DEV float row_sigmoid(float z) {
  if constexpr (TYPE == QR_F32) return 1.0f / (1.0f + expf(-z));
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return r;
}

}  // namespace d3
