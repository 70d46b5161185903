// Row quantisation to int8 in units of 8 elements (the definition is in
// quantize.cu), shared by the kernels that quantise on the way in.
#pragma once

#include "internal.cuh"

namespace mtp {

__device__ __forceinline__ void unpack(const __nv_bfloat16* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const __half* p, float* v) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const float* p, float* v) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ float one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float one(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float one(const float* p) { return *p; }

// Elements c .. c + 7 of a row of K (zeros past it).
template <typename T, bool WIDE>
__device__ __forceinline__ void load_unit(const T* row, int c, int K, float* v) {
  if (WIDE) {
    unpack(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < K ? one(row + c + i) : 0.f;
  }
}

// |x| as an integer orders like |x|, infinities above all numbers and NaNs
// above them.
__device__ __forceinline__ uint32_t magnitude(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
  return m;
}

struct RowScale {
  float factor;  // 127 / max, 0 for a row of zeros or with an infinity or NaN
  float pre;     // 2^64 for tiny rows
};

__device__ __forceinline__ RowScale row_scale(uint32_t most) {
  RowScale r;
  const float m = __uint_as_float(most);
  r.pre = m < 0x1p-64f ? 0x1p64f : 1.f;
  r.factor = most == 0 || most >= 0x7f800000u ? 0.f : __fdiv_rn(127.f, m * r.pre);
  return r;
}

// Four codes: adding 1.5 * 2^23 rounds half to even and leaves the integer in
// the low bits, four operations fewer than a conversion at its 16 a cycle and SM.
__device__ __forceinline__ uint32_t four_codes(const float* v, float factor) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], factor), 12582912.f));
  return __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
}

// Codes of N (4 or 8) values, as words; v is changed where the row is tiny.
template <int N>
__device__ __forceinline__ void codes_of(float* v, RowScale r, uint32_t* w) {
  if (r.pre != 1.f)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= r.pre;
#pragma unroll
  for (int i = 0; i < N; i += 4) w[i / 4] = r.factor != 0.f ? four_codes(v + i, r.factor) : 0u;
}

__device__ __forceinline__ void store_unit(int8_t* q, float* v, RowScale r) {
  uint32_t w[2];
  codes_of<8>(v, r, w);
  *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
}

}  // namespace mtp
