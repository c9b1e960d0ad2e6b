// Eight elements of bf16, fp16 or fp32 to and from floats by 16-byte accesses.
#pragma once
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

// eight elements as they lie in memory, and as floats
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
YF_DEVINL Raw8<T> load_raw8(const void* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.v[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
// eight floats as four pairs, for instructions that take two at a time
struct F8 {
  uint64_t p[4];
};
YF_DEVINL F8 splat8(float f) {
  const uint64_t v = f32x2(f, f);
  return {{v, v, v, v}};
}
YF_DEVINL F8 mul8(const F8& a, const F8& b) {
  return {{mul_f32x2(a.p[0], b.p[0]), mul_f32x2(a.p[1], b.p[1]), mul_f32x2(a.p[2], b.p[2]), mul_f32x2(a.p[3], b.p[3])}};
}
YF_DEVINL F8 mul8(const F8& a, float f) { return mul8(a, splat8(f)); }
YF_DEVINL F8 fma8(const F8& a, const F8& b, const F8& c) {
  return {{fma_f32x2(a.p[0], b.p[0], c.p[0]), fma_f32x2(a.p[1], b.p[1], c.p[1]), fma_f32x2(a.p[2], b.p[2], c.p[2]), fma_f32x2(a.p[3], b.p[3], c.p[3])}};
}
YF_DEVINL F8 fma8(const F8& a, float f, const F8& c) { return fma8(a, splat8(f), c); }
// sum += a . b, two partial sums
YF_DEVINL void dot8(uint64_t& sum, const F8& a, const F8& b) {
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = fma_f32x2(a.p[i], b.p[i], sum);
}
YF_DEVINL float both(uint64_t sum) {
  const float2 t = f32x2_split(sum);
  return t.x + t.y;
}
template <typename T>
YF_DEVINL F8 unpack8(const Raw8<T>& r) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
  F8 f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (sizeof(T) == 4) {
      f.p[i] = f32x2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else if (std::is_same<T, __half>::value) {
      const float2 t = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f.p[i] = f32x2(t.x, t.y);
    } else {
      f.p[i] = f32x2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  return f;
}
template <typename T>
YF_DEVINL void store8(T* p, const F8& f) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = f32x2_split(f.p[i]);
    if (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(t.x);
      w[2 * i + 1] = __float_as_uint(t.y);
    } else if (std::is_same<T, __half>::value) {
      const __half2 z = __floats2half2_rn(t.x, t.y);
      w[i] = *reinterpret_cast<const uint32_t*>(&z);
    } else {
      w[i] = pack_bf16x2(t.x, t.y);
    }
  }
  reinterpret_cast<uint4*>(p)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
