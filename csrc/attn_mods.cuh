// What the attention kernels do to a score between Q K^T and the softmax, and which keys a query sees, beyond the plain causal form:
//   score = cap tanh(scale q.k / cap) - slope_h |i - j|       (either part optional)
//   query i sees the keys spans[i] = [lo, hi); key j is seen by the queries key_spans[j]; padding sees and is seen by nothing
// The kernels are instantiated for sets of these bits:
#pragma once
#include "common.cuh"

constexpr int MOD_CAP = 1;
constexpr int MOD_BIAS = 2;

struct AttnMods {
  const int2* spans;    // [B, S] by query (forward) or by key (backward), cut to the row; null: causal
  const int* padding;   // [B, ceil(S / 128)] padded tokens of every 128; null with spans
  const float* slopes;  // [Hq]
  __nv_bfloat16* out_lo;  // forward: what rounding the output to bf16 left over, laid out like it; null: not kept.  D = rowsum(dO * O) wants
                          // it: over documents of 2 to 20 tokens the rounding of O puts dQ and dK 0.5 to 0.33 % off, 0.25 % without it
  float cap_log2;       // cap * log2(e)
  float cap_exp;        // 2 log2(e) scale / cap: tanh of a raw product s is 1 - 2 / (1 + 2^(s * cap_exp))
  float poly_max;       // |s| up to here: cap_log2 * tanh(s * scale / cap) = s * (poly[0] + poly[1] s^2 + ...)
  float poly[4];
};

// The host's part: tanh(x) / x as a polynomial in x^2, fitted for the least relative error (6e-7) on |x| <= 1/2, with the scale and
// the cap multiplied in.  Caps so small that the factors would leave fp32 do without.
inline AttnMods attn_mods(float scale, float softcap, const float* slopes, const int* spans, const int* padding) {
  AttnMods m = {};
  m.spans = reinterpret_cast<const int2*>(spans);
  m.padding = padding;
  m.slopes = slopes;
  if (softcap > 0.f) {
    const double fit[4] = {0.999999456, -0.333263172, 0.131902872, -0.0444019209};
    const double x = (double)scale / (double)softcap, cap = 1.4426950408889634 * (double)softcap;
    m.cap_log2 = (float)cap;
    m.cap_exp = (float)(2.8853900817779268 * x);
    m.poly_max = x < 1000. ? (float)(0.5 / x) : -1.f;
    double power = cap * x;
    for (int i = 0; i < 4; ++i, power *= x * x) m.poly[i] = x < 1000. ? (float)(fit[i] * power) : 0.f;
  }
  return m;
}

// cap * log2(e) * tanh(s * scale / cap) for a raw product s: the polynomial where it holds, else from the exponential (absolute error
// about 2^-22 of the cap; the hardware's tanh is good to 2^-11 relative, 2 % of a probability at a cap of 50).  Both in one:
YF_DEVINL float capped_small(float s, const AttnMods& m) {
  const float z = s * s;
  return s * fmaf(fmaf(fmaf(m.poly[3], z, m.poly[2]), z, m.poly[1]), z, m.poly[0]);
}
YF_DEVINL float capped_any(float s, const AttnMods& m) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + fast_exp2(s * m.cap_exp)));
  return fabsf(s) <= m.poly_max ? capped_small(s, m) : fmaf(-2.f * m.cap_log2, r, m.cap_log2);
}
// N scores in place.  What becomes of a score does not depend on its neighbours.
template <int N>
YF_DEVINL void cap_scores(uint32_t (&s)[N], const AttnMods& m) {
  float far = 0.f;
#pragma unroll
  for (int t = 0; t < N; t += 2) far = fmax3_abs(far, __uint_as_float(s[t]), __uint_as_float(s[t + 1]));
  if (far <= m.poly_max) {
    const uint64_t p0 = f32x2(m.poly[0], m.poly[0]), p1 = f32x2(m.poly[1], m.poly[1]), p2 = f32x2(m.poly[2], m.poly[2]),
                   p3 = f32x2(m.poly[3], m.poly[3]);
#pragma unroll
    for (int t = 0; t < N; t += 2) {  // capped_small, two at a time
      const uint64_t x = f32x2(__uint_as_float(s[t]), __uint_as_float(s[t + 1])), z = mul_f32x2(x, x);
      const float2 y = f32x2_split(mul_f32x2(x, fma_f32x2(fma_f32x2(fma_f32x2(p3, z, p2), z, p1), z, p0)));
      s[t] = __float_as_uint(y.x);
      s[t + 1] = __float_as_uint(y.y);
    }
  } else {
#pragma unroll
    for (int t = 0; t < N; ++t) s[t] = __float_as_uint(capped_any(__uint_as_float(s[t]), m));
  }
}

// N scores in place: s[e] = s[e] * scale - slope |d0 + e|.  `side`: 1 or -1 where d0 + e has that sign for all scores that count (those of the other
// sign are hidden anyway), 0 where both do (prefixes).  The distances are whole numbers and stay exact.
template <int N>
YF_DEVINL void add_bias(uint32_t (&s)[N], float scale, float slope, float d0, int side) {
  const uint64_t scale2 = f32x2(scale, scale);
  if (side != 0) {
    const float f = side > 0 ? -slope : slope;
    const uint64_t f2 = f32x2(f, f), two = f32x2(2.f, 2.f);
    uint64_t d = f32x2(d0, d0 + 1.f);
#pragma unroll
    for (int t = 0; t < N; t += 2) {
      const float2 y = f32x2_split(fma_f32x2(d, f2, mul_f32x2(f32x2(__uint_as_float(s[t]), __uint_as_float(s[t + 1])), scale2)));
      d = add_f32x2(d, two);
      s[t] = __float_as_uint(y.x);
      s[t + 1] = __float_as_uint(y.y);
    }
  } else {
#pragma unroll
    for (int t = 0; t < N; ++t) s[t] = __float_as_uint(fmaf(-slope, fabsf(d0 + (float)t), __uint_as_float(s[t]) * scale));
  }
}

// bits [from, to) of a word, for ends anywhere
YF_DEVINL uint32_t bit_range(int from, int to) {
  const uint32_t below_to = to >= 32 ? 0xffffffffu : to <= 0 ? 0u : (1u << to) - 1u;
  const uint32_t below_from = from >= 32 ? 0xffffffffu : from <= 0 ? 0u : (1u << from) - 1u;
  return below_to & ~below_from;
}

// Zeros in the padded rows of a shared-memory tile of `rows` tokens from `t0` on, two swizzled halves of 128 bytes a row `half_bytes`
// apart: padding is multiplied by probabilities of zero, but may hold anything, infinities and NaN included.  One warp; `spans` of
// the sequence (padding: an empty range).
YF_DEVINL void zero_padded_rows(uint8_t* tile, int half_bytes, int rows, int t0, int S, const int2* spans) {
  for (int r = threadIdx.x & 31; r < rows; r += 32) {
    if (t0 + r >= S) break;  // past the end: zeros already
    const int2 s = __ldg(spans + t0 + r);
    if (s.x < s.y) continue;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(tile + h * half_bytes + r * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
}
