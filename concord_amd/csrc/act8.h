// act8.h -- activations in 8 bits, and the functions whose input is kept so.
//
// 32 adjacent values of a row (a block; a row's last one may be shorter) share a
// step 2^e, the smallest power of two with max|x| <= 127 2^e and e >= -126:
//   code = x 2^-e rounded half to even, -127 .. 127;   exponent byte = e + 127 (1 .. 249)
//   value = code 2^e, limited to the type's largest finite number
// Scaling by a power of two is exact, so the codes have one definition whatever
// computes them, each value is off by at most half a step (less than 1/127 of the
// block's largest; 2^-127 where the step is held at 2^-126, in fp32 and bf16 blocks of
// nothing above 127 2^-127), and one significant byte fits bf16 and fp16 without a further
// rounding.
// A block that holds an infinity or NaN has exponent byte 255 and codes 0: all of it
// reads back as NaN.
#pragma once
#include "elem.h"

namespace concord {

constexpr int kBlock8 = 32;
constexpr uint32_t kBad8 = 255;

// exponent byte of a block whose largest magnitude has these bits: the exponent
// less 6, one more where the mantissa is above 127 / 64
CONCORD_DEV uint32_t exponent8(uint32_t top) {
  return top >= 0x7F800000u ? kBad8 : max((int)((top + 0x1FFFFu) >> 23) - 6, 1);
}
// 1 / step (byte 255: not used)
CONCORD_DEV float inverse_step8(uint32_t e8) { return __uint_as_float((254u - e8) << 23); }
CONCORD_DEV float step8(uint32_t e8) { return __uint_as_float(e8 << 23); }   // (byte 255: infinity)

// the low byte of 1.5 2^23 + x / step is the code: the sum rounds half to even
CONCORD_DEV uint32_t code8(float x, float inv) { return __float_as_uint(__builtin_fmaf(x, inv, 12582912.0f)); }

// four codes, in order
CONCORD_DEV uint32_t codes8(const float* x, float inv) {
  const uint32_t lo = __builtin_amdgcn_perm(code8(x[1], inv), code8(x[0], inv), 0x0C0C0400u);
  const uint32_t hi = __builtin_amdgcn_perm(code8(x[3], inv), code8(x[2], inv), 0x04000C0Cu);
  return lo | hi;
}

template <class T>
struct Largest;   // the type's largest finite number, and the exponent byte from which 128 steps exceed it
template <>
struct Largest<float> {
  static constexpr float value = 3.4028234663852886e38f;
  static constexpr uint32_t e8 = 248;
};
template <>
struct Largest<BF16> {
  static constexpr float value = 3.3895313892515355e38f;
  static constexpr uint32_t e8 = 248;
};
template <>
struct Largest<_Float16> {
  static constexpr float value = 65504.0f;
  static constexpr uint32_t e8 = 136;
};

// Four codes as values of T; NaN for a block of byte 255.  u = code + 128 is a byte
// without sign, which one instruction takes from its word, and u step - 128 step rounds
// nothing away.  Where 128 steps pass the largest number (a rare block, and byte 255,
// whose step is infinite) the product is formed from the code itself: 0 times infinity is
// NaN, and what exceeds T is limited.
template <class T>
CONCORD_DEV void values8(float* v, uint32_t w, uint32_t e8) {
  const float step = step8(e8), less = -128.0f * step;
  const uint32_t u = w ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf((float)((u >> (8 * i)) & 0xFFu), step, less);
  if (e8 >= Largest<T>::e8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = (float)(int)__builtin_amdgcn_sbfe(w, 8 * i, 8) * step;
      v[i] = fabsf(x) > Largest<T>::value ? copysignf(Largest<T>::value, x) : x;
    }
  }
}

// ---- gelu ---------------------------------------------------------------------
// With a = |x|, the lower tail of the normal distribution is Phi(-a) = exp(-a^2 / 2) q(a);
// q, half of the scaled complementary error function of a / sqrt(2), is t P(t), t = 1 /
// (1 + c a), P a polynomial fitted to q's values for a up to 17.  So the tail keeps its
// digits far out, where 1 + erf would have lost every one, and
//   x Phi(x) = max(x, 0) - a tail,   Phi(x) = tail or 1 - tail.
// Past a = 16 both are at their limits, and a stands at 16.
//   FINE (fp32): degree 8, relative error 5.2e-8 with its coefficients as they stand (at
// a = 0, where it is largest), and the exponent's rounding taken back with its remainder:
// 4e-7 of the tail in all.
//   else (bf16, fp16): degree 5, 8.8e-6, a 28th of half a step of fp16, and the
// exponent's rounding (at most a^2 2^-24 of the tail) stays.  The kernels are bound by their
// instructions as much as by memory.
template <bool FINE>
struct Gelu {
  // tail = Phi(-a) and e = exp(-a^2 / 2), a = min(|x|, 16)
  static CONCORD_DEV void parts(float a, float& tail, float& e) {
    const float s = a * a, y = s * -0.72134752f;
    e = __builtin_amdgcn_exp2f(y);
    if constexpr (FINE) {
      const float rest = __builtin_fmaf(a, a, -s);
      const float lost = __builtin_fmaf(s, -0.72134752f, -y) + __builtin_fmaf(rest, -0.72134752f, s * -9.6298149e-9f);
      e = __builtin_fmaf(e, lost * 0.69314718f, e);
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f));
      float p = __builtin_fmaf(-0.029165321961045265f, t, 0.14406773447990417f);
      p = __builtin_fmaf(p, t, -0.2559165060520172f);
      p = __builtin_fmaf(p, t, 0.1594100296497345f);
      p = __builtin_fmaf(p, t, -0.02327592857182026f);
      p = __builtin_fmaf(p, t, 0.10558006167411804f);
      p = __builtin_fmaf(p, t, 0.11981412768363953f);
      p = __builtin_fmaf(p, t, 0.13986453413963318f);
      p = __builtin_fmaf(p, t, 0.13962124288082123f);
      tail = p * t * e;
    } else {
      const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.46f, a, 1.0f));
      float p = __builtin_fmaf(0.07207910716533661f, t, -0.23614893853664398f);
      p = __builtin_fmaf(p, t, 0.1774096041917801f);
      p = __builtin_fmaf(p, t, 0.11628451943397522f);
      p = __builtin_fmaf(p, t, 0.18703024089336395f);
      p = __builtin_fmaf(p, t, 0.18334899842739105f);
      tail = p * t * e;
    }
  }
  // (0.5 x + 0.5 |x| rather than a maximum: it keeps a NaN)
  static CONCORD_DEV float value(float x) {
    float tail, e;
    const float a = fminf(fabsf(x), 16.0f);
    parts(a, tail, e);
    return __builtin_fmaf(-a, tail, __builtin_fmaf(fabsf(x), 0.5f, 0.5f * x));
  }
  static CONCORD_DEV float slope(float x) {
    float tail, e;
    parts(fminf(fabsf(x), 16.0f), tail, e);
    return __builtin_fmaf(x * 0.3989422804f, e, x < 0.0f ? tail : 1.0f - tail);
  }
  static CONCORD_DEV void both(float x, float& v, float& d) {
    float tail, e;
    const float a = fminf(fabsf(x), 16.0f);
    parts(a, tail, e);
    v = __builtin_fmaf(-a, tail, __builtin_fmaf(fabsf(x), 0.5f, 0.5f * x));
    d = __builtin_fmaf(x * 0.3989422804f, e, x < 0.0f ? tail : 1.0f - tail);
  }
};

// x (1 + tanh(u)) / 2 = x / (1 + exp(-2 u)), u = sqrt(2 / pi) (x + 0.044715 x^3).
// Past |x| = 16 the sigmoid is 0 or 1 to the last bit, and x^3 would overflow.
template <bool FINE>
struct GeluTanh {
  static CONCORD_DEV float limit(float x) { return fabsf(x) > 16.0f ? copysignf(16.0f, x) : x; }   // (NaN stays)
  // e = exp(-2 u), sig = 1 / (1 + e)
  static CONCORD_DEV void parts(float x, float& e, float& sig) {
    e = __builtin_amdgcn_exp2f(x * __builtin_fmaf(x * x, -0.1029432397f, -2.302208198f));
    sig = __builtin_amdgcn_rcpf(1.0f + e);
  }
  static CONCORD_DEV float value(float x) {
    float e, sig;
    parts(limit(x), e, sig);
    return x * sig;
  }
  static CONCORD_DEV void both(float x, float& v, float& d) {
    float e, sig;
    const float c = limit(x);
    parts(c, e, sig);
    v = x * sig;
    // sig + x sig (1 - sig) 2 u'; 1 - sig = e sig keeps its digits where sig is near 1
    const float rest = c > 0.0f ? e * sig : 1.0f - sig;
    d = __builtin_fmaf(c * sig * rest, __builtin_fmaf(c * c, 0.2140644488f, 1.5957691216f), sig);
  }
  static CONCORD_DEV float slope(float x) {
    float v, d;
    both(x, v, d);
    return d;
  }
};

}  // namespace concord
