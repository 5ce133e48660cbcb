// exp of the verification's logits (pages_kernels.hip); plain enough to be tested on the host.
#ifndef QWEN3_VERIFY_EXP_H
#define QWEN3_VERIFY_EXP_H

#include <stdint.h>

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)
#define VERIFY_FN __host__ __device__ __forceinline__
#else
#define VERIFY_FN inline
#endif

// 1 / v to a unit in the last place (on the host as VERIFY_RCP says, where it is defined)
VERIFY_FN float verify_rcp(float v) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_amdgcn_rcpf(v);
#elif defined(VERIFY_RCP)
  return VERIFY_RCP(v);
#else
  return 1.0f / v;
#endif
}

// exp((x - top) / T), 0 below 2^-996 and for a NaN, with unit = 256 log2(e) / T: 2^(1/256)
// to the power x unit - C, C = rint(top unit), times norm, which makes up for C.  y = x unit +
// (1.5 2^52 - C) holds the nearest integer's n = rint(x unit) - C in its low bits, y less
// that constant is rint(x unit), both exact, so that the rest has the rounding of one fma; n goes
// into the exponent by an addition (f64 roundings, conversions and ldexp have a fraction
// of the rate).  x becomes an f64 by a shift, 2^896 too small, which the unit makes up
// for.  table[n] = 2^(n / 256), n < 256.  For a top of +inf: of 0.
struct VerifyExp {
  const double* table;
  double unit, base, norm;
  double c1, c2, c3, c4;
  float least;  // x of 2^-996, about
  bool far;
  // unit_of_heat: verify_unit(T)
  VERIFY_FN VerifyExp(const double* table, float top_of, double unit_of_heat)
      : table(table), far(top_of == __builtin_inff()) {
    const float at = far ? 0.0f : top_of;
    // An f16 below `top` is further from it than |top| 2^-12, and 2^-24 at least: a larger unit
    // only takes 2^-996 to something smaller.
    unit = __builtin_fmin(
        far ? 1.0 : unit_of_heat,
        (double)(255000.0f * verify_rcp(__builtin_fmaxf(__builtin_fabsf(at) * 0x1p-12f, 0x1p-24f))));
    // Below the top by 2^-12 of it at least, so it is less, whatever its sign.  The shift in some()
    // moves it towards 0 by less than 2^-20 of itself: of 255000 steps of 2^(1/256) by 1000 at
    // most, and 1023 2^8 are what the exponent holds.
    least = at - 255000.0f * verify_rcp((float)unit);
    c1 = 0x1.62e42fefa39efp-9;
    c2 = 0x1.ebfbdff82c58fp-19;
    c3 = 0x1.c6b08d704a0c0p-29;
    c4 = 0x1.3b2ab6fba4e77p-39;
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+s"(c1), "+s"(c2), "+s"(c3), "+s"(c4));
#endif
    const double magic = 6755399441055744.0, z = (double)at * unit, c = (z + magic) - magic;
    base = magic - c;
    norm = poly(-__builtin_fma((double)at, unit, -c));
    unit *= 0x1p896;
  }
  VERIFY_FN double poly(double r) const {
    return __builtin_fma(
        __builtin_fma(__builtin_fma(__builtin_fma(c4, r, c3), r, c2), r, c1), r, 1.0);
  }
  // The same without norm and with 2^-996, about, in the place of 0: a product, of which
  // `to` is the second factor.  x: an f16's value.
  VERIFY_FN double some(float x, double& to) const {
    const uint32_t bits =
        (uint32_t)((int32_t)__builtin_bit_cast(uint32_t, __builtin_fmaxf(x, least)) >> 3) & 0x8fffffffu;
    const double v = __builtin_bit_cast(double, (uint64_t)bits << 32);
    const double y = __builtin_fma(v, unit, base);
    const uint32_t n = (uint32_t)__builtin_bit_cast(uint64_t, y);
    const uint64_t b = __builtin_bit_cast(uint64_t, table[n & 255]);
    uint32_t hi = (uint32_t)(b >> 32) + ((n & ~255u) << 12);
#if defined(__HIP_DEVICE_COMPILE__)
    asm("" : "+v"(hi));  // (or the compiler adds in 64 bits)
#endif
    to = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)b);
    return poly(__builtin_fma(v, unit, -(y - base)));
  }
  VERIFY_FN double raw(float x) const {  // without norm
    double to;
    const double w = some(x, to) * to;
    return x > least ? w : 0.0;
  }
  VERIFY_FN double operator()(float x) const { return raw(x) * norm; }
};

// 256 log2(e) / T; any where the maximum takes all
VERIFY_FN double verify_unit(float heat) {
  return heat > 0.0f ? __builtin_fmax(369.3299304675746 / (double)heat, 1e-30) : 1.0;
}

#endif
