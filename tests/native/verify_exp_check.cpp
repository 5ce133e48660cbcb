// The exp of kv_verify (verify_exp.h) against the C library's, over temperatures and row
// maxima of every size: no weight may be negative, above that of the maximum or, where the
// exact one is below 2^-1000, more than a trace.
#include <cmath>
#include <cstdint>

static int rcp_ulps = 0;
static float rcp_off(float v) {
  float r = 1.0f / v;
  for (int i = 0; i < rcp_ulps; ++i) r = std::nextafterf(r, INFINITY);
  for (int i = 0; i > rcp_ulps; --i) r = std::nextafterf(r, 0.0f);
  return r;
}
#define VERIFY_RCP rcp_off
#include "verify_exp.h"

#include <cstdio>
#include <vector>

static double table[256];
static long failures = 0;

// value of f16 bits
static float half(uint16_t h) {
  const int e = h >> 10 & 31, m = h & 1023;
  const float v = e == 31 ? (m ? NAN : INFINITY) : e ? std::ldexp(1024.0f + m, e - 25) : std::ldexp((float)m, -24);
  return h & 0x8000 ? -v : v;
}
// the f16 nearest to a value, within their range
static float to_half(double v) {
  const int e = v == 0.0 ? -14 : std::ilogb(v) < -14 ? -14 : std::ilogb(v);
  return (float)std::ldexp(std::rint(std::ldexp(v, 10 - e)), e - 10);
}
// the bits of the next f16 below a finite one
static uint16_t below(uint16_t h) { return h == 0 ? 0x8001 : h & 0x8000 ? h + 1 : h - 1; }

static void wrong(const char* what, float top, float heat, float x, double got, double want) {
  if (++failures <= 20)
    std::printf("%s: top %.9g T %.9g x %.9g: %.17g, exact %.17g\n", what, top, heat, x, got, want);
}

// Full 64 bits, 2^-53 each: the unit, its constant and the C library's (x - top) / T round their
// share of an exponent d, with one spare; 16 for table, norm, polynomials and products.
static double tolerance(double d) { return (4 * std::fabs(d) + 16) * 0x1p-53; }

static void check(uint16_t top_bits, float heat) {
  const float top = half(top_bits);
  const VerifyExp w(table, top, verify_unit(heat));
  if (!(w.least < top)) wrong("least", top, heat, w.least, w.least, top);
  auto one = [&](float x) {
    double to;
    const double all = w.some(x, to) * to * w.norm, got = w(x);
    const double d = ((double)x - (double)top) / (double)heat;
    const double exact = std::isnan(x) || x == -INFINITY ? 0.0 : std::exp(d);
    if (exact > 0x1p-990) {
      if (!(std::fabs(got - exact) <= tolerance(d) * exact) || got != all) wrong("weight", top, heat, x, got, exact);
    } else {
      if (!(got >= 0.0 && got <= 0x1p-985)) wrong("small", top, heat, x, got, exact);
      if (!(all >= 0.0 && all <= 0x1p-985)) wrong("sum's", top, heat, x, all, exact);
    }
  };
  one(top);
  uint16_t b = top_bits;
  for (int i = 0; i < 24 && (b & 0x7fff) < 0x7bff; ++i) one(half(b = below(b)));
  for (double d = 1e-7; d < 2e5; d *= 1.7) {  // f16 values at distances of every size
    const float x = to_half(top - d);
    if (x < top && x >= -65504.0f) one(x);
  }
  for (double d = 0.01; d < 2000; d *= 1.3) {  // and at exponents of every size
    const float x = to_half(top - d * heat);
    if (x < top && x >= -65504.0f) one(x);
  }
  one(-65504.0f);
  one(-INFINITY);
  one(NAN);
}

int main() {
  for (int n = 0; n < 256; ++n) table[n] = std::exp2(n / 256.0);
  std::vector<float> heats;
  for (double t = 1e-6; t <= 2e4; t *= 1.37) heats.push_back((float)t);
  for (double t : {1e-45, 1e-38, 1e-30, 1e-20, 1e-12, 1e6, 1e12, 1e20, 1e25, 1e30, 1e35, 1e36, 3.4e38,
                   (double)INFINITY}) heats.push_back((float)t);
  for (rcp_ulps = -1; rcp_ulps <= 1; ++rcp_ulps)
    for (float heat : heats)
      for (int sign = 0; sign < 2; ++sign)
        for (int h = 0; h < 0x7c00; h += h < 40 || h % 1024 < 3 || h % 1024 > 1020 ? 1 : 41)
          check((uint16_t)(h | sign << 15), heat);
  std::printf("%ld wrong\n", failures);
  return failures != 0;
}
