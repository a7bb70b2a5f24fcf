// The 8-bit code of a value next to a border between two, in plain C++ (tests/native/codes.cpp compiles it alone).
#pragma once

namespace came8 {

// The code nearest to 127 p / a, ties to even, where x is that quotient off by less than 1e-4 and c the whole number nearest to x.
// p and a > 0 are products of two float32 numbers, exact in 64 bits; 127 p is not (55 bits), nor does the quotient of two such
// numbers tell a tie from what is next to one.  So 127 p is compared with a times the border on x's side of c: both products
// as a rounded part and what is left (a fused multiply-add, exact).  Near the border the rounded parts are within a factor of 2,
// and what is left of both are a few units of bits at most 2^8 apart: both differences are exact, and their sum has the sign of the
// whole; elsewhere no rounding changes it.
template <typename F, typename D>
constexpr F nearest_code(F x, F c, D p, D a) {
  const D border = D(c) + (x > c ? D(0.5) : D(-0.5));
  const D u = D(127.0) * p, v = border * a;
  const D above = (u - v) + (__builtin_fma(D(127.0), p, -u) - __builtin_fma(border, a, -v));
  const int low = int(border - D(0.5));
  return F(above > D(0.0) || (above == D(0.0) && (low & 1) != 0) ? low + 1 : low);
}

}  // namespace came8
