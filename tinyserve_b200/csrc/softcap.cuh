// tanh(x) = x P(x^2) for |x| <= TANH_SMALL, P of degree four: relative error 7e-7, on the multiply-add units.  Away from 0, 1 - 2 / (e^(2x) + 1) has an
// error of some 2^-23 of 1, which a soft cap multiplies by the cap: scores far below their cap lose everything in it.
#pragma once

constexpr float TANH_SMALL = 0.75f;
constexpr float TANH_P0 = 9.999994059e-01f, TANH_P1 = -3.332809286e-01f, TANH_P2 = 1.325760377e-01f, TANH_P3 = -5.001763221e-02f, TANH_P4 = 1.289561170e-02f;
