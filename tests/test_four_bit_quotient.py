"""The four-bit quantiser's division (``quotient`` of ``ring4.h``) restated on the CPU.

A reciprocal within one unit of the last place and one Newton step give the correctly rounded n / d where d has at
most 11 significant bits, as the divisors there have (15, and scales rounded to bf16 or fp16). With t = fl(n r) the
residual n - t d is exact, and t + (n - t d) r lies within 2^-46 of n / d (relative: the step squares an error of
2^-23) before its one rounding. A midpoint m of two floats has 25 bits; n - m d is a whole multiple of the unit of
m d, and never 0 (m d has more than 24 bits, n has 24), so n / d keeps 2^-36 away from every midpoint and the
rounding cannot fall on the wrong side.
"""

from __future__ import annotations

import numpy as np
import pytest

F, X = np.float32, np.longdouble


def _quotient(n, d, r):
    t = n * r  # float32, one rounding
    residual = X(n) - X(t) * X(d)  # at most 35 bits: exact in 64
    assert np.array_equal(residual, X(F(residual)))
    return F(X(t) + residual * X(r))


def _numerators(d, g):
    """Floats spread over two binades, and for every divisor those whose quotients lie nearest to midpoints."""
    wide = (g.integers(2**23, 2**24, 64).astype(F) * F(2.0**-23))[None, :].repeat(len(d), 0)
    mid = (2 * g.integers(2**24, 2**25, (len(d), 64)) + 1).astype(X) * X(2.0**-26)  # 26 bits: any binade of the quotient
    near = F(mid * X(d)[:, None])
    return np.concatenate([wide, 2 * wide, near, np.nextafter(near, F(0)), np.nextafter(near, F(8))], 1)


@pytest.mark.parametrize("bits", [4, 8, 11])
@pytest.mark.parametrize("ulp", [-1, 0, 1])
def test_the_quotient_is_correctly_rounded(bits, ulp):
    assert np.finfo(X).nmant >= 63
    whole = np.array([15]) if bits == 4 else np.arange(2**(bits - 1), 2**bits)
    d = whole.astype(F) * F(2.0 ** (1 - bits))
    r = F(1) / d
    r = r if ulp == 0 else np.nextafter(r, F(0) if ulp < 0 else F(4))
    n = _numerators(d, np.random.default_rng(bits))
    assert np.array_equal(_quotient(n, d[:, None], r[:, None]), n / d[:, None])
