"""The arithmetic of the routing's exponential, step by step in exact numbers rounded to 64 bits: within a few
2^-53 of exp, which the series up to r^11 is not."""
import math
import random
from fractions import Fraction as F

LN2 = F(693147180559945309417232121458176568, 10 ** 36)
HI = F(math.floor(LN2 * 2 ** 32), 2 ** 32)
LO = F(float(LN2 - HI))


def fma(a, b, c):
    return F(float(a * b + c))


def exp(x):
    """exp of a fraction, to 2^-100."""
    s = t = F(1)
    for n in range(1, 40):
        t = t * x / n
        s += t
    return s


def error(v, terms):
    """Relative error of the series up to r^terms at v, in 2^-53."""
    n = round(v * 1.4426950408889634)
    r = fma(F(-n), LO, fma(F(-n), HI, F(v)))
    p = F(1 / math.factorial(terms))
    for i in range(terms - 1, 1, -1):
        p = fma(p, r, F(1 / math.factorial(i)))
    p = fma(fma(p, r, F(1)), r, F(1))
    want = exp(F(v) - n * LN2)
    return float(abs(p - want) / want) * 2 ** 53


def test_exponential():
    rng = random.Random(1)
    values = [0.0, 1e-300, 0.3465, -0.3465, 0.3466, 700.0, -700.0, 1000 * math.log(2)]
    values += [rng.uniform(-1, 1) for _ in range(100)] + [rng.uniform(-700, 700) for _ in range(100)]
    # r is rounded once (at |r| < 0.35), then the last two steps: at most 0.35 + 0.35 * 1.42 / 0.71 + 1.42 half steps
    # of what is 0.7 or more, and n times the part of ln 2 that a long double does not hold
    assert max(error(v, 13) for v in values) < 3
    assert error(-0.3465, 11) > 50
