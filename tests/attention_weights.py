"""Softmax weights of two keys whose scores are exact, and how far a result may be off by them.

q is one-hot, so a score is one product of representable numbers; the values are 0 and v. The result
v w / (1 + w), w = e^-delta, then holds one weight and little else. In units of 2^-24 of it: the exponential 2, its
argument's factor and rounding at most 5 (delta below 2, F16 lifted by 2^8), the sum 2, the products of up to
three terms 6, the join of four waves 4, division and last product 2, of which each is counted in full: 24
leaves some. On top the weight's own rounding: to one term of F16 (cut: 2^-10) or BF16 (2^-8), to two (2^-21,
cut; 2^-16), to three of BF16 (2^-24)."""
import numpy as np

import scrapgpulibrary_amd as sg
from tests.serving_util import U, to_bits, values

WEIGHT = {sg.F16: {1: 2.0**-10, 2: 2.0**-21}, sg.BF16: {1: 2.0**-8, 2: 2.0**-16, 3: 2.0**-24}}


def inputs(dtype, n, seed):
    """delta [n] and v [n, 64] of n requests, as the type holds them (bits)."""
    r = np.random.default_rng(seed)
    return to_bits(dtype, r.uniform(0, 2, n)), to_bits(dtype, r.standard_normal((n, 64)))


def result(dtype, delta, v):
    w = np.exp(-values(dtype, delta))[:, None]
    return values(dtype, v) * w / (1 + w)


def bound(dtype, out, terms, want):
    rel = WEIGHT[dtype][terms] + 24 * 2.0**-24 + (U[out] if out != sg.F32 else 0)
    return rel * np.abs(want) + (2.0**-25 if out == sg.F16 else 0)


def in_terms(dtype, terms, w):
    """f32 weights as the kernels may hold them: cut to the type's bits, the rest in the next term, the last one
    rounded (F16: cut)."""
    bits = 11 if dtype == sg.F16 else 8
    held, rest = np.zeros_like(w), w.astype(np.float64)
    for i in range(terms):
        m, e = np.frexp(rest)
        cut = np.ldexp(np.trunc(m * 2**bits) if dtype == sg.F16 or i + 1 < terms else np.rint(m * 2**bits), e - bits)
        held, rest = held + cut, rest - cut
    return held
