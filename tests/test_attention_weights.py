"""The bound of attention_weights, on the CPU: it holds for weights of as many terms as it says and not for
fewer, so that a kernel which lost a term would not pass."""
import numpy as np
import pytest

import scrapgpulibrary_amd as sg
from tests import attention_weights as aw
from tests.serving_util import to_bits, values


def model(dtype, out, terms, delta, v):
    w = np.exp(-values(dtype, delta)).astype(np.float32).astype(np.float64)
    held = aw.in_terms(dtype, terms, w)
    total = 1 + (held if terms == 1 else w)
    return values(out, to_bits(out, held[:, None] * values(dtype, v) / total[:, None]))


@pytest.mark.parametrize("dtype,out,terms", [(sg.F16, sg.F16, 2), (sg.F16, sg.F32, 2), (sg.BF16, sg.BF16, 2), (sg.BF16, sg.F32, 3), (sg.BF16, sg.F32, 2), (sg.F16, sg.F16, 1), (sg.BF16, sg.BF16, 1)])
def test_bound_tells_the_terms(dtype, out, terms):
    delta, v = aw.inputs(dtype, 64, 1)
    want = aw.result(dtype, delta, v)
    assert np.all(np.abs(model(dtype, out, terms, delta, v) - want) <= aw.bound(dtype, out, terms, want))
    if terms > 1:
        over = np.abs(model(dtype, out, terms - 1, delta, v) - want) > aw.bound(dtype, out, terms, want)
        assert np.mean(over) > 0.01, np.mean(over)
