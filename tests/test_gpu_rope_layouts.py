"""ROPE_AXES and ROPE_AXES_STORE at the ends of their sizes, and over caches of other layouts."""
import numpy as np
import pytest

import scrapgpulibrary_amd as sg
from tests.serving_util import Tensor, free_all, to_bits, values
from tests.test_gpu_rope_axes import close, turned

pytestmark = pytest.mark.gpu


def test_more_threads_than_32_bits_count(hip):
    """Tokens whose pairs of elements are more than 2^31, and whose elements lie up to 8 GiB apart: the first, the
    last and those around the thread of that number."""
    dev, st = hip
    d, t, n = 6, 715827882 + 4099, 500
    buf = dev.alloc(2 * d * t)
    pos = Tensor(hip, sg.I32, (1, 1)).put([[37]])
    x = sg.tdesc(sg.F16, (d, 1, t), buf)
    r = np.random.default_rng(1)
    at = [0, 715827882 - n // 2, t - n]
    old = [to_bits(sg.F16, r.standard_normal((n, 1, d))) for _ in at]
    for i, o in zip(at, old):
        st.write(buf, 2 * d * i, o)
    op, keep = sg.rope_axes_op(x, sg.tdesc(sg.I32, (1, t), pos.buf, nb=[4, 0, 0, 0]), x, d)
    status, why = dev.supported(op)
    assert status == sg.OK, why
    st.execute(op)
    st.sync()
    for i, o in zip(at, old):
        got = st.read(buf, 2 * d * i, o.nbytes).view(np.float16).reshape(o.shape)
        want, mag = turned(values(sg.F16, o), np.full((n, 1), 37, np.int32), d, None, 0, 0, 10000.0, 1.0)
        close(values(sg.F16, got), want, mag, sg.F16)
    free_all(pos)
    buf.free()
