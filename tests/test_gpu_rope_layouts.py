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


@pytest.mark.parametrize("layout", ["pages", "heads", "places"])
def test_k_and_v_in_one_buffer(hip, layout):
    """k and v in turn in one buffer: page by page, head by head inside a page, place by place inside a head, gaps
    between them untouched. What really overlaps is refused."""
    dev, st = hip
    r = np.random.default_rng(3)
    t, hq, hk, d, page, pages, gap = 40, 4, 2, 64, 16, 5, 16
    order = {"pages": "pkhsd", "heads": "phksd", "places": "phskd"}[layout]
    size = {"p": pages, "k": 2, "h": hk, "s": page, "d": d}
    whole = Tensor(hip, sg.F16, [size[c] for c in order], [gap if c in "ks" else 0 for c in order]).put(0)
    old = whole.get()
    step = dict(zip(order, whole.strides))
    cache = lambda at: sg.tdesc(sg.F16, (d, page, hk, pages), whole.buf, offset=at, nb=[2, step["s"], step["h"], step["p"]])  # noqa: E731
    x = to_bits(sg.F32, r.standard_normal((t, hq + 2 * hk, d)))
    parts = np.split(x, [hq, hq + hk], axis=1)
    q, k, v = (Tensor(hip, sg.F32, p.shape).put(p) for p in parts)
    y = Tensor(hip, sg.F16, (t, hq, d)).fill()
    pos, slots = r.integers(0, 5000, (t, 1)).astype(np.int32), r.permutation(pages * page)[:t].astype(np.int32)
    tp, ts = Tensor(hip, sg.I32, pos.shape).put(pos), Tensor(hip, sg.I32, (t,)).put(slots)

    def op(at):
        return sg.rope_axes_store_op(q.desc, k.desc, v.desc, tp.desc, ts.desc, y.desc, cache(0), cache(at), d)

    status, why = dev.supported(op(step["k"])[0])
    assert status == sg.OK, why
    st.execute(op(step["k"])[0])
    st.sync()
    got = whole.get()
    kc, vc = (np.transpose(c, [order.replace("k", "").index(a) for a in "phsd"]) for c in np.moveaxis(got, order.index("k"), 0))
    want, mag = turned(values(sg.F32, parts[1]), pos, d, None, 0, 0, 10000.0, 1.0)
    left = np.ones((pages, page), bool)
    for i, s in enumerate(slots):
        close(values(sg.F16, kc[s // page, :, s % page]), want[i], mag[i], sg.F16)
        assert np.array_equal(vc[s // page, :, s % page], to_bits(sg.F16, parts[2][i]))
        left[s // page, s % page] = False
    assert not np.swapaxes(kc, 1, 2)[left].any() and not np.swapaxes(vc, 1, 2)[left].any()
    assert whole.untouched()
    for at in (0, 16, step["k"] - 48, step["p"], step["p"] + 16, step["h"], step["s"]):
        status, why = dev.supported(op(at)[0])
        assert status == sg.INVALID_ARGUMENT and "overlap" in why, at
    free_all(whole, q, k, v, y, tp, ts)


@pytest.mark.parametrize("axes,d", [(2, 80), (2, 64), (4, 64)])
@pytest.mark.parametrize("adjacent", [0, 1])
def test_frequencies_that_start_anew_on_each_axis(hip, axes, d, adjacent):
    """An image encoder's rotation: each of `axes` equal shares of the pairs has the frequencies theta^(-2j / (d / axes)) of
    its own axis' position. By this op: base theta^axes, and the positions of axis a times theta^a."""
    theta, t, heads = 100, 50, 3
    r = np.random.default_rng(axes)
    x, pos = to_bits(sg.F32, r.standard_normal((t, heads, d))), r.integers(0, 20 if axes == 4 else 73, (t, axes))
    tx, y = Tensor(hip, sg.F32, x.shape).put(x), Tensor(hip, sg.F32, x.shape).fill()
    tp = Tensor(hip, sg.I32, pos.shape).put(pos * theta ** np.arange(axes))
    share = d // 2 // axes
    hip[1].execute(sg.rope_axes_op(tx.desc, tp.desc, y.desc, d, [share] * axes, adjacent, base=theta**axes)[0])
    hip[1].sync()
    ang = np.concatenate([pos[:, a : a + 1] * float(theta) ** (-2 * np.arange(share) / (d / axes)) for a in range(axes)], 1)[:, None]
    i, j = (np.arange(0, d, 2), np.arange(1, d, 2)) if adjacent else (np.arange(d // 2), np.arange(d // 2) + d // 2)
    v = values(sg.F32, x)
    want, mag = v.copy(), np.zeros_like(v)
    want[..., i], want[..., j] = v[..., i] * np.cos(ang) - v[..., j] * np.sin(ang), v[..., i] * np.sin(ang) + v[..., j] * np.cos(ang)
    mag[..., i] = mag[..., j] = np.abs(v[..., i]) + np.abs(v[..., j])
    close(y.get(), want, mag, sg.F32)
    free_all(tx, y, tp)
