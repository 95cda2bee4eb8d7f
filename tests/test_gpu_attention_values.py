"""ATTENTION_PROMPT and ATTENTION_PAGED where values or weights are at the ends of their ranges."""
import math
import time

import numpy as np
import pytest

import scrapgpulibrary_amd as sg
from tests import attention_weights as aw
from tests.serving_util import Tensor, attend, free_all, to_bits, values
from tests.test_gpu_attention import run, run_paged

pytestmark = pytest.mark.gpu

D = 64


def attention(hip, q, k, v, dtype, out, scale, form, hk=1):
    """The result [n, Hq, D] of one request with q [n, Hq, D] over k, v [m, Hk, D] (the type's bits),
    causal: `form` "rows" (few rows over pages), "tiles" (pages) or "prompt"."""
    n, m, page = len(q), len(k), 16
    tq, y = Tensor(hip, dtype, q.shape).put(q), Tensor(hip, out, q.shape).fill()
    if form == "prompt":
        rest = [Tensor(hip, dtype, x.shape).put(x) for x in (k, v)]
        rest += [Tensor(hip, sg.I32, (2,)).put([0, i]) for i in (n, m)]
        op, keep = sg.attention_prompt_op(tq.desc, rest[0].desc, rest[1].desc, rest[2].desc, y.desc, scale, k_start=rest[3].desc)
    else:
        pages = -(-m // page)
        rest = []
        for x in (k, v):
            c = np.zeros((pages * page,) + x.shape[1:], x.dtype)
            c[:m] = x
            c = c.reshape(pages, page, *x.shape[1:]).swapaxes(1, 2)
            rest.append(Tensor(hip, dtype, c.shape).put(c))
        rest += [Tensor(hip, sg.I32, (1, pages)).put(np.arange(pages)), Tensor(hip, sg.I32, (2,)).put([0, n]), Tensor(hip, sg.I32, (1,)).put([m])]
        op, keep = sg.attention_paged_op(tq.desc, *[t.desc for t in rest], y.desc, scale, max_query=n if form == "rows" else 0)
    run(hip, op)
    assert ("rows" in sg.last_launch()[0]) == (form == "rows")
    got = values(out, y.get())
    free_all(tq, y, *rest)
    return got


def one_hot(dtype, n, heads, scores):
    """q and k whose scores (scale 1) are `scores` [m] for every row."""
    q, k = np.zeros((n, heads, D)), np.zeros((len(scores), 1, D))
    q[..., 3] = 1
    k[:, 0, 3] = scores
    return to_bits(dtype, q), to_bits(dtype, k)


FORMS = [("rows", 1), ("rows", 4), ("tiles", 80), ("prompt", 80), ("prompt", 1)]


@pytest.mark.parametrize("dtype,out", [(sg.F16, sg.F16), (sg.F16, sg.F32), (sg.BF16, sg.BF16), (sg.BF16, sg.F32)], ids=["f16-f16", "f16-f32", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("form,n", FORMS, ids=[f"{f}-{n}" for f, n in FORMS])
@pytest.mark.parametrize("heads", [1, 16])
def test_infinities_of_small_weight(hip, dtype, out, form, n, heads):
    """A seen infinite value makes the result infinite however small its weight, in the first step, in
    the last (which holds keys past the end), alone and beside the other sign (NaN there)."""
    m = 459 + n
    for less in (10, 20, 40, 80):  # the weights are e^-less of the largest
        scores = np.zeros(m)
        v = np.random.default_rng(less).standard_normal((m, 1, D))
        for j, d, x in ((1, 5, np.inf), (200, 9, -np.inf), (m - n, 13, np.inf), (2, 17, np.inf), (300, 17, -np.inf), (33, 21, np.nan)):
            scores[j] = -less
            v[j, 0, d] = x
        q, k = one_hot(dtype, n, heads, scores)
        v = to_bits(dtype, v)
        got = attention(hip, q, k, v, dtype, out, 1.0, form)
        w = np.exp(scores)
        seen = np.arange(m) <= m - n + np.arange(n)[:, None]
        w = np.where(seen, w, 0.0)
        fine = np.nan_to_num(values(dtype, v)[:, 0], nan=0.0, posinf=0.0, neginf=0.0)
        want = (w / w.sum(1, keepdims=True)) @ fine
        want[:, [5, 13]], want[:, 9], want[:, [17, 21]] = np.inf, -np.inf, np.nan
        want = np.broadcast_to(want[:, None], got.shape)
        for sign in (1, -1):
            assert np.array_equal(got == sign * np.inf, want == sign * np.inf)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        # (the weights: rounded once to the type, as its result; sums of 500 f32 terms)
        few = np.isfinite(want)
        assert np.max(np.abs(got[few] - want[few])) < 2 * {sg.F16: 2.0**-10, sg.BF16: 2.0**-7}[dtype]


@pytest.mark.parametrize("out", [sg.BF16, sg.F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("form,n", FORMS, ids=[f"{f}-{n}" for f, n in FORMS])
def test_large_values_that_fade(hip, out, form, n):
    """A finite value near the type's largest, in a key that a later one outweighs by e^200: nothing of it
    is left, whether the later key comes in the same wave's steps, in another's or in another piece."""
    for m, p in ((260, 1), (260, 40), (260, 130), (4000, 2000), (4000, 3900)):
        scores, v = np.zeros(m), np.zeros((m, 1, D))
        scores[p] = 200
        v[3, 0, 5], v[7, 0, 9] = 8.5e37, -3e38
        v[p, 0, :] = 0.5
        q, k = one_hot(sg.BF16, n, 3, scores)
        got = attention(hip, q, k, to_bits(sg.BF16, v), sg.BF16, out, 1.0, form)
        sees = m - n + np.arange(n) + 1 > p
        assert sees.any()
        assert np.max(np.abs(got[sees] - 0.5)) < 2.0**-7, (m, p)


def two_keys(hip, dtype, out, form, delta, v):
    """Requests of one new token over two keys each (see attention_weights): the results [n, 64]."""
    n, page = len(delta), 16
    t = n + (100 if form == "tiles" else 0)  # (tokens of one more request, over the first page: so many that tiles run)
    q = np.zeros((t, 1, D))
    q[..., 3] = 1
    k, vals = np.zeros((n, 2, 1, D)), np.zeros((n, 2, 1, D))
    k[:, 1, 0, 3], vals[:, 1, 0] = -values(dtype, delta), values(dtype, v)
    tq, y = Tensor(hip, dtype, q.shape).put(to_bits(dtype, q)), Tensor(hip, out, q.shape).fill()
    starts = np.append(np.arange(n + 1), [t] if t > n else []).astype(np.int32)
    if form == "prompt":
        rest = [Tensor(hip, dtype, (2 * n, 1, D)).put(to_bits(dtype, x.reshape(2 * n, 1, D))) for x in (k, vals)]
        rest += [Tensor(hip, sg.I32, (n + 1,)).put(i) for i in (starts, 2 * starts)]
        op, keep = sg.attention_prompt_op(tq.desc, rest[0].desc, rest[1].desc, rest[2].desc, y.desc, 1.0, k_start=rest[3].desc)
    else:
        rest = []
        for x in (k, vals):
            c = np.zeros((n, 1, page, D))
            c[:, 0, :2] = x[:, :, 0]
            rest.append(Tensor(hip, dtype, c.shape).put(to_bits(dtype, c)))
        b = len(starts) - 1
        rest += [Tensor(hip, sg.I32, (b, 1)).put(np.arange(b).reshape(b, 1) % n), Tensor(hip, sg.I32, (b + 1,)).put(starts), Tensor(hip, sg.I32, (b,)).put(np.full(b, 2))]
        op, keep = sg.attention_paged_op(tq.desc, *[x.desc for x in rest], y.desc, 1.0, max_query=1 if form == "rows" else 0)
    run(hip, op)
    assert ("rows" in sg.last_launch()[0]) == (form == "rows")
    got = values(out, y.get())[:n, 0]
    free_all(tq, y, *rest)
    return got


@pytest.mark.parametrize("dtype,out", [(sg.F16, sg.F16), (sg.F16, sg.F32), (sg.BF16, sg.BF16), (sg.BF16, sg.F32)], ids=["f16-f16", "f16-f32", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("form", ["rows", "tiles", "prompt"])
def test_weights_have_the_bits_that_they_should(hip, dtype, out, form):
    """F32 results: weights of 22 (F16) or 24 bits (BF16). 16-bit results: two terms of the type in the kernel
    for few rows, one in the tiles."""
    terms = {sg.F16: 2, sg.BF16: 3}[dtype] if out == sg.F32 else 2 if form == "rows" else 1
    for seed in range(4):
        delta, v = aw.inputs(dtype, 64, seed)
        want = aw.result(dtype, delta, v)
        over = np.abs(two_keys(hip, dtype, out, form, delta, v) - want) - aw.bound(dtype, out, terms, want)
        assert np.max(over) <= 0, f"{np.max(over):.3e} over the bound, {np.mean(over > 0):.1%} of the elements"


@pytest.mark.parametrize("form", ["rows", "tiles"])
@pytest.mark.parametrize("out", [sg.F16, sg.F32], ids=["f16", "f32"])
@pytest.mark.parametrize("hq,hk,d", [(3, 1, 8), (8, 2, 64), (6, 6, 96), (7, 1, 128), (5, 1, 184), (4, 1, 256)])
def test_tokens_of_no_request_are_zero(hip, form, out, hq, hk, d):
    """A fixed batch of which some tokens, or none, live: the others' results are zero, in either kernel."""
    for reqs, rest in (([(1, 40), (0, 9), (2, 70)], 1), ([(1, 300)], 700), ([(0, 5), (0, 0)], 33), ([(3, 3)] * 70, 250)):
        run_paged(hip, reqs, hq, hk, d, sg.F16, out, seed=d, rest=rest, max_query=3 if form == "rows" else 0)
        assert ("rows" in sg.last_launch()[0]) == (form == "rows") or form == "tiles"


def test_tokens_of_no_request_cost_little(hip):
    """64 single tokens in a batch with places for 8192 take less than twice the time of a batch of 64 (their
    zeros are 64 MiB beside 350 MiB of keys and values)."""
    dev, st = hip
    b, kv, page, hk, hq, d = 64, 4096, 16, 8, 32, 128
    pages = b * kv // page
    bufs = [dev.alloc(pages * page * hk * d * 2) for _ in range(2)]
    for buf in bufs:
        st.write(buf, 0, np.zeros(buf.size, np.uint8))
    k, v = (sg.tdesc(sg.F16, (d, page, hk, pages), buf) for buf in bufs)
    table = Tensor(hip, sg.I32, (b, kv // page)).put(np.random.default_rng(1).permutation(pages).reshape(b, -1))
    starts, lens = Tensor(hip, sg.I32, (b + 1,)).put(np.arange(b + 1)), Tensor(hip, sg.I32, (b,)).put(np.full(b, kv))
    times = []
    for t in (b, 8192):
        q, y = Tensor(hip, sg.F16, (t, hq, d)).put(0), Tensor(hip, sg.F16, (t, hq, d)).fill()
        op, keep = sg.attention_paged_op(q.desc, k, v, table.desc, starts.desc, lens.desc, y.desc, 0.1, max_query=1)
        took = []
        for _ in range(8):
            at = time.perf_counter()
            for _ in range(10):
                st.execute(op)
            st.sync()
            took.append(time.perf_counter() - at)
        times.append(min(took))
        free_all(q, y)
    free_all(table, starts, lens)
    for buf in bufs:
        buf.free()
    assert times[1] < 2 * times[0], times


def test_more_keys_than_a_whole_number_counts(hip):
    """40 requests of 2^30 keys each (all in one page, which their tables repeat): 1.3e9 steps of 32 keys in
    pieces that must not be more than the launch has room for. All scores are 0 and every sum is a whole
    number that f32 holds, so each result is the mean of the page's values; the next call is right as well."""
    dev, st = hip
    b, page, d, w = 40, 65536, 8, 16383
    v = np.zeros((1, 1, page, d), np.float16)
    for e in range(d):
        v[0, 0, e :: 4 + e % 4 * 4, e] = 1
    table = Tensor(hip, sg.I32, (b, w)).put(0)
    tk, tv = Tensor(hip, sg.F16, v.shape).put(np.zeros_like(v)), Tensor(hip, sg.F16, v.shape).put(v)
    q, y = Tensor(hip, sg.F16, (b, 1, d)).put(np.ones((b, 1, d), np.float16)), Tensor(hip, sg.F32, (b, 1, d)).fill()
    starts, lens = Tensor(hip, sg.I32, (b + 1,)).put(np.arange(b + 1)), Tensor(hip, sg.I32, (b,)).put(np.full(b, w * page))
    run(hip, sg.attention_paged_op(q.desc, tk.desc, tv.desc, table.desc, starts.desc, lens.desc, y.desc, 1.0, max_query=1)[0])
    assert "rows" in sg.last_launch()[0]
    # (the waves' and pieces' sums are whole, their joins round)
    assert np.max(np.abs(y.get() / v.astype(np.float64).mean(2)[0] - 1)) < 2.0**-18
    free_all(table, tk, tv, q, y, starts, lens)
    run_paged(hip, [(1, 5000), (1, 3000)], 4, 1, 64, sg.F16, sg.F32, max_query=1)


def test_launches_too_large_are_refused(hip):
    """More work-groups than a launch has (2^32 threads) are refused by the rule; the most that fit, and as
    many tokens where requests have few, are not."""
    dev, st = hip
    buf = dev.alloc(256)

    def prompt(b, t, hk):
        q, i = sg.tdesc(sg.F16, (8, hk, t), buf), sg.tdesc(sg.I32, (b + 1,), buf)
        return dev.supported(sg.attention_prompt_op(q, q, q, i, sg.tdesc(sg.F16, (8, hk, t)), 1.0)[0])

    def paged(b, t, hk, mq):
        q, i = sg.tdesc(sg.F16, (8, hk, t), buf), sg.tdesc(sg.I32, (b + 1,), buf)
        c = sg.tdesc(sg.F16, (8, 16, hk, 4), buf)
        return dev.supported(sg.attention_paged_op(q, c, c, sg.tdesc(sg.I32, (4, b), buf), i, sg.tdesc(sg.I32, (b,), buf), sg.tdesc(sg.F16, (8, hk, t)), 1.0, max_query=mq)[0])

    for status, why in (prompt(65535, 65535, 256), prompt(1, 1 << 23, 256), prompt(65535, 65535, 65535), paged(65535, 65535, 256, 1)):
        assert status == sg.UNSUPPORTED and "too many" in why, why
    for status, why in (prompt(65535, 65535, 250), prompt(1, 1 << 23, 200), paged(60000, 60000, 1, 1), paged(64, (1 << 24) - 1, 16, 1)):
        assert status == sg.OK, why
    buf.free()


def test_starts_that_go_back_over_a_long_request(hip):
    """Starts that cover tokens again and again beside one request of 256000 keys: the tiles are more than the
    launch has places for, and the long one's would be cut. Nothing but results is written, what is written is the
    result of a request that has the token (or of two, in parts), and the next call is right."""
    dev, st = hip
    r = np.random.default_rng(40)
    t, hq, page, short, long, again = 512, 16, 4096, 64, 256000, 22
    w = -(-long // page)
    kc, vc = (to_bits(sg.F16, r.standard_normal((w, 1, page, D))) for _ in range(2))
    q = to_bits(sg.F16, r.standard_normal((t, hq, D)))
    starts = [0, t] * again + [0, 8, t]
    b = len(starts) - 1
    lens = [short] * (b - 2) + [long, short]
    tables = np.tile(np.arange(w, dtype=np.int32), (b, 1))
    tk, tv, tq = (Tensor(hip, sg.F16, x.shape).put(x) for x in (kc, vc, q))
    y = Tensor(hip, sg.F32, q.shape, (16, 0, 0), 64).fill()
    ti, tl, tt = Tensor(hip, sg.I32, (b + 1,)).put(starts), Tensor(hip, sg.I32, (b,)).put(lens), Tensor(hip, sg.I32, tables.shape).put(tables)
    run(hip, sg.attention_paged_op(tq.desc, tk.desc, tv.desc, tt.desc, ti.desc, tl.desc, y.desc, 0.125, causal=0)[0])
    form, grid = sg.last_launch()
    want, room = int(form.split("want=")[1]), grid - 1
    # the pieces that the requests' lengths ask for, by the kernel's rule for their length
    tiles = [-(-max(0, n) * hq // 128) for n in np.diff(starts)]
    steps = [-(-m // 64) for m in lens]
    per = max(8, sum(n * m for n, m in zip(tiles, steps)) // want + 1)
    for _ in range(3):
        n = sum(a * -(-m // per) for a, m in zip(tiles, steps))
        per = per if n <= want else max(per + 1, per * n // want)
    assert "tiles" in form and max(steps) > per + 6 and sum(a * -(-m // per) for a, m in zip(tiles, steps)) > room > 0
    assert y.untouched()
    got = y.get()
    of = {}
    for m in (short, long):
        k, v = (values(sg.F16, c.reshape(-1, 1, D)[:m]) for c in (kc, vc))
        of[m] = attend(values(sg.F16, q[:8] if m == long else q), k, v, 0.125, 0)[0]
    fine = np.isnan(got) | (np.abs(got - of[short]) < 1e-4)
    fine[:8] |= np.abs(got[:8] - of[long]) < 1e-4
    assert fine.all() and not np.isnan(got[-8:]).any()
    free_all(tk, tv, tq, y, ti, tl, tt)
    run_paged(hip, [(40, 2000), (3, 9)], 4, 1, 64, sg.F16, sg.F32, seed=41)


@pytest.mark.parametrize("d,hq,each", [(128, 4, 2), (64, 64, 2), (128, 64, 1), (96, 40, 1), (256, 2, 1)])
def test_pieces_follow_what_a_cu_holds(hip, d, hq, each):
    """Few rows: the keys go in as many pieces as the CUs hold work-groups, two each, or one where 64 rows of
    more than 64 elements, or heads of 256, fill the registers."""
    run_paged(hip, [(1, 3000), (1, 100)], hq, 1, d, sg.F16, sg.F16, seed=d, max_query=1)
    assert int(sg.last_launch()[0].split("want=")[1]) == each * 256


@pytest.mark.parametrize("dtype,out", [(sg.F16, sg.F16), (sg.F16, sg.F32), (sg.BF16, sg.BF16), (sg.BF16, sg.F32)], ids=["f16-f16", "f16-f32", "bf16-bf16", "bf16-f32"])
@pytest.mark.parametrize("form,n", FORMS, ids=[f"{f}-{n}" for f, n in FORMS])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_the_largest_magnitude(hip, dtype, out, form, n, sign):
    """Scores of 2^24 and somewhat less, of either sign, in steps of 2^13 and more: the mean of the values at the
    largest."""
    m = 300 + n
    r = np.random.default_rng(7)
    q, k, v = np.zeros((n, 2, D)), np.zeros((m, 1, D)), r.integers(-8, 9, (m, 1, D)).astype(float)
    q[..., 3] = sign * 256
    k[:, 0, 3] = 65504 - 512 * r.integers(0, 3, m)
    k, v = to_bits(dtype, k), to_bits(dtype, v)
    got = attention(hip, to_bits(dtype, q), k, v, dtype, out, 1.0, form)
    for i in range(n):
        s = sign * values(dtype, k[: m - n + i + 1, 0, 3])
        want = values(dtype, v)[: m - n + i + 1, 0][s == s.max()].mean(0)
        # (equal weights: their rounding cancels; sums of 300 f32 terms of up to 8)
        assert np.max(np.abs(got[i] - want)) < {sg.F32: 2.0**-18, sg.F16: 2.0**-9, sg.BF16: 2.0**-6}[out]


@pytest.mark.parametrize("form,n", FORMS, ids=[f"{f}-{n}" for f, n in FORMS])
@pytest.mark.parametrize("d", [64, 72, 256])
def test_nothing_but_infinities(hip, form, n, d):
    """All values of many keys infinite, or NaN, or infinite in every other element, with weights that round to zero
    among them."""
    m = 1500 + n
    r = np.random.default_rng(d)
    q, k = np.zeros((n, 1, d)), np.zeros((m, 1, d))
    q[..., 3], k[:, 0, 3] = 1, -40 * (r.integers(0, 3, m) > 0)
    k[100] = 0
    for i, fill in enumerate((np.inf, -np.inf, np.nan, None)):
        v = np.full((m, 1, d), fill if fill is not None else 0.25)
        if fill is None:
            v[:, :, ::2] = np.inf
        got = attention(hip, to_bits(sg.F16, q), to_bits(sg.F16, k), to_bits(sg.F16, v), sg.F16, (sg.F16, sg.F32)[i % 2], 1.0, form)
        want = np.broadcast_to(v[0, 0], got.shape)
        assert np.array_equal(got, want, equal_nan=True), fill
