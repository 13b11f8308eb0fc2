"""GPU tests of the token log probabilities against a plain 64-bit implementation.

Tolerances: an exponential of the hardware is within 2 units in the last place and the argument z log2(e) is rounded once,
so a term of the sum is off by at most (|z| + 4) 2^-24 relative, and the sum over lanes and slices adds at most 2^-18 for
the vocabularies here; weighted by the terms themselves (|z| e^z stays under 1/e of the largest term per token) log l is
off by less than 2^-17 + 2^-22 log V, and x - m - log l by another unit of |x - m| <= 2^7: 3e-5 absolute.  The entropy is
a ratio of two such sums, of numbers up to log V = 12: 2e-4 absolute bounds twelve times that error.  Identities of the
alternatives are exact."""
import numpy as np
import pytest

from gpu_util import act_rounded, act_to_device_array

pytestmark = pytest.mark.gpu
LOGPROB, ENTROPY = 3e-5, 2e-4


def plain(x, tokens, top):
    """x: float32 [rows, vocabulary] as the device reads them."""
    x = np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), np.finfo(np.float32).max))
    lp, h = np.full(len(x), -np.inf), np.zeros(len(x))
    ids, tops = np.full((len(x), top), -1, np.int32), np.full((len(x), top), -np.inf)
    for r, row in enumerate(x):
        alive = np.flatnonzero(row > -np.inf)
        if not alive.size:
            continue
        m = row.max()
        e = np.exp(row[alive] - m)
        log_z = np.log(e.sum())
        p = e / e.sum()
        h[r] = -np.sum(np.where(p > 0, p * (row[alive] - m - log_z), 0))
        if 0 <= tokens[r] < len(row):
            lp[r] = row[tokens[r]] - m - log_z
        order = alive[np.lexsort((alive, -row[alive]))][:top]
        ids[r, :len(order)] = order
        tops[r, :len(order)] = row[order] - m - log_z
    return lp, h, ids, tops


def run(pkg, ctx, x, dtype, tokens, top, pad=0, shift=0):
    """Rows `pad` elements apart beyond the vocabulary, the first `shift` elements behind an aligned address."""
    rows, v = x.shape
    stride = v + pad
    laid = np.full(shift + rows * stride, np.nan, np.float32)
    for r in range(rows):
        laid[shift + r * stride:shift + r * stride + v] = x[r]
    d = ctx.upload(act_to_device_array(laid, dtype, pkg))
    t = ctx.upload(np.asarray(tokens, np.int32))
    lp, h = (ctx.upload(np.full(rows, np.nan, np.float32)) for _ in range(2))
    ids, tops = ctx.upload(np.full((rows, max(top, 1)), -9, np.int32)), ctx.upload(np.full((rows, max(top, 1)), np.nan, np.float32))
    ctx.token_logprobs(d.ptr + shift * (4 if dtype == pkg.F32 else 2), dtype, rows, v, t, top, lp, h, ids, tops, row_stride=stride if pad else 0)
    ctx.synchronize()
    return (lp.download(np.float32, (rows,)), h.download(np.float32, (rows,)),
            ids.download(np.int32, (rows, max(top, 1)))[:, :top], tops.download(np.float32, (rows, max(top, 1)))[:, :top])


def check(pkg, ctx, x, dtype, tokens, top, **kw):
    seen = act_rounded(x, dtype, pkg)
    lp, h, ids, tops = run(pkg, ctx, x, dtype, tokens, top, **kw)
    want_lp, want_h, want_ids, want_tops = plain(seen, tokens, top)
    assert np.array_equal(ids, want_ids)
    for got, want, tol in ((lp, want_lp, LOGPROB), (tops, want_tops, LOGPROB), (h, want_h, ENTROPY)):
        fine = np.isfinite(want)
        assert np.array_equal(got[~fine], want[~fine].astype(np.float32))
        # numbers beyond 2^7 in magnitude are off by units of their own
        assert np.all(np.abs(got[fine] - want[fine]) <= tol * np.maximum(1, np.abs(want[fine]) / 128))


@pytest.mark.parametrize("dtype", ["F32", "BF16", "F16"])
@pytest.mark.parametrize("rows,vocabulary,top,pad,shift", [
    (1, 1, 1, 0, 0), (2, 2, 5, 0, 0), (3, 63, 32, 0, 1), (5, 64, 8, 3, 0), (1, 1023, 20, 0, 3), (4, 1025, 0, 0, 0),
    (2, 4096, 5, 0, 0), (3, 4099, 32, 1, 7), (1, 65536, 5, 0, 0), (7, 50021, 20, 2, 1), (2500, 77, 3, 0, 0),
    (1, 300007, 32, 0, 5)])
def test_shapes(pkg, ctx, dtype, rows, vocabulary, top, pad, shift):
    rng = np.random.default_rng(rows + vocabulary)
    x = (rng.standard_normal((rows, vocabulary)) * 4).astype(np.float32)
    check(pkg, ctx, x, getattr(pkg, dtype), rng.integers(0, vocabulary, rows), top, pad=pad, shift=shift)


@pytest.mark.parametrize("vocabulary", [50, 5000, 70001])
def test_orders_that_are_hard_on_the_alternatives(pkg, ctx, vocabulary):
    """Ascending (every logit is an alternative when it is met), descending, all equal, a few values, one peak."""
    rng = np.random.default_rng(7)
    v = np.arange(vocabulary, dtype=np.float32)
    rows = [v * np.float32(20 / vocabulary), -v * np.float32(20 / vocabulary), np.zeros(vocabulary, np.float32),
            rng.choice(np.array([1.0, 2.0, 3.0, -0.0, 0.0], np.float32), vocabulary), np.where(v == vocabulary - 1, 60, 0).astype(np.float32)]
    x = np.stack(rows).astype(np.float32)
    for dtype in (pkg.F32, pkg.BF16):
        check(pkg, ctx, x, dtype, [vocabulary - 1, 0, 3, 7, vocabulary - 1], 32)


def test_masked_logits(pkg, ctx):
    """-inf and NaN are masked, +inf the largest number, the lowest finite number a logit like any other."""
    rng = np.random.default_rng(8)
    v = 9001
    x = (rng.standard_normal((8, v)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1] = np.nan
    x[2] = -np.inf; x[2, 8000] = -3.0; x[2, 17] = -3.0
    x[3, rng.random(v) < 0.9] = -np.inf
    x[4, rng.random(v) < 0.5] = np.nan
    x[5, 100] = np.inf; x[5, 200] = np.inf
    x[6] = np.finfo(np.float32).min
    x[7, 1:] = np.finfo(np.float32).min
    check(pkg, ctx, x, pkg.F32, [3, 3, 17, int(np.flatnonzero(x[3] == -np.inf)[0]), int(np.flatnonzero(np.isnan(x[4]))[0]), 200, 5, 0], 9)
    check(pkg, ctx, x[:1], pkg.F32, [-1], 4)


def test_tokens_outside_the_vocabulary(pkg, ctx):
    x = np.random.default_rng(9).standard_normal((4, 333)).astype(np.float32)
    check(pkg, ctx, x, pkg.BF16, [-1, 333, 2 ** 31 - 1, 332], 3)


def test_entropy_ends(pkg, ctx):
    """log V for equal logits, 0 for a certain token."""
    x = np.zeros((2, 65536), np.float32)
    x[1] = -1000.0
    x[1, 4] = 0.0
    lp, h, ids, tops = run(pkg, ctx, x, pkg.F32, [9, 4], 2)
    assert abs(h[0] - np.log(65536)) <= ENTROPY and h[1] == 0 and lp[1] == 0
    assert ids.tolist() == [[0, 1], [4, 0]]


def test_parts_alone(pkg, ctx):
    """Only log probabilities, only the entropy, only the alternatives."""
    x = np.random.default_rng(10).standard_normal((3, 20000)).astype(np.float32)
    tokens = [5, 6, 7]
    lp, h, ids, tops = run(pkg, ctx, x, pkg.F32, tokens, 4)
    d, t = ctx.upload(x), ctx.upload(np.array(tokens, np.int32))
    a, b, c, e = ctx.alloc(12), ctx.alloc(12), ctx.alloc(48), ctx.alloc(48)
    ctx.token_logprobs(d, pkg.F32, 3, 20000, t, 0, a)
    ctx.token_logprobs(d, pkg.F32, 3, 20000, entropy=b)
    ctx.token_logprobs(d, pkg.F32, 3, 20000, top_count=4, top_ids=c, top_logprobs=e)
    ctx.synchronize()
    assert np.array_equal(a.download(np.float32), lp) and np.array_equal(b.download(np.float32), h)
    assert np.array_equal(c.download(np.int32, (3, 4)), ids) and np.array_equal(e.download(np.float32, (3, 4)), tops)


def test_refusals(pkg, ctx):
    x, t, o = ctx.alloc(400), ctx.alloc(400), ctx.alloc(400)
    for status, args, kw in [
            ("INVALID_ARGUMENT", (None, pkg.F32, 1, 50, t, 0, o), {}), ("INVALID_ARGUMENT", (x, 5, 1, 50, t, 0, o), {}),
            ("SHAPE", (x, pkg.F32, 0, 50, t, 0, o), {}), ("SHAPE", (x, pkg.F32, 1, 0, t, 0, o), {}),
            ("SHAPE", (x, pkg.F32, 1, 50, t, 0, o), {"row_stride": 49}), ("SHAPE", (x, pkg.F32, 1, 50, t, 33, o, o, o, o), {}),
            ("INVALID_ARGUMENT", (x, pkg.F32, 1, 50, t, 0, None, o), {}), ("INVALID_ARGUMENT", (x, pkg.F32, 1, 50, None, 0, o), {}),
            ("INVALID_ARGUMENT", (x, pkg.F32, 1, 50, t, 3, o, o, o), {}), ("INVALID_ARGUMENT", (x, pkg.F32, 1, 50), {}),
            ("INVALID_ARGUMENT", (x.ptr + 2, pkg.F32, 1, 50, t, 0, o), {})]:
        with pytest.raises(pkg.MI355QError) as e:
            ctx.token_logprobs(*args, **kw)
        assert e.value.status_name == status, (args, str(e.value))
