"""GPU tests of the attention over the 8-bit block cache against a plain 64-bit implementation of the definition.

Tolerances.  Scores: products of codes with f16 / bf16 queries are exact in fp32, a sum of HD of them is off by at most
HD 2^-24 of the sum of magnitudes (under 64 in these inputs, scaled): 1e-3 absolute at the very most, 2e-5 typically; lse
inherits that: 2e-4.  Weights are rounded to f16 in front of the product with the values: 2^-11 of each, so the output is
off by at most 2^-11 of the weighted mean of |v|, below 2^-11 max|v|, plus the output's own rounding, 2^-8 (bf16) or
2^-11 (f16) of |out| <= max|v|.  Weight sums are fp32 and inherit the scores' error relative to their size."""
import numpy as np
import pytest

from gpu_util import act_rounded, act_to_device_array, out_from_device
from test_gpu_kv_block_cache import TOKENS, Cache, deal, lay_out, sequences

pytestmark = pytest.mark.gpu


def plain(cache, tables, lengths, rows, q, group, scale, window):
    """q: [rows, heads, hd].  Returns out, lse [rows, heads] and the added weight sums, all in 64 bits."""
    total, heads, hd = q.shape
    out, lse = np.zeros((total, heads, hd)), np.full((total, heads), -np.inf)
    added = np.zeros(cache.sums.shape)
    at = 0
    for b, n in enumerate(rows):
        length = lengths[b]
        k, v = cache.numbers(tables[b], length).astype(np.float64)
        there = np.array([0 <= tables[b][t // TOKENS] < cache.blocks for t in range(length)], bool)
        for i in range(n):
            p = length - n + i
            t = np.arange(length)
            seen = (t <= p) & there & ((t > p - window) if window else True)
            idx = np.flatnonzero(seen)
            if idx.size:
                for h in range(heads):
                    kv = h // group
                    s = k[idx, kv] @ q[at + i, h].astype(np.float64) * scale
                    m = s.max()
                    e = np.exp(s - m)
                    w = e / e.sum()
                    out[at + i, h] = w @ v[idx, kv]
                    lse[at + i, h] = m + np.log(e.sum())
                    for x, t_ in zip(w, idx):
                        added[tables[b][t_ // TOKENS], kv, t_ % TOKENS] += x
        at += n
    return out, lse, added


def run(pkg, ctx, cache, seq, q, q_dtype, out_dtype, scale, window=0, weights=True, pad=0, lse=True):
    total, heads, hd = q.shape
    width = heads * hd
    laid = np.full((total, width + pad), 7.0, np.float32)
    laid[:, :width] = q.reshape(total, width)
    qd = ctx.upload(act_to_device_array(laid, q_dtype, pkg))
    od, ld = ctx.upload(np.full(total * (width + pad), 0x7FC0, np.uint16)), ctx.upload(np.full(total * heads, np.nan, np.float32))
    ctx.kv_block_attention(cache.c, seq, qd, q_dtype, heads, od, out_dtype, scale, window, ld if lse else None, weights,
                           width + pad if pad else 0, width + pad if pad else 0)
    ctx.synchronize()
    out = out_from_device(od, out_dtype, (total, width + pad), pkg)
    assert np.all(np.isnan(out[:, width:]))
    return out[:, :width].reshape(total, heads, hd), ld.download(np.float32, (total, heads))


def check(pkg, ctx, cache, tables, lengths, rows, q, q_dtype, out_dtype, window=0, pad=0, bounds=None, scale=None):
    heads, hd = q.shape[1:]
    scale = hd ** -0.5 if scale is None else scale
    q = act_rounded(q, q_dtype, pkg)
    seq = sequences(pkg, ctx, tables, lengths, rows, bounds)
    before = cache.download()[2].astype(np.float64)
    out, lse = run(pkg, ctx, cache, seq, q, q_dtype, out_dtype, scale, window, True, pad)
    want, want_lse, added = plain(cache, tables, lengths, rows, q, heads // cache.heads, scale, window)
    top = 127 * cache.scales[..., 1].max()
    step = 2.0 ** -8 if out_dtype == pkg.BF16 else 2.0 ** -11
    assert np.all(np.abs(out - want) <= 2.0 ** -11 * top + step * np.abs(want) + 1e-6)
    seen = np.isfinite(want_lse)
    assert np.array_equal(seen, np.isfinite(lse)) and np.all(lse[~seen] == -np.inf) and not out[~seen].any()
    assert np.all(np.abs(lse[seen] - want_lse[seen]) <= 2e-4)
    _, _, sums = cache.download()
    assert np.all(np.abs(sums - (before + added)) <= 2e-4 * np.maximum(added, 1e-3) + 2.0 ** -22 * np.abs(before))
    # the same again: weights have been added a second time, outputs have the same bits
    out2, lse2 = run(pkg, ctx, cache, seq, q, q_dtype, out_dtype, scale, window, True, pad)
    assert np.array_equal(out2, out) and np.array_equal(lse2, lse)
    # without weights and without lse: the same outputs up to the order of sums, and the sums untouched
    _, _, sums = cache.download()
    out3, _ = run(pkg, ctx, cache, seq, q, q_dtype, out_dtype, scale, window, False, pad, lse=False)
    assert np.all(np.abs(out3 - out) <= 2.0 ** -10 * top + 2 * step * np.abs(want) + 1e-6)
    assert np.array_equal(cache.download()[2], sums)


CASES = [
    # (head dimension, KV heads, group, lengths, rows, window)
    (128, 2, 4, [1], [1], 0),                                  # one token
    (128, 1, 8, [64, 65, 63, 128], [1, 1, 1, 1], 0),           # ends of blocks
    (64, 3, 1, [300, 5, 777], [1, 1, 1], 0),                   # one head each
    (256, 1, 3, [130, 1000], [1, 2], 0),
    (128, 2, 16, [515], [1], 0),
    (64, 1, 7, [200], [5], 0),                                 # 35 rows of a group
    (128, 1, 5, [2500, 40], [1, 1], 0),                        # several parts of a sequence
    (64, 2, 4, [70, 333, 64], [70, 100, 1], 0),                # prompts beside a decode step
    (128, 2, 3, [129], [129], 0),
    (256, 2, 2, [90, 260], [33, 7], 0),
    (128, 1, 2, [400], [200], 50),                             # sliding windows
    (64, 1, 4, [1000, 10], [3, 10], 1),
    (128, 2, 1, [700], [4], 65),
    (64, 1, 20, [100], [1], 0),                                # groups beyond sixteen and thirty-two
    (64, 1, 40, [100], [1], 0),
    (128, 1, 64, [70], [2], 0),
    (256, 1, 1, [600], [130], 300),
]


@pytest.mark.parametrize("types", [("BF16", "BF16"), ("F16", "F16"), ("F16", "BF16")])
@pytest.mark.parametrize("hd,heads,group,lengths,rows,window", CASES)
def test_attention(pkg, ctx, hd, heads, group, lengths, rows, window, types):
    rng = np.random.default_rng(hd + sum(lengths) + group)
    tables, _, blocks = deal(rng, lengths, spare=1)
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)
    q = (rng.standard_normal((sum(rows), heads * group, hd)) * 0.5).astype(np.float32)
    check(pkg, ctx, cache, tables, lengths, rows, q, getattr(pkg, types[0]), getattr(pkg, types[1]), window)


@pytest.mark.parametrize("rows", [1, 60])
def test_rows_that_see_nothing(pkg, ctx, rows):
    """Empty sequences, more rows than tokens, absent blocks, and a window that falls into an absent block."""
    rng = np.random.default_rng(11)
    cache = Cache(pkg, ctx, 1, 64, 3, rng)
    tables, lengths = [[0], [1], [2, -1, 7], [99]], [0, 20, 190, 64]
    n = [rows, rows, rows, rows]
    q = rng.standard_normal((sum(n), 2, 64)).astype(np.float32)
    check(pkg, ctx, cache, tables, lengths, n, q, pkg.BF16, pkg.F16)
    check(pkg, ctx, cache, tables, lengths, n, q, pkg.F16, pkg.BF16, window=30)


@pytest.mark.parametrize("rows", [1, 70])
def test_strides_and_wide_bounds(pkg, ctx, rows):
    """Rows apart, at odd strides, and bounds far above the real lengths and rows."""
    rng = np.random.default_rng(12)
    tables, _, blocks = deal(rng, [300, 100])
    cache = Cache(pkg, ctx, 2, 128, blocks, rng)
    q = rng.standard_normal((rows + 1, 6, 128)).astype(np.float32)
    for pad in (8, 3):
        check(pkg, ctx, cache, tables, [300, 100], [rows, 1], q, pkg.BF16, pkg.BF16, pad=pad, bounds=(rows + 1, 20000))


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("spread", [1e-4, 1.0, 1e4])
def test_scales_of_blocks_far_apart(pkg, ctx, rows, spread):
    """Blocks whose value scales differ by up to 10^8, zero scales among them, and scores from flat to one-hot."""
    rng = np.random.default_rng(13)
    tables, _, blocks = deal(rng, [500])
    cache = Cache(pkg, ctx, 1, 128, blocks, rng)
    cache.scales[:, :, 1] = spread * 10.0 ** rng.uniform(-4, 4, (blocks, 1))
    cache.scales[tables[0][1]] = 0.0
    cache.codes[tables[0][1]] = 0
    cache.d_codes.upload(lay_out(cache.codes))
    cache.d_scales.upload(cache.scales)
    q = rng.standard_normal((rows, 4, 128)).astype(np.float32) * np.array([0.0, 1e-3, 1.0, 4.0], np.float32)[None, :, None]
    out_dtype = pkg.BF16 if spread > 1 else pkg.F16 if spread < 1 else pkg.BF16
    check(pkg, ctx, cache, tables, [500], [rows], q, pkg.BF16, out_dtype)


@pytest.mark.parametrize("rows", [1, 40])
def test_large_and_small_queries(pkg, ctx, rows):
    """Rows of bf16 queries whose size is far outside the f16 range, brought back by the scales of the keys."""
    rng = np.random.default_rng(14)
    tables, _, blocks = deal(rng, [200])
    for size in (1e-30, 1e-6, 1e6, 1e30):
        cache = Cache(pkg, ctx, 1, 64, blocks, rng)
        cache.scales[:, :, 0] = (rng.uniform(0.01, 0.05, (blocks, 1)) / size).astype(np.float32)
        cache.d_scales.upload(cache.scales)
        q = (rng.standard_normal((rows, 3, 64)) * size).astype(np.float32)
        check(pkg, ctx, cache, tables, [200], [rows], q, pkg.BF16, pkg.BF16)


@pytest.mark.parametrize("rows", [1, 40])
def test_a_query_that_is_no_number_stays_in_its_row(pkg, ctx, rows):
    rng = np.random.default_rng(15)
    tables, _, blocks = deal(rng, [100])
    cache = Cache(pkg, ctx, 1, 64, blocks, rng)
    q = rng.standard_normal((rows, 4, 64)).astype(np.float32)
    seq = sequences(pkg, ctx, tables, [100], [rows])
    clean, _ = run(pkg, ctx, cache, seq, act_rounded(q, pkg.F16, pkg), pkg.F16, pkg.F16, 0.125, weights=False)
    q[0, 1, 3], q[0, 2, 0] = np.nan, np.inf
    out, lse = run(pkg, ctx, cache, seq, act_rounded(q, pkg.F16, pkg), pkg.F16, pkg.F16, 0.125, weights=False)
    assert np.all(np.isnan(out[0, 1])) and np.isnan(lse[0, 1]) and np.all(np.isnan(out[0, 2]))
    keep = np.ones((rows, 4), bool)
    keep[0, 1:3] = False
    assert np.array_equal(out[keep], clean[keep])


def test_long_cache_offsets(pkg, ctx):
    """Blocks beyond 2^31 bytes of codes: 140000 blocks of one head of 128 are 2.3 GB."""
    rng = np.random.default_rng(16)
    blocks, hd = 140000, 128
    small = Cache(pkg, ctx, 1, hd, 4, rng)
    codes, scales, sums = ctx.alloc(blocks * 2 * TOKENS * hd), ctx.alloc(blocks * 8), ctx.alloc(blocks * 256)
    ctx.fill(sums, 0)
    far = [139999, 5, 131072, 70000]
    laid = lay_out(small.codes)
    for i, b in enumerate(far):
        for buf, part in ((codes, laid[i]), (scales, small.scales[i])):
            size = part.nbytes
            piece = type(buf)(ctx, buf.ptr + b * size, size)
            piece.upload(part)
    q = act_rounded(rng.standard_normal((1, 4, hd)).astype(np.float32), pkg.BF16, pkg)
    wide = type("", (), {"c": pkg.KVBlockCache(1, hd, blocks, codes, scales, sums)})
    got, lse = run(pkg, ctx, wide, sequences(pkg, ctx, [far], [250], [1]), q, pkg.BF16, pkg.F16, 0.1)
    want, want_lse = run(pkg, ctx, small, sequences(pkg, ctx, [[0, 1, 2, 3]], [250], [1]), q, pkg.BF16, pkg.F16, 0.1)
    assert np.array_equal(got, want) and np.array_equal(lse, want_lse)
    for b in (codes, scales, sums):
        b.free()


def test_second_stream(pkg, ctx):
    """The call runs on the stream it is given: inputs uploaded there by a kernel of that stream are seen."""
    rng = np.random.default_rng(17)
    tables, _, blocks = deal(rng, [700])
    cache = Cache(pkg, ctx, 1, 128, blocks, rng)
    q = act_rounded(rng.standard_normal((1, 4, 128)).astype(np.float32), pkg.F16, pkg)
    seq = sequences(pkg, ctx, tables, [700], [1])
    want, _ = run(pkg, ctx, cache, seq, q, pkg.F16, pkg.F16, 0.1, weights=False)
    own = pkg.Context(0)
    stream = own.stream_create()
    src, qd, od = ctx.upload(act_to_device_array(q.reshape(1, -1), pkg.F16, pkg)), ctx.alloc(1024), ctx.alloc(1024)
    ctx.synchronize()
    own.copy(qd, src, 1024, stream)
    own.kv_block_attention(cache.c, seq, qd, pkg.F16, 4, od, pkg.F16, 0.1, stream=stream)
    own.synchronize(stream)
    assert np.array_equal(out_from_device(od, pkg.F16, (1, 4, 128), pkg), want)
    own.stream_destroy(stream)
    own.close()


def test_refusals(pkg, ctx):
    cache = Cache(pkg, ctx, 2, 64, 4)
    bare = Cache(pkg, ctx, 2, 64, 4, sums=False)
    seq = sequences(pkg, ctx, [[0, 1]], [100], [3])
    q, o = ctx.alloc(3 * 512), ctx.alloc(3 * 512)
    for status, args, kw in [
            ("INVALID_ARGUMENT", (cache.c, seq, q, pkg.F32, 4, o, pkg.F16, 0.1), {}),
            ("INVALID_ARGUMENT", (cache.c, seq, q, pkg.F16, 4, o, pkg.F32, 0.1), {}),
            ("INVALID_ARGUMENT", (cache.c, seq, None, pkg.F16, 4, o, pkg.F16, 0.1), {}),
            ("INVALID_ARGUMENT", (cache.c, seq, q, pkg.F16, 4, None, pkg.F16, 0.1), {}),
            ("SHAPE", (cache.c, seq, q, pkg.F16, 3, o, pkg.F16, 0.1), {}), ("SHAPE", (cache.c, seq, q, pkg.F16, 0, o, pkg.F16, 0.1), {}),
            ("INVALID_ARGUMENT", (cache.c, seq, q, pkg.F16, 4, o, pkg.F16, 0.0), {}),
            ("INVALID_ARGUMENT", (cache.c, seq, q, pkg.F16, 4, o, pkg.F16, float("nan")), {}),
            ("SHAPE", (cache.c, seq, q, pkg.F16, 4, o, pkg.F16, 0.1), {"q_row_stride": 255}),
            ("SHAPE", (cache.c, seq, q, pkg.F16, 4, o, pkg.F16, 0.1), {"out_row_stride": 255}),
            ("INVALID_ARGUMENT", (cache.c, seq, q.ptr + 1, pkg.F16, 4, o, pkg.F16, 0.1), {}),
            ("INVALID_ARGUMENT", (bare.c, seq, q, pkg.F16, 4, o, pkg.F16, 0.1), {"accumulate_weights": True})]:
        with pytest.raises(pkg.MI355QError) as e:
            ctx.kv_block_attention(*args, **kw)
        assert e.value.status_name == status, (args, str(e.value))


SPANS = [
    # (head dimension, KV heads, group, lengths, rows, window): tiles of 128 rows whose blocks are dealt to the workgroups
    (128, 1, 4, [6000], [70], 0),                              # many parts of a tile
    (128, 2, 3, [4000, 70, 0, 1500, 300], [60, 90, 5, 1, 200], 0),      # rows in front of the first token, an empty sequence
    (64, 3, 5, [5000, 64, 2000], [30, 64, 129], 0),
    (256, 1, 4, [3000, 129], [40, 129], 0),
    (256, 2, 2, [2600, 2600, 2600], [9, 30, 12], 2000),
    (128, 1, 2, [6000, 500], [100, 20], 3000),
]


@pytest.mark.parametrize("hd,heads,group,lengths,rows,window", SPANS)
def test_attention_in_spans(pkg, ctx, hd, heads, group, lengths, rows, window):
    rng = np.random.default_rng(hd + sum(lengths) + group)
    tables, _, blocks = deal(rng, lengths, spare=1)
    tables[0][len(tables[0]) // 2] = -1                        # an absent block in the middle of the longest sequence
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)
    q = (rng.standard_normal((sum(rows), heads * group, hd)) * 0.5).astype(np.float32)
    check(pkg, ctx, cache, tables, lengths, rows, q, pkg.BF16, pkg.F16, window)


def test_as_many_parts_as_there_can_be(pkg, ctx):
    """One tile of a single head over 200 000 tokens: 125 parts."""
    rng = np.random.default_rng(12)
    hd, length, rows = 64, 200_000, 40
    tables, _, blocks = deal(rng, [length])
    cache = Cache(pkg, ctx, 1, hd, blocks, rng)
    q = act_rounded((rng.standard_normal((rows, 1, hd)) * 0.5).astype(np.float32), pkg.F16, pkg)
    seq = sequences(pkg, ctx, tables, [length], [rows])
    out, lse = run(pkg, ctx, cache, seq, q, pkg.F16, pkg.F16, hd ** -0.5, weights=False)
    numbers = cache.codes[tables[0], 0].astype(np.float64) * cache.scales[tables[0], 0][:, :, None, None]
    k, v = numbers.transpose(1, 0, 2, 3).reshape(2, -1, hd)[:, :length]
    s = q[:, 0].astype(np.float64) @ k.T * hd ** -0.5
    s[np.arange(length)[None] > np.arange(length - rows, length)[:, None]] = -np.inf
    m = s.max(1, keepdims=True)
    e = np.exp(s - m)
    total = e.sum(1, keepdims=True)
    want = e @ v / total
    top = 127 * cache.scales[..., 1].max()
    assert np.all(np.abs(out[:, 0] - want) <= 2.0 ** -11 * top + 2.0 ** -11 * np.abs(want) + 1e-6)
    assert np.all(np.abs(lse - (m + np.log(total))) <= 2e-4)


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_more_tiles_than_the_chip_holds(pkg, ctx, hd, window):
    """Forty short prompts of ten heads: a workgroup a tile, with the wavefronts' other shape."""
    rng = np.random.default_rng(hd + window)
    lengths = rng.integers(30, 150, 40).tolist()
    rows = [33 if i % 7 else 34 for i in range(40)]
    tables, _, blocks = deal(rng, lengths)
    cache = Cache(pkg, ctx, 10, hd, blocks, rng)
    q = (rng.standard_normal((sum(rows), 10, hd)) * 0.5).astype(np.float32)
    check(pkg, ctx, cache, tables, lengths, rows, q, pkg.BF16, pkg.F16, window)


def test_long_prompt_with_all_tiles_whole(pkg, ctx):
    """A prompt of 1500 rows of 40 heads on 40: 480 tiles of up to 24 blocks, one of them absent; a sample of rows and heads
    against the definition."""
    rng = np.random.default_rng(21)
    hd, heads, length = 64, 40, 1500
    tables, _, blocks = deal(rng, [length])
    tables[0][5] = blocks + 3
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)
    q = act_rounded((rng.standard_normal((length, heads, hd)) * 0.5).astype(np.float32), pkg.BF16, pkg)
    out, lse = run(pkg, ctx, cache, sequences(pkg, ctx, tables, [length], [length]), q, pkg.BF16, pkg.BF16, hd ** -0.5, weights=False)
    k, v = cache.numbers(tables[0], length).astype(np.float64)
    there = np.array([0 <= tables[0][t // TOKENS] < blocks for t in range(length)])
    top = 127 * cache.scales[..., 1].max()
    for r in list(range(0, 140)) + list(rng.integers(140, length, 200)) + [length - 1]:
        for h in rng.integers(0, heads, 3):
            seen = there & (np.arange(length) <= r)
            s = k[seen, h] @ q[r, h].astype(np.float64) * hd ** -0.5
            e = np.exp(s - s.max())
            want = e @ v[seen, h] / e.sum()
            assert np.all(np.abs(out[r, h] - want) <= 2.0 ** -11 * top + 2.0 ** -8 * np.abs(want) + 1e-6)
            assert abs(lse[r, h] - (s.max() + np.log(e.sum()))) <= 2e-4
