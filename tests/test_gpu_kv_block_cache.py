"""GPU tests of the 8-bit block KV cache: append, read back and eviction through the C ABI, against a plain NumPy
implementation that follows the definition token by token.

The cache's scales are one fp32 product each and its codes one division and one rounding each, in the order the plain
implementation performs them in fp32, so codes, scales, weight sums and positions are compared for equality; numbers read
back are code * scale in fp32, rounded once."""
import numpy as np
import pytest

import oracle
from gpu_util import act_rounded, act_to_device_array, out_from_device

pytestmark = pytest.mark.gpu
INVERSE = np.float32(1 / 127.49)
TOKENS = 64


def key_byte(t, d, hd):
    return (((t // 16) * (hd // 64) + d // 64) * 4 + d // 16 % 4) * 256 + t % 16 * 16 + d % 16


def value_byte(t, d, hd):
    return (d // 16 * 4 + t // 4 % 4) * 256 + d % 16 * 16 + t // 32 * 8 + t // 16 % 2 * 4 + t % 4


def places(hd):
    """Byte of every (token, dimension) of a block's keys and values."""
    t, d = np.meshgrid(np.arange(TOKENS), np.arange(hd), indexing="ij")
    return key_byte(t, d, hd), value_byte(t, d, hd)


def lay_out(codes):
    """[block, head, 2, token, dimension] -> [block, head, 2, 64 x dimensions] as the cache holds it."""
    n, h, _, _, hd = codes.shape
    out = np.empty((n, h, 2, TOKENS * hd), np.int8)
    for part, place in enumerate(places(hd)):
        out[:, :, part, place.ravel()] = codes[:, :, part].reshape(n, h, -1)
    return out


def take_apart(laid, hd):
    n, h = laid.shape[:2]
    return np.stack([laid[:, :, part, place.ravel()].reshape(n, h, TOKENS, hd) for part, place in enumerate(places(hd))], 2)


class Cache:
    """A cache on the host, in plain order, and its copy on the device."""

    def __init__(self, pkg, ctx, heads, hd, blocks, rng=None, sums=True):
        self.pkg, self.ctx, self.heads, self.hd, self.blocks = pkg, ctx, heads, hd, blocks
        shape = (blocks, heads, 2, TOKENS, hd)
        self.codes = np.zeros(shape, np.int8) if rng is None else rng.integers(-127, 128, shape).astype(np.int8)
        self.scales = np.zeros((blocks, heads, 2), np.float32) if rng is None else rng.uniform(0.005, 0.05, (blocks, heads, 2)).astype(np.float32)
        self.sums = np.zeros((blocks, heads, TOKENS), np.float32) if rng is None else rng.uniform(0, 4, (blocks, heads, TOKENS)).astype(np.float32)
        self.d_codes, self.d_scales = ctx.upload(lay_out(self.codes)), ctx.upload(self.scales)
        self.d_sums = ctx.upload(self.sums) if sums else None
        self.c = pkg.KVBlockCache(heads, hd, blocks, self.d_codes, self.d_scales, self.d_sums)

    def download(self):
        self.ctx.synchronize()
        codes = take_apart(self.d_codes.download(np.int8, (self.blocks, self.heads, 2, TOKENS * self.hd)), self.hd)
        sums = self.d_sums.download(np.float32, self.sums.shape) if self.d_sums else None
        return codes, self.d_scales.download(np.float32, self.scales.shape), sums

    def numbers(self, table, length):
        """Tokens [0, length) of a sequence, [2, token, head, dimension] in fp32."""
        out = np.zeros((2, length, self.heads, self.hd), np.float32)
        for t in range(length):
            b = table[t // TOKENS]
            if 0 <= b < self.blocks:
                out[:, t] = (self.codes[b, :, :, t % TOKENS].astype(np.float32) * self.scales[b][..., None]).transpose(1, 0, 2)
        return out

    def append(self, table, first, x):
        """x: [2, token, head, dimension] at positions first, first + 1, ... (negative ones are dropped)."""
        n = x.shape[1]
        for j in range(max(first, 0) // TOKENS, -(-(first + n) // TOKENS)):
            lo, hi = max(first, 0, j * TOKENS) - j * TOKENS, min(first + n, (j + 1) * TOKENS) - j * TOKENS
            b = table[j]
            if not 0 <= b < self.blocks:
                continue
            for h in range(self.heads):
                for part in range(2):
                    y = x[part, j * TOKENS + lo - first:j * TOKENS + hi - first, h]
                    finite = np.abs(y[np.isfinite(y)])
                    top = np.float32(finite.max() if finite.size else 0)
                    old = self.scales[b, h, part] if lo else np.float32(0)
                    new = np.maximum(old, np.float32(top * INVERSE))
                    div = new if new > 0 else np.float32(1)
                    if new != old and lo:
                        ratio = np.float32(old / div)
                        self.codes[b, h, part, :lo] = np.rint(self.codes[b, h, part, :lo].astype(np.float32) * ratio).astype(np.int8)
                    q = np.clip(np.rint((y / div).astype(np.float32)), -127, 127)
                    self.codes[b, h, part, lo:hi] = np.where(np.isnan(y), 0, q).astype(np.int8)
                    self.scales[b, h, part] = new
                self.sums[b, h, lo:hi] = 0


def sequences(pkg, ctx, tables, lengths, rows, bounds=None):
    width = max(1, max(len(t) for t in tables))
    table = np.full((len(tables), width), -1, np.int32)
    for b, t in enumerate(tables):
        table[b, :len(t)] = t
    starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    most_rows, most = bounds or (max(rows), max(max(lengths), 1))
    return pkg.KVSequences(len(tables), ctx.upload(table), width, ctx.upload(np.array(lengths, np.int32)),
                           ctx.upload(starts), int(starts[-1]), most_rows, most)


def deal(rng, lengths, spare=0):
    """A table of distinct random blocks for every sequence, and the number of blocks."""
    counts = [-(-n // TOKENS) for n in lengths]
    ids = rng.permutation(sum(counts) + spare).astype(np.int32)
    at = np.concatenate([[0], np.cumsum(counts)])
    return [ids[at[i]:at[i + 1]].tolist() for i in range(len(counts))], ids[at[-1]:], len(ids)


def check_tokens(cache, tables, lengths):
    codes, scales, sums = cache.download()
    for table, n in zip(tables, lengths):
        for j, b in enumerate(table[:-(-n // TOKENS)]):
            if not 0 <= b < cache.blocks:
                continue
            have = min(TOKENS, n - j * TOKENS)
            assert np.array_equal(codes[b, :, :, :have], cache.codes[b, :, :, :have])
            assert np.array_equal(scales[b], cache.scales[b])
            if sums is not None:
                assert np.array_equal(sums[b, :, :have], cache.sums[b, :, :have])


ROUNDS = [
    # (head dimension, KV heads, dtype, row stride beyond the heads, appended rows of each sequence call after call)
    (128, 2, "BF16", 0, [[1, 1], [1, 1], [63, 130], [1, 5], [64, 1]]),
    (64, 3, "F16", 0, [[130, 1, 64], [1, 2, 1], [7, 200, 63]]),
    (256, 1, "F32", 0, [[65], [1], [62], [1], [200]]),
    (128, 1, "F32", 3, [[3, 90], [61, 1], [1, 1]]),          # rows that are not 16-byte aligned
    (64, 2, "BF16", 5, [[20], [44], [1]]),
    (256, 2, "F16", 8, [[1, 300], [2, 2]]),
]


@pytest.mark.parametrize("hd,heads,dtype,pad,calls", ROUNDS)
def test_append_and_read(pkg, ctx, hd, heads, dtype, pad, calls):
    rng = np.random.default_rng(hd + pad)
    dt = getattr(pkg, dtype)
    n = len(calls[0])
    total = np.sum(calls, 0)
    tables, _, blocks = deal(rng, total.tolist(), spare=2)
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)      # blocks hold what others left in them
    lengths = np.zeros(n, int)
    for rows in calls:
        lengths = lengths + rows
        x = rng.standard_normal((2, sum(rows), heads, hd)) * rng.choice([1e-3, 1.0, 30.0], (2, sum(rows), 1, 1))
        x = act_rounded(x.astype(np.float32), dt, pkg)
        seq = sequences(pkg, ctx, tables, lengths.tolist(), rows)
        width = heads * hd
        laid = np.zeros((2, sum(rows), width + pad), np.float32)
        laid[:, :, :width] = x.reshape(2, sum(rows), width)
        k, v = (ctx.upload(act_to_device_array(np.ascontiguousarray(y), dt, pkg)) for y in laid)
        ctx.kv_block_append(cache.c, seq, k, v, dt, width + pad if pad else 0)
        at = 0
        for b, r in enumerate(rows):
            cache.append(tables[b], int(lengths[b]) - r, x[:, at:at + r])
            at += r
        check_tokens(cache, tables, lengths.tolist())
        # what was written, read back, in every type
        for out_dtype in (pkg.F32, pkg.BF16, pkg.F16):
            nan = np.uint32(0x7FC00000) if out_dtype == pkg.F32 else np.uint16(0x7FC0)
            outs = [ctx.upload(np.full(sum(rows) * (width + pad), nan)) for _ in range(2)]
            ctx.kv_block_read(cache.c, seq, outs[0], outs[1], out_dtype, width + pad if pad else 0)
            ctx.synchronize()
            for part, o in enumerate(outs):
                got = out_from_device(o, out_dtype, (sum(rows), width + pad), pkg)
                want = np.concatenate([cache.numbers(tables[b], int(lengths[b]))[part, int(lengths[b]) - r:].reshape(r, width)
                                       for b, r in enumerate(rows)])
                assert np.array_equal(got[:, :width], act_rounded(want, out_dtype, pkg))
                assert np.all(np.isnan(got[:, width:]))


def test_values_that_are_no_numbers(pkg, ctx):
    """NaN becomes 0, infinities the ends of the scale, and neither sets the scale; an all-zero block has scale 0."""
    hd, heads = 64, 1
    cache = Cache(pkg, ctx, heads, hd, 2)
    x = np.zeros((2, 70, heads, hd), np.float32)
    x[0, :64] = np.linspace(-2, 2, 64)[None, None, :]
    x[0, 3, 0, :4] = [np.nan, np.inf, -np.inf, 1.0]
    x[1, 5, 0, 7] = np.inf                               # alone among zeros
    seq = sequences(pkg, ctx, [[1, 0]], [70], [70])
    ctx.kv_block_append(cache.c, seq, ctx.upload(x[0]), ctx.upload(x[1]), pkg.F32)
    cache.append([1, 0], 0, x)
    check_tokens(cache, [[1, 0]], [70])
    codes, scales, _ = cache.download()
    assert codes[1, 0, 0, 3, :3].tolist() == [0, 127, -127] and scales[1, 0, 0] == np.float32(np.float32(2) * INVERSE)
    assert scales[1, 0, 1] == 0 and scales[0, 0].tolist() == [0, 0]


def test_more_rows_than_tokens_and_absent_blocks(pkg, ctx):
    """Rows in front of the first token are dropped and read as zeros; so are tokens whose block id is out of range."""
    rng = np.random.default_rng(5)
    hd, heads = 128, 2
    cache = Cache(pkg, ctx, heads, hd, 3, rng)
    tables, lengths, rows = [[2, 7, 0], [1]], [150, 5], [150, 80]
    x = rng.standard_normal((2, 230, heads, hd)).astype(np.float32)
    seq = sequences(pkg, ctx, tables, lengths, rows)
    ctx.kv_block_append(cache.c, seq, ctx.upload(x[0]), ctx.upload(x[1]), pkg.F32)
    cache.append(tables[0], 0, x[:, :150])
    cache.append(tables[1], -75, x[:, 150:])
    check_tokens(cache, tables, lengths)
    outs = [ctx.alloc(230 * heads * hd * 4) for _ in range(2)]
    for o in outs:
        ctx.fill(o, 0x7FC00000)
    ctx.kv_block_read(cache.c, seq, outs[0], outs[1], pkg.F32)
    ctx.synchronize()
    for part in range(2):
        got = outs[part].download(np.float32, (230, heads, hd))
        assert np.array_equal(got[:150], cache.numbers(tables[0], 150)[part])
        assert not got[64:128].any() and not got[150:225].any()
        assert np.array_equal(got[225:], cache.numbers(tables[1], 5)[part])


def test_tables_that_make_no_sense_write_nothing(pkg, ctx):
    """Row starts that run backwards or past the rows, negative lengths, lengths beyond the table: no access outside."""
    hd, heads = 64, 1
    cache = Cache(pkg, ctx, heads, hd, 2)
    x = ctx.upload(np.ones((10, heads * hd), np.float32))
    table, lengths = ctx.upload(np.array([[0], [1], [0], [1]], np.int32)), ctx.upload(np.array([-5, 3, 4, 2 ** 30], np.int32))
    starts = ctx.upload(np.array([0, 2, 1, 99, -7], np.int32))
    seq = pkg.KVSequences(4, table, 1, lengths, starts, 10, 10, 1000)
    ctx.kv_block_append(cache.c, seq, x, x, pkg.F32)
    codes, scales, _ = cache.download()
    assert not codes.any() and not scales.any()


# ---- eviction ------------------------------------------------------------------------------------------------------------
def plain_evict(cache, table, length, budget, recent, sinks, new_table):
    """Returns per head the kept positions; brings the host copy of the new blocks up to date."""
    kept_of = []
    for h in range(cache.heads):
        if length <= budget:
            kept = list(range(length))
        else:
            weight = {}
            for t in range(sinks, length - recent):
                b = table[t // TOKENS]
                w = cache.sums[b, h, t % TOKENS] if 0 <= b < cache.blocks else np.float32(0)
                weight[t] = -np.inf if np.isnan(w) else w
            order = sorted(weight, key=lambda t: (-weight[t], t))
            kept = sorted(list(range(sinks)) + order[:budget - sinks - recent] + list(range(length - recent, length)))
        kept_of.append(kept)
    for j, target in enumerate(new_table[:-(-budget // TOKENS)]):
        codes = np.zeros((cache.heads, 2, TOKENS, cache.hd), np.int8)
        scales, sums = np.zeros((cache.heads, 2), np.float32), np.zeros((cache.heads, TOKENS), np.float32)
        for h in range(cache.heads):
            here = kept_of[h][j * TOKENS:(j + 1) * TOKENS]
            src = [(table[t // TOKENS], t % TOKENS) for t in here]
            for part in range(2):
                own = np.array([cache.scales[b, h, part] if 0 <= b < cache.blocks else 0 for b, _ in src] or [0], np.float32)
                scales[h, part] = own.max()
                for i, (b, t) in enumerate(src):
                    if 0 <= b < cache.blocks:
                        ratio = np.float32(own[i] / (own.max() if own.max() > 0 else np.float32(1)))
                        codes[h, part, i] = np.rint(cache.codes[b, h, part, t].astype(np.float32) * ratio).astype(np.int8)
                        sums[h, i] = cache.sums[b, h, t]
        yield target, codes, scales, sums
    yield None, kept_of, None, None


EVICTIONS = [
    # (head dimension, KV heads, lengths, budget, recent, sinks)
    (128, 2, [300, 64, 65, 129], 100, 20, 4),
    (64, 1, [1000], 64, 0, 0),
    (256, 3, [130, 1], 129, 129, 0),          # the budget is all recent tokens
    (64, 2, [5000, 2049], 1999, 100, 64),     # several rounds of the selecting workgroup
    (128, 1, [90], 1, 0, 1),                  # one token is left
    (64, 1, [200, 0, 100], 100, 0, 0),        # an empty sequence; one exactly on budget
    (64, 1, [333], 65, 0, 65),
]


@pytest.mark.parametrize("ties", [False, True])
@pytest.mark.parametrize("hd,heads,lengths,budget,recent,sinks", EVICTIONS)
def test_evict(pkg, ctx, hd, heads, lengths, budget, recent, sinks, ties):
    rng = np.random.default_rng(budget + ties)
    per = -(-budget // TOKENS)
    tables, free, blocks = deal(rng, lengths, spare=per * len(lengths) + 1)
    new_tables = free[:per * len(lengths)].reshape(len(lengths), per)
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)
    if ties:                                  # few different sums, zeros of both signs and no numbers among them
        cache.sums[:] = rng.choice(np.array([0.0, -0.0, 1.0, 2.5, np.nan, np.inf, -1.0], np.float32), cache.sums.shape)
        cache.d_sums.upload(cache.sums)
    seq = sequences(pkg, ctx, tables, lengths, [1] * len(lengths))
    new_lengths, positions = ctx.upload(np.full(len(lengths), -1, np.int32)), ctx.upload(np.full((len(lengths), heads, budget), -7, np.int32))
    ctx.kv_block_evict(cache.c, seq, budget, ctx.upload(new_tables), per, new_lengths, recent, sinks, positions)
    codes, scales, sums = cache.download()
    assert new_lengths.download(np.int32, (len(lengths),)).tolist() == [min(n, budget) for n in lengths]
    got = positions.download(np.int32, (len(lengths), heads, budget))
    for b, n in enumerate(lengths):
        for target, want_codes, want_scales, want_sums in plain_evict(cache, tables[b], n, budget, recent, sinks, new_tables[b].tolist()):
            if target is None:
                for h, kept in enumerate(want_codes):
                    assert got[b, h, :len(kept)].tolist() == kept
                    assert np.all(got[b, h, len(kept):] == -7)
                continue
            assert np.array_equal(codes[target], want_codes)
            assert np.array_equal(scales[target], want_scales)
            assert np.array_equal(sums[target], want_sums, equal_nan=True)
    # without positions (they live in the context's scratch then), the same blocks
    again = Cache(pkg, ctx, heads, hd, blocks, np.random.default_rng(1))
    again.d_codes.upload(lay_out(cache.codes)); again.d_scales.upload(cache.scales); again.d_sums.upload(cache.sums)
    ctx.kv_block_evict(again.c, seq, budget, ctx.upload(new_tables), per, new_lengths, recent, sinks)
    codes2, scales2, sums2 = again.download()
    picked = new_tables.ravel()
    assert np.array_equal(codes2[picked], codes[picked]) and np.array_equal(scales2[picked], scales[picked])
    assert np.array_equal(sums2[picked], sums[picked], equal_nan=True)


LONG = [
    # (KV heads, lengths, longest the host knows of, budget, recent, sinks)
    (2, [40000, 200, 16385, 0, 16384], 40000, 9001, 1000, 4),
    (1, [70003], 70003, 60000, 0, 0),
    (3, [20000, 33000], 50000, 1, 0, 0),
    (1, [17000, 30001], 30001, 5000, 4000, 1000),         # nothing competes
    (1, [100, 16000], 20000, 300, 5, 64),                 # chunks behind the sequences
    (1, [2_200_000], 2_200_000, 100_000, 64, 4),          # chunks of more than 1024 blocks
    (140, [16500] * 4, 16500, 1000, 64, 4),               # two chunks a sequence
]


@pytest.mark.parametrize("sums", ["spread", "ties", "zeros", "close"])
@pytest.mark.parametrize("heads,lengths,longest,budget,recent,sinks", LONG)
def test_evict_long(pkg, ctx, heads, lengths, longest, budget, recent, sinks, sums):
    """Sequences whose tokens are selected by several workgroups: positions against a stable sort, new lengths, and the sums
    that go along with the tokens."""
    rng = np.random.default_rng(len(lengths) + budget)
    hd, per = 64, -(-budget // TOKENS)
    tables, free, blocks = deal(rng, lengths, spare=per * len(lengths))
    new_tables = free.reshape(len(lengths), per)
    shape = (blocks, heads, TOKENS)
    if sums == "spread":
        own = (6 * rng.random(shape) ** 4).astype(np.float32)
    elif sums == "ties":
        own = rng.choice(np.array([0.0, -0.0, 1.0, 2.5, np.nan, np.inf, -1.0, 1.0000001], np.float32), shape)
    elif sums == "zeros":
        own = np.zeros(shape, np.float32)
    else:                                     # all sums begin with the same eleven bits, many are equal
        own = (1.0 + rng.integers(0, 3000, shape) * 2.0 ** -23).astype(np.float32)
    d_sums, scales = ctx.upload(own), ctx.alloc(blocks * heads * 2 * 4)
    codes = ctx.alloc(pkg.KVBlockCache.codes_bytes(heads, hd, blocks))
    ctx.fill(scales, 0x3F800000); ctx.fill(codes, 0)
    cache = pkg.KVBlockCache(heads, hd, blocks, codes, scales, d_sums)
    seq = sequences(pkg, ctx, tables, lengths, [1] * len(lengths), (1, longest))
    new_lengths, positions = ctx.upload(np.full(len(lengths), -1, np.int32)), ctx.upload(np.full((len(lengths), heads, budget), -7, np.int32))
    ctx.kv_block_evict(cache, seq, budget, ctx.upload(new_tables), per, new_lengths, recent, sinks, positions)
    ctx.synchronize()
    assert new_lengths.download(np.int32, (len(lengths),)).tolist() == [min(n, budget) for n in lengths]
    got = positions.download(np.int32, (len(lengths), heads, budget))
    after = d_sums.download(np.float32, shape)
    for b, n in enumerate(lengths):
        weight = own[tables[b]].transpose(1, 0, 2).reshape(heads, -1)[:, :n] if n else np.zeros((heads, 0), np.float32)
        moved = after[new_tables[b]].transpose(1, 0, 2).reshape(heads, -1)
        for h in range(heads):
            kept = np.arange(n)
            if n > budget:
                middle = np.nan_to_num(weight[h, sinks:n - recent], nan=-np.inf, posinf=np.inf, neginf=-np.inf)
                order = np.argsort(-middle, kind="stable")[:budget - sinks - recent] + sinks
                kept = np.concatenate([np.arange(sinks), np.sort(order), np.arange(n - recent, n)])
            assert np.array_equal(got[b, h, :len(kept)], kept)
            assert np.all(got[b, h, len(kept):] == -7)
            assert np.array_equal(moved[h, :len(kept)], weight[h, kept], equal_nan=True)
            assert not moved[h, len(kept):].any()
    for buf in (codes, scales, d_sums, positions, new_lengths):
        buf.free()


def test_evict_with_absent_blocks(pkg, ctx):
    rng = np.random.default_rng(3)
    cache = Cache(pkg, ctx, 1, 64, 8, rng)
    table, new_table = [3, 99, 1, -1], [5, 0]
    seq = sequences(pkg, ctx, [table], [240], [1])
    new_lengths, positions = ctx.alloc(4), ctx.alloc(100 * 4)
    ctx.kv_block_evict(cache.c, seq, 100, ctx.upload(np.array([new_table], np.int32)), 2, new_lengths, 10, 0, positions)
    codes, scales, sums = cache.download()
    for target, want_codes, want_scales, want_sums in plain_evict(cache, table, 240, 100, 10, 0, new_table):
        if target is None:
            assert positions.download(np.int32, (100,)).tolist() == want_codes[0]
        else:
            assert np.array_equal(codes[target], want_codes) and np.array_equal(scales[target], want_scales)
            assert np.array_equal(sums[target], want_sums)


# ---- refusals ------------------------------------------------------------------------------------------------------------
def test_refusals(pkg, ctx):
    cache = Cache(pkg, ctx, 2, 64, 4)
    seq = sequences(pkg, ctx, [[0, 1]], [100], [3])
    x = ctx.alloc(3 * 128 * 4)
    table, lengths = ctx.upload(np.zeros(4, np.int32)), ctx.alloc(4)

    def refused(status, call, *args, **kw):
        with pytest.raises(pkg.MI355QError) as e:
            call(*args, **kw)
        assert e.value.status_name == status, str(e.value)

    def other(**kw):
        c = cache.c._c
        values = {n: getattr(c, n) for n, _ in c._fields_}
        values.update(kw)
        new = pkg.KVBlockCache(1, 64, 1, 0, 0)
        for n, v in values.items():
            setattr(new._c, n, v)
        return new

    def others(**kw):
        c = seq._c
        new = pkg.KVSequences(1, 0, 1, 0, 0, 1, 1, 1)
        for n, _ in c._fields_:
            setattr(new._c, n, kw.get(n, getattr(c, n)))
        return new

    for call in (ctx.kv_block_append, ctx.kv_block_read):
        refused("UNSUPPORTED_FORMAT", call, other(head_dimension=96), seq, x, x, pkg.F32)
        refused("SHAPE", call, other(kv_head_count=0), seq, x, x, pkg.F32)
        refused("SHAPE", call, other(block_count=0), seq, x, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, other(codes_dev=None), seq, x, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, other(codes_dev=cache.d_codes.ptr + 8), seq, x, x, pkg.F32)
        refused("SHAPE", call, cache.c, others(sequence_count=0), x, x, pkg.F32)
        refused("SHAPE", call, cache.c, others(maximum_rows=4), x, x, pkg.F32)
        refused("SHAPE", call, cache.c, others(maximum_rows=0), x, x, pkg.F32)
        refused("SHAPE", call, cache.c, others(maximum_length=0), x, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, cache.c, others(lengths_dev=None), x, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, cache.c, others(row_starts_dev=None), x, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, cache.c, seq, None, x, pkg.F32)
        refused("INVALID_ARGUMENT", call, cache.c, seq, x, x, 7)
        refused("INVALID_ARGUMENT", call, cache.c, seq, x.ptr + 1, x, pkg.F16)
        refused("SHAPE", call, cache.c, seq, x, x, pkg.F32, 127)
    refused("INVALID_ARGUMENT", ctx.kv_block_evict, other(weight_sums_dev=None), seq, 64, table, 1, lengths)
    refused("INVALID_ARGUMENT", ctx.kv_block_evict, cache.c, seq, 64, None, 1, lengths)
    refused("SHAPE", ctx.kv_block_evict, cache.c, seq, 0, table, 1, lengths)
    refused("SHAPE", ctx.kv_block_evict, cache.c, seq, 65, table, 1, lengths)
    refused("SHAPE", ctx.kv_block_evict, cache.c, seq, 64, table, 1, lengths, recent=60, sinks=5)


@pytest.mark.parametrize("size", [1e-38, 1e-36, 1e-28, 1e-4, 1.0, 1e20, 3e38])
def test_codes_near_the_middle_of_two(pkg, ctx, size):
    """Numbers around the middles between codes, at scales from subnormal ones to the largest: the codes of a division."""
    rng = np.random.default_rng(8)
    hd, length = 128, 128
    tables, _, blocks = deal(rng, [length])
    cache = Cache(pkg, ctx, 1, hd, blocks)
    scale = np.float32(np.float32(size) * INVERSE)
    x = ((rng.integers(-126, 127, (2, length, 1, hd)) + rng.choice([0.0, 0.5, 0.49], (2, length, 1, hd))) * np.float64(scale)).astype(np.float32)
    step = rng.integers(-1, 2, x.shape)
    x = np.where(step > 0, np.nextafter(x, np.float32(np.inf)), np.where(step < 0, np.nextafter(x, np.float32(-np.inf)), x))
    x[:, ::64, 0, 0] = np.float32(size)                      # the largest of each block
    k, v = (ctx.upload(np.ascontiguousarray(x[i].reshape(length, hd))) for i in range(2))
    ctx.kv_block_append(cache.c, sequences(pkg, ctx, tables, [length], [length]), k, v, pkg.F32)
    cache.append(tables[0], 0, x)
    check_tokens(cache, tables, [length])


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("sinks", [1, 2, 31, 32, 33, 63])
def test_evict_across_the_first_block_of_the_pool(pkg, ctx, hd, sinks):
    """`sinks` tokens of a block and the others from block 0, which the second lane of a half meets first."""
    rng = np.random.default_rng(sinks)
    cache = Cache(pkg, ctx, 2, hd, 4, rng)
    table, new_table, budget = [2, 0], [1], 64
    seq = sequences(pkg, ctx, [table], [128], [1])
    ctx.kv_block_evict(cache.c, seq, budget, ctx.upload(np.array([new_table], np.int32)), 1, ctx.alloc(4), budget - sinks, sinks)
    codes, scales, sums = cache.download()
    for target, want_codes, want_scales, want_sums in plain_evict(cache, table, 128, budget, budget - sinks, sinks, new_table):
        if target is not None:
            assert np.array_equal(codes[target], want_codes) and np.array_equal(scales[target], want_scales)
            assert np.array_equal(sums[target], want_sums)
