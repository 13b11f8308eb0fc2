"""GPU tests of the block cache's operators together: plan steps replayed from a captured graph, and the serving loop."""
import importlib.util
import os
import sys

import numpy as np
import pytest

from gpu_util import act_rounded, act_to_device_array, out_from_device
from test_gpu_kv_block_attention import plain
from test_gpu_kv_block_cache import TOKENS, Cache, deal, sequences, take_apart

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(pkg):
    path = os.path.join(os.path.dirname(pkg.__file__), "block_cache_decode.py")
    spec = importlib.util.spec_from_file_location("block_cache_decode", path)
    mod = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = mod
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("hd,heads,group,rows", [(128, 2, 4, 1), (64, 2, 4, 7), (64, 1, 4, 33), (256, 1, 2, 40)])
def test_steps_in_a_graph_replayed_with_other_lengths(pkg, ctx, hd, heads, group, rows):
    """Append, attention with weight sums and log probabilities as plan steps: a graph built once, with lengths of 0, gives
    the bits of the direct calls for every length, block table and input it is replayed with, with other work of the
    context in between; codes, scales and sums stay equal as well."""
    rng = np.random.default_rng(hd + rows)
    count, longest, vocabulary = 3, 900, 5003
    tables, _, blocks = deal(rng, [longest] * count, spare=0)
    width = heads * group * hd
    one, two = Cache(pkg, ctx, heads, hd, blocks, np.random.default_rng(5)), Cache(pkg, ctx, heads, hd, blocks, np.random.default_rng(5))
    total = count * rows
    # tables with contents of their own for the graph; the direct calls get theirs afresh each time
    table = np.stack([np.asarray(t, np.int32) for t in tables])
    table_dev, lengths_dev = ctx.upload(table), ctx.upload(np.zeros(count, np.int32))
    starts_dev = ctx.upload(np.arange(count + 1, dtype=np.int32) * rows)
    seq = pkg.KVSequences(count, table_dev, table.shape[1], lengths_dev, starts_dev, total, rows, longest)
    q, k, v = (ctx.alloc(total * n * 2) for n in (width, heads * hd, heads * hd))
    logits, tokens = ctx.alloc(total * vocabulary * 4), ctx.alloc(total * 4)
    outs = [(ctx.alloc(total * width * 2), ctx.alloc(total * heads * group * 4), ctx.alloc(total * 4), ctx.alloc(total * 4),
             ctx.alloc(total * 12), ctx.alloc(total * 12)) for _ in range(2)]
    stream = ctx.stream_create()
    plan = pkg.DispatchPlan(ctx)
    out, lse, lp, ent, ids, tops = outs[0]
    plan.add_kv_block_append(one.c, seq, k, v, pkg.BF16, layer_index=3, tensor_name="layer.3.cache")
    plan.add_kv_block_attention(one.c, seq, q, pkg.BF16, heads * group, out, pkg.BF16, hd ** -0.5, lse=lse, accumulate_weights=True,
                                layer_index=3)
    plan.add_token_logprobs(logits, pkg.F32, total, vocabulary, tokens, 3, lp, ent, ids, tops)
    assert len(plan) == 3
    steps = [plan.step(i) for i in range(3)]
    assert [s[0].kernel_name for s in steps] == ["kv_block_append", "kv_block_attention", "token_logprobs"]
    before = one.download()
    plan.graph_build(stream)
    ctx.synchronize(stream)
    for was, now in zip(before, one.download()):
        assert np.array_equal(was, now), "building the graph has touched the cache"
    with pytest.raises(pkg.MI355QError):
        plan.add_kv_block_append(one.c, seq, k, v, pkg.BF16)
    lengths = np.array([rows, 0, 100])
    for rep in range(5):
        for buf, n in ((q, width), (k, heads * hd), (v, heads * hd)):
            buf.upload(act_to_device_array(rng.standard_normal((total, n)).astype(np.float32), pkg.BF16, pkg))
        logits.upload(rng.standard_normal((total, vocabulary)).astype(np.float32))
        tokens.upload(rng.integers(0, vocabulary, total).astype(np.int32))
        lengths = np.minimum(lengths + rng.integers(rows, 200 + rows, count), longest) if rep else lengths
        if rep == 3:
            table = table[:, ::-1].copy()                       # other blocks in the places
            table_dev.upload(table)
        lengths_dev.upload(lengths.astype(np.int32))
        for b in outs[0] + outs[1]:
            ctx.fill(b, 0x7FC07FC0)
        ctx.synchronize()
        plan.graph_launch(stream)
        ctx.synchronize(stream)
        out, lse, lp, ent, ids, tops = outs[1]
        ctx.kv_block_append(two.c, seq, k, v, pkg.BF16)
        ctx.kv_block_attention(two.c, seq, q, pkg.BF16, heads * group, out, pkg.BF16, hd ** -0.5, lse=lse, accumulate_weights=True)
        ctx.token_logprobs(logits, pkg.F32, total, vocabulary, tokens, 3, lp, ent, ids, tops)
        ctx.synchronize()
        for a, b in zip(outs[0], outs[1]):
            assert np.array_equal(a.download(np.uint32), b.download(np.uint32)), f"replay {rep}"
        for a, b in zip(one.download(), two.download()):
            assert np.array_equal(a, b), f"replay {rep}"
    plan.destroy()
    ctx.stream_destroy(stream)


def test_refusals_of_the_steps(pkg, ctx):
    cache = Cache(pkg, ctx, 2, 64, 4)
    bare = pkg.KVBlockCache(2, 64, 4, cache.d_codes, cache.d_scales)
    seq = sequences(pkg, ctx, [[0, 1]], [70], [1])
    buf = ctx.alloc(4096)
    plan = pkg.DispatchPlan(ctx)
    for call in (lambda: plan.add_kv_block_append(cache.c, seq, None, buf, pkg.BF16),
                 lambda: plan.add_kv_block_append(cache.c, seq, buf, buf, 9),
                 lambda: plan.add_kv_block_attention(cache.c, seq, buf, pkg.F32, 4, buf, pkg.BF16, 0.125),
                 lambda: plan.add_kv_block_attention(cache.c, seq, buf, pkg.BF16, 3, buf, pkg.BF16, 0.125),
                 lambda: plan.add_kv_block_attention(bare, seq, buf, pkg.BF16, 4, buf, pkg.BF16, 0.125, accumulate_weights=True),
                 lambda: plan.add_token_logprobs(buf, pkg.F32, 1, 100),
                 lambda: plan.add_token_logprobs(None, pkg.F32, 1, 100, entropy=buf)):
        with pytest.raises(pkg.MI355QError):
            call()
    assert len(plan) == 0
    plan.destroy()


def test_serving_loop(pkg, ctx, example):
    """Ragged prompts, then decoding across two evictions, from a graph and with direct launches of the same steps: the
    same tokens and the same bits of the log probabilities.  What the last step left in memory is checked in 64 bits: the
    attention of the last layer against the cache's numbers, the log probabilities against the logits."""
    runs = []
    for graph in (True, False):
        d = example.BlockCacheDecoder(pkg, ctx, sequences=3, limit=128, budget=70, sinks=2, recent=16, vocabulary=1000)
        prompts = [d.rng.integers(0, d.vocabulary, n) for n in (100, 1, 64)]
        scored = d.prompts(prompts)
        steps = [d.step(graph) for _ in range(100)]
        # 100 tokens reach 128 after 28 steps, then fall to 70 before every 58th further one; the prompt of one token has
        # 29 by then and 87 at the second eviction, that of 64 has 92 and falls to 70 with the others both times
        assert d.evictions == 2 and d.lengths.tolist() == [84, 84, 84]
        cache, b = d.caches[-1], d.buffers
        hd, total = d.head_dimension, cache.block_count
        codes, scales, _ = cache._keepalive
        host = Cache.__new__(Cache)
        host.blocks, host.heads, host.hd = total, d.kv_heads, hd
        host.codes = take_apart(codes.download(np.int8, (total, d.kv_heads, 2, TOKENS * hd)), hd)
        host.scales = scales.download(np.float32, (total, d.kv_heads, 2))
        host.sums = np.zeros((total, d.kv_heads, TOKENS))
        q = out_from_device(b["q"], pkg.BF16, (3, d.heads, hd), pkg)
        want, _, _ = plain(host, d.table_dev.download(np.int32, (3, d.blocks)), d.lengths, [1, 1, 1], q, d.heads // d.kv_heads,
                           hd ** -0.5, 0)
        got = out_from_device(b["attended"], pkg.BF16, (3, d.heads, hd), pkg)
        top = 127 * host.scales[..., 1].max()
        assert np.all(np.abs(got - want) <= 2.0 ** -11 * top + 2.0 ** -8 * np.abs(want) + 1e-6)
        z = b["logits"].download(np.float32, (3, d.vocabulary)).astype(np.float64)
        logs = z - z.max(1, keepdims=True)
        logs -= np.log(np.exp(logs).sum(1, keepdims=True))
        tokens, chosen, entropy = steps[-1]
        assert np.array_equal(tokens, z.argmax(1))
        # fp32 sums of 1000 terms and one logarithm: far below 2^-16 of the numbers' size
        assert np.all(np.abs(chosen - logs.max(1)) <= 2.0 ** -16 * (1 + np.abs(logs.max(1))))
        assert np.all(np.abs(entropy + (np.exp(logs) * logs).sum(1)) <= 2.0 ** -14 * (1 + np.abs(entropy)))
        runs.append((scored, steps, d.lengths.copy()))
        d.close()
    (scored, steps, lengths), (scored2, steps2, lengths2) = runs
    assert all(np.array_equal(a, b) for a, b in zip(scored, scored2)) and np.array_equal(lengths, lengths2)
    for a, b in zip(steps, steps2):
        assert all(np.array_equal(x, y) for x, y in zip(a, b))


def test_eviction_follows_the_weights_of_the_attention(pkg, ctx):
    """Attention with weight sums over several tiles and shares of rows, then eviction: the kept positions are the sinks,
    the last tokens and the tokens with most weight of the plain implementation; positions whose plain sums lie within the
    sums' tolerance of the lowest kept one are free to go either way."""
    rng = np.random.default_rng(77)
    hd, heads, group, length, rows, budget, recent, sinks = 64, 2, 4, 700, 300, 200, 32, 4
    tables, free, blocks = deal(rng, [length], spare=-(-budget // TOKENS))
    cache = Cache(pkg, ctx, heads, hd, blocks, rng)
    cache.sums[:] = 0
    cache.d_sums.upload(cache.sums)
    q = act_rounded((rng.standard_normal((rows, heads * group, hd)) * 0.2).astype(np.float32), pkg.BF16, pkg)
    seq = sequences(pkg, ctx, tables, [length], [rows])
    out = ctx.alloc(q.size * 2)
    ctx.kv_block_attention(cache.c, seq, ctx.upload(act_to_device_array(q.reshape(rows, -1), pkg.BF16, pkg)), pkg.BF16, heads * group,
                           out, pkg.BF16, hd ** -0.5, accumulate_weights=True)
    lengths, positions = ctx.alloc(4), ctx.alloc(heads * budget * 4)
    ctx.kv_block_evict(cache.c, seq, budget, ctx.upload(free), len(free), lengths, recent, sinks, positions)
    ctx.synchronize()
    assert lengths.download(np.int32)[0] == budget
    kept = positions.download(np.int32, (heads, budget))
    _, _, added = plain(cache, tables, [length], [rows], q, group, hd ** -0.5, 0)
    for h in range(heads):
        w = np.array([added[tables[0][t // TOKENS], h, t % TOKENS] for t in range(length)])
        assert np.all(np.diff(kept[h]) > 0)
        middle = np.arange(sinks, length - recent)
        assert set(range(sinks)) <= set(kept[h]) and set(range(length - recent, length)) <= set(kept[h])
        order = np.sort(w[middle])[::-1]
        limit, slack = order[budget - sinks - recent - 1], 4e-4 * max(order[budget - sinks - recent - 1], 1e-3)
        must = set(middle[w[middle] > limit + slack])
        may = set(middle[w[middle] >= limit - slack])
        mid = set(kept[h]) & set(middle)
        assert must <= mid <= may


def test_offsets_beyond_32_bits(pkg, ctx):
    """Blocks more than 2^32 bytes into the codes, and rows more than 2^32 elements into their tensors: the same bits as the
    same work on a small cache and dense rows."""
    rng = np.random.default_rng(9)
    hd, heads, group, small, far, lengths, rows = 256, 8, 1, 12, 20000, [300, 200], [68, 2]
    total, width, stride = sum(rows), heads * group * hd, 1 << 26
    assert far * heads * 2 * TOKENS * hd > 2 ** 32 and (total - 1) * stride > 2 ** 32
    near = Cache(pkg, ctx, heads, hd, small, rng)
    shift = far - small
    sizes = [heads * 2 * TOKENS * hd, heads * 2 * 4, heads * TOKENS * 4]                 # bytes of a block
    big = [ctx.alloc(far * n) for n in sizes]
    parts = [pkg.DeviceBuffer(ctx, b.offset(shift * n), small * n) for b, n in zip(big, sizes)]
    for part, own in zip(parts, (near.d_codes, near.d_scales, near.d_sums)):
        ctx.copy(part, own, own.nbytes)
    ctx.synchronize()
    cache = pkg.KVBlockCache(heads, hd, far, *big)
    tables = [[0, 3, 1, 5, 2], [4, 9, 6, 7]]
    seqs = sequences(pkg, ctx, tables, lengths, rows), sequences(pkg, ctx, [[b + shift for b in t] for t in tables], lengths, rows)
    q, k, v = (act_to_device_array(rng.standard_normal((total, width)).astype(np.float32), pkg.BF16, pkg) for _ in range(3))
    dense = [ctx.upload(x) for x in (q, k, v)] + [ctx.alloc(total * width * 2) for _ in range(3)]
    wide = ctx.alloc(total * stride * 2)                     # q, k, v, output and the rows read back, side by side
    columns = [pkg.DeviceBuffer(ctx, wide.offset(i * width * 2), 0) for i in range(6)]
    for column, x in zip(columns, (q, k, v)):
        for r in range(total):
            pkg.DeviceBuffer(ctx, column.offset(r * stride * 2), width * 2).upload(x[r])
    for c, seq, bufs, step in ((near.c, seqs[0], dense, 0), (cache, seqs[1], columns, stride)):
        ctx.kv_block_append(c, seq, bufs[1], bufs[2], pkg.BF16, step)
        ctx.kv_block_attention(c, seq, bufs[0], pkg.BF16, heads * group, bufs[3], pkg.BF16, hd ** -0.5, accumulate_weights=True,
                               q_row_stride=step, out_row_stride=step)
        ctx.kv_block_read(c, seq, bufs[4], bufs[5], pkg.BF16, step)
    ctx.synchronize()
    for i in (3, 4, 5):
        want = dense[i].download(np.uint16, (total, width))
        for r in range(total):
            got = pkg.DeviceBuffer(ctx, columns[i].offset(r * stride * 2), width * 2).download(np.uint16)
            assert np.array_equal(got, want[r]), f"tensor {i}, row {r}"
    for part, own in zip(parts, (near.d_codes, near.d_scales, near.d_sums)):
        assert np.array_equal(part.download(np.uint8), own.download(np.uint8))
    new = np.array([[8, 10], [11, -1]], np.int32)
    far_new = np.where(new < 0, far, new + shift).astype(np.int32)
    for c, seq, table in ((near.c, seqs[0], new), (cache, seqs[1], far_new)):
        ctx.kv_block_evict(c, seq, 100, ctx.upload(table), 2, ctx.alloc(8), 10, 4)
    ctx.synchronize()
    for part, own in zip(parts, (near.d_codes, near.d_scales, near.d_sums)):
        assert np.array_equal(part.download(np.uint8), own.download(np.uint8))
    vocabulary, pitch = 5000, stride // 2
    logits = rng.standard_normal((total, vocabulary)).astype(np.float32)
    for r in range(total):
        pkg.DeviceBuffer(ctx, wide.offset(r * pitch * 4), vocabulary * 4).upload(logits[r])
    results = []
    for buf, step in ((ctx.upload(logits), 0), (wide, pitch)):
        ids, tops, entropy = ctx.alloc(total * 12), ctx.alloc(total * 12), ctx.alloc(total * 4)
        ctx.token_logprobs(buf, pkg.F32, total, vocabulary, None, 3, None, entropy, ids, tops, step)
        ctx.synchronize()
        results.append((ids.download(np.int32), tops.download(np.float32), entropy.download(np.float32)))
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    for b in big + [wide] + dense:
        b.free()
