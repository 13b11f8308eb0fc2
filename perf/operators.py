"""The attention step over the 8-bit block cache and what stands behind the output head, as measurable cases.

Four kinds of pass, each one call (or the write and the read back of one cache) of the public entry points:

``append``    the keys and values of new tokens go into the block cache; the blocks they touched are read back as numbers.
``attend``    attention of the sequences' new rows over the cache: decode steps, a few tokens to verify, prompts and
              prompt chunks; with ``weights`` the attention weight every cached token received is added up for eviction.
``evict``     a cache over its budget is reduced to the tokens that received most weight; what is kept is read back.
``logprobs``  log probability of the given token, entropy and the likeliest alternatives of rows of logits.

4096 / 8 KV heads of 128 with 32 query heads is the layer of the benchmark at the root of the repository, 65536 the
vocabulary of its output head; other sizes are generic.

The cache: blocks of 64 tokens and one KV head, int8 codes with one fp32 scale for the block's keys and one for its
values.  Codes stand in the order the matrix cores take them: keys as [16-token tile][64 dimensions][16 dimensions]
[token][dimension], values as [16 dimensions][tokens 4c .. 4c+3 of each 16][dimension][32 tokens][16 tokens][token].
"""
import importlib
import math

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 64
STEPS = 127.49      # half of a block's largest magnitude is then no midpoint between two codes


def _append(name, sequences, history, rows, kv_heads=8, head_dim=128, x="bf16"):
    return {"name": name, "kind": "append", "sequences": sequences, "history": history, "rows": rows,
            "kv_heads": kv_heads, "head_dim": head_dim, "x": x}


def _attend(name, sequences, history, rows, heads=32, kv_heads=8, head_dim=128, x="bf16", window=0, weights=False):
    return {"name": name, "kind": "attend", "sequences": sequences, "history": history, "rows": rows, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "x": x, "window": window, "weights": weights}


def _evict(name, sequences, length, budget, recent, sinks, kv_heads=8, head_dim=128, x="bf16"):
    return {"name": name, "kind": "evict", "sequences": sequences, "history": length, "budget": budget, "recent": recent,
            "sinks": sinks, "kv_heads": kv_heads, "head_dim": head_dim, "x": x}


def _logprobs(name, rows, vocabulary, top, x="f32"):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocabulary": vocabulary, "top": top, "x": x}


def listed():
    return [
        # a serving batch adds one token to every sequence, most of them in the middle of a block
        _append("append_tokens_b48", 48, 3001, 1),
        # a long prompt is written at once
        _append("append_prompt_4096", 1, 0, 4096, x="f16"),
        # one sequence of a chat's length: two dependent launches of microseconds, where latency is everything
        _attend("attend_token_517", 1, 516, 1),
        # a serving batch of ragged lengths that keeps account of every token's weight for eviction
        _attend("attend_tokens_b32_weights", 32, 8191, 1, weights=True),
        # two sequences of very long context with groups of eight heads, f16 activations (the reference's decode type)
        _attend("attend_token_131071_f16", 2, 131070, 1, heads=64, x="f16"),
        # five draft tokens verified at once on a model with small heads and a sliding window
        _attend("attend_verify_window_hd64", 16, 4000, 5, heads=24, kv_heads=4, head_dim=64, window=1024),
        # a long prompt of odd length on the benchmark's layer
        _attend("attend_prompt_5001", 1, 0, 5001),
        # chunks of three prompts of ragged lengths on what is cached of them, wide heads, weights wanted
        _attend("attend_chunk_hd256_weights", 3, 5800, 509, heads=16, kv_heads=4, head_dim=256, x="f16", weights=True),
        # a batch at the end of its budget
        _evict("evict_b8_8192", 8, 8192, 2048, 256, 4),
        # one very long document reduced to an odd number of tokens
        _evict("evict_60001_hd64", 1, 60001, 5003, 1000, 0, kv_heads=4, head_dim=64, x="f16"),
        # the token that was just sampled, with its alternatives, from the head's fp32 logits
        _logprobs("logprobs_1_65536", 1, 65536, 5),
        # a prompt's own log probabilities over an odd vocabulary, bf16 logits full of equal values
        _logprobs("logprobs_777_100003_bf16", 777, 100003, 20, x="bf16"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choices(["append", "attend", "evict", "logprobs"], [2, 6, 2, 2])[0]
    x = rng.choice(["bf16", "f16"])
    head_dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    per_token = 2 * head_dim * kv_heads
    if kind == "append":
        x = rng.choice(["bf16", "f16", "f32"])
        if rng.random() < 0.5:
            return _nameless(_append("", _log_int(rng, 1, 64), _log_int(rng, 1, 4096), _log_int(rng, 1, 8), kv_heads, head_dim, x))
        return _nameless(_append("", _log_int(rng, 1, 4), rng.choice([0, _log_int(rng, 1, 2000)]),
                                 _log_int(rng, 64, 2048), kv_heads, head_dim, x))
    if kind == "attend":
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 6, 8])
        weights = rng.random() < 0.35
        if rng.random() < 0.6:      # decode steps and short verifications
            sequences = _log_int(rng, 1, 48)
            most = max(64, min(131072, 250_000_000 // (per_token * sequences)))
            window = rng.choice([0, 0, 0, _log_int(rng, 100, 4096)])
            return _nameless(_attend("", sequences, _log_int(rng, 16, most), rng.choice([1, 1, 1, rng.randint(2, 8)]),
                                     heads, kv_heads, head_dim, x, window, weights))
        rows = _log_int(rng, 16, 2048)
        sequences = rng.randint(1, max(1, min(4, 1024 // rows)))
        history = rng.choice([0, _log_int(rng, 1, 4096)])
        while sequences * rows * heads * (rows + history) > 2 * 10**8 and history + rows > 512:
            history, rows = history // 2, max(16, rows * 3 // 4)
        return _nameless(_attend("", sequences, history, rows, heads, kv_heads, head_dim, x,
                                 rng.choice([0, 0, _log_int(rng, 50, 2000)]), weights))
    if kind == "evict":
        sequences = _log_int(rng, 1, 16)
        length = _log_int(rng, 300, max(400, min(60000, 130_000_000 // (per_token * sequences))))
        budget = max(16, int(length * rng.uniform(0.05, 0.9)))
        recent = int(budget * rng.uniform(0.0, 0.6))
        return _nameless(_evict("", sequences, length, budget, recent, rng.choice([0, 4, budget // 16]), kv_heads, head_dim, x))
    vocabulary = _log_int(rng, 2000, 130000)
    rows = _log_int(rng, 1, max(2, min(777, 77_000_000 // vocabulary)))
    return _nameless(_logprobs("", rows, vocabulary, rng.choice([0, 1, 5, 8, 20]), rng.choice(["f32", "bf16", "f16"])))


def _nameless(case):
    del case["name"]
    return case


# ---- the ragged sizes of a batch, the same for every seed ------------------------------------------------------------
def _spread(b, low):
    """A factor in [low, 1] for sequence b; 1 for the first."""
    return 1.0 - (1.0 - low) * ((b * 7919) % 997) / 996.0


def _rows(case):
    """New rows of each sequence: alike at decode, ragged where prompts are cut."""
    n = case.get("rows", 0)
    return [n if n <= 8 else max(1, int(n * _spread(b + 5 * (b > 0), 0.3))) for b in range(case["sequences"])]


def _lengths(case):
    """Tokens of each sequence in the cache, the new rows among them."""
    return [int(case["history"] * _spread(b, 0.25)) + r for b, r in enumerate(_rows(case))]


def _blocks(tokens):
    return -(-tokens // BLOCK)


def _visible(case):
    """Per sequence: (tokens any row sees, (row, token) pairs)."""
    got = []
    for length, n in zip(_lengths(case), _rows(case)):
        w = case["window"] or length
        first = max(0, length - n - w + 1)
        pairs = sum(min(p + 1, w) for p in range(length - n, length))
        got.append((length - first, pairs))
    return got


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _table(case, g, spare=0):
    """Block ids of every sequence in random order, -1 behind its last block; and how many blocks there are."""
    counts = [_blocks(t) for t in _lengths(case)]
    ids = torch.randperm(sum(counts) + spare, device="cuda", generator=g).to(torch.int32)
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    return table, ids[at:], sum(counts) + spare


def _cached(case, blocks, g):
    """Codes [block, head, key or value, token, dimension] and scales of a filled cache."""
    shape = (blocks, case["kv_heads"], 2, BLOCK, case["head_dim"])
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    for i in range(0, blocks, 1024):      # keys and values about normal; the largest of a block near 127
        part = codes[i:i + 1024]
        part.copy_((torch.randn(part.shape, device="cuda", generator=g) * 32).round_().clamp_(-127, 127))
    scales = torch.rand((blocks, case["kv_heads"], 2), device="cuda", generator=g) * 0.03 + 0.02
    return codes, scales


def _new_rows(case, g, width):
    rows = sum(_rows(case))
    x = torch.randn((rows, width), device="cuda", generator=g)
    return (x * (0.5 + torch.rand((rows, 1), device="cuda", generator=g))).to(DTYPES[case["x"]])


def _inputs(case, seed):
    """Everything a pass reads, codes as [block, head, key or value, token, dimension]."""
    g = _generator(seed)
    kind, i = case["kind"], {}
    if kind == "logprobs":
        logits = torch.randn((case["rows"], case["vocabulary"]), device="cuda", generator=g).mul_(3.0)
        i["logits"] = logits.to(DTYPES[case["x"]])
        i["tokens"] = torch.randint(0, case["vocabulary"], (case["rows"],), device="cuda", dtype=torch.int32, generator=g)
        return i
    spare = _blocks(case["budget"]) * case["sequences"] if kind == "evict" else 0
    i["table"], free, blocks = _table(case, g, spare)
    i["codes"], i["scales"] = _cached(case, blocks, g)
    i["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    rows = _rows(case)
    i["starts"] = torch.tensor([sum(rows[:b]) for b in range(len(rows) + 1)], dtype=torch.int32, device="cuda")
    width = case["kv_heads"] * case["head_dim"]
    if kind == "append":
        i["k"], i["v"] = _new_rows(case, g, width), _new_rows(case, g, width)
    elif kind == "attend":
        i["q"] = _new_rows(case, g, case["heads"] * case["head_dim"])
        if case["weights"]:
            i["sums"] = torch.rand((blocks, case["kv_heads"], BLOCK), device="cuda", generator=g)
    else:
        i["sums"] = 6.0 * torch.rand((blocks, case["kv_heads"], BLOCK), device="cuda", generator=g) ** 4
        i["new_table"] = free.view(case["sequences"], -1).contiguous()
    return i


def _lay_out(codes):
    """[block, head, 2, token, dimension] as the cache holds it: [block, head, 2, 64 x dimensions]."""
    n, h, _, _, d = codes.shape
    out = torch.empty((n, h, 2, BLOCK * d), dtype=torch.int8, device=codes.device)
    out[:, :, 0] = codes[:, :, 0].reshape(n, h, 4, 16, d // 64, 4, 16).permute(0, 1, 2, 4, 5, 3, 6).reshape(n, h, -1)
    out[:, :, 1] = codes[:, :, 1].reshape(n, h, 2, 2, 4, 4, d // 16, 16).permute(0, 1, 6, 4, 7, 2, 3, 5).reshape(n, h, -1)
    return out


def _plain_order(laid, d):
    """The reverse, for blocks gathered in any leading shape: keys and values as [..., token, dimension]."""
    lead = laid.shape[:-2]
    k = laid[..., 0, :].reshape(-1, 4, d // 64, 4, 16, 16).permute(0, 1, 4, 2, 3, 5).reshape(*lead, BLOCK, d)
    v = laid[..., 1, :].reshape(-1, d // 16, 4, 16, 2, 2, 4).permute(0, 4, 5, 2, 6, 1, 3).reshape(*lead, BLOCK, d)
    return k, v


class _State:
    pass


_context = None


def prepare(case, seed):
    s = _State()
    s.case = case
    for name, value in _inputs(case, seed).items():
        setattr(s, name, value)
    if case["kind"] == "logprobs":
        n, k = case["rows"], case["top"]
        s.logprob, s.entropy = (torch.empty(n, device="cuda") for _ in range(2))
        s.top_ids = torch.empty((n, k), dtype=torch.int32, device="cuda")
        s.top_logprobs = torch.empty((n, k), device="cuda")
        torch.cuda.synchronize()
        return s
    s.codes = _lay_out(s.codes)
    s.max_rows, s.max_length = max(_rows(case)), max(_lengths(case))
    s.rows = sum(_rows(case))
    kv_heads, d, dtype = case["kv_heads"], case["head_dim"], DTYPES[case["x"]]
    if case["kind"] == "append":        # read back: every token of the blocks the new ones went into
        back = [t - (t - n) // BLOCK * BLOCK for t, n in zip(_lengths(case), _rows(case))]
        s.back_starts = torch.tensor([sum(back[:b]) for b in range(len(back) + 1)], dtype=torch.int32, device="cuda")
        s.back_rows, s.back_most = sum(back), max(back)
    elif case["kind"] == "evict":
        kept = [min(t, case["budget"]) for t in _lengths(case)]
        s.back_starts = torch.tensor([sum(kept[:b]) for b in range(len(kept) + 1)], dtype=torch.int32, device="cuda")
        s.back_rows, s.back_most = sum(kept), max(kept)
        s.new_lengths = torch.empty_like(s.lengths)
        s.positions = torch.full((case["sequences"], kv_heads, case["budget"]), -1, dtype=torch.int32, device="cuda")
    else:
        s.out = torch.empty((s.rows, case["heads"] * d), dtype=dtype, device="cuda")
        s.lse = torch.empty((s.rows, case["heads"]), device="cuda")
    if case["kind"] != "attend":
        s.k_back, s.v_back = (torch.empty((s.back_rows, kv_heads * d), dtype=dtype, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    return s


# ---- the framework's calls -------------------------------------------------------------------------------------------
def _run_own(s):
    global _context
    mi355q = importlib.import_module("swift-mlx-lm_amd")
    if _context is None:
        _context = mi355q.Context(0)
    ctx, case, stream = _context, s.case, torch.cuda.current_stream().cuda_stream
    dtype = {"f16": mi355q.F16, "bf16": mi355q.BF16, "f32": mi355q.F32}[case["x"]]
    if case["kind"] == "logprobs":
        ctx.token_logprobs(s.logits.data_ptr(), dtype, case["rows"], case["vocabulary"], s.tokens.data_ptr(), case["top"],
                           s.logprob.data_ptr(), s.entropy.data_ptr(), s.top_ids.data_ptr(), s.top_logprobs.data_ptr(),
                           stream=stream)
        return {"logprob": s.logprob, "entropy": s.entropy, "top_ids": s.top_ids, "top_logprobs": s.top_logprobs}
    sums = getattr(s, "sums", None)
    cache = mi355q.KVBlockCache(case["kv_heads"], case["head_dim"], s.codes.shape[0], s.codes.data_ptr(),
                                s.scales.data_ptr(), 0 if sums is None else sums.data_ptr())
    sequences = mi355q.KVSequences(case["sequences"], s.table.data_ptr(), s.table.shape[1], s.lengths.data_ptr(),
                                   s.starts.data_ptr(), s.rows, s.max_rows, s.max_length)
    if case["kind"] == "attend":
        ctx.kv_block_attention(cache, sequences, s.q.data_ptr(), dtype, case["heads"], s.out.data_ptr(), dtype,
                               scale=case["head_dim"] ** -0.5, window=case["window"], lse=s.lse.data_ptr(),
                               accumulate_weights=case["weights"], stream=stream)
        return {"out": s.out, "lse": s.lse, **({"sums": s.sums} if case["weights"] else {})}
    if case["kind"] == "append":
        ctx.kv_block_append(cache, sequences, s.k.data_ptr(), s.v.data_ptr(), dtype, stream=stream)
        back = mi355q.KVSequences(case["sequences"], s.table.data_ptr(), s.table.shape[1], s.lengths.data_ptr(),
                                  s.back_starts.data_ptr(), s.back_rows, s.back_most, s.max_length)
        ctx.kv_block_read(cache, back, s.k_back.data_ptr(), s.v_back.data_ptr(), dtype, stream=stream)
        return {"k": s.k_back, "v": s.v_back, "scales": s.scales}
    ctx.kv_block_evict(cache, sequences, case["budget"], s.new_table.data_ptr(), s.new_table.shape[1],
                       s.new_lengths.data_ptr(), recent=case["recent"], sinks=case["sinks"],
                       positions=s.positions.data_ptr(), stream=stream)
    back = mi355q.KVSequences(case["sequences"], s.new_table.data_ptr(), s.new_table.shape[1], s.new_lengths.data_ptr(),
                              s.back_starts.data_ptr(), s.back_rows, s.back_most, case["budget"])
    ctx.kv_block_read(cache, back, s.k_back.data_ptr(), s.v_back.data_ptr(), dtype, stream=stream)
    return {"positions": s.positions, "lengths": s.new_lengths, "sums": s.sums, "k": s.k_back, "v": s.v_back}


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _row_places(starts, lengths, rows):
    """Sequence and position of every row of a ragged row tensor."""
    row = torch.arange(rows, device="cuda")
    b = torch.searchsorted(starts[1:].long(), row, right=True)
    return b, lengths[b].long() - starts[b + 1].long() + row


def _plain_read(codes, scales, table, lengths, starts, rows, d, dtype):
    b, p = _row_places(starts, lengths, rows)
    block = table[b, p // BLOCK].long()
    h = codes.shape[1]
    k, v = _plain_order(codes, d)
    out = [(x[block, :, p % BLOCK].float() * scales[block, :, i, None]).view(rows, h * d).to(dtype) for i, x in enumerate((k, v))]
    return out


def _plain_append(s):
    case, d, h = s.case, s.case["head_dim"], s.case["kv_heads"]
    n = s.starts.diff().long()
    first = s.lengths.long() - n
    touched = (s.max_rows + BLOCK - 2) // BLOCK + 1
    j = first[:, None] // BLOCK + torch.arange(touched, device="cuda")            # block of the sequence
    live = j * BLOCK < s.lengths[:, None]
    block = torch.where(live, s.table.long().gather(1, j.clamp(max=s.table.shape[1] - 1)), -1)
    p = j[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")
    new = (p >= first[:, None, None]) & (p < s.lengths[:, None, None]) & live[:, :, None]
    row = torch.where(new, s.starts[:-1, None, None] + p - first[:, None, None], 0).long()
    x = torch.stack((s.k[row], s.v[row]), 3).float().view(*row.shape, 2, h, d)    # [b, j, token, 2, h, d]
    x = (x * new[..., None, None, None]).permute(0, 1, 4, 3, 2, 5)                # [b, j, h, 2, token, d]
    kept = (p < first[:, None, None])[:, :, None, None, :, None]
    at = block.clamp(min=0)
    old = torch.where((j * BLOCK < first[:, None])[:, :, None, None], s.scales[at], 0.0)
    scale = torch.maximum(old, x.abs().amax((4, 5)) * (1.0 / STEPS))
    safe = torch.where(scale > 0, scale, 1.0)[..., None, None]
    codes = torch.stack(_plain_order(s.codes[at], d), 3).float()
    codes = torch.where(kept, (codes * (old[..., None, None] / safe)).round(),
                        torch.where(new[:, :, None, None, :, None], (x / safe).round().clamp(-127, 127), codes))
    picked = live.flatten()
    s.codes[block.flatten()[picked]] = _lay_out(codes.to(torch.int8).flatten(0, 1))[picked]
    s.scales[block.flatten()[picked]] = scale.flatten(0, 1)[picked]
    k, v = _plain_read(s.codes, s.scales, s.table, s.lengths, s.back_starts, s.back_rows, d, DTYPES[case["x"]])
    return {"k": k, "v": v, "scales": s.scales}


def _plain_attend(s):
    case = s.case
    h, d, heads, batch = case["kv_heads"], case["head_dim"], case["heads"], case["sequences"]
    group, most = heads // h, s.max_rows
    table = s.table.long().clamp(min=0)
    k, v = (x.float() for x in _plain_order(s.codes[table], d))                   # [b, j, h, token, d]
    scales = s.scales[table]
    k = (k * scales[:, :, :, 0, None, None]).permute(0, 2, 1, 3, 4).reshape(batch, h, -1, d)
    v = (v * scales[:, :, :, 1, None, None]).permute(0, 2, 1, 3, 4).reshape(batch, h, -1, d)
    tokens = k.shape[2]
    n = s.starts.diff().long()
    i = torch.arange(most, device="cuda")
    row = (s.starts[:-1, None] + i).clamp(max=s.rows - 1).long()
    q = s.q.float().view(s.rows, h, group, d)[row].permute(0, 2, 3, 1, 4).reshape(batch, h, group * most, d)
    x = torch.matmul(q, k.transpose(2, 3).contiguous()).view(batch, h, group, most, tokens) * d ** -0.5
    del k
    p = (s.lengths.long() - n)[:, None] + i                                       # position of a row
    t = torch.arange(tokens, device="cuda")
    seen = (t <= p[:, :, None]) & (i < n[:, None])[:, :, None]
    if case["window"]:
        seen &= t > p[:, :, None] - case["window"]
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(4, keepdim=True).clamp(min=-3e38)
    x = (x - top).exp_()
    total = x.sum(4, keepdim=True)
    x /= torch.where(total > 0, total, 1.0)
    o = torch.matmul(x.view(batch, h, group * most, tokens), v).view(batch, h, group, most, d)
    lse = (top + total.log()).squeeze(4)
    b, p = _row_places(s.starts, s.lengths, s.rows)
    i = torch.arange(s.rows, device="cuda") - s.starts[b]
    out = {"out": o[b, :, :, i].reshape(s.rows, heads * d).to(DTYPES[case["x"]]), "lse": lse[b, :, :, i].reshape(s.rows, heads)}
    if case["weights"]:
        w = x.sum((2, 3)).view(batch, h, -1, BLOCK).permute(0, 2, 1, 3).flatten(0, 1)      # zero behind a sequence's end
        s.sums.index_add_(0, table.flatten(), w)
        out["sums"] = s.sums
    return out


def _plain_evict(s):
    case = s.case
    h, d, batch, budget = case["kv_heads"], case["head_dim"], case["sequences"], case["budget"]
    table = s.table.long().clamp(min=0)
    length = s.lengths.long()[:, None, None]
    sums = s.sums[table].permute(0, 2, 1, 3).flatten(2)                           # [b, h, token]
    t = torch.arange(sums.shape[2], device="cuda").expand_as(sums)
    rank = torch.where((t >= length - case["recent"]) | (t < case["sinks"]), math.inf, sums).masked_fill(t >= length, -math.inf)
    order = rank.sort(dim=2, descending=True, stable=True).indices[:, :, :budget]
    s.new_lengths.copy_(s.lengths.clamp(max=budget))
    count = s.new_lengths.long()[:, None, None]
    place = torch.arange(order.shape[2], device="cuda")
    kept = torch.where(place < count, order, 1 << 40).sort(2).values
    live = kept < 1 << 40
    s.positions[:, :, :kept.shape[2]] = torch.where(live, kept, -1).to(torch.int32)
    width = s.new_table.shape[1] * BLOCK
    pad = torch.nn.functional.pad(torch.where(live, kept, 0), (0, width - kept.shape[2]))
    live = torch.nn.functional.pad(live, (0, width - kept.shape[2]))
    source = table.gather(1, (pad // BLOCK).flatten(1)).view_as(pad)
    head = torch.arange(h, device="cuda")[:, None].expand_as(pad)
    k, v = _plain_order(s.codes, d)
    scale = s.scales[source, head] * live[..., None]                              # [b, h, token, 2]
    codes = torch.stack((k[source, head, pad % BLOCK], v[source, head, pad % BLOCK]), 3).float()
    blocked = scale.view(batch, h, -1, BLOCK, 2)
    new = blocked.amax(3)
    ratio = blocked / torch.where(new > 0, new, 1.0)[:, :, :, None]
    codes = (codes.view(batch, h, -1, BLOCK, 2, d) * ratio[..., None]).round()
    target = s.new_table.long()
    s.codes[target.flatten()] = _lay_out(codes.permute(0, 2, 1, 4, 3, 5).flatten(0, 1).to(torch.int8))
    s.scales[target.flatten()] = new.permute(0, 2, 1, 3).flatten(0, 1)
    moved = sums.gather(2, pad) * live
    s.sums[target.flatten()] = moved.view(batch, h, -1, BLOCK).permute(0, 2, 1, 3).flatten(0, 1)
    k, v = _plain_read(s.codes, s.scales, s.new_table, s.new_lengths, s.back_starts, s.back_rows, d, DTYPES[case["x"]])
    return {"positions": s.positions, "lengths": s.new_lengths, "sums": s.sums, "k": k, "v": v}


def _plain_logprobs(s):
    x = s.logits.float()
    top, ids = x.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :s.case["top"]], ids[:, :s.case["top"]]
    z = x - x.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1)
    lse = x.amax(1) + total.log()
    return {"logprob": x.gather(1, s.tokens.long()[:, None])[:, 0] - lse, "entropy": total.log() - (e * z).sum(1) / total,
            "top_ids": ids.to(torch.int32), "top_logprobs": top - lse[:, None]}


def run(s):
    if own:
        return _run_own(s)
    return {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "logprobs": _plain_logprobs}[s.case["kind"]](s)


# ---- the same in 64 bits, sequence by sequence -----------------------------------------------------------------------
def _exact_tokens(i, b, table="table", length=None):
    """Keys and values of sequence b as [2, h, token, d] codes with their scales [2, h, token]."""
    length = int(i["lengths"][b]) if length is None else length
    ids = i[table][b, :_blocks(length)].long()
    codes = i["codes"][ids].permute(2, 1, 0, 3, 4).flatten(2, 3)[:, :, :length]
    scales = i["scales"][ids].double().permute(2, 1, 0).repeat_interleave(BLOCK, 2)[:, :, :length]
    return codes.double(), scales


def _exact_append(case, i):
    starts, d, h = i["starts"].tolist(), case["head_dim"], case["kv_heads"]
    scales, back = i["scales"].double().clone(), []
    for b, length in enumerate(_lengths(case)):
        rows = range(starts[b], starts[b + 1])
        first = length - len(rows)
        x = torch.stack([i[n][rows.start:rows.stop].double().view(-1, h, d) for n in ("k", "v")])      # [2, token, h, d]
        for j in range(first // BLOCK, _blocks(length)):
            block, low, high = int(i["table"][b, j]), j * BLOCK, min(length, (j + 1) * BLOCK)
            y = x[:, max(low, first) - first:high - first].permute(2, 0, 1, 3)                         # [h, 2, token, d]
            before = scales[block] if low < first else torch.zeros_like(scales[block])
            after = torch.maximum(before, y.abs().amax((2, 3)) / STEPS)
            was = i["codes"][block, :, :, :max(0, first - low)].double() * (before / after)[..., None, None]
            codes = torch.cat((was.round(), (y / after[..., None, None]).round().clamp(-127, 127)), 2)
            back.append((codes * after[..., None, None]).permute(1, 2, 0, 3).flatten(2))                # [2, token, h d]
            scales[block] = after
    back = torch.cat(back, 1)
    return {"k": back[0], "v": back[1], "scales": scales}


def _exact_attend(case, i):
    starts, d, h = i["starts"].tolist(), case["head_dim"], case["kv_heads"]
    group = case["heads"] // h
    out, lse = [], []
    sums = i["sums"].double().clone() if case["weights"] else None
    for b, length in enumerate(_lengths(case)):
        n = starts[b + 1] - starts[b]
        codes, scales = _exact_tokens(i, b)
        k, v = codes * scales[..., None]
        q = i["q"][starts[b]:starts[b + 1]].double().view(n, h, group, d)
        p = torch.arange(length - n, length, device="cuda")[:, None]
        t = torch.arange(length, device="cuda")
        hidden = (t > p) | (t <= p - (case["window"] or length))
        o, l = torch.empty((n, h, group, d), dtype=torch.float64, device="cuda"), torch.empty((n, h, group), dtype=torch.float64, device="cuda")
        for head in range(h):
            x = (q[:, head].reshape(n * group, d) @ k[head].t().contiguous()).view(n, group, length) / math.sqrt(d)
            x = x.masked_fill(hidden[:, None], -math.inf)
            l[:, head] = torch.logsumexp(x, 2)
            w = torch.exp(x - l[:, head, :, None])
            o[:, head] = (w.view(n * group, length) @ v[head]).view(n, group, d)
            if sums is not None:
                added = torch.zeros(_blocks(length) * BLOCK, dtype=torch.float64, device="cuda")
                added[:length] = w.sum((0, 1))
                sums[i["table"][b, :_blocks(length)].long(), head] += added.view(-1, BLOCK)
        out.append(o.view(n, -1))
        lse.append(l.view(n, -1))
    return {"out": torch.cat(out), "lse": torch.cat(lse), **({"sums": sums} if case["weights"] else {})}


def _exact_evict(case, i):
    sums, back, budget = i["sums"].double().clone(), [], case["budget"]
    for b, length in enumerate(_lengths(case)):
        codes, scales = _exact_tokens(i, b)
        ids, new_ids = i["table"][b, :_blocks(length)].long(), i["new_table"][b].long()
        count = min(length, budget)
        rows = torch.empty((2, count, case["kv_heads"], case["head_dim"]), dtype=torch.float64, device="cuda")
        for head in range(case["kv_heads"]):
            weight = i["sums"][ids, head].double().flatten()[:length]
            weight[length - min(length, case["recent"]):] = math.inf
            weight[:case["sinks"]] = math.inf
            kept = torch.sort(weight, descending=True, stable=True).indices[:count].sort().values
            moved = torch.zeros(new_ids.numel() * BLOCK, dtype=torch.float64, device="cuda")
            moved[:count] = i["sums"][ids, head].double().flatten()[kept]
            sums[new_ids, head] = moved.view(-1, BLOCK)
            for part in range(2):
                for low in range(0, count, BLOCK):
                    at = kept[low:low + BLOCK]
                    scale = scales[part, head, at].max()
                    rows[part, low:low + BLOCK, head] = (codes[part, head, at] * (scales[part, head, at] / scale)[:, None]).round() * scale
        back.append(rows.flatten(2))
    back = torch.cat(back, 1)
    return {"positions": None, "lengths": None, "sums": sums, "k": back[0], "v": back[1]}


def exact(case, seed):
    i = _inputs(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, i)
    if case["kind"] == "attend":
        return _exact_attend(case, i)
    if case["kind"] == "evict":
        return _exact_evict(case, i)
    logits = i["logits"]
    got = {"logprob": [], "entropy": [], "top_ids": None, "top_logprobs": []}
    for r in range(0, case["rows"], 64):
        x = torch.log_softmax(logits[r:r + 64].double(), 1)
        got["logprob"].append(x.gather(1, i["tokens"][r:r + 64].long()[:, None])[:, 0])
        got["entropy"].append(-(x.exp() * x).sum(1))
        got["top_logprobs"].append(x.topk(case["top"], 1).values)
    return {n: v if v is None else torch.cat(v) for n, v in got.items()}


def work(case):
    size = DTYPES[case["x"]].itemsize
    if case["kind"] == "logprobs":
        n, v = case["rows"], case["vocabulary"]
        return {"bytes": n * (v * size + 4 + 8 + 8 * case["top"]), "flops": 6.0 * n * v}
    h, d = case["kv_heads"], case["head_dim"]
    rows, lengths = _rows(case), _lengths(case)
    if case["kind"] == "append":
        back = sum(t - (t - n) // BLOCK * BLOCK for t, n in zip(lengths, rows))
        scales = 8 * h * sum(_blocks(t) - (t - n) // BLOCK for t, n in zip(lengths, rows))
        per = 2 * h * d
        # rows in and codes out; tokens that were in a touched block in and out; everything out again as numbers
        return {"bytes": per * (sum(rows) * (size + 1) + 2 * (back - sum(rows)) + back * (1 + size)) + 3 * scales, "flops": 4.0 * per * back}
    if case["kind"] == "attend":
        seen = _visible(case)
        tokens = sum(t for t, _ in seen)
        moved = tokens * h * (2 * d + 8 / BLOCK) + 2 * sum(rows) * case["heads"] * d * size + sum(rows) * case["heads"] * 4
        return {"bytes": moved + (8 * tokens * h if case["weights"] else 0),
                "flops": 4.0 * d * case["heads"] * sum(pairs for _, pairs in seen)}
    kept = sum(min(t, case["budget"]) for t in lengths)
    # the weights; kept codes in, out, in again and out as numbers; kept weights and positions out
    return {"bytes": h * (4 * sum(lengths) + kept * (2 * d * (3 + size) + 8 + 32 / BLOCK)), "flops": 4.0 * h * d * kept}
