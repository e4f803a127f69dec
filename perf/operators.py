"""The cleartext operators that stand beside the encrypted layer, as cases that can be timed and compared.

Three operators: writing keys and values into 4-bit pages and reading them back, attention over such
pages (with the range of every row's scores, from which the encrypted softmax takes its intervals),
and the scoring of given tokens under clear logits.  ``run`` computes them in plain torch in 32 bits,
or, with ``own`` set, through ``holmes_amd.clear``.

A page holds 128 tokens.  Each run of 32 values along the head dimension shares a power of two
2^(b - 127), held as the byte b, and every value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, with a
sign.  b is the exponent of the run's largest magnitude rounded to one mantissa bit, less 2 (limited to
2..252), so that the largest value becomes 4 or 6 units; a run that holds an infinity or a NaN has
b = 255 and reads back as NaN.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 128   # tokens of a page
RUN = 32     # values that share a scale
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # the token that one decode step adds to the cache, and its check against what was written
        dict(name="pages-token", kind="pages", tokens=1, heads=8, dim=128, type="bf16"),
        # the keys and values of a long calibration prompt going into the cache, read back for the next layer's check
        dict(name="pages-prompt", kind="pages", tokens=32768, heads=8, dim=128, type="bf16"),
        # one token over two pages, the size of the encrypted decode step: latency
        dict(name="decode-one", kind="attend", seqs=1, low=257, high=257, new=1, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=True),
        # a served batch in which every sequence has a length of its own
        dict(name="decode-batch", kind="attend", seqs=32, low=63, high=8191, new=1, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=False),
        # one sequence with a very long history: few rows, so the history itself is what can be shared out
        dict(name="decode-long", kind="attend", seqs=1, low=131072, high=131072, new=1, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=False),
        # many sequences with long histories: the cache's bytes and nothing else
        dict(name="decode-large", kind="attend", seqs=48, low=12000, high=24576, new=1, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=False),
        # the 128-token page of the encrypted prefill layer, with its softmax's ranges
        dict(name="prompt-page", kind="attend", seqs=1, low=128, high=128, new=128, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=True),
        # a calibration prompt
        dict(name="prompt-long", kind="attend", seqs=1, low=4096, high=4096, new=4096, ragged=False, heads=8, group=4,
             dim=128, type="bf16", ranges=True),
        # continued prompts of different sizes behind histories of different lengths, an odd group, small heads
        dict(name="prompt-ragged", kind="attend", seqs=5, low=700, high=6001, new=611, ragged=True, heads=3, group=5,
             dim=64, type="fp16", ranges=False),
        # the next token of one sequence: latency
        dict(name="score-one", kind="score", rows=1, vocab=131072, top=8, type="fp32", hole=0.0),
        # a short answer, an odd vocabulary of which a part is masked
        dict(name="score-masked", kind="score", rows=61, vocab=50021, top=20, type="fp32", hole=0.3),
        # a whole prompt scored against the decrypted answer
        dict(name="score-prompt", kind="score", rows=4096, vocab=131072, top=5, type="bf16", hole=0.0),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["pages", "attend", "attend", "score"])
    if kind == "pages":
        return dict(kind=kind, tokens=_spread(rng, 1, 20000), heads=rng.randint(1, 10), dim=rng.choice([64, 128]),
                    type=rng.choice(sorted(TYPES)))
    if kind == "score":
        rows = _spread(rng, 1, 2000)
        return dict(kind=kind, rows=rows, vocab=_spread(rng, 40, min(200000, 200000000 // rows)), top=rng.randint(0, 20),
                    type=rng.choice(sorted(TYPES)), hole=rng.choice([0.0, 0.0, 0.5]))
    heads, group, dim = rng.randint(1, 8), rng.randint(1, 8), rng.choice([64, 128])
    shape = dict(kind=kind, heads=heads, group=group, dim=dim, type=rng.choice(["bf16", "fp16"]),
                 ranges=rng.choice([False, True]))
    if rng.random() < 0.6:  # single tokens
        seqs = _spread(rng, 1, 48)
        high = _spread(rng, 1, min(65536, 400000 // seqs))
        return dict(shape, seqs=seqs, low=_spread(rng, 1, high), high=high, new=1, ragged=False)
    seqs = rng.randint(1, 5)
    high = _spread(rng, 2, 4096)
    new = _spread(rng, 2, min(high, 1500))
    return dict(shape, seqs=seqs, low=_spread(rng, new, high), high=high, new=new, ragged=rng.choice([False, True]))


def _lengths(case):
    """The sequences' lengths, from the shortest to the longest in even ratios, every second one from the far end."""
    n, low, high = case["seqs"], case["low"], case["high"]
    got = [high] if n == 1 else [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]
    return got[::2] + got[1::2][::-1]


def _counts(case):
    """The new tokens of each sequence, at the end of it: all alike, or from one up."""
    n, new = case["seqs"], case["new"]
    if not case["ragged"] or n == 1:
        return [new] * n
    return [1 + (new - 1) * i // (n - 1) for i in range(n)]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _tokens(gen, n, heads, dim):
    """Keys or values of n tokens: channels of different widths about means of their own, as projections give them."""
    width = torch.exp(0.5 * _randn(gen, 1, heads, dim))
    return (_randn(gen, n, heads, dim) + 0.5 * _randn(gen, 1, heads, dim)) * width


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)
    kind, s = case["kind"], {"case": case}
    dtype = TYPES[case["type"]]
    if kind == "score":
        rows, vocab = case["rows"], case["vocab"]
        x = 2.0 * _randn(gen, rows, vocab)
        x += 6.0 * (torch.rand((rows, vocab), generator=gen, device="cuda") < 4.0 / vocab)  # what the model expects
        if case["hole"]:
            x.masked_fill_(torch.rand((rows, vocab), generator=gen, device="cuda") < case["hole"], -math.inf)
        s["logits"] = x.to(dtype)
        near, far = x.argmax(1), torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        s["tokens"] = torch.where(torch.rand((rows,), generator=gen, device="cuda") < 0.6, near, far)
        if rows > 8:
            s["tokens"][::9] = -1  # padding
        return s
    heads, dim = case["heads"], case["dim"]
    if kind == "pages":
        total = case["tokens"]
        pages = -(-total // PAGE) + 1
        s["keys"], s["values"] = (_tokens(gen, total, heads, dim).to(dtype) for _ in range(2))
        s["slots"] = _slots(gen, pages, torch.tensor([total]), 37)[0][0, :total].contiguous()
        _pool(s, pages, heads, dim)
        return s
    lengths, counts = _lengths(case), _counts(case)
    need = [-(-n // PAGE) for n in lengths]
    pages = sum(need) + 3
    slots, s["table"] = _slots(gen, pages, torch.tensor(lengths), 0)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    s["queries"] = (1.5 * _randn(gen, starts[-1], heads * case["group"], dim)).to(dtype)
    _pool(s, pages, heads, dim)
    for b, n in enumerate(lengths):  # the history, written as it came
        _append(s, _tokens(gen, n, heads, dim).to(dtype), _tokens(gen, n, heads, dim).to(dtype), slots[b, :n].contiguous())
    return s


def _slots(gen, pages, lengths, first):
    """Where each sequence's tokens lie (page * 128 + place), and its pages, in no order."""
    need = (lengths + first + PAGE - 1) // PAGE
    order = torch.randperm(pages, generator=gen, device="cuda")
    table = torch.full((len(lengths), int(need.max())), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need.tolist()):
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    place = torch.arange(first, first + int(lengths.max()), device="cuda")
    return table.long()[:, place // PAGE] * PAGE + place % PAGE, table


def _pool(s, pages, heads, dim):
    """The cache that the program keeps."""
    if own:
        from holmes_amd import clear

        s["pool"] = clear.ClearKVPages(pages, kv_heads=heads, head_dim=dim)
        return
    s["codes"] = torch.zeros((2, pages * PAGE, heads, dim // 2), dtype=torch.uint8, device="cuda")
    s["scales"] = torch.zeros((2, pages * PAGE, heads, dim // RUN), dtype=torch.uint8, device="cuda")


def _append(s, keys, values, slots):
    if own:
        s["pool"].append(keys, values, slots)
        return
    for i, x in enumerate((keys, values)):
        s["codes"][i, slots], s["scales"][i, slots] = _quantise(x)


def _quantise(x):
    """The codes (two to a byte, the first value low) and scale bytes of x, in runs of 32 along its last axis."""
    x = x.float().unflatten(-1, (-1, RUN))
    top = x.abs().amax(-1, keepdim=True)
    byte = (((top.view(torch.int32) + (1 << 21)) >> 23) - 2).clamp(2, 252)
    fine = torch.isfinite(x).all(-1, keepdim=True)
    unit = (byte << 23).view(torch.float32)
    y = x.abs() / unit
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = torch.where(fine, code + 8 * torch.signbit(x).to(torch.uint8), torch.zeros_like(code)).flatten(-2)
    byte = torch.where(fine, byte, torch.full_like(byte, 255)).squeeze(-1).to(torch.uint8)
    return code[..., ::2] + 16 * code[..., 1::2], byte


def _values(codes, scales):
    """What codes and scale bytes stand for, in 32 bits."""
    unit = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    unit = torch.cat([unit, -unit])
    pair = torch.stack([unit.repeat(16), unit.repeat_interleave(16)], 1)
    x = pair[codes.int()].flatten(-2).unflatten(-1, (-1, RUN))
    scale = (scales.int() << 23).view(torch.float32)
    scale = torch.where(scales == 255, torch.full_like(scale, math.nan), scale)
    return (x * scale.unsqueeze(-1)).flatten(-2)


def run(s):
    kind = s["case"]["kind"]
    if own:
        if kind == "pages":
            s["pool"].append(s["keys"], s["values"], s["slots"])
            return tuple(s["pool"].read(s["slots"], s["keys"].dtype))
        if kind == "attend":
            got = s["pool"].attend(s["queries"], s["table"], s["lengths"], starts=s["starts"], most=s["case"]["new"],
                                   ranges=s["case"]["ranges"])
            return tuple(x for x in got if x is not None)
        from holmes_amd import clear

        got = clear.token_logprobs(s["logits"], s["tokens"], top=s["case"]["top"])
        return tuple(x for x in got if x is not None)
    return {"pages": _plain_pages, "attend": _plain_attend, "score": _plain_score}[kind](s)


def _plain_pages(s):
    dtype = s["keys"].dtype
    _append(s, s["keys"], s["values"], s["slots"])
    most = torch.finfo(dtype).max
    x = _values(s["codes"][:, s["slots"]], s["scales"][:, s["slots"]]).clamp(-most, most).to(dtype)
    return x[0], x[1]


def _plain_attend(s):
    case, q = s["case"], s["queries"]
    heads, group, dim = case["heads"], case["group"], case["dim"]
    lengths, starts = s["lengths"].long(), s["starts"].long()
    seqs, most = lengths.numel(), case["new"]
    place = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    slots = s["table"].long().clamp(min=0)[:, place // PAGE] * PAGE + place % PAGE
    there = place < lengths[:, None]
    keys, values = (_values(s["codes"][i, slots], s["scales"][i, slots]).transpose(1, 2) for i in range(2))
    values = torch.where(there[:, None, :, None], values, torch.zeros((), device="cuda"))
    count = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + i).clamp(max=q.shape[0] - 1)
    x = q.float()[row].unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).reshape(seqs, heads, group * most, dim)
    score = torch.matmul(x, keys.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    position = lengths[:, None] - count[:, None] + i
    seen = (place[None, None, :] <= position[:, :, None]) & there[:, None, :]
    seen = seen[:, None, None].expand(seqs, 1, group, most, -1).reshape(seqs, 1, group * most, -1)
    score = torch.where(seen, score, torch.full((), -math.inf, device="cuda"))
    high = score.amax(-1, keepdim=True)
    weight = torch.exp(score - torch.where(torch.isinf(high), torch.zeros_like(high), high))
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values) / torch.where(total == 0, torch.ones_like(total), total)
    sums = [high + torch.log(total)]
    if case["ranges"]:
        sums += [torch.where(seen, score, torch.full((), math.inf, device="cuda")).amin(-1, keepdim=True), high]
    valid = i < count[:, None]

    def rows(t):  # [seqs][heads][group * most][n] back to [tokens][query heads][n]
        t = t.unflatten(2, (group, most)).permute(0, 3, 1, 2, 4)
        return t[valid].flatten(1, 2)

    return (rows(out).to(q.dtype), *(rows(t).squeeze(-1) for t in sums))


def _plain_score(s):
    x, tokens, top = s["logits"].float(), s["tokens"], s["case"]["top"]
    high = x.amax(1, keepdim=True)
    x = x - torch.where(torch.isinf(high), torch.zeros_like(high), high)
    weight = torch.exp(x)
    total = weight.sum(1, keepdim=True)
    total = torch.where(total == 0, torch.ones_like(total), total)  # a row that is masked as a whole
    log = torch.log(total)
    given = torch.where(tokens >= 0, (x.gather(1, tokens.clamp(min=0)[:, None]) - log)[:, 0], torch.zeros((), device="cuda"))
    spread = torch.where(weight == 0, torch.zeros_like(x), weight * x).sum(1, keepdim=True)
    entropy = (log - spread / total)[:, 0]
    if not top:
        return given, entropy
    bits = (s["logits"].float() + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long() * (1 << 32)  # the values' order, then the lowest index
    order += (1 << 32) - 1 - torch.arange(x.shape[1], device="cuda")
    ids = (1 << 32) - 1 - (order.topk(top, dim=1).values & 0xFFFFFFFF)
    return given, entropy, ids, x.gather(1, ids) - log


def work(case):
    kind, size = case["kind"], TYPES[case["type"]].itemsize
    if kind == "score":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        return {"bytes": rows * (vocab * size + 8 + 8 + 12 * top), "flops": 5 * rows * vocab}
    heads, dim = case["heads"], case["dim"]
    held = 2 * heads * (dim // 2 + dim // RUN)  # bytes of one token in the cache
    if kind == "pages":
        n = case["tokens"]
        return {"bytes": n * (2 * (2 * heads * dim * size + held) + 8), "flops": n * 2 * heads * dim * 4}
    rows, pairs = 0, 0
    for length, new in zip(_lengths(case), _counts(case)):
        rows += new
        pairs += new * length - new * (new - 1) // 2
    query_heads = heads * case["group"]
    sums = 3 if case["ranges"] else 1
    return {"bytes": sum(_lengths(case)) * held + rows * query_heads * (2 * dim * size + 4 * sums),
            "flops": pairs * query_heads * (4 * dim + 5)}


# ---------------------------------------------------------------------------- in 64 bits
def _held(x):
    """The values that the 4-bit form keeps of x, from its definition."""
    x = x.double().unflatten(-1, (-1, RUN))
    top = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(torch.where(torch.isfinite(top), top, torch.ones_like(top)))
    exponent = torch.where(top == 0, torch.full_like(exponent, -200), exponent - 3 + (mantissa >= 0.875).int())
    unit = torch.ldexp(torch.ones_like(top), exponent.clamp(2 - 127, 252 - 127))
    y = x.abs() / unit
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0).double())
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return torch.where(torch.isfinite(top), torch.copysign(y * unit, x), torch.full_like(y, math.nan)).flatten(-2)


def exact(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)
    dtype = TYPES[case["type"]]
    if case["kind"] == "score":
        s = prepare(case, seed)
        parts = [_exact_score(x, t, case["top"]) for x, t in zip(s["logits"].split(256), s["tokens"].split(256))]
        return tuple(torch.cat(p) for p in zip(*parts))
    if case["kind"] == "pages":
        s = prepare(case, seed)
        return _held(s["keys"]), _held(s["values"])
    # the same inputs as prepare's, in the order in which it makes them
    heads, group, dim = case["heads"], case["group"], case["dim"]
    lengths, counts = _lengths(case), _counts(case)
    _slots(gen, sum(-(-n // PAGE) for n in lengths) + 3, torch.tensor(lengths), 0)
    queries = (1.5 * _randn(gen, sum(counts), heads * group, dim)).to(dtype).double()
    outs, at = [], 0
    for length, new in zip(lengths, counts):
        keys, values = (_held(_tokens(gen, length, heads, dim).to(dtype)) for _ in range(2))
        outs.append(_exact_attend(queries[at:at + new], keys, values, group))
        at += new
    got = tuple(torch.cat(p) for p in zip(*outs))
    return got if case["ranges"] else got[:2]


def _exact_attend(queries, keys, values, group):
    new, length, dim = queries.shape[0], keys.shape[0], keys.shape[2]
    later = torch.arange(length, device="cuda")[None, :] > torch.arange(length - new, length, device="cuda")[:, None]
    out, lse, low, high = torch.zeros_like(queries), *(torch.zeros_like(queries[..., 0]) for _ in range(3))
    for h in range(queries.shape[1]):
        score = queries[:, h] @ keys[:, h // group].T / math.sqrt(dim)
        low[:, h] = score.masked_fill(later, math.inf).amin(1)
        score = score.masked_fill(later, -math.inf)
        high[:, h] = score.amax(1)
        lse[:, h] = torch.logsumexp(score, 1)
        out[:, h] = torch.softmax(score, 1) @ values[:, h // group]
    return out, lse, low, high


def _exact_score(logits, tokens, top):
    x = logits.double()
    logs = torch.where((x == -math.inf).all(1, keepdim=True), x, torch.log_softmax(x, 1))
    given = torch.where(tokens >= 0, logs.gather(1, tokens.clamp(min=0)[:, None])[:, 0], 0.0)
    entropy = -torch.where(x == -math.inf, 0.0, logs.exp() * logs).sum(1)
    if not top:
        return given, entropy
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
    return given, entropy, ids, logs.gather(1, ids)
