"""More of the cleartext operators that stand beside the encrypted layer, as cases that can be timed and compared.

Four operators, in the order in which a prompt meets them: rotary positions on queries and keys; attention over a whole
prompt whose keys and values are not rounded to 4 bits, as the encrypted layer has them; the attention weight that each
cached token has been given, over the 4-bit pages; and the eviction of all but the heaviest tokens of every key head into
other pages, which is how a long prompt comes down to the few pages that the encrypted layer keeps.  ``run`` computes them
in plain torch in 32 bits (angles in 64), or, with ``own`` set, through ``holmes_amd.clear``.

A page holds 128 tokens.  Each run of 32 values along the head dimension shares a power of two 2^(b - 127), held as the
byte b, and every value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 times it, with a sign.  b is the exponent of the run's largest
magnitude rounded to one mantissa bit, less 2 (limited to 2..252), so that the largest value becomes 4 or 6 units.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 128   # tokens of a page
RUN = 32     # values that share a scale
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BASE = 500000.0      # the encrypted layers' rope_theta
ORIGINAL = 8192      # tokens that the frequencies were made for, where they are scaled


def listed():
    return [
        # the query and the key of one decode step: latency
        dict(name="rotate-token", kind="rotate", tokens=1, heads=32, kv_heads=8, dim=128, rotated=128, interleaved=False,
             scaling="none", far=256, inverse=False, type="bf16"),
        # queries and keys of a long calibration prompt
        dict(name="rotate-prompt", kind="rotate", tokens=32768, heads=32, kv_heads=8, dim=128, rotated=128,
             interleaved=False, scaling="wavelength", far=0, inverse=False, type="bf16"),
        # neighbouring pairs in half of a small head, an odd number of tokens far behind the length the model was made for
        dict(name="rotate-part", kind="rotate", tokens=6001, heads=15, kv_heads=3, dim=64, rotated=32, interleaved=True,
             scaling="ramp", far=120000, inverse=False, type="fp16"),
        # the 128-token page of the encrypted prefill layer, with its softmax's ranges
        dict(name="prompt-page", kind="prompt", seqs=1, low=128, high=128, heads=8, group=4, dim=128, causal=True,
             ranges=True, type="bf16"),
        # prompts of very different lengths packed one behind the other, an odd group, small heads
        dict(name="prompt-packed", kind="prompt", seqs=12, low=1, high=2047, heads=3, group=5, dim=64, causal=True,
             ranges=True, type="fp16"),
        # a long calibration prompt
        dict(name="prompt-long", kind="prompt", seqs=1, low=8192, high=8192, heads=8, group=4, dim=128, causal=True,
             ranges=False, type="bf16"),
        # what one decode step over two pages adds: latency
        dict(name="weigh-token", kind="weigh", seqs=1, low=257, high=257, new=1, heads=8, group=4, dim=128, prior=True,
             type="bf16"),
        # a served batch with long histories
        dict(name="weigh-batch", kind="weigh", seqs=32, low=2000, high=24576, new=1, heads=8, group=4, dim=128, prior=True,
             type="bf16"),
        # a calibration prompt over its own tokens
        dict(name="weigh-prompt", kind="weigh", seqs=1, low=4096, high=4096, new=4096, heads=8, group=4, dim=128,
             prior=False, type="bf16"),
        # three pages down to the two of the encrypted decode step
        dict(name="evict-one", kind="evict", seqs=1, low=384, high=384, keep=256, recent=32, heads=8, dim=128),
        # a served batch brought down to eight pages each; some sequences have fewer tokens than that
        dict(name="evict-batch", kind="evict", seqs=32, low=63, high=8191, keep=1024, recent=128, heads=8, dim=128),
        # one very long history: few rows to choose from, each of them long
        dict(name="evict-long", kind="evict", seqs=1, low=131072, high=131072, keep=8192, recent=1000, heads=8, dim=128),
    ]


def _spread(rng, low, high):
    """A whole number between the two, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["rotate", "prompt", "weigh", "evict"])
    dim = rng.choice([64, 128])
    if kind == "rotate":
        heads = rng.randint(1, 8)
        return dict(kind=kind, tokens=_spread(rng, 1, 16000), heads=heads * rng.randint(1, 5), kv_heads=heads, dim=dim,
                    rotated=rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                    interleaved=rng.choice([False, True]), scaling=rng.choice(["none", "linear", "wavelength", "ramp"]),
                    far=_spread(rng, 1, 1000000), inverse=rng.choice([False, False, True]), type=rng.choice(sorted(TYPES)))
    heads, group = rng.randint(1, 8), rng.randint(1, 6)
    if kind == "prompt":
        seqs = rng.randint(1, 12)
        high = _spread(rng, 1, min(6000, int(math.sqrt(1.2e9 / (seqs * heads * group)))))
        return dict(kind=kind, seqs=seqs, low=_spread(rng, 1, high), high=high, heads=heads, group=group, dim=dim,
                    causal=rng.choice([True, True, False]), ranges=rng.choice([False, True]),
                    type=rng.choice(["bf16", "fp16"]))
    if kind == "weigh":
        shape = dict(kind=kind, heads=heads, group=group, dim=dim, prior=rng.choice([False, True]),
                     type=rng.choice(["bf16", "fp16"]))
        if rng.random() < 0.5:  # single tokens
            seqs = _spread(rng, 1, 48)
            high = _spread(rng, 1, min(65536, 400000 // seqs))
            return dict(shape, seqs=seqs, low=_spread(rng, 1, high), high=high, new=1)
        seqs = rng.randint(1, 4)
        high = _spread(rng, 2, 4096)
        new = _spread(rng, 2, min(high, 1500))
        return dict(shape, seqs=seqs, low=_spread(rng, new, high), high=high, new=new)
    seqs = _spread(rng, 1, 32)
    high = _spread(rng, 1, min(100000, 250000 // seqs))
    keep = _spread(rng, 1, min(high + 10, 8192))
    return dict(kind=kind, seqs=seqs, low=_spread(rng, 1, high), high=high, keep=keep, recent=rng.randint(0, keep),
                heads=heads, dim=dim)


def _lengths(case):
    """The sequences' lengths, from the shortest to the longest in even ratios, every second one from the far end."""
    n, low, high = case["seqs"], case["low"], case["high"]
    got = [high] if n == 1 else [int(round(low * (high / low) ** (i / (n - 1)))) for i in range(n)]
    return got[::2] + got[1::2][::-1]


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _tokens(gen, n, heads, dim):
    """Keys or values of n tokens: channels of different widths about means of their own, as projections give them."""
    width = torch.exp(0.5 * _randn(gen, 1, heads, dim))
    return (_randn(gen, n, heads, dim) + 0.5 * _randn(gen, 1, heads, dim)) * width


def _scaling(case):
    """The numbers of a scaled rotary embedding: the factor that lengths grow by, and the two ends of the blend."""
    return {"none": None, "linear": (8.0,), "wavelength": (8.0, 1.0, 4.0), "ramp": (16.0, 1.0, 32.0)}[case["scaling"]]


def _frequencies(case):
    """Radians per token of every pair in 64 bits, and what the rotated values are multiplied by."""
    f = BASE ** (-torch.arange(0, case["rotated"], 2, dtype=torch.float64) / case["rotated"])
    given, amount = _scaling(case), 1.0
    if case["scaling"] == "linear":
        f = f / given[0]
    elif case["scaling"] == "wavelength":  # whole below original / high tokens a turn, divided above original / low
        part = ((ORIGINAL * f / (2 * math.pi) - given[1]) / (given[2] - given[1])).clamp(0, 1)
        f = part * f + (1 - part) * f / given[0]
    elif case["scaling"] == "ramp":  # over the pairs' numbers, between those with `high` and `low` turns in the original
        ends = [case["rotated"] * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in given[:0:-1]]
        first, last = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), case["rotated"] - 1)
        part = ((torch.arange(len(f), dtype=torch.float64) - first) / max(last - first, 0.001)).clamp(0, 1)
        f = (1 - part) * f + part * f / given[0]
        amount = 0.1 * math.log(given[0]) + 1.0
    return f, amount


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)
    kind, s, heads, dim = case["kind"], {"case": case}, case["heads"], case["dim"]
    if kind == "rotate":
        n, dtype = case["tokens"], TYPES[case["type"]]
        # as a projection leaves them: queries and keys side by side
        both = _randn(gen, n, heads + case["kv_heads"], dim).to(dtype)
        s["queries"], s["keys"] = both[:, :heads], both[:, heads:]
        s["positions"] = case["far"] + torch.arange(n, device="cuda")
        if case["far"] and n > 4:  # packed prompts
            s["positions"][n // 3:] -= int(torch.randint(1, case["far"] + 1, (), generator=gen, device="cuda"))
        if own:
            from holmes_amd import clear

            given = _scaling(case)
            if given is not None:
                given = clear.RotaryScaling(case["scaling"], given[0], ORIGINAL, *given[1:])
            s["plan"] = clear.RotaryPositions(dim, base=BASE, rotated=case["rotated"], interleaved=case["interleaved"],
                                              scaling=given)
        else:
            frequencies, s["amount"] = _frequencies(case)
            s["frequencies"] = frequencies.cuda()
        return s
    lengths = _lengths(case)
    if kind == "prompt":
        dtype = TYPES[case["type"]]
        s["queries"] = (1.5 * _randn(gen, sum(lengths), heads * case["group"], dim)).to(dtype)
        s["keys"], s["values"] = (_tokens(gen, sum(lengths), heads, dim).to(dtype) for _ in range(2))
        s["starts"] = _starts(lengths)
        return s
    # pages in no order, then those that eviction fills
    need = [-(-n // PAGE) for n in lengths]
    fresh = -(-case["keep"] // PAGE) if kind == "evict" else 0
    pages = sum(need) + fresh * len(lengths) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    s["table"] = torch.full((len(lengths), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        s["table"][b, :n] = order[at:at + n]
        at += n
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    _pool(s, pages, heads, dim)
    if kind == "evict":
        s["into"] = order[at:at + fresh * len(lengths)].view(len(lengths), fresh).contiguous()
        s["slots"] = _slots(s["into"], case["keep"]).flatten()
        # what softmax rows leave behind: many small weights, few large ones, and none behind a sequence's end
        s["weights"] = torch.exp(2.0 * _randn(gen, len(lengths), heads, max(need) * PAGE))
        s["weights"] *= torch.arange(max(need) * PAGE, device="cuda") < s["lengths"][:, None, None]
    else:
        counts = [case["new"]] * len(lengths)
        s["starts"] = _starts(counts)
        s["queries"] = (1.5 * _randn(gen, sum(counts), heads * case["group"], dim)).to(TYPES[case["type"]])
        s["prior"] = torch.exp(_randn(gen, len(lengths), heads, max(need) * PAGE)) if case["prior"] else None
        s["lse"] = torch.empty(s["queries"].shape[:2], device="cuda")
    slots = _slots(s["table"].clamp(min=0), max(lengths))
    for b, n in enumerate(lengths):  # the history, written as it came
        keys, values = (_tokens(gen, n, heads, dim).to(torch.bfloat16) for _ in range(2))
        _append(s, keys, values, slots[b, :n].contiguous())
        if kind == "weigh":  # as the attention before this call left it
            rows = slice(b * case["new"], (b + 1) * case["new"])
            later = _later(n, case["new"])
            held = _values(*_quantise(keys)).transpose(0, 1)
            for h in range(heads):
                q = s["queries"][rows, h * case["group"]:(h + 1) * case["group"]].float().transpose(0, 1)
                score = torch.matmul(q, held[h].T.contiguous()) * (1.0 / math.sqrt(dim))
                score = torch.logsumexp(score.masked_fill(later, -math.inf), -1)
                s["lse"][rows, h * case["group"]:(h + 1) * case["group"]] = score.T
    return s


def _starts(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")


def _later(length, new):
    """Which tokens lie behind each of a sequence's last `new` ones."""
    return torch.arange(length, device="cuda") > torch.arange(length - new, length, device="cuda")[:, None]


def _slots(table, tokens):
    """Where the first tokens of each sequence lie: page * 128 + place."""
    place = torch.arange(tokens, device="cuda")
    return table.long()[:, place // PAGE] * PAGE + place % PAGE


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
    (s["codes"][0, slots], s["scales"][0, slots]), (s["codes"][1, slots], s["scales"][1, slots]) = _quantise(keys), _quantise(values)


def _quantise(x):
    """The codes (two to a byte, the first value low) and scale bytes of x, in runs of 32 along its last axis."""
    x = x.float().unflatten(-1, (-1, RUN))
    top = x.abs().amax(-1, keepdim=True)
    byte = (((top.view(torch.int32) + (1 << 21)) >> 23) - 2).clamp(2, 252)
    y = x.abs() / (byte << 23).view(torch.float32)
    code = ((y > 0.25).to(torch.uint8) + (y >= 0.75) + (y > 1.25) + (y >= 1.75) + (y > 2.5) + (y >= 3.5) + (y > 5.0))
    code = (code + 8 * torch.signbit(x).to(torch.uint8)).flatten(-2)
    return code[..., ::2] + 16 * code[..., 1::2], byte.squeeze(-1).to(torch.uint8)


def _values(codes, scales):
    """What codes and scale bytes stand for, in 32 bits."""
    unit = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    unit = torch.cat([unit, -unit])
    pair = torch.stack([unit.repeat(16), unit.repeat_interleave(16)], 1)
    x = pair[codes.int()].flatten(-2).unflatten(-1, (-1, RUN))
    return (x * (scales.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        from holmes_amd import clear

        if kind == "rotate":
            return tuple(s["plan"].rotate(s["positions"], s["queries"], s["keys"], inverse=case["inverse"]))
        if kind == "prompt":
            got = clear.prompt_attention(s["queries"], s["keys"], s["values"], s["starts"], most=case["high"],
                                         causal=case["causal"], ranges=case["ranges"])
            return tuple(x for x in got if x is not None)
        if kind == "weigh":
            return s["pool"].weigh(s["queries"], s["table"], s["lengths"], s["lse"], starts=s["starts"], most=case["new"],
                                   prior=s["prior"])
        got = s["pool"].evict(s["table"], s["lengths"], s["weights"], s["into"], case["keep"], recent=case["recent"])
        return (*got, *s["pool"].read(s["slots"], torch.bfloat16))
    return {"rotate": _plain_rotate, "prompt": _plain_prompt, "weigh": _plain_weigh, "evict": _plain_evict}[kind](s)


def _plain_rotate(s):
    case = s["case"]
    angle = s["positions"].double()[:, None] * s["frequencies"]
    sign = -1.0 if case["inverse"] else 1.0
    cos, sin = (s["amount"] * torch.cos(angle)).float()[:, None], (sign * s["amount"] * torch.sin(angle)).float()[:, None]

    def turned(x):
        y = x.float()
        part = y[..., :case["rotated"]]
        if case["interleaved"]:
            a, b = part[..., ::2], part[..., 1::2]
            part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = part.chunk(2, -1)
            part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([part, y[..., case["rotated"]:]], -1).to(x.dtype)

    return turned(s["queries"]), turned(s["keys"])


def _padded(starts, most, total):
    """For each sequence its first `most` rows, and which of them are its own."""
    count = starts[1:] - starts[:-1]
    i = torch.arange(most, device="cuda")
    return (starts[:-1, None] + i).clamp(max=total - 1), i < count[:, None]


def _rows_back(t, valid, group):
    """[sequences][heads][group * most][n] to [tokens][query heads][n]."""
    return t.unflatten(2, (group, -1)).permute(0, 3, 1, 2, 4)[valid].flatten(1, 2)


def _plain_prompt(s):
    case = s["case"]
    heads, group, dim, most = case["heads"], case["group"], case["dim"], case["high"]
    row, valid = _padded(s["starts"].long(), most, s["queries"].shape[0])
    x = s["queries"].float()[row].unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    keys, values = (t.float()[row].transpose(1, 2).contiguous() for t in (s["keys"], s["values"]))
    score = torch.matmul(x, keys.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(dim))
    seen = valid[:, None, None, None, :]
    if case["causal"]:
        i = torch.arange(most, device="cuda")
        seen = seen & (i <= i[:, None])
    seen = seen.expand(-1, 1, group, most, -1).flatten(2, 3)
    low = torch.where(seen, score, torch.full((), math.inf, device="cuda")).amin(-1, keepdim=True) if case["ranges"] else None
    score = torch.where(seen, score, torch.full((), -math.inf, device="cuda"))
    high = score.amax(-1, keepdim=True)
    weight = torch.exp(score - high)
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, values) / total
    sums = [high + torch.log(total)] + ([low, high] if case["ranges"] else [])
    return (_rows_back(out, valid, group).to(s["queries"].dtype), *(_rows_back(t, valid, group).squeeze(-1) for t in sums))


def _plain_weigh(s):
    case = s["case"]
    heads, group, dim, most = case["heads"], case["group"], case["dim"], case["new"]
    lengths = s["lengths"].long()
    slots = _slots(s["table"].clamp(min=0), s["table"].shape[1] * PAGE)
    keys = _values(s["codes"][0, slots], s["scales"][0, slots]).permute(0, 2, 3, 1).contiguous()
    row, valid = _padded(s["starts"].long(), most, s["queries"].shape[0])
    x = s["queries"].float()[row].unflatten(2, (heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    lse = s["lse"][row].unflatten(2, (heads, group)).permute(0, 2, 3, 1).flatten(2, 3)[..., None]
    weight = torch.exp(torch.matmul(x, keys) * (1.0 / math.sqrt(dim)) - lse)
    place = torch.arange(keys.shape[-1], device="cuda")
    there = place < lengths[:, None]
    seen = (place <= (lengths[:, None] - most + torch.arange(most, device="cuda"))[..., None]) & there[:, None]
    seen = seen[:, None, None].expand(-1, 1, group, most, -1).flatten(2, 3)
    weight = torch.where(seen, weight, torch.zeros((), device="cuda")).sum(2)
    if s["prior"] is not None:
        weight = weight + torch.where(there[:, None], s["prior"], torch.zeros((), device="cuda"))
    return weight


def _plain_evict(s):
    case = s["case"]
    keep, heads = case["keep"], case["heads"]
    lengths = s["lengths"].long()[:, None, None]
    place = torch.arange(s["table"].shape[1] * PAGE, device="cuda")
    # the weights' order (none is negative), then the lowest place; the last tokens go before all, what is none behind
    order = (s["weights"].view(torch.int32).long() << 31) + ((1 << 31) - 1 - place)
    order = torch.where(place >= lengths - case["recent"], order + (1 << 62), order)
    order = torch.where(place < lengths, order, -1 - place)
    width = min(keep, place.numel())
    kept = order.topk(width, dim=-1).indices
    kept = torch.where(kept < lengths, kept, torch.full((), place.numel(), device="cuda")).sort(-1).values
    kept = torch.nn.functional.pad(kept, (0, keep - width), value=place.numel())
    there = kept < place.numel()
    old = kept.clamp(max=place.numel() - 1)
    weights = torch.where(there, s["weights"].gather(2, old), torch.zeros((), device="cuda"))
    page = s["table"].long()[:, None].expand(-1, heads, -1).gather(2, old // PAGE)
    head = torch.arange(heads, device="cuda")[:, None].expand(kept.shape)
    new = _slots(s["into"], keep)[:, None].expand(kept.shape)
    slot, head, new = (page * PAGE + old % PAGE)[there], head[there], new[there]
    s["codes"][:, new, head], s["scales"][:, new, head] = s["codes"][:, slot, head], s["scales"][:, slot, head]
    got = _values(s["codes"][:, s["slots"]], s["scales"][:, s["slots"]]).to(torch.bfloat16)
    return (torch.where(there, kept, -1).to(torch.int32), torch.clamp(s["lengths"], max=keep), weights, got[0], got[1])


def work(case):
    kind, heads, dim = case["kind"], case["heads"], case["dim"]
    if kind == "rotate":
        n, size = case["tokens"], TYPES[case["type"]].itemsize
        values = n * (heads + case["kv_heads"]) * dim
        return {"bytes": 2 * values * size + 8 * n, "flops": 3 * values * case["rotated"] // dim}
    lengths = _lengths(case)
    held = heads * (dim // 2 + dim // RUN)  # bytes of one token's keys, or values, in the cache
    if kind == "evict":
        kept = [min(n, case["keep"]) for n in lengths]
        return {"bytes": sum(lengths) * heads * 4 + sum(kept) * (2 * 2 * held + heads * 8) +
                len(lengths) * case["keep"] * (2 * heads * dim * 2 + 8), "flops": sum(lengths) * heads * 4}
    query_heads, size = heads * case["group"], TYPES[case["type"]].itemsize
    if kind == "prompt":
        tokens, sums = sum(lengths), 3 if case["ranges"] else 1
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        return {"bytes": tokens * (2 * (query_heads + heads) * dim * size + query_heads * 4 * sums),
                "flops": pairs * query_heads * (4 * dim + 5)}
    new = case["new"]
    pairs = sum(new * n - new * (new - 1) // 2 for n in lengths)
    rows = new * len(lengths) * query_heads
    return {"bytes": sum(lengths) * (held + heads * 4 * (2 if case["prior"] else 1)) + rows * (dim * size + 4),
            "flops": pairs * query_heads * (2 * dim + 4)}


# ---------------------------------------------------------------------------- in 64 bits
def _held(x):
    """The values that the 4-bit form keeps of x, from its definition."""
    x = x.double().unflatten(-1, (-1, RUN))
    top = x.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(top)
    exponent = torch.where(top == 0, torch.full_like(exponent, -200), exponent - 3 + (mantissa >= 0.875).int())
    unit = torch.ldexp(torch.ones_like(top), exponent.clamp(2 - 127, 252 - 127))
    y = x.abs() / unit
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0).double())
    y = (torch.round(y / step) * step).clamp(max=6.0)
    return torch.copysign(y * unit, x).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "rotate":
        return _exact_rotate(case, s)
    lengths, heads = _lengths(case), case["heads"]
    if case["kind"] == "prompt":
        outs, at = [], 0
        for n in lengths:
            outs.append(_exact_attend(*(s[k][at:at + n].double() for k in ("queries", "keys", "values")), case))
            at += n
        return tuple(torch.cat(p) for p in zip(*outs))
    # the same inputs as prepare's, in the order in which it makes them
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + 13)
    need = [-(-n // PAGE) for n in lengths]
    width = max(need) * PAGE
    fresh = -(-case["keep"] // PAGE) if case["kind"] == "evict" else 0
    torch.randperm(sum(need) + fresh * len(lengths) + 3, generator=gen, device="cuda")
    if case["kind"] == "evict":
        _randn(gen, len(lengths), heads, width)
    else:
        _randn(gen, case["new"] * len(lengths), heads * case["group"], case["dim"])
        if case["prior"]:
            _randn(gen, len(lengths), heads, width)
    outs = []
    for b, n in enumerate(lengths):
        keys, values = (_held(_tokens(gen, n, heads, case["dim"]).to(torch.bfloat16)) for _ in range(2))
        if case["kind"] == "evict":
            outs.append(_exact_evict(case, s["weights"][b, :, :n], keys, values))
        else:
            rows = slice(b * case["new"], (b + 1) * case["new"])
            got = _exact_weigh(case, s["queries"][rows].double(), s["lse"][rows].double(), keys)
            if case["prior"]:
                got += s["prior"][b, :, :n].double()
            outs.append(torch.nn.functional.pad(got, (0, width - n)))
    if case["kind"] == "weigh":
        return torch.stack(outs)
    kept, weights, keys, values = (torch.stack(p) for p in zip(*outs))
    return (kept, torch.tensor([min(n, case["keep"]) for n in lengths]), weights, keys.flatten(0, 1), values.flatten(0, 1))


def _exact_rotate(case, s):
    pairs = case["rotated"] // 2
    f = [math.exp(-math.log(BASE) * i / pairs) for i in range(pairs)]
    given, amount = _scaling(case), 1.0
    if case["scaling"] == "linear":
        f = [x / 8.0 for x in f]
    elif case["scaling"] == "wavelength":
        for i, x in enumerate(f):
            length = 2 * math.pi / x
            if length > ORIGINAL / given[1]:
                f[i] = x / given[0]
            elif length > ORIGINAL / given[2]:
                part = (ORIGINAL / length - given[1]) / (given[2] - given[1])
                f[i] = (1 - part) * x / given[0] + part * x
    elif case["scaling"] == "ramp":
        amount = 1.0 + 0.1 * math.log(given[0])

        def pair_of(turns):  # the (fractional) pair that makes so many turns in the original length
            return pairs * math.log(ORIGINAL / (2 * math.pi * turns)) / math.log(BASE)

        first, last = max(0, math.floor(pair_of(given[2]))), min(2 * pairs - 1, math.ceil(pair_of(given[1])))
        for i, x in enumerate(f):
            part = min(1.0, max(0.0, (i - first) / max(last - first, 1e-3)))
            f[i] = x * (1 - part) + x / given[0] * part
    turn = torch.polar(torch.full((), amount, dtype=torch.float64, device="cuda"),
                       s["positions"].double()[:, None] * torch.tensor(f, dtype=torch.float64, device="cuda"))[:, None]
    turn = turn.conj() if case["inverse"] else turn

    def turned(x):
        x = x.double().clone()
        at = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
        if not case["interleaved"]:
            at = slice(0, pairs), slice(pairs, 2 * pairs)
        z = torch.complex(x[..., at[0]].contiguous(), x[..., at[1]].contiguous()) * turn
        x[..., at[0]], x[..., at[1]] = z.real, z.imag
        return x

    return turned(s["queries"]), turned(s["keys"])


def _exact_attend(queries, keys, values, case):
    n, group = keys.shape[0], case["group"]
    out = torch.zeros_like(queries)
    lse, low, high = (torch.zeros_like(queries[..., 0]) for _ in range(3))
    for h in range(queries.shape[1]):
        score = queries[:, h] @ keys[:, h // group].T / math.sqrt(case["dim"])
        hidden = _later(n, n) if case["causal"] else torch.zeros_like(score, dtype=torch.bool)
        low[:, h] = score.masked_fill(hidden, math.inf).amin(1)
        score = score.masked_fill(hidden, -math.inf)
        high[:, h] = score.amax(1)
        lse[:, h] = torch.logsumexp(score, 1)
        out[:, h] = torch.softmax(score, 1) @ values[:, h // group]
    return (out, lse, low, high) if case["ranges"] else (out, lse)


def _exact_weigh(case, queries, lse, keys):
    got = torch.zeros((keys.shape[1], keys.shape[0]), dtype=torch.float64, device="cuda")
    hidden = _later(keys.shape[0], queries.shape[0])
    for h in range(queries.shape[1]):
        score = queries[:, h] @ keys[:, h // case["group"]].T / math.sqrt(case["dim"])
        got[h // case["group"]] += torch.exp(score - lse[:, h, None]).masked_fill(hidden, 0.0).sum(0)
    return got


def _exact_evict(case, weights, keys, values):
    heads, n = weights.shape
    keep, all_kept, rest = case["keep"], [], []
    for h in range(heads):
        last = max(0, n - case["recent"])
        heavy = torch.sort(weights[h, :last], descending=True, stable=True).indices[:max(0, keep - (n - last))]
        kept = torch.sort(torch.cat([heavy, torch.arange(last, n, device="cuda")])).values
        spare = keep - kept.numel()
        all_kept.append(torch.nn.functional.pad(kept, (0, spare), value=-1))
        rest.append((torch.nn.functional.pad(weights[h, kept].double(), (0, spare)),
                     *(torch.nn.functional.pad(x[kept, h], (0, 0, 0, spare)) for x in (keys, values))))
    weights, keys, values = (torch.stack(p) for p in zip(*rest))
    return torch.stack(all_kept), weights, keys.transpose(0, 1), values.transpose(0, 1)
