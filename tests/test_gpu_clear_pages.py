"""The 4-bit cleartext pages and the attention over them (holmes_amd.clear) against plain float64 models.

Writing and reading are exact by the format's definition.  Attention's tolerance counts, for a row with
scores s = scale q.k over n tokens and probabilities p: the scores' 32-bit sums of D products, an fp16
query's two bf16 parts (2^-17 of each), the probabilities' two bf16 parts (2^-17) and the exponential's
and its argument's roundings; the sums over a lane's n / 16 tokens; half a step of the output's type (below its least normal number, one step).
"""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

PAGE = 128
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def held(x):
    """The values that a page keeps of x (CPU, float64), by nearest point of the grid, ties to the even code."""
    x = x.detach().cpu().double()
    runs = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = runs.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top)
    mant, exp = torch.frexp(torch.where(fine & (top > 0), top, torch.ones_like(top)))
    e = exp - 3 + (mant >= 0.875).int()
    e = torch.where(top == 0, torch.full_like(e, -125), e).clamp(-125, 125)
    unit = torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())
    y = torch.where(fine, runs.abs() / unit, torch.zeros_like(runs))
    mids = (GRID[1:] + GRID[:-1]) / 2
    code = (y.unsqueeze(-1) > mids).sum(-1)
    tie = (y.unsqueeze(-1) == mids).any(-1)
    code = code + (tie & (code % 2 == 1)).long()   # between an odd and an even code: the even one
    out = torch.where(fine, torch.copysign(GRID[code] * unit, runs), torch.full_like(runs, math.nan))
    return out.reshape(x.shape)


def same(got, want):
    want = want.to(got.dtype) if got.dtype != torch.float16 else want.clamp(-65504, 65504).to(torch.float16)
    got = got.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert torch.equal(got[ok], want[ok])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("tokens,heads", [(1, 1), (33, 3), (257, 8)])
def test_pages_hold_what_the_format_says(tokens, heads, kind, dim):
    from holmes_amd import clear

    print("pages", tokens, heads, kind, dim, flush=True)
    g = torch.Generator().manual_seed(tokens * 10 + heads)
    pool = clear.ClearKVPages(5, kv_heads=heads, head_dim=dim)
    slots = torch.randperm(5 * PAGE, generator=g)[:tokens]
    x = (torch.randn((2, tokens, heads, dim), generator=g) * torch.exp(3 * torch.randn((2, tokens, heads, 1), generator=g)))
    x = x.to(TYPES[kind])
    pool.append(x[0].cuda(), x[1].cuda(), slots.cuda())
    for out in TYPES.values():
        k, v = pool.read(slots.cuda(), out)
        same(k, held(x[0]))
        same(v, held(x[1]))


def test_pages_at_the_formats_borders():
    """Ties, the largest magnitudes that round up to the next unit, zeros, the types' least and largest
    values, infinities and NaN (of their run of 32 alone)."""
    from holmes_amd import clear

    print("pages borders", flush=True)
    ticks = torch.arange(0, 57) / 8.0          # every midpoint and point of the grid in steps of 1/8 up to 7
    rows = []
    for top in (4.0, 6.0, 6.9921875, 7.0, 7.5):
        for scale in (1.0, 2.0**-90, 2.0**100):
            r = torch.zeros(128)
            r[:57] = ticks.clamp(max=top)
            r[57] = -top
            r[64:121] = -ticks.clamp(max=top)
            r[31] = r[63] = r[95] = r[127] = top
            rows.append(r * scale)
    rows.append(torch.zeros(128))
    rows.append(torch.full((128,), 3.3895314e38))
    rows.append(torch.full((128,), 2.0**-126))
    odd = torch.randn(128, generator=torch.Generator().manual_seed(3))
    odd[5], odd[40], odd[70] = math.inf, math.nan, -math.inf
    rows.append(odd)
    x = torch.stack(rows)[:, None, :]
    pool = clear.ClearKVPages(1, kv_heads=1)
    slots = torch.arange(len(x))
    pool.append(x.cuda(), x.flip(0).cuda(), slots.cuda())
    k, v = pool.read(slots.cuda(), torch.float32)
    same(k, held(x))
    same(v, held(x.flip(0)))
    k, _ = pool.read(slots.cuda(), torch.float16)
    same(k, held(x))


def test_slots_outside_the_pool_and_strided_inputs():
    from holmes_amd import clear

    print("pages slots", flush=True)
    g = torch.Generator().manual_seed(5)
    pool = clear.ClearKVPages(2, kv_heads=3)
    first = torch.randn((256, 3, 128), generator=g)
    pool.append(first.cuda(), first.cuda(), torch.arange(256).cuda())
    wide = torch.randn((9, 3, 2, 129), generator=g).to(torch.bfloat16).cuda()   # keys and values interleaved, odd strides
    slots = torch.tensor([7, -1, 255, 256, 2**40, -5, 0, 128, 127]).cuda()
    pool.append(wide[:, :, 0, 1:], wide[:, :, 1, 1:], slots)
    want_k, want_v = held(first), held(first)
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < 256:
            want_k[s], want_v[s] = held(wide[i, :, 0, 1:]), held(wide[i, :, 1, 1:])
    k, v = pool.read(torch.arange(256).cuda(), torch.float32)
    same(k, want_k)
    same(v, want_v)
    k, v = pool.read(slots, torch.bfloat16)
    for i, s in enumerate(slots.tolist()):
        same(k[i], want_k[s] if 0 <= s < 256 else torch.zeros(3, 128))


# ---------------------------------------------------------------------------- attention
def build(seqs, heads, dim, g, spare=2, kind=torch.bfloat16, spread=1.0):
    """A pool with the sequences' tokens in shuffled pages, the table, and the held keys and values (float64)."""
    from holmes_amd import clear

    need = [-(-n // PAGE) for n in seqs]
    pool = clear.ClearKVPages(sum(need) + spare, kv_heads=heads, head_dim=dim)
    pool.buf.random_(0, 250)  # what earlier owners of the pages left
    order = torch.randperm(sum(need) + spare, generator=g)
    table = torch.full((len(seqs), max(max(need), 1)), 2**30, dtype=torch.int32)
    keys, values, at = [], [], 0
    for b, n in enumerate(seqs):
        table[b, :need[b]] = order[at:at + need[b]].int()
        at += need[b]
        k, v = (spread * torch.randn((n, heads, dim), generator=g).to(kind) for _ in range(2))
        t = torch.arange(n)
        slots = table[b].long()[t // PAGE] * PAGE + t % PAGE
        pool.append(k.cuda(), v.cuda(), slots.cuda())
        keys.append(held(k))
        values.append(held(v))
    return pool, table.cuda(), keys, values


def check(got, q, keys, values, counts, *, causal=True, scale=None, there=None):
    """Every row of ``got`` against float64, within the tolerance of the module's docstring."""
    dim, heads = q.shape[2], keys[0].shape[1]
    group = q.shape[1] // heads
    scale = scale or 1.0 / math.sqrt(dim)
    out, lse = got.out.cpu().double(), got.lse.cpu().double()
    half = torch.finfo(q.dtype).eps / 2
    qq = q.cpu().double()
    parts = 2.0**-17 if q.dtype == torch.float16 else 0.0
    at = 0
    for b, new in enumerate(counts):
        n = keys[b].shape[0]
        for i in range(new):
            see = torch.arange(n) <= n - new + i if causal else torch.ones(n, dtype=torch.bool)
            if there is not None:
                see = see & there[b]
            for h in range(q.shape[1]):
                o, x = out[at + i, h], lse[at + i, h]
                lo_hi = None if got.low is None else (got.low[at + i, h].item(), got.high[at + i, h].item())
                if not see.any():
                    assert (o == 0).all() and x == -math.inf and lo_hi in (None, (math.inf, -math.inf)), (b, i, h)
                    continue
                k, v = keys[b][see, h // group], values[b][see, h // group]
                s = scale * (k @ qq[at + i, h])
                d = scale * (k.abs() @ qq[at + i, h].abs()).max() * (2.0**-24 * (dim + 8) + parts)
                want = torch.logsumexp(s, 0)
                p = torch.softmax(s, 0)
                depth = 2.0**-24 * (len(s) / 16 + 64)
                e = 2 * d + 2.0**-22 * (2 + (s.max() - s.min()).item()) + depth
                assert abs(x - want) <= e + 2.0**-22 * abs(want), (b, i, h, float(x), float(want))
                w = p @ v
                tol = half * w.abs() + (2 * e + 2.0**-17) * (p @ v.abs()) + (2.0**-24 if q.dtype == torch.float16 else 2.0**-133)
                assert ((o - w).abs() <= tol).all(), (b, i, h, float(((o - w).abs() - tol).max()))
                if lo_hi:
                    t = d + 2.0**-22 * s.abs().max()
                    assert abs(lo_hi[0] - s.min()) <= t and abs(lo_hi[1] - s.max()) <= t, (b, i, h)
        at += new


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim", [(1, 1, 128), (2, 4, 128), (3, 5, 64), (1, 17, 64), (2, 8, 128)])
@pytest.mark.parametrize("ranges", [False, True])
def test_single_tokens(heads, group, dim, kind, ranges):
    print("single", heads, group, dim, kind, ranges, flush=True)
    g = torch.Generator().manual_seed(heads * 100 + group)
    seqs = [1, 2, 63, 64, 65, 127, 128, 129, 700, 0, 16, 1000]
    pool, table, keys, values = build(seqs, heads, dim, g)
    q = torch.randn((len(seqs), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    got = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=ranges)
    check(got, q, keys, values, [1] * len(seqs))
    again = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=ranges)
    assert torch.equal(got.out, again.out) and torch.equal(got.lse, again.lse)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (1, 7, 64), (2, 1, 128)])
def test_prompts(heads, group, dim, causal, kind):
    """New tokens behind histories, counts of 0 and 1 and all of a sequence among them, with a sequence that
    has more queries than tokens: its first rows see nothing."""
    print("prompts", heads, group, dim, causal, kind, flush=True)
    g = torch.Generator().manual_seed(7 + group)
    seqs, counts = [40, 300, 5, 129, 7], [40, 33, 0, 1, 12]
    pool, table, keys, values = build(seqs, heads, dim, g)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32).cuda()
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    for most in (None, 40):
        got = pool.attend(q, table, lengths, starts=starts, most=most, causal=causal, ranges=True)
        check(got, q, keys, values, counts, causal=causal)


def test_long_history_is_split_and_joined():
    print("long", flush=True)
    g = torch.Generator().manual_seed(11)
    seqs = [20011]
    pool, table, keys, values = build(seqs, 2, 128, g)
    q = torch.randn((1, 8, 128), generator=g).to(torch.bfloat16).cuda()
    got = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True)
    check(got, q, keys, values, [1])
    wide = torch.full((1, 3 * table.shape[1]), -1, dtype=torch.int32).cuda()   # a table with room to grow
    wide[:, :table.shape[1]] = table
    check(pool.attend(q, wide, torch.tensor(seqs, dtype=torch.int32).cuda()), q, keys, values, [1])


def test_a_longer_prompt():
    print("longer prompt", flush=True)
    g = torch.Generator().manual_seed(12)
    seqs = [777]
    pool, table, keys, values = build(seqs, 1, 128, g)
    q = torch.randn((777, 2, 128), generator=g).to(torch.bfloat16).cuda()
    starts = torch.tensor([0, 777], dtype=torch.int32).cuda()
    got = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts, ranges=True)
    check(got, q, keys, values, [777])


def test_strided_queries_scales_and_large_scores():
    print("strided", flush=True)
    g = torch.Generator().manual_seed(13)
    seqs = [200, 90]
    pool, table, keys, values = build(seqs, 2, 64, g, spread=30.0)
    q = torch.randn((2, 6, 67), generator=g).to(torch.bfloat16).cuda()[:, :, 3:]
    assert q.stride(1) == 67
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    check(pool.attend(q, table, lengths, scale=0.7, ranges=True), q, keys, values, [1, 1], scale=0.7)
    turned = torch.randn((6, 2, 64), generator=g).to(torch.float16).cuda().transpose(0, 1)
    check(pool.attend(turned, table, lengths), turned, keys, values, [1, 1])


def test_pages_that_are_not_there():
    """A page number outside the pool takes its 128 tokens away, wherever it stands."""
    print("missing pages", flush=True)
    g = torch.Generator().manual_seed(17)
    seqs = [500, 300, 100]
    pool, table, keys, values = build(seqs, 2, 128, g)
    q = torch.randn((3, 8, 128), generator=g).to(torch.bfloat16).cuda()
    table[0, 1], table[1, 2], table[2, 0] = -1, pool.pages, 2**31 - 1
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    there[0][128:256] = there[1][256:] = there[2][:] = False
    got = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True)
    check(got, q, keys, values, [1, 1, 1], there=there)


def test_lengths_beyond_the_table_and_empty_calls():
    print("lengths", flush=True)
    g = torch.Generator().manual_seed(19)
    pool, table, keys, values = build([128, 128], 1, 128, g)
    q = torch.randn((2, 4, 128), generator=g).to(torch.bfloat16).cuda()
    got = pool.attend(q, table, torch.tensor([10**6, -3], dtype=torch.int32).cuda())
    one = pool.attend(q[:1], table[:1], torch.tensor([128], dtype=torch.int32).cuda())
    assert torch.equal(got.out[:1], one.out) and (got.out[1] == 0).all() and (got.lse[1] == -math.inf).all()
    none = pool.attend(q[:0], table[:0], torch.zeros(0, dtype=torch.int32).cuda())
    assert none.out.shape == (0, 4, 128)
    bare = pool.attend(q, table[:, :0], torch.tensor([5, 5], dtype=torch.int32).cuda())
    assert (bare.out == 0).all() and (bare.lse == -math.inf).all()


@pytest.mark.parametrize("dim", [64, 128])
def test_nan_reaches_the_rows_that_see_it(dim):
    """A NaN in the cache is NaN for the rows that see its token (of a value: in its run's 32 dims) and
    changes nothing for the rows before it, nor from behind a sequence's end."""
    print("nan", dim, flush=True)
    g = torch.Generator().manual_seed(23)
    n, cut = 150, 20
    from holmes_amd import clear

    for side in ("key", "value"):
        x = torch.randn((2, n + 10, 1, dim), generator=g)
        clean = x.clone()
        x[0 if side == "key" else 1, n - cut, 0, 40] = math.nan
        x[:, n:] = math.inf                       # behind the end
        table = torch.tensor([[1, 0]], dtype=torch.int32).cuda()
        q = torch.randn((n, 2, dim), generator=g).to(torch.bfloat16).cuda()
        got = []
        for y in (x, clean):
            pool = clear.ClearKVPages(2, kv_heads=1, head_dim=dim)
            t = torch.arange(n + 10)
            pool.append(y[0].cuda(), y[1].cuda(), (table[0].long().cpu()[t // PAGE] * PAGE + t % PAGE).cuda())
            got.append(pool.attend(q, table, torch.tensor([n], dtype=torch.int32).cuda(), ranges=True,
                                   starts=torch.tensor([0, n], dtype=torch.int32).cuda()))
        a, b = got
        first = n - cut
        assert torch.equal(a.out[:first], b.out[:first]) and torch.equal(a.lse[:first], b.lse[:first])
        assert torch.equal(a.low[:first], b.low[:first]) and torch.equal(a.high[:first], b.high[:first])
        if side == "key":
            assert all(torch.isnan(t[first:]).all() for t in a)
        else:
            assert torch.isnan(a.out[first:, :, 32:64]).all()
            assert torch.equal(a.out[first:, :, :32], b.out[first:, :, :32])
            assert torch.equal(a.out[first:, :, 64:], b.out[first:, :, 64:])
            assert torch.equal(a.lse[first:], b.lse[first:])


def test_another_stream_and_a_graph():
    """On a stream of its own, and captured: every replay gives the eager result on new inputs."""
    print("stream and graph", flush=True)
    g = torch.Generator().manual_seed(29)
    seqs = [900, 31]
    pool, table, keys, values = build(seqs, 2, 128, g)
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    q = torch.randn((2, 8, 128), generator=g).to(torch.bfloat16).cuda()
    want = pool.attend(q, table, lengths, ranges=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.attend(q, table, lengths, ranges=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    k = torch.randn((2, 2, 128), generator=g).cuda()
    slots = torch.tensor([int(table[0, 899 // PAGE]) * PAGE + 899 % PAGE, -1]).cuda()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        pool.append(k, k, slots)
        rec = pool.attend(q, table, lengths, ranges=True)
    for i in range(3):
        k.copy_(torch.randn((2, 2, 128), generator=g))
        q.copy_(torch.randn((2, 8, 128), generator=g).to(torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in rec]
        pool.append(k, k, slots)
        want = pool.attend(q, table, lengths, ranges=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_softmax_ranges_hold_every_row():
    from holmes_amd import clear

    print("ranges", flush=True)
    g = torch.Generator().manual_seed(31)
    seqs = [400]
    pool, table, keys, values = build(seqs, 2, 128, g)
    q = torch.randn((400, 4, 128), generator=g).to(torch.bfloat16).cuda()
    got = pool.attend(q, table, torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True,
                      starts=torch.tensor([0, 400], dtype=torch.int32).cuda())
    r = clear.softmax_ranges(got.low, got.high, got.lse)
    for i in (0, 1, 57, 399):
        for h in range(4):
            s = keys[0][:i + 1, h // 2] @ q[i, h].cpu().double() / math.sqrt(128)
            mapped = (s - r.score_shift) / 2
            assert r.exp_interval[0] < mapped.min() and mapped.max() < r.exp_interval[1]
            total = torch.exp(2 * mapped).sum()
            assert r.rsqrt_interval[0] < total < r.rsqrt_interval[1]
