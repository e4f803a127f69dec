"""Attention over whole prompts (holmes_amd.clear.prompt_attention) against float64.

Tolerance, for a row with scores s = scale q.k over n tokens and probabilities p: the scores' 32-bit sums of D products
(e below: 2^-24 (D + 8) of the sum of magnitudes, twice, for the score and the reference's; the exponential's and its
argument's roundings, 2^-22 (2 + max s - min s); the sum over a lane's n / 2 tokens, 2^-24 (n / 2 + 64)); a probability in
the type of the values (half a step, 2^-8 or 2^-11 of it at the worst, taken twice); half a
step of the output's type (below its least normal number, one step)."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_prompt import starts_of  # noqa: E402

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def check(got, q, k, v, counts, *, causal=True, scale=None, first=0):
    """Every row of `got` against float64; rows before `first` belong to no sequence."""
    dim, heads = q.shape[2], k.shape[1]
    group = q.shape[1] // heads
    scale = scale or 1.0 / math.sqrt(dim)
    half = torch.finfo(q.dtype).eps / 2
    least = 2.0**-24 if q.dtype == torch.float16 else 2.0**-133
    q, k, v = (x.cpu().double() for x in (q, k, v))
    out, lse = got.out.cpu().double(), got.lse.cpu().double()
    at = first
    for n in counts:
        if n == 0:
            continue
        see = torch.ones(n, n, dtype=torch.bool)
        see = see.tril() if causal else see
        for h in range(q.shape[1]):
            x, y, z = q[at:at + n, h], k[at:at + n, h // group], v[at:at + n, h // group]
            s = scale * (x @ y.T)
            d = (scale * (x.abs() @ y.abs().T)).masked_fill(~see, 0.0).amax(1) * 2.0**-24 * (dim + 8)
            low, high = s.masked_fill(~see, math.inf).amin(1), s.masked_fill(~see, -math.inf).amax(1)
            s = s.masked_fill(~see, -math.inf)
            want = torch.logsumexp(s, 1)
            p = torch.softmax(s, 1)
            e = 2 * d + 2.0**-22 * (2 + high - low) + 2.0**-24 * (n / 2 + 64)
            off = (lse[at:at + n, h] - want).abs()
            assert (off <= e + 2.0**-22 * want.abs()).all(), (n, h, float((off - e).max()))
            w = p @ z
            tol = half * w.abs() + ((2 * e + 2 * half)[:, None]) * (p @ z.abs()) + least
            off = (out[at:at + n, h] - w).abs()
            assert (off <= tol).all(), (n, h, float((off - tol).max()))
            if got.low is not None:
                t = d + 2.0**-22 * torch.maximum(low.abs(), high.abs())
                assert ((got.low[at:at + n, h].cpu().double() - low).abs() <= t).all()
                assert ((got.high[at:at + n, h].cpu().double() - high).abs() <= t).all()
        at += n


def inputs(g, tokens, heads, group, dim, kind, spread=1.0):
    return [(spread * torch.randn((tokens, n, dim), generator=g)).to(TYPES[kind]).cuda() for n in (heads * group, heads, heads)]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal,ranges", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (1, 7, 64), (3, 1, 128), (8, 2, 64), (1, 150, 64)])
def test_packed(heads, group, dim, causal, ranges, kind):
    """One token and none; lengths at the borders of units and tiles."""
    print("packed", heads, group, dim, causal, ranges, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 10 + group)
    counts = [1, 0, 2, 63, 64, 65, 0, 128, 129, 31, 200, 1] if group < 100 else [1, 5, 70]
    q, k, v = inputs(g, sum(counts), heads, group, dim, kind)
    got = clear_call(q, k, v, starts_of(counts), causal=causal, ranges=ranges)
    check(got, q, k, v, counts, causal=causal)
    again = clear_call(q, k, v, starts_of(counts), most=200, causal=causal, ranges=ranges)
    assert torch.equal(got.out, again.out) and torch.equal(got.lse, again.lse)


def clear_call(*a, **k):
    from holmes_amd import clear

    return clear.prompt_attention(*a, **k)


@pytest.mark.parametrize("kind,heads,group,dim,tokens", [("bf16", 2, 4, 128, 1025), ("fp16", 3, 5, 64, 777), ("bf16", 1, 1, 64, 1),
                                                         ("fp16", 1, 2, 128, 2000)])
def test_one_sequence(kind, heads, group, dim, tokens):
    print("one", kind, heads, group, dim, tokens, flush=True)
    g = torch.Generator().manual_seed(tokens)
    q, k, v = inputs(g, tokens, heads, group, dim, kind, spread=2.0)
    for causal in (True, False):
        check(clear_call(q, k, v, causal=causal, ranges=True), q, k, v, [tokens], causal=causal)
    check(clear_call(q, k, v, scale=0.01), q, k, v, [tokens], scale=0.01)


@pytest.mark.parametrize("kind,heads,group,dim", [("bf16", 1, 2, 128), ("fp16", 2, 1, 64)])
@pytest.mark.parametrize("causal,ranges", [(True, True), (False, False), (True, False), (False, True)])
def test_rows_in_parts(kind, heads, group, dim, causal, ranges):
    """Few rows of many tokens: parts of a tile's tokens join; some tiles have one part, some rows see nothing of a part."""
    print("parts", kind, heads, group, dim, causal, ranges, flush=True)
    from holmes_amd import _native as nat

    g = torch.Generator().manual_seed(20)
    for counts in ([1500], [700, 3, 1300, 513]):
        n = sum(counts)
        assert nat.lib().hck_prompt_attend_workspace_bytes(n, len(counts), heads, group, dim, max(counts), causal) > 0
        q, k, v = inputs(g, n, heads, group, dim, kind, spread=1.5)
        got = clear_call(q, k, v, starts_of(counts), most=max(counts), causal=causal, ranges=ranges)
        check(got, q, k, v, counts, causal=causal)
        again = clear_call(q, k, v, starts_of(counts), most=max(counts), causal=causal, ranges=ranges)
        assert torch.equal(got.out, again.out) and torch.equal(got.lse, again.lse)
    k[1200, 0, 2], v[900, 0, 1] = math.nan, math.inf   # of the third sequence, 703 .. 2002, and the same parts of others
    bad = clear_call(q, k, v, starts_of(counts), most=max(counts), causal=causal)
    lost = torch.isnan(bad.lse).any(1).cpu()
    want = torch.zeros(n, dtype=torch.bool)
    want[(1200 if causal else 703):2003] = True
    assert torch.equal(lost, want) and torch.isnan(bad.out[want.cuda()][:, :group]).all()
    rows = torch.zeros(n, dtype=torch.bool)
    rows[(900 if causal else 703):2003] = True
    rows &= ~want
    assert torch.isposinf(bad.out[rows.cuda()][:, :group, 1]).all() and torch.isfinite(bad.out[~(rows | want).cuda()]).all()


def test_many_sequences():
    """More than a wave's lanes, of very different lengths, with `most` and without."""
    print("many", flush=True)
    g = torch.Generator().manual_seed(2)
    counts = [(7 * i) % 60 for i in range(150)] + [400, 1, 0, 33]
    q, k, v = inputs(g, sum(counts), 2, 3, 64, "bf16")
    for most in (None, 400):
        check(clear_call(q, k, v, starts_of(counts), most=most, ranges=True), q, k, v, counts)


def test_rows_that_no_sequence_covers_are_left_alone():
    print("uncovered", flush=True)
    from holmes_amd import _native as nat

    g = torch.Generator().manual_seed(3)
    counts, first, tail = [40, 70], 10, 25
    n = first + sum(counts) + tail
    q, k, v = inputs(g, n, 2, 2, 128, "bf16")
    starts = (starts_of(counts) + first).int()
    check(clear_call(q, k, v, starts, ranges=True), q, k, v, counts, first=first)
    # into buffers of the caller's
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 9.0).cuda()
    nat.check(nat.lib().hck_prompt_attend(q.data_ptr(), k.data_ptr(), v.data_ptr(), nat.HCK_BF16, n, 2, 2, 128, 512, 128, 256,
                                          128, 256, 128, starts.data_ptr(), 2, 60, 1, 0.1, out.data_ptr(), lse.data_ptr(), None,
                                          None, None, 0, torch.cuda.current_stream().cuda_stream), "hck_prompt_attend")
    torch.cuda.synchronize()
    rows = torch.zeros(n, dtype=torch.bool)
    rows[:first] = rows[-tail:] = rows[first + 40 + 60:first + 110] = True     # 60: the second sequence's rest
    assert (out.cpu()[rows] == 7).all() and (lse.cpu()[rows] == 9).all() and not (out.cpu()[~rows] == 7).any()


def test_strides():
    """Tensors side by side, heads before tokens, broadcast heads and tokens, odd addresses."""
    print("strides", flush=True)
    g = torch.Generator().manual_seed(4)
    n, heads, dim = 150, 2, 64
    both = torch.randn((n, 8 + 2 * heads, dim), generator=g).to(torch.bfloat16).cuda()
    cuts = [both[:, :8], both[:, 8:10], both[:, 10:]]
    odd = [torch.randn((n, h, dim + 1), generator=g).to(torch.bfloat16).cuda()[..., 1:] for h in (4, 2, 2)]
    across = [torch.randn((h, n, dim), generator=g).to(torch.float16).cuda().transpose(0, 1) for h in (4, 2, 2)]
    base = torch.randn((1, 1, dim), generator=g).to(torch.bfloat16).cuda()
    same = [torch.randn((n, 4, dim), generator=g).to(torch.bfloat16).cuda(), base.expand(n, 2, dim), base.expand(n, 2, dim)]
    apart = [both.new_zeros(12 * n * dim + 1)[1:].view(n, 12, dim).copy_(both)[:, a:b] for a, b in ((0, 8), (8, 10), (10, 12))]
    for q, k, v in (cuts, odd, across, same, apart):
        check(clear_call(q, k, v, starts_of([100, 50]), ranges=True), q, k, v, [100, 50])


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_infinities_and_nan_reach_who_sees_them(dim, kind):
    """A value that is none is seen by its own rows and later ones; a key by the same, in their sums; a query by its row."""
    print("odd", dim, kind, flush=True)
    g = torch.Generator().manual_seed(5)
    counts, heads, group = [130, 90], 1, 3
    q, k, v = inputs(g, 220, heads, group, dim, kind)
    clean = clear_call(q, k, v, starts_of(counts), ranges=True)
    for at, value in ((70, math.nan), (71, math.inf), (129, -math.inf), (0, math.nan), (128, math.nan)):
        x = v.clone()
        x[at, 0, 5] = value
        got = clear_call(q, k, x, starts_of(counts), ranges=True)
        assert torch.equal(got.lse, clean.lse) and torch.equal(got.low, clean.low)
        want = clean.out.clone()
        want[at:130, :, 5] = value
        same = (got.out == want) | (torch.isnan(got.out) & torch.isnan(want))
        near = (got.out.float() - want.float()).abs() <= 2 * torch.finfo(got.out.dtype).eps * (1 + want.float().abs())
        assert (same | near).all()
        assert torch.equal(got.out[130:], clean.out[130:])
        y = k.clone()
        y[at, 0, 3] = value if math.isnan(value) else math.nan
        got = clear_call(q, y, v, starts_of(counts), ranges=True)
        bad = torch.zeros(220, dtype=torch.bool)
        bad[at:130] = True
        for t in got:
            lost = torch.isnan(t).cpu().flatten(1)
            assert lost[bad].all() and not lost[~bad].any()
    x = q.clone()
    x[77, 1, 0] = math.nan
    got = clear_call(x, k, v, starts_of(counts), ranges=True)
    for t in got:
        lost = torch.isnan(t).cpu().flatten(2 if t.dim() == 3 else 1).reshape(220, heads * group, -1)
        assert lost[77, 1].all() and lost.flatten(1).any(1).sum() == 1 and not lost[77, [0, 2]].any()


def test_large_and_far_values():
    """Averages of values up to the type's largest stay finite; scores of 10^5 and beyond keep a sum."""
    print("large", flush=True)
    g = torch.Generator().manual_seed(6)
    for kind, size in (("bf16", 3.3e38), ("fp16", 65000.0)):
        q, k, v = inputs(g, 500, 1, 2, 64, kind)
        v = (torch.sign(v.float()) * size).to(TYPES[kind])
        check(clear_call(q, k, v, causal=False), q, k, v, [500], causal=False)
        v = torch.full_like(v, size)
        got = clear_call(q, k, v)
        assert torch.isfinite(got.out).all()
        assert ((got.out.double() / v[0, 0, 0].double() - 1).abs() <= 2 * torch.finfo(v.dtype).eps).all()
    q, k, v = inputs(g, 300, 1, 1, 128, "bf16", spread=100.0)
    check(clear_call(q, k, v, ranges=True), q, k, v, [300])
    got = clear_call(q * 1e6, k * 1e6, v, ranges=True)       # scores of 10^16: the largest one's value
    at = (q.cpu().double()[:, 0] * 1e6).to(torch.bfloat16).double() @ (k.cpu().double()[:, 0] * 1e6).to(torch.bfloat16).double().T
    assert torch.isfinite(got.out).all() and torch.isfinite(got.lse).all()
    best = at.masked_fill(torch.ones(300, 300).triu(1).bool(), -math.inf).argmax(1)
    assert torch.equal(got.out[:, 0].cpu(), v[:, 0].cpu()[best])


def test_graph():
    print("graph", flush=True)
    g = torch.Generator().manual_seed(7)
    q, k, v = inputs(g, 300, 2, 4, 128, "bf16")
    starts = starts_of([100, 200])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clear_call(q, k, v, starts, ranges=True)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = clear_call(q, k, v, starts, ranges=True)
    for cut in (100, 1, 299):
        starts[1] = cut
        q.mul_(1.01)
        graph.replay()
        torch.cuda.synchronize()
        check(got, q, k, v, [cut, 300 - cut])
