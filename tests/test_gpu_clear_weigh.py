"""What attention has given each cached token (ClearKVPages.weigh) against float64.

Tolerance of a term exp(s - lse): the scores' 32-bit sums of D products (2^-24 (D + 8) of the sum of their magnitudes), an
fp16 query's two bf16 parts (2^-17 of it); the exponent's roundings, 2^-23 of |s| and of |lse| each; 2^-22 for the
exponential, the row's factor and the fused sum; of a sum over n terms n / 2 more roundings at the worst, taken as 2^-24 n of it,
and one for the prior."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import TYPES, build  # noqa: E402
from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402


def check(got, q, keys, lse, counts, group, *, causal=True, scale=None, prior=None, there=None):
    dim = q.shape[2]
    scale = scale or 1.0 / math.sqrt(dim)
    part = 2.0**-17 if q.dtype == torch.float16 else 0.0
    q, lse, got = q.cpu().double(), lse.cpu().double(), got.cpu().double()
    at = 0
    for b, new in enumerate(counts):
        n = keys[b].shape[0]
        assert (got[b, :, n:] == 0).all()
        for h in range(keys[b].shape[1]):
            k = keys[b][:, h]
            x = q[at:at + new, h * group:(h + 1) * group].flatten(0, 1)
            y = lse[at:at + new, h * group:(h + 1) * group].flatten()
            s = scale * (x @ k.T)
            d = scale * (x.abs() @ k.abs().T) * (2.0**-24 * (dim + 8) + part)
            see = torch.arange(n) <= (n - new + torch.arange(new))[:, None] if causal else torch.ones(new, n, dtype=torch.bool)
            if there is not None:
                see = see & there[b]
            see = see.repeat_interleave(group, 0) & (y != -math.inf)[:, None]
            w = torch.where(see, torch.exp(s - y[:, None]), 0.0)
            e = torch.expm1(d + 2.0**-23 * (s.abs() + y.abs()[:, None]) + 2.0**-22)
            tol = torch.where(see, w * e, 0.0).sum(0) + 2.0**-24 * max(len(x), 1) * w.sum(0)
            want = w.sum(0)
            if prior is not None:
                p = torch.nn.functional.pad(prior[b, h].cpu().double(), (0, n))[:n]
                want, tol = want + p, tol + 2.0**-24 * (want + p).abs()
            off = (got[b, h, :n] - want).abs()
            assert (off <= tol + 2.0**-140).all(), (b, h, float((off - tol).max()))
        at += new


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim", [(1, 1, 128), (2, 4, 128), (3, 5, 64), (1, 17, 64)])
def test_single_tokens(heads, group, dim, kind):
    print("single", heads, group, dim, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 100 + group)
    seqs = [1, 2, 63, 64, 65, 127, 128, 129, 700, 0, 16, 1000]
    pool, table, keys, _ = build(seqs, heads, dim, g)
    q = torch.randn((len(seqs), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths).lse
    got = pool.weigh(q, table, lengths, lse)
    assert got.shape == (len(seqs), heads, table.shape[1] * 128)
    check(got, q, keys, lse, [1] * len(seqs), group)
    # every row's probabilities add up to 1 (a sum of n terms, each with the module's tolerance at scores below 8 or so)
    total = got.sum(2).cpu()
    want = torch.tensor([float(group) if n else 0.0 for n in seqs])[:, None]
    assert ((total - want).abs() <= group * 2.0**-12).all()
    for places in (0, 64, 70, table.shape[1] * 128 + 5):   # what earlier calls gave, with fewer places or more
        prior = torch.rand((len(seqs), heads, places + 3), generator=g).cuda()[..., :places]
        check(pool.weigh(q, table, lengths, lse, prior=prior), q, keys, lse, [1] * len(seqs), group, prior=prior)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim,causal", [(2, 4, 128, True), (1, 5, 64, True), (2, 1, 128, False), (1, 3, 64, False)])
def test_few_queries_each(heads, group, dim, causal, kind):
    """Up to 16 rows of several queries: some see a part of a unit, some sequences have fewer queries than others, or none."""
    print("few", heads, group, dim, causal, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 7 + group)
    seqs, counts = [3, 64, 130, 1, 65, 257, 0, 700], [3, 2, 3, 1, 0, 3, 2, 3]
    pool, table, keys, _ = build(seqs, heads, dim, g)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths, starts=starts_of(counts), most=3, causal=causal).lse
    got = pool.weigh(q, table, lengths, lse, starts=starts_of(counts), most=3, causal=causal)
    check(got, q, keys, lse, counts, group, causal=causal)


def test_units_in_turn():
    """A table with room for so much that a wave takes several units of 64 tokens, and most of them are behind the end."""
    print("turns", flush=True)
    g = torch.Generator().manual_seed(17)
    seqs, heads, group = [1, 2, 63, 64, 65, 127, 128, 129, 700, 0, 256, 1300], 2, 3
    pool, table, keys, _ = build(seqs, heads, 128, g)
    q = torch.randn((len(seqs), heads * group, 128), generator=g).to(torch.bfloat16).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths).lse
    prior = torch.rand((len(seqs), heads, 1100), generator=g).cuda()
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    there[11][256:384] = False
    table = widen(table, 700)
    table[11, 2] = -1
    got = pool.weigh(q, table, lengths, lse, prior=prior)
    check(got, q, keys, lse, [1] * len(seqs), group, prior=prior, there=there)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim,causal,most", [(2, 4, 128, True, 300), (1, 7, 64, False, 300), (3, 1, 128, True, None),
                                                         (2, 3, 64, True, 333)])
def test_many_rows(heads, group, dim, causal, most, kind):
    """Counts of 0 and 1, of a whole sequence, of more than the sequence holds; lengths at the units' borders."""
    print("many", heads, group, dim, causal, most, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 10 + group)
    seqs, counts = [150, 300, 5, 129, 64, 0, 193, 1025], [150, 33, 0, 1, 64, 2, 90, 300]
    seqs[4] = 50   # 14 of its queries see nothing
    pool, table, keys, _ = build(seqs, heads, dim, g)
    table = widen(table, table.shape[1] + 2)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths, starts=starts_of(counts), causal=causal).lse
    prior = torch.rand((len(seqs), heads, 200), generator=g).cuda()
    got = pool.weigh(q, table, lengths, lse, starts=starts_of(counts), most=most, causal=causal, prior=prior)
    check(got, q, keys, lse, counts, group, causal=causal, prior=prior)
    again = pool.weigh(q, table, lengths, lse, starts=starts_of(counts), most=most, causal=causal, prior=prior)
    assert torch.equal(got, again)


def test_a_whole_prompt():
    print("prompt", flush=True)
    g = torch.Generator().manual_seed(8)
    n, heads, group = 2100, 1, 3
    pool, table, keys, _ = build([n], heads, 128, g)
    q = (2 * torch.randn((n, heads * group, 128), generator=g)).to(torch.bfloat16).cuda()
    lengths = torch.tensor([n], dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths, starts=starts_of([n])).lse
    check(pool.weigh(q, table, lengths, lse, starts=starts_of([n])), q, keys, lse, [n], group)


def test_scale_strides_missing_pages_and_rows_of_nothing():
    print("strides", flush=True)
    g = torch.Generator().manual_seed(11)
    seqs, counts, heads, group, dim = [520, 300], [140, 60], 2, 2, 128
    pool, table, keys, _ = build(seqs, heads, dim, g)
    wide = torch.randn((200, heads * group, 2, 131), generator=g).to(torch.float16).cuda()
    q = wide[:, :, 1, 3:]
    table = widen(table, 9)
    table[0, 0], table[0, 2], table[1, 2] = -1, pool.pages, 2**31 - 1
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    there[0][:128] = there[0][256:384] = there[1][256:] = False
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths, starts=starts_of(counts), scale=0.3).lse
    lse = torch.stack([lse, lse], -1)[..., 0]              # every second value
    lse[7, 1] = -math.inf
    got = pool.weigh(q, table, lengths, lse, starts=starts_of(counts), scale=0.3)
    check(got, q, keys, lse, counts, group, scale=0.3, there=there)
    # a length beyond the table's room, and one below 0 (behind the written 520 tokens the page holds any bytes)
    far = pool.weigh(q[:2], table, torch.tensor([5000, -3], dtype=torch.int32).cuda(), lse[:2])
    assert (far[1] == 0).all() and torch.isfinite(far[0, :, :520]).all()


def test_nan_stays_with_its_token_and_its_rows():
    print("nan", flush=True)
    from holmes_amd import clear

    g = torch.Generator().manual_seed(12)
    n, heads = 200, 2
    x = torch.randn((2, n, heads, 64), generator=g)
    x[0, 77, 1, 3] = math.nan
    pool = clear.ClearKVPages(2, kv_heads=heads, head_dim=64)
    pool.append(x[0].cuda(), x[1].cuda(), torch.arange(n).cuda())
    table, lengths = torch.tensor([[0, 1]], dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    q = torch.randn((n, heads, 64), generator=g).to(torch.bfloat16).cuda()
    lse = torch.full((n, heads), 5.0).cuda()
    got = pool.weigh(q, table, lengths, lse, starts=starts_of([n]))
    nan = torch.zeros(got.shape, dtype=torch.bool)
    nan[0, 1, 77] = True
    assert torch.equal(torch.isnan(got).cpu(), nan)
    lse[100, 0] = math.nan                                 # of the row: the tokens that it sees
    nan[0, 0, :101] = True
    assert torch.equal(torch.isnan(pool.weigh(q, table, lengths, lse, starts=starts_of([n]))).cpu(), nan)


def test_graph():
    print("graph", flush=True)
    g = torch.Generator().manual_seed(13)
    seqs = [300, 40]
    pool, table, keys, _ = build(seqs, 2, 128, g)
    q = torch.randn((2, 8, 128), generator=g).to(torch.bfloat16).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths).lse
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.weigh(q, table, lengths, lse)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = pool.weigh(q, table, lengths, lse)
    for n in (300, 299, 5):
        lengths[0] = n
        lse.copy_(pool.attend(q, table, lengths).lse)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, pool.weigh(q, table, lengths, lse))
        check(got, q, [keys[0][:n], keys[1]], lse, [1, 1], 4)
