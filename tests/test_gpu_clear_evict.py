"""Eviction of cached tokens (ClearKVPages.evict): whole numbers and bytes, so all of it is exact."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import PAGE, build  # noqa: E402


def chosen(weights, n, keep, recent, there=None):
    """The places that stay of a row of n, in order."""
    there = range(n) if there is None else [j for j in range(n) if there[j]]
    last = [j for j in there if j >= n - recent]

    def order(j):
        w = float(weights[j]) if j < len(weights) else 0.0
        return (0, 0.0, j) if math.isnan(w) else (1, -w, j)
    rest = sorted((j for j in there if j < n - recent), key=order)
    return sorted(rest[:max(0, keep - len(last))] + last)


def check(pool, before, table, seqs, weights, into, keep, recent, got, there=None):
    """The kept places, their weights, and what the pool holds afterwards against what it held `before`."""
    heads = pool.kv_heads
    w = weights.cpu()
    k0, v0 = (x.cpu() for x in before)
    k1, v1 = (x.cpu() for x in pool.read(torch.arange(pool.pages * PAGE).cuda(), torch.float32))
    want_k, want_v = k0.clone(), v0.clone()
    t, to = table.cpu(), into.cpu()
    for b, n in enumerate(seqs):
        for h in range(heads):
            stay = chosen(w[b, h].tolist(), n, keep, recent, None if there is None else there[b])
            assert got.lengths[b].item() == len(stay)
            kept = got.kept[b, h].tolist()
            assert kept == stay + [-1] * (keep - len(stay)), (b, h)
            values = [float(w[b, h, j]) if j < w.shape[2] else 0.0 for j in stay]
            for x, y in zip(got.weights[b, h].tolist(), values + [0.0] * (keep - len(stay))):
                assert x == y or (math.isnan(x) and math.isnan(y))
            for i, j in enumerate(stay):
                page = int(to[b, i // PAGE])
                if 0 <= page < pool.pages:
                    src = int(t[b, j // PAGE]) * PAGE + j % PAGE
                    want_k[page * PAGE + i % PAGE, h], want_v[page * PAGE + i % PAGE, h] = k0[src, h], v0[src, h]
    for x, y in ((k1, want_k), (v1, want_v)):
        assert torch.equal(torch.nan_to_num(x, nan=1e30), torch.nan_to_num(y, nan=1e30))


def pages_for(pool, table, seqs, keep, g):
    """Pages of the pool that no table has, in any order."""
    used = {int(table[b, i]) for b, n in enumerate(seqs) for i in range(-(-n // PAGE))}
    free = torch.tensor([p for p in range(pool.pages) if p not in used])
    need = -(-keep // PAGE)
    free = free[torch.randperm(len(free), generator=g)][:need * len(seqs)]
    return free.view(len(seqs), need).int().cuda()


def everything(pool):
    return pool.read(torch.arange(pool.pages * PAGE).cuda(), torch.float32)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (37, 5), (128, 128), (129, 30), (256, 0), (400, 100), (0, 0)])
def test_lengths_and_numbers(keep, recent, dim):
    print("evict", keep, recent, dim, flush=True)
    g = torch.Generator().manual_seed(keep + dim)
    seqs = [1, 0, 2, 37, 63, 64, 128, 129, 500, 1300]
    heads = 3
    pool, table, _, _ = build(seqs, heads, dim, g, spare=len(seqs) * 4 + 3)
    weights = torch.exp(2 * torch.randn((len(seqs), heads, table.shape[1] * PAGE), generator=g)).cuda()
    into = pages_for(pool, table, seqs, keep, g)
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    before = everything(pool)
    got = pool.evict(table, lengths, weights, into, keep, recent=recent)
    check(pool, before, table.cpu(), seqs, weights, into, keep, recent, got)


@pytest.mark.parametrize("what", ["ties", "zeros", "odd", "negative", "narrow", "close"])
def test_weights_of_all_kinds(what):
    print("weights", what, flush=True)
    g = torch.Generator().manual_seed(5)
    seqs, heads, keep, recent = [700, 1500], 2, 300, 40
    pool, table, _, _ = build(seqs, heads, 64, g, spare=8)
    w = torch.rand((2, heads, 1536), generator=g)
    if what == "ties":
        w = torch.randint(0, 4, w.shape, generator=g).float()
    elif what == "zeros":
        w = torch.where(torch.rand(w.shape, generator=g) < 0.99, torch.where(w < 0.5, 0.0, -0.0), w)
    elif what == "odd":
        for value in (math.nan, -math.nan, math.inf, -math.inf):
            w[torch.rand(w.shape, generator=g) < 0.02] = value
    elif what == "negative":
        w = 1e-38 * (w - 0.7)     # subnormal ones among them
    elif what == "narrow":
        w = w[..., :333]
    elif what == "close":
        w = 1.0 + torch.randint(0, 50, w.shape, generator=g) * 2.0**-23   # only the last digit differs
    wide = torch.full((2, heads, w.shape[2] + 7), math.inf)
    wide[..., 3:3 + w.shape[2]] = w
    w = wide.cuda()[..., 3:3 + w.shape[2]]
    into = pages_for(pool, table, seqs, keep, g)
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    before = everything(pool)
    check(pool, before, table.cpu(), seqs, w, into, keep, recent, pool.evict(table, lengths, w, into, keep, recent=recent))


@pytest.mark.parametrize("keep,recent", [(5000, 100), (5000, 5000), (20000, 17000), (1, 0), (16500, 0)])
def test_long_rows(keep, recent):
    """Rows of one segment and of several, whole ones and ones with pages outside the pool."""
    print("long", keep, recent, flush=True)
    g = torch.Generator().manual_seed(6)
    seqs, heads = [40000, 9000, 0, 16384, 32769], 1
    pool, table, _, _ = build(seqs, heads, 64, g, spare=5 * -(-keep // PAGE))
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    into = pages_for(pool, table, seqs, keep, g)
    shape = (5, heads, table.shape[1] * PAGE)
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    for i, w in enumerate((torch.rand(shape, generator=g), torch.randint(0, 3, shape, generator=g).float(), torch.zeros(shape))):
        if i == 1:
            table[0, 5], table[0, 250], table[4, 255:] = -1, pool.pages, 2**31 - 1
            there[0][5 * PAGE:6 * PAGE] = there[0][250 * PAGE:251 * PAGE] = there[4][255 * PAGE:] = False
        before = everything(pool)
        got = pool.evict(table, lengths, w.cuda(), into, keep, recent=recent)
        check(pool, before, table.cpu(), seqs, w, into, keep, recent, got, there=there)


def test_pages_outside_the_pool_and_nan_tokens():
    print("missing", flush=True)
    g = torch.Generator().manual_seed(7)
    seqs, heads, keep, recent = [600, 300, 200], 2, 150, 90
    pool, table, _, _ = build(seqs, heads, 128, g, spare=9)
    bad = torch.randn((2, heads, 128), generator=g)
    bad[0, :, 5] = math.nan
    pool.append(bad.cuda(), bad.cuda(), table[0, 1].long() * PAGE + torch.tensor([3, 9]).cuda())
    into = pages_for(pool, table, seqs, keep, g)
    table = table.clone()
    table[0, 0], table[0, 3], table[1, 2], table[2, :] = -1, pool.pages, 2**31 - 1, -5
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    there[0][:128] = there[0][384:512] = there[1][256:] = there[2][:] = False
    w = torch.rand((3, heads, 640), generator=g).cuda()
    into[1, 1] = -1                                 # the second page of this one takes nothing
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    before = everything(pool)
    got = pool.evict(table, lengths, w, into, keep, recent=recent)
    check(pool, before, table.cpu(), seqs, w, into, keep, recent, got, there=there)


def test_graph_and_shared_pages():
    """A page that two sequences share goes to each of their targets; a captured call follows lengths and weights."""
    print("graph", flush=True)
    g = torch.Generator().manual_seed(8)
    pool, table, _, _ = build([256], 2, 64, g, spare=6)
    table = table.expand(2, 2)
    seqs, keep, recent = [256, 200], 100, 10
    into = pages_for(pool, table.cpu(), seqs, keep, g)
    w = torch.rand((2, 2, 256), generator=g).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        pool.evict(table, lengths, w, into, keep, recent=recent)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = pool.evict(table, lengths, w, into, keep, recent=recent)
    for n in (256, 130, 60):
        seqs[0] = n
        lengths[0] = n
        w.copy_(torch.rand((2, 2, 256), generator=g))
        before = everything(pool)
        graph.replay()
        torch.cuda.synchronize()
        check(pool, before, table.cpu(), seqs, w, into, keep, recent, got)
