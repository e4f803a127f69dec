"""Attention of many rows over 4-bit pages, against float64 with the tolerance of test_gpu_clear_pages.

Which kernel a call takes goes by the work that the table has room for, so the tables here have room for some
hundred pages (the columns behind a sequence's pages hold numbers that are none): tiles of 128 rows, of 256 where
there are many of them, histories that are split and joined, and sequences too many to be split."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import PAGE, TYPES, build, check  # noqa: E402


def widen(table, columns):
    wide = torch.full((table.shape[0], columns), -7, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    return wide


def starts_of(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32).cuda()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal,ranges", [(True, True), (False, False), (True, False)])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (1, 7, 64), (3, 1, 128)])
def test_many_rows(heads, group, dim, causal, ranges, kind):
    """Counts of 0 and 1, of a whole sequence, of more than the sequence holds; lengths at the units' borders."""
    print("many rows", heads, group, dim, causal, ranges, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 10 + group)
    seqs, counts = [150, 300, 5, 129, 64, 0, 193], [150, 33, 0, 1, 64, 2, 90]
    seqs[4] = 50   # 14 of its queries see nothing
    pool, table, keys, values = build(seqs, heads, dim, g)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    got = pool.attend(q, widen(table, 900), torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts_of(counts), most=150,
                      causal=causal, ranges=ranges)
    check(got, q, keys, values, counts, causal=causal)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_tiles_of_256_rows(kind):
    print("256 rows", kind, flush=True)
    g = torch.Generator().manual_seed(4)
    seqs = [1 + 37 * i % 211 for i in range(54)]
    counts = [1 + 5 * i % 12 for i in range(54)]
    seqs[7], counts[7] = 300, 70     # 280 rows: a tile and a part of one
    pool, table, keys, values = build(seqs, 4, 128, g)
    q = torch.randn((sum(counts), 16, 128), generator=g).to(TYPES[kind]).cuda()
    got = pool.attend(q, widen(table, 300), torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts_of(counts), most=70,
                      ranges=True)
    check(got, q, keys, values, counts)


@pytest.mark.parametrize("kind,heads,group,dim", [("bf16", 2, 4, 128), ("fp16", 1, 5, 64)])
def test_split_histories(kind, heads, group, dim):
    """New tokens behind histories of very different lengths: shares of the long one join."""
    print("split", kind, heads, group, dim, flush=True)
    g = torch.Generator().manual_seed(9)
    seqs, counts = [9000, 70, 2111], [30, 30, 17]
    pool, table, keys, values = build(seqs, heads, dim, g)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    for most in (30, 400):   # 400: tiles that no sequence has
        got = pool.attend(q, widen(table, 2000), torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts_of(counts),
                          most=most, ranges=True)
        check(got, q, keys, values, counts)


def test_uneven_single_tokens_and_more_sequences_than_are_shared_out():
    print("uneven", flush=True)
    g = torch.Generator().manual_seed(12)
    for seqs in ([15000, 3, 64, 2500, 0, 129], [1 + 7 * i % 150 for i in range(700)]):
        pool, table, keys, values = build(seqs, 1, 64, g)
        q = torch.randn((len(seqs), 3, 64), generator=g).to(torch.bfloat16).cuda()
        got = pool.attend(q, widen(table, table.shape[1] + 40), torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True)
        check(got, q, keys, values, [1] * len(seqs))


def test_missing_pages_under_many_rows():
    print("missing pages", flush=True)
    g = torch.Generator().manual_seed(13)
    seqs, counts = [520, 300], [140, 60]
    pool, table, keys, values = build(seqs, 2, 128, g)
    q = torch.randn((200, 4, 128), generator=g).to(torch.bfloat16).cuda()
    wide = widen(table, 900)
    wide[0, 0], wide[0, 2], wide[1, 2] = -1, pool.pages, 2**31 - 1
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    there[0][:128] = there[0][256:384] = there[1][256:] = False
    got = pool.attend(q, wide, torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts_of(counts), most=140, ranges=True)
    check(got, q, keys, values, counts, there=there)


@pytest.mark.parametrize("seqs", [1, 60])   # 60: tiles of 256 rows
@pytest.mark.parametrize("dim", [64, 128])
def test_nan_under_many_rows(dim, seqs):
    """A NaN in the cache is NaN for the rows that see its token, of a value in its run's dims, and for no other."""
    print("nan", dim, seqs, flush=True)
    from holmes_amd import clear

    g = torch.Generator().manual_seed(14)
    n, cut, heads = 150, 20, 6
    at = torch.arange(n + 10)
    slots = torch.tensor([1, 0])[at // PAGE] * PAGE + at % PAGE
    table = widen(torch.tensor([[1, 0]], dtype=torch.int32).cuda().expand(seqs, 2), 900)
    lengths = torch.full((seqs,), n, dtype=torch.int32).cuda()
    q = torch.randn((n, 2 * heads, dim), generator=g).to(torch.bfloat16).cuda().repeat(seqs, 1, 1)
    for side in ("key", "value"):
        x = torch.randn((2, n + 10, heads, dim), generator=g)
        clean = x.clone()
        x[0 if side == "key" else 1, n - cut, :, 40] = math.nan
        x[:, n:] = math.inf                       # behind the end
        got = []
        for y in (x, clean):
            pool = clear.ClearKVPages(2, kv_heads=heads, head_dim=dim)
            pool.append(y[0].cuda(), y[1].cuda(), slots.cuda())
            got.append(pool.attend(q, table, lengths, ranges=True, most=n, starts=starts_of([n] * seqs)))
        a, b = (clear.Attended(*(t.unflatten(0, (seqs, n)) for t in r)) for r in got)
        first = n - cut
        for i in range(4):
            assert torch.equal(a[i][:, :first], b[i][:, :first]), i
        if side == "key":
            assert all(torch.isnan(t[:, first:]).all() for t in a)
        else:
            assert torch.isnan(a.out[:, first:, :, 32:64]).all()
            assert torch.equal(a.out[:, first:, :, :32], b.out[:, first:, :, :32])
            assert torch.equal(a.out[:, first:, :, 64:], b.out[:, first:, :, 64:])
            assert torch.equal(a.lse[:, first:], b.lse[:, first:])


def test_many_rows_in_a_graph():
    """Captured with the join of split histories: every replay gives the eager result on new inputs, bit by bit
    (the second sequence grows into slots that hold an earlier owner's values, and so maybe NaN)."""
    print("graph", flush=True)
    g = torch.Generator().manual_seed(15)
    seqs, counts = [3000, 40], [40, 40]
    pool, table, keys, values = build(seqs, 2, 64, g)
    wide, lengths = widen(table, 1500), torch.tensor(seqs, dtype=torch.int32).cuda()
    starts = starts_of(counts)
    q = torch.randn((80, 4, 64), generator=g).to(torch.bfloat16).cuda()
    pool.attend(q, wide, lengths, starts=starts, most=40, ranges=True)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rec = pool.attend(q, wide, lengths, starts=starts, most=40, ranges=True)
    for i in range(3):
        q.copy_(torch.randn((80, 4, 64), generator=g).to(torch.bfloat16))
        lengths.copy_(torch.tensor([3000 - 700 * i, 40 + 17 * i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in rec]
        want = pool.attend(q, wide, lengths, starts=starts, most=40, ranges=True)
        for a, b in zip(got, want):
            bits = torch.int16 if a.dtype == torch.bfloat16 else torch.int32
            assert torch.equal(a.view(bits), b.view(bits)), i


def test_offsets_beyond_32_bits():
    """The last pages of a pool of 4.6 GB hold, read and attend as those of a small one."""
    from holmes_amd import clear

    print("large pool", flush=True)
    g = torch.Generator().manual_seed(16)
    n, heads = 300, 8
    k, v = (torch.randn((n, heads, 128), generator=g).to(torch.bfloat16).cuda() for _ in range(2))
    q = torch.randn((n, 2 * heads, 128), generator=g).to(torch.bfloat16).cuda()
    lengths, starts = torch.tensor([n], dtype=torch.int32).cuda(), starts_of([n])
    got = []
    for pages in (3, 33000):
        pool = clear.ClearKVPages(pages, kv_heads=heads)
        slots = torch.arange(pages * PAGE - n, pages * PAGE).cuda()
        table = torch.arange(pages - 3, pages, dtype=torch.int32).cuda()[None]
        first = (pages * PAGE - n) - (pages - 3) * PAGE   # the sequence begins inside its first page
        pool.append(k, v, slots)
        zero = torch.zeros((first, heads, 128), dtype=torch.bfloat16, device="cuda")
        pool.append(zero, zero, torch.arange((pages - 3) * PAGE, pages * PAGE - n).cuda())
        whole = lengths + first
        got.append((*pool.read(slots), *pool.attend(q[-1:], table, whole)[:2],
                    *pool.attend(q, widen(table, 900), whole, starts=starts, ranges=True)))
        del pool
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_logits_beyond_32_bits():
    """The last rows of 5 GB of logits score as alone."""
    from holmes_amd import clear

    print("many logits", flush=True)
    rows, vocab = 20000, 131072
    x = torch.zeros((rows, vocab), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(17)
    last = torch.randn((3, vocab), generator=g, device="cuda").to(torch.bfloat16)
    x[-3:] = last
    tokens = torch.arange(rows, device="cuda")
    got = clear.token_logprobs(x, tokens, top=4)
    want = clear.token_logprobs(last, tokens[-3:], top=4)
    assert torch.equal(got.top_ids[-3:], want.top_ids)
    # the few rows are split, so their sums come in another order
    for a, b in ((got.logprobs, want.logprobs), (got.entropy, want.entropy), (got.top_logprobs, want.top_logprobs)):
        assert ((a[-3:] - b).abs() <= 2.0**-24 * (vocab / 64 + 64) + 2.0**-21 * b.abs()).all()
    assert (got.logprobs[:-3] + math.log(vocab)).abs().max() < 1e-4


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (3, 7, 64), (2, 12, 128)])
def test_single_tokens_with_room_beyond_the_caches(heads, group, dim, kind):
    """Tables with room for more than the last cache holds: loads that pass it by."""
    print("room", heads, group, dim, kind, flush=True)
    g = torch.Generator().manual_seed(18)
    seqs = [1, 64, 65, 127, 700, 0, 16, 2100]
    pool, table, keys, values = build(seqs, heads, dim, g)
    q = torch.randn((len(seqs), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    for columns in (100, 2500):
        got = pool.attend(q, widen(table, columns), torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True)
        check(got, q, keys, values, [1] * len(seqs))


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_a_read_beyond_the_caches(out):
    from holmes_amd import clear
    from .test_gpu_clear_pages import held, same

    print("large read", out, flush=True)
    g = torch.Generator().manual_seed(19)
    pool = clear.ClearKVPages(70, kv_heads=8)
    x = torch.randn((2, 8900, 8, 128), generator=g).to(torch.bfloat16)
    slots = torch.randperm(70 * PAGE, generator=g)[:8900].cuda()
    slots[5] = -1
    pool.append(x[0].cuda(), x[1].cuda(), slots)
    k, v = pool.read(slots, out)
    assert (k[5] == 0).all() and (v[5] == 0).all()
    x[:, 5] = 0
    same(k, held(x[0]))
    same(v, held(x[1]))
