"""Calls with more room than they need and less than there is: a `most` below a sequence's queries in token weights, and eviction
through tables that are much wider than the lengths."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from . import test_gpu_clear_evict as evict  # noqa: E402
from .test_gpu_clear_pages import TYPES, build  # noqa: E402
from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402
from .test_gpu_clear_weigh import check  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group,dim,most", [(2, 4, 128, 3), (1, 5, 64, 3), (2, 4, 128, 40), (1, 3, 64, 100), (1, 1, 128, 0)])
def test_queries_beyond_most_give_nothing(heads, group, dim, most, causal, kind):
    """As rows whose lse is -inf would."""
    print("most", heads, group, dim, most, causal, kind, flush=True)
    g = torch.Generator().manual_seed(heads * 10 + group + most)
    seqs, counts = [150, 300, 5, 700, 64, 0], [150, 33, 5, 2, 1, 3]
    pool, table, keys, _ = build(seqs, heads, dim, g)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    lse = pool.attend(q, table, lengths, starts=starts_of(counts), causal=causal).lse
    got = pool.weigh(q, table, lengths, lse, starts=starts_of(counts), most=most, causal=causal)
    beyond = torch.cat([torch.arange(c) >= most for c in counts]).cuda()
    check(got, q, keys, torch.where(beyond[:, None], -math.inf, lse), counts, group, causal=causal)


@pytest.mark.parametrize("columns", [128, 129, 700])
@pytest.mark.parametrize("keep,recent", [(256, 32), (100, 100), (1, 0), (1000, 10)])
def test_tables_much_wider_than_the_lengths(keep, recent, columns):
    """By one workgroup a row with many keys a thread, and by segments most of which are empty."""
    print("wide", keep, recent, columns, flush=True)
    g = torch.Generator().manual_seed(keep + columns)
    seqs, heads = [384, 0, 1, 500, 129, 1200], 3
    pool, table, _, _ = build(seqs, heads, 128, g, spare=len(seqs) * 8 + 1)
    into = evict.pages_for(pool, table, seqs, keep, g)
    weights = torch.rand((len(seqs), heads, table.shape[1] * 128), generator=g).cuda()
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    before = evict.everything(pool)
    got = pool.evict(widen(table, columns), lengths, weights, into, keep, recent=recent)
    evict.check(pool, before, table.cpu(), seqs, weights, into, keep, recent, got)
