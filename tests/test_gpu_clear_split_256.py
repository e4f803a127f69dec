"""Tiles of 256 rows whose histories are split and joined, against float64 with the tolerance of test_gpu_clear_pages.

A workgroup of 256 rows takes a page (two units of 64 tokens) between two barriers; shares of an odd number of units
begin and end inside one."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import PAGE, TYPES, build  # noqa: E402
from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402

HEADS, GROUP, DIM, MOST = 4, 4, 128, 1300


def share_of(seqs, counts):
    """Units of a share: the smallest (to a sixteenth) for which the parts are no more than the 256 workgroups that run
    at once, at least 8."""
    units = [-(-n // 64) for n, c in zip(seqs, counts) for _ in range(-(-c * GROUP // 256))]
    base = max(8, -(-sum(units) * HEADS // 256))
    for f in range(16, 33):
        share = (base * f + 15) // 16
        if f == 32 or sum(-(-u // share) for u in units) <= 256 // HEADS:
            return share


def check(got, q, keys, values, counts, there, causal):
    at, group = 0, q.shape[1] // keys[0].shape[1]
    half = torch.finfo(q.dtype).eps / 2
    parts = 2.0**-17 if q.dtype == torch.float16 else 0.0
    for b, new in enumerate(counts):
        n = keys[b].shape[0]
        see = torch.arange(n)[None, :] <= (n - new + torch.arange(new))[:, None] if causal else torch.ones((new, n), dtype=torch.bool)
        see = (see & there[b]).cuda()
        for h in range(q.shape[1]):
            x = q[at:at + new, h].double()
            k, v = (t[b][:, h // group].cuda() for t in (keys, values))
            s = (x @ k.T / math.sqrt(DIM)).masked_fill(~see, -math.inf)
            size = (x.abs() @ k.abs().T / math.sqrt(DIM)).masked_fill(~see, 0.0).amax(1)
            d = size * (2.0**-24 * (DIM + 8) + parts)
            low, high = s.masked_fill(~see, math.inf).amin(1), s.amax(1)
            e = 2 * d + 2.0**-22 * (2 + high - low) + 2.0**-24 * (n / 16 + 64)
            lse = torch.logsumexp(s, 1)
            rows = slice(at, at + new)
            assert ((got.lse[rows, h] - lse).abs() <= e + 2.0**-22 * lse.abs()).all(), (b, h)
            t = d + 2.0**-22 * torch.maximum(low.abs(), high.abs())
            assert ((got.low[rows, h] - low).abs() <= t).all() and ((got.high[rows, h] - high).abs() <= t).all(), (b, h)
            p = torch.softmax(s, 1)
            want, most = p @ v, p @ v.abs()
            out = got.out[rows, h].double()
            assert torch.equal(torch.isnan(out), torch.isnan(want)), (b, h)
            tiny = 2.0**-24 if q.dtype == torch.float16 else 2.0**-133
            tol = half * want.abs() + (2 * e[:, None] + 2.0**-17) * most + tiny
            ok = ~torch.isnan(want)
            assert ((out - want).abs()[ok] <= tol[ok]).all(), (b, h, float(((out - want).abs() - tol)[ok].max()))
        at += new


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("seqs,counts,odd", [
    ([12000, 300, 9000, 40], [70, 33, 66, 5], True),
    ([5000, 1000, 2700, 129], [70, 128, 90, 129], False),
])
def test_split(seqs, counts, odd, causal, kind):
    print("split, 256 rows", seqs, causal, kind, flush=True)
    share = share_of(seqs, counts)
    assert share % 2 == odd and max(seqs) > 2 * 64 * share
    assert len(seqs) * HEADS * -(-MOST * GROUP // 256) >= 320      # what takes tiles of 256 rows
    g = torch.Generator().manual_seed(len(seqs) + odd)
    pool, table, keys, values = build(seqs, HEADS, DIM, g)
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    wide = widen(table, 400)
    wide[0, 7], there[0][7 * PAGE:8 * PAGE] = -1, False            # a page that is not there
    for t in (64 * share - 1, 64 * share):                         # a value that is NaN on either side of a share's border
        run = t % 4
        v = values[2][t].clone()
        v[1, 32 * run + 5] = math.nan
        slot = torch.tensor([int(table[2, t // PAGE]) * PAGE + t % PAGE]).cuda()
        pool.append(keys[2][t][None].float().cuda(), v[None].float().cuda(), slot)
        values[2][t, 1, 32 * run:32 * run + 32] = math.nan
    q = torch.randn((sum(counts), HEADS * GROUP, DIM), generator=g).to(TYPES[kind]).cuda()
    call = dict(starts=starts_of(counts), most=MOST, causal=causal, ranges=True)
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    got = pool.attend(q, wide, lengths, **call)
    check(got, q, keys, values, counts, there, causal)
    bits = torch.int16
    again = pool.attend(q, wide, lengths, **call)
    assert torch.equal(got.out.view(bits), again.out.view(bits)) and torch.equal(got.lse, again.lse)


def test_more_rows_than_given():
    """``most`` left out bounds every sequence's queries by all rows: the same results."""
    print("without most", flush=True)
    g = torch.Generator().manual_seed(3)
    seqs, counts = [700, 64, 1, 300], [1, 1, 1, 40]
    pool, table, keys, values = build(seqs, HEADS, DIM, g)
    q = torch.randn((sum(counts), HEADS * GROUP, DIM), generator=g).to(torch.bfloat16).cuda()
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    lengths = torch.tensor(seqs, dtype=torch.int32).cuda()
    for columns in (table.shape[1], 900):
        got = pool.attend(q, widen(table, columns), lengths, starts=starts_of(counts), ranges=True)
        check(got, q, keys, values, counts, there, True)
