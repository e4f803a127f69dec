"""Attention over whole prompts where every row's softmax is one token's: outputs are that token's values, bit for bit, so that no
other token's, no other head's and no value out of its place can stand in for it.

Keys are vectors of +1 and -1 and a query is one of them times 8, with a scale of 2 log 2: in units of log 2 the score of its own
token is 16 D, and every other seen token's is below that by 256 or more.  Exponentials are then a power of two and zeros, in any type
and against any whole reference, and the output is the token's value in exact arithmetic.  lse and the largest score are 16 D log 2,
a whole number times log 2 (2^-22 of it)."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_prompt import starts_of  # noqa: E402
from .test_gpu_clear_whole_prompt import TYPES, clear_call  # noqa: E402


def check(counts, heads, group, dim, kind, causal, parts, most=None):
    from holmes_amd import _native as nat

    n = sum(counts)
    size = nat.lib().hck_prompt_attend_workspace_bytes(n, len(counts), heads, group, dim, most or n, causal)
    assert (size > 0) == parts
    g = torch.Generator().manual_seed(n + heads + group + dim)
    keys = torch.randint(0, 2, (n, heads, dim), generator=g) * 2 - 1
    values = torch.randn((n, heads, dim), generator=g).to(TYPES[kind])
    at = torch.tensor(sum(([b] * c for b, c in enumerate(counts)), []))
    starts = starts_of(counts)
    first = starts.cpu()[at]
    own = torch.arange(n) - first
    room = own + 1 if causal else torch.tensor(counts)[at]
    # each row's token: any that it sees, its own and the first for some
    pick = (torch.rand((n, heads * group), generator=g) * room[:, None]).long().clamp(max=room[:, None] - 1)
    pick[::5] = own[::5, None] if causal else room[::5, None] - 1
    pick[1::7] = 0
    pick = pick + first[:, None]
    head = torch.arange(heads * group) // group
    queries = 8 * keys[pick, head]
    # far from every other token of its sequence (on integers, for all that a row may see)
    lo = 0
    for c in counts:
        for h in range(heads):
            k = keys[lo:lo + c, h].double()
            near = (k @ k.T - 2 * dim * torch.eye(c)).max() if c else -dim
            assert dim - near >= 16
        lo += c
    got = clear_call(queries.to(TYPES[kind]).cuda(), keys.to(TYPES[kind]).cuda(), values.cuda(), starts, most=most, causal=causal,
                     scale=2.0 * math.log(2.0), ranges=True)
    assert torch.equal(got.out.cpu(), values[pick, head])
    for x in (got.lse, got.high):
        want = 16 * dim * math.log(2.0)
        assert ((x.cpu().double() - want).abs() <= 2.0**-22 * want).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,group", [(2, 3), (1, 4)])
def test_packed(heads, group, causal, kind):
    print("packed", heads, group, causal, kind, flush=True)
    for dim in (64, 128):
        check([1, 0, 2, 63, 64, 65, 127, 129, 33, 200], heads, group, dim, kind, causal, parts=False, most=200)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_in_parts(causal, kind):
    print("parts", causal, kind, flush=True)
    for counts, heads, group, dim in (([1500], 1, 2, 128), ([700, 3, 1300, 513], 2, 1, 128), ([1100, 64, 0, 900], 1, 3, 64)):
        check(counts, heads, group, dim, kind, causal, parts=True, most=max(counts))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
def test_more_sequences_than_lanes_in_parts(causal, kind):
    """Sequences are looked through 64 at a time, here in three rounds, with cut tiles in each and tiles of one part beside them."""
    print("sequences", causal, kind, flush=True)
    counts = [(7 * i) % 60 for i in range(60)] + [1200] + [(11 * i) % 50 for i in range(66)] + [0, 1300, 520, 1] + [5] * 9
    assert len(counts) > 128
    check(counts, 1, 2, 128, kind, causal, parts=True, most=1300)
    check(counts, 1, 1, 128, kind, causal, parts=True)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,heads,group,dim", [([1500], 1, 2, 128), ([700, 3, 1300, 513], 2, 1, 64), ([130, 1, 64, 400], 2, 3, 128)])
def test_even_probabilities(counts, heads, group, dim, causal, kind):
    """Queries of 0, and values of whole numbers: exponentials are one power of two, sums are exact, and the mean of what a row sees is
    off by the reciprocal's and the product's rounding (2^-22 of it) and half a step of the output's type.  A value that is left
    out, or counted twice, is off by its n-th part, which is more."""
    print("even", counts, heads, group, dim, causal, kind, flush=True)
    g = torch.Generator().manual_seed(sum(counts))
    n = sum(counts)
    values = (torch.randint(1, 9, (n, heads, dim), generator=g) * (torch.randint(0, 2, (n, heads, dim), generator=g) * 2 - 1))
    keys = torch.randn((n, heads, dim), generator=g).to(TYPES[kind])
    queries = torch.zeros((n, heads * group, dim), dtype=TYPES[kind])
    got = clear_call(queries.cuda(), keys.cuda(), values.to(TYPES[kind]).cuda(), starts_of(counts), most=max(counts), causal=causal)
    at = 0
    for c in counts:
        v = values[at:at + c].double()
        seen = torch.arange(1, c + 1).double() if causal else torch.full((c,), float(c), dtype=torch.float64)
        want = (v.cumsum(0) if causal else v.sum(0, keepdim=True).expand(c, -1, -1)) / seen[:, None, None]
        want = want.repeat_interleave(group, 1)
        half = torch.finfo(TYPES[kind]).eps / 2
        off = (got.out[at:at + c].cpu().double() - want).abs()
        assert (off <= (half + 2.0**-22) * want.abs()).all()
        lse = got.lse[at:at + c].cpu().double()
        assert ((lse - seen.log()[:, None]).abs() <= 2.0**-22 * (1 + 40 * math.log(2.0))).all()
        at += c
