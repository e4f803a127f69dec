"""Attention over 4-bit pages where scores are far beyond the exponents of 2: the token of the largest takes all.

Keys and queries are multiples of one row of signs, so that scores are exact but for their scaling; the next largest
is a third below or more, which leaves it a probability of 0.  Outputs are then the token's held values, rounded once
(the probability is a power of 2 or, by the exponential, 2^-22 off one; its two parts 2^-17), and the logarithm of the
sum is the largest score to the roundings of scale, product and conversion (2^-24 each, 2^-21 in all)."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_clear_pages import PAGE, held  # noqa: E402
from tests.test_gpu_clear_prompt import widen  # noqa: E402


@pytest.mark.parametrize("kind,size", [("fp16", 2.0**15), ("bf16", 2.0**15), ("bf16", 2.0**40), ("bf16", 2.0**4)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("count,columns", [(1, 20), (3, 20), (40, 900), (300, 900)])
def test_the_largest_score_takes_all(count, columns, dim, kind, size):
    from holmes_amd import clear

    print("far", count, columns, dim, kind, size, flush=True)
    dtype = {"fp16": torch.float16, "bf16": torch.bfloat16}[kind]
    g = torch.Generator().manual_seed(dim + count)
    n, heads, group = 1500, 2, 4
    sign = torch.randint(0, 2, (heads, dim), generator=g).float() * 2 - 1
    grow = torch.tensor([2.0, 3.0, 4.0])[torch.randint(0, 3, (n, heads), generator=g)]
    most, least = torch.tensor([700, 1100]), torch.tensor([901, 37])
    grow[most, torch.arange(heads)], grow[least, torch.arange(heads)] = 6.0, 1.0
    k = 2.0**13 * grow[:, :, None] * sign
    v = torch.randn((n, heads, dim), generator=g)
    pages = -(-n // PAGE)
    pool = clear.ClearKVPages(pages, kv_heads=heads, head_dim=dim)
    pool.append(k.cuda(), v.cuda(), torch.arange(n).cuda())
    table = torch.arange(pages, dtype=torch.int32)[None].cuda()
    way = torch.tensor([1.0, -1.0, 0.5, -0.5])[torch.arange(count * heads * group).reshape(count, heads, group) % 4]
    q = (way[..., None] * size * sign[:, None]).reshape(count, heads * group, dim).to(dtype)
    got = pool.attend(q.cuda(), widen(table, columns), torch.tensor([n], dtype=torch.int32).cuda(),
                      starts=torch.tensor([0, count], dtype=torch.int32).cuda(), most=count, causal=False, ranges=True)
    win = torch.where(way > 0, most[None, :, None], least[None, :, None])
    lose = torch.where(way < 0, most[None, :, None], least[None, :, None])
    at = torch.arange(heads)[None, :, None].expand(count, heads, group)
    want = held(v)[win, at].reshape(count, heads * group, dim)
    out = got.out.cpu().double()
    assert ((out - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0**-15) * want.abs() + torch.finfo(dtype).tiny).all()
    unit = way.double() * size * 2.0**13 * dim / math.sqrt(dim)
    top, low = unit * grow[win, at].double(), unit * grow[lose, at].double()
    if size > 2.0**10:   # else the others' probabilities are 0 all the same, but scores are counted to 24 bits of them
        for name, want in (("lse", top), ("high", top), ("low", low)):
            have = getattr(got, name).cpu().double().reshape(want.shape)
            assert ((have - want).abs() <= 2.0**-21 * want.abs()).all(), name
