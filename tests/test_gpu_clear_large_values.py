"""Attention over 4-bit pages whose values go up to the format's largest: an average of finite values is finite.

The expectation is that of test_gpu_clear_pages (float64 over the held values, its tolerance).  A token of 2^70 or more
changes how its run of 32 dims is summed from there on, so such tokens stand in the first unit, in a late one, alone,
under a probability that is nearly 0, behind the rows that see them, and in every token."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import PAGE, TYPES, build, check, held  # noqa: E402
from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402

MOST = 6 * 2.0**125


def put(pool, table, keys, values, b, t, run, value):
    """Puts `value` (and its negative, in turn) into a run of token t's values, in the pool and in the expectation."""
    heads, dim = keys[b].shape[1:]
    v = values[b][t].clone()
    v[:, 32 * run:32 * run + 32] = value * torch.tensor([1.0, -1.0], dtype=torch.float64).repeat(16)
    slot = torch.tensor([int(table[b, t // PAGE]) * PAGE + t % PAGE]).cuda()
    pool.append(keys[b][t][None].float().cuda(), v[None].float().cuda(), slot)
    values[b][t] = held(v.float())
    assert torch.isfinite(values[b][t]).all()


def run(seqs, counts, heads, group, dim, places, columns=None, seed=41, kind="bf16"):
    print("large values", seqs[:4], counts[:4], heads, group, dim, kind, flush=True)
    g = torch.Generator().manual_seed(seed)
    pool, table, keys, values = build(seqs, heads, dim, g)
    for b, t, r, value in places:
        put(pool, table, keys, values, b, t, r, value)
    q = torch.randn((sum(counts), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    got = pool.attend(q, widen(table, columns or table.shape[1]), torch.tensor(seqs, dtype=torch.int32).cuda(),
                      starts=starts_of(counts), most=max(counts), ranges=True)
    assert torch.isfinite(got.out).all() or kind == "fp16"
    check(got, q, keys, values, counts)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 8, 16])
@pytest.mark.parametrize("value", [2.0**70, 2.0**76, 2.0**112, MOST])
def test_single_tokens(value, group, dim):
    run([1, 300, 700, 257], [1] * 4, 2, group, dim,
        [(0, 0, 0, value), (1, 0, 1, value), (2, 690, 0, -value), (2, 40, 1, value), (3, 256, 1, value)])


@pytest.mark.parametrize("dim", [64, 128])
def test_every_token(dim):
    """The sum of a history's values is beyond the type, their average is not."""
    n = 300
    run([n], [1], 1, 4, dim, [(0, t, r, MOST) for t in range(n) for r in range(dim // 32)])


def test_a_split_history():
    run([20011], [1], 2, 4, 128, [(0, 9000, 2, 2.0**112), (0, 20010, 3, MOST)])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("columns", [None, 900])
def test_prompts(columns, dim):
    """The rows before a large token are as they were."""
    run([150, 300, 64], [150, 33, 64], 2, 4, dim,
        [(0, 70, 0, 2.0**112), (0, 149, 1, MOST), (1, 5, 1, 2.0**80), (1, 290, 1, MOST), (2, 0, 0, 2.0**100)], columns)


@pytest.mark.parametrize("counts,columns", [([30, 30], 2000), ([9, 9], None)])
def test_split_prompts(counts, columns):
    run([5000, 700], counts, 2, 4, 128, [(0, 2500, 1, 2.0**112), (0, 4999, 2, MOST), (1, 64, 0, 2.0**90)], columns)


def test_tiles_of_256_rows():
    seqs, counts = [40 + 37 * i % 211 for i in range(54)], [1 + 5 * i % 12 for i in range(54)]
    seqs[7], counts[7] = 300, 70
    run(seqs, counts, 4, 4, 128, [(i, seqs[i] - 1 - i % 13, i % 4, 2.0**(74 + i % 50)) for i in range(54)], 300)


def test_a_large_value_of_little_probability():
    """2^112 times a probability of e^-80, beside values of 1: both count."""
    from holmes_amd import clear

    print("little probability", flush=True)
    for columns, count in ((1, 1), (900, 40)):
        k, v, q = torch.zeros((3, 1, 128)), torch.ones((3, 1, 128)), torch.zeros((count, 4, 128))
        k[0], k[1], q[..., 0] = 0.0, 0.0, 8.0
        k[2, 0, 0], v[2, 0, 64:] = -10.0, 2.0**112     # e2m1 keeps -8 of units of 2: -80 is asked of 10 as 8
        pool = clear.ClearKVPages(1, kv_heads=1)
        pool.append(k.cuda(), v.cuda(), torch.arange(3).cuda())
        table = widen(torch.zeros((1, 1), dtype=torch.int32).cuda(), columns)
        got = pool.attend(q.to(torch.bfloat16).cuda(), table, torch.tensor([3], dtype=torch.int32).cuda(), causal=False,
                          starts=starts_of([count]), scale=1.0)
        s = held(k)[:, 0] @ q[0, 0].double()
        want = torch.softmax(s, 0) @ held(v)[:, 0]
        assert want[64] > 1.01 and s[2] < -60
        # the exponential's argument of 64 counts to 24 bits of it, and bf16 to half a step
        assert ((got.out.cpu().double() - want).abs() <= (2.0**-9 + 2.0**-15) * want).all()


@pytest.mark.parametrize("value", [2.0**76, 60000.0])
def test_fp16_outputs(value):
    """An average beyond the type is its infinity, one within it a number."""
    from holmes_amd import clear

    print("fp16", value, flush=True)
    k, v = torch.zeros((4, 1, 128)), torch.ones((4, 1, 128))
    v[3, 0, 32:64] = value
    pool = clear.ClearKVPages(1, kv_heads=1)
    pool.append(k.cuda(), v.cuda(), torch.arange(4).cuda())
    got = pool.attend(torch.zeros((1, 4, 128), dtype=torch.float16).cuda(), torch.zeros((1, 1), dtype=torch.int32).cuda(),
                      torch.tensor([4], dtype=torch.int32).cuda()).out.cpu().double()
    want = held(v)[:, 0].mean(0)
    assert math.isinf(float(got[0, 0, 40])) == (float(want[40]) > 65520)
    ok = want < 65520
    assert ((got[0][:, ok] - want[ok]).abs() <= 2.0**-10 * want[ok]).all()


@pytest.mark.parametrize("seqs,counts", [([12000, 300, 9000, 40], [70, 33, 66, 5])])
def test_split_tiles_of_256_rows(seqs, counts):
    """Large tokens in some shares of a history and not in others, on either side of a border inside a page."""
    from .test_gpu_clear_split_256 import DIM, GROUP, HEADS, MOST as BOUND, check as compare, share_of

    print("large values, split 256 rows", flush=True)
    g = torch.Generator().manual_seed(6)
    pool, table, keys, values = build(seqs, HEADS, DIM, g)
    border = 64 * share_of(seqs, counts)
    assert border % PAGE == 64
    for t, r, value in ((border - 1, 0, 2.0**112), (3 * border, 1, MOST), (3 * border + 70, 0, 2.0**90), (0, 3, 2.0**74)):
        for b in (0, 2):
            put(pool, table, keys, values, b, t, r, value)
    put(pool, table, keys, values, 1, 299, 2, MOST)     # the last token: seen by the last query alone
    q = torch.randn((sum(counts), HEADS * GROUP, DIM), generator=g).to(torch.bfloat16).cuda()
    got = pool.attend(q, widen(table, 400), torch.tensor(seqs, dtype=torch.int32).cuda(), starts=starts_of(counts), most=BOUND,
                      ranges=True)
    there = [torch.ones(n, dtype=torch.bool) for n in seqs]
    assert torch.isfinite(got.out).all()
    compare(got, q, keys, values, counts, there, True)
