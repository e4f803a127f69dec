"""Weights of rows whose scores are far from 0 (ClearKVPages.weigh), against float64 and the lse that is given.

Scores here are exact in 32 bits, and what is left is the kernel's arithmetic.  At |lse| = 2^27 what rounding took from lse log2 e
is below 8 + 2.6 and from scale log2 e below 12 units of log 2, the last known to 2^-23 of itself and their sums rounded by 2^-24: 2^-18.1,
times log 2 a relative 2^-18.6 of the weight, and two exponentials and their product 2^-22.  The exponent's
difference rounds by 2^-24 of itself, and scale's part is counted where the score is lse: taken together as 2^-18 + 2^-21 |s - lse|."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def pool_of(dim):
    """Three tokens: 1 in dim 0 and 0, 1 and -1 in dim 1."""
    from holmes_amd import clear

    keys = torch.zeros((3, 1, dim))
    keys[:, 0, 0], keys[:, 0, 1] = 1.0, torch.tensor([0.0, 1.0, -1.0])
    pool = clear.ClearKVPages(1, kv_heads=1, head_dim=dim)
    pool.append(keys.cuda(), keys.cuda(), torch.arange(3).cuda())
    assert torch.equal(pool.read(torch.arange(3).cuda(), torch.float32)[0].cpu(), keys)
    return pool, keys[:, 0].double()


def weigh(pool, q, lse, scale, many):
    """What each row of q [rows][dim] gives by itself: a sequence for each, and with `many` 16 rows of nothing beside it."""
    n = q.shape[0]
    table = torch.zeros((n, 1), dtype=torch.int32).cuda()
    lengths = torch.full((n,), 3, dtype=torch.int32).cuda()
    if not many:
        return pool.weigh(q[:, None].cuda(), table, lengths, lse[:, None].cuda(), scale=scale)[:, 0, :3].cpu()
    wide = torch.zeros((n, 17, q.shape[1]), dtype=q.dtype)
    terms = torch.full((n, 17), -math.inf)
    wide[:, 16], terms[:, 16] = q, lse
    starts = torch.arange(0, 17 * n + 1, 17, dtype=torch.int32).cuda()
    return pool.weigh(wide.flatten(0, 1)[:, None].cuda(), table, lengths, terms.flatten()[:, None].cuda(), starts=starts, most=17,
                      causal=False, scale=scale)[:, 0, :3].cpu()


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("scale", [1.0, 0.3, 128**-0.5])
@pytest.mark.parametrize("dim", [64, 128])
def test_scores_far_from_0(dim, scale, many):
    print("far", dim, scale, many, flush=True)
    pool, keys = pool_of(dim)
    rows, lses = [], []
    for exponent in (8, 16, 20, 23, 25, 26):
        for mantissa in (1.0, 1.25, 1.7109375):
            for sign in (1, -1):
                size = sign * mantissa * 2.0**exponent
                step = max(2.0**(math.floor(math.log2(abs(size) / scale)) - 23), 1.0)   # the products' last place, or 1
                for delta in (-3, 0, 1, 7):
                    rows.append((size / scale, step))
                    lses.append(size + delta * step * scale / 2)
    q = torch.zeros((len(rows), dim))
    q[:, :2] = torch.tensor(rows)
    q = q.bfloat16()
    lse = torch.tensor(lses, dtype=torch.float64).float()
    if scale != 1.0:      # near the scores that the rounded queries have
        s = scale * q[:, 0].double()
        lse = (s + (lse.double() - torch.tensor([r[0] * scale for r in rows], dtype=torch.float64))).float()
    got = weigh(pool, q, lse, scale, many).double()
    s = scale * (q.double() @ keys.T)
    away = s - lse.double()[:, None]
    want = torch.exp(away)
    use = (away.abs() < 60)          # no sums of 2^100 and no differences of 2^-100
    assert use.any(1).all()
    tol = want * (2.0**-18 + 2.0**-21 * away.abs())
    off = (got - want).abs()
    assert (off[use] <= tol[use]).all(), float((off / want)[use].max())
    assert (got >= 0).all()


@pytest.mark.parametrize("many", [False, True])
def test_scores_beyond(many):
    """Any finite lse: no weight is negative or NaN, and the tokens keep the order of their scores."""
    print("beyond", many, flush=True)
    pool, keys = pool_of(64)
    sizes = [s * 2.0**e * m for s in (1, -1) for e in (27, 28, 29, 30, 40, 80, 120) for m in (1.0, 1.37, 1.99)] + [3e38, -3e38]
    q = torch.zeros((len(sizes), 64))
    q[:, 0] = torch.tensor(sizes)
    q[:, 1] = q[:, 0].abs() / 128
    q = q.bfloat16()
    lse = q[:, 0].float()
    got = weigh(pool, q, lse, 1.0, many)
    assert (got >= 0).all() and not torch.isnan(got).any()
    assert (got[:, 1] >= got[:, 0]).all() and (got[:, 0] >= got[:, 2]).all()
