"""The encrypted softmax's intervals from scores' ranges (torch on the host; no GPU needed)."""

import math

import pytest
import torch

from holmes_amd import clear

from .test_gpu_clear_pages import held

INF, NAN = math.inf, math.nan


def rows(*of):
    return [torch.tensor(x) for x in zip(*of)]


def test_empty_rows_do_not_count():
    r = clear.softmax_ranges(*rows((-2.0, 4.0, 4.5), (INF, -INF, -INF), (-1.0, 6.0, 6.25)))
    assert r.score_shift == 2.0 and r.exp_interval[0] == -r.exp_interval[1]
    assert 2.0 < r.exp_interval[1] < 2.5
    assert r.rsqrt_interval[0] < math.exp(2.5) < math.exp(4.25) < r.rsqrt_interval[1]
    with pytest.raises(ValueError, match="no row"):
        clear.softmax_ranges(*[torch.zeros((0, 4))] * 3)


@pytest.mark.parametrize("bad", [(NAN, NAN, NAN), (1.0, 2.0, NAN), (1.0, INF, INF), (-INF, 2.0, 2.5), (-INF, -INF, -INF)])
def test_a_row_with_a_nan_or_an_infinity_is_refused(bad):
    for at in (0, 2):
        of = [(-2.0, 4.0, 4.5), (-3.0, 1.0, 2.0)]
        of.insert(at, bad)
        with pytest.raises(ValueError, match="NaN or infinite"):
            clear.softmax_ranges(*rows(*of))


@pytest.mark.parametrize("row", [(-1000.0, 1000.0, 1000.0), (-1e6, 5.0, 5.0)])
def test_sums_beyond_float64_are_refused(row):
    with pytest.raises(ValueError, match="beyond float64"):
        clear.softmax_ranges(*rows(row, (-2.0, 4.0, 4.5)))
    low = (-1500.0, -1400.0, -1400.0)
    with pytest.raises(ValueError, match="beyond float64"):
        clear.softmax_ranges(*rows(low, (0.0, 0.0, 1.0)))


def kv(kind, g, tokens, heads, dim):
    """Plain normal keys; channels of different widths about means of their own; one strong channel in 32."""
    x = torch.randn((tokens, heads, dim), generator=g)
    if kind == "channels":
        x = (x + 0.5 * torch.randn((1, heads, dim), generator=g)) * torch.exp(0.5 * torch.randn((1, heads, dim), generator=g))
    if kind == "strong":
        x[..., ::32] *= 10.0
    return x


@pytest.mark.parametrize("kind", ["plain", "channels", "strong"])
def test_intervals_hold_the_unrounded_keys_scores(kind):
    """The ranges are those of keys in 4 bits; the encrypted layer's keys are not rounded, and its scores have to lie
    inside too.  Without the rounding's bound some of these sets leave the intervals."""
    tokens, heads, group, dim = 512, 2, 4, 128
    missed = 0
    for seed in range(16):
        g = torch.Generator().manual_seed(seed)
        k = kv(kind, g, tokens, heads, dim)
        q = 1.5 * torch.randn((tokens, heads * group, dim), generator=g)
        seen = torch.ones((tokens, tokens), dtype=torch.bool).tril()[127:]   # the rows that see a page

        def scores(keys):
            s = q.double().transpose(0, 1) @ keys.double().repeat_interleave(group, 1).permute(1, 2, 0) / math.sqrt(dim)
            s = s[:, 127:]
            return s.masked_fill(~seen, INF).amin(2), s.masked_fill(~seen, -INF).amax(2), s.masked_fill(~seen, -INF).logsumexp(2)

        rounded, true = scores(held(k)), scores(k)
        bound = clear.score_rounding(q[127:], k, held(k))
        assert 0 < bound and max(float((a - b).abs().max()) for a, b in zip(rounded, true)) <= bound
        assert bound <= 1.0001 * float(q.norm(dim=2).max() * (k - held(k)).norm(dim=2).max()) / math.sqrt(dim)   # Cauchy-Schwarz
        for rounding in (0.0, bound):
            r = clear.softmax_ranges(*rounded, rounding=rounding)
            low, high, lse = (t - r.score_shift for t in true)
            inside = (r.exp_interval[0] < float(low.min()) / 2 and float(high.max()) / 2 < r.exp_interval[1]
                      and r.rsqrt_interval[0] < math.exp(float(lse.min())) and math.exp(float(lse.max())) < r.rsqrt_interval[1])
            assert inside or rounding == 0.0, seed
            missed += not inside
    assert missed > 0 or kind != "strong"   # else this shows nothing


def test_rounding_is_checked():
    k = torch.randn((5, 2, 64))
    assert clear.score_rounding(torch.randn((3, 4, 64)), k, k) == 0.0
    assert clear.score_rounding(torch.randn((3, 4, 64)), k[:0], k[:0]) == 0.0
    assert clear.score_rounding(torch.ones((1, 2, 64)), k, k + 0.5, scale=2.0) == pytest.approx(2 * 64 * 0.5, rel=1e-4)
    for q, a, b in ((torch.zeros((3, 4, 64)), k, k[1:]), (torch.zeros((3, 4, 32)), k, k), (torch.zeros((3, 3, 64)), k, k)):
        with pytest.raises(ValueError, match="queries"):
            clear.score_rounding(q, a, b)
    for bad in (-1.0, INF, NAN):
        with pytest.raises(ValueError, match="rounding"):
            clear.softmax_ranges(*rows((-2.0, 4.0, 4.5)), rounding=bad)
