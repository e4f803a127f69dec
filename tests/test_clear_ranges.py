"""The encrypted softmax's intervals from scores' ranges (torch on the host; no GPU needed)."""

import math

import pytest
import torch

from holmes_amd import clear

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
