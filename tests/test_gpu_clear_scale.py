"""Scales at both ends of their range, against float64 with the tolerance of test_gpu_clear_pages."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import build, check  # noqa: E402
from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402


@pytest.mark.parametrize("count,columns", [(1, 2), (70, 900)])
@pytest.mark.parametrize("scale", [2.0**126, 2.0**120, 2.0**-100])
def test_ends(scale, count, columns):
    print("scale", scale, count, flush=True)
    g = torch.Generator().manual_seed(count)
    pool, table, keys, values = build([150], 2, 128, g, spread=2.0**-8)
    q = torch.randint(-8, 9, (count, 8, 128), generator=g).to(torch.bfloat16)
    q = (q * (2.0**4 / scale)).cuda()     # all within bf16's normal numbers
    got = pool.attend(q, widen(table, columns), torch.tensor([150], dtype=torch.int32).cuda(), starts=starts_of([count]),
                      most=count, scale=scale, ranges=True)
    check(got, q, keys, values, [count], scale=scale)


def test_refused():
    print("scales refused", flush=True)
    pool, table, _, _ = build([5], 1, 64, torch.Generator().manual_seed(1))
    q, lengths = torch.zeros((1, 2, 64), dtype=torch.bfloat16).cuda(), torch.tensor([5], dtype=torch.int32).cuda()
    for bad in (2.5e38, 1e-60, 1e60, -1.0, 0.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            pool.attend(q, table, lengths, scale=bad)
