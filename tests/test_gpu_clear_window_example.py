"""The example around a prompt and its window with less than a page of tokens, and with fewer kept than its last ones."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_window import example  # noqa: E402


@pytest.mark.parametrize("tokens,keep", [(100, 32), (1, 1), (127, 300), (200, 1), (128, 0)])
def test_small_prompts_and_windows(tokens, keep):
    print("example", tokens, keep, flush=True)
    got = example().run(tokens, keep)
    kept = min(tokens, keep)
    assert got["kept"].lengths.tolist() == [kept] and got["kept"].kept.shape == (1, 8, keep)
    last = list(range(tokens - kept, tokens)) if kept <= 64 else None
    for h in range(8):
        places = got["kept"].kept[0, h, :kept].tolist()
        assert places == (last if last is not None else sorted(set(places))) and (got["kept"].kept[0, h, kept:] == -1).all()
    # the last row sees the whole prompt, and the intervals hold it
    r, p = got["ranges"], got["prompt"]
    assert r.exp_interval[0] <= (float(p.low[-1].min()) - r.score_shift) / 2 <= (float(p.high[-1].max()) - r.score_shift) / 2 <= r.exp_interval[1]
    assert math.log(r.rsqrt_interval[0]) <= float(p.lse[-1].min()) - r.score_shift <= float(p.lse[-1].max()) - r.score_shift <= math.log(r.rsqrt_interval[1])
