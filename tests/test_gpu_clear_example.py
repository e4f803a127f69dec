"""The calibration example's calls together: pages, attention with ranges, the softmax's intervals, scores."""

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_calibration_example():
    path = Path(__file__).resolve().parent.parent / "examples" / "calibrate_decode.py"
    spec = importlib.util.spec_from_file_location("calibrate_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    print("example", flush=True)
    got = module.run(tokens=200, steps=2, vocab=1003)
    r = got["ranges"]
    assert r.exp_interval[0] < got["mapped"].min() and got["mapped"].max() < r.exp_interval[1]
    assert r.rsqrt_interval[0] < got["total"] < r.rsqrt_interval[1]
    # a degree-15 series for exp over |x| <= h errs by about 2 (h / 2)^16 / 16! of 1, twice that once squared
    h = r.exp_interval[1]
    assert got["softmax_error"] < 16 * math.exp(2 * h) * (h / 2) ** 16 / math.factorial(16) + 1e-9
    assert got["prompt"].logprobs.shape == (200,) and torch.isfinite(got["prompt"].logprobs).all()
    for a in got["answers"]:
        assert a.top_ids.shape == (1, 4) and bool((a.top_logprobs[0, 0] >= a.logprobs).all())
        assert bool((a.entropy >= 0).all()) and bool((a.entropy <= math.log(1003) + 1e-5).all())
