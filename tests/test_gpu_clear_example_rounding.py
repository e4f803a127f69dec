"""The calibration example's intervals hold the scores of the keys as they came, not only of those in 4 bits."""

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("tokens", [200, 700])
def test_unrounded_keys(tokens):
    path = Path(__file__).resolve().parent.parent / "examples" / "calibrate_decode.py"
    spec = importlib.util.spec_from_file_location("calibrate_decode", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    print("example", tokens, flush=True)
    got = module.run(tokens=tokens, steps=1, vocab=503, seed=3)
    r, q, k = got["ranges"], got["queries"].double().cpu(), got["keys"].double().cpu()
    assert got["rounding"] > 0
    for row in range(127, tokens, 40):
        s = (k[:row + 1].repeat_interleave(4, 1) * q[row]).sum(2) / math.sqrt(128) - r.score_shift
        assert r.exp_interval[0] < float(s.min()) / 2 and float(s.max()) / 2 < r.exp_interval[1]
        total = torch.exp(s).sum(0)
        assert r.rsqrt_interval[0] < float(total.min()) and float(total.max()) < r.rsqrt_interval[1]
