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


def test_the_history_that_is_encrypted():
    """Every head's kept tokens, unrounded, in the layout that the encrypted step's pages are packed from."""
    print("history", flush=True)
    import numpy as np

    from holmes_amd.decode import kv_head, pack_key_page, pack_value_page, page_slot

    tokens, keep = 400, 256
    got = example().run(tokens, keep)
    assert all(x.shape == (keep, 1024) and x.dtype == torch.bfloat16 for x in got["history"])
    kept, f = got["kept"].kept[0].cpu().numpy(), np.arange(64)
    for rows, of, pack, sign in ((got["history"][0], got["keys"], pack_key_page, -1), (got["history"][1], got["values"], pack_value_page, 1)):
        of = of.double().cpu().numpy()
        for page in range(2):
            for g in range(2):
                packed = pack(rows[128 * page:128 * page + 128].double().cpu().numpy(), g)
                for pair in range(2):
                    for lane in range(2):
                        h = int(kv_head(g, pair, lane))
                        for t in (0, 1, 77, 127):
                            x = of[kept[h, 128 * page + t], h]
                            assert np.array_equal(packed[page_slot(pair, f, t, lane)], x[f] + sign * 1j * x[f + 64])
