"""Token scores of rows with about as many values as a workgroup has threads, against float64 with the bounds of
test_gpu_clear_scores.py: more alternatives than threads with a piece of the row, each side of the lengths at which
all values are listed, rows at any distance, ties, masks, NaN first."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_clear_scores import TYPES, check  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab,top", [(32, 32), (40, 20), (68, 14), (127, 17), (128, 32), (129, 16), (129, 17), (136, 17), (200, 25),
                                       (255, 32), (256, 32), (256, 1), (257, 32), (271, 32)])
def test_short_rows(vocab, top, kind):
    from holmes_amd import clear

    print("short", vocab, top, kind, flush=True)
    g = torch.Generator().manual_seed(vocab * 33 + top)
    x = torch.randn((40, vocab + 3), generator=g)
    x[0:8] = torch.randint(-2, 3, (8, vocab + 3), generator=g).float()  # ties
    x[8] = 0.5
    x[9] = -math.inf
    x[10:14][torch.rand((4, vocab + 3), generator=g) < 0.7] = -math.inf
    x[14] = torch.arange(vocab + 3) / 16.0
    x[15] = -x[14]
    x[16] = 0.0
    x[16, ::3] = -0.0
    x = x.to(TYPES[kind])
    rows = x.cuda()[:, 1:vocab + 1]  # every border of 16 bytes
    tokens = torch.randint(0, vocab, (40,), generator=g)
    check(clear.token_logprobs(rows, tokens.cuda(), top=top), x[:, 1:vocab + 1], tokens, top)


@pytest.mark.parametrize("vocab", [50, 200, 256])
def test_short_rows_with_nan(vocab):
    """NaN stands before all other values, in the order of the row; its row's numbers are NaN, the others' their own."""
    from holmes_amd import clear

    print("short nan", vocab, flush=True)
    x = torch.randn((3, vocab), generator=torch.Generator().manual_seed(vocab))
    x[1, vocab - 1], x[1, 5] = math.nan, -math.nan
    tokens = torch.tensor([1, 2, 3])
    got = clear.token_logprobs(x.cuda(), tokens.cuda(), top=30)
    assert torch.isnan(got.logprobs[1]) and torch.isnan(got.entropy[1]) and torch.isnan(got.top_logprobs[1]).all()
    rest = [i for i in torch.sort(x[1].nan_to_num(math.inf), descending=True, stable=True).indices.tolist()][:30]
    assert got.top_ids[1].tolist() == rest
    check(clear.TokenScores(*(t[[0, 2]] for t in got)), x[[0, 2]], tokens[[0, 2]], 30)
