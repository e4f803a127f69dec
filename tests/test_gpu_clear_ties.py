"""Token scores of rows where few tokens may stand: the alternatives are those and then the first of the rest, by the
bounds of test_gpu_clear_scores.py.  Rows in one piece and in many, the allowed ones in front, at the end, in one
lane's reach or in many; masks of -inf and of a low value; every other value alike."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_clear_scores import TYPES, check  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rest", [-math.inf, -50.0])
@pytest.mark.parametrize("vocab,more", [(300, 0), (3001, 0), (50021, 0), (131072, 0), (50021, 1100)])
def test_few_allowed(vocab, more, rest, kind):
    from holmes_amd import clear

    print("allowed", vocab, more, rest, kind, flush=True)
    g = torch.Generator().manual_seed(vocab)
    rows = 14 + more
    x = torch.full((rows, vocab + 5), rest)
    x[0, 1:9] = 1.0                                         # in front
    x[1, vocab - 6:] = torch.arange(11.0)                   # at the end
    x[2, 150], x[2, 151], x[2, 299] = 3.0, 3.0, 2.0         # two alike
    x[3, 3:140] = torch.randn(137, generator=g)             # as many as the first places
    x[4, ::max(vocab // 25, 1)] = 0.5                       # alike, spread
    x[5, 5:295:3] = torch.randn(97, generator=g)
    x[7, 160] = 9.0
    x[8, 20:260:8] = torch.randn(30, generator=g)           # one lane's element of every piece
    x[9] = 2.0                                              # all alike
    x[10, 2:66] = 1.0                                       # the first places alike, above the rest
    x[11, 100:200] = -60.0                                  # below the rest
    x[12, 2:70] = -60.0                                     # the first places below the rest
    for r in range(13, rows):
        x[r, torch.randint(0, vocab, (int(1 + r % 40),), generator=g)] = torch.randn((), generator=g)
    x = x.to(TYPES[kind])
    for off, top in ((2, 20), (0, 32), (3, 1), (1, 5)):
        part = x[:, off:off + vocab]
        tokens = torch.randint(0, vocab, (rows,), generator=g)
        check(clear.token_logprobs(x.cuda()[:, off:off + vocab], tokens.cuda(), top=top), part, tokens, top)


@pytest.mark.parametrize("vocab", [3001, 131072])
def test_nan_beside_a_mask(vocab):
    from holmes_amd import clear

    print("nan beside a mask", vocab, flush=True)
    x = torch.full((3, vocab), -math.inf)
    x[:, 70], x[1, 2500], x[1, 90] = 1.0, math.nan, math.nan
    got = clear.token_logprobs(x.cuda(), torch.tensor([70, 70, 70]).cuda(), top=6)
    assert got.top_ids[1].tolist() == [90, 2500, 70, 0, 1, 2]
    assert torch.isnan(got.logprobs[1]) and torch.isnan(got.entropy[1])
    check(clear.TokenScores(*(t[[0, 2]] for t in got)), x[[0, 2]], torch.tensor([70, 70]), 6)
