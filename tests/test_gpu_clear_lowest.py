"""Token scores where logits are as low or as high as their type goes, as masks of the lowest value are: such a value
counts nothing beside an ordinary one, and alike ones share the row.  Tolerances as in test_gpu_clear_scores.py; a log
probability of a value that far below the others is the value's own, to the products' roundings."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from tests.test_gpu_clear_scores import TYPES, check  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,vocab", [(12, 77), (12, 3001), (12, 70001), (1, 131072)])
def test_rows_of_the_lowest_value(rows, vocab, kind):
    """Nothing but the lowest value, or the highest: every token 1 in vocabulary."""
    from holmes_amd import clear

    print("lowest", rows, vocab, kind, flush=True)
    x = torch.full((rows, vocab), torch.finfo(TYPES[kind]).min, dtype=TYPES[kind])
    x[1::2] = torch.finfo(TYPES[kind]).max
    tokens = torch.arange(rows)
    check(clear.token_logprobs(x.cuda(), tokens.cuda(), top=5), x, tokens, 5)


@pytest.mark.parametrize("low", ["type", -1e38, -2.2e38, -3e4])
@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("vocab,left", [(77, 0.3), (3001, 0.3), (3001, 0.01), (70001, 0.3), (70001, 0.001)])
def test_masks_of_a_low_value(vocab, left, kind, low):
    """The rest of the row is scored as if -inf stood there, and what stands there by its distance."""
    from holmes_amd import clear

    dtype = TYPES[kind]
    least = torch.finfo(dtype).min
    low = torch.tensor(least if low == "type" else max(low, least)).to(dtype)
    print("mask", vocab, left, kind, float(low), flush=True)
    g = torch.Generator().manual_seed(vocab)
    x = (3 * torch.randn((8, vocab), generator=g)).to(dtype)
    mask = torch.rand((8, vocab), generator=g) >= left
    mask[:, 40:43] = False
    x[mask] = low
    tokens = torch.full((8,), 41)
    got = clear.token_logprobs(x.cuda(), tokens.cuda(), top=3)
    check(got, x.masked_fill(mask, -math.inf), tokens, 3)
    masked = mask.int().argmax(1)
    got = clear.token_logprobs(x.cuda(), masked.cuda()).logprobs.cpu().double()
    want = x.double().gather(1, masked[:, None])[:, 0] - x.double().logsumexp(1)
    assert ((got - want).abs() <= 2.0**-21 * want.abs()).all()


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_of_both_ends(kind):
    """Values near the type's ends of different sizes: the largest takes all."""
    from holmes_amd import clear

    print("ends", kind, flush=True)
    x = torch.randn((4, 5000), generator=torch.Generator().manual_seed(9))
    x[0] = -1e38 - 1e38 * torch.rand(5000, generator=torch.Generator().manual_seed(1)) * 2
    x[1] = 3.2e38 - x[0].abs()
    x[2, ::7] = -3.3e38
    x[2, 4000] = 3.3e38
    x[3, 2500:] = -2.5e38
    x[0, 1234], x[1, 1234] = -0.9e38, 3.3e38
    x = x.to(TYPES[kind])
    got = clear.token_logprobs(x.cuda(), torch.tensor([1234, 1234, 4000, 5]).cuda(), top=1)
    assert got.top_ids[:3, 0].tolist() == [1234, 1234, 4000]
    assert got.logprobs[:3].tolist() == [0, 0, 0] and got.entropy[:3].tolist() == [0, 0, 0]
    check(clear.TokenScores(*(t[3:] for t in got)), x[3:].masked_fill(x[3:] < -1e38, -math.inf), torch.tensor([5]), 1)
