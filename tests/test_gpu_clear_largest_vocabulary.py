"""Token scores over 2^31 - 1 tokens: the last values' numbers, which a lane's own number on top would take past 31 bits."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("first", [0, 3])   # a row that begins on a 16-byte border, and one that does not
def test_largest_vocabulary(first):
    from holmes_amd import clear

    print("vocabulary of 2^31 - 1", first, flush=True)
    vocab = 2**31 - 1
    x = torch.zeros(vocab + first, dtype=torch.bfloat16, device="cuda")[first:][None]
    marks = {0: 8.0, 12345: 9.0, vocab - 9: 10.0, vocab - 2: 11.0, vocab - 1: 12.0}
    for i, v in marks.items():
        x[0, i] = v
    log = math.log(vocab - len(marks) + sum(math.exp(v) for v in marks.values()))
    got = clear.token_logprobs(x, torch.tensor([vocab - 1]).cuda(), top=6)
    assert got.top_ids[0].tolist() == [vocab - 1, vocab - 2, vocab - 9, 12345, 0, 1]
    want = torch.tensor([12.0, 11.0, 10.0, 9.0, 8.0, 0.0], dtype=torch.float64) - log
    # a lane's sum is of 2^17 powers of 2, exact but for the marks' few; then 256 lanes and 64 parts
    assert ((got.top_logprobs[0].cpu().double() - want).abs() <= 2.0**-18).all()
    assert abs(float(got.logprobs[0]) - float(want[0])) <= 2.0**-18
