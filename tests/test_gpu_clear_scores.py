"""Token scores (holmes_amd.clear.token_logprobs) against float64.

Tolerance of a log probability: the arguments x log2 e - r carry one rounding each (2^-24 of their size),
log2 e and ln 2 as 32-bit numbers change the logits' differences by 2^-24 of them, the exponentials and the
logarithm a step or two; a lane's chain of sums is at most vocabulary / 64 long."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(got, x, tokens, top):
    y = x.detach().cpu().double()
    rows, vocab = y.shape
    logs = torch.where((y == -math.inf).all(1, keepdim=True), y, torch.log_softmax(y, 1))
    p = logs.exp()
    entropy = -torch.where(p == 0, 0.0, p * logs).sum(1)
    span = torch.where(torch.isfinite(y), y, y.masked_fill(~torch.isfinite(y), -math.inf).amax(1, keepdim=True))
    span = (span.amax(1) - span.amin(1)).nan_to_num(0.0, 0.0, 0.0)
    sums = 2.0**-24 * (vocab / 64 + 32)
    ent_tol = 2.0**-22 * (span + 4) * 2 + sums * (1 + entropy.abs())
    if tokens is not None:
        t = tokens.cpu()
        want = torch.where(t >= 0, logs.gather(1, t.clamp(0, vocab - 1)[:, None])[:, 0], 0.0)
        want = torch.where(t >= vocab, math.nan, want)
        near(got.logprobs, want, 2.0**-22 * (want.abs().nan_to_num(0, 0, 0) + span + 4) + sums)
    near(got.entropy, entropy, ent_tol)
    if top:
        ids = torch.sort(y, dim=1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_ids.cpu(), ids)
        want = logs.gather(1, ids)
        near(got.top_logprobs, want, (2.0**-22 * (span + 4) + sums)[:, None] + 2.0**-22 * want.abs().nan_to_num(0, 0, 0))
    else:
        assert got.top_ids is None and got.top_logprobs is None


def near(got, want, tol):
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    assert ((got - want).abs() <= tol)[fine].all(), float(((got - want).abs() - tol)[fine].max())


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (2, 63, 0), (5, 1000, 32), (1, 131072, 8), (70, 50021, 20),
                                            (300, 4097, 5), (1100, 3001, 3), (2, 70001, 1)])
def test_scores(rows, vocab, top, kind):
    from holmes_amd import clear

    print("scores", rows, vocab, top, kind, flush=True)
    g = torch.Generator().manual_seed(rows + vocab)
    x = (3 * torch.randn((rows, vocab), generator=g)).to(TYPES[kind])
    tokens = torch.randint(0, vocab, (rows,), generator=g)
    tokens[::4] = x[::4].float().argmax(1)
    if rows > 2:
        tokens[1], tokens[2] = -100, vocab
    got = clear.token_logprobs(x.cuda(), tokens.cuda(), top=top)
    check(got, x, tokens, top)
    assert clear.token_logprobs(x.cuda(), top=top).logprobs is None


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_ties_masks_and_large_values(kind):
    """All values alike, two values only, sorted both ways (every one enters the list of the best), rows masked
    but for one or as a whole, values of both signs far from 0, zeros of both signs."""
    from holmes_amd import clear

    print("ties", kind, flush=True)
    vocab, top = 9001, 32
    g = torch.Generator().manual_seed(2)
    rows = [torch.full((vocab,), 1.25), (torch.arange(vocab) % 2).float(), torch.arange(vocab) / 64.0,
            -torch.arange(vocab) / 64.0, torch.full((vocab,), -math.inf), torch.full((vocab,), -math.inf),
            1e4 + torch.randn(vocab, generator=g), -3e4 + torch.randn(vocab, generator=g), torch.zeros(vocab),
            torch.randn(vocab, generator=g)]
    rows[4][vocab - 3] = 7.0
    rows[8][::2] = -0.0
    rows[9][torch.rand(vocab, generator=g) < 0.9] = -math.inf
    x = torch.stack(rows).to(TYPES[kind])
    tokens = torch.tensor([5, 0, vocab - 1, 0, vocab - 3, 17, 3, 4, 5, 6])
    check(clear.token_logprobs(x.cuda(), tokens.cuda(), top=top), x, tokens, top)


def test_nan_and_infinity():
    """A NaN makes its row's numbers NaN and stands first among its values; +inf does what the formulas say."""
    from holmes_amd import clear

    print("nan", flush=True)
    x = torch.randn((3, 5000), generator=torch.Generator().manual_seed(3))
    x[0, 4321], x[0, 77] = math.nan, -math.nan
    x[1, 100] = math.inf
    got = clear.token_logprobs(x.cuda(), torch.tensor([3, 3, 3]).cuda(), top=3)
    assert torch.isnan(got.logprobs[0]) and torch.isnan(got.entropy[0]) and torch.isnan(got.top_logprobs[0]).all()
    assert got.top_ids[0].tolist()[:2] == [77, 4321]
    assert got.logprobs[1] == -math.inf and got.top_ids[1, 0] == 100 and torch.isnan(got.entropy[1])
    check(clear.TokenScores(*(t[2:] for t in got)), x[2:], torch.tensor([3]), 3)


def test_strided_unaligned_rows_and_streams():
    from holmes_amd import clear

    print("strided", flush=True)
    g = torch.Generator().manual_seed(4)
    for dtype in TYPES.values():
        wide = torch.randn((6, 4099), generator=g).to(dtype).cuda()
        for cut in range(0, 9):
            x = wide[::2, cut:cut + 4001]
            tokens = torch.tensor([0, 4000, 1717]).cuda()
            check(clear.token_logprobs(x, tokens, top=4), x, tokens, 4)
    row = wide[:1].expand(3, -1)   # the same row three times
    check(clear.token_logprobs(row, tokens, top=4), row, tokens, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = clear.token_logprobs(wide, top=5)
    side.synchronize()
    check(got, wide, None, 5)
    assert clear.token_logprobs(wide[:0], top=5).top_ids.shape == (0, 5)


def test_scores_in_a_graph():
    from holmes_amd import clear

    print("graph", flush=True)
    g = torch.Generator().manual_seed(6)
    x = torch.randn((2, 60000), generator=g).cuda()
    tokens = torch.tensor([1, 2]).cuda()
    clear.token_logprobs(x, tokens, top=6)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        rec = clear.token_logprobs(x, tokens, top=6)
    for i in range(3):
        x.copy_(torch.randn((2, 60000), generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in rec]
        assert all(torch.equal(a, b) for a, b in zip(got, clear.token_logprobs(x, tokens, top=6))), i
        check(clear.TokenScores(*got), x, tokens, 6)
