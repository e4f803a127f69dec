"""A prompt's way to the window that is kept, all operators in a row as they are used, against float64; streams; and what the
calls refuse of tensors on the GPU."""

import importlib.util
import math
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_evict import chosen  # noqa: E402
from .test_gpu_clear_pages import held  # noqa: E402

ROOT = Path(__file__).resolve().parent.parent


def example():
    spec = importlib.util.spec_from_file_location("keep_window", ROOT / "examples" / "keep_window.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("tokens,keep,recent", [(500, 256, 64), (130, 256, 0), (300, 100, 100)])
def test_from_a_prompt_to_its_window(tokens, keep, recent):
    """Tolerances: of attention over the pages and of weights as in their own tests' docstrings, at scores below 8 and 500
    tokens (a term's relative error e below 2^-15, and two bf16 parts of a probability, 2^-17; an output's rounding is off by
    half a step, 2^-8 of it)."""
    print("window", tokens, keep, recent, flush=True)
    got = example().run(tokens, keep, recent)
    heads, group, dim, kept = 8, 4, 128, min(keep, tokens)
    q, k, v = (got[x].cpu().double() for x in ("queries", "keys", "values"))
    k4, v4 = held(got["keys"][:tokens]), held(got["values"][:tokens])
    # the ranges hold every score of rows that see a page, against keys as they came
    later = torch.ones(tokens, tokens, dtype=torch.bool).triu(1)
    lo, hi = math.inf, -math.inf
    for h in range(heads * group):
        s = (q[127:tokens, h] @ k[:tokens, h // group].T / math.sqrt(dim)).masked_fill(later[127:], math.nan)
        lo, hi = min(lo, float(s[~s.isnan()].min())), max(hi, float(s[~s.isnan()].max()))
    r = got["ranges"]
    assert r.exp_interval[0] <= (lo - r.score_shift) / 2 and (hi - r.score_shift) / 2 <= r.exp_interval[1]
    # the weights, with the lse that the attention gave
    e = 2.0**-15
    for h in range(heads):
        want = torch.zeros(tokens, dtype=torch.float64)
        for g in range(group):
            s = (q[:tokens, h * group + g] @ k4[:, h].T / math.sqrt(dim)).masked_fill(later, -math.inf)
            assert ((torch.logsumexp(s, 1) - got["cached"].lse[:, h * group + g].cpu()).abs() <= e).all()
            want += torch.softmax(s, 1).sum(0)
        w = got["weights"][0, h].cpu().double()
        assert ((w[:tokens] - want).abs() <= 2 * e * want).all() and (w[tokens:] == 0).all()
        # what was kept goes by the weights as they are
        stay = chosen(w.tolist(), tokens, keep, recent)
        assert got["kept"].kept[0, h].tolist() == stay + [-1] * (keep - kept)
        assert torch.equal(got["kept"].weights[0, h, :kept].cpu().double(), w[stay])
        assert torch.equal(got["held"][0][:, h].cpu().double(), k4[stay, h])
        assert torch.equal(got["held"][1][:, h].cpu().double(), v4[stay, h])
        # the next token over them, and what it adds
        for g in range(group):
            x = q[tokens, h * group + g]
            s = k4[stay, h] @ x / math.sqrt(dim)
            p = torch.softmax(s, 0)
            out, part = p @ v4[stay, h], got["part"].out[0, h * group + g].cpu().double()
            assert ((out - part).abs() <= torch.finfo(torch.bfloat16).eps / 2 * out.abs() + (2 * e + 2.0**-17) * (p @ v4[stay, h].abs()) + 2.0**-133).all()
            want_part = p if g == 0 else want_part + p
        after = got["after"][0, h].cpu().double()
        assert ((after[:kept] - want_part - w[stay]).abs() <= 2 * e * want_part + 2.0**-23 * w[stay]).all() and (after[kept:] == 0).all()
    assert int(got["kept"].lengths[0]) == kept


def test_two_streams_at_once():
    """Calls with workspaces on two streams do not share them."""
    from holmes_amd import clear

    print("streams", flush=True)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = [torch.randn((3000, n, 64), generator=g, device="cuda").bfloat16() for n in (2, 1, 1)]
    y = [torch.randn((2500, n, 64), generator=g, device="cuda").bfloat16() for n in (3, 1, 1)]
    want = clear.prompt_attention(*x), clear.prompt_attention(*y)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, t in zip(streams, (x, y)):
            with torch.cuda.stream(s):
                got.append(clear.prompt_attention(*t))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert torch.equal(r.out, want[i % 2].out) and torch.equal(r.lse, want[i % 2].lse)


def test_two_graphs_with_workspaces():
    """Two captured calls with workspaces, replayed in turn and between eager calls, keep their own results."""
    from holmes_amd import clear

    print("graphs", flush=True)
    g = torch.Generator(device="cuda").manual_seed(4)
    x = [torch.randn((2500, n, 64), generator=g, device="cuda").bfloat16() for n in (2, 1, 1)]
    n, heads = 17000, 1                                   # rows that are chosen from in segments
    pool = clear.ClearKVPages(-(-n // 128) + 8, kv_heads=heads, head_dim=64)
    k = torch.randn((n, heads, 64), generator=g, device="cuda")
    pool.append(k, k, torch.arange(n, device="cuda"))
    table = torch.arange(-(-n // 128), dtype=torch.int32, device="cuda")[None]
    into = torch.arange(table.shape[1], table.shape[1] + 8, dtype=torch.int32, device="cuda")[None]
    lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn((300, 2, 64), generator=g, device="cuda").bfloat16()
    starts = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    lse = torch.full((300, 2), 9.0, device="cuda")

    def chain():
        w = pool.weigh(q, table, lengths, lse, starts=starts)
        return (w, *pool.evict(table, lengths, w, into, 1000, recent=50))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(), clear.prompt_attention(*x)
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        with torch.cuda.graph(graphs[0], stream=side):
            a = chain()
        with torch.cuda.graph(graphs[1], stream=side):
            b = clear.prompt_attention(*x)
    for step in range(3):
        q.mul_(1.1), x[0].mul_(0.9), lengths.fill_(n - 3000 * step)
        graphs[0].replay(), graphs[1].replay()
        want = chain(), clear.prompt_attention(*x)
        torch.cuda.synchronize()
        for t, u in zip(a, want[0]):
            assert torch.equal(t, u)
        assert torch.equal(b.out, want[1].out) and torch.equal(b.lse, want[1].lse)


def test_largest_strides_and_offsets():
    """A pool and prompts whose bytes pass 2^32."""
    from holmes_amd import clear

    print("offsets", flush=True)
    g = torch.Generator(device="cuda").manual_seed(5)
    pages = 2**32 // (128 * 68) // 4 + 40                  # of 4 heads of 64 dims
    pool = clear.ClearKVPages(pages, kv_heads=4, head_dim=64)
    assert pool.nbytes > 2**32
    keys = torch.randn((200, 4, 64), generator=g, device="cuda")
    small = clear.ClearKVPages(8, kv_heads=4, head_dim=64)
    far = torch.tensor([[pages - 1, pages - 30]], dtype=torch.int32, device="cuda")
    near = torch.tensor([[6, 1]], dtype=torch.int32, device="cuda")
    place = torch.arange(200, device="cuda")
    lengths = torch.tensor([200], dtype=torch.int32, device="cuda")
    q = torch.randn((200, 8, 64), generator=g, device="cuda").bfloat16()
    starts = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    got = []
    for p, table, to in ((pool, far, pages - 5), (small, near, 4)):
        p.append(keys, keys, table[0].long()[place // 128] * 128 + place % 128)
        lse = p.attend(q, table, lengths, starts=starts).lse
        w = p.weigh(q, table, lengths, lse, starts=starts)
        single = p.weigh(q[-1:], table, lengths, lse[-1:])
        into = torch.tensor([[to]], dtype=torch.int32, device="cuda")
        got.append((w, single, *p.evict(table, lengths, w, into, 70, recent=9), *p.read(to * 128 + place[:70], torch.float32)))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    del pool
    # tokens 2^16 values apart: 40000 of them are 5 GB
    wide = torch.zeros((40000, 1 << 16), dtype=torch.bfloat16, device="cuda")
    x = [wide[:, i:i + 64].unsqueeze(1) for i in (0, 64, 128)]
    for t in x:
        t.copy_(torch.randn(t.shape, generator=g, device="cuda"))
    starts = torch.tensor([0, 39900, 40000], dtype=torch.int32, device="cuda")
    a = clear.prompt_attention(*x, starts, ranges=True)
    b = clear.prompt_attention(*(t.contiguous() for t in x), starts, ranges=True)
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    at = torch.arange(40000, device="cuda")
    plan = clear.RotaryPositions(64)
    assert torch.equal(plan.rotate(at, x[0]), plan.rotate(at, x[0].contiguous()))


def test_refusals():
    from holmes_amd import clear

    print("refusals", flush=True)
    pool = clear.ClearKVPages(4, kv_heads=2, head_dim=64)
    table = torch.zeros((3, 2), dtype=torch.int32).cuda()
    lengths, lse = torch.ones(3, dtype=torch.int32).cuda(), torch.zeros(3, 4).cuda()
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16).cuda()
    weights, into = torch.zeros(3, 2, 256).cuda(), torch.zeros((3, 2), dtype=torch.int32).cuda()

    def refused(match, call, error=(ValueError, TypeError)):
        with pytest.raises(error, match=match):
            call()
    for bad in (lse[:2], lse.half(), lse[:, :3], lse.flatten(), lse.cpu()):
        refused("lse", lambda: pool.weigh(q, table, lengths, bad))
    for bad in (weights[:2], weights[:, :1], weights.double(), weights[0], weights.cpu(), weights.transpose(1, 2)):
        refused("prior", lambda: pool.weigh(q, table, lengths, lse, prior=bad))
        refused("weights", lambda: pool.evict(table, lengths, bad, into, 5))
    for bad in (table[:2], table.long(), table[0], table.cpu()):
        refused("table", lambda: pool.weigh(q, bad, lengths, lse))
        refused("table", lambda: pool.evict(bad, lengths, weights, into, 5))
    for bad in (into[:2], into.long(), into[0], into.cpu()):
        refused("into", lambda: pool.evict(table, lengths, weights, bad, 5))
    refused("starts", lambda: pool.weigh(q[:2], table, lengths, lse[:2]))
    refused("starts", lambda: pool.weigh(q, table, lengths, lse, starts=lengths))
    refused("most", lambda: pool.weigh(q, table, lengths, lse, most=-1))
    refused("scale", lambda: pool.weigh(q, table, lengths, lse, scale=0.0))
    refused("multiple", lambda: pool.weigh(q[:, :3], table, lengths, lse[:, :3]))
    for keep, recent, match in ((257, 0, "keep"), (-1, 0, "keep"), (5, 6, "recent"), (5, -1, "recent")):
        refused(match, lambda: pool.evict(table, lengths, weights, into, keep, recent=recent))
    grad = [torch.zeros((3, n, 64), dtype=torch.bfloat16, device="cuda", requires_grad=True) for n in (4, 2, 2)]
    plan = clear.RotaryPositions(64)
    at = torch.arange(3).cuda()
    plain = [t.detach() for t in grad]
    for i in range(3):
        mixed = [grad[j] if i == j else plain[j] for j in range(3)]
        refused("gradient", lambda: clear.prompt_attention(*mixed))
    refused("gradient", lambda: plan.rotate(at, grad[0]))
    refused("gradient", lambda: plan.rotate(at, plain[0], grad[1]))
    refused("gradient", lambda: pool.weigh(grad[0], table, lengths, lse))
    refused("gradient", lambda: pool.evict(table, lengths, weights.clone().requires_grad_(), into, 5))
    with torch.no_grad():
        clear.prompt_attention(*grad), plan.rotate(at, grad[0])
    buf, pool.buf = pool.buf, pool.buf[:3]
    refused("buf", lambda: pool.weigh(q, table, lengths, lse))
    refused("buf", lambda: pool.evict(table, lengths, weights, into, 5))
    pool.buf = buf
    # nothing to do
    none = torch.zeros((0, 2), dtype=torch.int32).cuda()
    assert pool.weigh(q[:0], none, lengths[:0], lse[:0]).shape == (0, 2, 256)
    got = pool.evict(none, lengths[:0], weights[:0], none, 5)
    assert got.kept.shape == (0, 2, 5) and got.lengths.shape == (0,)
    got = pool.evict(table, lengths, weights, into, 0)
    assert got.kept.shape == (3, 2, 0) and got.lengths.tolist() == [0, 0, 0]
    assert pool.weigh(q, table[:, :0], lengths, lse).shape == (3, 2, 0)
    assert clear.prompt_attention(*(t[:0] for t in plain)).out.shape == (0, 4, 64)
