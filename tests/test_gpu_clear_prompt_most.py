"""Attention over whole prompts with a `most` that is less than a sequence's tokens: the rows that it allows for are right, and see
all of the sequence where `causal` is off, also where tiles come in parts; the others are left alone."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_prompt import starts_of  # noqa: E402
from .test_gpu_clear_whole_prompt import check, clear_call, inputs  # noqa: E402


@pytest.mark.parametrize("kind,heads,group,dim", [("bf16", 1, 2, 128), ("fp16", 2, 3, 64)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("counts,most", [([3000], 1500), ([4000], 2000), ([700, 2500, 3, 1300, 0, 1201], 1200)])
def test_longer_sequences_than_most(counts, most, causal, heads, group, dim, kind):
    print("most", counts, most, causal, heads, group, dim, kind, flush=True)
    from holmes_amd import _native as nat

    g = torch.Generator().manual_seed(sum(counts) + most)
    n = sum(counts)
    size = nat.lib().hck_prompt_attend_workspace_bytes(n, len(counts), heads, group, dim, most, causal)
    assert size > 0 or (heads == 2 and len(counts) > 1 and not causal)      # in parts, but where there are tiles enough
    q, k, v = inputs(g, n, heads, group, dim, kind)
    starts = starts_of(counts)
    rows = torch.cat([torch.arange(c) < most for c in counts]).cuda()
    want = clear_call(q, k, v, starts, causal=causal, ranges=True)
    got = clear_call(q, k, v, starts, most=most, causal=causal, ranges=True)
    # (the other rows are the whole call's, for the comparison's sake)
    got = got._make(torch.where(rows.view(-1, *[1] * (x.dim() - 1)), x, y) for x, y in zip(got, want))
    check(got, q, k, v, counts, causal=causal)
    # into buffers of the caller's, with a workspace that others' bytes follow
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 9.0).cuda()
    work = torch.full((size + 4096,), 0x55, dtype=torch.uint8, device="cuda")
    nat.check(nat.lib().hck_prompt_attend(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), nat.HCK_BF16 if kind == "bf16" else nat.HCK_F16, n, heads, group, dim,
        q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), starts.data_ptr(), len(counts), most, causal,
        dim**-0.5, out.data_ptr(), lse.data_ptr(), None, None, work.data_ptr(), size, torch.cuda.current_stream().cuda_stream),
        "hck_prompt_attend")
    torch.cuda.synchronize()
    assert torch.equal(out[rows], got.out[rows]) and torch.equal(lse[rows], got.lse[rows])
    assert (out[~rows] == 7).all() and (lse[~rows] == 9).all() and (work[size:] == 0x55).all()


def test_sequences_that_grow_past_most_in_a_graph():
    """Starts are read at each replay: the sequences that a captured call meets may be longer than those it was made for."""
    print("graph", flush=True)
    g = torch.Generator().manual_seed(21)
    n, most = 3000, 1500
    q, k, v = inputs(g, n, 1, 2, 64, "bf16")
    starts = starts_of([1500, 1500])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        clear_call(q, k, v, starts, most=most, causal=False)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = clear_call(q, k, v, starts, most=most, causal=False)
    for cut in (1500, 2900, 3000, 64):
        starts[1] = cut
        q.mul_(0.99)
        graph.replay()
        torch.cuda.synchronize()
        rows = torch.cat([torch.arange(c) < most for c in (cut, n - cut)]).cuda()
        want = clear_call(q, k, v, starts, causal=False)
        mixed = got._replace(out=torch.where(rows[:, None, None], got.out, want.out), lse=torch.where(rows[:, None], got.lse, want.lse))
        check(mixed, q, k, v, [c for c in (cut, n - cut)], causal=False)
