"""The probabilities' two bf16 parts leave 2^-17 of each, seen where two values all but cancel.

Two tokens have the values 1 and -1 and nearly equal scores, which are exact; out = p0 - p1 is some 2^-7 of what it is
summed from, so that half a step of fp16 (2^-19 of it all) hides nothing.  Beside the parts, an exponential's argument
(up to 32, half a step 2^-20) and the instruction (2^-23) count: 2^-19 in all."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_prompt import starts_of, widen  # noqa: E402


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("each,columns", [(1, 1), (1024, 900)])   # single tokens, tiles of 128 rows
def test_parts(each, columns, dim):
    from holmes_amd import clear

    print("parts", each, columns, dim, flush=True)
    g = torch.Generator().manual_seed(dim)
    rows = 1024
    k, v = torch.zeros((2, 1, dim)), torch.ones((2, 1, dim))
    k[0, 0, 0] = k[1, 0, 1] = 4.0
    v[1] = -1.0
    pool = clear.ClearKVPages(1, kv_heads=1, head_dim=dim)
    pool.append(k.cuda(), v.cuda(), torch.arange(2).cuda())
    q = torch.zeros((rows, 4, dim), dtype=torch.float16)
    q[..., 0] = (1 + torch.rand((rows, 4), generator=g)).half()
    q[..., 1] = q[..., 0] - 2.0**-10 * torch.randint(1, 8, (rows, 4), generator=g).half()
    seqs = rows // each
    table = widen(torch.zeros((seqs, 1), dtype=torch.int32).cuda(), columns)
    got = pool.attend(q.cuda(), table, torch.full((seqs,), 2, dtype=torch.int32).cuda(), starts=starts_of([each] * seqs),
                      most=each, causal=False, scale=1.0)
    d = 2 * (q[..., 0].double() - q[..., 1].double())   # half the scores' difference
    want = torch.tanh(d)[..., None]
    off = (got.out.cpu().double() - want).abs()
    assert (off <= 2.0**-12 * want.abs() + 2.0**-17 + 2.0**-19).all(), float(off.max() * 2**17)
