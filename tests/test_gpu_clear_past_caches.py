"""Single tokens over a pool that is more than the L2 caches hold: loads that pass it by, against float64 with the
tolerance of test_gpu_clear_pages."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_pages import TYPES, build, check  # noqa: E402
from .test_gpu_clear_prompt import widen  # noqa: E402


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,group,dim", [(2, 4, 128), (3, 7, 64), (2, 12, 128)])
def test_single_tokens_of_a_large_pool(heads, group, dim, kind):
    print("large pool", heads, group, dim, kind, flush=True)
    g = torch.Generator().manual_seed(18)
    seqs = [1, 64, 65, 127, 700, 0, 16, 2100]
    room = (33 << 20) // (heads * dim * 136) + 1
    pool, table, keys, values = build(seqs, heads, dim, g, spare=room)
    assert pool.nbytes > 32 << 20
    q = torch.randn((len(seqs), heads * group, dim), generator=g).to(TYPES[kind]).cuda()
    for columns in (100, room):
        got = pool.attend(q, widen(table, columns), torch.tensor(seqs, dtype=torch.int32).cuda(), ranges=True)
        check(got, q, keys, values, [1] * len(seqs))
