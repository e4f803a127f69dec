"""A pool's bytes belong to the tensor that its ``buf`` is at the time of a call."""

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_another_buffer():
    from holmes_amd import clear

    print("another buffer", flush=True)
    g = torch.Generator().manual_seed(2)
    pool = clear.ClearKVPages(3, kv_heads=2, head_dim=64)
    k = torch.randn((5, 2, 64), generator=g).cuda()
    slots = torch.arange(5).cuda()
    pool.append(k, k, slots)
    first, want = pool.buf, pool.read(slots)[0].clone()
    pool.buf = torch.zeros_like(first)
    assert (pool.read(slots)[0] == 0).all()
    pool.append(k, k, slots)
    assert torch.equal(pool.buf, first) and torch.equal(pool.read(slots)[0], want)
    short = torch.zeros_like(first)
    short.untyped_storage().resize_(100)
    for bad in (first[:2], first.cpu(), first.int(), first.transpose(0, 1), short):
        pool.buf = bad
        for call in (lambda: pool.append(k, k, slots), lambda: pool.read(slots),
                     lambda: pool.attend(k[:1].bfloat16(), slots[None, :1].int(), slots[1:2].int())):
            with pytest.raises(ValueError, match="buf"):
                call()
