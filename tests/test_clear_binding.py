"""The native calls behind holmes_amd.clear refuse what does not fit before anything is launched (no GPU needed:
every call here is refused for an argument, at the latest for its device)."""

import pytest
import torch

from holmes_amd import clear

POOL = (0x1000, 4, 2, 128, 0)   # an address that is never read, 4 pages, 2 heads of 128, device 0
BF16 = torch.bfloat16


def kv(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


def test_append_and_read():
    b = clear._bound()
    slots = torch.zeros(3, dtype=torch.int64)
    for bad in (slots[None], slots.int(), slots):   # the last for its device
        with pytest.raises(ValueError, match="slots"):
            b.append(*POOL, kv(3, 2, 128), kv(3, 2, 128), bad)
        with pytest.raises(ValueError, match="slots"):
            b.read(*POOL, bad, BF16)
    for bad in (None, 3, "keys"):
        with pytest.raises(TypeError, match="keys"):
            b.append(*POOL, bad, kv(3, 2, 128), slots)
    with pytest.raises(TypeError, match="arguments"):
        b.append(*POOL)
    with pytest.raises(TypeError, match="arguments"):
        b.read(*POOL, slots)


@pytest.mark.parametrize("change,match", [
    (dict(queries=kv(5, 4, 128, dtype=torch.float32)), "bfloat16 or float16"),
    (dict(queries=kv(5, 4, 64)), "queries"),
    (dict(queries=kv(5, 512)), "queries"),
    (dict(queries=kv(5, 4, 128).transpose(0, 2).contiguous().transpose(0, 2)), "queries"),
    (dict(), "queries"),                                     # all as it should be, but on the CPU
    (dict(queries=7), "tensor"),
])
def test_attend(change, match):
    got = dict(queries=kv(5, 4, 128), table=torch.zeros((5, 1), dtype=torch.int32),
               lengths=torch.ones(5, dtype=torch.int32), starts=None, most=None, causal=True, scale=None, ranges=False)
    got.update(change)
    with pytest.raises((ValueError, TypeError), match=match):
        clear._bound().attend(*POOL, *got.values())


def test_scores():
    for top in (-1, 6, 1 << 40):
        with pytest.raises(ValueError, match="top"):
            clear.token_logprobs(kv(2, 5), top=top)
    with pytest.raises(TypeError):
        clear.token_logprobs(kv(2, 5), top="three")
    with pytest.raises(TypeError, match="logits"):
        clear.token_logprobs([[1.0]])
    with pytest.raises(ValueError, match="logits"):
        clear.token_logprobs(torch.zeros((2, 5), dtype=torch.int32))
