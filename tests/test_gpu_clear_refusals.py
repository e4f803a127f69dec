"""What the cleartext operators refuse of GPU tensors, each by one thing that is wrong with it."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_pages_refuse():
    from holmes_amd import clear

    print("refusals: pages", flush=True)
    pool = clear.ClearKVPages(2, kv_heads=2, head_dim=64)
    good = torch.zeros((3, 2, 64), device="cuda")
    slots = torch.arange(3, device="cuda")
    before = pool.buf.clone()
    for bad in (good[:2], good[:, :1], good[..., :32], good[0], good.cpu(), good.half(), good.double(),
                torch.zeros((3, 2, 128), device="cuda")[..., ::2]):
        with pytest.raises(ValueError):
            pool.append(bad, good, slots)
        with pytest.raises(ValueError):
            pool.append(good, bad, slots)
    for bad in (slots[None], slots.int(), slots.cpu(), slots[:2]):
        with pytest.raises(ValueError):
            pool.append(good, good, bad)
    for bad in (slots[None], slots.int(), slots.cpu()):
        with pytest.raises(ValueError):
            pool.read(bad)
    for bad in (torch.float64, torch.int8):
        with pytest.raises(ValueError, match="dtype"):
            pool.read(slots, bad)
    with pytest.raises(TypeError):
        pool.read(slots, "bfloat16")
    torch.cuda.synchronize()
    assert torch.equal(pool.buf, before)
    pool.append(good, good, slots)                          # and the good ones are taken, none among them
    pool.append(good[:0], good[:0], slots[:0])
    assert pool.read(slots[:0])[0].shape == (0, 2, 64)


def test_attend_refuses():
    from holmes_amd import clear

    print("refusals: attend", flush=True)
    pool = clear.ClearKVPages(2, kv_heads=2, head_dim=64)
    q = torch.zeros((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((3, 1), dtype=torch.int32, device="cuda")
    lengths = torch.ones(3, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    pool.attend(q, table, lengths)
    pool.attend(q, table, lengths, starts=starts, most=0)
    wide = torch.zeros((3, 4), dtype=torch.int32, device="cuda")
    for bad in (q.float(), q.cpu(), q[:, :3], q[:, :0], q[..., :32], q[0], q[:2], q.repeat(1, 1, 2)[..., ::2]):
        with pytest.raises(ValueError):
            pool.attend(bad, table, lengths)
    for bad in (table.long(), table.cpu(), table[:2], table[0], wide[:, ::2]):
        with pytest.raises(ValueError):
            pool.attend(q, bad, lengths)
    for bad in (lengths.long(), lengths.cpu(), lengths[:2], lengths[None], torch.ones(6, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError):
            pool.attend(q, table, bad)
    for bad in (starts.long(), starts.cpu(), starts[:3], starts[None], starts.repeat_interleave(2)[::2]):
        with pytest.raises(ValueError, match="starts"):
            pool.attend(q, table, lengths, starts=bad)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="scale"):
            pool.attend(q, table, lengths, scale=bad)
    with pytest.raises(ValueError, match="most"):
        pool.attend(q, table, lengths, starts=starts, most=-1)
    with pytest.raises(TypeError):
        pool.attend(q, table, lengths, scale="one")


def test_scores_refuse():
    from holmes_amd import clear

    print("refusals: scores", flush=True)
    x = torch.zeros((3, 8), device="cuda")
    tokens = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (x[0], x.t(), x.double(), x[:, :0], x[:, ::2]):
        with pytest.raises(ValueError, match="logits"):
            clear.token_logprobs(bad)
    for bad in (tokens.int(), tokens.cpu(), tokens[:2], tokens[None]):
        with pytest.raises(ValueError, match="tokens"):
            clear.token_logprobs(x, bad)
    for bad in (-1, 9, 33):
        with pytest.raises(ValueError, match="top"):
            clear.token_logprobs(x, top=bad)
    assert clear.token_logprobs(x, tokens, top=8).top_ids.tolist() == [list(range(8))] * 3
