"""What the cleartext operators refuse, checked before anything is launched (no GPU needed)."""

import ctypes

import pytest
import torch

from holmes_amd import _native as nat
from holmes_amd import clear

P = ctypes.c_void_p(0x1000)   # never read: every call here is refused first


def append(pool=P, pages=1, heads=1, dim=128, kind=0, keys=P, values=P, slots=P, tokens=1):
    return nat.lib().hck_kv4_append(pool, pages, heads, dim, kind, keys, 0, 0, values, 0, 0, slots, tokens, None)


def read(pool=P, pages=1, heads=1, dim=128, kind=0, slots=P, tokens=1, keys=P, values=P):
    return nat.lib().hck_kv4_read(pool, pages, heads, dim, kind, slots, tokens, keys, values, None)


@pytest.mark.parametrize("call", [append, read])
def test_pages_refuse(call):
    assert nat.lib().hck_kv4_page_bytes(128) == 128 * 136 and nat.lib().hck_kv4_page_bytes(64) == 128 * 68
    assert nat.lib().hck_kv4_page_bytes(96) == 0
    assert call(dim=96) == call(kind=3) == call(kind=-1) == -2
    for bad in (dict(pool=None), dict(pages=0), dict(heads=0), dict(heads=65536), dict(tokens=-1), dict(keys=None),
                dict(values=None), dict(slots=None), dict(tokens=1 << 62)):
        assert call(**bad) == nat.HCK_ERR_ARG, bad
    assert call(tokens=0, keys=None, values=None, slots=None) == 0


def attend(pool=P, pages=1, heads=1, dim=128, kind=0, q=P, tokens=1, group=1, table=P, cols=1, lengths=P, starts=None,
           seqs=1, most=1, scale=1.0, out=P, lse=P, low=None, high=None, work=None, size=0):
    return nat.lib().hck_kv4_attend(pool, pages, heads, dim, kind, q, tokens, group, 0, 0, table, 0, cols, lengths,
                                    starts, seqs, most, 1, scale, out, lse, low, high, work, size, None)


def test_attend_refuses():
    assert attend(dim=80) == attend(kind=nat.HCK_F32) == -2
    for bad in (dict(pool=None), dict(pages=0), dict(heads=0), dict(q=None), dict(group=0), dict(group=2000),
                dict(table=None), dict(lengths=None), dict(seqs=2), dict(seqs=-1), dict(seqs=1 << 17), dict(most=-1),
                dict(cols=-1), dict(cols=1 << 25), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                dict(scale=float("inf")), dict(out=None), dict(lse=None), dict(low=P), dict(high=P), dict(tokens=-1),
                dict(tokens=1 << 40)):
        assert attend(**bad) == nat.HCK_ERR_ARG, bad
    need = nat.lib().hck_kv4_attend_workspace_bytes(1, 1, 1, 1, 128, 1, 1000)
    assert need > 0
    assert attend(cols=1000) == attend(cols=1000, work=P, size=need - 1) == nat.HCK_ERR_WORKSPACE
    assert attend(tokens=0, seqs=0, q=None, out=None) == 0


def scores(x=P, kind=2, rows=1, vocab=10, tokens=P, top=0, given=P, entropy=P, ids=None, logs=None, work=None, size=0):
    return nat.lib().hck_token_scores(x, kind, rows, vocab, 0, tokens, top, given, entropy, ids, logs, work, size, None)


def test_scores_refuse():
    assert scores(kind=3) == -2
    for bad in (dict(x=None), dict(rows=-1), dict(rows=1 << 31), dict(vocab=0), dict(top=-1), dict(top=33, vocab=100),
                dict(top=11), dict(top=1), dict(top=1, ids=P), dict(given=None), dict(entropy=None),
                dict(x=ctypes.c_void_p(0x1002))):
        assert scores(**bad) == nat.HCK_ERR_ARG, bad
    need = nat.lib().hck_token_scores_workspace_bytes(1, 100000, 2, 4)
    assert need > 0
    assert scores(vocab=100000, top=4, ids=P, logs=P) == nat.HCK_ERR_WORKSPACE
    assert scores(vocab=100000, top=4, ids=P, logs=P, work=P, size=need - 1) == nat.HCK_ERR_WORKSPACE
    assert scores(rows=0, x=None, entropy=None) == 0


def test_python_checks():
    with pytest.raises(ValueError, match="head_dim"):
        clear.ClearKVPages(4, head_dim=96)
    with pytest.raises(ValueError, match="pages"):
        clear.ClearKVPages(0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        clear.ClearKVPages(4, device="cpu")
    x = torch.zeros((2, 5))
    for bad in (x[0], x.t().contiguous().t(), x.double(), torch.zeros((2, 0))):
        with pytest.raises(ValueError, match="logits"):
            clear.token_logprobs(bad)
    with pytest.raises(ValueError, match="top"):
        clear.token_logprobs(x, top=6)
    with pytest.raises(ValueError, match="tokens"):
        clear.token_logprobs(x, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="tokens"):
        clear.token_logprobs(x, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        clear.token_logprobs(x)


def test_softmax_ranges_without_a_row():
    none = torch.tensor([-float("inf")])
    with pytest.raises(ValueError, match="no row"):
        clear.softmax_ranges(-none, none, none)
    r = clear.softmax_ranges(torch.tensor([-2.0, float("inf")]), torch.tensor([4.0, -float("inf")]),
                             torch.tensor([4.5, -float("inf")]))
    assert r.score_shift == 1.0 and r.exp_interval[0] < -1.5 and r.exp_interval[1] > 1.5
    assert r.rsqrt_interval[0] < 33.12 < r.rsqrt_interval[1]
