"""The largest calls of token weights, eviction, rotary positions and whole-prompt attention that are taken: one step beyond, the
C entry points refuse them (no GPU needed: nothing here is launched)."""

import ctypes

from holmes_amd import _native as nat

from .test_clear_window import evict, weigh

P = ctypes.c_void_p(0x1000)   # never read


def test_rows_of_weights():
    """A sequence's rows are counted in 31 bits by whole stages of 64.  (In parts, for which there is no workspace here.)"""
    most = (1 << 31) - 1 - 256
    for group in (1, 5):
        rows = most // group
        many = dict(tokens=(1 << 31) - 1, group=group, starts=P)
        assert weigh(**many, most=rows) == nat.HCK_ERR_WORKSPACE
        assert nat.lib().hck_kv4_weigh_workspace_bytes((1 << 31) - 1, 1, 1, group, rows, 1) > 0
        assert weigh(**many, most=rows + 1) == nat.HCK_ERR_ARG
        assert nat.lib().hck_kv4_weigh_workspace_bytes((1 << 31) - 1, 1, 1, group, rows + 1, 1) == 0


def test_sequences_times_key_heads():
    """Numbered in 31 bits."""
    for call, more in ((weigh, dict(tokens=65535)), (evict, {})):
        assert call(seqs=65535, heads=32769, **more) == nat.HCK_ERR_ARG
        assert call(seqs=65535, heads=32769, cols=200, **more) == nat.HCK_ERR_ARG
    assert evict(seqs=65535, heads=32768, cols=200) == nat.HCK_ERR_WORKSPACE     # the most that is taken, in segments
    assert nat.lib().hck_kv4_evict_workspace_bytes(65535, 32768, 200) > 0
    assert nat.lib().hck_kv4_evict_workspace_bytes(65535, 32769, 200) == 0
    assert nat.lib().hck_kv4_weigh_workspace_bytes(65535, 65535, 32769, 1, 1, 1) == 0
