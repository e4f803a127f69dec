"""The largest calls of token weights, eviction, rotary positions and whole-prompt attention that are taken: one step beyond, the
C entry points refuse them (no GPU needed: nothing here is launched)."""

import ctypes

from holmes_amd import _native as nat

from .test_clear_window import evict, prompt, rotary, weigh

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


def test_workgroups():
    """A launch counts its threads along an axis in 32 bits: 2^24 workgroups of 256 are refused before anything is launched."""
    one = dict(rotated=2, dim=2, heads=30000, kv=0)             # a token to a workgroup
    assert rotary(tokens=1 << 24, **one) == nat.HCK_ERR_ARG
    assert prompt(tokens=1 << 24, seqs=1 << 24, starts=P, most=1, heads=1, group=1) == nat.HCK_ERR_ARG
    assert prompt(tokens=1 << 21, seqs=1 << 21, starts=P, most=1, heads=8, group=1) == nat.HCK_ERR_ARG
    assert weigh(cols=(1 << 23) - 1, heads=64) == nat.HCK_ERR_ARG                              # few rows
    assert weigh(cols=(1 << 23) - 1, heads=4, tokens=100, most=100, starts=P) == nat.HCK_ERR_ARG   # many


def test_products_of_prompts():
    """More rows than any memory holds, and more sequences times key heads than 31 bits."""
    for bad in (dict(tokens=1 << 30, most=1, seqs=1 << 30, starts=P, heads=1 << 10, group=1 << 20),
                dict(tokens=1 << 30, most=1, starts=P, heads=1 << 20, group=1 << 10),
                dict(tokens=1 << 20, most=1 << 20, seqs=(1 << 31) - 1, starts=P, heads=2, group=1),
                dict(tokens=1 << 30, most=1 << 30, seqs=(1 << 31) - 1, starts=P, heads=(1 << 31) - 1, group=1)):
        assert prompt(**bad) == nat.HCK_ERR_ARG
        assert nat.lib().hck_prompt_attend_workspace_bytes(bad["tokens"], bad.get("seqs", 1), bad["heads"], bad["group"], 128,
                                                           bad["most"], 1) == 0
