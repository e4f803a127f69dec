"""Rotary frequencies, and what rotary positions, whole-prompt attention, token weights and eviction refuse before anything is
launched (no GPU needed: every call here is refused for an argument, at the latest for its device)."""

import ctypes
import math
from fractions import Fraction

import pytest
import torch

from holmes_amd import _native as nat
from holmes_amd import clear

P = ctypes.c_void_p(0x1000)   # never read
POOL = (0x1000, 4, 2, 128, 0)
BF16 = torch.bfloat16


# ---------------------------------------------------------------------------- frequencies
def test_frequencies():
    got, amount = clear._rotary_frequencies(8, 10000.0, None)
    assert amount == 1.0 and got == pytest.approx([1.0, 0.1, 0.01, 0.001], rel=1e-14)
    got, _ = clear._rotary_frequencies(8, 10000.0, clear.RotaryScaling("linear", 4.0))
    assert got == pytest.approx([0.25, 0.025, 0.0025, 0.00025], rel=1e-14)
    # the first pair as it was, the last divided
    got, _ = clear._rotary_frequencies(8, 10000.0, clear.RotaryScaling("base", 4.0))
    assert got[0] == 1.0 and got[3] == pytest.approx(0.001 / 4, rel=1e-13)
    assert got[1] / got[0] == pytest.approx(got[3] / got[2], rel=1e-13)


def test_turns():
    """Nearest multiples of 2^-64 turns, against 80 digits of pi."""
    turn = 2 * Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862089, 10**79)
    for f in [1.0, 0.1, 500000.0**-0.75, 1e-30, 0.0, 6.283185307179586, 3.0, *clear._rotary_frequencies(128, 500000.0, None)[0]]:
        want = Fraction(f) / turn * 2**64
        assert abs((clear._turns(f) - want + 2**63) % 2**64 - 2**63) <= Fraction(1, 2) + Fraction(1, 10**9), f


def test_blended_frequencies():
    plain, _ = clear._rotary_frequencies(128, 500000.0, None)
    turns = [8192 * f / (2 * math.pi) for f in plain]
    got, amount = clear._rotary_frequencies(128, 500000.0, clear.RotaryScaling("wavelength", 8.0, 8192, 1.0, 4.0))
    assert amount == 1.0
    for f, g, t in zip(plain, got, turns):
        part = min(max((t - 1.0) / 3.0, 0.0), 1.0)
        assert g == pytest.approx(f * (part + (1 - part) / 8), rel=1e-13)
    assert got[0] == plain[0] and got[-1] == plain[-1] / 8 and any(f / 8 < g < f for f, g in zip(plain, got))
    got, amount = clear._rotary_frequencies(128, 500000.0, clear.RotaryScaling("ramp", 16.0, 8192, 1.0, 32.0))
    assert amount == pytest.approx(1.2772588722239782, rel=1e-15)
    # between the pair before 32 turns and the one behind a single turn, in even steps
    first = max(i for i, t in enumerate(turns) if t >= 32.0)
    last = min(i for i, t in enumerate(turns) if t <= 1.0)
    for i, (f, g) in enumerate(zip(plain, got)):
        part = min(max((i - first) / (last - first), 0.0), 1.0)
        assert g == pytest.approx(f * (1 - part) + f / 16 * part, rel=1e-12)


@pytest.mark.parametrize("change,match", [
    (dict(head_dim=0), "head_dim"), (dict(head_dim=63), "head_dim"), (dict(head_dim=514), "head_dim"),
    (dict(rotated=130), "rotated"), (dict(rotated=0), "rotated"), (dict(rotated=3), "rotated"),
    (dict(base=0.0), "base"), (dict(base=5e-324), "base"), (dict(base=1e300), "base"), (dict(base=-1.0), "base"),
    (dict(scaling=clear.RotaryScaling("base", 1e300), rotated=4), "factor"), (dict(scaling=clear.RotaryScaling("ramp", 2.0, math.inf)), "blended"), (dict(base=math.nan), "base"), (dict(base=math.inf), "base"),
    (dict(scaling=clear.RotaryScaling("none", 2.0)), "kind"), (dict(scaling=clear.RotaryScaling("linear", 0.5)), "factor"),
    (dict(scaling=clear.RotaryScaling("linear", math.nan)), "factor"), (dict(rotated=2, scaling=clear.RotaryScaling("base", 2.0)), "pairs"),
    (dict(scaling=clear.RotaryScaling("wavelength", 2.0, 0)), "blended"),
    (dict(scaling=clear.RotaryScaling("ramp", 2.0, 100, 4.0, 4.0)), "blended"),
    (dict(base=1.0, scaling=clear.RotaryScaling("ramp", 2.0)), "above 1"),
])
def test_plans_refuse(change, match):
    with pytest.raises(ValueError, match=match):
        clear.RotaryPositions(**change)


def test_no_cpu_path():
    with pytest.raises(RuntimeError, match="GPU"):
        clear.RotaryPositions(device="cpu")
    x = torch.zeros((3, 2, 64), dtype=BF16)
    with pytest.raises(RuntimeError, match="GPU"):
        clear.prompt_attention(x, x, x)
    with pytest.raises(RuntimeError, match="GPU"):
        clear._window().rotate(torch.zeros(4, dtype=torch.int64), 64, 8, False, 1.0, torch.arange(3), x, None, False)


# ---------------------------------------------------------------------------- the C entry points
def rotary(positions=P, size=8, tokens=3, turns=P, rotated=128, inter=0, kind=0, dim=128, q=P, heads=2, out=P, k=P, kv=1, out_k=P):
    return nat.lib().hck_rotary(positions, size, tokens, turns, rotated, inter, 0, 1.0, kind, dim, q, 0, 0, heads, out, k, 0, 0,
                                kv, out_k, None)


def test_rotary_refuses():
    assert rotary(kind=3) == rotary(dim=1) == rotary(dim=7) == rotary(dim=514) == -2
    for bad in (dict(rotated=0), dict(rotated=5), dict(rotated=130), dict(tokens=-1), dict(heads=-1), dict(kv=-1),
                dict(heads=65535), dict(heads=9000), dict(size=2), dict(positions=None), dict(turns=None), dict(q=None),
                dict(out=None), dict(k=None), dict(out_k=None), dict(tokens=1 << 50)):
        assert rotary(**bad) == nat.HCK_ERR_ARG, bad
    assert rotary(tokens=0, q=None, positions=None) == 0
    assert rotary(heads=0, kv=0, q=None, k=None) == 0


def prompt(q=P, k=P, v=P, kind=0, tokens=10, heads=2, group=2, dim=128, strides=(512, 128, 256, 128, 256, 128), starts=None,
           seqs=1, most=10, scale=1.0, out=P, lse=P, low=None, high=None, work=None, size=0):
    return nat.lib().hck_prompt_attend(q, k, v, kind, tokens, heads, group, dim, *strides, starts, seqs, most, 1, scale, out,
                                       lse, low, high, work, size, None)


def test_prompt_refuses():
    assert prompt(kind=nat.HCK_F32) == prompt(dim=96) == -2
    odd = ctypes.c_void_p(0x1008)
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lse=None), dict(low=P), dict(high=P), dict(q=odd),
                dict(k=odd), dict(v=odd), dict(out=odd), dict(tokens=-1), dict(tokens=1 << 31), dict(heads=0), dict(group=0),
                dict(heads=1 << 20, group=1 << 20), dict(seqs=-1), dict(seqs=2), dict(most=-1), dict(scale=0.0),
                dict(scale=math.nan), dict(scale=math.inf), dict(scale=1e300), dict(scale=1e-300),
                dict(strides=(512, 128, 256, 128, 256, 4)), dict(strides=(511, 128, 256, 128, 256, 128)),
                dict(strides=(512, 128, 120, 128, 256, 128)), dict(strides=(512, 128, 256, 128, 0, 128)),
                dict(strides=(512, 128, 256, 128, 1 << 24, 128)), dict(tokens=1 << 30, most=1 << 30),
                dict(tokens=1 << 24, most=1 << 24, group=200)):
        assert prompt(**bad) == nat.HCK_ERR_ARG, bad
    need = nat.lib().hck_prompt_attend_workspace_bytes(4000, 1, 2, 2, 128, 4000, 1)
    assert need > 0
    long = dict(tokens=4000, most=4000)
    assert prompt(**long) == prompt(**long, work=P, size=need - 1) == prompt(**long, work=odd, size=need) == nat.HCK_ERR_WORKSPACE
    assert prompt(seqs=0, starts=P, q=None) == prompt(tokens=0, q=None) == prompt(most=0, q=None) == 0


def weigh(pool=P, pages=1, heads=1, dim=128, kind=0, q=P, tokens=1, group=1, table=P, cols=1, lengths=P, starts=None, seqs=1,
          most=1, scale=1.0, lse=P, prior=None, places=0, out=P, work=None, size=0):
    return nat.lib().hck_kv4_weigh(pool, pages, heads, dim, kind, q, tokens, group, 0, 0, table, 0, cols, lengths, starts, seqs,
                                   most, 1, scale, lse, prior, 0, 0, places, out, work, size, None)


def test_weigh_refuses():
    assert weigh(dim=96) == weigh(kind=nat.HCK_F32) == -2
    for bad in (dict(pool=None), dict(pages=0), dict(heads=0), dict(heads=65536), dict(q=None), dict(lse=None), dict(out=None),
                dict(table=None), dict(lengths=None), dict(tokens=-1), dict(tokens=2), dict(group=0), dict(group=1 << 30, most=4),
                dict(seqs=-1), dict(seqs=65536, tokens=65536), dict(most=-1), dict(cols=-1), dict(cols=1 << 23),
                dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(places=-1), dict(places=3),
                dict(cols=(1 << 23) - 1, heads=60000)):
        assert weigh(**bad) == nat.HCK_ERR_ARG, bad
    need = nat.lib().hck_kv4_weigh_workspace_bytes(1000, 1, 1, 4, 1000, 8)
    assert need > 0
    many = dict(tokens=1000, group=4, most=1000, cols=8, starts=P)
    assert weigh(**many) == weigh(**many, work=P, size=need - 1) == nat.HCK_ERR_WORKSPACE
    assert weigh(seqs=0, tokens=0, q=None, lse=None) == weigh(cols=0, out=None) == 0


def evict(pool=P, pages=1, heads=1, dim=128, table=P, cols=1, lengths=P, seqs=1, weights=P, places=128, into=P, into_cols=1,
          keep=10, recent=2, kept=P, now=P, left=P, work=None, size=0):
    return nat.lib().hck_kv4_evict(pool, pages, heads, dim, table, 0, cols, lengths, seqs, weights, 0, 0, places, into, 0,
                                   into_cols, keep, recent, kept, now, left, work, size, None)


def test_evict_refuses():
    assert evict(dim=96) == -2
    for bad in (dict(pool=None), dict(pages=0), dict(heads=0), dict(heads=65536), dict(table=None), dict(lengths=None),
                dict(weights=None), dict(into=None), dict(kept=None), dict(now=None), dict(left=None), dict(cols=-1),
                dict(cols=1 << 23), dict(seqs=-1), dict(seqs=65536), dict(places=-1), dict(into_cols=-1), dict(keep=-1),
                dict(keep=129), dict(recent=-1), dict(recent=11), dict(into_cols=1 << 23)):
        assert evict(**bad) == nat.HCK_ERR_ARG, bad
    need = nat.lib().hck_kv4_evict_workspace_bytes(1, 1, 129)
    assert need > 0 and nat.lib().hck_kv4_evict_workspace_bytes(1, 1, 128) == 0
    assert evict(cols=129) == evict(cols=129, work=P, size=need - 1) == nat.HCK_ERR_WORKSPACE
    assert evict(seqs=0, lengths=None, now=None) == 0


# ---------------------------------------------------------------------------- the Python side
def kv(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("change,match", [
    (dict(turns=7), "tensor"), (dict(positions=torch.arange(4)), "positions"), (dict(positions=torch.zeros(3)), "positions"),
    (dict(positions=torch.zeros((3, 1), dtype=torch.int64)), "positions"), (dict(queries=kv(3, 2, 64, dtype=torch.float64)), "queries"),
    (dict(queries=kv(3, 64)), "queries"), (dict(queries=kv(3, 2, 128)), "queries"), (dict(keys=kv(4, 2, 64)), "keys"),
    (dict(keys=kv(3, 2, 64, dtype=torch.float16)), "one type"), (dict(keys="none"), "tensor"),
    (dict(queries=kv(64, 2, 3).transpose(0, 2)), "contiguous"), (dict(queries=kv(3, 20000, 64)), "heads"),
])
def test_rotate(change, match):
    got = dict(turns=torch.zeros(4, dtype=torch.int64), head_dim=64, rotated=8, interleaved=False, amount=1.0,
               positions=torch.arange(3), queries=kv(3, 2, 64), keys=None, inverse=False)
    got.update(change)
    with pytest.raises((ValueError, TypeError), match=match):
        clear._window().rotate(*got.values())


@pytest.mark.parametrize("change,match", [
    (dict(queries=kv(5, 4, 64, dtype=torch.float32)), "bfloat16 or float16"), (dict(queries=kv(5, 4, 96)), "64 or 128"),
    (dict(queries=kv(5, 64)), "queries"), (dict(keys=kv(4, 2, 64)), "keys"), (dict(keys=kv(5, 2, 128)), "keys"),
    (dict(values=kv(5, 4, 64)), "keys"), (dict(values=kv(5, 2, 64, dtype=torch.float16)), "keys"), (dict(keys=kv(5, 3, 64)), "keys"),
    (dict(keys=kv(5, 3, 64), values=kv(5, 3, 64)), "multiple"), (dict(keys=kv(5, 0, 64), values=kv(5, 0, 64)), "multiple"),
    (dict(starts=torch.zeros(3, dtype=torch.int64)), "starts"), (dict(starts=torch.zeros(0, dtype=torch.int32)), "starts"),
    (dict(starts=torch.zeros((1, 2), dtype=torch.int32)), "starts"), (dict(most=-1), "most"), (dict(scale=0.0), "scale"),
    (dict(scale=-2.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"), (dict(scale="one"), "real|float"),
    (dict(queries=kv(64, 4, 5).transpose(0, 2)), "contiguous"),
])
def test_prompt_attention(change, match):
    got = dict(queries=kv(5, 4, 64), keys=kv(5, 2, 64), values=kv(5, 2, 64), starts=None, most=None, causal=True, scale=None,
               ranges=False)
    got.update(change)
    with pytest.raises((ValueError, TypeError), match=match):
        clear._window().prompt(*got.values())


@pytest.mark.parametrize("change,match", [
    (dict(queries=kv(5, 4, 128, dtype=torch.float32)), "bfloat16 or float16"), (dict(queries=kv(5, 4, 64)), "queries"),
    (dict(), "queries"),                                    # all as it should be, but on the CPU
    (dict(queries=7), "tensor"),
])
def test_weigh(change, match):
    got = dict(queries=kv(5, 4, 128), table=torch.zeros((5, 1), dtype=torch.int32), lengths=torch.ones(5, dtype=torch.int32),
               lse=kv(5, 4, dtype=torch.float32), starts=None, most=None, causal=True, scale=None, prior=None)
    got.update(change)
    with pytest.raises((ValueError, TypeError), match=match):
        clear._window().weigh(*POOL, *got.values())


@pytest.mark.parametrize("change,match", [
    (dict(table=torch.zeros(5, dtype=torch.int32)), "table"), (dict(lengths=torch.ones(4, dtype=torch.int32)), "table"),
    (dict(), "table"), (dict(weights="w"), "tensor"), (dict(into=3), "tensor"),
])
def test_evict(change, match):
    got = dict(table=torch.zeros((5, 1), dtype=torch.int32), lengths=torch.ones(5, dtype=torch.int32),
               weights=torch.zeros((5, 2, 128)), into=torch.zeros((5, 1), dtype=torch.int32), keep=3, recent=0)
    got.update(change)
    with pytest.raises((ValueError, TypeError), match=match):
        clear._window().evict(*POOL, *got.values())


@pytest.mark.parametrize("name,count", [("rotate", 9), ("prompt", 8), ("weigh", 14), ("evict", 11)])
def test_numbers_of_arguments(name, count):
    with pytest.raises(TypeError, match="arguments"):
        getattr(clear._window(), name)(*[None] * (count - 1))
