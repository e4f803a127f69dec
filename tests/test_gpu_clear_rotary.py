"""Rotary positions (holmes_amd.clear.RotaryPositions) against a model in exact turns and 64 bits.

Tolerance, of a pair (x0, x1) that becomes x0 c - x1 s: the cosine and sine in 32 bits, each within 2 steps (polynomials
below 2^-26, their and the argument's roundings), times ``amount`` one more half; two products and a sum, another half step
each: 4 2^-23 (|x0| + |x1|) amount in all, far positions' angles included (2^-34 turns); and half a step of the output's type (below its least
normal number, one step)."""

import math
from fractions import Fraction

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LEAST = {torch.bfloat16: 2.0**-133, torch.float16: 2.0**-24, torch.float32: 2.0**-149}
TURN = 2 * Fraction(314159265358979323846264338327950288419716939937510582097494459, 10**62)


def angles(plan, positions):
    """cos and sin of every position's pairs, by exact turns."""
    rows = []
    for p in positions.tolist():
        rows.append([2 * math.pi * float((p * Fraction(f) / TURN) % 1) for f in plan.frequencies])
    t = torch.tensor(rows, dtype=torch.float64)
    return torch.cos(t), torch.sin(t)


def check(plan, positions, x, got, sign=1.0):
    c, s = (plan.amount * y[:, None] for y in angles(plan, positions.cpu()))
    s = sign * s
    x, r = x.cpu().double(), plan.rotated
    part = x[..., :r]
    a, b = (part[..., ::2], part[..., 1::2]) if plan.interleaved else part.chunk(2, -1)
    u, v = a * c - b * s, b * c + a * s
    size = (a.abs() + b.abs()) * plan.amount
    if plan.interleaved:
        want, size = torch.stack([u, v], -1).flatten(-2), size.repeat_interleave(2, -1)
    else:
        want, size = torch.cat([u, v], -1), size.repeat(1, 1, 2)
    assert got.dtype in LEAST and got.is_contiguous()
    tol = 4 * 2.0**-23 * size + torch.finfo(got.dtype).eps / 2 * (1 + 2.0**-20) * want.abs() + LEAST[got.dtype]
    off = (got[..., :r].cpu().double() - want).abs()
    assert (off <= tol).all(), float((off - tol).max())
    assert torch.equal(got[..., r:].cpu().double(), x[..., r:])


@pytest.mark.parametrize("kind", sorted(TYPES))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated,heads,kv_heads,tokens", [
    (128, 128, 32, 8, 1), (128, 64, 5, 1, 7), (64, 32, 3, 3, 33), (64, 6, 1, 2, 5), (10, 6, 2, 1, 9), (512, 512, 2, 1, 3),
    (2, 2, 1, 1, 1), (96, 48, 3, 1, 1030), (64, 16, 2, 1, 4101)])
def test_rotate(dim, rotated, heads, kv_heads, tokens, interleaved, kind):
    from holmes_amd import clear

    print("rotate", dim, rotated, heads, kv_heads, tokens, interleaved, kind, flush=True)
    g = torch.Generator().manual_seed(dim + tokens)
    plan = clear.RotaryPositions(dim, rotated=rotated, interleaved=interleaved)
    positions = torch.randint(0, 5000, (tokens,), generator=g).cuda()
    q = torch.randn((tokens, heads, dim), generator=g).to(TYPES[kind]).cuda()
    k = torch.randn((tokens, kv_heads, dim), generator=g).to(TYPES[kind]).cuda()
    a, b = plan.rotate(positions, q, k)
    check(plan, positions, q, a)
    check(plan, positions, k, b)
    alone = plan.rotate(positions.int(), q, inverse=True)
    check(plan, positions, q, alone, sign=-1.0)


@pytest.mark.parametrize("scaling", [("linear", 8.0), ("base", 4.0), ("wavelength", 8.0, 8192, 1.0, 4.0),
                                     ("ramp", 16.0, 4096, 1.0, 32.0)])
def test_far_positions_and_scalings(scaling):
    from holmes_amd import clear

    print("far", scaling, flush=True)
    g = torch.Generator().manual_seed(3)
    positions = torch.tensor([0, 1, -1, 131071, 2**31 - 1, -2**31 + 1, 2**24 + 1, 999999937])
    x = torch.randn((8, 3, 128), generator=g).cuda()
    plan = clear.RotaryPositions(scaling=clear.RotaryScaling(*scaling))
    check(plan, positions, x, plan.rotate(positions.cuda(), x))
    check(plan, positions, x, plan.rotate(positions.int().cuda(), x))


def test_strides_and_odd_values():
    from holmes_amd import clear

    print("strides", flush=True)
    g = torch.Generator().manual_seed(4)
    plan = clear.RotaryPositions(64, base=10000.0)
    wide = torch.randn((11, 7, 2, 65), generator=g).to(torch.bfloat16).cuda()   # odd strides and addresses
    positions = torch.arange(40).cuda()[::2][:11]
    a, b = plan.rotate(positions, wide[:, :5, 0, 1:], wide[:, 5:, 1, :64])
    check(plan, positions, wide[:, :5, 0, 1:], a)
    check(plan, positions, wide[:, 5:, 1, :64], b)
    across = torch.randn((5, 9, 64), generator=g).cuda().transpose(0, 1)        # heads before tokens
    check(plan, positions[:9], across, plan.rotate(positions[:9], across))
    one = torch.randn((9, 1, 64), generator=g).cuda().expand(9, 4, 64)          # a broadcast head
    check(plan, positions[:9], one, plan.rotate(positions[:9], one))
    # a value that is none stays with its pair
    x = torch.randn((3, 2, 64), generator=g)
    x[1, 0, 5], x[2, 1, 40] = math.nan, math.inf
    y = plan.rotate(positions[:3], x.cuda()).cpu()
    odd = torch.zeros(3, 2, 64, dtype=torch.bool)
    odd[1, 0, [5, 37]] = odd[2, 1, [8, 40]] = True
    assert torch.equal(~torch.isfinite(y), odd)
    # nothing to do
    assert plan.rotate(positions[:0], x.cuda()[:0]).shape == (0, 2, 64)
    a, b = plan.rotate(positions[:3], x.cuda(), x.cuda()[:, :0])
    assert b.shape == (3, 0, 64)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_more_than_the_caches_hold(interleaved, kind):
    """Large calls, which go past the caches, give what their tokens do in small ones."""
    from holmes_amd import clear

    print("large", interleaved, kind, flush=True)
    g = torch.Generator(device="cuda").manual_seed(6)
    plan = clear.RotaryPositions(128, rotated=96, interleaved=interleaved)
    positions = torch.arange(3500, device="cuda") * 7
    q = torch.randn((3500, 32, 128), generator=g, device="cuda").to(TYPES[kind])
    k = torch.randn((3500, 8, 128), generator=g, device="cuda").to(TYPES[kind])
    a, b = plan.rotate(positions, q, k)
    check(plan, positions[::500], q[::500], a[::500].contiguous())
    for i in range(0, 3500, 500):
        c, d = plan.rotate(positions[i:i + 500], q[i:i + 500], k[i:i + 500])
        assert torch.equal(a[i:i + 500], c) and torch.equal(b[i:i + 500], d)


def test_back_and_forth_and_the_encrypted_layers_phases():
    """The default plan is DecodeSpec's embedding: its phases in 32 bits are off by the angle's rounding there."""
    from holmes_amd import clear
    from holmes_amd.decode import DecodeSpec, rope_phase

    print("phases", flush=True)
    plan = clear.RotaryPositions()
    ones = torch.zeros((1, 1, 128))
    ones[..., :64] = 1.0
    for at in (0, 1, 256):
        y = plan.rotate(torch.tensor([at]).cuda(), ones.cuda()).cpu()[0, 0].double()
        phase = torch.from_numpy(rope_phase(at, DecodeSpec()))
        assert (torch.complex(y[:64], y[64:]) - phase).abs().max() < (at + 1) * 2.0**-21   # a few steps of angles up to `at`
    x = torch.randn((50, 4, 128)).cuda()
    positions = torch.arange(1000000, 1000050).cuda()
    back = plan.rotate(positions, plan.rotate(positions, x), inverse=True)
    # twice the tolerance of one rotation, whose outputs are at most |x0| + |x1|
    assert ((back - x).abs() <= 16 * 2.0**-23 * (x.abs() + x.abs().roll(64, -1))).all()


def test_graph():
    from holmes_amd import clear

    print("graph", flush=True)
    plan = clear.RotaryPositions(64)
    x, at = torch.randn((70, 3, 64)).cuda(), torch.arange(70).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        plan.rotate(at, x, x)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a, b = plan.rotate(at, x, x)
    for step in range(3):
        at += 1000 * step
        graph.replay()
        torch.cuda.synchronize()
        check(plan, at, x, a)
        assert torch.equal(a, b)
