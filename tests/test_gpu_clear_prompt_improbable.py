"""Attention over whole prompts where most of the probability is with a token that has no value, and what is left with improbable ones.

A probability goes into its product in 16 bits, relative to the sum of exponentials: half a step, and in fp16, whose exponentials
are taken times 2^15 against a reference less than 2^8 above the row's largest, no less than half of 2^-24 / 2^7 = 2^-31 (so those below 2^-32
may count as 0).  bf16 keeps a relative half step down to 2^-100.  The rest of the tolerance is test_gpu_clear_whole_prompt's."""

import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from .test_gpu_clear_whole_prompt import TYPES, clear_call  # noqa: E402


def inputs(n, group, dim, kind, size):
    """Scores that are key's first values: 0 for one token, -7 to -42 for the others."""
    g = torch.Generator().manual_seed(n + group + dim)
    q = torch.zeros((n, group, dim))
    q[:, :, 0] = math.sqrt(dim) if dim == 64 else 8.0
    k = torch.zeros((n, 1, dim))
    k[:, 0, 0] = -7.0 - 35.0 * torch.rand(n, generator=g)
    sink = n // 3
    k[sink, 0, 0] = 0.0
    v = size * torch.randn((n, 1, dim), generator=g)
    v[sink] = 0.0
    return [x.to(TYPES[kind]) for x in (q, k, v)], 8.0**-1, sink


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("n,group,dim,size", [(1000, 2, 64, 1000.0), (1000, 2, 128, 1.0), (300, 8, 64, 10000.0)])
def test_a_token_without_a_value(n, group, dim, size, kind):
    print("sink", n, group, dim, size, kind, flush=True)
    (q, k, v), scale, sink = inputs(n, group, dim, kind, size)
    got = clear_call(q.cuda(), k.cuda(), v.cuda(), causal=False, scale=scale)
    s = scale * (q[:, 0].double() @ k[:, 0].double().T)
    p, z = torch.softmax(s, 1), v[:, 0].double()
    half = torch.finfo(TYPES[kind]).eps / 2
    each = torch.clamp(half * p, min=2.0**-32) if kind == "fp16" else half * p
    e = 2.0**-22 * (2 + 42) + 2.0**-24 * (n / 2 + 64)
    want = p @ z
    tol = half * want.abs() + (each + 2 * e * p) @ z.abs() + (2.0**-24 if kind == "fp16" else 2.0**-133)
    for h in range(group):
        assert ((got.out[:, h].cpu().double() - want).abs() <= tol).all()
        assert ((got.lse[:, h].cpu().double() - torch.logsumexp(s, 1)).abs() <= e).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_an_infinite_value_is_seen_however_improbable(kind):
    """Infinite where its probability counts as more than 0, NaN where it counts as 0: never a finite number."""
    print("infinite", kind, flush=True)
    (q, k, v), scale, sink = inputs(700, 2, 64, kind, 1.0)
    at = int(k[:, 0, 0].argmin())
    v[at, 0, 9] = math.inf
    got = clear_call(q.cuda(), k.cuda(), v.cuda(), scale=scale).out.cpu()
    assert not torch.isfinite(got[at:, :, 9]).any() and torch.isfinite(got[:at]).all()
    got[..., 9] = 0
    assert torch.isfinite(got).all()
