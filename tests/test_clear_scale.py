"""The scale of the cleartext attention's scores: what is beyond 2^126 or none in 32 bits is refused (no GPU needed)."""

import pytest

from holmes_amd import _native as nat

from .test_clear import attend


@pytest.mark.parametrize("scale", [2.4e38, 3.0e38, 2.0**126 * (1 + 2.0**-23), -0.0, 1e-46])
def test_refused(scale):
    assert attend(scale=scale) == attend(scale=scale, tokens=0, seqs=0) == nat.HCK_ERR_ARG


@pytest.mark.parametrize("scale", [2.0**126, 2.0**-126, 1.0])
def test_taken(scale):
    assert attend(scale=scale, tokens=0, seqs=0) == 0   # nothing to do
