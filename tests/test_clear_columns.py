"""The widest table of the cleartext attention (no GPU needed)."""

import pytest

from holmes_amd import _native as nat

from .test_clear import attend


@pytest.mark.parametrize("dim", [64, 128])
def test_columns(dim):
    """2^24 columns of 128 tokens are 2^31: numbers that a 32-bit integer does not hold."""
    assert attend(cols=1 << 24, dim=dim) == nat.HCK_ERR_ARG
    assert nat.lib().hck_kv4_attend_workspace_bytes(1, 1, 1, 1, dim, 1, 1 << 24) == 0
    need = nat.lib().hck_kv4_attend_workspace_bytes(1, 1, 1, 1, dim, 1, (1 << 24) - 1)
    assert need > 0 and attend(cols=(1 << 24) - 1, dim=dim) == nat.HCK_ERR_WORKSPACE
