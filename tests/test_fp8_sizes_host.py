"""Sizes beyond 32 bits are refused, not taken modulo 2^32 (CPU)."""
from __future__ import annotations

import pytest

pytest.importorskip("torch")


@pytest.mark.parametrize("sizes", [((1 << 32) + 5, 6, 7), (5, (1 << 32) + 6, 7), (5, 6, (1 << 32) + 7), (5, 1 << 31, 7)])
def test_the_workspace_of_a_linear_layer_too_large(fvsr, sizes):
    with pytest.raises(fvsr.FVSRError, match="too large") as e:
        fvsr.linear_fp8_workspace_size(*sizes, False)
    assert e.value.status == fvsr.FVSR_EUNSUPPORTED
