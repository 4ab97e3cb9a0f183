"""Refusals of the attention entry points at the ends of what their arguments can say (no GPU needed)."""
import numpy as np
import pytest

import fusedmm_amd as fa
from test_attention_cpu import desc, rows, rows4

NOT_FINITE = [float("nan"), float("inf"), float("-inf")]


@pytest.mark.parametrize("scale", NOT_FINITE)
def test_a_scale_that_is_not_finite(capfd, scale):
    for call in (lambda d: rows(d), lambda d: rows4(d),
                 lambda d: fa.fusedMM_attn_forward(d, None, 16, 16, 16, None, 16, None, None, None, 0, stream=0),
                 lambda d: fa.fusedMM_attn_backward(d, None, None, 16, 16, 16, None, 16, None, 16, 16, 16, 16, 16, None, None, 0, stream=0)):
        assert call(desc(scale=scale)) == fa.FAIL
        assert "scale is not a finite number" in capfd.readouterr().err
