"""Calls on 8-bit caches at the borders of what they take (no GPU needed)."""
import pytest

from dyllm_b200 import _lib
from tests.test_fp8_cache import ATTEND


@pytest.mark.parametrize("cap", [5e-7, 4.3e37, 3e38])
def test_caps_whose_quotient_is_no_normal_number_are_refused(cap):
    assert _lib.load().dyllm_attention_salient_rows_fp8(*{**ATTEND, "cap": cap}.values()) == -1
    assert "softcap" in _lib.load().dyllm_last_error().decode()
