"""Calls on 8-bit caches at the borders of what they take (no GPU needed)."""
import pytest

from dyllm_b200 import _lib
from tests.test_fp8_cache import ATTEND


@pytest.mark.parametrize("cap", [5e-7, 4.3e37, 3e38])
def test_caps_whose_quotient_is_no_normal_number_are_refused(cap):
    assert _lib.load().dyllm_attention_salient_rows_fp8(*{**ATTEND, "cap": cap}.values()) == -1
    assert "softcap" in _lib.load().dyllm_last_error().decode()


@pytest.mark.parametrize("args", [(0, 1, 1, 4, 4), (3, 0, 1, 4, 4), (3, 1, 0, 4, 4), (3, 1, 1, 0, 4), (3, 1, 1, 4, 0), (3, 1, 1, 2, 4), (3, 1, 1, 6, 4)])
def test_calls_without_work_and_refused_ones_launch_nothing(args):
    assert _lib.load().dyllm_attention_salient_rows_fp8_launches(*args, 1000, 1) == 0
