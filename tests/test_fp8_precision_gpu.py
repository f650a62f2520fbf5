"""Attention over 8-bit caches: what a row's result may depend on, and how exact its parts are held."""
import pytest
import torch

from tests.test_fp8_cache_gpu import SHAPES, Batch, _attend, _check, _cuda, _far, _to_cache

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------------------------------
# rows of all sizes side by side
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", SHAPES[1:])
@pytest.mark.parametrize("far", [False, True])
def test_a_row_does_not_depend_on_the_size_of_others(cuda_device, lens, qlens, counts, heads, hkv, far):
    """Neighbouring rows and heads that differ by up to 2^40, most of them of usual size."""
    b = Batch(lens, qlens, seed=31 + heads)
    sizes = torch.tensor([1.0, 1e9, 1.0, 1e-3, 1.0, 2.0 ** 10, 1.0, 1.0, 1e6])
    _check(*_attend(b, heads, hkv, counts, q_size=sizes[torch.arange(sum(qlens) * heads) % 9].view(-1, heads, 1), far=far))


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", [SHAPES[1], SHAPES[4], SHAPES[6]])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("far", [False, True])
def test_rows_that_see_nothing_may_hold_any_number(cuda_device, lens, qlens, counts, heads, hkv, cap, far):
    """Rows of empty ranges (padding) near the end of the type's range, in the tiles of rows that see keys."""
    b = Batch(lens, qlens, seed=37)
    size = torch.cat([torch.where(torch.arange(n) % 4 == 3, 1.0, 5e37) for n in qlens])      # as _ranges("empty") has them
    _check(*_attend(b, heads, hkv, counts, "empty", cap=cap, q_size=size.view(-1, 1, 1), far=far))
