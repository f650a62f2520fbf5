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


# ---------------------------------------------------------------------------------------------------------------------
# the weights
# ---------------------------------------------------------------------------------------------------------------------
def _check_weights(got, want, mag, big, floor, cap):
    """Half a step of bf16 for the result (2^-8), half a step of half precision for each weight (2^-11, so as much of the
    weighted sum of magnitudes).  The largest weight of a row is taken as 2^12 or more, and numbers down to 2^-6 are held as the
    half-precision numbers that they are; a smaller one is off by at most a step of the smallest codes, 2^-16, 2^-28 of the
    largest weight, times codes that are at most twice the largest of the heaviest key.  Scores as in ``_check``."""
    delta = 2.0 ** -16 * (big + cap).unsqueeze(-1)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -20 + 2 * delta) * mag + 2.0 ** -27 * floor.unsqueeze(-1) + 1e-30
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol).max()))


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", SHAPES)
@pytest.mark.parametrize("far", [False, True])
def test_weights_are_held_in_half_precision(cuda_device, lens, qlens, counts, heads, hkv, far):
    _check_weights(*_attend(Batch(lens, qlens, seed=41), heads, hkv, counts, far=far))
    _check_weights(*_attend(Batch(lens, qlens, seed=43), heads, hkv, counts, q_size=4.0, spread=2.0, far=far))


@pytest.mark.parametrize("rows,cache_rows", [(20, 2001), (100, 30000)])
def test_many_keys_of_small_weights_beside_a_heavy_one(cuda_device, rows, cache_rows):
    """One key, and 2000 that are alike, each with 2^-14 to 2^-19 of its weight: what is lost in each of them adds up.  (As many
    batch entries and heads as keep the tiles in one piece: a part has its own largest weight.)"""
    from dyllm_b200.attention_ops import attention_salient_rows_fp8
    from tests.test_fp8_cache_gpu import FP8, _cum

    n, batch, heads = 2001, 20, 32
    k, v = (torch.zeros(cache_rows, heads, 128, device="cuda") for _ in range(2))
    k[0, :, 0] = 8.0
    v[0, :, :64] = 1.0
    v[1:n, :, 64:] = 1.0
    caches = [(t.flatten(1).to(FP8), torch.ones(cache_rows, heads, device="cuda")) for t in (k, v)]
    q = torch.zeros(rows, heads, 128).bfloat16()
    q[:, :, 0] = torch.linspace(9.7, 13.2, rows * heads).view(rows, heads).div(8.0).bfloat16()
    starts = torch.zeros(batch, dtype=torch.int64)      # every entry of the batch has the same rows of the cache
    cu, idx = _cum([rows] * batch), torch.arange(rows * batch, dtype=torch.int32)
    out = attention_salient_rows_fp8(q.repeat(batch, 1, 1).cuda(), *caches, *_cuda(starts, starts, torch.arange(batch), cu, _cum([n] * batch), cu, idx),
                                     max_rows_per_seq=rows, scale=1.0)
    tail = (n - 1) * torch.exp(-8.0 * q[:, :, 0].double())
    want = torch.stack([1 / (1 + tail), tail / (1 + tail)], -1).repeat_interleave(64, -1)
    # bf16 2^-8; half precision 2^-11 of each weight; scores below 32 in powers of two, rounded four times to 2^-20, under 2^-18;
    # a sum in fp32 in chains of 32 terms a warp or 2001 / 2 a thread: 2^-14
    tol = (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -18 + 2.0 ** -14) * want
    err = (out.view(batch, rows, heads, 128).cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / want).max())


# ---------------------------------------------------------------------------------------------------------------------
# capped scores
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", [SHAPES[1], SHAPES[4], SHAPES[6]])
@pytest.mark.parametrize("cap,q_size", [(1e-6, 1.0), (0.5, 1.0), (5.0, 3.0), (50.0, 8.0), (1e4, 3.0), (1e6, 3.0), (1e9, 3.0), (1e30, 3.0), (4e37, 3.0)])
@pytest.mark.parametrize("far", [False, True])
def test_a_cap_of_any_size_costs_its_scores_no_digits(cuda_device, lens, qlens, counts, heads, hkv, cap, q_size, far):
    """The bound of a score's error is that of the score: the cap takes no part (tanh by itself: 2^-18 of the score)."""
    got, want, mag, big, floor, _ = _attend(Batch(lens, qlens, seed=47), heads, hkv, counts, cap=cap, q_size=q_size, far=far)
    _check(got, want, mag, big, floor, 0.0)


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", [SHAPES[1], SHAPES[3], SHAPES[6]])
@pytest.mark.parametrize("mask", [None, "empty"])
@pytest.mark.parametrize("far", [False, True])
def test_a_query_without_numbers_is_alone_with_that(cuda_device, lens, qlens, counts, heads, hkv, mask, far):
    """A head of a row with a NaN or an infinity gives NaN (zeros where it sees no key); rows and heads beside it are as ever."""
    size = torch.ones(sum(qlens) * heads)
    size[2::5], size[3::11] = float("inf"), float("nan")
    got, want, mag, big, floor, cap = _attend(Batch(lens, qlens, seed=71), heads, hkv, counts, mask, q_size=size.view(-1, heads, 1), far=far)
    assert not bool(torch.isnan(want).all())      # of three listed rows none may be such a one
    fine = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~fine)
    _check(got.masked_fill(~fine, 0), want.masked_fill(~fine, 0), mag.nan_to_num(), big.nan_to_num(posinf=0.0), floor.nan_to_num(), cap)
