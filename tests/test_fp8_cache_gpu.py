"""8-bit caches on the GPU: written, updated and read bit for bit as defined, and the attention over them against 64 bits."""
import math

import pytest
import torch

from oracle import dyllm_oracle as orc

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _cum(v):
    return torch.tensor([0] + torch.tensor(v).cumsum(0).tolist(), dtype=torch.int32)


class Batch:
    """Sequences of the given lengths in shuffled order in caches with rows of nobody between them; queries = last rows."""

    def __init__(self, lens, qlens=None, seed=0, gap=3):
        g = self.g = torch.Generator().manual_seed(seed)
        n = len(lens)
        qlens = lens if qlens is None else qlens
        self.lens, self.qlens, self.n = lens, qlens, n
        self.cu_k, self.cu_q = _cum(lens), _cum(qlens)
        self.ids = torch.randperm(3 * n + 1, generator=g)[:n]
        self.k_starts, self.v_starts = (torch.full((3 * n + 1,), -1, dtype=torch.int64) for _ in range(2))
        for starts in (self.k_starts, self.v_starts):
            pos = gap
            for b in torch.randperm(n, generator=g).tolist():
                starts[self.ids[b]] = pos
                pos += lens[b] + gap
            self.rows = pos

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.g)

    def cache(self, heads, spread=0.5):
        x = self.randn(self.rows, heads, 128) * torch.exp(spread * self.randn(self.rows, heads, 1))
        code, scale = orc.fp8_quantise(x)
        return code, scale

    def picks(self, counts):
        """Listed rows per sequence: (cu, int32 query rows, int64 key rows)."""
        rows, rows_k = [], []
        for b, m in enumerate(counts):
            at = torch.randperm(self.qlens[b], generator=self.g)[:m].sort().values
            rows.append(at + int(self.cu_q[b]))
            rows_k.append(at + int(self.cu_k[b]) + self.lens[b] - self.qlens[b])
        return _cum([len(r) for r in rows]), torch.cat(rows).int(), torch.cat(rows_k).long()


def _far(b, code, scale):
    """The same cache with rows of nobody behind it: more than 1024 a sequence, so that the call cannot take it for a short one."""
    n = 1025 * b.n
    return torch.cat([code, torch.zeros(n, *code.shape[1:]).double()]), torch.cat([scale, torch.ones(n, scale.size(1)).double()])


def _to_cache(code, scale):
    return code.flatten(1).float().cuda().to(FP8), scale.float().cuda()


def _same(cache, code, scale):
    codes, scales = cache
    assert torch.equal(codes.cpu().float().view_as(code).double(), code)
    assert torch.equal(torch.nan_to_num(scales.cpu().double(), nan=-1.0), torch.nan_to_num(scale.double(), nan=-1.0))


def _cuda(*ts):
    return [t.cuda() for t in ts]


def _values_with_edges(b, rows, heads):
    x = (b.randn(rows, heads, 128) * torch.exp(2.0 * b.randn(rows, heads, 1))).bfloat16()
    if rows > 3:
        x[0] = 0.0
        x[1, 0] = 1e-30                                              # below the smallest scale's steps
        x[2, -1, 17] = float("nan")
        x[3, 0, 100] = float("-inf")
        x[rows // 2] = 448.0
        x[rows - 1, 0] = 3.0e38
    return x


LENS = [([1], 1), ([5, 1, 0, 33], 3), ([130, 257], 32), ([64] * 9, 4), ([700], 5)]


@pytest.mark.parametrize("lens,heads", LENS)
@pytest.mark.parametrize("block", [False, True])
@pytest.mark.parametrize("sliced", [False, True])
def test_write_and_read(cuda_device, lens, heads, block, sliced):
    from dyllm_b200 import ops

    b = Batch(lens, [v // 2 for v in lens] if block else None, seed=heads)
    total = sum(b.qlens)
    code, scale = b.cache(heads)
    cache = _to_cache(code, scale)
    x = _values_with_edges(b, total, heads)
    xd = x.cuda()
    if sliced:      # the second half of a fused product
        xd = torch.cat([torch.full_like(xd, 7.0), xd], 1)[:, heads:]
    starts, cu_q, cu_k, ids = _cuda(b.k_starts, b.cu_q, b.cu_k, b.ids)
    k = cu_k if block else None
    ops.fp8_cache_write(xd, *cache, starts, cu_q, ids, cu_seqlens_k=k)
    orc.fp8_cache_write(code, scale, x, b.k_starts, b.cu_q, b.ids, b.cu_k if block else None)
    _same(cache, code, scale)
    out = torch.full((total + 2, heads, 128), 9.0, dtype=torch.bfloat16, device="cuda")
    got = ops.fp8_cache_read(*cache, starts, cu_q, ids, total + 2, cu_seqlens_k=k, out=out)
    assert got is out and bool((out[total:] == 9.0).all())
    want = orc.fp8_cache_read(code, scale, b.k_starts, b.cu_q, b.ids, b.cu_k if block else None)
    assert torch.equal(torch.nan_to_num(out[:total].cpu().double(), nan=-5.0), torch.nan_to_num(want, nan=-5.0))
    fresh = ops.fp8_cache_read(*cache, starts, cu_q, ids, total, cu_seqlens_k=k)
    assert torch.equal(torch.nan_to_num(fresh, nan=-5.0), torch.nan_to_num(out[:total], nan=-5.0))


def test_rows_outside_the_cache_are_not_written_and_read_as_zeros(cuda_device):
    from dyllm_b200 import ops

    heads = 2
    codes = torch.full((10, 256), 1.0).cuda().to(FP8)
    scales = torch.ones(10, heads).cuda()
    starts, cu, ids = _cuda(torch.tensor([-1, 8, 0]), torch.tensor([0, 2, 6, 7], dtype=torch.int32), torch.tensor([0, 1, 2]))
    x = torch.full((7, heads, 128), 3.0).bfloat16().cuda()
    ops.fp8_cache_write(x, codes, scales, starts, cu, ids)              # two rows of nobody, two in and two behind the cache, one
    got = codes.float()
    assert bool((got[1:8] == 1.0).all()) and bool((scales[1:8] == 1.0).all())
    assert bool((got[[0, 8, 9]] * scales[[0, 8, 9]].repeat_interleave(128, 1) == 3.0).all())
    out = ops.fp8_cache_read(codes, scales, starts, cu, ids, 7)
    assert out[:, 0, 0].tolist() == [0.0, 0.0, 3.0, 3.0, 0.0, 0.0, 3.0]


UPDATES = [([40], [40], [1], 4), ([64, 1, 300, 20], [64, 1, 100, 20], [9, 1, 0, 20], 3), ([512] * 5, [128] * 5, [31, 0, 64, 5, 17], 32)]


@pytest.mark.parametrize("lens,qlens,counts,heads", UPDATES)
@pytest.mark.parametrize("live", [None, 0, 7])
def test_update(cuda_device, lens, qlens, counts, heads, live):
    from dyllm_b200 import ops

    b = Batch(lens, qlens, seed=heads + len(lens))
    cu, rows, rows_k = b.picks(counts)
    n = len(rows)
    kc, ks = b.cache(heads)
    vc, vs = b.cache(heads)
    k_cache, v_cache = _to_cache(kc, ks), _to_cache(vc, vs)
    fused = torch.cat([_values_with_edges(b, n, heads), _values_with_edges(b, n, heads)], 1)
    k_new, v_new = fused[:, :heads], fused[:, heads:]
    positions = torch.cat([torch.arange(a - q, a) for a, q in zip(lens, qlens)])
    angle = torch.outer(torch.arange(400).double(), 10000.0 ** (-torch.arange(64).double() / 64))
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    positions[0] = 10 ** 6                                              # clamped to the table
    fd = fused.cuda()
    pos_idx = rows.long()
    args = _cuda(rows_k, positions, pos_idx, cos_sin, b.cu_k, b.k_starts, b.v_starts, b.ids)
    dv = torch.full((n, heads, 128), 5.0, dtype=torch.bfloat16, device="cuda")
    count = None if live is None else torch.tensor([live], dtype=torch.int32, device="cuda")
    got = ops.fp8_kv_cache_update(fd[:, :heads], fd[:, heads:], *args, k_cache, v_cache, num_rows_dev=count, dv=dv)
    m = n if live is None else min(live, n)
    want = orc.fp8_kv_cache_update(k_new[:m], v_new[:m], rows_k[:m], positions.clamp(0, 399), pos_idx[:m], cos_sin, b.cu_k, b.k_starts,
                                   b.v_starts, b.ids, kc, ks, vc, vs)
    _same(k_cache, kc, ks)
    _same(v_cache, vc, vs)
    assert got is dv and bool((dv[m:] == 5.0).all())
    # the difference of two four-bit numbers, rounded to fp32 (exact unless the scales are far apart), then to bf16
    assert torch.equal(torch.nan_to_num(dv[:m].cpu(), nan=-5.0), torch.nan_to_num(want.float().bfloat16(), nan=-5.0))
    # the same rows once more: nothing changes, and nothing is added to a context
    again = ops.fp8_kv_cache_update(fd[:, :heads], fd[:, heads:], *args, k_cache, v_cache, num_rows_dev=count)
    assert bool((torch.nan_to_num(again[:m], nan=0.0) == 0).all())
    _same(v_cache, vc, vs)


def test_update_of_rows_that_no_cache_holds(cuda_device):
    from dyllm_b200 import ops

    cache = [(torch.full((6, 128), 2.0).cuda().to(FP8), torch.ones(6, 1).cuda()) for _ in range(2)]
    starts, cu, ids = _cuda(torch.tensor([-1, 4]), torch.tensor([0, 3, 7], dtype=torch.int32), torch.tensor([0, 1]))
    rows_k, positions = _cuda(torch.tensor([1, 4, 6]), torch.tensor([0, 0, 0]))      # no start; row 5; row 7 of 6
    cos_sin = torch.cat([torch.ones(4, 64), torch.zeros(4, 64)], 1).cuda()
    x = torch.full((3, 1, 128), 8.0).bfloat16().cuda()
    dv = ops.fp8_kv_cache_update(x, x, rows_k, positions, None, cos_sin, cu, starts, starts, ids, *cache)
    assert dv[:, 0, 0].tolist() == [0.0, 6.0, 0.0]
    for codes, scales in cache:
        value = codes.float() * scales
        assert bool((value[:5] == 2.0).all()) and bool((value[5] == 8.0).all())


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def _ranges(kind, b, g):
    got = []
    for length, q in zip(b.lens, b.qlens):
        pos = torch.arange(length - q, length)
        if kind == "prefix":
            got.append(torch.stack([torch.zeros_like(pos), (pos // 16 + 1) * 16], 1))           # past the end: cut
        elif kind == "window":
            got.append(torch.stack([pos - 9, pos + 10], 1))                                     # below zero: cut
        elif kind == "empty":
            r = torch.stack([pos * 0, pos * 0 + length], 1)
            r[::2] = torch.tensor([5, 5])
            r[1::4] = torch.tensor([2 ** 31 - 1, -2 ** 31])
            got.append(r)
        elif kind == "extremes":
            ends = torch.tensor([[-2 ** 31, length // 2], [0, -2 ** 31], [-2 ** 31, 2 ** 31 - 1], [length // 3, 2 ** 31 - 1]])
            got.append(ends[torch.arange(q) % 4])
        else:
            a = torch.randint(0, max(length, 1), (q,), generator=g)
            got.append(torch.stack([a, a + torch.randint(0, length + 2, (q,), generator=g)], 1))
    return torch.cat(got).int()


def _attend(b, heads, hkv, counts, mask=None, cap=0.0, slopes=False, scale=None, seed=0, q_size=1.0, spread=0.5, sliced=False,
            most=None, edit=None, far=False):
    from dyllm_b200 import _lib
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    cu, rows, _ = b.picks(counts)
    total_q = sum(b.qlens)
    q = (b.randn(total_q, heads, 128) * q_size).bfloat16()
    (kc, ks), (vc, vs) = b.cache(hkv, spread), b.cache(hkv, spread)
    if edit:
        edit(b, kc, ks, vc, vs)
    if far:
        (kc, ks), (vc, vs) = _far(b, kc, ks), _far(b, vc, vs)
    ranges = None if mask is None else _ranges(mask, b, b.g)
    slope = 2.0 ** -torch.arange(1, heads + 1).float() if slopes else None
    qd = q.cuda()
    if sliced:
        qd = torch.cat([qd, torch.full_like(qd, float("nan"))], 1)[:, :heads]
    n = len(rows)
    out = torch.full((n + 3, heads, 128), 11.0, dtype=torch.bfloat16, device="cuda")
    dev = _cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu)
    pad = torch.cat([rows, torch.full((3,), 2 ** 30, dtype=torch.int32)]).cuda()               # capacity above the live count
    most = max(max(counts), 1) if most is None else most

    def run(o):
        return attention_salient_rows_fp8(qd, _to_cache(kc, ks), _to_cache(vc, vs), *dev, pad, max_rows_per_seq=most, scale=scale,
                                          softcap=cap, slopes=None if slope is None else slope.cuda(),
                                          key_ranges=None if ranges is None else ranges.cuda(), out=o)

    assert run(out) is out
    assert _lib.load().dyllm_device_status() == 0
    assert bool((out[n:] == 11.0).all())
    again = run(torch.full_like(out, 11.0))
    assert torch.equal(torch.nan_to_num(again, nan=-5.0), torch.nan_to_num(out, nan=-5.0))      # run to run the same bits
    k = orc.fp8_cache_read(kc, ks, b.k_starts, b.cu_k, b.ids)
    v = orc.fp8_cache_read(vc, vs, b.v_starts, b.cu_k, b.ids)
    want, mag, big, floor = orc.attention_rows_fp8(q, k, v, b.cu_q, b.cu_k, cu, rows, scale, cap, slope, ranges)
    return out[:n].cpu().double(), want, mag, big, floor, cap


def _check(got, want, mag, big, floor, cap):
    """Half a step of bf16 for the result (2^-8).

    A weight w (within 2^2.8 of its row's largest, 1, the values' scales included) is taken as 64 w in half precision (2^-11) and
    split into e4m3 and what that leaves, |r| <= 2^-4 of it (half a step), in e5m2, rounded by 2^-3 of itself: off by at most
    (2^-7 + 2^-11) w, or by half a step of the smallest numbers, 2^-17 / 64 <= 2^-22.  The first moves the result by as much of
    sum(weight * |v|); the second by 2^-22 of the largest weight for each key, times its codes, which are at most twice the largest
    of the heaviest key.

    The score is a sum of 128 products in fp32 (2^-24 a term, 2^-17 in all) of queries that are exact above 2^-18 of their row's
    largest and off by 2^-26 of it below, times a scale, capped and biased (a few 2^-24 of the cap and the bias): 2^-16 of what
    it is made of, which moves weights and sum by as much, relatively.  Exponential and quotient: 2^-20."""
    delta = 2.0 ** -16 * (big + cap).unsqueeze(-1)
    tol = 2.0 ** -8 * want.abs() + (2.0 ** -7 + 2.0 ** -11 + 2.0 ** -20 + 2 * delta) * mag + 2.0 ** -21 * floor.unsqueeze(-1) + 1e-30
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got - want).abs() / tol).nan_to_num().max()))


SHAPES = [
    ([1], [1], [1], 1, 1),                                      # one token
    ([300], [300], [3], 2, 2),
    ([17, 1, 64, 33, 5], [17, 1, 10, 33, 5], [5, 1, 0, 33, 2], 4, 2),
    ([129, 31, 32, 128, 127, 0], [20, 5, 32, 7, 6, 0], [16, 5, 17, 1, 0, 0], 7, 1),      # seven queries a key head, no keys at all
    ([513, 260], [100, 200], [70, 40], 6, 3),
    ([1500], [64], [40], 8, 2),
    ([700, 90], [700, 90], [400, 90], 2, 2),
]


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", SHAPES)
@pytest.mark.parametrize("mask", [None, "prefix", "window", "empty", "random"])
@pytest.mark.parametrize("far", [False, True])
def test_attention(cuda_device, lens, qlens, counts, heads, hkv, mask, far):
    _check(*_attend(Batch(lens, qlens, seed=len(lens) + heads), heads, hkv, counts, mask, far=far))


@pytest.mark.parametrize("counts", [[10, 2, 7], [40, 2, 33]])                              # pairs: 20, 80 a sequence and key head
@pytest.mark.parametrize("mask,slopes", [(None, False), (None, True), ("prefix", False), ("random", True)])
def test_attention_of_sequences_that_many_ctas_hold(cuda_device, counts, mask, slopes):
    """Hundreds of parts, joined in their order; a short sequence between long ones."""
    _check(*_attend(Batch([20011, 5, 9000], [64, 5, 300], seed=13), 4, 2, counts, mask, slopes=slopes))


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", SHAPES[2:])
@pytest.mark.parametrize("far", [False, True])
def test_attention_with_ranges_at_the_ends_of_their_type(cuda_device, lens, qlens, counts, heads, hkv, far):
    _check(*_attend(Batch(lens, qlens, seed=11), heads, hkv, counts, "extremes", far=far))


@pytest.mark.parametrize("lens,qlens,counts,heads,hkv", SHAPES[1:6])
@pytest.mark.parametrize("mask,cap,slopes,scale,sliced", [
    (None, 20.0, False, None, False), (None, 0.0, True, None, True), ("prefix", 30.0, True, 0.2, True), (None, 5.0, False, -0.1, False),
    (None, 0.0, False, 0.0, False),
])
@pytest.mark.parametrize("far", [False, True])
def test_attention_scores(cuda_device, lens, qlens, counts, heads, hkv, mask, cap, slopes, scale, sliced, far):
    _check(*_attend(Batch(lens, qlens, seed=7), heads, hkv, counts, mask, cap, slopes, scale, sliced=sliced, far=far))


@pytest.mark.parametrize("heads,hkv,counts", [(4, 4, [6, 20]), (8, 2, [9, 30]), (2, 1, [100, 70])])
@pytest.mark.parametrize("q_size,spread", [(8.0, 3.0), (1e-3, 0.0), (1e4, 0.5), (30.0, 6.0)])
@pytest.mark.parametrize("far", [False, True])
def test_attention_with_peaked_scores_and_values_of_all_sizes(cuda_device, heads, hkv, counts, q_size, spread, far):
    _check(*_attend(Batch([400, 333], [200, 100], seed=3), heads, hkv, counts, q_size=q_size, spread=spread,
                    scale=128 ** -0.5 / max(q_size / 8.0, 1.0), far=far))


@pytest.mark.parametrize("counts", [[3, 5], [60, 90]])
@pytest.mark.parametrize("most", [1, 1000])
@pytest.mark.parametrize("far", [False, True])
def test_the_bound_of_listed_rows_only_chooses_kernels(cuda_device, counts, most, far):
    _check(*_attend(Batch([210, 340], [100, 340], seed=5), 4, 2, counts, most=most, far=far))


@pytest.mark.parametrize("counts", [[4], [100]])
@pytest.mark.parametrize("far", [False, True])
def test_nan_of_unseen_keys_stays_unseen(cuda_device, counts, far):
    """Keys 20.. of the sequence hold NaN in K or V; the rows of a window that ends before them are finite, the others NaN."""
    def edit(b, kc, ks, vc, vs):
        k0, v0 = int(b.k_starts[b.ids[0]]), int(b.v_starts[b.ids[0]])
        kc[k0 + 150], ks[k0 + 150] = 0.0, math.nan
        vc[v0 + 170], vs[v0 + 170] = 0.0, math.nan

    got, want, mag, big, floor, cap = _attend(Batch([200], [200], seed=2), 2, 2, counts, "window", edit=edit, far=far)
    bad = torch.isnan(got).any(-1).any(-1)
    assert bool(bad.any()) == bool(torch.isnan(want).any()) and not bool(bad.all())
    fine = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~fine)
    _check(got.masked_fill(~fine, 0), want.masked_fill(~fine, 0), mag.nan_to_num(), big.nan_to_num(), floor.nan_to_num(), cap)


@pytest.mark.parametrize("counts", [[4], [100]])
@pytest.mark.parametrize("gap", [150, 1100])
def test_rows_of_nobody_may_hold_any_byte(cuda_device, counts, gap):
    """Rows between the sequences are never part of a result, be they NaN codes (an arena comes uninitialised)."""
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch([133], [133], seed=4, gap=gap)
    cu, rows, _ = b.picks(counts)
    (kc, ks), (vc, vs) = b.cache(2), b.cache(2)
    q = b.randn(133, 2, 128).bfloat16().cuda()
    outs = []
    for byte in (0x00, 0x7f, 0xff):
        caches = []
        for code, scale, starts in ((kc, ks, b.k_starts), (vc, vs, b.v_starts)):
            codes, scales = _to_cache(code, scale)
            own = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
            own[int(starts[b.ids[0]]):int(starts[b.ids[0]]) + 133] = True
            codes.view(torch.uint8)[~own] = byte
            scales[~own] = math.nan if byte else 0.0
            caches.append((codes, scales))
        outs.append(attention_salient_rows_fp8(q, *caches, *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, rows),
                                               max_rows_per_seq=max(counts)))
    assert bool(torch.isfinite(outs[0]).all())
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("times,far", [(1, False), (30, False), (30, True)])
def test_sequences_without_a_cache_and_rows_out_of_range_give_zeros(cuda_device, times, far):
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch([40, 50], seed=6)
    (kc, ks), (vc, vs) = b.cache(2), b.cache(2)
    if far:
        (kc, ks), (vc, vs) = _far(b, kc, ks), _far(b, vc, vs)
    q = b.randn(90, 4, 128).bfloat16().cuda()
    b.v_starts[b.ids[1]] = -1
    cu, rows = torch.tensor([0, 3 * times, 5 * times], dtype=torch.int32), torch.tensor([0, -4, 90] * times + [41, 60] * times, dtype=torch.int32)
    out = torch.full((5 * times, 4, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    attention_salient_rows_fp8(q, _to_cache(kc, ks), _to_cache(vc, vs), *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, rows),
                               max_rows_per_seq=3 * times, out=out)
    there = torch.zeros(5 * times, dtype=torch.bool)
    there[0 : 3 * times : 3] = True
    assert bool((out[there.cuda()] != 0).any(-1).all()) and bool((out[~there.cuda()] == 0).all())


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("most", [3, 60])
def test_attention_of_a_batch_of_more_than_a_warps_sequences(cuda_device, most, far):
    g = torch.Generator().manual_seed(21)
    lens = torch.randint(0, 300, (75,), generator=g).tolist()
    counts = [min(n, int(torch.randint(0, most + 1, (1,), generator=g))) for n in lens]
    _check(*_attend(Batch(lens, seed=21), 4, 2, counts, far=far))
    _check(*_attend(Batch(lens, seed=22), 4, 2, counts, "window", far=far))


@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("heads,hkv", [(160, 1), (66, 2), (33, 33)])
def test_attention_of_more_heads_than_a_tile_has_rows(cuda_device, heads, hkv, far):
    _check(*_attend(Batch([70, 3, 140], seed=17), heads, hkv, [2, 1, 3], "prefix", far=far))


@pytest.mark.parametrize("far", [False, True])
def test_a_replayed_call_follows_the_lists(cuda_device, far):
    """Captured with lists of one length and replayed with others: counts, rows and sequences are read on the device."""
    from dyllm_b200 import ops
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch([500, 90, 333], [200, 90, 100], seed=19)
    total_q, heads, hkv = sum(b.qlens), 6, 2
    caches = [_to_cache(*(_far(b, *c) if far else c)) for c in (b.cache(hkv), b.cache(hkv))]
    q = b.randn(total_q, heads, 128).bfloat16().cuda()
    ks, vs, ids, cu_q, cu_k = _cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k)
    k_new, v_new = (b.randn(total_q, hkv, 128).bfloat16().cuda() for _ in range(2))
    angle = torch.outer(torch.arange(600).double(), 10000.0 ** (-torch.arange(64).double() / 64))
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).float().cuda()
    cu, rows = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(total_q, dtype=torch.int32, device="cuda")
    rows_k, count = torch.zeros(total_q, dtype=torch.int64, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    positions = torch.arange(total_q, device="cuda")

    def fill(counts):
        c, r, rk = b.picks(counts)
        cu.copy_(c)
        rows[: len(r)], rows_k[: len(rk)] = r.cuda(), rk.cuda()
        count.fill_(len(r))

    def run(caches):
        dv = torch.zeros_like(v_new)
        ops.fp8_kv_cache_update(k_new, v_new, rows_k, positions, None, cos_sin, cu_k, ks, vs, ids, *caches, num_rows_dev=count, dv=dv)
        out = torch.zeros(total_q, heads, 128, dtype=torch.bfloat16, device="cuda")
        attention_salient_rows_fp8(q, *caches, ks, vs, ids, cu_q, cu_k, cu, rows, max_rows_per_seq=200, out=out)
        return dv, out, ops.fp8_cache_read(*caches[0], ks, cu_k, ids, sum(b.lens))

    def copy():
        return [tuple(t.clone() for t in c) for c in caches]

    fill([3, 1, 2])
    run(copy())
    torch.cuda.synchronize()
    mine = copy()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(mine)
    for counts in ([3, 1, 2], [200, 90, 100], [0, 0, 0], [0, 17, 1], [150, 0, 0], [1, 1, 1]):
        fill(counts)
        for m, c in zip(mine, caches):
            for x, y in zip(m, c):
                x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(got, run(copy())):
            assert torch.equal(x, y)


def test_calls_from_two_threads_on_two_streams(cuda_device):
    import threading

    from dyllm_b200 import _lib
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    jobs, results = [], {}
    for n, counts in enumerate(([9, 4], [130, 90])):
        b = Batch([300, 1500], [300, 200], seed=23 + n)
        kc, vc = _to_cache(*b.cache(2)), _to_cache(*b.cache(2))
        cu, rows, _ = b.picks(counts)
        args = (b.randn(500, 4, 128).bfloat16().cuda(), kc, vc, *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, rows), max(counts))
        jobs.append((args, attention_salient_rows_fp8(*args)))
    torch.cuda.synchronize()

    def work(n):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            results[n] = [attention_salient_rows_fp8(*jobs[n][0]) for _ in range(40)]
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert _lib.load().dyllm_device_status() == 0
    for n, (_, want) in enumerate(jobs):
        assert len(results[n]) == 40 and all(torch.equal(got, want) for got in results[n])


@pytest.mark.parametrize("listed", [3, 200])
def test_caches_without_rows_and_batches_without_queries(cuda_device, listed):
    """An arena that holds nobody yet: nothing is written, everything reads as zeros; lists of a batch that has no query rows."""
    from dyllm_b200 import _lib, ops
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    cache = torch.empty(0, 256, device="cuda").to(FP8), torch.empty(0, 2, device="cuda")
    starts, ids, cu = _cuda(torch.tensor([0, -1]), torch.tensor([0, 1]), torch.tensor([0, listed, listed + 2], dtype=torch.int32))
    x = torch.ones(listed + 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    ops.fp8_cache_write(x, *cache, starts, cu, ids)
    assert bool((ops.fp8_cache_read(*cache, starts, cu, ids, listed + 2) == 0).all())
    rows = torch.arange(listed + 2, device="cuda")
    dv = ops.fp8_kv_cache_update(x, x, rows, rows, None, torch.ones(listed + 2, 128, device="cuda"), cu, starts, starts, ids, cache, cache)
    assert bool((dv == 0).all())
    for q in (x, x[:0]):
        out = torch.full_like(x, 5.0)
        got = attention_salient_rows_fp8(q, cache, cache, starts, starts, ids, cu if len(q) else cu * 0, cu, cu, rows.int(), listed, out=out)
        assert got is out and bool((out == 0).all())
    assert _lib.load().dyllm_device_status() == 0


def test_python_refusals(cuda_device):
    from dyllm_b200 import ops
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.zeros(8, 256, device="cuda").to(FP8), torch.zeros(8, 2, device="cuda")
    cu, ids = torch.tensor([0, 4], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    for bad, text in ((x.float(), "bfloat16"), (x[0], "3-D"), (x.transpose(0, 1), "contiguous"), (x[..., ::2], "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            ops.fp8_cache_write(bad, codes, scales, ids, cu, ids)
    for c, s in ((codes.view(torch.uint8), scales), (codes[:, :128], scales), (codes, scales.double()), (codes, scales[:4]),
                 (codes.float(), scales), (codes, scales.t())):
        with pytest.raises(RuntimeError):
            ops.fp8_cache_write(x, c, s, ids, cu, ids)
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        ops.fp8_cache_write(x, codes, scales, ids, cu[:1], ids)
    with pytest.raises(RuntimeError, match="int64"):
        ops.fp8_cache_write(x, codes, scales, ids.int(), cu, ids)
    with pytest.raises(RuntimeError, match="out"):
        ops.fp8_cache_read(codes, scales, ids, cu, ids, 4, out=x[:3])
    table = torch.zeros(4, 128, device="cuda")
    rows = torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="an entry per"):
        ops.fp8_kv_cache_update(x, x, rows[:3], rows, None, table, cu, ids, ids, ids, (codes, scales), (codes, scales))
    with pytest.raises(RuntimeError, match="same shape"):
        ops.fp8_kv_cache_update(x, x[:3], rows, rows, None, table, cu, ids, ids, ids, (codes, scales), (codes, scales))
    with pytest.raises(RuntimeError, match="128"):
        ops.fp8_kv_cache_update(x, x, rows, rows, None, table[:, :64].contiguous(), cu, ids, ids, ids, (codes, scales), (codes, scales))
    idx = torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(q=x, k_cache=(codes, scales), v_cache=(codes, scales), k_seq_starts=ids, v_seq_starts=ids, seq_ids=ids, cu_seqlens_q=cu,
                cu_seqlens_k=cu, cu_salientlens=cu, idx_salient_row=idx, max_rows_per_seq=2)
    for change, text in ((dict(q=x.float()), "bfloat16"), (dict(idx_salient_row=idx.long()), "int32"), (dict(slopes=torch.ones(3, device="cuda")), "slopes"),
                         (dict(key_ranges=torch.zeros(4, 3, dtype=torch.int32, device="cuda")), "key_ranges"), (dict(num_salient=3), "num_salient"),
                         (dict(cu_salientlens=cu[:1]), "cu_salientlens"), (dict(out=x[:1]), "out"), (dict(softcap=-1.0), "softcap"),
                         (dict(key_ranges=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), "key_ranges"),
                         (dict(q=torch.zeros(4, 3, 128, dtype=torch.bfloat16, device="cuda")), "multiple")):
        with pytest.raises(RuntimeError, match=text):
            attention_salient_rows_fp8(**{**good, **change})
