"""Calls on 8-bit caches that the formulas allow and few programs make."""
import pytest
import torch

from tests.test_fp8_cache_gpu import FP8, Batch, _attend, _check, _cuda, _far, _to_cache

pytestmark = pytest.mark.gpu


def test_update_of_rows_behind_the_last_sequence_of_the_batch(cuda_device):
    """The caches go on behind it, with a sequence of another batch: its rows stay, delta-V is zero."""
    from dyllm_b200 import ops

    cache = [(torch.full((12, 128), 2.0).cuda().to(FP8), torch.ones(12, 1).cuda()) for _ in range(2)]
    starts, cu, ids = _cuda(torch.tensor([5, 0, 8]), torch.tensor([0, 3, 6], dtype=torch.int32), torch.tensor([0, 1]))
    rows_k, positions = _cuda(torch.tensor([6, 2, 7, 5, 2 ** 40, 10]), torch.zeros(6, dtype=torch.int64))
    cos_sin = torch.cat([torch.ones(4, 64), torch.zeros(4, 64)], 1).cuda()
    x = torch.full((6, 1, 128), 8.0).bfloat16().cuda()
    dv = ops.fp8_kv_cache_update(x, x, rows_k, positions, None, cos_sin, cu, starts, starts, ids, *cache)
    assert dv[:, 0, 0].tolist() == [0.0, 6.0, 0.0, 6.0, 0.0, 0.0]
    want = torch.full((12,), 2.0)
    want[[7, 2]] = 8.0
    for codes, scales in cache:
        assert torch.equal((codes.float() * scales).cpu(), want.unsqueeze(1).expand(12, 128))


def test_a_bound_of_no_rows_loses_none(cuda_device):
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch([70, 90], [70, 90], seed=53)
    kc, vc = _to_cache(*b.cache(2)), _to_cache(*b.cache(2))
    cu, rows, _ = b.picks([5, 3])
    args = (b.randn(160, 4, 128).bfloat16().cuda(), kc, vc, *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, rows))
    want = attention_salient_rows_fp8(*args, max_rows_per_seq=5)
    out = torch.full_like(want, 7.0)
    assert attention_salient_rows_fp8(*args, max_rows_per_seq=0, out=out) is out
    assert torch.equal(out, want)


def _launches(call):
    """Kernels that a call launches, as a graph holds them."""
    import ctypes

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        call()
    n = ctypes.c_size_t()
    runtime = ctypes.CDLL("libcudart.so.12")
    assert runtime.cudaGraphGetNodes(ctypes.c_void_p(graph.raw_cuda_graph()), None, ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("lens,counts,heads,hkv,ranges,launches", [
    ([300, 64], [5, 3], 4, 2, False, 1),                  # few rows
    ([300, 64], [5, 3], 4, 2, True, 2),                   # and keys per tile
    ([32011, 900], [32, 3], 4, 4, False, 2),              # a tile in many parts: joined by a launch
    ([1500, 900], [200, 90], 4, 2, False, 2),             # many rows
    ([1500, 900], [200, 90], 4, 2, True, 3),
    ([300, 64], [0, 0], 4, 2, False, 1),                  # lists that turn out empty on the device
])
def test_launches_are_counted(cuda_device, lens, counts, heads, hkv, ranges, launches):
    from dyllm_b200 import _lib
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch(lens, [min(n, 400) for n in lens], seed=59)
    kc, vc = _to_cache(*b.cache(hkv)), _to_cache(*b.cache(hkv))
    cu, rows, _ = b.picks(counts)
    total_q = sum(b.qlens)
    rows = torch.cat([rows, torch.zeros(3, dtype=torch.int32)])
    args = (b.randn(total_q, heads, 128).bfloat16().cuda(), kc, vc, *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, rows))
    seen = torch.tensor([[0, 200]], dtype=torch.int32).repeat(total_q, 1).cuda() if ranges else None

    def call():
        return attention_salient_rows_fp8(*args, max_rows_per_seq=max(max(counts), 1), key_ranges=seen)

    assert _launches(call) == launches
    before = _lib.launch_count
    call()
    assert _lib.launch_count - before == launches
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    attention_salient_rows_fp8(*args[:-1], empty, max_rows_per_seq=1)
    assert _lib.launch_count - before == launches


@pytest.mark.parametrize("rows,far", [(2, False), (70, True)])
def test_a_long_sequence_among_many_short_ones(cuda_device, rows, far):
    """Tiles of one unit by the hundred, and between them some that are cut into parts."""
    lens = [100, 1, 0, 90] * 9 + [5003] + [100] * 34
    _check(*_attend(Batch(lens, seed=61), 8, 8, [min(n, rows) for n in lens], far=far))


@pytest.mark.parametrize("rows,far", [(5, False), (90, True)])
@pytest.mark.parametrize("size", [-1e20, -1e13, 1.0, 1e13, 1e20])
def test_a_key_that_is_alone_has_all_the_weight(cuda_device, rows, far, size):
    """However far below zero its score is: rows of a window of one key give that key's value."""
    from dyllm_b200.attention_ops import attention_salient_rows_fp8

    b = Batch([100], [100], seed=67)
    (_, _), (vc, vs) = b.cache(2), b.cache(2)
    kc, ks = torch.ones(b.rows, 2, 128).double(), torch.full((b.rows, 2), 2.0 ** 50).double()
    caches = [_to_cache(*(_far(b, *c) if far else c)) for c in ((kc, ks), (vc, vs))]
    q = torch.full((100, 4, 128), size).bfloat16()
    pos = torch.arange(100, dtype=torch.int32)
    cu, idx = torch.tensor([0, rows], dtype=torch.int32), pos[:rows].flip(0)
    out = attention_salient_rows_fp8(q.cuda(), *caches, *_cuda(b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k, cu, idx), rows,
                                     key_ranges=torch.stack([pos, pos + 1], 1).cuda())
    at = int(b.v_starts[b.ids[0]]) + idx.long()
    want = (vc[at] * vs[at].unsqueeze(-1)).repeat_interleave(2, 1)
    # a weight of 2^12 exactly, over its own sum: the quotient's rounding, and a value that bf16 holds
    assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs()).all())
