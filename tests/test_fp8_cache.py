"""8-bit caches without a GPU: the definition in 64 bits, and the refusals of the entry points (all of them come before any
CUDA call)."""
import pytest
import torch

from dyllm_b200 import _lib, attention_ops, ops
from oracle import dyllm_oracle as orc

SOME = 1 << 20          # an address that is only looked at


def test_e4m3_grid_is_the_types_grid():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn)
    assert torch.equal(codes.double(), torch.from_numpy(orc.E4M3))


@pytest.mark.parametrize("size", [1.0, 448.0, 3e-30, 1e30, 0.0])
def test_quantised_values_are_the_nearest_of_the_grid(size):
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(64, 128, generator=g) * size).bfloat16()
    x[3], x[4, 7], x[5] = 0.0, 448.0, 448.0 * 2.0 ** 3
    code, scale = orc.fp8_quantise(x)
    assert torch.equal(code, (x.double() / scale.unsqueeze(-1)).float().to(torch.float8_e4m3fn).double())
    amax = x.double().abs().amax(-1)
    assert bool((amax <= 448 * scale).all())
    assert bool(((amax > 224 * scale) | (scale == 2.0 ** -60)).all())
    # half a step of e4m3, relative above the subnormals, absolute in them
    err = (code * scale.unsqueeze(-1) - x.double()).abs()
    assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, scale.unsqueeze(-1) * 2.0 ** -10)).all())


def test_a_head_with_a_nan_or_an_infinity_reads_as_nan():
    x = torch.ones(3, 2, 128)
    x[1, 0, 5], x[2, 1, 9] = float("inf"), float("nan")
    code, scale = orc.fp8_quantise(x)
    assert bool(torch.isnan(scale)[1, 0]) and bool(torch.isnan(scale)[2, 1]) and int(torch.isnan(scale).sum()) == 2
    assert bool((code[1, 0] == 0).all()) and bool(torch.isfinite(code).all())


def _error():
    return _lib.load().dyllm_last_error().decode()


WRITE = dict(x=SOME, ldx=512, heads=4, dim=128, codes=SOME, scales=SOME, rows=64, starts=SOME, cu=SOME, cu_k=None, ids=SOME, batch=1,
             total=8, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dim=64), "head_dim 64"), (dict(heads=0), "heads 0"), (dict(batch=-1), "batch -1"), (dict(total=-1), "rows -1"),
    (dict(rows=-1), "cache rows -1"), (dict(x=None), "null x"), (dict(x=SOME + 2), "16-byte aligned"), (dict(ldx=516), "row pitch"),
    (dict(ldx=504), "row pitch"), (dict(codes=SOME + 8), "codes must be 16-byte"), (dict(scales=SOME + 2), "aligned"),
    (dict(codes=None), "null"), (dict(starts=None), "null"), (dict(cu=None), "null"), (dict(ids=None), "null"),
])
def test_write_refusals(change, text):
    assert _lib.load().dyllm_fp8_cache_write(*{**WRITE, **change}.values()) in (-1, -2)
    assert text in _error()


READ = dict(codes=SOME, scales=SOME, rows=64, heads=4, dim=128, out=SOME, starts=SOME, cu=SOME, cu_k=None, ids=SOME, batch=1, total=8,
            stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dim=256), "head_dim 256"), (dict(heads=-1), "heads -1"), (dict(out=None), "null"), (dict(out=SOME + 8), "out must be 16-byte"),
    (dict(codes=SOME + 4), "16-byte"), (dict(scales=None), "null"), (dict(total=-3), "rows -3"),
])
def test_read_refusals(change, text):
    assert _lib.load().dyllm_fp8_cache_read(*{**READ, **change}.values()) in (-1, -2)
    assert text in _error()


UPDATE = dict(k=SOME, ldk=512, v=SOME, ldv=512, rows_k=SOME, positions=SOME, pos_idx=None, cs=SOME, max_pos=16, cu=SOME, kst=SOME, vst=SOME,
              ids=SOME, batch=1, n=8, n_dev=None, heads=4, dim=128, kc=SOME, ks=SOME, kr=64, vc=SOME, vs=SOME, vr=64, dv=SOME, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dim=96), "head_dim 96"), (dict(heads=0), "heads 0"), (dict(max_pos=0), "0 positions"), (dict(k=SOME + 8), "k_new must be"),
    (dict(ldv=130), "v_new must be"), (dict(v=None), "null v_new"), (dict(rows_k=None), "null"), (dict(dv=None), "null"),
    (dict(dv=SOME + 8), "16-byte"), (dict(cs=SOME + 4), "16-byte"), (dict(vr=-1), "cache rows -1"), (dict(n=-1), "rows -1"),
])
def test_update_refusals(change, text):
    assert _lib.load().dyllm_fp8_kv_cache_update(*{**UPDATE, **change}.values()) in (-1, -2)
    assert text in _error()


ATTEND = dict(q=SOME, ldq=1024, tq=8, kc=SOME, ks=SOME, kr=64, vc=SOME, vs=SOME, vr=64, kst=SOME, vst=SOME, ids=SOME, out=SOME, cu_q=SOME,
              cu_k=SOME, batch=1, most=4, heads=8, kv=4, dim=128, cu_r=SOME, idx=SOME, n=4, scale=0.1, cap=0.0, slopes=None, ranges=None,
              ws=SOME, ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dim=64), "head_dim 64"), (dict(heads=6), "positive multiple"), (dict(heads=0), "positive multiple"), (dict(kv=0), "positive multiple"),
    (dict(n=-1), "rows -1"), (dict(batch=-1), "batch -1"), (dict(most=-1), "max rows -1"), (dict(tq=-1), "Tq -1"), (dict(kr=-1), "batch"),
    (dict(cap=-1.0), "softcap -1"), (dict(cap=1e-9), "softcap"), (dict(cap=float("nan")), "softcap"), (dict(cap=float("inf")), "softcap"),
    (dict(scale=float("nan")), "scale"), (dict(q=None), "null"), (dict(idx=None), "null"), (dict(cu_r=None), "null"), (dict(vs=None), "null"),
    (dict(q=SOME + 8), "16-byte"), (dict(vc=SOME + 8), "16-byte"), (dict(out=SOME + 2), "16-byte"), (dict(ldq=1020), "row pitch"),
    (dict(ldq=512), "row pitch"), (dict(ranges=SOME + 4), "key_ranges"),
])
def test_attention_refusals(change, text):
    assert _lib.load().dyllm_attention_salient_rows_fp8(*{**ATTEND, **change}.values()) in (-1, -2)
    assert text in _error()


@pytest.mark.parametrize("change", [dict(batch=0), dict(n=0), dict(most=0)])
def test_calls_without_work_launch_nothing(change):
    """No GPU here: a launch would return an error."""
    lib = _lib.load()
    assert lib.dyllm_attention_salient_rows_fp8(*{**ATTEND, **change}.values()) == 0
    for args, rows in ((WRITE, "total"), (READ, "total"), (UPDATE, "n")):
        name = {id(WRITE): "dyllm_fp8_cache_write", id(READ): "dyllm_fp8_cache_read", id(UPDATE): "dyllm_fp8_kv_cache_update"}[id(args)]
        assert getattr(lib, name)(*{**args, rows: 0}.values()) == 0
        assert getattr(lib, name)(*{**args, "batch": 0}.values()) == 0


def test_workspace_size_of_nothing():
    assert _lib.load().dyllm_attention_salient_rows_fp8_workspace_bytes(0, 0, 0, 0) >= 0


def test_python_refuses_tensors_of_the_cpu():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    codes, scales = torch.zeros(8, 256, dtype=torch.float8_e4m3fn), torch.zeros(8, 2)
    cu, ids = torch.tensor([0, 4], dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        ops.fp8_cache_write(x, codes, scales, ids, cu, ids)
    with pytest.raises(RuntimeError, match="codes must be a CUDA tensor"):
        ops.fp8_cache_read(codes, scales, ids, cu, ids, 4)
    with pytest.raises(RuntimeError, match="k_new must be a CUDA tensor"):
        ops.fp8_kv_cache_update(x, x, ids, ids, None, scales, cu, ids, ids, ids, (codes, scales), (codes, scales))
    with pytest.raises(RuntimeError, match="q must be a CUDA tensor"):
        attention_ops.attention_salient_rows_fp8(x, (codes, scales), (codes, scales), ids, ids, ids, cu, cu, cu, cu, 4)
