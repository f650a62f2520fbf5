"""The choice of the caches' type, and what an attention block with 8-bit caches refuses (no GPU needed)."""
import pytest
import torch


def test_unknown_cache_type_is_refused():
    from dyllm_b200 import layers

    with pytest.raises(ValueError, match="int4"):
        layers.set_kv_cache_dtype("int4")
    assert layers._kv_cache_dtype == "bf16"


def test_attention_with_8_bit_caches_wants_their_update_from_its_caller(monkeypatch):
    from dyllm_b200 import cache_manager, context, layers

    monkeypatch.setattr(cache_manager.CacheManager.__init__, "__defaults__", (64, torch.float32, torch.device("cpu")))
    monkeypatch.setattr(cache_manager.Fp8CacheManager.__init__, "__defaults__", (128, 64, torch.device("cpu")))
    layers.set_kv_cache_dtype("fp8")
    try:
        attn = layers.Attention(2, 128, 128 ** -0.5, 1)
    finally:
        layers.set_kv_cache_dtype("bf16")
    assert type(attn.v_cache) is cache_manager.Fp8CacheManager and type(attn.context_cache) is cache_manager.CacheManager
    assert type(layers.Attention(2, 128, 128 ** -0.5, 1).v_cache) is cache_manager.CacheManager
    codes, scales = attn.v_cache.pair
    assert codes.shape == (0, 128) and scales.shape == (0, 1) and codes.dtype == torch.float8_e4m3fn
    rows = torch.tensor([1], dtype=torch.int64)
    context.set_context(False, idx_salient_row=rows, idx_salient_row32=rows.int(), total_seqlen=4, total_seqlen_k=4)
    try:
        q, k, v = torch.zeros(4, 2, 128), torch.zeros(4, 1, 128), torch.zeros(1, 1, 128)
        for kw in ({}, {"dv": v}, {"k_cache": attn.v_cache}):
            with pytest.raises(RuntimeError, match="pass dv and k_cache"):
                attn(q, k, v, **kw)
    finally:
        context.reset_context()
