"""Captured steps after a change of the batch's geometry, which drops every graph of the one before."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_steps_are_captured_again_for_another_batch(cuda_device):
    from dyllm_b200 import _lib, runner
    from dyllm_b200.model import LLaDAForDLM, LLaDAShape, init_weights_

    shape = LLaDAShape(hidden_size=256, num_attention_heads=2, n_kv_heads=2, head_dim=128, mlp_hidden_size=512,
                       num_hidden_layers=2, vocab_size=1024, mask_token_id=1000, max_sequence_length=256)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(cuda_device):
            model = LLaDAForDLM(shape, 0.99)
    finally:
        torch.set_default_dtype(torch.float32)
    init_weights_(model, seed=3, std=0.05)
    model.eval()
    eager, graphs = (runner.StepRunner(model, 1000, block_length=8, steps=16, num_full_steps=3, refresh_period=4, use_graphs=u)
                     for u in (False, True))
    g = torch.Generator().manual_seed(0)
    for batch, length in ((3, 40), (2, 25), (3, 40)):
        prompts = torch.randint(0, 900, (batch, length), generator=g).tolist()
        want = eager.generate(prompts, 16)
        assert graphs.generate(prompts, 16) == want and graphs.generate(prompts, 16) == want
    assert _lib.load().dyllm_device_status() == 0
