"""The operators on 8-bit caches together, as the models run them: every call of a generation against 64 bits, and the ways of
driving a generation against one another."""
import pytest
import torch

from oracle import dyllm_oracle as orc
from tests.test_fp8_cache_gpu import _check

pytestmark = pytest.mark.gpu
TAU = 0.99


def _model(kind, device, cache="fp8", seed=3):
    from dyllm_b200 import layers, model as M

    common = dict(hidden_size=256, head_dim=128, num_hidden_layers=2, vocab_size=1024, mask_token_id=1000)
    layers.set_kv_cache_dtype(cache)
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(device):
            if kind == "llada":
                m = M.LLaDAForDLM(M.LLaDAShape(num_attention_heads=2, n_kv_heads=2, mlp_hidden_size=512, max_sequence_length=256,
                                               **common), TAU)
            elif kind == "dream":
                m = M.DreamForDLM(M.DreamShape(num_attention_heads=6, num_key_value_heads=2, intermediate_size=512,
                                               max_position_embeddings=256, **common), TAU)
            else:
                m = M.LLaDAMoEForDLM(M.LLaDAMoEShape(num_attention_heads=2, num_key_value_heads=2, num_experts=8,
                                                     num_experts_per_tok=2, expert_intermediate_size=128,
                                                     max_position_embeddings=256, **common), TAU)
    finally:
        torch.set_default_dtype(torch.float32)
        layers.set_kv_cache_dtype("bf16")
    M.init_weights_(m, seed=seed, std=0.05)
    return m.eval()


def _runner(model, **kw):
    from dyllm_b200 import runner

    return runner.StepRunner(model, 1000, block_length=8, steps=16, num_full_steps=3, refresh_period=4, **kw)


def _prompts(lens, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 900, (n,), generator=g).tolist() for n in lens]


def _cpu(pair):
    codes, scales = (t.cpu() for t in pair)
    return codes.float().double().view(codes.size(0), scales.size(1), 128), scales.double()


def _check_every_call(monkeypatch, seen):
    """Each operator replaced by itself with its result compared: caches and delta-V bit for bit, the attention within bounds."""
    from dyllm_b200 import layers, ops

    real = {n: getattr(ops, n) for n in ("fp8_cache_write", "fp8_cache_read", "fp8_kv_cache_update")}
    attend = layers.attention_salient_rows_fp8

    def write(x, codes, scales, starts, cu, ids, cu_seqlens_k=None):
        kc, ks = _cpu((codes, scales))
        real["fp8_cache_write"](x, codes, scales, starts, cu, ids, cu_seqlens_k=cu_seqlens_k)
        orc.fp8_cache_write(kc, ks, x.cpu(), starts.cpu(), cu.cpu(), ids.cpu(), None if cu_seqlens_k is None else cu_seqlens_k.cpu())
        at = orc._fp8_rows(starts.cpu(), cu.cpu(), ids.cpu())
        got = _cpu((codes, scales))
        assert torch.equal(got[0][at], kc[at]) and torch.equal(got[1][at], ks[at])
        seen.append("write")

    def read(codes, scales, starts, cu, ids, total, **kw):
        got = real["fp8_cache_read"](codes, scales, starts, cu, ids, total, **kw)
        want = orc.fp8_cache_read(*_cpu((codes, scales)), starts.cpu(), cu.cpu(), ids.cpu())
        assert got.size(0) == want.size(0) and torch.equal(got.cpu().double(), want)
        seen.append("read")
        return got

    def update(k, v, rows_k, positions, pos_idx, cos_sin, cu_k, k_starts, v_starts, ids, kc, vc, count=None, dv=None):
        torch.cuda.synchronize()
        live = k.size(0) if count is None else int(count)
        before = [*_cpu(kc), *_cpu(vc)]
        got = real["fp8_kv_cache_update"](k, v, rows_k, positions, pos_idx, cos_sin, cu_k, k_starts, v_starts, ids, kc, vc, count, dv=dv)
        torch.cuda.synchronize()
        want = orc.fp8_kv_cache_update(k[:live].cpu(), v[:live].cpu(), rows_k[:live].cpu(), positions.cpu(), pos_idx[:live].cpu(),
                                       cos_sin.cpu(), cu_k.cpu(), k_starts.cpu(), v_starts.cpu(), ids.cpu(), *before)
        at = orc._fp8_rows(k_starts.cpu(), cu_k.cpu(), ids.cpu())
        for have, should in zip([*_cpu(kc), *_cpu(vc)], before):
            assert torch.equal(have[at], should[at])
        assert torch.equal(got[:live].cpu().double(), want.bfloat16().double())
        seen.append("update")
        return got

    def attention(q, kc, vc, k_starts, v_starts, ids, cu_q, cu_k, cu_rows, rows, **kw):
        got = attend(q, kc, vc, k_starts, v_starts, ids, cu_q, cu_k, cu_rows, rows, **kw)
        cu_q, cu_k, cu_rows, ids = (t.cpu() for t in (cu_q, cu_k, cu_rows, ids))
        live = int(cu_rows[-1])
        k = orc.fp8_cache_read(*_cpu(kc), k_starts.cpu(), cu_k, ids)
        v = orc.fp8_cache_read(*_cpu(vc), v_starts.cpu(), cu_k, ids)
        _check(got[:live].cpu().double(), *orc.attention_rows_fp8(q.cpu(), k, v, cu_q, cu_k, cu_rows, rows[:live].cpu()), 0.0)
        seen.append("attention")
        return got

    monkeypatch.setattr(ops, "fp8_cache_write", write)
    monkeypatch.setattr(ops, "fp8_cache_read", read)
    monkeypatch.setattr(ops, "fp8_kv_cache_update", update)
    monkeypatch.setattr(layers, "attention_salient_rows_fp8", attention)


@pytest.mark.parametrize("kind,lens", [("llada", [40, 23, 61]), ("dream", [33, 33]), ("moe", [17])])
@pytest.mark.parametrize("one_stream", [False, True])
def test_every_call_of_a_generation(cuda_device, monkeypatch, kind, lens, one_stream):
    from dyllm_b200 import _lib

    if one_stream:
        monkeypatch.setenv("DYLLM_KV_OVERLAP", "0")
    model = _model(kind, cuda_device)
    sr = _runner(model, use_graphs=False)
    seen = []
    _check_every_call(monkeypatch, seen)
    out = sr.generate(_prompts(lens), 16, device_state=False)
    assert _lib.load().dyllm_device_status() == 0
    assert all(t != 1000 for row in out for t in row)
    dense, sparse = 3, 13
    assert seen.count("write") == dense * 2 * 2 and seen.count("attention") == seen.count("read") == sparse * 2
    assert 0 < seen.count("update") <= sparse * 2


@pytest.mark.parametrize("kind", ["llada", "dream", "moe"])
def test_generations_driven_by_host_device_and_graphs_agree(cuda_device, monkeypatch, kind):
    from dyllm_b200 import _lib, layers

    # the estimate of the rows chooses kernels, whose results differ in their last bits: one estimate for all
    monkeypatch.setattr(layers.Attention, "_next_hint", lambda self, count, capacity, fixed=0: min(20, capacity))
    model = _model(kind, cuda_device)
    prompts, other = _prompts([40] * 3), _prompts([40] * 3, seed=9)
    sr, gr = _runner(model, use_graphs=False), _runner(model, use_graphs=True)
    host = sr.generate(prompts, 16, device_state=False)
    dev = sr.generate(prompts, 16, device_state=True)
    assert host == dev == gr.generate(prompts, 16) == gr.generate(prompts, 16)
    assert gr.generate(other, 16) == sr.generate(other, 16)
    assert gr.generate(_prompts([25] * 2), 16) == sr.generate(_prompts([25] * 2), 16)          # other geometry: captured anew
    assert gr.generate(prompts, 16) == host
    assert _lib.load().dyllm_device_status() == 0


def test_caches_take_half_the_memory_and_16_bits_stay_the_default(cuda_device):
    from dyllm_b200.cache_manager import CacheManager, Fp8CacheManager

    with torch.no_grad():
        size = {}
        for cache in ("bf16", "fp8"):
            model = _model("llada", cuda_device, cache)
            attn = model.model.layers[0].self_attn
            assert type(attn.k_cache) is type(attn.attn.v_cache) is (Fp8CacheManager if cache == "fp8" else CacheManager)
            assert type(attn.attn.context_cache) is CacheManager
            _runner(model, use_graphs=False).generate(_prompts([40]), 16)
            kept = attn.k_cache.pair if cache == "fp8" else [attn.k_cache.cache]
            size[cache] = sum(t.numel() * t.element_size() for t in kept)
    assert size["bf16"] == 56 * 2 * 256 and size["fp8"] == 56 * 2 * 132


def test_manager_keeps_sequences_as_the_16_bit_one(cuda_device):
    from dyllm_b200.cache_manager import CacheManager, Fp8CacheManager
    from dyllm_b200.context import reset_context, set_context

    g = torch.Generator().manual_seed(1)
    heads = 3
    plain, fp8 = CacheManager(heads * 128), Fp8CacheManager(heads)
    for seq, n in [(4, 700), (9, 1), (2, 600), (7, 33)]:                    # grows past its first arena
        c = torch.randn(n, heads * 128, generator=g).bfloat16().cuda()
        code, scale = orc.fp8_quantise(c.view(n, heads, 128))
        plain.add_seq((code * scale.unsqueeze(-1)).flatten(1).bfloat16().cuda(), seq)
        fp8.add_seq(c, seq)

    def compare(ids, lens, qlens=None):
        qlens = qlens or lens
        cum = lambda v: torch.tensor([0] + torch.tensor(v).cumsum(0).tolist(), dtype=torch.int32).cuda()
        set_context(True, cu_seqlens_q=cum(qlens), cu_seqlens_k=cum(lens), total_seqlen=sum(qlens), total_seqlen_k=sum(lens),
                    context_lens_cpu=lens, cu_seqlens_q_cpu=cum(qlens).tolist())
        t = torch.tensor(ids).cuda()
        assert torch.equal(fp8.get_seqs(t), plain.get_seqs(t))
        assert torch.equal(fp8.get_seqs_block(t), plain.get_seqs_block(t))
        return t

    try:
        compare([7, 4, 2, 9], [33, 700, 600, 1], [3, 70, 600, 0])
        for m in (plain, fp8):
            m.finish([4, 9])
        t = compare([7, 2], [33, 600], [33, 100])
        c = torch.randn(133, heads * 128, generator=g).bfloat16().cuda()
        code, scale = orc.fp8_quantise(c.view(133, heads, 128))
        fp8.reset_block(c, t)
        plain.reset_block((code * scale.unsqueeze(-1)).flatten(1).bfloat16().cuda(), t)
        compare([2, 7], [600, 33])
        for n in (33, 50):                                                   # in place, then of another length
            c = torch.randn(n, heads * 128, generator=g).bfloat16().cuda()
            code, scale = orc.fp8_quantise(c.view(n, heads, 128))
            fp8.reset_seq(c, 7)
            plain.reset_seq((code * scale.unsqueeze(-1)).flatten(1).bfloat16().cuda(), 7)
            compare([7, 2], [n, 600])
        assert fp8._seq_to_start == plain._seq_to_start and torch.equal(fp8.seq_start_gpu, plain.seq_start_gpu)
        with pytest.raises(RuntimeError, match="fp8_kv_cache_update"):
            fp8.scatter_update(t, t, c)
        with pytest.raises(ValueError, match="head dimension"):
            Fp8CacheManager(2, 64)
    finally:
        reset_context()


def test_two_captured_graphs_on_two_streams_keep_apart(cuda_device):
    """Two generations' operators captured over shared caches, replayed at the same time on two streams: same bits as alone."""
    from dyllm_b200 import ops
    from dyllm_b200.attention_ops import attention_salient_rows_fp8
    from tests.test_fp8_cache_gpu import Batch, _far, _to_cache

    b = Batch([900, 333, 64], [300, 333, 64], seed=8)
    kc, vc = _to_cache(*_far(b, *b.cache(2))), _to_cache(*_far(b, *b.cache(2)))
    ks, vs, ids, cu_q, cu_k = (t.cuda() for t in (b.k_starts, b.v_starts, b.ids, b.cu_q, b.cu_k))
    jobs = []
    for counts in ([7, 2, 9], [250, 333, 64]):
        cu, rows, _ = b.picks(counts)
        q = b.randn(sum(b.qlens), 8, 128).bfloat16().cuda()
        cu, rows = cu.cuda(), rows.cuda()

        def run(q=q, cu=cu, rows=rows, most=max(counts)):
            k = ops.fp8_cache_read(*kc, ks, cu_k, ids, sum(b.lens))
            return k, attention_salient_rows_fp8(q, kc, vc, ks, vs, ids, cu_q, cu_k, cu, rows, max_rows_per_seq=most)

        alone = run()
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):
            got = run()
        jobs.append((alone, got, graph, stream, run))         # a graph reads the inputs where they were: `run` holds them
    for _ in range(5):
        for _, got, graph, stream, _ in jobs:
            with torch.cuda.stream(stream):
                got[1].fill_(3.0)
                graph.replay()
        torch.cuda.synchronize()
        for alone, got, *_ in jobs:
            assert torch.equal(alone[0], got[0]) and torch.equal(alone[1], got[1])
