"""GPU: what ``PagedEngine.generate_paged`` decodes over.  Before its first step the pool, read through the
block tables, holds exactly the K/V that each prompt's prefill worked on: the reused chunks as
assembled, then the prompt's other tokens."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 (B200) device")
    from kvboost_b200 import ops
    ops.read_status(torch.device("cuda"))
    yield
    assert ops.read_status(torch.device("cuda")) == 0


def _model():
    """Two layers whose tokens differ in K and V and attend to some more than to others."""
    from transformers import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=501, hidden_size=512, intermediate_size=1024,
                      num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                      max_position_embeddings=4096, rms_norm_eps=1e-6, rope_theta=1e6,
                      tie_word_embeddings=False, attn_implementation="sdpa")
    torch.manual_seed(0)
    m = Qwen2ForCausalLM(cfg)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "norm" in name:
                p.fill_(1.0)
            elif name.endswith("bias"):
                p.zero_()
            else:
                p.normal_(0, 1.0 if "embed" in name else p.shape[-1] ** -0.5)
    return m.to("cuda", torch.bfloat16).eval()


def _prompts(lens, shared, seed=3):
    g = torch.Generator().manual_seed(seed)
    head = torch.randint(0, 501, (shared,), generator=g).tolist()
    return [(head + torch.randint(0, 501, (max(0, n - shared),), generator=g).tolist())[:n] for n in lens]


def _pool_and_prefill(eng, prompts, monkeypatch, **kw):
    """Per prompt and layer: (K, V) of the pool before the first step, and the prefill's cache."""
    from kvboost_b200 import paged_engine
    pool, prefill = [], []
    suffix, install = eng._prefill_suffix, paged_engine.install_paged_attention

    def record_suffix(*a):
        logits, layers = suffix(*a)
        prefill.append([(k[0].clone(), v[0].clone()) for k, v in layers])
        return logits, layers

    def record_pool(model, state):
        for table, n in zip(state["block_tables"].tolist(), state["seq_lens"].tolist()):
            table = table[:-(-n // 16)]
            pool.append([tuple(t.clone() for t in eng.allocator.read_kv(layer, table, n))
                         for layer in range(eng.allocator.num_layers)])
        return install(model, state)

    monkeypatch.setattr(eng, "_prefill_suffix", record_suffix)
    monkeypatch.setattr(paged_engine, "install_paged_attention", record_pool)
    got = eng.generate_paged(prompts, **kw)
    monkeypatch.undo()
    return got, pool, prefill


def _equal(pool, prefill, prompts):
    assert len(pool) == len(prefill) == len(prompts)
    for p, a, b in zip(prompts, pool, prefill):
        for (k, v), (kk, vv) in zip(a, b):
            assert k.shape[1] == len(p) and torch.equal(k, kk) and torch.equal(v, vv)


@pytest.mark.parametrize("chunk_size", [40, 24, 16, 33, 128])
def test_the_pool_holds_what_the_prefill_saw(monkeypatch, chunk_size):
    """Chunks that fill their blocks and chunks that do not, two or more of them reused, one prompt
    without reuse and one fully cached."""
    from kvboost_b200.paged_engine import PagedEngine
    prompts = _prompts([300, 256, 5, 281, 80], 256)
    eng = PagedEngine(_model(), num_blocks=256, chunk_size=chunk_size, min_chunk_tokens=8, recompute_strategy="none")
    eng.warm(prompts[0][:256])
    for _ in range(2):                       # the second time the prompts' own chunks are cached too
        got, pool, prefill = _pool_and_prefill(eng, prompts, monkeypatch, max_new_tokens=3)
        assert got[0].cached_tokens >= 2 * chunk_size and got[2].cached_tokens == 0
        _equal(pool, prefill, prompts)
        assert eng.allocator.used_blocks == eng.chunk_mapper.blocks_used_by_chunks()
        assert all(rc == 1 for rc in eng.allocator._ref_count.values())
