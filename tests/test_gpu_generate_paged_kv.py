"""GPU: what ``PagedEngine.generate_paged`` decodes over.  Before its first step the pool, read through the
block tables, holds exactly the K/V that each prompt's prefill worked on: the reused chunks as
assembled, seams repaired, then the prompt's other tokens."""

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
    """Per prompt and layer: (K, V) of the pool before the first step, and the prefill's cache; the
    prompts' block tables."""
    from kvboost_b200 import paged_engine
    pool, prefill, tables = [], [], []
    suffix, install = eng._prefill_suffix, paged_engine.install_paged_attention

    def record_suffix(*a):
        logits, layers = suffix(*a)
        prefill.append([(k[0].clone(), v[0].clone()) for k, v in layers])
        return logits, layers

    def record_pool(model, state):
        for table, n in zip(state["block_tables"].tolist(), state["seq_lens"].tolist()):
            table = table[:-(-n // 16)]
            tables.append(table)
            pool.append([tuple(t.clone() for t in eng.allocator.read_kv(layer, table, n))
                         for layer in range(eng.allocator.num_layers)])
        return install(model, state)

    monkeypatch.setattr(eng, "_prefill_suffix", record_suffix)
    monkeypatch.setattr(paged_engine, "install_paged_attention", record_pool)
    got = eng.generate_paged(prompts, **kw)
    monkeypatch.undo()
    return got, pool, prefill, tables


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
        got, pool, prefill, _ = _pool_and_prefill(eng, prompts, monkeypatch, max_new_tokens=3)
        assert got[0].cached_tokens >= 2 * chunk_size and got[2].cached_tokens == 0
        _equal(pool, prefill, prompts)
        assert eng.allocator.used_blocks == eng.chunk_mapper.blocks_used_by_chunks()
        assert all(rc == 1 for rc in eng.allocator._ref_count.values())


@pytest.mark.parametrize("chunk_size", [128, 40])
@pytest.mark.parametrize("strategy", ["selective", "cacheblend"])
def test_repaired_seams_reach_the_decode_steps(monkeypatch, strategy, chunk_size):
    """The default seam repair and CacheBlend: the pool holds the repaired K/V, and blocks that the
    repair left as they were stay shared among the prompts.  (The default one recomputes the end of
    a chunk over what comes before it: three chunks, for the first was encoded over just that.)"""
    from kvboost_b200.paged_engine import PagedEngine
    prompts = _prompts([428, 384, 409], 384)
    eng = PagedEngine(_model(), num_blocks=256, chunk_size=chunk_size, min_chunk_tokens=8, recompute_strategy=strategy)
    eng.warm(prompts[0][:384])
    for again in range(2):
        raw = torch.cat([c.keys for c in eng._assemble_run(prompts[0])[4]], 2)
        _, pool, prefill, tables = _pool_and_prefill(eng, prompts, monkeypatch, max_new_tokens=3)
        _equal(pool, prefill, prompts)
        n = min(raw.shape[2], 384)
        changed = [bool((prefill[0][layer][0][:, :n] != raw[layer, :, :n]).any()) for layer in range(2)]
        assert changed[1]                          # there is something that the repair changed
        assert eng.allocator.used_blocks == eng.chunk_mapper.blocks_used_by_chunks()
        assert all(rc == 1 for rc in eng.allocator._ref_count.values())
        if strategy == "selective" and chunk_size == 128:
            # the 16 tokens before the seam at 256, and at 384 once the last chunk is cached too: a
            # block of each prompt's own
            own = [15, 23] if again else [15]
            same = [a == b for a, b in zip(tables[0][:24], tables[2][:24])]
            assert same[:7] + same[8:] == [i not in own for i in range(24) if i != 7]
