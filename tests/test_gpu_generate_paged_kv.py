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


@pytest.mark.parametrize("chunk_size,bits", [(40, 16), (24, 16), (16, 16), (33, 16), (128, 16), (128, 8), (32, 8)])
def test_the_pool_holds_what_the_prefill_saw(monkeypatch, chunk_size, bits):
    """Chunks that fill their blocks and chunks that do not, two or more of them reused, one prompt
    without reuse and one fully cached."""
    from kvboost_b200.paged_engine import PagedEngine
    prompts = _prompts([300, 256, 5, 281, 80], 256)
    eng = PagedEngine(_model(), num_blocks=256, chunk_size=chunk_size, min_chunk_tokens=8, recompute_strategy="none",
                      kv_cache_bits=bits)
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


def test_steps_append_in_order(monkeypatch):
    """After the last step the pool holds the prefill's K/V and, behind them, what the steps appended,
    and every step attended to its own token and all before it."""
    from kvboost_b200 import paged_decode, paged_engine
    from kvboost_b200.paged_engine import PagedEngine
    prompts = _prompts([100, 31, 16, 1, 77], 64)
    new = 20
    eng = PagedEngine(_model(), num_blocks=64, chunk_size=32, min_chunk_tokens=8)
    eng.warm(prompts[0][:64])
    append, attend, uninstall = (paged_decode.append_paged_kv, paged_decode.paged_decode_attention,
                                 paged_engine.uninstall_paged_attention)
    added, seen, last, state_of = [], [], [], []

    def record_append(k, v, pool, slots):
        added.append((k.clone(), v.clone()))
        append(k, v, pool, slots)

    def record_attend(q, pool, tables, lens, *a, **kw):
        seen.append(lens.tolist())
        state_of[:] = [tables.tolist(), lens.tolist()]
        return attend(q, pool, tables, lens, *a, **kw)

    def record_last(model):
        for table, n in zip(*state_of):
            last.append([eng.allocator.read_kv(layer, table[:-(-n // 16)], n) for layer in range(2)])
        return uninstall(model)

    monkeypatch.setattr(paged_decode, "append_paged_kv", record_append)
    monkeypatch.setattr(paged_decode, "paged_decode_attention", record_attend)
    monkeypatch.setattr(paged_engine, "uninstall_paged_attention", record_last)
    _, _, prefill, _ = _pool_and_prefill(eng, prompts, monkeypatch, max_new_tokens=new)
    assert len(added) == len(seen) == 2 * (new - 1)
    assert seen[::2] == seen[1::2] == [[len(p) + i + 1 for p in prompts] for i in range(new - 1)]
    for b, p in enumerate(prompts):
        for layer in range(2):
            for kv in range(2):
                steps = [added[2 * i + layer][kv][b] for i in range(new - 1)]
                want = torch.cat([prefill[b][layer][kv], torch.stack(steps, 1)], 1)
                assert torch.equal(last[b][layer][kv], want)


# Logits of magnitude up to 4 in bfloat16: two of them compared, each in two evaluations, rounded by at
# most 4 * 2^-8 = 0.016 apiece, and as much again from the activations below.
CLOSE = 0.12


def _behind(model, ids, reuse, keys, values, tokens):
    """How far each token lies behind the best of a dense forward over the reused K/V, the prompt's
    other tokens and the tokens before it."""
    from kvboost_b200.engine import KVBoost
    cache = KVBoost._cache_from(keys[:, :, :reuse].contiguous(), values[:, :, :reuse].contiguous())
    x = torch.tensor([ids[reuse:] + tokens[:-1]], device="cuda")
    pos = torch.arange(reuse, reuse + x.shape[1], device="cuda")[None]
    with torch.no_grad():
        logits = model(input_ids=x, position_ids=pos, past_key_values=cache, use_cache=True).logits[0]
    logits = logits[-len(tokens):].float()
    return logits.amax(-1) - logits[torch.arange(len(tokens)), torch.tensor(tokens)]


def test_greedy_tokens_follow_the_repaired_context():
    """Short prompts, where each block carries weight: the tokens are the best over the repaired K/V, and
    with one block of the reference zeroed they are not (the comparison can tell)."""
    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    prompts = _prompts([36, 40, 33], 32, seed=5)
    eng = PagedEngine(m, num_blocks=64, chunk_size=16, min_chunk_tokens=8, recompute_overlap=4)
    eng.warm(prompts[0][:32])
    want = [eng._assemble(p) for p in prompts]
    got = eng.generate_paged(prompts, max_new_tokens=12)
    for block in (0, 1):
        far = 0.0
        for p, r, (keys, values, n, _) in zip(prompts, got, want):
            assert n == r.cached_tokens == 32
            assert (_behind(m, p, 32, keys, values, r.generated_ids) <= CLOSE).all()
            keys, values = keys.clone(), values.clone()
            keys[:, :, 16 * block:16 * block + 16] = 0
            values[:, :, 16 * block:16 * block + 16] = 0
            far = max(far, float(_behind(m, p, 32, keys, values, r.generated_ids).max()))
        assert far > 2 * CLOSE


@pytest.mark.parametrize("chunk_size", [40, 24, 32])
def test_generate_with_chunks_that_end_inside_a_block(chunk_size):
    """The one-prompt loop, two and more chunks reused: greedy tokens follow the assembled K/V, and no
    cached chunk's block is freed while the mapper holds it."""
    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    prompts = _prompts([84, 90, 85], 80, seed=11)
    eng = PagedEngine(m, num_blocks=64, chunk_size=chunk_size, min_chunk_tokens=chunk_size, recompute_strategy="none")
    eng.warm(prompts[0][:80])
    n = 80 // chunk_size * chunk_size
    for p in prompts:
        keys, values, cached, _ = eng._assemble(p)
        tokens = eng.generate(p, max_new_tokens=12).generated_ids
        assert cached == n
        assert (_behind(m, p, n, keys, values, tokens) <= CLOSE).all()
        held = [b for blocks in eng.chunk_mapper._chunk_blocks.values() for b in blocks]
        assert not set(held) & set(eng.allocator._free)
        assert eng.allocator.used_blocks == len(held)


def test_a_refused_step_raises(monkeypatch):
    """A block id outside the pool, which the kernels skip and report: no tokens, the pool whole, the bit
    left for ``read_status``; bits that others left do not stop a call and are there after it."""
    from kvboost_b200 import ops, paged_engine
    from kvboost_b200.paged_engine import PagedEngine
    eng = PagedEngine(_model(), num_blocks=64, chunk_size=32, min_chunk_tokens=8)
    prompts = _prompts([50, 20], 0)
    dev = torch.device("cuda")
    ops.status_word(dev).fill_(64)
    assert len(eng.generate_paged(prompts, max_new_tokens=4)[0].generated_ids) == 4
    assert ops.read_status(dev) == 64
    tables = paged_engine.block_table_tensor

    def spoiled(lists, device):
        t = tables(lists, device)
        t[0, 0] = 1 << 20               # a block of the reused chunk
        return t

    monkeypatch.setattr(paged_engine, "block_table_tensor", spoiled)
    with pytest.raises(RuntimeError, match="status 0x10"):
        eng.generate_paged([p[:-1] + [7] for p in prompts], max_new_tokens=4)
    assert ops.read_status(dev) == 16
    assert eng.allocator.used_blocks == eng.chunk_mapper.blocks_used_by_chunks()


def test_one_call_at_a_time():
    """Calls from ``allowed_tokens`` and from another thread are refused, and the outer one's tokens are
    those of a call on its own."""
    import threading

    from kvboost_b200.paged_engine import PagedEngine
    eng = PagedEngine(_model(), num_blocks=64, chunk_size=32, min_chunk_tokens=8)
    prompts = _prompts([50], 0)
    eng.warm(prompts[0])                      # every call reuses the same chunks
    want = eng.generate_paged(prompts, max_new_tokens=6)[0].generated_ids
    refused = []

    def attempt(call):
        try:
            call()
        except RuntimeError as e:
            refused.append("running" in str(e))

    def allowed(i, out):
        calls = [lambda: eng.generate_paged(prompts, 3), lambda: eng.generate(prompts[0], 3),
                 lambda: eng.generate([5], 2, mode="baseline")]
        for call in calls:
            attempt(call)
        t = threading.Thread(target=attempt, args=(calls[0],))
        t.start()
        t.join()
        return None

    got = eng.generate_paged(prompts, max_new_tokens=6, allowed_tokens=allowed)[0].generated_ids
    assert got == want and refused == [True] * 24
    assert eng.generate_paged(prompts, max_new_tokens=6)[0].generated_ids == want
