"""GPU: ``PagedEngine.generate_paged``, the batched decode loop over the block pool: its greedy
tokens are the best of a dense-cache forward over the same reused K/V, the pool's blocks
come back, and penalties, biases and masks follow the 64-bit restatement on the model's
logits.

"Best" within 0.12: these random-weight models' two best logits often lie closer than
bfloat16 tells apart.  A logit of magnitude up to 4 is rounded by at most 4 * 2^-8 = 0.016;
the comparison has two logits in each of two evaluations (0.06), and the bfloat16
activations below them add as much again.  A wrong K/V moves logits by their spread, about 1.
"""

import pytest
import torch

from oracle import step as ostep

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
    from transformers import Qwen2Config, Qwen2ForCausalLM
    cfg = Qwen2Config(vocab_size=501, hidden_size=512, intermediate_size=1024,
                      num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2,
                      max_position_embeddings=4096, rms_norm_eps=1e-6, rope_theta=1e6,
                      tie_word_embeddings=False, attn_implementation="sdpa")
    torch.manual_seed(0)
    m = Qwen2ForCausalLM(cfg)
    with torch.no_grad():
        for name, p in m.named_parameters():
            p.normal_(0, 1.0 if "lm_head" in name else 0.02)  # decisive greedy choices
    return m.to("cuda", torch.bfloat16).eval()


def _prompts(lens, shared, seed=3):
    g = torch.Generator().manual_seed(seed)
    head = torch.randint(0, 501, (shared,), generator=g).tolist()
    return [(head + torch.randint(0, 501, (max(0, n - shared),), generator=g).tolist())[:n] for n in lens]


CLOSE = 0.12


def _check_greedy(model, ids, reuse, keys, values, tokens):
    """Every token is the best of a forward over the reused K/V, the prompt's other tokens and
    the tokens before it."""
    from kvboost_b200.engine import KVBoost
    from transformers import DynamicCache
    cache = KVBoost._cache_from(keys[:, :, :reuse].contiguous(), values[:, :, :reuse].contiguous()) \
        if reuse else DynamicCache()
    x = torch.tensor([ids[reuse:] + tokens[:-1]], device="cuda")
    pos = torch.arange(reuse, reuse + x.shape[1], device="cuda")[None]
    with torch.no_grad():
        logits = model(input_ids=x, position_ids=pos, past_key_values=cache, use_cache=True).logits[0]
    logits = logits[-len(tokens):].float()
    picked = logits[torch.arange(len(tokens)), torch.tensor(tokens)]
    assert (picked >= logits.amax(-1) - CLOSE).all(), (logits.amax(-1) - picked).tolist()


def test_greedy_tokens():
    """Ragged prompts sharing two chunks, one fully cached, one of a single token, one whose
    cached run ends inside a block; new tokens cross block boundaries."""
    from kvboost_b200.engine import KVBoost
    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    prompts = _prompts([300, 256, 1, 413, 275, 97], 256)
    eng = PagedEngine(m, num_blocks=256, recompute_strategy="none")
    eng.warm(prompts[0][:256])
    eng.warm(prompts[5])                                   # a lone chunk of 97 tokens
    free = eng.allocator.free_blocks
    got = eng.generate_paged(prompts, max_new_tokens=20)
    assert eng.allocator.free_blocks == free - eng.chunk_mapper.blocks_used_by_chunks()
    assert all(rc == 1 for rc in eng.allocator._ref_count.values())
    again = eng.generate_paged(prompts, max_new_tokens=20)  # more of the prompts cached now
    assert eng.allocator.free_blocks == eng.allocator.num_blocks - eng.chunk_mapper.blocks_used_by_chunks()
    assert all(rc == 1 for rc in eng.allocator._ref_count.values())
    assert [r.cached_tokens for r in got] == [256, 256, 0, 256, 256, 97]
    full = KVBoost(m, recompute_strategy="none")
    full.warm(prompts[0][:256])
    full.warm(prompts[5])
    for p, r, r2 in zip(prompts, got, again):
        assert len(r.generated_ids) == len(r2.generated_ids) == 20 and r.prompt_tokens == len(p)
        keys, values, n, _ = full._assemble(p)
        assert n == r.cached_tokens
        _check_greedy(m, p, min(n, len(p) - 1), keys, values, r.generated_ids)
    full.generate_batch(prompts, max_new_tokens=1)          # stores the prompts' other chunks
    for p, r in zip(prompts, again):
        keys, values, n, _ = full._assemble(p)
        assert n == r.cached_tokens
        _check_greedy(m, p, min(n, len(p) - 1), keys, values, r.generated_ids)
    assert eng.generate_paged([]) == []


def _reference_step(model, ids, n_prompt, rep, freq, pres, bias, allowed):
    with torch.no_grad():
        x = model(input_ids=torch.tensor([ids], device="cuda"), use_cache=False).logits[0, -1]
    mask = None
    if allowed is not None:
        import numpy as np
        words = np.zeros((1, 16), dtype=np.int64)
        for t in allowed:
            words[0, t // 32] |= 1 << (t % 32)
        mask = words
    import numpy as np
    return ostep.logits(x.double().cpu().numpy()[None], np.array([ids]), [n_prompt], [len(ids)], [rep], [freq],
                        [pres], np.array([list(bias)]), np.array([list(bias.values())]), mask)[0]


def test_penalties_biases_and_masks():
    """Each token generate_paged picks is the restatement's best on the model's logits for the
    tokens so far (times 1.3, the largest factor the penalties put on a logit), and is allowed."""
    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    prompts = _prompts([150, 40], 0)
    bias = {7: 3.0, 400: -50.0, 33: 1.5}

    def allowed(i, out):
        return None if i == 0 else range(len(out) % 2, 501, 2)      # prompt 1: even, odd, even, ...

    eng = PagedEngine(m, num_blocks=64, recompute_strategy="none")
    res = eng.generate_paged(prompts, max_new_tokens=12, repetition_penalty=1.3, frequency_penalty=0.7,
                             presence_penalty=0.4, logit_bias=bias, allowed_tokens=allowed)
    for i, (p, r) in enumerate(zip(prompts, res)):
        ids = list(p)
        for n, t in enumerate(r.generated_ids):
            want = _reference_step(m, ids, len(p), 1.3, 0.7, 0.4, bias, allowed(i, r.generated_ids[:n]))
            assert want[t] >= want.max() - 1.3 * CLOSE, (i, n, t)
            if i == 1:
                assert t % 2 == n % 2
            ids.append(t)
    sampled = eng.generate_paged(prompts, max_new_tokens=5, temperature=0.7, do_sample=True)
    assert [len(r.generated_ids) for r in sampled] == [5, 5]


def test_pool_too_small_leaves_the_pool_as_it_was():
    from kvboost_b200.paged_engine import PagedEngine
    eng = PagedEngine(_model(), num_blocks=8, recompute_strategy="none")
    with pytest.raises(RuntimeError, match="OOM"):
        eng.generate_paged(_prompts([100, 100], 0), max_new_tokens=10)
    assert eng.allocator.free_blocks == 8


def test_a_prompt_without_a_token_left_is_refused():
    from kvboost_b200.paged_engine import PagedEngine
    eng = PagedEngine(_model(), num_blocks=64, recompute_strategy="none")
    p = _prompts([20, 30], 0)
    for sample in (False, True):
        with pytest.raises(ValueError, match="prompt 1"):
            eng.generate_paged(p, max_new_tokens=4, do_sample=sample, allowed_tokens=lambda i, out: [3, 4] if i == 0 else [])
    with pytest.raises(ValueError, match="lie in"):
        eng.generate_paged(p, max_new_tokens=4, allowed_tokens=lambda i, out: [501])
    assert eng.allocator.free_blocks == 64
    twice = eng.generate_paged([p[0], p[0]], max_new_tokens=6)
    assert twice[0].generated_ids == twice[1].generated_ids


def test_the_end_id_stops_a_prompt_and_keeps_the_others_going():
    """A prompt that met the end id takes no more tokens and is asked for none; zero new tokens
    means one, as in ``generate``."""
    from types import SimpleNamespace

    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    p = _prompts([20, 33, 50], 0)
    eng = PagedEngine(m, num_blocks=64, recompute_strategy="none")
    free = [r.generated_ids for r in eng.generate_paged(p, max_new_tokens=8)]
    eos = free[1][2]
    eng.tokenizer = SimpleNamespace(eos_token_id=eos, pad_token_id=None,
                                    decode=lambda ids, skip_special_tokens: " ".join(map(str, ids)))
    asked = []

    def allowed(i, out):
        asked.append((i, len(out)))
        assert eos not in out
        return None

    got = eng.generate_paged(p, max_new_tokens=8, allowed_tokens=allowed)
    for ids, r in zip(free, got):
        n = ids.index(eos) + 1 if eos in ids else 8
        assert r.generated_ids == ids[:n]
    assert max(n for i, n in asked if i == 1) == free[1].index(eos)
    assert eng.generate_paged(p, max_new_tokens=0)[2].generated_ids == free[2][:1]
    assert eng.allocator.free_blocks == 64 - eng.chunk_mapper.blocks_used_by_chunks()


@pytest.mark.parametrize("n", [33, 48, 49, 97, 128, 129, 144, 145])
def test_reuse_that_ends_at_and_around_block_borders(n):
    """The prompt's chunks cached or not, its last token runs again: the same tokens, within the
    pool's blocks (the status word stays clear)."""
    from kvboost_b200.paged_engine import PagedEngine
    m = _model()
    p = _prompts([n], 0, seed=n)
    eng = PagedEngine(m, num_blocks=2 * -(-(n + 17) // 16) + 1, recompute_strategy="none")
    eng.warm(p[0])
    for _ in range(2):
        r = eng.generate_paged(p, max_new_tokens=17)[0]
        keys, values, cached, _ = eng._assemble(p[0])
        assert r.cached_tokens == cached
        _check_greedy(m, p[0], min(cached, n - 1), keys, values, r.generated_ids)
