"""Paged-pool generation engine: the drop-in for KVBoost's ``CPUPagedEngine``.

Mirrors ``src/kvboost/cpu_paged/cpu_engine.py:72-516``: the chunk-reuse engine
(``KVBoost``) whose single-prompt generation keeps the sequence's K/V in a
16-token block pool instead of a growing cache tensor:

1. the reused chunks are loaded into the pool through the chunk mapper (a
   chunk already in the pool is forked, so its blocks are shared), giving the
   sequence's block table (``cpu_engine.py:187-206``);
2. the prompt's new tokens run as one model forward over the assembled
   (seam-repaired) prefix, and their K/V are appended to the pool after the
   prefix -- every layer at the same slots, new blocks taken from the free list
   by the first layer (``:208-248``, ``:440-475``); a fully cached prompt
   re-feeds its last token and appends it after the prefix (``:250-282``);
3. each decode step runs the model with no cache: the paged interceptor
   (``flash_attn_ext.install_paged_attention``) appends the step's K/V at the
   next slot and attends over the pool (``:284-310``, ``:344-408``);
4. the sequence's own blocks (past the reused prefix) go back to the free list,
   then the prompt's new chunks are stored (``:312-319``, ``:499-512``).

The block bookkeeping (free-list order, forks, copy-on-write, which blocks are
freed) follows the reference step for step, so block tables are identical.
What differs is where it runs: the pool lives in GPU memory in the model's
dtype (the reference's pool is float16 because its ``from_pretrained`` loads
the model in float16), the appends are device scatters, the prefill runs on the
sm_100a prefill kernel and the decode steps on the paged attention path.  The
reference class raises under transformers 5.x (it indexes the returned
``DynamicCache`` as a tuple, ``cpu_engine.py:451``); this one reads the cache's
layers.  ``generate_batch`` / ``generate_many`` are ``KVBoost``'s (the
reference's paged engine inherits them unchanged), and ``BASELINE`` mode runs
the whole prompt as in ``KVBoost``.

``generate_paged`` has no counterpart in the reference: it decodes several prompts
over the pool at once, each step's block tables, slots, K/V writes, attention and
logits on the device (``paged_decode``, ``logits``).
"""

from __future__ import annotations

import threading
import time
from typing import Callable, Dict, List, Optional, Sequence, Tuple, Union

import torch

from .engine import GenerationMode, GenerationResult, KVBoost, RecomputeStrategy, TokenIds
from .flash_attn_ext import install_paged_attention, uninstall_paged_attention
from .logits import process_logits
from .ops import read_status, status_word
from .paged import BLOCK_SIZE, DeviceBlockAllocator, DeviceChunkMapper, block_table_tensor
from .paged_decode import append_paged_kv, extend_block_tables


def _model_dims(model) -> Tuple[int, int, int]:
    """(layers, KV heads, head dim) as ``_infer_model_dims`` (``cpu_engine.py:56-69``)
    reads them, with the config's explicit ``head_dim`` where it has one."""
    cfg = model.config
    heads = cfg.num_attention_heads
    kv = getattr(cfg, "num_key_value_heads", None) or heads
    d = getattr(cfg, "head_dim", None) or cfg.hidden_size // heads
    return cfg.num_hidden_layers, kv, d


class PagedEngine(KVBoost):
    """``KVBoost`` with the paged decode loop of ``CPUPagedEngine``.

    ``block_size`` (16, the paged kernels' block) and ``num_blocks`` (pool size)
    as in the reference; ``pool_dtype`` defaults to the model's dtype.
    """

    def __init__(self, model, tokenizer=None, *, max_cache_bytes: int = 16 << 30,
                 block_size: int = BLOCK_SIZE, num_blocks: int = 4096,
                 pool_dtype: Optional[torch.dtype] = None, **kwargs) -> None:
        super().__init__(model, tokenizer, max_cache_bytes=max_cache_bytes, **kwargs)
        L, H, D = _model_dims(self.model)
        dt = pool_dtype or next(self.model.parameters()).dtype
        self.allocator = DeviceBlockAllocator(L, H, D, num_blocks, block_size,
                                              device=self.device, dtype=dt)
        self.chunk_mapper = DeviceChunkMapper(self.allocator)
        self._num_layers, self._block_size = L, block_size
        self._stepping = threading.Lock()    # held while the model's attention is a batched step's
        store_evict = self.store.on_evict

        def on_evict(chunk):      # chunk blocks leave the pool with the chunk (:124-126)
            store_evict(chunk)
            self.chunk_mapper.on_evict(chunk.chunk_id)
        self.store.on_evict = on_evict

    # ── generation ────────────────────────────────────────────────────────────
    def generate(self, prompt: Union[str, Sequence[int]], max_new_tokens: int = 64,
                 mode: Union[str, GenerationMode] = GenerationMode.CHUNK_KV_REUSE,
                 temperature: float = 1.0, do_sample: bool = False,
                 cacheable_prefix_len: Optional[int] = None) -> GenerationResult:
        mode = GenerationMode(mode)
        if self._stepping.locked():
            raise RuntimeError("generate_paged is running on this engine")
        if mode == GenerationMode.BASELINE:
            return super().generate(prompt, max_new_tokens, mode, temperature, do_sample)
        self._sync()
        t0 = time.perf_counter()
        token_ids = self._encode(prompt)
        reuse = mode == GenerationMode.CHUNK_KV_REUSE
        keys, values, cached_len, _, chunks = self._assemble_run(token_ids, repair_seams=reuse)
        res = self._paged_decode(prompt, token_ids, chunks, keys, values, cached_len,
                                 max_new_tokens, temperature, do_sample, mode.value, t0,
                                 # the reference passes its hit ratio only in reuse mode
                                 cached_len / max(len(token_ids), 1) if reuse else 0.0)
        self._store_prompt_chunks(token_ids, cacheable_prefix_len=cacheable_prefix_len)
        return res

    def _append_layers(self, layers, table: List[int], slot: int,
                       skip: int) -> Tuple[List[int], int]:
        """The tokens from ``skip`` on of each layer's cache appended at ``slot``
        (``_append_new_kv_to_pool``, ``cpu_engine.py:440-475``)."""
        n_new = layers[0][0].shape[2] - skip
        if n_new <= 0:
            return table, slot
        for layer, (k, v) in enumerate(layers):
            table, _ = self.allocator.append_kv(layer, table, slot, k[0, :, skip:],
                                                v[0, :, skip:])
        return table, slot + n_new

    def _paged_decode(self, prompt, token_ids: TokenIds, chunks, keys, values, cached_len: int,
                      max_new_tokens: int, temperature: float, do_sample: bool, mode_name: str,
                      t0: float, hit_ratio: float) -> GenerationResult:
        from transformers import DynamicCache
        table: List[int] = []
        in_pool = shared_blocks = 0
        if keys is not None and cached_len > 0:
            in_pool = cached_len
            if any(c.length % self._block_size for c in chunks[:-1]):
                # chunks that begin inside a block cannot lend their blocks: the sequence's own
                n = -(-cached_len // self._block_size)
                table = self.allocator.allocate(n)
                kv = [self._chunk_kv([c]) for c in chunks]
                self._write_blocks(table, list(range(n)), torch.cat([k for k, _ in kv], 2),
                                   torch.cat([v for _, v in kv], 2))
            else:
                shared_blocks = -(-cached_len // self._block_size)
                for c in chunks:      # the chunks as cached (before any seam repair)
                    k, v = self._chunk_kv([c])
                    table.extend(self.chunk_mapper.load_chunk(
                        c.chunk_id, [(k[l][None], v[l][None]) for l in range(k.shape[0])]))
        live = token_ids[cached_len:]
        if live:
            cache = self._cache_from(keys, values) if keys is not None else DynamicCache()
            x = torch.tensor([live], dtype=torch.long, device=self.device)
            pos = torch.arange(cached_len, cached_len + len(live), device=self.device)[None]
            skip = cached_len
        else:     # fully cached: re-feed the last token at its position
            cache = (self._cache_from(keys[:, :, :cached_len - 1].contiguous(),
                                      values[:, :, :cached_len - 1].contiguous())
                     if cached_len > 1 else DynamicCache())
            x = torch.tensor([[token_ids[-1]]], dtype=torch.long, device=self.device)
            pos = torch.tensor([[cached_len - 1]], dtype=torch.long, device=self.device)
            skip = cached_len - 1
        out = self._forward(x, pos, cache)
        first_logits = out.logits[0, -1, :].float()
        generated = [int(self._sample(out.logits[:, -1, :], temperature, do_sample)[0])]
        t_first = time.perf_counter()
        table, in_pool = self._append_layers(self._layers(out.past_key_values), table, in_pool,
                                             skip)
        del out, cache
        cur = cached_len + len(live)
        state = {"allocator": self.allocator, "block_table": table, "_write_slot": in_pool}
        eos = self._eos
        install_paged_attention(self.model, state)
        try:
            while len(generated) < max_new_tokens and generated[-1] != eos:
                x = torch.tensor([[generated[-1]]], dtype=torch.long, device=self.device)
                p = torch.tensor([[cur]], dtype=torch.long, device=self.device)
                with torch.no_grad():
                    logits = self.model(input_ids=x, position_ids=p, use_cache=False,
                                        logits_to_keep=1).logits
                state["_write_slot"] += 1
                generated.append(int(self._sample(logits[:, -1, :], temperature, do_sample)[0]))
                cur += 1
        finally:
            uninstall_paged_attention(self.model)
        table = state["block_table"]
        t1 = time.perf_counter()
        # the sequence's own blocks (past the reused prefix's) return to the free list
        if table[shared_blocks:]:
            self.allocator.free(table[shared_blocks:])
        self.last_block_table = table
        return GenerationResult(
            mode=mode_name, prompt=prompt if isinstance(prompt, str) else "",
            output_text=self._decode_text(generated), generated_tokens=len(generated),
            ttft_ms=(t_first - t0) * 1e3, total_ms=(t1 - t0) * 1e3,
            tokens_per_sec=len(generated) / max(t1 - t0, 1e-9), kv_reuse_ratio=hit_ratio,
            prompt_tokens=len(token_ids), cached_tokens=cached_len,
            first_token_logits=first_logits.cpu().numpy(), generated_ids=generated)

    # ── several prompts over the pool at once ──────────────────────────────────
    def generate_paged(self, prompts: List[Union[str, Sequence[int]]], max_new_tokens: int = 64,
                       temperature: float = 1.0, do_sample: bool = False,
                       repetition_penalty: float = 1.0, frequency_penalty: float = 0.0,
                       presence_penalty: float = 0.0,
                       logit_bias: Optional[Dict[int, float]] = None,
                       allowed_tokens: Optional[Callable[[int, List[int]],
                                                         Optional[Sequence[int]]]] = None,
                       ) -> List[GenerationResult]:
        """Decode several prompts together, their K/V in the block pool.

        Each prompt reuses its cached chunks, seams repaired by the engine's strategy for the
        prefill and for every step (as in ``KVBoost.generate``; this engine's ``generate``
        decodes over the chunks as cached).  The blocks that a chunk fills are shared through
        the mapper; those that the repair changed, those with tokens of two chunks (where
        ``chunk_size`` is no multiple of 16) and a part-filled last block are written anew.
        Then it prefills its new tokens, and every step runs one token of every prompt: block
        tables and slots from the lengths (``extend_block_tables``), K/V into the pool and
        attention over it in every layer, and the logits' processing
        (``process_logits``): ``repetition_penalty`` over prompt and output,
        ``frequency_penalty`` and ``presence_penalty`` over the output, ``logit_bias`` by
        token id, and ``allowed_tokens(i, output ids)``, the ids prompt i may continue with
        (None: any).  A prompt that has met the end id keeps its place in the steps until
        all have ended.  The blocks of the longest outputs are reserved before the first
        step and returned at the end; the prompts' new chunks are then stored.  A step that the
        device refused a part of (``ops.read_status``; the word is the device's, so a report of
        other work on it counts) raises, and so does a call while another
        runs on the engine (from ``allowed_tokens``, or from another thread): its steps would
        go through the other's tables.
        """
        if not self._stepping.acquire(blocking=False):
            raise RuntimeError("generate_paged is running on this engine")
        try:
            return self._generate_paged(prompts, max_new_tokens, temperature, do_sample,
                                        repetition_penalty, frequency_penalty, presence_penalty,
                                        logit_bias, allowed_tokens)
        finally:
            self._stepping.release()

    def _generate_paged(self, prompts, max_new_tokens, temperature, do_sample, repetition_penalty,
                        frequency_penalty, presence_penalty, logit_bias,
                        allowed_tokens) -> List[GenerationResult]:
        if self.allocator.dtype != next(self.model.parameters()).dtype:
            raise RuntimeError("generate_paged needs a pool in the model's dtype")
        if not prompts:
            return []
        self._sync()
        t0 = time.perf_counter()
        all_ids = [self._encode(p) for p in prompts]
        if any(not ids for ids in all_ids):
            raise ValueError("empty prompt")
        # the device's status word is read with every step's tokens; what others left in it waits
        status = status_word(self.device)
        before = read_status(self.device)
        B, bs, dev = len(prompts), self._block_size, self.device
        most = max(1, int(max_new_tokens))   # a first token comes with the prompt, as in generate
        prefixes: List[List[int]] = []     # each prompt's blocks of reused chunks
        forked: List[int] = []             # references to hand back
        reserved: List[int] = []
        try:
            first_logits, kv_new, cached, reused = [], [], [], []
            for ids in all_ids:
                keys, values, cached_len, bounds, chunks = self._assemble_run(ids)
                reuse = min(cached_len, len(ids) - 1)   # a fully cached prompt's last token runs again
                table = [-1] * -(-reuse // bs)
                repaired = len(chunks) > 1 and self.recompute_strategy != RecomputeStrategy.NONE
                for c, (start, end) in zip(chunks, bounds):
                    # a chunk that begins on a block's border shares the blocks it fills, but for
                    # those whose K/V the seam repair changed
                    whole = range(start // bs, min(end, reuse) // bs) if start % bs == 0 else ()
                    if not whole:
                        continue
                    k, v = self._chunk_kv([c])
                    if repaired:
                        n = len(whole) * bs
                        same = ((keys[:, :, start:start + n] == k[:, :, :n]) &
                                (values[:, :, start:start + n] == v[:, :, :n]))
                        same = same.unflatten(2, (len(whole), bs)).all(-1).all(-1).all(1).all(0)
                        whole = [i for i, ok in zip(whole, same.tolist()) if ok]
                        if not whole:
                            continue
                    shared = c.chunk_id in self.chunk_mapper._chunk_blocks
                    blocks = self.chunk_mapper.load_chunk(
                        c.chunk_id, [(k[l][None], v[l][None]) for l in range(k.shape[0])])
                    # a reference of this call's own, whether or not the chunk was in the pool
                    forked.extend(blocks if shared else self.allocator.fork(blocks))
                    for i in whole:
                        table[i] = blocks[i - start // bs]
                own = [i for i, block in enumerate(table) if block < 0]
                if own:     # changed blocks, blocks with parts of two chunks, the one that new tokens begin in
                    blocks = self.allocator.allocate(len(own))
                    reserved.extend(blocks)
                    self._write_blocks(blocks, own, keys[:, :, :reuse], values[:, :, :reuse])
                    for i, block in zip(own, blocks):
                        table[i] = block
                prefixes.append(table)
                cached.append(cached_len)
                reused.append(reuse)
                logits, layers = self._prefill_suffix(ids, keys, values, reuse)
                first_logits.append(logits)
                kv_new.append([(k[0, :, reuse:], v[0, :, reuse:]) for k, v in layers])
            lens = [len(ids) for ids in all_ids]
            want = [-(-(n + most) // bs) for n in lens]
            free = self.allocator.allocate(sum(w - len(t) for w, t in zip(want, prefixes)))
            reserved.extend(free)
            i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
            tables = block_table_tensor([t + [0] * (w - len(t)) for t, w in zip(prefixes, want)], dev)
            seq_lens, free_blocks, num_free = i32(reused), i32(free), i32([len(free)])
            new = [n - c for n, c in zip(lens, reused)]
            # the prompts' new tokens, packed, layer by layer
            step = extend_block_tables(tables, seq_lens, i32(new), free_blocks, num_free,
                                       self.allocator.num_blocks, sum(new), seq_lens_out=seq_lens,
                                       num_free_out=num_free)
            for layer, pool in enumerate(self.allocator.pools):
                parts = [kv[layer] for kv in kv_new]
                append_paged_kv(torch.cat([k for k, _ in parts], 1).transpose(0, 1).to(pool.dtype),
                                torch.cat([v for _, v in parts], 1).transpose(0, 1).to(pool.dtype),
                                pool, step.slots)
            del kv_new
            logits = torch.stack(first_logits)
            V = logits.shape[-1]
            history = torch.zeros(B, max(lens) + most, dtype=torch.int32, device=dev)
            for b, ids in enumerate(all_ids):
                history[b, :lens[b]] = i32(ids)
            prompt_lens, total_lens = i32(lens), i32(lens)
            f32 = lambda x: torch.full((B,), float(x), dtype=torch.float32, device=dev)  # noqa: E731
            penalised = repetition_penalty != 1.0 or frequency_penalty or presence_penalty
            kw = {}
            if penalised:
                kw.update(token_ids=history, prompt_lens=prompt_lens, total_lens=total_lens,
                          repetition_penalty=f32(repetition_penalty),
                          frequency_penalty=f32(frequency_penalty),
                          presence_penalty=f32(presence_penalty))
            if logit_bias:
                kw.update(bias_ids=i32([list(logit_bias)] * B),
                          bias_values=torch.tensor([[float(w) for w in logit_bias.values()]] * B,
                                                   dtype=torch.float32, device=dev))
            if do_sample:
                kw["temperature"] = f32(temperature)
            generated: List[List[int]] = [[] for _ in range(B)]
            done = [False] * B
            ones, rows = i32([1] * B), torch.arange(B, device=dev)
            eos = self._eos
            state = {"allocator": self.allocator, "block_tables": tables, "seq_lens": seq_lens}
            install_paged_attention(self.model, state)
            try:
                t_first = 0.0
                while True:
                    if allowed_tokens is not None:
                        kw["allowed_mask"] = self._token_masks(
                            [None if done[b] else allowed_tokens(b, list(generated[b]))
                             for b in range(B)], V)
                    x = process_logits(logits.contiguous(), **kw)
                    # a row without a finite best (all masked, NaN) cannot be sampled from
                    lost = ~torch.isfinite(x.amax(-1))
                    nxt = self._sample(x.masked_fill_(lost[:, None], 0.0), 1.0, do_sample)
                    history[rows, total_lens.long()] = nxt.to(torch.int32)
                    total_lens += 1
                    picked, lost, refused = torch.stack(
                        [nxt, lost.long(), status.long().expand(B)]).tolist()
                    if refused[0]:
                        raise RuntimeError(f"the device refused part of a step (status {refused[0]:#x}, "
                                           "KVB_STATUS_*): no tokens are returned")
                    for b, t in enumerate(picked):
                        if done[b]:
                            continue
                        if lost[b]:
                            raise ValueError(f"no token is left for prompt {b}: its logits are all "
                                             "masked or not finite")
                        generated[b].append(int(t))
                        done[b] = eos is not None and int(t) == eos
                    t_first = t_first or time.perf_counter()
                    n_out = int(max(len(g) for g in generated))
                    if all(done) or n_out >= most:
                        break
                    step = extend_block_tables(tables, seq_lens, ones, free_blocks, num_free,
                                               self.allocator.num_blocks, B, seq_lens_out=seq_lens,
                                               num_free_out=num_free)
                    state["slots"], state["max_seq_len"] = step.slots, max(lens) + n_out
                    with torch.no_grad():
                        logits = self.model(input_ids=nxt[:, None], position_ids=step.positions[:, None],
                                            use_cache=False, logits_to_keep=1).logits[:, -1]
            finally:
                uninstall_paged_attention(self.model)
            t1 = time.perf_counter()
        finally:
            if before:
                status.bitwise_or_(before)
            self.allocator.free(reserved)
            self.allocator.free(forked)
        results = [GenerationResult(
            mode="paged_batch", prompt=p if isinstance(p, str) else "",
            output_text=self._decode_text(generated[b]), generated_tokens=len(generated[b]),
            ttft_ms=(t_first - t0) * 1e3, total_ms=(t1 - t0) * 1e3,
            tokens_per_sec=len(generated[b]) / max(t1 - t0, 1e-9),
            kv_reuse_ratio=cached[b] / max(lens[b], 1), prompt_tokens=lens[b],
            cached_tokens=cached[b], first_token_logits=first_logits[b].float().cpu().numpy(),
            generated_ids=generated[b]) for b, p in enumerate(prompts)]
        for ids in all_ids:
            self._store_prompt_chunks(ids)
        return results

    def _write_blocks(self, blocks: List[int], places: List[int], keys: torch.Tensor,
                      values: torch.Tensor) -> None:
        """The 16-token pieces ``places`` of ``[L, H, P, D]`` K/V into ``blocks`` of every layer;
        slots past P repeat the last token."""
        bs = self._block_size
        at = torch.tensor(places, device=keys.device)[:, None] * bs + torch.arange(bs, device=keys.device)
        at = at.flatten().clamp(max=keys.shape[2] - 1)
        for layer in range(keys.shape[0]):
            self.allocator.write_chunk(layer, blocks, keys[layer][:, at], values[layer][:, at])

    def _prefill_suffix(self, ids: TokenIds, keys, values, reuse: int):
        """The prompt's tokens from ``reuse`` on over its reused prefix: the last logits
        ``[V]`` and the cache's layers."""
        from transformers import DynamicCache
        cache = (self._cache_from(keys[:, :, :reuse].contiguous(), values[:, :, :reuse].contiguous())
                 if reuse else DynamicCache())
        x = torch.tensor([ids[reuse:]], dtype=torch.long, device=self.device)
        pos = torch.arange(reuse, len(ids), device=self.device)[None]
        out = self._forward(x, pos, cache)
        return out.logits[0, -1], self._layers(out.past_key_values)

    def _token_masks(self, allowed: List[Optional[Sequence[int]]], vocab: int) -> torch.Tensor:
        """Bit masks ``[B, ceil(vocab / 32)]`` of the ids each row may take (None: any)."""
        words = -(-vocab // 32)
        bits = torch.zeros(len(allowed), words * 32, dtype=torch.int64)
        for row, ids in zip(bits, allowed):
            if ids is None:
                row.fill_(1)
                continue
            at = torch.as_tensor(list(ids), dtype=torch.long)
            if at.numel() and not 0 <= int(at.min()) <= int(at.max()) < vocab:
                raise ValueError(f"allowed token ids must lie in [0, {vocab})")
            row[at] = 1
        masks = (bits.view(len(allowed), words, 32) << torch.arange(32)).sum(-1)
        return (masks - ((masks >> 31) << 32)).to(torch.int32).to(self.device)

    def paged_stats(self) -> dict:
        """``paged_stats`` (``cpu_engine.py:514-522``)."""
        return {"block_utilization": self.allocator.utilization(),
                "free_blocks": self.allocator.free_blocks,
                "used_blocks": self.allocator.used_blocks,
                "num_blocks": self.allocator.num_blocks,
                "loaded_chunks": self.chunk_mapper.loaded_chunks(),
                "blocks_used_by_chunks": self.chunk_mapper.blocks_used_by_chunks()}


# the reference's name for it
CPUPagedEngine = PagedEngine
