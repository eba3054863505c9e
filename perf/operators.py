"""Cases of the operators that carry one decode step of a batch of requests over the
16-token block pool: the step's block tables and slot map, the new tokens' K/V written
into the pool, the attention of each request's new token over its blocks, and the logits
with penalties, biases and a grammar mask.

``run`` computes them from elementary torch operations, or, where ``own`` is true, by the
framework's calls.  Shapes are the framework's own (Qwen2.5-3B heads 16/2, D 128,
vocabulary 151936; the 64/8-head long prefix; 16-token blocks; 128-token int8 chunks) or
generic ones in the ranges between.
"""

import math

import torch

own = False

BLOCK = 16
CHUNK_BLOCKS = 8        # an int8 chunk is 128 tokens: its blocks share the V scales
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EL = {"bf16": 2, "fp16": 2, "fp32": 4}


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, evenly spread over their logarithm."""
    if n == 1:
        return [hi]
    a, b = math.log(max(lo, 1)), math.log(max(hi, 1))
    out = [int(round(math.exp(a + (b - a) * i / (n - 1)))) for i in range(n)]
    return [max(lo, min(hi, x)) for x in out]


def _lens(case):
    """Cached tokens of each request; ``idle`` rows of the batch hold no request."""
    n, idle = case["batch"], case.get("idle", 0)
    return _spread(n - idle, case["len_lo"], case["len_hi"]) + [0] * idle


def _new_lens(case):
    """New tokens of each request: one for a decode row, a suffix for a prefill row."""
    p = case["prefill_rows"]
    return [1] * (case["batch"] - p - case["idle"]) + \
        (_spread(p, case["new_lo"], case["new_hi"]) if p else []) + [0] * case["idle"]


def _cdiv(a, b):
    return -(-a // b)


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # the smallest step: a few requests decode one token each, every call latency
        dict(name="tables_decode_b8", op="tables", batch=8, len_lo=40, len_hi=1500, prefill_rows=0,
             new_lo=1, new_hi=1, idle=1),
        # a serving step that mixes decode rows with reuse prefills' suffixes
        dict(name="tables_mixed_b256", op="tables", batch=256, len_lo=1, len_hi=20000,
             prefill_rows=56, new_lo=17, new_hi=4099, idle=3),
        # one layer's new K/V of a decode batch
        dict(name="append_decode_b64_h8", op="append", tokens=64, heads=8, dim=128, dtype="bf16",
             skip=0, layout="thd"),
        # one layer's K/V of packed suffix prefills, straight from the projections
        dict(name="append_prefill_t8192_h8", op="append", tokens=8192, heads=8, dim=128,
             dtype="bf16", skip=0, layout="thd"),
        # odd token count, MHA heads of D 96, a model cache's [heads, tokens] storage, padding
        dict(name="append_odd_t1777_h32_d96", op="append", tokens=1777, heads=32, dim=96,
             dtype="fp16", skip=29, layout="htd"),
        # a lone short request: launch latency
        dict(name="attn_b1_short", op="attn", batch=1, q_heads=16, kv_heads=2, dim=128,
             dtype="bf16", pool="bf16", len_lo=333, len_hi=333),
        # the framework's decode batch: 8 prompts of 4096 tokens, 16/2 heads
        dict(name="attn_b8_4096", op="attn", batch=8, q_heads=16, kv_heads=2, dim=128,
             dtype="bf16", pool="bf16", len_lo=4096, len_hi=4097),
        # continuous batching: ragged lengths up to 16 K, an idle row
        dict(name="attn_ragged_b64_16k", op="attn", batch=64, q_heads=32, kv_heads=8, dim=128,
             dtype="bf16", pool="bf16", len_lo=700, len_hi=16381, idle=1),
        # the int8 chunk cache read in place: 64/8 heads over 32 K reused tokens
        dict(name="attn_int8_b4_32k", op="attn", batch=4, q_heads=64, kv_heads=8, dim=128,
             dtype="bf16", pool="int8", len_lo=32768, len_hi=32768),
        # MHA of D 96 in fp16, many requests, from one token on
        dict(name="attn_mha_d96_b24", op="attn", batch=24, q_heads=32, kv_heads=32, dim=96,
             dtype="fp16", pool="fp16", len_lo=1, len_hi=2051),
        # one request's logits, all of the processing on
        dict(name="logits_b1", op="logits", batch=1, vocab=151936, dtype="bf16", history=1200,
             bias=24, mask=True, penalties=True),
        # a large batch's logits
        dict(name="logits_b192", op="logits", batch=192, vocab=151936, dtype="bf16", history=2500,
             bias=64, mask=True, penalties=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "append", "attn", "attn", "attn", "logits"])
    if op == "tables":
        batch = _log(rng, 1, 256)
        rows = rng.choice([0, rng.randint(0, batch)])
        rows = min(rows, 56)
        hi = _log(rng, 2, 20000)
        new_hi = _log(rng, 2, 4099)
        return dict(op=op, batch=batch, len_lo=rng.randint(0, hi), len_hi=hi, prefill_rows=rows,
                    new_lo=rng.randint(1, new_hi), new_hi=new_hi,
                    idle=rng.randint(0, min(5, max(0, batch - rows - 1))))
    if op == "append":
        dim = rng.choice([64, 96, 128])
        heads = rng.choice([1, 2, 3, 4, 8, 16, 32])
        tokens = _log(rng, 1, max(2, 8192 * 8 * 128 // (heads * dim)))
        tokens = min(tokens, 8192)
        return dict(op=op, tokens=tokens, heads=heads, dim=dim, dtype=rng.choice(["bf16", "fp16"]),
                    skip=rng.randint(0, min(40, tokens - 1)), layout=rng.choice(["thd", "htd"]))
    if op == "attn":
        dtype = rng.choice(["bf16", "fp16"])
        heads = rng.choice([1, 2, 3, 4, 8, 16, 32])
        group = rng.choice([1, 2, 3, 4, 7, 8, 12, 16] if heads <= 8 else [1, 2, 4])
        dim = rng.choice([64, 96, 128])
        hi = _log(rng, 1, 32768)
        batch = min(_log(rng, 1, 128), max(1, 300000 * 8 * 128 // (hi * heads * dim)))
        idle = rng.randint(0, min(3, batch - 1))
        return dict(op=op, batch=batch, q_heads=heads * group, kv_heads=heads, dim=dim, dtype=dtype,
                    pool=rng.choice([dtype, dtype, "int8"]), len_lo=rng.randint(max(1, hi // 20), hi),
                    len_hi=hi, idle=idle)
    return dict(op="logits", batch=_log(rng, 1, 160), vocab=_log(rng, 1000, 151936),
                dtype=rng.choice(["bf16", "fp16", "fp32"]) if rng.random() < 0.5 else "bf16",
                history=_log(rng, 1, 2500), bias=rng.choice([0, 1, rng.randint(2, 64)]),
                mask=rng.random() < 0.7, penalties=rng.random() < 0.8)


# ── inputs ───────────────────────────────────────────────────────────────────

def _tables(nblk, width, ids):
    """Block tables [B, width] from the blocks of each row and a shuffled list of ids."""
    n = torch.tensor(nblk, device=ids.device)
    col = torch.arange(width, device=ids.device)[None]
    start = (torch.cumsum(n, 0) - n)[:, None]
    at = (start + col).clamp(max=max(0, ids.numel() - 1))
    return torch.where(col < n[:, None], ids[at], 0).to(torch.int32).contiguous()


def _make_tables(case, g, dev):
    order = torch.randperm(case["batch"], generator=torch.Generator().manual_seed(g.initial_seed()))
    new = _new_lens(case)
    live = case["batch"] - case["idle"]
    lens = _spread(live, case["len_lo"], case["len_hi"]) + [0] * case["idle"]
    shuffled = torch.randperm(live, generator=torch.Generator().manual_seed(g.initial_seed() + 1))
    lens = [lens[i] for i in shuffled.tolist()] + lens[live:]
    lens, new = [lens[i] for i in order.tolist()], [new[i] for i in order.tolist()]
    have = [_cdiv(x, BLOCK) for x in lens]
    want = [_cdiv(x + y, BLOCK) for x, y in zip(lens, new)]
    need = sum(want) - sum(have)
    num_blocks = sum(want) + 100
    ids = torch.randperm(num_blocks, generator=g, device=dev).to(torch.int32)
    used = sum(have)
    return dict(case=case, block_tables=_tables(have, max(want) + 5, ids),
                seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev),
                new_lens=torch.tensor(new, dtype=torch.int32, device=dev),
                free_blocks=ids[used:].contiguous(),
                num_free=torch.tensor([need + 90], dtype=torch.int32, device=dev),
                num_blocks=num_blocks, tokens=sum(new))


def _make_append(case, g, dev):
    T, H, D, dt = case["tokens"], case["heads"], case["dim"], _DT[case["dtype"]]
    num_blocks = _cdiv(T, BLOCK) * 5 // 4 + 3
    pool = torch.randn(num_blocks, 2, H, BLOCK, D, generator=g, device=dev).to(dt)
    shape = (2, T, H, D) if case["layout"] == "thd" else (2, H, T, D)
    kv = torch.randn(*shape, generator=g, device=dev).to(dt)
    if case["layout"] == "htd":
        kv = kv.transpose(1, 2)
    # tokens of one request fill blocks in turn; requests are short runs of them
    blocks = torch.randperm(num_blocks, generator=g, device=dev)
    t = torch.arange(T, device=dev)
    slots = (blocks[t // BLOCK] * BLOCK + t % BLOCK).to(torch.int32)
    if case["skip"]:
        off = torch.randperm(T, generator=g, device=dev)[:case["skip"]]
        slots[off] = -1
    return dict(case=case, kv_pool=pool, k_new=kv[0], v_new=kv[1], slots=slots)


def _make_attn(case, g, dev):
    B, Hq, H, D = case["batch"], case["q_heads"], case["kv_heads"], case["dim"]
    dt = _DT[case["dtype"]]
    order = torch.randperm(B, generator=torch.Generator().manual_seed(g.initial_seed()))
    lens = _lens(case)
    lens = [lens[i] for i in order.tolist()]
    nblk = [_cdiv(x, BLOCK) for x in lens]
    num_blocks = _cdiv(sum(nblk) + 9, CHUNK_BLOCKS) * CHUNK_BLOCKS
    ids = torch.randperm(num_blocks, generator=g, device=dev).to(torch.int32)
    s = dict(case=case, block_tables=_tables(nblk, max(nblk) + 2, ids),
             seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), k_scale=None, v_scale=None)
    # queries somewhat larger than keys: attention that prefers some tokens
    s["q"] = (1.5 * torch.randn(B, Hq, 1, D, generator=g, device=dev)).to(dt)
    if case["pool"] != "int8":
        s["kv_pool"] = torch.randn(num_blocks, 2, H, BLOCK, D, generator=g, device=dev,
                                   dtype=torch.float32 if num_blocks < 4096 else dt).to(dt)
        return s
    # int8 chunks of 128 tokens: K with a scale per token, V with one per channel and chunk
    n = num_blocks // CHUNK_BLOCKS
    kv = torch.randn(n, CHUNK_BLOCKS, 2, H, BLOCK, D, generator=g, device=dev, dtype=torch.float16)
    ks = kv[:, :, 0].abs().amax(-1) / 127                                # [n, 8, H, 16]
    vs = kv[:, :, 1].abs().amax(3).amax(1, keepdim=True) / 127           # [n, 1, H, D]
    pool = torch.empty(kv.shape, dtype=torch.int8, device=dev)
    pool[:, :, 0] = (kv[:, :, 0] / ks[..., None]).round().clamp(-128, 127).to(torch.int8)
    pool[:, :, 1] = (kv[:, :, 1] / vs[:, :, :, None]).round().clamp(-128, 127).to(torch.int8)
    s["kv_pool"] = pool.view(num_blocks, 2, H, BLOCK, D)
    s["k_scale"] = ks.reshape(num_blocks, H, BLOCK).contiguous()
    s["v_scale"] = vs.expand(n, CHUNK_BLOCKS, H, D).reshape(num_blocks, H, D).contiguous()
    return s


def _make_logits(case, g, dev):
    B, V, L = case["batch"], case["vocab"], case["history"]
    s = dict(case=case, logits=(3 * torch.randn(B, V, generator=g, device=dev)).to(_DT[case["dtype"]]))
    for name in ("token_ids", "prompt_lens", "total_lens", "repetition_penalty",
                 "frequency_penalty", "presence_penalty", "bias_ids", "bias_values", "allowed_mask"):
        s[name] = None
    cpu = torch.Generator().manual_seed(g.initial_seed())
    if case["penalties"]:
        # text repeats itself: token ids from a skewed distribution
        u = torch.rand(B, L, generator=g, device=dev)
        s["token_ids"] = (u.pow(4) * (V - 1)).to(torch.int32)
        total = torch.tensor(_spread(B, max(1, L // 5), L))[torch.randperm(B, generator=cpu)]
        s["total_lens"] = total.to(torch.int32).to(dev)
        s["prompt_lens"] = (total * 2 // 3).to(torch.int32).to(dev)
        s["repetition_penalty"] = 1.0 + 0.4 * torch.rand(B, generator=g, device=dev)
        s["frequency_penalty"] = 0.5 * torch.rand(B, generator=g, device=dev)
        s["presence_penalty"] = torch.rand(B, generator=g, device=dev) - 0.2
    if case["bias"]:
        n = min(case["bias"], V)
        base = torch.randperm(V, generator=g, device=dev)[:n].to(torch.int32)
        shift = torch.randint(0, V, (B, 1), generator=g, device=dev, dtype=torch.int32)
        s["bias_ids"] = ((base[None] + shift) % V).to(torch.int32).contiguous()
        s["bias_values"] = 4 * torch.randn(B, n, generator=g, device=dev)
    if case["mask"]:
        # a grammar leaves runs of the vocabulary open
        words = _cdiv(V, 32)
        r = torch.randint(-2**31, 2**31, (B, words), generator=g, device=dev)
        keep = torch.rand(B, words, generator=g, device=dev)
        r = torch.where(keep < 0.5, 0, torch.where(keep < 0.6, -1, r))
        s["allowed_mask"] = r.to(torch.int32)
    s["temperature"] = 0.6 + 0.8 * torch.rand(B, generator=g, device=dev)
    return s


_MAKE = {"tables": _make_tables, "append": _make_append, "attn": _make_attn, "logits": _make_logits}


def prepare(case, seed):
    dev = torch.device("cuda")
    return _MAKE[case["op"]](case, torch.Generator(device=dev).manual_seed(seed), dev)


# ── the operators ────────────────────────────────────────────────────────────

def _plain_tables(s):
    tab, lens, new, free = s["block_tables"], s["seq_lens"].long(), s["new_lens"].long(), s["free_blocks"]
    B, width = tab.shape
    have, want = (lens + BLOCK - 1) // BLOCK, (lens + new + BLOCK - 1) // BLOCK
    need = want - have
    cum = torch.cumsum(need, 0)
    n_free = s["num_free"].long()
    fits = (want <= width) & ((need == 0) | (cum <= n_free))
    col = torch.arange(width, device=tab.device)[None]
    fresh = fits[:, None] & (col >= have[:, None]) & (col < want[:, None])
    at = n_free - 1 - ((cum - need)[:, None] + col - have[:, None])       # popped from the end
    tab.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], tab))
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=tab.device), torch.cumsum(new, 0)])
    t = torch.arange(s["tokens"], device=tab.device)
    row = torch.searchsorted(cu[1:], t, right=True).clamp(max=B - 1)
    pos = lens[row] + t - cu[row]
    slot = tab[row, (pos // BLOCK).clamp(max=width - 1)].long() * BLOCK + pos % BLOCK
    live = fits[row] & (t < cu[-1])
    taken = torch.where(fits, need, 0).sum().reshape(1)
    return (torch.where(live, slot, -1).to(torch.int32), torch.where(live, pos, 0),
            cu.to(torch.int32), torch.where(fits, lens + new, lens).to(torch.int32),
            (n_free - taken).to(torch.int32), tab)


def _plain_append(s):
    pool, keep = s["kv_pool"], s["slots"] >= 0
    at = s["slots"][keep].long()
    block, off = at // BLOCK, at % BLOCK
    pool[block, 0, :, off] = s["k_new"][keep]
    pool[block, 1, :, off] = s["v_new"][keep]
    return pool


def _plain_attn(s):
    q, tab, lens = s["q"], s["block_tables"].long(), s["seq_lens"].long()
    B, Hq, _, D = q.shape
    H, width = s["kv_pool"].shape[2], tab.shape[1]
    S = width * BLOCK
    kv = s["kv_pool"][tab]                                               # [B, w, 2, H, 16, D]
    k = kv[:, :, 0].permute(0, 2, 1, 3, 4).reshape(B, H, S, D).float()
    v = kv[:, :, 1].permute(0, 2, 1, 3, 4).reshape(B, H, S, D).float()
    del kv
    if s["k_scale"] is not None:
        k = k * s["k_scale"][tab].permute(0, 2, 1, 3).reshape(B, H, S, 1).float()
        v = v * s["v_scale"][tab].permute(0, 2, 1, 3).float().repeat_interleave(BLOCK, 2)
    seen = torch.arange(S, device=q.device)[None] < lens[:, None]
    k = torch.where(seen[:, None, :, None], k, 0.0)
    v = torch.where(seen[:, None, :, None], v, 0.0)
    qs = q.reshape(B, H, Hq // H, D).float() * (1.0 / math.sqrt(D))
    x = torch.matmul(qs, k.transpose(2, 3))
    x = torch.where(seen[:, None, None, :], x, -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = torch.log(total) + torch.where(total > 0, top, 0.0)
    return o.reshape(B, Hq, 1, D).to(q.dtype), lse.reshape(B, Hq, 1)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    if s["token_ids"] is not None:
        ids = s["token_ids"].long()
        at = torch.arange(ids.shape[1], device=x.device)[None]
        here = at < s["total_lens"][:, None]
        made = here & (at >= s["prompt_lens"][:, None])
        zero = torch.zeros(B, V, dtype=torch.int32, device=x.device)
        seen = zero.scatter_add(1, ids, here.to(torch.int32)) > 0
        count = zero.scatter_add(1, ids, made.to(torch.int32)).float()
        r = s["repetition_penalty"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency_penalty"][:, None] * count
        x = x - s["presence_penalty"][:, None] * (count > 0).float()
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    x = x / s["temperature"][:, None]
    if s["allowed_mask"] is not None:
        v = torch.arange(V, device=x.device)
        bit = (s["allowed_mask"][:, v // 32] >> (v % 32).to(torch.int32)) & 1
        x = torch.where(bit == 1, x, -math.inf)
    return x


_PLAIN = {"tables": _plain_tables, "append": _plain_append, "attn": _plain_attn, "logits": _plain_logits}


def _own_tables(s):
    from kvboost_b200.paged_decode import extend_block_tables
    step = extend_block_tables(s["block_tables"], s["seq_lens"], s["new_lens"], s["free_blocks"],
                               s["num_free"], s["num_blocks"], s["tokens"])
    return (step.slots, step.positions, step.cu_new, step.seq_lens, step.num_free, s["block_tables"])


def _own_append(s):
    from kvboost_b200.paged_decode import append_paged_kv
    append_paged_kv(s["k_new"], s["v_new"], s["kv_pool"], s["slots"])
    return s["kv_pool"]


def _own_attn(s):
    from kvboost_b200.paged_decode import paged_decode_attention
    return paged_decode_attention(s["q"], s["kv_pool"], s["block_tables"], s["seq_lens"],
                                  k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_logits(s):
    from kvboost_b200.logits import process_logits
    return process_logits(
        s["logits"], token_ids=s["token_ids"], prompt_lens=s["prompt_lens"],
        total_lens=s["total_lens"], repetition_penalty=s["repetition_penalty"],
        frequency_penalty=s["frequency_penalty"], presence_penalty=s["presence_penalty"],
        bias_ids=s["bias_ids"], bias_values=s["bias_values"], allowed_mask=s["allowed_mask"],
        temperature=s["temperature"])


_OWN = {"tables": _own_tables, "append": _own_append, "attn": _own_attn, "logits": _own_logits}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    op = case["op"]
    if op == "tables":
        B, T = case["batch"], sum(_new_lens(case))
        fresh = _cdiv(T, BLOCK)
        # lengths in and out, counts, popped ids and their table entries, slots and positions
        return {"bytes": 4 * (4 * B + 3) + 8 * fresh + 12 * T + 4 * B, "flops": 0}
    if op == "append":
        n = case["tokens"] - case["skip"]
        return {"bytes": 4 * n * case["heads"] * case["dim"] * _EL[case["dtype"]] + 4 * case["tokens"],
                "flops": 0}
    if op == "attn":
        lens = _lens(case)
        B, Hq, H, D, T = case["batch"], case["q_heads"], case["kv_heads"], case["dim"], sum(lens)
        nblk = sum(_cdiv(x, BLOCK) for x in lens)
        io = 2 * B * Hq * D * 2 + 4 * B * Hq + 4 * nblk + 4 * B
        if case["pool"] == "int8":
            # codes and a K scale per token; V scales per channel of each block
            kv = 2 * T * H * D + 2 * T * H + 2 * nblk * H * D
        else:
            kv = 4 * T * H * D
        return {"bytes": io + kv, "flops": 4 * Hq * D * T}
    B, V = case["batch"], case["vocab"]
    n = B * V * (_EL[case["dtype"]] + 4) + 4 * B
    if case["penalties"]:
        n += 4 * sum(_spread(B, max(1, case["history"] // 5), case["history"])) + 20 * B
    n += 8 * B * case["bias"]
    if case["mask"]:
        n += 4 * B * _cdiv(V, 32)
    return {"bytes": n, "flops": 6 * B * V}


# ── the definitions in 64 bits ───────────────────────────────────────────────

def _exact_append(s):
    pool = s["kv_pool"].double()
    flat = pool.permute(0, 3, 1, 2, 4).reshape(-1, 2, pool.shape[2], pool.shape[4])
    for i, slot in enumerate(s["slots"].tolist()):
        if slot >= 0:
            flat[slot, 0] = s["k_new"][i].double()
            flat[slot, 1] = s["v_new"][i].double()
    n, _, H, _, D = pool.shape
    return flat.reshape(n, BLOCK, 2, H, D).permute(0, 2, 3, 1, 4).contiguous()


def _exact_attn(s):
    q = s["q"].double()
    B, Hq, _, D = q.shape
    H = s["kv_pool"].shape[2]
    o = torch.zeros_like(q)
    lse = torch.full((B, Hq, 1), -math.inf, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["seq_lens"].tolist()):
        if n == 0:
            continue
        blocks = s["block_tables"][b, :_cdiv(n, BLOCK)].long()
        kv = s["kv_pool"][blocks].double()
        k, v = kv[:, 0], kv[:, 1]                                        # [w, H, 16, D]
        if s["k_scale"] is not None:
            k = k * s["k_scale"][blocks].double()[..., None]
            v = v * s["v_scale"][blocks].double()[:, :, None]
        for h in range(H):
            kh, vh = k[:, h].reshape(-1, D)[:n], v[:, h].reshape(-1, D)[:n]
            rows = slice(h * (Hq // H), (h + 1) * (Hq // H))
            x = q[b, rows, 0] @ kh.T / math.sqrt(D)
            lse[b, rows, 0] = torch.logsumexp(x, -1)
            o[b, rows, 0] = torch.softmax(x, -1) @ vh
    return o, lse


def _exact_logits(s):
    x = s["logits"].double()
    for b in range(x.shape[0]):
        if s["token_ids"] is not None:
            p, n = int(s["prompt_lens"][b]), int(s["total_lens"][b])
            row, r = x[b], s["repetition_penalty"][b].double()
            ids = torch.unique(s["token_ids"][b, :n].long())
            old = row[ids]
            row[ids] = torch.where(old > 0, old / r, old * r)
            made, times = torch.unique(s["token_ids"][b, p:n].long(), return_counts=True)
            row[made] -= s["frequency_penalty"][b].double() * times + s["presence_penalty"][b].double()
        if s["bias_ids"] is not None:
            x[b].index_add_(0, s["bias_ids"][b].long(), s["bias_values"][b].double())
    x /= s["temperature"].double()[:, None]
    if s["allowed_mask"] is not None:
        shifts = torch.arange(32, device=x.device)
        bits = (s["allowed_mask"].long()[:, :, None] >> shifts) & 1
        x[bits.flatten(1)[:, :x.shape[1]] == 0] = -math.inf
    return x


def exact(case, seed):
    if case["op"] == "tables":
        return None                 # whole numbers
    s = prepare(case, seed)
    return {"append": _exact_append, "attn": _exact_attn, "logits": _exact_logits}[case["op"]](s)
