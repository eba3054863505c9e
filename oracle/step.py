"""64-bit restatement of a batched decode step over the block pool: block tables and
slots (the allocator's order, ``cpu_paged/block_allocator.py:85-96``), the K/V append, the
attention of one token per request, and the logits' processing.  Test infrastructure."""

import numpy as np

BLOCK = 16
BAD_BLOCK, BAD_LENGTH, POOL_EMPTY = 16, 32, 128


def extend_tables(tables, seq_lens, new_lens, free, num_free, num_blocks, max_new):
    """Row by row.  Returns (tables, slots, positions, cu, seq_lens, num_free, status)."""
    tables = np.array(tables, dtype=np.int64)
    B, width = tables.shape
    num_free = min(max(int(num_free), 0), len(free))
    slots = np.full(max_new, -1, dtype=np.int64)
    pos = np.zeros(max_new, dtype=np.int64)
    cu, out, status = [0], [], 0
    place = asked = taken = 0
    for b in range(B):
        l, n = int(seq_lens[b]), int(new_lens[b])
        out.append(l)
        if l < 0 or n < 0 or n > max_new:
            status |= BAD_LENGTH
            cu.append(min(place, max_new))
            continue
        first = place
        place += n
        cu.append(min(place, max_new))
        if l + n > width * BLOCK or (n and place > max_new):
            status |= BAD_LENGTH
            continue
        have, want = -(-l // BLOCK), -(-(l + n) // BLOCK)
        before = asked
        asked += want - have
        if want > have and asked > num_free:
            status |= POOL_EMPTY
            continue
        for i in range(want - have):
            tables[b, have + i] = free[num_free - 1 - before - i]
        taken += want - have
        out[b] = l + n
        for t in range(n):
            p = l + t
            pos[first + t] = p
            blk = tables[b, p // BLOCK]
            if 0 <= blk < num_blocks:
                slots[first + t] = blk * BLOCK + p % BLOCK
            else:
                status |= BAD_BLOCK
    return tables, slots, pos, np.array(cu), np.array(out), num_free - taken, status


def append(pool, k, v, slots):
    """pool [n, 2, H, 16, D]; k, v [T, H, D]."""
    pool = np.array(pool)
    for t, s in enumerate(slots):
        if 0 <= s < pool.shape[0] * BLOCK:
            pool[s // BLOCK, 0, :, s % BLOCK] = k[t]
            pool[s // BLOCK, 1, :, s % BLOCK] = v[t]
    return pool


def gather(pool, table, n, k_scale=None, v_scale=None):
    """K, V [H, n, D] in float64 of one row; blocks outside the pool are zeros."""
    nb, _, H, _, D = pool.shape
    K, V = np.zeros((H, n, D)), np.zeros((H, n, D))
    for i in range(-(-n // BLOCK)):
        b, m = int(table[i]), min(BLOCK, n - i * BLOCK)
        if not 0 <= b < nb:
            continue
        k, v = pool[b, 0].astype(np.float64), pool[b, 1].astype(np.float64)
        if k_scale is not None:
            k = k * k_scale[b].astype(np.float64)[:, :, None]
            v = v * v_scale[b].astype(np.float64)[:, None, :]
        K[:, i * BLOCK:i * BLOCK + m], V[:, i * BLOCK:i * BLOCK + m] = k[:, :m], v[:, :m]
    return K, V


def decode_attention(q, pool, tables, lens, scale, k_scale=None, v_scale=None):
    """q [B, Hq, D].  Returns o, lse and, for error bounds, ``a`` = sum_t w_t |v_t| (as o) and, as
    lse, ``x`` = max_t scale * sum_d |q_d k_td|, ``vmax`` = max|v|, ``kq`` = max_t scale * max_d|q| *
    sum_d |k_td| and ``kb`` = scale * sum_d|q| * max|k|."""
    B, Hq, D = q.shape
    H = pool.shape[2]
    g = Hq // H
    o, a = np.zeros((B, Hq, D)), np.zeros((B, Hq, D))
    lse = np.full((B, Hq), -np.inf)
    x, vmax, kq, kb = (np.zeros((B, Hq)) for _ in range(4))
    cap = tables.shape[1] * BLOCK
    for b in range(B):
        n = min(int(lens[b]), cap)
        if n <= 0:
            continue
        K, V = gather(pool, tables[b], n, k_scale, v_scale)
        for h in range(Hq):
            k, v, qq = K[h // g], V[h // g], q[b, h].astype(np.float64)
            s = k @ qq * scale
            top = s.max()
            p = np.exp(s - top)
            o[b, h] = p @ v / p.sum()
            a[b, h] = p @ np.abs(v) / p.sum()
            lse[b, h] = top + np.log(p.sum())
            x[b, h] = scale * (np.abs(k) @ np.abs(qq)).max()
            vmax[b, h] = np.abs(v).max()
            kq[b, h] = scale * np.abs(qq).max() * np.abs(k).sum(-1).max()
            kb[b, h] = scale * np.abs(qq).sum() * np.abs(k).max()
    return o, lse, a, x, vmax, kq, kb


def logits(x, token_ids=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None,
           presence=None, bias_ids=None, bias_values=None, mask=None, temperature=None):
    """Row by row, entry by entry."""
    x = np.array(x, dtype=np.float64)
    B, V = x.shape
    for b in range(B):
        if token_ids is not None:
            n = min(max(int(total_lens[b]), 0), token_ids.shape[1])
            p = min(max(int(prompt_lens[b]), 0), n) if prompt_lens is not None else 0
            seen, count = set(), {}
            for i in range(n):
                t = int(token_ids[b, i])
                if 0 <= t < V:
                    seen.add(t)
                    if i >= p:
                        count[t] = count.get(t, 0) + 1
            for t in seen:
                if repetition is not None:
                    r = float(repetition[b])
                    x[b, t] = x[b, t] / r if x[b, t] > 0 else x[b, t] * r
                c = count.get(t, 0)
                if frequency is not None:
                    x[b, t] -= float(frequency[b]) * c
                if presence is not None and c:
                    x[b, t] -= float(presence[b])
        if bias_ids is not None:
            for t, w in zip(bias_ids[b], bias_values[b]):
                if 0 <= t < V:
                    x[b, t] += float(w)
        if temperature is not None:
            x[b] /= max(float(temperature[b]), float(np.float32(1e-5)))
        if mask is not None:
            words = np.asarray(mask[b]).astype(np.int64) & 0xffffffff
            v = np.arange(V)
            x[b, (words[v // 32] >> (v % 32)) & 1 == 0] = -np.inf
    return x
