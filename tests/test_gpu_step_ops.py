"""GPU: the operators of a batched decode step over the block pool, each against its
64-bit restatement (``oracle/step.py``), and all of them together as a step.

Tolerances.  u = 2^-24 is float32's half step.  Attention: a score is a dot of D products
in float32, off by at most (D + 6) u times scale * sum|q k| (``x``).  The exponential and the
scale's product add 2^-21 of relative error, so a weight is off by e = (D + 6) u x + 2^-20
relative.  The sums of n weights add n u; the weights themselves are carried in two 16-bit
halves (2^-16 of relative error in bfloat16; in float16 2^-21 and at worst 2^-24 absolute, of a
largest weight >= 1).  So |o - o64| <= half a step of the output's type times |o| + (2 e + 2 n u +
2^-16) a + n 2^-23 max|v| with a = sum w|v|, and |lse - lse64| <= e + 2 n u + 2^-20 + 2 u |lse|.

Over int8 pools a code c is multiplied as c + 128 <= 255 and the bias taken out of the sum, so
a score's terms are at most 255 scales = 2.1 max|k| times |q| (``kb``) instead of |q k|: e has
(D + 6) u (x + 2.1 kb); the query is rounded to multiples of 2^-25 of its row maximum (``kq`` *
2^-24 with the normalisation).  The same bias in V adds 18 roundings of 2.1 max|v|: 48 u max|v|.
Under bfloat16 the weights are single float16 numbers: 2^-11 a instead of 2^-16 a.
"""

import math

import numpy as np
import pytest
import torch

from oracle import step as ostep

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 (B200) device")
    from kvboost_b200 import ops
    ops.read_status(torch.device("cuda"))
    yield
    assert ops.read_status(torch.device("cuda")) == 0


def _status():
    from kvboost_b200 import ops
    return ops.read_status(torch.device("cuda"))


# ── block tables ─────────────────────────────────────────────────────────────

def _run_tables(tables, lens, new, free, num_free, num_blocks, max_new, in_place=False):
    from kvboost_b200.paged_decode import extend_block_tables
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)  # noqa: E731
    tab, ln, nf = i32(tables), i32(lens), i32([num_free])
    kw = dict(seq_lens_out=ln, num_free_out=nf) if in_place else {}
    s = extend_block_tables(tab, ln, i32(new), i32(free), nf, num_blocks, max_new, **kw)
    if in_place:
        assert s.seq_lens is ln and s.num_free is nf
    torch.cuda.synchronize()
    return [t.cpu().numpy() for t in (tab, s.slots, s.positions, s.cu_new, s.seq_lens)] + \
        [int(s.num_free.item())]


def _tables_case(rng, B, width, max_len, max_new_len, spare=50):
    lens = rng.integers(0, max_len + 1, B)
    new = rng.integers(0, max_new_len + 1, B)
    have = -(-lens // 16)
    need = int((-(-(lens + new) // 16) - have).sum())
    num_blocks = int(have.sum()) + need + spare
    ids = rng.permutation(num_blocks)
    tables, at = np.full((B, width), -7, dtype=np.int64), 0
    for b in range(B):
        m = min(int(have[b]), width)
        tables[b, :m] = ids[at:at + m]
        at += m
    return tables, lens, new, ids[at:], num_blocks, need


@pytest.mark.parametrize("B,max_len,max_new", [(1, 0, 1), (1, 16, 40), (3, 31, 17), (8, 1000, 1),
                                               (33, 700, 300), (257, 90, 65), (1025, 40, 20),
                                               (8192, 33, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_extend_tables(B, max_len, max_new, in_place):
    rng = np.random.default_rng(B * 7 + max_new)
    tables, lens, new, free, nblk, need = _tables_case(rng, B, -(-(max_len + max_new) // 16) + 1,
                                                       max_len, max_new)
    for extra in (0, 37):
        total = int(new.sum()) + extra
        nfree = need + (extra > 0)
        want = ostep.extend_tables(tables, lens, new, free, nfree, nblk, total)
        got = _run_tables(tables, lens, new, free, nfree, nblk, total, in_place)
        assert want[-1] == 0
        for g, w in zip(got, want):
            assert np.array_equal(g, w)


def test_extend_tables_long_prefill():
    """65 537 tokens in one call, one row of 60 001."""
    rng = np.random.default_rng(2)
    lens, new = np.array([5, 0, 16, 100]), np.array([60001, 5535, 1, 0])
    free = rng.permutation(5000)
    tables = np.full((4, 4000), -1, dtype=np.int64)
    for b in range(4):
        tables[b, :8] = 5000 + b * 8 + np.arange(8)
    args = (tables, lens, new, free, 4900, 5100, 65537)
    for g, w in zip(_run_tables(*args), ostep.extend_tables(*args)):
        assert np.array_equal(g, w)


def test_extend_tables_refusals_leave_rows_alone():
    """Rows that do not fit: their length, table and slots stay as they were."""
    tables = np.arange(40).reshape(8, 5)
    lens = np.array([10, -1, 79, 20, 16, 0, 33, 16])
    new = np.array([10, 3, 2, -4, 40, 0, 1, 16])
    free = np.array([101, 102, 103, 104, 105, 106])
    for num_free in (6, 4, 3, 1, 0, -3, 900):
        for max_new in (200, 70, 60, 12):
            args = (tables, lens, new, free, num_free, 300, max_new)
            want = ostep.extend_tables(*args)
            got = _run_tables(*args)
            assert _status() == want[-1]
            for g, w in zip(got, want):
                assert np.array_equal(g, w), (num_free, max_new)


def test_extend_tables_bad_ids():
    """Table and free-list entries outside the pool give slot -1 and a status bit."""
    tables = np.array([[500, 0], [3, 0]])
    args = (tables, [3, 16], [2, 2], [7, -5], 2, 100, 4)
    want = ostep.extend_tables(*args)
    got = _run_tables(*args)
    assert _status() == want[-1] == ostep.BAD_BLOCK
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


def test_extend_tables_sliced_rows_and_no_tokens():
    from kvboost_b200.paged_decode import extend_block_tables
    big = torch.full((6, 32), 9, dtype=torch.int32, device=DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    s = extend_block_tables(big[1:4, 4:10], i32([16, 0, 1]), i32([1, 1, 0]), i32([50, 51, 52]),
                            i32([3]), 100, 2)
    assert s.slots.tolist() == [52 * 16, 51 * 16] and s.num_free.item() == 1
    want = torch.full((6, 32), 9, dtype=torch.int32)
    want[1, 5], want[2, 4] = 52, 51
    assert torch.equal(big.cpu(), want)
    s = extend_block_tables(big[1:4, 4:10], i32([16, 0, 1]), i32([0, 0, 0]), i32([]), i32([0]), 100, 0)
    assert s.slots.numel() == 0 and s.cu_new.tolist() == [0, 0, 0, 0]


# ── append ───────────────────────────────────────────────────────────────────

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D", [(1, 1, 64), (1, 8, 128), (5, 3, 96), (64, 2, 128), (333, 32, 96),
                                   (777, 5, 8), (40, 2, 256)])
@pytest.mark.parametrize("layout", ["thd", "htd", "bhsd_slice", "odd"])
def test_append(dtype, T, H, D, layout):
    from kvboost_b200.paged_decode import append_paged_kv
    g = torch.Generator().manual_seed(T * 31 + D)
    nb = T // 16 + 4
    pool = torch.randn(nb, 2, H, 16, D, generator=g).to(dtype)
    kv = torch.randn(2, T, H, D, generator=g).to(dtype)
    slots = torch.randperm(nb * 16, generator=g)[:T].to(torch.int32)
    slots[torch.rand(T, generator=g) < 0.2] = -1
    want = ostep.append(pool.float().numpy(), kv[0].float().numpy(), kv[1].float().numpy(), slots.numpy())
    if layout == "thd":
        k, v = kv.cuda()
    elif layout == "htd":
        k, v = (t.transpose(0, 1) for t in kv.transpose(1, 2).contiguous().cuda())
    elif layout == "bhsd_slice":      # the tail of a longer cache, K and V strided apart
        big = torch.zeros(1, H, T + 9, D, dtype=dtype, device=DEV)
        big[0, :, 9:] = kv[0].transpose(0, 1).cuda()
        k, v = big[0, :, 9:].transpose(0, 1), kv[1].cuda()
    else:                             # rows that start off a 16-byte boundary
        odd = torch.zeros(2, T, H, D + 1, dtype=dtype, device=DEV)
        odd[..., 1:] = kv.cuda()
        k, v = odd[0, ..., 1:], odd[1, ..., 1:]
    p = pool.cuda()
    append_paged_kv(k, v, p, slots.cuda())
    assert np.array_equal(p.float().cpu().numpy(), want)


def test_append_slots_outside_the_pool():
    from kvboost_b200.paged_decode import append_paged_kv
    pool = torch.zeros(3, 2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    kv = torch.ones(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    append_paged_kv(kv, kv, pool, torch.tensor([48, -2, 47, 2 ** 31 - 1], dtype=torch.int32, device=DEV))
    assert _status() == ostep.BAD_BLOCK
    assert pool.sum().item() == 2 * 2 * 64 and pool[2, :, :, 15].sum().item() == 2 * 2 * 64
    append_paged_kv(kv[:0], kv[:0], pool, torch.empty(0, dtype=torch.int32, device=DEV))


# ── attention ────────────────────────────────────────────────────────────────

def _pool(g, lens, H, D, dtype, int8, spare=5, poison=True):
    """A pool whose blocks belong to the rows in shuffled order; slots no row owns hold NaN
    (int8: extreme codes), table entries past a row's blocks hold ids far outside the pool."""
    nblk = [-(-n // 16) for n in lens]
    nb = sum(nblk) + spare
    ids = torch.randperm(nb, generator=g)
    width = max(1, max(nblk) + 2)
    tables = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
    kv = torch.randn(nb, 2, H, 16, D, generator=g)
    owned, at = torch.zeros(nb, 16, dtype=torch.bool), 0
    for b, n in enumerate(lens):
        mine = ids[at:at + nblk[b]]
        at += nblk[b]
        tables[b, :nblk[b]] = mine.to(torch.int32)
        for i, blk in enumerate(mine.tolist()):
            owned[blk, :min(16, n - 16 * i)] = True
    if not int8:
        pool = kv.to(dtype)
        if poison:
            pool.masked_fill_(~owned[:, None, None, :, None], float("nan"))
        return pool, tables, None, None
    ks = (kv[:, 0].abs().amax(-1) / 127).to(torch.float16)
    vs = (kv[:, 1].abs().amax(2) / 127).to(torch.float16)
    q = torch.empty(kv.shape, dtype=torch.int8)
    q[:, 0] = (kv[:, 0] / ks.float()[..., None]).round().clamp(-128, 127).to(torch.int8)
    q[:, 1] = (kv[:, 1] / vs.float()[:, :, None]).round().clamp(-128, 127).to(torch.int8)
    if poison:
        q.masked_fill_(~owned[:, None, None, :, None], -128)
        ks.masked_fill_(~owned[:, None], float("nan"))
    return q, tables, ks, vs


def _np(t):
    return None if t is None else t.float().numpy() if t.dtype != torch.int8 else t.numpy()


def _check_attention(o, lse, q, pool, tables, lens, scale, ks=None, vs=None):
    dtype, int8 = q.dtype, ks is not None
    D = q.shape[-1]
    want, wl, a, x, vmax, kq, kb = ostep.decode_attention(
        _np(q[:, :, 0]), _np(pool), tables.numpy(), lens, scale, _np(ks), _np(vs))
    n = np.minimum(np.maximum(np.asarray(lens), 0), tables.shape[1] * 16)[:, None]
    e = x * (D + 6) * U + 2.0 ** -20
    if int8:
        e = e + kb * 2.1 * (D + 6) * U + kq * 2.0 ** -24
    weights = 2.0 ** -11 if int8 and dtype == torch.bfloat16 else 2.0 ** -16
    half = torch.finfo(dtype).eps / 2
    small = torch.finfo(dtype).tiny
    bound = half * np.abs(want) + ((2 * e + 2 * n * U + weights)[..., None]) * a + \
        ((n * 2.0 ** -23 + (48 * U if int8 else 0.0)) * vmax)[..., None] + small
    got = o[:, :, 0].double().cpu().numpy()
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > bound
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want).max())
    if lse is not None:
        gl = lse[:, :, 0].double().cpu().numpy()
        empty = np.isinf(wl)
        assert np.array_equal(np.isneginf(gl), empty)
        lb = e + 2 * n * U + 2.0 ** -20 + 2 * U * np.abs(np.where(empty, 0, wl))
        assert (np.abs(np.where(empty, 0, gl) - np.where(empty, 0, wl)) <= lb).all()
    return want


def _attend(q, pool, tables, lens, ks=None, vs=None, **kw):
    from kvboost_b200.paged_decode import paged_decode_attention
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    return paged_decode_attention(c(q), c(pool), c(tables),
                                  torch.tensor(lens, dtype=torch.int32, device=DEV),
                                  k_scale=c(ks), v_scale=c(vs), **kw)


_LENS = {"one": [1], "block": [16], "edges": [0, 1, 15, 16, 17, 31, 32, 33, 0, 100],
         "long": [5003, 0, 1, 2048], "many": [(i * 37) % 200 for i in range(70)],
         "skew": [1] * 9 + [9001] + [40] * 20}


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("lens", list(_LENS))
@pytest.mark.parametrize("H,group", [(2, 8), (3, 1), (1, 5)])
def test_paged_decode(pool_kind, dtype, D, lens, H, group):
    ln = _LENS[lens]
    g = torch.Generator().manual_seed(D + len(ln) + H * 10 + group)
    pool, tables, ks, vs = _pool(g, ln, H, D, dtype, pool_kind == "int8")
    q = (1.5 * torch.randn(len(ln), H * group, 1, D, generator=g)).to(dtype)
    o, lse = _attend(q, pool, tables, ln, ks, vs)
    _check_attention(o, lse, q, pool, tables, ln, 1 / math.sqrt(D), ks, vs)


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
@pytest.mark.parametrize("H,group", [(1, 2), (2, 7), (1, 9), (2, 12), (2, 16), (1, 17), (1, 24), (1, 32),
                                     (1, 71), (16, 1), (8, 4)])
def test_paged_decode_groups(pool_kind, H, group):
    ln = [300, 0, 17, 1025]
    g = torch.Generator().manual_seed(H * 100 + group)
    pool, tables, ks, vs = _pool(g, ln, H, 128, torch.bfloat16, pool_kind == "int8")
    q = torch.randn(len(ln), H * group, 1, 128, generator=g).to(torch.bfloat16)
    o, lse = _attend(q, pool, tables, ln, ks, vs)
    _check_attention(o, lse, q, pool, tables, ln, 1 / math.sqrt(128), ks, vs)


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
@pytest.mark.parametrize("amp,scale", [(40.0, None), (1.0, 2.0), (0.0, None), (1e4, 1e-5), (1.0, -0.1),
                                       (3e-6, 3e4)])
def test_paged_decode_score_ranges(pool_kind, amp, scale):
    """Peaked rows (late maxima), a zero query, large and tiny queries under other scales."""
    ln = [2000, 129, 1]
    g = torch.Generator().manual_seed(11)
    pool, tables, ks, vs = _pool(g, ln, 2, 128, torch.bfloat16, pool_kind == "int8")
    q = (amp * torch.randn(3, 8, 1, 128, generator=g)).to(torch.bfloat16)
    o, lse = _attend(q, pool, tables, ln, ks, vs, softmax_scale=scale)
    _check_attention(o, lse, q, pool, tables, ln, abs(scale) * np.sign(scale) if scale else 1 / math.sqrt(128),
                     ks, vs) if scale is None or scale > 0 else _check_neg(o, lse, q, pool, tables, ln, scale, ks, vs)


def _check_neg(o, lse, q, pool, tables, lens, scale, ks, vs):
    """A negative scale is the positive one with the query negated."""
    _check_attention(o, lse, -q, pool, tables, lens, -scale, ks, vs)


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
def test_paged_decode_bad_blocks_and_lengths(pool_kind):
    """Ids outside the pool read as zeros and set a bit; a length past the table is cut."""
    g = torch.Generator().manual_seed(4)
    ln = [70, 40]
    pool, tables, ks, vs = _pool(g, ln, 2, 64, torch.bfloat16, pool_kind == "int8", poison=False)
    q = torch.randn(2, 4, 1, 64, generator=g).to(torch.bfloat16)
    bad = tables.clone()
    bad[0, 1], bad[1, 2], bad[0, 4] = -1, pool.shape[0], 1 << 30
    o, lse = _attend(q, pool, bad, ln, ks, vs)
    assert _status() == ostep.BAD_BLOCK
    _check_attention(o, lse, q, pool, bad, ln, 0.125, ks, vs)
    cut = tables[:, :2].contiguous()
    o, lse = _attend(q, pool, cut, [1000, 32], ks, vs)
    assert _status() == ostep.BAD_LENGTH
    _check_attention(o, lse, q, pool, cut, [1000, 32], 0.125, ks, vs)
    o, lse = _attend(q, pool, tables, [-5, 40], ks, vs)
    _check_attention(o, lse, q, pool, tables, [-5, 40], 0.125, ks, vs)


def test_paged_decode_non_finite_values_stay_in_their_rows():
    """inf / NaN in one head's visible K or V reach that KV head's outputs only, as in the
    formula; -inf scores weigh nothing."""
    g = torch.Generator().manual_seed(5)
    ln = [200, 200]
    pool, tables, _, _ = _pool(g, ln, 2, 64, torch.bfloat16, False)
    q = torch.randn(2, 8, 1, 64, generator=g).to(torch.bfloat16)
    q[0, :4, 0, 0] = -1.0
    clean, _ = _attend(q, pool, tables, ln)
    p2 = pool.clone()
    p2[tables[0, 3], 0, 0, 5, 0] = float("inf")          # score -inf for row 0, head 0's group
    p2[tables[1, 2], 1, 1, 7, 3] = float("nan")          # feature 3 of row 1, KV head 1
    o, lse = _attend(q, p2, tables, ln)
    want = clean.clone()
    K = p2.float()
    x = torch.einsum("htd,hd->ht", K[tables[0, :13].long(), 0, 0].reshape(1, -1, 64)[:, :200].expand(4, -1, -1),
                     q[0, :4, 0].float()) / 8
    assert torch.isneginf(x[:, 53]).all()
    w = torch.softmax(x.double(), -1)
    ref = w @ K[tables[0, :13].long(), 1, 0].reshape(-1, 64)[:200].double()
    assert torch.allclose(o[0, :4, 0].double().cpu(), ref, atol=2 ** -7)
    want[0, :4] = o[0, :4]
    want[1, 4:, 0, 3] = float("nan")
    assert torch.isnan(o[1, 4:, 0, 3]).all()
    assert torch.equal(torch.nan_to_num(o), torch.nan_to_num(want))
    p2[tables[0, 0], 0, 1, 0] = float("nan")             # a NaN key: the whole head row
    o, lse = _attend(q, p2, tables, ln)
    assert torch.isnan(o[0, 4:]).all() and torch.isnan(lse[0, 4:]).all() and not torch.isnan(o[0, :4]).any()


def test_paged_decode_layouts_and_streams():
    """HF's transposed query, a misaligned one, a caller's output view, sliced tables, no
    LSE, another stream; the same bits every time.  (A hint that changes the launch's shape
    changes the order of the sums: ``test_paged_decode_shapes_of_the_launch_agree``.)"""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(6)
    ln = [1700, 3, 0, 513]
    pool, tables, _, _ = _pool(g, ln, 4, 128, torch.bfloat16, False)
    q = torch.randn(4, 16, 1, 128, generator=g).to(torch.bfloat16)
    want, lse = _attend(q, pool, tables, ln)
    _check_attention(want, lse, q, pool, tables, ln, 1 / math.sqrt(128))
    lens = torch.tensor(ln, dtype=torch.int32, device=DEV)
    P, wide = pool.cuda(), torch.zeros(7, tables.shape[1] + 6, dtype=torch.int32, device=DEV)
    wide[2:6, 3:3 + tables.shape[1]] = tables.cuda()
    view = wide[2:6, 3:3 + tables.shape[1]]
    hf = q.cuda().transpose(1, 2).contiguous().transpose(1, 2)
    odd = torch.zeros(4, 16, 1, 129, dtype=torch.bfloat16, device=DEV)
    odd[..., 1:] = q.cuda()
    room = torch.full((4, 1, 20, 128), 5.0, dtype=torch.bfloat16, device=DEV)
    out = room[:, :, 2:18].transpose(1, 2)
    for qq, kw in ((hf, {}), (odd[..., 1:], dict(return_lse=False)), (q.cuda(), dict(out=out)),
                   (q.cuda(), dict(max_seq_len=1700))):
        o, l2 = paged_decode_attention(qq, P, view, lens, **kw)
        assert torch.equal(o, want), kw
        assert (l2 is None) if "return_lse" in kw else torch.equal(l2, lse)
    assert (room[:, :, :2] == 5).all() and (room[:, :, 18:] == 5).all()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        o, _ = paged_decode_attention(q.cuda(), P, view, lens)
    s.synchronize()
    assert torch.equal(o, want)


def test_paged_decode_shapes_of_the_launch_agree():
    """The hint picks the launch shape only: results agree to the rounding bound."""
    g = torch.Generator().manual_seed(8)
    for ln in ([260] * 3, [7] * 300, [4000, 10]):
        pool, tables, _, _ = _pool(g, ln, 2, 64, torch.float16, False)
        q = torch.randn(len(ln), 4, 1, 64, generator=g).to(torch.float16)
        for hint in (None, 16, 512, 100000):
            o, lse = _attend(q, pool, tables, ln, max_seq_len=hint)
            _check_attention(o, lse, q, pool, tables, ln, 0.125)


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
@pytest.mark.parametrize("B,longest", [(40, 3000), (256, 2300), (257, 2300), (700, 1200), (8193, 1100)])
def test_paged_decode_batch_sizes(pool_kind, B, longest):
    """Every way the rows are divided: a row per lane, eight, sums over the CTA, a CTA per item;
    idle rows between, one long row."""
    g = torch.Generator().manual_seed(B)
    ln = (torch.randint(0, 50, (B,), generator=g) * (torch.rand(B, generator=g) < 0.7)).tolist()
    ln[B // 3] = longest
    ln[-1] = 0
    pool, tables, ks, vs = _pool(g, ln, 1, 64, torch.bfloat16, pool_kind == "int8")
    q = torch.randn(B, 2, 1, 64, generator=g).to(torch.bfloat16)
    o, lse = _attend(q, pool, tables, ln, ks, vs)
    _check_attention(o, lse, q, pool, tables, ln, 0.125, ks, vs)


@pytest.mark.parametrize("pool_kind", ["same", "int8"])
@pytest.mark.parametrize("B,H,group,D,longest", [(300, 8, 1, 64, 300), (200, 16, 2, 128, 160), (90, 20, 9, 64, 700)])
def test_paged_decode_many_short_items(pool_kind, B, H, group, D, longest):
    """More items than warps: a share's end leaves an item that is short enough whole, with one
    warp or the next, and cuts the others; idle rows, one-token rows and one long row among them."""
    g = torch.Generator().manual_seed(B + D)
    ln = torch.randint(1, longest + 1, (B,), generator=g)
    ln[::17] = 1
    ln[::23] = 0
    ln[B // 2] = 6000
    ln = ln.tolist()
    pool, tables, ks, vs = _pool(g, ln, H, D, torch.float16, pool_kind == "int8")
    q = torch.randn(B, H * group, 1, D, generator=g).to(torch.float16)
    o, lse = _attend(q, pool, tables, ln, ks, vs)
    _check_attention(o, lse, q, pool, tables, ln, D ** -0.5, ks, vs)


@pytest.mark.parametrize("ln", [[50, 20], [5000, 3000, 9]])
def test_paged_decode_over_its_own_query(ln):
    """out=q: the output takes the query's place."""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(17)
    pool, tables, _, _ = _pool(g, ln, 2, 128, torch.float16, False)
    q = torch.randn(len(ln), 16, 1, 128, generator=g).to(torch.float16)
    want, _ = _attend(q, pool, tables, ln)
    qc = q.cuda()
    o, _ = paged_decode_attention(qc, pool.cuda(), tables.cuda(),
                                  torch.tensor(ln, dtype=torch.int32, device=DEV), out=qc)
    assert o is qc and torch.equal(qc, want)


def test_paged_decode_offsets_past_32_bits():
    """A pool of 2.6e9 elements: the last blocks are written and read."""
    from kvboost_b200.paged_decode import append_paged_kv, paged_decode_attention
    nb, H, D = 80000, 8, 128
    pool = torch.empty(nb, 2, H, 16, D, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator().manual_seed(3)
    kv = torch.randn(2, 40, H, D, generator=g).to(torch.bfloat16)
    blocks = [nb - 1, 65536, nb - 2]
    slots = torch.tensor([blocks[t // 16] * 16 + t % 16 for t in range(40)], dtype=torch.int32)
    append_paged_kv(kv[0].cuda(), kv[1].cuda(), pool, slots.cuda())
    tables = torch.tensor([blocks], dtype=torch.int32)
    q = torch.randn(1, 16, 1, D, generator=g).to(torch.bfloat16)
    o, lse = paged_decode_attention(q.cuda(), pool, tables.cuda(),
                                    torch.tensor([40], dtype=torch.int32, device=DEV))
    small = torch.zeros(3, 2, H, 16, D, dtype=torch.bfloat16)
    for t in range(40):
        small[t // 16, :, :, t % 16] = kv[:, t]
    _check_attention(o, lse, q, small, torch.tensor([[0, 1, 2]], dtype=torch.int32), [40], 1 / math.sqrt(D))
    del pool
    i8 = torch.empty(nb, 2, H, 16, D, dtype=torch.int8, device=DEV)
    ks = torch.full((nb, H, 16), 0.01, dtype=torch.float16, device=DEV)
    vs = torch.full((nb, H, D), 0.02, dtype=torch.float16, device=DEV)
    codes = torch.randint(-127, 128, (3, 2, H, 16, D), generator=g).to(torch.int8)
    i8[torch.tensor(blocks, device=DEV)] = codes.cuda()
    o, lse = paged_decode_attention(q.cuda(), i8, tables.cuda(),
                                    torch.tensor([40], dtype=torch.int32, device=DEV), ks, vs)
    _check_attention(o, lse, q, codes, torch.tensor([[0, 1, 2]], dtype=torch.int32), [40],
                     1 / math.sqrt(D), ks[:3].cpu(), vs[:3].cpu())


# ── logits ───────────────────────────────────────────────────────────────────

def _logits_case(B, V, L, N, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.rand(*s, generator=g)  # noqa: E731
    c = dict(logits=(3 * torch.randn(B, V, generator=g)).to(dtype))
    if L:
        c["token_ids"] = torch.randint(-2, min(V + 2, 50), (B, L), generator=g).to(torch.int32)
        c["total_lens"] = torch.randint(-1, L + 3, (B,), generator=g).to(torch.int32)
        c["prompt_lens"] = torch.randint(-1, L + 3, (B,), generator=g).to(torch.int32)
        c.update(repetition_penalty=1 + r(B), frequency_penalty=r(B), presence_penalty=r(B) - 0.5)
    if N:
        c["bias_ids"] = torch.randint(-1, V + 1, (B, N), generator=g).to(torch.int32)
        c["bias_ids"][:, N // 2] = c["bias_ids"][:, 0]       # an id given twice adds twice
        c["bias_values"] = 4 * torch.randn(B, N, generator=g)
    c["allowed_mask"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32 + 1), generator=g).to(torch.int32)
    c["temperature"] = 0.5 + r(B)
    return c


def _oracle_logits(c):
    n = lambda k: c[k].numpy() if c.get(k) is not None else None  # noqa: E731
    return ostep.logits(c["logits"].double().numpy(), n("token_ids"), n("prompt_lens"), n("total_lens"),
                        n("repetition_penalty"), n("frequency_penalty"), n("presence_penalty"),
                        n("bias_ids"), n("bias_values"), n("allowed_mask"), n("temperature"))


def _check_logits(got, want, c, dtype):
    """At most 6 + N float32 roundings, each half a step of a value no larger than the sum of
    the terms' magnitudes (x * r, the penalties, the biases) over the temperature."""
    got = got.double().cpu().numpy()
    fin = np.isfinite(want)
    assert np.array_equal(np.isneginf(got), np.isneginf(want))
    mag = np.abs(c["logits"].double().numpy())
    if c.get("repetition_penalty") is not None:
        mag = mag * np.maximum(c["repetition_penalty"].numpy(), 1)[:, None]
    for k in ("frequency_penalty", "presence_penalty"):
        if c.get(k) is not None:
            mag = mag + np.abs(c[k].double().numpy())[:, None] * c["token_ids"].shape[1]
    n = 0
    if c.get("bias_values") is not None:
        mag = mag + np.abs(c["bias_values"].double().numpy()).sum(1)[:, None]
        n = c["bias_values"].shape[1]
    if c.get("temperature") is not None:
        mag = mag / np.maximum(c["temperature"].numpy(), 1e-5)[:, None]
    # below the smallest normal number values are spaced eps * smallest_normal (float16: 2^-24
    # below 2^-14), so the last rounding is off by up to half of that however small the value is:
    # float16(-2.7018e-5) is 1.74e-8 off, more than 2^-11 of it (1.32e-8), less than 2^-25
    info = torch.finfo(dtype)
    bound = (6 + n) * U * mag + info.eps / 2 * (np.abs(np.where(fin, want, 0)) + info.smallest_normal) + 1e-38
    assert (np.abs(np.where(fin, got, 0) - np.where(fin, want, 0)) <= bound).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,L,N", [(1, 1, 3, 1), (1, 31, 0, 0), (2, 33, 40, 5), (3, 1000, 1, 0),
                                     (5, 4097, 300, 17), (2, 50001, 5000, 300), (1, 151936, 77, 3),
                                     (70, 2048, 33, 2), (2, 33, 9, 300), (200, 20000, 50, 3),
                                     (100, 30000, 17000, 2)])
def test_process_logits(dtype, B, V, L, N):
    from kvboost_b200.logits import process_logits
    c = _logits_case(B, V, L, N, dtype, V + L)
    want = _oracle_logits(c)
    d = {k: t.cuda() for k, t in c.items()}
    _check_logits(process_logits(**d), want, c, torch.float32)
    # parts alone
    for drop in (("allowed_mask",), ("temperature",), ("bias_ids", "bias_values"), ("prompt_lens",),
                 ("repetition_penalty",), ("frequency_penalty",), ("presence_penalty",),
                 ("token_ids", "prompt_lens", "total_lens", "repetition_penalty", "frequency_penalty",
                  "presence_penalty")):
        c2 = {k: t for k, t in c.items() if k not in drop}
        _check_logits(process_logits(**{k: d[k] for k in c2}), _oracle_logits(c2), c2, torch.float32)
    # in place, in the logits' dtype, through a strided view
    wide = torch.full((B, V + 5), 7.0, dtype=dtype, device=DEV)
    wide[:, 3:3 + V] = d["logits"]
    d["logits"] = wide[:, 3:3 + V]
    assert process_logits(**d, out=d["logits"]) is d["logits"]
    _check_logits(d["logits"], want, c, dtype)
    assert (wide[:, :3] == 7).all() and (wide[:, 3 + V:] == 7).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V,pad", [(1, 5, 0), (5, 4100, 0), (5, 4096, 4), (3, 8191, 1), (150, 10004, 0),
                                     (150, 10000, 8), (40, 33000, 2)])
def test_process_logits_without_history(dtype, B, V, pad):
    """Mask and temperature alone, rows on 8, 4 or single values, a new result and in place."""
    from kvboost_b200.logits import process_logits
    c = _logits_case(B, V, 0, 0, dtype, V + pad)
    want = _oracle_logits(c)
    d = {k: t.cuda() for k, t in c.items()}
    wide = torch.full((B, V + pad), 7.0, dtype=dtype, device=DEV)
    wide[:, :V] = d["logits"]
    d["logits"] = wide[:, :V]
    _check_logits(process_logits(**d), want, c, torch.float32)
    for drop in ("allowed_mask", "temperature"):
        c2 = {k: t for k, t in c.items() if k != drop}
        _check_logits(process_logits(**{k: d[k] for k in c2}), _oracle_logits(c2), c2, torch.float32)
    process_logits(**d, out=d["logits"])
    _check_logits(d["logits"], want, c, dtype)
    assert (wide[:, V:] == 7).all()


@pytest.mark.parametrize("V", [4104, 4100, 4101])
def test_process_logits_same_for_every_alignment(V):
    """Rows on 8, 4 or single values, counted in 16 and in 32 bits: the
    same bits as the same rows one by one on their own."""
    from kvboost_b200.logits import process_logits
    c = _logits_case(6, V, 700, 9, torch.bfloat16, V)
    d = {k: t.cuda() for k, t in c.items()}
    got = process_logits(**d)
    one = torch.cat([process_logits(**{k: t[b:b + 1].clone() for k, t in d.items()}) for b in range(6)])
    assert torch.equal(got, one)
    long = torch.full((6, 17000), -1, dtype=torch.int32, device=DEV)
    long[:, :700] = d["token_ids"]
    # the lengths stay, so the longer buffer changes the counters' width alone
    lens = {k: d[k].clamp(max=700) for k in ("total_lens", "prompt_lens")}
    assert torch.equal(got, process_logits(**{**d, "token_ids": long, **lens}))


def test_process_logits_captured():
    """A captured call follows its inputs' new values at each replay."""
    from kvboost_b200.logits import process_logits
    c = _logits_case(3, 5000, 60, 4, torch.bfloat16, 8)
    d = {k: t.cuda() for k, t in c.items()}
    process_logits(**d)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = process_logits(**d)
    for seed in (1, 2):
        c = _logits_case(3, 5000, 60, 4, torch.bfloat16, seed)
        for k, t in c.items():
            d[k].copy_(t)
        graph.replay()
        _check_logits(o, _oracle_logits(c), c, torch.float32)


def test_process_logits_special_values():
    """A mask that leaves nothing, infinities and NaN, temperature 0, a count past 65 535."""
    from kvboost_b200.logits import process_logits
    V = 300
    x = torch.linspace(-3, 3, V, device=DEV).repeat(4, 1)
    x[1, 5], x[1, 6], x[1, 7] = float("inf"), float("-inf"), float("nan")
    mask = torch.full((4, 10), -1, dtype=torch.int32, device=DEV)
    mask[0] = 0
    mask[1, 0] = ~(1 << 7)
    ids = torch.full((4, 70000), 9, dtype=torch.int32, device=DEV)
    n = torch.full((4,), 70000, dtype=torch.int32, device=DEV)
    f = torch.full((4,), 0.5, device=DEV)
    t = torch.tensor([1.0, 1.0, 0.0, 2.0], device=DEV)
    o = process_logits(x, token_ids=ids, total_lens=n, frequency_penalty=f, allowed_mask=mask, temperature=t)
    assert torch.isneginf(o[0]).all()
    assert o[1, 5] == float("inf") and torch.isneginf(o[1, 6]) and torch.isneginf(o[1, 7])
    assert torch.allclose(o[2, 10:], x[2, 10:] / 1e-5)
    assert torch.allclose(o[3, 9], (x[3, 9] - 35000) / 2)
    keep = torch.ones(V, dtype=torch.bool, device=DEV)
    keep[9] = False
    assert torch.equal(o[3][keep], x[3][keep] / 2)
    assert process_logits(x[:0]).shape == (0, V)


# ── together ─────────────────────────────────────────────────────────────────

def test_a_step_of_all_operators():
    """Eight requests decode 40 tokens through extend / append / attend, a captured graph per
    step shape replayed with in-place lengths: outputs equal attention over the dense history,
    blocks follow the host allocator's order, and no slot is used twice."""
    from kvboost_b200.paged_decode import append_paged_kv, extend_block_tables, paged_decode_attention
    B, H, G, D, steps = 8, 2, 4, 64, 40
    g = torch.Generator().manual_seed(1)
    plens = [0, 1, 15, 16, 17, 40, 100, 33]
    nb = 64
    pool = torch.full((nb, 2, H, 16, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    tables = torch.full((B, 12), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    free = torch.arange(nb, dtype=torch.int32, device=DEV)
    nfree = torch.tensor([nb], dtype=torch.int32, device=DEV)
    hist = [torch.randn(2, n, H, D, generator=g).to(torch.bfloat16) for n in plens]
    # prompts: one packed append
    T = sum(plens)
    s = extend_block_tables(tables, lens, torch.tensor(plens, dtype=torch.int32, device=DEV), free,
                            nfree, nb, T, seq_lens_out=lens, num_free_out=nfree)
    packed = torch.cat(hist, 1).cuda()
    append_paged_kv(packed[0], packed[1], pool, s.slots)
    assert s.positions.tolist() == [p for n in plens for p in range(n)]
    # the decode step, captured
    ones = torch.ones(B, dtype=torch.int32, device=DEV)
    k, v = (torch.zeros(B, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(B, H * G, 1, D, dtype=torch.bfloat16, device=DEV)

    def step():
        s = extend_block_tables(tables, lens, ones, free, nfree, nb, B, seq_lens_out=lens,
                                num_free_out=nfree)
        append_paged_kv(k, v, pool, s.slots)
        return (*paged_decode_attention(q, pool, tables, lens), s.slots)

    saved = [t.clone() for t in (tables, lens, nfree, pool)]
    step()                                       # warm-up, undone
    for t, x in zip((tables, lens, nfree, pool), saved):
        t.copy_(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse, slots = step()
    used = set(s.slots.tolist())
    for i in range(steps):
        kv = torch.randn(2, B, H, D, generator=g).to(torch.bfloat16)
        qq = torch.randn(B, H * G, 1, D, generator=g).to(torch.bfloat16)
        k.copy_(kv[0])
        v.copy_(kv[1])
        q.copy_(qq)
        graph.replay()
        new = slots.tolist()
        assert min(new) >= 0 and not used.intersection(new) and len(set(new)) == B
        used.update(new)
        hist = [torch.cat([h, kv[:, b:b + 1]], 1) for b, h in enumerate(hist)]
        n = [p + i + 1 for p in plens]
        assert lens.tolist() == n
        if i % 13 == 0 or i == steps - 1:
            dense = torch.zeros(B, 2, H, 12 * 16, D, dtype=torch.bfloat16)
            for b, h in enumerate(hist):
                dense[b, :, :, :h.shape[1]] = h.permute(0, 2, 1, 3)
            p = dense.view(B, 2, H, 12, 16, D).permute(0, 3, 1, 2, 4, 5).reshape(-1, 2, H, 16, D)
            _check_attention(o, lse, qq, p, torch.arange(B * 12).view(B, 12), n, 1 / math.sqrt(D))
    assert nfree.item() == nb - sum(-(-(p + steps) // 16) for p in plens)


def test_two_captured_graphs_do_not_share_workspaces():
    """Two attention graphs replayed on two streams at once give the eager results."""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(21)
    sets = []
    for ln in ([3000, 5], [1777, 2500]):
        pool, tables, _, _ = _pool(g, ln, 2, 128, torch.bfloat16, False)
        q = torch.randn(2, 16, 1, 128, generator=g).to(torch.bfloat16)
        args = (q.cuda(), pool.cuda(), tables.cuda(), torch.tensor(ln, dtype=torch.int32, device=DEV))
        sets.append((args, paged_decode_attention(*args)[0].clone()))
    graphs = []
    for args, _ in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            o, _ = paged_decode_attention(*args)
        graphs.append((gr, o, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for gr, o, s in graphs:
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for (_, want), (_, o, _) in zip(sets, graphs):
        assert torch.equal(o, want)
