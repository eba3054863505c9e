"""GPU: the batched step's operators where host code and device meet: torch without private bindings, calls
from several threads, captured calls whose inputs change, results that overlap."""

import math

import numpy as np
import pytest
import torch

from oracle import step as ostep

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability()[0] != 10:
        pytest.skip("needs an sm_100 (B200) device")
    from kvboost_b200 import ops
    ops.read_status(torch.device("cuda"))
    yield
    assert ops.read_status(torch.device("cuda")) == 0


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _step(g, n=700):
    """One call of each operator; the results."""
    from kvboost_b200.logits import process_logits
    from kvboost_b200.paged_decode import append_paged_kv, extend_block_tables, paged_decode_attention
    tables = torch.zeros(2, 200, dtype=torch.int32, device=DEV)
    s = extend_block_tables(tables, _i32([0, 0]), _i32([n, 5]), torch.arange(300, dtype=torch.int32, device=DEV), _i32([300]),
                            300, n + 5)
    pool = torch.zeros(300, 2, 2, 16, 64, dtype=torch.bfloat16, device=DEV)
    kv = torch.randn(2, n + 5, 2, 64, generator=g).to(DEV, torch.bfloat16)
    append_paged_kv(kv[0], kv[1], pool, s.slots)
    q = torch.randn(2, 8, 1, 64, generator=g).to(DEV, torch.bfloat16)
    o, lse = paged_decode_attention(q, pool, tables, s.seq_lens)
    x = process_logits(torch.randn(2, 1001, generator=g).to(DEV), temperature=torch.full((2,), 0.7, device=DEV))
    return [*s, tables, pool, o, lse, x]


def test_torch_without_private_bindings(monkeypatch):
    """The public functions in their place give the same results, on another stream too."""
    from kvboost_b200 import paged_decode as pd
    want = _step(torch.Generator().manual_seed(1))
    monkeypatch.setattr(pd, "_raw_stream", pd._stream_of)
    monkeypatch.setattr(pd, "_current_device", torch.cuda.current_device)
    monkeypatch.setattr(pd, "_empty_strided", pd._new_strided)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _step(torch.Generator().manual_seed(1))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                             (torch.float32, torch.float32)])
def test_logits_beside_their_result_in_one_buffer(dtype, out_dtype):
    """Rows of the logits and of the result in turn in one buffer do not overlap; rows that do are
    refused."""
    from kvboost_b200.logits import process_logits
    B, V = 5, 1004
    wide = torch.zeros(B, 3 * V * 4, dtype=torch.uint8, device=DEV)
    x = wide[:, :V * dtype.itemsize].view(dtype)
    o = wide[:, V * 8:V * 8 + V * out_dtype.itemsize].view(out_dtype)
    x.copy_(torch.randn(B, V, device=DEV))
    want = x.float() * 2
    t = torch.full((B,), 0.5, device=DEV)
    assert process_logits(x, temperature=t, out=o) is o
    assert torch.equal(o.float(), want)
    with pytest.raises(Exception, match="overlap"):
        process_logits(x, temperature=t, out=wide[:, 8:8 + V * out_dtype.itemsize].view(out_dtype))


def _tables_args(B, seed):
    rng = np.random.default_rng(seed)
    lens, new = rng.integers(0, 34, B), rng.integers(0, 4, B)
    tables = np.full((B, 4), -7)
    ids = rng.permutation(B * 4 + 10)
    have = -(-lens // 16)
    at = 0
    for b in range(B):
        tables[b, :have[b]] = ids[at:at + have[b]]
        at += have[b]
    return tables, lens, new, ids[at:], len(ids) - at, B * 4 + 10, int(new.sum())


def test_tables_of_large_and_small_batches_from_two_threads():
    """Host threads that build the tables of batches of different size at once get their own results."""
    import threading

    from kvboost_b200 import _lib
    lib = _lib.load()
    work = []
    for B in (8192, 3500):
        tables, lens, new, free, nfree, nblk, total = _tables_args(B, B)
        want = ostep.extend_tables(tables, lens, new, free, nfree, nblk, total)
        ins = [_i32(x) for x in (tables, lens, new, free, [nfree])]
        outs = [torch.zeros(n, dtype=t, device=DEV) for n, t in
                ((total, torch.int32), (total, torch.int64), (B + 1, torch.int32), (B, torch.int32), (1, torch.int32),
                 (1, torch.int32))]
        p = _lib.pack_extend_tables(B, 4, 16, nblk, total, len(free), 4, *[t.data_ptr() for t in ins + outs])
        work.append((p, torch.cuda.Stream(), ins, outs, want))
    torch.cuda.synchronize()
    refused = []

    def run(p, stream):
        for _ in range(20000):
            if lib.kvb_extend_block_tables(p, stream.cuda_stream):
                refused.append(lib.kvb_last_error())

    threads = [threading.Thread(target=run, args=w[:2]) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for _, _, ins, outs, want in work:
        for got, w in zip((ins[0], *outs[:4]), want):
            assert np.array_equal(got.cpu().numpy(), w)
        assert outs[4].item() == want[5] and outs[5].item() == 0


def test_first_call_on_a_device_inside_a_capture():
    """The status word that it makes is zero before the first replay, and replays add to it."""
    from kvboost_b200 import ops
    from kvboost_b200.paged_decode import extend_block_tables
    dev = torch.device(DEV)
    args = (torch.zeros(2, 4, dtype=torch.int32, device=DEV), _i32([0, 0]), _i32([1, 99]), _i32([5, 6]), _i32([2]), 10, 100)
    extend_block_tables(*args)
    assert ops.read_status(dev) == ostep.BAD_LENGTH
    words = dict(ops._status_words)
    ops._status_words.clear()
    try:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s = extend_block_tables(*args)
        assert ops.read_status(dev, reset=False) == 0
        ops.status_word(dev).fill_(ostep.BAD_BLOCK)
        graph.replay()
        assert ops.read_status(dev) == ostep.BAD_BLOCK | ostep.BAD_LENGTH
        assert s.slots[:2].tolist() == [6 * 16, -1]
        ops._status_words.clear()
        with torch.inference_mode():
            extend_block_tables(*args)
        assert ops.read_status(dev) == ostep.BAD_LENGTH and ops.read_status(dev) == 0
    finally:
        ops._status_words.clear()
        ops._status_words.update(words)


@pytest.mark.parametrize("lens", [[3000, 5, 64], [40, 0, 333]])
def test_attention_into_the_query_and_into_other_layouts(lens):
    """``out=q``, a result with the heads outermost, both launch shapes; a broadcast one is refused."""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(2)
    nblk = [-(-n // 16) for n in lens]
    tables = torch.zeros(3, max(nblk), dtype=torch.int32)
    ids = torch.randperm(sum(nblk), generator=g).to(torch.int32)
    for b in range(3):
        tables[b, :nblk[b]] = ids[sum(nblk[:b]):sum(nblk[:b + 1])]
    pool = torch.randn(sum(nblk), 2, 2, 16, 64, generator=g).to(DEV, torch.bfloat16)
    q = torch.randn(3, 8, 1, 64, generator=g).to(DEV, torch.bfloat16)
    args = (pool, tables.to(DEV), _i32(lens))
    want, _ = paged_decode_attention(q, *args)
    own = q.clone()
    assert paged_decode_attention(own, *args, out=own)[0] is own
    assert torch.equal(own, want)
    turned = torch.empty(8, 3, 1, 64, dtype=q.dtype, device=DEV).transpose(0, 1)
    assert torch.equal(paged_decode_attention(q, *args, out=turned)[0], want)
    with pytest.raises(Exception, match="overlap"):
        paged_decode_attention(q, *args, out=torch.empty(1, 8, 1, 64, dtype=q.dtype, device=DEV).expand(3, -1, -1, -1))


def _scene(g, B, H, group, D, dtype, int8, width, most):
    """Fixed buffers of a captured call and a function that fills them anew."""
    nb = B * width if B * width < 4000 else 4000
    pool = torch.zeros(nb, 2, H, 16, D, dtype=torch.int8 if int8 else dtype, device=DEV)
    ks = torch.zeros(nb, H, 16, dtype=torch.float16, device=DEV) if int8 else None
    vs = torch.zeros(nb, H, D, dtype=torch.float16, device=DEV) if int8 else None
    q = torch.zeros(B, H * group, 1, D, dtype=dtype, device=DEV)
    tables = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)

    def fill(i):
        n = torch.randint(0, most + 1, (B,), generator=g)
        n[i % B] = most if i % 3 else 1           # a long row that moves, and replays without one
        n[(i + 1) % B] = 0
        lens.copy_(n.to(torch.int32))
        tables.copy_(torch.stack([torch.randperm(nb, generator=g)[:width] for _ in range(B)]).to(torch.int32))
        q.copy_(torch.randn(q.shape, generator=g))
        if int8:
            pool.copy_(torch.randint(-127, 128, pool.shape, generator=g))
            ks.copy_((0.5 + torch.rand(ks.shape, generator=g)) / 64)
            vs.copy_((0.5 + torch.rand(vs.shape, generator=g)) / 64)
        else:
            pool.copy_(torch.randn(pool.shape, generator=g))

    return (q, pool, tables, lens, ks, vs), fill


def _expect(o, lse, args):
    from test_gpu_step_ops import _check_attention
    q, pool, tables, lens, ks, vs = (None if t is None else t.cpu() for t in args)
    _check_attention(o, lse, q, pool, tables, lens.tolist(), 1 / math.sqrt(q.shape[-1]), ks, vs)


@pytest.mark.parametrize("B,H,group,D,dtype,int8", [
    (2, 1, 4, 64, torch.bfloat16, False), (3, 2, 12, 96, torch.float16, False), (3, 2, 8, 128, torch.bfloat16, True),
    (40, 1, 2, 64, torch.float16, True), (300, 1, 1, 64, torch.bfloat16, False)])
def test_split_launch_replayed_with_other_inputs(B, H, group, D, dtype, int8):
    """A captured call whose items span CTAs, its queries, lengths, tables and pool new at every replay and
    its results wiped before: each replay's results are its own."""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(B + D)
    args, fill = _scene(g, B, H, group, D, dtype, int8, 200, 3200 if B < 100 else 600)
    fill(0)
    paged_decode_attention(*args[:4], k_scale=args[4], v_scale=args[5])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = paged_decode_attention(*args[:4], k_scale=args[4], v_scale=args[5])
    for i in range(6):
        fill(i)
        o.fill_(float("nan"))
        lse.fill_(float("nan"))
        graph.replay()
        _expect(o, lse, args)


def test_two_split_graphs_on_two_streams_with_other_inputs():
    """As above, both graphs in flight at once."""
    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(5)
    sides = []
    for H, D in ((2, 128), (1, 64)):
        args, fill = _scene(g, 2, H, 8, D, torch.bfloat16, False, 200, 3200)
        fill(0)
        paged_decode_attention(*args[:4])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = paged_decode_attention(*args[:4])
        sides.append((graph, torch.cuda.Stream(), o, lse, args, fill))
    for i in range(8):
        for _, _, o, lse, _, fill in sides:
            fill(i)
            o.fill_(float("nan"))
            lse.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream, *_ in sides:
            with torch.cuda.stream(stream):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for _, _, o, lse, args, _ in sides:
            _expect(o, lse, args)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("H,group", [(1, 9), (2, 12), (1, 16), (1, 17)])
@pytest.mark.parametrize("lens", [[300, 0, 17, 1000], [2500, 0, 17, 33]])
def test_groups_above_eight(lens, H, group, D, dtype, int8):
    """16 query heads an item, every width and type, a CTA an item (tables of up to 64 blocks) and split."""
    from test_gpu_step_ops import _check_attention, _pool

    from kvboost_b200.paged_decode import paged_decode_attention
    g = torch.Generator().manual_seed(D + group)
    pool, tables, ks, vs = _pool(g, lens, H, D, dtype, int8)
    if max(lens) <= 1000:
        tables = tables[:, :64].contiguous()
    q = torch.randn(len(lens), H * group, 1, D, generator=g).to(dtype)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    o, lse = paged_decode_attention(c(q), c(pool), c(tables), _i32(lens), k_scale=c(ks), v_scale=c(vs))
    _check_attention(o, lse, q, pool, tables, lens, 1 / math.sqrt(D), ks, vs)
