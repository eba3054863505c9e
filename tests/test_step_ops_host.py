"""Host side of the batched decode step's operators (CPU): the C entries refuse what the
kernels do not take before anything launches, and the Python ops refuse CPU tensors."""

import ctypes

import numpy as np
import pytest
import torch

from kvboost_b200 import _build, _lib


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_build.LIB_PATH):
        _build.build(verbose=False)
    return _lib.load()


def _tables(**kw):
    p = _lib.KvbExtendTablesParams(2, 4, 16, 100, 8, 10, 4, *([4096] * 11))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _append(**kw):
    p = _lib.KvbAppendPagedParams(128, 2, 3, 10, 4096, 4096, 256, 128, 256, 128, 4096, 4096, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _decode(**kw):
    p = _lib.KvbPagedDecodeParams(0, 128, 2, 8, 2, 16, 1, 0.1, 4096, 4096, 4096, 1024, 128, 1024, 128, 8,
                                  4096, None, None, 10, 4, 4, 4096, 4096, 0, 0, 4096, None, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _logits(**kw):
    p = _lib.KvbLogitsParams(0, 2, 2, 1000, 0, 0, 4096, 8192, 1000, 1000)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


INV, UNS = _lib.KVB_ERR_INVALID, _lib.KVB_ERR_UNSUPPORTED


@pytest.mark.parametrize("make,fn,field,value,rc,needle", [
    (_tables, "kvb_extend_block_tables", "batch", 0, INV, "batch"),
    (_tables, "kvb_extend_block_tables", "batch", 8193, UNS, "batch"),
    (_tables, "kvb_extend_block_tables", "block_size", 32, INV, "block_size"),
    (_tables, "kvb_extend_block_tables", "max_blocks_per_seq", 5, INV, "block_table_stride"),
    (_tables, "kvb_extend_block_tables", "num_blocks", 1 << 27, INV, "num_blocks"),
    (_tables, "kvb_extend_block_tables", "max_new_tokens", -1, INV, "max_new_tokens"),
    (_tables, "kvb_extend_block_tables", "free_capacity", -1, INV, "free_capacity"),
    (_tables, "kvb_extend_block_tables", "seq_lens", None, INV, "non-null"),
    (_tables, "kvb_extend_block_tables", "slots", None, INV, "non-null"),
    (_append, "kvb_append_paged_kv", "head_dim", 100, INV, "head_dim"),
    (_append, "kvb_append_paged_kv", "head_dim", 264, INV, "head_dim"),
    (_append, "kvb_append_paged_kv", "num_kv_heads", 0, INV, "num_kv_heads"),
    (_append, "kvb_append_paged_kv", "num_tokens", -1, INV, "num_tokens"),
    (_append, "kvb_append_paged_kv", "num_blocks", 0, INV, "num_blocks"),
    (_append, "kvb_append_paged_kv", "k_new", 4098, INV, "aligned"),
    (_append, "kvb_append_paged_kv", "v_token_stride", 12, INV, "multiples of 8"),
    (_append, "kvb_append_paged_kv", "slots", None, INV, "non-null"),
    (_decode, "kvb_paged_decode_fwd", "dtype", 2, INV, "dtype"),
    (_decode, "kvb_paged_decode_fwd", "head_dim", 80, INV, "head_dim"),
    (_decode, "kvb_paged_decode_fwd", "batch", -1, INV, "batch"),
    (_decode, "kvb_paged_decode_fwd", "num_q_heads", 7, INV, "divisible"),
    (_decode, "kvb_paged_decode_fwd", "num_kv_heads", 0, INV, "divisible"),
    (_decode, "kvb_paged_decode_fwd", "block_size", 8, INV, "block_size"),
    (_decode, "kvb_paged_decode_fwd", "pool_format", 2, INV, "pool_format"),
    (_decode, "kvb_paged_decode_fwd", "pool_format", 0, INV, "k_scale16"),
    (_decode, "kvb_paged_decode_fwd", "num_blocks", 0, INV, "num_blocks"),
    (_decode, "kvb_paged_decode_fwd", "block_table_stride", 3, INV, "block_table_stride"),
    (_decode, "kvb_paged_decode_fwd", "q", None, INV, "non-null"),
    (_decode, "kvb_paged_decode_fwd", "kv_pool", 4104, INV, "aligned"),
    (_decode, "kvb_paged_decode_fwd", "o_head_stride", 132, INV, "multiples of 8"),
    (_logits, "kvb_process_logits", "dtype", 3, INV, "dtype"),
    (_logits, "kvb_process_logits", "out_dtype", 1, INV, "out_dtype"),
    (_logits, "kvb_process_logits", "vocab", 0, INV, "vocab"),
    (_logits, "kvb_process_logits", "batch", 65536, UNS, "batch"),
    (_logits, "kvb_process_logits", "vocab", (1 << 30) + 1, UNS, "vocab"),
    (_tables, "kvb_extend_block_tables", "max_new_tokens", (1 << 30) + 1, UNS, "max_new_tokens"),
    (_tables, "kvb_extend_block_tables", "positions", 4104, INV, "aligned"),
    (_decode, "kvb_paged_decode_fwd", "max_blocks_per_seq", 1 << 30, INV, "block_table_stride"),
    (_logits, "kvb_process_logits", "logits", 4097, INV, "aligned"),
    (_logits, "kvb_process_logits", "out_stride", 999, INV, "strides"),
    (_logits, "kvb_process_logits", "out", 4096, INV, "in place"),
    (_logits, "kvb_process_logits", "token_ids", 4096, INV, "total_lens"),
    (_logits, "kvb_process_logits", "presence_penalty", 4096, INV, "token_ids"),
    (_logits, "kvb_process_logits", "num_bias", 3, INV, "bias_ids"),
    (_logits, "kvb_process_logits", "allowed_mask", 4096, INV, "mask_stride"),
])
def test_c_entries_refuse_before_launch(lib, make, fn, field, value, rc, needle):
    p = make(**{field: value})
    assert getattr(lib, fn)(ctypes.byref(p), None) == rc
    assert needle in lib.kvb_last_error().decode()
    assert getattr(lib, fn)(None, None) == INV


def test_decode_workspace_refuses_what_the_call_refuses(lib):
    assert lib.kvb_paged_decode_workspace_bytes(ctypes.byref(_decode(head_dim=80))) == -1
    assert lib.kvb_paged_decode_workspace_bytes(ctypes.byref(_decode())) >= 0


def test_python_ops_refuse_cpu_tensors():
    from kvboost_b200.logits import process_logits
    from kvboost_b200.paged_decode import append_paged_kv, extend_block_tables, paged_decode_attention
    i = torch.zeros(1, dtype=torch.int32)
    h = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    pool = torch.zeros(2, 2, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        extend_block_tables(torch.zeros(1, 2, dtype=torch.int32), i, i, i, i, 2, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        append_paged_kv(h, h, pool, i)
    with pytest.raises(RuntimeError, match="CUDA"):
        paged_decode_attention(h[:, :, None], pool, torch.zeros(1, 2, dtype=torch.int32), i)
    with pytest.raises(RuntimeError, match="CUDA"):
        process_logits(torch.zeros(1, 8))


def test_decode_split_launch_needs_its_workspace(lib):
    p = _decode(max_blocks_per_seq=4096, block_table_stride=4096)
    need = lib.kvb_paged_decode_workspace_bytes(ctypes.byref(p))
    assert need > 0
    assert lib.kvb_paged_decode_fwd(ctypes.byref(p), None) == INV
    assert b"workspace" in lib.kvb_last_error()
    p.workspace, p.workspace_bytes = 4100, need
    assert lib.kvb_paged_decode_fwd(ctypes.byref(p), None) == INV
    assert b"aligned" in lib.kvb_last_error()
    p = _decode(max_blocks_per_seq=(1 << 27) - 1, block_table_stride=1 << 27, batch=100)
    assert lib.kvb_paged_decode_fwd(ctypes.byref(p), None) == UNS


def test_token_masks():
    """Bit v % 32 of word v // 32, the sign bit included."""
    from types import SimpleNamespace

    from kvboost_b200.paged_engine import PagedEngine
    eng = SimpleNamespace(device="cpu")
    m = PagedEngine._token_masks(eng, [None, [0, 31, 32, 69], []], 70)
    assert m.dtype == torch.int32 and m.shape == (3, 3)
    assert m[0].tolist() == [-1, -1, -1]
    assert m[1].tolist() == [1 - 2 ** 31, 1, 32] and m[2].tolist() == [0, 0, 0]
    for bad in ([70], [-1]):
        with pytest.raises(ValueError):
            PagedEngine._token_masks(eng, [bad], 70)


def test_struct_layouts_match_the_header(tmp_path):
    import subprocess
    structs = {c.__name__: c for c in (_lib.KvbExtendTablesParams, _lib.KvbAppendPagedParams,
                                       _lib.KvbPagedDecodeParams, _lib.KvbLogitsParams)}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "kvb_attn.h"', 'int main(){']
    for name, cls in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-I", _build.INCLUDE, "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    got = dict(line.split() for line in out.splitlines())
    for name, cls in structs.items():
        assert int(got[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{name}.{f}"]) == getattr(cls, f).offset, f"{name}.{f}"


def test_oracle_tables_follow_the_host_allocator():
    """The restatement pops blocks in ``BlockAllocator.allocate``'s order."""
    from oracle import paged as opaged
    from oracle import step as ostep
    model = opaged.AllocatorModel(20)
    t0 = model.allocate(2)
    free = list(range(20))[:18]
    tables = np.full((2, 6), -1)
    tables[0, :2] = t0
    out = ostep.extend_tables(tables, [32, 0], [17, 3], free, 18, 20, 20)
    assert out[0][0, 2:4].tolist() == model.allocate(2)
    assert out[0][1, :1].tolist() == model.allocate(1)
    assert out[5] == 15 and out[-1] == 0


def test_packed_parameters_equal_the_structures(lib):
    """``packer`` lays the fields out as the ctypes mirrors do."""
    for cls, pack in ((_lib.KvbExtendTablesParams, _lib.pack_extend_tables),
                      (_lib.KvbAppendPagedParams, _lib.pack_append_paged),
                      (_lib.KvbPagedDecodeParams, _lib.pack_paged_decode),
                      (_lib.KvbLogitsParams, _lib.pack_logits)):
        values = [0.25 if t is ctypes.c_float else 3 + i + (1 << 40 if ctypes.sizeof(t) == 8 else 0)
                  for i, (_, t) in enumerate(cls._fields_)]
        assert pack(*values) == bytes(cls(*values))
    p = _lib.pack_paged_decode(*[0] * len(_lib.KvbPagedDecodeParams._fields_))
    assert lib.kvb_paged_decode_workspace_bytes(p) == -1 and b"head_dim" in lib.kvb_last_error()
