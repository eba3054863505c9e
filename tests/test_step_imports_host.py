"""Host side of the paged paths (CPU): they import on a torch whose C binding lacks the private names that
the batched step's operators use to save host time, and the step refuses attention it does not have."""

import subprocess
import sys

import pytest

from kvboost_b200 import _build

NAMES = ["_cuda_getCurrentRawStream", "_cuda_getDevice", "_dynamo.guards._empty_strided_cuda"]


@pytest.mark.parametrize("missing", NAMES + ["all"])
def test_import_without_private_names(missing):
    code = """
import sys, torch
for name in sys.argv[1:]:
    at = torch._C
    *way, last = name.split(".")
    for part in way:
        at = getattr(at, part)
    if hasattr(at, last):
        delattr(at, last)
import kvboost_b200.paged_engine, kvboost_b200.logits
from kvboost_b200 import paged_decode as pd
from kvboost_b200.flash_attn_ext import _make_paged_attn_fn
_make_paged_attn_fn(0, {})
public = {"_cuda_getCurrentRawStream": (pd._raw_stream, pd._stream_of),
          "_cuda_getDevice": (pd._current_device, torch.cuda.current_device),
          "_dynamo.guards._empty_strided_cuda": (pd._empty_strided, pd._new_strided)}
for name in sys.argv[1:]:
    assert public[name][0] is public[name][1], name
"""
    names = NAMES if missing == "all" else [missing]
    subprocess.run([sys.executable, "-c", code, *names], check=True, cwd=_build.ROOT, timeout=300)


@pytest.mark.parametrize("kw", [{"sliding_window": 128}, {"softcap": 30.0}])
def test_a_batched_step_refuses_attention_it_does_not_have(kw):
    """As the other attention paths do, and before anything is written to the pool."""
    import torch

    from kvboost_b200.flash_attn_ext import _make_paged_attn_fn
    fn = _make_paged_attn_fn(0, {"allocator": None, "slots": torch.zeros(1, dtype=torch.int32)})
    x = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="sliding-window"):
        fn(None, x, x, x, **kw)
