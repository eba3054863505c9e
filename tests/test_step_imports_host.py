"""The paged paths import on a torch whose C binding lacks the private names that the batched step's
operators use to save host time (CPU)."""

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
