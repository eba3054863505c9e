"""A decode step of a batch of requests over the block pool, on the device.

What ``append_kv_to_blocks`` and ``paged_attention_fwd`` do per sequence and token on
the host (``cpu_paged/paged_attn_cpu.py:33-163``), for all requests of a step at once:

* ``extend_block_tables`` -- block tables, pool slots and positions of the step's new
  tokens from the requests' lengths (``kvb_extend_block_tables``);
* ``append_paged_kv`` -- their K/V into a 16-bit pool (``kvb_append_paged_kv``);
* ``paged_decode_attention`` -- each request's new token over its blocks, 16-bit or
  KIVI int8, read in place (``kvb_paged_decode_fwd``).

Lengths, tables, slots and the free list are device tensors and nothing is read back,
so a step can be captured in a CUDA graph.  Device-side findings (a bad block id, a
length that does not fit, an empty free list) go to the device's status word
(``ops.read_status``).
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .ops import _DTYPES, _check_tensor, _status_words, status_word

BLOCK_SIZE = 16

def _stream_of(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


def _new_strided(shape, strides, dtype) -> torch.Tensor:
    return torch.empty_strided(shape, strides, dtype=dtype, device="cuda")


def _binding(name: str, public):
    """A function of torch's C binding, or ``public`` on a torch without it."""
    f = torch._C
    for part in name.split("."):
        f = getattr(f, part, None)
    return f or public


# A decode step calls these operators once per layer, so the host's cost per call is kept
# to a few checks: the stream handle comes from torch's C binding (2 us less than building a
# Stream object), results from its allocation of a strided tensor on the current device
# (0.8 us, ``new_empty`` 1.3 to 1.5), the device is switched only where it differs.
_raw_stream = _binding("_cuda_getCurrentRawStream", _stream_of)
_current_device = _binding("_cuda_getDevice", torch.cuda.current_device)
_empty_strided = _binding("_dynamo.guards._empty_strided_cuda", _new_strided)


def _allocator(device):
    """``f(shape, strides, dtype)``: a new tensor on the device."""
    if _current_device() == device.index:
        return _empty_strided
    return lambda shape, strides, dtype: torch.empty_strided(shape, strides, dtype=dtype, device=device)


def _launch(fn, params, device, what: str) -> None:
    """One library call on the device's current stream."""
    idx = device.index
    if _current_device() == idx:
        rc = fn(params, _raw_stream(idx))
    else:
        with torch.cuda.device(device):
            rc = fn(params, _raw_stream(idx))
    _lib.check(rc, what)


def _status_ptr(device) -> int:
    w = _status_words.get(device.index)
    return (status_word(device) if w is None else w).data_ptr()


def _check_int32(name: str, t: torch.Tensor, ndim: int, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype is not torch.int32 or t.dim() != ndim or t.device != device:
        raise RuntimeError(f"{name} must be a {ndim}-D int32 tensor on {device}, got "
                           f"{t.dim()}-D {t.dtype} on {t.device}")
    if not t.is_contiguous():
        if ndim == 1:
            raise RuntimeError(f"{name} must be contiguous")
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            raise RuntimeError(f"{name} must have contiguous rows")


def _check_tables(block_tables: torch.Tensor, batch: int, device) -> int:
    """Row stride of the block tables (rows may be a slice of a wider buffer)."""
    _check_int32("block_tables", block_tables, 2, device)
    rows, width = block_tables.shape
    if rows != batch or width < 1:
        raise RuntimeError(f"block_tables must be [{batch}, >= 1], got {tuple(block_tables.shape)}")
    stride = block_tables.stride()[0] if batch > 1 else width
    if stride < width:
        raise RuntimeError("block_tables rows must not overlap")
    return stride


class BlockTableStep(NamedTuple):
    """What ``extend_block_tables`` returns, all on the device."""
    slots: torch.Tensor       # int32 [max_new_tokens]: pool slot of each packed token, -1 unused
    positions: torch.Tensor   # int64 [max_new_tokens]: its position in its sequence
    cu_new: torch.Tensor      # int32 [B + 1]: row b's tokens are cu_new[b] .. cu_new[b + 1] - 1
    seq_lens: torch.Tensor    # int32 [B]: lengths with the new tokens
    num_free: torch.Tensor    # int32 [1]: blocks left on the free list


def extend_block_tables(block_tables: torch.Tensor, seq_lens: torch.Tensor,
                        new_lens: torch.Tensor, free_blocks: torch.Tensor,
                        num_free: torch.Tensor, num_blocks: int, max_new_tokens: int,
                        seq_lens_out: Optional[torch.Tensor] = None,
                        num_free_out: Optional[torch.Tensor] = None) -> BlockTableStep:
    """Give every request of a step the blocks its new tokens need.

    Row b of ``block_tables`` (int32 ``[B, max_blocks]``) holds ``seq_lens[b]`` tokens and
    gets ``new_lens[b]`` more (0: idle).  New blocks are popped from the end of
    ``free_blocks[:num_free]``, rows in order (the order of ``BlockAllocator.allocate``),
    and written to the table in place; the new tokens, packed row after row, get their
    pool slots (``block * 16 + offset``) and positions.  ``max_new_tokens`` bounds the
    step's tokens (the host knows it: B for a decode step).

    A row that does not fit (its table or ``max_new_tokens`` too small, a negative
    length, or no free blocks left for it) keeps its length, its tokens get slot -1, and
    the status word says why (``KVB_STATUS_BAD_LENGTH`` / ``KVB_STATUS_POOL_EMPTY``).
    ``seq_lens_out`` / ``num_free_out`` may be ``seq_lens`` / ``num_free`` themselves: the
    step then advances in place.
    """
    if not isinstance(block_tables, torch.Tensor):
        raise TypeError("block_tables must be a torch.Tensor")
    if not block_tables.is_cuda:
        raise RuntimeError("block_tables must be on CUDA (kvboost_b200 has no CPU path)")
    dev = block_tables.device
    B, width = block_tables.shape if block_tables.dim() == 2 else (0, 0)
    stride = _check_tables(block_tables, B, dev)
    _check_int32("seq_lens", seq_lens, 1, dev)
    _check_int32("new_lens", new_lens, 1, dev)
    _check_int32("num_free", num_free, 1, dev)
    _check_int32("free_blocks", free_blocks, 1, dev)
    if seq_lens.numel() != B or new_lens.numel() != B or num_free.numel() != 1:
        raise RuntimeError(f"seq_lens and new_lens must have {B} entries, num_free one")
    if not 1 <= B <= _lib.KVB_MAX_STEP_ROWS:
        raise RuntimeError(f"a step has 1 to {_lib.KVB_MAX_STEP_ROWS} rows, got {B}")
    T = int(max_new_tokens)
    if T < 0:
        raise RuntimeError("max_new_tokens must be >= 0")
    # the int32 results share one allocation: slots first (16-byte aligned)
    new = _allocator(dev)
    slots, cu, lens_out, free_out = new((T + 2 * B + 2,), (1,), torch.int32).split_with_sizes((T, B + 1, B, 1))
    positions = new((T,), (1,), torch.int64)
    if seq_lens_out is None:
        seq_lens_out = lens_out
    else:
        _check_int32("seq_lens_out", seq_lens_out, 1, dev)
    if num_free_out is None:
        num_free_out = free_out
    else:
        _check_int32("num_free_out", num_free_out, 1, dev)
    if seq_lens_out.numel() != B or num_free_out.numel() != 1:
        raise RuntimeError(f"seq_lens_out must have {B} entries, num_free_out one")
    p = _lib.pack_extend_tables(
        B, width, BLOCK_SIZE, int(num_blocks), T, free_blocks.numel(), stride,
        block_tables.data_ptr(), seq_lens.data_ptr(), new_lens.data_ptr(), free_blocks.data_ptr(),
        num_free.data_ptr(), slots.data_ptr(), positions.data_ptr(), cu.data_ptr(),
        seq_lens_out.data_ptr(), num_free_out.data_ptr(), _status_ptr(dev))
    _launch(_lib.load().kvb_extend_block_tables, p, dev, "kvb_extend_block_tables")
    return BlockTableStep(slots, positions, cu, seq_lens_out, num_free_out)


def _check_pool(kv_pool: torch.Tensor, device):
    """(num_blocks, kv_heads, head_dim) of one layer's pool."""
    if not isinstance(kv_pool, torch.Tensor):
        raise TypeError("kv_pool must be a torch.Tensor")
    shape = kv_pool.shape
    if len(shape) != 5 or shape[1] != 2 or shape[3] != BLOCK_SIZE or not kv_pool.is_contiguous() \
            or kv_pool.device != device:
        raise RuntimeError(f"kv_pool must be a contiguous [num_blocks, 2, kv_heads, 16, head_dim] "
                           f"tensor on {device}, got {tuple(shape)} on {kv_pool.device}")
    return shape[0], shape[2], shape[4]


def append_paged_kv(k_new: torch.Tensor, v_new: torch.Tensor, kv_pool: torch.Tensor,
                    slots: torch.Tensor) -> None:
    """Write the new tokens' K/V into a 16-bit pool at their slots.

    ``k_new`` / ``v_new``: ``[T, Hkv, D]`` views (a model cache's ``[Hkv, T, D]`` storage is
    read in place through its transpose) in the pool's dtype; ``kv_pool``: one layer's
    ``[num_blocks, 2, Hkv, 16, D]`` (``DeviceBlockAllocator.pools[layer]``); ``slots``: int32
    ``[T]`` from ``extend_block_tables``, all different, -1 where a token is not stored.
    Slots outside the pool are skipped and set ``KVB_STATUS_BAD_BLOCK``.  Sources inside the pool
    itself are refused.
    """
    _check_tensor("k_new", k_new, 3)
    _check_tensor("v_new", v_new, 3)
    dev = k_new.device
    if k_new.shape != v_new.shape or v_new.device != dev:
        raise RuntimeError("k_new and v_new must have the same shape and device")
    T, H, D = k_new.shape
    num_blocks, heads, dim = _check_pool(kv_pool, dev)
    if heads != H or dim != D:
        raise RuntimeError("pool heads / head_dim do not match k_new")
    dtype = kv_pool.dtype
    if k_new.dtype != dtype or v_new.dtype != dtype:
        raise RuntimeError(f"k_new and v_new must have the pool's dtype {dtype} "
                           "(int8 pools hold whole KIVI chunks)")
    if D % 8 or D > 256:
        raise RuntimeError(f"head_dim must be a multiple of 8 up to 256, got {D}")
    _check_int32("slots", slots, 1, dev)
    if slots.numel() != T:
        raise RuntimeError(f"slots must have {T} entries, got {slots.numel()}")
    if T == 0:
        return
    kt, kh, _ = k_new.stride()
    vt, vh, _ = v_new.stride()
    if kt % 8 or kh % 8 or k_new.data_ptr() % 16:
        k_new = k_new.clone(memory_format=torch.contiguous_format)
        kt, kh, _ = k_new.stride()
    if vt % 8 or vh % 8 or v_new.data_ptr() % 16:
        v_new = v_new.clone(memory_format=torch.contiguous_format)
        vt, vh, _ = v_new.stride()
    p = _lib.pack_append_paged(
        D, H, T, num_blocks, k_new.data_ptr(), v_new.data_ptr(), kt, kh, vt, vh,
        kv_pool.data_ptr(), slots.data_ptr(), _status_ptr(dev))
    _launch(_lib.load().kvb_append_paged_kv, p, dev, "kvb_append_paged_kv")


def paged_decode_attention(q: torch.Tensor, kv_pool: torch.Tensor, block_tables: torch.Tensor,
                           seq_lens: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None,
                           softmax_scale: Optional[float] = None,
                           max_seq_len: Optional[int] = None,
                           out: Optional[torch.Tensor] = None, return_lse: bool = True,
                           ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Attention of one new token per request over its blocks of the pool, read in place.

    q: ``[B, Hq, 1, D]``; ``kv_pool``: one layer's ``[num_blocks, 2, Hkv, 16, D]`` in q's
    dtype, or int8 with its float16 scales ``k_scale [num_blocks, Hkv, 16]`` and ``v_scale
    [num_blocks, Hkv, D]`` (``DeviceBlockAllocator.k_scale16`` / ``v_scale16``; such a pool holds
    whole KIVI chunks and takes no single tokens, so the rows attend to reused chunks alone);
    ``block_tables``: int32 ``[B, max_blocks]``; ``seq_lens``: int32 ``[B]`` device tensor, the
    tokens row b attends to (its own included, once appended).  ``Hq % Hkv == 0``.
    Returns ``(o [B, Hq, 1, D] in q's dtype, lse float32 [B, Hq, 1] or None)``; a row of
    length 0 gives zeros and -inf.  ``out``: q's shape and dtype, in heads that do not overlap
    (``out=q`` works in place).  ``max_seq_len``, a host-known bound of the lengths,
    only tunes the launch.
    """
    _check_tensor("q", q, 4)
    B, Hq, Sq, D = q.shape
    dev = q.device
    if Sq != 1:
        raise RuntimeError(f"q must hold one token per request [B, Hq, 1, D], got {tuple(q.shape)}")
    if D not in (64, 96, 128):
        raise RuntimeError(f"head_dim must be one of 64, 96, 128, got {D}")
    num_blocks, Hkv, dim = _check_pool(kv_pool, dev)
    if dim != D:
        raise RuntimeError(f"pool head_dim {dim} does not match the query's {D}")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise RuntimeError(f"num_q_heads ({Hq}) must be divisible by num_kv_heads ({Hkv})")
    stride = _check_tables(block_tables, B, dev)
    _check_int32("seq_lens", seq_lens, 1, dev)
    if seq_lens.numel() != B:
        raise RuntimeError(f"seq_lens must have {B} entries, got {seq_lens.numel()}")
    dtype, pool_dtype = q.dtype, kv_pool.dtype
    if pool_dtype == torch.int8:
        fmt = _lib.KVB_POOL_INT8_KIVI
        for name, t, shape in (("k_scale", k_scale, (num_blocks, Hkv, BLOCK_SIZE)),
                               ("v_scale", v_scale, (num_blocks, Hkv, D))):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.float16 or t.device != dev \
                    or t.shape != shape or not t.is_contiguous():
                raise RuntimeError(f"int8 pools need {name}: contiguous float16 {list(shape)} on {dev}")
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    else:
        fmt, ks, vs = _lib.KVB_POOL_COMPUTE, 0, 0
        if pool_dtype != dtype:
            raise RuntimeError("a 16-bit pool must hold the compute dtype")
        if k_scale is not None or v_scale is not None:
            raise RuntimeError("scales belong to int8 pools")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(D)
    if max_seq_len is not None and not 0 <= max_seq_len < 1 << 31:
        raise RuntimeError(f"max_seq_len must be in [0, 2^31), got {max_seq_len}")
    new = _allocator(dev)
    if out is None:
        ob, oh = Hq * D, D
        out = new((B, Hq, 1, D), (ob, D, D, 1), dtype)
    else:
        ob, oh = out.stride()[:2] if out.dim() == 4 else (1, 1)
        if out.shape != q.shape or out.dtype != dtype or out.device != dev or out.stride(3) != 1 \
                or ob % 8 or oh % 8 or out.data_ptr() % 16:
            raise RuntimeError("out must match q in shape, dtype and device, with 16-byte aligned heads")
    lse = new((B, Hq, 1), (Hq, 1, 1), torch.float32) if return_lse else None
    if B == 0:
        return out, lse
    qb, qh, _, _ = q.stride()
    if qb % 8 or qh % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        qb, qh, _, _ = q.stride()
    fields = (_DTYPES[dtype], D, B, Hq, Hkv, BLOCK_SIZE, fmt, softmax_scale, q.data_ptr(),
              out.data_ptr(), lse.data_ptr() if return_lse else 0, qb, qh, ob, oh, Hq,
              kv_pool.data_ptr(), ks, vs, num_blocks, block_tables.shape[1], stride,
              block_tables.data_ptr(), seq_lens.data_ptr(), max_seq_len or 0, 0, _status_ptr(dev))
    lib = _lib.load()
    p = _lib.pack_paged_decode(*fields, 0, 0)
    need = lib.kvb_paged_decode_workspace_bytes(p)
    if need > 0:
        # partial results of this call: torch's caching allocator orders their reuse on the
        # current stream, so calls on concurrent streams never share them
        ws = new((need,), (1,), torch.uint8)
        p = _lib.pack_paged_decode(*fields, ws.data_ptr(), need)
    _launch(lib.kvb_paged_decode_fwd, p, dev, "kvb_paged_decode_fwd")
    return out, lse
