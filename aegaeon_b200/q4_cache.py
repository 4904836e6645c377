"""A paged KV cache held in 4 bits: write rows into it, read them back, attend
over it.

The cache of one layer is two uint8 tensors (K and V) of pages,
``[num_blocks, kv_heads, block_size * (head_dim // 2 + 4)]``: for each block and
kv head the 4-bit codes of the block's tokens, then an fp16 scale and zero for
each token (a value is ``scale * code + zero``).  At head_dim 128 a token and
head takes 68 bytes where 16-bit values take 256, and a page is plain bytes of
one block, so the swap and migration paths move it unchanged: pass the page
tensors as the segments of a ``KVSwapper``, or a view of them in a 2-byte type
(which is what it assumes) as the ``kv_cache`` of ``ops.swap``.  A request swapped out and in again crosses the host link with
3.8 times fewer bytes.

  write      quantises new K and V rows into their slots;
  read       gives rows back in 16 or 32 bits;
  attention  causal attention over the pages through block tables, for single
             tokens and for pieces of prompts, with an optional sliding window
             and first tokens that stay visible.

Slot ``s`` is token ``s % block_size`` of block ``s // block_size``.  Every call
is queued on the current stream of its tensors' device and may be captured into
a CUDA graph; nothing is read back.  What the host can see is checked before
anything is queued (ValueError, TypeError); a slot, block id or length in device
memory that is outside its buffer is skipped by the kernels and shows in
``_lib.device_status``.  The reference has no counterpart (its caches hold
16-bit values).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _lib

HEAD_DIMS = (64, 128, 256)
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16,
           torch.float32: _lib.DTYPE_FP32}
_workspace_bytes: dict = {}


def head_bytes(block_size: int, head_dim: int) -> int:
    """Bytes of one block's tokens of one kv head."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if block_size < 16 or block_size % 16 or block_size > 4096:
        raise ValueError(f"block_size must be a multiple of 16 up to 4096, got {block_size}")
    return block_size * (head_dim // 2 + 4)


def page_bytes(block_size: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of a page: one block of one tensor (K or V)."""
    return kv_heads * head_bytes(block_size, head_dim)


def allocate(num_blocks: int, block_size: int, kv_heads: int, head_dim: int,
             device: Union[str, torch.device] = "cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """Zeroed key and value pages of one layer."""
    shape = (num_blocks, kv_heads, head_bytes(block_size, head_dim))
    return (torch.zeros(shape, dtype=torch.uint8, device=device),
            torch.zeros(shape, dtype=torch.uint8, device=device))


def _cache(key_pages: torch.Tensor, value_pages: torch.Tensor, head_dim: int):
    """Checks a cache's tensors and gives (pointers, strides, shape) as the C
    entry points take them."""
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
    if key_pages.dtype is not torch.uint8 or value_pages.dtype is not torch.uint8:
        raise TypeError("cache pages must be uint8 tensors")
    shape = key_pages.shape
    if len(shape) != 3 or value_pages.shape != shape:
        raise ValueError("key and value pages must have one shape, [num_blocks, kv_heads, bytes]")
    if not key_pages.is_cuda or value_pages.device != key_pages.device:
        raise ValueError("key and value pages must be on one CUDA device")
    blocks, heads, size = shape
    per_token = head_dim // 2 + 4
    if size == 0 or size % (16 * per_token):
        raise ValueError(f"{size} bytes for each head are no multiple of 16 tokens of "
                         f"{per_token} bytes (head_dim {head_dim})")
    ks, vs = key_pages.stride(), value_pages.stride()
    if (ks[2] != 1 or vs[2] != 1 or (heads > 1 and (ks[1] != size or vs[1] != size))):
        raise ValueError("the bytes of a page must be contiguous")
    if blocks > 1 and ks[0] != vs[0]:
        raise ValueError("key and value pages must have the same stride")
    return (key_pages.data_ptr(), value_pages.data_ptr(), ks[0] if blocks > 1 else heads * size,
            blocks, heads, size // per_token, head_dim)


def _rows(key: torch.Tensor, value: torch.Tensor, tokens: int, heads: int, head_dim: int,
          device: torch.device):
    """Checks key and value rows; (type code, four strides)."""
    kind = _DTYPES.get(key.dtype)
    if kind is None or value.dtype is not key.dtype:
        raise TypeError("key and value must both be bfloat16, float16 or float32, "
                        f"got {key.dtype} and {value.dtype}")
    shape = (tokens, heads, head_dim)
    if tuple(key.shape) != shape or tuple(value.shape) != shape:
        raise ValueError(f"key and value must be [tokens, kv_heads, head_dim] = {list(shape)}, "
                         f"got {list(key.shape)} and {list(value.shape)}")
    if key.device != device or value.device != device:
        raise ValueError("key and value must be on the device of the cache")
    ks, vs = key.stride(), value.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("the elements of a row must be contiguous")
    return kind, ks[0], ks[1], vs[0], vs[1]


def _slots(slots: torch.Tensor, device: torch.device) -> int:
    if slots.dtype is not torch.int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise ValueError("slots must be a contiguous int64 tensor of one dimension")
    if slots.device != device:
        raise ValueError("slots must be on the device of the cache")
    return slots.shape[0]


def _call(device: torch.device, name: str, *args) -> None:
    fn = getattr(_lib.lib(), name)
    index = device.index
    if torch.cuda.current_device() == index:
        status = fn(*args, _lib.current_stream_handle(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _lib.current_stream_handle(index))
    if status:
        _lib.check(status)


def write(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
          value_pages: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise ``key`` and ``value`` ``[tokens, kv_heads, head_dim]`` (bfloat16,
    float16 or float32; any strides with contiguous rows) into ``slots``
    (int64 ``[tokens]``; negative: the row is skipped).  The slots of one call
    must be distinct.

    For each row: ``scale = fp16((max - min) / 15)``, ``zero = fp16(min)`` and
    ``code = rint((x - zero) / scale)`` in [0, 15].  Values beyond +-65504 are
    clamped; a row with a NaN or an infinity reads back as NaN."""
    if key.dim() != 3:
        raise ValueError("key must be [tokens, kv_heads, head_dim]")
    device = key_pages.device
    c = _cache(key_pages, value_pages, key.shape[2])
    tokens = _slots(slots, device)
    kind, *strides = _rows(key, value, tokens, c[4], c[6], device)
    if tokens:
        _call(device, "kvx_q4_write", key.data_ptr(), value.data_ptr(), kind, tokens, *strides,
              slots.data_ptr(), *c)


def read(key_pages: torch.Tensor, value_pages: torch.Tensor, slots: torch.Tensor, *,
         head_dim: int, dtype: torch.dtype = torch.bfloat16,
         out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The key and value rows of ``slots`` (int64 ``[tokens]``; negative: a row
    of zeros) as ``[tokens, kv_heads, head_dim]`` in ``dtype``, or into the
    tensors of ``out``."""
    device = key_pages.device
    c = _cache(key_pages, value_pages, head_dim)
    tokens = _slots(slots, device)
    if out is None:
        if dtype not in _DTYPES:
            raise TypeError(f"rows are read as bfloat16, float16 or float32, not {dtype}")
        key = torch.empty((tokens, c[4], head_dim), dtype=dtype, device=device)
        value = torch.empty_like(key)
    else:
        key, value = out
    kind, *strides = _rows(key, value, tokens, c[4], head_dim, device)
    if tokens:
        _call(device, "kvx_q4_read", *c, slots.data_ptr(), tokens, key.data_ptr(),
              value.data_ptr(), kind, *strides)
    return key, value


def _workspace(device: torch.device, head_dim: int, rows: int) -> int:
    rows = min(rows, 33)  # more rows than the largest tile make no difference
    got = _workspace_bytes.get((device.index, head_dim, rows))
    if got is None:
        import ctypes

        n = ctypes.c_uint64()
        with torch.cuda.device(device):
            _lib.check(_lib.lib().kvx_q4_attention_workspace(head_dim, rows, ctypes.byref(n)))
        got = _workspace_bytes[(device.index, head_dim, rows)] = n.value
    return got


def attention(query: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor,
              block_tables: torch.Tensor, seq_lens: torch.Tensor, *,
              query_starts: Optional[torch.Tensor] = None, scale: Optional[float] = None,
              window: Optional[int] = None, sinks: int = 0,
              out: Optional[torch.Tensor] = None, return_lse: bool = False
              ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Causal attention of ``query`` ``[tokens, heads, head_dim]`` (bfloat16 or
    float16) over the cache; ``heads`` is a multiple of the cache's kv heads.

    ``seq_lens`` (int32 ``[batch]``) counts the tokens of each sequence in the
    cache, those of this call's queries among them (``write`` them first);
    ``block_tables`` (int32 ``[batch, width]``) names their blocks.  The queries
    of a sequence are its last tokens: ``tokens / batch`` each, or rows
    ``query_starts[b]`` to ``query_starts[b + 1]`` (int32 ``[batch + 1]``).
    A length of 0 marks a padded sequence: its rows are 0.

    ``window``: a query sees itself and the ``window - 1`` tokens before it, and
    besides them the first ``sinks`` tokens of its sequence.  ``scale``:
    1 / sqrt(head_dim) by default.  ``return_lse``: also the natural
    log-sum-exp of each row's scores, float32 ``[tokens, heads]`` (-inf for a
    row that sees nothing, whose output is 0).  Rows of ``out`` behind the last
    sequence of ``query_starts`` are left as they were."""
    if query.dim() != 3:
        raise ValueError("query must be [tokens, heads, head_dim]")
    device = key_pages.device
    tokens, heads, head_dim = query.shape
    c = _cache(key_pages, value_pages, head_dim)
    kind = _DTYPES.get(query.dtype)
    if kind is None or kind == _lib.DTYPE_FP32:
        raise TypeError(f"query must be bfloat16 or float16, got {query.dtype}")
    if heads == 0 or heads % c[4]:
        raise ValueError(f"{heads} query heads are no multiple of {c[4]} kv heads")
    if block_tables.dtype is not torch.int32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be an int32 tensor [batch, width]")
    if seq_lens.dtype is not torch.int32 or seq_lens.dim() != 1 or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 tensor [batch]")
    batch, width = block_tables.shape
    if seq_lens.shape[0] != batch:
        raise ValueError(f"block_tables has {batch} sequences but seq_lens has "
                         f"{seq_lens.shape[0]}")
    ts = block_tables.stride()
    if width > 1 and ts[1] != 1:
        raise ValueError("the entries of a block table must be contiguous")
    qs = query.stride()
    if qs[2] != 1:
        raise ValueError("the elements of a query row must be contiguous")
    if query.device != device or block_tables.device != device or seq_lens.device != device:
        raise ValueError("all tensors must be on the device of the cache")
    if query_starts is None:
        if batch == 0 or tokens % batch:
            if tokens:
                raise ValueError(f"{tokens} query tokens cannot be shared by {batch} sequences "
                                 "alike; pass query_starts")
        rows = tokens // batch if batch else 0
        starts = None
    else:
        if (query_starts.dtype is not torch.int32 or query_starts.dim() != 1
                or not query_starts.is_contiguous() or query_starts.shape[0] != batch + 1):
            raise ValueError("query_starts must be a contiguous int32 tensor [batch + 1]")
        if query_starts.device != device:
            raise ValueError("all tensors must be on the device of the cache")
        rows = tokens
        starts = query_starts.data_ptr()
    if window is not None and window < 1:
        raise ValueError("window must be at least 1 (None: no window)")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    elif not math.isfinite(scale):
        raise ValueError("scale must be finite")
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=query.dtype, device=device)
    elif (out.shape != query.shape or out.dtype is not query.dtype or out.device != device
          or out.stride(2) != 1):
        raise ValueError("out must have the shape, type and device of query and contiguous rows")
    lse = (torch.empty((tokens, heads), dtype=torch.float32, device=device)
           if return_lse else None)
    if tokens and batch:
        size = _workspace(device, head_dim, rows * (heads // c[4]))
        work = torch.empty(size, dtype=torch.uint8, device=device)
        os_ = out.stride()
        _call(device, "kvx_q4_attention", query.data_ptr(), qs[0], qs[1], out.data_ptr(), os_[0],
              os_[1], None if lse is None else lse.data_ptr(), kind, tokens, heads, *c,
              block_tables.data_ptr(), ts[0], width, seq_lens.data_ptr(), starts, batch, scale,
              window or 0, sinks, work.data_ptr(), size)
    return (out, lse) if return_lse else out
