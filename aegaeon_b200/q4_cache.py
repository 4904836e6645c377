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
anything is queued (ValueError, TypeError), also that what a call writes overlaps
neither itself nor what it reads.  What is in device memory the kernels check: a
slot or block id outside its buffer is skipped and a length is cut to its block
table, which shows in ``_lib.device_status``; a length below 0 counts as 0.  None
of them has a gradient: a tensor that requires one is refused unless gradients are
off, one that carries a forward-mode gradient always is.  What they write to counts a version
on.  The reference has no counterpart (its caches hold 16-bit values).
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib

HEAD_DIMS = (64, 128, 256)


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


def write(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor,
          value_pages: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise ``key`` and ``value`` ``[tokens, kv_heads, head_dim]`` (bfloat16,
    float16 or float32; any strides with contiguous rows) into ``slots``
    (int64 ``[tokens]``; negative: the row is skipped).  The slots of one call
    must be distinct.

    For each row: ``scale = fp16((max - min) / 15)``, ``zero = fp16(min)`` and
    ``code = rint((x - zero) / scale)`` in [0, 15].  Values beyond +-65504 are
    clamped; a row with a NaN or an infinity reads back as NaN."""
    status = _lib.q4().write(key, value, key_pages, value_pages, slots)
    if status:
        _lib.check(status)


def read(key_pages: torch.Tensor, value_pages: torch.Tensor, slots: torch.Tensor, *,
         head_dim: int, dtype: torch.dtype = torch.bfloat16,
         out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
         ) -> Tuple[torch.Tensor, torch.Tensor]:
    """The key and value rows of ``slots`` (int64 ``[tokens]``; negative: a row
    of zeros) as ``[tokens, kv_heads, head_dim]`` in ``dtype``, or into the
    tensors of ``out``.  Scale and zero are rounded, so the top of a row that reaches
    65504 may lie above it, by less than 80: from 65520 on that is infinity in
    float16, in an attention's output too; bfloat16 and float32 hold it."""
    key, value = (None, None) if out is None else out
    status, key, value = _lib.q4().read(key_pages, value_pages, slots, head_dim, dtype, key, value)
    if status:
        _lib.check(status)
    return key, value


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
    ``query_starts[b]`` to ``query_starts[b + 1]`` (int32 ``[batch + 1]``, not decreasing;
    the call's kernel is then chosen by all its rows, so single tokens of long
    sequences are better called apart from pieces of prompts).
    A length of 0 marks a padded sequence: its rows are 0.

    ``window``: a query sees itself and the ``window - 1`` tokens before it, and
    besides them the first ``sinks`` tokens of its sequence.  ``scale``:
    1 / sqrt(head_dim) by default.  ``return_lse``: also the natural
    log-sum-exp of each row's scores, float32 ``[tokens, heads]`` (-inf for a
    row that sees nothing, whose output is 0).  Rows of ``out`` behind the last
    sequence of ``query_starts`` are left as they were, and the log-sum-exp has
    nothing there."""
    status, out, lse = _lib.q4().attention(query, key_pages, value_pages, block_tables, seq_lens,
                                           query_starts, scale, window, sinks, out, return_lse)
    if status:
        _lib.check(status)
    return (out, lse) if return_lse else out
