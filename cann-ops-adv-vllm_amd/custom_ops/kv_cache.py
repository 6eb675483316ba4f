"""KV-cache operators: what fills the paged cache that the sparse attention ops read, a cache held in 4 bits, and dense
attention over it.  No counterpart in the reference, whose ops only read the cache (extension/custom_ops/add_custom.py);
conventions (block_table, seq_len, block_size, antiquant parameters, GPU tensors only, torch's current stream) are those of
`add_custom`.

Tokens of a call.  Rows query_start[b] .. query_start[b + 1] belong to sequence b (query_start [B + 1] int32 on the GPU;
None: row b, one per sequence).  The i-th of n rows stands at position seq_len[b] - n + i — seq_len [B] int32 counts the
sequence with its new rows — and lives in row pos % block_size of page block_table[b][pos // block_size].

The 4-bit cache is four tensors (`empty_int4_cache`): a token of a kv head is D codes and a (scale, zero) pair,
x = scale * code + zero.
    key_cache    uint8 [blocks, Hkv, bs, D / 2]         byte i: channel 2 i (low bits), channel 2 i + 1 (high bits)
    value_cache  uint8 [blocks, Hkv, bs / 4, D / 2, 4]  the same bytes, those of four consecutive tokens side by side
    key_params, value_params  float16 [blocks, Hkv, bs, 2]
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _abi


class Int4Cache(NamedTuple):
    key_cache: torch.Tensor
    value_cache: torch.Tensor
    key_params: torch.Tensor
    value_params: torch.Tensor


def empty_int4_cache(num_blocks: int, num_key_value_heads: int, block_size: int, head_dim: int, device="cuda") -> Int4Cache:
    """The tensors of a 4-bit cache, zeroed (every token reads as zeros)."""
    if block_size <= 0 or block_size % 16 or head_dim not in (32, 64, 128, 256):
        raise _abi.AclError("a 4-bit cache needs a block size that is a multiple of 16 and a head dim of 32, 64, 128 or 256")
    n, h, bs, d = int(num_blocks), int(num_key_value_heads), int(block_size), int(head_dim)
    zeros = lambda shape, dt: torch.zeros(shape, dtype=dt, device=device)   # noqa: E731
    return Int4Cache(zeros((n, h, bs, d // 2), torch.uint8), zeros((n, h, bs // 4, d // 2, 4), torch.uint8),
                     zeros((n, h, bs, 2), torch.float16), zeros((n, h, bs, 2), torch.float16))


def append_kv_cache(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                    block_table: torch.Tensor, seq_len: torch.Tensor, *, query: Optional[torch.Tensor] = None,
                    query_out: Optional[torch.Tensor] = None, query_start: Optional[torch.Tensor] = None,
                    cos_sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                    interleaved: bool = False, block_size: int = 128, antiquant_scale: Optional[torch.Tensor] = None,
                    antiquant_offset: Optional[torch.Tensor] = None, antiquant_mode: int = 0,
                    key_params: Optional[torch.Tensor] = None, value_params: Optional[torch.Tensor] = None
                    ) -> Optional[torch.Tensor]:
    """Write the new rows key, value [T, Hkv, D] (float16 / bfloat16, any token and head stride) into the paged cache,
    rotated by position on the way; query [T, Hq, D] is rotated along and returned (None without query).  One launch.

    cos_sin [rows, R] (float32 or the rows' dtype): R / 2 cosines, then R / 2 sines of a position; the channel pairs
    (i, i + R / 2) — (2 i, 2 i + 1) with interleaved — of q and K turn by them, channels from R on pass through.  positions
    [T] int32 names the table rows (default: the position in the sequence).  No cos_sin: no rotation.

    The caches have the rows' dtype ([blocks, bs, Hkv * D], [blocks, bs, Hkv, D] or [blocks, Hkv, bs, D]), are int8 in the
    same shapes (antiquant_scale / antiquant_offset as the attention ops take them, modes 0 and 2) or uint8: 4 bits, with
    key_params / value_params.  query_out may be query itself; where it is given, rows in no sequence are left as they are
    (a new tensor holds zeros there)."""
    return _abi.native.append(key, value, key_cache, value_cache, block_table, seq_len, query, query_out, query_start, cos_sin,
                              positions, antiquant_scale, antiquant_offset, key_params, value_params, block_size,
                              bool(interleaved), antiquant_mode)


def gather_kv_cache(key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor, seq_len: torch.Tensor,
                    num_key_value_heads: int, *, query_start: Optional[torch.Tensor] = None, num_tokens: Optional[int] = None,
                    block_size: int = 128, antiquant_scale: Optional[torch.Tensor] = None,
                    antiquant_offset: Optional[torch.Tensor] = None, antiquant_mode: int = 0,
                    key_params: Optional[torch.Tensor] = None, value_params: Optional[torch.Tensor] = None,
                    out_dtype: Optional[torch.dtype] = None, key_out: Optional[torch.Tensor] = None,
                    value_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The last rows of every sequence (query_start; None: the last one) out of a paged cache of any type, in 16 bits:
    (K [T, Hkv, D], V).  num_tokens is T (needed with query_start, which lives on the GPU).  Tokens without a place in the
    cache read as zeros; rows in no sequence are zeros in new tensors and left as they are in key_out / value_out.
    out_dtype: float16 or bfloat16 (default: the cache's, the antiquant parameters' or float16); where key_out is given out_dtype and
    num_key_value_heads have to agree with it and num_tokens must not exceed its rows."""
    if (key_out is None) != (value_out is None):
        raise _abi.AclError("gather_kv_cache: key_out and value_out come together")
    n = heads = d = 0
    if num_key_value_heads < 1:
        raise _abi.AclError("gather_kv_cache: num_key_value_heads must be positive")
    if key_out is not None:
        # the outputs say it all: what else was said must not contradict them
        if out_dtype not in (None, key_out.dtype):
            raise _abi.AclError(f"gather_kv_cache: out_dtype is {out_dtype}, key_out's {key_out.dtype}")
        if key_out.dim() == 3 and num_key_value_heads != key_out.shape[1]:
            raise _abi.AclError(f"gather_kv_cache: num_key_value_heads is {num_key_value_heads}, key_out has {key_out.shape[1]} heads")
        if key_out.dim() == 3 and num_tokens is not None and num_tokens > key_out.shape[0]:
            raise _abi.AclError(f"gather_kv_cache: num_tokens is {num_tokens}, key_out has {key_out.shape[0]} rows")
    else:
        if num_tokens is None:
            if query_start is not None:
                raise _abi.AclError("gather_kv_cache: num_tokens must be given with query_start")
            num_tokens = seq_len.shape[0]
        n, heads, d = int(num_tokens), int(num_key_value_heads), key_cache.shape[-1]
        if key_cache.dtype == torch.uint8:
            d *= 2
        elif key_cache.dim() != 4:
            d //= heads
        if out_dtype is None:
            out_dtype = {torch.uint8: torch.float16, torch.int8: getattr(antiquant_scale, "dtype", torch.float16)}.get(
                key_cache.dtype, key_cache.dtype)
        if out_dtype not in (torch.float16, torch.bfloat16):
            raise _abi.AclError("gather_kv_cache: out_dtype must be float16 or bfloat16")
    return _abi.native.gather(key_cache, value_cache, key_params, value_params, block_table, seq_len, query_start, antiquant_scale,
                              antiquant_offset, key_out, value_out, block_size, antiquant_mode, n, heads, d, out_dtype == torch.bfloat16)


def paged_attention_int4(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, key_params: torch.Tensor,
                         value_params: torch.Tensor, block_table: torch.Tensor, seq_len: torch.Tensor, scale_value: float,
                         num_key_value_heads: int, *, query_start: Optional[torch.Tensor] = None,
                         max_query_len: Optional[int] = None, causal: bool = True,
                         block_position: Optional[torch.Tensor] = None, block_size: int = 128,
                         softmax_lse: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                         out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Attention of query [T, Hq, D] over a 4-bit cache; returns [T, Hq, D] in query's dtype (out_dtype=torch.float32: not
    rounded).  One launch.

    query_start None: decode, one row per sequence.  With query_start: several rows per sequence (candidate tokens, prompt
    chunks; append_kv_cache has stored their K and V), max_query_len the most rows of one sequence (default T).  It decides how
    the work is shared out, so the exact number is the quickest — a batch of single rows planned for T rows may take half as
    much time again — while the results of any other one differ in rounding only.  causal: a row sees the tokens up to its own position;
    False: all seq_len[b] tokens (an encoder's states).
    block_position [B, Hq | Hkv, P] int32 (decode only): the logical pages each row attends, as cent_select returns them.
    softmax_lse: float32 [T, Hq], filled with the rows' log-sum-exp.  A row that sees no token is zero; rows in no sequence
    are zero in a new tensor and left as they are in `out`."""
    want = out.dtype if out is not None else query.dtype
    if out_dtype is not None and out_dtype != want:
        if out is not None or out_dtype != torch.float32:
            raise _abi.AclError("paged_attention_int4: out_dtype must be query's dtype or float32, and out's where out is given")
        want = out_dtype
    return _abi.native.attention(query, key_cache, value_cache, key_params, value_params, block_table, seq_len, query_start,
                                 block_position, out, softmax_lse, scale_value, num_key_value_heads, block_size,
                                 -1 if max_query_len is None else max_query_len, bool(causal), want == torch.float32)
