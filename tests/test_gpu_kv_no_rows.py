"""Calls of the KV-cache operators without rows: nothing happens, and an operand that has rows all the same is refused (its
output would come back unwritten)."""
import pytest
import torch

import custom_ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows(n, heads=2, dtype=torch.float16):
    return torch.zeros((n, heads, 64), dtype=dtype, device=DEV)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_nothing_to_do_and_refusals():
    cache = custom_ops.empty_int4_cache(3, 2, 32, 64, device=DEV)
    table, seq, start = i32(0, 1)[None], i32(5), i32(0, 0)
    par = dict(key_params=cache[2], value_params=cache[3])

    def append(k=rows(0), v=rows(0), **kw):
        return custom_ops.append_kv_cache(k, v, *cache[:2], table, seq, query_start=start, block_size=32, **par, **kw)

    def gather(**kw):
        return custom_ops.gather_kv_cache(*cache[:2], table, seq, 2, query_start=start, block_size=32, **par, **kw)

    def attend(q=rows(0, 4), **kw):
        return custom_ops.paged_attention_int4(q, *cache, table, seq, 0.1, 2, query_start=start, block_size=32, **kw)

    mine = rows(0, 4)
    assert append() is None and append(query=rows(0, 4)).shape == (0, 4, 64) and append(query=rows(0, 4), query_out=mine) is mine
    assert gather(num_tokens=0)[0].shape == (0, 2, 64) and gather(key_out=rows(0), value_out=rows(0))[1].shape == (0, 2, 64)
    assert attend().shape == (0, 4, 64) and attend(out=mine, softmax_lse=torch.empty((0, 4), device=DEV)) is mine
    for f, word in ((lambda: append(query=rows(5, 4)), "query"), (lambda: append(v=rows(5)), "value"),
                    (lambda: append(query=rows(0, 4), query_out=rows(5, 4)), "query_out"), (lambda: gather(key_out=rows(0), value_out=rows(5)), "value_out"),
                    (lambda: attend(out=rows(5, 4)), "out"), (lambda: attend(softmax_lse=torch.empty((5, 4), device=DEV)), "softmax_lse")):
        with pytest.raises(RuntimeError, match=f"no rows.* {word} "):
            f()
    assert not any(bool(t.any()) for t in cache)
