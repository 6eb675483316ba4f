"""Outputs of the KV-cache operators that share memory with another operand: refused where that would be a race, right where
the documentation allows it (attention into query itself, rotation in place)."""
import pytest
import torch

import custom_ops
from test_gpu_int4_attention import call, dev, make

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("n,s,Hq,Hkv,D", [([1] * 3, [9000, 40, 700], 8, 2, 128), ([5, 2, 9], [3000, 40, 90], 8, 1, 64), ([300, 5], [400, 70], 4, 2, 128),
                                          ([3, 1], [64, 500], 20, 1, 256)])
def test_attention_into_its_query(n, s, Hq, Hkv, D):
    c = make(51, n, s, Hq, Hkv, D, 32, "f16")
    want = call(c)
    q = dev(c["q"]).clone()
    assert call(c, q=q, out=q) is q and torch.equal(q, want)


def test_overlaps():
    c = make(52, [2, 1], [30, 40], 4, 2, 64, 32, "f16")
    room = torch.zeros(8 * 3 * 4 * 64, dtype=torch.float16, device=DEV)
    q = room[:768].view(3, 4, 64)
    for out in (room[64:832].view(3, 4, 64), room[:1536].view(torch.float32).view(3, 4, 64)):
        with pytest.raises(RuntimeError, match="overlap"):
            call(c, q=q, out=out)
    with pytest.raises(RuntimeError, match="overlap"):
        call(c, q=room[:1536].view(3, 4, 128)[..., :64], out=q)
    call(c, q=q, out=room[768:1536].view(3, 4, 64))
    cache = custom_ops.empty_int4_cache(3, 2, 32, 64, device=DEV)
    table, seq = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), torch.tensor([5], dtype=torch.int32, device=DEV)
    kw = dict(block_size=32, key_params=cache[2], value_params=cache[3])
    k = room[:128].view(1, 2, 64)
    for v in (k, room[64:192].view(1, 2, 64)):
        with pytest.raises(RuntimeError, match="overlap"):
            custom_ops.gather_kv_cache(*cache[:2], table, seq, 2, key_out=k, value_out=v, **kw)
    custom_ops.gather_kv_cache(*cache[:2], table, seq, 2, key_out=k, value_out=room[128:256].view(1, 2, 64), **kw)
    torch.cuda.synchronize()
