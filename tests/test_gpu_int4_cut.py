"""A call over the first rows of a batch only: query_start goes on behind them.  The rows keep the positions that they have in
the whole batch, for the append, the read-back and the attention alike."""
import pytest
import torch

import custom_ops
from test_gpu_int4_attention import DEV, check, dev, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,s,Hq,Hkv,D,cut", [([5, 4, 9], [40, 300, 20], 4, 2, 64, 7), ([70, 60], [90, 200], 4, 2, 128, 101),
                                              ([3, 300], [64, 310], 8, 1, 128, 5), ([6, 8], [6, 8], 2, 2, 256, 9)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_over_the_first_rows(n, s, Hq, Hkv, D, cut, causal):
    c = make(61, n, s, Hq, Hkv, D, 32, "f16")
    c["q"], c["T"] = c["q"][:cut].contiguous(), cut
    check(c, causal)


def test_the_same_rows_as_in_the_whole_call():
    c = make(62, [5, 60], [50, 400], 8, 2, 64, 32, "f16")
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((65, 2, 64), generator=g).half().to(DEV) for _ in range(2))
    table, seq, start = dev(c["table"]), dev(c["seq"]), dev(c["start"])
    out = []
    for T in (65, 30):
        cache = custom_ops.empty_int4_cache(c["blocks"], 2, 32, 64, device=DEV)
        kw = dict(query_start=start, block_size=32)
        par = dict(key_params=cache[2], value_params=cache[3])
        custom_ops.append_kv_cache(k, v, *cache[:2], table, seq, **kw, **par)
        if T < 65:                                                     # again, the first rows only: the same places, the same bits
            custom_ops.append_kv_cache(k[:T], v[:T], *cache[:2], table, seq, **kw, **par)
        back = custom_ops.gather_kv_cache(*cache[:2], table, seq, 2, num_tokens=T, **kw, **par)
        out.append((*cache, *(b[:30] for b in back),
                    custom_ops.paged_attention_int4(dev(c["q"])[:T], *cache, table, seq, 0.125, 2, max_query_len=60, **kw)[:30]))
    torch.cuda.synchronize()
    for a, b in zip(out[0][:-1], out[1][:-1]):
        assert torch.equal(a, b)
    assert (out[0][-1] - out[1][-1]).abs().max() <= 2.0 ** -9       # (another plan; a row off by one position is far from it)
