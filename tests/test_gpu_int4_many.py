"""paged_attention_int4 where the distribution of the work changes: more sequences than lanes of a wave, more items than
workgroups, a line of steps too long for 32-bit arithmetic, and rows few enough for weights in two parts (fp32 output)."""
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo
from test_gpu_int4_attention import DEV, check, dev, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,Hq,Hkv,D,bs,dtype", [(70, 4, 2, 128, 32, "f16"), (64, 2, 1, 64, 16, "bf16"), (130, 8, 1, 32, 48, "f16"),
                                                 (65, 3, 3, 256, 16, "f16")])
def test_many_sequences(B, Hq, Hkv, D, bs, dtype):
    s = [(37 * i * i + 11) % 260 for i in range(B)]
    s[3] = s[B - 1] = 0
    check(make(B + D, [1] * B, s, Hq, Hkv, D, bs, dtype, decode=True))


@pytest.mark.parametrize("B,Hkv,bs", [(40, 8, 32), (90, 16, 16), (8, 40, 128)])
def test_more_items_than_workgroups(B, Hkv, bs):
    """320 to 1440 items over 512 workgroups: pieces of the line end inside items, single items span several pieces."""
    s = [3 + (i * 53) % 90 for i in range(B)]
    s[1], s[B // 2] = 1900, 700
    check(make(B + Hkv, [1] * B, s, Hkv, Hkv, 64, bs, "f16", decode=True))


@pytest.mark.parametrize("n,Hq,Hkv,D", [([40, 3, 0, 77, 1, 130], 8, 2, 64), ([5] * 70, 4, 1, 128), ([33, 2, 65, 1] * 17, 2, 2, 32)])
def test_rows_of_many_tiles(n, Hq, Hkv, D):
    s = [x + (7 * i) % 64 for i, x in enumerate(n)]
    check(make(sum(n) + D, n, s, Hq, Hkv, D, 16, "f16", extra_rows=2))


def test_a_line_beyond_32_bits():
    """128 sequences x 8 heads x a table of 2^26 tokens: the longest lengths that the table allows add up beyond 2^31 steps, so
    the line is counted in 64 bits, though the lengths of this call are short."""
    B, Hkv, bs = 128, 8, 512
    s = [1 + (i * 29) % 200 for i in range(B)]
    c = make(9, [1] * B, s, Hkv, Hkv, 32, bs, "f16", decode=True)
    short = c["table"]
    wide = torch.full((B, (1 << 26) // bs), -1, dtype=torch.int32)
    wide[:, :short.shape[1]] = short
    c["table"] = wide
    check(c)


def test_two_parts_of_the_weights():
    """At most eight rows: a weight is held in two float16 parts, off by 2^-22 of itself and 2^-30 of the largest V scale
    absolutely; with flat scores (q so small that the score's own error is below 2^-20) and fp32 output the bound of
    attention_bound tightens from 2^-10 vmax to (2^-21 + 2^-30 n) vmax for the weights.  The single part misses it."""
    s = [1, 2, 3, 5, 17, 40]
    c = make(11, [1] * 6, s, 8, 1, 128, 16, "f16", decode=True, peaky=0.002)
    out = custom_ops.paged_attention_int4(dev(c["q"]), dev(kvo.pack_k(c["kc"])), dev(kvo.pack_v(c["vc"])), dev(c["kp"]), dev(c["vp"]),
                                          dev(c["table"]), dev(c["seq"]), c["D"] ** -0.5, 1, block_size=16, out_dtype=torch.float32)
    want, _, big = kvo.attention(c["q"], kvo.values4(c["kc"], c["kp"]), kvo.values4(c["vc"], c["vp"]), c["table"], c["seq"], c["D"] ** -0.5, 1, 16)
    vmax, A = big[..., :1], big[..., 1:]
    delta = 2.0 ** -24 * (c["D"] + 8) * A + 2.0 ** -21 * (1 + A)
    bound = (2 * delta + 2.0 ** -21 + 2.0 ** -30 * 40 + 2.0 ** -20) * vmax + 2.0 ** -24 * want.abs() + 2.0 ** -24
    assert ((out.cpu().double() - want).abs() <= bound).all()
    lists = torch.arange(3, dtype=torch.int32).repeat(6, 8, 1).to(DEV)
    lists[:, :, 1:] = torch.where(lists[:, :, 1:] * 16 < dev(c["seq"])[:, None, None], lists[:, :, 1:], -1)
    again = custom_ops.paged_attention_int4(dev(c["q"]), dev(kvo.pack_k(c["kc"])), dev(kvo.pack_v(c["vc"])), dev(c["kp"]), dev(c["vp"]),
                                            dev(c["table"]), dev(c["seq"]), c["D"] ** -0.5, 1, block_size=16, block_position=lists,
                                            out_dtype=torch.float32)
    assert ((again.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("D,bs,dtype,causal", [(128, 48, "f16", True), (64, 32, "bf16", True), (32, 16, "f16", False), (256, 16, "bf16", True)])
def test_many_rows(D, bs, dtype, causal):
    """512 rows x 64 heads: enough tiles for the four waves of a workgroup to share the rows."""
    check(make(D + bs, [300, 0, 212], [300, 5, 260], 64, 8, D, bs, dtype), causal)


@pytest.mark.parametrize("n,s,Hq,Hkv,D", [([16] * 8, [900 + 37 * i for i in range(8)], 8, 1, 64), ([9, 3, 16, 12], [3000, 70, 1200, 12], 8, 1, 128)])
def test_rows_of_two_waves(n, s, Hq, Hkv, D):
    """65 to 128 rows of a kv head in few items: two waves share the rows, two the tokens, parts of one item each."""
    check(make(sum(s), n, s, Hq, Hkv, D, 32, "f16"))
