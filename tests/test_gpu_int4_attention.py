"""paged_attention_int4 against the 64-bit restatement in oracle/kv_cache.py (tolerances derived there, attention_bound)."""
import numpy as np
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def make(seed, n, s, Hq, Hkv, D, bs, dtype, decode=False, extra_rows=0, peaky=1.0, spare_pages=0):
    g = torch.Generator().manual_seed(seed)
    B, T = len(n), sum(n) + extra_rows
    width = max(1, max(-(-x // bs) for x in s)) + spare_pages
    blocks = B * width + 2
    table = torch.randperm(blocks, generator=g)[:B * width].reshape(B, width).to(torch.int32)
    kc, vc = (torch.randint(0, 16, (blocks, Hkv, bs, D), generator=g, dtype=torch.uint8) for _ in range(2))
    pars = []
    for _ in range(2):
        sc = 0.3 * torch.exp(0.5 * torch.randn((blocks, Hkv, bs), generator=g))
        pars.append(torch.stack((sc, -7.5 * sc + 0.3 * torch.randn(sc.shape, generator=g)), -1).half())
    q = (peaky * torch.randn((T, Hq, D), generator=g)).to(DT[dtype])
    start = None if decode else torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32)
    return dict(n=n, s=s, Hq=Hq, Hkv=Hkv, D=D, bs=bs, dt=DT[dtype], kc=kc, vc=vc, kp=pars[0], vp=pars[1], q=q, table=table,
                seq=torch.tensor(s, dtype=torch.int32), start=start, blocks=blocks, T=T)


def dev(t):
    return None if t is None else t.to(DEV)


def call(c, causal=True, lists=None, q=None, **kw):
    return custom_ops.paged_attention_int4(dev(c["q"]) if q is None else q, dev(kvo.pack_k(c["kc"])), dev(kvo.pack_v(c["vc"])), dev(c["kp"]),
                                           dev(c["vp"]), dev(c["table"]), dev(c["seq"]), c["D"] ** -0.5, c["Hkv"],
                                           query_start=dev(c["start"]), max_query_len=max(c["n"]), causal=causal,
                                           block_position=dev(lists), block_size=c["bs"], **kw)


def want_of(c, causal=True, lists=None):
    return kvo.attention(c["q"], kvo.values4(c["kc"], c["kp"]), kvo.values4(c["vc"], c["vp"]), c["table"], c["seq"], c["D"] ** -0.5,
                         c["Hkv"], c["bs"], c["start"], causal, lists)


def check(c, causal=True, lists=None, out_dtype=None):
    lse = torch.full((c["T"], c["Hq"]), 5.0, device=DEV)
    out = call(c, causal, lists, softmax_lse=lse, out_dtype=out_dtype)
    torch.cuda.synchronize()
    want, wlse, big = want_of(c, causal, lists)
    got, glse = out.cpu().double(), lse.cpu().double()
    live = ~torch.isnan(wlse)
    assert not got[~live].any() and bool((glse[~live] < -3.3e38).all())
    bound = kvo.attention_bound(want, big, c["D"], out.dtype)
    err = (got - want).abs()
    worst = (err / bound)[live].max().item()
    assert worst <= 1.0, f"off by {worst:.2f} of the bound"
    seen = live & (wlse > -3e38)
    A = big[..., 1]
    slack = 2.0 ** -24 * (c["D"] + 8) * A + 2.0 ** -20 * (2 + A)
    assert ((glse - wlse).abs()[seen] <= slack[seen]).all()
    assert bool((glse[live & ~seen] < -3.3e38).all()) and not got[live & ~seen].any()
    return out


DECODE = [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 127, 129, 257, 700]


@pytest.mark.parametrize("Hq,Hkv,D,bs,dtype", [
    (4, 4, 128, 128, "f16"), (8, 2, 128, 16, "f16"), (16, 1, 128, 48, "bf16"), (5, 1, 64, 64, "f16"), (8, 8, 64, 16, "bf16"),
    (4, 2, 256, 128, "f16"), (3, 3, 32, 32, "f16"), (24, 1, 128, 128, "f16"), (40, 1, 64, 16, "bf16"), (64, 1, 128, 64, "f16"),
    (20, 1, 256, 16, "bf16"), (64, 1, 256, 32, "f16"), (48, 1, 32, 16, "f16"),
])
def test_decode(Hq, Hkv, D, bs, dtype):
    check(make(Hq + D, [1] * len(DECODE), DECODE, Hq, Hkv, D, bs, dtype, decode=True))


@pytest.mark.parametrize("peaky", [0.0, 8.0, 60.0])
def test_flat_and_peaked_scores(peaky):
    check(make(5, [1] * 4, [300, 64, 65, 1000], 4, 2, 128, 64, "f16", decode=True, peaky=peaky))


def test_one_long_sequence_is_shared():
    c = make(6, [1], [20000], 4, 2, 64, 128, "f16", decode=True)
    check(c)
    c = make(7, [1, 1, 1], [9000, 3, 4000], 2, 1, 128, 16, "bf16", decode=True)
    check(c)


@pytest.mark.parametrize("Hq,Hkv,D,bs,dtype,causal", [
    (4, 4, 128, 128, "f16", True), (8, 2, 128, 16, "bf16", True), (32, 4, 64, 48, "f16", True), (4, 2, 256, 64, "f16", True),
    (6, 2, 32, 32, "bf16", True), (8, 2, 128, 64, "f16", False), (16, 2, 256, 16, "bf16", False),
])
def test_several_rows(Hq, Hkv, D, bs, dtype, causal):
    """Candidate tokens: a few rows per sequence, some longer than the sequence itself (its first rows see nothing)."""
    c = make(Hq * D, [1, 4, 2, 7, 0, 3, 5], [100, 4, 33, 300, 50, 1, 64], Hq, Hkv, D, bs, dtype, extra_rows=3)
    check(c, causal)


@pytest.mark.parametrize("Hq,Hkv,D,bs,dtype,causal", [
    (4, 2, 128, 128, "f16", True), (2, 2, 64, 16, "bf16", True), (10, 2, 128, 48, "f16", True), (2, 1, 256, 64, "bf16", True),
    (3, 1, 32, 32, "f16", True), (2, 2, 128, 64, "f16", False),
])
def test_prompts(Hq, Hkv, D, bs, dtype, causal):
    c = make(Hq + D + bs, [130, 1, 257, 70], [130, 40, 400, 71], Hq, Hkv, D, bs, dtype, extra_rows=2)
    check(c, causal)


def _lists(c, rows, seed, P=9):
    g = np.random.default_rng(seed)
    out = np.full((len(c["s"]), rows, P), kvo.END, dtype=np.int32)
    for b, s in enumerate(c["s"]):
        pages = -(-s // c["bs"])
        for r in range(rows):
            k = int(g.integers(0, min(P, pages) + 1))
            out[b, r, :k] = np.sort(g.permutation(pages)[:k])
    return torch.from_numpy(out)


@pytest.mark.parametrize("Hq,Hkv,D,bs,per_head", [
    (4, 4, 128, 128, True), (8, 2, 128, 16, True), (8, 2, 64, 48, False), (24, 1, 128, 16, False), (2, 2, 256, 32, True),
    (64, 1, 64, 64, False), (4, 2, 32, 16, True),
])
def test_page_lists(Hq, Hkv, D, bs, per_head):
    c = make(D + bs, [1] * 6, [1, 20, 333, 64, 700, 0], Hq, Hkv, D, bs, "f16", decode=True)
    lists = _lists(c, Hq if per_head else Hkv, 3)
    lists[4, 0, :3] = torch.tensor([3, 1, 1])            # neither ascending nor distinct
    lists[4, -1, 1] = c["table"].shape[1]                # outside the table: the list ends here
    lists[2, 0, 0] = -5
    check(c, lists=lists)


def test_a_long_list_is_shared():
    c = make(8, [1], [16000], 2, 2, 128, 16, "f16", decode=True)
    lists = torch.arange(1000, dtype=torch.int32).flip(0).repeat(1, 2, 1).contiguous()
    check(c, lists=lists)
    check(c, lists=torch.cat((lists, torch.full((1, 2, 300), kvo.END, dtype=torch.int32)), -1))


def test_pages_that_are_not_there():
    c = make(9, [1, 3, 90], [200, 300, 150], 4, 2, 128, 32, "f16")
    c["table"][0, 1], c["table"][1, 0], c["table"][2, 4] = -1, c["blocks"], 2 ** 31 - 1
    check(c)
    c["table"][0] = -1                                   # a sequence with no page at all
    out = check(c)
    assert not out[0].any()


def test_what_lies_behind_a_sequence_is_not_seen():
    """Parameters of rows behind the end hold NaN and infinities; pages behind it are never named."""
    c = make(10, [1, 40, 5], [37, 45, 100], 4, 2, 64, 64, "f16", spare_pages=1)
    base = call(c)
    for b, s in enumerate(c["s"]):
        for pos in range(s, c["table"].shape[1] * 64):
            for p in (c["kp"], c["vp"]):
                p[int(c["table"][b, pos // 64]), :, pos % 64] = torch.tensor([float("inf"), float("nan")])
    assert torch.equal(call(c), base)


def test_a_row_with_nan_reaches_only_those_who_see_it():
    c = make(11, [40], [60], 4, 2, 64, 16, "f16")
    base = call(c)
    page, row = int(c["table"][0, 40 // 16]), 40 % 16     # position 40: rows 20 .. 39 of the call see it
    c["vp"][page, 0, row, 1] = float("nan")
    got = call(c)
    assert torch.equal(got[:20], base[:20]) and torch.equal(got[20:, 2:], base[20:, 2:])
    assert bool(torch.isnan(got[20:, :2]).all())
    c["vp"][page, 0, row, 1], c["kp"][page, 1, row, 1] = 0.0, float("nan")
    got = call(c)
    assert torch.equal(got[:20], base[:20]) and bool(torch.isnan(got[20:, 2:]).all()) and bool(torch.isfinite(got[20:, :2]).all())


def test_extreme_queries_and_scales():
    c = make(12, [1] * 4, [70, 300, 33, 128], 2, 1, 128, 32, "bf16", decode=True)
    c["q"][0] = 0.0
    c["q"][1] *= 1e-30
    c["q"][2] *= 3000.0                                   # one token takes all
    c["vp"][:, :, ::7] = 0.0                              # rows of zeros
    c["vp"][:, :, 1::5] *= 1000.0                         # scales of very different sizes
    c["vp"][:, :, 2::5] *= 2.0 ** -10
    check(c)


def test_float32_output_and_strided_queries():
    c = make(13, [1, 9, 70], [50, 80, 300], 8, 2, 128, 64, "f16")
    out = check(c, out_dtype=torch.float32)
    wide = torch.zeros((c["T"], 12, 131), dtype=c["dt"], device=DEV)
    wide[:, 2:10, 1:129] = dev(c["q"])
    assert torch.equal(call(c, q=wide[:, 2:10, 1:129], out_dtype=torch.float32), out)


def test_rows_in_no_sequence_keep_a_callers_values():
    c = make(14, [3, 4], [50, 80], 4, 2, 64, 16, "f16", extra_rows=6)
    mine, lse = torch.full((13, 4, 64), 9.0, dtype=c["dt"], device=DEV), torch.full((13, 4), 9.0, device=DEV)
    out = call(c, out=mine, softmax_lse=lse)
    base = call(c)
    assert out is mine and torch.equal(mine[:7], base[:7]) and bool((mine[7:] == 9).all()) and bool((lse[7:] == 9).all())
    assert not base[7:].any()


def test_table_shorter_than_the_sequence():
    c = make(15, [1, 5, 90], [64, 64, 64], 4, 2, 64, 16, "f16")
    c["seq"] = torch.tensor([70, 66, 100], dtype=torch.int32)
    check(c)


def test_repeats_are_bit_equal():
    c = make(16, [1] * 5 , [5000, 3, 900, 12000, 64], 8, 2, 128, 64, "f16", decode=True)
    base = call(c)
    for _ in range(5):
        assert torch.equal(call(c), base)


def test_streams_and_workspaces():
    """Launches that interleave on two streams keep their counters and partial states apart."""
    cs = [make(17 + i, [1] * 3, [4000 + 700 * i, 30, 2000], 4, 2, 128, 64, "f16", decode=True) for i in range(2)]
    base = [call(c) for c in cs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(call(cs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g, base[i])


def test_offsets_beyond_32_bits():
    D, Hkv, bs = 256, 8, 128
    blocks = (5 << 30) // (Hkv * bs * D // 2)
    c = make(21, [1], [300], 8, Hkv, D, bs, "f16", decode=True)
    want = call(c)
    kc = torch.empty((blocks, Hkv, bs, D // 2), dtype=torch.uint8, device=DEV)
    vc = torch.empty((blocks, Hkv, bs // 4, D // 2, 4), dtype=torch.uint8, device=DEV)
    kp, vp = (torch.empty((blocks, Hkv, bs, 2), dtype=torch.float16, device=DEV) for _ in range(2))
    at = blocks - c["blocks"]
    for big, small in ((kc, kvo.pack_k(c["kc"])), (vc, kvo.pack_v(c["vc"])), (kp, c["kp"]), (vp, c["vp"])):
        big[at:] = small.to(DEV)
    out = custom_ops.paged_attention_int4(dev(c["q"]), kc, vc, kp, vp, dev(c["table"]) + at, dev(c["seq"]), D ** -0.5, Hkv, block_size=bs)
    assert torch.equal(out, want)
    del kc, vc, kp, vp
    torch.cuda.empty_cache()
