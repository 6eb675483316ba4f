"""append_kv_cache / gather_kv_cache against the 64-bit restatement in oracle/kv_cache.py.

Tolerances (derived, not tuned).  Rotation: two products and a sum in fp32 on exact inputs, at most 3 roundings of
2^-24 (|x| + |y|), then one rounding to the row's type (half a step: fp16 2^-11, bf16 2^-8; fp16 subnormals 2^-25).  V is
copied: bit-equal in a 16-bit cache.  int8: the code of (x / s - o) may differ by one where the quotient lies within its own fp32
error of a border; the value read back is within s / 2 + that error (or the code is saturated).  4 bits: against the
parameters that were stored, every code is the nearest representable one (same reasoning); the stored zero of a V row is
exactly f16(lo), its scale within one f16 step of f16((hi - lo) / 15) (two roundings)."""
import numpy as np
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def make(seed, n, old, Hq, Hkv, D, bs, cache, dtype, layout="BSH", rot=None, interleaved=False, decode=False, extra_rows=0,
         cs_dtype=torch.float32, view=True):
    g = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    rot = D if rot is None else rot
    s = [a + b for a, b in zip(n, old)]
    B, T = len(n), sum(n) + extra_rows
    width = max(1, max(-(-x // bs) for x in s)) + 1
    blocks = B * width + 2
    table = torch.randperm(blocks, generator=g)[:B * width].reshape(B, width).to(torch.int32)
    start = None if decode else torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32)
    qkv = torch.randn((T, (Hq + 2 * Hkv) * D), generator=g).to(dt)
    pos_max = max(max(s), 1)
    ang = torch.arange(pos_max)[:, None].double() * 10000.0 ** (-torch.arange(0, rot, 2).double() / rot)
    cs = torch.cat((ang.cos(), ang.sin()), -1).to(cs_dtype)
    c = dict(n=n, s=s, B=B, T=T, Hq=Hq, Hkv=Hkv, D=D, bs=bs, cache=cache, dt=dt, layout=layout, rot=rot, interleaved=interleaved,
             table=table, seq=torch.tensor(s, dtype=torch.int32), start=start, qkv=qkv, cs=cs, blocks=blocks, kw={})
    if cache == "int4":
        c["bufs"] = [torch.randint(0, 256, sh, generator=g, dtype=torch.uint8) for sh in
                     ((blocks, Hkv, bs, D // 2), (blocks, Hkv, bs // 4, D // 2, 4))]
        c["pars"] = [torch.randn((blocks, Hkv, bs, 2), generator=g).half() for _ in range(2)]
    else:
        sh = (blocks, bs, Hkv, D) if layout == "BSH" else (blocks, Hkv, bs, D) if layout == "BNSD" else (blocks, bs, Hkv * D)
        if cache == "int8":
            c["bufs"] = [torch.randint(-128, 128, sh, generator=g, dtype=torch.int8) for _ in range(2)]
            c["scale"] = (0.02 + 0.02 * torch.rand((2, Hkv, D), generator=g)).to(dt)
            c["offset"] = torch.randint(-9, 10, (2, Hkv, D), generator=g).to(dt)
        else:
            c["bufs"] = [torch.randn(sh, generator=g).to(dt) for _ in range(2)]
    return c


def split(c, qkv):
    q, k, v = qkv.split([c["Hq"] * c["D"], c["Hkv"] * c["D"], c["Hkv"] * c["D"]], 1)
    return tuple(t.unflatten(1, (-1, c["D"])) for t in (q, k, v))


def to_dev(t):
    return None if t is None else t.to(DEV)


def call(c, positions=None, q_out=None, qkv=None, in_place=False, query=True, cos_sin="table"):
    qkv = to_dev(c["qkv"]) if qkv is None else qkv
    q, k, v = split(c, qkv)
    bufs = [to_dev(t) for t in c["bufs"]]
    kw = {}
    if c["cache"] == "int4":
        pars = [to_dev(t) for t in c["pars"]]
        kw = dict(key_params=pars[0], value_params=pars[1])
    if c["cache"] == "int8":
        kw = dict(antiquant_scale=to_dev(c["scale"]), antiquant_offset=to_dev(c["offset"]), antiquant_mode=c.get("mode", 0))
    out = custom_ops.append_kv_cache(k, v, bufs[0], bufs[1], to_dev(c["table"]), to_dev(c["seq"]), query=q if query else None,
                                     query_out=q if in_place else q_out, query_start=to_dev(c["start"]),
                                     cos_sin=to_dev(c["cs"]) if cos_sin == "table" else None, positions=to_dev(positions),
                                     interleaved=c["interleaved"], block_size=c["bs"], **kw)
    back = custom_ops.gather_kv_cache(bufs[0], bufs[1], to_dev(c["table"]), to_dev(c["seq"]), c["Hkv"], query_start=to_dev(c["start"]),
                                      num_tokens=c["T"], block_size=c["bs"], out_dtype=c["dt"], **kw)
    torch.cuda.synchronize()
    return out, bufs, kw, back


def row_of(c, buf, page, row):
    """[Hkv, ...] of one token"""
    if c["cache"] == "int4" and buf.dim() == 5:
        return buf[page, :, row // 4, :, row % 4]
    if c["cache"] == "int4" or c["layout"] == "BNSD":
        return buf[page, :, row]
    return buf[page, row].reshape(c["Hkv"], c["D"])


def check(c, got, positions=None, query=True, turned=True):
    out, bufs, kw, back = got
    q, k, v = split(c, c["qkv"])
    half, tiny = HALF[c["dt"]], TINY[c["dt"]]
    places = kvo.tokens(c["table"], c["seq"], c["start"], c["T"], c["bs"], c["blocks"])
    bufs = [b.cpu() for b in bufs]
    pars = [kw["key_params"].cpu(), kw["value_params"].cpu()] if c["cache"] == "int4" else None
    back = [b.cpu() for b in back]
    left = [b.clone() for b in c["bufs"]]           # what must still be there
    left_p = [p.clone() for p in c["pars"]] if pars else None
    for t, (b, pos, page, row) in enumerate(places):
        cs = int(positions[t]) if positions is not None and b >= 0 else pos
        live = pos >= 0 and (not turned or 0 <= cs < c["cs"].shape[0])
        turn = (lambda x: kvo.rotate(x, c["cs"][cs], c["interleaved"])) if turned else (lambda x: x.double())
        if query:
            if not live:
                assert not out[t].any(), f"row {t}"
            else:
                want = turn(q[t])
                slack = half * want.abs() + 2.0 ** -22 * (2 * q[t].double().abs().amax(-1, keepdim=True)) + tiny
                assert ((out[t].cpu().double() - want).abs() <= slack).all(), f"query row {t}"
        if page < 0 or not live:
            if page < 0:
                assert not back[0][t].any() and not back[1][t].any()
            continue
        for which, x in ((0, turn(k[t])), (1, v[t].double())):
            err = 2.0 ** -22 * 2 * k[t].double().abs().amax(-1, keepdim=True) if which == 0 else torch.zeros(c["Hkv"], 1).double()
            stored = row_of(c, bufs[which], page, row)
            row_of(c, left[which], page, row).copy_(stored)
            if c["cache"] == "int4":
                s, z = (pars[which][page, :, row, i].double()[:, None] for i in (0, 1))
                left_p[which][page, :, row].copy_(pars[which][page, :, row])
                ws, wz = kvo.params4(x)
                step = 2.0 ** -10 * ws.double()[:, None] + 2.0 ** -24 + err / 7
                assert ((s - ws.double()[:, None]).abs() <= step).all()
                zstep = (2.0 ** -10 * wz.double().abs()[:, None] + 2.0 ** -24) * (which == 0)
                assert ((z - wz.double()[:, None]).abs() <= zstep + err).all()
                code = kvo.unpack_k(stored).double()
                val = code * s + z
                near = (val - x).abs() <= s * (0.5 + 2.0 ** -18) + err + 2.0 ** -22 * x.abs()
                low, high = (code == 0) & (x < z), (code == 15) & (x > z + 15 * s)
                assert (near | low | high | (s == 0)).all(), f"token {t}"
            elif c["cache"] == "int8":
                sc, of = c["scale"].double(), c["offset"].double()
                if sc.dim() == 2:                   # per kv head
                    sc, of = sc[..., None].expand(2, c["Hkv"], c["D"]), of[..., None].expand(2, c["Hkv"], c["D"])
                sc, of = sc[which], of[which]
                code = stored.double().reshape(c["Hkv"], c["D"])
                val = (code + of) * sc
                near = (val - x).abs() <= sc * (0.5 + 2.0 ** -14) + err
                assert (near | ((code == 127) & (x > val)) | ((code == -128) & (x < val))).all(), f"token {t}"
            else:
                val = stored.double().reshape(c["Hkv"], c["D"])
                if which == 1 or not turned:
                    assert torch.equal(stored.reshape(c["Hkv"], c["D"]), (k, v)[which][t])
                else:
                    assert ((val - x).abs() <= half * x.abs() + err + tiny).all()
            got_back = back[which][t].double()
            assert ((got_back - val).abs() <= half * val.abs() * 1.01 + 2.0 ** -20 + tiny).all(), f"read-back of token {t}"
    for a, b in zip(bufs, left):                    # nothing else was written
        assert torch.equal(a.view(torch.uint8) if a.dtype != torch.uint8 else a, b.view(torch.uint8) if b.dtype != torch.uint8 else b)
    if pars:
        for a, b in zip(pars, left_p):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


RAGGED = ([5, 1, 16, 3, 40], [0, 130, 7, 63, 9])
CASES = [
    # n, old, Hq, Hkv, D, bs, cache, dtype, layout, rot, interleaved, decode
    (*RAGGED, 8, 2, 128, 128, "f16", "f16", "BSH", 128, False, False),
    (*RAGGED, 8, 2, 128, 16, "int4", "f16", "BSH", 128, False, False),
    (*RAGGED, 4, 4, 64, 48, "int4", "bf16", "BSH", 32, False, False),
    (*RAGGED, 6, 2, 256, 64, "int4", "f16", "BSH", 64, True, False),
    (*RAGGED, 5, 1, 32, 32, "int4", "bf16", "BSH", 32, False, False),
    (*RAGGED, 8, 2, 128, 64, "int8", "f16", "BNSD", 96, False, False),      # pairs 48 apart
    (*RAGGED, 4, 2, 256, 32, "int8", "bf16", "3D", 64, True, False),
    (*RAGGED, 2, 1, 512, 16, "bf16", "bf16", "BNSD", 256, False, False),
    (*RAGGED, 4, 2, 64, 80, "f16", "f16", "3D", 20, False, False),          # pairs 10 apart: no whole chunks
    ([1] * 9, [0, 1, 2, 15, 16, 17, 127, 128, 300], 8, 8, 128, 128, "int4", "f16", "BSH", 128, False, True),
    ([1] * 70, list(range(70)), 4, 1, 64, 16, "f16", "f16", "BSH", 64, False, True),
    ([700, 0, 1, 1400, 3], [0, 5, 0, 1, 2], 2, 1, 64, 16, "int4", "f16", "BSH", 64, False, False),   # 4 tokens a workgroup
    ([2500], [3], 2, 1, 64, 128, "int4", "bf16", "BSH", 64, False, False),                           # 16 tokens a workgroup
    ([2200, 100], [0, 0], 1, 1, 32, 128, "int8", "f16", "BSH", 16, True, False),
]


@pytest.mark.parametrize("n,old,Hq,Hkv,D,bs,cache,dtype,layout,rot,inter,decode", CASES)
def test_append_and_read_back(n, old, Hq, Hkv, D, bs, cache, dtype, layout, rot, inter, decode):
    c = make(3 + D + len(n), n, old, Hq, Hkv, D, bs, cache, dtype, layout, rot, inter, decode)
    check(c, call(c))


@pytest.mark.parametrize("cache", ["f16", "int4", "int8"])
def test_rows_without_a_place(cache):
    """Negative table entries and entries beyond the pool, positions before the sequence and behind the table, rows in no
    sequence: nothing else is written for them and nothing out of bounds is touched."""
    c = make(11, [6, 9, 30, 4], [20, 0, 100, 0], 4, 2, 64, 32, cache, "f16", extra_rows=5)
    c["table"][0, 0] = -1
    c["table"][2, 3] = c["blocks"]
    c["table"][2, 0] = 2 ** 31 - 1
    c["seq"][1] = 5                       # nine rows, five tokens: the first four have no position
    c["seq"][3] = c["table"].shape[1] * c["bs"] + 2     # the last rows lie behind the table
    c["cs"] = c["cs"][:1].repeat(c["table"].shape[1] * c["bs"], 1)
    got = call(c)
    check(c, got)
    assert not got[0][-5:].any()
    # rows in no sequence keep what a caller's own tensor holds
    mine = torch.full((c["T"], 4, 64), 7.0, dtype=c["dt"], device=DEV)
    out = call(c, q_out=mine)[0]
    assert out is mine and bool((mine[-5:] == 7).all()) and torch.equal(mine[:-5], got[0][:-5])


def test_positions_and_short_tables_of_angles():
    c = make(12, [4, 7], [30, 2], 4, 2, 64, 16, "f16", "f16")
    positions = torch.tensor([0, 3, 1, 33, 2, 2, 33, 0, 1, 2, 3], dtype=torch.int32)
    check(c, call(c, positions), positions)
    positions[2], positions[5] = -1, c["cs"].shape[0]     # no such row: neither stored nor turned
    for cache in ("f16", "int4"):
        c = make(12, [4, 7], [30, 2], 4, 2, 64, 16, cache, "f16")
        out, bufs, kw, back = call(c, positions)
        q = split(c, c["qkv"])[0]
        assert not out[2].any() and not out[5].any() and out[1].any()
        places = kvo.tokens(c["table"], c["seq"], c["start"], c["T"], c["bs"], c["blocks"])
        for t in (2, 5):
            _, _, page, row = places[t]
            for b, b0 in zip(bufs, c["bufs"]):
                assert torch.equal(row_of(c, b.cpu(), page, row), row_of(c, b0, page, row))


@pytest.mark.parametrize("cache", ["f16", "int4"])
def test_without_rotation_and_without_query(cache):
    c = make(13, [4, 17, 1], [3, 0, 5], 4, 2, 64, 16, cache, "f16")
    check(c, call(c, cos_sin=None), turned=False)
    check(c, call(c, query=False), query=False)


@pytest.mark.parametrize("D,inter", [(64, False), (128, True)])
def test_in_place_and_unaligned_rows(D, inter):
    c = make(14, [9, 33], [0, 5], 4, 2, D, 16, "f16", "bf16" if inter else "f16", interleaved=inter)
    c["cache"] = "f16" if not inter else "bf16"
    base = call(c)
    qkv = to_dev(c["qkv"].clone())
    out = call(c, qkv=qkv, in_place=True)[0]              # query_out is query: a view of the projection
    assert torch.equal(out, base[0]) and out.data_ptr() == qkv.data_ptr()
    wide = torch.zeros((c["T"], c["qkv"].shape[1] + 3), dtype=c["dt"], device=DEV)
    wide[:, 1:-2] = to_dev(c["qkv"])
    got = call(c, qkv=wide[:, 1:-2])                      # odd strides, rows at 2-byte alignment
    assert torch.equal(got[0], base[0])
    for a, b in zip(got[1], base[1]):
        assert torch.equal(a, b)


def test_half_precision_table_of_angles():
    c = make(15, [9, 33], [0, 5], 4, 2, 128, 16, "f16", "f16", cs_dtype=torch.float16)
    check(c, call(c))


@pytest.mark.parametrize("mode", ["tensor", "head"])
def test_int8_parameter_layouts(mode):
    c = make(16, [9, 3], [0, 5], 4, 2, 64, 32, "int8", "f16")
    if mode == "tensor":
        c["scale"], c["offset"] = torch.tensor([0.03, 0.02]).half(), torch.tensor([3.0, -2.0]).half()
        got = call(c)
        c["scale"], c["offset"] = (x[:, None].repeat(1, 2) for x in (c["scale"], c["offset"]))
    else:
        c["scale"], c["offset"] = torch.tensor([[0.03, 0.02], [0.04, 0.01]]).half(), torch.tensor([[3.0, -2.0], [0.0, 1.0]]).half()
        c["mode"] = 2
        got = call(c)
    check(c, got)


def test_special_values():
    """Constant rows, rows at float16's border, bfloat16 beyond it, NaN and infinities."""
    c = make(17, [8], [0], 2, 1, 64, 16, "int4", "bf16")
    q, k, v = split(c, c["qkv"])
    v[0] = 3.0                                            # scale 0: every code 0, the zero is the value
    v[1] = 0.0
    v[2] = torch.linspace(-1e30, 1e30, 64)[None]          # saturates
    v[3, 0, 5] = float("nan")
    v[4, 0, 9] = float("inf")
    v[5] = torch.linspace(-60000, 60000, 64)[None]
    v[6] = torch.linspace(1e-6, 3e-6, 64)[None]           # float16 subnormal steps
    _, _, kw, back = call(c, cos_sin=None)
    got = back[1].cpu().float()
    assert bool((got[0] == 3).all()) and not got[1].any()
    assert bool(torch.isfinite(got[2]).all()) and float(got[2].min()) <= -65000
    assert bool(torch.isnan(got[3]).all()) and bool(torch.isnan(got[4]).all()) and bool(torch.isfinite(got[5]).all())
    assert ((got[5] - v[5].float()).abs() <= 4001 + 2.0 ** -7 * v[5].float().abs()).all()
    # steps of 2^-24 (1.3e-7 of span / 15): off by half a step, the rounding of the zero and 15 half-roundings of the scale
    assert ((got[6] - v[6].float()).abs() <= 2.0 ** -24 * (0.5 + 0.5 + 7.5)).all()
    c = make(18, [3], [0], 2, 1, 64, 32, "int8", "f16")
    q, k, v = split(c, c["qkv"])
    v[0, 0, 0], v[0, 0, 1], v[0, 0, 2] = float("nan"), float("inf"), -float("inf")
    c["scale"][1, 0, 3] = 0
    _, bufs, _, _ = call(c)
    row = row_of(c, bufs[1].cpu(), int(c["table"][0, 0]), 0)[0]
    assert row[:4].tolist() == [0, 127, -128, 0]


def test_no_rows_and_empty_sequences():
    c = make(19, [0, 0, 3, 0], [4, 0, 1, 9], 2, 1, 64, 16, "int4", "f16")
    check(c, call(c))
    k = torch.empty((0, 1, 64), dtype=torch.float16, device=DEV)
    cache = custom_ops.empty_int4_cache(3, 1, 16, 64)
    out = custom_ops.append_kv_cache(k, k, cache.key_cache, cache.value_cache, torch.zeros((1, 2), dtype=torch.int32, device=DEV),
                                     torch.zeros(1, dtype=torch.int32, device=DEV), query=k, block_size=16,
                                     query_start=torch.zeros(2, dtype=torch.int32, device=DEV), key_params=cache.key_params,
                                     value_params=cache.value_params)
    assert out.shape == (0, 1, 64)


def test_offsets_beyond_32_bits():
    """Pages behind 4 GiB of codes (and 2^31 elements of a 16-bit cache)."""
    D, Hkv, bs = 256, 8, 128
    blocks = (5 << 30) // (Hkv * bs * D // 2)
    c = make(20, [5], [126], 2, Hkv, D, bs, "int4", "f16")
    small_table = c["table"].clone()
    bufs = [torch.empty((blocks, Hkv, bs, D // 2), dtype=torch.uint8, device=DEV),
            torch.empty((blocks, Hkv, bs // 4, D // 2, 4), dtype=torch.uint8, device=DEV)]
    pars = [torch.empty((blocks, Hkv, bs, 2), dtype=torch.float16, device=DEV) for _ in range(2)]
    table = (blocks - 1 - small_table).to(DEV)
    want = call(c)
    q, k, v = split(c, to_dev(c["qkv"]))
    kw = dict(query_start=to_dev(c["start"]), block_size=bs, key_params=pars[0], value_params=pars[1])
    custom_ops.append_kv_cache(k, v, bufs[0], bufs[1], table, to_dev(c["seq"]), query=q, cos_sin=to_dev(c["cs"]), **kw)
    back = custom_ops.gather_kv_cache(bufs[0], bufs[1], table, to_dev(c["seq"]), Hkv, num_tokens=5, out_dtype=c["dt"], **kw)
    for a, b in zip(back, want[3]):
        assert torch.equal(a, b)
    del bufs, pars
    torch.cuda.empty_cache()
