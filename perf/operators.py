"""Workloads of the KV-cache operators: appending to a paged cache, reading rows back, attention over a 4-bit cache and
cluster ids of its pages.

`listed()` and `draw()` name workloads, `prepare()` makes a program's tensors, `run()` makes one pass — through the
framework's operators where `own` is true, in plain torch operations otherwise — and `work()` / `exact()` say what a pass
cannot do without and what it yields in 64 bits.

The 4-bit cache: a token of a kv head is D codes (0 .. 15) and a (scale, zero) pair in float16, x = scale * code + zero.
  key cache    uint8 [blocks, Hkv, bs, D / 2]        byte i: channel 2 i in the low bits, channel 2 i + 1 in the high bits
  value cache  uint8 [blocks, Hkv, bs / 4, D / 2, 4] the same bytes, those of four consecutive tokens side by side
  parameters   float16 [blocks, Hkv, bs, 2] each
Token i of sequence b (rows query_start[b] .. query_start[b + 1], or row b when every sequence has one) stands at position
seq_len[b] - n_b + i; position p lies in row p % bs of page block_table[b][p // bs].
"""
import math
import os
import sys

import torch

own = False

F16_MAX = 65504.0


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cann-ops-adv-vllm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import custom_ops
    return custom_ops


# ----------------------------------------------------------------------------------------------------------------
# workloads
# ----------------------------------------------------------------------------------------------------------------
def listed():
    append = dict(op="append", D=128, rot=128, interleaved=False, bs=128, layout="BSH")
    attn = dict(op="attention", D=128, bs=128, causal=True, n_min=1, n_max=1, lists=0)
    return [
        # one new token per sequence of a serving batch into a 16-bit cache: a small call, latency counts
        dict(append, name="append_decode_f16", dtype="f16", cache="f16", B=64, Hq=32, Hkv=8, n_min=1, n_max=1, old=500),
        # a few prompts at once into the 4-bit cache, ragged lengths; the stored rows are read back in 16 bits
        dict(append, name="append_prompt_int4", dtype="f16", cache="int4", B=5, Hq=32, Hkv=8, n_min=700, n_max=4096, old=0),
        # chunks behind existing contexts into an int8 cache of head-major pages, a quarter of the channels rotated in pairs
        dict(append, name="append_chunk_int8", dtype="bf16", cache="int8", B=7, Hq=16, Hkv=4, D=256, rot=64,
             interleaved=True, bs=64, layout="BNSD", n_min=1, n_max=513, old=900),
        # whole contexts out of the 4-bit cache (a shared prefix for a 16-bit attention, a cache that changes its type)
        dict(op="gather", name="gather_contexts_int4", dtype="f16", cache="int4", B=16, Hkv=8, D=128, bs=128, layout="BSH",
             n_min=3000, n_max=8192, old=0),
        # the last rows of a few sequences out of a 16-bit cache
        dict(op="gather", name="gather_tails_bf16", dtype="bf16", cache="bf16", B=9, Hkv=8, D=64, bs=16, layout="BSH",
             n_min=1, n_max=33, old=400),
        # one short sequence: the latency of a call
        dict(attn, name="attn_decode_one", dtype="f16", B=1, Hq=8, Hkv=8, D=64, s_min=700, s_max=700),
        # a serving batch, grouped heads, ragged contexts up to 32k tokens
        dict(attn, name="attn_decode_32k", dtype="f16", B=64, Hq=32, Hkv=8, s_min=8000, s_max=32768),
        # page lists per q head, as the page selection yields them
        dict(attn, name="attn_decode_lists", dtype="f16", B=64, Hq=32, Hkv=32, s_min=16000, s_max=32768, lists=48),
        # a few candidate tokens per sequence checked at once
        dict(attn, name="attn_verify", dtype="bf16", B=24, Hq=32, Hkv=4, n_min=2, n_max=5, s_min=1000, s_max=16384),
        # prompt chunks, causal, some behind existing context
        dict(attn, name="attn_prompt", dtype="f16", B=4, Hq=32, Hkv=8, n_min=1000, n_max=4096, s_min=4096, s_max=6000),
        # cluster ids of the pages that a decode step filled
        dict(op="assign", name="assign_decode", dtype="f16", B=64, Hkv=8, D=128, bs=128, C=2048, pages=4, new=1),
        # cluster ids of all pages of long prompts
        dict(op="assign", name="assign_prompt", dtype="f16", B=16, Hkv=8, D=128, bs=128, C=2048, pages=64, new=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "gather", "attention", "attention", "attention", "assign"])
    dtype = rng.choice(["f16", "bf16"])
    D = rng.choice([64, 128, 128, 256])
    bs = rng.choice([16, 48, 64, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    G = rng.choice([1, 2, 4, 5, 8])
    if op in ("append", "gather"):
        cache = rng.choice([dtype, "int8", "int4", "int4"])
        if cache == "int8":
            bs = rng.choice([32, 64, 128])
        layout = rng.choice(["BSH", "BNSD"])
        B = _log(rng, 1, 64)
        n_max = 1 if op == "append" and rng.random() < 0.3 else _log(rng, 1, max(2, 8192 // B))
        case = dict(op=op, dtype=dtype, cache=cache, B=B, Hkv=Hkv, D=D, bs=bs, layout=layout,
                    n_min=rng.randint(1, n_max), n_max=n_max, old=rng.randint(0, 700))
        if op == "append":
            case.update(Hq=Hkv * G, rot=rng.choice([D, D // 2, D // 4]), interleaved=rng.random() < 0.3)
        return case
    if op == "assign":
        pages = rng.randint(1, 24)
        return dict(op=op, dtype=dtype, B=_log(rng, 1, 48), Hkv=Hkv, D=D, bs=bs, C=rng.choice([200, 512, 1024, 2048]),
                    pages=pages, new=rng.randint(1, pages))
    kind = rng.choice(["decode", "decode", "lists", "verify", "prompt"])
    case = dict(op=op, dtype=dtype, Hkv=Hkv, Hq=Hkv * G, D=D, bs=bs, causal=True, n_min=1, n_max=1, lists=0)
    if kind == "prompt":
        n = _log(rng, 20, 1500)
        return dict(case, B=rng.randint(1, 4), n_min=rng.randint(1, n), n_max=n, s_min=n, s_max=n + rng.randint(0, 1500),
                    causal=rng.random() < 0.8)
    B, s = _log(rng, 1, 64), _log(rng, 1, 12000)
    if kind == "verify":
        s = max(s, 8)
        return dict(case, B=min(B, 24), n_min=1, n_max=rng.randint(2, 8), s_min=max(8, s // 3), s_max=s)
    if kind == "lists":
        return dict(case, B=min(B, 16), s_min=max(1, s // 2), s_max=s, lists=rng.randint(1, max(1, min(40, s // bs + 1))))
    return dict(case, B=B, s_min=max(1, s // rng.choice([1, 2, 10])), s_max=s)


# ----------------------------------------------------------------------------------------------------------------
# what a program holds
# ----------------------------------------------------------------------------------------------------------------
def _torch_type(name):
    return {"f16": torch.float16, "bf16": torch.bfloat16}[name]


def _lengths(case, rng):
    """(n, s) per sequence on the host: rows of this call, and tokens of the sequence with them."""
    B = case["B"]
    n = [rng.randint(case.get("n_min", 1), case.get("n_max", 1)) for _ in range(B)]
    if case["op"] == "attention":
        s = [max(x, rng.randint(case["s_min"], case["s_max"])) for x in n]
    else:
        s = [x + (rng.randint(case["old"] // 2, case["old"]) if case["old"] else 0) for x in n]
    return n, s


def _host_lengths(case):
    import random
    return _lengths(case, random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name"))))


def _tables(case, s, gen, dev):
    bs = case["bs"]
    pages = [-(-x // bs) for x in s]
    width, total = max(pages), sum(pages)
    perm = torch.randperm(total + 3, generator=gen, device=dev).to(torch.int32)   # three pages belong to nobody
    table = torch.full((len(s), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, k in enumerate(pages):
        table[b, :k] = perm[at:at + k]
        at += k
    return table, total + 3


def _int4_cache(blocks, Hkv, bs, D, gen, dev, center=None):
    """Pages as an append leaves them: codes of bell-shaped rows, their scales and lowest values."""
    k = torch.empty((blocks, Hkv, bs, D // 2), dtype=torch.uint8, device=dev)
    v = torch.empty((blocks, Hkv, bs // 4, D // 2, 4), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 27) // (Hkv * bs * D))
    for at in range(0, blocks, step):
        m = min(step, blocks - at)
        for dst, like in ((k, (m, Hkv, bs, D // 2)), (v, (m, Hkv, bs // 4, D // 2, 4))):
            codes = (torch.randn(like + (2,), generator=gen, device=dev) * 2.7 + 7.5).round_().clamp_(0, 15).to(torch.uint8)
            dst[at:at + m] = codes[..., 0] | (codes[..., 1] << 4)
    params = []
    for _ in range(2):
        scale = 0.36 * torch.exp(0.2 * torch.randn((blocks, Hkv, bs), generator=gen, device=dev))
        zero = -7.5 * scale + 0.1 * torch.randn((blocks, Hkv, bs), generator=gen, device=dev)
        params.append(torch.stack((scale, zero), -1).to(torch.float16))
    return k, v, params[0], params[1]


def _empty_cache(case, blocks, dt, gen, dev):
    Hkv, D, bs = case["Hkv"], case["D"], case["bs"]
    if case["cache"] == "int4":
        return dict(key_cache=torch.zeros((blocks, Hkv, bs, D // 2), dtype=torch.uint8, device=dev),
                    value_cache=torch.zeros((blocks, Hkv, bs // 4, D // 2, 4), dtype=torch.uint8, device=dev),
                    key_params=torch.zeros((blocks, Hkv, bs, 2), dtype=torch.float16, device=dev),
                    value_params=torch.zeros((blocks, Hkv, bs, 2), dtype=torch.float16, device=dev))
    shape = (blocks, bs, Hkv, D) if case["layout"] == "BSH" else (blocks, Hkv, bs, D)
    kind = torch.int8 if case["cache"] == "int8" else dt
    out = dict(key_cache=torch.zeros(shape, dtype=kind, device=dev), value_cache=torch.zeros(shape, dtype=kind, device=dev))
    if case["cache"] == "int8":
        scale = 0.03 + 0.01 * torch.rand((2, Hkv, D), generator=gen, device=dev)
        out["antiquant_scale"] = scale.to(dt)
        out["antiquant_offset"] = (4 * torch.randn((2, Hkv, D), generator=gen, device=dev)).round().to(dt)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _torch_type(case["dtype"])
    Hkv, D, bs = case["Hkv"], case["D"], case["bs"]
    randn = lambda *shape: torch.randn(shape, generator=gen, device=dev)   # noqa: E731
    st = dict(case=case)
    if case["op"] == "assign":
        B, C, pages = case["B"], case["C"], case["pages"]
        s = [pages * bs - (b * 7) % bs for b in range(B)]   # the last page is filled to different heights
        st["table"], blocks = _tables(case, s, gen, dev)
        k, _, kp, _ = _int4_cache(blocks, Hkv, bs, D, gen, dev)
        cent = randn(Hkv, C, D)
        # keys of a page gather around a cluster's centroid: codes follow it, the scale is that of the sum
        home = torch.randint(0, C, (blocks, Hkv), generator=gen, device=dev)
        mean = cent[torch.arange(Hkv, device=dev)[None], home]
        for at in range(0, blocks, 64):
            x = mean[at:at + 64, :, None] + 0.5 * randn(min(64, blocks - at), Hkv, bs, D)
            lo, hi = x.amin(-1), x.amax(-1)
            z, sc = lo.half().float(), ((hi - lo) / 15).half().float()
            codes = ((x - z[..., None]) / sc[..., None]).round().clamp(0, 15).to(torch.uint8)
            k[at:at + 64] = codes[..., 0::2] | (codes[..., 1::2] << 4)
            kp[at:at + 64] = torch.stack((sc, z), -1).half()
        st.update(key_cache=k, key_params=kp, cent=cent.to(dt),
                  seq_len=torch.tensor(s, dtype=torch.int32, device=dev),
                  first=torch.full((B,), pages - case["new"], dtype=torch.int32, device=dev),
                  ids=torch.zeros((Hkv, blocks), dtype=torch.int32, device=dev))
        return st
    n, s = _host_lengths(case)
    T = sum(n)
    st["table"], blocks = _tables(case, s, gen, dev)
    st["seq_len"] = torch.tensor(s, dtype=torch.int32, device=dev)
    start = [0]
    for x in n:
        start.append(start[-1] + x)
    st["start"] = torch.tensor(start, dtype=torch.int32, device=dev) if case.get("n_max", 1) > 1 else None
    # row -> its sequence and position: what the plain form indexes with
    seq = torch.repeat_interleave(torch.arange(case["B"], device=dev), torch.tensor(n, device=dev))
    pos = torch.cat([torch.arange(x - m, x, device=dev) for m, x in zip(n, s)])
    st.update(T=T, seq=seq, pos=pos, n_max=max(n), s_max=max(s))
    if case["op"] == "append":
        # one projection's output, taken apart by views as a model does; the table of angles is float32
        Hq, rot = case["Hq"], case["rot"]
        qkv = randn(T, (Hq + 2 * Hkv) * D).to(dt)
        st["q"], st["k"], st["v"] = (t.view(T, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        angle = torch.arange(max(s), device=dev, dtype=torch.float64)[:, None] * freq
        st["cos_sin"] = torch.cat((angle.cos(), angle.sin()), -1).float()
        st.update(_empty_cache(case, blocks, dt, gen, dev))
    elif case["op"] == "gather":
        if case["cache"] == "int4":
            k, v, kp, vp = _int4_cache(blocks, Hkv, bs, D, gen, dev)
            st.update(key_cache=k, value_cache=v, key_params=kp, value_params=vp)
        else:
            st.update(_empty_cache(case, blocks, dt, gen, dev))
            for name in ("key_cache", "value_cache"):
                c = st[name]
                if c.dtype == torch.int8:
                    c.copy_(torch.randint(-128, 128, c.shape, generator=gen, device=dev, dtype=torch.int8))
                else:
                    c.copy_(randn(*c.shape))
    else:
        k, v, kp, vp = _int4_cache(blocks, Hkv, bs, D, gen, dev)
        st.update(key_cache=k, value_cache=v, key_params=kp, value_params=vp, q=randn(T, case["Hq"], D).to(dt))
        if case["lists"]:
            # per q head an ascending list of distinct pages of the sequence, shorter ones among them
            width = st["table"].shape[1]
            have = (st["seq_len"] + bs - 1) // bs
            score = torch.rand((case["B"], case["Hq"], width), generator=gen, device=dev)
            score.masked_fill_(torch.arange(width, device=dev) >= have[:, None, None], 2.0)
            order = score.argsort(-1)[..., :case["lists"]].to(torch.int32)
            take = torch.randint(max(1, case["lists"] // 2), case["lists"] + 1, (case["B"], case["Hq"], 1), generator=gen, device=dev)
            take = torch.minimum(take, have[:, None, None])
            end = torch.iinfo(torch.int32).max
            order.masked_fill_(torch.arange(order.shape[-1], device=dev) >= take, end)
            st["lists"] = order.sort(-1).values.contiguous()
    return st


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"append": _append, "gather": _gather, "attention": _attention, "assign": _assign}[case["op"]](case, state)


def _antiquant(st):
    return {k: st[k] for k in ("antiquant_scale", "antiquant_offset", "key_params", "value_params") if k in st}


def _append(case, st):
    if own:
        ops = _ops()
        q = ops.append_kv_cache(st["k"], st["v"], st["key_cache"], st["value_cache"], st["table"], st["seq_len"],
                                query=st["q"], query_start=st["start"], cos_sin=st["cos_sin"],
                                interleaved=case["interleaved"], block_size=case["bs"], **_antiquant(st))
    else:
        q = _rotate(st["q"], st["cos_sin"][st["pos"]], case["interleaved"]).to(st["q"].dtype)
        _store(case, st, _rotate(st["k"], st["cos_sin"][st["pos"]], case["interleaved"]), st["v"].float())
    if case["cache"] in ("f16", "bf16"):
        return q, st["key_cache"], st["value_cache"]
    return (q,) + tuple(_gather(case, st))   # what is held in few bits, as the values it stands for


def _gather(case, st):
    if own:
        return _ops().gather_kv_cache(st["key_cache"], st["value_cache"], st["table"], st["seq_len"], case["Hkv"],
                                      query_start=st["start"], num_tokens=st["T"], block_size=case["bs"],
                                      out_dtype=_torch_type(case["dtype"]), **_antiquant(st))
    page, row = _places(case, st)
    k, v = _rows(case, st, page, row)
    return k.to(_torch_type(case["dtype"])), v.to(_torch_type(case["dtype"]))


def _assign(case, st):
    if own:
        return _ops().assign_block_ids(st["key_cache"], st["table"], st["seq_len"], st["cent"], st["ids"], st["first"],
                                       block_size=case["bs"], antiquant_scale=st["key_params"])
    B, bs, new = case["B"], case["bs"], case["new"]
    page = st["first"].long()[:, None] + torch.arange(new, device=st["table"].device)
    phys = st["table"].gather(1, page).long().reshape(-1)
    live = (st["seq_len"].long()[:, None] - page * bs).clamp(max=bs).reshape(-1)
    x = _unpack(st["key_cache"][phys]).float() * st["key_params"][phys][..., :1].float() + st["key_params"][phys][..., 1:].float()
    x = x * (torch.arange(bs, device=x.device) < live[:, None])[:, None, :, None]
    mean = (x.sum(2) / live[:, None, None]).to(st["cent"].dtype).float()
    score = torch.matmul(mean.transpose(0, 1), st["cent"].float().transpose(1, 2))     # [Hkv, pages, C]
    st["ids"][:, phys] = score.argmax(-1).int()
    return st["ids"]


def _attention(case, st):
    if own:
        return _ops().paged_attention_int4(st["q"], st["key_cache"], st["value_cache"], st["key_params"], st["value_params"],
                                           st["table"], st["seq_len"], case["D"] ** -0.5, case["Hkv"], query_start=st["start"],
                                           max_query_len=st["n_max"], causal=case["causal"], block_position=st.get("lists"),
                                           block_size=case["bs"])
    B, Hq, Hkv, D, bs = case["B"], case["Hq"], case["Hkv"], case["D"], case["bs"]
    G, dev = Hq // Hkv, st["q"].device
    if case["lists"]:
        # every q head its own pages: [B, Hq, pages * bs, D]
        end = torch.iinfo(torch.int32).max
        logical = st["lists"].long()
        there = logical < end
        phys = st["table"].gather(1, torch.where(there, logical, 0).reshape(B, -1)).long().reshape(logical.shape)
        head = (torch.arange(Hq, device=dev) // G)[None, :, None]
        S = logical.shape[-1] * bs
        k = _unpack(st["key_cache"][phys, head]).float() * st["key_params"][phys, head][..., :1].float() + st["key_params"][phys, head][..., 1:].float()
        v = _unpack_v(st["value_cache"][phys, head]).float() * st["value_params"][phys, head][..., :1].float() + st["value_params"][phys, head][..., 1:].float()
        t = logical[..., None] * bs + torch.arange(bs, device=dev)
        seen = (there[..., None] & (t < st["seq_len"].long()[:, None, None, None])).reshape(B, Hq, 1, S)
        p = _softmax(torch.matmul(st["q"].float()[:, :, None], k.reshape(B, Hq, S, D).transpose(2, 3)) * D ** -0.5, seen)
        return torch.matmul(p, v.reshape(B, Hq, S, D))[:, :, 0].to(st["q"].dtype)
    # all pages of a sequence, padded to the longest: [B, Hkv, S, D]; rows padded to the most of one sequence
    N, pages = st["n_max"], st["table"].shape[1]
    S = pages * bs
    phys = st["table"].clamp(min=0).long()
    k = _unpack(st["key_cache"][phys]).float() * st["key_params"][phys][..., :1].float() + st["key_params"][phys][..., 1:].float()
    k = k.transpose(1, 2).reshape(B, Hkv, S, D)
    q = torch.zeros((B, N, Hq, D), device=dev)
    first = st["pos"][torch.searchsorted(st["seq"], torch.arange(B, device=dev))]      # position of a sequence's first row
    q[st["seq"], st["pos"] - first[st["seq"]]] = st["q"].float()
    q = q.reshape(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, D)
    last = first[:, None] + torch.arange(N, device=dev) if case["causal"] else st["seq_len"].long()[:, None].expand(B, N)
    t = torch.arange(S, device=dev)
    seen = (t <= last[..., None]) & (t < st["seq_len"].long()[:, None, None])          # [B, N, S]
    score = torch.matmul(q, k.transpose(2, 3)).reshape(B, Hkv, G, N, S) * D ** -0.5
    del k
    p = _softmax(score, seen[:, None, None])
    v = _unpack_v(st["value_cache"][phys]).float() * st["value_params"][phys][..., :1].float() + st["value_params"][phys][..., 1:].float()
    o = torch.matmul(p.reshape(B, Hkv, G * N, S), v.transpose(1, 2).reshape(B, Hkv, S, D))
    o = o.reshape(B, Hkv, G, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)
    return o[st["seq"], st["pos"] - first[st["seq"]]].to(st["q"].dtype)


# plain forms ------------------------------------------------------------------------------------------------------
def _rotate(x, cos_sin, interleaved):
    rot, x = cos_sin.shape[-1], x.float()
    c, s = (t[:, None] for t in cos_sin.chunk(2, -1))
    a, b = (x[..., :rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    ra, rb = a * c - b * s, b * c + a * s
    turned = torch.stack((ra, rb), -1).flatten(-2) if interleaved else torch.cat((ra, rb), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _places(case, st):
    page = st["table"][st["seq"], torch.div(st["pos"], case["bs"], rounding_mode="floor")].long()
    return page, st["pos"] % case["bs"]


def _quantise(x):
    lo, hi = x.amin(-1), x.amax(-1)
    s = ((hi - lo) / 15).clamp(max=F16_MAX).half()
    z = lo.clamp(-F16_MAX, F16_MAX).half()
    codes = ((x - z.float()[..., None]) / s.float()[..., None]).round().clamp(0, 15)
    codes = torch.where(s[..., None] > 0, codes, torch.zeros_like(codes)).to(torch.uint8)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.stack((s, z), -1)


def _store(case, st, k, v):
    page, row = _places(case, st)
    if case["cache"] == "int4":
        (kb, kp), (vb, vp) = _quantise(k), _quantise(v)
        st["key_cache"][page, :, row] = kb
        st["key_params"][page, :, row] = kp
        st["value_cache"][page, :, row // 4, :, row % 4] = vb
        st["value_params"][page, :, row] = vp
        return
    for name, x, i in (("key_cache", k, 0), ("value_cache", v, 1)):
        if case["cache"] == "int8":
            x = (x / st["antiquant_scale"][i].float() - st["antiquant_offset"][i].float()).round().clamp(-128, 127)
        if case["layout"] == "BSH":
            st[name][page, row] = x.to(st[name].dtype)
        else:
            st[name][page, :, row] = x.to(st[name].dtype)


def _unpack(b):
    """bytes [..., D / 2] -> codes [..., D]"""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def _unpack_v(b):
    """bytes [..., bs / 4, D / 2, 4] -> codes [..., bs, D]"""
    return _unpack(b.transpose(-1, -2)).flatten(-3, -2)


def _rows(case, st, page, row):
    if case["cache"] == "int4":
        kp, vp = st["key_params"][page, :, row].float(), st["value_params"][page, :, row].float()
        k = _unpack(st["key_cache"][page, :, row]).float() * kp[..., :1] + kp[..., 1:]
        v = _unpack(st["value_cache"][page, :, row // 4, :, row % 4]).float() * vp[..., :1] + vp[..., 1:]
        return k, v
    out = []
    for name, i in (("key_cache", 0), ("value_cache", 1)):
        x = (st[name][page, row] if case["layout"] == "BSH" else st[name][page, :, row]).float()
        if case["cache"] == "int8":
            x = (x + st["antiquant_offset"][i].float()) * st["antiquant_scale"][i].float()
        out.append(x)
    return out


def _softmax(score, seen):
    score = score.masked_fill(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


# ----------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ----------------------------------------------------------------------------------------------------------------
def _stored_row(case):
    D = case["D"]
    return {"f16": 2 * D, "bf16": 2 * D, "int8": D, "int4": D // 2 + 4}[case["cache"]]


def work(case):
    D, Hkv, B = case["D"], case["Hkv"], case["B"]
    if case["op"] == "assign":
        tokens = sum(case["new"] * case["bs"] - (b * 7) % case["bs"] for b in range(B))
        pages = B * case["new"]
        return {"bytes": tokens * Hkv * (D // 2 + 4) + Hkv * case["C"] * D * 2 + pages * Hkv * 4 + pages * 4,
                "flops": 2 * pages * Hkv * case["C"] * D + 2 * tokens * Hkv * D}
    n, s = _host_lengths(case)
    T = sum(n)
    if case["op"] == "append":
        low = case["cache"] in ("int8", "int4")
        moved = T * ((2 * case["Hq"] + 2 * Hkv) * D * 2 + 2 * Hkv * _stored_row(case)) + T * case["rot"] * 4
        moved += T * 2 * Hkv * (_stored_row(case) + 2 * D) if low else 0     # the stored rows are read back
        return {"bytes": moved, "flops": 3 * T * (case["Hq"] + Hkv) * case["rot"]}
    if case["op"] == "gather":
        return {"bytes": T * 2 * Hkv * (_stored_row(case) + 2 * D), "flops": T * 2 * Hkv * D * 2}
    Hq, row = case["Hq"], 2 * (D // 2 + 4)
    if case["lists"]:
        mean = 0.5 * (max(1, case["lists"] // 2) + case["lists"]) * case["bs"]
        tokens = sum(min(mean, x) for x in s)
        return {"bytes": tokens * Hkv * row + 4 * T * Hq * D, "flops": 4 * tokens * Hq * D}
    pairs = sum(sum(x - m + 1 + i for i in range(m)) if case["causal"] else m * x for m, x in zip(n, s))
    return {"bytes": sum(s) * Hkv * row + 4 * T * Hq * D, "flops": 4 * pairs * Hq * D}


# ----------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, row by row of the sequences
# ----------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "assign":
        return None
    with torch.no_grad():
        return {"append": _exact_append, "gather": _exact_gather, "attention": _exact_attention}[case["op"]](case, st)


def _exact_turn(x, pos, case):
    rot, half = case["rot"], case["rot"] // 2
    angle = torch.outer(pos.double(), 10000.0 ** (-torch.arange(half, device=x.device, dtype=torch.float64) * 2 / rot))
    spin = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.double().clone()
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
    z = torch.complex(x[..., a], x[..., b]) * spin
    x[..., a], x[..., b] = z.real, z.imag
    return x


def _exact_codes(x):
    """the values that 4-bit rows of x stand for"""
    lo, hi = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    s, z = ((hi - lo) / 15).to(torch.float16).double(), lo.to(torch.float16).double()
    return torch.where(s > 0, torch.round((x - z) / s).clip(0, 15) * s + z, z)


def _exact_append(case, st):
    q, k, v = _exact_turn(st["q"], st["pos"], case), _exact_turn(st["k"], st["pos"], case), st["v"].double()
    if case["cache"] == "int4":
        return q, _exact_codes(k), _exact_codes(v)
    if case["cache"] == "int8":
        sc, of = st["antiquant_scale"].double(), st["antiquant_offset"].double()
        return (q,) + tuple((torch.round(x / sc[i] - of[i]).clip(-128, 127) + of[i]) * sc[i] for i, x in enumerate((k, v)))
    kc, vc = st["key_cache"].double(), st["value_cache"].double()
    n, s = _host_lengths(case)
    at, bs = 0, case["bs"]
    for b, (m, x) in enumerate(zip(n, s)):
        for p0 in range(((x - m) // bs) * bs, x, bs):            # page by page
            lo, hi = max(p0, x - m), min(p0 + bs, x)
            page = int(st["table"][b, p0 // bs])
            r = slice(at + lo - (x - m), at + hi - (x - m))
            kc[page] = _put(kc[page], lo - p0, hi - p0, k[r], case)
            vc[page] = _put(vc[page], lo - p0, hi - p0, v[r], case)
        at += m
    return q, kc, vc


def _put(page, lo, hi, rows, case):
    page = page.clone()
    if case["layout"] == "BSH":
        page[lo:hi] = rows
    else:
        page[:, lo:hi] = rows.transpose(0, 1)
    return page


def _values_of(codes, params, quads):
    """4-bit pages -> float64 [pages, Hkv, bs, D]"""
    if quads:
        codes = codes.movedim(-1, -2).reshape(codes.shape[0], codes.shape[1], -1, codes.shape[-2])
    out = torch.empty(codes.shape[:-1] + (codes.shape[-1] * 2,), dtype=torch.float64, device=codes.device)
    out[..., 0::2] = (codes % 16).double()
    out[..., 1::2] = torch.div(codes, 16, rounding_mode="floor").double()
    return out * params[..., 0, None].double() + params[..., 1, None].double()


def _exact_pages(case, st, b, upto):
    """K and V of the first `upto` tokens of sequence b in 64 bits: [Hkv, upto, D]"""
    pages = st["table"][b, :-(-upto // case["bs"])].long()
    if case["op"] == "attention" or case["cache"] == "int4":
        k = _values_of(st["key_cache"][pages], st["key_params"][pages], False)
        v = _values_of(st["value_cache"][pages], st["value_params"][pages], True)
    else:
        k, v = st["key_cache"][pages].double(), st["value_cache"][pages].double()
        if case["layout"] == "BSH":
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        if case["cache"] == "int8":
            sc, of = st["antiquant_scale"].double(), st["antiquant_offset"].double()
            k, v = (k + of[0][:, None]) * sc[0][:, None], (v + of[1][:, None]) * sc[1][:, None]
    return tuple(x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, :upto] for x in (k, v))


def _exact_gather(case, st):
    n, s = _host_lengths(case)
    ks, vs = [], []
    for b, (m, x) in enumerate(zip(n, s)):
        k, v = _exact_pages(case, st, b, x)
        ks.append(k[:, x - m:].transpose(0, 1))
        vs.append(v[:, x - m:].transpose(0, 1))
    return torch.cat(ks), torch.cat(vs)


def _exact_attention(case, st):
    n, s = _host_lengths(case)
    if 4 * max(work(case)["flops"], 1) > 4e13:
        return None
    Hq, Hkv, D, bs = case["Hq"], case["Hkv"], case["D"], case["bs"]
    G, at, out = Hq // Hkv, 0, []
    for b, (m, x) in enumerate(zip(n, s)):
        k, v = _exact_pages(case, st, b, x)
        t = torch.arange(x, device=k.device)
        rows = []
        for h in range(Hq):
            q = st["q"][at:at + m, h].double()
            e = (q @ k[h // G].T) / math.sqrt(D)
            if case["causal"]:
                e = e.where(t[None] <= (x - m + torch.arange(m, device=t.device))[:, None], -math.inf)
            if case["lists"]:
                listed_pages = st["lists"][b, h]
                mine = listed_pages[listed_pages < torch.iinfo(torch.int32).max].long()
                keep = torch.zeros(-(-x // bs), dtype=torch.bool, device=t.device)
                keep[mine] = True
                e = e.where(keep[t // bs][None], -math.inf)
            rows.append(torch.softmax(e, -1) @ v[h // G])
        out.append(torch.stack(rows, 1))
        at += m
    return torch.cat(out)
