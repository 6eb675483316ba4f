"""The KV-cache operators as a decode loop uses them: prompt rows appended to a 4-bit cache, cluster ids of its pages,
page selection, attention over the selected pages — eagerly and replayed from a HIP graph."""
import numpy as np
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _cluster_ids(keys, cent, table, seq, first, bs, dt):
    """float64: ids of the pages from `first` on, and the gap between the best and the second score relative to what the
    rounding of the page mean can move a score by."""
    out = {}
    for b, s in enumerate(seq):
        for page in range(first[b], -(-s // bs)):
            live = min(bs, s - page * bs)
            mean = keys[int(table[b, page]), :, :live].mean(1).to(dt).double()          # [Hkv, D]
            sc = torch.einsum("nd,ncd->nc", mean, cent.double())
            top2 = sc.topk(2, -1)
            # the device's fp32 mean may round to a neighbour in dt (one step of every element) before the scores are taken
            half = torch.finfo(dt).eps
            noise = (half * mean.abs()[:, None] * cent.double().abs()).sum(-1).amax(-1)
            out[(b, page)] = (top2.indices[:, 0], (top2.values[:, 0] - top2.values[:, 1]) > 2 * noise, sc)
    return out


@pytest.mark.parametrize("Hkv,D,C,bs,dt", [(2, 128, 256, 128, "f16"), (4, 64, 300, 16, "f16"), (1, 256, 128, 48, "bf16"), (2, 32, 64, 32, "bf16")])
def test_cluster_ids_of_4_bit_pages(Hkv, D, C, bs, dt):
    tdt = torch.float16 if dt == "f16" else torch.bfloat16
    g = torch.Generator().manual_seed(D + C)
    seq, first = [5 * bs, 1, 3 * bs + 7, 2 * bs - 1], [0, 0, 1, 2]
    blocks, width = 30, 6
    table = torch.randperm(blocks, generator=g)[:4 * width].reshape(4, width).to(torch.int32)
    table[2, 2] = -1                                       # names no page: skipped
    codes = torch.randint(0, 16, (blocks, Hkv, bs, D), generator=g, dtype=torch.uint8)
    par = torch.stack((0.1 + 0.1 * torch.rand((blocks, Hkv, bs), generator=g), torch.randn((blocks, Hkv, bs), generator=g)), -1).half()
    cent = torch.randn((Hkv, C, D), generator=g).to(tdt)
    ids0 = torch.randint(0, C, (Hkv, blocks), generator=g, dtype=torch.int32)
    ids = ids0.clone().to(DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    out = custom_ops.assign_block_ids(kvo.pack_k(codes).to(DEV), table.to(DEV), i32(seq), cent.to(DEV), ids, i32(first), block_size=bs,
                                      antiquant_scale=par.to(DEV))
    got = out.cpu()
    untouched = torch.ones(blocks, dtype=torch.bool)
    sure = 0
    for (b, page), (want, clear, sc) in _cluster_ids(kvo.values4(codes, par), cent, table, seq, first, bs, tdt).items():
        if (b, page) == (2, 2):
            continue
        phys = int(table[b, page])
        untouched[phys] = False
        for n in range(Hkv):
            sure += int(clear[n])
            if clear[n]:
                assert int(got[n, phys]) == int(want[n])
            else:
                assert float(sc[n, got[n, phys]]) >= float(sc[n].max()) * (1 - 0.05) - 0.05 * D
    assert sure >= 1 and torch.equal(got[:, untouched], ids0[:, untouched])


def _setup(seed, B, Hq, Hkv, D, bs, pages):
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * pages, generator=g).reshape(B, pages).to(torch.int32).to(DEV)
    cache = custom_ops.empty_int4_cache(B * pages, Hkv, bs, D, DEV)
    pos = torch.arange(pages * bs, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
    return g, table, cache, torch.cat((pos.cos(), pos.sin()), -1).float().to(DEV)


def test_decode_loop_over_a_4_bit_cache():
    B, Hq, Hkv, D, bs, pages, C, k = 3, 8, 2, 128, 16, 24, 64, 12
    g, table, cache, cs = _setup(1, B, Hq, Hkv, D, bs, pages)
    cent = torch.randn((Hkv, C, D), generator=g).half().to(DEV)
    ids = torch.zeros((Hkv, B * pages), dtype=torch.int32, device=DEV)
    n = [200, 33, 130]
    start = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device=DEV)
    seq = torch.tensor(n, dtype=torch.int32, device=DEV)
    par = dict(key_params=cache.key_params, value_params=cache.value_params)
    draw = lambda T: torch.randn((T, (Hq + 2 * Hkv) * D), generator=g).half().to(DEV)   # noqa: E731
    cut = lambda x: [t.unflatten(1, (-1, D)) for t in x.split([Hq * D, Hkv * D, Hkv * D], 1)]   # noqa: E731
    q, key, val = cut(draw(sum(n)))
    q = custom_ops.append_kv_cache(key, val, cache.key_cache, cache.value_cache, table, seq, query=q, query_start=start, cos_sin=cs,
                                   block_size=bs, **par)
    prompt = custom_ops.paged_attention_int4(q, *cache, table, seq, D ** -0.5, Hkv, query_start=start, max_query_len=max(n), block_size=bs)
    first = torch.zeros(B, dtype=torch.int32, device=DEV)
    custom_ops.assign_block_ids(cache.key_cache, table, seq, cent, ids, first, block_size=bs, antiquant_scale=cache.key_params)
    steps = []
    for _ in range(3):
        first = torch.div(seq, bs, rounding_mode="floor").int()          # the page that the next token lands in
        seq += 1
        q, key, val = cut(draw(B))
        q = custom_ops.append_kv_cache(key, val, cache.key_cache, cache.value_cache, table, seq, query=q, cos_sin=cs, block_size=bs, **par)
        custom_ops.assign_block_ids(cache.key_cache, table, seq, cent, ids, first, block_size=bs, max_new_pages=1,
                                    antiquant_scale=cache.key_params)
        lists, length, _ = custom_ops.cent_select(q, cent, ids, table, seq, k=k, max_page_num=pages, page_size=bs)
        out = custom_ops.paged_attention_int4(q, *cache, table, seq, D ** -0.5, Hkv, block_size=bs, block_position=lists)
        steps.append((q.cpu(), seq.cpu().clone(), lists.cpu(), out.cpu(), [t.cpu().clone() for t in cache]))
    torch.cuda.synchronize()
    for q, s, lists, out, bufs in steps:
        kk = kvo.values4(kvo.unpack_k(bufs[0]), bufs[2])
        vv = kvo.values4(kvo.unpack_v(bufs[1]), bufs[3])
        # (12 of 64 clusters: a row may find none of its sequence's pages among them and is then zero)
        assert bool((lists[:, :, 0] < pages).any())
        want, _, big = kvo.attention(q, kk, vv, table.cpu(), s, D ** -0.5, Hkv, bs, lists=lists)
        assert ((out.double() - want).abs() <= kvo.attention_bound(want, big, D, torch.float16)).all()
    assert bool(torch.isfinite(prompt).all())


def test_prompt_in_chunks_is_the_prompt():
    """A prompt appended and attended in chunks sees what it sees in one piece (chunk borders anywhere)."""
    Hq, Hkv, D, bs, N = 8, 2, 64, 16, 333
    g, table, cache, cs = _setup(2, 1, Hq, Hkv, D, bs, 21)
    x = torch.randn((3, N, Hq, D), generator=g).half().to(DEV)
    par = lambda c: dict(key_params=c.key_params, value_params=c.value_params)   # noqa: E731
    whole = None
    for cuts in ([0, N], [0, 1, 2, 50, 51, 53, 120, 280, N]):
        c = custom_ops.empty_int4_cache(21, Hkv, bs, D, DEV)
        outs = []
        for a, b in zip(cuts, cuts[1:]):
            seq = torch.tensor([b], dtype=torch.int32, device=DEV)
            start = torch.tensor([0, b - a], dtype=torch.int32, device=DEV)
            q = custom_ops.append_kv_cache(x[1, a:b, :Hkv], x[2, a:b, :Hkv], c.key_cache, c.value_cache, table, seq, query=x[0, a:b],
                                           query_start=start, cos_sin=cs, block_size=bs, **par(c))
            outs.append(custom_ops.paged_attention_int4(q, *c, table, seq, D ** -0.5, Hkv, query_start=start, block_size=bs,
                                                        out_dtype=torch.float32))
        got = torch.cat(outs)
        if whole is None:
            whole, bufs = got, c
        else:
            for a, b in zip(bufs, c):
                assert torch.equal(a, b)                   # the same cache, bit for bit
            # other cuts, other orders of summation: fp32 noise and the float16 rounding of p * s' (2^-11 of |V| <= 6)
            assert float((got - whole).abs().max()) <= 2 * 2.0 ** -11 * 6


def test_decode_step_in_a_graph():
    """A decode step (append + attention) captured once and replayed over growing sequences, with eager work between the
    replays; every replay is bit-equal to the eager step."""
    B, Hq, Hkv, D, bs, pages = 5, 8, 2, 128, 64, 40
    g, table, cache, cs = _setup(3, B, Hq, Hkv, D, bs, pages)
    for t in (cache.key_cache, cache.value_cache):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, dtype=torch.uint8))
    for t in (cache.key_params, cache.value_params):
        t.copy_(torch.stack((0.2 + 0.1 * torch.rand(t.shape[:-1], generator=g), -2 + 0.1 * torch.randn(t.shape[:-1], generator=g)), -1))
    seq = torch.tensor([2100, 3, 900, 64, 1500], dtype=torch.int32, device=DEV)
    qkv = torch.zeros((B, Hq + 2 * Hkv, D), dtype=torch.float16, device=DEV)

    def step(c):
        q = custom_ops.append_kv_cache(qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], c.key_cache, c.value_cache, table, seq, query=qkv[:, :Hq],
                                       cos_sin=cs, block_size=bs, key_params=c.key_params, value_params=c.value_params)
        return custom_ops.paged_attention_int4(q, *c, table, seq, D ** -0.5, Hkv, block_size=bs)

    twin = custom_ops.Int4Cache(*(t.clone() for t in cache))
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    step(twin)                                             # the warm-up below stores a row: the twin's cache gets it too
    with torch.cuda.stream(side):
        step(cache)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            out = step(cache)
    for i in range(5):
        seq += 1
        qkv.copy_(torch.randn(qkv.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step(twin))
        torch.cuda.synchronize()
    for name, a, b in zip(cache._fields, cache, twin):
        for s_ in range(5):
            pos = int(seq[s_]) - 1
            p, r = int(table[s_, pos // bs]), pos % bs
            assert torch.equal(a[p, :, r // 4, :, r % 4], b[p, :, r // 4, :, r % 4]) if a.dim() == 5 else torch.equal(a[p, :, r], b[p, :, r]), name


def test_launches_per_call():
    """One kernel per call on a stream whose counters are the library's."""
    B, Hq, Hkv, D, bs, pages = 2, 4, 2, 64, 16, 8
    g, table, cache, cs = _setup(4, B, Hq, Hkv, D, bs, pages)
    seq = torch.tensor([70, 100], dtype=torch.int32, device=DEV)
    x = torch.randn((B, Hq, D), generator=g).half().to(DEV)
    from custom_ops import _abi
    par = dict(key_params=cache.key_params, value_params=cache.value_params)

    def step():
        custom_ops.append_kv_cache(x[:, :Hkv], x[:, Hkv:], cache.key_cache, cache.value_cache, table, seq, query=x, cos_sin=cs, block_size=bs, **par)
        custom_ops.paged_attention_int4(x, *cache, table, seq, 0.125, Hkv, block_size=bs)
        custom_ops.gather_kv_cache(cache.key_cache, cache.value_cache, table, seq, Hkv, block_size=bs, **par)

    step()
    before = _abi.spfaKernelLaunches()
    step()
    assert _abi.spfaKernelLaunches() - before == 3
