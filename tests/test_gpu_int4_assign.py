"""Cluster ids of 4-bit pages over the ranges that change how the work is split: one new page, a page per sequence of many
sequences (clusters sliced over workgroups), hundreds of pages (16 to 32 of them per workgroup), duplicate clusters.

Every page's tokens follow the signs of one centroid: token values are +-(1 - 2 r / 15), r in 0 .. 3, so every mean has the
centroid's signs and magnitudes in [0.6, 1].  The score of that centroid is the sum of the magnitudes, any other sign vector
loses at least 2 x 0.6 = 1.2; rounding the mean moves a score by at most D x 2^-9 (bfloat16 half a step, magnitudes <= 1)
<= 0.5 for D = 256.  The expected id is therefore exact, and among equal centroids the smallest."""
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I32 = torch.int32


def _problem(seed, seq, first, Hkv, D, C, bs, dt, most=0, twins=False, short_ids=0, bad=()):
    g = torch.Generator().manual_seed(seed)
    B = len(seq)
    width = max(1, max(-(-s // bs) for s in seq))
    blocks = B * width + 3
    table = torch.randperm(blocks, generator=g)[:B * width].reshape(B, width).to(I32)
    for (b, i), v in bad:
        table[b, i] = v
    signs = torch.randint(0, 2, (Hkv, C, D), generator=g)
    if twins:
        signs[:, C // 2:2 * (C // 2)] = signs[:, :C // 2]
    goal = torch.randint(0, C, (blocks, Hkv), generator=g)
    sign = torch.stack([signs[n, goal[:, n]] for n in range(Hkv)], 1)                     # [blocks, Hkv, D]
    r = torch.randint(0, 4, (blocks, Hkv, bs, D), generator=g)
    codes = torch.where(sign[:, :, None] == 1, 15 - r, r).to(torch.uint8)
    par = torch.empty((blocks, Hkv, bs, 2), dtype=torch.float16)
    par[..., 0], par[..., 1] = 2 / 15, -1.0
    cent = (2 * signs - 1).to(dt)
    ids = torch.full((Hkv, blocks - short_ids), -7, dtype=I32)
    want = ids.clone()
    for b, s in enumerate(seq):
        pages = range(max(0, first[b]), -(-s // bs))
        for i in list(pages)[:most] if most else pages:
            p = int(table[b, i])
            if not 0 <= p < blocks - short_ids:
                continue
            for n in range(Hkv):
                c = int(goal[p, n])
                want[n, p] = c - C // 2 if twins and C // 2 <= c < 2 * (C // 2) else c
    # rows behind a sequence's end hold anything
    for b, s in enumerate(seq):
        if s % bs and 0 <= int(table[b, s // bs]) < blocks:
            par[int(table[b, s // bs]), :, s % bs:] = float("nan")
    up = lambda x: torch.tensor(x, dtype=I32, device=DEV)   # noqa: E731
    args = [kvo.pack_k(codes).to(DEV), table.to(DEV), up(seq), cent.to(DEV)]
    return args, ids, up(first), par.to(DEV), want, bs, most


def _run(pr, ids):
    args, _, first, par, _, bs, most = pr
    return custom_ops.assign_block_ids(*args, ids, first, block_size=bs, antiquant_scale=par, max_new_pages=most)


CASES = {
    "one_page": dict(seq=[7], first=[0], Hkv=1, D=128, C=100, bs=16, dt=torch.float16),
    "one_long_page": dict(seq=[501], first=[0], Hkv=2, D=128, C=2048, bs=512, dt=torch.float16),
    "three_pages": dict(seq=[33, 40], first=[0, 1], Hkv=2, D=64, C=17, bs=16, dt=torch.bfloat16),
    "few_clusters": dict(seq=[100, 31], first=[0, 0], Hkv=5, D=64, C=1, bs=32, dt=torch.float16),
    "none": dict(seq=[32, 0, -3], first=[1, 0, 0], Hkv=2, D=64, C=64, bs=32, dt=torch.float16),
    "decode": dict(seq=[128 * (i % 3) + 1 + i for i in range(70)], first=[(128 * (i % 3) + i) // 128 for i in range(70)], Hkv=8, D=64, C=2048,
                   bs=128, dt=torch.float16),
    "decode_wide": dict(seq=[50 + i for i in range(20)], first=[(49 + i) // 16 for i in range(20)], Hkv=1, D=256, C=1500, bs=16, dt=torch.bfloat16),
    "many_sequences": dict(seq=[16 * (i % 4) + 5 for i in range(200)], first=[0] * 200, Hkv=3, D=32, C=1024, bs=16, dt=torch.float16),
    "twenty_each": dict(seq=[16 * 210, 16 * 215 - 3, 16 * 215], first=[0, 0, 0], Hkv=8, D=32, C=512, bs=16, dt=torch.float16),
    "thirty_two_each": dict(seq=[16 * 400 - 1, 16 * 400, 16 * 333], first=[0, 3, 0], Hkv=8, D=32, C=300, bs=16, dt=torch.bfloat16),
    "limited": dict(seq=[160, 160], first=[0, 4], Hkv=2, D=64, C=128, bs=16, dt=torch.float16, most=3),
    "odd_heads": dict(seq=[48 * 5 + 11] * 9, first=[0] * 9, Hkv=7, D=256, C=333, bs=48, dt=torch.float16),
    "bad_pages": dict(seq=[160, 160], first=[0, 0], Hkv=2, D=64, C=600, bs=16, dt=torch.float16, bad=[((0, 0), -1), ((0, 9), 1 << 30), ((1, 5), 23)],
                      short_ids=4),
    "twins": dict(seq=[64 + i for i in range(40)], first=[0] * 40, Hkv=4, D=64, C=2047, bs=16, dt=torch.float16, twins=True),
}


@pytest.mark.parametrize("name", list(CASES))
def test_ids(name):
    pr = _problem(3, **CASES[name])
    out = _run(pr, pr[1].to(DEV))
    assert torch.equal(out.cpu(), pr[4])


def test_nan_page_takes_cluster_zero():
    pr = _problem(5, seq=[40, 33], first=[0, 0], Hkv=2, D=64, C=700, bs=16, dt=torch.float16)
    args, _, _, par, want, _, _ = pr
    page = int(args[1][0, 1])
    par[page, :, 3, 1] = float("nan")
    want[:, page] = 0
    assert torch.equal(_run(pr, pr[1].to(DEV)).cpu(), want)


def test_replays_and_streams():
    """A captured call replayed with other lengths, with eager calls on two streams between the replays."""
    a = _problem(7, seq=[100 + i for i in range(24)], first=[6] * 24, Hkv=4, D=64, C=1024, bs=16, dt=torch.float16)
    b = _problem(8, seq=[70 + i for i in range(30)], first=[0] * 30, Hkv=2, D=128, C=2048, bs=16, dt=torch.bfloat16)
    side = torch.cuda.Stream()
    ids = a[1].to(DEV)
    with torch.cuda.stream(side):
        _run(a, ids)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _run(a, ids)
    full = a[0][2].clone()
    for turn in range(4):
        a[0][2].copy_(full - 16 * (turn % 2))
        want = a[1].clone()
        for s in range(24):
            for i in range(6, -(-int(a[0][2][s]) // 16)):
                p = int(a[0][1][s, i])
                want[:, p] = a[4][:, p]
        ids.copy_(a[1])
        two = [b[1].to(DEV), b[1].to(DEV)]
        torch.cuda.synchronize()
        graph.replay()
        _run(b, two[0])
        with torch.cuda.stream(side):
            _run(b, two[1])
        torch.cuda.synchronize()
        assert torch.equal(ids.cpu(), want)
        assert torch.equal(two[0].cpu(), b[4]) and torch.equal(two[1].cpu(), b[4])
