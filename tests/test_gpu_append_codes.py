"""append_kv_cache: codes and parameters bit for bit, on values that lie on the borders between two of them.

Without rotation every step is determined: the inputs are exact in fp32, a difference, a quotient and an offset are one
fp32 rounding each (numpy's are the correctly rounded ones), and the code is the nearest integer, ties to even.  4 bits:
scale = f16((hi - lo) / 15) and zero = f16(lo), ties to even."""
import numpy as np
import pytest
import torch

import custom_ops
from oracle import kv_cache as kvo

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
BS, HKV = 32, 2


def store(k, v, cache, **kw):
    """rows [T, HKV, D] appended as one sequence into pages 0, 1, ..."""
    T = k.shape[0]
    pages = -(-T // BS)
    table = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)   # noqa: E731
    custom_ops.append_kv_cache(k.to(DEV), v.to(DEV), cache[0], cache[1], table, i32(T), query_start=i32(0, T), block_size=BS, **kw)
    torch.cuda.synchronize()


def rows4(x):
    """codes [T, H, D], scale and zero [T, H] of rows x (fp32 holding 16-bit values)"""
    x = x.float().numpy()
    lo, hi = x.min(-1), x.max(-1)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        s = np.minimum((hi - lo) / np.float32(15), np.float32(65504)).astype(np.float16)
        z = np.clip(lo, -65504, 65504).astype(np.float16)
        q = (x - z.astype(np.float32)[..., None]) / s.astype(np.float32)[..., None]
        code = np.where(s[..., None] > 0, np.clip(np.rint(q), 0, 15), 0)
    return code.astype(np.uint8), s, z


def check4(x, dtype):
    x = x.to(DT[dtype])
    T, _, D = x.shape
    cache = custom_ops.empty_int4_cache(-(-T // BS), HKV, BS, D, device=DEV)
    v = x.flip(0).contiguous()
    store(x, v, cache[:2], key_params=cache[2], value_params=cache[3])
    kc, vc, kp, vp = (t.cpu() for t in cache)
    for rows, codes, pars, name in ((x, kvo.unpack_k(kc), kp, "K"), (v, kvo.unpack_v(vc), vp, "V")):
        flat = lambda t: t.transpose(1, 2).reshape(-1, HKV, t.shape[-1])[:T].numpy()      # noqa: E731
        code, s, z = rows4(rows)
        par = flat(pars)
        assert (par[..., 0].view(np.uint16) == s.view(np.uint16)).all(), f"{name}: scales of {np.argwhere(par[..., 0] != s)[:3].tolist()}"
        assert (par[..., 1] == z).all(), f"{name}: zeros"
        assert (flat(codes) == code).all(), f"{name}: codes at {np.argwhere(flat(codes) != code)[:3].tolist()}"


@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("T", [70, 700, 2100])
def test_int4_scales_half_way_between_two(T, D):
    """hi - lo = 15 (k / 64 + 2^-11) 2^e, k = 64 .. 127: half-way between two float16 scales, the even one is k / 64."""
    g = torch.Generator().manual_seed(T + D)
    k = torch.randint(64, 128, (T, HKV, 1), generator=g).double()
    e = torch.randint(-8, 9, (T, HKV, 1), generator=g).double()
    lo, hi = -15 * 2.0 ** -11 * 2.0 ** e, 15 * k / 64 * 2.0 ** e
    x = lo + (hi - lo) * torch.rand((T, HKV, D), generator=g).double()
    x = x.half().double().clamp(min=lo.expand_as(x), max=hi.expand_as(x))
    x[..., :1], x[..., D - 1:] = lo, hi
    check4(x.half(), "f16")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("T,D", [(70, 64), (700, 128), (2100, 32), (600, 256)])
def test_int4_codes_half_way_between_two(T, D, dtype):
    """Rows on a grid of half steps: every second value lies exactly between two codes."""
    g = torch.Generator().manual_seed(T + D)
    m = torch.tensor([1.0, 3.0, 5.0, 7.0])[torch.randint(0, 4, (T, HKV, 1), generator=g)]
    step = m * 2.0 ** torch.randint(-6, 4, (T, HKV, 1), generator=g)
    j = torch.randint(0, 31, (T, HKV, D), generator=g).float()
    j[..., 3], j[..., D - 2] = 0.0, 30.0
    base = torch.randint(-3, 2, (T, HKV, 1), generator=g).float()
    x = step * (j / 2 + base)
    assert torch.equal(x.to(DT[dtype]).float(), x)
    check4(x, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("spread", [0.0, 6.0])
def test_int4_codes_of_any_rows(spread, dtype):
    g = torch.Generator().manual_seed(9)
    x = torch.randn((2100, HKV, 64), generator=g) * torch.exp(spread * torch.randn((2100, HKV, 1), generator=g))
    x[5], x[6] = 0.25, 0.0                               # rows of one value
    x[7, :, :4] = 60000.0
    x[9, :, :2] = torch.tensor([-3e38, 3e38])            # (bfloat16: the difference is infinite)
    if dtype == "f16":
        x.clamp_(-60000, 60000)
        x[8] = 2.0 ** -24 * torch.arange(64)             # subnormal
    check4(x, dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("offset", [False, True])
@pytest.mark.parametrize("T,D", [(70, 64), (700, 128), (2100, 32), (600, 512)])
def test_int8_codes_half_way_between_two(T, D, offset, dtype):
    """x = s (j / 2 + offset): every second value lies exactly between two codes.  bfloat16: scales from 2^-80 to 2^80, both
    sides of where the quotient is formed without a division."""
    g = torch.Generator().manual_seed(T + D)
    dt = DT[dtype]
    m = torch.tensor([1.0, 3.0, 5.0, 7.0])[torch.randint(0, 4, (2, HKV, D), generator=g)]
    span = 4 if dtype == "f16" else 80
    e = torch.randint(-span, span + 1, (2, HKV, D // 8), generator=g).repeat_interleave(8, -1)
    e[..., :8] = torch.randint(-4, 5, (2, HKV, 8), generator=g)
    s = (m.double() * 2.0 ** e.double()).to(dt)
    o = torch.randint(-9, 10, (2, HKV, D), generator=g).to(dt) if offset else None
    top = 150 if dtype == "f16" else 31                  # (products of 8 bits)
    j = torch.randint(-top, top + 1, (2, T, HKV, D), generator=g).double()
    x = s.double()[:, None] * (j / 2)
    x[:, ::3] = s.double()[:, None] * (2.0 ** -2 * torch.randn((2, len(range(0, T, 3)), HKV, D), generator=g).double() * top)
    x = x.to(dt)
    shape = (-(-T // BS), BS, HKV, D)
    cache = [torch.zeros(shape, dtype=torch.int8, device=DEV) for _ in range(2)]
    store(x[0].contiguous(), x[1].contiguous(), cache, antiquant_scale=s.to(DEV), antiquant_offset=None if o is None else o.to(DEV))
    for which in range(2):
        q = x[which].float().numpy() / s[which].float().numpy()
        y = q - (o[which].float().numpy() if offset else np.float32(0))
        want = np.rint(np.clip(y, -128, 127)).astype(np.int8)
        got = cache[which].cpu().numpy().reshape(-1, HKV, D)[:T]
        assert (got == want).all(), f"at {np.argwhere(got != want)[:3].tolist()}"


def test_int8_codes_saturate_and_scales_of_zero():
    D = 64
    s = torch.full((2, HKV, D), 0.5, dtype=torch.float16)
    s[:, :, 5] = 0.0
    x = torch.zeros((40, HKV, D))
    x[:, :, 0], x[:, :, 1], x[:, :, 2], x[:, :, 3] = 60000.0, -60000.0, float("inf"), float("nan")
    x[:, :, 4], x[:, :, 5], x[:, :, 6], x[:, :, 7] = float("-inf"), 3.0, 63.75, -64.25
    cache = [torch.ones((2, BS, HKV, D), dtype=torch.int8, device=DEV) for _ in range(2)]
    store(x.half(), x.half(), cache, antiquant_scale=s.to(DEV))
    want = torch.zeros((D,), dtype=torch.int8)
    want[:8] = torch.tensor([127, -128, 127, 0, -128, 0, 127, -128], dtype=torch.int8)
    for c in cache:
        assert torch.equal(c.cpu().reshape(-1, HKV, D)[:40], want.expand(40, HKV, D))
