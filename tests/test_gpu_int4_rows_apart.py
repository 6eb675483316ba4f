"""paged_attention_int4: a row's result is its own, whatever the rows beside it hold (other heads of the group, other tokens
of the sequence — a wave keeps up to 32 of them).  Helpers and tolerances of test_gpu_int4_attention.py."""
import pytest
import torch

from oracle import kv_cache as kvo
from test_gpu_int4_attention import call, check, make

pytestmark = pytest.mark.gpu

# rows side by side: one sequence of decode rows (a group of 8 heads), candidate rows (two tiles of a wave), a prompt's rows
SHAPES = [([1], [300], 8, 1, 128, True), ([1], [300], 24, 1, 64, True), ([5], [300], 8, 1, 128, False), ([70], [300], 4, 1, 128, False),
          ([9], [80], 8, 1, 256, False), ([3], [64], 4, 1, 32, False)]


def rows_of(c):
    """the call's query rows as [rows, D], row 0 the first token's first head"""
    return c["q"].view(-1, c["D"])


@pytest.mark.parametrize("n,s,Hq,Hkv,D,decode", SHAPES)
def test_rows_of_very_different_sizes(n, s, Hq, Hkv, D, decode):
    """Row r is multiplied by a power of ten of its own; every row stays within its own bound, and a row's value does not
    change with the sizes of the others."""
    c = make(31, n, s, Hq, Hkv, D, 32, "bf16", decode=decode)
    base = call(c).view(-1, D)
    factors = torch.tensor([1.0, 1e8, 1.0, 1e12, 1e-6, 1e-12, 1.0, 1e4])
    f = factors[torch.arange(rows_of(c).shape[0]) % 8]
    c["q"] = (rows_of(c).float() * f[:, None]).to(c["dt"]).view_as(c["q"])
    got = check(c).view(-1, D)
    same = (f == 1.0).to(got.device)
    assert torch.equal(got[same], base[same])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("n,s,Hq,Hkv,D,decode", SHAPES)
def test_a_query_row_that_is_not_finite_stays_alone(n, s, Hq, Hkv, D, decode, bad, dtype):
    """Its neighbours, one of them with elements of 6000 and one with elements of 1e-4, come out as without it."""
    c = make(32, n, s, Hq, Hkv, D, 32, dtype, decode=decode)
    q = rows_of(c)
    q[2] = 6000.0 * (q[2] > 0)
    q[3] *= 1e-4
    base = call(c).view(-1, D)
    assert bool(torch.isfinite(base).all())
    q[1, D // 2 + 1] = bad
    got = call(c).view(-1, D)
    assert bool(torch.isnan(got[1]).any())
    others = torch.arange(got.shape[0], device=got.device) != 1
    assert torch.equal(got[others], base[others])


def test_rows_near_the_end_of_bfloat16():
    """Elements up to 2^119 times a scale of 2^-3.5: the largest score takes all, and nothing overflows on the way."""
    c = make(33, [1, 3], [40, 90], 8, 1, 128, 32, "bf16")
    q = rows_of(c)
    q[::3] = torch.sign(q[::3]) * 2.0 ** 119
    out = call(c)
    want = kvo.attention(c["q"], kvo.values4(c["kc"], c["kp"]), kvo.values4(c["vc"], c["vp"]), c["table"], c["seq"], c["D"] ** -0.5, 1, 32, c["start"])[0]
    assert ((out.cpu().double() - want).abs() <= 2.0 ** -6 * want.abs() + 2.0 ** -7).all()
