"""paged_attention_int4 over parameters of any sign and size.  Helpers and tolerances of test_gpu_int4_attention.py."""
import pytest
import torch

from oracle import kv_cache as kvo
from test_gpu_int4_attention import call, make

pytestmark = pytest.mark.gpu


def turned(pars, at):
    """The same values with the codes counted from the top: scale -s, zero z + 15 s, codes 15 - c."""
    s, z = pars[..., 0], pars[..., 1]
    return torch.stack((torch.where(at, -s, s), torch.where(at, (z.float() + 15 * s.float()).half(), z)), -1)


def within(c, rows=slice(None)):
    """float32 outputs of `rows` against the oracle, without the 2^-24 that the bound allows for outputs near zero: the values
    here may be much smaller than that."""
    got = call(c, out_dtype=torch.float32)
    want, _, big = kvo.attention(c["q"], kvo.values4(c["kc"], c["kp"]), kvo.values4(c["vc"], c["vp"]), c["table"], c["seq"], c["D"] ** -0.5,
                                 c["Hkv"], c["bs"], c["start"])
    bound = kvo.attention_bound(want, big, c["D"], torch.float32) - 2.0 ** -24
    err = (got.cpu().double() - want).abs()
    assert (err <= bound)[rows].all(), f"off by {(err / bound)[rows].max().item():.2f} of the bound"
    return got


@pytest.mark.parametrize("factor", [1.0, 2000.0, 2.0 ** -18])
@pytest.mark.parametrize("n,s,Hq,Hkv,D,decode", [([1] * 3, [300, 33, 1000], 4, 2, 128, True), ([5, 3], [300, 64], 8, 1, 64, False),
                                                 ([70], [200], 4, 2, 256, False)])
@pytest.mark.parametrize("every", [1, 3])
def test_negative_scales(n, s, Hq, Hkv, D, decode, factor, every):
    """Scales below zero: all of them, or one in three beside positive ones that are 2^8 times smaller."""
    c = make(41, n, s, Hq, Hkv, D, 32, "f16", decode=decode)
    at = (torch.arange(32) % every == 0).expand(c["kp"].shape[:-1])
    c["vp"] = (c["vp"].float() * factor * torch.where(at, 1.0, 2.0 ** -8)[..., None]).half()
    for codes, pars in (("kc", "kp"), ("vc", "vp")):
        c[pars] = turned(c[pars], at)
        c[codes] = torch.where(at[..., None], 15 - c[codes], c[codes])
    assert bool(torch.isfinite(c["vp"]).all())
    within(c)


@pytest.mark.parametrize("top", [60000.0, float("inf")])
@pytest.mark.parametrize("n,s,Hq,Hkv,D", [([40], [40], 4, 2, 64), ([40], [60], 4, 2, 128), ([5], [29], 8, 1, 128), ([20], [52], 2, 2, 256)])
def test_a_large_value_scale_reaches_only_those_who_see_it(n, s, Hq, Hkv, D, top):
    """Rows before a token with a huge scale: within the bound of the small values that they see, and the same for whatever
    the token's parameters hold.  (Scales of 2^-14: huge ones are 2^30 times larger, more than float16 spans.)"""
    c = make(42, n, s, Hq, Hkv, D, 16, "f16")
    c["vp"] = (c["vp"].float() * 2.0 ** -12).half()
    first = s[0] - n[0] + 2                              # rows 0 and 1 do not see it, row 2 on do
    for pos in (first, s[0] - 1):
        c["vp"][int(c["table"][0, pos // 16]), :, pos % 16, 0] = top
    got = within(c, slice(0, 2))
    seen = got[2:].cpu()
    assert bool(torch.isfinite(seen).all()) == (top < 1e5)


def test_infinite_scales_do_not_wear_out_the_reference():
    """Many tokens with an infinite scale, each in a step of its own, behind the rows that are asked for."""
    c = make(43, [200], [200], 2, 1, 64, 16, "f16")
    base = call(c)
    for pos in range(40, 200, 32):
        c["vp"][int(c["table"][0, pos // 16]), 0, pos % 16, 0] = float("inf")
    got = call(c)
    assert bool(torch.isfinite(got[:40]).all()) and not bool(torch.isfinite(got[40:]).all(-1).any())
    want, _, big = kvo.attention(c["q"][:40], kvo.values4(c["kc"], c["kp"]), kvo.values4(c["vc"], c["vp"]), c["table"],
                                 torch.tensor([40], dtype=torch.int32), 64 ** -0.5, 1, 16, torch.tensor([0, 40], dtype=torch.int32))
    assert ((got[:40].cpu().double() - want).abs() <= kvo.attention_bound(want, big, 64, torch.float16)).all()
    assert bool((base[:40] - got[:40]).abs().max() < 0.1)
