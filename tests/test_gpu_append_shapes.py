"""append_kv_cache / gather_kv_cache where the way the rows are dealt changes: one, four or eight tokens per workgroup, more and
fewer groups of lanes than tokens, whole 16-byte pieces and rows element by element.  Tolerances as in test_gpu_append."""
import pytest
import torch

from test_gpu_append import DEV, call, check, make

pytestmark = pytest.mark.gpu

# lengths of the new rows: 1 .. 512 tokens go one per workgroup, up to 2048 four, more eight
FEW, SOME, MANY = [130, 0, 257, 1], [513, 90, 2, 0, 31], [1500, 3, 700, 50]


@pytest.mark.parametrize("n", [FEW, SOME, MANY], ids=["few", "some", "many"])
@pytest.mark.parametrize("Hq,Hkv,D,bs,cache,dtype,layout,rot,inter", [
    (5, 2, 32, 16, "int4", "f16", None, 32, False), (3, 1, 256, 48, "int4", "bf16", None, 64, True), (1, 3, 64, 64, "int4", "f16", None, 48, False),
    (2, 1, 512, 16, "f16", "f16", "BSH", 512, False), (6, 2, 128, 32, "bf16", "bf16", "BNSD", 24, True), (7, 1, 32, 32, "int8", "f16", "BSH", 16, False),
    (4, 4, 256, 64, "int8", "bf16", "BNSD", 256, True),
])
def test_shapes(n, Hq, Hkv, D, bs, cache, dtype, layout, rot, inter):
    c = make(D + sum(n), n, [3 * i for i in range(len(n))], Hq, Hkv, D, bs, cache, dtype, layout=layout or "BSH", rot=rot, interleaved=inter, extra_rows=5)
    check(c, call(c))


@pytest.mark.parametrize("n", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("Hq,Hkv,D,cache,dtype,rot,inter", [(3, 2, 64, "int4", "f16", 20, False), (3, 2, 64, "int4", "bf16", 12, True),
                                                            (2, 1, 128, "f16", "f16", 30, False), (2, 1, 32, "int8", "f16", 4, True)])
def test_rotations_of_odd_widths(n, Hq, Hkv, D, cache, dtype, rot, inter):
    c = make(rot + sum(n), n, [0] * len(n), Hq, Hkv, D, 32, cache, dtype, rot=rot, interleaved=inter)
    check(c, call(c))


@pytest.mark.parametrize("cache,dtype,inter", [("int4", "f16", False), ("int8", "bf16", True), ("bf16", "bf16", False)])
def test_rows_off_by_one_element(cache, dtype, inter):
    """The same values from rows that start two bytes off are the same bits: the two paths round alike."""
    c = make(77, SOME, [4] * len(SOME), 4, 2, 64, 32, cache, dtype, interleaved=inter, extra_rows=2)
    plain = call(c)
    check(c, plain)
    wide = torch.zeros((c["T"], c["qkv"].shape[1] + 9), dtype=c["dt"], device=DEV)
    wide[:, 1:-8] = c["qkv"].to(DEV)
    off = call(c, qkv=wide[:, 1:-8])
    assert torch.equal(plain[0], off[0])
    for a, b in zip(plain[1] + list(plain[3]), off[1] + list(off[3])):
        assert torch.equal(a, b)


def test_rows_that_are_not_finite():
    """NaN or an infinity in a row: its stored zero is NaN, everything the row stands for with it, and no other row."""
    c = make(5, [600, 40], [0, 9], 2, 2, 128, 16, "int4", "f16", rot=64)
    clean = call(c)
    q0 = c["qkv"].clone()
    k0 = 2 * 128
    c["qkv"][100, k0 + 5] = float("nan")              # K, head 0
    c["qkv"][101, k0 + 2 * 128 + 7] = float("inf")    # V, head 0
    c["qkv"][620, k0 + 128 + 100] = float("-inf")     # K, head 1
    got = call(c)
    c["qkv"] = q0
    for which, t, h in ((0, 100, 0), (1, 101, 0), (0, 620, 1)):
        assert torch.isnan(got[3][which][t, h]).all()
        got[3][which][t, h] = clean[3][which][t, h]
    assert torch.equal(got[3][0], clean[3][0]) and torch.equal(got[3][1], clean[3][1]) and torch.equal(got[0], clean[0])
