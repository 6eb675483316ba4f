"""paged_attention_int4: page lists per kv head with groups that take two or all four waves of a workgroup for their rows.
Helpers and tolerances of test_gpu_int4_attention.py."""
import pytest
import torch

from test_gpu_int4_attention import _lists, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,bs,dtype", [(24, 1, 256, 32, "f16"), (48, 1, 256, 16, "bf16"), (64, 1, 256, 32, "f16"), (34, 2, 256, 64, "bf16"),
                                               (80, 2, 128, 48, "f16"), (96, 2, 64, 16, "bf16"), (33, 1, 32, 16, "f16")])
def test_wide_groups(Hq, Hkv, D, bs, dtype):
    c = make(Hq + D, [1] * 5, [1, 20, 333, 700, 0], Hq, Hkv, D, bs, dtype, decode=True)
    check(c, lists=_lists(c, Hkv, 5))


@pytest.mark.parametrize("G,D", [(24, 256), (48, 256), (40, 128)])
def test_a_long_list_of_a_wide_group_is_shared(G, D):
    c = make(G, [1], [6000], G, 1, D, 16, "f16", decode=True)
    lists = torch.arange(375, dtype=torch.int32).flip(0).repeat(1, 1, 1).contiguous()
    out = check(c, lists=lists)
    assert torch.equal(check(c, lists=lists), out)
